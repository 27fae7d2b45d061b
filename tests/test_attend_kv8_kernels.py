"""Each kernel that an attention over the 8-bit cache can be run by, to the last position and the last bits.

Scores are exact here, so that the bound is that of the probabilities alone: each key has one code, of -2, -1, 1 or 2, in one of
four dims; queries are multiples of 2^-19 below 1 there, and the scale is ln 2.  A product and its distance to the maximum are
then f32 values.  Values are +-127 by the key's kind and the dim, so that errors of one kind's probability do not average out.
"""
import numpy as np
import pytest

from blog_amd import qlin
from test_attend_kv8_scores import LN2
from test_kv8 import BLOCK, Cache, HEAD_DIMS, _attend, _device_cache, _gpu, attend, attend_tolerance

# sequences, rows, heads, key heads, blocks of a sequence
SHAPES = [(2, 1, 6, 2, 3), (3, 1, 4, 2, 20), (1, 2, 4, 1, 70), (1, 1, 4, 2, 1100), (26, 1, 8, 8, 9), (1, 9, 8, 2, 3), (2, 9, 8, 2, 20),
          (1, 9, 8, 2, 90), (66, 9, 4, 1, 3), (1, 300, 4, 4, 11)]


def plan(n, rows, heads, kv, d, blocks):
    """Tiles a wave, waves a workgroup, splits, and tiles of the launch (plan_of, qlin_attend_kv8.hip)."""
    pairs = rows * (heads // kv)
    tiles = 2 if pairs > 16 and d <= 128 else 1
    work = -(-pairs // (16 * tiles)) * kv * n
    few = blocks <= 64
    alike = lambda slots: n == 1 and 8 * work >= 7 * slots
    waves = 8 if 4 * work > (2 if tiles == 2 else 3) * 256 and work <= 256 and (few or alike(256)) else 4
    one = waves == 8 or work > 512 or (work > 256 and (few or alike(512)))
    return tiles, waves, min(1 if one else -(-512 // work), (blocks + 8) // 8, 128), work * tiles


def kernels_of(n, rows, heads, kv, d, blocks):
    tiles, waves, splits, _ = plan(n, rows, heads, kv, d, blocks)
    join = "no join" if splits == 1 else "a wave a row" if splits <= 8 else "a workgroup a row"
    return {("attention", d, tiles, waves), ("join", d, join)}


def test_the_restated_plan_is_the_launchs():
    rng = np.random.default_rng(1)
    for _ in range(5000):
        kv = int(rng.choice([1, 2, 3, 4, 8]))
        a = (int(rng.choice([1, 1, 2, 5, 24, 60])), int(rng.choice([1, 1, 2, 5, 20, 100, 600])), kv * int(rng.choice([1, 2, 4, 7])), kv,
             int(rng.choice(HEAD_DIMS)), int(rng.choice([1, 4, 8, 9, 30, 64, 65, 200, 1000, 30000])))
        _, _, splits, tiles = plan(*a)
        assert qlin.attend_kv8_workspace_bytes(*a) == (tiles * splits * 16 * (a[4] + 4) * 4 if splits > 1 else 0), a


def test_every_kernel_is_run():
    every = {("attention", d, t, w) for d in HEAD_DIMS for t in ((1, 2) if d <= 128 else (1,)) for w in (4, 8)}
    every |= {("join", d, j) for d in HEAD_DIMS for j in ("no join", "a wave a row", "a workgroup a row")}
    run = set().union(*(kernels_of(n, rows, heads, kv, d, blocks) for n, rows, heads, kv, blocks in SHAPES for d in HEAD_DIMS))
    assert run == every


def _case(n, rows, heads, kv, blocks, d):
    """The cache, queries, and starts: the first sequence fills its blocks, the last ends in its first one."""
    rng = np.random.default_rng(n * rows + blocks + d)
    ref = Cache(n, blocks, kv, d, rng.permutation(n * blocks + 2)[:n * blocks].reshape(n, blocks), n * blocks + 2)
    codes, signs = np.array([-2, -1, 1, 2]), rng.choice([-1, 1], (16, d))

    def fill(keys, values, one):
        dim, code = rng.integers(0, 4, keys.shape[:-1]), rng.integers(0, 4, keys.shape[:-1])
        keys[:] = 0
        np.put_along_axis(keys, dim[..., None], codes[code][..., None].astype(keys.dtype), -1)
        values[:] = signs[4 * dim + code] * one
    fill(ref.kc, ref.vc, 127)
    ring = np.empty((n, kv, 2, 64, d), np.float32)
    fill(ring[:, :, 0], ring[:, :, 1], 127 / 128)
    ref.ring = ring
    ref.scales[:, :, 0], ref.scales[:, :, 1] = 1.0, 2.0 ** -7
    q = np.zeros((n, rows, heads, d), np.float32)
    q[..., :4] = rng.integers(-2 ** 19 + 1, 2 ** 19, q.shape[:-1] + (4,)) * 2.0 ** -19
    starts = [int(x) for x in rng.integers(0, blocks * BLOCK - rows + 1, n)]
    starts[-1], starts[0] = 5, blocks * BLOCK - rows
    return ref, q, starts


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("d", HEAD_DIMS)
def test_attend_by_every_kernel(shape, d):
    torch = _gpu()
    from gpu_util import banner
    n, rows, heads, kv, blocks = shape
    ref, q, starts = _case(n, rows, heads, kv, blocks, d)
    banner(f"attend n={n} rows={rows} heads={heads}/{kv} blocks={blocks} d={d}: {kernels_of(n, rows, heads, kv, d, blocks)}")
    got = _attend(torch, ref, _device_cache(torch, ref, paged=True), q, starts, None, heads, LN2)
    for s in range(n):
        k, v, there = ref.values(s, starts[s] + rows)
        want, _ = attend(q[s].astype(np.float64), k, v, there, starts[s], LN2)
        assert np.abs(got[s] - want).max() <= attend_tolerance(0.0, v), s


def _bits(x, n):
    """x rounded to n significant bits."""
    m, e = np.frexp(x)
    return np.ldexp(np.rint(np.ldexp(m, n)), e - n)


@pytest.mark.parametrize("shape", SHAPES[:9], ids=str)
@pytest.mark.parametrize("d", [64, 256])
def test_the_bound_sees_what_is_lost(shape, d):
    """Planted in the oracle: queries or probabilities without their low halves (11 bits of 22), and a position that is left
    out (of the middle weight of those that the first sequence's last row sees)."""
    n, rows, heads, kv, blocks = shape
    ref, q, starts = _case(n, rows, heads, kv, blocks, d)
    k, v, there = ref.values(0, starts[0] + rows)
    q, last = q[0].astype(np.float64), starts[0] + rows - 1
    want, _ = attend(q, k, v, there, starts[0], LN2)
    bound = attend_tolerance(0.0, v)
    assert np.abs(attend(_bits(q, 11), k, v, there, starts[0], LN2)[0] - want).max() > 2 * bound
    short, less = 0.0, 0.0
    for h in range(heads):
        g = h // (heads // kv)
        e = np.exp(k[:, g] @ q[-1, h] * LN2)
        o = e @ v[:, g] / e.sum()
        assert np.abs(o - want[-1, h]).max() < 1e-12
        short = max(short, np.abs(_bits(e, 11) @ v[:, g] / _bits(e, 11).sum() - o).max())
        j = np.argsort(e)[len(e) // 2]
        f = np.where(np.arange(last + 1) == j, 0.0, e)
        less = max(less, np.abs(f @ v[:, g] / f.sum() - o).max())
    assert short > 2 * bound and less > 2 * bound, (short, less, bound)
