"""Attention over the 8-bit cache where scores are far from zero.

A softmax of finite scores is finite, whatever their size.  Queries and keys are powers of two times small integers here
and the scale is ln 2, so that every score (in units of log 2) is an integer that f32 holds exactly, next to which the
probabilities' own roundings are all there is."""
import numpy as np
import pytest

from test_kv8 import BLOCK, RING, _attend, _device_cache, _filled, _gpu, attend, attend_tolerance

LN2 = float(np.float32(np.log(2.0)))


def _far_cache(rng, per, kv, d, code):
    """Keys code in dim 0, -1, 0 or 1 in dim 1; complete blocks and the ring alike."""
    ref = _filled(rng, 1, per, kv, d)
    ref.kc[:] = 0
    ref.kc[..., 0] = code
    ref.kc[..., 1] = rng.integers(-1, 2, ref.kc.shape[:-1])
    ref.scales[:, :, 0] = 1.0
    ref.ring[:, :, 0] = 0
    ref.ring[:, :, 0, :, 0] = code
    ref.ring[:, :, 0, :, 1] = rng.integers(-1, 2, (1, kv, RING))
    return ref


@pytest.mark.parametrize("e,step", [(10, 1), (13, 4), (17, 4), (18, 4), (20, 16), (21, 32), (26, 1024)])
@pytest.mark.parametrize("code", [127, -127])
def test_the_scores_are_exact(e, step, code):
    """Each product and each sum of them is an f32 value, and neighbours are at least f32's spacing there apart."""
    values = np.float32(code * 2.0 ** e) + np.float32(step) * np.arange(-1, 2, dtype=np.float32)
    assert np.array_equal(values.astype(np.float64), code * 2.0 ** e + step * np.arange(-1.0, 2.0))
    # q_scale, as the launch computes it, is 1
    assert np.float32(LN2 * 1.4426950408889634) == 1.0


@pytest.mark.gpu
@pytest.mark.parametrize("d,heads,kv,rows,start", [(64, 4, 2, 1, 200), (128, 8, 2, 40, 90), (96, 3, 1, 17, 150), (192, 2, 2, 5, 100),
                                                   (256, 2, 1, 9, 60), (128, 4, 2, 1, 5000)])
@pytest.mark.parametrize("code", [127, -127])
def test_attend_scores_far_from_zero(d, heads, kv, rows, start, code):
    """Maxima from 2^17 to 2^33, of either sign: complete blocks, the open one, waves and splits that are joined."""
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(d + start)
    ref = _far_cache(rng, (start + rows) // BLOCK + 1, kv, d, code)
    cache = _device_cache(torch, ref, paged=False)
    for e, step in ((10, 1), (13, 4), (17, 4), (18, 4), (20, 16), (21, 32), (26, 1024)):
        banner(f"attend scores of {code} * 2^{e}, steps of {step}, d={d} rows={rows} start={start}")
        q = np.zeros((1, rows, heads, d), np.float32)
        q[..., 0] = 2.0 ** e
        q[..., 1] = step * rng.choice([-1.0, 1.0], (rows, heads))
        got = _attend(torch, ref, cache, q, [start], None, heads, LN2)
        k, v, there = ref.values(0, start + rows)
        want, _ = attend(q[0].astype(np.float64), k, v, there, start, LN2)
        assert np.isfinite(got).all()
        # scores without an error of their own
        assert np.abs(got[0] - want).max() <= attend_tolerance(0.0, v)


@pytest.mark.gpu
def test_attend_maxima_that_grow_from_near_to_far():
    """Each block's scores above the ones before, from 1 to 2^31: what came before no longer counts."""
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(5)
    kv, d, heads, per = 1, 64, 2, 33
    ref = _far_cache(rng, per, kv, d, 1)
    for b in range(per):
        ref.scales[b, :, 0] = 2.0 ** b
    cache = _device_cache(torch, ref, paged=False)
    for sign in (1.0, -1.0):
        q = np.zeros((1, 40, heads, d), np.float32)
        q[..., 0] = sign
        q[..., 1] = 2.0 ** -3
        for start in (0, 500, 960, 1000):
            banner(f"growing maxima, sign {sign}, start {start}")
            got = _attend(torch, ref, cache, q, [start], None, heads, LN2)
            k, v, there = ref.values(0, start + 40)
            want, _ = attend(q[0].astype(np.float64), k, v, there, start, LN2)
            assert np.isfinite(got).all()
            # all scores are multiples of an eighth of their block's power of two: exact too
            assert np.abs(got[0] - want).max() <= attend_tolerance(0.0, v)
