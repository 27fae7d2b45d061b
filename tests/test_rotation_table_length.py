"""Rotation tables of fewer positions than the cache: what the table has is as with a whole one, and what it does not have is
not a number, in the queries, in either cache and in the attention of the rows that see it."""
import numpy as np
import pytest

from blog_amd import qlin
from test_kv8 import EPS, _gpu, table64

pytestmark = pytest.mark.gpu


def _inputs(torch, rows, heads, kv, d, n=1):
    from gpu_util import dev
    rng = np.random.default_rng(rows + d)
    return dev(rng.standard_normal((n, rows, heads + 2 * kv, d)).astype(np.float32))


@pytest.mark.parametrize("d,rd,pairing", [(64, 64, 0), (128, 64, 1), (40, 40, 0)])
def test_f32_cache(d, rd, pairing):
    torch = _gpu()
    from gpu_util import banner, dev, empty_f32, host
    heads, kv, rows, start, ms, have = 4, 2, 20, 50, 80, 63
    table = dev(table64(ms, rd, 1e4).astype(np.float32))
    x = _inputs(torch, rows, heads, kv, d)
    a, width, got = x.data_ptr(), (heads + 2 * kv) * d, []
    banner(f"table of {have} positions, f32 cache d={d} rd={rd}")
    for t in (table, table[:have].contiguous()):
        q, kc, vc = empty_f32(rows, heads, d), empty_f32(ms, kv, d), empty_f32(ms, kv, d)
        qlin.qk_norm_rope_store_kv(qlin.QkRope(None, None, 0, EPS, 0, t, rd, pairing), a, width, a + 4 * heads * d, width,
                                   a + 4 * (heads + kv) * d, width, q, kc, vc, rows, heads, kv, d, ms,
                                   torch.tensor([start], dtype=torch.int32, device="cuda"))
        got.append((host(q), host(kc)[start:start + rows], host(vc)[start:start + rows]))
    (q, k, v), (qs, ks, vs) = got
    n = have - start
    assert np.array_equal(vs, v)
    for whole, part in ((q, qs), (k, ks)):
        assert np.array_equal(part[:n], whole[:n]) and np.isfinite(whole).all()
        assert np.isnan(part[n:, :, :rd]).all() and np.array_equal(part[n:, :, rd:], whole[n:, :, rd:])


@pytest.mark.parametrize("d,rd,pairing", [(64, 64, 0), (256, 64, 1)])
def test_8_bit_cache(d, rd, pairing):
    torch = _gpu()
    from gpu_util import banner, dev, empty_f32, host
    heads, kv, cap, have = 4, 2, 128, 100
    table = dev(table64(cap, rd, 1e4).astype(np.float32))
    x = _inputs(torch, 110, heads, kv, d)
    a, width, got = x.data_ptr(), (heads + 2 * kv) * d, []
    banner(f"table of {have} positions, 8-bit cache d={d} rd={rd}")
    for t in (table, table[:have].contiguous()):
        how = qlin.QkRope(None, None, 0, EPS, 0, t, rd, pairing)
        cache = qlin.Kv8Cache.empty(torch, 1, kv, d, cap)
        q, out = empty_f32(1, 110, heads, d), empty_f32(1, 110, heads, d)
        zero = torch.zeros(1, dtype=torch.int32, device="cuda")
        qlin.qk_norm_rope_store_kv8(how, cache, a, width, a + 4 * heads * d, width, a + 4 * (heads + kv) * d, width, q, 110, heads, zero)
        q_ok = torch.nan_to_num(q)
        need = qlin.attend_kv8_workspace_bytes(1, 110, heads, kv, d, cache.blocks_per_seq)
        qlin.attend_kv8(cache, q_ok, out, 110, heads, zero, None, d ** -0.5, torch.empty(max(need, 16), dtype=torch.uint8, device="cuda"))
        got.append((host(q), host(cache.pages), host(cache.recent), host(out)))
    (q, pages, ring, out), (qs, pages_s, ring_s, out_s) = got
    assert np.array_equal(qs[:, :have], q[:, :have]) and np.isnan(qs[:, have:, :, :rd]).all()
    assert np.array_equal(qs[:, have:, :, rd:], q[:, have:, :, rd:])
    assert np.array_equal(pages_s, pages)  # three complete blocks, 0 .. 95
    for p in range(96, 110):
        k, ks = ring[0, :, 0, p % 64], ring_s[0, :, 0, p % 64]
        assert np.array_equal(ks[:, rd:], k[:, rd:]) and (np.array_equal(ks, k) if p < have else np.isnan(ks[:, :rd]).all())
    assert np.isfinite(out).all() and np.array_equal(out_s[:, :have], out[:, :have]) and np.isnan(out_s[:, have:]).all()


def test_positions_outside_the_cache_are_the_nearest_in_it():
    """With a table of the cache's positions nothing is missing, however far a start lies outside."""
    torch = _gpu()
    from gpu_util import banner, dev, empty_f32, host
    heads, kv, d = 2, 1, 64
    table = table64(64, d, 1e4).astype(np.float32)
    x = _inputs(torch, 3, heads, kv, d)
    a, width = x.data_ptr(), (heads + 2 * kv) * d
    how = qlin.QkRope(None, None, 0, EPS, 0, dev(table), d)
    for start in (62, 64, 1000, 2 ** 31 - 1, -2, -2 ** 31):
        banner(f"start {start}")
        cache = qlin.Kv8Cache.empty(torch, 1, kv, d, 64)
        q = empty_f32(1, 3, heads, d)
        qlin.qk_norm_rope_store_kv8(how, cache, a, width, a + 4 * heads * d, width, a + 4 * (heads + kv) * d, width, q, 3, heads,
                                    torch.tensor([start], dtype=torch.int32, device="cuda"))
        assert np.isfinite(host(q)).all() and np.isfinite(host(cache.recent)).all()
