"""Rows of a call past the f32 caches' ends: each position has the row whose own it is, and where there is none the nearest one; the
other rows are stored nowhere."""
import numpy as np
import pytest

from blog_amd import qlin
from test_kv8 import EPS, norm_rope, table64

pytestmark = pytest.mark.gpu


def _kept(start, rows, end):
    """position -> the row that it holds"""
    kept = {}
    for r in sorted(range(rows), key=lambda r: abs(start + r - min(max(start + r, 0), end - 1)), reverse=True):
        kept[min(max(start + r, 0), end - 1)] = r
    return kept


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("rows,start", [(5, 37), (5, 39), (7, 40), (3, 100), (33, 20), (5, -2), (3, -9), (60, -7), (4, 2 ** 31 - 1), (4, -2 ** 31)])
def test_rows_past_the_ends(normed, rows, start):
    import torch
    from gpu_util import banner, bind_stream, dev, empty_f32, host
    bind_stream()
    heads, kv, d, end, theta = 4, 2, 64, 40, 1e4
    banner(f"rows past the ends: normed={normed} rows={rows} start={start}")
    rng = np.random.default_rng(rows)
    q, k, v = (rng.standard_normal((rows, n * d)).astype(np.float32) for n in (heads, kv, kv))
    kc, vc = empty_f32(end, kv, d), empty_f32(end, kv, d)
    pos = torch.tensor([start], dtype=torch.int32, device="cuda")
    table = table64(end, d, theta).astype(np.float32)
    qd = dev(q)
    if normed:
        qlin.qk_norm_rope_store_kv(qlin.QkRope(None, None, 0, EPS, 0, dev(table), d), qd, heads * d, dev(k), kv * d, dev(v), kv * d, qd, kc, vc,
                                   rows, heads, kv, d, end, pos)
    else:
        qlin.call("qlin_launch_rope_store_kv", qd, dev(k), dev(v), kc, vc, rows, heads, kv, d, end, pos, theta)
    kept, at = _kept(start, rows, end), np.clip(start + np.arange(rows, dtype=np.int64), 0, end - 1)
    turned = norm_rope(k.reshape(rows, kv, d).astype(np.float64), None, table, at, d, 0)
    # An f32 angle of up to 39 from a frequency that is off by two steps of f32 at most, 39 * 2^-22, its cosine and sine by as much,
    # and a sum of two products: below 2^-15 of the head's largest value.
    bound = 2.0 ** -15
    got_k, got_v = host(kc), host(vc)
    for p in range(end):
        if p in kept:
            assert np.array_equal(got_v[p].reshape(-1), v[kept[p]]), p
            assert np.abs(got_k[p] - turned[kept[p]]).max() <= bound * np.abs(turned[kept[p]]).max(), p
        else:
            assert np.isnan(got_k[p]).all() and np.isnan(got_v[p]).all(), p
    q_turned = norm_rope(q.reshape(rows, heads, d).astype(np.float64), None, table, at, d, 0)
    assert np.abs(host(qd).reshape(rows, heads, d) - q_turned).max() <= bound * np.abs(q_turned).max()
