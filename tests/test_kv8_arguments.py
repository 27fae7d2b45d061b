"""The 8-bit cache's calls refuse tensors that would be read past their end, or as other values."""
import pytest
import torch

from blog_amd import qlin
from test_kv8 import EPS


def _calls(how, cache, rows=1, heads=4, start=0x10000, n_rows=None):
    """Both stores, up to the launch: their checks of the arguments come first."""
    kv, d = cache.kv_heads, cache.head_dim
    a, qw, kw = 0x100000, heads * d, kv * d
    return (lambda: qlin.qk_norm_rope_store_kv(how, a, qw, a, kw, a, kw, a, a, a, rows, heads, kv, d, 64, start),
            lambda: qlin.qk_norm_rope_store_kv8(how, cache, a, qw, a, kw, a, kw, a, rows, heads, start, n_rows))


def test_norm_weights_of_a_whole_head():
    table = torch.zeros(64, 32)
    cache = qlin.Kv8Cache.empty(torch, 1, 2, 64, 64, device="cpu")
    w, short = torch.ones(64, dtype=torch.bfloat16), torch.ones(32, dtype=torch.bfloat16)
    for q, k in ((short, w), (w, short), (short, None), (None, short)):
        for call in _calls(qlin.QkRope(q, k, 0, EPS, 0, table, 32), cache):
            with pytest.raises(ValueError):
                call()
    # nothing to do: these are taken
    long = torch.ones(128, dtype=torch.bfloat16)
    for q, k in ((w, w), (None, None), (long, w), (0x10000, 0x10000)):
        for call in _calls(qlin.QkRope(q, k, 0, EPS, 0, table, 32), cache, rows=0):
            call()


def _of_cache(cache):
    """Every call's positions and counts: name, and the call with given ones."""
    how = qlin.QkRope(None, None, 0, EPS, 0, None, 0)
    a, ws = 0x100000, None
    ok = torch.zeros(cache.n_seqs, dtype=torch.int32)
    f32, kv8 = (lambda start, n_rows=None, i=i: _calls(how, cache, rows=0, start=start, n_rows=n_rows)[i]() for i in (0, 1))
    yield "start_pos of the 8-bit store", lambda t: kv8(t)
    yield "n_rows of the 8-bit store", lambda t: kv8(ok, t)
    yield "start_pos of the attention", lambda t: qlin.attend_kv8(cache, a, a, 0, 4, t, None, 1.0, ws)
    yield "n_rows of the attention", lambda t: qlin.attend_kv8(cache, a, a, 0, 4, ok, t, 1.0, ws)
    yield "first of the read back", lambda t: qlin.kv8_read(cache, t, ok, 0, a, a)
    yield "lens of the read back", lambda t: qlin.kv8_read(cache, ok, t, 0, a, a)
    if cache.n_seqs == 1:
        yield "start_pos of the f32 store", lambda t: f32(t)


@pytest.mark.parametrize("n", [1, 3])
def test_positions_and_counts_are_int32(n):
    """(With calls of no rows, which launch nothing.)"""
    cache = qlin.Kv8Cache.empty(torch, n, 2, 64, 64, device="cpu")
    i32 = lambda k: torch.zeros(k, dtype=torch.int32)
    bad = [torch.zeros(n, dtype=d) for d in (torch.int64, torch.float32, torch.int16)] + [i32(n)[:n - 1]]
    if n > 1:
        bad.append(i32(2 * n)[::2])
    for name, call in _of_cache(cache):
        for t in bad:
            with pytest.raises(ValueError):
                call(t)
                pytest.fail(name)
        for t in (i32(n), i32(n + 2), 0x10000):
            call(t)
