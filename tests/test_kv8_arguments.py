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
