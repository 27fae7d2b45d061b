"""Routing by scores (qlin_launch_moe_route) against the formula in 64 bits.

Scores are rounded to f32 once; a pick's weight is a quotient of such scores in 64 bits, rounded once, where a score next to the
middle between two f32 values may have gone to either (a step of 2^-23 of it): weights within 2^-22 of theirs."""
import ctypes as C

import numpy as np
import pytest

from blog_amd import qlin

OK, UNSUP, SHAPE, NULL, ROWB, LIMIT, LAUNCH, ALIGN = range(8)
FAKE = 0x10000


def reference(logits, k, sigmoid=False, bias=None, n_groups=1, top_groups=1, group_pairs=False, renormalise=False, scaling=1.0):
    tokens, ne = logits.shape
    ids, weights = np.full((tokens, k), -1, np.int32), np.zeros((tokens, k))
    for t in range(tokens):
        l = logits[t].astype(np.float64)
        fine = np.isfinite(l)
        s = np.zeros(ne)
        if fine.any():
            with np.errstate(over="ignore"):
                s[fine] = 1 / (1 + np.exp(-l[fine])) if sigmoid else np.exp(l[fine] - l[fine].max())
            if not sigmoid:
                s /= s.sum()
        s = s.astype(np.float32)
        c = s + bias if bias is not None else s.copy()
        c[~fine | ~(c > -np.inf)] = -np.inf
        size = ne // n_groups
        if n_groups > 1:
            of = np.sort(c.reshape(n_groups, size), 1)[:, ::-1]
            score = of[:, 0].copy()
            if group_pairs and size > 1:
                score = np.where(of[:, 1] > -np.inf, of[:, 0] + of[:, 1], score)
            best = sorted(range(n_groups), key=lambda g: (-score[g], g))[:top_groups]
            c[~np.isin(np.arange(ne) // size, best)] = -np.inf
        order = [e for e in sorted(range(ne), key=lambda e: (-c[e], e)) if c[e] > -np.inf][:k]
        ids[t, :len(order)] = order
        w = s[order].astype(np.float64)
        if renormalise:
            w = w / (w.sum() + 1e-20)
        weights[t, :len(order)] = w * np.float64(np.float32(scaling))
    return ids, weights


def test_reference_by_hand():
    l = np.log(np.array([[0.1, 0.4, 0.2, 0.3]], np.float32))
    ids, w = reference(l, 2)
    assert ids.tolist() == [[1, 3]] and np.allclose(w, [[0.4, 0.3]])
    ids, w = reference(l, 1, n_groups=2, top_groups=1, group_pairs=True, renormalise=True, scaling=3.0)  # 0.5 each: the first group
    assert ids.tolist() in ([[1]], [[3]]) and np.allclose(w, [[3.0]])
    ids, _ = reference(l, 3, bias=np.array([0, -np.inf, 1, 0], np.float32))
    assert ids.tolist() == [[2, 3, 0]]


def test_validation():
    def run(null=False, logits=FAKE, stride=64, ids=FAKE, w=FAKE, tokens=2, ne=64, k=4, **kw):
        a = dict(bias=FAKE, sigmoid=0, n_groups=8, top_groups=4, group_pairs=0, renormalise=0, scaling=1.0)
        a.update(kw)
        c = qlin.MoeRoutingArgs(*a.values())
        return qlin.status("qlin_launch_moe_route", None if null else C.addressof(c), logits, stride, ids, w, tokens, ne, k)
    assert run(null=True) == NULL and run(logits=0) == NULL and run(ids=0) == NULL and run(w=0) == NULL
    assert run(tokens=-1) == SHAPE and run(ne=0) == SHAPE and run(k=-1) == SHAPE and run(n_groups=0) == SHAPE and run(top_groups=0) == SHAPE
    assert run(stride=63) == SHAPE and run(n_groups=7) == SHAPE and run(top_groups=9) == SHAPE and run(k=33) == SHAPE
    assert run(ne=1025, stride=1025, n_groups=1, top_groups=1) == LIMIT and run(ne=130, stride=130, n_groups=65) == LIMIT
    assert run(ne=128, stride=128, n_groups=1, top_groups=1, k=65) == LIMIT
    for kw in (dict(logits=FAKE + 2), dict(ids=FAKE + 1), dict(w=FAKE + 2), dict(bias=FAKE + 2)):
        assert run(**kw) == ALIGN
    assert run(tokens=0, logits=0) == OK and run(k=0, logits=0) == OK


def test_python_refusals():
    import torch
    with pytest.raises(ValueError):
        qlin.moe_route(qlin.MoeRouting(), torch.zeros(2, 8), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2))
    with pytest.raises(ValueError):
        qlin.MoeRouting(bias=torch.zeros(8, dtype=torch.float64))


# ---- GPU ---------------------------------------------------------------------------------------

def _gpu():
    import torch
    from gpu_util import bind_stream
    assert torch.cuda.is_available(), "GPU tests need the MI355X"
    bind_stream()
    return torch


def _check(torch, logits, k, bias=None, pad=0, **kw):
    from gpu_util import dev, host
    tokens, ne = logits.shape
    wide = np.full((tokens, ne + pad), 99.0, np.float32)  # (what stands beside the experts would win)
    wide[:, :ne] = logits
    ids = torch.full((tokens + 1, k), -7, dtype=torch.int32, device="cuda")
    w = torch.full((tokens + 1, k), 7.0, device="cuda")
    how = qlin.MoeRouting(bias=None if bias is None else dev(bias), **kw)
    qlin.moe_route(how, dev(wide)[:, :ne], ids, w)
    got, gw = host(ids), host(w)
    assert (got[tokens] == -7).all() and (gw[tokens] == 7.0).all()
    want, ww = reference(logits, k, bias=bias, **kw)
    assert np.array_equal(got[:tokens], want)
    assert (np.abs(gw[:tokens] - ww) <= 2.0 ** -22 * np.abs(ww) + 2.0 ** -149).all()


@pytest.mark.gpu
@pytest.mark.parametrize("ne,n_groups", [(1, 1), (2, 1), (6, 3), (8, 8), (60, 1), (64, 8), (65, 1), (96, 12), (128, 64), (160, 8), (256, 8), (257, 1),
                                         (320, 16), (500, 10), (512, 1), (1000, 50), (1024, 64), (1024, 1)])
def test_routes(ne, n_groups):
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(ne)
    for tokens, k, top in ((1, 1, 1), (5, 6, (n_groups + 1) // 2), (37, 64, n_groups)):
        k = min(k, ne // n_groups * top)
        logits = (2 * rng.standard_normal((tokens, ne))).astype(np.float32)
        bias = (0.2 * rng.standard_normal(ne)).astype(np.float32)
        for sigmoid in (False, True):
            for pairs, renormalise, b in ((False, False, None), (True, True, bias)):
                banner(f"moe_route experts={ne} groups={n_groups} kept={top} k={k} tokens={tokens} sigmoid={sigmoid} pairs={pairs}")
                _check(torch, logits, k, bias=b, pad=tokens % 3, sigmoid=sigmoid, n_groups=n_groups, top_groups=top, group_pairs=pairs,
                       renormalise=renormalise, scaling=2.5)


@pytest.mark.gpu
def test_odd_values():
    """Ties (the lowest index, experts and groups), saturated scores, logits that are not finite, experts that are switched
    off, fewer experts than picks."""
    torch = _gpu()
    from gpu_util import banner
    banner("moe_route odd values")
    rng = np.random.default_rng(4)
    ne = 32
    x = rng.integers(-2, 3, (12, ne)).astype(np.float32)
    x[1] = 0.5
    x[2] = 1e4
    x[3] = -1e4
    x[4, 5], x[4, 9], x[4, 11] = np.inf, -np.inf, np.nan
    x[5] = np.nan
    x[6] = -np.inf
    x[6, 30] = 1.0
    x[7] = 3e38
    x[8] = -3e38
    x[9, ::2] = np.nan
    x[10, :16] = -np.inf
    bias = (0.1 * rng.standard_normal(ne)).astype(np.float32)
    off = bias.copy()
    off[[0, 7, 8, 9]] = -np.inf
    off[20] = np.nan
    off[3] = np.inf
    for sigmoid in (False, True):
        for b in (None, bias, off):
            for renormalise in (False, True):
                kw = dict(bias=b, sigmoid=sigmoid, renormalise=renormalise)
                _check(torch, x, 6, **kw)
                _check(torch, x, 32, **kw)
                _check(torch, x, 6, n_groups=8, top_groups=3, group_pairs=True, **kw)
                _check(torch, x, 6, n_groups=8, top_groups=2, **kw)
                _check(torch, x, 3, n_groups=32, top_groups=3, group_pairs=True, **kw)


@pytest.mark.gpu
def test_as_the_softmax_router():
    """Without bias, groups and renormalisation: qlin_launch_moe_router_topk's picks, and its weights to f32's accuracy (its
    exponentials and its sum of n_experts terms are in f32: n_experts + 8 half steps)."""
    torch = _gpu()
    from gpu_util import banner, dev, host
    banner("moe_route and moe_router_topk")
    rng = np.random.default_rng(5)
    for ne in (16, 64, 200):
        x = dev(rng.standard_normal((50, ne)).astype(np.float32))
        a, b = (torch.zeros(50, 6, dtype=torch.int32, device="cuda") for _ in range(2))
        u, v = (torch.zeros(50, 6, device="cuda") for _ in range(2))
        qlin.moe_route(qlin.MoeRouting(scaling=1.5), x, a, u)
        qlin.call("qlin_launch_moe_router_topk", x, b, v, 50, ne, 6, 1.5)
        assert np.array_equal(host(a), host(b))
        assert (np.abs(host(u) - host(v)) <= (ne + 8) * 2.0 ** -24 * host(u)).all()
