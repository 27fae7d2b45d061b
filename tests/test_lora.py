"""Low-rank adapters of many requests beside a shared projection (qlin_launch_lora_add) against the formula in 64 bits.

Accuracy: products are exact, sums in f32.  A sum of n terms t in f32, added one after the other, is off by n roundings of half a
step of a partial sum, which for terms of random signs is about sqrt(k) |t|; together 2^-24 sqrt(sum k) rms(t) = 2^-24 n rms(t) /
sqrt 2, or 2^-24 sqrt(n / 2) |t|_2.  Blocks that are added up apart are off by less.  A value of y has the errors of A x (in
units of its terms' norm, through B) and its own sum's; four times that, and half a step of y and of scale z, is what a value may be
off by; the root of the mean square error of an output is held to once that.  With small whole numbers everything is exact and
has to be equal."""
import ctypes as C

import numpy as np
import pytest

from blog_amd import qlin

OK, UNSUP, SHAPE, NULL, ROWB, LIMIT, LAUNCH, ALIGN = range(8)
FAKE = 0x10000
STEP = 2.0 ** -24


def test_validation():
    def run(null=False, n=1, t=0, slots=4, rank=8, n_in=64, ranks=FAKE, scales=FAKE, x=FAKE, xs=64, ids=FAKE, rows=2, ws=FAKE, nws=1 << 30, **kw):
        m = dict(a=FAKE, b=FAKE, base=FAKE, y=FAKE * 2, base_stride=32, y_stride=32, out_dim=32)
        m.update(kw)
        s = (qlin.LoraArgs * 2)(qlin.LoraArgs(*m.values()), qlin.LoraArgs(*m.values()))
        return qlin.status("qlin_launch_lora_add", None if null else C.addressof(s), n, t, slots, rank, n_in, ranks, scales, x, xs, ids, rows, ws, nws)
    assert run(t=3) == UNSUP and run(t=-1) == UNSUP
    assert run(n=-1) == SHAPE and run(slots=-1) == SHAPE and run(rank=-8) == SHAPE and run(n_in=-8) == SHAPE and run(rows=-1) == SHAPE
    assert run(rank=12) == SHAPE and run(n_in=60) == SHAPE and run(xs=63) == SHAPE and run(out_dim=-1) == SHAPE
    assert run(base_stride=31) == SHAPE and run(y_stride=31) == SHAPE and run(y=FAKE, y_stride=40) == SHAPE
    assert run(n=5) == LIMIT and run(rank=264) == LIMIT and run(slots=1025) == LIMIT and run(rows=65537) == LIMIT
    assert run(null=True) == NULL and run(ids=0) == NULL and run(x=0) == NULL and run(ws=0) == NULL
    for name in ("a", "b", "base", "y"):
        assert run(**{name: 0}) == NULL, name
    for name in ("a", "b"):
        assert run(**{name: FAKE + 8}) == ALIGN, name
    for name in ("base", "y", "x", "ids", "ranks", "scales"):
        assert run(**{name: FAKE + 2}) == ALIGN, name
    assert run(ws=FAKE + 8) == ALIGN
    need = qlin.lora_workspace_bytes(2, 1, 4, 8, 64)
    assert need > 0 and run(nws=need - 1) == LIMIT
    assert run(n=0, null=True) == OK and run(rows=0, x=0) == OK and run(out_dim=0, base=0, y=0) == OK
    for bad in ((0, 1, 4, 8, 64), (2, 0, 4, 8, 64), (2, 1, 0, 8, 64), (2, 1, 4, 0, 64), (2, 1, 4, 8, 0)):
        assert qlin.lora_workspace_bytes(*bad) == 0


def test_python_refusals():
    import torch
    bf = torch.bfloat16
    with pytest.raises(ValueError):
        qlin.Lora(torch.zeros(2, 8, 64, dtype=bf), torch.zeros(2, 32, 8))  # types
    with pytest.raises(ValueError):
        qlin.Lora(torch.zeros(2, 8, 64, dtype=bf), torch.zeros(3, 32, 8, dtype=bf))  # slots
    with pytest.raises(ValueError):
        qlin.Lora(torch.zeros(2, 8, 64, dtype=bf), torch.zeros(2, 32, 16, dtype=bf))  # ranks
    with pytest.raises(ValueError):
        qlin.Lora(torch.zeros(2, 8, 64, dtype=torch.float64), torch.zeros(2, 32, 8, dtype=torch.float64))
    with pytest.raises(ValueError):
        qlin.Lora(torch.zeros(2, 64, 8, dtype=bf).transpose(1, 2), torch.zeros(2, 32, 8, dtype=bf))
    w = qlin.Lora(torch.zeros(2, 8, 64), torch.zeros(2, 32, 8))
    x, y, ids = torch.zeros(3, 64), torch.zeros(3, 32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError):  # not on a GPU
        qlin.lora_add(x, ids, [(w, y, y)])


# ---- GPU ---------------------------------------------------------------------------------------

def _gpu():
    import torch
    from gpu_util import bind_stream
    assert torch.cuda.is_available(), "GPU tests need the MI355X"
    bind_stream()
    return torch


TYPES = ["bfloat16", "float16", "float32"]


def _case(torch, seed, rows, n_in, outs, slots, rank, kind, ids=None, whole=False):
    gen = torch.Generator().manual_seed(seed)
    t = getattr(torch, TYPES[kind])
    if whole:
        # |A| <= 1 with few entries, x of 20 bits, |B| <= 1: every sum below 2^24 (x's sums of 8 terms at most, the rest in B's)
        x = torch.randint(-2 ** 17, 2 ** 17, (rows, n_in), generator=gen).float()
        mats = []
        for out in outs:
            a = torch.zeros(slots, rank, n_in)
            a.scatter_(2, torch.randint(0, n_in, (slots, rank, 8), generator=gen), torch.randint(-1, 2, (slots, rank, 8), generator=gen).float())
            b = torch.zeros(slots, out, rank)
            b.scatter_(2, torch.randint(0, rank, (slots, out, 4), generator=gen), torch.randint(-1, 2, (slots, out, 4), generator=gen).float())
            mats.append((a.to(t), b.to(t), torch.randint(-2 ** 20, 2 ** 20, (rows, out), generator=gen).float()))
    else:
        x = torch.randn(rows, n_in, generator=gen)
        mats = [((torch.randn(slots, rank, n_in, generator=gen) * n_in ** -0.5).to(t), (torch.randn(slots, out, rank, generator=gen)).to(t),
                 torch.randn(rows, out, generator=gen)) for out in outs]
    if ids is None:
        ids = torch.randint(-1, slots + 1, (rows,), generator=gen)  # (slots itself: no adapter)
    ranks = torch.tensor([[rank, max(1, rank - 3), rank // 2, 0, rank + 5, 1][i % 6] for i in range(slots)])
    scales = torch.tensor([[1.0, 2.0, -1.0, 0.5][i % 4] for i in range(slots)]) if whole else 0.5 + torch.rand(slots, generator=gen)
    return dict(x=x, mats=mats, ids=ids.int(), ranks=ranks.int(), scales=scales.float(), whole=whole)


def _check(torch, c, *, in_place=False, wide=0, ranks=True, scales=True, spoil=True):
    """Runs a case and holds it to the formula; what a slot has beyond its adapter's rank is NaN."""
    from gpu_util import host
    rows, n_in = c["x"].shape
    slots, rank = c["mats"][0][0].shape[:2]
    use = c["ranks"].clamp(0, rank).tolist() if ranks else [rank] * slots

    def padded(t, left):
        out = torch.full((t.shape[0], t.shape[1] + 2 * wide), 7.0)
        out[:, left:left + t.shape[1]] = t
        return out.cuda()
    x = padded(c["x"], wide)[:, wide:wide + n_in]
    loras, args, keep = [], [], []
    for a, b, base in c["mats"]:
        a, b = a.clone(), b.clone()
        if spoil and ranks:
            for s in range(slots):
                a[s, use[s]:] = float("nan")
                b[s, :, use[s]:] = float("nan")
        loras.append(qlin.Lora(a.cuda(), b.cuda()))
        out = base.shape[1]
        was = padded(base, wide)
        y = was if in_place else torch.full((rows + 1, out + wide), 7.0, device="cuda")
        at = y[:, wide:wide + out] if in_place else y[:rows, :out]
        keep.append((was, y, at))
        args.append((loras[-1], at if in_place else was[:, wide:wide + out], at))
    need = qlin.lora_workspace_bytes(rows, len(args), slots, rank, n_in)
    ws = torch.full((need + 16,), 0xFF, dtype=torch.uint8, device="cuda")  # (NaN)
    qlin.lora_add(x, c["ids"].cuda(), args, ranks=c["ranks"].cuda() if ranks else None, scales=c["scales"].cuda() if scales else None,
                  workspace=ws[:need])
    torch.cuda.synchronize()
    assert (ws[need:] == 0xFF).all()
    x64, ids = c["x"].double().numpy(), c["ids"].numpy()
    for (a, b, base), (was, y, at) in zip(c["mats"], keep):
        out = base.shape[1]
        if in_place:
            assert (y[:, :wide] == 7).all() and (y[:, wide + out:] == 7).all()
        else:
            assert (y[rows:] == 7).all() and (y[:, out:] == 7).all() and torch.equal(was[:, wide:wide + out].cpu(), base)
        got, want = host(at.contiguous()), base.double().numpy().copy()
        tol, mean = np.zeros_like(want), np.zeros_like(want)
        for s in range(slots):
            r, k = np.flatnonzero(ids == s), use[s]
            if not len(r) or not k:
                continue
            a64, b64 = a[s, :k].double().numpy(), b[s, :, :k].double().numpy()
            scale = float(c["scales"][s]) if scales else 1.0
            z = scale * (x64[r] @ a64.T)
            want[r] += z @ b64.T
            # of z: its terms' norm, times sqrt(n / 2) and half a step; through B; then B's own sum's terms' norm
            zn = abs(scale) * np.sqrt((x64[r] ** 2) @ (a64.T ** 2)) * np.sqrt(n_in / 2) + np.abs(z)
            mean[r] = STEP * (np.sqrt((zn ** 2) @ (b64.T ** 2)) + np.sqrt((z ** 2) @ (b64.T ** 2)) * np.sqrt(k / 2))
            tol[r] = 4 * mean[r]
        none = (ids < 0) | (ids >= slots)
        assert np.array_equal(got[none], base.numpy()[none])
        if c["whole"]:
            assert np.array_equal(got, want.astype(np.float32))
            continue
        mean += STEP * np.abs(want)
        tol += STEP * np.abs(want)
        err = np.abs(got - want)
        assert (err <= tol).all(), float((err / np.maximum(tol, 1e-300)).max())
        assert np.sqrt((err ** 2).mean()) <= np.sqrt((mean ** 2).mean())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1, 2], ids=TYPES)
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 33, 64, 65, 130, 400])
def test_rows(rows, kind):
    torch = _gpu()
    from gpu_util import banner
    for n_in, outs, slots, rank in ((256, [96], 5, 16), (896, [896, 128, 128], 7, 24), (64, [33], 40, 64)):
        banner(f"lora_add rows={rows} in={n_in} out={outs} slots={slots} rank={rank} {TYPES[kind]}")
        c = _case(torch, rows, rows, n_in, outs, slots, rank, kind)
        _check(torch, c)
        _check(torch, c, in_place=True)
        _check(torch, _case(torch, rows, rows, n_in, outs, slots, rank, kind, whole=True))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1, 2], ids=TYPES)
@pytest.mark.parametrize("n_in,out,rank", [(8, 1, 8), (8, 5, 256), (24, 17, 40), (40, 64, 8), (1000, 100, 16), (4096, 257, 128), (18944, 63, 72), (2048, 1000, 256)])
def test_sizes(n_in, out, rank, kind):
    torch = _gpu()
    from gpu_util import banner
    for rows in (1, 21, 90):
        banner(f"lora_add rows={rows} in={n_in} out={out} rank={rank} {TYPES[kind]}")
        _check(torch, _case(torch, out, rows, n_in, [out], 3, rank, kind))
        _check(torch, _case(torch, out, rows, n_in, [out, out + 3, 8, 1], 3, rank, kind), ranks=False, scales=False, wide=1)
        _check(torch, _case(torch, out, rows, n_in, [out], 3, rank, kind, whole=True), wide=5, in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1, 2], ids=TYPES)
def test_order_of_requests(kind):
    """One adapter for all, none at all, runs of requests, every row another adapter, more slots than rows, many rows of many
    adapters in no order."""
    torch = _gpu()
    from gpu_util import banner
    t = torch.tensor
    runs = torch.repeat_interleave(t([2, -1, 0, 2, 1, 5]), t([40, 3, 17, 1, 100, 39]))
    for name, ids, slots in (("one", torch.full((200,), 3), 4), ("none", torch.full((200,), -1), 4), ("past the slots", torch.full((200,), 4), 4),
                             ("runs", runs, 6), ("each its own", torch.arange(200), 200), ("backwards", 199 - torch.arange(200), 1024),
                             ("int32's ends", t([2 ** 31 - 1, -2 ** 31, 0, 1]), 2), ("two in turn", torch.arange(333) % 2, 2)):
        banner(f"lora_add order: {name} {TYPES[kind]}")
        c = _case(torch, 5, len(ids), 320, [130, 24], slots, 16, kind, ids=ids)
        _check(torch, c)
        _check(torch, c, ranks=False, in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1], ids=TYPES[:2])
@pytest.mark.parametrize("rows,slots", [(1000, 3), (2011, 30), (5000, 200)])
def test_many_rows(rows, slots, kind):
    torch = _gpu()
    from gpu_util import banner
    banner(f"lora_add rows={rows} slots={slots} {TYPES[kind]}")
    _check(torch, _case(torch, rows, rows, 512, [300], slots, 32, kind))
    runs = torch.sort(torch.randint(-1, slots, (rows,), generator=torch.Generator().manual_seed(1))).values
    _check(torch, _case(torch, rows, rows, 512, [300], slots, 32, kind, ids=runs), in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("slots", [1, 1024])
def test_most_rows(slots):
    """More tiles than workgroups, with more projections; and no tile at all."""
    torch = _gpu()
    from gpu_util import banner
    banner(f"lora_add rows=65536 slots={slots}")
    c = _case(torch, slots, 65536, 64, [40, 8, 33], slots, 8, 0)
    _check(torch, c)
    c["ids"] = torch.full_like(c["ids"], -1)
    _check(torch, c, in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1, 2], ids=TYPES)
@pytest.mark.parametrize("rank", [72, 200, 256])
def test_many_rows_of_large_ranks(rank, kind):
    torch = _gpu()
    from gpu_util import banner
    banner(f"lora_add rows=300 rank={rank} {TYPES[kind]}")
    _check(torch, _case(torch, rank, 300, 1000, [200, 31], 3, rank, kind))
    _check(torch, _case(torch, rank, 300, 1000, [200, 31], 3, rank, kind, whole=True), in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1, 2], ids=TYPES)
def test_wide_ranges(kind):
    """Values of one row far apart, subnormal weights, and rows of infinities and NaN, which stay in their rows."""
    torch = _gpu()
    from gpu_util import banner, host
    banner(f"lora_add wide ranges {TYPES[kind]}")
    t = getattr(torch, TYPES[kind])
    rows, n_in, out, rank = 40, 128, 50, 8
    # one nonzero weight a rank: z is one product each, y one product more: exact to f32's half steps
    x = (torch.randn(rows, n_in, generator=torch.Generator().manual_seed(2)).double() * 10.0 ** torch.linspace(-30, 25, n_in).double()).float()
    a, b = torch.zeros(1, rank, n_in, dtype=t), torch.zeros(1, out, rank, dtype=t)
    pick = torch.tensor([0, 9, 20, 40, 64, 90, 110, 127])
    a[0, torch.arange(rank), pick] = torch.tensor([1.0, -1.5, 2.0, 6e-8 if kind == 1 else 1e-30 if kind == 0 else 1.17e-37, 0.75, 1.0, -3.0, 0.5]).to(t)
    for o in range(out):
        b[0, o, o % rank] = [1.0, 0.5, -1.25][o % 3]
    c = dict(x=x, mats=[(a, b, torch.zeros(rows, out))], ids=torch.zeros(rows, dtype=torch.int32), ranks=torch.tensor([rank]).int(), scales=torch.ones(1))
    x[5, 0], x[6, 1], x[7, 127] = float("inf"), float("nan"), float("-inf")
    base = torch.zeros(rows, out, device="cuda")
    y = torch.zeros(rows, out, device="cuda")
    ws = torch.empty(qlin.lora_workspace_bytes(rows, 1, 1, rank, n_in) + 16, dtype=torch.uint8, device="cuda")
    qlin.lora_add(x.cuda(), c["ids"].cuda(), [(qlin.Lora(a.cuda(), b.cuda()), base, y)], ranks=c["ranks"].cuda(), scales=c["scales"].cuda(), workspace=ws)
    got = host(y)
    fine = [r for r in range(rows) if r not in (5, 6, 7)]
    z = (x[fine].double() @ a[0].double().T)
    want = (z @ b[0].double().T).numpy()
    # z is rounded once, its product with B once; below 2^-126 in steps of 2^-149
    assert (np.abs(got[fine] - want) <= 3 * STEP * np.abs(want) + 2.0 ** -147).all()
    assert not np.isfinite(got[[5, 6, 7]]).all(1).any()
