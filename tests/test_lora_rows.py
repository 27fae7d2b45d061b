"""A row's adapter gives the same bits whatever stands in the rows beside it, of the same adapter too, and wherever the row stands:
values that the products' parts cannot hold (2^60 and more, infinities, NaN) go apart."""
import pytest

from blog_amd import qlin
from test_lora import TYPES, _case, _check, _gpu

pytestmark = pytest.mark.gpu


def _run(torch, c, x=None, order=None):
    """y of the case's projections (with other x; with the rows in another order, put back)."""
    x = c["x"] if x is None else x
    rows, n_in = x.shape
    order = torch.arange(rows) if order is None else order
    slots, rank = c["mats"][0][0].shape[:2]
    args = [(qlin.Lora(a.cuda(), b.cuda()), base[order].cuda(), torch.zeros_like(base).cuda()) for a, b, base in c["mats"]]
    ws = torch.full((qlin.lora_workspace_bytes(rows, len(args), slots, rank, n_in),), 0xFF, dtype=torch.uint8, device="cuda")
    qlin.lora_add(x[order].cuda(), c["ids"][order].cuda(), args, ranks=c["ranks"].cuda(), scales=c["scales"].cuda(), workspace=ws)
    back = torch.empty_like(order)
    back[order] = torch.arange(rows)
    return [y.cpu()[back] for _, _, y in args]


@pytest.mark.parametrize("kind", [0, 1, 2], ids=TYPES)
@pytest.mark.parametrize("rows,n_in,outs,slots,rank", [(5, 256, [40], 1, 8), (48, 3584, [512, 96], 5, 32), (200, 512, [300], 2, 24), (300, 1000, [200, 31], 3, 72),
                                                       (2011, 512, [130], 3, 64)])
def test_rows_beside_large_ones(rows, n_in, outs, slots, rank, kind):
    torch = _gpu()
    from gpu_util import banner
    banner(f"lora_add large rows: rows={rows} in={n_in} out={outs} slots={slots} rank={rank} {TYPES[kind]}")
    c = _case(torch, rows, rows, n_in, outs, slots, rank, kind)
    want = _run(torch, c)
    gen = torch.Generator().manual_seed(7)
    touched = torch.unique(torch.randint(0, rows, (max(1, rows // 20),), generator=gen))
    others = torch.ones(rows, dtype=torch.bool)
    others[touched] = False
    for value in (2.0 ** 60, -2.0 ** 70, 2.0 ** 59.9, float("inf"), float("nan")):
        x = c["x"].clone()
        x[touched, torch.randint(0, n_in, (len(touched),), generator=gen)] = value
        got = _run(torch, c, x)
        for y, w in zip(got, want):
            assert torch.equal(y[others], w[others]), value
        for turn in range(3):  # (in another order each time: other rows share a tile)
            for y, w in zip(_run(torch, c, x, torch.randperm(rows, generator=gen)), got):
                assert torch.equal(y.view(torch.int32)[others], w.view(torch.int32)[others]), (value, turn)
                assert torch.equal(torch.nan_to_num(y[touched], 7.0), torch.nan_to_num(w[touched], 7.0)), (value, turn)
        if abs(value) < float("inf"):
            _check(torch, {**c, "x": x})


@pytest.mark.parametrize("kind", [0, 1], ids=TYPES[:2])
@pytest.mark.parametrize("rows", [3, 40, 400])
def test_rows_of_large_products(rows, kind):
    """z alone is too large for parts, x is not: rows of x near 2^59, and an adapter whose scale makes it so; in place too."""
    torch = _gpu()
    from gpu_util import banner
    banner(f"lora_add large products: rows={rows} {TYPES[kind]}")
    c = _case(torch, rows, rows, 640, [200, 33], 3, 40, kind)
    want = _run(torch, c)
    mine = torch.arange(rows) % 5 == 2
    x = c["x"].clone()
    x[mine] *= 2.0 ** 57
    got = _run(torch, c, x)
    for y, w in zip(got, want):
        assert torch.equal(y[~mine], w[~mine])
    _check(torch, {**c, "x": x})
    _check(torch, {**c, "x": x}, in_place=True, wide=3)
    scales = c["scales"].clone()
    scales[1] = 2.0 ** 62
    _check(torch, {**c, "scales": scales})
    for y, w in zip(_run(torch, {**c, "scales": scales}), want):
        assert torch.equal(y[c["ids"] != 1], w[c["ids"] != 1])
