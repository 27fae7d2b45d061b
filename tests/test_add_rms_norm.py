"""The residual's addition with the RMSNorm into f32 and Q8_1 blocks (qlin_launch_add_rms_norm), and Q8_1 blocks read back
(qlin_launch_dequantize_q8_1).

The sum is one f32 addition and has to be equal; y is computed in 64 bits and rounded once, so it is off by at most half a step
of f32 (2^-24 of the value; 2^-50 more for the 64-bit arithmetic); the blocks are, byte for byte, those of the documented steps
for the y that the same call returns.  Sums of the values themselves (raw_sum) are f32 sums of 32 terms (a tree of depth 5: 5
half steps of f32 of the sum of magnitudes) rounded to f16 once (half a step, 2^-11, or half of its smallest, 2^-25)."""
import numpy as np
import pytest

from blog_amd import qlin

OK, UNSUP, SHAPE, NULL, ROWB, LIMIT, LAUNCH, ALIGN = range(8)
FAKE = 0x10000


def reference(s, weight64, eps, hidden):
    s = s.astype(np.float64)
    return s / np.sqrt((s * s).sum(1, keepdims=True) / hidden + np.float64(np.float32(eps))) * weight64


def test_validation():
    def run(x=FAKE, xs=64, delta=FAKE, ds=64, sum=FAKE * 2, ss=64, w=FAKE, t=0, normed=FAKE * 3, ns=64, q8=FAKE * 4, mmq=0, rows=2, hidden=64):
        return qlin.status("qlin_launch_add_rms_norm", x, xs, delta, ds, sum, ss, w, t, 1e-6, 0, normed, ns, q8, mmq, 0, rows, hidden)
    assert run(t=2) == UNSUP and run(t=-1) == UNSUP
    assert run(rows=-1) == SHAPE and run(hidden=-1) == SHAPE
    assert run(xs=63) == SHAPE and run(ds=63) == SHAPE and run(ss=63) == SHAPE and run(ns=63) == SHAPE
    assert run(x=0) == NULL and run(w=0) == NULL and run(normed=0, q8=0) == NULL
    for name in ("x", "delta", "sum", "normed", "q8"):
        assert run(**{name: FAKE * 5 + 2}) == ALIGN, name
    assert run(w=FAKE + 1) == ALIGN
    assert run(sum=FAKE, ss=65) == SHAPE  # in place with another stride
    assert run(delta=FAKE * 6, sum=FAKE * 6, ss=65) == SHAPE and run(normed=FAKE * 2) == SHAPE and run(normed=FAKE, ns=65) == SHAPE
    assert run(hidden=(1 << 24) + 1, xs=1 << 25, ds=1 << 25, ss=1 << 25, ns=1 << 25) == LIMIT
    assert run(rows=0, x=0) == OK and run(hidden=0, x=0) == OK
    back = lambda q=FAKE, x=FAKE, n=40, m=2, mmq=0: qlin.status("qlin_launch_dequantize_q8_1", q, x, n, m, mmq)
    assert back(n=-1) == SHAPE and back(m=-1) == SHAPE and back(q=0) == NULL and back(x=0) == NULL
    assert back(q=FAKE + 2) == ALIGN and back(x=FAKE + 1) == ALIGN and back(n=0, q=0) == OK and back(m=0, x=0) == OK


def test_python_refusals():
    import torch
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError):  # not on a GPU
        qlin.add_rms_norm(x, None, None, torch.zeros(64, dtype=torch.bfloat16), 0, 1e-6, 0, normed=x)
    with pytest.raises(ValueError):
        qlin.dequantize_q8_1(torch.zeros(144, dtype=torch.uint8), x, 64, 2)


# ---- GPU ---------------------------------------------------------------------------------------

def _gpu():
    import torch
    from gpu_util import bind_stream
    assert torch.cuda.is_available(), "GPU tests need the MI355X"
    bind_stream()
    return torch


def _weights(torch, rng, hidden, kind, one_plus):
    t = torch.from_numpy((1 + 0.3 * rng.standard_normal(hidden)).astype(np.float32)).to(torch.float16 if kind else torch.bfloat16)
    return t.cuda(), t.double().numpy() + one_plus


def _run(torch, rng, rows, hidden, *, delta=True, kind=0, one_plus=0, mmq=False, raw=False, f32=True, blocks=True, wide=0, in_place=False,
         x=None):
    from gpu_util import dev, host
    w, w64 = _weights(torch, rng, hidden, kind, one_plus)
    xn = (4 * rng.standard_normal((rows, hidden + wide))).astype(np.float32) if x is None else x
    dn = rng.standard_normal((rows, hidden + 2 * wide)).astype(np.float32)
    xd, dd = dev(xn)[:, wide:], dev(dn)[:, wide:wide + hidden] if delta else None
    s = xd if in_place else torch.full((rows + 1, hidden + wide), 7.0, device="cuda")[:rows, :hidden]
    y = torch.full((rows + 1, hidden + 3), 7.0, device="cuda") if f32 or blocks else None
    size = qlin.q8_1_bytes(hidden, rows, mmq)
    q = torch.full((size + 64,), 0x55, dtype=torch.uint8, device="cuda") if blocks else None
    qlin.add_rms_norm(xd, dd, s, w, kind, 1e-5, one_plus, normed=y[:rows, :hidden] if f32 else None, q8_1=q, mmq=mmq, raw_sum=raw)
    sums = xn[:, wide:] + dn[:, wide:wide + hidden] if delta else xn[:, wide:]
    assert np.array_equal(host(s)[:rows, :hidden], sums, equal_nan=True)
    if not in_place:
        assert np.array_equal(host(xd), xn[:, wide:], equal_nan=True)
    want = reference(sums, w64, 1e-5, hidden)
    if not f32:  # (the blocks' own check needs y)
        qlin.add_rms_norm(s, None, None, w, kind, 1e-5, one_plus, normed=y[:rows, :hidden])
    got = host(y)
    assert (got[rows:] == 7.0).all() and (got[:, hidden:] == 7.0).all()
    got = got[:rows, :hidden]
    if blocks:
        unit = 128 if mmq else 32
        v = np.zeros((rows, -(-hidden // unit) * unit), np.float32)
        v[:, :hidden] = got
        v = v.reshape(rows, -1, 32)
        scale = np.abs(v).max(2) * (np.float32(1) / np.float32(127))
        inverse = np.where(scale >= 2.0 ** -126, np.float32(1) / np.maximum(scale, np.float32(2.0 ** -126)), np.float32(0))
        q_want = np.clip(np.rint(v * inverse[:, :, None]), -127, 127).astype(np.int8)
        b = host(q)
        assert (b[size:] == 0x55).all()
        if mmq:
            b = b[:size].reshape(-1, rows, 144).transpose(1, 0, 2)
            heads, codes = b[:, :, :16].copy().view(np.float16).reshape(rows, -1, 2), b[:, :, 16:].copy().view(np.int8)
        else:
            b = b[:size].reshape(rows, -1, 36)
            heads, codes = b[:, :, :4].copy().view(np.float16).reshape(rows, -1, 2), b[:, :, 4:].copy().view(np.int8)
        assert np.array_equal(codes.reshape(q_want.shape), q_want)
        assert np.array_equal(heads[:, :, 0], scale.astype(np.float16))
        if raw:
            v64 = v.astype(np.float64)
            sums = v64.sum(2)
            assert (np.abs(heads[:, :, 1] - sums) <= 2.0 ** -11 * np.abs(sums) + 2.0 ** -25 + 6 * 2.0 ** -24 * np.abs(v64).sum(2)).all()
        else:
            assert np.array_equal(heads[:, :, 1], (scale * q_want.sum(2, dtype=np.int32).astype(np.float32)).astype(np.float16))
        d, codes = heads[:, :, 0], codes.reshape(rows, -1)
        back = torch.full((rows * hidden + 5,), 7.0, device="cuda")
        qlin.dequantize_q8_1(q, back, hidden, rows, mmq=mmq)
        values = d.astype(np.float32).repeat(32, 1) * codes.astype(np.float32)
        back = host(back)
        assert np.array_equal(back[:rows * hidden].reshape(rows, hidden), values[:, :hidden], equal_nan=True) and (back[rows * hidden:] == 7.0).all()
    return got, want


HALF_STEP = 2.0 ** -24 + 2.0 ** -50


@pytest.mark.gpu
@pytest.mark.parametrize("hidden", [1, 2, 31, 33, 64, 127, 129, 255, 256, 257, 500, 896, 1024, 1025, 2047, 2048, 3584, 4096, 4100, 8192, 8193,
                                    16384, 16400, 20001])
@pytest.mark.parametrize("mmq", [False, True])
def test_sizes(hidden, mmq):
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(hidden)
    for rows in (1, 2, 7):
        banner(f"add_rms_norm rows={rows} hidden={hidden} mmq={mmq}")
        got, want = _run(torch, rng, rows, hidden, mmq=mmq)
        assert (np.abs(got - want) <= HALF_STEP * np.abs(want) + 2.0 ** -149).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(delta=False), dict(kind=1), dict(one_plus=1), dict(kind=1, one_plus=1), dict(raw=True), dict(raw=True, mmq=True),
                                dict(f32=False), dict(blocks=False), dict(wide=3), dict(wide=4), dict(in_place=True), dict(in_place=True, wide=1),
                                dict(delta=False, f32=False, mmq=True)], ids=lambda kw: ",".join(f"{k}={v}" for k, v in kw.items()))
@pytest.mark.parametrize("rows,hidden", [(5, 200), (300, 896), (3, 4096), (2, 20000)])
def test_forms(rows, hidden, kw):
    torch = _gpu()
    from gpu_util import banner
    banner(f"add_rms_norm rows={rows} hidden={hidden} {kw}")
    got, want = _run(torch, np.random.default_rng(rows), rows, hidden, **kw)
    assert (np.abs(got - want) <= HALF_STEP * np.abs(want) + 2.0 ** -149).all()


@pytest.mark.gpu
def test_outputs_in_the_inputs_place():
    """normed over x and over delta, where the sum is stored elsewhere or not at all; the sum over delta."""
    torch = _gpu()
    from gpu_util import banner
    gen = torch.Generator(device="cuda").manual_seed(3)
    for rows, hidden in ((3, 900), (2, 17000)):
        banner(f"add_rms_norm in place rows={rows} hidden={hidden}")
        x, d = (torch.randn(rows, hidden, device="cuda", generator=gen) for _ in range(2))
        w = torch.ones(hidden, dtype=torch.bfloat16, device="cuda")
        want, total = torch.empty_like(x), torch.empty_like(x)
        qlin.add_rms_norm(x, d, total, w, 0, 1e-6, 0, normed=want)
        for where in ("x", "delta", "sum over delta", "x and delta", "sum and x"):
            a, b = x.clone(), d.clone()
            y = a if where in ("x", "sum and x") else b if where in ("delta", "x and delta") else torch.empty_like(x)
            s = b if where in ("sum over delta", "sum and x") else a if where == "x and delta" else None
            qlin.add_rms_norm(a, b, s, w, 0, 1e-6, 0, normed=y)
            torch.cuda.synchronize()
            assert torch.equal(y, want), where
            assert s is None or torch.equal(s, total), where


@pytest.mark.gpu
def test_odd_values():
    """Rows of zeros, tiny and huge values, infinities and NaN, which stay in their rows."""
    torch = _gpu()
    from gpu_util import banner
    banner("add_rms_norm odd values")
    rng = np.random.default_rng(9)
    x = rng.standard_normal((8, 300)).astype(np.float32)
    x[1] = 0
    x[2] *= np.float32(1e-42)
    x[3] *= np.float32(1e37)
    x[4, 7] = np.inf
    x[5, 8] = np.nan
    x[6, :] = np.float32(3e38)
    with np.errstate(invalid="ignore"):
        got, want = _run(torch, rng, 8, 300, delta=False, x=x, blocks=False)
    for r in (0, 1, 2, 3, 6, 7):
        assert (np.abs(got[r] - want[r]) <= HALF_STEP * np.abs(want[r]) + 2.0 ** -149).all(), r
    assert np.isnan(got[4, 7]) and (np.delete(got[4], 7) == 0).all() and np.isnan(got[5]).all()


@pytest.mark.gpu
def test_many_rows():
    torch = _gpu()
    from gpu_util import banner
    for rows, hidden in ((2011, 4096), (3001, 128), (1500, 1000)):
        banner(f"add_rms_norm rows={rows} hidden={hidden}")
        got, want = _run(torch, np.random.default_rng(rows), rows, hidden, mmq=True)
        assert (np.abs(got - want) <= HALF_STEP * np.abs(want) + 2.0 ** -149).all()


@pytest.mark.gpu
@pytest.mark.parametrize("mmq", [False, True])
def test_blocks_as_the_quantizers(mmq):
    """qlin_launch_quantize_q8_1's blocks of the same y: scales a step of f16 apart at most (2^-10 of 127 steps) and codes one,
    which few are."""
    torch = _gpu()
    from gpu_util import banner, host
    banner(f"add_rms_norm and quantize_q8_1 mmq={mmq}")
    rows, hidden = 50, 4096
    x = torch.randn(rows, hidden, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    y, size = torch.empty_like(x), qlin.q8_1_bytes(hidden, rows, mmq)
    q, ref = (torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in range(2))
    qlin.add_rms_norm(x, None, None, torch.ones(hidden, dtype=torch.bfloat16, device="cuda"), 0, 1e-6, 0, normed=y, q8_1=q, mmq=mmq)
    qlin.call("qlin_launch_quantize_q8_1_mmq" if mmq else "qlin_launch_quantize_q8_1", y, ref, hidden, rows, 0)
    a, b = torch.empty_like(x), torch.empty_like(x)
    qlin.dequantize_q8_1(q, a, hidden, rows, mmq=mmq)
    qlin.dequantize_q8_1(ref, b, hidden, rows, mmq=mmq)
    step = np.abs(host(y)).reshape(rows, -1, 32).max(2).repeat(32, 1) / 127
    assert (np.abs(host(a) - host(b)) <= 1.13 * step).all() and (host(a) != host(b)).mean() <= 1e-2


@pytest.mark.gpu
def test_blocks_that_are_not_finite():
    torch = _gpu()
    from gpu_util import banner, host
    banner("add_rms_norm blocks that are not finite")
    x = torch.ones(3, 96, device="cuda")
    x[1, 40] = float("nan")
    x[2, 40] = float("inf")
    q = torch.zeros(qlin.q8_1_bytes(96, 3), dtype=torch.uint8, device="cuda")
    y = torch.zeros(3, 96, device="cuda")
    qlin.add_rms_norm(x, None, None, torch.ones(96, dtype=torch.bfloat16, device="cuda"), 0, 1e-6, 0, q8_1=q)
    qlin.dequantize_q8_1(q, y, 96, 3)
    got = host(y)
    assert np.isfinite(got[0]).all() and np.isnan(got[1]).all()
    assert (got[2, :32] == 0).all() and np.isnan(got[2, 32:64]).all() and (got[2, 64:] == 0).all()  # 1 / inf, inf / inf
