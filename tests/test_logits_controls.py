"""Penalties, biases and masks on logits, and the greedy pick (qlin_launch_logits_controls).

The reference takes the documented steps in f32, one rounding each, so results have to be equal bit for bit."""
import ctypes as C

import numpy as np
import pytest

from blog_amd import qlin

OK, UNSUP, SHAPE, NULL, ROWB, LIMIT, LAUNCH, ALIGN = range(8)
FAKE = 0x10000


def reference(logits, vocab, history=None, lens=None, rep=None, freq=None, pres=None, ids=None, values=None, mask=None):
    f = np.float32
    rows = len(logits)
    out = logits[:, :vocab].astype(f)
    picks = np.zeros(rows, np.int32)
    for r in range(rows):
        x = out[r].copy()
        if history is not None:
            h = history[r][:history.shape[1] if lens is None else max(0, min(int(lens[r]), history.shape[1]))]
            h = h[(h >= 0) & (h < vocab)]
            count = np.bincount(h, minlength=vocab)
            seen = count > 0
            p, q, s = (f(d if a is None else a[r]) for a, d in ((rep, 1), (freq, 0), (pres, 0)))
            with np.errstate(over="ignore", invalid="ignore"):
                y = np.where(x > 0, x / p, x * p)
                y = (y - q * count.astype(f)) - s
            x = np.where(seen, y, x).astype(f)
        if ids is not None:
            total = {}
            for t, b in zip(ids[r].tolist(), values[r]):
                if 0 <= t < vocab:
                    total[t] = f(total[t] + b) if t in total else f(b)
            for t, b in total.items():
                x[t] = f(x[t] + b)
        if mask is not None:
            bits = (mask[r][np.arange(vocab) // 32] >> (np.arange(vocab) % 32).astype(np.uint32)) & 1
            x = np.where(bits == 1, x, f(-np.inf))
        out[r] = x
        ok = ~np.isnan(x)
        if ok.any() and x[ok].max() > -np.inf:
            picks[r] = np.flatnonzero(ok & (x == x[ok].max()))[0]
    return out, picks


def test_reference_by_hand():
    x = np.array([[2.0, -2.0, 1.0, 0.5, 3.0, 3.0]], np.float32)
    hist = np.array([[0, 0, 1, 7, -1, 4]], np.int32)
    out, pick = reference(x, 6, hist, np.array([5]), [2.0], [0.25], [0.5], np.array([[3, 3, 9]]), np.array([[1.0, 0.5, 8.0]], np.float32),
                          np.array([[0b101111]], np.uint32))
    assert out.tolist() == [[1.0 - 0.5 - 0.5, -4.0 - 0.25 - 0.5, 1.0, 2.0, -np.inf, 3.0]] and pick[0] == 5


def test_validation():
    def run(null=False, logits=FAKE, ls=100, out=FAKE, os=100, rows=2, vocab=100, picks=FAKE, ws=FAKE, nws=1 << 30, **kw):
        a = dict(history=FAKE, history_lens=FAKE, repetition=FAKE, frequency=FAKE, presence=FAKE, bias_ids=FAKE, bias_values=FAKE,
                 mask=FAKE, mask_stride=4, max_history=10, max_bias=4)
        a.update(kw)
        c = qlin.LogitsControlsArgs(*a.values())
        return qlin.status("qlin_launch_logits_controls", None if null else C.addressof(c), logits, ls, out, os, rows, vocab, picks, ws, nws)
    assert run(null=True) == NULL
    assert run(rows=-1) == SHAPE and run(vocab=-1) == SHAPE and run(max_history=-1) == SHAPE and run(max_bias=-1) == SHAPE
    assert run(ls=99) == SHAPE and run(os=99) == SHAPE and run(os=101) == SHAPE and run(mask_stride=3) == SHAPE
    assert run(max_history=(1 << 20) + 1) == LIMIT and run(max_bias=4097) == LIMIT and run(vocab=(1 << 28) + 1, ls=1 << 29, os=1 << 29, mask_stride=1 << 24) == LIMIT
    assert run(logits=0) == NULL and run(out=0) == NULL and run(bias_values=0) == NULL
    for name in ("history", "history_lens", "repetition", "frequency", "presence", "bias_ids", "bias_values", "mask"):
        assert run(**{name: FAKE + 2}) == ALIGN, name
    for name in ("logits", "out", "picks", "ws"):
        assert run(**{name: FAKE + 1}) == ALIGN, name
    need = qlin.logits_controls_scratch_bytes(3, 151936)
    assert need > 0
    assert run(rows=3, vocab=151936, ls=151936, os=151936, mask_stride=4748, ws=0, nws=0) == NULL
    assert run(rows=3, vocab=151936, ls=151936, os=151936, mask_stride=4748, nws=need - 1) == LIMIT
    assert run(rows=0, logits=0, out=0) == OK and run(vocab=0, logits=0, out=0) == OK
    assert qlin.logits_controls_scratch_bytes(0, 5) == 0 and qlin.logits_controls_scratch_bytes(5, -1) == 0


def test_python_layouts():
    import torch
    x, wide = torch.zeros(2, 64), torch.zeros(2, 128)
    ids = torch.zeros(2, 8, dtype=torch.int32)
    for kw in (dict(logits=wide[:, ::2]), dict(out=wide[:, ::2]), dict(history=ids[:, ::2]), dict(mask=ids[:, :2]),
               dict(bias_ids=ids[:, :4], bias_values=x[:, :4].contiguous()),
               dict(bias_ids=ids, bias_values=x[:, :8]), dict(bias_ids=ids, bias_values=x)):
        with pytest.raises(ValueError):
            qlin.logits_controls(**{**dict(logits=x, out=x, rows=2, vocab=64), **kw})


# ---- GPU ---------------------------------------------------------------------------------------

def _gpu():
    import torch
    from gpu_util import bind_stream
    assert torch.cuda.is_available(), "GPU tests need the MI355X"
    bind_stream()
    return torch


def _case(rng, rows, vocab, max_history, max_bias, masked, spread=3.0):
    a = dict(logits=(spread * rng.standard_normal((rows, vocab))).astype(np.float32))
    if max_history:
        a["history"] = rng.integers(-3, vocab + 3, (rows, max_history)).astype(np.int32)
        a["history"][:, ::2] = a["history"][:, :1]  # one token many times
        a["lens"] = rng.integers(-1, max_history + 2, rows).astype(np.int32)
        a["lens"][0] = max_history
        a["rep"], a["freq"], a["pres"] = (rng.uniform(lo, hi, rows).astype(np.float32) for lo, hi in ((0.7, 1.6), (-0.1, 0.3), (-0.2, 0.5)))
    if max_bias:
        a["ids"] = rng.integers(-2, vocab + 2, (rows, max_bias)).astype(np.int32)
        a["ids"][:, max_bias // 2:] = a["ids"][:, :max_bias - max_bias // 2]  # tokens twice, some more often
        a["ids"][:, -2:] = a["ids"][:, :1]
        a["values"] = (5 * rng.standard_normal((rows, max_bias))).astype(np.float32)
    if masked:
        a["mask"] = rng.integers(0, 1 << 32, (rows, (vocab + 31) // 32 + 1), dtype=np.uint32)
    return a


def _run(torch, a, vocab, in_place=False, picks=True, pad=0, lead=0):
    from gpu_util import dev, host
    rows = len(a["logits"])
    wide = np.full((rows, lead + vocab + pad), 7.0, np.float32)
    wide[:, lead:lead + vocab] = a["logits"]
    x = dev(wide)[:, lead:]
    out = x if in_place else torch.full((rows, vocab + pad), 7.0, dtype=torch.float32, device="cuda")
    pick = torch.full((rows,), -9, dtype=torch.int32, device="cuda")
    need = qlin.logits_controls_scratch_bytes(rows, vocab)
    ws = torch.full((need + 16,), 0xFF, dtype=torch.uint8, device="cuda")
    t = {k: dev(v.view(np.int32) if v.dtype == np.uint32 else v) for k, v in a.items() if k != "logits"}
    qlin.logits_controls(x, out, rows, vocab, history=t.get("history"), history_lens=t.get("lens"), repetition=t.get("rep"),
                         frequency=t.get("freq"), presence=t.get("pres"), bias_ids=t.get("ids"), bias_values=t.get("values"),
                         mask=t.get("mask"), picks=pick if picks else None, scratch=ws if picks else None)
    got = host(out)
    assert (got[:, vocab:] == 7.0).all()  # past the vocabulary, as it was
    assert (ws[need:] == 0xFF).all()
    if not in_place:
        assert np.array_equal(host(x)[:, :vocab], a["logits"], equal_nan=True)
    return got[:, :vocab], host(pick)


def _check(torch, a, vocab, **kw):
    got, pick = _run(torch, a, vocab, **kw)
    want, best = reference(a["logits"], vocab, *(a.get(k) for k in ("history", "lens", "rep", "freq", "pres", "ids", "values", "mask")))
    assert np.array_equal(got, want, equal_nan=True)
    if kw.get("picks", True):
        assert np.array_equal(pick, best)
    else:
        assert (pick == -9).all()


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 1023, 1024, 1025, 4099, 32000, 50257])
@pytest.mark.parametrize("rows,max_history,max_bias,masked", [(1, 40, 0, True), (3, 700, 9, True), (2, 0, 300, False), (5, 1, 1, False), (2, 0, 0, True)])
def test_logits_controls(vocab, rows, max_history, max_bias, masked):
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(vocab + rows)
    banner(f"logits_controls vocab={vocab} rows={rows} history={max_history} biases={max_bias} masked={masked}")
    a = _case(rng, rows, vocab, max_history, max_bias, masked)
    _check(torch, a, vocab)
    _check(torch, a, vocab, in_place=True)
    _check(torch, a, vocab, pad=3, lead=1)  # rows at 4-byte alignment
    _check(torch, a, vocab, picks=False)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,max_history,max_bias", [(1, 151936, 600, 20), (40, 102400, 3000, 64), (300, 32000, 50, 4096), (2, 151936, 70000, 0),
                                                             (130, 60001, 100, 3)])
def test_logits_controls_large(rows, vocab, max_history, max_bias):
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(rows)
    banner(f"logits_controls vocab={vocab} rows={rows} history={max_history} biases={max_bias}")
    _check(torch, _case(rng, rows, vocab, max_history, max_bias, True), vocab)


@pytest.mark.gpu
def test_logits_controls_odd_values():
    """NaN and infinities among the logits, ties, rows whose mask or biases leave nothing, defaults of absent arrays."""
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(6)
    vocab = 5000
    banner("logits_controls odd values")
    a = _case(rng, 9, vocab, 50, 8, True)
    x = a["logits"]
    x[0, ::3] = np.nan
    x[1, 17], x[1, 4000] = np.inf, np.inf
    x[2, :] = -np.inf
    x[3, :] = np.nan
    a["mask"][4, :] = 0
    x[5, :] = 1.25  # ties: the lowest index that is left
    a["ids"][6, :4], a["values"][6, :4] = [9, 10, 9, 11], [-np.inf, np.inf, 1.0, np.nan]
    x[7, 100] = np.nan
    a["mask"][7, 3] &= ~np.uint32(1 << 4)  # a masked NaN is -inf
    x[8, :] = -3.0e38  # the type's lowest, scaled beyond it
    a["rep"][8] = 1.5
    _check(torch, a, vocab)
    for drop in (("lens",), ("rep",), ("freq", "pres"), ("rep", "freq", "pres"), ("history", "lens", "rep", "freq", "pres")):
        _check(torch, {k: v for k, v in a.items() if k not in drop}, vocab)


@pytest.mark.gpu
def test_logits_pick_is_the_argmax_entrys():
    torch = _gpu()
    from gpu_util import banner, dev, host
    rng = np.random.default_rng(7)
    for vocab in (100, 151936):
        banner(f"pick against qlin_launch_argmax, vocab={vocab}")
        x = rng.integers(-5, 6, (3, vocab)).astype(np.float32)  # many ties
        got, pick = _run(torch, dict(logits=x), vocab)
        one = torch.zeros(1, dtype=torch.int32, device="cuda")
        for r in range(3):
            qlin.call("qlin_launch_argmax", dev(x[r]), vocab, one)
            assert host(one)[0] == pick[r]
