"""Drafted tokens checked against the target's probabilities (qlin_launch_verify_drafts) against the formula in 64 bits.

Tokens and counts have to be equal.  rates and logprobs are computed in 64 bits and rounded once: half a step (2^-24 of the value),
and 1e-11 for exponentials and sums of up to 2^18 terms in 64 bits."""
import numpy as np
import pytest

from blog_amd import qlin

OK, UNSUP, SHAPE, NULL, ROWB, LIMIT, LAUNCH, ALIGN = range(8)
FAKE = 0x10000
NEXT = np.nextafter(np.float32(1), np.float32(0))


def probabilities(l, t):
    """softmax(l / t), and its logarithms; all of it at the first largest for t = 0; zeros where no logit is above -inf."""
    l = np.where(np.isnan(l), -np.inf, l).astype(np.float64)
    top = l.max()
    if top == -np.inf:
        return np.zeros(len(l)), np.full(len(l), -np.inf)
    if not t > 0:
        one = np.zeros(len(l))
        one[np.flatnonzero(l == top)[0]] = 1
    elif top == np.inf:
        one = (l == top).astype(np.float64)
        one /= one.sum()
    else:
        with np.errstate(over="ignore", invalid="ignore"):
            x = np.where(l > -np.inf, np.where(l == top, 0.0, l - top) / np.float64(np.float32(t)), -np.inf)
        e = np.exp(x)
        return e / e.sum(), x - np.log(e.sum())
    with np.errstate(divide="ignore"):
        return one, np.log(one)


def number(u):
    return 0.0 if np.isnan(u) else float(min(max(u, np.float32(0)), NEXT))


def reference(target, drafts, uniform, draft=None, n_drafts=None, temperature=None):
    n, rows, vocab = target.shape
    d = rows - 1
    tokens, accepted = np.full((n, rows), -1, np.int32), np.zeros(n, np.int32)
    logprobs, rates = np.zeros((n, rows)), np.zeros((n, d))
    for s in range(n):
        t = 1.0 if temperature is None else temperature[s]
        most = d if n_drafts is None else max(0, min(int(n_drafts[s]), d))
        going = True
        for i in range(most + 1):
            p, logs = probabilities(target[s, i], t)
            rest = p
            if i < most:
                x = int(drafts[s, i])
                there = 0 <= x < vocab
                if draft is not None:
                    q = probabilities(draft[s, i], t)[0]
                else:
                    q = np.zeros(vocab)
                    if there:
                        q[x] = 1
                px, qx = (p[x], q[x]) if there else (0.0, 0.0)
                rates[s, i] = min(1.0, px / qx) if qx > 0 else float(px > 0)
                if not going:
                    continue
                if number(uniform[s, i]) * qx < px:
                    tokens[s, i], logprobs[s, i] = x, logs[x]
                    continue
                rest = np.maximum(p - q, 0)
                if not rest.sum() > 0:
                    rest = p
            if going:
                going = False
                accepted[s] = i
                if not p.sum() > 0:
                    tokens[s, i], logprobs[s, i] = 0, -np.inf
                    continue
                # (in units of the largest: of 3000 equal weights, half of their sum is that of 1500, which 1 / 3001 each
                # would miss by a rounding)
                sums = np.cumsum(rest / rest.max())
                y = int(np.flatnonzero(sums > number(uniform[s, d]) * sums[-1])[0])
                tokens[s, i], logprobs[s, i] = y, logs[y]
    return tokens, accepted, logprobs, rates


def test_reference_by_hand():
    target = np.log(np.array([[[0.5, 0.3, 0.2], [0.1, 0.1, 0.8]]], np.float32))
    u = lambda *v: np.array([v], np.float32)
    # by lookup: taken with the target's own probability
    assert [a.tolist() for a in reference(target, np.array([[0]]), u(0.4, 0.5))[:2]] == [[[0, 2]], [1]]
    assert [a.tolist() for a in reference(target, np.array([[0]]), u(0.6, 0.5))[:2]] == [[[1, -1]], [0]]  # 0.3 and 0.2 are left
    assert [a.tolist() for a in reference(target, np.array([[0]]), u(0.6, 0.7))[:2]] == [[[2, -1]], [0]]
    draft = np.log(np.array([[[0.25, 0.5, 0.25]]], np.float32))
    got = reference(target, np.array([[1]]), u(0.7, 0.99), draft=draft)  # 0.3 / 0.5; what is left: 0.25 at the first token
    assert got[0].tolist() == [[0, -1]] and np.allclose(got[3], 0.6) and np.allclose(got[2], [[np.log(0.5), 0]])


def test_validation():
    def run(target=FAKE, ts=100, draft=FAKE, ds=100, drafts=FAKE, n_drafts=FAKE, temp=FAKE, uni=FAKE, tok=FAKE, acc=FAKE, logs=FAKE, rates=FAKE,
            n=2, d=3, vocab=100, ws=FAKE, nws=1 << 30):
        return qlin.status("qlin_launch_verify_drafts", target, ts, draft, ds, drafts, n_drafts, temp, uni, tok, acc, logs, rates, n, d, vocab, ws, nws)
    assert run(n=-1) == SHAPE and run(d=-1) == SHAPE and run(vocab=-1) == SHAPE and run(vocab=0) == SHAPE
    assert run(ts=99) == SHAPE and run(ds=99) == SHAPE
    assert run(d=64) == LIMIT and run(vocab=(1 << 21) + 1, ts=1 << 29, ds=1 << 29) == LIMIT
    assert run(n=1 << 22, vocab=151936, ts=151936, ds=151936, nws=1 << 60) == LIMIT
    for name in ("target", "uni", "tok", "acc", "drafts", "ws"):
        assert run(**{name: 0}) == NULL, name
    for name in ("target", "draft", "drafts", "n_drafts", "temp", "uni", "tok", "acc", "logs", "rates"):
        assert run(**{name: FAKE + 2}) == ALIGN, name
    assert run(ws=FAKE + 8) == ALIGN
    need = qlin.verify_drafts_workspace_bytes(2, 3, 100)
    assert need > 0 and run(nws=need - 1) == LIMIT
    assert run(n=0, target=0) == OK
    for bad in ((0, 3, 100), (2, -1, 100), (2, 64, 100), (2, 3, 0), (2, 3, (1 << 21) + 1)):
        assert qlin.verify_drafts_workspace_bytes(*bad) == 0


def test_python_refusals():
    import torch
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    with pytest.raises(ValueError):
        qlin.verify_drafts(torch.zeros(2, 3, 50), i32(2, 2), torch.zeros(2, 3), i32(2, 3), i32(2))


# ---- GPU ---------------------------------------------------------------------------------------

def _gpu():
    import torch
    from gpu_util import bind_stream
    assert torch.cuda.is_available(), "GPU tests need the MI355X"
    bind_stream()
    return torch


def _case(rng, n, d, vocab, with_draft, spread=2.5):
    target = (spread * rng.standard_normal((n, d + 1, vocab))).astype(np.float32)
    a = dict(target=target, uniform=rng.random((n, d + 1)).astype(np.float32), drafts=np.zeros((n, d), np.int32))
    near = (target[:, :d] + 0.7 * rng.standard_normal((n, d, vocab))).astype(np.float32)
    if d:
        a["drafts"][:] = (near + rng.gumbel(size=near.shape)).argmax(2) if with_draft else near.argmax(2)
    if with_draft:
        a["draft"] = near
    return a


def _run(torch, a, pad=0, optional=True):
    from gpu_util import dev, host
    n, rows, vocab = a["target"].shape
    d = rows - 1

    def wide(x):
        w = np.full(x.shape[:2] + (vocab + pad,), 1e4, np.float32)  # (what stands beside the vocabulary would win)
        w[:, :, :vocab] = x
        return dev(w)[:, :, :vocab]
    t = {k: dev(a[k]) for k in ("drafts", "uniform", "n_drafts", "temperature") if k in a}
    tokens = torch.full((n + 1, rows), -9, dtype=torch.int32, device="cuda")
    accepted = torch.full((n + 1,), -9, dtype=torch.int32, device="cuda")
    logs, rates = torch.full((n + 1, rows), 7.0, device="cuda"), torch.full((n + 1, d), 7.0, device="cuda")
    need = qlin.verify_drafts_workspace_bytes(n, d, vocab)
    ws = torch.full((need + 16,), 0xFF, dtype=torch.uint8, device="cuda")
    qlin.verify_drafts(wide(a["target"]), t["drafts"], t["uniform"], tokens[:n], accepted[:n],
                       draft_logits=wide(a["draft"]) if "draft" in a else None, n_drafts=t.get("n_drafts"), temperature=t.get("temperature"),
                       logprobs=logs[:n] if optional else None, rates=rates[:n] if optional else None, workspace=ws[:need])
    out = [host(x) for x in (tokens, accepted, logs, rates)]
    assert (ws[need:] == 0xFF).all() and (out[0][n] == -9).all() and out[1][n] == -9 and (out[2][n] == 7).all() and (out[3][n] == 7).all()
    return [x[:n] for x in out]


def _check(torch, a, **kw):
    tokens, accepted, logs, rates = _run(torch, a, **kw)
    want = reference(a["target"], a["drafts"], a["uniform"], a.get("draft"), a.get("n_drafts"), a.get("temperature"))
    assert np.array_equal(accepted, want[1])
    assert np.array_equal(tokens, want[0])
    if kw.get("optional", True):
        for got, w in ((logs, want[2]), (rates, want[3])):
            fine = np.isfinite(w)
            assert np.array_equal(got[~fine], w[~fine])
            assert (np.abs(got[fine] - w[fine]) <= 2.0 ** -24 * np.abs(w[fine]) + 1e-11).all()
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 257, 1000, 1023, 1024, 1025, 4099, 32000])
@pytest.mark.parametrize("n,d,with_draft", [(1, 0, False), (3, 1, False), (4, 4, True), (9, 3, True), (2, 7, False), (1, 63, True)])
def test_verify(vocab, n, d, with_draft):
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(vocab + d)
    a = _case(rng, n, d, vocab, with_draft)
    banner(f"verify_drafts vocab={vocab} seqs={n} drafts={d} draft logits={with_draft}")
    _check(torch, a)
    a["temperature"] = rng.uniform(0.3, 1.5, n).astype(np.float32)
    a["temperature"][::3] = [0.0, -1.0, np.nan][(n + d) % 3]
    a["n_drafts"] = rng.integers(-1, d + 2, n).astype(np.int32)
    _check(torch, a, pad=1)
    _check(torch, a, pad=3, optional=False)


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,vocab,with_draft", [(1, 4, 151936, False), (24, 4, 151936, True), (150, 0, 102400, False), (40, 2, 60001, True),
                                                (1, 1, 1 << 21, True), (2, 1, 600000, False)])
def test_verify_large(n, d, vocab, with_draft):
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(n)
    banner(f"verify_drafts vocab={vocab} seqs={n} drafts={d} draft logits={with_draft}")
    a = _case(rng, n, d, vocab, with_draft)
    a["temperature"] = rng.uniform(0.0, 1.2, n).astype(np.float32)
    _check(torch, a)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [196608, 196609, 400003, 524288])
@pytest.mark.parametrize("with_draft", [False, True])
def test_few_rows_of_many_slices(vocab, with_draft):
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(vocab)
    banner(f"verify_drafts vocab={vocab} 2 sequences, draft logits={with_draft}")
    a = _case(rng, 2, 1, vocab, with_draft)
    for temperature in ([0.0, 0.8], [0.9, 0.0]):
        a["temperature"] = np.array(temperature, np.float32)
        for u in (0.0, 0.5, NEXT):
            a["uniform"][:, 1] = u
            _check(torch, a)


@pytest.mark.gpu
@pytest.mark.parametrize("with_draft", [False, True])
def test_odd_values(with_draft):
    """Masked tokens, rows that a mask leaves empty, infinities and NaN, ties, drafts outside the vocabulary, random numbers at
    and outside the ends, equal distributions, temperatures far from one."""
    torch = _gpu()
    from gpu_util import banner
    banner(f"verify_drafts odd values, draft logits={with_draft}")
    rng = np.random.default_rng(11)
    n, d, vocab = 24, 3, 3001
    a = _case(rng, n, d, vocab, with_draft)
    t = a["target"]
    lowest = np.finfo(np.float32).min
    t[0, 0, ::2] = -np.inf  # masked
    t[1, 1, :] = -np.inf    # a mask that leaves nothing
    t[2, 0, :] = np.nan
    t[3, 2, ::3] = np.nan
    t[4, 0, [5, 2999]] = np.inf
    t[5, 0, :] = lowest     # a mask of the type's lowest value
    t[6, 0, :] = lowest
    t[6, 0, 77] = 1.0
    t[7] = 2.0              # ties
    a["drafts"][8] = [-1, 5, 7]
    a["drafts"][9] = [vocab, 5, 7]
    a["uniform"][10] = 0.0
    a["uniform"][11] = NEXT
    a["uniform"][12] = 1.0
    a["uniform"][13] = -0.5
    a["uniform"][14] = np.nan
    a["uniform"][15] = np.inf
    t[16, :, :] = -np.inf
    t[16, :, 1500] = 0.25   # one token is left, drafted or not
    a["drafts"][16] = [1500, 1500, 3]
    t[17, 0, a["drafts"][17, 0]] = -np.inf  # the target never says what was drafted
    if with_draft:
        a["draft"][18] = t[18, :d]  # the same distribution
        a["uniform"][18] = NEXT
        a["draft"][19, 0] = -np.inf
        a["draft"][20, 1] = np.nan
        a["draft"][21, 0, a["drafts"][21, 0]] = -np.inf  # drafted against its own distribution
        a["draft"][1, 1, :] = -np.inf
    for temperature in (None, np.full(n, 0.0), np.full(n, 1e-30), np.full(n, 0.05), np.full(n, 50.0), np.full(n, np.inf), rng.uniform(0, 1, n)):
        if temperature is not None:
            a["temperature"] = temperature.astype(np.float32)
        for u in (None, 0.0, 0.5, NEXT):
            b = dict(a) if u is None else {**a, "uniform": np.concatenate([a["uniform"][:, :d], np.full((n, 1), u, np.float32)], 1)}
            _check(torch, b)


@pytest.mark.gpu
def test_what_comes_out_is_the_targets_distribution():
    """Tokens drafted from q, random numbers of one seed: the first token's counts over 40000 sequences against the target's
    probabilities, each within 5 standard deviations (a chance of 6e-7 each to be outside of them)."""
    torch = _gpu()
    from gpu_util import banner
    banner("verify_drafts, counts of 40000 draws")
    rng = np.random.default_rng(12)
    n, vocab = 40000, 7
    p, q = rng.standard_normal(vocab).astype(np.float32), rng.standard_normal(vocab).astype(np.float32)
    a = dict(target=np.broadcast_to(p, (n, 2, vocab)).copy(), draft=np.broadcast_to(q, (n, 1, vocab)).copy(),
             drafts=(q + rng.gumbel(size=(n, 1, vocab))).argmax(2).astype(np.int32), uniform=rng.random((n, 2)).astype(np.float32))
    for with_draft in (True, False):
        if not with_draft:
            del a["draft"]
        tokens, accepted, _, _ = _run(torch, a)
        want = probabilities(p, 1.0)[0]
        count = np.bincount(tokens[:, 0], minlength=vocab)
        assert (np.abs(count - n * want) <= 5 * np.sqrt(n * want * (1 - want))).all(), (count, n * want)
        assert 0 < accepted.sum() < n
