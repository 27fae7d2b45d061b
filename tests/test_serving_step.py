"""A server's step for many requests at once, as the operators are used one after the other: the residual's addition and the norm
into Q8_1 blocks, a product of these with adapters beside it, routing into the experts' products, the head and the check of drafted
tokens; captured and replayed, on another stream, with one workspace; and the decoder with adapters and drafts."""
import numpy as np
import pytest

import oracle as orc
import qgen
from blog_amd import qlin
from qgen import Q4_K, Q5_0, Q8_0
from test_add_rms_norm import HALF_STEP
from test_add_rms_norm import reference as norm_reference
from test_decoder_kv8 import Twin, _close, _config, _env
from test_moe_route import reference as route_reference
from test_verify_drafts import reference as verify_reference

pytestmark = pytest.mark.gpu

SEQS, DRAFTS, HIDDEN, OUT, VOCAB, E, FFN, K = 5, 2, 512, 300, 1200, 32, 256, 4
ROWS = SEQS * (DRAFTS + 1)


class Step:
    """The buffers and calls of one step."""

    def __init__(self, torch, seed=0):
        from gpu_util import dev
        self.torch = torch
        rng = np.random.default_rng(seed)
        f = lambda *s: rng.standard_normal(s).astype(np.float32)
        self.n = n = dict(x=f(ROWS, HIDDEN), delta=f(ROWS, HIDDEN), norm=(1 + 0.2 * f(HIDDEN)), bias=0.1 * f(E), router=f(HIDDEN, E) / 16,
                          uniform=rng.random((SEQS, DRAFTS + 1)).astype(np.float32), temperature=rng.uniform(0.5, 1.2, SEQS).astype(np.float32),
                          drafts=rng.integers(0, VOCAB, (SEQS, DRAFTS)).astype(np.int32), ids=rng.integers(-1, 3, ROWS).astype(np.int32))
        n["temperature"][1] = 0
        self.w, self.rb, _ = qgen.random_matrix(Q8_0, OUT, HIDDEN, seed=1)
        self.head, self.head_rb, _ = qgen.random_matrix(Q8_0, VOCAB, HIDDEN, seed=2)
        self.experts = [qgen.random_matrix(t, E * r, c, seed=3 + i)[0] for i, (t, r, c) in enumerate(((Q4_K, FFN, HIDDEN), (Q4_K, FFN, HIDDEN), (Q5_0, HIDDEN, FFN)))]
        self.d = {k: dev(v) for k, v in n.items()}
        self.d["norm"] = self.d["norm"].bfloat16()
        self.dw, self.dhead, self.dexperts = dev(self.w), dev(self.head), [dev(e) for e in self.experts]
        g = torch.Generator().manual_seed(seed)
        self.a = (torch.randn(3, 16, HIDDEN, generator=g) * HIDDEN ** -0.5).bfloat16()
        self.b = (0.3 * torch.randn(3, OUT, 16, generator=g)).bfloat16()
        self.ranks = torch.tensor([16, 5, 9], dtype=torch.int32)
        self.lora = qlin.Lora(self.a.cuda(), self.b.cuda())
        self.dranks = self.ranks.cuda()
        z = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device="cuda")
        i32 = torch.int32
        self.normed, self.blocks, self.y = z(ROWS, HIDDEN), z(qlin.q8_1_bytes(HIDDEN, ROWS), t=torch.uint8), z(ROWS, OUT)
        self.sum, self.experts_out, self.rlogits = z(ROWS, HIDDEN), z(ROWS, HIDDEN), z(ROWS, E)
        self.picks, self.weights, self.logits = z(ROWS, K, t=i32), z(ROWS, K), z(SEQS, DRAFTS + 1, VOCAB)
        self.tokens, self.accepted = z(SEQS, DRAFTS + 1, t=i32), z(SEQS, t=i32)
        self.logprobs, self.rates = z(SEQS, DRAFTS + 1), z(SEQS, DRAFTS)
        self.how = qlin.MoeRouting(sigmoid=True, bias=self.d["bias"], n_groups=4, top_groups=2, group_pairs=True, renormalise=True, scaling=1.5)
        self.moe_bytes = qlin.lib().qlin_moe_grouped_workspace_bytes(ROWS, K, E, FFN, HIDDEN)
        need = max(self.moe_bytes, qlin.lora_workspace_bytes(ROWS, 1, 3, 16, HIDDEN), qlin.verify_drafts_workspace_bytes(SEQS, DRAFTS, VOCAB))
        self.ws = torch.full((need + 512,), 0xFF, dtype=torch.uint8, device="cuda")  # one for all, of any contents
        self.ws = self.ws[-self.ws.data_ptr() % 256:]
        self.results = [self.sum, self.normed, self.blocks, self.y, self.picks, self.weights, self.experts_out, self.logits, self.tokens,
                        self.accepted, self.logprobs, self.rates]

    def run(self):
        torch, d = self.torch, self.d
        qlin.set_stream(torch.cuda.current_stream())
        qlin.add_rms_norm(d["x"], d["delta"], self.sum, d["norm"], 0, 1e-6, 0, normed=self.normed, q8_1=self.blocks)
        qlin.quant_matmul_q8_1(Q8_0, self.dw, self.rb, self.blocks, self.y, OUT, HIDDEN, ROWS)
        qlin.lora_add(self.normed, d["ids"], [(self.lora, self.y, self.y)], ranks=self.dranks, workspace=self.ws)
        torch.mm(self.normed, d["router"], out=self.rlogits)
        qlin.moe_route(self.how, self.rlogits, self.picks, self.weights)
        self.experts_out.copy_(self.sum)
        gate, up, down = self.dexperts
        qlin.call("qlin_moe_routed_decode_grouped", Q4_K, gate, up, gate.numel(), Q5_0, down, down.numel(), E, FFN, HIDDEN, HIDDEN, self.normed,
                  self.picks, self.weights, self.ws.data_ptr(), self.moe_bytes, self.experts_out, ROWS, K)
        qlin.quant_matmul(Q8_0, self.dhead, self.head_rb, self.experts_out, self.logits, VOCAB, HIDDEN, ROWS)
        qlin.verify_drafts(self.logits, d["drafts"], d["uniform"], self.tokens, self.accepted, temperature=d["temperature"],
                           logprobs=self.logprobs, rates=self.rates, workspace=self.ws)


def test_step_of_a_batch():
    torch = _env()
    from gpu_util import banner, dev, host
    banner("a server's step")
    s = Step(torch)
    s.run()
    n = s.n
    total = n["x"] + n["delta"]
    assert np.array_equal(host(s.sum), total)
    gain = s.d["norm"].double().cpu().numpy()
    want = norm_reference(total, gain, 1e-6, HIDDEN)
    normed = host(s.normed)
    assert (np.abs(normed - want) <= HALF_STEP * np.abs(want)).all()
    # the product of the blocks (f64 in the oracle), and the adapters' of the normed rows
    y = orc.matmul_q8_1(Q8_0, s.w, s.rb, host(s.blocks), OUT, HIDDEN, ROWS)
    for a in range(3):
        r, k = n["ids"] == a, int(s.ranks[a])
        y[r] += normed[r].astype(np.float64) @ s.a[a, :k].double().numpy().T @ s.b[a, :, :k].double().numpy().T
    assert qgen.normwise_rel_err(host(s.y), y) <= 1e-4
    picks, weights = route_reference(host(s.rlogits), K, sigmoid=True, bias=n["bias"], n_groups=4, top_groups=2, group_pairs=True, renormalise=True,
                                     scaling=1.5)
    assert np.array_equal(host(s.picks), picks) and (np.abs(host(s.weights) - weights) <= 2.0 ** -22 * weights).all()
    # the experts, a token at a time
    out = dev(total)
    act = torch.zeros(K * FFN, device="cuda")
    gate, up, down = s.dexperts
    for t in range(ROWS):
        qlin.call("qlin_moe_routed_decode_indexed", Q4_K, gate, up, gate.numel(), Q5_0, down, down.numel(), E, FFN, HIDDEN, HIDDEN, s.normed[t],
                  s.picks[t], s.weights[t], act, out[t], K)
    assert qgen.normwise_rel_err(host(s.experts_out), host(out)) <= 1e-5
    logits = host(s.logits)
    assert qgen.normwise_rel_err(logits.reshape(ROWS, VOCAB), orc.matmul_f64(Q8_0, s.head, s.head_rb, host(s.experts_out), VOCAB, HIDDEN)) <= 1e-3
    tokens, accepted, logprobs, rates = verify_reference(logits, n["drafts"], n["uniform"], temperature=n["temperature"])
    assert np.array_equal(host(s.tokens), tokens) and np.array_equal(host(s.accepted), accepted)
    assert np.abs(host(s.logprobs) - logprobs).max() <= 1e-5 and np.abs(host(s.rates) - rates).max() <= 1e-6


def test_captured_steps_of_two_graphs():
    """Two steps captured into graphs of their own, which share nothing but the allocator; replays between eager steps and on
    another stream give what the eager step gave, and nothing is allocated."""
    torch = _env()
    from gpu_util import banner
    steps = [Step(torch, seed) for seed in (0, 7)]
    steps[1].ws = steps[0].ws  # (replayed one after the other)
    want = []
    for i, s in enumerate(steps):
        banner(f"step {i}, eager")
        s.run()
        torch.cuda.synchronize()
        want.append([r.clone() for r in s.results])
    graphs = []
    for i, s in enumerate(steps):
        banner(f"step {i}, captured")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.run()
        graphs.append(g)
    qlin.set_stream(torch.cuda.current_stream())
    other = torch.cuda.Stream()
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    free = lambda: torch.cuda.mem_get_info()[0] + torch.cuda.memory_reserved()
    before = None
    for turn in range(8):
        for i, s in enumerate(steps):
            for r in s.results:
                r.fill_(3)
            if turn % 2:
                with torch.cuda.stream(other):
                    other.wait_stream(torch.cuda.default_stream())
                    s.run() if turn % 4 == 3 else graphs[i].replay()
                torch.cuda.default_stream().wait_stream(other)
            else:
                graphs[i].replay()
            torch.cuda.synchronize()
            for r, w in zip(s.results, want[i]):
                assert torch.equal(r, w), (turn, i)
            qlin.set_stream(torch.cuda.current_stream())
            s.run()
        torch.cuda.synchronize()
        if turn == 3:  # (torch's product allots its own workspace when it first meets a stream)
            before = free()
    assert free() >= before


# ---- the decoder -------------------------------------------------------------------------------

def _adapters(torch, cfg, slots, rank, seed, names=("wq", "wk", "wv", "wo", "wd")):
    g = torch.Generator().manual_seed(seed)
    dims = {"wq": (cfg.hidden, cfg.q_dim), "wk": (cfg.hidden, cfg.kv_dim), "wv": (cfg.hidden, cfg.kv_dim), "wo": (cfg.q_dim, cfg.hidden),
            "wd": (cfg.ffn, cfg.hidden)}
    return [{n: ((torch.randn(slots, rank, dims[n][0], generator=g) * dims[n][0] ** -0.5).bfloat16(),
                 (0.1 * torch.randn(slots, dims[n][1], rank, generator=g)).bfloat16()) for n in names} for _ in range(cfg.layers)]


@pytest.mark.parametrize("qk_norm,kv8", [(False, False), (True, True)])
@pytest.mark.parametrize("names", [("wq", "wk", "wv", "wo", "wd"), ("wv", "wd")])
def test_decoder_with_adapters(qk_norm, kv8, names):
    """Against the float64 decoder with each adapter's product in the weights; the slot rewritten between replays."""
    torch = _env()
    from gpu_util import banner, host
    from blog_amd.decoder import Qwen2Decoder, make_weights
    cfg = _config(qk_norm=qk_norm, kv8=kv8)
    w = make_weights(torch, cfg, seed=5)
    dec = Qwen2Decoder(torch, cfg, w, max_seq=96, max_prompt=32)
    made = _adapters(torch, cfg, 3, 8, 6, names)
    slot = torch.zeros(1, dtype=torch.int32, device="cuda")
    scales = torch.tensor([1.0, 0.5, 2.0], device="cuda")
    dec.set_adapters([{n: qlin.Lora(a.cuda(), b.cuda()) for n, (a, b) in L.items()} for L in made], slot, scales=scales)
    prompt = np.random.default_rng(1).integers(0, cfg.vocab, 21)
    graph = None
    outs = {}
    for use in (1, -1, 2, 1):
        banner(f"decoder with adapters {names}, slot {use}")
        twin = Twin(cfg, w, 96)
        if use >= 0:
            for L, W in zip(made, twin.layers):
                for n, (a, b) in L.items():
                    W[n] = W[n] + float(scales[use]) * (b[use].double().numpy() @ a[use].double().numpy())
        slot.fill_(use)
        dec.prefill(torch.tensor(prompt, dtype=torch.int32, device="cuda"))
        want, seen = twin.run(prompt, 0), []
        for step in range(6):
            got = host(dec.logits)
            assert _close(got, want), (use, step, np.linalg.norm(got - want) / np.linalg.norm(want))
            seen.append(got)
            token = int(host(dec.token)[0])
            want = twin.run(np.array([token]), len(prompt) + step)
            if graph is None:
                torch.cuda.synchronize()
                state = [t.clone() for t in (dec.token, dec.pos)]
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    dec.step()
                qlin.set_stream(torch.cuda.current_stream())
                dec.token.copy_(state[0]), dec.pos.copy_(state[1])
            graph.replay() if step % 2 else dec.step()
        if use in outs:
            assert all(np.array_equal(a, b) for a, b in zip(outs[use], seen))
        outs[use] = seen
    plain = Qwen2Decoder(torch, cfg, w, max_seq=96, max_prompt=32)
    plain.prefill(torch.tensor(prompt, dtype=torch.int32, device="cuda"))
    dec.set_adapters(None, 0)
    dec.prefill(torch.tensor(prompt, dtype=torch.int32, device="cuda"))
    assert torch.equal(plain.logits, dec.logits)


def test_decoder_refuses_adapters():
    torch = _env()
    from blog_amd.decoder import Qwen2Decoder, make_weights
    cfg = _config()
    dec = Qwen2Decoder(torch, cfg, make_weights(torch, cfg, seed=5), max_seq=64, max_prompt=8)
    make = lambda rank, n_in, out: qlin.Lora(torch.zeros(2, rank, n_in, device="cuda"), torch.zeros(2, out, rank, device="cuda"))
    good = {"wq": make(8, cfg.hidden, cfg.q_dim)}
    for layers in ([good], [good, {"wg": make(8, cfg.hidden, cfg.ffn)}], [good, {"wo": make(8, cfg.hidden, cfg.q_dim)}],
                   [good, {**good, "wk": make(16, cfg.hidden, cfg.kv_dim)}]):
        with pytest.raises(ValueError):
            dec.set_adapters(layers, 0)
    with pytest.raises(ValueError):
        dec.set_adapters([good, good], torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        dec.drafts(8)
    assert dec.adapters is None
    dec.set_controls(presence=1.0)
    with pytest.raises(ValueError):
        dec.step_drafts(dec.drafts(2))


class Rows(Twin):
    """The float64 decoder with the logits of all rows of a call."""

    def rms(self, x, w):
        return super().rms(x.base if w is self.final else x, w)  # (its last row is a view of all)

    def back(self, pos):
        for k, v in self.exact:
            del k[pos:], v[pos:]


@pytest.mark.parametrize("qk_norm,kv8", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("with_logits", [False, True])
def test_decoder_by_drafts(qk_norm, kv8, with_logits):
    """Each row's logits against the float64 decoder, tokens and counts as the formula has them from those logits, positions taken
    back after each rejection, greedy and not; captured and replayed alike."""
    torch = _env()
    from gpu_util import banner, host
    from blog_amd.decoder import Qwen2Decoder, make_weights
    cfg = _config(qk_norm=qk_norm, kv8=kv8, vocab=200)
    w = make_weights(torch, cfg, seed=9)
    dec, again, twin = (Qwen2Decoder(torch, cfg, w, max_seq=192, max_prompt=48) for _ in range(2)), None, Rows(cfg, w, 192)
    dec, again = dec
    rng = np.random.default_rng(3)
    prompt = rng.integers(0, cfg.vocab, 40)
    ids = torch.tensor(prompt, dtype=torch.int32, device="cuda")
    n = 5
    d, e = dec.drafts(n), again.drafts(n)
    draft_logits = torch.zeros(1, n, cfg.vocab, device="cuda") if with_logits else None
    dec.prefill(ids), again.prefill(ids)
    torch.cuda.synchronize()
    state = [t.clone() for t in (again.token, again.pos)]
    again.step_drafts(e, draft_logits)  # (the first call of its kernels, outside of the capture)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        again.step_drafts(e, draft_logits)
    qlin.set_stream(torch.cuda.current_stream())
    again.token.copy_(state[0]), again.pos.copy_(state[1])
    twin.run(prompt, 0)
    pos, token, taken = len(prompt), int(host(dec.token)[0]), []
    for call in range(9):
        banner(f"drafts, call {call}, qk_norm={qk_norm} kv8={kv8} logits={with_logits}")
        # what the float64 decoder would say, with a few other tokens among them
        guess, at, own, rows = [], pos, token, []
        most = [n, 0, n, 3, n, n, 1, n, n][call]
        for i in range(n + 1):
            rows.append(twin.run(np.array([own]), at)[0])
            at += 1
            if i < n:
                own = int(np.argmax(rows[-1])) if rng.random() < 0.8 else int(rng.integers(0, cfg.vocab))
                guess.append(own)
        # (in one call, as the 8-bit cache reads a block that the drafts complete in codes, for all of them)
        near = np.array(rows[:n])
        twin.back(pos)
        rows = twin.run(np.array([token] + guess), pos)
        d["drafts"].copy_(torch.tensor([guess], dtype=torch.int32))
        d["uniform"].copy_(torch.tensor(rng.random((1, n + 1)), dtype=torch.float32))
        d["temperature"].fill_(0.0 if call < 5 else 0.02)
        d["n_drafts"].fill_(most)
        if with_logits:
            draft_logits.copy_(torch.tensor(near + 0.02 * rng.standard_normal((n, cfg.vocab)), dtype=torch.float32)[None])
        for name in ("drafts", "uniform", "temperature", "n_drafts"):
            e[name].copy_(d[name])
        dec.step_drafts(d, draft_logits)
        g.replay()
        logits = host(d["logits"])
        for i in range(n + 1):
            assert _close(logits[0, i], rows[i]), (call, i)
        want = verify_reference(logits, np.array([guess]), host(d["uniform"]), None if draft_logits is None else host(draft_logits),
                                host(d["n_drafts"]), host(d["temperature"]))
        m = int(want[1][0])
        assert np.array_equal(host(d["tokens"]), want[0]) and int(host(d["accepted"])[0]) == m
        taken.append(m)
        pos, token = pos + m + 1, int(want[0][0, m])
        assert int(host(dec.token)[0]) == token and int(host(dec.pos)[0]) == pos
        for a, b in ((dec.token, again.token), (dec.pos, again.pos), *((d[k], e[k]) for k in ("tokens", "logits", "logprobs", "rates"))):
            assert torch.equal(a, b)
        twin.back(pos)
    assert max(taken) >= 2 and min(taken) < n
    want = twin.run(np.array([token]), pos)[0]
    dec.step()
    assert _close(host(dec.logits), want)
