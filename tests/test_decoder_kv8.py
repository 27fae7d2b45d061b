"""The decoder with normed query and key heads, the 8-bit cache and controls on the logits: the operators as one decode
runs them, against a float64 decoder, captured and replayed, on another stream, and with buffers shared by graphs."""
import numpy as np
import pytest

from blog_amd import qlin
from test_kv8 import Cache, _check_attend, _device_cache, _filled, attend, norm_rope, table64
from test_logits_controls import reference

pytestmark = pytest.mark.gpu


def _env():
    import torch
    from gpu_util import bind_stream
    assert torch.cuda.is_available(), "GPU tests need the MI355X"
    bind_stream()
    return torch


def _config(**kw):
    from blog_amd.decoder import Qwen2Config
    return Qwen2Config(**{**dict(layers=2, hidden=256, n_heads=6, kv_heads=2, head_dim=64, ffn=512, vocab=1000, theta=1e5), **kw})


def _bf16(t):
    return (t.cpu().numpy().view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def _q8_0(t, cols):
    b = t.cpu().numpy().reshape(-1, cols // 32, 34)
    d = b[:, :, :2].copy().view(np.float16).astype(np.float64)
    return (b[:, :, 2:].view(np.int8) * d).reshape(-1, cols)


class Twin:
    """The decoder in float64, its cache (8 bits or exact) position by position."""

    def __init__(self, cfg, weights, max_seq):
        self.c = cfg
        self.table = table64(max_seq, cfg.head_dim, cfg.theta).astype(np.float32)
        self.emb = _q8_0(weights["table"], cfg.hidden)
        self.final = _bf16(weights["final_norm"])
        dims = dict(wq=cfg.hidden, wk=cfg.hidden, wv=cfg.hidden, wo=cfg.q_dim, wg=cfg.hidden, wu=cfg.hidden, wd=cfg.ffn)
        self.layers = [{**{n: _q8_0(W[n], k) for n, k in dims.items()},
                        **{n: _bf16(W[n]) for n in W if n.endswith("norm")}} for W in weights["layers"]]
        per = (max_seq + 31) // 32
        self.caches = [Cache(1, per, cfg.kv_heads, cfg.head_dim) for _ in self.layers]
        self.exact = [([], []) for _ in self.layers]

    def rms(self, x, w):
        return x / np.sqrt(np.mean(x * x, -1, keepdims=True) + self.c.eps) * w

    def run(self, tokens, start):
        """Logits of the last of the tokens at positions start .."""
        c, h, n = self.c, self.emb[tokens], len(tokens)
        pos = start + np.arange(n)
        for i, W in enumerate(self.layers):
            x = self.rms(h, W["attn_norm"])
            q = norm_rope((x @ W["wq"].T).reshape(n, c.n_heads, -1), W.get("q_norm"), self.table, pos, c.head_dim, 0, c.eps)
            k = norm_rope((x @ W["wk"].T).reshape(n, c.kv_heads, -1), W.get("k_norm"), self.table, pos, c.head_dim, 0, c.eps)
            v = (x @ W["wv"].T).reshape(n, c.kv_heads, -1)
            if c.kv8:
                self.caches[i].store(0, start, k.astype(np.float32), v.astype(np.float32))
                kk, vv, there = self.caches[i].values(0, start + n)
            else:
                self.exact[i][0].extend(k)
                self.exact[i][1].extend(v)
                kk, vv = np.array(self.exact[i][0]), np.array(self.exact[i][1])
                there = np.ones(len(kk), bool)
            a, _ = attend(q, kk, vv, there, start, c.head_dim ** -0.5)
            h = h + a.reshape(n, -1) @ W["wo"].T
            x = self.rms(h, W["ffn_norm"])
            g = x @ W["wg"].T
            h = h + (g / (1 + np.exp(-g)) * (x @ W["wu"].T)) @ W["wd"].T
        return self.rms(h[-1], self.final) @ self.emb.T


# Logits against the twin, of the largest: the linears' own bound of this repository's decoder tests (1e-3 normwise; their
# activations are held to 2^-17), and in the 8-bit cache keys and values next to a border between two codes: an error of
# 2^-17 moves at most 127 * 2^-16 = 0.2% of the codes, each by 1/127 of its block's largest (about 4 rms), which is
# sqrt(0.002) * 4 / 127 = 1.4e-3 of the attention's output.
BOUND = 1e-3 + 1.4e-3


def _close(got, want):
    return np.linalg.norm(got - want) <= BOUND * np.linalg.norm(want)


@pytest.mark.parametrize("qk_norm,kv8", [(True, True), (False, True), (True, False)])
@pytest.mark.parametrize("prompt", [1, 37, 64])
def test_decoder_against_float64(qk_norm, kv8, prompt):
    torch = _env()
    from gpu_util import banner, host
    from blog_amd.decoder import Qwen2Decoder, make_weights
    cfg = _config(qk_norm=qk_norm, kv8=kv8)
    w = make_weights(torch, cfg, seed=3)
    dec, twin = Qwen2Decoder(torch, cfg, w, max_seq=160, max_prompt=64), Twin(cfg, w, 160)
    ids = np.random.default_rng(prompt).integers(0, cfg.vocab, prompt)
    banner(f"decoder qk_norm={qk_norm} kv8={kv8} prompt={prompt}")
    dec.prefill(torch.tensor(ids, dtype=torch.int32, device="cuda"))
    want = twin.run(ids, 0)
    for step in range(40):
        got = host(dec.logits)
        assert _close(got, want), (step, np.linalg.norm(got - want) / np.linalg.norm(want))
        token = int(host(dec.token)[0])
        assert token == int(np.argmax(got))
        want = twin.run(np.array([token]), prompt + step)
        dec.step()


def test_decoder_controls():
    """Penalties, a bias and a mask that changes from step to step, in the decoder's own loop; off, the pick is the plain one."""
    torch = _env()
    from gpu_util import banner, host
    from blog_amd.decoder import Qwen2Decoder, make_weights
    cfg = _config(qk_norm=True, kv8=True)
    w = make_weights(torch, cfg, seed=4)
    rng = np.random.default_rng(2)
    words = (cfg.vocab + 31) // 32
    mask = torch.zeros(1, words, dtype=torch.int32, device="cuda")
    dec = Qwen2Decoder(torch, cfg, w, max_seq=96, max_prompt=64)
    bias = {5: 3.0, 900: -1.0, 17: 0.5}
    dec.set_controls(repetition=1.3, frequency=0.2, presence=0.4, bias=bias, mask=mask)
    ids = list(rng.integers(0, cfg.vocab, 20))
    banner("decoder controls")
    for step in range(30):
        m = rng.integers(0, 1 << 32, (1, words), dtype=np.uint32)
        mask.copy_(torch.from_numpy(m.view(np.int32)))
        if step == 0:
            dec.prefill(torch.tensor(np.array(ids), dtype=torch.int32, device="cuda"))
        else:
            dec.step()
        f = lambda v: np.array([v], np.float32)
        out, pick = reference(host(dec.logits)[None], cfg.vocab, np.array([ids], np.int32), None, f(1.3), f(0.2), f(0.4),
                              np.array([list(bias)]), np.array([list(bias.values())], np.float32), m)
        assert np.array_equal(host(dec.controlled), out)
        assert int(host(dec.token)[0]) == pick[0]
        ids.append(int(pick[0]))
    with pytest.raises(ValueError):
        dec.set_controls(mask=mask[:, 1:])
    plain = Qwen2Decoder(torch, cfg, w, max_seq=96, max_prompt=64)
    prompt = torch.tensor(np.array(ids[:20]), dtype=torch.int32, device="cuda")
    neutral = Qwen2Decoder(torch, cfg, w, max_seq=96, max_prompt=64)
    neutral.set_controls()
    assert plain.generate(prompt, 12) == neutral.generate(prompt, 12)


@pytest.mark.parametrize("controls", [False, True])
def test_captured_step_replays_as_the_eager_one(controls):
    torch = _env()
    from gpu_util import banner
    from blog_amd.decoder import Qwen2Decoder, make_weights
    cfg = _config(qk_norm=True, kv8=True)
    w = make_weights(torch, cfg, seed=5)
    prompt = torch.randint(0, cfg.vocab, (50,), dtype=torch.int32, device="cuda",
                           generator=torch.Generator(device="cuda").manual_seed(6))
    n = 25
    banner(f"captured decode step, controls={controls}")
    eager, dec = (Qwen2Decoder(torch, cfg, w, max_seq=512, max_prompt=64) for _ in range(2))
    for d in (eager, dec):
        if controls:
            d.set_controls(repetition=1.2, frequency=0.1)
    ref = torch.zeros(n, cfg.vocab, device="cuda")
    tokens = eager.generate(prompt, n, logits_out=ref)
    dec.prefill(prompt)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dec.step()
    qlin.set_stream(torch.cuda.current_stream())
    got = [int(dec.token.item())]
    for i in range(1, n):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(dec.logits, ref[i]), f"step {i}"
        got.append(int(dec.token.item()))
    assert got == tokens


def test_a_graph_keeps_the_controls_it_was_captured_with():
    """A step captured under one set of controls, replayed after others were set (and their memory used again)."""
    torch = _env()
    from gpu_util import banner
    from blog_amd.decoder import Qwen2Decoder, make_weights
    cfg = _config(qk_norm=True, kv8=True)
    w = make_weights(torch, cfg, seed=8)
    prompt = torch.randint(0, cfg.vocab, (20,), dtype=torch.int32, device="cuda",
                           generator=torch.Generator(device="cuda").manual_seed(9))
    banner("controls of a captured step")
    words = (cfg.vocab + 31) // 32
    odd = lambda: torch.full((1, words), 0x2AAAAAAA, dtype=torch.int32, device="cuda")  # odd tokens, but for the words' last
    eager, dec = (Qwen2Decoder(torch, cfg, w, max_seq=64, max_prompt=32) for _ in range(2))
    for d in (eager, dec):
        d.set_controls(repetition=1.3, presence=0.5, bias={3: 2.0, 9: 1.0}, mask=odd())
    tokens = eager.generate(prompt, 12)
    assert all(t % 2 == 1 for t in tokens)
    dec.prefill(prompt)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dec.step()
    qlin.set_stream(torch.cuda.current_stream())
    dec.set_controls(repetition=0.9)
    filler = [torch.full((n,), 0x7F7F7F7F, dtype=torch.int32, device="cuda") for n in [1, 1, 1, 2, 2, words] * 8]
    got = [int(dec.token.item())]
    for _ in range(11):
        g.replay()
        torch.cuda.synchronize()
        got.append(int(dec.token.item()))
    assert got == tokens
    del filler
    for bad in (dict(repetition=0.0), dict(repetition=-1.0), dict(mask=odd().cpu()), dict(mask=odd().long()), dict(mask=odd()[:, 1:])):
        with pytest.raises(ValueError):
            dec.set_controls(**bad)


@pytest.mark.parametrize("kv8", [False, True])
def test_steps_past_the_last_position(kv8):
    """As without controls: the last position is taken again."""
    torch = _env()
    from gpu_util import banner
    from blog_amd.decoder import Qwen2Decoder, make_weights
    cfg = _config(qk_norm=True, kv8=kv8)
    w = make_weights(torch, cfg, seed=8)
    banner(f"steps past the last position, kv8={kv8}")
    dec = Qwen2Decoder(torch, cfg, w, max_seq=32, max_prompt=32)
    dec.set_controls(frequency=0.2)
    tokens = dec.generate(torch.arange(30, dtype=torch.int32, device="cuda"), 8)
    assert all(0 <= t < cfg.vocab for t in tokens) and int(dec.pos.item()) == 37
    assert torch.isfinite(dec.logits).all()


def test_graphs_that_share_a_workspace():
    """Two captured attentions (one row over a long cache, many rows) and a captured pick that share one workspace, replayed in
    turns between eager calls that use it too: bit for bit the eager results, whatever the workspace held."""
    torch = _env()
    from gpu_util import banner, dev
    rng = np.random.default_rng(1)
    heads, kv, d, per = 8, 2, 128, 200
    ref = _filled(rng, 1, per, kv, d)
    cache = _device_cache(torch, ref, paged=False)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    calls = []
    for rows, start in ((1, 6000), (70, 3000), (3, 40)):
        calls.append((dev(rng.standard_normal((1, rows, heads, d)).astype(np.float32)), rows, i32([start])))
    logits = torch.randn(2, 50000, device="cuda")
    need = max([qlin.attend_kv8_workspace_bytes(1, r, heads, kv, d, per) for _, r, _ in calls]
               + [qlin.logits_controls_scratch_bytes(2, 50000)])
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    outs = [torch.empty_like(q) for q, _, _ in calls]
    picked, pick = torch.empty_like(logits), torch.zeros(2, dtype=torch.int32, device="cuda")

    def run(i):
        if i < len(calls):
            q, rows, start = calls[i]
            qlin.attend_kv8(cache, q, outs[i], rows, heads, start, None, d ** -0.5, ws)
        else:
            qlin.logits_controls(logits, picked, 2, 50000, picks=pick, scratch=ws)
    banner("graphs that share a workspace")
    want, graphs = [], []
    results = lambda i: [outs[i]] if i < len(calls) else [picked, pick]
    for i in range(4):
        run(i)
        torch.cuda.synchronize()
        want.append([r.clone() for r in results(i)])
    for i in range(4):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            qlin.set_stream(torch.cuda.current_stream())
            run(i)
        graphs.append(g)
    qlin.set_stream(torch.cuda.current_stream())
    for turn in range(4):
        for i in np.random.default_rng(turn).permutation(4):
            for r in results(i):
                r.zero_()
            ws.fill_(255 if turn % 2 else 0)
            run((i + 1) % 4)
            graphs[i].replay()
            torch.cuda.synchronize()
            for a, b in zip(results(i), want[i]):
                assert torch.equal(a, b), (turn, i)


def test_another_stream_and_two_caches_at_once():
    """Calls on two streams, each with its own cache, outputs and workspace, that run at the same time."""
    torch = _env()
    from gpu_util import banner, dev
    rng = np.random.default_rng(11)
    heads, kv, d, per = 6, 2, 64, 120
    banner("two streams")
    sets = []
    for i in range(2):
        ref = _filled(rng, 1, per, kv, d)
        q = rng.standard_normal((1, 2, heads, d)).astype(np.float32)
        need = qlin.attend_kv8_workspace_bytes(1, 2, heads, kv, d, per)
        sets.append((ref, _device_cache(torch, ref, False), q, dev(q), torch.zeros(1, 2, heads, d, device="cuda"),
                     torch.empty(need, dtype=torch.uint8, device="cuda"), torch.tensor([3700 - i], dtype=torch.int32, device="cuda")))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for s, (ref, cache, q, qd, out, ws, start) in zip(streams, sets):
            qlin.set_stream(s)
            qlin.attend_kv8(cache, qd, out, 2, heads, start, None, 0.125, ws)
    torch.cuda.synchronize()
    qlin.set_stream(torch.cuda.current_stream())
    for i, (ref, cache, q, qd, out, ws, start) in enumerate(sets):
        want = out.clone()
        _check_attend(torch, ref, cache, q, [3700 - i], None, heads, 0.125)
        qlin.attend_kv8(cache, qd, out, 2, heads, start, None, 0.125, ws)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
