"""What the decoder's options say is what it does."""
import numpy as np
import pytest

from test_decoder_kv8 import _config, _env

pytestmark = pytest.mark.gpu


def _prompt(torch, cfg, n, seed=1):
    return torch.randint(0, cfg.vocab, (n,), dtype=torch.int32, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def test_head_norms_are_the_configurations():
    """Weights that hold head norms do not switch them on, and a configuration with them does not do without."""
    torch = _env()
    from gpu_util import banner
    from blog_amd.decoder import Qwen2Decoder, make_weights
    plain, normed = _config(qk_norm=False, kv8=True), _config(qk_norm=True, kv8=True)
    w = make_weights(torch, normed, seed=3)
    without = {**w, "layers": [{n: t for n, t in W.items() if n not in ("q_norm", "k_norm")} for W in w["layers"]]}
    prompt = _prompt(torch, plain, 20)
    logits = []
    for cfg, weights in ((plain, w), (plain, without), (normed, w)):
        banner(f"head norms: qk_norm={cfg.qk_norm}")
        dec = Qwen2Decoder(torch, cfg, weights, max_seq=64, max_prompt=32)
        dec.prefill(prompt)
        dec.step()
        logits.append(dec.logits.clone())
    assert torch.equal(logits[0], logits[1]) and not torch.equal(logits[0], logits[2])
    for kv8 in (False, True):
        with pytest.raises(KeyError):
            Qwen2Decoder(torch, _config(qk_norm=True, kv8=kv8), without, max_seq=64, max_prompt=32)


@pytest.mark.parametrize("qk_norm,kv8", [(True, True), (False, True), (True, False)])
@pytest.mark.parametrize("max_seq", [100, 96, 33])
def test_steps_across_the_last_position(qk_norm, kv8, max_seq):
    """Past the last position a step takes it again, with the token's key and value in place of the former ones, in either
    cache, also where max_seq is not a whole number of the 8-bit cache's blocks; captured and replayed alike."""
    torch = _env()
    from gpu_util import banner, host
    from blog_amd import qlin
    from blog_amd.decoder import Qwen2Decoder, make_weights
    from test_decoder_kv8 import Twin, _close
    cfg = _config(qk_norm=qk_norm, kv8=kv8)
    w = make_weights(torch, cfg, seed=7)
    prompt = _prompt(torch, cfg, max_seq - 4 if max_seq < 64 else 64)
    eager, dec = (Qwen2Decoder(torch, cfg, w, max_seq=max_seq, max_prompt=64) for _ in range(2))
    twin = Twin(cfg, w, max_seq)
    n = max_seq + 40 - len(prompt)
    banner(f"across the last position, max_seq={max_seq} qk_norm={qk_norm} kv8={kv8}")
    tokens = _prompt(torch, cfg, n, seed=2)  # (given: picks of their own soon repeat one token there)
    eager.prefill(prompt)
    ref, ids, at = [], host(prompt), 0
    for i in range(n):
        got, want = host(eager.logits), twin.run(ids, at)
        assert _close(got, want), (i, np.linalg.norm(got - want) / np.linalg.norm(want))
        ref.append(eager.logits.clone())
        ids, at = host(tokens[i:i + 1]), min(len(prompt) + i, max_seq - 1)
        for k, v in twin.exact:  # (the position that is taken again)
            del k[at:], v[at:]
        eager.token.copy_(tokens[i:i + 1])
        eager.step()
    dec.prefill(prompt)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dec.step()
    qlin.set_stream(torch.cuda.current_stream())
    for i in range(1, n):
        dec.token.copy_(tokens[i - 1:i])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(dec.logits, ref[i]), i
    assert int(dec.pos.item()) == len(prompt) + n - 1


def test_history_past_the_last_position():
    """The last row of the history is taken again too."""
    torch = _env()
    from gpu_util import banner, host
    from blog_amd.decoder import Qwen2Decoder, make_weights
    cfg = _config(qk_norm=True, kv8=True)
    dec = Qwen2Decoder(torch, cfg, make_weights(torch, cfg, seed=8), max_seq=40, max_prompt=32)
    dec.set_controls(presence=1.0, frequency=0.3)
    prompt = _prompt(torch, cfg, 30)
    banner("history past the last position")
    tokens = dec.generate(prompt, 20)
    seen = host(prompt).tolist() + tokens[:-1]
    assert host(dec.history)[0].tolist() == seen[:39] + seen[-1:]


def test_controls_that_are_replaced_while_a_step_waits():
    """A step on another stream than the controls' own reads those it was launched with, also where they are replaced, and
    their memory asked for again, before it runs."""
    torch = _env()
    from gpu_util import banner
    from blog_amd import qlin
    from blog_amd.decoder import Qwen2Decoder, make_weights
    cfg = _config(qk_norm=True, kv8=True)
    w = make_weights(torch, cfg, seed=8)
    prompt = _prompt(torch, cfg, 20)
    words = (cfg.vocab + 31) // 32
    controls = lambda: dict(repetition=1.3, frequency=0.1, presence=0.5, bias={3: 2.0, 9: 1.0},
                            mask=torch.full((1, words), 0x2AAAAAAA, dtype=torch.int32, device="cuda"))
    banner("controls replaced while a step waits")
    side = torch.cuda.Stream()
    results = []
    for replaced in (False, True):
        dec = Qwen2Decoder(torch, cfg, w, max_seq=64, max_prompt=32)
        dec.set_controls(**controls())
        dec.prefill(prompt)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)  # (about 10 ms)
            dec.step()
        if replaced:
            dec.set_controls(repetition=0.9)
            filler = [torch.full((n,), 0x7F7F7F7F, dtype=torch.int32, device="cuda") for n in [1, 1, 1, 2, 2, words] * 8]
        torch.cuda.synchronize()
        results.append((dec.controlled.clone(), dec.token.clone()))
        qlin.set_stream(torch.cuda.current_stream())
    del filler
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])


def test_more_biases_than_a_pick_takes():
    """Refused by set_controls, which then leaves what was set as it was, and not by the step after it."""
    torch = _env()
    from gpu_util import banner
    from blog_amd import qlin
    from blog_amd.decoder import Qwen2Decoder, make_weights
    cfg = _config(vocab=5000)
    dec = Qwen2Decoder(torch, cfg, make_weights(torch, cfg, seed=8), max_seq=64, max_prompt=32)
    dec.set_controls(repetition=1.3)
    banner("as many biases as a pick takes")
    with pytest.raises(ValueError):
        dec.set_controls(bias={t: 1.0 for t in range(qlin.MAX_BIAS + 1)})
    assert dec.controls["repetition"].item() == np.float32(1.3)
    dec.set_controls(bias={t: -100.0 for t in range(qlin.MAX_BIAS)})
    assert all(t >= qlin.MAX_BIAS for t in dec.generate(_prompt(torch, cfg, 5), 4))


def test_steps_without_controls_between():
    """A step captured before there were controls does not count its token; no token of the text before is counted for it."""
    torch = _env()
    from gpu_util import banner, host
    from blog_amd import qlin
    from blog_amd.decoder import Qwen2Decoder, make_weights
    cfg = _config(qk_norm=True, kv8=True)
    dec = Qwen2Decoder(torch, cfg, make_weights(torch, cfg, seed=8), max_seq=64, max_prompt=32)
    dec.prefill(_prompt(torch, cfg, 4))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dec.step()
    qlin.set_stream(torch.cuda.current_stream())
    banner("steps without controls between")
    dec.set_controls(frequency=1.0)
    dec.generate(_prompt(torch, cfg, 20, seed=3), 20)
    prompt = _prompt(torch, cfg, 10, seed=4)
    dec.prefill(prompt)
    for _ in range(5):
        g.replay()
    token = dec.token.clone()
    dec.step()
    torch.cuda.synchronize()
    assert host(dec.history)[0, :16].tolist() == host(prompt).tolist() + 5 * [-1] + host(token).tolist()
    counts = np.bincount(np.append(host(prompt), host(token)), minlength=cfg.vocab).astype(np.float32)
    assert np.array_equal(host(dec.controlled)[0], host(dec.logits) - counts)
