"""Adapters and drafts that are set up on a stream with work of its own, and used on another one at once."""
import numpy as np
import pytest

from blog_amd import qlin
from test_decoder_kv8 import _config, _env

pytestmark = pytest.mark.gpu


def _busy(torch):
    """Some milliseconds of work on the current stream."""
    a = torch.randn(4096, 4096, device="cuda")
    for _ in range(20):
        a = a @ a
        a /= a.norm()
    return a


def _loras(torch, cfg, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: 0.2 * torch.randn(*s, device="cuda", generator=g)
    dims = {"wq": (cfg.hidden, cfg.q_dim), "wo": (cfg.q_dim, cfg.hidden), "wd": (cfg.ffn, cfg.hidden)}
    return [{n: qlin.Lora(r(3, 8, i), r(3, o, 8)) for n, (i, o) in dims.items()} for _ in range(cfg.layers)]


def test_set_up_on_another_stream():
    torch = _env()
    from gpu_util import banner
    from blog_amd.decoder import Qwen2Decoder, make_weights
    cfg = _config(vocab=200)
    w = make_weights(torch, cfg, seed=5)
    layers = _loras(torch, cfg, 1)
    prompt = torch.arange(20, dtype=torch.int32, device="cuda")
    fixed = torch.tensor([[3, 5, 7]], dtype=torch.int32, device="cuda")

    def use(dec, d):
        dec.prefill(prompt)
        first = dec.logits.clone()
        d["drafts"].copy_(fixed)
        d["uniform"].fill_(0.5)
        dec.step_drafts(d)
        return [first, d["logits"].clone(), d["tokens"].clone(), d["logprobs"].clone(), d["rates"].clone()]
    want = {}
    for slot in (0, 2):
        banner(f"adapters of slot {slot}, one stream")
        dec = Qwen2Decoder(torch, cfg, w, max_seq=64, max_prompt=32)
        dec.set_adapters(layers, slot)
        want[slot] = use(dec, dec.drafts(3))
    assert not torch.equal(want[0][0], want[2][0])
    dec = Qwen2Decoder(torch, cfg, w, max_seq=64, max_prompt=32)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for turn in range(6):
        banner(f"adapters set up on another stream, turn {turn}")
        slot = 2 * (turn % 2)
        with torch.cuda.stream(a):
            junk = torch.full((1 << 20,), 7, dtype=torch.int32, device="cuda")  # (memory that the stream still writes when it is free again)
            held = _busy(torch)
            junk.fill_(-3)
            del junk
            dec.set_adapters(layers, slot)
            d = dec.drafts(3)
        with torch.cuda.stream(b):
            got = use(dec, d)
        torch.cuda.synchronize()
        for x, y in zip(got, want[slot]):
            assert torch.equal(x, y), turn
        del held
    qlin.set_stream(torch.cuda.current_stream())


def test_adapters_workspace(monkeypatch):
    """Enough for every number of rows and linear, asked for once for layers that are alike."""
    torch = _env()
    from gpu_util import banner
    from blog_amd.decoder import Qwen2Decoder, make_weights
    banner("the adapters' workspace")
    cfg = _config(vocab=200, layers=6)
    dec = Qwen2Decoder(torch, cfg, make_weights(torch, cfg, seed=5), max_seq=96, max_prompt=80)
    layers = _loras(torch, cfg, 1)
    layers[3] = {"wq": layers[3]["wq"], "wv": qlin.Lora(torch.zeros(3, 8, cfg.hidden, device="cuda"), torch.zeros(3, cfg.kv_dim, 8, device="cuda"))}
    asked, real = [], qlin.lora_workspace_bytes
    monkeypatch.setattr(qlin, "lora_workspace_bytes", lambda *a: asked.append(a) or real(*a))
    dec.set_adapters(layers, 1)
    forms = {(len(ws), ws[0].like) for L in layers for names in dec.LINEARS if (ws := [L[n] for n in names if n in L])}
    want = max(real(rows, n, *like[1:]) for n, like in forms for rows in range(1, 81))
    assert len(forms) == 4 and dec.adapters["ws"].numel() == want and len(asked) <= len(forms) * 80
