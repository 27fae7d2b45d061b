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
