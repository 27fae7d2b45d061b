"""A row of a step by drafts is the model's answer to the tokens up to it, whatever drafts follow: over the 8-bit cache too, where
the drafts complete a block."""
import numpy as np
import pytest

from blog_amd import qlin
from test_decoder_kv8 import _close, _config, _env
from test_serving_step import Rows

pytestmark = pytest.mark.gpu


def _start(torch, n, prompt, *, qk_norm, kv8, max_seq=128, seed=9):
    from blog_amd.decoder import Qwen2Decoder, make_weights
    cfg = _config(qk_norm=qk_norm, kv8=kv8, vocab=200)
    w = make_weights(torch, cfg, seed=seed)
    dec, twin = Qwen2Decoder(torch, cfg, w, max_seq=max_seq, max_prompt=64), Rows(cfg, w, max_seq)
    rng = np.random.default_rng(prompt)
    ids = rng.integers(0, cfg.vocab, prompt)
    for part in range(0, prompt, 48):  # (a prompt, then tokens)
        if part == 0:
            dec.prefill(torch.tensor(ids[:48], dtype=torch.int32, device="cuda"))
            twin.run(ids[:48], 0)
        else:
            for i in range(part, min(prompt, part + 48)):
                dec.token.fill_(int(ids[i]))
                dec.step()
                twin.run(ids[i:i + 1], i)
    return cfg, dec, twin, dec.drafts(n), rng


def _fill(torch, d, drafts, most, uniform=0.5):
    d["drafts"].copy_(torch.tensor(np.array([drafts]), dtype=torch.int32))
    d["uniform"].fill_(uniform)
    d["n_drafts"].fill_(most)


@pytest.mark.parametrize("qk_norm,kv8", [(True, True), (False, True), (True, False), (False, False)])
@pytest.mark.parametrize("prompt,n", [(27, 5), (31, 5), (32, 5), (58, 5), (61, 5), (62, 1), (63, 5), (63, 0), (64, 5), (40, 31), (32, 31), (33, 31)])
def test_rows_are_those_of_single_steps(qk_norm, kv8, prompt, n):
    """Every row's logits against the float64 decoder that takes the tokens one after the other; then a step after the last
    accepted one, over what the rejected ones left behind."""
    torch = _env()
    from gpu_util import banner, host
    banner(f"rows of drafts: qk_norm={qk_norm} kv8={kv8} prompt={prompt} n={n}")
    cfg, dec, twin, d, rng = _start(torch, n, prompt, qk_norm=qk_norm, kv8=kv8)
    token = int(host(dec.token)[0])
    rows, own, drafts = [], token, []
    for i in range(n + 1):
        rows.append(twin.run(np.array([own]), prompt + i)[0])
        own = int(np.argmax(rows[-1])) if i % 4 < 2 else int(rng.integers(0, cfg.vocab))
        drafts.append(own)
    _fill(torch, d, drafts[:n], n)
    dec.step_drafts(d)
    logits = host(d["logits"])
    for i in range(n + 1):
        assert _close(logits[0, i], rows[i]), (i, np.linalg.norm(logits[0, i] - rows[i]) / np.linalg.norm(rows[i]))
    m = int(host(d["accepted"])[0])
    token = int(host(dec.token)[0])
    assert int(host(dec.pos)[0]) == prompt + m + 1 and token == int(host(d["tokens"])[0, m])
    twin.back(prompt + m + 1)
    want = twin.run(np.array([token]), prompt + m + 1)[0]
    dec.step()
    assert _close(host(dec.logits), want)


# Rows of one call that differ in later rows' tokens only: the same products in the same order, but for the power of two that a
# tile's rows take their probabilities by, which other rows of the tile can move.  A probability is then rounded to 22 bits elsewhere
# (2^-22 of it), and sums of up to 96 of them are f32 sums (96 half steps of 2^-24 at most): 2^-17 of an attention's output.
# Two layers, whose linears and norms pass a relative error on at most about fourfold.
SAME = 4 * 2 * 2.0 ** -17


@pytest.mark.parametrize("kv8", [True, False])
@pytest.mark.parametrize("prompt,n", [(59, 5), (62, 5), (30, 5), (40, 31), (63, 3)])
def test_rows_do_not_depend_on_later_drafts(kv8, prompt, n):
    """The same positions taken again with other drafts after row i, also past n_drafts: the rows up to i, what is accepted of them
    and their rates are as before."""
    torch = _env()
    from gpu_util import banner, host
    banner(f"later drafts: kv8={kv8} prompt={prompt} n={n}")
    cfg, dec, _, d, rng = _start(torch, n, prompt, qk_norm=True, kv8=kv8)
    d["temperature"].fill_(0.7)
    token, pos = dec.token.clone(), dec.pos.clone()
    drafts = rng.integers(0, cfg.vocab, n)
    _fill(torch, d, drafts, n)
    dec.step_drafts(d)
    first, rates = host(d["logits"]).copy(), host(d["rates"]).copy()
    for i in sorted({0, 1, n // 2, n - 1}):
        for junk in (int(rng.integers(0, cfg.vocab)), -7):
            other = drafts.copy()
            other[i:] = junk
            dec.token.copy_(token), dec.pos.copy_(pos)
            _fill(torch, d, other, i)
            dec.step_drafts(d)
            got = host(d["logits"])
            for r in range(i + 1):
                assert np.linalg.norm(got[0, r] - first[0, r]) <= SAME * np.linalg.norm(first[0, r]), (i, r, junk)
            # (by lookup a rate is a probability: a logit and the sum's logarithm, each off by SAME times the row's norm at most)
            off = 2 * SAME * np.linalg.norm(first[0], axis=1).max() / 0.7
            assert np.allclose(host(d["rates"])[0, :i], rates[0, :i], rtol=2 * off, atol=0) and (host(d["rates"])[0, i:] == 0).all()
