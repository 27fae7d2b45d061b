"""The logits' controls refuse tensors whose values would be read as others, or past their end."""
import pytest
import torch

from blog_amd import qlin

ROWS, VOCAB = 3, 64


def _tensors(rows=ROWS, device="cpu"):
    i32 = dict(dtype=torch.int32, device=device)
    f32 = dict(dtype=torch.float32, device=device)
    return dict(logits=torch.zeros(rows, VOCAB, **f32), out=torch.zeros(rows, VOCAB, **f32), history=torch.zeros(rows, 5, **i32),
                history_lens=torch.zeros(rows, **i32), repetition=torch.ones(rows, **f32), frequency=torch.zeros(rows, **f32),
                presence=torch.zeros(rows, **f32), bias_ids=torch.zeros(rows, 4, **i32), bias_values=torch.zeros(rows, 4, **f32),
                mask=torch.zeros(rows, 2, **i32), picks=torch.zeros(rows, **i32))


def _refused(**kw):
    with pytest.raises(ValueError):
        qlin.logits_controls(**{**_tensors(), **dict(rows=ROWS, vocab=VOCAB), **kw})


@pytest.mark.parametrize("name", list(_tensors()))
def test_other_types(name):
    t = _tensors()[name]
    for dtype in (torch.int64, torch.float64, torch.int16, torch.float16, torch.float32 if t.dtype is torch.int32 else torch.int32):
        _refused(**{name: t.to(dtype)})
        # (as many bytes as the right type has)
        _refused(**{name: torch.zeros(t.shape[:-1] + (max(1, t.shape[-1] * 4 // dtype.itemsize),), dtype=dtype)})


@pytest.mark.parametrize("name", list(_tensors()))
def test_fewer_rows(name):
    _refused(**{name: _tensors()[name][:ROWS - 1]})
    _refused(**{name: _tensors()[name][:0]})
    with pytest.raises(ValueError):  # one row, of which a tensor has none
        qlin.logits_controls(**{**_tensors(1), **dict(rows=1, vocab=VOCAB), name: _tensors()[name][:0]})


def test_fewer_tokens():
    _refused(logits=torch.zeros(ROWS, VOCAB - 1))
    _refused(out=torch.zeros(ROWS, VOCAB - 1))


@pytest.mark.parametrize("name", ["history_lens", "repetition", "frequency", "presence", "picks"])
def test_values_apart(name):
    t = _tensors()[name]
    _refused(**{name: torch.zeros(2 * ROWS, dtype=t.dtype)[::2]})


def test_calls_without_rows():
    """Nothing to do, with tensors of any number of rows (and no vocabulary: the same)."""
    for rows, have in ((0, 0), (0, 3)):
        qlin.logits_controls(**_tensors(have), rows=rows, vocab=VOCAB)
    qlin.logits_controls(**_tensors(), rows=ROWS, vocab=0)


@pytest.mark.gpu
def test_what_is_taken():
    """More rows than the call has, addresses for what has a value for each row, and single rows of any stride."""
    from gpu_util import banner, bind_stream
    bind_stream()
    banner("layouts that are taken")
    t = _tensors(5, "cuda")
    t["logits"].copy_(torch.arange(5 * VOCAB, device="cuda").view(5, VOCAB) % 37)
    t["mask"].fill_(-1)
    t["bias_values"].fill_(0.5)
    t["history"].copy_(torch.arange(25, device="cuda").view(5, 5))
    t["history_lens"].fill_(5)
    t["repetition"].fill_(1.5)
    scratch = torch.zeros(max(16, qlin.logits_controls_scratch_bytes(5, VOCAB)), dtype=torch.uint8, device="cuda")
    qlin.logits_controls(**t, rows=5, vocab=VOCAB, scratch=scratch)
    torch.cuda.synchronize()
    out, picks = t["out"].clone(), t["picks"].clone()
    t["out"].zero_(), t["picks"].fill_(-1)
    addresses = {n: t[n].data_ptr() for n in ("history_lens", "repetition", "frequency", "presence", "picks")}
    qlin.logits_controls(**{**t, **addresses}, rows=3, vocab=VOCAB, scratch=scratch)
    torch.cuda.synchronize()
    assert torch.equal(t["out"][:3], out[:3]) and (t["out"][3:] == 0).all()
    assert torch.equal(t["picks"][:3], picks[:3]) and (t["picks"][3:] == -1).all()
    t["out"].zero_()
    wide = torch.zeros(1, 2 * VOCAB, device="cuda")
    wide[0, 3:VOCAB + 3] = t["logits"][1]
    one = {n: v[1:2] for n, v in t.items()}
    qlin.logits_controls(**{**one, "logits": wide[:, 3:VOCAB + 3]}, rows=1, vocab=VOCAB, scratch=scratch)
    torch.cuda.synchronize()
    assert torch.equal(t["out"][1], out[1]) and int(t["picks"][1]) == int(picks[1])
    t["out"].zero_()
    qlin.logits_controls(**{**t, "mask": t["mask"].view(torch.uint32)}, rows=5, vocab=VOCAB, scratch=scratch)
    torch.cuda.synchronize()
    assert torch.equal(t["out"], out)
