"""The calls around a step's linears refuse tensors that would be read as other values, before anything is launched (a library that
counts its calls stands in for the real one)."""
import pytest
import torch

from blog_amd import qlin


@pytest.fixture
def calls(monkeypatch):
    qlin.lib()
    made = []

    class Counted:
        def __getattr__(self, name):
            return lambda *a: made.append(name) or 0
    monkeypatch.setattr(qlin, "_lib", Counted())
    monkeypatch.setattr(qlin, "_device_of", lambda t, name: t.get_device())
    return made


f32, i32, u8, bf16, f16 = torch.float32, torch.int32, torch.uint8, torch.bfloat16, torch.float16


def z(*shape, dtype=f32):
    return torch.zeros(*shape, dtype=dtype)


def _verify(n=3, d=4, vocab=10, **kw):
    a = dict(target=z(n, d + 1, vocab), drafts=z(n, d, dtype=i32), uniform=z(n, d + 1), tokens=z(n, d + 1, dtype=i32), accepted=z(n, dtype=i32),
             n_drafts=z(n, dtype=i32), temperature=z(n), logprobs=z(n, d + 1), rates=z(n, d), workspace=z(64, dtype=u8))
    a.update(kw)
    qlin.verify_drafts(a.pop("target"), a.pop("drafts"), a.pop("uniform"), a.pop("tokens"), a.pop("accepted"), **a)


@pytest.mark.parametrize("bad", [dict(uniform=z(3, 8)), dict(uniform=z(5, 3)), dict(uniform=z(3, 4)), dict(drafts=z(3, 5, dtype=i32)), dict(drafts=z(4, 3, dtype=i32)),
                                 dict(tokens=z(3, 8, dtype=i32)), dict(logprobs=z(3, 6)), dict(rates=z(3, 5)), dict(rates=z(4, 4)[:, :3]),
                                 dict(accepted=z(3, 2, dtype=i32)), dict(n_drafts=z(3, 5, dtype=i32)), dict(temperature=z(4, 3)), dict(temperature=z(2)),
                                 dict(uniform=z(3, 5, dtype=torch.float64)), dict(tokens=z(3, 5))],
                         ids=lambda b: ",".join(f"{k}{list(v.shape)}" for k, v in b.items()))
def test_verify_drafts_refuses(calls, bad):
    with pytest.raises(ValueError):
        _verify(**bad)
    assert not calls


@pytest.mark.parametrize("good", [{}, dict(uniform=z(7, 5), tokens=z(4, 5, dtype=i32), rates=z(9, 4)), dict(uniform=z(15), drafts=z(20, dtype=i32)),
                                  dict(accepted=z(3, 1, dtype=i32), temperature=z(1, 3)), dict(accepted=z(8, dtype=i32)), dict(accepted=z(8, 1, dtype=i32))])
def test_verify_drafts_takes(calls, good):
    _verify(**good)
    assert calls == ["qlin_launch_verify_drafts"]


def test_verify_drafts_of_one_sequence_and_without_drafts(calls):
    _verify(n=1, uniform=z(1, 9), drafts=z(1, 32, dtype=i32))  # the values stand where they are read
    _verify(d=0, uniform=z(3, 1), drafts=None, rates=None)
    _verify(d=0, uniform=z(3), tokens=z(3, dtype=i32), rates=z(3, 0))
    assert len(calls) == 3
    with pytest.raises(ValueError):
        _verify(d=0, uniform=z(3, 4))
    assert len(calls) == 3


def test_lora_add_refuses(calls):
    w = qlin.Lora(z(2, 8, 64), z(2, 32, 8))

    def run(ids=z(3, dtype=i32), ranks=z(2, dtype=i32), scales=z(2)):
        qlin.lora_add(z(3, 64), ids, [(w, z(3, 32), z(3, 32))], ranks=ranks, scales=scales, workspace=z(64, dtype=u8))
    run()
    run(ids=z(9, dtype=i32), ranks=z(1, 2, dtype=i32), scales=z(2, 1))
    assert len(calls) == 2
    for bad in (dict(ids=z(3, 2, dtype=i32)), dict(ids=z(2, dtype=i32)), dict(ids=z(3, dtype=torch.int64)), dict(ranks=z(2, 3, dtype=i32)), dict(scales=z(4, 2))):
        with pytest.raises(ValueError):
            run(**bad)
    assert len(calls) == 2


def test_moe_route_refuses(calls):
    for bias in (z(2, 8), z(7)):
        with pytest.raises(ValueError):
            qlin.moe_route(qlin.MoeRouting(bias=bias), z(3, 8), z(3, 2, dtype=i32), z(3, 2))
    assert not calls
    qlin.moe_route(qlin.MoeRouting(bias=z(8)), z(3, 8), z(4, 2, dtype=i32), z(4, 2))
    qlin.moe_route(qlin.MoeRouting(bias=z(1, 8)), z(3, 8), z(3, 2, dtype=i32), z(3, 2))
    assert len(calls) == 2


def test_blocks_read_back_refuse(calls):
    blocks = z(qlin.q8_1_bytes(64, 3), dtype=u8)
    qlin.dequantize_q8_1(blocks, z(3, 64), 64, 3)
    qlin.dequantize_q8_1(blocks, z(200), 64, 3)
    qlin.dequantize_q8_1(blocks, z(1, 70), 64, 1)
    assert len(calls) == 3
    for bad in (z(3, 70), z(2, 64), z(64, 3)):
        with pytest.raises(ValueError):
            qlin.dequantize_q8_1(blocks, bad, 64, 3)
    assert len(calls) == 3


def test_add_rms_norm_refuses_weights_of_several_rows(calls):
    x = z(2, 64)
    qlin.add_rms_norm(x, None, None, z(80, dtype=bf16), 0, 1e-6, 0, normed=z(2, 64))
    qlin.add_rms_norm(x, None, None, z(1, 64, dtype=bf16), 0, 1e-6, 0, normed=z(2, 64))
    for bad in (z(2, 64, dtype=bf16), z(64, 2, dtype=bf16), z(63, dtype=bf16), z(64)):
        with pytest.raises(ValueError):
            qlin.add_rms_norm(x, None, None, bad, 0, 1e-6, 0, normed=z(2, 64))
    assert len(calls) == 2


def test_add_rms_norm_refuses_weights_of_the_other_type(calls):
    x = z(2, 64)
    run = lambda w, kind: qlin.add_rms_norm(x, None, None, w, kind, 1e-6, 0, normed=z(2, 64))
    for w, kind in ((z(64, dtype=bf16), 0), (z(64, dtype=f16), 1), (z(64, dtype=torch.int16), 0), (z(64, dtype=torch.int16), 1), (z(64, dtype=torch.uint16), 1)):
        run(w, kind)  # (patterns of 16 bits may be either)
    assert len(calls) == 5
    for w, kind in ((z(64, dtype=bf16), 1), (z(64, dtype=f16), 0)):
        with pytest.raises(ValueError):
            run(w, kind)
    assert len(calls) == 5


def test_tensors_of_another_device_than_the_current_one(calls, monkeypatch):
    monkeypatch.undo()
    qlin.lib()
    monkeypatch.setattr(qlin, "_current_device", lambda: 0, raising=False)

    class There:
        device = "cuda"

        def __init__(self, at):
            self.at = at

        def get_device(self):
            return self.at
    assert qlin._device_of(There(0), "x") == 0
    for at in (1, -1):
        with pytest.raises(ValueError):
            qlin._device_of(There(at), "x")
