"""The targets that OrthoSSMLM.loss makes of its input: the next token of each
position, whatever integer type the ids have, none around padding."""
import pytest
import torch

import orthossm_b200.lm as lm


class _Stop(Exception):
    pass


def made(monkeypatch, ids, **kw):
    """The targets a call of loss hands on, taken where the network begins (no GPU)."""
    model = lm.OrthoSSMLM(lm.OrthoLMConfig(vocab_size=300, n_layers=1)).to(torch.bfloat16)
    got = []

    def end(h, w, targets, **_):
        got.append(targets)
        raise _Stop

    monkeypatch.setattr(lm, "embed_tokens", lambda ids, w: torch.zeros(*ids.shape, w.shape[1], dtype=w.dtype))
    monkeypatch.setattr(lm, "residual_norm", lambda x, y, *a, **k: (x, x))
    monkeypatch.setattr(lm.V8Layer, "paths", lambda self, h, c, e: (h, h, None))
    monkeypatch.setattr(lm, "linear_cross_entropy", end)
    with pytest.raises(_Stop):
        model.loss(ids, **kw)
    return got[0]


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64])
@pytest.mark.parametrize("ignore", [-100, -1000, 1 << 40])
def test_any_integer_type(monkeypatch, dtype, ignore):
    ids = torch.tensor([[3, 100, 7, 120], [0, 1, 2, 3]], dtype=dtype)
    t = made(monkeypatch, ids, ignore_index=ignore)
    assert t.long().tolist() == [[100, 7, 120, ignore], [1, 2, 3, ignore]]


def test_the_last_byte_is_a_token(monkeypatch):
    """255 of a byte vocabulary is no padding, although uint8 compares it equal to -1."""
    ids = torch.tensor([[255, 7, 255, 255, 0]], dtype=torch.uint8)
    assert made(monkeypatch, ids).tolist() == [[7, 255, 255, 0, -100]]


def test_padding_anywhere(monkeypatch):
    """Padding (-1) before, between or after tokens has no target, and is none: what follows it begins a text."""
    ids = torch.tensor([[-1, -1, 4, 5, 6], [7, -1, -1, 8, 9], [1, 2, 3, -1, -1]])
    assert made(monkeypatch, ids, ignore_index=-7).tolist() == [[-7, -7, 5, 6, -7], [-7, -7, -7, 9, -7],
                                                                [2, 3, -7, -7, -7]]


@pytest.mark.gpu
def test_loss_of_left_padding_and_gaps():
    """No loss where a position or the one after it is padding, and the mean is over the others."""
    torch.manual_seed(0)
    model = lm.OrthoSSMLM(lm.OrthoLMConfig(vocab_size=300, n_layers=1, window=64)).to("cuda", torch.bfloat16)
    ids = torch.randint(0, 300, (2, 150), device="cuda")
    ids[0, :40] = -1
    ids[1, 60:70] = -1
    st = model.fresh_states(2, "cuda", generator_seed=1)
    with torch.no_grad():
        each = model.loss(ids, states=st, reduction="none")
        mean = model.loss(ids, states=st)
    has = torch.zeros_like(ids, dtype=torch.bool)
    has[0, 40:-1] = True
    has[1, :59] = True
    has[1, 70:-1] = True
    assert torch.equal(each != 0, has) and each.isfinite().all()
    # a mean and a sum of 247 fp32 losses, each rounded to 2^-24
    assert abs(float(mean) - float(each.double().sum() / has.sum())) <= 2.0 ** -23 * float(mean)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int16, torch.int32])
def test_loss_of_small_id_types(dtype):
    """A byte vocabulary's ids as bytes: the losses and gradients of the same ids in int64."""
    torch.manual_seed(0)
    model = lm.OrthoSSMLM(lm.OrthoLMConfig(vocab_size=256, n_layers=1, window=64)).to("cuda", torch.bfloat16)
    ids = torch.randint(0, 256, (2, 130), device="cuda")
    ids[0, ::9], ids[1, -1] = 255, 255
    st = model.fresh_states(2, "cuda", generator_seed=1)
    out = []
    for i in (ids, ids.to(dtype)):
        loss = model.loss(i, states=st)
        out.append((loss.detach(), *torch.autograd.grad(loss, [model.embedding.weight, model.final_norm.weight])))
        with torch.no_grad():
            out[-1] += (model.loss(i, states=st, reduction="none"),)
    for a, b in zip(*out):
        assert torch.equal(a, b)
    assert (out[1][3][:, -1] == 0).all() and (out[1][3][:, :-1] > 0).all()
