"""OrthoSSMLM.loss with its three operators in place and with their plain fp32
forms in their places: the rest of the network is the same in both."""
import pytest
import torch
import torch.nn.functional as F

import orthossm_b200.lm as lm
from tests.test_gpu_lm_loss import model_and_ids, rel

pytestmark = pytest.mark.gpu


def plain_embed(ids, w):
    return w.float()[ids.clamp(min=0)].mul((ids >= 0)[..., None]).to(w.dtype)


def plain_norm(x, y, w, b=None, *, norm="rms", eps):
    s = x.float() if y is None else x.float() + y.float()
    v = s - s.mean(-1, keepdim=True) if norm == "layer" else s
    h = v * (v.square().mean(-1, keepdim=True) + eps).rsqrt() * w.float()
    return s.to(x.dtype), (h if b is None else h + b.float()).to(x.dtype)


def plain_loss(h, w, targets, *, ignore_index, z_loss, reduction):
    z = h.float() @ w.float().t()
    on = targets != ignore_index
    lse = z.logsumexp(-1)
    each = F.cross_entropy(z.flatten(0, 1), targets.flatten(), ignore_index=ignore_index, reduction="none")
    each = each.view(targets.shape) + z_loss * torch.where(on, lse, 0.0).square()
    return each if reduction == "none" else each.sum() / (on.sum() if reduction == "mean" else 1)


@pytest.mark.parametrize("reduction,z_loss", [("mean", 0.0), ("sum", 1e-3)])
def test_gradients_of_all_parameters(monkeypatch, reduction, z_loss):
    """Both round at the same places, the operators beside that dz and each
    gradient once: 7 calls, 2^-9 / sqrt(3) = 1.1e-3 of the norm each, two of them
    a call, sqrt(14) 1.1e-3 = 4.2e-3 in all, and the flips that follow in the rest
    of the network.  1e-2 is asked, so no contribution of a hundredth can be missing."""
    model, ids = model_and_ids()
    ids = ids.clone()
    ids[0, :30], ids[1, 200:210] = -1, -1
    st = model.fresh_states(2, "cuda", generator_seed=1)
    ps = dict(model.named_parameters())

    def step():
        loss = model.loss(ids, states=st, reduction=reduction, z_loss=z_loss)
        return loss.detach(), torch.autograd.grad(loss, list(ps.values()), allow_unused=True)

    loss, got = step()
    monkeypatch.setattr(torch.backends.cuda.matmul, "allow_tf32", False)
    for name, f in (("embed_tokens", plain_embed), ("residual_norm", plain_norm), ("linear_cross_entropy", plain_loss)):
        monkeypatch.setattr(lm, name, f)
    want_loss, want = step()
    assert abs(float(loss) / float(want_loss) - 1) < 1e-3
    for name, a, b in zip(ps, got, want):
        assert (a is None) == (b is None), name
        if a is not None:
            assert rel(a, b) < 1e-2, (name, rel(a, b))
