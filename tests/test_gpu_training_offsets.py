"""Tensors of more than 2^32 elements: the rows at their ends are what a call on
those rows alone makes of them."""
import pytest
import torch

import orthossm_b200 as O
from tests.test_gpu_training import BF, gen

pytestmark = pytest.mark.gpu
T, D = (1 << 22) + 37, 1024  # 8.6 GB in bf16


@pytest.fixture(autouse=True)
def free():
    yield
    torch.cuda.empty_cache()


def rows(T, d):
    """Random rows, the same 4096 again and again (filled in pieces: small in memory beside them)."""
    some = torch.randn(4096, d, device="cuda", generator=gen(0)).to(BF)
    out = torch.empty(T, d, dtype=BF, device="cuda")
    for a in range(0, T, 4096):
        out[a:a + 4096] = some[:min(4096, T - a)]
    return out


def test_norm():
    x = rows(T, D).requires_grad_()
    w = torch.ones(D, device="cuda").requires_grad_()
    r, h = O.residual_norm(x, None, w, norm="layer")
    dx, dw = torch.autograd.grad(h, (x, w), h.detach())
    xe = x.detach()[-100:].clone().requires_grad_()
    _, he = O.residual_norm(xe, None, w.detach(), norm="layer")
    dxe, = torch.autograd.grad(he, xe, he.detach())
    assert torch.equal(h[-100:], he) and torch.equal(dx[-100:], dxe)
    # the weight's: 1024 times the sum over the 4096 different rows, and the first 37 again; terms of one sign, at
    # most T / 148 of them and 32 runs of blocks added up one by one in fp32
    v = torch.nn.functional.layer_norm(x.detach()[:4096].double(), (D,), eps=1e-6) * h.detach()[:4096].double()
    want = 1024 * v.sum(0) + v[:37].sum(0)
    assert float((dw.double() / want - 1).abs().max()) < (T / 148 + 64) * 2.0 ** -24 + 1e-5


def test_embed():
    g = gen(1)
    w = torch.randn(500, D, device="cuda", generator=g).to(BF).requires_grad_()
    ids = torch.randint(0, 400, (T,), device="cuda", generator=g)
    ids[-100:] = torch.arange(400, 500, device="cuda")  # these rows' only positions
    out = O.embed_tokens(ids, w)
    assert torch.equal(out[-100:], w[400:]) and torch.equal(out[:50], w[ids[:50]])
    up = rows(T, D)
    dw, = torch.autograd.grad(out, w, up)
    assert torch.equal(dw[400:], up[-100:])


def test_loss():
    d, V = 2048, 300
    n = (1 << 21) + 37
    h = rows(n, d).requires_grad_()
    w = (torch.randn(V, d, device="cuda", generator=gen(2)) / d ** 0.5).to(BF)
    t = torch.randint(0, V, (n,), device="cuda", generator=gen(3))
    t[5] = -100  # the others' states are laid side by side: as many again
    loss = O.linear_cross_entropy(h, w, t, reduction="none")
    up = torch.ones_like(loss)
    dh, = torch.autograd.grad(loss, h, up)
    he = h.detach()[-100:].clone().requires_grad_()
    le = O.linear_cross_entropy(he, w, t[-100:], reduction="none")
    dhe, = torch.autograd.grad(le, he, up[-100:])
    # other panels of columns, so other orders of fp32 sums of 300 terms; and the gradient rounded to bf16
    loss, le = loss.detach(), le.detach()
    assert float((loss[-100:] - le).abs().max()) <= 2.0 ** -20 * float(le.abs().max())
    assert float((dh[-100:].float() - dhe.float()).abs().max()) <= 2.0 ** -7 * float(dhe.abs().max())
