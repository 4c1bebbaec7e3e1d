"""residual_norm's gradients where roundings on the way would show: from the sum
itself, not from the rounded stream that forward returns."""
import pytest
import torch

import orthossm_b200 as O
from tests.test_gpu_training import BF, FP, HF, gen, norm_inputs
from tests.training_ref import assert_within, norm_ref, u

pytestmark = pytest.mark.gpu


def norm_ref_of_the_sum(ts, opts, dr, dh):
    """norm_ref's values with the bounds of a backward pass that starts from x
    and y: a gate of ones changes no value, and no bound but that one."""
    one = torch.ones(ts["x"].shape[-1], device="cuda")
    ref = norm_ref({**ts, "gate": one}, opts, dr, dh)
    del ref["dgate"]
    return ref


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("shape", [(400, 1), (300, 3), (37, 8), (20, 257), (50, 512), (9, 2048), (2, 8192)])
@pytest.mark.parametrize("norm,scale", [("rms", 1.0), ("rms", 0.7), ("rms", 2.0 ** -10), ("layer", 0.7)])
def test_from_the_sum(shape, norm, scale, dt):
    ts = norm_inputs(shape, dt, dt, norm, None, None)
    if scale < 0.01:  # a stream among fp16's subnormal numbers
        with torch.no_grad():
            ts["x"].mul_(2.0 ** -16)
            ts["y"].mul_(2.0 ** -6)
    eps = 1e-14 if scale < 0.01 else 1e-5
    r, h = O.residual_norm(ts["x"], ts["y"], ts["weight"], ts["bias"], norm=norm, eps=eps, scale=scale)
    dr = torch.randn(shape, device="cuda", generator=gen(5)).to(dt)
    for dh in (torch.randn(shape, device="cuda", generator=gen(6)).to(dt), h.detach()):
        dh = dh * 2.0 ** -6 if scale < 0.01 else dh  # dx stays within fp16
        names = [k for k, t in ts.items() if t is not None]
        got = dict(zip(names, torch.autograd.grad((r, h), [ts[k] for k in names], (dr, dh), retain_graph=True)))
        want = norm_ref_of_the_sum(ts, dict(norm=norm, post_norm=None, scale=scale, eps=eps), dr, dh)
        for k in names:
            v, b = want["d" + k]
            # one channel, r of 1e-7: dx of 1e7 dh eps / (r^2 + eps) passes fp16's range.  65504 and half of its
            # step of 32 round to infinity, so a value that may lie there may be infinite
            over = got[k].isinf() & (v.abs() + b >= 65520) & (got[k].sign() == v.sign()) & (dt is HF)
            assert_within(torch.where(over, 0, got[k]), torch.where(over, 0, v), b, k)


@pytest.mark.parametrize("dt", [BF, HF])
def test_upstream_parallel_to_the_normed_row(dt):
    """dx = inv (e - v mean(e v)) takes off what is parallel to v.  With e = h,
    the rounded v, what is left is e's own rounding, some 0.3 u of its norm; fp32
    statistics and sums of 512 terms lose at most 512 2^-24 = 3e-5 of e, a 40th
    of that in bf16 and a fifth in fp16, the output's rounding u of the result.
    (From the rounded sum it is off by its whole norm.)"""
    g = gen(0)
    x, y = ((torch.randn(1000, 512, device="cuda", generator=g)).to(dt).requires_grad_() for _ in range(2))
    _, h = O.residual_norm(x, y)
    dx, dy = torch.autograd.grad(h, (x, y), h.detach())
    xd, yd = x.detach().double().requires_grad_(), y.detach().double().requires_grad_()
    s = xd + yd
    v = s / (s.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    want, = torch.autograd.grad(v, xd, h.detach().double())
    for got in (dx, dy):
        off = float((got.double() - want).norm() / want.norm())
        assert off < u(dt) + (0.03 if dt is BF else 0.2), off


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("d", [1, 512])
def test_weight_gradient_of_the_sum(d, dt):
    """A weight's gradient is a sum over 8 rows of normed values: fp32 terms within
    (d + 32) 2^-23 of their own, and their sum; the weight is fp32.  The terms'
    signs are alike, so that the sum is as large as its terms."""
    g = gen(1)
    x, y = ((torch.randn(8, d, device="cuda", generator=g)).to(dt) for _ in range(2))
    w = torch.ones(d, device="cuda").requires_grad_()
    _, h = O.residual_norm(x, y, w, eps=0.05)
    dh = (h.detach().sign() * (0.5 + torch.rand(8, d, device="cuda", generator=g))).to(dt)
    dw, = torch.autograd.grad(h, w, dh)
    s = x.double() + y.double()
    want = (dh.double() * s / (s.square().mean(-1, keepdim=True) + 0.05).sqrt()).sum(0)
    assert float(((dw.double() - want).abs() / want).max()) < (2 * d + 64 + 8) * 2.0 ** -24


@pytest.mark.parametrize("xdt,ydt", [(BF, BF), (HF, HF), (FP, FP), (FP, BF)])
@pytest.mark.parametrize("gate,post", [(None, None), ("channel", "rms"), ("token", None), (None, "layer")])
def test_gradient_of_the_stream_alone(gate, post, xdt, ydt):
    """Only r is used: h's norm has no part in the gradients."""
    ts = norm_inputs((70, 264), xdt, ydt, "rms", post, gate)
    r, h = O.residual_norm(ts["x"], ts["y"], ts["weight"], gate=ts["gate"], scale=0.5, eps=1e-5, post_norm=post,
                           post_weight=ts["post_weight"], post_bias=ts["post_bias"])
    dr = torch.randn(r.shape, device="cuda", generator=gen(2)).to(xdt)
    names = [k for k, t in ts.items() if t is not None and k != "weight"]
    got = torch.autograd.grad(r, [ts[k] for k in names], dr)
    want = norm_ref(ts, dict(norm="rms", post_norm=post, scale=0.5, eps=1e-5), dr, torch.zeros_like(h))
    for k, v in zip(names, got):
        assert_within(v, *want["d" + k], k)


@pytest.mark.parametrize("dt", [BF, HF, FP])
def test_one_tensor_as_stream_and_output(dt):
    """x + x, both returned values and x again: the gradients of all uses add up.
    Three gradients of dt are added up, each and each sum rounded once: 5 u of
    their magnitudes, beside the norm's own four times (64 + 32) 2^-23."""
    x = torch.randn(30, 64, device="cuda", generator=gen(1)).to(dt).requires_grad_()
    c = [torch.randn(30, 64, device="cuda", generator=gen(k)).to(dt) for k in (2, 3, 4)]
    r, h = O.residual_norm(x, x, scale=0.5)
    got, = torch.autograd.grad((r * c[0]).float().sum() + (h * c[1]).float().sum() + (x * c[2]).float().sum(), x)
    xd = x.detach().double().requires_grad_()
    s = 1.5 * xd
    n = s / (s.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    parts = [torch.autograd.grad((v * k.double()).sum(), xd, retain_graph=True)[0] for v, k in zip((s, n, xd), c)]
    mag = sum(p.abs() for p in parts) + (s.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * 2 * c[1].double().abs()
    assert_within(got, sum(parts), 5 * u(dt) * mag + 4 * 96 * 2.0 ** -23 * mag)
