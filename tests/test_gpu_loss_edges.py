"""linear_cross_entropy where few tests reach: rows of very different weights,
sure tokens, several groups of rows, several pieces, very wide states, and
differences."""
import pytest
import torch

import orthossm_b200 as O
from tests.test_gpu_training import BF, HF, check_lce, gen, lce_inputs
from tests.training_ref import assert_within, lce_ref, u

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_weight_that_is_not_finite(bad, dt):
    """One token's upstream gradient has overflowed: its own row and the weight's
    gradient show it, the other rows are what they are without it."""
    h, w, t = lce_inputs(300, 64, 1000, dt, 0.2)
    loss = O.linear_cross_entropy(h, w, t, reduction="none")
    k = int((t != -100).nonzero()[7, 0])
    up = torch.rand(300, device="cuda", generator=gen(1))
    up[k] = 0.0
    want, _ = torch.autograd.grad(loss, (h, w), up, retain_graph=True)
    up[k] = bad
    dh, dw = torch.autograd.grad(loss, (h, w), up)
    rest = torch.arange(300, device="cuda") != k
    assert float(want[rest].float().norm()) > 0 and torch.equal(dh[rest], want[rest])
    assert not dh[k].isfinite().any() and not dw.isfinite().any()


def sure_inputs(T, V, dt, gap, shift):
    """Tokens whose target's logit lies about ``gap`` above log of the others' sum,
    all logits near ``shift``: the first channel shifts, the others tell targets apart."""
    d = 64
    g = gen(4)
    w = torch.randn(V, d, device="cuda", generator=g) / 8
    w[:, 0] = 1.0
    w = w.to(dt)
    t = torch.randperm(V, device="cuda", generator=g)[:T]
    rest = w.double().clone()
    rest[:, 0] = 0
    h = torch.zeros(T, d, device="cuda", dtype=torch.float64)
    for _ in range(60):  # along the target's row until it is as far above the others
        h[:, 0] = 0
        z = h @ rest.t()
        zt = z.gather(1, t[:, None])[:, 0]
        z.scatter_(1, t[:, None], -torch.inf)
        h += (gap - (zt - z.logsumexp(1)))[:, None].clamp(-2, 2) * 0.7 * rest[t] / rest[t].square().sum(1, keepdim=True)
    h[:, 0] = shift
    return h.to(dt).requires_grad_(), w.requires_grad_(), t


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("gap", [5.0, 9.0])
@pytest.mark.parametrize("shift", [0.0, 20.0, 100.0])
def test_sure_tokens(shift, gap, dt):
    """A token of probability 1 - q has gradients of the size of q.  dW of the
    targets' rows is -g q h: q's own error is at most exp's of the logits' fp32
    sums (64 + 8 terms within 2^-23 of their magnitudes, of the target and of the
    others), and beside it, relative to 1 and not to q, the softmax's fp32 sum
    and 2^x: 42 additions of 2^-24 that the largest term sees (the 32 of its run,
    and those of the runs, halves and tiles of 1000 columns) and twice 2^-22."""
    V, T = 1000, 200
    h, w, t = sure_inputs(T, V, dt, gap, shift)
    loss = O.linear_cross_entropy(h, w, t, reduction="sum")
    dh, dw = torch.autograd.grad(loss, (h, w))
    H, W = h.detach().double(), w.detach().double()
    z = H @ W.t()
    p = z.softmax(1)
    q = 1 - p.gather(1, t[:, None])[:, 0]
    assert q.median() < 2 * torch.tensor(-gap).exp()
    ez = 72 * 2.0 ** -23 * (H.abs() @ W.abs().t()).amax(1)
    eq = q * 2 * ez * 1.01 + 42 * 2.0 ** -24 + 2 * 2.0 ** -22
    dz = p.clone()
    dz.scatter_add_(1, t[:, None], torch.full_like(q, -1.0)[:, None])
    want = -q[:, None] * H + (dz.scatter(1, t[:, None], 0.0).t() @ H)[t]  # other tokens' small part too
    mag = q[:, None] * H.abs() + (dz.scatter(1, t[:, None], 0.0).t() @ H.abs())[t]
    bound = eq[:, None] * H.abs() + 2.02 * u(dt) * mag + 2e-3 * (mag - q[:, None] * H.abs()) + T * 2.0 ** -23 * mag
    if dt is HF:  # probabilities below 2^-28 of the largest factor, outputs below the normal numbers
        bound = bound + 2.0 ** -39 * H.abs().sum(0) + 2.0 ** -25
    assert_within(dw[t], want, bound, "dweight")
    with torch.no_grad():  # the loss, -log(1 - q), of that size too
        each = O.linear_cross_entropy(h, w, t, reduction="none")
    assert_within(each, -torch.log1p(-q), 1.1 * eq + q * 2.0 ** -24, "loss")


@pytest.mark.parametrize("dt", [BF, HF])
def test_weights_over_decades(dt):
    """Per-token weights from 4096 down to 2^-12: dz is in units of the largest
    weight of the call, so a row of a share rho of it keeps probabilities down to
    2^-28 / rho in fp16.  Each element within lce_ref's bound, which counts that."""
    T, d, V = 260, 128, 4000
    h, w, t = lce_inputs(T, d, V, dt, 0.1)
    loss = O.linear_cross_entropy(h, w, t, reduction="none")
    up = 4096.0 * 2.0 ** (-24 * torch.arange(T, device="cuda") / (T - 1))
    got = torch.autograd.grad(loss, (h, w), up)
    want, bound = lce_ref(h, w, t, up, reduction="none")
    for a, b, c, what in zip(got, want[1:], bound[1:], ("dhidden", "dweight")):
        assert_within(a, b, c, what)
    # in norm: a row's softmax part loses at most 2^-25 2^-14 of the largest weight an element, as noise over the columns
    on = t != -100
    off = (got[0].double() - want[1]).norm(dim=1)[on]
    tiny = 2.0 ** -25 if dt is HF else 0.0  # half of the output's smallest step
    allowed = (2.02 * u(dt) * want[1].norm(dim=1) + tiny * d ** 0.5)[on]
    allowed = allowed + (4096.0 * 2.0 ** -39 * w.detach().double().norm() if dt is HF else 0.0) + 1e-4 * up[on]
    assert (off <= allowed).all()


@pytest.mark.parametrize("T,d,V,ignored", [(8400, 2048, 700, 0.0), (8900, 2048, 300, 0.05), (33500, 512, 600, 0.0)])
def test_several_groups_of_row_blocks(T, d, V, ignored):
    """More than 32 MB of states: the blocks of rows stand in two groups, the last one smaller."""
    check_lce(*lce_inputs(T, d, V, BF, ignored), z_loss=1e-4)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_several_pieces_and_no_token_ignored(reduction):
    """40000 tokens take pieces of 6656 columns: two, the second a ragged one; the states are read where they lie."""
    check_lce(*lce_inputs(40000, 24, 7003, HF, 0.0), reduction=reduction)


@pytest.mark.parametrize("T,d,V", [(130, 16392, 300), (5, 65536, 257)])
def test_very_wide_states(T, d, V):
    check_lce(*lce_inputs(T, d, V, BF, 0.1))


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("of", ["hidden", "weight"])
def test_differences(of, dt):
    """The slope along a direction from the loss alone, in float64: central
    differences at two steps (their difference bounds what the finer one is off
    by), along the gradient's own signs, along its positive part, and at random.
    The allowance is the gradient's rounding bound along the direction; it has to
    be a small part of the slope, so a gradient that is 0 or twice as large fails."""
    h, w, t = lce_inputs(64, 64, 500, dt, 0.2)
    loss = O.linear_cross_entropy(h, w, t, reduction="sum", z_loss=1e-3)
    grad = torch.autograd.grad(loss, (h, w))[of == "weight"].double()
    on = t != -100
    H, W = h.detach().double(), w.detach().double()

    def f(v):
        z = (v if of == "hidden" else H)[on] @ (W if of == "hidden" else v).t()
        lse = z.logsumexp(1)
        return (lse - z.gather(1, t[on][:, None])[:, 0] + 1e-3 * lse ** 2).sum()

    at = H if of == "hidden" else W
    _, bound = lce_ref(h, w, t, torch.ones((), device="cuda"), z_loss=1e-3, reduction="sum")
    bound = bound[1 + (of == "weight")]
    exact = torch.autograd.grad(f(at.requires_grad_()), at)[0]
    at = at.detach()
    noise = torch.randn(at.shape, device="cuda", dtype=torch.float64, generator=gen(3))
    for e in (exact.sign(), exact.clamp(min=0), noise + 2 * exact.abs().mean() ** -1 * exact):
        e = e / e.norm()
        d1, d2 = ((f(at + s * e) - f(at - s * e)) / (2 * s) for s in (2.0 ** -6, 2.0 ** -7))
        allowed = (bound * e.abs()).sum() + 2 * (d1 - d2).abs()
        assert allowed < 0.1 * d2.abs()
        assert ((grad * e).sum() - d2).abs() <= allowed
