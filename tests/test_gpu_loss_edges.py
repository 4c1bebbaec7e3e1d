"""linear_cross_entropy where few tests reach: rows of very different weights."""
import pytest
import torch

import orthossm_b200 as O
from tests.test_gpu_training import BF, HF, gen, lce_inputs

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
