"""Scalars of the training operators beyond fp32, in which the kernels take them, are refused as others are."""
import ctypes as C

import pytest
import torch

import orthossm_b200 as O
from orthossm_b200 import _lib as L
from tests.test_training_host import EMBED


@pytest.mark.parametrize("scale", [float("inf"), float("-inf"), float("nan")])
def test_embed_scale_at_the_c_entry(scale):
    lib = L.lib()
    a = L.EmbedArgs(**{**EMBED, "scale": scale})
    assert lib.ossm_embed_workspace_bytes(C.byref(a)) == 0
    assert lib.ossm_embed_fwd(C.byref(a), None) == L.OSSM_EINVAL
    assert lib.ossm_embed_bwd(C.byref(a), 4096, 1 << 40, None) == L.OSSM_EINVAL


@pytest.mark.gpu
@pytest.mark.parametrize("big", [1e39, 1e300])
def test_beyond_fp32(big):
    x = torch.zeros(4, 64, device="cuda", dtype=torch.bfloat16)
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    for call in (lambda: O.linear_cross_entropy(x, x, t, z_loss=big), lambda: O.embed_tokens(t, x, scale=big),
                 lambda: O.embed_tokens(t, x, scale=-big), lambda: O.residual_norm(x, x, scale=big),
                 lambda: O.residual_norm(x, x, scale=-big), lambda: O.residual_norm(x, eps=big),
                 lambda: O.residual_norm(x, x, post_norm="rms", post_eps=big)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: O.linear_cross_entropy(x, x, t, z_loss=3e38), lambda: O.embed_tokens(t, x, scale=-3e38),
                 lambda: O.residual_norm(x, x, scale=3e38, eps=3e38)):
        call()
