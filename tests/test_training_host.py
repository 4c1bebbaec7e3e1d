"""Argument checks of the training operators' C entry points: none of these
reaches the GPU."""
import ctypes as C

import pytest
import torch

import orthossm_b200 as O
from orthossm_b200 import _lib as L


def _with(cls, base, **kw):
    return cls(**{**base, **kw})


LCE = dict(tokens=64, dim=512, vocab=1000, dtype=L.OSSM_BF16, hidden=4096, hidden_stride=512, weight=4096,
           weight_stride=512, targets=4096, ignore_index=-100, reduction=L.OSSM_LOSS_MEAN, loss=4096, lse=4096)


@pytest.mark.parametrize("bad", [dict(tokens=0), dict(tokens=(1 << 27) + 1), dict(dim=12), dict(dim=0), dict(vocab=0),
                                 dict(dtype=L.OSSM_F32), dict(hidden=4098), dict(hidden=None), dict(hidden_stride=500),
                                 dict(weight_stride=516), dict(targets=None), dict(reduction=3), dict(z_loss=-1.0),
                                 dict(z_loss=float("nan")), dict(lse=None)])
def test_lce_arguments(bad):
    lib = L.lib()
    for back in (0, 1):
        ok = dict(LCE, grad_loss=4096, grad_hidden=4096, grad_weight=4096)
        assert lib.ossm_lce_workspace_bytes(C.byref(_with(L.LceArgs, ok)), back) > 0
        a = _with(L.LceArgs, ok, **bad)
        assert lib.ossm_lce_workspace_bytes(C.byref(a), back) == 0
        f = lib.ossm_lce_bwd if back else lib.ossm_lce_fwd
        assert f(C.byref(a), 4096, 1 << 40, None) == L.OSSM_EINVAL
        assert f(C.byref(_with(L.LceArgs, ok)), None, 1 << 40, None) == L.OSSM_EWORKSPACE
        assert f(C.byref(_with(L.LceArgs, ok)), 4096, 16, None) == L.OSSM_EWORKSPACE
        assert f(C.byref(_with(L.LceArgs, ok)), 4100, 1 << 40, None) == L.OSSM_EWORKSPACE
    assert lib.ossm_lce_bwd(C.byref(_with(L.LceArgs, LCE)), 4096, 1 << 40, None) == L.OSSM_EINVAL  # no grad_loss


def test_lce_workspace_is_bounded():
    """dz of a piece of the vocabulary, not of all of it."""
    lib = L.lib()
    grads = dict(grad_loss=4096, grad_hidden=4096, grad_weight=4096)
    for T, V in ((16384, 32000), (131072, 32000), (8192, 131072), (1 << 20, 131072)):
        a = _with(L.LceArgs, dict(LCE, **grads), tokens=T, vocab=V)
        n = lib.ossm_lce_workspace_bytes(C.byref(a), 1)
        assert n <= max(512 << 20, T * 4096 * 2) + T * 512 * (2 + 4) + (112 << 20)


EMBED = dict(tokens=64, dim=512, vocab=1000, dtype=L.OSSM_BF16, ids=4096, weight=4096, weight_stride=512, scale=1.0,
             out=4096, grad_out=4096, grad_out_stride=512, grad_weight=4096)


@pytest.mark.parametrize("bad", [dict(tokens=-1), dict(tokens=1 << 31), dict(dim=0), dict(dim=65537), dict(vocab=0),
                                 dict(vocab=1 << 27), dict(dtype=3), dict(ids=None)])
def test_embed_arguments(bad):
    lib = L.lib()
    assert lib.ossm_embed_workspace_bytes(C.byref(_with(L.EmbedArgs, EMBED))) > 0
    a = _with(L.EmbedArgs, EMBED, **bad)
    assert lib.ossm_embed_workspace_bytes(C.byref(a)) == 0
    assert lib.ossm_embed_fwd(C.byref(a), None) == L.OSSM_EINVAL
    assert lib.ossm_embed_bwd(C.byref(a), 4096, 1 << 40, None) == L.OSSM_EINVAL
    assert lib.ossm_embed_bwd(C.byref(_with(L.EmbedArgs, EMBED)), None, 1 << 40, None) == L.OSSM_EWORKSPACE


NORM = dict(tokens=64, dim=512, stream_dtype=L.OSSM_BF16, dtype=L.OSSM_BF16, x=4096, x_stride=512, y=4096, y_stride=512,
            scale=1.0, norm=L.OSSM_NORM_RMS, eps=1e-6, post_eps=1e-6, r=4096, h=4096, stats=4096, grad_r=4096,
            grad_r_stride=512, grad_h=4096, grad_h_stride=512)


@pytest.mark.parametrize("bad", [dict(tokens=-1), dict(dim=0), dict(dim=8193), dict(stream_dtype=5),
                                 dict(stream_dtype=L.OSSM_F16), dict(norm=0), dict(norm=3), dict(post_norm=3),
                                 dict(gate_kind=1), dict(gate_kind=4, gate=4096), dict(eps=-1.0),
                                 dict(scale=float("inf")), dict(y=None, post_norm=1), dict(post_weight=4096),
                                 dict(gate_kind=3, gate=4096, gate_stride=100)])
def test_norm_arguments(bad):
    lib = L.lib()
    assert lib.ossm_norm_workspace_bytes(C.byref(_with(L.NormArgs, NORM))) > 0
    a = _with(L.NormArgs, NORM, **bad)
    assert lib.ossm_norm_workspace_bytes(C.byref(a)) == 0
    assert lib.ossm_residual_norm_fwd(C.byref(a), None) == L.OSSM_EINVAL
    assert lib.ossm_residual_norm_bwd(C.byref(a), 4096, 1 << 40, None) == L.OSSM_EINVAL


def test_no_cpu_path():
    t = torch.zeros(4, 64)
    for call in (lambda: O.linear_cross_entropy(t, t, torch.zeros(4, dtype=torch.int64)),
                 lambda: O.embed_tokens(torch.zeros(4, dtype=torch.int64), t), lambda: O.residual_norm(t, t)):
        with pytest.raises(RuntimeError):
            call()
