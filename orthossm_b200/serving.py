"""Serving operators: attention over packed prompts and over a cache, and the
choice of the next token.

The reference stops at the logits of dense batches (model.py:23-187) and runs
its local attention as a masked SDPA over one batch (slr_module.py:83-243); a
server has prompts of different lengths, a cache, and tokens to draw.  Both
operators run in this package's sm_100a kernels behind the C ABI
(``ossm_attention_fwd``, ``ossm_sample_tokens``) on the current stream, and
have no backward pass.
"""
from __future__ import annotations

import math
from typing import Optional, Union

import torch
from torch.autograd import forward_ad

from . import _lib as L
from .sdpc_kernel import _WS_ATTN, _captured_workspace, _need_cuda, _ptr, _workspace

_DT_ATTN = {torch.bfloat16: L.OSSM_BF16, torch.float16: L.OSSM_F16}
_DT_SAMPLE = {torch.float32: L.OSSM_F32, torch.bfloat16: L.OSSM_BF16, torch.float16: L.OSSM_F16}


_raw_stream = torch._C._cuda_getCurrentRawStream  # the current stream's handle without a Stream object (2 us)
# (device index, stream) -> (workspace address, bytes) of the tensors in _WS_ATTN: one size fits all
# arguments, so none is ever replaced
_ATTN_WS: dict = {}


def _rows_ok(st, sh, sd, n, heads, ptr):
    """Strides and base of a [n, heads, head_dim] tensor that suit 16-byte accesses."""
    return sd == 1 and not (st % 8 or sh % 8 or ptr % 16) and (st > 0 or n <= 1) and (sh > 0 or heads <= 1)


def _tma_rows(t):
    """t [rows, heads, head_dim] itself where it can be read as it is, else a contiguous copy."""
    return t if _rows_ok(*t.stride(), t.shape[0], t.shape[1], t.data_ptr()) else \
        t.clone(memory_format=torch.contiguous_format)


_I32 = torch.int32


def _vector(t, n, dev):
    return t.dtype is _I32 and t.shape == (n,) and t.get_device() == dev


def _refuse_attention(q, k, v, cu_q, cu_k, kv_lengths, window, scale, out):
    """Raises for the first argument of packed_attention that does not fit."""
    _need_cuda(q, k, v, cu_q, cu_k, kv_lengths, out)
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape:
        raise ValueError(f"packed_attention: q [Tq,H,hd] and k, v [Tk,Hkv,hd] expected, got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    if q.dtype not in _DT_ATTN or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"packed_attention: q, k, v must share bf16 or fp16, got {q.dtype}, {k.dtype}, {v.dtype}")
    dev = q.get_device()
    if k.get_device() != dev or v.get_device() != dev:
        raise ValueError("packed_attention: q, k, v must be on one device")
    B = cu_q.shape[0] - 1 if cu_q.dim() == 1 else 0
    if not 1 <= B <= 16384:
        raise ValueError(f"packed_attention: 1 to 16384 sequences, got {B}")
    for t, n, what in ((cu_q, B + 1, "cu_seqlens_q"), (cu_k, B + 1, "cu_seqlens_k"), (kv_lengths, B, "kv_lengths")):
        if t is not None and not _vector(t, n, dev):
            raise ValueError(f"packed_attention: {what} must be an int32 vector of {n} on {q.device}")
    if window is not None and window < 1:
        raise ValueError(f"packed_attention: window must be at least 1, got {window}")
    if not 0.0 < scale < math.inf:
        raise ValueError(f"packed_attention: scale must be positive and finite, got {scale}")
    if out is not None:
        if out.shape != q.shape or out.dtype != q.dtype or out.get_device() != dev:
            raise ValueError("packed_attention: out must have q's shape, dtype and device")
        if _tma_rows(out) is not out:
            raise ValueError("packed_attention: out needs a unit channel stride and 16-byte aligned rows")
    hd, H, Hkv = q.shape[2], q.shape[1], k.shape[1]
    raise ValueError(f"packed_attention: head_dim {hd} and {k.shape[2]} (equal, a multiple of 8, at most 128) or heads "
                     f"{H} / {Hkv} (a multiple) not supported")


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                     cu_seqlens_k: Optional[torch.Tensor] = None, *, max_seqlen_q: int,
                     kv_lengths: Optional[torch.Tensor] = None, window: Optional[int] = None,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal softmax attention of sequences packed along the first axis.

    q: [Tq, H, hd]; k, v: [Tk, Hkv, hd], bf16 or fp16 (CUDA), H a multiple of
    Hkv (query head h reads key head h // (H // Hkv)), hd a multiple of 8, at
    most 128.  Token and head strides are free.
    cu_seqlens_q / cu_seqlens_k: [B+1] int32 on the device, non-decreasing:
    sequence b owns queries cu_seqlens_q[b] .. cu_seqlens_q[b+1] and the keys
    of the same range of cu_seqlens_k (default: cu_seqlens_q).  At most 16384
    sequences.
    kv_lengths: [B] int32 on the device: only the first kv_lengths[b] of a
    sequence's key slots are held (a cache [B, slots, Hkv, hd] viewed as
    [B*slots, Hkv, hd], with cu_seqlens_k = slots * arange(B+1)).
    max_seqlen_q: the most queries a sequence has, known on the host (it
    chooses the kernels: a small one runs the form for single tokens).

    The queries are the sequence's last tokens: query i of Lq stands at
    position i + Lk - Lq and sees the keys at or before it, with ``window``
    the last ``window`` of them.  A query that sees none gives zeros.  Keys
    and values that a query does not see do not reach its output, whatever
    they hold.  scale: default 1 / sqrt(hd).  Rows of q outside every sequence
    are not written.  Returns [Tq, H, hd] in q's dtype (``out`` if given)."""
    dev = q.get_device()
    dt = _DT_ATTN.get(q.dtype)
    scale_ = scale
    ok = dev >= 0 and dt is not None and q.dim() == 3 and k.dim() == 3 and cu_seqlens_q.dim() == 1
    if ok:
        Tq, H, hd = q.shape
        Tk, Hkv, hdk = k.shape
        B = cu_seqlens_q.shape[0] - 1
        cu_k = cu_seqlens_q if cu_seqlens_k is None else cu_seqlens_k
        scale_ = hd ** -0.5 if scale is None and hd else scale
        ok = (v.shape == k.shape and k.dtype == q.dtype and v.dtype == q.dtype and k.get_device() == dev
              and v.get_device() == dev and hdk == hd and hd % 8 == 0 and 8 <= hd <= 128 and Hkv > 0 and H > 0
              and H % Hkv == 0 and 1 <= B <= 16384 and _vector(cu_seqlens_q, B + 1, dev)
              and (cu_k is cu_seqlens_q or _vector(cu_k, B + 1, dev))
              and (kv_lengths is None or _vector(kv_lengths, B, dev)) and (window is None or window >= 1)
              and 0.0 < scale_ < math.inf
              and (out is None or (out.shape == q.shape and out.dtype == q.dtype and out.get_device() == dev)))
    if not ok:
        _refuse_attention(q, k, v, cu_seqlens_q, cu_seqlens_k, kv_lengths, window, 1.0 if scale_ is None else scale_,
                          out)
    if (q.requires_grad or k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        raise NotImplementedError("packed_attention has no backward pass: call it under torch.no_grad()")
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in (q, k, v)):
        raise NotImplementedError("packed_attention has no forward-mode derivative")
    ot, oh = H * hd, hd
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        ot, oh, unit = out.stride()
        if not _rows_ok(ot, oh, unit, Tq, H, out.data_ptr()):
            _refuse_attention(q, k, v, cu_seqlens_q, cu_seqlens_k, kv_lengths, window, scale_, out)
    if Tq == 0:
        return out
    (qt, qh, qu), (kt, kh, ku), (vt, vh, vu) = q.stride(), k.stride(), v.stride()
    qp, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if (qu != 1 or ku != 1 or vu != 1 or (qt | qh | kt | kh | vt | vh) & 7 or (qp | kp | vp) & 15
            or not (qt and qh and kt and kh and vt and vh)):
        q, k, v = _tma_rows(q), _tma_rows(k), _tma_rows(v)  # copies of what cannot be read as it is
        (qt, qh, _), (kt, kh, _), (vt, vh, _) = q.stride(), k.stride(), v.stride()
        qp, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if not cu_seqlens_q.is_contiguous():
        cu_seqlens_q, cu_k = cu_seqlens_q.contiguous(), cu_k.contiguous()
    elif not cu_k.is_contiguous():
        cu_k = cu_k.contiguous()
    if kv_lengths is not None and not kv_lengths.is_contiguous():
        kv_lengths = kv_lengths.contiguous()
    a = L.AttnArgs(B, H, Hkv, hd, Tq, Tk, min(int(max_seqlen_q), 0x7fffffff), dt, qp, kp, vp, out.data_ptr(), qt, qh,
                   kt, kh, vt, vh, ot, oh, cu_seqlens_q.data_ptr(), cu_k.data_ptr(),
                   None if kv_lengths is None else kv_lengths.data_ptr(),
                   0 if window is None else min(int(window), 0x7fffffff), scale_, L.OSSM_ATTN_NO_CAPTURE)
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            _attention(a, dev)
    else:
        _attention(a, dev)
    return out


def _attn_workspace(device, stream, nbytes, capturing):
    """The stream's workspace, or under capture one of the graph's own: a graph
    may be replayed beside calls on the stream that it was captured on."""
    if capturing:
        return _captured_workspace("attention", device, stream.cuda_stream, nbytes, L.OSSM_ATTN_WS_ZERO)
    return _workspace(device, stream, nbytes, cache=_WS_ATTN)


def _attention(a, dev):
    lib = L.lib()
    stream = _raw_stream(dev)
    ref = L.C.byref(a)
    ws = _ATTN_WS.get((dev, stream))
    status = L.OSSM_EWORKSPACE if ws is None else lib.ossm_attention_fwd(ref, ws[0], ws[1], stream)
    if status == L.OSSM_EWORKSPACE:  # the first call on this stream, or one that is captured
        nbytes = lib.ossm_attn_workspace_bytes(ref)
        if nbytes == 0:
            L.check(L.OSSM_EINVAL, "packed_attention (argument check)")
        device = torch.device("cuda", dev)
        capturing = torch.cuda.is_current_stream_capturing()
        t = _attn_workspace(device, torch.cuda.current_stream(device), nbytes, capturing)
        if capturing:
            a.flags = 0
        else:
            _ATTN_WS[dev, stream] = t.data_ptr(), t.numel()
        status = lib.ossm_attention_fwd(ref, t.data_ptr(), t.numel(), stream)
    if status != L.OSSM_OK:
        L.check(status, "packed_attention")


def _setting(x, dtype, B, what, dev, most=None):
    """A setting given as a tensor [B], in the kernel's type; of counts, ``most``
    and more are the same."""
    if x.dim() != 1 or x.shape[0] != B or x.get_device() != dev:
        raise ValueError(f"sample_tokens: {what} must be a number or a vector of {B} on the logits' device")
    if x.dtype != dtype:
        x = (x if most is None else x.clamp(0, most)).to(dtype)  # a larger type's counts do not wrap
    return x.contiguous()


def sample_tokens(logits: torch.Tensor, noise: Optional[torch.Tensor] = None, *,
                  temperature: Union[float, torch.Tensor] = 1.0, top_k: Union[int, torch.Tensor] = 0,
                  top_p: Union[float, torch.Tensor] = 1.0, min_p: Union[float, torch.Tensor] = 0.0,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The next token of each row of logits [B, V] (fp32, bf16 or fp16, CUDA;
    V below 2^23, B at most 2^27).

    Candidates are ordered by logit, at equal logits by index.  The first
    ``top_k`` stay (0: all); of these the shortest prefix whose probability
    under softmax(logits / temperature) over the first top_k reaches ``top_p``
    (1: all; at least one stays); of these the ones at least ``min_p`` times
    as likely as the first.  The token is the candidate with the largest
    ``logit / temperature - log(noise)``, ties to the lowest index: with
    ``noise`` [B, V] fp32 from the standard exponential distribution
    (``torch.empty(B, V).exponential_()``) it is drawn from the softmax over
    the candidates, and the same row and noise give the same token, alone or
    in any batch.

    ``noise=None`` or a temperature of 0 takes the largest logit.  Each
    setting is a number or a tensor [B] on the device (float32; top_k int32),
    one value a row; a tensor's temperature that is not positive is 0, and an
    infinite one makes all candidates equally likely.  NaN and -inf logits are
    never drawn; a row that has nothing else gives -1.
    Returns int64 [B] (``out`` if given)."""
    _need_cuda(logits, noise, out)
    dt = _DT_SAMPLE.get(logits.dtype)
    if logits.dim() != 2 or dt is None:
        raise ValueError(f"sample_tokens: logits [B,V] in fp32, bf16 or fp16 expected, got {tuple(logits.shape)} "
                         f"{logits.dtype}")
    B, V = logits.shape
    dev = logits.get_device()
    if not 1 <= V < 1 << 23 or B > 1 << 27:
        raise ValueError(f"sample_tokens: 1 to 2^23 - 1 candidates in at most 2^27 rows, got {V} in {B}")
    lst, unit = logits.stride()
    if unit != 1:
        logits = logits.contiguous()
        lst = logits.stride(0)
    nst = 0
    if noise is not None:
        if noise.shape != logits.shape or noise.dtype != torch.float32 or noise.get_device() != dev:
            raise ValueError("sample_tokens: noise must be fp32 with the logits' shape and device")
        nst, unit = noise.stride()
        if unit != 1:
            noise = noise.contiguous()
            nst = noise.stride(0)
    if out is None:
        out = torch.empty(B, dtype=torch.int64, device=logits.device)
    elif out.shape != (B,) or out.dtype != torch.int64 or out.get_device() != dev or not out.is_contiguous():
        raise ValueError("sample_tokens: out must be a contiguous int64 [B] on the logits' device")
    t, k, p, m = temperature, top_k, top_p, min_p
    t_row = k_row = p_row = m_row = None  # kept until the launch
    if isinstance(t, torch.Tensor):
        t_row, t = _setting(t, torch.float32, B, "temperature", dev), 0.0
    if isinstance(k, torch.Tensor):
        k_row, k = _setting(k, torch.int32, B, "top_k", dev, V), 0
    if isinstance(p, torch.Tensor):
        p_row, p = _setting(p, torch.float32, B, "top_p", dev), 0.0
    if isinstance(m, torch.Tensor):
        m_row, m = _setting(m, torch.float32, B, "min_p", dev), 0.0
    if not (0.0 <= t < math.inf and k >= 0 and 0.0 <= p <= 1.0 and 0.0 <= m <= 1.0):
        raise ValueError(f"sample_tokens: temperature {t} must be >= 0 and finite, top_k {k} >= 0, top_p {p} and "
                         f"min_p {m} in [0, 1]")
    if B == 0:
        return out
    a = L.SampleArgs(B, V, logits.data_ptr(), dt, lst, _ptr(noise), nst, max(1.0 / t, 2.0 ** -149) if t > 0 else 0.0, p, m,
                     min(int(k), V), _ptr(t_row), _ptr(p_row), _ptr(m_row), _ptr(k_row), out.data_ptr())
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            status = L.lib().ossm_sample_tokens(L.C.byref(a), _raw_stream(dev))
    else:
        status = L.lib().ossm_sample_tokens(L.C.byref(a), _raw_stream(dev))
    if status != L.OSSM_OK:
        L.check(status, "sample_tokens")
    return out
