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

from . import _lib as L
from .sdpc_kernel import _WS_ATTN, _need_cuda, _ptr, _workspace

_DT_ATTN = {torch.bfloat16: L.OSSM_BF16, torch.float16: L.OSSM_F16}
_DT_SAMPLE = {torch.float32: L.OSSM_F32, torch.bfloat16: L.OSSM_BF16, torch.float16: L.OSSM_F16}


def _tma_rows(t):
    """t [rows, heads, head_dim] itself where its strides and base suit 16-byte
    accesses, else a contiguous copy."""
    st, sh, sd = t.stride()
    ok = (sd == 1 and st % 8 == 0 and sh % 8 == 0 and (st > 0 or t.shape[0] <= 1) and (sh > 0 or t.shape[1] <= 1)
          and t.data_ptr() % 16 == 0)
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _index(t, n, what, dev):
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n or t.device != dev:
        raise ValueError(f"packed_attention: {what} must be an int32 vector of {n} on {dev}")
    return t if t.is_contiguous() else t.contiguous()


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
    _need_cuda(q, k, v, cu_seqlens_q, cu_seqlens_k, kv_lengths, out)
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape:
        raise ValueError(f"packed_attention: q [Tq,H,hd] and k, v [Tk,Hkv,hd] expected, got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    dt = _DT_ATTN.get(q.dtype)
    if dt is None or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"packed_attention: q, k, v must share bf16 or fp16, got {q.dtype}, {k.dtype}, {v.dtype}")
    Tq, H, hd = q.shape
    Tk, Hkv, _ = k.shape
    if k.shape[2] != hd or hd % 8 or not 8 <= hd <= 128 or Hkv < 1 or H < 1 or H % Hkv:
        raise ValueError(f"packed_attention: head_dim {hd} (a multiple of 8 up to 128, the same in k) or heads "
                         f"{H} / {Hkv} (a multiple) not supported")
    dev = q.device
    if k.device != dev or v.device != dev:
        raise ValueError("packed_attention: q, k, v must be on one device")
    B = cu_seqlens_q.shape[0] - 1
    if not 1 <= B <= 16384:
        raise ValueError(f"packed_attention: 1 to 16384 sequences, got {B}")
    cu_q = _index(cu_seqlens_q, B + 1, "cu_seqlens_q", dev)
    cu_k = cu_q if cu_seqlens_k is None else _index(cu_seqlens_k, B + 1, "cu_seqlens_k", dev)
    if kv_lengths is not None:
        kv_lengths = _index(kv_lengths, B, "kv_lengths", dev)
    if window is not None and window < 1:
        raise ValueError(f"packed_attention: window must be at least 1, got {window}")
    scale = 1.0 / math.sqrt(hd) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"packed_attention: scale must be positive and finite, got {scale}")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        raise NotImplementedError("packed_attention has no backward pass: call it under torch.no_grad()")
    if out is None:
        out = torch.empty(Tq, H, hd, dtype=q.dtype, device=dev)
    else:
        if out.shape != q.shape or out.dtype != q.dtype or out.device != dev:
            raise ValueError("packed_attention: out must have q's shape, dtype and device")
        if _tma_rows(out) is not out:
            raise ValueError("packed_attention: out needs a unit channel stride and 16-byte aligned rows")
    if Tq == 0:
        return out
    q, k, v = _tma_rows(q), _tma_rows(k), _tma_rows(v)
    a = L.AttnArgs(B, H, Hkv, hd, Tq, Tk, int(max_seqlen_q), dt, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                   out.data_ptr(), q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
                   out.stride(0), out.stride(1), cu_q.data_ptr(), cu_k.data_ptr(), _ptr(kv_lengths),
                   min(int(window), 0x7fffffff) if window is not None else 0, scale)
    lib = L.lib()
    ref = L.C.byref(a)
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _attention(lib, ref, dev, out)
    return _attention(lib, ref, dev, out)


def _attention(lib, ref, dev, out):
    nbytes = lib.ossm_attn_workspace_bytes(ref)
    if nbytes == 0:
        L.check(L.OSSM_EINVAL, "packed_attention (argument check)")
    stream = torch.cuda.current_stream(dev)
    ws = _workspace(dev, stream, nbytes, cache=_WS_ATTN)
    L.check(lib.ossm_attention_fwd(ref, ws.data_ptr(), ws.numel(), stream.cuda_stream), "packed_attention")
    return out


def _setting(x, dtype, B, what, dev):
    """(scalar, pointer, tensor to keep) of a setting given as a number or as a tensor [B]."""
    if isinstance(x, torch.Tensor):
        if x.dim() != 1 or x.shape[0] != B or x.device != dev:
            raise ValueError(f"sample_tokens: {what} must be a number or a vector of {B} on {dev}")
        x = x.to(dtype).contiguous()
        return 0, x.data_ptr(), x
    return x, None, None


def sample_tokens(logits: torch.Tensor, noise: Optional[torch.Tensor] = None, *,
                  temperature: Union[float, torch.Tensor] = 1.0, top_k: Union[int, torch.Tensor] = 0,
                  top_p: Union[float, torch.Tensor] = 1.0, min_p: Union[float, torch.Tensor] = 0.0,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The next token of each row of logits [B, V] (fp32, bf16 or fp16, CUDA).

    Candidates are ordered by logit, at equal logits by index.  The first
    ``top_k`` stay (0: all); of these the shortest prefix whose probability
    under softmax(logits / temperature) over the first top_k reaches ``top_p``
    (1: all; at least one stays); of these the ones at least ``min_p`` times
    as likely as the first.  The token is the candidate with the largest
    ``logit / temperature - log(noise)``, ties to the lowest index: with
    ``noise`` [B, V] fp32 from the standard exponential distribution
    (``torch.empty(B, V).exponential_()``) it is drawn from the softmax over
    the candidates, and the same noise gives the same token.

    ``noise=None`` or a temperature of 0 takes the largest logit.  Each
    setting is a number or a tensor [B] on the device (float32; top_k int32),
    one value a row; a tensor's temperature that is not positive is 0.  NaN
    and -inf logits are never drawn; a row that has nothing else gives -1.
    Returns int64 [B] (``out`` if given)."""
    _need_cuda(logits, noise, out)
    if logits.dim() != 2 or logits.dtype not in _DT_SAMPLE:
        raise ValueError(f"sample_tokens: logits [B,V] in fp32, bf16 or fp16 expected, got {tuple(logits.shape)} "
                         f"{logits.dtype}")
    B, V = logits.shape
    dev = logits.device
    if V < 1:
        raise ValueError("sample_tokens: no candidates")
    if noise is not None:
        if noise.shape != logits.shape or noise.dtype != torch.float32 or noise.device != dev:
            raise ValueError("sample_tokens: noise must be fp32 with the logits' shape and device")
        if noise.stride(1) != 1:
            noise = noise.contiguous()
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    if out is None:
        out = torch.empty(B, dtype=torch.int64, device=dev)
    elif out.shape != (B,) or out.dtype != torch.int64 or out.device != dev or not out.is_contiguous():
        raise ValueError("sample_tokens: out must be a contiguous int64 [B] on the logits' device")
    t, t_row, t_keep = _setting(temperature, torch.float32, B, "temperature", dev)
    k, k_row, k_keep = _setting(top_k, torch.int32, B, "top_k", dev)
    p, p_row, p_keep = _setting(top_p, torch.float32, B, "top_p", dev)
    m, m_row, m_keep = _setting(min_p, torch.float32, B, "min_p", dev)
    if not (0.0 <= t < math.inf and k >= 0 and 0.0 <= p <= 1.0 and 0.0 <= m <= 1.0):
        raise ValueError(f"sample_tokens: temperature {t} must be >= 0 and finite, top_k {k} >= 0, top_p {p} and "
                         f"min_p {m} in [0, 1]")
    if B == 0:
        return out
    a = L.SampleArgs(B, V, logits.data_ptr(), _DT_SAMPLE[logits.dtype], logits.stride(0), _ptr(noise),
                     0 if noise is None else noise.stride(0), 1.0 / t if t > 0 else 0.0, p, m, min(int(k), V), t_row,
                     p_row, m_row, k_row, out.data_ptr())
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _sample(a, dev, out)
    return _sample(a, dev, out)


def _sample(a, dev, out):
    L.check(L.lib().ossm_sample_tokens(L.C.byref(a), torch.cuda.current_stream(dev).cuda_stream), "sample_tokens")
    return out
