"""Training operators: token embeddings, the norms around a block with its
residual, and the loss from hidden states without the logits.

The reference's training script composes them of torch's own operators
(model.py:23-187, sdpc_engine.py:420-426): nn.Embedding, nn.RMSNorm, and a cross
entropy of whole logits.  Here each is one operator with its gradients, in this
package's sm_100a kernels behind the C ABI (``ossm_embed_*``,
``ossm_residual_norm_*``, ``ossm_lce_*``), on the current stream.  Results
depend on the arguments alone: no atomics add up values.  Gradients of
gradients and forward-mode derivatives are refused.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L
from .sdpc_kernel import _WS_TRAIN, _captured_workspace, _is_capturing, _need_cuda, _ptr, _workspace

_DT = {torch.float32: L.OSSM_F32, torch.bfloat16: L.OSSM_BF16, torch.float16: L.OSSM_F16}
_INTS = (torch.int64, torch.int32, torch.int16, torch.uint8, torch.int8)
_NORMS = {"rms": L.OSSM_NORM_RMS, "layer": L.OSSM_NORM_LAYER}
_REDUCTIONS = {"none": L.OSSM_LOSS_NONE, "mean": L.OSSM_LOSS_MEAN, "sum": L.OSSM_LOSS_SUM}

_raw_stream = torch._C._cuda_getCurrentRawStream  # the current stream's handle without a Stream object (2 us)
_STATUS: dict = {}  # (device index, stream) -> address of the status word in the tensor of _WS_TRAIN


def _no_tangents(what, *ts):
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                              for t in ts):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def _needs_grad(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _status(dev, stream):
    """Address of the stream's status word, which ``workspace_status`` reads."""
    at = _STATUS.get((dev, stream))
    if at is None or _is_capturing():
        device = torch.device("cuda", dev)
        if _is_capturing():
            return _captured_workspace("training", device, stream, 256, 256).data_ptr() + 8
        at = _workspace(device, torch.cuda.current_stream(device), 256, cache=_WS_TRAIN).data_ptr() + 8
        _STATUS[dev, stream] = at
    return at


def _run(dev, what, fn, a, ws_bytes=None):
    """Calls a C entry point on the current stream of device ``dev``."""
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _run(dev, what, fn, a, ws_bytes)
    if ws_bytes is None:
        status = fn(L.C.byref(a), _raw_stream(dev))
    else:
        if ws_bytes == 0:
            L.check(L.OSSM_EINVAL, f"{what} (argument check)")
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=torch.device("cuda", dev))
        status = fn(L.C.byref(a), ws.data_ptr(), ws_bytes, _raw_stream(dev))
    if status != L.OSSM_OK:
        L.check(status, what)


def _rows(t, d, align=False):
    """t [..., d] as rows [T, d] with a unit channel stride, and their stride;
    a copy where it cannot be read as it is.  ``align``: rows start on 16 bytes."""
    r = t if t.dim() == 2 else t.reshape(-1, d)
    st, unit = r.stride()
    n = r.shape[0]
    if n <= 1:
        st = d
    if (unit != 1 and d > 1) or st < d or (align and (st * r.element_size() % 16 or r.data_ptr() % 16)):
        r, st = r.clone(memory_format=torch.contiguous_format), d
    return r, st


# ----------------------------------------------------------------------------
# loss
# ----------------------------------------------------------------------------

def _lce_args(h, hst, w, wst, targets, ignore, z_loss, reduction, loss, lse, dev):
    return L.LceArgs(h.shape[0], h.shape[1], w.shape[0], _DT[h.dtype], h.data_ptr(), hst, w.data_ptr(), wst,
                     targets.data_ptr(), ignore, z_loss, reduction, _ptr(loss), lse.data_ptr(), None, None, None,
                     _status(dev, _raw_stream(dev)))


def _lce_forward(hidden, weight, targets, ignore, z_loss, reduction):
    d, dev = hidden.shape[-1], hidden.get_device()
    h, hst = _rows(hidden, d, align=True)
    w, wst = _rows(weight, d, align=True)
    t = targets.reshape(-1).contiguous()
    T = h.shape[0]
    if T == 0:
        return torch.zeros((0,) if reduction == 0 else (), device=h.device), torch.empty(0, device=h.device)
    loss = torch.empty(T if reduction == 0 else (), device=h.device)
    lse = torch.empty(T, device=h.device)
    a = _lce_args(h, hst, w, wst, t, ignore, z_loss, reduction, loss, lse, dev)
    lib = L.lib()
    _run(dev, "linear_cross_entropy", lib.ossm_lce_fwd, a, lib.ossm_lce_workspace_bytes(L.C.byref(a), 0))
    return loss, lse


class _LceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore, z_loss, reduction):
        loss, lse = _lce_forward(hidden, weight, targets, ignore, z_loss, reduction)
        ctx.save_for_backward(hidden, weight, targets, lse)
        ctx.opts = ignore, z_loss, reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        hidden, weight, targets, lse = ctx.saved_tensors
        ignore, z_loss, reduction = ctx.opts
        want_h, want_w = ctx.needs_input_grad[:2]
        if lse.numel() == 0:
            return (torch.zeros_like(hidden) if want_h else None, torch.zeros_like(weight) if want_w else None,
                    None, None, None, None)
        d, dev = hidden.shape[-1], hidden.get_device()
        h, hst = _rows(hidden, d, align=True)
        w, wst = _rows(weight, d, align=True)
        t = targets.reshape(-1).contiguous()
        g = g.float().contiguous()
        dh = torch.empty(hidden.shape, dtype=hidden.dtype, device=hidden.device) if want_h else None
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device) if want_w else None
        a = _lce_args(h, hst, w, wst, t, ignore, z_loss, reduction, None, lse, dev)
        a.grad_loss, a.grad_hidden, a.grad_weight = g.data_ptr(), _ptr(dh), _ptr(dw)
        lib = L.lib()
        _run(dev, "linear_cross_entropy backward", lib.ossm_lce_bwd, a,
             lib.ossm_lce_workspace_bytes(L.C.byref(a), 1))
        return dh, dw, None, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *,
                         ignore_index: int = -100, z_loss: float = 0.0, reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of the logits ``hidden @ weight.T`` against ``targets``,
    without the logits: they are formed and used a tile at a time, forward and
    again backward.

    hidden: [..., d], weight: [V, d], bf16 or fp16 (CUDA), d a multiple of 8;
    targets: [...] integers.  A token whose target is ``ignore_index`` has no
    loss and no gradient, and its state does not reach anything, whatever it
    holds.  Another target outside 0 .. V-1 gives NaN.
    ``z_loss`` adds ``z_loss * lse**2`` to a token's loss (lse: log of the sum
    of the exponentials of its logits).
    reduction: "mean" over the tokens that have a target (0 if none has),
    "sum", or "none": the losses [...], 0 where there is no target.
    Returns fp32.  Differentiable in ``hidden`` and ``weight``; the gradients
    have their types.  Memory beside inputs and gradients: a piece of the
    logits' gradient of at most 512 MB (or 4096 of the V columns, if more) in
    the inputs' type and, if that is not all columns, fp32 sums of hidden's
    size; with ignored tokens a copy of the others' states."""
    _need_cuda(hidden, weight, targets)
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear_cross_entropy: hidden [..., d] and weight [V, d] expected, got {tuple(hidden.shape)} "
                         f"and {tuple(weight.shape)}")
    if hidden.dtype not in (torch.bfloat16, torch.float16) or weight.dtype != hidden.dtype:
        raise ValueError(f"linear_cross_entropy: hidden and weight must share bf16 or fp16, got {hidden.dtype}, "
                         f"{weight.dtype}")
    V, d = weight.shape
    if d % 8 or not 8 <= d <= 1 << 16 or not 1 <= V <= 1 << 27:
        raise ValueError(f"linear_cross_entropy: d a multiple of 8 up to 65536 and V from 1 to 2^27 expected, got {d} "
                         f"and {V}")
    if targets.shape != hidden.shape[:-1] or targets.dtype not in _INTS:
        raise ValueError(f"linear_cross_entropy: integer targets of shape {tuple(hidden.shape[:-1])} expected, got "
                         f"{tuple(targets.shape)} {targets.dtype}")
    if targets.numel() > 1 << 27:
        raise ValueError(f"linear_cross_entropy: at most 2^27 tokens, got {targets.numel()}")
    dev = hidden.get_device()
    if weight.get_device() != dev or targets.get_device() != dev:
        raise ValueError("linear_cross_entropy: hidden, weight and targets must be on one device")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"linear_cross_entropy: reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if not 0.0 <= z_loss < math.inf:
        raise ValueError(f"linear_cross_entropy: z_loss must be finite and not negative, got {z_loss}")
    _no_tangents("linear_cross_entropy", hidden, weight)
    if targets.dtype != torch.int64:
        targets = targets.long()
    args = (hidden, weight, targets, int(ignore_index), float(z_loss), _REDUCTIONS[reduction])
    loss = _LceFn.apply(*args) if _needs_grad(hidden, weight) else _lce_forward(*args)[0]
    return loss.view(targets.shape) if reduction == "none" and loss.dim() != targets.dim() else loss


# ----------------------------------------------------------------------------
# embeddings
# ----------------------------------------------------------------------------

def _embed_forward(ids, weight, scale):
    V, d = weight.shape
    w, wst = _rows(weight, d)
    i = ids.contiguous()
    out = torch.empty(*ids.shape, d, dtype=weight.dtype, device=weight.device)
    a = L.EmbedArgs(i.numel(), d, V, _DT[weight.dtype], i.data_ptr(), w.data_ptr(), wst, scale, out.data_ptr(),
                    None, 0, None)
    if out.numel():
        _run(weight.get_device(), "embed_tokens", L.lib().ossm_embed_fwd, a)
    return out


class _EmbedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale):
        ctx.save_for_backward(ids)
        ctx.opts = weight.shape, weight.dtype, scale
        return _embed_forward(ids, weight, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        ids, = ctx.saved_tensors
        (V, d), dtype, scale = ctx.opts
        g, gst = _rows(g, d)
        i = ids.contiguous()
        dw = torch.empty(V, d, dtype=dtype, device=g.device)
        a = L.EmbedArgs(i.numel(), d, V, _DT[dtype], i.data_ptr(), None, 0, scale, None, g.data_ptr(), gst,
                        dw.data_ptr())
        lib = L.lib()
        _run(dw.get_device(), "embed_tokens backward", lib.ossm_embed_bwd, a,
             lib.ossm_embed_workspace_bytes(L.C.byref(a)))
        return None, dw, None


def embed_tokens(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0) -> torch.Tensor:
    """``scale * weight[ids]``, zeros where an id is no row of the weight (a
    padded position can hold -1).

    ids: integers of any shape, weight: [V, d] fp32, bf16 or fp16 (CUDA), V
    below 2^27, d at most 65536.  Returns [..., d] in weight's dtype.
    Differentiable in ``weight``: a row's gradient is the scaled sum over the
    positions that hold its token, added up in fp32 in their order (cut into
    fixed pieces) and rounded once; rows without a position get zeros."""
    _need_cuda(ids, weight)
    if weight.dim() != 2 or weight.dtype not in _DT:
        raise ValueError(f"embed_tokens: weight [V, d] in fp32, bf16 or fp16 expected, got {tuple(weight.shape)} "
                         f"{weight.dtype}")
    V, d = weight.shape
    if not (1 <= V < 1 << 27 and 1 <= d <= 1 << 16):
        raise ValueError(f"embed_tokens: V from 1 below 2^27 and d from 1 to 65536 expected, got {V} and {d}")
    if ids.dtype not in _INTS or ids.numel() >= 1 << 31:
        raise ValueError(f"embed_tokens: below 2^31 integer ids expected, got {ids.numel()} {ids.dtype}")
    if ids.get_device() != weight.get_device():
        raise ValueError("embed_tokens: ids and weight must be on one device")
    if not math.isfinite(scale):
        raise ValueError(f"embed_tokens: scale must be finite, got {scale}")
    _no_tangents("embed_tokens", weight)
    if ids.dtype != torch.int64:
        ids = ids.long()
    return (_EmbedFn.apply if _needs_grad(weight) else _embed_forward)(ids, weight, float(scale))


# ----------------------------------------------------------------------------
# residual and norms
# ----------------------------------------------------------------------------

def _vec(t):
    """A parameter's address and type code (0 where there is none)."""
    return (None, 0) if t is None else (t.data_ptr(), _DT[t.dtype])


def _norm_args(T, d, sdt, dt, gate, gate_kind, gst, scale, norm, post, eps, post_eps, w, b, pw, pb):
    (wp, wd), (bp, bd), (pwp, pwd), (pbp, pbd), (gp, gd) = _vec(w), _vec(b), _vec(pw), _vec(pb), _vec(gate)
    return L.NormArgs(T, d, _DT[sdt], _DT[dt], None, d, None, d, gp, gate_kind, gd, gst, scale, norm, post, eps,
                      post_eps, wp, bp, pwp, pbp, wd, bd, pwd, pbd)


def _gate_rows(gate, kind, d):
    if gate is None:
        return None, 0
    if kind == L.OSSM_GATE_FULL:
        return _rows(gate, d)
    return gate.contiguous(), 0


def _norm_forward(x, y, w, b, gate, pw, pb, opts, want_stats):
    norm, post, kind, scale, eps, post_eps, dt = opts
    d, dev = x.shape[-1], x.get_device()
    xr, xst = _rows(x, d)
    T = xr.shape[0]
    w, b, pw, pb = (None if t is None else t.contiguous() for t in (w, b, pw, pb))
    g, gst = _gate_rows(gate, kind, d)
    a = _norm_args(T, d, x.dtype, dt, g, kind, gst, scale, norm, post, eps, post_eps, w, b, pw, pb)
    a.status = _status(dev, _raw_stream(dev))
    a.x, a.x_stride = xr.data_ptr(), xst
    r = x
    if y is not None:
        yr, a.y_stride = _rows(y, d)
        r = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        a.y, a.r = yr.data_ptr(), r.data_ptr()
    h = torch.empty(x.shape, dtype=dt, device=x.device)
    a.h = h.data_ptr()
    stats = torch.empty(4 if post else 2, T, device=x.device) if want_stats else None
    a.stats = _ptr(stats)
    if T:
        _run(dev, "residual_norm", L.lib().ossm_residual_norm_fwd, a)
    return r, h, stats


class _NormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, w, b, gate, pw, pb, opts):
        r, h, stats = _norm_forward(x, y, w, b, gate, pw, pb, opts, True)
        ctx.full = bool(opts[1]) or gate is not None
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*((x, y) if ctx.full else (r, None)), w, b, gate, pw, pb, stats)
        ctx.opts = opts
        ctx.has_y = y is not None
        return r, h

    @staticmethod
    @once_differentiable
    def backward(ctx, gr, gh):
        x, y, w, b, gate, pw, pb, stats = ctx.saved_tensors
        norm, post, kind, scale, eps, post_eps, dt = ctx.opts
        if gr is None and gh is None:
            return (None,) * 8
        d, dev = x.shape[-1], x.get_device()
        xr, xst = _rows(x, d)
        T = xr.shape[0]
        need = ctx.needs_input_grad
        wc, bc, pwc, pbc = (None if t is None else t.contiguous() for t in (w, b, pw, pb))
        g, gst = _gate_rows(gate, kind, d)
        a = _norm_args(T, d, x.dtype, dt, g, kind, gst, scale, norm, post, eps, post_eps, wc, bc, pwc, pbc)
        a.status = _status(dev, _raw_stream(dev))
        a.stats = stats.data_ptr()
        a.x_stride = xst
        if ctx.full:
            yr, a.y_stride = _rows(y, d)
            a.x, a.y = xr.data_ptr(), yr.data_ptr()
        else:
            a.r = xr.data_ptr()
        if gr is not None:
            gr, a.grad_r_stride = _rows(gr, d)
            a.grad_r = gr.data_ptr()
        if gh is not None:
            gh, a.grad_h_stride = _rows(gh, d)
            a.grad_h = gh.data_ptr()
        like = lambda t, want: torch.empty(t.shape, dtype=t.dtype, device=t.device) if want and t is not None else None  # noqa: E731
        dw, db, dpw, dpb = like(w, need[2]), like(b, need[3]), like(pw, need[5]), like(pb, need[6])
        dgate = like(gate, need[4])
        # without a norm or gate of y, and a scale of 1, its gradient is x's
        same = not ctx.full and scale == 1.0 and dt == x.dtype
        dx = like(x, need[0] or (same and need[1]))
        dy = torch.empty(x.shape, dtype=dt, device=x.device) if ctx.has_y and need[1] and not same else None
        a.grad_x, a.grad_y, a.grad_gate = _ptr(dx), _ptr(dy), _ptr(dgate)
        a.grad_weight, a.grad_bias, a.grad_post_weight, a.grad_post_bias = _ptr(dw), _ptr(db), _ptr(dpw), _ptr(dpb)
        lib = L.lib()
        if T:
            _run(dev, "residual_norm backward", lib.ossm_residual_norm_bwd, a,
                 lib.ossm_norm_workspace_bytes(L.C.byref(a)))
        else:
            for t in (dw, db, dpw, dpb, dgate):
                if t is not None:
                    t.zero_()
        if gh is None:  # h was not used: its parameters get nothing
            dw, db = None, None
        if same and ctx.has_y and need[1]:
            dy = dx
        return (dx if need[0] else None), dy, dw, db, dgate, dpw, dpb, None


def _refuse_norm(why):
    raise ValueError("residual_norm: " + why)


def residual_norm(x: torch.Tensor, y: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                  bias: Optional[torch.Tensor] = None, *, norm: str = "rms", eps: float = 1e-6,
                  gate: Optional[torch.Tensor] = None, scale: float = 1.0, post_norm: Optional[str] = None,
                  post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                  post_eps: Optional[float] = None,
                  out_dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """A block's residual and the norms on its two sides, in one pass:

        n = post_norm(y);  r = x + scale * gate * n;  h = norm(r)

    Returns ``(r, h)``: the residual stream and the next block's input.

    x: [..., d], the stream (CUDA); y: the block's output, of its shape, or None
    (then r is x).  d at most 16384.  Both of one dtype (fp32, bf16, fp16), or
    an fp32 stream beside a 16-bit y.  r has x's dtype and h y's (without y:
    ``out_dtype``, by default x's).
    norm, post_norm: "rms" (v * weight / sqrt(mean(v^2) + eps), plus a bias if
    one is given), "layer" (the same of v less its mean); post_norm None: n = y.
    Weights and biases: [d] or None, of any of the three dtypes; post_eps: eps
    by default.
    gate: None, [d] (a value per channel), [..., 1] (per token), or y's shape.

    Differentiable in all tensors.  Arithmetic, statistics and sums are fp32; h
    is the norm of r before its rounding."""
    _need_cuda(x, y, weight, bias, gate, post_weight, post_bias)
    if x.dim() < 1 or x.dtype not in _DT or not 1 <= x.shape[-1] <= 16384 or x.numel() // x.shape[-1] >= 1 << 31:
        _refuse_norm(f"x [..., d] in fp32, bf16 or fp16 with d from 1 to 16384 and below 2^31 rows expected, got "
                     f"{tuple(x.shape)} {x.dtype}")
    d, dev = x.shape[-1], x.get_device()
    dt = out_dtype or (x.dtype if y is None else y.dtype)
    if dt not in _DT or (dt != x.dtype and x.dtype != torch.float32) or (y is not None and y.dtype != dt):
        _refuse_norm(f"x, y and h must share a dtype, or a 16-bit y and h stand beside an fp32 x; got {x.dtype}, "
                     f"{None if y is None else y.dtype}, {dt}")
    if y is not None and y.shape != x.shape:
        _refuse_norm(f"y must have x's shape {tuple(x.shape)}, got {tuple(y.shape)}")
    if norm not in _NORMS or post_norm not in (None, *_NORMS):
        _refuse_norm(f"norm must be 'rms' or 'layer', post_norm also None, got {norm!r}, {post_norm!r}")
    if y is None and (post_norm or gate is not None):
        _refuse_norm("post_norm and gate need y")
    if not post_norm and (post_weight is not None or post_bias is not None):
        _refuse_norm("post_weight and post_bias need post_norm")
    for t, what in ((weight, "weight"), (bias, "bias"), (post_weight, "post_weight"), (post_bias, "post_bias")):
        if t is not None and (t.shape != (d,) or t.dtype not in _DT):
            _refuse_norm(f"{what} must be [{d}] in fp32, bf16 or fp16, got {tuple(t.shape)} {t.dtype}")
    kind = L.OSSM_GATE_NONE
    if gate is not None:
        kind = (L.OSSM_GATE_CHANNEL if gate.shape == (d,) else L.OSSM_GATE_FULL if gate.shape == x.shape else
                L.OSSM_GATE_TOKEN if gate.shape == (*x.shape[:-1], 1) else None)
        if kind is None or gate.dtype not in _DT:
            _refuse_norm(f"gate must be [{d}], {(*x.shape[:-1], 1)} or {tuple(x.shape)} in fp32, bf16 or fp16, got "
                         f"{tuple(gate.shape)} {gate.dtype}")
    for t in (y, weight, bias, gate, post_weight, post_bias):
        if t is not None and t.get_device() != dev:
            _refuse_norm("all tensors must be on one device")
    post_eps = eps if post_eps is None else post_eps
    if not (0.0 <= eps < math.inf and 0.0 <= post_eps < math.inf and math.isfinite(scale)):
        _refuse_norm(f"eps {eps} and post_eps {post_eps} must be finite and not negative, scale {scale} finite")
    ts = (x, y, weight, bias, gate, post_weight, post_bias)
    _no_tangents("residual_norm", *ts)
    opts = (_NORMS[norm], _NORMS[post_norm] if post_norm else L.OSSM_NORM_NONE, kind, float(scale), float(eps),
            float(post_eps), dt)
    if _needs_grad(*ts):
        return _NormFn.apply(*ts, opts)
    return _norm_forward(*ts, opts, False)[:2]
