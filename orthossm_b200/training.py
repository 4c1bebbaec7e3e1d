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

import struct
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L
from .sdpc_kernel import _WS_TRAIN, _captured_workspace, _is_capturing, _need_cuda, _workspace

_DT = {torch.float32: L.OSSM_F32, torch.bfloat16: L.OSSM_BF16, torch.float16: L.OSSM_F16}
_F32_MAX = torch.finfo(torch.float32).max  # the kernels take scalars in fp32
_INTS = (torch.int64, torch.int32, torch.int16, torch.uint8, torch.int8)
_NORMS = {"rms": L.OSSM_NORM_RMS, "layer": L.OSSM_NORM_LAYER}
_REDUCTIONS = {"none": L.OSSM_LOSS_NONE, "mean": L.OSSM_LOSS_MEAN, "sum": L.OSSM_LOSS_SUM}

_raw_stream = torch._C._cuda_getCurrentRawStream  # the current stream's handle without a Stream object (2 us)
_current_device = torch._C._cuda_getDevice
# The argument structs of the C ABI as bytes, with its alignment: packed in a third of a ctypes struct's time.
_LCE = struct.Struct("@qiiiPqPqPqfiPPPPPPP")
_EMBED = struct.Struct("@qiiiPPqfPPqP")
_NORM = struct.Struct("@qiiiPqPqPiiqfiiffPPPPiiiiPPPPqPqPPPPPPPP")
for _s, _c in ((_LCE, L.LceArgs), (_EMBED, L.EmbedArgs), (_NORM, L.NormArgs)):
    if -(-_s.size // 8) * 8 != L.C.sizeof(_c):
        raise RuntimeError("orthossm_b200: packed struct layout does not match the C ABI")
_STATUS: dict = {}  # (device index, stream) -> address of the status word in the tensor of _WS_TRAIN


def _no_tangents(what, *ts):
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def _at(t):
    """A tensor's address, 0 where there is none."""
    return 0 if t is None else t.data_ptr()


def _status(dev, stream):
    """Address of the stream's status word, which ``workspace_status`` reads."""
    if _is_capturing():
        return _captured_workspace("training", torch.device("cuda", dev), stream, 256, 256).data_ptr() + 8
    at = _STATUS.get((dev, stream))
    if at is None:
        device = torch.device("cuda", dev)
        at = _workspace(device, torch.cuda.current_stream(device), 256, cache=_WS_TRAIN).data_ptr() + 8
        _STATUS[dev, stream] = at
    return at


class _On:
    """The device of the tensors as the current one, where it is another."""

    def __init__(self, dev):
        self.to = dev if dev != _current_device() else None

    def __enter__(self):
        if self.to is not None:
            self.back = _current_device()
            torch.cuda.set_device(self.to)

    def __exit__(self, *exc):
        if self.to is not None:
            torch.cuda.set_device(self.back)


def _run(what, fn, args, stream, ws_bytes=None, device=None):
    """Calls a C entry point with the packed arguments, and a workspace of its own if it takes one."""
    if ws_bytes is None:
        status = fn(args, stream)
    else:
        if ws_bytes == 0:
            L.check(L.OSSM_EINVAL, f"{what} (argument check)")
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
        status = fn(args, ws.data_ptr(), ws_bytes, stream)
    if status != L.OSSM_OK:
        L.check(status, what)


def _rows(t, d, align=False):
    """t [..., d] as rows with a unit channel stride, and their stride;
    a copy where it cannot be read as it is.  ``align``: rows start on 16 bytes."""
    if t.is_contiguous() and not (align and (t.data_ptr() % 16 or d * t.element_size() % 16)):
        return t, d
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

def _lce_call(hidden, weight, targets, opts, loss, lse, dev, bwd, grads=(0, 0, 0)):
    """Forward (loss, lse: None or [2, T], its value and what rounding left) or backward (grads: of the loss, where to)."""
    ignore, z_loss, reduction = opts
    V, d = weight.shape
    h, hst = _rows(hidden, d, align=True)
    w, wst = _rows(weight, d, align=True)
    if not targets.is_contiguous():
        targets = targets.contiguous()
    T = targets.numel()
    with _On(dev):
        lib, stream = L.lib(), _raw_stream(dev)
        values = [T, d, V, _DT[weight.dtype], h.data_ptr(), hst, w.data_ptr(), wst, targets.data_ptr(), ignore, z_loss,
                  reduction, _at(loss), 1 if lse is None else lse.data_ptr(), *grads, _status(dev, stream),
                  0 if lse is None else lse.data_ptr() + 4 * T]
        nbytes = lib.ossm_lce_workspace_bytes(_LCE.pack(*values), bwd)
        if nbytes == 0:
            L.check(L.OSSM_EINVAL, "linear_cross_entropy (argument check)")
        # lse is kept for a backward pass only
        ws = torch.empty(nbytes + (4 * T if lse is None else 0), dtype=torch.uint8, device=weight.device)
        at = ws.data_ptr()
        if lse is None:
            values[13] = at + nbytes
        status = (lib.ossm_lce_bwd if bwd else lib.ossm_lce_fwd)(_LCE.pack(*values), at, nbytes, stream)
        if status != L.OSSM_OK:
            L.check(status, "linear_cross_entropy")


def _lce_forward(hidden, weight, targets, opts, keep_lse=False):
    T, dev = targets.numel(), hidden.get_device()
    if T == 0:
        loss = torch.zeros(targets.shape if opts[2] == 0 else (), device=hidden.device)
        return loss, torch.empty(0, device=hidden.device)
    loss = torch.empty(targets.shape if opts[2] == 0 else (), device=hidden.device)
    lse = torch.empty(2, T, device=hidden.device) if keep_lse else None
    _lce_call(hidden, weight, targets, opts, loss, lse, dev, 0)
    return loss, lse


class _LceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, opts):
        loss, lse = _lce_forward(hidden, weight, targets, opts, True)
        ctx.save_for_backward(hidden, weight, targets, lse)
        ctx.opts = opts
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        hidden, weight, targets, lse = ctx.saved_tensors
        want_h, want_w = ctx.needs_input_grad[:2]
        if lse.numel() == 0:
            return (torch.zeros_like(hidden) if want_h else None, torch.zeros_like(weight) if want_w else None, None, None)
        g = g.float().contiguous()
        dh = torch.empty(hidden.shape, dtype=hidden.dtype, device=hidden.device) if want_h else None
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device) if want_w else None
        _lce_call(hidden, weight, targets, ctx.opts, None, lse, hidden.get_device(), 1,
                  (g.data_ptr(), _at(dh), _at(dw)))
        return dh, dw, None, None


def _refuse_loss(hidden, weight, targets, ignore_index, z_loss, reduction):
    """Raises for the first argument of linear_cross_entropy that does not fit."""
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
    if not -1 << 63 <= ignore_index < 1 << 63:
        raise ValueError(f"linear_cross_entropy: ignore_index must fit 64 bits, got {ignore_index}")
    raise ValueError(f"linear_cross_entropy: z_loss must be finite in fp32 and not negative, got {z_loss}")


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
    have their types.  The gradient of the logits is rounded to the inputs' type
    for its two products, in units of the largest upstream gradient of the call:
    fp16 keeps a token's probabilities down to 2^-28 over its share of that.
    Logits are fp32 sums that the tensor core cuts: a loss is within some 2e-7
    of its value at 512 channels, 1e-5 at 2000 (6e-7 for means of thousands).
    Memory beside inputs and gradients: forward 16
    bytes a token for each panel of columns (2048, fewer for few tokens); backward a piece of the logits' gradient of
    at most 512 MB (or 4096 of the V columns, if more) in the inputs' type, 40
    MB of sums and, if the piece is not all columns, fp32 sums of hidden's
    size; in both room for a copy of hidden, used if tokens are ignored."""
    dev, dt, shape = hidden.get_device(), hidden.dtype, targets.shape
    code = _REDUCTIONS.get(reduction)
    ok = (dev >= 0 and (dt is torch.bfloat16 or dt is torch.float16) and weight.dtype is dt and weight.dim() == 2
          and hidden.dim() == len(shape) + 1 and code is not None and 0.0 <= z_loss <= _F32_MAX
          and -1 << 63 <= ignore_index < 1 << 63
          and weight.get_device() == dev and targets.get_device() == dev and targets.dtype in _INTS)
    if ok:
        V, d = weight.shape
        ok = hidden.shape == (*shape, d) and d % 8 == 0 and 8 <= d <= 1 << 16 and 1 <= V <= 1 << 27 \
            and targets.numel() <= 1 << 27
    if not ok:
        _refuse_loss(hidden, weight, targets, ignore_index, z_loss, reduction)
    if forward_ad._current_level >= 0:
        _no_tangents("linear_cross_entropy", hidden, weight)
    if targets.dtype is not torch.int64:
        targets = targets.long()
    opts = int(ignore_index), float(z_loss), code
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return _LceFn.apply(hidden, weight, targets, opts)
    return _lce_forward(hidden, weight, targets, opts)[0]


# ----------------------------------------------------------------------------
# embeddings
# ----------------------------------------------------------------------------

def _embed_forward(ids, weight, scale):
    V, d = weight.shape
    dev = weight.get_device()
    w, wst = _rows(weight, d)
    if not ids.is_contiguous():
        ids = ids.contiguous()
    out = torch.empty(*ids.shape, d, dtype=weight.dtype, device=weight.device)
    n = ids.numel()
    if n:
        with _On(dev):
            _run("embed_tokens", L.lib().ossm_embed_fwd,
                 _EMBED.pack(n, d, V, _DT[weight.dtype], ids.data_ptr(), w.data_ptr(), wst, scale, out.data_ptr(), 0, 0,
                             0), _raw_stream(dev))
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
        dev = g.get_device()
        g, gst = _rows(g, d)
        if not ids.is_contiguous():
            ids = ids.contiguous()
        dw = torch.empty(V, d, dtype=dtype, device=g.device)
        a = _EMBED.pack(ids.numel(), d, V, _DT[dtype], ids.data_ptr(), 0, 0, scale, 0, g.data_ptr(), gst, dw.data_ptr())
        lib = L.lib()
        with _On(dev):
            _run("embed_tokens backward", lib.ossm_embed_bwd, a, _raw_stream(dev), lib.ossm_embed_workspace_bytes(a),
                 g.device)
        return None, dw, None


def _refuse_embed(ids, weight, scale):
    """Raises for the first argument of embed_tokens that does not fit."""
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
    raise ValueError(f"embed_tokens: scale must be finite in fp32, got {scale}")


def embed_tokens(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0) -> torch.Tensor:
    """``scale * weight[ids]``, zeros where an id is no row of the weight (a
    padded position can hold -1).

    ids: integers of any shape, weight: [V, d] fp32, bf16 or fp16 (CUDA), V
    below 2^27, d at most 65536.  Returns [..., d] in weight's dtype.
    Differentiable in ``weight``: a row's gradient is the scaled sum over the
    positions that hold its token, added up in fp32 in their order (cut into
    fixed pieces) and rounded once; rows without a position get zeros."""
    dev = weight.get_device()
    ok = (dev >= 0 and ids.get_device() == dev and weight.dim() == 2 and weight.dtype in _DT and ids.dtype in _INTS
          and ids.numel() < 1 << 31 and -_F32_MAX <= scale <= _F32_MAX)
    if ok:
        V, d = weight.shape
        ok = 1 <= V < 1 << 27 and 1 <= d <= 1 << 16
    if not ok:
        _refuse_embed(ids, weight, scale)
    if forward_ad._current_level >= 0:
        _no_tangents("embed_tokens", weight)
    if ids.dtype is not torch.int64:
        ids = ids.long()
    if weight.requires_grad and torch.is_grad_enabled():
        return _EmbedFn.apply(ids, weight, float(scale))
    return _embed_forward(ids, weight, float(scale))


# ----------------------------------------------------------------------------
# residual and norms
# ----------------------------------------------------------------------------

def _like(t, want=True):
    """An uninitialised contiguous tensor like t, or None."""
    if not want or t is None:
        return None
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _norm_static(ts, opts, d, T):
    """What forward and backward pack alike: contiguous parameters (kept by the
    caller until the launch) and the struct's fields that describe them."""
    x, y, w, b, gate, pw, pb = ts
    norm, post, kind, scale, eps, post_eps, dt = opts
    gst = 0
    if gate is not None:
        if kind == L.OSSM_GATE_FULL:
            gate, gst = _rows(gate, d)
        elif not gate.is_contiguous():
            gate = gate.contiguous()
    held = [t if t is None or t.is_contiguous() else t.contiguous() for t in (w, b, pw, pb)]
    code = lambda t: 0 if t is None else _DT[t.dtype]  # noqa: E731
    held.append(gate)
    return held, (T, d, _DT[x.dtype], _DT[dt]), (
        _at(gate), kind, code(gate), gst, scale, norm, post, eps, post_eps, *map(_at, held[:4]), *map(code, held[:4]))


def _norm_forward(ts, opts, want_stats):
    x, y = ts[0], ts[1]
    d, dev, dt, post = x.shape[-1], x.get_device(), opts[6], opts[1]
    T = x.numel() // d
    xr, xst = _rows(x, d)
    yr, yst = (None, d) if y is None else _rows(y, d)
    r = x if y is None else _like(x)
    h = _like(x) if dt is x.dtype else torch.empty(x.shape, dtype=dt, device=x.device)
    stats = torch.empty(4 if post else 2, T, device=x.device) if want_stats else None
    if T:
        held, head, mid = _norm_static(ts, opts, d, T)
        with _On(dev):
            stream = _raw_stream(dev)
            _run("residual_norm", L.lib().ossm_residual_norm_fwd,
                 _NORM.pack(*head, xr.data_ptr(), xst, _at(yr), yst, *mid, 0 if y is None else r.data_ptr(),
                            h.data_ptr(), _at(stats), 0, d, 0, d, 0, 0, 0, 0, 0, 0, 0, _status(dev, stream)), stream)
    return r, h, stats


class _NormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, w, b, gate, pw, pb, opts):
        r, h, stats = _norm_forward((x, y, w, b, gate, pw, pb), opts, True)
        ctx.full = bool(opts[1]) or gate is not None
        ctx.set_materialize_grads(False)
        # an fp32 r stands for x and y; a rounded one may have lost what the gradients are a difference of
        ctx.sum = ctx.full or (y is not None and x.dtype is not torch.float32)
        ctx.save_for_backward(*((x, y) if ctx.sum else (r, None)), w, b, gate, pw, pb, stats)
        ctx.opts = opts
        ctx.has_y = y is not None
        return r, h

    @staticmethod
    @once_differentiable
    def backward(ctx, gr, gh):
        if gr is None and gh is None:
            return (None,) * 8
        *ts, stats = ctx.saved_tensors
        x, y, w, b, gate, pw, pb = ts
        opts, full = ctx.opts, ctx.full
        need_x, need_y, need_w, need_b, need_gate, need_pw, need_pb = ctx.needs_input_grad[:7]
        scale, dt = opts[3], opts[6]
        d, dev = x.shape[-1], x.get_device()
        T = x.numel() // d
        xr, xst = _rows(x, d)
        yr, yst = (None, d) if y is None else _rows(y, d)
        gr, grst = (None, d) if gr is None else _rows(gr, d)
        ghr, ghst = (None, d) if gh is None else _rows(gh, d)
        dw, db, dgate, dpw, dpb = (_like(w, need_w), _like(b, need_b), _like(gate, need_gate), _like(pw, need_pw),
                                   _like(pb, need_pb))
        # without a norm or gate of y, and a scale of 1, its gradient is x's
        same = not full and scale == 1.0 and dt is x.dtype
        dx = _like(x, need_x or (same and need_y))
        dy = torch.empty(x.shape, dtype=dt, device=x.device) if ctx.has_y and need_y and not same else None
        if T:
            held, head, mid = _norm_static(ts, opts, d, T)
            lib = L.lib()
            with _On(dev):
                stream = _raw_stream(dev)
                at = xr.data_ptr()
                a = _NORM.pack(*head, at if ctx.sum else 0, xst, _at(yr), yst, *mid, 0 if ctx.sum else at, 0, stats.data_ptr(),
                               _at(gr), grst, _at(ghr), ghst, _at(dx), _at(dy), _at(dgate), _at(dw), _at(db), _at(dpw),
                               _at(dpb), _status(dev, stream))
                _run("residual_norm backward", lib.ossm_residual_norm_bwd, a, stream, lib.ossm_norm_workspace_bytes(a),
                     x.device)
        else:
            for t in (dw, db, dpw, dpb, dgate):
                if t is not None:
                    t.zero_()
        if gh is None:  # h was not used: its parameters get nothing
            dw = db = None
        if same and ctx.has_y and need_y:
            dy = dx
        return (dx if need_x else None), dy, dw, db, dgate, dpw, dpb, None


def _refuse_norm(x, y, weight, bias, norm, eps, gate, scale, post_norm, post_weight, post_bias, post_eps, dt):
    """Raises for the first argument of residual_norm that does not fit."""
    def refuse(why):
        raise ValueError("residual_norm: " + why)

    _need_cuda(x, y, weight, bias, gate, post_weight, post_bias)
    if x.dim() < 1 or x.dtype not in _DT or not 1 <= x.shape[-1] <= 8192 or x.numel() // x.shape[-1] >= 1 << 31:
        refuse(f"x [..., d] in fp32, bf16 or fp16 with d from 1 to 8192 and below 2^31 rows expected, got "
               f"{tuple(x.shape)} {x.dtype}")
    d = x.shape[-1]
    if dt not in _DT or (dt != x.dtype and x.dtype != torch.float32) or (y is not None and y.dtype != dt):
        refuse(f"x, y and h must share a dtype, or a 16-bit y and h stand beside an fp32 x; got {x.dtype}, "
               f"{None if y is None else y.dtype}, {dt}")
    if y is not None and y.shape != x.shape:
        refuse(f"y must have x's shape {tuple(x.shape)}, got {tuple(y.shape)}")
    if norm not in _NORMS or post_norm not in (None, *_NORMS):
        refuse(f"norm must be 'rms' or 'layer', post_norm also None, got {norm!r}, {post_norm!r}")
    if y is None and (post_norm or gate is not None):
        refuse("post_norm and gate need y")
    if not post_norm and (post_weight is not None or post_bias is not None):
        refuse("post_weight and post_bias need post_norm")
    for t, what in ((weight, "weight"), (bias, "bias"), (post_weight, "post_weight"), (post_bias, "post_bias")):
        if t is not None and (t.shape != (d,) or t.dtype not in _DT):
            refuse(f"{what} must be [{d}] in fp32, bf16 or fp16, got {tuple(t.shape)} {t.dtype}")
    if gate is not None and (gate.dtype not in _DT or gate.shape not in ((d,), x.shape, (*x.shape[:-1], 1))):
        refuse(f"gate must be [{d}], {(*x.shape[:-1], 1)} or {tuple(x.shape)} in fp32, bf16 or fp16, got "
               f"{tuple(gate.shape)} {gate.dtype}")
    if any(t is not None and t.get_device() != x.get_device() for t in (y, weight, bias, gate, post_weight, post_bias)):
        refuse("all tensors must be on one device")
    refuse(f"eps {eps} and post_eps {post_eps} must be finite in fp32 and not negative, scale {scale} finite in fp32")


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
    (then r is x).  d at most 8192.  Both of one dtype (fp32, bf16, fp16), or
    an fp32 stream beside a 16-bit y.  r has x's dtype and h y's (without y:
    ``out_dtype``, by default x's).
    norm, post_norm: "rms" (v * weight / sqrt(mean(v^2) + eps), plus a bias if
    one is given), "layer" (the same of v less its mean); post_norm None: n = y.
    Weights and biases: [d] or None, of any of the three dtypes; post_eps: eps
    by default.
    gate: None, [d] (a value per channel), [..., 1] (per token), or y's shape.

    Differentiable in all tensors.  Arithmetic, statistics and sums are fp32; h
    is the norm of r before its rounding.  Backward keeps x and y (r alone where
    it is fp32 and y has neither norm nor gate)."""
    dev, xdt = x.get_device(), x.dtype
    shape = x.shape
    d = shape[-1] if shape else 0
    dt = out_dtype or (xdt if y is None else y.dtype)
    code, post = _NORMS.get(norm), 0 if post_norm is None else _NORMS.get(post_norm)
    post_eps = eps if post_eps is None else post_eps
    kind = L.OSSM_GATE_NONE
    ok = (dev >= 0 and xdt in _DT and dt in _DT and (dt is xdt or xdt is torch.float32) and 1 <= d <= 8192
          and x.numel() < d << 31 and code and post is not None
          and 0.0 <= eps <= _F32_MAX and 0.0 <= post_eps <= _F32_MAX and -_F32_MAX <= scale <= _F32_MAX)
    if ok:
        if y is not None:
            ok = y.shape == shape and y.dtype is dt and y.get_device() == dev
        else:
            ok = not post and gate is None
        if gate is not None and ok:
            g = gate.shape
            kind = (L.OSSM_GATE_CHANNEL if g == (d,) else L.OSSM_GATE_FULL if g == shape else
                    L.OSSM_GATE_TOKEN if g == (*shape[:-1], 1) else None)
            ok = kind is not None and gate.dtype in _DT and gate.get_device() == dev
        if not post and (post_weight is not None or post_bias is not None):
            ok = False
        for t in (weight, bias, post_weight, post_bias):
            if t is not None and not (t.dim() == 1 and t.shape[0] == d and t.dtype in _DT and t.get_device() == dev):
                ok = False
    if not ok:
        _refuse_norm(x, y, weight, bias, norm, eps, gate, scale, post_norm, post_weight, post_bias, post_eps, dt)
    ts = (x, y, weight, bias, gate, post_weight, post_bias)
    if forward_ad._current_level >= 0:
        _no_tangents("residual_norm", *ts)
    opts = (code, post, kind, float(scale), float(eps), float(post_eps), dt)
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return _NormFn.apply(*ts, opts)
    return _norm_forward(ts, opts, False)[:2]
