"""Cases of the training operators: the language-model loss from hidden states, token embeddings with their gradient,
and the norms around a block with its residual.

``run`` computes an operator in its plain form (elementary torch operations in
fp32) or, with ``own`` set, through this package's public functions.  A case
is a dict of plain values.  A training case returns the outputs and every
gradient, a scoring or serving case the outputs.
"""
import math

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ----------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------

def _loss(name, tokens, dim, vocab, dtype, train, reduction="mean", ignored=0.0, z_loss=0.0):
    """ignored: the share of tokens that have no target."""
    return {"name": name, "op": "loss", "tokens": tokens, "dim": dim, "vocab": vocab, "dtype": dtype, "train": train,
            "reduction": reduction, "ignored": ignored, "z_loss": z_loss}


def _embed(name, tokens, dim, vocab, dtype, train, scale=1.0, skewed=True, padded=0.0):
    """skewed: token v about as often as 1 / (v + 1); padded: the share of positions that hold no token (id -1)."""
    return {"name": name, "op": "embed", "tokens": tokens, "dim": dim, "vocab": vocab, "dtype": dtype, "train": train,
            "scale": scale, "skewed": skewed, "padded": padded}


def _norm(name, tokens, dim, stream, dtype, train, norm="rms", post="", gate="", scale=1.0):
    """stream: type of the residual stream x; dtype: type of the block's output y and of the normed h.
    post: the norm of the block's output; gate: "", "channel", "token" or "full"."""
    return {"name": name, "op": "norm", "tokens": tokens, "dim": dim, "stream": stream, "dtype": dtype, "train": train,
            "norm": norm, "post": post, "gate": gate, "scale": scale}


def listed():
    return [
        # one short continuation scored token by token at the language model's sizes: a call whose latency counts
        _loss("loss_score_one", 33, 512, 32000, "bf16", False, "none"),
        # evaluation of a few documents, a loss per token
        _loss("loss_score", 4096, 512, 32000, "bf16", False, "none"),
        # the language model's training step: 8 sequences of 2048, a few positions without a target
        _loss("loss_train", 16384, 512, 32000, "bf16", True, "mean", 0.02),
        # fine-tuning: prompts carry no loss, nothing divides evenly, fp16 with a penalty on lse
        _loss("loss_ragged", 5003, 1000, 49999, "fp16", True, "sum", 0.5, 1e-4),
        # a wide model at the engine's vocabulary
        _loss("loss_wide", 8192, 2048, 131072, "bf16", True, "mean"),
        # one decode step of a batch of streams
        _embed("embed_step", 32, 512, 32000, "bf16", False),
        # a training batch of 8 x 16384 tokens, as frequent as words are
        _embed("embed_train", 131072, 512, 32000, "bf16", True),
        # the engine's fp32 embedding at its vocabulary, scaled, a padded batch of odd length
        _embed("embed_wide", 20001, 256, 131072, "fp32", True, 16.0, False, 0.1),
        # a decode step between two blocks
        _norm("norm_step", 32, 512, "bf16", "bf16", False),
        # the language model's step between two blocks: residual, then RMSNorm
        _norm("norm_train", 131072, 512, "bf16", "bf16", True),
        # the combine of the global and the local path: their sum, then LayerNorm
        _norm("norm_combine", 30011, 512, "bf16", "bf16", True, "layer"),
        # norms on both sides of the block, a gate per channel and a residual scale, fp32 stream beside bf16 blocks
        _norm("norm_sandwich", 16384, 2048, "fp32", "bf16", True, "rms", "rms", "channel", 0.5),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["loss", "loss", "embed", "norm"])
    train = rng.random() < 0.7
    if kind == "loss":
        tokens, dim, vocab = _log_between(rng, 1, 16384), 8 * _log_between(rng, 8, 256), _log_between(rng, 500, 131072)
        while tokens * vocab > 1 << 30 or tokens * dim * vocab > 1 << 41:
            tokens = tokens * 2 // 3
        c = _loss("", tokens, dim, vocab, rng.choice(["bf16", "bf16", "fp16"]), train,
                  rng.choice(["mean", "mean", "sum", "none"]), rng.choice([0.0, 0.02, 0.5, 0.9]),
                  rng.choice([0.0, 0.0, 1e-4]))
    elif kind == "embed":
        tokens, vocab = _log_between(rng, 1, 131072), _log_between(rng, 100, 131072)
        dim = rng.choice([8 * _log_between(rng, 1, 256), _log_between(rng, 1, 1024)])
        while (tokens + vocab) * dim > 1 << 27:
            dim = dim * 2 // 3
        c = _embed("", tokens, dim, vocab, rng.choice(["bf16", "bf16", "fp16", "fp32"]), train,
                   rng.choice([1.0, round(math.sqrt(dim), 3)]), rng.random() < 0.6, rng.choice([0.0, 0.0, 0.1, 0.6]))
    else:
        tokens = _log_between(rng, 1, 131072)
        dim = rng.choice([8 * _log_between(rng, 2, 1024), 8 * _log_between(rng, 2, 1024), _log_between(rng, 3, 8192)])
        while tokens * dim > 1 << 26:
            tokens = tokens * 2 // 3
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        c = _norm("", tokens, dim, rng.choice([dtype, "fp32"]), dtype, train, rng.choice(["rms", "layer"]),
                  rng.choice(["", "", "rms", "layer"]), rng.choice(["", "", "channel", "token", "full"]),
                  rng.choice([1.0, 0.5, round(rng.uniform(0.1, 1.5), 3)]))
    del c["name"]
    return c


def work(case):
    T, d = case["tokens"], case["dim"]
    size = 2 if case["dtype"] in ("bf16", "fp16") else 4
    if case["op"] == "loss":
        V = case["vocab"]
        rows = T - int(T * case["ignored"])  # the others have no part in any product
        b = size * (T * d + V * d) + 8 * T + 4 * T
        return {"bytes": b + (size * (T * d + V * d) if case["train"] else 0),
                "flops": (6 if case["train"] else 2) * rows * d * V}
    if case["op"] == "embed":
        V = case["vocab"]
        used = min(V, T)
        b = 8 * T + size * (used + T) * d
        return {"bytes": b + (8 * T + size * (T + V) * d if case["train"] else 0),
                "flops": T * d * (2 if case["train"] else 1)}
    stream = 2 if case["stream"] in ("bf16", "fp16") else 4
    full = size if case["gate"] == "full" else 0
    b = T * d * (2 * stream + 2 * size + full)  # x, y (and the gate) in, r and h out
    if case["train"]:  # x, y, dr, dh (and the gate) in, dx, dy (and the gate's) out
        b += T * d * (3 * stream + 3 * size + 2 * full)
    return {"bytes": b, "flops": T * d * (25 if case["train"] else 8)}


# ----------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DTYPE[case["dtype"]]
    T, d, train = case["tokens"], case["dim"], case["train"]
    randn = lambda *n: torch.randn(*n, device="cuda", generator=g)  # noqa: E731
    rand = lambda *n: torch.rand(*n, device="cuda", generator=g)    # noqa: E731
    s = {"op": case["op"], "train": train}
    if case["op"] == "loss":
        V = case["vocab"]
        w = randn(V, d).mul_(1.4 / math.sqrt(d)).to(dt)
        targets = (V ** rand(T)).long().sub_(1).clamp_(0, V - 1)
        # states that point at their target more or less, as a trained model's do
        s["hidden"] = randn(T, d).addcmul_(w[targets].float(), 4.0 * rand(T, 1)).to(dt).requires_grad_(train)
        s["weight"] = w.requires_grad_(train)
        targets[torch.randperm(T, device="cuda", generator=g)[:int(T * case["ignored"])]] = -100
        s["targets"], s["reduction"], s["z_loss"] = targets, case["reduction"], case["z_loss"]
        # per-token losses come back with weights of their own
        s["d_loss"] = rand(T) if case["reduction"] == "none" else torch.ones((), device="cuda")
    elif case["op"] == "embed":
        V = case["vocab"]
        ids = ((V ** rand(T)) - 1 if case["skewed"] else rand(T) * V).long().clamp_(0, V - 1)
        ids[rand(T) < case["padded"]] = -1
        s["ids"], s["scale"] = ids, case["scale"]
        s["weight"] = randn(V, d).mul_(0.02).to(dt).requires_grad_(train)
        s["d_out"] = randn(T, d).to(dt) if train else None
    else:
        st = _DTYPE[case["stream"]]
        s["x"] = randn(T, d).mul_(2.0).to(st).requires_grad_(train)
        s["y"] = randn(T, d).mul_(0.7).to(dt).requires_grad_(train)
        s["norm"], s["post_norm"], s["scale"] = case["norm"], case["post"] or None, case["scale"]
        affine = lambda kind: ((1.0 + 0.1 * randn(d)).to(dt).requires_grad_(train),  # noqa: E731
                               (0.1 * randn(d)).to(dt).requires_grad_(train) if kind == "layer" else None)
        s["weight"], s["bias"] = affine(case["norm"])
        s["post_weight"], s["post_bias"] = affine(case["post"]) if case["post"] else (None, None)
        shape = {"channel": (d,), "token": (T, 1), "full": (T, d)}.get(case["gate"])
        s["gate"] = None if shape is None else rand(*shape).to(dt).requires_grad_(train)
        s["d_r"], s["d_h"] = (randn(T, d).to(st), randn(T, d).to(dt)) if train else (None, None)
    return s


# ----------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------

_EPS = 1e-6


def run(state):
    s = {k: v for k, v in state.items() if k != "op"}
    if own:
        return {"loss": _own_loss, "embed": _own_embed, "norm": _own_norm}[state["op"]](s)
    with torch.no_grad():
        return {"loss": _plain_loss, "embed": _plain_embed, "norm": _plain_norm}[state["op"]](**s)


def _own_loss(s):
    import orthossm_b200 as O
    loss = O.linear_cross_entropy(s["hidden"], s["weight"], s["targets"], z_loss=s["z_loss"], reduction=s["reduction"])
    if not s["train"]:
        return [loss]
    return [loss.detach(), *torch.autograd.grad(loss, (s["hidden"], s["weight"]), s["d_loss"])]


def _own_embed(s):
    import orthossm_b200 as O
    out = O.embed_tokens(s["ids"], s["weight"], scale=s["scale"])
    if not s["train"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, (s["weight"],), s["d_out"])]


_NORM_INPUTS = ("x", "y", "weight", "bias", "gate", "post_weight", "post_bias")


def _own_norm(s):
    import orthossm_b200 as O
    r, h = O.residual_norm(s["x"], s["y"], s["weight"], s["bias"], norm=s["norm"], eps=_EPS, gate=s["gate"],
                           scale=s["scale"], post_norm=s["post_norm"], post_weight=s["post_weight"],
                           post_bias=s["post_bias"], post_eps=_EPS)
    if not s["train"]:
        return [r, h]
    leaves = [s[k] for k in _NORM_INPUTS if s[k] is not None]
    return [r.detach(), h.detach(), *torch.autograd.grad((r, h), leaves, (s["d_r"], s["d_h"]))]


def _plain_loss(hidden, weight, targets, reduction, z_loss, d_loss, train):
    """z = h . w over the vocabulary; a token's loss is lse - z[target] + z_loss lse^2 with lse = log sum exp z, 0
    without a target.  Its gradient in z is (1 + 2 z_loss lse) softmax(z), less 1 at the target."""
    has = targets >= 0
    rows = has.nonzero()[:, 0]
    t = targets[rows]
    h, w = hidden[rows].float(), weight.float()
    z = h @ w.t()
    m = z.amax(-1, keepdim=True)
    zt = z.gather(1, t[:, None])[:, 0]
    z.sub_(m).exp_()
    total = z.sum(-1, keepdim=True)
    lse = (m + total.log())[:, 0]
    each = torch.zeros(targets.shape, device=h.device)
    each[rows] = lse - zt + z_loss * lse * lse
    n = rows.numel()
    loss = each if reduction == "none" else each.sum() if reduction == "sum" else each.sum() / max(n, 1)
    if not train:
        return [loss]
    g = d_loss[rows] if reduction == "none" else d_loss.expand(n) / (max(n, 1) if reduction == "mean" else 1)
    z.mul_((g * (1 + 2 * z_loss * lse))[:, None] / total)
    z[torch.arange(n, device=h.device), t] -= g
    dh = torch.zeros(hidden.shape, device=h.device)
    dh[rows] = z @ w
    return [loss, dh.to(hidden.dtype), (z.t() @ h).to(weight.dtype)]


def _plain_embed(ids, weight, scale, d_out, train):
    """Row ids[t] of the weight, scaled; zeros where the id is no row.  The gradient of a row is the scaled sum over
    the positions that hold it (float64: a frequent token has thousands)."""
    has = ids >= 0
    out = (weight[ids.clamp(min=0)].float() * scale * has[:, None]).to(weight.dtype)
    if not train:
        return [out]
    dw = torch.zeros(weight.shape, device=ids.device, dtype=torch.float64)
    dw.index_add_(0, ids[has], d_out[has].double())
    return [out, dw.mul_(scale).to(weight.dtype)]


def _normed(v, kind):
    """v less its mean (layer) over its root mean square, and the inverse of that."""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    inv = 1.0 / ((v * v).mean(-1, keepdim=True) + _EPS).sqrt()
    return v * inv, inv


def _norm_grad(dv, v, inv, kind):
    """Gradient of the normed values v in what was normed, from theirs."""
    g = dv - v * (dv * v).mean(-1, keepdim=True)
    if kind == "layer":
        g = g - dv.mean(-1, keepdim=True)
    return g * inv


def _plain_norm(x, y, weight, bias, norm, gate, scale, post_norm, post_weight, post_bias, d_r, d_h, train):
    """n = post_norm(y), r = x + scale gate n, h = norm(r)."""
    f = lambda t: None if t is None else t.float()  # noqa: E731
    w, pw, gt, n = f(weight), f(post_weight), f(gate), f(y)
    if post_norm:
        pv, pinv = _normed(n, post_norm)
        n = pv * pw if post_bias is None else pv * pw + post_bias.float()
    step = scale * n if gt is None else scale * gt * n
    r = x.float() + step
    v, inv = _normed(r, norm)
    h = v * w if bias is None else v * w + bias.float()
    out = [r.to(x.dtype), h.to(y.dtype)]
    if not train:
        return out
    dh = d_h.float()
    dr = d_r.float() + _norm_grad(dh * w, v, inv, norm)
    dn = dr * scale
    grads = {"x": dr, "weight": (dh * v).sum(0), "bias": None if bias is None else dh.sum(0)}
    if gt is not None:
        dg = dn * n
        grads["gate"] = dg.sum(0) if gt.dim() == 1 else dg.sum(1, keepdim=True) if gt.shape != y.shape else dg
        dn = dn * gt
    if post_norm:
        grads["post_weight"] = (dn * pv).sum(0)
        grads["post_bias"] = None if post_bias is None else dn.sum(0)
        dn = _norm_grad(dn * pw, pv, pinv, post_norm)
    grads["y"] = dn
    have = {"x": x, "y": y, "weight": weight, "bias": bias, "gate": gate, "post_weight": post_weight,
            "post_bias": post_bias}
    return out + [grads[k].to(have[k].dtype) for k in _NORM_INPUTS if have[k] is not None]


# ----------------------------------------------------------------------------
# float64
# ----------------------------------------------------------------------------

def exact(case, seed):
    """The outputs from their definitions in float64."""
    s = prepare(case, seed)
    return {"loss": _exact_loss, "embed": _exact_embed, "norm": _exact_norm}[case["op"]](s)


def _exact_loss(s):
    """A block of tokens at a time: log-softmax of the block's logits, gradients as softmax less the target's row."""
    H, W, targets, lam = s["hidden"].detach(), s["weight"].detach().double(), s["targets"], s["z_loss"]
    T, count = targets.shape[0], int((targets >= 0).sum())
    each = torch.zeros(T, dtype=torch.float64, device=H.device)
    dh = torch.zeros(H.shape, dtype=torch.float64, device=H.device)
    dw = torch.zeros_like(W)
    block = max(1, (1 << 27) // W.shape[0])
    for a in range(0, T, block):
        b = min(T, a + block)
        hb, tb = H[a:b].double(), targets[a:b]
        on = (tb >= 0).double()
        at = tb.clamp(min=0)
        z = torch.einsum("td,vd->tv", hb, W)
        lse = torch.logsumexp(z, 1)
        each[a:b] = on * (lse - torch.take_along_dim(z, at[:, None], 1).squeeze(1) + lam * lse.square())
        if s["train"]:
            up = s["d_loss"].double()
            up = up[a:b] if s["reduction"] == "none" else up / (max(count, 1) if s["reduction"] == "mean" else 1.0)
            p = torch.exp(z - lse[:, None]) * (1.0 + 2.0 * lam * lse)[:, None]
            p.scatter_add_(1, at[:, None], -torch.ones_like(p[:, :1]))
            p *= (up * on)[:, None]
            dh[a:b] = p @ W
            dw += torch.einsum("tv,td->vd", p, hb)
        del z
    loss = each if s["reduction"] == "none" else each.sum() / (max(count, 1) if s["reduction"] == "mean" else 1.0)
    return [loss, dh, dw] if s["train"] else [loss]


def _exact_embed(s):
    ids, W = s["ids"], s["weight"].detach()
    held = torch.where(ids >= 0)[0]
    out = torch.zeros(ids.shape[0], W.shape[1], dtype=torch.float64, device=W.device)
    out[held] = s["scale"] * W.double()[ids[held]]
    if not s["train"]:
        return [out]
    # tokens in order of their id: a row's gradient is a difference of running sums of its run
    order = held[torch.sort(ids[held], stable=True).indices]
    counts = torch.bincount(ids[held], minlength=W.shape[0])
    dw = torch.zeros(W.shape, dtype=torch.float64, device=W.device)
    used = counts > 0
    if order.numel():
        dw[used] = torch.segment_reduce(s["d_out"][order].double(), "sum", lengths=counts[used], axis=0)
    return [out, s["scale"] * dw]


def _exact_norm(s):
    """The definition in float64, gradients by automatic differentiation."""
    v = {k: None if s[k] is None else s[k].detach().double().requires_grad_(s["train"]) for k in _NORM_INPUTS}

    def normed(u, kind, w, b):
        if kind == "layer":
            return torch.nn.functional.layer_norm(u, u.shape[-1:], w, b, _EPS)
        return u * torch.rsqrt(u.square().mean(-1, keepdim=True) + _EPS) * w

    n = normed(v["y"], s["post_norm"], v["post_weight"], v["post_bias"]) if s["post_norm"] else v["y"]
    r = v["x"] + s["scale"] * (n if v["gate"] is None else v["gate"] * n)
    h = normed(r, s["norm"], v["weight"], v["bias"])
    if not s["train"]:
        return [r, h]
    leaves = [v[k] for k in _NORM_INPUTS if v[k] is not None]
    grads = torch.autograd.grad((r, h), leaves, (s["d_r"].double(), s["d_h"].double()))
    return [r.detach(), h.detach(), *grads]
