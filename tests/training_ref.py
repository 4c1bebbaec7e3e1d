"""float64 restatements of the training operators, with elementwise error
bounds that follow from the roundings the kernels make.

u(t): half a step of a type relative to the value (bf16 2^-8, fp16 2^-11, fp32
2^-24).  fp32 sums of n terms are within n 2^-23 of the sum of their magnitudes
(the tensor core may cut where it could round: a whole step, not half)."""
import torch

F = 2.0 ** -23


def u(dtype):
    return torch.finfo(dtype).eps / 2


def lce_ref(hidden, weight, targets, g, ignore=-100, z_loss=0.0, reduction="mean"):
    """(loss, dH, dW) and their bounds; g: the upstream gradient."""
    dt = hidden.dtype
    V, d = weight.shape
    H, W, t = hidden.detach().reshape(-1, d).double(), weight.detach().double(), targets.reshape(-1)
    on = t != ignore
    H = torch.where(on[:, None], H, 0.0)
    n = int(on.sum())
    at = torch.where(on, t, 0)[:, None]
    z = H @ W.t()
    ez = (d + 8) * F * (H.abs() @ W.abs().t()).amax(1)  # of a row's logits
    lse = torch.logsumexp(z, 1)
    p = (z - lse[:, None]).exp()
    # 2^x is good to 2^-22; a row's sum is added up in runs of 64 within panels of 8 tiles, then V / 256 of them
    el = ez + 2.0 ** -21 + (80 + V / 256) * F + lse.abs() * 2.0 ** -22
    each = torch.where(on, lse - z.gather(1, at)[:, 0] + z_loss * lse ** 2, 0.0)
    eeach = torch.where(on, el + ez + z_loss * (2 * lse.abs() * el + el ** 2), 0.0) + each.abs() * u(torch.float32)
    share = 1.0 / max(n, 1) if reduction == "mean" else 1.0
    loss, eloss = each, eeach
    if reduction != "none":
        loss, eloss = each.sum() * share, eeach.sum() * share + (each.sum() * share).abs() * u(torch.float32)
    gt = (g.detach().double().reshape(-1).expand(t.shape[0]) * share) * on
    a = (gt * (1 + 2 * z_loss * lse))[:, None]
    dz = a * p
    dz.scatter_add_(1, at, -gt[:, None])
    ep = 2 * el[:, None] + ez[:, None] + 2.0 ** -20 + z_loss * 2 * el[:, None]  # of a p, relative
    edz = a.abs() * p * ep + gt.abs()[:, None] * F + (a * p).abs() * 4 * F
    edz = edz + u(dt) * (dz.abs() + edz)  # rounded for the products
    if dt == torch.float16:  # or, below fp16's normal numbers, to steps of 2^-24 of 2^-14 of the largest factor
        edz = edz + on[:, None] * 2.0 ** -25 * 2.0 ** -14 * torch.maximum(a.abs(), gt.abs()[:, None]).max()
    dh, dw = dz @ W, dz.t() @ H
    edh = edz @ W.abs() + V * F * (dz.abs() @ W.abs())
    edw = edz.t() @ H.abs() + max(n, 1) * F * (dz.abs().t() @ H.abs())
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps if dt == torch.float16 else 0.0
    edh, edw = edh + u(dt) * (dh.abs() + edh) + tiny, edw + u(dt) * (dw.abs() + edw) + tiny
    return (loss, dh.view(hidden.shape), dw), (eloss, edh.view(hidden.shape), edw)


def embed_ref(ids, weight, g, scale=1.0):
    """(out, dW) and their bounds."""
    V, d = weight.shape
    i, W, dt = ids.reshape(-1), weight.detach().double(), weight.dtype
    on = (i >= 0) & (i < V)
    out = torch.where(on[:, None], W[torch.where(on, i, 0)] * scale, 0.0)
    G = g.detach().reshape(-1, d).double()[on]
    dw, mag = torch.zeros_like(W), torch.zeros_like(W)
    dw.index_add_(0, i[on], G)
    mag.index_add_(0, i[on], G.abs())
    count = torch.bincount(i[on], minlength=V).double()[:, None]
    edw = (count + 2) * F * mag * abs(scale)
    eout = 1.01 * (u(dt) + u(torch.float32)) * out.abs()
    return (out.view(*ids.shape, d), dw * scale), (eout.view(*ids.shape, d), edw + 1.01 * u(dt) * (dw * scale).abs())


def norm_ref(ts, opts, dr, dh):
    """ts: dict of x, y, weight, bias, gate, post_weight, post_bias (or None);
    opts: norm, post_norm, scale, eps.  {name: (value, bound)} of r, h and the
    gradient of each tensor.  Gradients by automatic differentiation in
    float64, bounds from the formulas' magnitudes."""
    v = {k: None if t is None else t.detach().double().requires_grad_() for k, t in ts.items()}
    norm, post, scale, eps = opts["norm"], opts["post_norm"], opts["scale"], opts["eps"]
    x, y = v["x"], v["y"]
    d = x.shape[-1]

    def normed(q, kind):
        if kind == "layer":
            q = q - q.mean(-1, keepdim=True)
        inv = 1 / (q.square().mean(-1, keepdim=True) + eps).sqrt()
        return q * inv, inv

    one = lambda t: 1.0 if t is None else t   # noqa: E731
    zero = lambda t: 0.0 if t is None else t  # noqa: E731
    pv = pinv = None
    r = x
    if y is not None:
        n = y
        if post:
            pv, pinv = normed(y, post)
            n = pv * one(v["post_weight"]) + zero(v["post_bias"])
        r = x + scale * one(v["gate"]) * n
    q, inv = normed(r, norm)
    h = q * one(v["weight"]) + zero(v["bias"])
    outs, ups = [h], [dh.double()]
    if dr is not None:
        outs.append(r)
        ups.append(dr.double())
    names = [k for k, t in v.items() if t is not None]
    grads = dict(zip(names, torch.autograd.grad(outs, [v[k] for k in names], ups)))
    with torch.no_grad():
        fp = (d + 32) * F  # relative to the magnitudes below, of what fp32 statistics and sums lose
        ux = u(ts["x"].dtype)
        dt = ts["y"].dtype if y is not None else dh.dtype
        rmag = x.abs() + (0 if y is None else abs(scale) * (one(v["gate"]) * (
            n if not post else pv.abs() * one(v["post_weight"]) + zero(v["post_bias"]))).abs())
        if post:  # a mean is taken from y: what is lost is relative to |y|
            pm = pv.abs() + (y.abs() + y.abs().mean(-1, keepdim=True)) * pinv
            rmag = rmag + abs(scale) * (one(v["gate"]) * one(v["post_weight"])).__abs__() * pm
        bounds = {"r": (r, 1.01 * ux * r.abs() + fp * rmag)}
        qm = q.abs() + (rmag + rmag.mean(-1, keepdim=True)) * inv  # magnitude of the normed values' terms
        wa = abs(one(v["weight"])) if v["weight"] is None else v["weight"].abs()
        bounds["h"] = (h, 1.01 * u(dt) * h.abs() + 4 * fp * (qm * wa + abs(zero(v["bias"]) if v["bias"] is None
                                                                            else v["bias"].abs())))
        # backward; without norm or gate of y it starts from the rounded r (or x itself),
        # but LayerNorm's of a 16-bit stream from x and y
        dhd = dh.double()
        rounded = y is not None and not post and v["gate"] is None and (
            norm == "rms" or ts["x"].dtype == torch.float32)
        eq = 4 * fp * qm + (1.01 * ux * r.abs() * inv * (1 + q.abs()) if rounded else 0.0)  # of q
        e = dhd * (wa if v["weight"] is None else v["weight"])
        m0 = (e * q).mean(-1, keepdim=True)
        m0m = (e.abs() * q.abs()).mean(-1, keepdim=True)
        em0 = (e.abs() * eq).mean(-1, keepdim=True) + 2 * fp * m0m
        m1m = e.abs().mean(-1, keepdim=True) if norm == "layer" else 0.0
        egr = inv * (eq * m0.abs() + (q.abs() + eq) * em0 + 4 * fp * (e.abs() + q.abs() * m0m + m1m))
        gr = grads["x"]
        if dr is not None:
            egr = egr + 4 * F * dr.abs()
        bounds["dx"] = (gr, egr + 1.01 * ux * (gr.abs() + egr))
        T = max(1, x.numel() // d)
        flat = lambda t: t.reshape(-1, d)  # noqa: E731
        col = lambda name, val, err, mag: (val, flat(err).sum(0) + 2 * T * F * flat(mag).sum(0)  # noqa: E731
                                           + 1.01 * u(ts[name].dtype) * val.abs())
        if v["weight"] is not None:
            bounds["dweight"] = col("weight", grads["weight"], dhd.abs() * eq, (dhd * q).abs())
        if v["bias"] is not None:
            bounds["dbias"] = col("bias", grads["bias"], 0 * dhd, dhd.abs())
        if y is None:
            return bounds
        gm = one(v["gate"]) if v["gate"] is None else v["gate"].abs()
        dn, edn = (gr * scale * one(v["gate"])), egr * abs(scale) * gm + 4 * F * (gr * scale * one(v["gate"])).abs()
        nv = n
        en = 4 * fp * (pm * abs(one(v["post_weight"])) if v["post_weight"] is None else pm * v["post_weight"].abs()) \
            if post else 0 * n
        if v["gate"] is not None:
            val, err, mag = grads["gate"], abs(scale) * (egr * (nv.abs() + en) + gr.abs() * en), \
                (gr * scale * nv).abs()
            err = err + 4 * F * mag
            k = u(ts["gate"].dtype)
            if v["gate"].shape == (d,):
                bounds["dgate"] = col("gate", val, err, mag)
            elif v["gate"].shape == x.shape:
                bounds["dgate"] = (val, err + 1.01 * k * (val.abs() + err))
            else:
                bounds["dgate"] = (val, err.sum(-1, keepdim=True) + d * F * mag.sum(-1, keepdim=True)
                                   + 1.01 * k * val.abs())
        if post:
            epv = 4 * fp * pm
            if v["post_weight"] is not None:
                bounds["dpost_weight"] = col("post_weight", grads["post_weight"], edn * pv.abs() + dn.abs() * epv,
                                             (dn * pv).abs())
            if v["post_bias"] is not None:
                bounds["dpost_bias"] = col("post_bias", grads["post_bias"], edn, dn.abs())
            pw = 1.0 if v["post_weight"] is None else v["post_weight"].abs()
            f, ef = dn * one(v["post_weight"]), edn * pw
            k0 = (f.abs() * pv.abs()).mean(-1, keepdim=True)
            ek0 = (ef * pv.abs() + f.abs() * epv).mean(-1, keepdim=True) + 2 * fp * k0
            k1 = (ef + 2 * fp * f.abs()).mean(-1, keepdim=True) if post == "layer" else 0.0
            edy = pinv * (ef + k1 + epv * k0 + (pv.abs() + epv) * ek0
                          + 4 * fp * (f.abs() + pv.abs() * k0 + f.abs().mean(-1, keepdim=True)))
        else:
            edy = edn
        dy = grads["y"]
        bounds["dy"] = (dy, edy + 1.01 * u(dt) * (dy.abs() + edy)
                        + (1.01 * ux * dy.abs() if rounded else 0.0))
        return bounds


def assert_within(got, want, bound, what=""):
    """|got - want| <= bound, and below a type's normal numbers half of their
    step: they lie smallest_normal eps apart (fp16: 2^-14 2^-10 = 2^-24), so that
    rounding to them is off by up to half of that (fp16: 2^-25 = 2.98e-8), more
    than u relative to the value."""
    half = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    got, want, bound = got.detach().double(), want.double(), bound.double() + half
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    bad = ~(off <= bound + 1e-30)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst {float(off[bad].max()):.3e} "
                           f"where {float(bound[bad].min()):.3e} is allowed")
