"""Training operators on the GPU against float64 (tests/training_ref.py holds
the definitions and derives the bounds)."""
import pytest
import torch

import orthossm_b200 as O
from tests.training_ref import assert_within, embed_ref, lce_ref, norm_ref

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def lce_inputs(T, d, V, dt, ignored, seed=0):
    g = gen(seed)
    w = (torch.randn(V, d, device="cuda", generator=g) * 1.4 / d ** 0.5).to(dt)
    t = torch.randint(0, V, (T,), device="cuda", generator=g)
    h = (torch.randn(T, d, device="cuda", generator=g) + 3 * torch.rand(T, 1, device="cuda", generator=g) * w[t]).to(dt)
    off = torch.rand(T, device="cuda", generator=g) < ignored
    t[off] = -100
    return h.requires_grad_(), w.requires_grad_(), t


def check_lce(h, w, t, reduction="mean", z_loss=0.0, seed=1, scale=1.0, **kw):
    loss = O.linear_cross_entropy(h, w, t, reduction=reduction, z_loss=z_loss, **kw)
    up = torch.rand(loss.shape, device="cuda", generator=gen(seed)) * 2 * scale
    up = up - 0.5 * scale if reduction == "none" else up
    got = (loss, *torch.autograd.grad(loss, (h, w), up))
    want, bound = lce_ref(h, w, t, up, z_loss=z_loss, reduction=reduction,
                          ignore=kw.get("ignore_index", -100))
    assert got[0].dtype == FP and got[1].dtype == h.dtype and got[2].dtype == w.dtype
    for a, b, c, what in zip(got, want, bound, ("loss", "dhidden", "dweight")):
        assert_within(a, b.view(a.shape), c.view(a.shape), what)
    with torch.no_grad():  # without a graph: the same losses
        assert torch.equal(O.linear_cross_entropy(h, w, t, reduction=reduction, z_loss=z_loss, **kw), loss)
    return got


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("T,d,V,ignored,reduction,z_loss", [
    (1, 8, 1, 0.0, "mean", 0.0), (1, 512, 32000, 0.0, "none", 0.0), (2, 64, 2, 0.0, "sum", 1e-2),
    (129, 72, 1001, 0.3, "mean", 0.0), (128, 128, 256, 0.0, "none", 1e-3), (300, 512, 777, 0.9, "none", 0.0),
    (257, 320, 4097, 0.02, "sum", 1e-4), (5, 1000, 257, 0.4, "mean", 1e-1), (640, 2048, 513, 0.5, "mean", 0.0),
    (4000, 264, 9999, 0.1, "mean", 0.0), (127, 8, 50001, 1.0, "mean", 0.0), (1000, 16, 300, 1.0, "none", 0.0),
    (2500, 256, 40000, 0.0, "none", 0.0), (64, 512, 50000, 0.1, "mean", 0.0)])
def test_loss(T, d, V, ignored, reduction, z_loss, dt):
    check_lce(*lce_inputs(T, d, V, dt, ignored), reduction=reduction, z_loss=z_loss)


def test_loss_pieces_of_the_vocabulary():
    """More tokens than one piece of dz takes: three pieces, the last a ragged one."""
    check_lce(*lce_inputs(65600, 40, 8500, BF, 0.2), reduction="mean", z_loss=1e-3)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("scale", [65536.0, 2.0 ** -20])
def test_loss_scaled_gradients(dt, scale):
    """An upstream factor (a loss scale) reaches the gradients whole: dz is in units of the largest."""
    T, d, V = 200, 64, 1000
    h, w, t = lce_inputs(T, d, V, dt, 0.1)
    loss = O.linear_cross_entropy(h, w, t)
    up = torch.tensor(scale / 4096, device="cuda")
    g1 = torch.autograd.grad(loss, (h, w), up, retain_graph=True)
    want, bound = lce_ref(h, w, t, up)
    for a, b, c in zip(g1, want[1:], bound[1:]):
        assert_within(a, b, c)


def test_loss_ignored_states_reach_nothing():
    h, w, t = lce_inputs(300, 128, 1000, BF, 0.4)
    clean = check_lce(h, w, t)
    with torch.no_grad():
        h[t == -100] = float("nan")
        h[(t == -100).nonzero()[::2, 0]] = float("inf")
    dirty = check_lce(h, w, t)
    for a, b in zip(clean, dirty):
        assert torch.equal(a, b)
    assert (dirty[1][t == -100] == 0).all()


def test_loss_no_targets_at_all():
    h, w, t = lce_inputs(40, 64, 300, BF, 1.0)
    with torch.no_grad():
        h.fill_(float("nan"))
    for reduction in ("mean", "sum", "none"):
        loss = O.linear_cross_entropy(h, w, t, reduction=reduction)
        assert (loss == 0).all()
        dh, dw = torch.autograd.grad(loss.sum(), (h, w))
        assert (dh == 0).all() and (dw == 0).all()
    h0 = torch.empty(0, 64, device="cuda", dtype=BF, requires_grad=True)
    loss = O.linear_cross_entropy(h0, w, t[:0])
    dh, dw = torch.autograd.grad(loss, (h0, w))
    assert loss == 0 and dh.shape == (0, 64) and (dw == 0).all()
    assert O.linear_cross_entropy(h0, w, t[:0], reduction="none").shape == (0,)


def test_loss_unknown_targets_and_values():
    h, w, t = lce_inputs(200, 64, 300, BF, 0.2)
    good = O.linear_cross_entropy(h, w, t, reduction="none")
    bad = t.clone()
    bad[3], bad[150] = 300, -1
    loss = O.linear_cross_entropy(h, w, bad, reduction="none")
    assert loss.isnan().nonzero()[:, 0].tolist() == [3, 150]
    rest = ~loss.isnan()
    assert torch.equal(loss[rest], torch.where(t != -100, good, 0.0)[rest])
    dh, = torch.autograd.grad(loss, h, torch.ones_like(loss))
    assert dh[[3, 150]].isnan().all() and not dh[rest].isnan().any()
    assert O.linear_cross_entropy(h, w, bad).isnan()
    # another mark for tokens without a target
    check_lce(h, w, torch.where(t == -100, -1, t), ignore_index=-1)
    check_lce(h, w, torch.where(t == -100, 7, t), ignore_index=7)
    with torch.no_grad():  # a state that is not finite has no finite loss, the others theirs
        k = int((t != -100).nonzero()[5, 0])
        h[k, 3] = float("inf")
        loss = O.linear_cross_entropy(h, w, t, reduction="none")
    assert not loss[k].isfinite() and torch.equal(loss[torch.arange(200, device="cuda") != k],
                                                  good[torch.arange(200, device="cuda") != k])


def test_loss_large_logits():
    """Logits of a few hundred: the sums follow the maximum."""
    h, w, t = lce_inputs(150, 64, 3000, BF, 0.0)
    with torch.no_grad():
        h.mul_(60.0)
    check_lce(h, w, t, reduction="none")
    with torch.no_grad():  # columns in rising order: the maximum moves with every tile
        w.copy_(torch.linspace(-1, 1, 3000, device="cuda")[:, None].expand(-1, 64))
        h.fill_(4.0)
    check_lce(h, w, t, reduction="none")


def test_loss_layouts():
    """Batches, strides, addresses off 16 bytes, int32 targets, gradients of one input alone."""
    B, S, d, V = 3, 50, 64, 500
    h, w, t = lce_inputs(B * S, d, V, BF, 0.1)
    want = O.linear_cross_entropy(h, w, t, reduction="none")
    gh, gw = torch.autograd.grad(want.sum(), (h, w))
    wide = torch.zeros(B, S, d + 24, device="cuda", dtype=BF)
    wide[..., 8:8 + d] = h.detach().view(B, S, d)
    off = torch.zeros(V * d + 3, device="cuda", dtype=BF)
    off[3:] = w.detach().reshape(-1)
    for hh in (h.detach().view(B, S, d), wide[..., 8:8 + d], h.detach().view(B, S, d).transpose(0, 1).contiguous().transpose(0, 1)):
        for ww in (w.detach(), off[3:].view(V, d), w.detach().t().contiguous().t()):
            hh, ww = hh.detach().requires_grad_(), ww.detach().requires_grad_()
            loss = O.linear_cross_entropy(hh, ww, t.view(B, S).int(), reduction="none")
            assert loss.shape == (B, S) and torch.equal(loss.reshape(-1), want)
            a, = torch.autograd.grad(loss.sum(), hh, retain_graph=True)
            b, = torch.autograd.grad(loss.sum(), ww)
            assert torch.equal(a.reshape(-1, d), gh) and torch.equal(b, gw)
    one = O.linear_cross_entropy(h[5], w, t[5], reduction="none")
    assert one.shape == () and torch.equal(one, want[5])


def test_loss_gradient_by_differences():
    """Along a direction: (loss(h + s e) - loss(h - s e)) / 2s in float64 of the rounded points."""
    h, w, t = lce_inputs(64, 64, 500, HF, 0.2)
    loss = O.linear_cross_entropy(h, w, t, reduction="sum")
    dh, dw = torch.autograd.grad(loss, (h, w))
    for x, g, at in ((h, dh, 0), (w, dw, 1)):
        e = (torch.randn(x.shape, device="cuda", generator=gen(3)) * 2.0 ** -6).to(HF)
        hi, lo = (x + e).detach(), (x - e).detach()
        f = lambda v: float(lce_ref(*((v, w) if at == 0 else (h, v)), t, torch.ones((), device="cuda"),
                                    reduction="sum")[0][0])  # noqa: E731
        step = hi.double() - lo.double()
        slope = float((g.double() * step).sum())
        # third order along the step, and the gradient's own rounding
        third = float(sum(((hi.double() - x.double()).abs().flatten() ** 3).tolist())) * 8
        assert abs(f(hi) - f(lo) - slope) <= 2.0 ** -9 * float((g.double() * step).abs().sum()) + third + 1e-3 * abs(slope)


def test_loss_repeats_and_batches_alike():
    h, w, t = lce_inputs(3000, 128, 5000, BF, 0.1)
    first = check_lce(h, w, t)
    for _ in range(3):
        again = check_lce(h, w, t)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_loss_captured_and_on_other_streams():
    h, w, t = lce_inputs(500, 128, 3000, BF, 0.2)
    side = torch.cuda.Stream()

    def step():
        loss = O.linear_cross_entropy(h, w, t)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w)))

    want = step()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (7, 8):
        h2, w2, t2 = lce_inputs(500, 128, 3000, BF, 0.5, seed)
        with torch.no_grad():
            h.copy_(h2), w.copy_(w2), t.copy_(t2)
        graph.replay()
        torch.cuda.synchronize()
        now = step()
        assert all(torch.equal(a, b) for a, b in zip(got, now))
    assert O.workspace_status() == 0


def test_calls_at_once():
    """The three operators on two streams at the same time, eagerly and as two
    graphs: each call has its own workspace."""
    sets = [(lce_inputs(700, 264, 9000, BF, 0.2, seed), torch.randint(0, 900, (5000,), device="cuda", generator=gen(seed)),
             torch.randn(5000, 264, device="cuda", generator=gen(seed)).to(BF)) for seed in (1, 2)]

    def step(inputs):
        (h, w, t), ids, g = inputs
        loss = O.linear_cross_entropy(h, w, t, z_loss=1e-3)
        out = O.embed_tokens(ids, w)
        r, n = O.residual_norm(out, g, norm="layer", post_norm="rms")
        return (loss.detach(), *torch.autograd.grad(loss, (h, w)), *torch.autograd.grad((r, n), w, (g, g)))

    want = [step(s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append([step(s) for _ in range(3)])
        torch.cuda.synchronize()
        for a, many in zip(want, got):
            assert all(torch.equal(x, y) for b in many for x, y in zip(a, b))
    graphs, held = [torch.cuda.CUDAGraph() for _ in sets], []
    for gr, s in zip(graphs, sets):
        with torch.cuda.graph(gr):
            held.append(step(s))
    for _ in range(3):
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, held):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert O.workspace_status() == 0


def test_loss_refusals():
    h, w, t = lce_inputs(10, 64, 100, BF, 0.0)
    f = O.linear_cross_entropy
    for bad in (lambda: f(h.float(), w.float(), t), lambda: f(h, w.half(), t), lambda: f(h[:, :32], w, t),
                lambda: f(h[:, :60].contiguous(), w[:, :60].contiguous(), t), lambda: f(h, w, t[:5]),
                lambda: f(h, w, t.float()), lambda: f(h, w, t, reduction="max"), lambda: f(h, w, t, z_loss=-1.0),
                lambda: f(h, w, t, z_loss=float("nan")), lambda: f(h, w[:0], t),
                lambda: f(h, w, t, ignore_index=1 << 63)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        f(h.cpu(), w.cpu(), t.cpu())
    g, = torch.autograd.grad(f(h, w, t), h, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError):
        f(fwd.make_dual(h.detach(), torch.ones_like(h)), w, t)


# ----------------------------------------------------------------------------
# embeddings
# ----------------------------------------------------------------------------

def check_embed(ids, w, scale=1.0, seed=2):
    out = O.embed_tokens(ids, w, scale=scale)
    g = torch.randn(out.shape, device="cuda", generator=gen(seed)).to(w.dtype)
    dw, = torch.autograd.grad(out, w, g)
    want, bound = embed_ref(ids, w, g, scale)
    assert out.dtype == w.dtype and dw.dtype == w.dtype
    assert_within(out, want[0], bound[0], "out")
    assert_within(dw, want[1], bound[1], "dweight")
    return out, dw


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("T,d,V,scale", [(1, 1, 1, 1.0), (1, 512, 32000, 2.0), (7, 3, 2, 1.0), (300, 64, 50, 22.6),
                                         (2049, 100, 1000, 1.0), (5000, 513, 700, 0.5), (4096, 512, 300, 1.0),
                                         (70000, 24, 5, 1.0), (3000, 1040, 140000, 1.0), (300000, 8, 300000, 1.0)])
def test_embed(T, d, V, scale, dt):
    g = gen(T)
    w = torch.randn(V, d, device="cuda", generator=g).to(dt).requires_grad_()
    ids = (V ** torch.rand(T, device="cuda", generator=g)).long().sub_(1).clamp_(0, V - 1)
    check_embed(ids, w, scale)


def test_embed_padding_and_one_token_everywhere():
    w = torch.randn(500, 72, device="cuda", generator=gen(0)).to(BF).requires_grad_()
    ids = torch.randint(0, 500, (3, 4000), device="cuda", generator=gen(1))
    ids[:, ::3] = -1
    ids[0, 5], ids[1, 7], ids[2, 8] = 500, 1 << 40, -(1 << 50)
    out, _ = check_embed(ids, w)
    assert (out[:, ::3] == 0).all() and (out[0, 5] == 0).all()
    check_embed(torch.full((20000,), 499, device="cuda"), w)      # one token's sum over all chunks
    _, dw = check_embed(torch.full((9000,), -1, device="cuda"), w)  # none at all
    assert (dw == 0).all()
    one = torch.full((5000,), 3, device="cuda")
    one[2500:] = -1
    check_embed(one, w)


def test_embed_layouts():
    V, d = 300, 64
    w = torch.randn(V, d, device="cuda", generator=gen(0)).to(BF)
    ids = torch.randint(0, V, (40, 6), device="cuda", generator=gen(1))
    want = w[ids]
    off = torch.zeros(V * d + 3, device="cuda", dtype=BF)
    off[3:] = w.reshape(-1)
    wide = torch.zeros(V, d + 5, device="cuda", dtype=BF)
    wide[:, 2:2 + d] = w
    for ww in (w, off[3:].view(V, d), wide[:, 2:2 + d], w.t().contiguous().t()):
        assert torch.equal(O.embed_tokens(ids, ww), want)
        assert torch.equal(O.embed_tokens(ids.int().t(), ww), want.transpose(0, 1))
        assert torch.equal(O.embed_tokens(ids[:, ::2], ww), want[:, ::2])
    p = w.clone().requires_grad_()
    out = O.embed_tokens(ids, p)
    g = torch.randn(out.shape, device="cuda", generator=gen(2)).to(BF)
    dw, = torch.autograd.grad(out, p, g, retain_graph=True)
    stretched = torch.randn(40, 1, d, device="cuda", generator=gen(3)).to(BF).expand(40, 6, d)
    for gg in (g.transpose(0, 1).contiguous().transpose(0, 1), off.new_zeros(40 * 6 * d + 1)[1:].view(g.shape).copy_(g)):
        assert torch.equal(torch.autograd.grad(out, p, gg, retain_graph=True)[0], dw)
    assert torch.equal(torch.autograd.grad(out, p, stretched, retain_graph=True)[0],
                       torch.autograd.grad(out, p, stretched.contiguous())[0])
    e = torch.empty(0, 5, dtype=torch.int64, device="cuda")
    out = O.embed_tokens(e, p)
    assert out.shape == (0, 5, d)
    assert (torch.autograd.grad(out.sum(), p)[0] == 0).all()
    assert torch.equal(O.embed_tokens(torch.tensor(5, device="cuda"), w), w[5])


def test_embed_repeats_captured_and_refused():
    w = torch.randn(1000, 256, device="cuda", generator=gen(0)).requires_grad_()
    ids = torch.randint(0, 40, (9000,), device="cuda", generator=gen(1))
    g = torch.randn(9000, 256, device="cuda", generator=gen(2))

    def step():
        out = O.embed_tokens(ids, w, scale=3.0)
        return out.detach(), torch.autograd.grad(out, w, g)[0]

    want = step()
    assert all(torch.equal(a, b) for a, b in zip(want, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    ids.copy_(torch.randint(0, 1000, (9000,), device="cuda", generator=gen(5)))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))
    f = O.embed_tokens
    for bad in (lambda: f(ids.float(), w), lambda: f(ids, w.double()), lambda: f(ids, w[0]),
                lambda: f(ids, w, scale=float("inf"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        f(ids.cpu(), w)


# ----------------------------------------------------------------------------
# residual and norms
# ----------------------------------------------------------------------------

def norm_inputs(shape, xdt, ydt, norm, post, gate, affine=True, wdt=None, y=True, seed=0):
    g, d = gen(seed), shape[-1]
    rn = lambda *n: torch.randn(*n, device="cuda", generator=g)  # noqa: E731
    wdt = wdt or ydt
    ts = dict.fromkeys(("x", "y", "weight", "bias", "gate", "post_weight", "post_bias"))
    ts["x"] = rn(*shape).mul_(2).add_(0.3).to(xdt)
    if y:
        ts["y"] = rn(*shape).add_(-0.2).to(ydt)
    if affine:
        ts["weight"] = (1 + 0.3 * rn(d)).to(wdt)
        ts["bias"] = rn(d).to(wdt) if norm == "layer" else None
        if post:
            ts["post_weight"] = (1 + 0.3 * rn(d)).to(wdt)
            ts["post_bias"] = rn(d).to(wdt) if post == "layer" else None
    if gate:
        ts["gate"] = rn(*{"channel": (d,), "token": (*shape[:-1], 1), "full": shape}[gate]).to(wdt)
    return {k: None if t is None else t.requires_grad_() for k, t in ts.items()}


def check_norm(ts, norm="rms", post=None, scale=1.0, eps=1e-5, use_r=True, out_dtype=None, seed=3):
    r, h = O.residual_norm(ts["x"], ts["y"], ts["weight"], ts["bias"], norm=norm, eps=eps, gate=ts["gate"], scale=scale,
                           post_norm=post, post_weight=ts["post_weight"], post_bias=ts["post_bias"],
                           out_dtype=out_dtype)
    g = gen(seed)
    dr = torch.randn(r.shape, device="cuda", generator=g).to(r.dtype) if use_r else None
    dh = torch.randn(h.shape, device="cuda", generator=g).to(h.dtype)
    names = [k for k, t in ts.items() if t is not None]
    grads = torch.autograd.grad((h, r) if use_r else h, [ts[k] for k in names], (dh, dr) if use_r else dh)
    got = {"r": r, "h": h, **{"d" + k: v for k, v in zip(names, grads)}}
    want = norm_ref(ts, dict(norm=norm, post_norm=post, scale=scale, eps=eps), dr, dh)
    for k, (v, b) in want.items():
        assert got[k].dtype == (h.dtype if k == "h" else r.dtype if k == "r" else ts[k[1:]].dtype)
        assert_within(got[k], v, b, k)
    with torch.no_grad():
        r2, h2 = O.residual_norm(ts["x"], ts["y"], ts["weight"], ts["bias"], norm=norm, eps=eps, gate=ts["gate"],
                                 scale=scale, post_norm=post, post_weight=ts["post_weight"],
                                 post_bias=ts["post_bias"], out_dtype=out_dtype)
    assert torch.equal(r2, r) and torch.equal(h2, h)
    return got


@pytest.mark.parametrize("xdt,ydt", [(BF, BF), (HF, HF), (FP, FP), (FP, BF), (FP, HF)])
@pytest.mark.parametrize("shape", [(1, 1), (3, 8), (2, 5, 37), (33, 256), (9, 512), (130, 513), (5, 1000), (40, 2048),
                                   (3, 4100), (6, 8192)])
def test_norm_plain(shape, xdt, ydt):
    for norm in ("rms", "layer"):
        check_norm(norm_inputs(shape, xdt, ydt, norm, None, None), norm, scale=1.0)
        check_norm(norm_inputs(shape, xdt, ydt, norm, None, None, wdt=FP), norm, scale=0.7, use_r=False)
        check_norm(norm_inputs(shape, xdt, ydt, norm, None, None, affine=False, y=False), norm, out_dtype=ydt)


@pytest.mark.parametrize("xdt,ydt", [(BF, BF), (FP, HF), (FP, FP)])
@pytest.mark.parametrize("shape", [(1, 3), (2, 300, 64), (50, 384), (20, 520), (17, 1111), (5, 6000), (3, 8191), (2, 8192)])
@pytest.mark.parametrize("gate,post", [(g, p) for g in (None, "channel", "token", "full")
                                       for p in (None, "rms", "layer") if g or p])
def test_norm_gated(shape, gate, post, xdt, ydt):
    norm = "layer" if gate in ("token", None) else "rms"
    check_norm(norm_inputs(shape, xdt, ydt, norm, post, gate, wdt=FP if shape[-1] == 384 else None), norm, post, 0.5)


@pytest.mark.parametrize("dt", [BF, HF])
def test_norm_rows_of_close_values(dt):
    """Rows whose spread is below a step of the stream's type: backward norms the sum, not what was returned of it."""
    ts = norm_inputs((400, 3), dt, dt, "layer", None, None)
    check_norm(ts, "layer", scale=0.5)
    ts = norm_inputs((50, 512), dt, dt, "layer", None, None)
    with torch.no_grad():
        ts["x"].fill_(100.0)
        ts["y"].mul_(0.05)
    check_norm(ts, "layer")


def test_norm_many_rows():
    """Sums over more rows than blocks, in fixed order."""
    a = check_norm(norm_inputs((70001, 64), BF, BF, "rms", None, None), "rms")
    b = check_norm(norm_inputs((70001, 64), BF, BF, "rms", None, None), "rms")
    assert all(torch.equal(a[k], b[k]) for k in a)
    check_norm(norm_inputs((20011, 96), FP, BF, "layer", "rms", "channel"), "layer", "rms", 0.3)


def test_norm_layouts():
    """Strided, misaligned and stretched inputs give what their copies give."""
    d = 64
    base = norm_inputs((4, 10, d), BF, BF, "rms", "rms", "full")
    want = check_norm(base, "rms", "rms", 0.5)

    def moved(t, how):
        if t.dim() == 1:
            buf = torch.zeros(t.numel() + 1, device="cuda", dtype=t.dtype)
            buf[1:] = t.detach()
            return buf[1:].requires_grad_()
        if how == 0:
            buf = torch.zeros(*t.shape[:-1], d + 5, device="cuda", dtype=t.dtype)
            buf[..., 3:3 + d] = t.detach()
            return buf[..., 3:3 + d].requires_grad_()
        return t.detach().transpose(0, 1).contiguous().transpose(0, 1).requires_grad_()

    for how in (0, 1):
        ts = {k: None if t is None else moved(t, how) for k, t in base.items()}
        got = check_norm(ts, "rms", "rms", 0.5)
        assert torch.equal(got["h"], want["h"]) and torch.equal(got["r"], want["r"])
    x = torch.randn(1, d, device="cuda", generator=gen(0)).to(BF)
    r, h = O.residual_norm(x.expand(6, d), x.expand(6, d))
    r1, h1 = O.residual_norm(x, x)
    assert torch.equal(r, r1.expand(6, d)) and torch.equal(h, h1.expand(6, d))
    # a gradient that is a stretched value
    x = torch.randn(30, d, device="cuda", generator=gen(1)).to(BF).requires_grad_()
    r, h = O.residual_norm(x, x.detach())
    a, = torch.autograd.grad(h.sum() + r.sum(), x)
    r, h = O.residual_norm(x, x.detach())
    b, = torch.autograd.grad((r, h), x, (torch.ones_like(r), torch.ones_like(h)))
    assert torch.equal(a, b)
    # the same tensor as stream and block output, and used again
    r, h = O.residual_norm(x, x)
    a, = torch.autograd.grad(h.float().square().sum() + (x * 2).float().sum(), x)
    assert a.isfinite().all()
    r, h = O.residual_norm(torch.empty(0, d, device="cuda", dtype=BF, requires_grad=True))
    assert h.shape == (0, d)


def test_norm_zero_rows_and_values():
    x = torch.zeros(5, 64, device="cuda")
    r, h = O.residual_norm(x, torch.zeros_like(x), norm="layer", eps=1e-5)
    assert (h == 0).all()
    x[2] = float("nan")
    x[3, 4] = float("inf")
    r, h = O.residual_norm(x, torch.ones_like(x), eps=1e-5)
    assert torch.equal(h[[0, 1, 4]], h[:1].expand(3, 64)) and h[2].isnan().all() and h[3, 4].isnan()
    x = torch.full((3, 512), 200.0, device="cuda", dtype=HF)  # the sum of squares passes fp16's range
    assert_within(O.residual_norm(x)[1], torch.ones(3, 512, device="cuda"), torch.full((3, 512), 2.0 ** -11, device="cuda"))
    x = torch.full((2, 1000), 4096.0, device="cuda")
    x[:, ::2] += 1
    assert_within(O.residual_norm(x, norm="layer", eps=0.0)[1].abs(), torch.ones(2, 1000, device="cuda"),
                  torch.full((2, 1000), 2e-3, device="cuda"))


def test_norm_captured_and_streams():
    ts = norm_inputs((300, 512), BF, BF, "rms", None, None)
    dh = torch.randn(300, 512, device="cuda", generator=gen(4)).to(BF)

    def step():
        r, h = O.residual_norm(ts["x"], ts["y"], ts["weight"])
        return (r.detach(), h.detach(), *torch.autograd.grad((r, h), [ts["x"], ts["y"], ts["weight"]], (dh, dh)))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        ts["x"].add_(1)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_norm_refusals():
    x = torch.zeros(4, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    f = O.residual_norm
    for bad in (lambda: f(x.double()), lambda: f(x, x[:2]), lambda: f(x.half(), x), lambda: f(x.half(), x.bfloat16()),
                lambda: f(x, x, w[:3]), lambda: f(x, x, w.double()), lambda: f(x, norm="batch"),
                lambda: f(x, x, post_norm="batch"), lambda: f(x, gate=w), lambda: f(x, post_norm="rms"),
                lambda: f(x, x, post_weight=w), lambda: f(x, x, gate=w[:5]), lambda: f(x, x, gate=torch.ones(4, device="cuda")),
                lambda: f(x, eps=-1.0), lambda: f(x, x, scale=float("nan")),
                lambda: f(torch.zeros(2, 8193, device="cuda")), lambda: f(x.bfloat16(), out_dtype=FP)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        f(x.cpu())
