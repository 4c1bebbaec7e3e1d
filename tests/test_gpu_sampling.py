"""sample_tokens on the GPU against its definition in float64, row by row."""
import math

import pytest
import torch

import orthossm_b200 as O

pytestmark = pytest.mark.gpu
INF = float("inf")


def ref_row(l, e, t, k, p, m):
    """(token, decided): the definition in float64 on one row; decided is False
    where fp32 rounding could turn the choice: it falls otherwise with top_p or
    min_p moved by 2^-20 of itself, or another score is within 2^-18 of the
    best one's size."""
    l, e = l.double().cpu(), None if e is None else e.double().cpu()
    idx = torch.arange(l.numel())[l > -INF]  # drops NaN and -inf
    if idx.numel() == 0:
        return -1, True
    order = idx[torch.sort(l[idx], descending=True, stable=True).indices]
    if e is None or not t > 0:
        return int(order[0]), True
    x = l[order]
    w = torch.where(x == x[0], torch.ones_like(x), ((x - x[0]) / t).exp())
    score = x / t - e[order].log()
    score[score.isnan()] = -INF

    def choice(move):
        n = k if 0 < k < x.numel() else x.numel()
        if p < 1.0:
            c = w[:n].cumsum(0)
            n = max(1, int((c - w[:n] < p * move * c[-1]).sum()))
        if m > 0:
            n = max(1, int(((w[:n] >= m * move) | (w[:n] == 1)).sum()))  # equals of the first are exact
        s = score[:n]
        best = order[:n][s == s.max()].min()
        near = (s < s.max()) & (s >= s.max() - (s.max().abs() + 1) * 2.0 ** -18)
        return int(best), not bool(near.any())

    token, clear = choice(1.0)
    return token, clear and all(choice(1.0 + d)[0] == token for d in (2.0 ** -20, -2.0 ** -20))


def check(logits, noise, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    got = O.sample_tokens(logits, noise, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p).tolist()
    at = lambda x, b: x[b].item() if isinstance(x, torch.Tensor) else x  # noqa: E731
    loose = 0
    for b in range(logits.shape[0]):
        want, decided = ref_row(logits[b], None if noise is None else noise[b], at(temperature, b), at(top_k, b),
                                at(top_p, b), at(min_p, b))
        if decided:
            assert got[b] == want, (b, got[b], want)
        else:
            loose += 1
    assert loose <= 1 + logits.shape[0] // 20
    return got


def inputs(B, V, dtype, seed=0, spread=2.5, grid=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    l = torch.randn(B, V, device="cuda", generator=g) * spread
    if grid:
        l = (l / grid).round() * grid  # many equal logits
    return l.to(dtype), torch.empty(B, V, device="cuda").exponential_(generator=g)


FILTERS = [dict(), dict(top_k=1), dict(top_k=5), dict(top_k=50), dict(top_k=700), dict(top_p=0.05), dict(top_p=0.9),
           dict(top_p=0.999), dict(min_p=0.05), dict(top_k=40, top_p=0.8), dict(top_k=40, min_p=0.1),
           dict(top_p=0.95, min_p=0.02), dict(top_k=2000, top_p=0.9, min_p=0.001), dict(top_p=0.0), dict(min_p=1.0)]


@pytest.mark.parametrize("f", FILTERS, ids=lambda f: "_".join(f"{k}{v}" for k, v in f.items()) or "open")
@pytest.mark.parametrize("V", [1, 7, 1000, 32000, 50257])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_filters(f, V, dtype):
    l, e = inputs(6, V, dtype, seed=V)
    check(l, e, temperature=0.8, **f)


@pytest.mark.parametrize("f", FILTERS, ids=lambda f: "_".join(f"{k}{v}" for k, v in f.items()) or "open")
@pytest.mark.parametrize("V,spread", [(3000, 0.3), (40000, 0.05), (40000, 30.0)])
def test_ties_flat_and_peaked_rows(f, V, spread):
    """Logits on a coarse grid: thousands of equal ones at every threshold, kept
    by index; nearly flat rows (the nucleus is most of the row) and peaked ones."""
    l, e = inputs(4, V, torch.bfloat16, seed=1, spread=spread, grid=0.25)
    check(l, e, **f)


@pytest.mark.parametrize("f", [dict(), dict(top_k=50), dict(top_k=3000, top_p=0.7), dict(top_p=0.95), dict(top_p=0.5),
                               dict(top_p=0.9, min_p=0.001)],
                         ids=lambda f: "_".join(f"{k}{v}" for k, v in f.items()) or "open")
@pytest.mark.parametrize("B,V,spread", [(1, 150001, 1.0), (3, 131072, 2.5), (40, 30011, 1.0)])
def test_long_rows(f, B, V, spread):
    """Rows shared by several CTAs, wide prefixes, and rows beyond 2^17 logits."""
    l, e = inputs(B, V, torch.bfloat16, seed=B, spread=spread)
    check(l, e, temperature=1.1, **f)


@pytest.mark.parametrize("f", [dict(top_p=0.8), dict(top_p=0.97, min_p=1e-4), dict(top_p=0.3, min_p=0.02)],
                         ids=lambda f: "_".join(f"{k}{v}" for k, v in f.items()))
@pytest.mark.parametrize("period", [2, 3, 8])
@pytest.mark.parametrize("high", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_uneven_rows(dtype, high, period, f):
    """Rows whose large and small logits alternate in blocks of 16 bytes, so that
    what a few blocks show of the tail can be far from the whole row's."""
    V, block = 32768, 16 // dtype.itemsize
    l, e = inputs(76, V, torch.float32, seed=period, spread=1.0)
    every = (torch.arange(V, device="cuda") // block) % period == 0
    l[:, every if not high else ~every] -= 25.0
    check(l.to(dtype), e, **f)


@pytest.mark.parametrize("V,low,p,B", [(131072, -20.2, 0.9999, 3), (131072, -20.2, 0.9999, 80),
                                       (1 << 20, -21.5, 0.9998, 2), ((1 << 22) + 5, -22.5, 0.99965, 1)])
def test_peak_over_a_flat_tail(V, low, p, B):
    """Candidates of less than 2^-29 of the first one's weight, so many that
    together they decide where the nucleus ends: half of them stay."""
    l = torch.full((1, V), low, device="cuda")
    l[:, 0] = 0.0
    w = math.exp(low)
    whole = 1.0 + (V - 1) * w
    stay = 1 + (p * whole - 1.0) / w  # so many stay
    assert V / 4 < stay < 3 * V / 4
    off = 2.0 ** -18 * whole / w      # the masses' and the sums' fp32 roundings, in candidates
    for i in (int(stay - off - 2), int(stay + off + 2)):
        e = torch.ones(1, V, device="cuda")
        e[:, i] = 1e-30  # wins if it stays
        got = O.sample_tokens(l.expand(B, V), e.expand(B, V), top_p=p)
        assert got.tolist() == [i if i < stay else 0] * B


@pytest.mark.parametrize("V,spread,dtype", [(131072, 0.5, torch.float32), (50257, 1.5, torch.float32),
                                            (131072, 1.0, torch.bfloat16), (9001, 1.0, torch.float16)])
def test_prefix_end_in_any_batch(V, spread, dtype):
    """Noise that makes the last candidate of the prefix win, so that the token
    shows where it ends: the same for a row alone and in batches of any size,
    and where float64 has it, as far as fp32 weights can tell."""
    g = torch.Generator(device="cuda").manual_seed(V)
    l = (torch.randn(1, V, device="cuda", generator=g) * spread).to(dtype)
    order = torch.sort(l[0].double(), descending=True, stable=True).indices
    T = 0.9
    e = torch.empty(1, V, device="cuda")  # the score of the candidate in place r is r * 80 / V
    e[0, order] = (l[0].double()[order] / T - 80.0 / V * torch.arange(V, device="cuda")).exp().float()
    rank = torch.empty(V, dtype=torch.long, device="cuda")
    rank[order] = torch.arange(V, device="cuda")
    n = 160
    p = torch.linspace(0.35, 0.97, n, device="cuda")
    f = lambda b, **kw: O.sample_tokens(l.expand(b, V), e.expand(b, V), temperature=T, **kw)  # noqa: E731
    many = f(n, top_p=p)
    some = torch.cat([f(40, top_p=x) for x in p.split(40)])
    one = torch.cat([f(1, top_p=x) for x in p.split(1)])
    x = l[0].double()[order] / T
    w = (x - x[0]).exp()
    upto = w.cumsum(0)
    for b in range(n):
        end = int((upto - w < float(p[b]) * upto[-1]).sum()) - 1
        off = 2.0 ** -18 * float(upto[-1] / w[end]) + 1
        assert abs(int(rank[many[b]]) - end) <= off, (b, int(rank[many[b]]), end)
    assert torch.equal(many, some) and torch.equal(many, one)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_open_rows_of_every_length(dtype):
    """Unfiltered rows that end at any lane of a warp, at odd alignments."""
    for V in [*range(1, 20), 127, 128, 129, 255, 256, 257, 511, 513, 2047, 4095, 4097, 8191, 16383, 16385, 40001]:
        l, e = inputs(5, V, dtype, seed=V)
        s = l.double() - e.double().log()
        best = s.argmax(-1)
        second = s.scatter(1, best[:, None], -INF).amax(-1) if V > 1 else torch.full_like(s[:, 0], -INF)
        clear = s.amax(-1) - second > 2.0 ** -18 * (s.amax(-1).abs() + 1)
        got = O.sample_tokens(l, e)
        assert bool((got == best)[clear].all()), V


def test_all_equal():
    """One logit everywhere: the first k by index."""
    for val in (0.0, -0.0, 3.0, -7.5):
        l = torch.full((2, 9000), val, device="cuda")
        l[1, ::2] = -0.0 if val == 0.0 else val
        e = torch.empty_like(l).exponential_()
        e[:, 3] = 1e-30  # wins wherever index 3 stays
        assert O.sample_tokens(l, e, top_k=3).tolist()[0] < 3
        assert O.sample_tokens(l, e, top_k=4).tolist() == [3, 3]
        assert O.sample_tokens(l, e, top_p=4 / 9000 - 1e-5).tolist() == [3, 3]
        assert O.sample_tokens(l, e, top_p=2 / 9000 - 1e-5).tolist()[1] < 3
        assert O.sample_tokens(l, e, min_p=1.0).tolist() == [3, 3]
        assert O.sample_tokens(l, e).tolist() == [3, 3]
        assert O.sample_tokens(l).tolist() == [0, 0]
    for val in (INF, -1e30):  # noise cannot move such a score: the lowest index
        l = torch.full((2, 9000), val, device="cuda")
        for f in (dict(), dict(top_k=4), dict(top_p=0.3), dict(min_p=1.0)):
            assert O.sample_tokens(l, torch.empty_like(l).exponential_(), **f).tolist() == [0, 0]


@pytest.mark.parametrize("f", [dict(), dict(top_k=3), dict(top_p=0.5), dict(min_p=0.1), dict(top_k=9, top_p=0.9)])
def test_non_finite(f):
    V = 5000
    l, e = inputs(7, V, torch.float32, seed=2)
    l[0] = -INF                      # nothing left: -1
    l[1] = float("nan")
    l[2] = -INF
    l[2, 4321] = -5.0                # one left
    l[3, ::3] = float("nan")
    l[4, 17], l[4, 900] = INF, INF   # only the infinite ones have weight
    l[5] = -INF
    l[5, 7:40] = torch.finfo(torch.float32).min  # the type's lowest value is a candidate
    l[6, 100:] = -INF
    got = check(l, e, **f)
    assert got[:3] == [-1, -1, 4321] and got[4] in (17, 900) and 7 <= got[5] < 40 and got[6] < 100


def test_greedy():
    l, e = inputs(5, 4000, torch.bfloat16, grid=0.5)
    want = [int((r == r.max()).nonzero()[0]) for r in l.float().cpu()]
    assert O.sample_tokens(l).tolist() == want
    assert O.sample_tokens(l, e, temperature=0.0, top_p=0.9).tolist() == want
    t = torch.tensor([0.0, -1.0, float("nan"), 0.0, 0.0], device="cuda")
    assert O.sample_tokens(l, e, temperature=t, top_k=7).tolist() == want


def test_endless_temperature():
    """A temperature so high that its inverse is 0: every candidate is as likely."""
    l, e = inputs(4, 3000, torch.float32, seed=11)
    l[:, 7] = -INF
    e[:, 7] = 1e-30
    t = torch.tensor([INF, 3e38, 1.0, INF], device="cuda")
    for f in (dict(), dict(top_k=50), dict(min_p=0.5), dict(top_p=0.5)):
        check(l, e, temperature=t, **f)
        check(l, e, temperature=1e300, **f)


@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 32000), (torch.float32, 4001)])
def test_settings_of_each_row(dtype, V):
    B = 24
    l, e = inputs(B, V, dtype, seed=4)
    g = torch.Generator(device="cuda").manual_seed(0)
    u = torch.rand(4, B, device="cuda", generator=g)
    t = 0.5 + u[0]
    k = (u[1] * 100).to(torch.int32)
    p = u[2].clone()
    p[::5] = 1.0
    m = u[3] * 0.2
    m[::3] = 0.0
    k[::4] = 0
    check(l, e, temperature=t, top_k=k, top_p=p, min_p=m)
    check(l, e, temperature=0.7, top_k=k)
    check(l, e, temperature=t, top_p=p)
    check(l, e, temperature=t, min_p=m)
    check(l, e, temperature=t)


def test_widest_row():
    l = torch.zeros(2, 1 << 23, device="cuda")
    for f in (dict(), dict(top_p=0.5)):
        with pytest.raises(ValueError, match="candidates"):
            O.sample_tokens(l, l, **f)
    V = (1 << 23) - 1
    l, e = l[:, :V], torch.ones(2, V, device="cuda")
    e[0, V // 2 - 1], e[0, V // 2 + 1], e[1, V - 1] = 1e-20, 1e-30, 1e-30
    assert O.sample_tokens(l, e, top_p=0.5).tolist() == [V // 2 - 1, 0]
    assert O.sample_tokens(l, e).tolist() == [V // 2 + 1, V - 1]
    assert O.sample_tokens(l, e, top_k=V // 2).tolist() == [V // 2 - 1, 0]


def test_counts_of_a_wider_type():
    l, e = inputs(5, 3000, torch.float32, seed=12)
    want = O.sample_tokens(l, e).tolist()
    k = torch.tensor([2 ** 32 + 1, 2 ** 31, 2 ** 40, -2 ** 33 + 1, 1], device="cuda")
    got = O.sample_tokens(l, e, top_k=k).tolist()
    assert got[:4] == want[:4] and got[4] == int(l[4].argmax())
    assert O.sample_tokens(l, e, top_k=k.clamp(-9, 9)).tolist()[3] == want[3]


def test_layouts_and_output():
    l, e = inputs(6, 3001, torch.bfloat16, seed=5)
    want = O.sample_tokens(l, e, top_k=20, top_p=0.9).tolist()
    wide = torch.full((6, 3007), 9.0, device="cuda", dtype=torch.bfloat16)
    for off in (0, 1, 3):
        wide[:, off:off + 3001] = l
        assert O.sample_tokens(wide[:, off:off + 3001], e, top_k=20, top_p=0.9).tolist() == want
        we = torch.empty(6, 3010, device="cuda")
        we[:, off:off + 3001] = e
        assert O.sample_tokens(l, we[:, off:off + 3001], top_k=20, top_p=0.9).tolist() == want
        assert O.sample_tokens(wide[:, off:off + 3001], we[:, off:off + 3001]).tolist() == \
            O.sample_tokens(l, e).tolist()
    assert O.sample_tokens(l.t().contiguous().t(), e.t().contiguous().t(), top_k=20, top_p=0.9).tolist() == want
    assert O.sample_tokens(l[:1].expand(6, -1), e, top_k=20).shape == (6,)
    out = torch.zeros(6, dtype=torch.int64, device="cuda")
    assert O.sample_tokens(l, e, top_k=20, top_p=0.9, out=out) is out and out.tolist() == want
    assert O.sample_tokens(l[:0], e[:0]).shape == (0,)


def test_noise_extremes():
    """Zero noise wins outright, infinite and NaN noise lose to all others."""
    l = torch.zeros(3, 2000, device="cuda")
    e = torch.ones_like(l)
    e[0, 1234] = 0.0
    e[1] = INF
    e[1, 7] = 5.0
    e[2] = float("nan")
    e[2, 1999] = 1.0
    assert O.sample_tokens(l, e).tolist() == [1234, 7, 1999]
    assert O.sample_tokens(l, e, top_k=2000).tolist() == [1234, 7, 1999]
    assert O.sample_tokens(l, e, top_p=0.9999).tolist()[:2] == [1234, 7]


@pytest.mark.parametrize("f", [dict(), dict(top_k=6), dict(top_p=0.8), dict(min_p=0.2)])
def test_frequencies(f):
    """Tokens of 40000 rows of one distribution against its probabilities
    (chi-square; 5 standard deviations above the mean of its distribution)."""
    n, V = 40000, 12
    base = torch.linspace(2.0, -1.0, V, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(8)
    e = torch.empty(n, V, device="cuda").exponential_(generator=g)
    got = torch.bincount(O.sample_tokens(base.expand(n, V), e, **f), minlength=V).double().cpu()
    w = base.double().cpu().exp()
    w = w / w.sum()
    keep = torch.ones(V, dtype=torch.bool)
    if "top_k" in f:
        keep[f["top_k"]:] = False
    if "top_p" in f:
        keep &= w.cumsum(0) - w < f["top_p"]
    if "min_p" in f:
        keep &= w >= f["min_p"] * w[0]
    w = w * keep
    w = w / w.sum()
    assert float(got[~keep].sum()) == 0
    x2 = float(((got - n * w) ** 2 / (n * w))[keep].sum())
    dof = int(keep.sum()) - 1
    assert x2 < dof + 5 * math.sqrt(2 * dof) + 5


def test_repeats_streams_and_graphs():
    l, e = inputs(9, 32000, torch.bfloat16, seed=6)
    f = dict(temperature=0.9, top_k=50, top_p=0.9)
    want = O.sample_tokens(l, e, **f)
    assert all(torch.equal(want, O.sample_tokens(l, e, **f)) for _ in range(3))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.empty_like(want)
    with torch.cuda.stream(side):
        O.sample_tokens(l, e, **f, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            O.sample_tokens(l, e, **f, out=out)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    e.exponential_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, O.sample_tokens(l, e, **f))


def test_refusals():
    l = torch.zeros(2, 8, device="cuda")
    e = torch.ones(2, 8, device="cuda")
    f = O.sample_tokens
    for bad in [lambda: f(l[0], e[0]), lambda: f(l.double(), e), lambda: f(l, e.half()), lambda: f(l, e[:1]),
                lambda: f(l, e, temperature=-1.0), lambda: f(l, e, temperature=INF),
                lambda: f(l, e, temperature=float("nan")), lambda: f(l, e, top_k=-1),
                lambda: f(l, e, top_p=1.5), lambda: f(l, e, top_p=-0.1), lambda: f(l, e, min_p=2.0),
                lambda: f(l, e, top_k=torch.ones(3, dtype=torch.int32, device="cuda")),
                lambda: f(l, e, top_p=torch.ones(2)), lambda: f(l, e, out=torch.zeros(2, device="cuda")),
                lambda: f(l[:, :0], e[:, :0])]:
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="CUDA"):
        f(l.cpu(), e)
