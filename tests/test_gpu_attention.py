"""packed_attention on the GPU against a float64 restatement that looks at the
seen keys alone (tests/attention_ref.py), at the lengths, masks, layouts and
values where it can go wrong; every bound is derived there."""
import pytest
import torch

import orthossm_b200 as O
from tests.attention_ref import bound, packed_attention_ref

pytestmark = pytest.mark.gpu


def cum(v):
    return torch.tensor([0] + list(v), device="cuda").cumsum(0).to(torch.int32)


def check(out, q, k, v, cu_q, cu_k, **kw):
    ref, mag, owned = packed_attention_ref(q, k, v, cu_q, cu_k, **kw)
    got = out.double().cpu()
    vmax = float(torch.nan_to_num(v, 0.0, 0.0, 0.0).abs().max()) if v.numel() else 0.0
    lim = bound(ref, mag, q.dtype, k.shape[0], vmax)
    bad = ((got - ref).abs() > lim) | ~torch.isfinite(got)
    assert not bool(bad[owned].any()), f"{int(bad[owned].sum())} values off, worst " \
        f"{float(((got - ref).abs() / lim)[owned].max())} of the bound"
    return owned


def packed(lens, H, Hkv, hd, dtype, seed=0):
    """q, k, v of self-attending prompts as one projection leaves them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = sum(lens)
    qkv = torch.randn(T, H + 2 * Hkv, hd, device="cuda", generator=g).to(dtype)
    return (*qkv.split([H, Hkv, Hkv], 1), cum(lens))


HEADS = [(8, 8, 64), (4, 1, 64), (6, 2, 128), (2, 2, 32), (3, 3, 8), (4, 2, 80), (2, 1, 96), (1, 1, 120), (16, 2, 128)]


@pytest.mark.parametrize("H,Hkv,hd", HEADS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_packed_prompts(H, Hkv, hd, dtype):
    """Prompts of lengths around every tile edge, with empty ones between."""
    lens = [1, 0, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 0, 255, 256, 257, 300, 390]
    q, k, v, cu = packed(lens, H, Hkv, hd, dtype)
    out = O.packed_attention(q, k, v, cu, max_seqlen_q=max(lens))
    check(out, q, k, v, cu, cu)


@pytest.mark.parametrize("window", [1, 2, 16, 100, 128, 129, 512, 5000])
@pytest.mark.parametrize("H,Hkv,hd,dtype", [(2, 2, 64, torch.bfloat16), (4, 2, 128, torch.float16)])
def test_windows(window, H, Hkv, hd, dtype):
    lens = [1, 130, 700, 257, 1100]
    q, k, v, cu = packed(lens, H, Hkv, hd, dtype, seed=window)
    out = O.packed_attention(q, k, v, cu, max_seqlen_q=max(lens), window=window)
    check(out, q, k, v, cu, cu, window=window)


# (queries, keys) of each sequence: tokens and pieces against longer caches, no keys at all, more queries than keys
# (the first queries then see nothing), no queries
PAIRS = [
    [(1, 1)], [(1, 0)], [(1, 1), (1, 17), (1, 0), (1, 1000), (1, 128)], [(1, 5000)],
    [(2, 2), (3, 100), (5, 3), (0, 50), (4, 64), (2, 1500)], [(16, 16), (16, 1000), (7, 2), (17, 40)],
    [(64, 3000), (1, 10), (33, 33)], [(200, 100), (130, 1), (5, 0)], [(300, 900), (128, 2000), (1, 1500)],
    [(100, 4000)],
]


@pytest.mark.parametrize("pairs", PAIRS, ids=lambda p: "_".join(f"{a}x{b}" for a, b in p))
@pytest.mark.parametrize("H,Hkv,hd,dtype", [(8, 8, 64, torch.bfloat16), (8, 1, 128, torch.bfloat16),
                                            (6, 2, 64, torch.float16), (24, 1, 32, torch.float16),
                                            (2, 2, 80, torch.bfloat16)])
@pytest.mark.parametrize("window", [None, 40])
def test_against_a_cache(pairs, H, Hkv, hd, dtype, window):
    """Queries against a cache with room left: NaN and infinities in the free
    slots, in front of the first sequence and behind the last must not matter."""
    g = torch.Generator(device="cuda").manual_seed(len(pairs))
    slots = max(b for _, b in pairs) + 37
    n = len(pairs)
    q = torch.randn(sum(a for a, _ in pairs), H, hd, device="cuda", generator=g).to(dtype)
    k, v = (torch.randn(n, slots, Hkv, hd, device="cuda", generator=g).to(dtype) for _ in range(2))
    for b, (_, nk) in enumerate(pairs):
        k[b, nk:] = float("nan")
        v[b, nk:] = float("inf") if b % 2 else float("nan")
    k, v = k.view(n * slots, Hkv, hd), v.view(n * slots, Hkv, hd)
    cu_q, cu_k = cum(a for a, _ in pairs), cum([slots] * n)
    kv = torch.tensor([b for _, b in pairs], device="cuda", dtype=torch.int32)
    out = O.packed_attention(q, k, v, cu_q, cu_k, max_seqlen_q=max(a for a, _ in pairs), kv_lengths=kv, window=window)
    check(out, q, k, v, cu_q, cu_k, kv_lengths=kv, window=window)


@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nq,nk", [(400, 400), (3, 300), (140, 700)])
def test_hidden_values_do_not_matter(what, hd, nq, nk):
    """Non-finite keys and values inside the sequence reach the queries that
    see them and no others: ahead of the query, and behind its window."""
    dtype, H, W = torch.bfloat16, 2, 150
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(nq, H, hd, device="cuda", generator=g).to(dtype)
    k, v = (torch.randn(nk, H, hd, device="cuda", generator=g).to(dtype) for _ in range(2))
    clean_k, clean_v = k.clone(), v.clone()
    cu_q, cu_k = cum([nq]), cum([nk])
    places = [nk - 1, nk - 2, max(0, nk - 170), 5]
    for j in places:
        v[j, 0, 3], v[j, 1, hd - 1] = what, what
    k[nk - 1, 0, 0] = what
    out = O.packed_attention(q, k, v, cu_q, cu_k, max_seqlen_q=nq, window=W)
    ref, mag, _ = packed_attention_ref(q, clean_k, clean_v, cu_q, cu_k, window=W)
    at = torch.arange(nq) + nk - nq
    seen = torch.stack([(at >= j) & (at - j < W) for j in places]).any(0)
    blind = ~seen
    assert int(blind.sum()) > 0 or nq < 10
    got, lim = out.double().cpu(), bound(ref, mag, dtype, nk, 6.0)
    assert bool(((got - ref).abs() <= lim)[blind].all())
    # the other channels of a query that sees a bad value are not touched by it
    body = torch.ones(H, hd, dtype=torch.bool)
    body[0], body[1, hd - 1] = False, False
    assert bool(((got - ref).abs() <= lim)[:, body].all())
    # a seen value arrives: channel hd - 1 of head 1 (finite weights)
    if what == what:
        assert bool((got[seen][:, 1, hd - 1] == what).all())
    else:
        assert bool(got[seen][:, 1, hd - 1].isnan().all())


@pytest.mark.parametrize("what", [float("nan"), float("inf")])
@pytest.mark.parametrize("G,hd,nq,window,most", [(16, 64, 2, None, 2), (16, 64, 2, 40, 2), (8, 64, 3, 40, 3),
                                                 (4, 64, 5, 40, 5), (2, 64, 9, 40, 9), (1, 64, 17, 40, 17),
                                                 (3, 32, 6, 17, 6), (16, 128, 5, 40, 1), (24, 80, 4, None, 1),
                                                 (1, 128, 40, 33, 1)])
def test_hidden_values_of_grouped_heads(G, hd, nq, window, most, what):
    """One key at a time is not finite: the newest ones, which only the last
    queries see, and the oldest within a window, which only the first ones see.
    With many heads on one key head a block of rows is a single query of the
    sequence; ``max_seqlen_q`` (most) is no bound."""
    dtype, Hkv, nk = torch.bfloat16, 2, 150
    g = torch.Generator(device="cuda").manual_seed(G)
    q = torch.randn(nq, G * Hkv, hd, device="cuda", generator=g).to(dtype)
    k, v = (torch.randn(nk, Hkv, hd, device="cuda", generator=g).to(dtype) for _ in range(2))
    cu_q, cu_k = cum([nq]), cum([nk])
    ref, mag, _ = packed_attention_ref(q, k, v, cu_q, cu_k, window=window)
    lim = bound(ref, mag, dtype, nk, 6.0)
    at = torch.arange(nq) + nk - nq
    places = {nk - 1, nk - nq // 2} | ({nk - nq - window + 1, nk - window - 1} if window else set())
    for j in places:
        seen = (at >= j) & ((at - j < window) if window else True)
        assert 0 < int(seen.sum()) < nq
        kj, vj = k.clone(), v.clone()
        kj[j], vj[j] = what, what
        for kk, vv in ((k, vj), (kj, vj), (kj, v)):
            out = O.packed_attention(q, kk, vv, cu_q, cu_k, max_seqlen_q=most, window=window).double().cpu()
            assert bool(((out - ref).abs() <= lim)[~seen].all()), j
            assert kk is kj or not bool(torch.isfinite(out[seen]).any()), j


@pytest.mark.parametrize("G,hd", [(1, 64), (3, 128), (8, 64)])
@pytest.mark.parametrize("nq,nk,window", [(700, 700, 100), (700, 1200, 33), (700, 732, None), (333, 5000, 900)])
def test_many_queries_in_the_form_for_few(nq, nk, window, G, hd):
    """max_seqlen_q far too small: blocks whose windows begin and end anywhere
    within the pieces that their keys are cut into."""
    dtype = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(nk)
    q = torch.randn(nq, G, hd, device="cuda", generator=g).to(dtype)
    k, v = (torch.randn(nk, 1, hd, device="cuda", generator=g).to(dtype) for _ in range(2))
    cu_q, cu_k = cum([nq]), cum([nk])
    check(O.packed_attention(q, k, v, cu_q, cu_k, max_seqlen_q=1, window=window), q, k, v, cu_q, cu_k, window=window)


@pytest.mark.parametrize("nq,nk", [(1, 300), (200, 300)])
def test_layouts(nq, nk):
    """Head-major tensors, odd strides (copied), a shared head of stride zero, a given output with gaps."""
    H, hd, dtype = 4, 64, torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(9)
    mk = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    cu_q, cu_k = cum([nq]), cum([nk])
    q = mk(H, nq, hd).transpose(0, 1)
    k = mk(H, nk, hd).transpose(0, 1)
    v = mk(nk, H, hd + 1)[..., 1:]          # rows not 16-byte aligned
    out = torch.full((nq, H + 1, hd), 7.0, device="cuda", dtype=dtype)
    got = O.packed_attention(q, k, v, cu_q, cu_k, max_seqlen_q=nq, out=out[:, :H])
    assert got.data_ptr() == out.data_ptr()
    check(got, q, k, v, cu_q, cu_k)
    assert bool((out[:, H] == 7.0).all())
    k1 = mk(nk, 1, hd).expand(nk, H, hd)
    check(O.packed_attention(q, k1, v, cu_q, cu_k, max_seqlen_q=nq), q, k1, v, cu_q, cu_k)


@pytest.mark.parametrize("H,Hkv,hd", [(3, 3, 128), (8, 2, 64), (6, 1, 96)])
@pytest.mark.parametrize("nq,nk,window",
                         [(9000, 9000, None), (7000, 7000, 300), (900, 20000, None), (260, 40000, None)])
def test_long_sequences(H, Hkv, hd, nq, nk, window):
    """Many items a CTA, and items cut between CTAs: rows spread over the
    sequence against the reference."""
    dtype = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(nq)
    mk = lambda n, h: torch.randn(n, h, hd, device="cuda", generator=g).to(dtype)  # noqa: E731
    q, k, v = mk(nq + 5, H), mk(nk + 7, Hkv), mk(nk + 7, Hkv)
    cu_q, cu_k = cum([5, nq]), cum([7, nk])
    out = O.packed_attention(q, k, v, cu_q, cu_k, max_seqlen_q=nq, window=window)
    assert bool(torch.isfinite(out).all())
    for i in [0, 1, 127, 128, nq // 3, nq // 2, nq - 200, nq - 130, nq - 2, nq - 1]:
        end = i + nk - nq + 1  # the row as a sequence of one query and the keys before it
        one = torch.tensor([0, 1]), torch.tensor([0, end])
        ref, mag, _ = packed_attention_ref(q[5 + i:6 + i], k[7:7 + end], v[7:7 + end], *one, window=window)
        lim = bound(ref, mag, dtype, end, 6.0)
        assert bool(((out[5 + i].double().cpu() - ref[0]).abs() <= lim[0]).all()), i
    assert O.workspace_status() == 0


@pytest.mark.parametrize("nq", [1, 150])
def test_rows_outside_the_sequences_are_left_alone(nq):
    H, hd = 2, 64
    q, k, v = (torch.randn(nq + 40, H, hd, device="cuda").to(torch.bfloat16) for _ in range(3))
    cu = torch.tensor([20, 20 + nq], device="cuda", dtype=torch.int32)
    out = torch.full_like(q, 3.0)
    O.packed_attention(q, k, v, cu, max_seqlen_q=nq, out=out)
    owned = check(out, q, k, v, cu, cu)
    assert bool((out[~owned.cuda()] == 3.0).all())


@pytest.mark.parametrize("nq", [1, 300])
def test_large_scores_and_scale(nq):
    """Scores of several hundred: the running maximum has to carry them; a
    scale of its own."""
    H, hd, nk, dtype = 2, 64, 700, torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randn(nq, H, hd, device="cuda", generator=g)
    k = torch.randn(nk, H, hd, device="cuda", generator=g)
    k = k + q[-1] * torch.linspace(-1, 1, nk, device="cuda")[:, None, None]  # a maximum that rises along the keys
    q, k = (q * 4).to(dtype), (k * 2).to(dtype)
    v = torch.randn(nk, H, hd, device="cuda", generator=g).to(dtype)
    cu_q, cu_k = cum([nq]), cum([nk])
    out = O.packed_attention(q, k, v, cu_q, cu_k, max_seqlen_q=nq, scale=0.25)
    check(out, q, k, v, cu_q, cu_k, scale=0.25)


@pytest.mark.parametrize("H,Hkv,hd,nq", [(8, 8, 64, 1), (4, 4, 32, 3), (6, 3, 64, 2), (8, 2, 128, 1)])
def test_long_caches_of_a_batch(H, Hkv, hd, nq):
    """A line of keys long enough that each item takes two key heads (where
    their number is even and a head has up to 64 channels), cut between CTAs."""
    n, slots = 24, 20000
    g = torch.Generator(device="cuda").manual_seed(H)
    lens = [slots - (i * 997) % 9000 for i in range(n)]
    q = torch.randn(n * nq, H, hd, device="cuda", generator=g).to(torch.bfloat16)
    k, v = (torch.randn(n * slots, Hkv, hd, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    kv = torch.tensor(lens, device="cuda", dtype=torch.int32)
    cu_q, cu_k = cum([nq] * n), cum([slots] * n)
    out = O.packed_attention(q, k, v, cu_q, cu_k, max_seqlen_q=nq, kv_lengths=kv)
    for b in (0, 1, 11, n - 1):
        qs = slice(b * nq, (b + 1) * nq)
        ks = slice(b * slots, b * slots + lens[b])
        check(out[qs], q[qs], k[ks], v[ks], torch.tensor([0, nq]), torch.tensor([0, lens[b]]))


def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes and 2^31 elements, read at its end."""
    H, hd, slots, n = 4, 128, 1 << 20, 5
    k, v = (torch.empty(n * slots, H, hd, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    L0, tail = 700, (n - 1) * slots
    for t in (k, v):
        t[tail:tail + L0] = torch.randn(L0, H, hd, device="cuda").to(torch.bfloat16)
    kv = torch.tensor([0] * (n - 1) + [L0], device="cuda", dtype=torch.int32)
    for nq in (1, 200):
        q = torch.randn(nq, H, hd, device="cuda").to(torch.bfloat16)
        cu_q, cu_k = cum([0] * (n - 1) + [nq]), cum([slots] * n)
        out = O.packed_attention(q, k, v, cu_q, cu_k, max_seqlen_q=nq, kv_lengths=kv)
        small = torch.tensor([0, L0], dtype=torch.int32)
        check(out, q, k[tail:tail + L0], v[tail:tail + L0], cum([nq]), small)


@pytest.mark.parametrize("n", [1, 1000])
def test_many_sequences(n):
    lens = [(i * 7) % 5 for i in range(n)]
    q, k, v, cu = packed(lens, 2, 1, 64, torch.bfloat16)
    if sum(lens) == 0:
        assert O.packed_attention(q, k, v, cu, max_seqlen_q=1).shape == q.shape
        return
    check(O.packed_attention(q, k, v, cu, max_seqlen_q=max(lens)), q, k, v, cu, cu)
    kv = torch.tensor([min(x, 2) for x in lens], device="cuda", dtype=torch.int32)
    check(O.packed_attention(q, k, v, cu, max_seqlen_q=max(lens), kv_lengths=kv), q, k, v, cu, cu, kv_lengths=kv)


@pytest.mark.parametrize("nq,nk", [(1, 3000), (260, 900)])
def test_repeats_streams_and_graphs(nq, nk):
    """Bitwise the same on repeated calls, on a side stream and replayed from a
    graph on new inputs (nothing is kept from one call for the next)."""
    H, hd = 4, 64
    mk = lambda t: torch.randn(t, H, hd, device="cuda").to(torch.bfloat16)  # noqa: E731
    cu_q, cu_k = cum([nq, nq]), cum([nk, nk // 2])
    q, k, v = mk(2 * nq), mk(nk + nk // 2), mk(nk + nk // 2)
    call = lambda o=None: O.packed_attention(q, k, v, cu_q, cu_k, max_seqlen_q=nq, out=o)  # noqa: E731
    first = call()
    assert all(torch.equal(first, call()) for _ in range(3))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
        out = torch.empty_like(first)
        call(out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call(out)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(first, other)
    for t in (q, k, v):
        t.copy_(torch.randn_like(t))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, call())
    check(out, q, k, v, cu_q, cu_k)
    assert O.workspace_status() == 0


def _waste(nbytes=1 << 28):
    """Fills memory that is free with a pattern that no counter has."""
    x = [torch.full((nbytes // 4,), 0x5a5a5a5a, dtype=torch.int32, device="cuda") for _ in range(4)]
    del x


def _pieces(hd):
    """A call of each kernel whose items are cut between CTAs: (call(out), out, check())."""
    r = []
    for nq, nk in ((1, 40000), (300, 9000)):
        H = 4
        q = torch.randn(nq, H, hd, device="cuda").to(torch.bfloat16)
        k, v = (torch.randn(nk, H, hd, device="cuda").to(torch.bfloat16) for _ in range(2))
        cu_q, cu_k = cum([nq]), cum([nk])
        out = torch.empty_like(q)

        def call(q=q, k=k, v=v, cu_q=cu_q, cu_k=cu_k, nq=nq, out=out):
            return O.packed_attention(q, k, v, cu_q, cu_k, max_seqlen_q=nq, out=out)
        r.append((call, out, call().clone()))
    return r


@pytest.mark.parametrize("side", [False, True])
def test_workspace_after_a_timeout(side):
    """What a call that gave up leaves, its status and counters that are not 0,
    is gone once the status has been read."""
    from orthossm_b200 import sdpc_kernel
    calls = _pieces(64)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream() if side else torch.cuda.current_stream()):
        for call, _, want in calls:
            assert torch.equal(call(), want)
        stream = torch.cuda.current_stream()
        words = sdpc_kernel._WS_ATTN[(stream.device, stream.cuda_stream)].view(torch.int32)
        words[64:64 + 2048] = 1  # the counters follow a header of 256 bytes
        words[2] = 3             # its status word
        stream.synchronize()
        assert O.workspace_status(clear=False) == 3 and O.workspace_status() == 3 and O.workspace_status() == 0
        for _ in range(2):
            for call, _, want in calls:
                assert torch.equal(call(), want)
        stream.synchronize()


def test_graphs_and_larger_heads_after_them():
    """Calls captured at 64 channels, replayed after calls at 128 and with the
    freed memory overwritten."""
    calls = _pieces(64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for call, _, _ in calls:
            call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for call, _, _ in calls:
            call()
    with torch.cuda.stream(side):
        large = _pieces(128)
        _waste()
    torch.cuda.synchronize()
    for _ in range(3):
        for _, out, _ in calls:
            out.zero_()
        graph.replay()
        for call, out, want in large:
            assert torch.equal(call(), want)
        torch.cuda.synchronize()
        for _, out, want in calls:
            assert torch.equal(out, want)
    assert O.workspace_status() == 0


def test_graphs_without_a_call_before():
    """Two graphs captured on a stream that has seen no call, the second one
    replayed first, and calls on that stream beside them."""
    calls = _pieces(64)
    side = torch.cuda.Stream()
    graphs = []
    for call, _, _ in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            call()
        graphs.append(g)
    _waste()
    for i in (1, 0, 1, 1, 0):
        call, out, want = calls[i]
        out.zero_()
        torch.cuda.synchronize()
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        with torch.cuda.stream(side):
            assert torch.equal(call(), want)
        torch.cuda.synchronize()
    del graphs
    assert O.workspace_status() == 0


def test_refusals():
    q = torch.zeros(4, 4, 64, device="cuda", dtype=torch.bfloat16)
    k = torch.zeros(4, 2, 64, device="cuda", dtype=torch.bfloat16)
    cu = cum([4])
    ok = dict(max_seqlen_q=4)
    f = O.packed_attention
    for bad in [lambda: f(q.float(), k.float(), k.float(), cu, **ok), lambda: f(q, k.half(), k, cu, **ok),
                lambda: f(q, k, k[:, :1], cu, **ok), lambda: f(q[:, :3], k, k, cu, **ok),
                lambda: f(q[..., :60], k[..., :60], k[..., :60], cu, **ok),
                lambda: f(q[0], k, k, cu, **ok), lambda: f(q, k, k, cu.long(), **ok),
                lambda: f(q, k, k, cu, cu[:1], **ok), lambda: f(q, k, k, cu, window=0, **ok),
                lambda: f(q, k, k, cu, scale=-1.0, **ok), lambda: f(q, k, k, cu, scale=float("inf"), **ok),
                lambda: f(q, k, k, cu, kv_lengths=cu, **ok), lambda: f(q, k, k, cu, out=q[:2], **ok),
                lambda: f(q, k, k, cu[:1], **ok),
                lambda: f(torch.zeros(4, 4, 136, device="cuda", dtype=torch.bfloat16),
                          torch.zeros(4, 4, 136, device="cuda", dtype=torch.bfloat16),
                          torch.zeros(4, 4, 136, device="cuda", dtype=torch.bfloat16), cu, **ok)]:
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="CUDA"):
        f(q.cpu(), k, k, cu, **ok)
    with pytest.raises(NotImplementedError):
        f(q.requires_grad_(), k, k, cu, **ok)
    with torch.no_grad():
        f(q, k, k, cu, **ok)


def test_forward_mode_is_refused():
    """A tangent of q, k or v must not be dropped in silence."""
    q, k, v = (torch.randn(4, 2, 64, device="cuda").to(torch.bfloat16) for _ in range(3))
    cu = cum([4])
    want = O.packed_attention(q, k, v, cu, max_seqlen_q=4)
    with torch.autograd.forward_ad.dual_level():
        for i in range(3):
            x = [q, k, v]
            x[i] = torch.autograd.forward_ad.make_dual(x[i], torch.ones_like(x[i]))
            with pytest.raises(NotImplementedError), torch.no_grad():
                O.packed_attention(*x, cu, max_seqlen_q=4)
        assert torch.equal(O.packed_attention(q, k, v, cu, max_seqlen_q=4), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("G,hd,nq", [(1, 64, 1), (4, 128, 1), (8, 64, 2), (2, 80, 3)])
def test_weights_of_few_queries_are_not_rounded(G, hd, nq, dtype):
    """Values of one size and either sign, so that outputs are differences of
    weights: the form for few queries keeps these to fp32.  Bound: the output's
    rounding, u |o|; the weights' two 16-bit parts, u^2, and their fp32 errors:
    scores off by hd 2^-24 sum |q k| scale (below 2^-14 here), the rest by a
    few 2^-22.  Weights rounded to the type would not pass."""
    n, Hkv = 150, 2
    g = torch.Generator(device="cuda").manual_seed(hd)
    lk = [nq + i % 9 for i in range(n)]
    q = torch.randn(n * nq, G * Hkv, hd, device="cuda", generator=g).to(dtype)
    k = torch.randn(sum(lk), Hkv, hd, device="cuda", generator=g).to(dtype)
    v = torch.randint(0, 2, (sum(lk), Hkv, hd), device="cuda", generator=g).mul(2).sub(1).to(dtype)
    cu_q, cu_k = cum([nq] * n), cum(lk)
    out = O.packed_attention(q, k, v, cu_q, cu_k, max_seqlen_q=nq).double().cpu()
    ref, mag, _ = packed_attention_ref(q, k, v, cu_q, cu_k)
    u = 2.0 ** (-8 if dtype == torch.bfloat16 else -11)
    lim = u * ref.abs() + (2.0 ** -13 + u * u) * mag + 1e-6
    assert bool(((out - ref).abs() <= lim).all())
    # a pair of weights p, 1 - p in the type: their difference off by more than the bound
    p = torch.rand(4000, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    d, r = p.to(dtype).double() - (1 - p).to(dtype).double(), 2 * p - 1
    assert bool(((d - r).abs() > u * r.abs() + 2.0 ** -13 + u * u + 1e-6).any())
