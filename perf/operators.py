"""Cases of the serving operators: attention over packed prompts and over a cache, and the choice of the next token.

``run`` computes an operator in its plain form (elementary torch operations in
fp32) or, with ``own`` set, through this package's public functions.  A case
is a dict of plain values; ``lengths`` turns it into the token counts of its
sequences, so that the work of a case is known without its inputs.
"""
import math

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ----------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------

def _attend(name, seqs, keys, new, heads, kv_heads, head_dim, dtype, window=0, ragged=True):
    """seqs sequences of at most `keys` keys.  new = 0: a whole prompt (as many queries as keys, packed);
    new > 0: the last `new` tokens of each sequence against a cache of `keys` slots a sequence."""
    return {"name": name, "op": "attend", "seqs": seqs, "keys": keys, "new": new, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "window": window, "ragged": ragged}


def _sample(name, rows, vocab, dtype, temperature, top_k=0, top_p=1.0, min_p=0.0, per_row=False):
    """top_k = 0, top_p = 1, min_p = 0: that filter is off.  per_row: each row has settings of its own."""
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": temperature,
            "top_k": top_k, "top_p": top_p, "min_p": min_p, "per_row": per_row}


def listed():
    return [
        # one user's next token early in a reply, at the language model's heads: a call whose latency counts
        _attend("token_one_user", 1, 385, 1, 8, 8, 64, "bf16"),
        # the language model's decode step for a batch of long streams: 512 tokens of each are seen
        _attend("token_window", 32, 16384, 1, 8, 8, 64, "bf16", window=512),
        # a serving batch in decode, grouped heads, every stream at a length of its own
        _attend("token_grouped", 64, 8192, 1, 32, 8, 128, "bf16"),
        # one stream at the million-token length, a few rows only: the keys have to be split over the GPU
        _attend("token_million", 1, 1048576, 1, 8, 8, 64, "bf16"),
        # a few short prompts together, at the engine's 4 heads
        _attend("prompt_short", 4, 300, 0, 4, 4, 64, "bf16"),
        # the language model's prompt pass: window of 512 over long prompts
        _attend("prompt_window", 2, 16384, 0, 8, 8, 64, "bf16", window=512),
        # packed prompts of different lengths, grouped heads
        _attend("prompt_grouped", 6, 4096, 0, 32, 8, 128, "bf16"),
        # one long document
        _attend("prompt_long", 1, 16384, 0, 16, 16, 128, "fp16", ragged=False),
        # a prompt that comes in pieces: the next 500 tokens against what the cache holds
        _attend("prompt_piece", 3, 16384, 500, 16, 4, 128, "bf16"),
        # one user's next token out of the language model's vocabulary
        _sample("sample_one_user", 1, 32000, "bf16", 0.8, top_k=50, top_p=0.95),
        # a batch drawn from the whole distribution, fp32 logits
        _sample("sample_open", 256, 32000, "fp32", 1.0),
        # a batch at the engine's vocabulary, every user with settings of their own
        _sample("sample_nucleus", 128, 131072, "bf16", 0.9, top_p=0.92, min_p=0.01, per_row=True),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["token", "prompt", "piece", "sample", "sample"])
    if kind == "sample":
        rows, vocab = _log_between(rng, 1, 256), _log_between(rng, 1000, 131072)
        top_k, top_p, min_p = 0, 1.0, 0.0
        if rng.random() < 0.5:
            top_k = _log_between(rng, 1, 200)
        if rng.random() < 0.5:
            top_p = round(rng.uniform(0.3, 0.99), 3)
        if rng.random() < 0.3:
            min_p = round(rng.uniform(0.01, 0.2), 3)
        c = _sample("", rows, vocab, rng.choice(["bf16", "fp16", "fp32"]), round(rng.uniform(0.5, 1.5), 2), top_k,
                    top_p, min_p, rng.random() < 0.5)
    else:
        head_dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
        window = rng.choice([0, 0, 0, 512, _log_between(rng, 16, 4096)])
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        if kind == "token":
            new = rng.choice([1, 1, 1, 2, 5])
            seqs = _log_between(rng, 1, 128)
            keys = min(_log_between(rng, 64, 200000), (1 << 29) // (seqs * kv_heads * head_dim))
        else:
            new = 0 if kind == "prompt" else _log_between(rng, 8, 1000)
            seqs = _log_between(rng, 1, 16)
            keys = _log_between(rng, 100, 8192 if kind == "prompt" else 32768)
            while seqs * heads * keys * (new or keys) > 1 << 31:
                keys = keys * 2 // 3
        c = _attend("", seqs, keys, min(new, keys), heads, kv_heads, head_dim, dtype, window, rng.random() < 0.75)
    del c["name"]
    return c


def lengths(case):
    """(queries, keys) of each sequence."""
    n, most = case["seqs"], case["keys"]
    keys = [most] + [most if not case["ragged"] else max(1, int(most * (0.1 + 0.9 * ((i * 0.6180339887) % 1.0))))
                     for i in range(1, n)]
    return [min(case["new"], k) if case["new"] else k for k in keys], keys


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        # every logit is read; the noise of all candidates only where no filter leaves a few of them
        open_ = not case["top_k"] and case["top_p"] >= 1.0 and not case["min_p"]
        return {"bytes": n * (size + (4 if open_ else 0)) + 8 * case["rows"], "flops": 2 * n}
    H, Hkv, hd, w = case["heads"], case["kv_heads"], case["head_dim"], case["window"]
    pairs = rows = read = 0
    for q, k in zip(*lengths(case)):
        rows += q
        read += min(k, w + q - 1) if w else k
        if not w:
            pairs += q * (k - q) + q * (q + 1) // 2
        else:  # query i sees min(w, k - q + i + 1) keys
            full = max(0, min(q, k - w + 1 if k >= w else 0))  # queries that see w keys
            part = q - full
            first = k - q + 1
            pairs += full * w + part * first + part * (part - 1) // 2
    return {"bytes": size * hd * (2 * rows * H + 2 * read * Hkv), "flops": 4 * hd * H * pairs}


# ----------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DTYPE[case["dtype"]]
    if case["op"] == "sample":
        B, V = case["rows"], case["vocab"]
        logits = torch.randn(B, V, device="cuda", generator=g).mul_(2.5)
        # a few likely continuations above the rest, as a trained model's logits have
        top = torch.randint(0, V, (B, 24), device="cuda", generator=g)
        logits.scatter_add_(1, top, torch.rand(B, 24, device="cuda", generator=g).mul_(9.0))
        noise = torch.empty(B, V, device="cuda").exponential_(generator=g)
        s = {"op": "sample", "logits": logits.to(dt), "noise": noise, "temperature": case["temperature"],
             "top_k": case["top_k"], "top_p": case["top_p"], "min_p": case["min_p"]}
        if case["per_row"]:
            u = torch.rand(3, B, device="cuda", generator=g)
            s["temperature"] = case["temperature"] * (0.75 + 0.5 * u[0])
            if case["top_k"]:
                s["top_k"] = (1 + u[1] * case["top_k"]).to(torch.int32)
            if case["top_p"] < 1.0:
                s["top_p"] = case["top_p"] - 0.2 * u[1]
            if case["min_p"]:
                s["min_p"] = case["min_p"] * u[2]
        return s
    H, Hkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    lq, lk = lengths(case)
    cum = lambda v: torch.tensor([0] + v, device="cuda").cumsum(0).to(torch.int32)  # noqa: E731
    s = {"op": "attend", "cu_q": cum(lq), "max_q": max(lq), "max_k": max(lk), "window": case["window"] or None,
         "lengths": None}
    if case["new"]:  # a cache of `keys` slots a sequence, filled up to the sequence's length
        n, cap = case["seqs"], case["keys"]
        s["q"] = torch.randn(sum(lq), H, hd, device="cuda", generator=g).to(dt)
        s["k"], s["v"] = (torch.randn(n * cap, Hkv, hd, device="cuda", generator=g).to(dt) for _ in range(2))
        s["cu_k"] = torch.arange(n + 1, device="cuda", dtype=torch.int32) * cap
        s["lengths"] = torch.tensor(lk, device="cuda", dtype=torch.int32)
    else:  # q, k, v as one projection leaves them
        qkv = torch.randn(sum(lq), H + 2 * Hkv, hd, device="cuda", generator=g).to(dt)
        s["q"], s["k"], s["v"] = qkv.split([H, Hkv, Hkv], 1)
        s["cu_k"] = s["cu_q"]
    return s


# ----------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------

def run(state):
    if state["op"] == "sample":
        return _own_sample(state) if own else _plain_sample(**{k: v for k, v in state.items() if k != "op"})
    return _own_attend(state) if own else _plain_attend(**{k: v for k, v in state.items() if k != "op"})


def _own_attend(s):
    import orthossm_b200 as O
    return O.packed_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], max_seqlen_q=s["max_q"],
                              kv_lengths=s["lengths"], window=s["window"])


def _own_sample(s):
    import orthossm_b200 as O
    return O.sample_tokens(s["logits"], s["noise"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                           min_p=s["min_p"])


def _plain_attend(q, k, v, cu_q, cu_k, max_q, max_k, window, lengths):
    """Query i of a sequence with Lq queries and Lk keys stands at position i + Lk - Lq and sees the keys at or
    before it, the last `window` of them if there is a window: softmax(q.k / sqrt(hd)) over these, times v;
    zeros where it sees none."""
    Tq, H, hd = q.shape
    Tk, Hkv = k.shape[0], k.shape[1]
    dev = q.device
    lq = cu_q[1:] - cu_q[:-1]
    lk = cu_k[1:] - cu_k[:-1] if lengths is None else lengths
    B = lq.shape[0]
    iq, ik = (torch.arange(n, device=dev, dtype=torch.int32) for n in (max_q, max_k))
    rows = (cu_q[:-1, None] + iq).clamp_(max=Tq - 1).long()
    keys = (cu_k[:-1, None] + ik).clamp_(max=Tk - 1).long()
    qp = q[rows].float().view(B, max_q, Hkv, H // Hkv, hd).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, hd)
    kp = k[keys].float().permute(0, 2, 3, 1)
    s = (qp @ kp).mul_(1.0 / math.sqrt(hd)).view(B, Hkv, H // Hkv, max_q, max_k)
    del kp
    at = (iq + (lk - lq)[:, None])[:, :, None]
    hidden = (ik > at) | (ik >= lk[:, None, None])
    if window is not None:
        hidden |= ik <= at - window
    s.masked_fill_(hidden[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = s.sub_(m.masked_fill_(m == float("-inf"), 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(total.masked_fill_(total == 0, 1.0))
    o = p.view(B, Hkv, -1, max_k) @ v[keys].float().permute(0, 2, 1, 3)
    o = o.view(B, Hkv, H // Hkv, max_q, hd).permute(0, 3, 1, 2, 4).reshape(B, max_q, H, hd)
    t = torch.arange(Tq, device=dev, dtype=torch.int32)
    b = torch.searchsorted(cu_q[1:], t, right=True)
    return o[b, (t - cu_q[b]).long()].to(q.dtype)


def _plain_sample(logits, noise, temperature, top_k, top_p, min_p):
    """Of the candidates, ordered by logit and at equal logits by index, the first top_k stay; of these the shortest
    prefix whose probability (softmax(logits / temperature) over the first top_k) reaches top_p; of these the ones
    at least min_p times as likely as the first.  The token is the candidate with the largest
    logit / temperature - log(noise), noise from the standard exponential distribution: candidate i wins with
    the probability that the softmax over the candidates gives it."""
    col = lambda x: x[:, None] if isinstance(x, torch.Tensor) else x  # noqa: E731
    l = logits.float()
    inv = 1.0 / col(temperature)
    order = None
    if isinstance(top_k, torch.Tensor) or isinstance(top_p, torch.Tensor) or isinstance(min_p, torch.Tensor) \
            or top_k or top_p < 1.0 or min_p:
        l, order = torch.sort(l, dim=-1, descending=True, stable=True)
        noise = noise.gather(1, order)
        w = ((l - l[:, :1]) * inv).exp()
        keep = torch.ones_like(l, dtype=torch.bool)
        if isinstance(top_k, torch.Tensor) or top_k:
            keep &= torch.arange(l.shape[1], device=l.device) < col(top_k)
        kept = w * keep
        if isinstance(top_p, torch.Tensor) or top_p < 1.0:
            keep &= kept.cumsum(-1) - kept < col(top_p) * kept.sum(-1, keepdim=True)
            keep[:, 0] = True
        if isinstance(min_p, torch.Tensor) or min_p:
            keep &= w >= col(min_p)
    score = l * inv - noise.log()
    if order is None:
        return score.argmax(-1)
    score.masked_fill_(~keep, float("-inf"))
    # of equal scores the lowest index wins
    best = score == score.amax(-1, keepdim=True)
    return order.masked_fill(~best, l.shape[1]).amin(-1)


def exact(case, seed):
    """The attention of each sequence in float64, a block of queries at a time; tokens are whole numbers and have
    no such value."""
    if case["op"] == "sample":
        return None
    s = prepare(case, seed)
    q, k, v = s["q"], s["k"], s["v"]
    H, Hkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    lq, lk = lengths(case)
    out, q0 = [], 0
    for b in range(case["seqs"]):
        k0 = b * case["keys"] if case["new"] else q0
        kb = k[k0:k0 + lk[b]].double().permute(1, 2, 0)
        vb = v[k0:k0 + lk[b]].double().transpose(0, 1)
        j = torch.arange(lk[b], device=q.device)
        for i0 in range(0, lq[b], 512):
            i1 = min(i0 + 512, lq[b])
            qb = q[q0 + i0:q0 + i1].double().view(i1 - i0, Hkv, H // Hkv, hd)
            x = torch.einsum("ihgd,hdj->hgij", qb, kb) / math.sqrt(hd)
            at = (torch.arange(i0, i1, device=q.device) + lk[b] - lq[b])[:, None]
            seen = j <= at
            if case["window"]:
                seen &= j > at - case["window"]
            x = torch.where(seen, x, torch.full((), float("-inf"), dtype=x.dtype, device=x.device))
            o = torch.einsum("hgij,hjd->ihgd", torch.softmax(x, -1), vb)
            out.append(o.reshape(i1 - i0, H, hd))
        q0 += lq[b]
    return torch.cat(out)
