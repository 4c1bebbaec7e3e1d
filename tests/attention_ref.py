"""float64 restatement of packed_attention, one sequence, head and query at a
time, that looks at the seen keys alone; returns the outputs, the weighted sum
of |v| that the rounding bounds need, and which rows belong to a sequence."""
import torch


def packed_attention_ref(q, k, v, cu_q, cu_k, kv_lengths=None, window=None, scale=None):
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    Tq, H, hd = q.shape
    G = H // k.shape[1]
    scale = hd ** -0.5 if scale is None else scale
    out, mag = torch.zeros(Tq, H, hd, dtype=torch.float64), torch.zeros(Tq, H, hd, dtype=torch.float64)
    owned = torch.zeros(Tq, dtype=torch.bool)
    cu_q, cu_k = cu_q.tolist(), cu_k.tolist()
    for b in range(len(cu_q) - 1):
        nq, nk = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        if kv_lengths is not None:
            nk = min(nk, int(kv_lengths[b]))
        owned[cu_q[b]:cu_q[b + 1]] = True
        for i in range(nq):
            at = i + nk - nq
            lo = 0 if window is None else max(0, at - window + 1)
            if at < lo:
                continue
            kk, vv = k[cu_k[b] + lo:cu_k[b] + at + 1], v[cu_k[b] + lo:cu_k[b] + at + 1]
            kk, vv = kk.repeat_interleave(G, 1), vv.repeat_interleave(G, 1)
            p = torch.softmax(torch.einsum("hd,jhd->hj", q[cu_q[b] + i], kk) * scale, -1)
            out[cu_q[b] + i] = torch.einsum("hj,jhd->hd", p, vv)
            mag[cu_q[b] + i] = torch.einsum("hj,jhd->hd", p, vv.abs())
    return out, mag, owned


def bound(ref, mag, dtype, keys, vmax):
    """Elementwise error bound.  Roundings to the type (8 significant bits in
    bf16, 11 in fp16: to within u = 2^-8 and 2^-11 of the value): the
    output's, u |o|, and each weight's before the product with v, u sum p|v|.  fp32: the scores (sums of hd products, |s| up to a few
    tens) and the exponential move each weight by less than 2^-12 of itself.
    fp16 weights below 2^-14 of the largest are rounded to steps of 2^-24."""
    u = 2.0 ** (-8 if dtype == torch.bfloat16 else -11)
    sub = keys * 2.0 ** -25 * vmax if dtype == torch.float16 else 0.0
    return u * ref.abs() + (u * 1.01 + 2.0 ** -12) * mag + sub + 1e-6
