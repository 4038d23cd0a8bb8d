"""Sigmoid attention with a learned bias by relative position in 64 bits, with
bounds, on top of reference64 (whose arithmetic holds here: the score's additive
term is then a matrix).

The table's gradient is a sum of dS as the kernels hold it in fp32, before any
rounding to the I/O dtype: each dS is off by reference64's share of it without that
rounding, the sum of a bucket by (longest chain of additions) e of the sum of their
sizes, and it is rounded once to the table's dtype.
"""

import math

import torch

from reference64 import E32, half_step, one_head


def line_of(table, buckets, h, d):
    """table[buckets[R + d], h] in 64 bits, 0 where the bucket is none of the table's;
    and the buckets (-1: none)."""
    R = buckets.numel() // 2
    u = buckets.long()[d.clamp(-R, R) + R]
    ok = (u >= 0) & (u < table.shape[0])
    u = torch.where(ok, u, -1)
    return torch.where(ok, table.double()[u.clamp(min=0), h], 0.0), u


def grad_of_scores(q, k, v, do, add, causal):
    """dS of one head in 64 bits and what an fp32 one may be off by."""
    D, n, m = q.shape[1], q.shape[0], k.shape[0]
    q, k, v, do = (t.double() for t in (q, k, v, do))
    scale = 1.0 / math.sqrt(D)
    p = torch.sigmoid(q @ k.t() * scale + add)
    if causal:
        p = torch.where(torch.arange(m, device=q.device)[None] <= torch.arange(n, device=q.device)[:, None], p, 0.0)
    finite = torch.where(torch.isfinite(add), add, 0.0)
    share = (D + 8) * E32 * (q.abs() @ k.abs().t() * scale + finite.abs()) + 2.0 ** -21
    dp, adp = do @ v.t(), do.abs() @ v.abs().t()
    return p * (1.0 - p) * dp, p * adp * ((D + 16) * E32 + share)


def packed_rel(q, k, v, do, table, buckets, cu_q, cu_k, causal, bias=None):
    """{name: (value, bound)} of O, dQ, dK, dV and dtable.  bias: of all sequences, or
    a list of theirs."""
    H, G, dtype, dev = q.shape[1], q.shape[1] // k.shape[1], q.dtype, q.device
    u, tiny = half_step(dtype)
    names = {"o": q} if do is None else {"o": q, "dq": q, "dk": k, "dv": k, "dtable": table}
    out = {x: [torch.zeros(t.shape, dtype=torch.float64, device=dev) for _ in range(2)] for x, t in names.items()}
    size = torch.zeros(table.shape, dtype=torch.float64, device=dev)
    longest = 0
    for b in range(len(cu_q) - 1):
        n, m = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        if n <= 0 or m <= 0:
            continue
        longest = max(longest, n + m)
        qa, ka = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        d = torch.arange(m, device=dev)[None] - torch.arange(n, device=dev)[:, None]
        for h in range(H):
            line, bucket = line_of(table, buckets, h, d)
            add = line + (-math.log(m) if bias is None else bias[b] if isinstance(bias, list) else bias)
            heads = q[qa, h], k[ka, h // G], v[ka, h // G], None if do is None else do[qa, h]
            for x, (val, err) in one_head(*heads, add, dtype, 0 if causal else None).items():
                at = (qa, h) if x in ("o", "dq") else (ka, h // G)
                out[x][0][at] += val
                out[x][1][at] += err
            if do is None:
                continue
            ds, eds = grad_of_scores(*heads, add, causal)
            at = torch.where(bucket >= 0, bucket, table.shape[0]).flatten()
            for to, what in ((out["dtable"][0], ds), (out["dtable"][1], eds), (size, ds.abs())):
                col = torch.zeros(table.shape[0] + 1, dtype=torch.float64, device=dev)
                to[:, h] += col.index_add_(0, at, what.flatten())[:-1]
    for x in ("dk", "dv"):
        if x in out:  # rounded once, after the sum over the query heads
            val, err = out[x]
            out[x][1] = torch.where(err > 0, err + u * (val.abs() + err) + tiny, err)
    if do is not None:
        ut, tt = half_step(table.dtype)
        val, err = out["dtable"]
        err = err + (longest + buckets.numel() + 200) * E32 * size
        out["dtable"][1] = torch.where(size > 0, err + ut * (val.abs() + err) + tt, 0.0)
    return {x: tuple(t) for x, t in out.items()}
