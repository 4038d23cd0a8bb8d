"""Sigmoid attention of one sequence in 64 bits, with bounds on what kernels
that work as these do may be off by, element by element.

The bounds follow the arithmetic.  u is half a step of the I/O dtype
(finfo.eps / 2, and `tiny` for subnormal results); e = 2^-24 is fp32's.
  * S = q·k·scale + add in fp32 from exact products: off by (D + 8) e A with
    A = |q|·|k| |scale| + |add|, so P = sigmoid(S) is off by that share of P
    (dP/dS = P(1 - P) <= P), and by 2^-21 of P for the hardware's exp2 and
    reciprocal; rounded to the I/O dtype before its product: u P + tiny.
  * a sum of n terms in fp32: n e of the sum of their sizes; the result is
    rounded once: u of it + tiny.
  * dS = P (1 - P) dP likewise, with dP off by (D + 8) e |dO|·|V|.
A `shared` head's dK and dV are sums over its query heads: so are the bounds.
"""

import math

import torch

E32 = 2.0 ** -24


def half_step(dtype):
    f = torch.finfo(dtype)
    return f.eps / 2, f.tiny * f.eps / 2


def one_head(q, k, v, do, add, dtype, causal_offset=None, scale=None):
    """(values, bounds) of O, dQ, dK, dV for one query head ([n, D] tensors of
    `dtype`; add: float or [keys]); query i sees keys <= i + causal_offset."""
    D, n, m = q.shape[1], q.shape[0], k.shape[0]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    u, tiny = half_step(dtype)
    q, k, v = q.double(), k.double(), v.double()
    if isinstance(add, torch.Tensor):
        add = add.double()
    else:
        add = torch.full((m,), add, dtype=torch.float64, device=q.device)
    seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
    if causal_offset is not None:
        i = torch.arange(n, device=q.device)[:, None] + causal_offset
        seen = torch.arange(m, device=q.device)[None] <= i
    finite = torch.where(torch.isfinite(add), add, 0.0)
    s = q @ k.t() * scale + add
    p = torch.where(seen, torch.sigmoid(s), 0.0)
    # Share of P that its fp32 value may be off by.
    share = (D + 8) * E32 * (q.abs() @ k.abs().t() * abs(scale) + finite.abs()) + 2.0 ** -21
    ep = torch.where(seen, p * (share + u) + tiny, 0.0)
    o = p @ v
    eo = ep @ v.abs() + (m + 2) * E32 * (p @ v.abs())
    out = {"o": (o, eo + u * (o.abs() + eo) + tiny)}
    if do is None:
        return out
    do = do.double()
    dp, adp = do @ v.t(), do.abs() @ v.abs().t()
    ds = p * (1.0 - p) * dp
    # fma(-P, P dP, P dP): off by a few e of P |dP|; P's own error moves P (1 - P)
    # by at most its share of P, dP's by (D + 8) e |dO|·|V|.
    eds = torch.where(seen, p * adp * ((D + 16) * E32 + share) + u * ds.abs() + tiny, 0.0)
    dq = ds @ k * scale
    edq = abs(scale) * (eds @ k.abs() + (m + 2) * E32 * (ds.abs() @ k.abs()))
    dk = ds.t() @ q * scale
    edk = abs(scale) * (eds.t() @ q.abs() + (n + 2) * E32 * (ds.abs().t() @ q.abs()))
    dv = p.t() @ do
    edv = ep.t() @ do.abs() + (n + 2) * E32 * (p.t() @ do.abs())
    out.update(dq=(dq, edq + u * (dq.abs() + edq) + tiny), dk=(dk, edk), dv=(dv, edv))
    return out


def packed(q, k, v, do, cu_q, cu_k, causal=False, mod=None, bias=None, scale=None):
    """{name: (value, bound)} of packed sequences with grouped heads, [rows,
    heads, D] each; rows outside every sequence are zeros with bound 0."""
    H, G, dtype = q.shape[1], q.shape[1] // k.shape[1], q.dtype
    u, tiny = half_step(dtype)
    names = {"o": q} if do is None else {"o": q, "dq": q, "dk": k, "dv": k}
    out = {x: [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for _ in range(2)] for x, t in names.items()}
    for b in range(len(cu_q) - 1):
        qa, ka = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        n = cu_k[b + 1] - cu_k[b]
        if n <= 0 or cu_q[b + 1] <= cu_q[b]:
            continue
        add = -math.log(n) if bias is None else bias
        if mod is not None:
            add = add + mod[ka].double()
        for h in range(H):
            one = one_head(q[qa, h], k[ka, h // G], v[ka, h // G], None if do is None else do[qa, h], add, dtype,
                           0 if causal else None, scale)
            for x, (val, err) in one.items():
                at = (qa, h) if x in ("o", "dq") else (ka, h // G)
                out[x][0][at] += val
                out[x][1][at] += err
    for x in ("dk", "dv"):
        if x in out:  # rounded once, after the sum over the query heads
            val, err = out[x]
            out[x][1] = torch.where(err > 0, err + u * (val.abs() + err) + tiny, err)
    return {x: tuple(t) for x, t in out.items()}


def assert_within(got, want, name=""):
    val, err = want
    got = got.detach().double().to(val.device)
    assert got.shape == val.shape, (name, got.shape, val.shape)
    assert torch.isfinite(got).all(), f"{name}: values that are not finite"
    over = (got - val).abs() - err
    if over.numel():
        worst = over.argmax()
        assert over.max() <= 0, (f"{name}: off by {(got - val).abs().flatten()[worst]:.3e}, bound "
                                 f"{err.flatten()[worst]:.3e}, value {val.flatten()[worst]:.3e}, "
                                 f"{int((over > 0).sum())} of {over.numel()} over")
