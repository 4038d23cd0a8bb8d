"""Performance cases of the operators that tell sigmoid attention where its tokens are:
`sigmoid_attention_varlen` and `sigmoid_attention_paged` with a learned bias by
buckets of the relative position, `rotary_embedding`, and
`paged_cache_write_rotary`.

A case is a dict of plain values:
  kind       "bias" | "paged" | "append" | "rotate"
  H, Hkv, D  query heads, key/value heads, head dim
  dtype      "float16" | "bfloat16" | "float32" (the learned table's too)
  lens       seed of the case's lengths (a case's work is fixed, so its
             lengths are; the values of the tensors follow `seed`)
  bias, paged: buckets learned values per head, for relative positions up to dist
             (two-sided: half of the buckets for keys after the query)
  bias:    B sequences of lo..T tokens packed back to back; train (forward and
           backward: returns O, dQ, dK, dV and the table's gradient; else O)
  paged:   B sequences with ctx_lo..ctx tokens before the call's own, of which
           the first `ones` bring one and the others new_lo..new; pages of ps
  append, rotate: the first `rot` columns of a head turn by angles of a table of
           P positions, in pairs of neighbours (pairs) or of halves
  append:  N new tokens of up to `run` in a row, into a cache of `slots` slots in
           pages of ps, `pad` of them without a slot
  rotate:  N packed tokens of sequences of up to `run`, forward and backward
"""

import functools
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
_SIZE = {"float16": 2, "bfloat16": 2, "float32": 4}
_BIAS = dict(kind="bias", B=1, T=128, lo=0, H=8, Hkv=8, D=64, dtype="bfloat16", causal=False, train=True, buckets=32,
             dist=128, lens=0)
_PAGED = dict(kind="paged", B=1, ctx_lo=0, ctx=1024, ones=0, new_lo=1, new=1, ps=16, H=8, Hkv=2, D=128,
              dtype="bfloat16", causal=True, buckets=32, dist=128, lens=0)
_APPEND = dict(kind="append", N=1, run=1, slots=1024, ps=16, pad=0, P=8192, H=32, Hkv=8, D=128, rot=128, pairs=False,
               dtype="bfloat16", lens=0)
_ROTATE = dict(kind="rotate", N=256, run=256, P=8192, H=16, Hkv=16, D=64, rot=64, pairs=False, dtype="bfloat16", lens=0)
_BASE = {"bias": _BIAS, "paged": _PAGED, "append": _APPEND, "rotate": _ROTATE}


def _case(name, kind, **kw):
    return dict(_BASE[kind], **kw, name=name)


def listed():
    return [
        # One short text through a small encoder, forward only: launches and host time.
        _case("bias-short", "bias", B=1, T=128, H=8, Hkv=8, D=64, dtype="float16", train=False),
        # An encoder's training step on texts of odd lengths packed back to back.
        _case("bias-train-encoder", "bias", B=16, T=1001, lo=101, H=12, Hkv=12, D=64, lens=3),
        # A decoder's training step on long documents, grouped heads.
        _case("bias-train-causal", "bias", B=3, T=4096, lo=1500, H=16, Hkv=4, D=128, causal=True, lens=5),
        # The same in fp32 with narrow heads, short sequences and a wide table.
        _case("bias-train-fp32", "bias", B=5, T=777, lo=1, H=8, Hkv=8, D=32, dtype="float32", buckets=64, dist=300,
              lens=6),
        # Decoding: one token each for 16 requests with ragged contexts.
        _case("bias-decode", "paged", B=16, ctx_lo=1024, ctx=8191, ones=16, H=32, Hkv=8, lens=4),
        # A chunk of a long prompt after most of it is in the cache.
        _case("bias-chunk", "paged", B=2, ctx_lo=5000, ctx=12000, new_lo=1024, new=1024, H=32, Hkv=8, lens=11),
        # A step that mixes running requests with prompt chunks, 64-wide heads.
        _case("bias-mixed", "paged", B=24, ctx_lo=300, ctx=4096, ones=20, new_lo=100, new=700, ps=32, H=12, Hkv=4,
              D=64, dtype="float16", lens=12),
        # One decoding step's queries, keys and values.
        _case("append-decode", "append", N=64, slots=65536, lens=8),
        # A prompt step's, with padding rows; half of a head turns, neighbours in pairs.
        _case("append-prompt", "append", N=16383, run=2048, slots=40960, ps=64, pad=77, H=16, Hkv=8, D=64, rot=32,
              pairs=True, dtype="float16", lens=9),
        # A training step's queries and keys, a few short texts.
        _case("rotate-short", "rotate", N=509, run=200, lens=10),
        # The same for long documents, grouped heads.
        _case("rotate-long", "rotate", N=16384, run=8192, H=32, Hkv=8, D=128, rot=128, lens=13),
    ]


def _log_int(r, lo, hi):
    return int(round(math.exp(r.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges: packed sequences of 1 to 4096 tokens,
    forward and training; 1 to 256 sequences of up to 65536 cached tokens with 1
    to 2048 new ones; 1 to 16384 tokens appended or rotated; every head dim and
    dtype, groups of 1 to 16, 4 to 256 buckets of distances up to 8 to 1024."""
    while True:
        kind = rng.choice(("bias", "bias", "bias", "paged", "paged", "paged", "append", "rotate"))
        c = dict(_BASE[kind], lens=rng.randrange(1 << 20))
        c["Hkv"] = rng.choice((1, 2, 3, 4, 8, 8, 12, 16))
        c["D"] = rng.choice((128, 128, 64, 64, 64, 32, 16))
        c["dtype"] = rng.choice(("bfloat16", "bfloat16", "bfloat16", "float16", "float16", "float32"))
        c["H"] = c["Hkv"] * rng.choice((1, 1, 1, 2, 3, 4, 8, 16))
        if c["H"] > 64:
            continue
        if kind in ("append", "rotate"):
            c.update(N=_log_int(rng, 1 if kind == "append" else 16, 16384), rot=c["D"] // rng.choice((1, 1, 2)),
                     pairs=rng.random() < 0.4, P=_log_int(rng, 256, 32768))
            c["run"] = min(_log_int(rng, 1, 4096), c["P"])
            if c["N"] * (c["H"] + c["Hkv"]) * c["D"] * _SIZE[c["dtype"]] > 16384 * 40 * 256:
                continue
            if kind == "rotate":
                return c
            c["ps"] = rng.choice((16, 32, 64, 128))
            c["pad"] = rng.choice((0, 0, rng.randint(0, c["N"])))
            c["slots"] = -(-int(c["N"] * rng.uniform(1.2, 4.0)) // c["ps"]) * c["ps"]
            if c["slots"] * c["Hkv"] * c["D"] * _SIZE[c["dtype"]] > 1 << 27:
                continue
            return c
        c["causal"] = rng.random() < 0.6
        c.update(buckets=2 * _log_int(rng, 2, 128), dist=_log_int(rng, 8, 1024))
        if c["dist"] < c["buckets"]:
            continue
        if kind == "bias":
            c.update(B=_log_int(rng, 1, 16), T=_log_int(rng, 1, 4096), train=rng.random() < 0.7)
            c["lo"] = rng.randint(0, c["T"])
            if work(c)["flops"] > (2e10 if c["dtype"] == "float32" else 3.5e11):
                continue
            return c
        c.update(B=_log_int(rng, 1, 256), ctx=_log_int(rng, 1, 65536), ps=rng.choice((16, 16, 32, 64, 128)),
                 new=_log_int(rng, 1, 2048))
        c["ones"] = rng.choice((0, c["B"], c["B"], rng.randint(0, c["B"])))
        c["new_lo"] = rng.randint(0, c["new"])
        c["ctx_lo"] = rng.randint(0, c["ctx"])
        ctx, new = _requests(c)
        total = sum(ctx) + sum(new)
        if sum(new) == 0 or sum(new) * c["H"] * c["D"] > 8192 * 32 * 128:
            continue
        if total * c["Hkv"] * c["D"] * _SIZE[c["dtype"]] > 1 << 29:
            continue
        if work(c)["flops"] > (2e10 if c["dtype"] == "float32" else 3.5e11):
            continue
        return c


def _lens(c):
    """Lengths of the packed sequences (the longest is T)."""
    r = random.Random(c["lens"])
    if c["B"] == 1:
        return [c["T"]]
    n = [r.randint(c["lo"], c["T"]) for _ in range(c["B"])]
    n[r.randrange(c["B"])] = c["T"]
    return n


def _requests(c):
    """Tokens in the cache and new tokens of every request."""
    r = random.Random(c["lens"])
    ctx = [r.randint(c["ctx_lo"], c["ctx"]) for _ in range(c["B"])]
    new = [1 if b < c["ones"] else r.randint(c["new_lo"], c["new"]) for b in range(c["B"])]
    return ctx, new


def _positions(c):
    """Positions of the packed tokens: runs of neighbours."""
    r, at = random.Random(c["lens"]), []
    while len(at) < c["N"]:
        n = min(c["N"] - len(at), c["run"] if not at else r.randint(1, c["run"]))
        first = r.randint(0, c["P"] - n) if c["kind"] == "append" else 0
        at.extend(range(first, first + n))
    return at


def _seen(n, total, causal):
    """Visible (query, key) pairs of the last n of `total` tokens."""
    return n * (total - n) + n * (n + 1) // 2 if causal else n * total


def _offsets(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _pages(tokens, ps):
    return -(-tokens // ps)


@functools.lru_cache(64)
def _bucket_line(buckets, dist, two_sided):
    """Buckets of the relative positions -dist .. dist: one each for the near
    ones, logarithmic ones up to `dist`, half of them for keys after the query
    (one-sided: these share the first)."""
    n = buckets // 2 if two_sided else buckets
    near = n // 2
    far, i, m = list(range(near)), 0, n - near
    for d in range(near, dist + 1):
        # i = floor(log(d / near) / log(dist / near) * m), in whole numbers
        while i < m - 1 and d ** m * near ** (i + 1) >= dist ** (i + 1) * near ** m:
            i += 1
        far.append(near + i)
    after = [n + x for x in far[1:]] if two_sided else [0] * dist
    return tuple(far[::-1] + after)


def _inputs(c, seed):
    """The case's tensors, on the GPU, and its lengths."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(1000003 * (seed % (1 << 40)) + 31)
    dt = _DTYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dt)

    def shuffled(n):
        return torch.randperm(n, generator=g, device=dev).to(torch.int32)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    s = {"case": c}
    if c["kind"] in ("bias", "paged"):
        s["table"] = normal(c["buckets"], c["H"])
        s["buckets"] = ints(_bucket_line(c["buckets"], c["dist"], not c["causal"]))
    else:
        angle = torch.arange(c["P"], device=dev, dtype=torch.float64)[:, None] * torch.pow(
            10000.0, -torch.arange(0, c["rot"], 2, device=dev, dtype=torch.float64) / c["rot"])
        s["angles"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        s["at"] = ints(_positions(c))
        s["q"], s["k"] = normal(c["N"], c["H"], c["D"]), normal(c["N"], c["Hkv"], c["D"])
    if c["kind"] == "bias":
        n = _lens(c)
        s["q"], s["k"], s["v"] = normal(sum(n), c["H"], c["D"]), normal(sum(n), c["Hkv"], c["D"]), normal(
            sum(n), c["Hkv"], c["D"])
        s["do"] = normal(sum(n), c["H"], c["D"]) if c["train"] else None
        s["lens"], s["cu"] = n, ints(_offsets(n))
    elif c["kind"] == "paged":
        ctx, new = _requests(c)
        lens = [x + y for x, y in zip(ctx, new)]
        pages = [_pages(x, c["ps"]) for x in lens]
        pool, first, width = shuffled(sum(pages) + 3), _offsets(pages), max(1, max(pages))
        j = torch.arange(width, device=dev)[None]
        at = (ints(first[:-1])[:, None] + j).clamp(max=pool.numel() - 1)
        s["pages"] = torch.where(j < ints(pages)[:, None], pool[at.long()], -1).to(torch.int32).contiguous()
        shape = (pool.numel(), c["ps"], c["Hkv"], c["D"])
        s["kc"], s["vc"], s["q"] = normal(*shape), normal(*shape), normal(sum(new), c["H"], c["D"])
        s["new"], s["lens"], s["longest"] = new, lens, max(new)
        s["cu"], s["seq_lens"] = ints(_offsets(new)), ints(lens)
    elif c["kind"] == "append":
        shape = (c["slots"] // c["ps"], c["ps"], c["Hkv"], c["D"])
        s["v"], s["kc"], s["vc"] = normal(c["N"], c["Hkv"], c["D"]), normal(*shape), normal(*shape)
        # Runs of consecutive slots, as pages give them, then the padding rows.
        runs = shuffled(shape[0]).long()[:, None] * c["ps"] + torch.arange(c["ps"], device=dev)[None]
        s["slots"] = runs.reshape(-1)[:c["N"]].to(torch.int32).contiguous()
        if c["pad"]:
            s["slots"][c["N"] - c["pad"]:] = -1
    else:
        s["dq"], s["dk"] = normal(c["N"], c["H"], c["D"]), normal(c["N"], c["Hkv"], c["D"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["kind"] == "bias" and case["train"]:
        for x in ("q", "k", "v", "table"):
            s[x].requires_grad_(True)
    if own and case["kind"] == "rotate":
        for x in ("q", "k"):
            s[x].requires_grad_(True)
    return s


# ---- the framework's operators ------------------------------------------------

@functools.lru_cache(None)
def _framework():
    sys.path.insert(0, os.path.join(os.getcwd(), "triton-sigmoid_amd"))
    import triton_sigmoid
    return triton_sigmoid


def _run_own(s):
    ts, c = _framework(), s["case"]
    if c["kind"] == "bias":
        def attend():
            return ts.sigmoid_attention_varlen(s["q"], s["k"], s["v"], s["cu"], s["cu"], c["T"], c["T"],
                                               is_causal=c["causal"], bias_table=s["table"], bias_buckets=s["buckets"])
        if not c["train"]:
            with torch.no_grad():
                return {"o": attend()}
        o = attend()
        dq, dk, dv, dtable = torch.autograd.grad(o, (s["q"], s["k"], s["v"], s["table"]), s["do"])
        return {"o": o, "dq": dq, "dk": dk, "dv": dv, "dtable": dtable}
    if c["kind"] == "rotate":
        q, k = ts.rotary_embedding(s["q"], s["k"], s["at"], s["angles"], interleaved=c["pairs"])
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    with torch.no_grad():
        if c["kind"] == "append":
            q = ts.paged_cache_write_rotary(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["slots"], s["at"], s["angles"],
                                            interleaved=c["pairs"])
            return {"q": q, "kc": s["kc"], "vc": s["vc"]}
        return ts.sigmoid_attention_paged(s["q"], s["kc"], s["vc"], s["pages"], s["seq_lens"], s["cu"], s["longest"],
                                          is_causal=c["causal"], bias_table=s["table"], bias_buckets=s["buckets"])


# ---- plain forms ----------------------------------------------------------------

def _plain_line(s, lo, hi):
    """The learned values [H, hi - lo + 1] of the relative positions lo .. hi."""
    dist = s["case"]["dist"]
    d = torch.arange(lo, hi + 1, device="cuda").clamp(-dist, dist) + dist
    return s["table"].float()[s["buckets"].long()[d]].t()


def _plain_bias(s):
    """Per sequence, all heads of one key/value head at a time, in 32 bits."""
    c = s["case"]
    G, scale, dt = c["H"] // c["Hkv"], 1.0 / math.sqrt(c["D"]), s["q"].dtype
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    do = s["do"].float() if c["train"] else None
    o = torch.empty_like(q)
    dq, dk, dv = (torch.empty_like(t) for t in (q, k, v)) if c["train"] else (None, None, None)
    dtable = torch.zeros(s["table"].shape, dtype=torch.float64, device=q.device)
    first = 0
    for n in s["lens"]:
        at = slice(first, first + n)
        first += n
        if n == 0:
            continue
        line = _plain_line(s, 1 - n, n - 1) - math.log(n)
        for hk in range(c["Hkv"]):
            hs = slice(hk * G, (hk + 1) * G)
            qh = q[at, hs].transpose(0, 1).contiguous()  # [G, n, D]
            kh, vh = k[at, hk].contiguous(), v[at, hk].contiguous()
            add = line[hs].unfold(1, n, 1).flip(1)  # row i: the values of positions -i .. n - 1 - i
            p = torch.sigmoid(torch.matmul(qh, kh.t()) * scale + add)
            if c["causal"]:
                p = torch.tril(p)
            o[at, hs] = torch.matmul(p, vh).transpose(0, 1)
            if not c["train"]:
                continue
            doh = do[at, hs].transpose(0, 1).contiguous()
            ds = torch.matmul(doh, vh.t()) * (p * (1.0 - p))
            dq[at, hs] = (torch.matmul(ds, kh) * scale).transpose(0, 1)
            dk[at, hk] = torch.matmul(ds.reshape(G * n, n).t(), qh.reshape(G * n, -1)) * scale
            dv[at, hk] = torch.matmul(p.reshape(G * n, n).t(), doh.reshape(G * n, -1))
            # Diagonals as columns: row n - 1 - i begins i places further on.
            skew = torch.nn.functional.pad(ds.flip(1), (0, n)).reshape(G, -1)[:, :n * (2 * n - 1)]
            diagonal = skew.reshape(G, n, 2 * n - 1).sum(1, dtype=torch.float64)
            d = torch.arange(1 - n, n, device=q.device).clamp(-c["dist"], c["dist"]) + c["dist"]
            dtable[:, hs] = dtable[:, hs].index_add(0, s["buckets"].long()[d], diagonal.t())
    if not c["train"]:
        return {"o": o.to(dt)}
    return {"o": o.to(dt), "dq": dq.to(dt), "dk": dk.to(dt), "dv": dv.to(dt), "dtable": dtable.to(dt)}


def _plain_paged(s):
    c, q = s["case"], s["q"]
    G, scale, ps = c["H"] // c["Hkv"], 1.0 / math.sqrt(c["D"]), c["ps"]
    out, first = torch.empty(q.shape, dtype=torch.float32, device=q.device), 0
    for b, (n, total) in enumerate(zip(s["new"], s["lens"])):
        if n == 0:
            continue
        pages = s["pages"][b, :_pages(total, ps)].long()
        k = s["kc"][pages].reshape(-1, c["Hkv"], c["D"])[:total].float().permute(1, 2, 0).contiguous()
        v = s["vc"][pages].reshape(-1, c["Hkv"], c["D"])[:total].float().transpose(0, 1).contiguous()
        qb = q[first:first + n].float().reshape(n, c["Hkv"], G, c["D"]).permute(1, 2, 0, 3).reshape(c["Hkv"], G * n, -1)
        # Query i sits at position total - n + i.
        line = _plain_line(s, 1 - total, n - 1) - math.log(total)
        add = line.unfold(1, total, 1).flip(1).reshape(c["Hkv"], G * n, total)
        p = torch.sigmoid(torch.matmul(qb, k) * scale + add)
        if c["causal"]:
            i = torch.arange(n, device=q.device).repeat(G) + (total - n)
            p = torch.where(torch.arange(total, device=q.device)[None] <= i[:, None], p, 0.0)
        o = torch.matmul(p, v).reshape(c["Hkv"], G, n, c["D"]).permute(2, 0, 1, 3)
        out[first:first + n] = o.reshape(n, c["H"], c["D"])
        first += n
    return out.to(q.dtype)


def _plain_turn(s, x, back=False):
    """Rows [N, heads, D] turned by their positions' angles, in 32 bits."""
    c, half = s["case"], s["case"]["rot"] // 2
    row = s["angles"][s["at"].long()]
    cos, sin = row[:, None, :half], row[:, None, half:]
    if back:
        sin = -sin
    y = x.float().clone()
    a, b = (slice(0, c["rot"], 2), slice(1, c["rot"], 2)) if c["pairs"] else (slice(0, half), slice(half, c["rot"]))
    u, w = x[..., a].float(), x[..., b].float()
    y[..., a] = u * cos - w * sin
    y[..., b] = w * cos + u * sin
    return y.to(x.dtype)


def _plain_append(s):
    slots = s["slots"].long()
    at = torch.nonzero(slots >= 0)[:, 0]
    for rows, cache in ((_plain_turn(s, s["k"]), s["kc"]), (s["v"], s["vc"])):
        cache.view(-1, *cache.shape[2:])[slots[at]] = rows[at]
    return {"q": _plain_turn(s, s["q"]), "kc": s["kc"], "vc": s["vc"]}


def _plain_rotate(s):
    return {"q": _plain_turn(s, s["q"]), "k": _plain_turn(s, s["k"]), "dq": _plain_turn(s, s["dq"], True),
            "dk": _plain_turn(s, s["dk"], True)}


def run(state):
    if own:
        return _run_own(state)
    return {"bias": _plain_bias, "paged": _plain_paged, "append": _plain_append,
            "rotate": _plain_rotate}[state["case"]["kind"]](state)


def work(case):
    """Bytes: every input read once and every output written once (the cache's
    rows in use and the slots written only, the angles of the positions that
    occur); flops: 4·D per visible pair and query head forward and 10·D backward,
    3 for each turned element."""
    c = case
    size = _SIZE[c["dtype"]]
    if c["kind"] in ("append", "rotate"):
        angles = 4 * c["rot"] * len(set(_positions(c)))
        if c["kind"] == "append":
            there = c["N"] - c["pad"]
            return {"bytes": 2 * (c["N"] * c["H"] + 2 * there * c["Hkv"]) * c["D"] * size + 8 * c["N"] + angles,
                    "flops": 3 * (c["N"] * c["H"] + there * c["Hkv"]) * c["rot"]}
        rows = c["N"] * (c["H"] + c["Hkv"])
        return {"bytes": 4 * rows * c["D"] * size + 4 * c["N"] + angles, "flops": 6 * rows * c["rot"]}
    table = c["buckets"] * c["H"] * size + 4 * (2 * c["dist"] + 1)
    if c["kind"] == "bias":
        n = _lens(c)
        pairs = sum(_seen(x, x, c["causal"]) for x in n)
        times = 4 if c["train"] else 2  # Q, O (dO, dQ); K, V (dK, dV)
        return {"bytes": sum(n) * times * (c["H"] + c["Hkv"]) * c["D"] * size + times // 2 * table,
                "flops": (14 if c["train"] else 4) * c["D"] * c["H"] * pairs}
    ctx, new = _requests(c)
    keys = sum(x + y for x, y in zip(ctx, new) if y)
    pairs = sum(_seen(y, x + y, c["causal"]) for x, y in zip(ctx, new))
    return {"bytes": (2 * keys * c["Hkv"] + 2 * sum(new) * c["H"]) * c["D"] * size + 4 * (keys // c["ps"]) + table,
            "flops": 4 * c["D"] * c["H"] * pairs}


# ---- the definitions in 64 bits ---------------------------------------------------

def _exact_head(c, q, k, v, do, column, add, offset, dcolumn):
    """O (and dQ, dK, dV, the last two summed by the caller) of one query head,
    by blocks of queries; query i sits at position i + offset. `column`: the learned
    values of the head by bucket, whose gradient is added to `dcolumn`."""
    scale = q.shape[1] ** -0.5
    o, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    step = max(64, (1 << 25) // max(k.shape[0], 1))
    kt, vt = k.t().contiguous(), v.t().contiguous()
    line = torch.tensor(_bucket_line(c["buckets"], c["dist"], not c["causal"]), device="cuda")
    for i in range(0, q.shape[0], step):
        j = min(q.shape[0], i + step)
        away = torch.arange(k.shape[0], device="cuda")[None] - (torch.arange(i, j, device="cuda")[:, None] + offset)
        bucket = line[torch.clamp(away, -c["dist"], c["dist"]) + c["dist"]]
        p = 1.0 / (1.0 + torch.exp(-((q[i:j] @ kt) * scale + add + column[bucket])))
        if c["causal"]:
            p = torch.where(away > 0, 0.0, p)
        o[i:j] = p @ v
        if do is not None:
            ds = (p - p * p) * (do[i:j] @ vt)
            dq[i:j] = scale * (ds @ k)
            dk += scale * (ds.t().contiguous() @ q[i:j])
            dv += p.t().contiguous() @ do[i:j]
            for u in range(c["buckets"]):
                dcolumn[u] += torch.where(bucket == u, ds, 0.0).sum()
    return o, dq, dk, dv


def _exact_bias(c, s):
    at = _offsets(_lens(c))
    out = {x: torch.zeros(s[y].shape, dtype=torch.float64, device="cuda")
           for x, y in (("o", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v"), ("dtable", "table"))}
    for a, b in zip(at[:-1], at[1:]):
        for h in range(c["H"] if b > a else 0):
            hk = h * c["Hkv"] // c["H"]
            one = [None if t is None else t[a:b, x].double().contiguous()
                   for t, x in ((s["q"], h), (s["k"], hk), (s["v"], hk), (s["do"], h))]
            o, dq, dk, dv = _exact_head(c, *one, s["table"][:, h].double(), -math.log(b - a), 0, out["dtable"][:, h])
            out["o"][a:b, h], out["dq"][a:b, h] = o, dq
            out["dk"][a:b, hk] += dk
            out["dv"][a:b, hk] += dv
    return out if c["train"] else {"o": out["o"]}


def _exact_paged(c, s):
    ctx, new = _requests(c)
    at, out = _offsets(new), torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (x, n) in enumerate(zip(ctx, new)):
        if n == 0:
            continue
        pos = torch.arange(x + n, device="cuda")
        page, row = s["pages"][b].long()[pos // c["ps"]], pos % c["ps"]
        for hk in range(c["Hkv"]):
            k, v = s["kc"][page, row, hk].double(), s["vc"][page, row, hk].double()
            for h in range(hk * c["H"] // c["Hkv"], (hk + 1) * c["H"] // c["Hkv"]):
                q = s["q"][at[b]:at[b + 1], h].double().contiguous()
                out[at[b]:at[b + 1], h] = _exact_head(c, q, k, v, None, s["table"][:, h].double(), -math.log(x + n), x,
                                                      None)[0]
    return out


def _exact_turn(c, s, x, sign=1.0):
    """Rows as complex numbers times unit ones; the angles are the given table's."""
    half, x = c["rot"] // 2, x.double()
    row = s["angles"].double()[s["at"].long()]
    unit = torch.complex(row[:, :half], sign * row[:, half:])[:, None]
    turned, rest = x[..., :c["rot"]], x[..., c["rot"]:]
    pair = turned.unflatten(-1, (half, 2)) if c["pairs"] else turned.unflatten(-1, (2, half)).transpose(-1, -2)
    z = torch.view_as_real(torch.complex(pair[..., 0].contiguous(), pair[..., 1].contiguous()) * unit)
    z = z if c["pairs"] else z.transpose(-1, -2)
    return torch.cat([z.reshape(turned.shape), rest], -1)


def _exact_append(c, s):
    slots = s["slots"].tolist()
    row_of = torch.full((c["slots"],), -1, dtype=torch.long)
    for t, slot in enumerate(slots):
        if slot >= 0:
            row_of[slot] = t
    row_of = row_of.cuda()
    got = {"q": _exact_turn(c, s, s["q"])}
    for name, rows in (("kc", _exact_turn(c, s, s["k"])), ("vc", s["v"].double())):
        flat = s[name].double().reshape(c["slots"], -1)
        new = rows.reshape(c["N"], -1)[row_of.clamp(min=0)]
        got[name] = torch.where((row_of >= 0)[:, None], new, flat).reshape(s[name].shape)
    return got


def _exact_rotate(c, s):
    return {"q": _exact_turn(c, s, s["q"]), "k": _exact_turn(c, s, s["k"]), "dq": _exact_turn(c, s, s["dq"], -1.0),
            "dk": _exact_turn(c, s, s["dk"], -1.0)}


def exact(case, seed):
    c = case
    s = _inputs(c, seed)
    if c["kind"] in ("bias", "paged") and work(c)["flops"] > 3e12:
        return None
    return {"bias": _exact_bias, "paged": _exact_paged, "append": _exact_append, "rotate": _exact_rotate}[c["kind"]](c, s)
