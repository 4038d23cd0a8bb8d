"""Paged cache: the plan, the writer and the attention against plain
implementations (the attention's in 64 bits), and a run of them together."""

import math
import random

import pytest
import torch
from torch.autograd import forward_ad

import triton_sigmoid as ts
from reference64 import assert_within, one_head

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
I32 = torch.int32


def ints(v):
    return torch.tensor(v, dtype=I32, device="cuda")


def offsets(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


# --- plan ---------------------------------------------------------------------------

def plain_plan(ctx, new, table, free, ps, N):
    table, taken, slots = [list(r) for r in table], 0, []
    for b, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        for j in range(-(-c // ps), -(-(c + n) // ps)):
            if j < len(table[b]):
                table[b][j] = free[taken] if taken < len(free) else -1
            taken += 1
        for x in range(c, c + n):
            page = table[b][x // ps] if x // ps < len(table[b]) else -1
            slots.append(page * ps + x % ps if page >= 0 else -1)
    slots = (slots + [-1] * N)[:N]
    cu = offsets([max(n, 0) for n in new])
    return table, slots, cu, [max(c, 0) + max(n, 0) for c, n in zip(ctx, new)], taken


def check_plan(ctx, new, ps, N, pages=None, width=None, seed=0, ids=None):
    r = random.Random(seed)
    held = [-(-max(c, 0) // ps) for c in ctx]
    total = [-(-(max(c, 0) + max(n, 0)) // ps) for c, n in zip(ctx, new)]
    width = max(total, default=0) if width is None else width
    pool = r.sample(range(sum(total) + 9), sum(total) + 9)
    table = [[pool.pop() if j < h else -7 for j in range(width)] for h in held]
    free = pool if pages is None else pool[:pages]
    got = ts.paged_plan(ints(ctx), ints(new), ints(table).reshape(len(ctx), width), ints(free), ps, N)
    want = plain_plan(ctx, new, table, free, ps, N)
    for name, g, w in zip(got._fields, got, want):
        assert g.dtype == I32
        assert g.tolist() == w, name


@pytest.mark.parametrize("B", [0, 1, 2, 63, 64, 65, 255, 256, 257, 1000, 8192])
def test_plan_of_batches(B):
    r = random.Random(B)
    ctx = [r.randint(0, 90) for _ in range(B)]
    new = [r.choice((0, 1, 1, r.randint(0, 40))) for _ in range(B)]
    check_plan(ctx, new, 16, sum(new) + r.choice((0, 5)), seed=B)


@pytest.mark.parametrize("ps", [16, 32, 128, 256, 1 << 20])
def test_plan_page_borders(ps):
    p = min(ps, 512)
    ctx = [0, 0, p - 1, p, p + 1, 2 * p, 0, p - 1]
    new = [0, 1, 1, 1, p, p, 2 * p + 1, 2]
    check_plan(ctx, new, ps, sum(new) + 3)


def test_plan_of_many_tokens():
    check_plan([5, 0, 100], [40000, 0, 27001], 16, 67100)


def test_plan_without_enough_pages_or_columns():
    check_plan([10, 20, 30], [30, 30, 30], 16, 90, pages=3)  # the last request goes without
    check_plan([10, 20, 30], [30, 30, 30], 16, 90, pages=0)
    check_plan([10, 20, 0], [30, 3, 100], 16, 133, width=3)  # more pages than columns
    check_plan([10, 20], [30, 30], 16, 25)  # fewer rows than tokens
    check_plan([-3, 20], [5, -2], 16, 9)  # negative lengths count as none


def test_plan_of_sums_past_32_bits_ends():
    big, wide = (1 << 31) - 1, torch.full((4, 5), 99, dtype=I32, device="cuda")
    table = wide[:3, 1:4]
    ts.paged_plan(ints([big, 0, 5]), ints([big, 7, big]), table, ints([50, 51]), 1 << 20, 300)
    torch.cuda.synchronize()
    assert (wide[:, 0] == 99).all() and (wide[:, 4] == 99).all() and (wide[3] == 99).all()


@pytest.mark.parametrize("binding", ["node", "python"])
def test_autograd_sees_what_is_changed(monkeypatch, binding):
    if binding == "python":
        monkeypatch.setenv("SIGATTN_EAGER_BINDING", "python")
    kc, vc = (torch.randn(4, 16, 2, 32, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    table = torch.zeros(1, 2, dtype=I32, device="cuda")
    at = table._version
    plan = ts.paged_plan(ints([0]), ints([3]), table, ints([2, 1]), 16, 3)
    assert table._version == at + 1
    w = torch.ones((), device="cuda", requires_grad=True)
    y = (w * kc).sum()
    at = kc._version, vc._version
    new = torch.randn(3, 2, 32, device="cuda", dtype=torch.bfloat16)
    ts.paged_cache_write(new, new, kc, vc, plan.slot_mapping)
    assert (kc._version, vc._version) == (at[0] + 1, at[1] + 1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        kc, vc = torch.zeros_like(kc), torch.zeros_like(vc)
    ts.paged_cache_write(new, new, kc, vc, plan.slot_mapping)
    assert torch.equal(kc[2, :3], new)


def test_plan_keeps_other_entries_and_strides():
    wide = torch.full((3, 10), 99, dtype=I32, device="cuda")
    plan = ts.paged_plan(ints([17, 0, 3]), ints([16, 0, 1]), wide[:, 2:7], ints([50, 51, 52]), 16, 17)
    want = torch.full((3, 10), 99, dtype=I32)
    want[0, 4] = 50
    assert torch.equal(wide.cpu(), want) and plan.pages_needed.item() == 1
    assert plan.block_table.data_ptr() == wide[:, 2:7].data_ptr()
    assert plan.slot_mapping.tolist() == [99 * 16 + i for i in range(1, 16)] + [-1] * 0 + [50 * 16] + [99 * 16 + 3]


# --- writer ---------------------------------------------------------------------------

@pytest.mark.parametrize("layout", ["rows", "heads first", "joint"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("N, heads, D, ps", [(1, 1, 16, 16), (3, 3, 32, 16), (100, 8, 128, 64), (1031, 5, 64, 32)])
def test_write(N, heads, D, ps, dtype, layout):
    g = torch.Generator().manual_seed(N)
    pages = -(-N // ps) + 3

    def caches():
        if layout == "rows":
            return torch.zeros(2, pages, ps, heads, D, dtype=DT[dtype]).cuda()
        if layout == "heads first":
            return torch.zeros(2, pages, heads, ps, D, dtype=DT[dtype]).cuda().transpose(2, 3)
        return torch.zeros(pages, 2, ps, heads, D, dtype=DT[dtype]).cuda().transpose(0, 1)

    both = caches()
    both.copy_(torch.randn(both.shape, generator=g))
    k, v = (torch.randn(N, heads, D, generator=g).to(DT[dtype]).cuda() for _ in range(2))
    slots = torch.randperm(pages * ps, generator=g)[:N]
    slots[torch.rand(N, generator=g) < 0.2] = -1
    if N > 3:
        slots[1], slots[2] = pages * ps, 2 ** 31 - 1  # past the cache: not written
    want = both.clone()
    ok = (slots >= 0) & (slots < pages * ps)
    for c, rows in zip(want, (k, v)):
        at = slots[ok].cuda()
        c[at // ps, at % ps] = rows[ok.cuda()]
    ts.paged_cache_write(k, v, both[0], both[1], slots.to(I32).cuda())
    assert torch.equal(both, want)


def test_write_of_strided_and_unaligned_rows():
    g = torch.Generator().manual_seed(1)
    wide = torch.randn(50, 10, 32, generator=g).half().cuda()
    kc, vc = (torch.zeros(5, 16, 3, 32, dtype=torch.half, device="cuda") for _ in range(2))
    slots = torch.randperm(80, generator=g)[:50].to(I32).cuda()
    ts.paged_cache_write(wide[:, 4:7], wide[:, 7:], kc, vc, slots)
    flat = wide.cpu()
    for c, rows in ((kc, flat[:, 4:7]), (vc, flat[:, 7:])):
        assert torch.equal(c.cpu().view(80, 3, 32)[slots.cpu().long()], rows)
    odd = torch.randn(50 * 96 + 1, generator=g).half().cuda()[1:].view(50, 3, 32)  # off 16 bytes
    ts.paged_cache_write(odd, wide[:, 7:], kc, vc, slots.long())
    assert torch.equal(kc.cpu().view(80, 3, 32)[slots.cpu().long()], odd.cpu())
    ts.paged_cache_write(wide[:0, :3], wide[:0, :3], kc, vc, slots[:0])


# --- attention --------------------------------------------------------------------------

def make(ctx, new, ps, H, Hkv, D, dtype, seed=0, spare=3, fill=float("nan"), layout="rows"):
    """A cache in shuffled pages whose unused rows hold `fill`."""
    g = torch.Generator().manual_seed(seed)
    lens = [c + n for c, n in zip(ctx, new)]
    pages = [-(-x // ps) for x in lens]
    pool = torch.randperm(sum(pages) + spare, generator=g).tolist()
    width = max(pages, default=0) + 1
    table = torch.full((len(lens), width), -1, dtype=I32)
    if layout == "heads first":
        caches = torch.full((2, len(pool), Hkv, ps, D), fill).transpose(2, 3)
    else:
        caches = torch.full((2, len(pool), ps, Hkv, D), fill)
    rows = []
    for b, x in enumerate(lens):
        kv = torch.randn(2, x, Hkv, D, generator=g)
        rows.append(kv.to(dtype).cuda())
        for j in range(pages[b]):
            table[b, j] = pool.pop()
            m = min(ps, x - j * ps)
            caches[:, table[b, j], :m] = kv[:, j * ps:j * ps + m]
    caches = caches.to(dtype).cuda()
    q = torch.randn(sum(new), H, D, generator=g).to(dtype).cuda()
    return q, caches[0], caches[1], table.cuda(), ints(lens), ints(offsets(new)), rows


def reference(q, rows, new, causal, mod=None, bias=None, scale=None, absent=None):
    """(value, bound) of O; absent[b]: positions whose pages are not there."""
    H = q.shape[1]
    val, err = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    at = offsets(new)
    for b, n in enumerate(new):
        k, v = rows[b]
        L = k.shape[0]
        if n == 0 or L == 0:
            continue
        add = torch.full((L,), -math.log(L) if bias is None else bias, dtype=torch.float64, device="cuda")
        if mod is not None:
            add = add + mod[b, :L].double()
        if absent is not None and absent[b]:
            add[absent[b]] = -torch.inf  # P = 0
        for h in range(H):
            hk = h // (H // k.shape[1])
            o = one_head(q[at[b]:at[b + 1], h], k[:, hk], v[:, hk], None, add, q.dtype, L - n if causal else None,
                         scale)["o"]
            val[at[b]:at[b + 1], h], err[at[b]:at[b + 1], h] = o
    return val, err


def check(ctx, new, ps, H, Hkv, D, dtype, causal=True, mod=False, max_q="longest", seed=0, layout="rows", **kw):
    q, kc, vc, table, lens, cu, rows = make(ctx, new, ps, H, Hkv, D, dtype, seed, layout=layout)
    term = None
    if mod:
        term = torch.randn(table.shape[0], table.shape[1] * ps, generator=torch.Generator().manual_seed(7)).cuda()
        term[:, 3] = -torch.inf
    longest = max(new, default=0) if max_q == "longest" else max_q
    got = ts.sigmoid_attention_paged(q, kc, vc, table, lens, cu, longest, is_causal=causal, score_mod=term, **kw)
    assert_within(got, reference(q, rows, new, causal, term, kw.get("sigmoid_bias"), kw.get("scale")), "o")
    return got


SHAPES = {
    "one of one": ([0], [1]),
    "decode": ([0, 14, 15, 16, 31, 32, 33, 63, 64, 127, 200, 515], [1] * 12),
    "few": ([0, 30, 100, 513, 5], [4, 3, 0, 2, 4]),
    "chunk": ([0, 100, 301], [130, 33, 64]),
    "mixed": ([250, 0, 77, 129, 600, 31], [1, 97, 1, 0, 40, 1]),
    "long": ([1500, 900], [70, 300]),
}


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("heads", [(4, 4), (8, 2), (6, 2), (16, 1)], ids=lambda h: f"{h[0]}x{h[1]}")
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_against_64_bits(shape, dtype, D, heads, causal):
    ctx, new = SHAPES[shape]
    if dtype == "f32" and shape == "long":
        ctx, new = [300], [70]
    check(ctx, new, 16 if D != 64 else 64, *heads, D, DT[dtype], causal)


@pytest.mark.parametrize("ps", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("layout", ["rows", "heads first"])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_page_sizes_and_layouts(D, layout, ps):
    check([5, 100, 1000, 0], [1, 1, 1, 1], ps, 8, 2, D, torch.bfloat16, layout=layout)
    check([5, 100, 700, 0], [50, 9, 1, 129], ps, 8, 2, D, torch.bfloat16, layout=layout)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape", ["decode", "few", "mixed", "long"])
def test_terms_per_key_bias_and_scale(shape, dtype):
    ctx, new = SHAPES[shape]
    for D in (64, 128):
        check(ctx, new, 16, 8, 2, D, DT[dtype], mod=True)
        check(ctx, new, 32, 8, 2, D, DT[dtype], causal=False, mod=True, sigmoid_bias=-3.0, scale=0.05)


@pytest.mark.parametrize("B", [65, 130, 300])
def test_many_sequences(B):
    r = random.Random(B)
    ctx = [r.choice((0, r.randint(0, 60), r.randint(0, 400))) for _ in range(B)]
    check(ctx, [1] * B, 16, 4, 2, 64, torch.bfloat16)
    check(ctx, [r.choice((0, 1, 1, 1, r.randint(2, 30))) for _ in range(B)], 16, 4, 1, 128, torch.float16)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads", [(8, 8), (8, 1), (32, 2)], ids=lambda h: f"{h[0]}x{h[1]}")
def test_long_contexts_are_split(heads, D):
    check([9000], [1], 16, *heads, D, torch.bfloat16)
    check([5000, 17, 2500], [1, 1, 1], 64, *heads, D, torch.bfloat16)
    check([4000, 900], [60, 1], 32, *heads, D, torch.bfloat16)


def test_longest_query_not_given_or_cut():
    ctx, new = [100, 0, 40], [1, 37, 4]
    whole = check(ctx, new, 16, 8, 2, 128, torch.bfloat16)
    loose = check(ctx, new, 16, 8, 2, 128, torch.bfloat16, max_q=None)
    assert whole.shape == loose.shape
    # A bound below a length cuts the sequence: its first rows end at its length.
    q, kc, vc, table, lens, cu, rows = make(ctx, new, 16, 8, 2, 128, torch.bfloat16)
    got = ts.sigmoid_attention_paged(q, kc, vc, table, lens, cu, 4, is_causal=True)
    keep = torch.cat([torch.arange(0, 5), torch.arange(38, 42)]).cuda()
    val, err = reference(q[keep], rows, [1, 4, 4], True)
    assert_within(got[keep], (val, err), "cut")
    rest = torch.ones(42, dtype=torch.bool)
    rest[keep.cpu()] = False
    assert not got[rest.cuda()].any()


def test_more_queries_than_keys_and_no_keys():
    """Rows before position 0 see nothing; a sequence without keys is zeros."""
    for dtype in (torch.bfloat16, torch.float32):
        for D in (64, 128):
            q, kc, vc, table, lens, cu, rows = make([20, 30], [10, 40], 16, 4, 2, D, dtype)
            lens = ints([30, 5])  # 40 queries over 5 keys
            got = ts.sigmoid_attention_paged(q, kc, vc, table, lens, cu, 40, is_causal=True)
            rows[1] = rows[1][:, :5]
            val, err = reference(q, rows, [10, 40], True)
            assert_within(got, (val, err), "o")
            assert not got[10:45].any()
            for causal in (True, False):
                got = ts.sigmoid_attention_paged(q, kc, vc, table, ints([0, 0]), cu, 40, is_causal=causal)
                assert not got.any()


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 70]], ids=["decode", "mixed"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_pages_that_are_not_there(dtype, new):
    """Bad page ids and lengths past the table: no keys there, no fault."""
    ctx = [100, 20, 200]
    q, kc, vc, table, lens, cu, rows = make(ctx, new, 16, 4, 2, 128, DT[dtype], fill=0.0)
    table[0, 2], table[2, 0], table[2, 5] = -1, kc.shape[0], 2 ** 31 - 1
    absent = [list(range(32, 48)), [], [*range(0, 16), *range(80, 96)]]
    got = ts.sigmoid_attention_paged(q, kc, vc, table, lens, cu, max(new), is_causal=True)
    assert_within(got, reference(q, rows, new, True, absent=absent), "o")
    # Lengths past the table are cut to it; its last column is -1 here.
    wide = table.shape[1] * 16
    got = ts.sigmoid_attention_paged(q, kc, vc, table, ints([2 ** 31 - 1] * 3), cu, max(new), sigmoid_bias=-5.0)
    short = ts.sigmoid_attention_paged(q, kc, vc, table, ints([wide] * 3), cu, max(new), sigmoid_bias=-5.0)
    assert torch.equal(got, short) and torch.isfinite(got).all()
    got = ts.sigmoid_attention_paged(q, kc, vc, table, ints([-4] * 3), cu, max(new))
    assert not got.any()


@pytest.mark.parametrize("new", [[1, 1], [50, 3]], ids=["decode", "chunk"])
def test_rows_outside_every_sequence_are_zero(new):
    for dtype in (torch.float16, torch.float32):
        q, kc, vc, table, lens, cu, rows = make([40, 100], new, 16, 4, 2, 64, dtype)
        more = torch.cat([q, q, q])[:sum(new) + 70].contiguous()
        got = ts.sigmoid_attention_paged(more, kc, vc, table, lens, cu, max(new), is_causal=True)
        assert torch.equal(got[:sum(new)],
                           ts.sigmoid_attention_paged(q, kc, vc, table, lens, cu, max(new), is_causal=True))
        assert not got[sum(new):].any()


@pytest.mark.parametrize("B", [2, 70])
@pytest.mark.parametrize("new", [1, 200], ids=["decode", "chunk"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_rows_before_the_first_sequence_are_zero(dtype, new, B):
    # Contexts long enough to be cut: the sums of parts know the rows of no sequence too.
    n = [new] + [1] * (B - 1)
    q, kc, vc, table, lens, cu, _ = make([4000, 3000] + [5] * (B - 2), n, 16, 4, 2, 32, dtype)
    want = ts.sigmoid_attention_paged(q, kc, vc, table, lens, cu, new, is_causal=True)
    more = torch.cat([q, q, q])[:sum(n) + 60] if sum(n) > 60 else q.repeat(80, 1, 1)[:sum(n) + 60]
    more[37:37 + sum(n)] = q
    got = ts.sigmoid_attention_paged(more.contiguous(), kc, vc, table, lens, cu + 37, new, is_causal=True)
    assert not got[:37].any() and not got[37 + sum(n):].any()
    assert torch.equal(got[37:37 + sum(n)], want)


@pytest.mark.parametrize("chunk, longest", [(0, 400), (40, 400), (40, 3000)], ids=["decode", "mixed", "chunk cut"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_thousand_sequences(dtype, chunk, longest):
    # Enough that decoding is not cut and its units are found without the other
    # lengths; a chunk of new tokens on many keys is.
    r = random.Random(11)
    ctx = [r.choice((0, 1, 15, 16, 40, 90)) for _ in range(1030)]
    new = [r.choice((0, 1, 1, 1)) for _ in ctx]
    ctx[700], new[3] = longest, chunk or 1
    if longest > 1024:
        new[700] = chunk
    check(ctx, new, 16, 2, 1, 32, DT[dtype])


def test_caches_and_tables_without_pages():
    q = torch.randn(5, 4, 64, device="cuda", dtype=torch.bfloat16)
    none = torch.empty(0, 16, 2, 64, device="cuda", dtype=torch.bfloat16)
    some = torch.full((3, 16, 2, 64), float("nan"), device="cuda", dtype=torch.bfloat16)
    cu = ints([0, 2, 5])
    for cache, table in ((none, torch.zeros(2, 40, dtype=I32, device="cuda")), (some, ints([]).reshape(2, 0))):
        got = ts.sigmoid_attention_paged(q, cache, cache.clone(), table, ints([600, 17]), cu, 3, is_causal=True)
        assert got.shape == q.shape and not got.any()
    ts.paged_cache_write(q[:, :2], q[:, 2:], none, none.clone(), ints([0, 1, 2, 3, 4]))


def test_no_sequences_and_no_rows():
    q, kc, vc, table, lens, cu, _ = make([4], [3], 16, 4, 2, 64, torch.bfloat16)
    none = ts.sigmoid_attention_paged(q, kc, vc, table[:0], lens[:0], cu[:1])
    assert none.shape == q.shape and not none.any()
    assert ts.sigmoid_attention_paged(q[:0], kc, vc, table, lens, ints([0, 0])).shape == (0, 4, 64)
    assert not ts.sigmoid_attention_paged(q, kc[:0], vc[:0], table, lens, cu).any()


@pytest.mark.parametrize("D", [64, 128])
def test_strided_and_unaligned_tensors(D):
    ctx, new = [100, 33, 400], [1, 20, 1]
    q, kc, vc, table, lens, cu, rows = make(ctx, new, 32, 6, 2, D, torch.float16)
    want = ts.sigmoid_attention_paged(q, kc, vc, table, lens, cu, 20, is_causal=True)
    wide = torch.cat([q, q], dim=1)
    joint = torch.stack([kc, vc], dim=1)
    table2 = torch.full((3, 40), -1, dtype=I32, device="cuda")
    table2[:, 3:3 + table.shape[1]] = table
    got = ts.sigmoid_attention_paged(wide[:, 6:], joint[:, 0], joint[:, 1], table2[:, 3:3 + table.shape[1]],
                                     lens.long(), cu.long(), 20, is_causal=True)
    assert torch.equal(got, want)

    def off(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        buf[1:] = t.reshape(-1)
        return buf[1:].view(t.shape)

    got = ts.sigmoid_attention_paged(off(q), off(kc), off(vc), table, lens, cu, 20, is_causal=True)
    assert_within(got, reference(q, rows, new, True), "unaligned")
    got = ts.sigmoid_attention_paged(off(q), kc, vc, table, lens, cu, 20, is_causal=True)
    assert_within(got, reference(q, rows, new, True), "unaligned query")


def test_other_streams_and_repeats():
    ctx, new = [3000, 100, 700], [1, 1, 1]
    q, kc, vc, table, lens, cu, _ = make(ctx, new, 16, 16, 2, 128, torch.bfloat16)
    want = ts.sigmoid_attention_paged(q, kc, vc, table, lens, cu, 1)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ts.sigmoid_attention_paged(q, kc, vc, table, lens, cu, 1))
    torch.cuda.synchronize()
    for o in got:
        assert torch.equal(o, want)


@pytest.mark.parametrize("N, longest", [(8, 1), (200, 150)])
def test_captured_step_on_other_lengths(N, longest):
    """A captured step (plan, write, attention) replayed on other lengths
    equals the eager one; two graphs of it take turns."""
    B, ps, H, Hkv, D, width = 4, 16, 8, 2, 128, 80
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(N, Hkv, D, generator=g).bfloat16().cuda() for _ in range(2))
    q = torch.randn(N, H, D, generator=g).bfloat16().cuda()
    pages = B * width + 7
    order = torch.randperm(pages, generator=g).to(I32).cuda()
    start = torch.randn(2, pages, ps, Hkv, D, generator=g).bfloat16().cuda()
    caches = start.clone()
    table = torch.empty(B, width, dtype=I32, device="cuda")
    ctx, new = ints([0] * B), ints([0] * B)

    def step():
        plan = ts.paged_plan(ctx, new, table, order[B * 40:], ps, N)
        ts.paged_cache_write(k, v, caches[0], caches[1], plan.slot_mapping)
        return plan.slot_mapping, ts.sigmoid_attention_paged(q, caches[0], caches[1], plan.block_table, plan.seq_lens,
                                                             plan.cu_seqlens, longest, is_causal=True)

    def reset(c, n):
        ctx.copy_(ints(c)), new.copy_(ints(n))
        table.copy_(order[:B * width].view(B, width))
        caches.copy_(start)

    reset([5] * B, [1] * B)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    lengths = [([5, 600, 0, 33], [1, 1, 1, 1]), ([100, 0, 639, 1], [1, 0, 1, 1])]
    if longest > 1:
        lengths = [([5, 600, 0, 33], [1, 20, 150, 1]), ([100, 0, 300, 1], [1, 140, 0, 3])]
    for c, n in lengths * 2:
        for graph, out in graphs:
            reset(c, n)
            graph.replay()
            torch.cuda.synchronize()
            have, cached = [t.clone() for t in out], caches.clone()
            reset(c, n)
            want = step()
            assert torch.equal(have[0], want[0]) and torch.equal(have[1], want[1]) and torch.equal(cached, caches)


def test_compiled_step():
    ctx, new = [40, 7], [1, 9]
    q, kc, vc, table, lens, cu, _ = make(ctx, new, 16, 4, 2, 64, torch.bfloat16, fill=0.0)
    k, v = (torch.randn(10, 2, 64).bfloat16().cuda() for _ in range(2))

    def step(q, k, v, kc, vc, table):
        plan = ts.paged_plan(ints(ctx), ints(new), table, free, 16, 10)
        ts.paged_cache_write(k, v, kc, vc, plan.slot_mapping)
        return ts.sigmoid_attention_paged(q, kc, vc, plan.block_table, plan.seq_lens, plan.cu_seqlens, 9,
                                          is_causal=True)

    ctx_t, new_t = ints(ctx), ints(new)
    free = ints([0, 1, 2, 3])

    def graph_step(q, k, v, kc, vc, table):
        plan = ts.paged_plan(ctx_t, new_t, table, free, 16, 10)
        ts.paged_cache_write(k, v, kc, vc, plan.slot_mapping)
        return ts.sigmoid_attention_paged(q, kc, vc, plan.block_table, plan.seq_lens, plan.cu_seqlens, 9,
                                          is_causal=True)

    one = [t.clone() for t in (kc, vc, table)]
    two = [t.clone() for t in (kc, vc, table)]
    want = step(q, k, v, *one)
    got = torch.compile(graph_step, fullgraph=True)(q, k, v, *two)
    assert torch.equal(got, want)
    for a, b in zip(one, two):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
def test_serving_equals_the_prompt_at_once(D, dtype):
    """Prompts in chunks and then token by token through plan, write and
    attention, against the packed attention of the whole sequences."""
    H, Hkv, ps, bias = 8, 2, 16, -5.0
    lens = [150, 37, 90]
    g = torch.Generator().manual_seed(5)
    data = [[torch.randn(n, h, D, generator=g).to(DT[dtype]).cuda() for h in (H, Hkv, Hkv)] for n in lens]
    cu = ints(offsets(lens))
    whole = ts.sigmoid_attention_varlen(*(torch.cat(x) for x in zip(*data)), cu, cu, is_causal=True, sigmoid_bias=bias)
    free = torch.randperm(40, generator=g).to(I32).cuda()
    table = torch.full((3, 12), -1, dtype=I32, device="cuda")
    kc, vc = (torch.full((40, ps, Hkv, D), float("nan"), dtype=DT[dtype], device="cuda") for _ in range(2))
    done, out = [0, 0, 0], [[], [], []]
    for step in range(60):
        take = [min(n - d, (50, 17, 1)[b] if step < 2 else (1, 3, 2)[b]) for b, (n, d) in enumerate(zip(lens, done))]
        if not any(take):
            break
        q, k, v = (torch.cat([data[b][x][done[b]:done[b] + take[b]] for b in range(3)]) for x in range(3))
        plan = ts.paged_plan(ints(done), ints(take), table, free, ps, sum(take))
        free = free[plan.pages_needed.item():]
        ts.paged_cache_write(k, v, kc, vc, plan.slot_mapping)
        o = ts.sigmoid_attention_paged(q, kc, vc, table, plan.seq_lens, plan.cu_seqlens, max(take), is_causal=True,
                                       sigmoid_bias=bias)
        at = offsets(take)
        for b in range(3):
            out[b].append(o[at[b]:at[b + 1]])
        done = [d + t for d, t in zip(done, take)]
    got = torch.cat([x for o in out for x in o])
    at = offsets(lens)
    val, err = (torch.zeros(whole.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    for b in range(3):
        for h in range(H):
            q, k, v = data[b]
            o = one_head(q[:, h], k[:, h // 4], v[:, h // 4], None, bias, DT[dtype], 0)["o"]
            val[at[b]:at[b + 1], h], err[at[b]:at[b + 1], h] = o
    assert_within(got, (val, err), "served")
    assert_within(whole, (val, err), "at once")


@pytest.mark.parametrize("B", [3, 64, 65, 200])
def test_cuts_of_ragged_batches(B):
    """Long and short contexts in one batch, with and without the candidates of
    small batches: every unit finds its chunk, every row its sums."""
    r = random.Random(B)
    top = {3: 6000, 64: 1500, 65: 1500, 200: 700}[B]
    ctx = [r.choice((0, 3, r.randint(0, 300), r.randint(0, top))) for _ in range(B)]
    ctx[r.randrange(B)] = 2 * top
    check(ctx, [1] * B, 16, 4, 2, 64, torch.bfloat16)
    new = [r.choice((1, 1, 0, 5, 40)) for _ in range(B)]
    check([min(c, 1500) for c in ctx], new, 32, 4, 2, 128, torch.bfloat16)


def test_workspace_of_other_calls_does_not_matter():
    """The same with a workspace full of NaN, and without one (nothing is cut)."""
    import ctypes

    from triton_sigmoid import _capi
    q, kc, vc, table, lens, cu, rows = make([3000, 10, 900, 500], [1, 1, 50, 33], 16, 8, 2, 128, torch.bfloat16)
    new = [1, 1, 50, 33]
    want = ts.sigmoid_attention_paged(q, kc, vc, table, lens, cu, 50, is_causal=True)
    lib = _capi.load_library()
    p = _capi.SigattnPagedProblem()
    p.abi_version, p.dtype = _capi.ABI_VERSION, _capi.BF16
    p.B, p.H, p.kv_heads, p.D, p.rows_q, p.max_seqlen_q = 4, 8, 2, 128, q.shape[0], 50
    p.num_pages, p.page_size, p.max_pages = kc.shape[0], 16, table.shape[1]
    p.q_stride_t, p.q_stride_h = 1024, 128
    p.k_stride_p, p.k_stride_t, p.k_stride_h = kc.stride()[:3]
    p.table_stride = table.stride(0)
    p.q, p.k_cache, p.v_cache = q.data_ptr(), kc.data_ptr(), vc.data_ptr()
    p.block_table, p.seq_lens_k, p.cu_seqlens_q = table.data_ptr(), lens.data_ptr(), cu.data_ptr()
    p.scale, p.causal = 128 ** -0.5, 1
    n = lib.sigattn_paged_fwd_workspace_bytes(ctypes.byref(p))
    assert n > 0
    ws = torch.full((n // 4 + 4,), float("nan"), device="cuda")
    out = torch.full_like(q, float("nan"))
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.sigattn_paged_fwd(ctypes.byref(p), out.data_ptr(), ws.data_ptr(), n, stream) == 0
    assert torch.equal(out, want)
    assert lib.sigattn_paged_fwd(ctypes.byref(p), out.data_ptr(), ws.data_ptr(), n - 1, stream) == -10
    assert lib.sigattn_paged_fwd(ctypes.byref(p), out.data_ptr(), ws.data_ptr() + 4, n, stream) == -10
    out.fill_(float("nan"))
    assert lib.sigattn_paged_fwd(ctypes.byref(p), out.data_ptr(), None, 0, stream) == 0
    assert_within(out, reference(q, rows, new, True), "uncut")


def test_python_binding(monkeypatch):
    """The Python layer's own calls equal the C++ module's."""
    from triton_sigmoid import _capi
    ctx, new = [100, 33, 900], [1, 40, 1]
    q, kc, vc, table, lens, cu, _ = make(ctx, new, 16, 6, 2, 64, torch.float16)
    k, v = (torch.randn(42, 2, 64, device="cuda").half() for _ in range(2))

    def step():
        t, a, b = table.clone(), kc.clone(), vc.clone()
        plan = ts.paged_plan(ints(ctx), ints(new), t, ints([1, 2, 3, 4]), 16, 44)
        ts.paged_cache_write(k, v, a, b, plan.slot_mapping[:42].contiguous())
        return (*plan, a, b, ts.sigmoid_attention_paged(q, kc, vc, table, lens, cu, 40, is_causal=True))

    assert _capi.autograd_node() is not None
    calls = []
    for name in ("quick_plan", "quick_write", "quick_paged"):
        whole = getattr(_capi.quick_module, name)

        def spy(*args, whole=whole, name=name):
            got = whole(*args)
            calls.append((name, got is not None and got is not False))
            return got

        monkeypatch.setattr(_capi.quick_module, name, spy)
    one = step()
    assert calls == [("quick_plan", True), ("quick_write", True), ("quick_paged", True)]
    monkeypatch.setenv("SIGATTN_EAGER_BINDING", "python")
    two = step()
    assert [took for _, took in calls[3:]] == [False] * 3
    for a, b in zip(one, two):
        assert torch.equal(a.nan_to_num(7.0) if a.is_floating_point() else a,
                           b.nan_to_num(7.0) if b.is_floating_point() else b)


@pytest.mark.parametrize("heads", [(64, 1), (48, 1), (33, 1), (40, 2)], ids=lambda h: f"{h[0]}x{h[1]}")
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_groups_of_more_heads_than_a_block(heads, dtype):
    for D in (64, 128):
        check([0, 700, 40], [1, 1, 1], 16, *heads, D, DT[dtype])
        check([100, 30], [5, 1], 16, *heads, D, DT[dtype])


def test_wide_integers():
    """int64 tables, slots and lengths; values past 32 bits are clamped: a slot
    or page there is none, not another one."""
    ctx, new = [40, 100], [1, 1]
    q, kc, vc, table, lens, cu, rows = make(ctx, new, 16, 4, 2, 64, torch.bfloat16, fill=0.0)
    wide = table.long()
    wide[0, 0] = 2 ** 32 + int(table[0, 1])
    got = ts.sigmoid_attention_paged(q, kc, vc, wide, lens.long(), cu.long(), 1)
    assert_within(got, reference(q, rows, new, False, absent=[list(range(16)), []]), "o")
    k = torch.ones(2, 2, 64, device="cuda").bfloat16()
    before = kc.clone()
    ts.paged_cache_write(k, k, kc, vc, torch.tensor([2 ** 32, -(2 ** 40)], device="cuda"))
    assert torch.equal(kc, before)
    plan = ts.paged_plan(ints([40, 100]).long(), ints(new).long(), table, ints([0]).long(), 16, 2)
    assert plan.slot_mapping.dtype == I32


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_offsets_past_32_bits(dtype):
    """A cache of more than 2^32 bytes a tensor (pages far apart): the last pages
    are written and read."""
    ps, Hkv, D, H = 16, 2, 64, 4
    pages = 9
    stride = 2 ** 29 // (1 if dtype == "bf16" else 2) + 64  # elements from page to page: 1 GiB
    buf = torch.empty(2, (pages - 1) * stride + ps * Hkv * D, dtype=DT[dtype], device="cuda")
    kc, vc = (t.as_strided((pages, ps, Hkv, D), (stride, Hkv * D, D, 1)) for t in buf)
    g = torch.Generator().manual_seed(1)
    lens, new = [70, 40], [1, 20]
    rows = [torch.randn(2, n, Hkv, D, generator=g).to(DT[dtype]).cuda() for n in lens]
    table = ints([[8, 0, 7, 5, 6], [4, 3, 1, -1, -1]])
    pos = [torch.arange(n) for n in lens]
    slots = torch.cat([table[b].cpu()[p // ps] * ps + p % ps for b, p in enumerate(pos)]).to(I32).cuda()
    k, v = (torch.cat([r[i] for r in rows]) for i in range(2))
    ts.paged_cache_write(k, v, kc, vc, slots)
    assert torch.equal(kc[8, 3], rows[0][0][3]) and torch.equal(vc[6, 5], rows[0][1][69])
    q = torch.randn(21, H, D, generator=g).to(DT[dtype]).cuda()
    got = ts.sigmoid_attention_paged(q, kc, vc, table, ints(lens), ints(offsets(new)), 20, is_causal=True)
    assert_within(got, reference(q, rows, new, True), "o")
    got = ts.sigmoid_attention_paged(q[:2], kc, vc, table, ints(lens), ints([0, 1, 2]), 1)
    assert_within(got, reference(q[:2], rows, [1, 1], False), "o")


def test_two_calls_at_once_on_one_cache():
    """Attention on two streams at once, of other sequences of one cache."""
    ctx, new = [2000, 100, 900, 50], [1, 30, 1, 30]
    q, kc, vc, table, lens, cu, rows = make(ctx, new, 16, 8, 2, 64, torch.bfloat16)
    at = offsets(new)
    halves = [(slice(0, 2), slice(0, at[2])), (slice(2, 4), slice(at[2], at[4]))]
    want = [ts.sigmoid_attention_paged(q[r], kc, vc, table[b], lens[b], ints(offsets(new[b])), 30, is_causal=True)
            for b, r in halves]
    cus = [ints(offsets(new[b])) for b, _ in halves]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for s, (b, r), c in zip(streams, halves, cus):
            with torch.cuda.stream(s):
                got.append(ts.sigmoid_attention_paged(q[r], kc, vc, table[b], lens[b], c, 30, is_causal=True))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("binding", ["node", "python"])
def test_tangents_are_refused(monkeypatch, binding):
    """Canonical arguments too: the C++ module leaves a dual tensor to the
    Python layer, which refuses it, also under no_grad."""
    if binding == "python":
        monkeypatch.setenv("SIGATTN_EAGER_BINDING", "python")
    q, kc, vc, table, lens, cu, _ = make([20, 5], [1, 3], 16, 4, 2, 64, torch.bfloat16, fill=0.0)
    mod = torch.zeros(2, table.shape[1] * 16, device="cuda")
    rows = torch.randn(4, 2, 64, device="cuda").bfloat16()
    before = kc.clone(), vc.clone()
    with forward_ad.dual_level():
        for i in range(4):
            a = [q, kc, vc, mod]
            a[i] = forward_ad.make_dual(a[i], torch.ones_like(a[i]))
            for call in (ts.sigmoid_attention_paged, torch.no_grad()(ts.sigmoid_attention_paged)):
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call(a[0], a[1], a[2], table, lens, cu, 3, score_mod=a[3])
            w = [rows, rows, kc, vc]
            w[i] = forward_ad.make_dual(w[i], torch.ones_like(w[i]))
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                ts.paged_cache_write(*w, ints([0, 1, 2, 3]))
        # Without a tangent the calls run inside a dual level as outside.
        got = ts.sigmoid_attention_paged(q, kc, vc, table, lens, cu, 3, score_mod=mod)
    assert torch.equal(got, ts.sigmoid_attention_paged(q, kc, vc, table, lens, cu, 3, score_mod=mod))
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])


@pytest.mark.parametrize("heads", [(4, 1), (4, 2)], ids=lambda h: f"{h[0]}x{h[1]}")
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_as_many_chunks_as_a_sequence_takes(dtype, heads):
    """Contexts whose chunks of the least length would be more than are summed:
    longer ones (24576 keys and more, for one sequence or two)."""
    for ctx in ([29999], [65900], [40001, 27]):
        check(ctx, [1] * len(ctx), 64, *heads, 64, DT[dtype])
    check([26000], [5], 128, *heads, 128, DT[dtype], causal=False, mod=True)


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 3]], ids=["decode", "chunk"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_tables_of_many_keys(dtype, new):
    """A table row that can hold 2^23 keys (lengths that floats hold no longer
    exactly), for short sequences and one that passes a page of 2^20."""
    ps, H, Hkv, D = 1 << 20, 4, 1, 32
    lens = [3000, 77, ps + 513]
    g = torch.Generator(device="cuda").manual_seed(8)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda").to(DT[dtype])  # noqa: E731
    rows = [normal(2, n, Hkv, D) for n in lens]
    caches = torch.full((2, 5, ps, Hkv, D), float("nan"), dtype=DT[dtype], device="cuda")
    pages = [[3], [0], [4, 2]]
    for r, p in zip(rows, pages):
        for j, page in enumerate(p):
            part = r[:, j * ps:(j + 1) * ps]
            caches[:, page, :part.shape[1]] = part
    q = normal(sum(new), H, D)
    for width in (2, 8, 13):
        table = ints([p + [-1] * (width - len(p)) for p in pages])
        got = ts.sigmoid_attention_paged(q, caches[0], caches[1], table, ints(lens), ints(offsets(new)), max(new),
                                         is_causal=True)
        assert_within(got, reference(q, rows, new, True), f"{width} pages a row")


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_rows_off_16_bytes(dtype, D, causal):
    """Caches off a 16-byte boundary take the portable kernel: a term per key,
    pages that are not there, rows of no sequence and a sequence without keys."""
    ctx, new, ps = [100, 33, 0, 700], [1, 20, 3, 2], 32
    q, kc, vc, table, lens, cu, rows = make(ctx, new, ps, 6, 2, D, DT[dtype], fill=0.0)

    def off(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        buf[1:] = t.reshape(-1)
        return buf[1:].view(t.shape)

    table[0, 1], table[3, 0], table[3, 5] = -1, kc.shape[0], 2 ** 31 - 1
    absent = [list(range(32, 64)), [], [], [*range(32), *range(160, 192)]]
    mod = torch.randn(4, table.shape[1] * ps, generator=torch.Generator().manual_seed(7)).cuda()
    mod[:, 3], mod[3, 100] = -torch.inf, torch.finfo(torch.float32).min
    more = torch.cat([q, q[:9]])
    for term in (None, mod):
        got = ts.sigmoid_attention_paged(more, off(kc), off(vc), table, lens, cu, 20, is_causal=causal, score_mod=term)
        assert_within(got[:sum(new)], reference(q, rows, new, causal, term, absent=absent), "o")
        assert not got[sum(new):].any()
    got = ts.sigmoid_attention_paged(q, off(kc), off(vc), table, ints([0, 53, 0, -5]), cu, 20, is_causal=causal)
    assert got[1:21].any() and not got[:1].any() and not got[21:].any()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [16, 32])
def test_terms_per_key_of_small_heads(D, dtype):
    for shape in ("decode", "few", "chunk", "mixed", "long"):
        ctx, new = SHAPES[shape]
        check(ctx, new, 16, 8, 2, D, DT[dtype], mod=True)
        check(ctx, new, 32, 6, 3, D, DT[dtype], causal=False, mod=True, sigmoid_bias=-2.0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_cuts_among_more_lengths_than_are_kept(dtype):
    """Batches of more than 256 sequences (whose lengths the waves hold) that are
    cut: decoding, chunks, and both."""
    r = random.Random(21)
    ctx = [r.choice((0, 1, 17, r.randint(0, 300), r.randint(0, 900))) for _ in range(300)]
    ctx[290], ctx[3] = 2600, 1500
    check(ctx, [1] * 300, 16, 4, 2, 32, DT[dtype])
    new = [r.choice((0, 1, 1, 1, 2)) for _ in ctx]
    new[290], new[270] = 40, 20
    check(ctx, new, 32, 4, 1, 64, DT[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_graphs_of_one_pool(dtype):
    """Two captured calls whose workspaces lie in one pool, replayed in turn on
    changing lengths: each equals the eager call."""
    sets = [make([3000, 50, 900], [1, 1, 1], 16, 8, 2, 64, DT[dtype], 1),
            make([1500, 2500], [40, 1], 16, 8, 2, 64, DT[dtype], 2)]
    longest, calls = (1, 40), []
    call = lambda i: ts.sigmoid_attention_paged(*sets[i][:6], longest[i], is_causal=True)  # noqa: E731
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call(0), call(1)
    side.synchronize()
    pool = None
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = call(i)
        pool = graph.pool()
        calls.append((graph, out))
    for cut in (0, 700, 1234):
        for i in (0, 1, 1, 0):
            lens = sets[i][4]
            whole = lens.clone()
            lens.sub_(cut).clamp_(min=longest[i])
            calls[i][0].replay()
            torch.cuda.synchronize()
            have = calls[i][1].clone()
            assert torch.equal(have, call(i))
            lens.copy_(whole)
