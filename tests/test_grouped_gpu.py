"""Grouped heads in packed sequences (sigmoid_attention_varlen with fewer
key/value heads than query heads) against the formulas in 64 bits."""

import os

import pytest
import torch

import triton_sigmoid as ts
from reference64 import assert_within, packed
from triton_sigmoid import _capi

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def offsets(lens, first=0):
    at = [first]
    for n in lens:
        at.append(at[-1] + n)
    return at


def make(rows_q, rows_k, H, Hkv, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)

    def normal(rows, heads):
        return torch.randn(rows, heads, D, generator=g).to(dtype).cuda()

    return normal(rows_q, H), normal(rows_k, Hkv), normal(rows_k, Hkv), normal(rows_q, H)


def run(q, k, v, do, cu_q, cu_k, **kw):
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    cq, ck = (torch.tensor(c, dtype=torch.int32, device="cuda") for c in (cu_q, cu_k))
    o = ts.sigmoid_attention_varlen(q, k, v, cq, ck, **kw)
    return dict(zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, (q, k, v), do))))


def check(q, k, v, do, cu_q, cu_k, causal, mod=None, **kw):
    got = run(q, k, v, do, cu_q, cu_k, is_causal=causal, score_mod=mod, **kw)
    want = packed(q, k, v, do, cu_q, cu_k, causal, mod)
    for x in got:
        assert_within(got[x], want[x], x)
    return got


LENS = {
    "one": [1],
    "short": [1, 0, 31, 32, 33],
    "odd": [63, 200, 0, 129, 1, 64],
    "block": [128, 256],
    "long": [515, 1, 1030],
}


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("heads", [(4, 2), (6, 2), (8, 1), (7, 7)], ids=lambda h: f"{h[0]}x{h[1]}")
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lens", ["one", "short", "odd", "long"])
def test_against_64_bits(lens, dtype, D, heads, causal):
    n = LENS[lens]
    if lens == "long" and (D in (16, 32) or heads == (7, 7)):
        n = [515]
    cu = offsets(n)
    q, k, v, do = make(cu[-1], cu[-1], *heads, D, DT[dtype])
    check(q, k, v, do, cu, cu, causal)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_score_mod_and_other_key_lengths(dtype, D):
    """Queries and keys of different lengths, a sequence without keys, a term
    per key with -inf (a masked key) in it."""
    nq, nk = [40, 3, 0, 130], [77, 0, 5, 300]
    cq, ck = offsets(nq), offsets(nk)
    q, k, v, do = make(cq[-1], ck[-1], 6, 3, D, DT[dtype], 1)
    mod = torch.randn(ck[-1], generator=torch.Generator().manual_seed(2)).cuda()
    mod[5], mod[-1] = -torch.inf, -torch.inf
    for causal in (False, True):
        check(q, k, v, do, cq, ck, causal, mod)


@pytest.mark.parametrize("D", [64, 128])
def test_rows_outside_every_sequence_are_zero(D):
    cu = offsets([70, 0, 33], first=5)
    q, k, v, do = make(cu[-1] + 9, cu[-1] + 9, 4, 2, D, torch.bfloat16, 3)
    got = check(q, k, v, do, cu, cu, True)
    for x in got.values():
        assert not x[:5].any() and not x[cu[-1]:].any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_more_sequences_than_the_ordered_batches(dtype):
    n = [(7 * i) % 41 for i in range(90)]
    cu = offsets(n)
    q, k, v, do = make(cu[-1], cu[-1], 8, 2, 64, DT[dtype], 4)
    check(q, k, v, do, cu, cu, True)
    q, k, v, do = make(cu[-1], cu[-1], 4, 1, 128, DT[dtype], 5)
    check(q, k, v, do, cu, cu, True)


@pytest.mark.parametrize("D", [32, 128])
def test_rows_off_16_bytes(D):
    """Tensors that start off a 16-byte boundary take the portable kernels."""
    cu = offsets([33, 0, 70])
    q, k, v, do = make(cu[-1], cu[-1], 6, 2, D, torch.float16, 6)

    def off(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        buf[1:] = t.reshape(-1)
        return buf[1:].view(t.shape)

    check(off(q), off(k), off(v), off(do), cu, cu, True)


def test_strided_inputs():
    cu = offsets([50, 90])
    q, k, v, do = make(cu[-1], cu[-1], 4, 2, 64, torch.bfloat16, 7)
    wide = torch.cat([q, k, v], dim=1)  # a fused projection's output
    got = run(wide[:, :4], wide[:, 4:6], wide[:, 6:], do, cu, cu, is_causal=True)
    same = run(q, k, v, do, cu, cu, is_causal=True)
    for x in got:
        assert torch.equal(got[x], same[x])


@pytest.mark.parametrize("binding", ["node", "python"])
@pytest.mark.parametrize("mb", ["0", "1", "2048"])
def test_backward_workspace_limits(monkeypatch, mb, binding):
    """The two-pass backward in whole groups of heads, and without a workspace."""
    monkeypatch.setenv("SIGATTN_BWD_WORKSPACE_MB", mb)
    if binding == "python":
        monkeypatch.setenv("SIGATTN_EAGER_BINDING", "python")
    cu = offsets([300, 700])
    q, k, v, do = make(cu[-1], cu[-1], 6, 2, 128, torch.bfloat16, 8)
    check(q, k, v, do, cu, cu, True)


def test_workspace_of_one_head_runs_without_it():
    """A dS workspace below one group of heads: the library recomputes."""
    cu = offsets([256, 256])
    q, k, v, do = make(cu[-1], cu[-1], 4, 2, 128, torch.bfloat16, 9)
    cut = torch.tensor(cu, dtype=torch.int32, device="cuda")
    scale = torch.tensor(128 ** -0.5, device="cuda")
    bias = -torch.log(torch.full((2,), 256.0, device="cuda"))
    pr = _capi._problem(q, k, v, bias, None, scale, None, None, True, packed=(cut, cut, 256, 256))
    lib = _capi.load_library()
    import ctypes
    full = lib.sigattn_bwd_workspace_bytes(ctypes.byref(pr))
    want = packed(q, k, v, do, cu, cu, True)
    stream = torch.cuda.current_stream().cuda_stream
    for share in (4, 3, 2, 1):  # of four heads: one, one, one group, two groups
        n = full // share
        ws = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
        g = [torch.full_like(t, float("nan")) for t in (q, k, v)]
        rc = lib.sigattn_bwd_ws(ctypes.byref(pr), do.data_ptr(), *(t.data_ptr() for t in g), ws.data_ptr(), n, stream)
        assert rc == 0
        for x, t in zip(("dq", "dk", "dv"), g):
            assert_within(t, want[x], f"{x}, workspace of {n}")


def test_equals_repeated_heads():
    """The same as each query head with a copy of its key/value head: O and dQ
    bit for bit, dK and dV within the bounds of the sum."""
    cu = offsets([100, 400])
    q, k, v, do = make(cu[-1], cu[-1], 8, 2, 128, torch.bfloat16, 10)
    got = run(q, k, v, do, cu, cu, is_causal=True)
    rep = run(q, k.repeat_interleave(4, 1), v.repeat_interleave(4, 1), do, cu, cu, is_causal=True)
    assert torch.equal(got["o"], rep["o"]) and torch.equal(got["dq"], rep["dq"])


def test_deterministic_and_on_another_stream():
    cu = offsets([333, 5, 600])
    q, k, v, do = make(cu[-1], cu[-1], 8, 2, 64, torch.float16, 11)
    one = run(q, k, v, do, cu, cu, is_causal=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        two = run(q, k, v, do, cu, cu, is_causal=True)
    side.synchronize()
    for x in one:
        assert torch.equal(one[x], two[x])


@pytest.mark.parametrize("D", [64, 128])
def test_captured_forward_and_backward(D):
    cu = offsets([130, 77])
    q, k, v, do = make(cu[-1], cu[-1], 4, 2, D, torch.bfloat16, 12)
    cut = torch.tensor(cu, dtype=torch.int32, device="cuda")

    def step():
        a, b, c = (t.detach().requires_grad_(True) for t in (q, k, v))
        o = ts.sigmoid_attention_varlen(a, b, c, cut, cut, 130, 130, is_causal=True)
        return (o.detach(), *torch.autograd.grad(o, (a, b, c), do))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        for t, new in zip((q, k, v, do), make(cu[-1], cu[-1], 4, 2, D, torch.bfloat16, 20 + seed)):
            t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_gradients_against_differences():
    """fp32 gradients against central differences of the 64-bit forward."""
    cu = offsets([9, 14])
    q, k, v, do = make(cu[-1], cu[-1], 4, 2, 32, torch.float32, 13)
    got = run(q, k, v, do, cu, cu, is_causal=True)
    step = 1e-4

    def loss(a, b, c):
        return (packed_value(a, b, c) * do.double()).sum()

    def packed_value(a, b, c):
        from reference64 import one_head
        o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        import math
        for x, y in zip(cu[:-1], cu[1:]):
            for h in range(4):
                o[x:y, h] = one_head(a[x:y, h], b[x:y, h // 2], c[x:y, h // 2], None, -math.log(y - x),
                                     torch.float32, 0)["o"][0]
        return o

    args = [t.double() for t in (q, k, v)]
    g = torch.Generator().manual_seed(14)
    for i, x in enumerate(("dq", "dk", "dv")):
        d = torch.randn(args[i].shape, generator=g, dtype=torch.float64).cuda()
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + step * d, args[i] - step * d
        want = (loss(*hi) - loss(*lo)) / (2 * step)
        have = (got[x].double() * d).sum()
        # fp32 sums of a few thousand terms of size one; the differences' own
        # error is step^2 of the third derivative.
        size = (got[x].double() * d).abs().sum()
        assert abs(have - want) <= 1e-5 * size + 1e-6


def test_compiled_forward_and_backward():
    cu = offsets([60, 100])
    q, k, v, do = make(cu[-1], cu[-1], 4, 2, 64, torch.bfloat16, 15)
    cut = torch.tensor(cu, dtype=torch.int32, device="cuda")

    def fn(a, b, c):
        return ts.sigmoid_attention_varlen(a, b, c, cut, cut, 100, 100, is_causal=True)

    want = run(q, k, v, do, cu, cu, is_causal=True)
    a, b, c = (t.detach().requires_grad_(True) for t in (q, k, v))
    o = torch.compile(fn, fullgraph=True)(a, b, c)
    got = dict(zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, (a, b, c), do))))
    for x in got:
        assert torch.equal(got[x], want[x])


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("heads", [(6, 2), (10, 2), (16, 1)], ids=lambda h: f"{h[0]}x{h[1]}")
def test_head_split_parts(heads, D, causal):
    """Few K / V heads: their groups run in parts whose sums are added; rows
    outside every sequence stay zero, and the parts' workspace may hold anything."""
    cu = offsets([140, 0, 300], first=3)
    q, k, v, do = make(cu[-1] + 7, cu[-1] + 7, *heads, D, torch.bfloat16, 16)
    junk = torch.full((64 << 20,), float("nan"), device="cuda")
    del junk  # the allocator hands it out again
    got = check(q, k, v, do, cu, cu, causal)
    for x in got.values():
        assert not x[:3].any() and not x[cu[-1]:].any()
    same = run(q, k, v, do, cu, cu, is_causal=causal)
    for x in got:
        assert torch.equal(got[x], same[x])


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("heads", [(10, 2), (16, 1)], ids=lambda h: f"{h[0]}x{h[1]}")
def test_head_split_parts_of_fp32(heads, D, causal):
    """As above, on the fp32 kernels; values past what their splits hold take
    the exact products, in parts too."""
    cu = offsets([140, 0, 300], first=3)
    q, k, v, do = make(cu[-1] + 7, cu[-1] + 7, *heads, D, torch.float32, 18)
    junk = torch.full((64 << 20,), float("nan"), device="cuda")
    del junk
    got = check(q, k, v, do, cu, cu, causal)
    for x in got.values():
        assert not x[:3].any() and not x[cu[-1]:].any()
    same = run(q, k, v, do, cu, cu, is_causal=causal)
    for x in got:
        assert torch.equal(got[x], same[x])
    small = do.clone()
    small[3:143] *= 1e-30
    check(q, k, v, small, cu, cu, causal)


def test_head_split_asks_for_its_workspace():
    import ctypes
    cut = torch.tensor([0, 256, 400], dtype=torch.int32, device="cuda")
    lib = _capi.load_library()
    for D, entry in ((64, "split"), (128, "ws")):
        q, k, v, do = make(400, 400, 8, 2, D, torch.float16, 17)
        scale, bias = torch.tensor(0.1, device="cuda"), torch.zeros(2, device="cuda")
        pr = _capi._problem(q, k, v, bias, None, scale, None, None, True, packed=(cut, cut, 256, 256))
        size = lib.sigattn_bwd_split_workspace_bytes if entry == "split" else lib.sigattn_bwd_workspace_bytes
        call = lib.sigattn_bwd_split if entry == "split" else lib.sigattn_bwd_ws
        n = size(ctypes.byref(pr))
        parts = 4 * 2 * 400 * 2 * D * 4  # a head each
        assert n > parts if entry == "ws" else n == parts
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        g = [torch.full_like(t, float("nan")) for t in (q, k, v)]
        args = (ctypes.byref(pr), do.data_ptr(), *(t.data_ptr() for t in g), ws.data_ptr())
        stream = torch.cuda.current_stream().cuda_stream
        want = packed(q, k, v, do, cut.tolist(), cut.tolist(), True, bias=0.0, scale=float(scale))
        for nbytes in (n, n - 16):
            rc = call(*args, nbytes, stream)
            if entry == "split" and nbytes < n:
                assert rc == -10
                continue
            assert rc == 0  # ws: without room for the parts the groups run whole
            for x, t in zip(("dq", "dk", "dv"), g):
                assert_within(t, want[x], x)


def test_short_way_of_eager_calls(monkeypatch):
    """Canonical eager calls go straight to the C++ node, with the same results
    and refusals as the Python layer's."""
    assert _capi.autograd_node() is not None
    cu = offsets([30, 0, 70])
    q, k, v, do = make(cu[-1], cu[-1], 4, 2, 64, torch.bfloat16, 18)
    whole, took = _capi.quick_module.quick_varlen, []

    def spy(*args):
        got = whole(*args)
        took.append(got is not None)
        return got

    monkeypatch.setattr(_capi.quick_module, "quick_varlen", spy)
    mod = torch.randn(cu[-1], device="cuda")
    for kw in (dict(), dict(score_mod=mod), dict(scale=0.3, sigmoid_bias=-2.0)):
        given = run(q, k, v, do, cu, cu, max_seqlen_q=70, max_seqlen_k=70, is_causal=True, **kw)
        assert took.pop()
        monkeypatch.setenv("SIGATTN_EAGER_BINDING", "python")
        same = run(q, k, v, do, cu, cu, max_seqlen_q=70, max_seqlen_k=70, is_causal=True, **kw)
        monkeypatch.delenv("SIGATTN_EAGER_BINDING")
        assert not took.pop()
        for x in given:
            assert torch.equal(given[x], same[x])
    cut = torch.tensor(cu, device="cuda", dtype=torch.int32)
    with pytest.raises(ValueError, match="heads mismatch"):
        ts.sigmoid_attention_varlen(q[:, :3].contiguous(), k, v, cut, cut, 70, 70)
    with pytest.raises(ValueError, match="non-negative"):
        ts.sigmoid_attention_varlen(q, k, v, cut, cut, -1, 70)
    run(q.float(), k.float(), v.float(), do.float(), cu, cu)  # no longest lengths: the Python layer reads them
    assert not took.pop()


# Few queries on many keys, not causal: the split-KV forward.  Its forms: waves
# that share a chunk, with parts to add or one chunk each; a wave for each chunk,
# with one each, cut by the lengths, or (more sequences than a wave has lanes)
# of one length.  (lengths, heads, bytes of partials a call asks for: none or some)
SHORT_QUERIES = {
    "shared": ([1, 0, 17, 32], [900, 300, 0, 2000], (8, 2), True),
    "shared, three to a head": ([5, 2], [700, 1500], (6, 2), True),
    "shared, one chunk": ([3] * 40, [(37 * i) % 257 for i in range(39)] + [256], (16, 2), False),
    "wave each, one chunk": ([1 + i % 2 for i in range(130)], [(53 * i) % 401 for i in range(129)] + [400], (16, 4),
                             False),
    "wave each, cut": ([1, 8, 0, 5], [16000, 17, 400, 9000], (16, 1), True),
    "wave each, one length": ([1 + i % 3 for i in range(70)], [(97 * i) % 1031 for i in range(69)] + [1031], (6, 2),
                              True),
}


@pytest.mark.parametrize("mod", [False, True], ids=["plain", "terms"])
@pytest.mark.parametrize("dtype, D", [("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("shape", list(SHORT_QUERIES))
def test_short_queries_on_long_keys(shape, dtype, D, mod):
    import ctypes
    nq, nk, heads, parts = SHORT_QUERIES[shape]
    cq, ck = offsets(nq), offsets(nk)
    q, k, v, do = make(cq[-1], ck[-1], *heads, D, DT[dtype], 30)
    term = None
    if mod:
        term = torch.randn(ck[-1], generator=torch.Generator().manual_seed(31)).cuda()
        term[5], term[-1] = -torch.inf, torch.finfo(torch.float32).min
    check(q, k, v, do, cq, ck, False, term)
    cut = [torch.tensor(c, dtype=torch.int32, device="cuda") for c in (cq, ck)]
    pr = _capi._problem(q, k, v, torch.zeros(len(nq), device="cuda"), term, torch.tensor(1.0, device="cuda"), None, None,
                        False, packed=(*cut, max(nq), max(nk)))
    assert (_capi.load_library().sigattn_fwd_decode_workspace_bytes(ctypes.byref(pr)) > 0) == parts


def test_gradients_of_repeated_heads_add_up():
    """dK and dV of a shared head are the sums of those of its copies: within
    the group's bound and those of the copies, each rounded once."""
    cu = offsets([100, 400])
    for D in (64, 128):
        q, k, v, do = make(cu[-1], cu[-1], 8, 2, D, torch.bfloat16, 10)
        got = run(q, k, v, do, cu, cu, is_causal=True)
        rk, rv = k.repeat_interleave(4, 1), v.repeat_interleave(4, 1)
        rep = run(q, rk, rv, do, cu, cu, is_causal=True)
        bound, each = packed(q, k, v, do, cu, cu, True), packed(q, rk, rv, do, cu, cu, True)
        for x in ("dk", "dv"):
            total = rep[x].double().unflatten(1, (2, 4)).sum(2)
            assert_within(got[x], (total, bound[x][1] + each[x][1].unflatten(1, (2, 4)).sum(2)), x)


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_two_pass_backward_in_several_passes(dtype, causal):
    """The dS of some K / V heads at a time: workspaces of one query head (none:
    recomputed), of one group, of two, of three (passes of two then), of all four,
    and of all with the parts of a head split behind them."""
    import ctypes
    lens = [300, 77, 0, 513]
    H, Hkv, D, G = 12, 4, 128, 3
    cu = offsets(lens)
    q, k, v, do = make(cu[-1], cu[-1], H, Hkv, D, DT[dtype], 32)
    cut = torch.tensor(cu, dtype=torch.int32, device="cuda")
    bias = -torch.log(torch.tensor(lens, device="cuda").clamp(min=1).float())
    scale = torch.tensor(D ** -0.5, device="cuda")  # (the problem holds addresses alone)
    pr = _capi._problem(q, k, v, bias, None, scale, None, None, causal, packed=(cut, cut, 513, 513))
    lib, blocks = _capi.load_library(), -(-513 // 32)
    per_head = len(lens) * (blocks * (blocks + 1) // 2 if causal else blocks * blocks) * 2048
    full = lib.sigattn_bwd_workspace_bytes(ctypes.byref(pr))
    assert full > H * per_head
    want = packed(q, k, v, do, cu, cu, causal)
    stream = torch.cuda.current_stream().cuda_stream
    for n in (per_head, G * per_head, 2 * G * per_head, 3 * G * per_head + 16, H * per_head, full):
        ws = torch.full((n // 4,), float("nan"), device="cuda")
        g = [torch.full_like(t, float("nan")) for t in (q, k, v)]
        rc = lib.sigattn_bwd_ws(ctypes.byref(pr), do.data_ptr(), *(t.data_ptr() for t in g), ws.data_ptr(), n, stream)
        assert rc == 0
        for x, t in zip(("dq", "dk", "dv"), g):
            assert_within(t, want[x], f"{x}, workspace of {n / per_head:.2f} heads")


@pytest.mark.parametrize("binding", ["node", "python"])
def test_backward_past_the_workspace_limit(monkeypatch, binding):
    """A training step whose dS is over the limit runs in passes of whole K / V
    heads, through either binding."""
    import ctypes
    monkeypatch.setenv("SIGATTN_BWD_WORKSPACE_MB", "180")
    if binding == "python":
        monkeypatch.setenv("SIGATTN_EAGER_BINDING", "python")
    lens = [1024 + (i % 5 - 2) * 38 for i in range(34)]
    cu = offsets(lens)
    q, k, v, do = make(cu[-1], cu[-1], 8, 4, 128, torch.bfloat16, 33)
    cut = torch.tensor(cu, dtype=torch.int32, device="cuda")
    pr = _capi._problem(q, k, v, torch.zeros(len(lens), device="cuda"), None, torch.tensor(1.0, device="cuda"), None,
                        None, True, packed=(cut, cut, max(lens), max(lens)))
    lib = _capi.load_library()
    full, size = lib.sigattn_bwd_workspace_bytes(ctypes.byref(pr)), _capi.bwd_workspace_bytes(lib, pr, q.device)
    assert 0 < size <= 180 << 20 < full
    check(q, k, v, do, cu, cu, True)


def test_dense_and_padded_tensors_as_packed_ones():
    """[B, T, H, D] tensors with grouped heads through views and the valid rows."""
    B, T, H, Hkv, D = 3, 70, 4, 2, 64
    q, k, v, do = make(B * T, B * T, H, Hkv, D, torch.bfloat16, 34)
    cu = torch.arange(0, (B + 1) * T, T, dtype=torch.int32, device="cuda")
    leaves = [t.view(B, T, -1, D).requires_grad_(True) for t in (q.clone(), k.clone(), v.clone())]
    a, b, c = leaves
    out = ts.sigmoid_attention_varlen(a.flatten(0, 1), b.flatten(0, 1), c.flatten(0, 1), cu, cu, T, T,
                                      is_causal=True).view_as(a)
    got = dict(zip(("o", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, do.view_as(out)))))
    want = packed(q, k, v, do, cu.tolist(), cu.tolist(), True)
    for x in got:
        assert_within(got[x].flatten(0, 1), want[x], x)
    lens = torch.tensor([70, 0, 33], device="cuda")
    valid = torch.arange(T, device="cuda") < lens[:, None]
    cu = torch.nn.functional.pad(lens.cumsum(0, dtype=torch.int32), (1, 0))
    out = torch.zeros_like(a).masked_scatter(valid[..., None, None], ts.sigmoid_attention_varlen(
        a[valid], b[valid], c[valid], cu, cu, T, T, is_causal=True))
    got = dict(zip(("o", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, do.view_as(out)))))
    rows = valid.flatten()
    want = packed(q[rows], k[rows], v[rows], do[rows], cu.tolist(), cu.tolist(), True)
    for x in got:
        assert_within(got[x].flatten(0, 1)[rows], want[x], x)
        assert not got[x].flatten(0, 1)[~rows].any()


def test_large_ragged_grids():
    """Not causal, D = 64, eight row blocks a compute unit: dQ beside dK/dV on a
    second stream; with few K / V heads their groups in parts there."""
    for heads, lens in (((16, 4), [512 - 7 * i for i in range(34)]), ((64, 1), [400, 1, 0, 257, 512, 130, 511, 300, 64])):
        cu = offsets(lens)
        q, k, v, do = make(cu[-1], cu[-1], *heads, 64, torch.float16, 35)
        units = torch.cuda.get_device_properties(0).multi_processor_count
        assert len(lens) * heads[0] * (512 // 128) >= 8 * units
        got = check(q, k, v, do, cu, cu, False)
        same = run(q, k, v, do, cu, cu, is_causal=False)
        for x in got:
            assert torch.equal(got[x], same[x])


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_fp32_of_many_blocks(D, causal):
    """Grids from a workgroup per compute unit on, where fewer waves share rows;
    lengths that end inside a block, and short ones between them."""
    for heads, lens in (((32, 8), [700, 5, 513, 640, 128, 0, 699, 1]), ((12, 6), [130] * 70)):
        cu = offsets(lens)
        q, k, v, do = make(cu[-1], cu[-1], *heads, D, torch.float32, 36)
        check(q, k, v, do, cu, cu, causal)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_off_16_bytes_in_other_types(dtype):
    cu = offsets([33, 0, 70, 200])
    q, k, v, do = make(cu[-1], cu[-1], 6, 2, 64, DT[dtype], 37)
    mod = torch.randn(cu[-1], generator=torch.Generator().manual_seed(38)).cuda()
    mod[7] = -torch.inf

    def off(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        buf[1:] = t.reshape(-1)
        return buf[1:].view(t.shape)

    for causal in (False, True):
        check(off(q), off(k), off(v), off(do), cu, cu, causal, mod)


@pytest.mark.parametrize("D", [64, 128])
def test_training_steps_on_two_streams(D):
    """Two grouped steps at once, each on a stream of its own and with the parts of
    its groups in a workspace of its own: as one after the other."""
    cus, data, want = [offsets([300, 70, 512]), offsets([411, 0, 200])], [], []
    for i, cu in enumerate(cus):
        data.append(make(cu[-1], cu[-1], 16, 2, D, torch.bfloat16, 40 + i))
        want.append(run(*data[i], cu, cu, max_seqlen_q=512, max_seqlen_k=512, is_causal=True))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for s, d, cu in zip(streams, data, cus):
            with torch.cuda.stream(s):
                got.append(run(*d, cu, cu, max_seqlen_q=512, max_seqlen_k=512, is_causal=True))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for x in a:
                assert torch.equal(a[x], b[x])
