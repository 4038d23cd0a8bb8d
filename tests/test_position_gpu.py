"""The learned bias by relative position, in packed sequences (forward, backward
and the table's gradient) and over a paged cache, against its definition in 64 bits."""

import math
import random

import pytest
import torch

import triton_sigmoid as ts
from reference64 import assert_within, one_head
from reference64_rel import grad_of_scores, line_of, packed_rel

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
I32 = torch.int32


def ints(v):
    return torch.tensor(v, dtype=I32, device="cuda")


def offsets(lens, first=0):
    at = [first]
    for n in lens:
        at.append(at[-1] + n)
    return at


def randn(g, *shape, dtype, f=1.0):
    return (f * torch.randn(shape, generator=g)).to(dtype).cuda()


def make(lens_q, lens_k, H, Hkv, D, dtype, num, R, seed=0, table_dtype=None, first=0, rest=0):
    g = torch.Generator().manual_seed(seed)
    nq, nk = first + sum(lens_q) + rest, first + sum(lens_k) + rest
    q, do = (randn(g, nq, H, D, dtype=dtype) for _ in range(2))
    k, v = (randn(g, nk, Hkv, D, dtype=dtype) for _ in range(2))
    table = randn(g, num, H, dtype=table_dtype or dtype, f=2.0)
    buckets = torch.randint(0, num, (2 * R + 1,), generator=g).to(I32).cuda()
    return q, k, v, do, table, buckets, offsets(lens_q, first), offsets(lens_k, first)


def run(q, k, v, do, table, buckets, cu_q, cu_k, causal, bias=None, mq=None, mk=None):
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, table)]
    mq = max(b - a for a, b in zip(cu_q, cu_q[1:])) if mq is None else mq
    mk = max(b - a for a, b in zip(cu_k, cu_k[1:])) if mk is None else mk
    o = ts.sigmoid_attention_varlen(*leaves[:3], ints(cu_q), ints(cu_k), mq, mk, is_causal=causal, sigmoid_bias=bias,
                                    bias_table=leaves[3], bias_buckets=buckets)
    return dict(zip(("o", "dq", "dk", "dv", "dtable"), (o, *torch.autograd.grad(o, leaves, do))))


def check(args, causal, bias=None):
    got = run(*args, causal, bias)
    want = packed_rel(*args, causal, bias)
    for x in want:
        assert_within(got[x], want[x], x)
    return got


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_types_and_head_dims(dtype, D, causal):
    lens = [131, 1, 70, 0, 33]
    check(make(lens, lens, 4, 2, D, DT[dtype], 8, 20, seed=D), causal)


@pytest.mark.parametrize("R", [0, 1, 7, 31, 32, 33, 64, 128, 300, 2048])
@pytest.mark.parametrize("causal", [False, True])
def test_reaches(R, causal):
    lens = [290, 65]
    check(make(lens, lens, 2, 2, 64, torch.bfloat16, 11, R, seed=R), causal)


@pytest.mark.parametrize("dtype, D", [("bf16", 64), ("f16", 128), ("f32", 64), ("bf16", 32)])
@pytest.mark.parametrize("R", [1000, 2048])
def test_far_reaches(R, dtype, D):
    check(make([2150, 70], [2150, 70], 1, 1, D, DT[dtype], 40, R, seed=R), False)


@pytest.mark.parametrize("num", [1, 2, 255, 256, 257, 700, 4096])
def test_numbers_of_buckets(num):
    check(make([150, 40], [150, 40], 2, 1, 32, torch.float16, num, 200, seed=num), False)


@pytest.mark.parametrize("H, Hkv", [(1, 1), (3, 1), (8, 8), (12, 4), (16, 1), (6, 2)])
@pytest.mark.parametrize("D", [64, 128])
def test_heads(H, Hkv, D):
    lens = [100, 200, 37]
    check(make(lens, lens, H, Hkv, D, torch.bfloat16, 16, 50, seed=H), True)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 513])
@pytest.mark.parametrize("dtype, D", [("bf16", 64), ("f16", 128), ("f32", 64), ("bf16", 32)])
def test_lengths(n, dtype, D):
    for causal in (False, True):
        check(make([n], [n], 2, 2, D, DT[dtype], 12, 40, seed=n), causal)


@pytest.mark.parametrize("dtype, D", [("bf16", 64), ("f16", 128), ("f32", 32), ("bf16", 16)])
@pytest.mark.parametrize("causal", [False, True])
def test_keys_of_other_lengths(dtype, D, causal):
    """Positions count from both starts; sequences without queries or without keys."""
    check(make([5, 150, 0, 40, 70], [200, 30, 17, 0, 71], 4, 2, D, DT[dtype], 12, 40, seed=D), causal)


@pytest.mark.parametrize("dtype, D", [("bf16", 64), ("bf16", 128), ("f32", 64)])
def test_long_sequences(dtype, D):
    lens = [1500, 777]
    check(make(lens, lens, 2, 1, D, DT[dtype], 32, 128, seed=3), True)
    check(make(lens, lens, 2, 2, D, DT[dtype], 32, 128, seed=4), False)


@pytest.mark.parametrize("dtype, D", [("bf16", 64), ("f16", 128), ("f32", 64), ("f16", 32)])
def test_many_sequences(dtype, D):
    """More of them than a wave has lanes, many empty."""
    r = random.Random(5)
    lens = [r.choice((0, 1, 3, r.randint(1, 90))) for _ in range(150)]
    for causal in (False, True):
        check(make(lens, lens, 2, 1, D, DT[dtype], 10, 25, seed=7), causal)


@pytest.mark.parametrize("dtype, D", [("bf16", 64), ("f16", 128), ("f32", 64)])
def test_rows_outside_every_sequence_are_zeros(dtype, D):
    q, k, v, do, table, buckets, cu, _ = make([60, 100], [60, 100], 2, 2, D, DT[dtype], 8, 16, first=13, rest=70)
    got = run(q, k, v, do, table, buckets, cu, cu, True, mq=80, mk=80)
    cut = [13, 73, 153]  # the second sequence to 80 rows; its default bias is the whole one's
    want = packed_rel(q[:153], k[:153], v[:153], do[:153], table, buckets, cut, cut, True, [-math.log(60), -math.log(100)])
    for x in ("o", "dq", "dk", "dv"):
        assert_within(got[x][:153], want[x], x)
        assert not got[x][153:].any() and not got[x][:13].any(), x
    assert_within(got["dtable"], want["dtable"], "dtable")


@pytest.mark.parametrize("table_dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_the_table_has_a_type_of_its_own(dtype, table_dtype):
    args = make([90, 30], [90, 30], 3, 3, 64, DT[dtype], 8, 30, table_dtype=DT[table_dtype])
    assert check(args, True)["dtable"].dtype == DT[table_dtype]


@pytest.mark.parametrize("dtype, D", [("bf16", 64), ("f16", 128), ("f32", 64), ("f32", 16)])
def test_values_at_the_types_ends(dtype, D):
    """Buckets of -inf and of the type's lowest value leave nothing, huge ones all."""
    q, k, v, do, table, buckets, cu, _ = make([140, 3], [140, 3], 2, 2, D, DT[dtype], 8, 30, seed=9)
    table[0], table[1], table[2] = -math.inf, torch.finfo(table.dtype).min, torch.finfo(table.dtype).max
    check((q, k, v, do, table, buckets, cu, cu), False)
    table[:] = -math.inf  # rows that see nothing
    got = check((q, k, v, do, table, buckets, cu, cu), True)
    assert all(not got[x].any() for x in got)


def test_buckets_outside_the_table_add_nothing():
    q, k, v, do, table, buckets, cu, _ = make([100, 31], [100, 31], 2, 2, 64, torch.float32, 8, 20)
    buckets[::3], buckets[1], buckets[5] = 8, -1, 1 << 30
    check((q, k, v, do, table, buckets, cu, cu), False)
    wide = buckets.long()
    wide[0] = 1 << 40
    got = run(q, k, v, do, table, wide, cu, cu, False)
    assert torch.equal(got["o"], run(q, k, v, do, table, buckets, cu, cu, False)["o"])


@pytest.mark.parametrize("dtype, D", [("bf16", 64), ("f32", 64), ("f16", 128)])
def test_strides_and_alignment(dtype, D):
    """Views with other strides, and rows off 16-byte boundaries."""
    q, k, v, do, table, buckets, cu, _ = make([75, 20], [75, 20], 2, 2, D, DT[dtype], 8, 20)
    want = packed_rel(q, k, v, do, table, buckets, cu, cu, True)

    def odd(t):
        s = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
        return s.copy_(t)

    for f in (odd, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)):
        views = [f(t).requires_grad_() for t in (q, k, v)] + [table.t().contiguous().t().requires_grad_()]
        o = ts.sigmoid_attention_varlen(*views[:3], ints(cu), ints(cu), 75, 75, is_causal=True, bias_table=views[3],
                                        bias_buckets=buckets)
        got = (o, *torch.autograd.grad(o, views, f(do)))
        for x, t in zip(("o", "dq", "dk", "dv", "dtable"), got):
            assert_within(t, want[x], x)


def test_zero_values_change_nothing():
    """A table of zeros: within the bounds, as the attention without one is."""
    q, k, v, do, table, buckets, cu, _ = make([200, 90], [200, 90], 4, 4, 64, torch.bfloat16, 8, 20)
    plain = ts.sigmoid_attention_varlen(q, k, v, ints(cu), ints(cu), 200, 200, is_causal=True)
    none = torch.zeros_like(table)
    check((q, k, v, do, none, buckets, cu, cu), True)
    assert_within(plain, packed_rel(q, k, v, do, none, buckets, cu, cu, True)["o"])


@pytest.mark.parametrize("dtype, D", [("bf16", 64), ("f16", 128), ("f32", 32), ("bf16", 32)])
def test_deterministic(dtype, D):
    args = make([700, 333, 90], [700, 333, 90], 4, 2, D, DT[dtype], 32, 128)
    first = run(*args, True)
    for _ in range(3):
        again = run(*args, True)
        assert all(torch.equal(first[x], again[x]) for x in first)


def test_gradient_against_differences():
    """fp32 against central differences of the op in the table's own direction: off by
    step^2 / 6 times the third derivative (|sigmoid'''| <= 1/8, of every score that the
    bucket reaches), and by the two values' rounding over the step."""
    args = q, k, v, do, table, buckets, cu, _ = make([40, 25], [40, 25], 2, 2, 32, torch.float32, 6, 12, seed=2)
    got = run(*args, False)["dtable"]
    want = packed_rel(*args, False)
    step, dO = 2.0 ** -6, do.double()
    for u, h in ((0, 0), (3, 1), (5, 0)):
        values = []
        for sign in (1.0, -1.0):
            moved = table.clone()
            moved[u, h] += sign * step
            o = run(q, k, v, do, moved, buckets, cu, cu, False)["o"].double()
            values.append((o * dO).sum())
        slope = (values[0] - values[1]) / (2 * step)
        third = sum((do[a:b, h].double() @ v[a:b, h].double().t()).abs().sum() for a, b in zip(cu, cu[1:])) / 8
        noise = (want["o"][1] * dO.abs()).sum() / step
        assert (slope - got[u, h].double()).abs() <= step ** 2 / 6 * third + noise + want["dtable"][1][u, h]


@pytest.mark.parametrize("frozen", [True, False])
def test_a_table_without_gradient(frozen):
    q, k, v, do, table, buckets, cu, _ = make([200], [200], 2, 2, 64, torch.bfloat16, 8, 20)
    full = run(q, k, v, do, table, buckets, cu, cu, True)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)] if frozen else [q, k, v]
    t = table.clone().requires_grad_(not frozen)
    o = ts.sigmoid_attention_varlen(*leaves, ints(cu), ints(cu), 200, 200, is_causal=True, bias_table=t,
                                    bias_buckets=buckets)
    got = torch.autograd.grad(o, leaves if frozen else [t], do)
    for x, y in zip(("dq", "dk", "dv") if frozen else ("dtable",), got):
        assert torch.equal(full[x], y)


@pytest.mark.parametrize("binding", ["node", "python"])
def test_a_table_without_gradient_takes_no_room_for_one(monkeypatch, binding):
    if binding == "python":
        monkeypatch.setenv("SIGATTN_EAGER_BINDING", "python")
    n, H, R = 4096, 8, 2048
    q, k, v, do, table, buckets, cu, _ = make([n], [n], H, H, 64, torch.bfloat16, 8, R)
    sums = n // 64 * H * (2 * R + 1) * 4
    peak = {}
    for frozen in (True, False):
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        t = table.clone().requires_grad_(not frozen)
        o = ts.sigmoid_attention_varlen(*leaves, ints(cu), ints(cu), n, n, bias_table=t, bias_buckets=buckets)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        got = torch.autograd.grad(o, leaves + ([] if frozen else [t]), do)
        peak[frozen] = torch.cuda.max_memory_allocated() - before
        del o, got
    assert peak[False] >= sums > 2 ** 23 and peak[True] < 3 * q.numel() * 2 + 2 ** 21


def test_captured_step_replays():
    q, k, v, do, table, buckets, cu, _ = make([300, 170, 64], [300, 170, 64], 4, 2, 64, torch.bfloat16, 32, 100)
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    at = ints(cu)

    def step():
        o = ts.sigmoid_attention_varlen(*leaves[:3], at, at, 300, 300, is_causal=True, bias_table=leaves[3],
                                        bias_buckets=buckets)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            for t in leaves:
                t.copy_(torch.roll(t, 1, 0))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        del want


def test_streams_and_two_calls_at_once():
    a = make([400, 100], [400, 100], 4, 4, 64, torch.bfloat16, 16, 60, seed=1)
    b = make([350, 222], [350, 222], 4, 4, 64, torch.bfloat16, 16, 60, seed=2)
    want = run(*a, True), run(*b, True)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = [None, None]
    for _ in range(3):
        for i, (s, x) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[i] = run(*x, True)
        torch.cuda.synchronize()
        for w, y in zip(want, got):
            assert all(torch.equal(w[x], y[x]) for x in w)


def test_compiled_and_eager_alike():
    q, k, v, do, table, buckets, cu, _ = make([90, 40], [90, 40], 2, 2, 64, torch.bfloat16, 8, 20)
    at = ints(cu)

    def f(q, k, v, t):
        return ts.sigmoid_attention_varlen(q, k, v, at, at, 90, 90, is_causal=True, bias_table=t, bias_buckets=buckets)

    want = run(q, k, v, do, table, buckets, cu, cu, True)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
    o = torch.compile(f, fullgraph=True, backend="aot_eager")(*leaves)
    got = (o, *torch.autograd.grad(o, leaves, do))
    assert all(torch.equal(want[x], y) for x, y in zip(("o", "dq", "dk", "dv", "dtable"), got))


def test_empty_calls():
    z = lambda n, h: torch.zeros(n, h, 64, device="cuda", requires_grad=True)  # noqa: E731
    table = torch.ones(4, 2, device="cuda", requires_grad=True)
    buckets = ints([0, 1, 2])
    for nq, nk, cu_q, cu_k in ((0, 0, [0, 0], [0, 0]), (3, 0, [0, 3], [0, 0]), (0, 3, [0, 0], [0, 3]), (3, 3, [0], [0])):
        q, k, v = z(nq, 2), z(nk, 2), z(nk, 2)
        o = ts.sigmoid_attention_varlen(q, k, v, ints(cu_q), ints(cu_k), nq, nk, bias_table=table, bias_buckets=buckets)
        assert o.shape == q.shape and not o.any()
        for t, g in zip((q, k, v, table), torch.autograd.grad(o, (q, k, v, table), torch.ones_like(o))):
            assert g.shape == t.shape and not g.any()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("R", [140, 150, 600, 1100, 1200])
def test_128_columns_and_the_room_for_sums(R, causal):
    """Workgroups of four waves, of eight where longer lines leave room for those alone, and of four again."""
    lens = [1250, 257, 0, 33]
    check(make(lens, lens, 1, 1, 128, torch.bfloat16, 40, R, seed=R), causal)


# Where dQ at D = 128 takes workgroups of eight waves: reaches 159 .. 1190.
@pytest.mark.parametrize("dtype, R", [("bf16", 158), ("bf16", 159), ("f16", 159), ("bf16", 1190), ("f16", 1190),
                                      ("bf16", 1191)])
@pytest.mark.parametrize("causal", [False, True])
def test_128_columns_on_either_side_of_eight_waves(dtype, R, causal):
    lens = [1250, 0, 33] if R > 1000 else [500, 0, 33]  # (a line reaches no further than the longest)
    check(make(lens, lens, 2, 1, 128, DT[dtype], 400, R, seed=R), causal)


@pytest.mark.parametrize("H, Hkv", [(3, 1), (8, 8), (12, 4), (16, 1)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_eight_waves_and_grouped_heads(H, Hkv, dtype):
    lens = [180, 300, 37, 257]
    check(make(lens, lens, H, Hkv, 128, DT[dtype], 16, 170, seed=H), True)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_eight_waves_and_many_sequences(dtype):
    r = random.Random(9)
    lens = [200, 290] + [r.choice((0, 1, 3, r.randint(1, 90))) for _ in range(100)]
    for causal in (False, True):
        check(make(lens, lens, 2, 1, 128, DT[dtype], 10, 180, seed=7), causal)
    check(make(lens, lens[::-1], 2, 1, 128, DT[dtype], 10, 180, seed=8), False)


@pytest.mark.parametrize("dtype, D, R", [("bf16", 128, 200), ("f16", 128, 200), ("bf16", 64, 200), ("f32", 128, 200),
                                         ("f32", 32, 200)])
def test_far_reaches_and_rows_outside_every_sequence(dtype, D, R):
    q, k, v, do, table, buckets, cu, _ = make([210, 300], [210, 300], 2, 1, D, DT[dtype], 8, R, first=70, rest=70)
    got = run(q, k, v, do, table, buckets, cu, cu, True, mq=280, mk=280)
    cut = [70, 280, 560]  # the second sequence to 280 rows; its default bias is the whole one's
    want = packed_rel(q[:560], k[:560], v[:560], do[:560], table, buckets, cut, cut, True, [-math.log(210), -math.log(300)])
    for x in ("o", "dq", "dk", "dv"):
        assert_within(got[x][:560], want[x], x)
        assert not got[x][560:].any() and not got[x][:70].any(), x
    assert_within(got["dtable"], want["dtable"], "dtable")


@pytest.mark.parametrize("lens, H, R, causal", [([300, 290], 2, 300, True), ([600], 3, 1000, False),
                                                ([1800, 70], 1, 2048, True)])
def test_fp32_far_reaches_at_128_columns(lens, H, R, causal):
    """The longest leave room for the tiles of one wave to 32 rows instead of two."""
    check(make(lens, lens, H, 1, 128, torch.float32, 40, R, seed=R), causal)


@pytest.mark.parametrize("D, dtype", [(64, "bf16"), (128, "f16"), (32, "f32")])
def test_bindings_alike(monkeypatch, D, dtype):
    args = make([300, 1, 77], [300, 1, 77], 4, 2, D, DT[dtype], 16, 60, seed=D)
    node = run(*args, True)
    monkeypatch.setenv("SIGATTN_EAGER_BINDING", "python")
    python = run(*args, True)
    assert all(torch.equal(node[x], python[x]) for x in node)


@pytest.mark.parametrize("D, dtype", [(64, "bf16"), (128, "f16"), (32, "f32")])
def test_the_library_makes_the_default_bias(monkeypatch, D, dtype):
    """A problem without one: in the forward, and in a backward that has no lines either."""
    from triton_sigmoid import _capi

    monkeypatch.setenv("SIGATTN_EAGER_BINDING", "python")
    args = make([300, 0, 77], [200, 5, 77], 4, 2, D, DT[dtype], 16, 60, seed=D)
    given, problem = run(*args, True), _capi._problem

    def without(*a, **k):
        p = problem(*a, **k)
        p.bias = None
        return p

    monkeypatch.setattr(_capi, "_problem", without)
    made = run(*args, True)
    assert all(torch.equal(given[x], made[x]) for x in given)


@pytest.mark.parametrize("binding", ["node", "python"])
def test_gradients_have_none_of_their_own(monkeypatch, binding):
    if binding == "python":
        monkeypatch.setenv("SIGATTN_EAGER_BINDING", "python")
    q, k, v, do, table, buckets, cu, _ = make([50], [50], 2, 2, 64, torch.bfloat16, 8, 20)
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    o = ts.sigmoid_attention_varlen(*leaves[:3], ints(cu), ints(cu), 50, 50, bias_table=table, bias_buckets=buckets)
    grads = torch.autograd.grad(o, leaves, do, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        sum(g.float().sum() for g in grads).backward()


@pytest.mark.parametrize("dtype, D", [("bf16", 64), ("f16", 128), ("bf16", 32), ("f32", 32), ("f32", 128)])
@pytest.mark.parametrize("causal", [False, True])
def test_infinite_keys_reach_no_sum_through_rows_that_are_not_there(dtype, D, causal):
    """A key of +-inf has sigmoids of 0 and 1, so dS = 0: the pairs of a key block with
    the rows that fill up a sequence's last block of queries are no pairs."""
    n, R, at = 37, 12, 33
    q, k, v, do, table, buckets, cu, _ = make([n], [n], 2, 2, D, DT[dtype], 2 * R + 1, R, seed=D)
    buckets = torch.arange(2 * R + 1, dtype=I32, device="cuda")
    k[at, :, 3] = math.inf
    got = run(q, k, v, do, table, buckets, cu, cu, causal)["dtable"].double()
    finite, u = torch.where(torch.isfinite(k), k, 0.0), torch.finfo(table.dtype).eps / 2
    pos = torch.arange(n, device="cuda")
    d = pos[None] - pos[:, None]
    for h in range(2):
        line, place = line_of(table, buckets, h, d)
        ds, err = grad_of_scores(q[:, h], finite[:, h], v[:, h], do[:, h], line - math.log(n), causal)
        ds[:, at] = err[:, at] = 0.0
        want, bound, size = (torch.zeros(2 * R + 1, dtype=torch.float64, device="cuda").index_add_(0, place.flatten(), x.flatten())
                             for x in (ds, err, ds.abs()))
        bound = bound + 300 * 2.0 ** -24 * size  # (fewer additions than that)
        assert ((got[:, h] - want).abs() <= bound + u * (want.abs() + bound) + torch.finfo(table.dtype).tiny).all()


def test_more_sequences_than_the_sums_keep():
    r = random.Random(6)
    lens = [r.choice((0, 1, 2, r.randint(1, 12))) for _ in range(1300)]
    check(make(lens, lens, 1, 1, 32, torch.bfloat16, 10, 9, seed=6), True)


def test_more_sums_than_31_bits_count():
    """2^31 sums of blocks and more: a batch's gradients are its sequences' in smaller batches, and
    the table's is the sum of theirs (fp32 sums of as many terms, in another order)."""
    n, B, H, D, R = 4096, 264, 64, 16, 2048
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("not enough free memory")
    assert n * B // 128 * H * (2 * R + 1) > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v, do = (torch.randn(n * B, H, D, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(4))
    table, buckets = torch.zeros(40, H, device="cuda"), torch.randint(0, 40, (2 * R + 1,), generator=g, device="cuda")

    def grads(first, count):
        at = slice(first * n, (first + count) * n)
        leaves = [t[at].requires_grad_() for t in (q, k, v)] + [table.clone().requires_grad_()]
        cu = torch.arange(count + 1, dtype=I32, device="cuda") * n
        o = ts.sigmoid_attention_varlen(*leaves[:3], cu, cu, n, n, is_causal=True, bias_table=leaves[3],
                                        bias_buckets=buckets.to(I32))
        return torch.autograd.grad(o, leaves, do[at])

    *whole, dtable = grads(0, B)
    parts = torch.zeros(40, H, dtype=torch.float64, device="cuda")
    for first, count in ((0, 100), (100, 100), (200, 64)):
        *some, t = grads(first, count)
        parts += t.double()
        for x, y in zip(whole, some):
            assert torch.equal(x[first * n:(first + count) * n], y)
    # dS have either sign, so running sums stay near the result S's size / sqrt(100) (a bucket's
    # places) and their rounding adds up as its square: 8448 blocks x 100 places of 2^-24 S / 10,
    # 6e-6 S.  The last 258 blocks, those past 2^31, make up a share of sqrt(3 %) of S.
    assert (dtable.double() - parts).abs().max() <= 2.0 ** -12 * parts.abs().max()
    assert dtable.abs().min() > 0


def test_fp32_sums_do_not_drift():
    """Four million dS of either sign in one bucket: what each may be off by adds up as
    its square where it has no preferred sign (six standard deviations; each within its
    bound), beside what all share: the fp32 bias and additive term, 2^-20 of the sum."""
    n = 2000
    q, k, v, do, table, buckets, cu, _ = make([n], [n], 2, 2, 32, torch.float32, 1, 0, seed=8)
    got = run(q, k, v, do, table, buckets, cu, cu, False)["dtable"].double()
    for h in range(2):
        add = (table.double()[0, h] - math.log(n)).expand(n, n)
        ds, err = grad_of_scores(q[:, h], k[:, h], v[:, h], do[:, h], add, False)
        bound = 6 * err.square().sum().sqrt() + 2.0 ** -20 * ds.sum().abs()
        assert (got[0, h] - ds.sum()).abs() <= bound


def test_fp32_sums_would_show_a_drift():
    """Sixty-four million dS of either sign in one bucket, with a bound that a drift of
    2^-27 of each dP to one side would be twice of (what the matrix cores' truncations add
    up to here: 9.1e-5 when nothing was done about it, 6e-8 now).  What has no preferred
    sign adds up as its square.  A truncation to 24 bits leaves 2^-23 / sqrt(12) of its value
    about the mean, three of them, of partial sums up to |dO|·|V|, 2^-24 of those: dP; of
    |q|·|k| scale: S, whose sum with the bias and the table's value is rounded once more; P is
    off by 2^-21.  Then the additions: 16 dS, and a lane's running sum of the keys before.
    Six standard deviations, and 2^-18 of the sum for what all share (the rounded bias
    and table)."""
    n, D = 8000, 32
    q, k, v, do, table, buckets, cu, _ = make([n], [n], 1, 1, D, torch.float32, 1, 0, seed=8)
    got = run(q, k, v, do, table, buckets, cu, cu, False)["dtable"].double()[0, 0]
    q, k, v, do = (t[:, 0].double() for t in (q, k, v, do))
    e, scale = 2.0 ** -24, 1.0 / math.sqrt(D)
    s = q @ k.t().contiguous() * scale + (table.double()[0, 0] - math.log(n))
    p = torch.sigmoid(s)
    w, dp = p * (1.0 - p), do @ v.t().contiguous()
    ds = w * dp
    var = (e * w * (do.abs() @ v.abs().t().contiguous())).square().sum()
    var += (e * ds * (q.abs() @ k.abs().t().contiguous() * scale + s.abs())).square().sum()
    var += (2.0 ** -21 * ds).square().sum()
    var += (e * ds.cumsum(1)[:, 31::32]).square().sum() * 2 + (16 * e * ds).square().sum()
    bound = 6 * var.sqrt() + 2.0 ** -18 * ds.sum().abs()
    assert 2.0 ** -27 * (w * dp.abs()).sum() >= 2 * bound
    assert (got - ds.sum()).abs() <= bound


@pytest.mark.parametrize("f", [(1e-13, 1e12, 1e30, 1e-30), (1.0, 1.0, 1e-15, 1e-14), (1e10, 1e-10, 1e15, 1e10)])
def test_fp32_values_far_from_one(f):
    """What three bf16 parts cannot hold takes the fp32 instruction, the sums by position too."""
    q, k, v, do, table, buckets, cu, _ = make([140, 33], [140, 33], 2, 1, 64, torch.float32, 12, 40)
    q, k, v, do = (x * y for x, y in zip((q, k, v, do), f))
    check((q, k, v, do, table, buckets, cu, cu), True)


# --- over a paged cache ---------------------------------------------------------------

def check_paged(ctx, new, H, Hkv, D, dtype, ps=16, num=16, R=40, causal=True, bias=None, mq="longest", seed=0,
                drop_page=False, layout="nhd", extra=0):
    g, r = torch.Generator().manual_seed(seed), random.Random(seed)
    lens = [c + n for c, n in zip(ctx, new)]
    pages = [-(-x // ps) for x in lens]
    pool = r.sample(range(sum(pages) + 3), sum(pages) + 3)
    width = max(1, max(pages)) + 1
    table = torch.full((len(ctx), width), -1, dtype=I32)
    for b, n in enumerate(pages):
        for j in range(n):
            table[b, j] = pool.pop()
    shape = (sum(pages) + 3, ps, Hkv, D)
    if layout == "nhd":
        kc, vc = (randn(g, *shape, dtype=dtype) for _ in range(2))
    else:  # heads before tokens
        kc, vc = (randn(g, shape[0], Hkv, ps, D, dtype=dtype).transpose(1, 2) for _ in range(2))
    q = randn(g, sum(new) + extra, H, D, dtype=dtype)
    values, buckets = randn(g, num, H, dtype=dtype, f=2.0), torch.randint(0, num, (2 * R + 1,), generator=g).to(I32).cuda()
    gone = {}
    if drop_page:
        for b, n in enumerate(pages):
            if n > 1:
                gone[b] = n // 2
                table[b, n // 2] = -1
    # What no sequence holds is never read.
    held = torch.zeros(shape[:2], dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        for j in range(pages[b]):
            if table[b, j] >= 0:
                held[table[b, j], : min(ps, n - j * ps)] = True
    for c in (kc, vc):
        c[~held] = math.nan
    table = table.cuda()
    mq = max(new) if mq == "longest" else mq
    got = ts.sigmoid_attention_paged(q, kc, vc, table, ints(lens), ints(offsets(new)), mq, is_causal=causal,
                                     sigmoid_bias=bias, bias_table=values, bias_buckets=buckets)
    want = torch.zeros(2, *q.shape, dtype=torch.float64, device="cuda")
    for b, (n, L, first) in enumerate(zip(new, lens, offsets(new))):
        if n == 0 or L == 0:
            continue
        pos = torch.arange(L, device="cuda")
        there = torch.ones(L, dtype=torch.bool, device="cuda")
        if b in gone:
            there = pos // ps != gone[b]
        pos = pos[there]
        rows = table[b].long()[pos // ps], pos % ps
        d = pos[None] - (torch.arange(n, device="cuda")[:, None] + L - n)
        for h in range(H):
            add = line_of(values, buckets, h, d)[0] + (-math.log(L) if bias is None else bias)
            if causal:
                add = torch.where(d > 0, -math.inf, add)
            at = slice(first, first + n)
            val, err = one_head(q[at, h], kc[rows][:, h // (H // Hkv)], vc[rows][:, h // (H // Hkv)], None, add, dtype)["o"]
            want[0][at, h], want[1][at, h] = val, err
    assert_within(got, tuple(want), "o")
    return got


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_paged_types_and_head_dims(dtype, D, causal):
    check_paged([100, 0, 33, 7], [1, 1, 1, 1], 8, 2, D, DT[dtype], causal=causal, seed=D)  # decoding
    check_paged([50, 0, 100], [70, 131, 40], 4, 2, D, DT[dtype], causal=causal, seed=D)  # chunks
    check_paged([100, 0, 33], [1, 60, 2], 8, 2, D, DT[dtype], causal=causal, seed=D)  # both


@pytest.mark.parametrize("H, Hkv", [(1, 1), (8, 1), (6, 2), (32, 8), (16, 16), (40, 1)])
def test_paged_heads(H, Hkv):
    check_paged([200, 31], [1, 1], H, Hkv, 64, torch.bfloat16, seed=H)
    check_paged([200, 31], [5, 60], H, Hkv, 64, torch.bfloat16, seed=H)


@pytest.mark.parametrize("dtype, D", [("bf16", 128), ("f16", 64), ("f32", 64), ("bf16", 32)])
@pytest.mark.parametrize("R", [0, 1, 31, 64, 500, 2048])
def test_paged_reaches(dtype, D, R):
    check_paged([700, 64, 1], [1, 1, 1], 8, 2, D, DT[dtype], R=R, num=9, seed=R)
    check_paged([700, 64, 1], [200, 33, 1], 8, 2, D, DT[dtype], R=R, num=9, causal=R % 2 == 0, seed=R)


@pytest.mark.parametrize("dtype, D", [("bf16", 128), ("f16", 64), ("f32", 128), ("f32", 32)])
def test_paged_long_contexts_are_cut(dtype, D):
    check_paged([9000], [1], 8, 2, D, DT[dtype], ps=64, R=128, seed=1)
    check_paged([5000, 300], [1, 1], 4, 4, D, DT[dtype], ps=32, R=700, seed=2)
    check_paged([4000], [150], 4, 2, D, DT[dtype], ps=16, R=128, seed=3)


@pytest.mark.parametrize("dtype, D", [("bf16", 128), ("f16", 64), ("f32", 64)])
def test_paged_page_sizes_pages_that_are_gone_and_padding(dtype, D):
    for ps in (16, 128, 1024):
        check_paged([300, 40], [1, 3], 8, 2, D, DT[dtype], ps=ps, drop_page=True, seed=ps)
    got = check_paged([300, 40, 5], [1, 90, 0], 8, 2, D, DT[dtype], extra=9, mq=None)
    assert not got[-9:].any()
    check_paged([60, 500], [4, 1], 8, 2, D, DT[dtype], layout="hnd", seed=4)
    check_paged([60, 500], [4, 1], 8, 2, D, DT[dtype], bias=-3.0, causal=False, seed=5)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_paged_rows_off_boundaries(dtype):
    g = torch.Generator().manual_seed(3)
    kc, vc = (randn(g, 4, 16, 2, 65, dtype=DT[dtype])[..., :64] for _ in range(2))
    q, values = randn(g, 2, 4, 64, dtype=DT[dtype]), randn(g, 6, 4, dtype=DT[dtype])
    buckets = torch.randint(0, 6, (21,), generator=g).to(I32).cuda()
    table, args = ints([[2, 0], [3, 1]]), (ints([20, 31]), ints([0, 1, 2]), 1)
    got = ts.sigmoid_attention_paged(q, kc, vc, table, *args, is_causal=True, bias_table=values, bias_buckets=buckets)
    want = ts.sigmoid_attention_paged(q, kc.contiguous(), vc.contiguous(), table, *args, is_causal=True,
                                      bias_table=values, bias_buckets=buckets)
    # Both within the bounds of the definition: apart by two of them at most.
    assert (got.float() - want.float()).abs().max() <= 4 * torch.finfo(DT[dtype]).eps * want.float().abs().max() + 1e-5


def test_paged_captured_step_replays():
    g = torch.Generator().manual_seed(0)
    kc, vc = (randn(g, 40, 16, 2, 64, dtype=torch.bfloat16) for _ in range(2))
    q, values = randn(g, 4, 8, 64, dtype=torch.bfloat16), randn(g, 16, 8, dtype=torch.bfloat16)
    buckets = torch.randint(0, 16, (201,), generator=g).to(I32).cuda()
    table, lens, cu = torch.arange(40, dtype=I32, device="cuda").view(4, 10), ints([100, 3, 64, 160]), ints([0, 1, 2, 3, 4])
    step = lambda: ts.sigmoid_attention_paged(q, kc, vc, table, lens, cu, 1, is_causal=True, bias_table=values,  # noqa: E731
                                              bias_buckets=buckets)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for new in ([100, 3, 64, 160], [1, 160, 17, 33], [159, 158, 2, 90]):
        lens.copy_(ints(new))
        values.copy_(torch.roll(values, 1, 0))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, step())


@pytest.mark.parametrize("dtype, D", [("bf16", 128), ("f16", 64), ("bf16", 32), ("f32", 128), ("f32", 32)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("new", [[1, 1], [90, 40], [90, 1]])
def test_paged_values_of_positions_that_hold_no_key(dtype, D, causal, new):
    """NaN at relative positions that lie behind every sequence: no pair's, so of no consequence."""
    g, R, ctx = torch.Generator().manual_seed(4), 200, (37, 71)
    lens = [c + n for c, n in zip(ctx, new)]
    kc, vc = (randn(g, 24, 16, 2, D, dtype=DT[dtype]) for _ in range(2))
    q, values = randn(g, sum(new), 4, D, dtype=DT[dtype]), randn(g, 2 * R + 1, 4, dtype=DT[dtype])
    table, buckets = torch.arange(24, dtype=I32, device="cuda").view(2, 12), torch.arange(2 * R + 1, dtype=I32, device="cuda")
    first = 1 if causal else max(new)  # the nearest position that no pair has

    def attend(t):
        return ts.sigmoid_attention_paged(q, kc, vc, table, ints(lens), ints(offsets(new)), max(new), is_causal=causal,
                                          bias_table=t, bias_buckets=buckets)

    want = attend(values)
    values[R + first:] = math.nan
    assert torch.equal(attend(values), want) and want.isfinite().all()


def _f16_bound(q, k, add, *vectors):
    """P v (and, of a second one, its transpose times do) of one head in 64 bits, and the bounds with
    P rounded to 11 bits however small it is (to 2^-37 below 2^-26): reference64's, without
    what rounding next to zero costs."""
    D, u, e = q.shape[1], 2.0 ** -11, 2.0 ** -24
    q, k = q.double(), k.double()
    p = torch.sigmoid(q @ k.t().contiguous() / math.sqrt(D) + add)
    share = (D + 8) * e * (q.abs() @ k.abs().t().contiguous() / math.sqrt(D) + add.abs()) + 2.0 ** -21
    off = p * (share + u) + 2.0 ** -37 * (p < 2.0 ** -26)
    out = []
    for x in vectors:
        val, err = p @ x.double(), off @ x.double().abs() + (p.shape[1] + 2) * e * (p @ x.double().abs())
        out.append((val, err + u * (val.abs() + err) + 2.0 ** -25))
        p, off = p.t().contiguous(), off.t().contiguous()
    return out


@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("odd", [False, True])
def test_f16_sigmoids_next_to_zero(D, odd):
    """Long contexts have sigmoids near one over their length, and less with negative values:
    below 2^-14 fp16 has fewer bits of them."""
    g, n, value = torch.Generator().manual_seed(D), 800, -8.0
    q, k, v = (randn(g, n * 2 * D + odd, dtype=torch.float16)[odd:].view(n, 2, D) for _ in range(3))
    v.mul_(4096)  # (so that an output's own rounding is no matter)
    table, buckets, cu = torch.full((1, 2), value, device="cuda"), ints([0]), ints([0, n])
    do = randn(g, n, 2, D, dtype=torch.float16) * 4096
    got = ts.sigmoid_attention_varlen(q, k, v.requires_grad_(), cu, cu, n, n, bias_table=table, bias_buckets=buckets)
    dv = torch.autograd.grad(got, v, do)[0]
    add = torch.full((), value - math.log(n), dtype=torch.float64, device="cuda")
    for h in range(2):
        o, dv_h = _f16_bound(q[:, h], k[:, h], add, v.detach()[:, h], do[:, h])
        assert_within(got[:, h], o)
        assert_within(dv[:, h], dv_h)


@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("new", [[1, 1], [70, 1], [70, 100]])
@pytest.mark.parametrize("odd", [False, True])
def test_paged_f16_sigmoids_next_to_zero(D, new, odd):
    g, ctx, value = torch.Generator().manual_seed(D), (700, 2900), -7.0
    lens = [c + n for c, n in zip(ctx, new)]
    kc, vc = (randn(g, 400, 16, 2, D + odd, dtype=torch.float16)[..., :D] for _ in range(2))
    vc.mul_(4096)
    q = randn(g, sum(new), 4, D, dtype=torch.float16)
    pages = torch.arange(400, dtype=I32, device="cuda").view(2, 200)
    got = ts.sigmoid_attention_paged(q, kc, vc, pages, ints(lens), ints(offsets(new)), max(new),
                                     bias_table=torch.full((1, 4), value, device="cuda"), bias_buckets=ints([0]))
    for b, (n, L, first) in enumerate(zip(new, lens, offsets(new))):
        rows = [c[200 * b: 200 * b + 200].reshape(3200, 2, D)[:L] for c in (kc, vc)]
        add = torch.full((), value - math.log(L), dtype=torch.float64, device="cuda")
        for h in range(4):
            o, = _f16_bound(q[first:first + n, h], rows[0][:, h // 2], add, rows[1][:, h // 2])
            assert_within(got[first:first + n, h], o)


@pytest.mark.parametrize("dtype, D", [("bf16", 64), ("f16", 128), ("f32", 32), ("f32", 128)])
@pytest.mark.parametrize("causal", [False, True])
def test_values_of_positions_that_hold_no_pair(dtype, D, causal):
    lens, R = [37, 70], 200
    q, k, v, do, table, _, cu, _ = make(lens, lens, 2, 1, D, DT[dtype], 2 * R + 1, R)
    buckets = torch.arange(2 * R + 1, dtype=I32, device="cuda")
    want = run(q, k, v, do, table, buckets, cu, cu, causal)
    table[R + (1 if causal else 70):] = table[:R - 69] = math.nan
    got = run(q, k, v, do, table, buckets, cu, cu, causal)
    assert all(torch.equal(got[x], want[x]) and want[x].isfinite().all() for x in want)


def test_what_was_trained_is_served():
    """A sequence in one training-shaped call, and token by token over a paged cache."""
    g = torch.Generator().manual_seed(8)
    n, H, Hkv, D, dtype = 75, 4, 2, 64, torch.float32
    q, k, v = randn(g, n, H, D, dtype=dtype), randn(g, n, Hkv, D, dtype=dtype), randn(g, n, Hkv, D, dtype=dtype)
    values, buckets = randn(g, 16, H, dtype=dtype), ts.relative_position_buckets(16, 40, False, device="cuda")
    cu = ints([0, n])
    whole = ts.sigmoid_attention_varlen(q, k, v, cu, cu, n, n, is_causal=True, sigmoid_bias=-2.0, bias_table=values,
                                        bias_buckets=buckets)
    want = packed_rel(q, k, v, None, values, buckets, [0, n], [0, n], True, bias=-2.0)["o"]
    assert_within(whole, want)
    kc, vc = (torch.zeros(8, 16, Hkv, D, dtype=dtype, device="cuda") for _ in range(2))
    table, free = torch.full((1, 8), -1, dtype=I32, device="cuda"), torch.arange(8, dtype=I32, device="cuda").flip(0)
    at, rows = 0, []
    for step in (30, 1, 1, 17, 1, 25):
        plan = ts.paged_plan(ints([at]), ints([step]), table, free, 16, step)
        free = free[int(plan.pages_needed):].contiguous()
        new = slice(at, at + step)
        ts.paged_cache_write(k[new], v[new], kc, vc, plan.slot_mapping)
        rows.append(ts.sigmoid_attention_paged(q[new], kc, vc, plan.block_table, plan.seq_lens, plan.cu_seqlens, step,
                                               is_causal=True, sigmoid_bias=-2.0, bias_table=values,
                                               bias_buckets=buckets))
        at += step
    assert_within(torch.cat(rows), want)


def test_paged_streams_and_two_calls_at_once():
    g = torch.Generator().manual_seed(1)
    kc, vc = (randn(g, 40, 16, 2, 64, dtype=torch.bfloat16) for _ in range(2))
    table, cu = torch.arange(40, dtype=I32, device="cuda").view(4, 10), ints([0, 1, 2, 3, 4])
    buckets = torch.randint(0, 16, (201,), generator=g).to(I32).cuda()
    calls = [(randn(g, 4, 8, 64, dtype=torch.bfloat16), randn(g, 16, 8, dtype=torch.bfloat16), ints(x))
             for x in ([100, 3, 64, 160], [1, 160, 17, 33])]

    def one(q, values, lens):
        return ts.sigmoid_attention_paged(q, kc, vc, table, lens, cu, 1, is_causal=True, bias_table=values,
                                          bias_buckets=buckets)

    want = [one(*c) for c in calls]
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        got = []
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append(one(*c))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("new", [[1, 1], [90, 1]])
def test_paged_bindings_alike(monkeypatch, new):
    args = [300, 40], new, 8, 2, 64, torch.bfloat16
    node = check_paged(*args, seed=9)
    monkeypatch.setenv("SIGATTN_EAGER_BINDING", "python")
    assert torch.equal(node, check_paged(*args, seed=9))


@pytest.mark.parametrize("new", [[1, 1], [70, 1]])
def test_paged_offsets_beyond_31_bits(new):
    """A cache of more than 2^31 values: the same rows at its front and at its end."""
    pages, ps, Hkv, D = 2 ** 31 // (16 * 2 * 128) + 40, 16, 2, 128
    kc, vc = (torch.empty(pages, ps, Hkv, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    g = torch.Generator().manual_seed(2)
    for c in (kc, vc):
        c[:20] = randn(g, 20, ps, Hkv, D, dtype=torch.bfloat16)
        c[-20:] = c[:20]
    q, values = randn(g, sum(new), 8, D, dtype=torch.bfloat16), randn(g, 16, 8, dtype=torch.bfloat16)
    buckets = torch.randint(0, 16, (101,), generator=g).to(I32).cuda()
    front = torch.arange(20, dtype=I32, device="cuda").view(2, 10)
    near, far = (ts.sigmoid_attention_paged(q, kc, vc, t, ints([160, 101]), ints(offsets(new)), max(new), is_causal=True,
                                            bias_table=values, bias_buckets=buckets)
                 for t in (front, front + (pages - 20)))
    assert torch.equal(near, far) and near.any()
