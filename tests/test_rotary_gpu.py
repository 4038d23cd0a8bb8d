"""Rotary embedding and the cache writer that turns keys on the way, against the
definition in 64 bits: two fp32 products and their sum (each off by 2^-24 of its
size; the sum too), rounded once to the I/O dtype."""

import pytest
import torch

import triton_sigmoid as ts
from reference64 import E32, assert_within, half_step

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
I32 = torch.int32


def randn(g, *shape, dtype):
    return torch.randn(shape, generator=g).to(dtype).cuda()


def turned(x, positions, angles, pairs, inverse=False):
    """(value, bound) of rows [N, heads, D]."""
    rot, u, tiny = angles.shape[1], *half_step(x.dtype)
    half, y = rot // 2, x.double()
    row = angles.double()[positions.long().clamp(0, angles.shape[0] - 1)][:, None]
    cos, sin = row[..., :half], row[..., half:] * (-1.0 if inverse else 1.0)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, half), slice(half, rot))
    val, err = y.clone(), torch.zeros_like(y)
    val[..., a], val[..., b] = y[..., a] * cos - y[..., b] * sin, y[..., b] * cos + y[..., a] * sin
    err[..., a] = 2 * E32 * ((y[..., a] * cos).abs() + (y[..., b] * sin).abs())
    err[..., b] = 2 * E32 * ((y[..., b] * cos).abs() + (y[..., a] * sin).abs())
    err[..., :rot] += u * (val[..., :rot].abs() + err[..., :rot]) + tiny
    return val, err


def tables(P, rot):
    return ts.rotary_table(P, rot, device="cuda")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D, rot", [(16, 16), (16, 2), (32, 32), (32, 12), (64, 64), (64, 32), (64, 6), (128, 128), (128, 64),
                                    (128, 126)])
@pytest.mark.parametrize("pairs", [False, True])
def test_values_and_gradients(dtype, D, rot, pairs):
    g = torch.Generator().manual_seed(D + rot)
    for N, H, Hkv in ((1, 1, 1), (37, 6, 2), (130, 5, 5)):
        q, k = randn(g, N, H, D, dtype=DT[dtype]).requires_grad_(), randn(g, N, Hkv, D, dtype=DT[dtype]).requires_grad_()
        dq, dk = randn(g, N, H, D, dtype=DT[dtype]), randn(g, N, Hkv, D, dtype=DT[dtype])
        at, angles = torch.randint(0, 500, (N,), generator=g).to(I32).cuda(), tables(500, rot)
        got = ts.rotary_embedding(q, k, at, angles, interleaved=pairs)
        grads = torch.autograd.grad(got, (q, k), (dq, dk))
        for x, y in zip((q, k), got):
            assert y.is_contiguous() and y.dtype == x.dtype
            assert_within(y, turned(x.detach(), at, angles, pairs))
        for x, y in zip((dq, dk), grads):
            assert_within(y, turned(x, at, angles, pairs, inverse=True))


def test_gradient_against_differences():
    """The op is linear: a difference over a step of one element is its column, off by
    the rounding of the two values over the step."""
    g = torch.Generator().manual_seed(1)
    q, k = (randn(g, 3, 2, 16, dtype=torch.float32) for _ in range(2))
    at, angles, do = torch.tensor([0, 7, 3], device="cuda"), tables(9, 12), randn(g, 3, 2, 16, dtype=torch.float32)
    leaf = q.clone().requires_grad_()
    (grad,) = torch.autograd.grad(ts.rotary_embedding(leaf, k, at, angles)[0], leaf, do)
    for i in ((0, 0, 0), (1, 1, 7), (2, 0, 11), (1, 0, 15)):
        ends = []
        for sign in (1.0, -1.0):
            x = q.clone()
            x[i] += sign
            ends.append((ts.rotary_embedding(x, k, at, angles)[0].double() * do.double()).sum())
        moved = (turned(q, at, angles, False)[1] + 8 * E32) * do.double().abs()
        assert ((ends[0] - ends[1]) / 2 - grad[i].double()).abs() <= moved.sum() + 4 * E32 * grad[i].abs()


def test_second_derivative_is_the_rotation():
    g = torch.Generator().manual_seed(1)
    q, k = (randn(g, 3, 2, 16, dtype=torch.float32).requires_grad_() for _ in range(2))
    at, angles, w = torch.tensor([0, 7, 3], device="cuda"), tables(9, 16), randn(g, 3, 2, 16, dtype=torch.float32)
    do = randn(g, 3, 2, 16, dtype=torch.float32).requires_grad_()
    (dq,) = torch.autograd.grad(ts.rotary_embedding(q, k, at, angles)[0], q, do, create_graph=True)
    (back,) = torch.autograd.grad(dq, do, w)
    assert_within(back, turned(w, at, angles, False))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_batched_tensors_strides_and_positions(dtype):
    g = torch.Generator().manual_seed(2)
    qkv = randn(g, 3, 20, 8, 64, dtype=DT[dtype])  # [B, T, H + 2 Hkv, D] of one projection
    q, k = qkv[:, :, :4], qkv[:, :, 4:6]
    angles = tables(50, 64)
    for at in (torch.arange(20, device="cuda"), torch.randint(0, 50, (3, 20), generator=g).cuda()):
        got = ts.rotary_embedding(q, k, at, angles)
        rows = at.expand(3, 20).reshape(-1)
        for x, y in zip((q, k), got):
            val, err = turned(x.flatten(0, 1), rows, angles, False)
            assert_within(y, (val.view(x.shape), err.view(x.shape)))
    flat = qkv.flatten(0, 1)
    for view in (flat[:, :5], flat[:, ::2], flat.transpose(0, 1).contiguous().transpose(0, 1)[:, 1:4], flat[::3]):
        rows = torch.arange(view.shape[0], device="cuda")
        for y in ts.rotary_embedding(view, view[:, :1], rows, angles, interleaved=True):
            assert_within(y, turned(view[:, :y.shape[1]], rows, angles, True))
    odd = torch.empty(flat.numel() + 1, dtype=flat.dtype, device="cuda")[1:].view(flat.shape).copy_(flat)
    rows = torch.arange(60, device="cuda")
    assert_within(ts.rotary_embedding(odd, odd, rows, angles)[1], turned(flat, rows, angles, False))


def test_positions_are_clamped_and_none_are_needed():
    g = torch.Generator().manual_seed(3)
    q = randn(g, 6, 2, 32, dtype=torch.bfloat16)
    at, angles = torch.tensor([-5, 0, 9, 10, 1 << 30, 1 << 40], device="cuda"), tables(10, 32)
    assert_within(ts.rotary_embedding(q, q, at, angles)[0], turned(q, at, angles, False))
    a, b = ts.rotary_embedding(q[:0], q[:0, :1], at[:0], angles)
    assert a.shape == (0, 2, 32) and b.shape == (0, 1, 32)


def test_far_positions_keep_their_angles():
    """Angles of positions past 2^17, from the table in 64 bits rounded to fp32."""
    table = ts.rotary_table(200000, 16)
    p = torch.tensor([131071, 199999], dtype=torch.float64)[:, None]
    angle = p * 10000.0 ** (-torch.arange(0, 16, 2, dtype=torch.float64) / 16)
    want = torch.cat([angle.cos(), angle.sin()], 1)
    # The fp64 angle itself is off by 2^-53 of up to 2e5 and its frequency's rounding.
    assert (table[[131071, 199999]].double() - want).abs().max() <= E32 + 1e-10


def check_write(N, H, Hkv, D, rot, dtype, pairs=False, ps=16, pages=9, layout="nhd", seed=0, long=False):
    g = torch.Generator().manual_seed(seed)
    q, k, v = randn(g, N, H, D, dtype=dtype), randn(g, N, Hkv, D, dtype=dtype), randn(g, N, Hkv, D, dtype=dtype)
    if layout == "nhd":
        kc, vc = (randn(g, pages, ps, Hkv, D, dtype=dtype) for _ in range(2))
    elif layout == "hnd":
        kc, vc = (randn(g, pages, Hkv, ps, D, dtype=dtype).transpose(1, 2) for _ in range(2))
    else:  # keys and values of a page side by side
        both = randn(g, pages, 2, ps, Hkv, D, dtype=dtype)
        kc, vc = both[:, 0], both[:, 1]
    slots = torch.randperm(pages * ps, generator=g)[:N].to(I32)
    slots[::7] = -1
    slots[3::11] = pages * ps
    slots, at = slots.cuda(), torch.randint(0, 300, (N,), generator=g).cuda()
    at = at if long else at.to(I32)
    angles, was = tables(300, rot), (kc.clone(), vc.clone())
    out = ts.paged_cache_write_rotary(q, k, v, kc, vc, slots.long() if long else slots, at, angles, interleaved=pairs)
    assert_within(out, turned(q, at, angles, pairs))
    there = (slots >= 0) & (slots < pages * ps)
    val, err = turned(k, at, angles, pairs)
    for cache, old, rows, bound in ((kc, was[0], val, err), (vc, was[1], v.double(), torch.zeros_like(err))):
        want, off = old.double(), torch.zeros_like(old, dtype=torch.float64)
        s = slots[there].long()
        want[s // ps, s % ps], off[s // ps, s % ps] = rows[there], bound[there]
        assert_within(cache, (want, off))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D, rot", [(16, 16), (32, 20), (64, 64), (64, 32), (128, 128), (128, 2)])
@pytest.mark.parametrize("pairs", [False, True])
def test_writes(dtype, D, rot, pairs):
    check_write(90, 6, 2, D, rot, DT[dtype], pairs, seed=D + rot)


@pytest.mark.parametrize("N, H, Hkv", [(0, 2, 1), (1, 1, 1), (1, 32, 8), (3, 7, 7), (64, 32, 8), (500, 3, 1)])
@pytest.mark.parametrize("layout", ["nhd", "hnd", "joint"])
def test_writes_of_sizes_and_layouts(N, H, Hkv, layout):
    check_write(N, H, Hkv, 64, 64, torch.bfloat16, ps=32, pages=20, layout=layout, seed=N, long=N % 2 == 0)


def test_write_from_one_projection_and_off_boundaries():
    g = torch.Generator().manual_seed(4)
    qkv = randn(g, 20, 8, 64, dtype=torch.float16)
    angles, at, slots = tables(64, 48), torch.arange(20, device="cuda"), torch.arange(20, device="cuda").flip(0)
    got = []
    for t in (qkv, torch.empty(qkv.numel() + 1, dtype=qkv.dtype, device="cuda")[1:].view(qkv.shape).copy_(qkv)):
        kc, vc = (torch.zeros(2, 16, 2, 64, dtype=qkv.dtype, device="cuda") for _ in range(2))
        out = ts.paged_cache_write_rotary(t[:, :4], t[:, 4:6], t[:, 6:], kc, vc, slots, at, angles)
        assert_within(out, turned(qkv[:, :4], at, angles, False))
        got.append((out, kc, vc))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert torch.equal(got[0][2].flatten(0, 1)[:20], qkv[:, 6:].flip(0))


@pytest.mark.parametrize("binding", ["node", "python"])
def test_autograd_sees_what_is_changed(monkeypatch, binding):
    if binding == "python":
        monkeypatch.setenv("SIGATTN_EAGER_BINDING", "python")
    kc, vc = (torch.randn(4, 16, 2, 32, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    new, at = torch.randn(3, 2, 32, device="cuda", dtype=torch.bfloat16), torch.arange(3, dtype=I32, device="cuda")
    was = kc._version, vc._version
    ts.paged_cache_write_rotary(new, new, new, kc, vc, at, at, tables(8, 32))
    assert (kc._version, vc._version) == (was[0] + 1, was[1] + 1)


@pytest.mark.parametrize("binding", ["node", "python"])
def test_refusals_on_the_gpu(monkeypatch, binding):
    if binding == "python":
        monkeypatch.setenv("SIGATTN_EAGER_BINDING", "python")
    kc, vc = (torch.zeros(4, 16, 2, 32, device="cuda") for _ in range(2))
    new, at, angles = torch.zeros(3, 2, 32, device="cuda"), torch.arange(3, device="cuda"), tables(8, 32)
    with pytest.raises(RuntimeError, match="no backward"):
        ts.paged_cache_write_rotary(new.clone().requires_grad_(), new, new, kc, vc, at, at, angles)
    with pytest.raises(RuntimeError, match="expected cuda"):
        ts.paged_cache_write_rotary(new.cpu(), new, new, kc, vc, at, at, angles)
    with pytest.raises(RuntimeError, match="expected cuda"):
        ts.rotary_embedding(new, new.cpu(), at, angles)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(new, new)
        with pytest.raises(RuntimeError, match="forward-mode"):
            ts.paged_cache_write_rotary(dual, new, new, kc, vc, at, at, angles)


def test_captured_step_replays():
    g = torch.Generator().manual_seed(6)
    q, k, v = randn(g, 8, 4, 64, dtype=torch.bfloat16), randn(g, 8, 2, 64, dtype=torch.bfloat16), randn(g, 8, 2, 64, dtype=torch.bfloat16)
    kc, vc = (torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slots, at, angles = torch.arange(8, dtype=I32, device="cuda"), torch.arange(8, dtype=I32, device="cuda"), tables(99, 64)
    step = lambda: ts.paged_cache_write_rotary(q, k, v, kc, vc, slots, at, angles)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        at.add_(7)
        slots.add_(8)
        graph.replay()
        torch.cuda.synchronize()
        got, keys = out.clone(), kc.clone()
        assert torch.equal(got, step()) and torch.equal(keys, kc), i
        assert_within(kc.flatten(0, 1)[8 + 8 * i:16 + 8 * i], turned(k, at, angles, False))


def test_compiled_and_eager_alike():
    g = torch.Generator().manual_seed(7)
    q, k = randn(g, 9, 4, 64, dtype=torch.bfloat16).requires_grad_(), randn(g, 9, 2, 64, dtype=torch.bfloat16).requires_grad_()
    at, angles = torch.arange(9, dtype=I32, device="cuda"), tables(16, 64)
    f = lambda q, k: ts.rotary_embedding(q, k, at, angles)  # noqa: E731
    do = randn(g, 9, 4, 64, dtype=torch.bfloat16), randn(g, 9, 2, 64, dtype=torch.bfloat16)
    want, got = f(q, k), torch.compile(f, fullgraph=True, backend="aot_eager")(q, k)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(want, (q, k), do), torch.autograd.grad(got, (q, k), do)))


def test_scores_depend_on_the_difference_alone():
    """Trained in one call and served over the cache, keys turned on the way: the same
    rows, and the same as every position moved by 11 (fp32)."""
    g = torch.Generator().manual_seed(8)
    n, H, Hkv, D = 50, 4, 2, 64
    q, k, v = (randn(g, n, h, D, dtype=torch.float32) for h in (H, Hkv, Hkv))
    angles, at, cu = tables(128, D), torch.arange(n, dtype=I32, device="cuda"), torch.tensor([0, n], dtype=I32, device="cuda")

    def whole(move):
        a, b = ts.rotary_embedding(q, k, at + move, angles)
        return ts.sigmoid_attention_varlen(a, b, v, cu, cu, n, n, is_causal=True, sigmoid_bias=-2.0)

    base = whole(0)
    # A turned row is off by 4e per element, the angles by e: scores by 10 e |q| |k| / 8,
    # and O by that share of sum |v|; the attention's own by (D + 8) e and 2^-21 of P.
    size = (q.norm(dim=-1).max() * k.norm(dim=-1).max() / 8).item()
    bound = ((10 + D + 8) * E32 * size + 2 ** -20 + n * E32) * v.abs().sum(0).max().item()
    assert (base - whole(11)).abs().max() <= 2 * bound
    kc, vc = (torch.zeros(4, 16, Hkv, D, device="cuda") for _ in range(2))
    table, rows = torch.arange(4, dtype=I32, device="cuda").flip(0)[None].contiguous(), []
    for first, step in ((0, 20), (20, 1), (21, 1), (22, 28)):
        new = slice(first, first + step)
        plan = ts.paged_plan(torch.tensor([first], dtype=I32, device="cuda"), torch.tensor([step], dtype=I32, device="cuda"),
                             table, table[0, -(-first // 16):].contiguous(), 16, step)
        a = ts.paged_cache_write_rotary(q[new], k[new], v[new], kc, vc, plan.slot_mapping, at[new], angles)
        rows.append(ts.sigmoid_attention_paged(a, kc, vc, plan.block_table, plan.seq_lens, plan.cu_seqlens, step,
                                               is_causal=True, sigmoid_bias=-2.0))
    assert (torch.cat(rows) - base).abs().max() <= 2 * bound


def test_slots_beyond_31_bits():
    """A cache of more than 2^31 values: rows at its end as at its front."""
    pages, ps, Hkv, D, N = 2 ** 31 // (16 * 2 * 128) + 4, 16, 2, 128, 40
    g = torch.Generator().manual_seed(4)
    kc, vc = (torch.empty(pages, ps, Hkv, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q, k, v = (randn(g, N, h, D, dtype=torch.bfloat16) for h in (4, Hkv, Hkv))
    pos, angles = torch.arange(N, dtype=torch.int32, device="cuda"), ts.rotary_table(N, D, device="cuda")
    slots = torch.arange(N, dtype=torch.int32, device="cuda")
    for first in (0, pages * ps - N):
        ts.paged_cache_write_rotary(q, k, v, kc, vc, slots + first, pos, angles)
    for c in (kc, vc):
        rows = c.view(-1, Hkv, D)
        assert torch.equal(rows[:N], rows[-N:])
    assert torch.equal(vc.view(-1, Hkv, D)[-N:], v)


@pytest.mark.parametrize("D, pairs", [(64, False), (128, True), (16, False)])
def test_bindings_alike(monkeypatch, D, pairs):
    g = torch.Generator().manual_seed(5)
    q, k, dq, dk = (randn(g, 100, h, D, dtype=torch.bfloat16) for h in (6, 2, 6, 2))
    pos, angles = torch.arange(100, dtype=torch.int32, device="cuda"), ts.rotary_table(128, D, device="cuda")

    def both():
        a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
        out = ts.rotary_embedding(a, b, pos, angles, pairs)
        return (*out, *torch.autograd.grad(out, (a, b), (dq, dk)))

    node = both()
    monkeypatch.setenv("SIGATTN_EAGER_BINDING", "python")
    assert all(torch.equal(x, y) for x, y in zip(node, both()))


def test_streams_and_two_calls_at_once():
    g = torch.Generator().manual_seed(6)
    angles = ts.rotary_table(4096, 64, device="cuda")
    pos = torch.arange(4000, dtype=torch.int32, device="cuda")
    calls = [tuple(randn(g, 4000, h, 64, dtype=torch.float16) for h in (8, 2)) for _ in range(2)]
    want = [ts.rotary_embedding(*c, pos, angles) for c in calls]
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        got = []
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append(ts.rotary_embedding(*c, pos, angles))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(want, got) for a, b in zip(x, y))


@pytest.mark.parametrize("off", [0, 1])
def test_more_rows_than_a_launch_has_workgroups(off):
    """2^24 rows and more, on 16-byte boundaries and off them: each as its copy among a few."""
    N, D, g = 2 ** 24 + 300, 16, torch.Generator().manual_seed(off)
    few = randn(g, 4099, 1, D, dtype=torch.bfloat16)
    at, angles = torch.arange(4099, dtype=I32, device="cuda"), tables(5000, D)
    q = torch.empty(N * D + off, dtype=torch.bfloat16, device="cuda")[off:].view(N, 1, D)
    rows = torch.arange(N, device="cuda") % 4099
    q.copy_(few[rows])
    got, _ = ts.rotary_embedding(q, few[:1].expand(N, 1, D), rows.to(I32), angles)
    want, _ = ts.rotary_embedding(few, few, at, angles)
    assert torch.equal(got, want[rows])


def test_more_units_than_a_launch_has_threads():
    """2^32 pieces and more (of an expanded query, whose copy is 137 GB): as in calls of a few rows."""
    N, H, D = 2 ** 23 + 70, 64, 128
    if torch.cuda.mem_get_info()[0] < 180 << 30:
        pytest.skip("not enough free memory")
    g = torch.Generator().manual_seed(0)
    q, k = randn(g, 1, H, D, dtype=torch.bfloat16), randn(g, 1, 1, D, dtype=torch.bfloat16)
    angles, at = tables(1000, D), (torch.arange(N, device="cuda") % 1000).to(I32)
    got, keys = ts.rotary_embedding(q.expand(N, H, D), k.expand(N, 1, D), at, angles)
    want, want_keys = ts.rotary_embedding(q.expand(1000, H, D), k.expand(1000, 1, D), at[:1000].contiguous(), angles)
    for first in (0, 2 ** 22, 2 ** 23 - 1000, 2 ** 23, N - 500):
        n = min(1000, N - first)
        assert torch.equal(got[first:first + n], want[at[first:first + n].long()]), first
    assert torch.equal(keys, want_keys[at.long()])
    del got
    torch.cuda.empty_cache()
