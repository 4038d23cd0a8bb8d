"""Positions: tables, refusals and the C ABI's checks, on the CPU."""

import ctypes
import math
from fractions import Fraction

import pytest
import torch
from torch.autograd import forward_ad

import triton_sigmoid as ts
from triton_sigmoid import _capi

CU = torch.tensor([0, 5, 12], dtype=torch.int32)


@pytest.mark.parametrize("num, far, both", [(32, 128, True), (32, 128, False), (4, 8, True), (2, 5, False), (64, 300, True),
                                            (320, 800, True), (8, 2048, False)])
def test_buckets(num, far, both):
    got = ts.relative_position_buckets(num, far, both)
    assert got.dtype == torch.int32 and got.shape == (2 * far + 1,)
    n = num // 2 if both else num
    near = n // 2
    for d in range(-far, far + 1):
        u, dist = got[far + d].item(), abs(d) if both else max(-d, 0)
        if both and d > 0:
            u -= n
        if dist < near:
            assert u == dist
            continue
        i = u - near
        assert 0 <= i < n - near
        # near * (far / near)^(i / m) <= dist < the next border, in exact numbers
        m, ratio = n - near, Fraction(far, near)
        assert Fraction(dist, near) ** m >= ratio ** i
        assert i == n - near - 1 or Fraction(dist, near) ** m < ratio ** (i + 1)


@pytest.mark.parametrize("kw", [dict(num_buckets=3), dict(num_buckets=2), dict(num_buckets=1, bidirectional=False),
                                dict(max_distance=8), dict(max_distance=2049), dict(num_buckets=-4)])
def test_buckets_that_are_none(kw):
    with pytest.raises(ValueError):
        ts.relative_position_buckets(**kw)


def test_rotary_table():
    got = ts.rotary_table(100, 24, base=500.0)
    assert got.dtype == torch.float32 and got.shape == (100, 24)
    for p, i in ((0, 0), (1, 0), (99, 5), (42, 11)):
        angle = p * 500.0 ** (-2 * i / 24)
        assert abs(got[p, i].item() - math.cos(angle)) <= 2.0 ** -24
        assert abs(got[p, 12 + i].item() - math.sin(angle)) <= 2.0 ** -24
    for bad in ((0, 8), (4, 7), (4, 0)):
        with pytest.raises(ValueError):
            ts.rotary_table(*bad)


def _varlen(**kw):
    args = dict(bias_table=torch.zeros(8, 4), bias_buckets=torch.zeros(5, dtype=torch.int32))
    args.update(kw)
    q, k = torch.zeros(12, 4, 16), torch.zeros(12, 2, 16)
    return ts.sigmoid_attention_varlen(q, k, k, CU, CU, 7, 7, **args)


def _paged(**kw):
    args = dict(bias_table=torch.zeros(8, 4), bias_buckets=torch.zeros(5, dtype=torch.int32))
    args.update(kw)
    cache = torch.zeros(3, 16, 2, 16)
    return ts.sigmoid_attention_paged(torch.zeros(2, 4, 16), cache, cache, torch.zeros(2, 2, dtype=torch.int32),
                                      torch.ones(2, dtype=torch.int32), torch.arange(3, dtype=torch.int32), 1, **args)


@pytest.mark.parametrize("call", [_varlen, _paged])
@pytest.mark.parametrize("kw, error, match", [
    (dict(bias_table=None), ValueError, "go together"), (dict(bias_buckets=None), ValueError, "go together"),
    (dict(bias_table=torch.zeros(8, 2)), ValueError, "bias_table must have shape"),
    (dict(bias_table=torch.zeros(0, 4)), ValueError, "bias_table must have shape"),
    (dict(bias_table=torch.zeros(32)), ValueError, "bias_table must have shape"),
    (dict(bias_table=torch.zeros(1, 1).expand(4097, 4)), ValueError, "bias_table must have shape"),
    (dict(bias_buckets=torch.zeros(4, dtype=torch.int32)), ValueError, "bias_buckets must have shape"),
    (dict(bias_buckets=torch.zeros(1, 5, dtype=torch.int32)), ValueError, "bias_buckets must have shape"),
    (dict(bias_buckets=torch.zeros(4099, dtype=torch.int32)), ValueError, "bias_buckets must have shape"),
    (dict(bias_buckets=torch.zeros(5)), ValueError, "int32 or int64"),
    (dict(bias_table=torch.zeros(8, 4, dtype=torch.float64)), RuntimeError, "unsupported bias_table dtype"),
    (dict(), RuntimeError, "gfx950"),
])
def test_bias_refusals(call, kw, error, match):
    with pytest.raises(error, match=match):
        call(**kw)


def test_bias_excludes_score_mod():
    with pytest.raises(ValueError, match="exclude each other"):
        _varlen(score_mod=torch.zeros(12))
    with pytest.raises(ValueError, match="exclude each other"):
        _paged(score_mod=torch.zeros(2, 32))


def test_paged_bias_has_no_gradient():
    with pytest.raises(RuntimeError, match="no backward"):
        _paged(bias_table=torch.zeros(8, 4, requires_grad=True))


@pytest.mark.parametrize("kw, error, match", [
    (dict(query=torch.zeros(12, 16)), ValueError, "3D tensors"),
    (dict(key=torch.zeros(11, 2, 16)), ValueError, "same tokens"),
    (dict(key=torch.zeros(12, 2, 32)), ValueError, "Head dimension mismatch"),
    (dict(angles=torch.zeros(9, 15)), ValueError, "angles must have shape"),
    (dict(angles=torch.zeros(9, 18)), ValueError, "angles must have shape"),
    (dict(angles=torch.zeros(0, 16)), ValueError, "angles must have shape"),
    (dict(angles=torch.zeros(16)), ValueError, "angles must have shape"),
    (dict(positions=torch.zeros(11, dtype=torch.int32)), ValueError, "positions must have shape"),
    (dict(positions=torch.zeros(12)), ValueError, "int32 or int64"),
    (dict(key=torch.zeros(12, 2, 16, dtype=torch.float16)), RuntimeError, "share a dtype"),
    (dict(query=torch.zeros(12, 4, 24), key=torch.zeros(12, 2, 24)), RuntimeError, "unsupported head dimension"),
    (dict(query=torch.zeros(12, 4, 16).double(), key=torch.zeros(12, 2, 16).double()), RuntimeError, "unsupported dtype"),
    (dict(), RuntimeError, "gfx950"),
])
def test_rotary_refusals(kw, error, match):
    args = dict(query=torch.zeros(12, 4, 16), key=torch.zeros(12, 2, 16), positions=torch.zeros(12, dtype=torch.int32),
                angles=torch.zeros(9, 16))
    args.update(kw)
    with pytest.raises(error, match=match):
        ts.rotary_embedding(**args)


@pytest.mark.parametrize("kw, error, match", [
    (dict(query=torch.zeros(4, 4, 16)), ValueError, "Expected query"),
    (dict(query=torch.zeros(5, 4, 32)), ValueError, "Head dimension mismatch"),
    (dict(key=torch.zeros(5, 4, 16), value=torch.zeros(5, 4, 16)), ValueError, "do not fit cache rows"),
    (dict(value=torch.zeros(4, 2, 16)), ValueError, "same shape"),
    (dict(slot_mapping=torch.zeros(4, dtype=torch.int32)), ValueError, "slot_mapping must have shape"),
    (dict(positions=torch.zeros(4, dtype=torch.int32)), ValueError, "positions must have shape"),
    (dict(angles=torch.zeros(9, 32)), ValueError, "angles must have shape"),
    (dict(query=torch.zeros(5, 4, 16, dtype=torch.float16)), RuntimeError, "share a dtype"),
    (dict(key_cache=torch.zeros(1, 16, 2, 16).expand(3, 16, 2, 16),
          value_cache=torch.zeros(1, 16, 2, 16).expand(3, 16, 2, 16)), ValueError, "must not repeat"),
    (dict(query=torch.zeros(5, 4, 16, requires_grad=True)), RuntimeError, "no backward"),
    (dict(), RuntimeError, "gfx950"),
])
def test_rotary_write_refusals(kw, error, match):
    args = dict(query=torch.zeros(5, 4, 16), key=torch.zeros(5, 2, 16), value=torch.zeros(5, 2, 16),
                key_cache=torch.zeros(3, 16, 2, 16), value_cache=torch.zeros(3, 16, 2, 16),
                slot_mapping=torch.zeros(5, dtype=torch.int32), positions=torch.zeros(5, dtype=torch.int32),
                angles=torch.zeros(9, 16))
    args.update(kw)
    with pytest.raises(error, match=match):
        ts.paged_cache_write_rotary(**args)


@pytest.mark.parametrize("name", ["query", "key", "value", "key_cache", "value_cache", "angles"])
def test_tangents_are_not_written(name):
    args = dict(query=torch.zeros(5, 4, 16), key=torch.zeros(5, 2, 16), value=torch.zeros(5, 2, 16),
                key_cache=torch.zeros(3, 16, 2, 16), value_cache=torch.zeros(3, 16, 2, 16),
                slot_mapping=torch.zeros(5, dtype=torch.int32), positions=torch.zeros(5, dtype=torch.int32),
                angles=torch.zeros(9, 16))
    with forward_ad.dual_level():
        args[name] = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            ts.paged_cache_write_rotary(**args)


# --- C ABI -----------------------------------------------------------------------------

FAKE = 1 << 20  # never dereferenced


def _set(s, **kw):
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def _problem(**kw):
    p = _set(_capi.SigattnProblem(), abi_version=_capi.ABI_VERSION, dtype=_capi.BF16, B=2, Tq=7, Tk=7, H=4, D=64, kv_heads=2,
             q_stride_t=256, q_stride_h=64, k_stride_t=128, k_stride_h=64, rows_q=12, rows_k=12, q=FAKE, k=FAKE, v=FAKE,
             bias=FAKE, scale=FAKE, cu_seqlens_q=FAKE, cu_seqlens_k=FAKE)
    return _set(p, **kw)


def _paged_problem(**kw):
    p = _set(_capi.SigattnPagedProblem(), abi_version=_capi.ABI_VERSION, dtype=_capi.BF16, B=2, H=4, kv_heads=2, D=64,
             rows_q=2, max_seqlen_q=1, num_pages=4, page_size=16, max_pages=2, q_stride_t=256, q_stride_h=64, k_stride_p=2048,
             k_stride_t=128, k_stride_h=64, table_stride=2, q=FAKE, k_cache=FAKE, v_cache=FAKE, block_table=FAKE,
             seq_lens_k=FAKE, cu_seqlens_q=FAKE, scale=0.1)
    return _set(p, **kw)


def _rel(**kw):
    return _set(_capi.SigattnRelBias(), **dict(dict(dtype=_capi.F32, num_buckets=8, max_distance=20, table=FAKE,
                                                    buckets=FAKE), **kw))


@pytest.mark.parametrize("kw, rc", [
    (dict(), 0), (dict(max_distance=0), 0), (dict(max_distance=2048), 0), (dict(num_buckets=4096), 0),
    (dict(max_distance=-1), -13), (dict(max_distance=2049), -13), (dict(num_buckets=0), -13), (dict(num_buckets=4097), -13),
    (dict(dtype=3), -2), (dict(table=None), -1), (dict(buckets=None), -1),
])
def test_rel_check(kw, rc):
    lib, r = _capi.load_library(), _rel(**kw)
    assert lib.sigattn_rel_check(ctypes.byref(_problem()), ctypes.byref(r)) == rc
    assert lib.sigattn_paged_rel_check(ctypes.byref(_paged_problem()), ctypes.byref(r)) == rc
    assert "relative bias" in lib.sigattn_strerror(-13).decode()


def test_rel_check_of_the_problem():
    lib, r = _capi.load_library(), ctypes.byref(_rel())
    for kw, rc in ((dict(score_mod=FAKE), -13), (dict(cu_seqlens_k=None, kv_heads=4), -13), (dict(H=65536, kv_heads=1), -4),
                   (dict(D=65), -3), (dict(abi_version=9), -7)):
        assert lib.sigattn_rel_check(ctypes.byref(_problem(**kw)), r) == rc, kw
    assert lib.sigattn_paged_rel_check(ctypes.byref(_paged_problem(score_mod=FAKE)), r) == -13
    assert lib.sigattn_rel_check(None, r) == lib.sigattn_rel_check(ctypes.byref(_problem()), None) == -1


def test_rel_calls_need_their_workspace():
    lib, p, r = _capi.load_library(), ctypes.byref(_problem()), ctypes.byref(_rel())
    need = lib.sigattn_rel_fwd_workspace_bytes(p, r)
    assert need >= 4 * 4 * 15  # four heads' lines, as far as seven tokens reach
    assert lib.sigattn_rel_fwd(p, r, FAKE, None, 0, None) == -10
    assert lib.sigattn_rel_fwd(p, r, FAKE, FAKE, need - 1, None) == -10
    assert lib.sigattn_rel_fwd(p, r, FAKE, FAKE + 8, need, None) == -10
    assert lib.sigattn_rel_fwd(p, r, None, FAKE, need, None) == -1
    need = lib.sigattn_rel_bwd_workspace_bytes(p, r)
    assert lib.sigattn_rel_bwd(p, r, None, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, need - 1, None) == -10
    assert lib.sigattn_rel_bwd(p, r, FAKE, None, FAKE, FAKE, FAKE, FAKE, FAKE, need, None) == -1
    pp = ctypes.byref(_paged_problem())
    need = lib.sigattn_paged_rel_fwd_workspace_bytes(pp, r)
    assert lib.sigattn_paged_rel_fwd(pp, r, FAKE, FAKE, need - 1, None) == -10
    assert lib.sigattn_paged_rel_fwd(pp, r, FAKE, None, 0, None) == -10


@pytest.mark.parametrize("dtype, D, rows", [(_capi.BF16, 64, 64), (_capi.BF16, 128, 64), (_capi.F32, 64, 32),
                                            (_capi.F32, 128, 64)])
def test_workspaces_with_and_without_a_gradient_of_the_table(dtype, D, rows):
    """A sum per block of queries, head and position; a call that wants none pays for none."""
    lib, N, H, R = _capi.load_library(), 65536, 32, 2048
    p = _problem(dtype=dtype, D=D, B=4, Tq=N, Tk=N, rows_q=N, rows_k=N, H=H, kv_heads=H, q_stride_t=H * D, q_stride_h=D,
                 k_stride_t=H * D, k_stride_h=D)
    r = _rel(max_distance=R)
    parts = (N // rows + 4) * H * (2 * R + 1) * 4
    full = lib.sigattn_rel_bwd_workspace_bytes(ctypes.byref(p), ctypes.byref(r))
    frozen = lib.sigattn_rel_bwd_frozen_workspace_bytes(ctypes.byref(p), ctypes.byref(r))
    line = lib.sigattn_rel_fwd_workspace_bytes(ctypes.byref(p), ctypes.byref(r))
    assert frozen == line < 1 << 20
    assert parts <= full - frozen - line <= parts + 256
    assert lib.sigattn_rel_bwd(ctypes.byref(p), ctypes.byref(r), None, FAKE, FAKE, FAKE, FAKE, None, FAKE, frozen - 1,
                               None) == -10
    assert lib.sigattn_rel_bwd(ctypes.byref(p), ctypes.byref(r), None, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, frozen,
                               None) == -10
    assert lib.sigattn_rel_bwd_frozen_workspace_bytes(None, ctypes.byref(r)) == 0


def _rotary(**kw):
    r = _set(_capi.SigattnRotary(), dtype=_capi.BF16, rows=3, q_heads=4, kv_heads=2, D=64, rot_dim=64, num_positions=9,
             q_stride_t=256, q_stride_h=64, k_stride_t=128, k_stride_h=64, cache_stride_p=2048, cache_stride_t=128,
             cache_stride_h=64, num_pages=4, page_size=16, q=FAKE, k=FAKE, v=FAKE, q_out=FAKE, k_out=FAKE, k_cache=FAKE,
             v_cache=FAKE, positions=FAKE, angles=FAKE, slot_mapping=FAKE)
    return _set(r, **kw)


@pytest.mark.parametrize("kw, rc", [
    (dict(dtype=7), -2), (dict(D=48), -3), (dict(rows=-1), -4), (dict(rows=1 << 31), -4), (dict(q_heads=65536), -4),
    (dict(kv_heads=-1), -4), (dict(num_positions=1 << 31), -4), (dict(rot_dim=0), -14), (dict(rot_dim=63), -14),
    (dict(rot_dim=66), -14), (dict(num_positions=0), -14), (dict(q_stride_t=-1), -5), (dict(k_stride_h=-1), -5),
    (dict(positions=None), -1), (dict(angles=None), -1), (dict(q=None), -1), (dict(q_out=None), -1), (dict(k=None), -1),
    (dict(rows=0), 0), (dict(q_heads=0, kv_heads=0), 0),
])
def test_rotary_checks(kw, rc):
    lib, r = _capi.load_library(), _rotary(**kw)
    assert lib.sigattn_rotary_apply(ctypes.byref(r), None) == rc
    assert lib.sigattn_paged_write_rotary(ctypes.byref(r), None) == rc
    assert "rot_dim" in lib.sigattn_strerror(-14).decode()


@pytest.mark.parametrize("kw, rc", [
    (dict(page_size=24), -4), (dict(page_size=8), -4), (dict(num_pages=1 << 28), -4), (dict(num_pages=-1), -4),
    (dict(cache_stride_p=-1), -5), (dict(k_cache=None), -1), (dict(v_cache=None), -1), (dict(v=None), -1),
    (dict(slot_mapping=None), -1), (dict(rows=0, v=None), 0),
])
def test_rotary_write_checks(kw, rc):
    assert _capi.load_library().sigattn_paged_write_rotary(ctypes.byref(_rotary(**kw)), None) == rc


def test_ops_trace_without_a_gpu():
    """Fake kernels: shapes and types under torch.compile's tracing."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q, k = torch.empty(12, 4, 16, dtype=torch.bfloat16), torch.empty(12, 2, 16, dtype=torch.bfloat16)
        table, buckets, i = torch.empty(8, 4), torch.empty(5, dtype=torch.int32), torch.empty(3, dtype=torch.int32)
        b, s = torch.empty(2), torch.empty(())
        o = torch.ops.myops.sigmoid_attn_varlen_rel_fwd(q, k, k, table, buckets, i, i, 7, 7, b, s, True)
        assert o.shape == q.shape and o.dtype == q.dtype
        g = torch.ops.myops.sigmoid_attn_varlen_rel_bwd(q, k, k, q, table, buckets, i, i, 7, 7, b, s, True)
        assert [t.shape for t in g] == [q.shape, k.shape, k.shape, table.shape] and g[3].dtype == table.dtype
        a, c = torch.ops.myops.rotary_embedding(q, k, i, torch.empty(9, 16), False, False)
        assert a.shape == q.shape and c.shape == k.shape
