"""Grouped heads: refusals and the C ABI's checks, on the CPU."""

import ctypes

import pytest
import torch

import triton_sigmoid as ts
from triton_sigmoid import _capi

CU = torch.tensor([0, 5, 12], dtype=torch.int32)


@pytest.mark.parametrize("H, Hk, Hv", [(4, 3, 3), (2, 4, 4), (4, 2, 4), (4, 2, 1), (4, 0, 0)])
def test_heads_that_do_not_group(H, Hk, Hv):
    q, k, v = (torch.zeros(12, h, 16) for h in (H, Hk, Hv))
    with pytest.raises(ValueError, match="Number of heads mismatch"):
        ts.sigmoid_attention_varlen(q, k, v, CU, CU)


@pytest.mark.parametrize("fn", [ts.sigmoid_attention, ts.sigmoid_attention_padded])
def test_the_other_layouts_keep_one_head_each(fn):
    with pytest.raises(ValueError, match="Number of heads mismatch"):
        fn(torch.zeros(1, 8, 4, 16), torch.zeros(1, 8, 2, 16), torch.zeros(1, 8, 2, 16))


def test_grouped_cpu_tensors_fail_loudly():
    with pytest.raises(RuntimeError, match="gfx950"):
        ts.sigmoid_attention_varlen(torch.zeros(12, 4, 16), torch.zeros(12, 2, 16), torch.zeros(12, 2, 16), CU, CU)


def _problem(**kw):
    p = _capi.SigattnProblem()
    p.abi_version, p.dtype = _capi.ABI_VERSION, _capi.BF16
    p.B, p.Tq, p.Tk, p.H, p.D = 2, 7, 7, 4, 64
    p.q_stride_t, p.q_stride_h, p.k_stride_t, p.k_stride_h = 256, 64, 128, 64
    p.rows_q = p.rows_k = 12
    fake = 1 << 20  # never dereferenced
    p.q = p.k = p.v = p.bias = p.scale = p.cu_seqlens_q = p.cu_seqlens_k = fake
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw, rc", [
    (dict(kv_heads=2), 0), (dict(kv_heads=0), 0), (dict(kv_heads=4), 0), (dict(kv_heads=1), 0),
    (dict(kv_heads=3), -12), (dict(kv_heads=8), -12), (dict(kv_heads=-2), -12),
    (dict(kv_heads=2, cu_seqlens_q=None, cu_seqlens_k=None), -12),
    (dict(kv_heads=2, cu_seqlens_k=None), -12),
    (dict(kv_heads=3, abi_version=2), 0),  # version 2 ends before the field
    (dict(abi_version=1), -7), (dict(abi_version=4), -7),
])
def test_check(kw, rc):
    lib = _capi.load_library()
    assert lib.sigattn_check(ctypes.byref(_problem(**kw))) == rc
    assert "kv_heads" in lib.sigattn_strerror(-12).decode()


def test_workspace_policy_takes_whole_groups(monkeypatch):
    """The Python layer's two-pass workspace: the whole problem's within the
    limit, else passes of whole K / V heads of one size that fill the GPU."""
    lib = _capi.load_library()
    p = _problem(D=128, Tq=4096, Tk=4096, H=24, kv_heads=4, rows_q=8192, rows_k=8192)
    full = lib.sigattn_bwd_workspace_bytes(ctypes.byref(p))
    per_head = full // 24
    monkeypatch.setattr(_capi, "_compute_units", lambda dev: 8)
    for heads, want in ((5, 0), (6, 6), (11, 6), (12, 12), (17, 12), (18, 12), (23, 12), (24, 24)):
        monkeypatch.setattr(_capi, "bwd_workspace_limit", lambda grouped: heads * per_head)
        assert _capi.bwd_workspace_bytes(lib, p, torch.device("cuda:0")) == want * per_head
    monkeypatch.setattr(_capi, "_compute_units", lambda dev: 64)  # 64 key blocks a K / V head
    for heads, want in ((6, 0), (12, 12)):
        monkeypatch.setattr(_capi, "bwd_workspace_limit", lambda grouped: heads * per_head)
        assert _capi.bwd_workspace_bytes(lib, p, torch.device("cuda:0")) == want * per_head


def test_workspace_limit(monkeypatch):
    monkeypatch.delenv("SIGATTN_BWD_WORKSPACE_MB", raising=False)
    assert _capi.bwd_workspace_limit() == 2048 << 20 and _capi.bwd_workspace_limit(True) == 8192 << 20
    monkeypatch.setenv("SIGATTN_BWD_WORKSPACE_MB", "64")
    assert _capi.bwd_workspace_limit() == _capi.bwd_workspace_limit(True) == 64 << 20
