"""Paged cache: refusals, the C ABI's checks and struct layouts, on the CPU."""

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch
from torch.autograd import forward_ad

import triton_sigmoid as ts
from triton_sigmoid import _capi

ROOT = Path(__file__).resolve().parent.parent
I32 = torch.int32


def _plan_args(**kw):
    a = dict(context_lens=torch.tensor([3, 40], dtype=I32), new_lens=torch.tensor([1, 2], dtype=I32),
             block_table=torch.full((2, 4), -1, dtype=I32), free_pages=torch.arange(8, dtype=I32), page_size=16,
             num_tokens=3)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw, match", [
    (dict(block_table=torch.zeros(4, dtype=I32)), r"block_table must have shape \(B, max_pages\)"),
    (dict(context_lens=torch.zeros(3, dtype=I32)), r"context_lens must have shape \(2,\)"),
    (dict(new_lens=torch.zeros(2, 1, dtype=I32)), r"new_lens must have shape \(2,\)"),
    (dict(free_pages=torch.zeros(2, 2, dtype=I32)), r"free_pages must have shape \(F,\)"),
    (dict(block_table=torch.zeros(2, 4, dtype=torch.int64)), "must be int32 with unit stride"),
    (dict(block_table=torch.zeros(4, 2, dtype=I32).t()), "must be int32 with unit stride"),
    (dict(block_table=torch.zeros(1, 4, dtype=I32).expand(2, 4)), "must not overlap"),
    (dict(page_size=8), "power of two"), (dict(page_size=24), "power of two"), (dict(page_size=0), "power of two"),
    (dict(num_tokens=-1), "non-negative"),
    (dict(context_lens=torch.zeros(8193, dtype=I32), new_lens=torch.zeros(8193, dtype=I32),
          block_table=torch.zeros(8193, 1, dtype=I32)), "up to 8192 requests"),
])
def test_plan_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        ts.paged_plan(**_plan_args(**kw))


def _caches(pages=4, ps=16, heads=2, D=32, dtype=torch.bfloat16):
    return torch.zeros(pages, ps, heads, D, dtype=dtype), torch.zeros(pages, ps, heads, D, dtype=dtype)


def _write_args(**kw):
    kc, vc = _caches()
    rows = torch.zeros(3, 2, 32, dtype=torch.bfloat16)
    a = dict(key=rows, value=rows, key_cache=kc, value_cache=vc, slot_mapping=torch.zeros(3, dtype=I32))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw, err, match", [
    (dict(key=torch.zeros(3, 64, dtype=torch.bfloat16)), ValueError, "3D tensors"),
    (dict(value=torch.zeros(4, 2, 32, dtype=torch.bfloat16)), ValueError, "same shape"),
    (dict(key_cache=torch.zeros(4, 16, 64, dtype=torch.bfloat16)), ValueError, "4D tensors"),
    (dict(key_cache=_caches(pages=5)[0]), ValueError, "same shape"),
    (dict(key_cache=_caches(heads=3)[0], value_cache=_caches(heads=3)[0]), ValueError, "do not fit"),
    (dict(key_cache=torch.zeros(4, 2, 16, 32, dtype=torch.bfloat16).transpose(1, 2)), ValueError, "same strides"),
    (dict(slot_mapping=torch.zeros(4, dtype=I32)), ValueError, r"slot_mapping must have shape \(3,\)"),
    (dict(key=torch.zeros(3, 2, 32)), RuntimeError, "share a dtype"),
    (dict(zip(("key_cache", "value_cache"), (t[:, :, :1].expand(-1, -1, 2, -1) for t in _caches()))), ValueError,
     "must not repeat rows"),
    (dict(key_cache=_caches(ps=24)[0], value_cache=_caches(ps=24)[0]), ValueError, "power of two"),
    (dict(zip(("key_cache", "value_cache"), _caches(dtype=torch.float64))), RuntimeError, "unsupported dtype"),
    (dict(zip(("key_cache", "value_cache"), _caches(D=48))), RuntimeError, "unsupported head dimension"),
])
def test_write_refusals(kw, err, match):
    with pytest.raises(err, match=match):
        ts.paged_cache_write(**_write_args(**kw))


def _attn_args(**kw):
    kc, vc = _caches()
    a = dict(query=torch.zeros(3, 4, 32, dtype=torch.bfloat16), key_cache=kc, value_cache=vc,
             block_table=torch.zeros(2, 3, dtype=I32), seq_lens_k=torch.ones(2, dtype=I32),
             cu_seqlens_q=torch.tensor([0, 1, 3], dtype=I32))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw, err, match", [
    (dict(query=torch.zeros(3, 128, dtype=torch.bfloat16)), ValueError, "3D tensor"),
    (dict(query=torch.zeros(3, 3, 32, dtype=torch.bfloat16)), ValueError, "Number of heads mismatch"),
    (dict(query=torch.zeros(3, 1, 32, dtype=torch.bfloat16)), ValueError, "Number of heads mismatch"),
    (dict(query=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), ValueError, "Head dimension mismatch"),
    (dict(query=torch.zeros(3, 4, 32)), RuntimeError, "share a dtype"),
    (dict(block_table=torch.zeros(3, dtype=I32)), ValueError, "block_table"),
    (dict(seq_lens_k=torch.ones(3, dtype=I32)), ValueError, r"seq_lens_k must have shape \(2,\)"),
    (dict(cu_seqlens_q=torch.zeros(2, dtype=I32)), ValueError, r"cu_seqlens_q must have shape \(3,\)"),
    (dict(score_mod=torch.zeros(2, 47)), ValueError, r"score_mod must have shape \(2, 48\)"),
    (dict(max_seqlen_q=-1), ValueError, "non-negative"),
])
def test_attention_refusals(kw, err, match):
    with pytest.raises(err, match=match):
        ts.sigmoid_attention_paged(**_attn_args(**kw))


def test_gradients_are_refused():
    q = torch.zeros(3, 4, 32, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        ts.sigmoid_attention_paged(**_attn_args(query=q))
    rows = torch.zeros(3, 2, 32, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        ts.paged_cache_write(**_write_args(key=rows))


def test_cpu_tensors_fail_loudly():
    for call in (lambda: ts.paged_plan(**_plan_args()), lambda: ts.paged_cache_write(**_write_args()),
                 lambda: ts.sigmoid_attention_paged(**_attn_args())):
        with pytest.raises(RuntimeError, match="gfx950"):
            call()


# --- C ABI ------------------------------------------------------------------------

FAKE = 1 << 20  # never dereferenced


def _problem(**kw):
    p = _capi.SigattnPagedProblem()
    p.abi_version, p.dtype = _capi.ABI_VERSION, _capi.BF16
    p.B, p.H, p.kv_heads, p.D, p.rows_q, p.max_seqlen_q = 2, 8, 2, 64, 5, 4
    p.num_pages, p.page_size, p.max_pages = 10, 16, 4
    p.q_stride_t, p.q_stride_h = 512, 64
    p.k_stride_p, p.k_stride_t, p.k_stride_h = 2048, 128, 64
    p.table_stride = 4
    p.q = p.k_cache = p.v_cache = p.block_table = p.seq_lens_k = p.cu_seqlens_q = FAKE
    p.scale = 0.125
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw, rc", [
    (dict(), 0), (dict(rows_q=0, q=None), 0), (dict(H=0), 0),
    (dict(abi_version=2), -7), (dict(dtype=3), -2), (dict(D=48), -3),
    (dict(B=-1), -4), (dict(rows_q=-1), -4), (dict(max_seqlen_q=-1), -4), (dict(page_size=8), -4),
    (dict(page_size=48), -4), (dict(num_pages=1 << 28), -4), (dict(max_pages=1 << 27), -4),
    (dict(rows_q=1 << 25, H=4096, kv_heads=4096), -4),
    (dict(kv_heads=3), -12), (dict(kv_heads=0), -12), (dict(kv_heads=16), -12),
    (dict(k_stride_t=-1), -5), (dict(table_stride=-4), -5),
    (dict(q=None), -1), (dict(block_table=None), -1), (dict(k_cache=None), -1), (dict(seq_lens_k=None), -1),
    (dict(cu_seqlens_q=None), -1), (dict(B=0, block_table=None, seq_lens_k=None, k_cache=None), 0),
    (dict(num_pages=0, k_cache=None, v_cache=None), 0), (dict(max_pages=0, block_table=None), 0),
])
def test_attention_check(kw, rc):
    assert _capi.load_library().sigattn_paged_check(ctypes.byref(_problem(**kw))) == rc


def test_attention_call_errors():
    lib = _capi.load_library()
    assert lib.sigattn_paged_check(None) == -1
    assert lib.sigattn_paged_fwd(ctypes.byref(_problem()), None, None, 0, None) == -1  # out
    assert lib.sigattn_paged_fwd(ctypes.byref(_problem(rows_q=0)), None, None, 0, None) == 0  # nothing to do
    assert lib.sigattn_paged_fwd_workspace_bytes(ctypes.byref(_problem(D=48))) == 0


@pytest.mark.parametrize("kw, rc", [
    (dict(esize=1), -2), (dict(D=20), -3), (dict(rows=-1), -4), (dict(page_size=17), -4),
    (dict(num_pages=1 << 28), -4), (dict(src_stride_t=-1), -5), (dict(k=None), -1), (dict(slot_mapping=None), -1),
    (dict(rows=0, k=None), 0), (dict(num_pages=0, k_cache=None), 0),
])
def test_write_call_errors(kw, rc):
    r = _capi.SigattnPagedRows()
    r.esize, r.rows, r.kv_heads, r.D, r.num_pages, r.page_size = 2, 3, 2, 64, 4, 16
    r.k = r.v = r.k_cache = r.v_cache = r.slot_mapping = FAKE
    for k, v in kw.items():
        setattr(r, k, v)
    assert _capi.load_library().sigattn_paged_write(ctypes.byref(r), None) == rc


@pytest.mark.parametrize("kw, rc", [
    (dict(B=-1), -4), (dict(B=8193), -4), (dict(page_size=12), -4), (dict(num_tokens=-1), -4),
    (dict(table_stride=-1), -5), (dict(cu=None), -1), (dict(table=None), -1), (dict(free=None), -1),
    (dict(slots=None), -1), (dict(needed=None), -1), (dict(max_pages=1 << 28), -4),
])
def test_plan_call_errors(kw, rc):
    a = dict(B=2, ctx=FAKE, new=FAKE, table=FAKE, table_stride=4, max_pages=4, free=FAKE, num_free=3, page_size=16,
             num_tokens=5, slots=FAKE, cu=FAKE, lens=FAKE, needed=FAKE)
    a.update(kw)
    assert _capi.load_library().sigattn_paged_plan(*a.values(), None) == rc
    assert _capi.PLAN_MAX_BATCH == 8192


def test_struct_layouts_match_the_header(tmp_path):
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    body, want = "", {}
    for name, cls in (("sigattn_paged_rows", _capi.SigattnPagedRows),
                      ("sigattn_paged_problem", _capi.SigattnPagedProblem), ("sigattn_problem", _capi.SigattnProblem)):
        for f, _ in cls._fields_:
            body += f'  printf("{name}.{f} %zu\\n", offsetof({name}, {f}));\n'
            want[f"{name}.{f}"] = getattr(cls, f).offset
        body += f'  printf("{name} %zu\\n", sizeof({name}));\n'
        want[name] = ctypes.sizeof(cls)
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "sigattn.h"\nint main(void) {\n' + body
                   + '  printf("plan %d\\n", SIGATTN_PLAN_MAX_BATCH);\n  return 0;\n}\n')
    want["plan"] = _capi.PLAN_MAX_BATCH
    subprocess.run([cc, f"-I{ROOT / 'include'}", str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    got = {k: int(v) for k, v in (line.split() for line in out.splitlines())}
    assert got == want


@pytest.mark.parametrize("name", ["query", "key_cache", "value_cache", "score_mod"])
def test_tangents_are_refused(name):
    """Forward mode has no rule here: a tangent is refused, not dropped."""
    args = _attn_args(score_mod=torch.zeros(2, 48))
    with forward_ad.dual_level():
        args[name] = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        for call in (ts.sigmoid_attention_paged, torch.no_grad()(ts.sigmoid_attention_paged)):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call(**args)
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            torch.ops.myops.sigmoid_attn_paged_fwd(
                args["query"], args["key_cache"], args["value_cache"], args["block_table"], args["seq_lens_k"],
                args["cu_seqlens_q"], 2, args["score_mod"], 0.5, None, False)


@pytest.mark.parametrize("name", ["key", "value", "key_cache", "value_cache"])
def test_tangents_are_not_written(name):
    args = _write_args()
    with forward_ad.dual_level():
        args[name] = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            ts.paged_cache_write(**args)


def test_functional_forward_mode_is_refused():
    args = _attn_args()
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(lambda q: ts.sigmoid_attention_paged(**dict(args, query=q)), (args["query"],),
                       (torch.ones_like(args["query"]),))
