"""Paged key/value cache: its bookkeeping, its writer, and sigmoid attention
of new tokens over it.

The reference has no cache; its padded forward with short queries
(sigmoid_triton_padded.py:853-1010) is what a decoding step computes.  Here
the keys and values of every sequence live in pages of `page_size` tokens
anywhere in two caches [num_pages, page_size, H_kv, D], listed in a block table
[B, max_pages]; one serving step is

    plan = paged_plan(context_lens, new_lens, block_table, free_pages, page_size, num_tokens)
    for each layer:
        paged_cache_write(key, value, key_cache, value_cache, plan.slot_mapping)
        out = sigmoid_attention_paged(query, key_cache, value_cache, plan.block_table, plan.seq_lens,
                                      plan.cu_seqlens, max_new, is_causal=True)

with query / key / value the packed rows of the step's new tokens, one for
each decoding request and many for a prompt.  Nothing synchronises the host, so
a step can be captured into a graph and replayed on other lengths.

Ops: `myops::paged_plan`, `myops::paged_cache_write`,
`myops::sigmoid_attn_paged_fwd` and `myops::sigmoid_attn_paged_rel_fwd` (torch.compile traces them without graph
breaks).  Forward only.
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _capi


class PagedPlan(NamedTuple):
    """What paged_plan returns; int32 tensors on the requests' device."""

    block_table: torch.Tensor  # the table given, with the new pages entered
    slot_mapping: torch.Tensor  # [num_tokens] slot of each packed token row, -1: none
    cu_seqlens: torch.Tensor  # [B + 1] offsets of the requests' new tokens
    seq_lens: torch.Tensor  # [B] tokens in the cache after the step
    pages_needed: torch.Tensor  # [] pages the step takes from free_pages


def _page_size_ok(page_size: int) -> bool:
    return 16 <= page_size <= 1 << 20 and page_size & (page_size - 1) == 0


def _check_page_size(page_size: int) -> None:
    if not _page_size_ok(page_size):
        raise ValueError(f"page_size must be a power of two, 16 at least, got {page_size}")


def _no_grad(what: str, *tensors: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no backward: call it under torch.no_grad() or on detached tensors")


def _no_tangent(what: str, *tensors: Optional[torch.Tensor]) -> None:
    # Where the kernels are called, so that the custom ops refuse them too: a
    # dual tensor's requires_grad is False, and no_grad does not stop forward mode.
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative: call it on tensors without tangents")


def _quick():
    """The C++ module for eager calls on canonical arguments, or None."""
    if torch.compiler.is_compiling():
        return None
    return _capi.quick_module if _capi.quick_module is not None else _bind()


def _bind():
    # The first call binds the module (which then serves every entry point);
    # without the library the call fails with its own error further on.
    if not _capi.LIB_PATH.exists():
        return None
    _capi.autograd_node()
    return _capi.quick_module


def _unit(t: torch.Tensor) -> torch.Tensor:
    """t with unit stride along its last dim."""
    return t if t.stride(-1) == 1 else t.contiguous()


def _ints(t: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """t as contiguous int32 on `dev`; wider integers are clamped, not wrapped."""
    if t.dtype == torch.int64:
        t = t.clamp(-(1 << 31), (1 << 31) - 1)
    return _capi._as(t, torch.int32, dev)


def _changed(*tensors: torch.Tensor) -> None:
    """Tells autograd of tensors that were changed in place."""
    for t in tensors:
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


# --- plan -----------------------------------------------------------------------

def _plan(context_lens, new_lens, block_table, free_pages, page_size, num_tokens):
    lib = _capi.load_library()
    _capi._check_device(block_table)
    dev = block_table.device
    context_lens, new_lens, free_pages = (_ints(t, dev) for t in (context_lens, new_lens, free_pages))
    B = block_table.shape[0]
    slots = torch.empty(num_tokens, dtype=torch.int32, device=dev)
    cu = torch.empty(B + 1, dtype=torch.int32, device=dev)
    lens = torch.empty(B, dtype=torch.int32, device=dev)
    needed = torch.empty((), dtype=torch.int32, device=dev)
    _capi._on_device(dev, lambda stream: _capi._raise(lib.sigattn_paged_plan(
        B, context_lens.data_ptr(), new_lens.data_ptr(), block_table.data_ptr(), block_table.stride(0),
        block_table.shape[1], free_pages.data_ptr(), free_pages.numel(), page_size, num_tokens, slots.data_ptr(),
        cu.data_ptr(), lens.data_ptr(), needed.data_ptr(), stream), "sigattn_paged_plan"))
    return slots, cu, lens, needed


@torch.library.custom_op("myops::paged_plan", mutates_args=("block_table",))
def paged_plan_op(context_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor,
                  free_pages: torch.Tensor, page_size: int, num_tokens: int
                  ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(slot_mapping, cu_seqlens, seq_lens, pages_needed); enters pages into block_table."""
    return _plan(context_lens, new_lens, block_table, free_pages, page_size, num_tokens)


@paged_plan_op.register_fake
def _(context_lens, new_lens, block_table, free_pages, page_size, num_tokens):
    B = block_table.shape[0]
    new = lambda *n: block_table.new_empty(n, dtype=torch.int32)  # noqa: E731
    return new(num_tokens), new(B + 1), new(B), new()


def paged_plan(
    context_lens: torch.Tensor,
    new_lens: torch.Tensor,
    block_table: torch.Tensor,
    free_pages: torch.Tensor,
    page_size: int,
    num_tokens: int,
) -> PagedPlan:
    """Pages and slots of one serving step's new tokens, on the device.

    Request b has context_lens[b] tokens in the cache and adds new_lens[b].
    The pages it needs beyond those it holds (ceil(context / page_size)) are
    taken from free_pages, in request order, and entered into block_table.

    Args:
        context_lens / new_lens: [B] integers (negative ones count as 0).
        block_table: int32 [B, max_pages], changed in place; entries outside
            the new pages stay as they are.
        free_pages: [F] ids of free pages; the step takes the first
            pages_needed of them (the list itself is not changed).
        page_size: tokens per page, a power of two, 16 at least.
        num_tokens: rows of the step's packed tokens, at least the sum of
            new_lens for every token to get a slot; rows past the last request
            get slot -1 (a batch of fixed size, as a captured graph has).

    Returns:
        PagedPlan.  If pages_needed is more than F, the last requests' missing
        pages are -1 in the table and their tokens' slots -1: check it before
        the plan is relied on.  A request that needs more than max_pages pages
        gets no slots for the tokens past them.  Up to 8192 requests; sums of
        lengths have to fit 31 bits.
    """
    quick = _quick()
    if quick is not None:
        got = quick.quick_plan(context_lens, new_lens, block_table, free_pages, page_size, num_tokens)
        if got is not None:
            return PagedPlan(block_table, *got)
    if block_table.dim() != 2:
        raise ValueError(f"block_table must have shape (B, max_pages), got {tuple(block_table.shape)}")
    B = block_table.shape[0]
    for name, t in (("context_lens", context_lens), ("new_lens", new_lens)):
        if t.shape != (B,):
            raise ValueError(f"{name} must have shape ({B},), got {tuple(t.shape)}")
    if free_pages.dim() != 1:
        raise ValueError(f"free_pages must have shape (F,), got {tuple(free_pages.shape)}")
    if block_table.dtype != torch.int32 or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError("block_table must be int32 with unit stride along its rows (it is changed in place)")
    if B > 1 and block_table.stride(0) < block_table.shape[1]:
        raise ValueError("block_table rows must not overlap (it is changed in place)")
    _check_page_size(page_size)
    if num_tokens < 0:
        raise ValueError(f"num_tokens must be non-negative, got {num_tokens}")
    if B > _capi.PLAN_MAX_BATCH:
        raise ValueError(f"paged_plan takes up to {_capi.PLAN_MAX_BATCH} requests, got {B}")
    if torch.compiler.is_compiling():
        got = paged_plan_op(context_lens, new_lens, block_table, free_pages, page_size, num_tokens)
    else:
        got = _plan(context_lens, new_lens, block_table, free_pages, page_size, num_tokens)
        _changed(block_table)
    return PagedPlan(block_table, *got)


# --- writer -----------------------------------------------------------------------

def _write(key, value, key_cache, value_cache, slot_mapping):
    _no_tangent("paged_cache_write", key, value, key_cache, value_cache)
    lib = _capi.load_library()
    _capi._check_device(key_cache)
    dev = key_cache.device
    for name, t in (("key", key), ("value", value), ("value_cache", value_cache)):
        if t.device != dev:
            raise RuntimeError(f"{name} is on {t.device}, expected {dev}")
    key, value = _unit(key), _unit(value)
    if key.stride() != value.stride():
        key, value = key.contiguous(), value.contiguous()
    slot_mapping = _ints(slot_mapping, dev)
    r = _capi.SigattnPagedRows()
    r.esize = key.element_size()
    r.rows, r.kv_heads, r.D = key.shape
    r.src_stride_t, r.src_stride_h = key.stride(0), key.stride(1)
    r.cache_stride_p, r.cache_stride_t, r.cache_stride_h = key_cache.stride()[:3]
    r.num_pages, r.page_size = key_cache.shape[:2]
    r.k, r.v, r.k_cache, r.v_cache = key.data_ptr(), value.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr()
    r.slot_mapping = slot_mapping.data_ptr()
    _capi._on_device(dev, lambda stream: _capi._raise(lib.sigattn_paged_write(ctypes.byref(r), stream),
                                                      "sigattn_paged_write"))


@torch.library.custom_op("myops::paged_cache_write", mutates_args=("key_cache", "value_cache"))
def paged_cache_write_op(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                         slot_mapping: torch.Tensor) -> None:
    """Rows of key and value into the caches' slots."""
    _write(key, value, key_cache, value_cache, slot_mapping)


@paged_cache_write_op.register_fake
def _(key, value, key_cache, value_cache, slot_mapping):
    return None


def _check_caches(key_cache: torch.Tensor, value_cache: torch.Tensor) -> None:
    if key_cache.dim() != 4 or value_cache.dim() != 4:
        raise ValueError("Expected key_cache and value_cache to be 4D tensors (num_pages, page_size, H_kv, D)")
    if key_cache.shape != value_cache.shape:
        raise ValueError(f"key_cache and value_cache must have the same shape, got {tuple(key_cache.shape)} and "
                         f"{tuple(value_cache.shape)}")
    if key_cache.stride() != value_cache.stride() or key_cache.stride(3) != 1:
        raise ValueError("key_cache and value_cache must have the same strides, and stride 1 along D, got "
                         f"{key_cache.stride()} and {value_cache.stride()}")
    if key_cache.dtype != value_cache.dtype:
        raise RuntimeError(f"key_cache and value_cache must share a dtype, got {key_cache.dtype}, {value_cache.dtype}")
    if key_cache.dtype not in _capi._DTYPE_CODE:
        raise RuntimeError(f"unsupported dtype {key_cache.dtype}; expected float16, bfloat16 or float32")
    if key_cache.shape[3] not in (16, 32, 64, 128):
        raise RuntimeError(f"unsupported head dimension {key_cache.shape[3]} (expected 16, 32, 64 or 128)")
    _check_page_size(key_cache.shape[1])


def _check_write(key, value, key_cache, value_cache, slot_mapping) -> None:
    _check_caches(key_cache, value_cache)
    if any(n > 1 and s == 0 for n, s in zip(key_cache.shape[:3], key_cache.stride())):
        raise ValueError(f"the caches must not repeat rows (they are changed in place), got strides "
                         f"{key_cache.stride()}")
    if key.dim() != 3 or value.dim() != 3:
        raise ValueError("Expected key and value to be 3D tensors (total_tokens, H_kv, D)")
    if key.shape != value.shape:
        raise ValueError(f"key and value must have the same shape, got {tuple(key.shape)} and {tuple(value.shape)}")
    if key.shape[1:] != key_cache.shape[2:]:
        raise ValueError(f"key rows {tuple(key.shape[1:])} do not fit cache rows {tuple(key_cache.shape[2:])}")
    if slot_mapping.shape != (key.shape[0],):
        raise ValueError(f"slot_mapping must have shape ({key.shape[0]},), got {tuple(slot_mapping.shape)}")
    if key.dtype != key_cache.dtype or value.dtype != key_cache.dtype:
        raise RuntimeError(f"key, value and the caches must share a dtype, got {key.dtype}, {value.dtype}, "
                           f"{key_cache.dtype}")


def paged_cache_write(
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
) -> None:
    """Writes the packed rows of a step's new tokens into the paged caches.

    Args:
        key, value: [N, H_kv, D].
        key_cache, value_cache: [num_pages, page_size, H_kv, D] of the same
            dtype, shape and strides (pages, tokens and heads may be strided,
            so [num_pages, H_kv, page_size, D] buffers are written through a
            transposed view); changed in place.
        slot_mapping: [N] slot page * page_size + row of each token, as
            paged_plan gives it; rows with a slot outside the cache (-1) are not
            written.  The slots of one call have to be distinct: of two rows
            with one slot either may stay, or pieces of both.
    """
    quick = _quick()
    if quick is not None and quick.quick_write(key, value, key_cache, value_cache, slot_mapping):
        return
    _check_write(key, value, key_cache, value_cache, slot_mapping)
    _no_grad("paged_cache_write", key, value, key_cache, value_cache)
    if torch.compiler.is_compiling():
        paged_cache_write_op(key, value, key_cache, value_cache, slot_mapping)
    else:
        _write(key, value, key_cache, value_cache, slot_mapping)
        _changed(key_cache, value_cache)


# --- attention ----------------------------------------------------------------------

def _attend(query, key_cache, value_cache, block_table, seq_lens_k, cu_seqlens_q, max_seqlen_q, score_mod, scale,
            bias, is_causal, rel=None):
    """bias None: -log(key length).  rel: (bias_table, bias_buckets)."""
    _no_tangent("sigmoid_attention_paged", query, key_cache, value_cache, score_mod, *(rel or ())[:1])
    lib = _capi.load_library()
    _capi._check_device(query)
    dev = query.device
    for name, t in (("key_cache", key_cache), ("value_cache", value_cache)):
        if t.device != dev:
            raise RuntimeError(f"{name} is on {t.device}, expected {dev}")
    query = _unit(query)
    seq_lens_k, cu_seqlens_q = (_ints(t, dev) for t in (seq_lens_k, cu_seqlens_q))
    if block_table.dtype != torch.int32 or block_table.device != dev or (
            block_table.shape[1] > 1 and block_table.stride(1) != 1):
        block_table = _ints(block_table, dev)
    score_mod = _capi._as(score_mod, torch.float32, dev)
    out = torch.empty(query.shape, dtype=query.dtype, device=dev)
    if out.numel() == 0:
        return out
    p = _capi.SigattnPagedProblem()
    p.abi_version, p.dtype = _capi.ABI_VERSION, _capi._DTYPE_CODE[query.dtype]
    p.rows_q, p.H, p.D = query.shape
    p.num_pages, p.page_size, p.kv_heads = key_cache.shape[:3]
    p.B, p.max_pages = block_table.shape
    p.max_seqlen_q = max_seqlen_q
    p.q_stride_t, p.q_stride_h = query.stride(0), query.stride(1)
    p.k_stride_p, p.k_stride_t, p.k_stride_h = key_cache.stride()[:3]
    p.table_stride = block_table.stride(0)
    p.q, p.k_cache, p.v_cache = query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr()
    p.block_table, p.seq_lens_k, p.cu_seqlens_q = (block_table.data_ptr(), seq_lens_k.data_ptr(),
                                                   cu_seqlens_q.data_ptr())
    if score_mod is not None:
        p.score_mod, p.mod_stride = score_mod.data_ptr(), score_mod.stride(0)
    p.scale, p.causal = scale, 1 if is_causal else 0
    if bias is not None:
        p.bias, p.own_bias = bias, 1

    def run(stream):
        if rel is not None:
            r, *kept = _capi.rel_bias(*rel, dev)
            nbytes = int(lib.sigattn_paged_rel_fwd_workspace_bytes(ctypes.byref(p), ctypes.byref(r)))
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            _capi._raise(lib.sigattn_paged_rel_fwd(ctypes.byref(p), ctypes.byref(r), out.data_ptr(), ws.data_ptr(),
                                                   nbytes, stream), "sigattn_paged_rel_fwd")
            return
        nbytes = int(lib.sigattn_paged_fwd_workspace_bytes(ctypes.byref(p)))
        ws, nbytes = _capi._bwd_workspace(nbytes, dev)  # without it: unsplit
        _capi._raise(lib.sigattn_paged_fwd(ctypes.byref(p), out.data_ptr(), _capi._ptr(ws), nbytes, stream),
                     "sigattn_paged_fwd")

    _capi._on_device(dev, run)
    return out


@torch.library.custom_op("myops::sigmoid_attn_paged_fwd", mutates_args=())
def sigmoid_attn_paged_fwd_op(
    Q: torch.Tensor,
    K_cache: torch.Tensor,
    V_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens_k: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    max_seqlen_q: int,
    score_mod: Optional[torch.Tensor],
    sm_scale: float,
    bias: Optional[float],
    is_causal: bool,
) -> torch.Tensor:
    """Forward over a paged cache."""
    return _attend(Q, K_cache, V_cache, block_table, seq_lens_k, cu_seqlens_q, max_seqlen_q, score_mod, sm_scale, bias,
                   is_causal)


@sigmoid_attn_paged_fwd_op.register_fake
def _(Q, K_cache, V_cache, block_table, seq_lens_k, cu_seqlens_q, max_seqlen_q, score_mod, sm_scale, bias, is_causal):
    return Q.new_empty(Q.shape)


@torch.library.custom_op("myops::sigmoid_attn_paged_rel_fwd", mutates_args=())
def sigmoid_attn_paged_rel_fwd_op(
    Q: torch.Tensor,
    K_cache: torch.Tensor,
    V_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens_k: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    max_seqlen_q: int,
    bias_table: torch.Tensor,
    bias_buckets: torch.Tensor,
    sm_scale: float,
    bias: Optional[float],
    is_causal: bool,
) -> torch.Tensor:
    """Forward over a paged cache with the learned bias by relative position."""
    return _attend(Q, K_cache, V_cache, block_table, seq_lens_k, cu_seqlens_q, max_seqlen_q, None, sm_scale, bias,
                   is_causal, (bias_table, bias_buckets))


@sigmoid_attn_paged_rel_fwd_op.register_fake
def _(Q, K_cache, V_cache, block_table, seq_lens_k, cu_seqlens_q, max_seqlen_q, bias_table, bias_buckets, sm_scale, bias,
      is_causal):
    return Q.new_empty(Q.shape)


def sigmoid_attention_paged(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens_k: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    max_seqlen_q: Optional[int] = None,
    is_causal: bool = False,
    scale: Optional[float] = None,
    sigmoid_bias: Optional[float] = None,
    score_mod: Optional[torch.Tensor] = None,
    bias_table: Optional[torch.Tensor] = None,
    bias_buckets: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Sigmoid attention of new tokens over a paged cache that holds them already.

    output = sigmoid(Q·Kᵀ·scale + sigmoid_bias + score_mod[k_idx]) · V over the
    keys of each sequence; with bias_table, that of the relative position
    (k_idx - seq_lens_k + n - i) is added.

    Args:
        query: [N, H, D] packed new tokens: sequence b's are rows
            cu_seqlens_q[b] .. cu_seqlens_q[b+1]-1, the last of its
            seq_lens_k[b] tokens.
        key_cache, value_cache: [num_pages, page_size, H_kv, D] of the query's
            dtype and the same strides (stride 1 along D), page_size a power
            of two from 16 on; H a multiple of H_kv, query head h reads head
            h // (H // H_kv).
        block_table: [B, max_pages] page of tokens j * page_size .. of each
            sequence; entries past a sequence's length are not read.  Pages
            outside the cache (-1) hold no keys: their positions add nothing.
        seq_lens_k: [B] tokens of each sequence in the cache, its new ones
            among them (clamped to [0, max_pages * page_size]).
        cu_seqlens_q: [B + 1] non-decreasing offsets, cu[0] = 0.
        max_seqlen_q: most new tokens of a sequence (a longer one is cut to
            its first max_seqlen_q rows, whose places among the keys then
            end seq_lens_k too); None takes N.  It picks the kernels and sizes
            the workspace, so give it for decoding.
        is_causal: query i of n new tokens sees keys up to position
            seq_lens_k - n + i (bottom-right: the last query sees every key); a
            row whose position is negative sees none and is zeros.
        scale: default 1/sqrt(D).
        sigmoid_bias: default -log(seq_lens_k[b]) per sequence.
        score_mod: optional [B, max_pages * page_size] per-key term by position
            (no NaN below seq_lens_k).
        bias_table, bias_buckets: the learned bias by relative position, as
            sigmoid_attention_varlen takes it (not with score_mod); query i of n
            sits at position seq_lens_k - n + i.

    Returns:
        [N, H, D] output, contiguous.  Rows outside every sequence are zeros.
        Slots of the cache past a sequence's length are never read; the query,
        and keys and values of a sequence itself, have to be finite.  Deterministic.
        Forward only: tensors that ask for a gradient (under grad mode) or
        carry a forward-mode tangent are refused.
    """
    quick = _quick()
    if quick is not None:
        out = quick.quick_paged(query, key_cache, value_cache, block_table, seq_lens_k, cu_seqlens_q, max_seqlen_q,
                                is_causal, scale, sigmoid_bias, score_mod, bias_table, bias_buckets)
        if out is not None:
            return out
    if query.dim() != 3:
        raise ValueError("Expected query to be a 3D tensor (total_tokens, H, D)")
    _check_caches(key_cache, value_cache)
    N, H, D = query.shape
    H_kv = key_cache.shape[2]
    if D != key_cache.shape[3]:
        raise ValueError(f"Head dimension mismatch: Q={D}, cache={key_cache.shape[3]}")
    if H != H_kv and (H_kv == 0 or H % H_kv):
        raise ValueError(f"Number of heads mismatch: Q={H}, cache={H_kv}")
    if block_table.dim() != 2:
        raise ValueError(f"block_table must have shape (B, max_pages), got {tuple(block_table.shape)}")
    B, max_pages = block_table.shape
    if seq_lens_k.shape != (B,):
        raise ValueError(f"seq_lens_k must have shape ({B},), got {tuple(seq_lens_k.shape)}")
    if cu_seqlens_q.shape != (B + 1,):
        raise ValueError(f"cu_seqlens_q must have shape ({B + 1},), got {tuple(cu_seqlens_q.shape)}")
    if score_mod is not None and score_mod.shape != (B, max_pages * key_cache.shape[1]):
        raise ValueError(f"score_mod must have shape ({B}, {max_pages * key_cache.shape[1]}), got "
                         f"{tuple(score_mod.shape)}")
    if max_seqlen_q is None:
        max_seqlen_q = N
    elif max_seqlen_q < 0:
        raise ValueError(f"max_seqlen_q must be non-negative, got {max_seqlen_q}")
    if query.dtype != key_cache.dtype:
        raise RuntimeError(f"query and the caches must share a dtype, got {query.dtype}, {key_cache.dtype}")
    rel = _capi.check_rel(bias_table, bias_buckets, H, score_mod)
    _no_grad("sigmoid_attention_paged", query, key_cache, value_cache, score_mod, bias_table)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    bias = None if sigmoid_bias is None else float(sigmoid_bias)
    if rel is not None and torch.compiler.is_compiling():
        return sigmoid_attn_paged_rel_fwd_op(query, key_cache, value_cache, block_table, seq_lens_k, cu_seqlens_q,
                                             int(max_seqlen_q), *rel, scale, bias, is_causal)
    if torch.compiler.is_compiling():
        return sigmoid_attn_paged_fwd_op(query, key_cache, value_cache, block_table, seq_lens_k, cu_seqlens_q,
                                         int(max_seqlen_q), score_mod, scale, bias, is_causal)
    return _attend(query, key_cache, value_cache, block_table, seq_lens_k, cu_seqlens_q, max_seqlen_q, score_mod, scale,
                   bias, is_causal, rel)
