"""Positions in sigmoid attention: the learned bias by buckets of the relative
position, and rotary embedding.

The reference has neither (its only additive term is score_mod, per key and
without a gradient).  The bias belongs to `sigmoid_attention_varlen` (training)
and `sigmoid_attention_paged` (serving), which take

    bias_table    [num_buckets, H] learned values
    bias_buckets  [2 R + 1] bucket of each relative position -R .. R (key minus
                  query; farther keys take the ends' buckets),
                  e.g. relative_position_buckets(32, 128, bidirectional=True)

and add bias_table[bias_buckets[R + j - i], h] to the score of query i and key j.

Rotary embedding turns pairs of a head's columns by angles that grow with the
position: `rotary_embedding` for queries and keys in training (its backward turns
by the negative angles), `paged_cache_write_rotary` for a serving step, whose keys
turn on their way into the paged cache:

    angles = rotary_table(max_positions, head_dim)                 # once
    q, k = rotary_embedding(q, k, positions, angles)               # training
    q = paged_cache_write_rotary(q, k, v, key_cache, value_cache,  # serving, per layer
                                 plan.slot_mapping, positions, angles)

Ops: `myops::rotary_embedding` and `myops::paged_cache_write_rotary` (torch.compile
traces them without graph breaks).
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _capi
from .sigmoid_paged import _changed, _check_write, _ints, _no_grad, _no_tangent, _quick, _unit


# --- tables ---------------------------------------------------------------------

def relative_position_buckets(
    num_buckets: int = 32,
    max_distance: int = 128,
    bidirectional: bool = True,
    device: Optional[torch.device] = None,
) -> torch.Tensor:
    """Buckets [2 max_distance + 1] (int32) of the relative positions
    -max_distance .. max_distance (key minus query), for `bias_buckets`.

    One direction has n buckets: num_buckets, or half of them each for keys up to
    the query and after it (bidirectional; else keys after the query share bucket
    0 with the query's own).  Its first n // 2 are for one distance each, the others
    logarithmic: distance d >= n // 2 has bucket
    n // 2 + floor(log(d / (n // 2)) / log(max_distance / (n // 2)) * (n - n // 2)),
    n - 1 at most -- in whole numbers, so that no border depends on rounding.
    """
    n = num_buckets // 2 if bidirectional else num_buckets
    near = n // 2
    if near < 1 or (bidirectional and num_buckets % 2):
        raise ValueError(f"num_buckets must be {'even and 4' if bidirectional else '2'} at least, got {num_buckets}")
    if max_distance <= near or max_distance > _capi.REL_MAX_DISTANCE:
        raise ValueError(f"max_distance must lie above {near} (the buckets of one distance) and up to "
                         f"{_capi.REL_MAX_DISTANCE}, got {max_distance}")
    one, i, m = list(range(near)), 0, n - near
    for d in range(near, max_distance + 1):
        # (d / near)^m >= (max_distance / near)^(i + 1)
        while i < m - 1 and d ** m * near ** (i + 1) >= max_distance ** (i + 1) * near ** m:
            i += 1
        one.append(near + i)
    after = [n + u for u in one[1:]] if bidirectional else [0] * max_distance
    return torch.tensor(one[::-1] + after, dtype=torch.int32, device=device)


def rotary_table(
    num_positions: int,
    rot_dim: int,
    base: float = 10000.0,
    device: Optional[torch.device] = None,
) -> torch.Tensor:
    """Angles [num_positions, rot_dim] (fp32) of the rotary functions: row p has
    the cosines of p * base**(-2 i / rot_dim), i < rot_dim / 2, then their sines.
    Computed in fp64, so that far positions keep their angles."""
    if num_positions < 1 or rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rotary_table needs positions and an even rot_dim, got {num_positions} and {rot_dim}")
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device)
    angle = torch.arange(num_positions, dtype=torch.float64, device=device)[:, None] * base ** (-i / rot_dim)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


# --- rotary embedding -------------------------------------------------------------

def _rotary(q, k, positions, angles, interleaved, inverse=False) -> "_capi.SigattnRotary":
    """The C struct over [N, heads, D] tensors of unit stride along D."""
    r = _capi.SigattnRotary()
    r.dtype = _capi._DTYPE_CODE[q.dtype]
    r.interleaved, r.inverse = int(interleaved), int(inverse)
    r.rows, r.q_heads, r.D = q.shape
    r.kv_heads = k.shape[1]
    r.num_positions, r.rot_dim = angles.shape
    r.q_stride_t, r.q_stride_h = q.stride(0), q.stride(1)
    r.k_stride_t, r.k_stride_h = k.stride(0), k.stride(1)
    r.q, r.k = q.data_ptr(), k.data_ptr()
    r.positions, r.angles = positions.data_ptr(), angles.data_ptr()
    return r


def _on(dev, **tensors) -> None:
    for name, t in tensors.items():
        if t.device != dev:
            raise RuntimeError(f"{name} is on {t.device}, expected {dev}")


def _apply(query, key, positions, angles, interleaved, inverse):
    """Turned copies of query and key [N, heads, D], contiguous."""
    lib = _capi.load_library()
    _capi._check_device(query)
    dev = query.device
    _on(dev, key=key)
    query, key = _unit(query), _unit(key)
    positions, angles = _ints(positions, dev), _capi._as(angles, torch.float32, dev)
    q, k = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (query, key))
    r = _rotary(query, key, positions, angles, interleaved, inverse)
    r.q_out, r.k_out = q.data_ptr(), k.data_ptr()
    _capi._on_device(dev, lambda stream: _capi._raise(lib.sigattn_rotary_apply(ctypes.byref(r), stream),
                                                      "sigattn_rotary_apply"))
    return q, k


@torch.library.custom_op("myops::rotary_embedding", mutates_args=())
def rotary_embedding_op(query: torch.Tensor, key: torch.Tensor, positions: torch.Tensor, angles: torch.Tensor,
                        interleaved: bool, inverse: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """query and key [N, heads, D] turned by (inverse: back by) their positions' angles."""
    return _apply(query, key, positions, angles, interleaved, inverse)


@rotary_embedding_op.register_fake
def _(query, key, positions, angles, interleaved, inverse):
    return query.new_empty(query.shape), key.new_empty(key.shape)


def _rotary_setup(ctx, inputs, output):
    _, _, positions, angles, ctx.interleaved, ctx.inverse = inputs
    ctx.save_for_backward(positions, angles)


def _rotary_backward(ctx, dq, dk):
    # A rotation's transpose is the rotation back.
    positions, angles = ctx.saved_tensors
    dq, dk = rotary_embedding_op(dq, dk, positions, angles, ctx.interleaved, not ctx.inverse)
    return dq, dk, None, None, None, None


rotary_embedding_op.register_autograd(_rotary_backward, setup_context=_rotary_setup)


class _RotaryEager(torch.autograd.Function):
    """Eager rotary_embedding: the op's kernels and gradients without its dispatch."""

    @staticmethod
    def forward(ctx, query, key, positions, angles, interleaved, inverse):
        _rotary_setup(ctx, (query, key, positions, angles, interleaved, inverse), None)
        return _apply(query, key, positions, angles, interleaved, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        positions, angles = ctx.saved_tensors
        dq, dk = _RotaryEager.apply(dq, dk, positions, angles, ctx.interleaved, not ctx.inverse)
        return dq, dk, None, None, None, None


def _check_rotary(query, key, angles) -> None:
    if query.shape[-1] != key.shape[-1]:
        raise ValueError(f"Head dimension mismatch: Q={query.shape[-1]}, K={key.shape[-1]}")
    if angles.dim() != 2 or angles.shape[0] < 1 or angles.shape[1] < 2 or angles.shape[1] % 2 or \
            angles.shape[1] > query.shape[-1]:
        raise ValueError(f"angles must have shape (positions, rot_dim) with rot_dim even and up to {query.shape[-1]}, "
                         f"got {tuple(angles.shape)}")
    if query.dtype not in _capi._DTYPE_CODE:
        raise RuntimeError(f"unsupported dtype {query.dtype}; expected float16, bfloat16 or float32")
    if key.dtype != query.dtype:
        raise RuntimeError(f"query and key must share a dtype, got {query.dtype}, {key.dtype}")
    if query.shape[-1] not in (16, 32, 64, 128):
        raise RuntimeError(f"unsupported head dimension {query.shape[-1]} (expected 16, 32, 64 or 128)")


def _check_positions(positions: torch.Tensor, shape: tuple) -> None:
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
    if positions.shape != shape:
        raise ValueError(f"positions must have shape {tuple(shape)}, got {tuple(positions.shape)}")


def rotary_embedding(
    query: torch.Tensor,
    key: torch.Tensor,
    positions: torch.Tensor,
    angles: torch.Tensor,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Turns queries and keys by the angles of their positions, with autograd.

    Pair (a, b) of a head's first rot_dim columns becomes
    (a cos - b sin, b cos + a sin); the other columns stay.

    Args:
        query, key: [N, H, D] and [N, H_kv, D] packed rows, or [B, T, H, D] and
            [B, T, H_kv, D] (float16, bfloat16 or float32; D 16, 32, 64 or 128; unit
            stride along D, other strides as they are).
        positions: [N], or [B, T] or [T], int32 or int64 row of `angles` of each token;
            clamped to the table's rows.
        angles: [positions, rot_dim] fp32 cosines, then sines, as rotary_table gives
            them; receives no gradient.
        interleaved: pair i is columns 2i and 2i + 1, else i and i + rot_dim / 2.

    Returns:
        (query, key) turned, contiguous, in their shapes and dtype (computed in
        fp32 and rounded once).
    """
    quick = _quick()
    if quick is not None:
        got = quick.quick_rotary(query, key, positions, angles, interleaved)
        if got is not None:
            return got
    if query.dim() not in (3, 4) or key.dim() != query.dim():
        raise ValueError("Expected query and key to be 3D tensors (total_tokens, H, D) or 4D tensors (B, T, H, D)")
    lead = query.shape[:-2]
    if key.shape[:-2] != lead:
        raise ValueError(f"query and key must have the same tokens, got {tuple(lead)} and {tuple(key.shape[:-2])}")
    _check_rotary(query, key, angles)
    if query.dim() == 4 and positions.dim() == 1:
        _check_positions(positions, lead[1:])
        positions = positions.expand(lead)
    else:
        _check_positions(positions, lead)
    q, k = query.flatten(0, -3), key.flatten(0, -3)
    args = (q, k, positions.reshape(-1), angles, bool(interleaved), False)
    q, k = rotary_embedding_op(*args) if torch.compiler.is_compiling() else _RotaryEager.apply(*args)
    return q.view(query.shape), k.view(key.shape)


# --- rotary embedding on the way into the cache -----------------------------------

def _write_rotary(query, key, value, key_cache, value_cache, slot_mapping, positions, angles, interleaved):
    _no_tangent("paged_cache_write_rotary", query, key, value, key_cache, value_cache, angles)
    lib = _capi.load_library()
    _capi._check_device(key_cache)
    dev = key_cache.device
    _on(dev, query=query, key=key, value=value, value_cache=value_cache)
    query, key, value = _unit(query), _unit(key), _unit(value)
    if key.stride() != value.stride():
        key, value = key.contiguous(), value.contiguous()
    slot_mapping, positions = _ints(slot_mapping, dev), _ints(positions, dev)
    angles = _capi._as(angles, torch.float32, dev)
    out = torch.empty(query.shape, dtype=query.dtype, device=dev)
    r = _rotary(query, key, positions, angles, interleaved)
    r.cache_stride_p, r.cache_stride_t, r.cache_stride_h = key_cache.stride()[:3]
    r.num_pages, r.page_size = key_cache.shape[:2]
    r.v, r.q_out, r.slot_mapping = value.data_ptr(), out.data_ptr(), slot_mapping.data_ptr()
    r.k_cache, r.v_cache = key_cache.data_ptr(), value_cache.data_ptr()
    _capi._on_device(dev, lambda stream: _capi._raise(lib.sigattn_paged_write_rotary(ctypes.byref(r), stream),
                                                      "sigattn_paged_write_rotary"))
    return out


@torch.library.custom_op("myops::paged_cache_write_rotary", mutates_args=("key_cache", "value_cache"))
def paged_cache_write_rotary_op(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor,
                                value_cache: torch.Tensor, slot_mapping: torch.Tensor, positions: torch.Tensor,
                                angles: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """The turned query; rows of the turned key and of value into the caches' slots."""
    return _write_rotary(query, key, value, key_cache, value_cache, slot_mapping, positions, angles, interleaved)


@paged_cache_write_rotary_op.register_fake
def _(query, key, value, key_cache, value_cache, slot_mapping, positions, angles, interleaved):
    return query.new_empty(query.shape)


def paged_cache_write_rotary(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    positions: torch.Tensor,
    angles: torch.Tensor,
    interleaved: bool = False,
) -> torch.Tensor:
    """paged_cache_write with the step's queries and keys turned by their positions.

    Args:
        query: [N, H, D] packed new tokens; key, value: [N, H_kv, D].
        key_cache, value_cache, slot_mapping: as for paged_cache_write; the keys are
            written turned, the values as they are.
        positions: [N] int32 or int64, clamped to the table's rows (any number on
            rows without a slot, whose query comes back turned by it).
        angles, interleaved: as for rotary_embedding.

    Returns:
        The turned query, [N, H, D], contiguous.  Forward only: tensors that ask for a
        gradient (under grad mode) or carry a forward-mode tangent are refused.
    """
    quick = _quick()
    if quick is not None:
        got = quick.quick_write_rotary(query, key, value, key_cache, value_cache, slot_mapping, positions, angles,
                                       interleaved)
        if got is not None:
            return got
    _check_write(key, value, key_cache, value_cache, slot_mapping)
    if query.dim() != 3 or query.shape[0] != key.shape[0]:
        raise ValueError(f"Expected query to be a 3D tensor ({key.shape[0]}, H, D), got {tuple(query.shape)}")
    _check_rotary(query, key, angles)
    _check_positions(positions, key.shape[:1])
    _no_grad("paged_cache_write_rotary", query, key, value, key_cache, value_cache, angles)
    args = (query, key, value, key_cache, value_cache, slot_mapping, positions, angles, bool(interleaved))
    if torch.compiler.is_compiling():
        return paged_cache_write_rotary_op(*args)
    out = _write_rotary(*args)
    _changed(key_cache, value_cache)
    return out
