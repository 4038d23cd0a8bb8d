// Rotary embedding: pairs of a head's columns turned by the angles of the row's
// position, for queries and keys (and their gradients, by the negative angles), or
// with the keys and values going straight to their slots of a paged cache.
#include <hip/hip_runtime.h>

#include "../../include/sigattn.h"
#include "launch.h"

namespace sigattn {
namespace {

struct RotaryArgs {
  const char *src[3];  // q, k, v (v: only copied; nullptr without a cache)
  char *out[3];        // q_out; k_out, or the caches
  const int32_t *positions, *slots;
  const float *angles;
  int64_t src_t[3], src_h[3], dst_p, dst_t, dst_h, out_t[2];  // bytes
  int64_t rows, num_slots;
  int heads[3], D, rot, num_positions, lp;
  float sign;
};

template <typename T> __device__ __forceinline__ float rot_ld(const char *row, int i) {
  if constexpr (sizeof(T) == 4) return ((const float *)row)[i];
  else return Elem<T>::to_f32(((const uint16_t *)row)[i]);
}
template <typename T> __device__ __forceinline__ void rot_st(char *row, int i, float x) {
  if constexpr (sizeof(T) == 4) ((float *)row)[i] = x;
  else ((uint16_t *)row)[i] = Elem<T>::from_f32(x);
}

// (a, b) turned; one rounding each besides the first product's, in every kernel alike.
__device__ __forceinline__ void turn_pair(float a, float b, float cs, float sn, float &u, float &w) {
  u = __builtin_fmaf(-b, sn, a * cs), w = __builtin_fmaf(a, sn, b * cs);
}

// Any strides, alignment and rot_dim: a workgroup per row, a thread per pair (or two
// copied columns); bound by its narrow loads (bf16 16384 rows H=32 Hkv=8 D=128 384 us
// forward and backward, where the other kernel takes 119).  A launch has fewer than 2^32
// threads: a workgroup goes on to the row kRotaryRows behind its own.
constexpr int64_t kRotaryRows = 1 << 20;
template <typename T, bool PAIRS> __device__ __forceinline__ void rotary_row(const RotaryArgs &a, const int64_t t) {
  const int half = a.rot / 2, dh = a.D / 2;
  const int pos = min(max(a.positions[t], 0), a.num_positions - 1);
  const float *row = a.angles + (int64_t)pos * a.rot;
  const int32_t slot = a.slots != nullptr ? a.slots[t] : 0;
  const bool there = a.slots == nullptr || (slot >= 0 && slot < a.num_slots);
  const int all = (a.heads[0] + a.heads[1] + a.heads[2]) * dh;
  for (int i = threadIdx.x; i < all; i += 256) {
    int h = i / dh;
    const int c = i - h * dh;
    const int which = h < a.heads[0] ? 0 : (h < a.heads[0] + a.heads[1] ? 1 : 2);
    h -= which > 0 ? a.heads[0] : 0;
    h -= which > 1 ? a.heads[1] : 0;
    const char *src = a.src[which] + t * a.src_t[which] + h * a.src_h[which];
    char *dst;
    if (which == 0 || a.slots == nullptr) {
      dst = a.out[which] + t * a.out_t[which] + (int64_t)h * a.D * sizeof(T);
    } else {
      if (!there) continue;
      dst = a.out[which] + (int64_t)(slot >> a.lp) * a.dst_p + (slot & ((1 << a.lp) - 1)) * a.dst_t + h * a.dst_h;
    }
    const bool turn = which < 2 && c < half;
    const int x = turn ? (PAIRS ? 2 * c : c) : (which < 2 ? a.rot + 2 * (c - half) : 2 * c);
    const int y = turn && !PAIRS ? c + half : x + 1;
    float u = rot_ld<T>(src, x), w = rot_ld<T>(src, y);
    if (turn) {
      const float p = u, q = w;
      turn_pair(p, q, row[c], row[c + half] * a.sign, u, w);
    }
    rot_st<T>(dst, x, u), rot_st<T>(dst, y, w);
  }
}
template <typename T, bool PAIRS> __global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
  for (int64_t t = blockIdx.x; t < a.rows; t += kRotaryRows) rotary_row<T, PAIRS>(a, t);
}

// Rows on 16-byte boundaries: a thread's unit is two 16-byte pieces, E pairs
// of columns (pieces of the two halves, or neighbours), or two pieces to copy.
// Units of all rows and heads follow one another; the quotient by a row's units is
// exact in fp32 (a workgroup's span and a row's units lie below 2^22).  The grid's second
// dimension counts kRotarySlice workgroups each (fewer than 2^32 threads in the first).  Bound by
// memory, at the rate of a large copy (5.1 TB/s): bf16 16384 rows H=32 Hkv=8 D=128
// (337 MB) 60.6 us, 5.6 TB/s, fp16 16383 rows H=16 Hkv=8 D=64 into a cache 23.6 us;
// 64 rows into a cache 3.4 us.  (Two units a thread 62.0 and 23.7, four 69.3 and
// 25.2: more loads in flight, fewer waves.)
template <typename T> struct RotaryPiece {
  static constexpr int E = 16 / sizeof(T);
  static __device__ __forceinline__ float get(const u32x4 &v, int i) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(f32x4, v)[i];
    else return Elem<T>::to_f32((uint16_t)(i % 2 == 0 ? v[i / 2] & 0xffffu : v[i / 2] >> 16));
  }
  static __device__ __forceinline__ u32x4 put(const float (&x)[E]) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(u32x4, (f32x4){x[0], x[1], x[2], x[3]});
    else return (u32x4){Elem<T>::pack(x[0], x[1]), Elem<T>::pack(x[2], x[3]), Elem<T>::pack(x[4], x[5]),
                        Elem<T>::pack(x[6], x[7])};
  }
};

constexpr int64_t kRotarySlice = 1 << 23;
template <typename T, bool PAIRS, bool CACHE>
__global__ __launch_bounds__(256) void rotary_wide_kernel(const RotaryArgs a, const int lu) {
  using Piece = RotaryPiece<T>;
  constexpr int E = Piece::E;
  const int half = a.rot / 2;
  const int n = (a.heads[0] + a.heads[1] + a.heads[2]) << lu;  // units of a row, 1 << lu of a head
  const int64_t base = (blockIdx.y * kRotarySlice + blockIdx.x) * 256, row0 = base / n;
  const int i = (int)(base - row0 * n) + (int)threadIdx.x, q = (int)(((float)i + 0.5f) * (1.0f / (float)n));
  const int64_t t = row0 + q;
  if (t >= a.rows) return;
  const int r = i - q * n, u = r & ((1 << lu) - 1);
  int h = r >> lu;
  const int which = h < a.heads[0] ? 0 : (h < a.heads[0] + a.heads[1] ? 1 : 2);
  h -= which > 0 ? a.heads[0] : 0;
  h -= which > 1 ? a.heads[1] : 0;
  const bool turn = (!CACHE || which < 2) && u * E < half;
  // Bytes of the unit's first piece within its head, and to its second.
  const int at = turn && !PAIRS ? 16 * u : 32 * u, step = turn && !PAIRS ? half * (int)sizeof(T) : 16;
  const char *src = (which == 0 ? a.src[0] : which == 1 ? a.src[1] : a.src[2]) +
                    t * (which == 0 ? a.src_t[0] : a.src_t[1]) + h * (which == 0 ? a.src_h[0] : a.src_h[1]) + at;
  char *dst;
  if (CACHE && which > 0) {
    const int32_t slot = a.slots[t];
    if (slot < 0 || slot >= a.num_slots) return;
    dst = (which == 1 ? a.out[1] : a.out[2]) + (int64_t)(slot >> a.lp) * a.dst_p +
          (slot & ((1 << a.lp) - 1)) * a.dst_t + h * a.dst_h + at;
  } else {
    dst = (which == 0 ? a.out[0] : a.out[1]) + t * (which == 0 ? a.out_t[0] : a.out_t[1]) +
          (int64_t)h * a.D * sizeof(T) + at;
  }
  u32x4 x = *(const u32x4 *)src, y = *(const u32x4 *)(src + step);
  if (turn) {
    const float *row = a.angles + (int64_t)min(max(a.positions[t], 0), a.num_positions - 1) * a.rot + u * E;
    float lo[E], hi[E];  // the two pieces, turned
#pragma unroll
    for (int e = 0; e < E; ++e) {
      // Pair e: elements 2e and 2e + 1 of the two pieces in a row, or e of each.
      const float cs = row[e], sn = row[half + e] * a.sign;
      if constexpr (PAIRS) {
        float(&to)[E] = e < E / 2 ? lo : hi;
        const u32x4 &from = e < E / 2 ? x : y;
        const int j = 2 * e % E;
        turn_pair(Piece::get(from, j), Piece::get(from, j + 1), cs, sn, to[j], to[j + 1]);
      } else {
        turn_pair(Piece::get(x, e), Piece::get(y, e), cs, sn, lo[e], hi[e]);
      }
    }
    x = Piece::put(lo), y = Piece::put(hi);
  }
  *(u32x4 *)dst = x, *(u32x4 *)(dst + step) = y;
}

// Whether that kernel takes the call; lu: log2 of a head's units.
template <typename T> bool rotary_wide(const RotaryArgs &a, int &lu) {
  constexpr int E = RotaryPiece<T>::E;
  uint64_t bits = (uintptr_t)a.angles;
  const bool cache = a.slots != nullptr;
  for (int i = 0; i < 3; ++i)
    if (a.heads[i] > 0) {
      bits |= (uintptr_t)a.src[i] | (uintptr_t)a.out[i] | (uint64_t)(a.src_t[i] | a.src_h[i]);
      if (cache && i > 0) bits |= (uint64_t)(a.dst_p | a.dst_t | a.dst_h);
    }
  lu = 31 - __builtin_clz((unsigned)(a.D / (2 * E)));
  return (bits & 15) == 0 && a.rot % (2 * E) == 0 && (int64_t)(a.heads[0] + a.heads[1] + a.heads[2]) << lu < 1 << 21;
}

template <typename T, bool PAIRS, bool CACHE> void rotary_launch(const RotaryArgs &a, int lu, hipStream_t st) {
  const int64_t units = a.rows * ((int64_t)(a.heads[0] + a.heads[1] + a.heads[2]) << lu), groups = (units + 255) / 256;
  const int64_t slices = (groups + kRotarySlice - 1) / kRotarySlice;
  const dim3 grid((unsigned)(slices > 1 ? kRotarySlice : groups), (unsigned)slices);
  rotary_wide_kernel<T, PAIRS, CACHE><<<grid, dim3(256), 0, st>>>(a, lu);
}

template <typename T> void rotary_t(const RotaryArgs &a, bool pairs, hipStream_t st) {
  int lu = 0;
  if (rotary_wide<T>(a, lu)) {
    if (a.slots != nullptr) {
      if (pairs) rotary_launch<T, true, true>(a, lu, st);
      else rotary_launch<T, false, true>(a, lu, st);
    } else if (pairs) rotary_launch<T, true, false>(a, lu, st);
    else rotary_launch<T, false, false>(a, lu, st);
    return;
  }
  const dim3 grid((unsigned)(a.rows < kRotaryRows ? a.rows : kRotaryRows));
  if (pairs) rotary_kernel<T, true><<<grid, dim3(256), 0, st>>>(a);
  else rotary_kernel<T, false><<<grid, dim3(256), 0, st>>>(a);
}

int rotary_run(const sigattn_rotary *r, bool cache, hipStream_t st) {
  RotaryArgs a{};
  const int64_t es = r->dtype == SIGATTN_F32 ? 4 : 2;
  a.src[0] = (const char *)r->q, a.src[1] = (const char *)r->k, a.src[2] = cache ? (const char *)r->v : nullptr;
  a.out[0] = (char *)r->q_out, a.out[1] = (char *)(cache ? r->k_cache : r->k_out);
  a.out[2] = cache ? (char *)r->v_cache : nullptr;
  a.positions = r->positions, a.slots = cache ? r->slot_mapping : nullptr, a.angles = r->angles;
  a.src_t[0] = r->q_stride_t * es, a.src_h[0] = r->q_stride_h * es;
  for (int i = 1; i < 3; ++i) a.src_t[i] = r->k_stride_t * es, a.src_h[i] = r->k_stride_h * es;
  a.dst_p = r->cache_stride_p * es, a.dst_t = r->cache_stride_t * es, a.dst_h = r->cache_stride_h * es;
  a.out_t[0] = r->q_heads * r->D * es, a.out_t[1] = r->kv_heads * r->D * es;
  a.rows = r->rows, a.num_slots = r->num_pages * r->page_size;
  a.heads[0] = (int)r->q_heads, a.heads[1] = (int)r->kv_heads, a.heads[2] = cache ? (int)r->kv_heads : 0;
  a.D = (int)r->D, a.rot = (int)r->rot_dim, a.num_positions = (int)r->num_positions;
  a.lp = cache ? 63 - __builtin_clzll((unsigned long long)r->page_size) : 0;
  a.sign = r->inverse != 0 ? -1.0f : 1.0f;
  (void)hipGetLastError();
  const bool pairs = r->interleaved != 0;
  if (r->dtype == SIGATTN_F32) rotary_t<float>(a, pairs, st);
  else if (r->dtype == SIGATTN_BF16) rotary_t<__bf16>(a, pairs, st);
  else rotary_t<_Float16>(a, pairs, st);
  return hipGetLastError() == hipSuccess ? SIGATTN_OK : SIGATTN_ERR_LAUNCH;
}

int rotary_check(const sigattn_rotary *r) {
  if (r == nullptr) return SIGATTN_ERR_NULL_ARG;
  if (r->dtype != SIGATTN_F16 && r->dtype != SIGATTN_BF16 && r->dtype != SIGATTN_F32) return SIGATTN_ERR_DTYPE;
  if (r->D != 16 && r->D != 32 && r->D != 64 && r->D != 128) return SIGATTN_ERR_HEAD_DIM;
  // (A row's heads times columns fit 31 bits.)
  if (r->rows < 0 || r->rows > INT32_MAX / 2 || r->q_heads < 0 || r->kv_heads < 0 || r->q_heads > 65535 ||
      r->kv_heads > 65535 || r->num_positions > INT32_MAX)
    return SIGATTN_ERR_SHAPE;
  // (Units of 16 columns, in fp32 8, in workgroups of 256: 2^8 slices at most.)
  if (r->rows > 0 && (r->q_heads + 2 * r->kv_heads) * r->D > ((int64_t)1 << 42) / r->rows) return SIGATTN_ERR_SHAPE;
  if (r->rot_dim < 2 || r->rot_dim > r->D || r->rot_dim % 2 != 0 || r->num_positions < 1) return SIGATTN_ERR_ROTARY;
  const int64_t strides[4] = {r->q_stride_t, r->q_stride_h, r->k_stride_t, r->k_stride_h};
  for (int64_t s : strides)
    if (s < 0) return SIGATTN_ERR_STRIDE;
  return SIGATTN_OK;
}

}  // namespace
}  // namespace sigattn

extern "C" int sigattn_rotary_apply(const sigattn_rotary *r, void *stream) {
  const int rc = sigattn::rotary_check(r);
  if (rc != SIGATTN_OK) return rc;
  if (r->rows == 0 || r->q_heads + r->kv_heads == 0) return SIGATTN_OK;
  if (r->positions == nullptr || r->angles == nullptr || (r->q_heads > 0 && (r->q == nullptr || r->q_out == nullptr)) ||
      (r->kv_heads > 0 && (r->k == nullptr || r->k_out == nullptr)))
    return SIGATTN_ERR_NULL_ARG;
  return sigattn::rotary_run(r, false, (hipStream_t)stream);
}

extern "C" int sigattn_paged_write_rotary(const sigattn_rotary *r, void *stream) {
  const int rc = sigattn::rotary_check(r);
  if (rc != SIGATTN_OK) return rc;
  if (r->num_pages < 0 || r->page_size < 16 || r->page_size > (1 << 20) || (r->page_size & (r->page_size - 1)) != 0 ||
      r->num_pages > INT32_MAX / r->page_size)
    return SIGATTN_ERR_SHAPE;
  const int64_t strides[3] = {r->cache_stride_p, r->cache_stride_t, r->cache_stride_h};
  for (int64_t s : strides)
    if (s < 0) return SIGATTN_ERR_STRIDE;
  if (r->rows == 0 || r->q_heads + r->kv_heads == 0) return SIGATTN_OK;
  if (r->positions == nullptr || r->angles == nullptr || r->slot_mapping == nullptr ||
      (r->q_heads > 0 && (r->q == nullptr || r->q_out == nullptr)) ||
      (r->kv_heads > 0 && (r->k == nullptr || r->v == nullptr ||
                           (r->num_pages > 0 && (r->k_cache == nullptr || r->v_cache == nullptr)))))
    return SIGATTN_ERR_NULL_ARG;
  return sigattn::rotary_run(r, true, (hipStream_t)stream);
}
