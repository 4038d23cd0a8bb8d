// Learned bias by relative position: sigmoid(q·k·scale + bias + x[key - query])
// with x a line of values per query head, what a table of buckets holds for each
// relative position within `reach`, and its ends' values for all beyond.
#pragma once

#include "../../include/sigattn.h"
#include "common.h"
#include "paged.h"

namespace sigattn {

// Values and sums by relative position d = key - query, -reach .. reach.  The
// caller's table may reach further than any two tokens of a call lie apart: `reach`
// is then what those need.  A head's line of values has kRelPad places more on either
// side (the ends' values), so that of a block of 32 keys or queries the first
// place is all that is clamped.
constexpr int kRelPad = 64;
__host__ __device__ constexpr int line_places(int reach) { return 2 * (reach + kRelPad) + 1; }

struct RelParams : KParams {
  static constexpr bool kRel = true;
  const float *line;  // [H, line_places(reach)]
  int reach;
  // dQ kernels: sums of dS of each (query block of part_rows rows, query head),
  // [part_slots(), H, places()], place reach + d.  Blocks of batch b follow one
  // another from slot first row / part_rows + b on, which leaves none without a
  // place of its own.
  float *part;        // nullptr: no sums
  int part_rows;

  __host__ __device__ __forceinline__ int places() const { return 2 * reach + 1; }
  __host__ __device__ __forceinline__ int64_t part_slots() const { return rows_q / part_rows + B; }
  __device__ __forceinline__ int64_t first_slot(int b) const { return packed_first(cu_q, rows_q, b) / part_rows + b; }
  __device__ __forceinline__ float *part_row(int b, int blk, int h) const {
    return part + ((first_slot(b) + blk) * H + h) * places();
  }
};

// Over a paged cache: query i of n at position L - n + i (forward only).
struct PagedRelParams : PagedParams {
  static constexpr bool kRel = true;
  const float *line;
  int reach;
};

// Place 0 of query head h's line, and its value at relative position d.
template <class P> __device__ __forceinline__ const float *rel_row(const P &p, int h) {
  return p.line + (int64_t)h * line_places(p.reach) + kRelPad + p.reach;
}
template <class P> __device__ __forceinline__ float rel_at(const P &p, int h, int d) {
  if constexpr (P::kRel) return rel_row(p, h)[min(max(d, -p.reach), p.reach)];
  else return 0.0f;
}

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// What a lane's column of scores has added beyond scale, times -log2(e), a block of
// 32 rows at a time, for kernels whose lanes read it themselves.  Blocks that lie
// beyond the line's end for every lane, nearly all of a long context, cost nothing:
// their value is the lane's constant.
struct RelColumn {
  const float *row;  // relative position 0
  float nbl, ends[2];
  int reach, pos;    // the column's position
  template <class P> __device__ __forceinline__ void init(const P &p, int h, int position, float bias) {
    row = rel_row(p, h), reach = p.reach, pos = position;
    nbl = -bias * kLog2e;
    ends[0] = __builtin_fmaf(row[-reach], -kLog2e, nbl), ends[1] = __builtin_fmaf(row[reach], -kLog2e, nbl);
  }
  // Rows are keys from position `first` on: 16 (or the first 2) of this half of the wave.
  template <int N> __device__ __forceinline__ void block(int first, int hi, float (&c)[N]) const {
    const int d = first - pos;  // of the block's first key
    const bool before = d + 31 <= -reach, after = d >= reach;
    if (__all(before || after)) return fill(before, c);
    const float *at = row + min(max(d, -reach - 32), reach) + 4 * hi;
#pragma unroll
    for (int g = 0; g < (N + 3) / 4; ++g) {
      const f32x4 v = *(const f32x4_any *)(at + 8 * g);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (4 * g + j < N) c[4 * g + j] = __builtin_fmaf(v[j], -kLog2e, nbl);
    }
  }
  template <int N> __device__ __forceinline__ void fill(bool before, float (&c)[N]) const {
    const float x = before ? ends[0] : ends[1];
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = x;
  }
};

// dS by relative position, of a dQ workgroup of NW waves.  A 32x32 block of scores
// (lane: query, accumulator rows: keys) whose places all lie beyond the line's end
// adds to one sum per lane.  Any other goes through LDS eight keys at a time,
// written so that a place's scores (a diagonal's) are neighbours: a lane reads those
// of its place, sums them and adds the sum to a line of the wave's own, which no
// other lane or wave touches, so every addition has its order.  (LDS atomics, no two
// lanes of an instruction on one place, took about 100 cycles each: bf16 H=12 D=64, 16
// sequences of 101 .. 1001, reach 128, 262 us instead of 74; 55 without the bias.)
// LDS: the waves' lines, a block's places more on either side of the ends, then the
// pieces that diagonals go through, [39 places][8 keys] in rows of 12 (so that a
// row's two 16-byte reads meet no other lane's banks).
constexpr int kNearMargin = 64, kSkewRow = 12, kSkew = 39 * kSkewRow;
__host__ __device__ constexpr int near_places(int reach) { return 2 * reach + 2 * kNearMargin; }
__host__ __device__ constexpr int near_floats(int reach, int waves = 4) { return waves * (near_places(reach) + kSkew); }

// What the wave's lanes wrote to LDS before is what its lanes read behind this.  The
// hardware keeps a wave's LDS accesses in order, so no instruction comes of it.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <int NW> struct PlaceSums {
  float beyond[2] = {0.0f, 0.0f};
  float *mine, *skew;  // relative position 0 of the wave's line; its piece
  int reach;
  bool on;

  // A barrier follows before the first add() or finish().
  __device__ __forceinline__ void init(const RelParams &p, float *near, int w, int tid) {
    on = p.part != nullptr, reach = p.reach;
    mine = near + w * near_places(reach) + reach + kNearMargin;
    skew = near + NW * near_places(reach) + w * kSkew;
    beyond[0] = beyond[1] = 0.0f;
    if (on)
      for (int i = tid; i < near_floats(reach, NW); i += 64 * NW) near[i] = 0.0f;
  }
  // A block whose first key lies `off` (a multiple of 32) after the wave's first query;
  // sgn: what the lane's dS are to be times.
  __device__ __forceinline__ void add(const float (&ds)[16], int off, int l32, int hi, float sgn = 1.0f) {
    if (!on) return;
    if (off + 31 <= -reach || off - 31 >= reach) {
      float x = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) x += ds[i];
      if (off < 0) beyond[0] = __builtin_fmaf(x, sgn, beyond[0]);
      else beyond[1] = __builtin_fmaf(x, sgn, beyond[1]);
      return;
    }
    const int lane = l32 + 32 * hi;
    float *to = skew + (31 + 4 * hi - l32) * kSkewRow + 4 * hi;
    float x = 0.0f;
#pragma unroll
    for (int g = 0; g < 4; ++g) {  // keys 8g .. 8g + 7, places 8g - 31 .. 8g + 7 from `off` on
#pragma unroll
      for (int j = 0; j < 4; ++j) to[j * (kSkewRow + 1)] = ds[4 * g + j] * sgn;
      wave_order();
      const int row = lane - 8 * g;
      const float *from = skew + min(max(row, 0), 38) * kSkewRow;
      const f32x4 u = *(const f32x4 *)from, v = *(const f32x4 *)(from + 4);
      const float y = ((u.x + u.y) + (u.z + u.w)) + ((v.x + v.y) + (v.z + v.w));
      x += row >= 0 && row <= 38 ? y : 0.0f;
      wave_order();
    }
    mine[off - 31 + lane] += x;
  }
  // The waves' lines, in their order, to the block's row of p.part; what lies on
  // either side of the ends goes to these, as do the waves' sums per lane.
  __device__ __forceinline__ void finish(const RelParams &p, const float *near, int b, int blk, int h, int w, int tid) {
    if (!on) return;
    const int n = near_places(reach), places = p.places(), lane = tid & 63;
    __shared__ float ends[NW][2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float x = wave_sum(beyond[e]);
      if (lane == 0) ends[w][e] = x;
    }
    __syncthreads();
    float *row = p.part_row(b, blk, h);
    const auto all = [&](int i) SIGATTN_INLINE {
      float x = near[i];
#pragma unroll
      for (int v = 1; v < NW; ++v) x += near[v * n + i];
      return x;
    };
    const auto end = [&](int e) SIGATTN_INLINE {
      float x = ends[0][e];
#pragma unroll
      for (int v = 1; v < NW; ++v) x += ends[v][e];
      return x;
    };
    if (w < 2) {
      // Wave 0: places up to the lower end, wave 1: from the upper one on.
      const float x = wave_sum(all(w == 0 ? lane + 1 : kNearMargin + places - 1 + lane));
      if (places > 1 && lane == 0) row[w == 0 ? 0 : places - 1] = x + end(w);
      if (places == 1 && lane == 0 && w == 0) {
        float y = x + end(0) + end(1);
        for (int i = 1; i < kNearMargin; ++i) y += all(kNearMargin + i);
        row[0] = y;
      }
    }
    for (int i = tid + 1; i < places - 1; i += 64 * NW) row[i] = all(kNearMargin + i);
  }
};

// The learned table: [buckets, H] of `dtype` (enum sigattn_dtype), and the bucket
// of each relative position -max_distance .. max_distance.
struct RelTable {
  const void *table;
  const int32_t *bucket;
  int dtype, buckets, max_distance, H, reach;
};

__device__ __forceinline__ int bucket_of(const RelTable &t, int place) {
  return t.bucket[t.max_distance + place - t.reach];
}

// The host's side: the caller's table for H heads and two lengths (reach: no two
// tokens lie further apart), and the bytes of its lines.
inline bool rel_table_ok(const sigattn_rel_bias *r) {
  return r->max_distance >= 0 && r->max_distance <= SIGATTN_REL_MAX_DISTANCE && r->num_buckets >= 1 &&
         r->num_buckets <= SIGATTN_REL_MAX_BUCKETS;
}
inline RelTable rel_table(const sigattn_rel_bias *r, int64_t H, int64_t Tq, int64_t Tk) {
  const int64_t longest = Tq > Tk ? Tq : Tk;
  RelTable t{};
  t.table = r->table, t.bucket = r->buckets;
  t.dtype = r->dtype, t.buckets = r->num_buckets, t.max_distance = (int)r->max_distance, t.H = (int)H;
  t.reach = (int)(r->max_distance < longest ? r->max_distance : longest);
  return t;
}
inline int64_t rel_line_bytes(const RelTable &t) {
  return ((int64_t)t.H * line_places(t.reach) * (int64_t)sizeof(float) + 255) / 256 * 256;
}

// line [H, line_places(reach)] from the table, and bias [B] (nullptr: not wanted), the
// default one of the key sequences.
void launch_rel_line(const RelTable &t, float *line, const int32_t *cu_k, int64_t B, float *bias, hipStream_t st);
// The table's gradient (`grad`, the table's type) from the dQ kernels' sums in
// p.part (nullptr: zeros); sums: [H, 2 reach + 1] floats of scratch.
void launch_rel_grad(const RelTable &t, const RelParams &p, float *sums, void *grad, hipStream_t st);

// MFMA forward, as launch_fwd_mfma.
void launch_rel_fwd_mfma(const RelParams &p, int dtype, int D, bool causal, hipStream_t st);

// MFMA backward, as launch_bwd_dq_mfma and launch_bwd_dkdv_mfma; the dQ kernel fills
// RelParams::part in blocks of rel_dq_rows rows.
int rel_dq_rows(const RelParams &p, int D, bool causal);
void launch_rel_dq_mfma(const RelParams &p, int dtype, int D, bool causal, hipStream_t st);
void launch_rel_dkdv_mfma(const RelParams &p, int dtype, int D, bool causal, hipStream_t st);
// Both in one launch; false (and nothing launched) where two are better.
bool launch_rel_bwd_mfma(const RelParams &pq, const RelParams &pk, int dtype, int D, bool causal, hipStream_t st);

// Portable kernels (launch.h); the dQ one fills RelParams::part, in blocks of
// kGenericRows rows.
constexpr int kGenericRows = 64;
void launch_rel_fwd_generic(const RelParams &p, int dtype, int D, bool causal, hipStream_t st);
void launch_rel_dq_generic(const RelParams &p, int dtype, int D, bool causal, hipStream_t st);
void launch_rel_dkdv_generic(const RelParams &p, int dtype, int D, bool causal, hipStream_t st);
// fp32 (launch_fwd_f32 and so on), D in {32, 64, 128} (16 as 32).
void launch_rel_fwd_f32(const RelParams &p, int D, bool causal, hipStream_t st);
int rel_dq_rows_f32(const RelParams &p, int D, bool causal);
void launch_rel_dq_f32(const RelParams &p, int D, bool causal, hipStream_t st);
void launch_rel_dkdv_f32(const RelParams &p, int D, bool causal, hipStream_t st);
// Both in one launch; false (and nothing launched) where their workgroups differ or
// the sums by position would leave dK/dV fewer of them per CU.
bool launch_rel_bwd_f32(const RelParams &pq, const RelParams &pk, int D, bool causal, hipStream_t st);
void launch_paged_rel_f32(const PagedRelParams &p, int units, int D, bool causal, hipStream_t st);
void launch_paged_rel_decode_f32(const PagedRelParams &p, int units, int D, bool causal, hipStream_t st);

// MFMA kernels over a paged cache, as launch_paged_fwd, launch_paged_decode and
// launch_paged_mixed (paged.h).
void launch_paged_rel_fwd(const PagedRelParams &p, int units, int dtype, int D, bool causal, hipStream_t st);
void launch_paged_rel_decode(const PagedRelParams &p, int units, int dtype, int D, bool causal, hipStream_t st);
void launch_paged_rel_mixed(const PagedRelParams &pf, int nf, const PagedRelParams &pd, int nd, int dtype, int D,
                            bool causal, hipStream_t st);
void launch_paged_rel_generic(const PagedRelParams &p, int dtype, int D, bool causal, hipStream_t st);

}  // namespace sigattn
