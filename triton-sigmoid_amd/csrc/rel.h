// Learned bias by relative position: sigmoid(q·k·scale + bias + x[key - query])
// with x a line of values per query head, what a table of buckets holds for each
// relative position within `reach`, and its ends' values for all beyond.
#pragma once

#include "../../include/sigattn.h"
#include "common.h"
#include "paged.h"

namespace sigattn {

// Values and sums are rows of 2 reach + 1 places, place reach + d for relative
// position d = key - query.  The caller's table may reach further than any two
// tokens of a call lie apart: `reach` is then what those need.
struct RelParams : KParams {
  static constexpr bool kRel = true;
  const float *line;  // [H, places]
  int reach;
  // dQ kernels: sums of dS of each (query block of part_rows rows, query head),
  // [part_slots(), H, places].  Blocks of batch b follow one another from slot
  // first row / part_rows + b on, which leaves none without a place of its own.
  float *part;        // nullptr: no sums
  int part_rows;

  __host__ __device__ __forceinline__ int places() const { return 2 * reach + 1; }
  __host__ __device__ __forceinline__ int64_t part_slots() const { return rows_q / part_rows + B; }
  __device__ __forceinline__ int64_t first_slot(int b) const { return packed_first(cu_q, rows_q, b) / part_rows + b; }
  __device__ __forceinline__ float *part_row(int b, int blk, int h) const {
    return part + ((first_slot(b) + blk) * H + h) * places();
  }
};

// Over a paged cache: query i of n at position L - n + i (forward only).  A lane of
// the matrix kernels has a column, so a head and a position of its own: it reads the
// values of a 32-key block itself, from a line with kRelPad places more on either
// side, so that the block's first place is all that is clamped.  Blocks that lie
// beyond the line's end for every lane, nearly all of a long context, cost nothing:
// their value is the lane's constant.
constexpr int kRelPad = 64;
struct PagedRelParams : PagedParams {
  static constexpr bool kRel = true;
  const float *line;  // [H, 2 reach + 1 + 2 kRelPad], places from the padding's first
  int reach;

  __device__ __forceinline__ const float *row(int h) const {
    return line + (int64_t)h * (2 * reach + 1 + 2 * kRelPad) + kRelPad + reach;
  }
};

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// What a lane's scores have added beyond scale, times -log2(e), block by block.
struct RelColumn {
  const float *row;  // relative position 0
  float nbl, ends[2];
  int reach, pos;    // the query's position, from the chunk's first key
  __device__ __forceinline__ void init(const PagedRelParams &p, int h, int position, float bias) {
    row = p.row(h), reach = p.reach, pos = position;
    nbl = -bias * kLog2e;
    ends[0] = __builtin_fmaf(row[-reach], -kLog2e, nbl), ends[1] = __builtin_fmaf(row[reach], -kLog2e, nbl);
  }
  // The 32-key block from key `first` on, 16 keys of this half of the wave; `n` of
  // them (2 or 16) are wanted.
  template <int N> __device__ __forceinline__ void block(int first, int hi, float (&c)[N]) const {
    const int d = first - pos;  // of the block's first key
    const bool before = d + 31 <= -reach, after = d >= reach;
    if (__all(before || after)) {
      const float x = before ? ends[0] : ends[1];
#pragma unroll
      for (int i = 0; i < N; ++i) c[i] = x;
      return;
    }
    const float *at = row + min(max(d, -reach - 32), reach) + 4 * hi;
#pragma unroll
    for (int g = 0; g < (N + 3) / 4; ++g) {
      const f32x4 v = *(const f32x4_any *)(at + 8 * g);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (4 * g + j < N) c[4 * g + j] = __builtin_fmaf(v[j], -kLog2e, nbl);
    }
  }
};

// Value of query head h at relative position d.
template <class P> __device__ __forceinline__ float rel_at(const P &p, int h, int d) {
  if constexpr (P::kRel && P::kPaged) return p.row(h)[min(max(d, -p.reach), p.reach)];
  else if constexpr (P::kRel) return p.line[(int64_t)h * (2 * p.reach + 1) + p.reach + min(max(d, -p.reach), p.reach)];
  else return 0.0f;
}

// The learned table: [buckets, H] of `dtype` (enum sigattn_dtype), and the bucket
// of each relative position -max_distance .. max_distance.
struct RelTable {
  const void *table;
  const int32_t *bucket;
  int dtype, buckets, max_distance, H, reach;
  int pad;  // places of the lines before -reach and after reach

  __host__ __device__ __forceinline__ int places() const { return 2 * (reach + pad) + 1; }
};

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
  return ((int64_t)t.H * t.places() * (int64_t)sizeof(float) + 255) / 256 * 256;
}

// line [H, places] from the table.
void launch_rel_line(const RelTable &t, float *line, hipStream_t st);
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

// Portable kernels (launch.h); the dQ one fills RelParams::part, in blocks of
// kGenericRows rows.
constexpr int kGenericRows = 64;
void launch_rel_fwd_generic(const RelParams &p, int dtype, int D, bool causal, hipStream_t st);
void launch_rel_dq_generic(const RelParams &p, int dtype, int D, bool causal, hipStream_t st);
void launch_rel_dkdv_generic(const RelParams &p, int dtype, int D, bool causal, hipStream_t st);
// MFMA kernels over a paged cache, as launch_paged_fwd, launch_paged_decode and
// launch_paged_mixed (paged.h).
void launch_paged_rel_fwd(const PagedRelParams &p, int units, int dtype, int D, bool causal, hipStream_t st);
void launch_paged_rel_decode(const PagedRelParams &p, int units, int dtype, int D, bool causal, hipStream_t st);
void launch_paged_rel_mixed(const PagedRelParams &pf, int nf, const PagedRelParams &pd, int nd, int dtype, int D, bool causal,
                            hipStream_t st);
void launch_paged_rel_generic(const PagedRelParams &p, int dtype, int D, bool causal, hipStream_t st);

}  // namespace sigattn
