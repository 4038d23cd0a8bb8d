// Paged key/value cache: parameters and launchers of the kernels that read it.
#pragma once

#include "common.h"

namespace sigattn {

// Attention over a paged cache.  The base's q, out, k, v, score_mod, cu_q,
// rows_q, sq_*, sk_t, sk_h, B, H, Tq (longest query sequence), Tk (tokens a
// block-table row can hold) and dmem mean what they do there; H counts query
// heads.
struct PagedParams : KParams {
  const int32_t *table;  // [B, max_pages], row stride table_stride
  const int32_t *lens;   // [B] keys
  int64_t table_stride, mod_stride, sk_p;
  int Hkv, G;            // K / V heads, query heads of each
  int lp, num_pages;     // log2 of the page size
  float fscale, fbias;
  int own_bias;          // 0: the bias is -log(keys)

  __device__ __forceinline__ int keys(int b) const { return clamp_len(lens, b, Tk); }
  __device__ __forceinline__ float bias_of(int Lk) const { return own_bias ? fbias : -logf((float)Lk); }
};

void launch_paged_generic(const PagedParams &p, int dtype, int D, bool causal, hipStream_t st);

}  // namespace sigattn
