// C ABI of the attention over a paged cache (include/sigattn.h): validation on
// the host, before any HIP call, and the choice of kernels.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>

#include "../../include/sigattn.h"
#include "launch.h"
#include "paged.h"

using sigattn::PagedParams;

namespace {

PagedParams make_params(const sigattn_paged_problem *p, void *out) {
  PagedParams k{};
  k.ncu = sigattn::device_compute_units();
  k.q = p->q, k.k = p->k_cache, k.v = p->v_cache, k.out = out;
  k.score_mod = p->score_mod;
  k.cu_q = p->cu_seqlens_q;
  k.rows_q = p->rows_q;
  k.sq_t = p->q_stride_t, k.sq_h = p->q_stride_h;
  k.sk_p = p->k_stride_p, k.sk_t = p->k_stride_t, k.sk_h = p->k_stride_h;
  k.B = (int)p->B, k.H = (int)p->H, k.Hkv = (int)p->kv_heads, k.G = (int)(p->H / p->kv_heads);
  k.Tq = (int)(p->max_seqlen_q < p->rows_q ? p->max_seqlen_q : p->rows_q);
  k.Tk = (int)(p->max_pages * p->page_size);
  k.dmem = (int)p->D;
  k.hgroup = k.qgroup = 1;
  k.table = p->block_table, k.table_stride = p->table_stride;
  k.lens = p->seq_lens_k;
  k.mod_stride = p->mod_stride;
  k.lp = 63 - __builtin_clzll((unsigned long long)p->page_size);
  k.num_pages = (int)p->num_pages;
  k.fscale = p->scale, k.fbias = p->bias, k.own_bias = p->own_bias;
  return k;
}

int launch_status() { return hipGetLastError() == hipSuccess ? SIGATTN_OK : SIGATTN_ERR_LAUNCH; }

}  // namespace

extern "C" {

int sigattn_paged_check(const sigattn_paged_problem *p) {
  if (p == nullptr) return SIGATTN_ERR_NULL_ARG;
  if (p->abi_version != SIGATTN_ABI_VERSION) return SIGATTN_ERR_ABI_VERSION;
  if (p->dtype != SIGATTN_F16 && p->dtype != SIGATTN_BF16 && p->dtype != SIGATTN_F32) return SIGATTN_ERR_DTYPE;
  if (p->D != 16 && p->D != 32 && p->D != 64 && p->D != 128) return SIGATTN_ERR_HEAD_DIM;
  if (p->B < 0 || p->H < 0 || p->rows_q < 0 || p->max_seqlen_q < 0 || p->num_pages < 0 || p->max_pages < 0 ||
      p->B > INT_MAX / 64 || p->H > 65535 || p->rows_q > INT_MAX / 64 || p->page_size < 16 ||
      p->page_size > (1 << 20) || (p->page_size & (p->page_size - 1)) != 0 ||
      p->num_pages > INT_MAX / p->page_size || p->max_pages > INT_MAX / 2 / p->page_size)
    return SIGATTN_ERR_SHAPE;
  if (p->H > 0 && (p->kv_heads <= 0 || p->kv_heads > p->H || p->H % p->kv_heads != 0)) return SIGATTN_ERR_KV_HEADS;
  // Work items of any kernel: one per query row and head at most.
  if (p->H > 0 && p->rows_q + p->B > INT_MAX / p->H) return SIGATTN_ERR_SHAPE;
  const int64_t strides[7] = {p->q_stride_t, p->q_stride_h, p->k_stride_p, p->k_stride_t,
                              p->k_stride_h, p->table_stride, p->mod_stride};
  for (int64_t s : strides)
    if (s < 0) return SIGATTN_ERR_STRIDE;
  if (p->rows_q == 0 || p->H == 0) return SIGATTN_OK;
  if (p->q == nullptr || p->cu_seqlens_q == nullptr) return SIGATTN_ERR_NULL_ARG;
  if (p->B > 0 && (p->seq_lens_k == nullptr ||
                   (p->max_pages > 0 && (p->block_table == nullptr ||
                                         (p->num_pages > 0 && (p->k_cache == nullptr || p->v_cache == nullptr))))))
    return SIGATTN_ERR_NULL_ARG;
  return SIGATTN_OK;
}

size_t sigattn_paged_fwd_workspace_bytes(const sigattn_paged_problem *) { return 0; }

int sigattn_paged_fwd(const sigattn_paged_problem *p, void *out, void *workspace, size_t workspace_bytes,
                      void *stream) {
  const int rc = sigattn_paged_check(p);
  if (rc != SIGATTN_OK) return rc;
  if (p->rows_q == 0 || p->H == 0) return SIGATTN_OK;
  if (out == nullptr) return SIGATTN_ERR_NULL_ARG;
  (void)workspace, (void)workspace_bytes;
  const hipStream_t st = (hipStream_t)stream;
  const PagedParams k = make_params(p, out);
  (void)hipGetLastError();
  if (p->B == 0) {  // no sequence: every row is outside
    sigattn::GapAxis a;
    a.H = k.H, a.D = (int)p->D, a.rows = p->rows_q, a.st = p->H * p->D, a.sh = p->D, a.out[0] = out;
    sigattn::launch_zero_gaps(a, sigattn::GapAxis{}, p->dtype == SIGATTN_F32 ? 4 : 2, st);
    return launch_status();
  }
  sigattn::launch_paged_generic(k, p->dtype, (int)p->D, p->causal != 0, st);
  return launch_status();
}

}  // extern "C"
