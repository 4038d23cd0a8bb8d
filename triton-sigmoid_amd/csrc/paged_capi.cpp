// C ABI of the attention over a paged cache (include/sigattn.h): validation on
// the host, before any HIP call, and the choice of kernels.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>

#include "../../include/sigattn.h"
#include "launch.h"
#include "paged_problem.h"

using namespace sigattn;

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

size_t sigattn_paged_fwd_workspace_bytes(const sigattn_paged_problem *p) {
  if (sigattn_paged_check(p) != SIGATTN_OK || p->rows_q == 0 || p->H == 0 || p->B == 0) return 0;
  const PagedParams k = make_params(p, nullptr);
  return use_mfma(p, nullptr) ? make_plan(p, k, kernel_dim(p)).bytes : 0;
}

int sigattn_paged_fwd(const sigattn_paged_problem *p, void *out, void *workspace, size_t workspace_bytes,
                      void *stream) {
  const int rc = sigattn_paged_check(p);
  if (rc != SIGATTN_OK) return rc;
  if (p->rows_q == 0 || p->H == 0) return SIGATTN_OK;
  if (out == nullptr) return SIGATTN_ERR_NULL_ARG;
  const hipStream_t st = (hipStream_t)stream;
  PagedParams k = make_params(p, out);
  const bool mfma = p->B > 0 && use_mfma(p, out), causal = p->causal != 0;
  const int D = kernel_dim(p), dt = p->dtype;
  PagedPlan pl;
  if (mfma) pl = make_plan(p, k, D);
  if (workspace != nullptr && pl.bytes > 0 && (workspace_bytes < pl.bytes || !aligned16(workspace)))
    return SIGATTN_ERR_WORKSPACE;
  if (workspace == nullptr) {  // nothing is cut
    pl.fwd.split_units = pl.decode.split_units = 0;
  }
  (void)hipGetLastError();
  if (p->B == 0) {  // no sequence: every row is outside
    launch_zero_gaps(paged_gap(p, k, out), GapAxis{}, dt == SIGATTN_F32 ? 4 : 2, st);
    return launch_status();
  }
  if (!mfma) {
    launch_paged_generic(k, dt, (int)p->D, causal, st);
    return launch_status();
  }
  run_plan(p, k, pl, (char *)workspace, out, st, [&](const PagedParams &first, int nf, const PagedParams &kd, int nd) {
    if (nf > 0 && nd > 0) launch_paged_mixed(first, nf, kd, nd, dt, D, causal, st);
    else if (nd > 0 && dt == SIGATTN_F32) launch_paged_decode_f32(first, nd, D, causal, st);
    else if (nd > 0) launch_paged_decode(first, nd, dt, D, causal, st);
    else if (dt == SIGATTN_F32) launch_paged_f32(first, nf, D, causal, st);
    else launch_paged_fwd(first, nf, dt, D, causal, st);
  });
  return launch_status();
}

}  // extern "C"
