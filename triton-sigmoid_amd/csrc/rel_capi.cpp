// C ABI of the learned bias by relative position (include/sigattn.h): validation on
// the host, before any HIP call, and the choice of kernels.
#include "paged_problem.h"
#include "rel.h"

using namespace sigattn;

namespace {

// What the line's launch leaves: the lines, then (without a bias of the caller's) the
// sequences' default ones.
int64_t rel_head_bytes(const sigattn_problem *p, const RelTable &t) {
  return rel_line_bytes(t) + (p->bias == nullptr ? (p->B * (int64_t)sizeof(float) + 255) / 256 * 256 : 0);
}

RelParams rel_params(const sigattn_problem *p, const RelTable &t, const void *line) {
  RelParams k{};
  (KParams &)k = make_params(p);
  k.line = (const float *)line;
  if (p->bias == nullptr) k.bias = (const float *)((const char *)line + rel_line_bytes(t));
  k.reach = t.reach;
  k.part_rows = kGenericRows;  // of calls without blocks of queries too, which divide by it
  return k;
}

void make_line(const sigattn_problem *p, const RelTable &t, void *to, hipStream_t st) {
  launch_rel_line(t, (float *)to, p->cu_seqlens_k, p->B,
                  p->bias == nullptr ? (float *)((char *)to + rel_line_bytes(t)) : nullptr, st);
}

int64_t rel_part_bytes(const sigattn_problem *p, const RelTable &t) {
  // (The shortest blocks' rows: whether the portable kernel's are taken depends on pointers
  // that a query of the size does not have.  A multiple of 256 bytes.)
  const int rows = p->dtype == SIGATTN_F32 && p->D < 128 ? 32 : kGenericRows;
  return ((p->rows_q / rows + p->B) * p->H * (2 * t.reach + 1) * (int64_t)sizeof(float) + 255) / 256 * 256;
}

// The backward's workspace: what the line's launch leaves, then (grad: a gradient of the
// table) the sums over blocks and those of each block, then grouped heads' parts.
struct RelSpace {
  int64_t sums, part, kv_part, bytes;
};
RelSpace rel_space(const sigattn_problem *p, const RelTable &t, bool grad) {
  RelSpace s;
  s.sums = rel_head_bytes(p, t);
  s.part = s.sums + (grad ? rel_line_bytes(t) : 0);
  s.kv_part = s.part + (grad ? rel_part_bytes(p, t) : 0);
  // (Pointers are not known to a query: aligned rows, as everywhere.)
  const void *none[1] = {nullptr};
  s.bytes = s.kv_part + head_split(p, use_mfma(p, none, 0) || use_f32_mfma(p, none, 0)).bytes;
  return s;
}

RelParams rel_kv_items(const RelParams &k) {
  RelParams s = k;
  (KParams &)s = kv_items(k);
  return s;
}

// The learned bias's table as far as the cache's sequences reach.
RelTable rel_table_of(const sigattn_paged_problem *p, const sigattn_rel_bias *r) {
  return rel_table(r, p->H, p->max_seqlen_q < p->rows_q ? p->max_seqlen_q : p->rows_q, p->max_pages * p->page_size);
}

}  // namespace

extern "C" {

int sigattn_rel_check(const sigattn_problem *p, const sigattn_rel_bias *r) {
  if (p == nullptr || r == nullptr) return SIGATTN_ERR_NULL_ARG;
  sigattn_problem with_bias = *p;
  if (p->bias == nullptr) with_bias.bias = p->scale;  // (its own: any pointer)
  const int rc = sigattn_check(&with_bias);
  if (rc != SIGATTN_OK) return rc;
  if (r->dtype != SIGATTN_F16 && r->dtype != SIGATTN_BF16 && r->dtype != SIGATTN_F32) return SIGATTN_ERR_DTYPE;
  if (!rel_table_ok(r) || p->score_mod != nullptr || p->cu_seqlens_q == nullptr || p->cu_seqlens_k == nullptr)
    return SIGATTN_ERR_REL_BIAS;
  if (p->H > 65535) return SIGATTN_ERR_SHAPE;  // the launches' second dimension
  if (p->H > 0 && (r->table == nullptr || r->buckets == nullptr)) return SIGATTN_ERR_NULL_ARG;
  return SIGATTN_OK;
}

size_t sigattn_rel_fwd_workspace_bytes(const sigattn_problem *p, const sigattn_rel_bias *r) {
  return sigattn_rel_check(p, r) == SIGATTN_OK ? (size_t)rel_head_bytes(p, rel_table(r, p->H, p->Tq, p->Tk)) : 0;
}

int sigattn_rel_fwd(const sigattn_problem *p, const sigattn_rel_bias *r, void *out, void *workspace,
                    size_t workspace_bytes, void *stream) {
  const int rc = sigattn_rel_check(p, r);
  if (rc != SIGATTN_OK) return rc;
  if (p->H == 0 || p->rows_q == 0) return SIGATTN_OK;
  if (out == nullptr) return SIGATTN_ERR_NULL_ARG;
  const hipStream_t st = (hipStream_t)stream;
  if (p->B == 0 || p->Tq == 0) {
    (void)hipGetLastError();
    zero_packed_gaps(p, out, nullptr, nullptr, st);
    return launch_status();
  }
  const RelTable t = rel_table(r, p->H, p->Tq, p->Tk);
  if (workspace == nullptr || !aligned16(workspace) || (int64_t)workspace_bytes < rel_head_bytes(p, t))
    return SIGATTN_ERR_WORKSPACE;
  RelParams k = rel_params(p, t, workspace);
  k.out = out;
  (void)hipGetLastError();
  make_line(p, t, workspace, st);
  const void *ptrs[4] = {p->q, p->k, p->v, out};
  const bool f32 = use_f32_mfma(p, ptrs, 4);
  if (f32 || use_mfma(p, ptrs, 4)) {
    GapAxis gq, gk;
    gap_axes(p, out, nullptr, nullptr, gq, gk);
    use_gaps(k, gq, gk);
    if (f32) launch_rel_fwd_f32(k, mfma_head_dim(p), p->causal != 0, st);
    else launch_rel_fwd_mfma(k, p->dtype, mfma_head_dim(p), p->causal != 0, st);
    return launch_status();
  }
  zero_packed_gaps(p, out, nullptr, nullptr, st);
  launch_rel_fwd_generic(k, p->dtype, (int)p->D, p->causal != 0, st);
  return launch_status();
}

size_t sigattn_rel_bwd_workspace_bytes(const sigattn_problem *p, const sigattn_rel_bias *r) {
  if (sigattn_rel_check(p, r) != SIGATTN_OK) return 0;
  return (size_t)rel_space(p, rel_table(r, p->H, p->Tq, p->Tk), true).bytes;
}

size_t sigattn_rel_bwd_frozen_workspace_bytes(const sigattn_problem *p, const sigattn_rel_bias *r) {
  if (sigattn_rel_check(p, r) != SIGATTN_OK) return 0;
  return (size_t)rel_space(p, rel_table(r, p->H, p->Tq, p->Tk), false).bytes;
}

int sigattn_rel_bwd(const sigattn_problem *p, const sigattn_rel_bias *r, const void *line, const void *dout, void *dq,
                    void *dk, void *dv, void *dtable, void *workspace, size_t workspace_bytes, void *stream) {
  const int rc = sigattn_rel_check(p, r);
  if (rc != SIGATTN_OK) return rc;
  if (p->H == 0) return SIGATTN_OK;
  const RelTable t = rel_table(r, p->H, p->Tq, p->Tk);
  if ((p->rows_q > 0 && (dq == nullptr || dout == nullptr)) ||
      (p->rows_k > 0 && (dk == nullptr || dv == nullptr)))
    return SIGATTN_ERR_NULL_ARG;
  const RelSpace space = rel_space(p, t, dtable != nullptr);
  if (workspace == nullptr || !aligned16(workspace) || (int64_t)workspace_bytes < space.bytes)
    return SIGATTN_ERR_WORKSPACE;
  const hipStream_t st = (hipStream_t)stream;
  RelParams k = rel_params(p, t, line != nullptr ? line : workspace);
  float *sums = (float *)((char *)workspace + space.sums);
  k.dout = dout;
  k.dq = dq;
  k.dk = dk;
  k.dv = dv;
  const void *ptrs[7] = {p->q, p->k, p->v, dout, dq, dk, dv};
  const bool f32 = use_f32_mfma(p, ptrs, 7), causal = p->causal != 0;
  const bool mfma = (f32 || use_mfma(p, ptrs, 7)) && p->Tq > 0 && p->Tk > 0;
  const int D = mfma ? mfma_head_dim(p) : (int)p->D;
  (void)hipGetLastError();
  if (!mfma) zero_packed_gaps(p, dq, dk, dv, st);
  if (p->B == 0 || p->Tq == 0) {  // no query row is in a sequence
    if (p->B > 0 && p->Tk > 0) launch_rel_dkdv_generic(rel_kv_items(k), p->dtype, D, causal, st);
    if (dtable != nullptr) launch_rel_grad(t, k, sums, dtable, st);
    return launch_status();
  }
  if (line == nullptr) make_line(p, t, workspace, st);
  if (dtable != nullptr) k.part = (float *)((char *)workspace + space.part);
  if (mfma) {
    const HeadSplit hs = head_split(p, mfma);
    k.qsplit = hs.n;
    k.kv_part = (float *)((char *)workspace + space.kv_part);
    k.part_rows = f32 ? rel_dq_rows_f32(k, D, causal) : rel_dq_rows(k, D, causal);
    RelParams kq = k;
    GapAxis gq, gk;
    gap_axes(p, dq, dk, dv, gq, gk);
    use_gaps(kq, gq, gk);
    const RelParams kk = rel_kv_items(k);
    if (f32 ? launch_rel_bwd_f32(kq, kk, D, causal, st) : launch_rel_bwd_mfma(kq, kk, p->dtype, D, causal, st)) {
      // one launch
    } else if (f32) {
      launch_rel_dq_f32(kq, D, causal, st);
      launch_rel_dkdv_f32(kk, D, causal, st);
    } else {
      launch_rel_dq_mfma(kq, p->dtype, D, causal, st);
      launch_rel_dkdv_mfma(kk, p->dtype, D, causal, st);
    }
  } else {
    launch_rel_dq_generic(k, p->dtype, D, causal, st);
    if (p->Tk > 0) launch_rel_dkdv_generic(rel_kv_items(k), p->dtype, D, causal, st);
  }
  if (dtable != nullptr) launch_rel_grad(t, k, sums, dtable, st);
  return launch_status();
}

int sigattn_paged_rel_check(const sigattn_paged_problem *p, const sigattn_rel_bias *r) {
  const int rc = sigattn_paged_check(p);
  if (rc != SIGATTN_OK) return rc;
  if (r == nullptr) return SIGATTN_ERR_NULL_ARG;
  if (r->dtype != SIGATTN_F16 && r->dtype != SIGATTN_BF16 && r->dtype != SIGATTN_F32) return SIGATTN_ERR_DTYPE;
  if (!rel_table_ok(r) || p->score_mod != nullptr) return SIGATTN_ERR_REL_BIAS;
  if (p->H > 0 && (r->table == nullptr || r->buckets == nullptr)) return SIGATTN_ERR_NULL_ARG;
  return SIGATTN_OK;
}

size_t sigattn_paged_rel_fwd_workspace_bytes(const sigattn_paged_problem *p, const sigattn_rel_bias *r) {
  if (sigattn_paged_rel_check(p, r) != SIGATTN_OK || p->rows_q == 0 || p->H == 0 || p->B == 0) return 0;
  const size_t plan = use_mfma(p, nullptr) ? make_plan(p, make_params(p, nullptr), kernel_dim(p)).bytes : 0;
  return (size_t)rel_line_bytes(rel_table_of(p, r)) + plan;
}

int sigattn_paged_rel_fwd(const sigattn_paged_problem *p, const sigattn_rel_bias *r, void *out, void *workspace,
                          size_t workspace_bytes, void *stream) {
  const int rc = sigattn_paged_rel_check(p, r);
  if (rc != SIGATTN_OK) return rc;
  if (p->rows_q == 0 || p->H == 0 || p->B == 0) return sigattn_paged_fwd(p, out, nullptr, 0, stream);
  if (out == nullptr) return SIGATTN_ERR_NULL_ARG;
  const RelTable t = rel_table_of(p, r);
  PagedRelParams k{};
  (PagedParams &)k = make_params(p, out);
  const bool mfma = use_mfma(p, out), causal = p->causal != 0;
  const int D = kernel_dim(p);
  PagedPlan pl;
  if (mfma) pl = make_plan(p, k, D);
  if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < (size_t)rel_line_bytes(t) + pl.bytes)
    return SIGATTN_ERR_WORKSPACE;
  const hipStream_t st = (hipStream_t)stream;
  k.line = (const float *)workspace, k.reach = t.reach;
  (void)hipGetLastError();
  launch_rel_line(t, (float *)workspace, nullptr, 0, nullptr, st);
  if (!mfma) {
    launch_paged_rel_generic(k, p->dtype, (int)p->D, causal, st);
    return launch_status();
  }
  run_plan(p, k, pl, (char *)workspace + rel_line_bytes(t), out, st,
           [&](const PagedRelParams &first, int nf, const PagedRelParams &kd, int nd) {
             const bool f32 = p->dtype == SIGATTN_F32;
             if (nf > 0 && nd > 0) launch_paged_rel_mixed(first, nf, kd, nd, p->dtype, D, causal, st);
             else if (nd > 0 && f32) launch_paged_rel_decode_f32(first, nd, D, causal, st);
             else if (f32) launch_paged_rel_f32(first, nf, D, causal, st);
             else if (nd > 0) launch_paged_rel_decode(first, nd, p->dtype, D, causal, st);
             else launch_paged_rel_fwd(first, nf, p->dtype, D, causal, st);
           });
  return launch_status();
}

}  // extern "C"
