// C ABI of the attention over a paged cache (include/sigattn.h): validation on
// the host, before any HIP call, and the choice of kernels.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>

#include "../../include/sigattn.h"
#include "launch.h"
#include "paged.h"
#include "rel.h"

using sigattn::kDecodeCols;
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

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool aligned16(const void *ptr) { return ((uintptr_t)ptr & 15u) == 0; }

// The MFMA kernels take rows that start on 16-byte boundaries (and 16 of which
// lie within 2^31 bytes).
bool use_mfma(const sigattn_paged_problem *p, const void *out) {
  const int64_t strides[5] = {p->q_stride_t, p->q_stride_h, p->k_stride_p, p->k_stride_t, p->k_stride_h};
  for (int64_t s : strides)
    if (s % (p->dtype == SIGATTN_F32 ? 4 : 8) != 0) return false;
  return p->k_stride_t < (int64_t)1 << 25 && aligned16(p->q) && aligned16(p->k_cache) && aligned16(p->v_cache) &&
         aligned16(out);
}

// Head dim of the kernel instance: head_dim 16 runs in the D = 32 kernels.
int kernel_dim(const sigattn_paged_problem *p) { return p->D == 16 ? 32 : (int)p->D; }

// What one kernel runs: its units at most (the device finds out how many there
// are), how it cuts sequences (PagedParams) and the partials that takes.
struct Part {
  int64_t units = 0;
  int split_units = 0, total_units = 0, min_chunk = 0, block = 0;
  size_t partial_bytes = 0;
};

// Sequences of up to kDecodeCols columns run in the decode kernel, longer ones
// in the forward's; a batch of one, whose length the host knows to be a long
// one or does not know, runs in the forward's alone.
// The decode kernel's chunks: a round of the waves that the GPU runs at a time
// at D = 128 (four per CU), of 64 keys at least.  Whole call, us, bf16 H=32 Hkv=8
// D=128: waves per CU 4 / 8, B=16 contexts 1024..8191 49 / 55, B=64 1024..3000 100 /
// 101, B=64 8000..9000 H=8 338 / 343 (6.57 TB/s); chunks of 64 / 128 / 192 keys at
// least, B=1 2000 keys 13.9 / 16.1 / 17.3, B=16 200..300 18.2 / 20.2 / 21.4, B=3
// up to 8000 15.2 / 16.6 / 18.7, longer ones alike.
constexpr int64_t kDecodeWavesPerCu = 4, kDecodeChunk = 64;
// The forward kernel's chunks, where its blocks do not fill the GPU: a round of
// its workgroups, of 1024 keys at least.  Whole call, us, one / two rounds: bf16
// H=32 Hkv=8 D=128, 2 x 1024 tokens on up to 12000 keys 324 / 343, 256 on 12000
// 57 / 77, 4 x 128 114 / 132, 2000 on none 59 / 89; chunks of 512 / 1024 / 2048
// keys, 24 requests, 4 of up to 700 tokens on up to 4096 keys, H=12 Hkv=4 D=128
// 87 / 69 / 83.
constexpr int64_t kChunk = 1024;
// (fp32 blocks: two rounds' worth of workgroups; chunks of 64 / 128 / 256 keys, us,
// B=1 2000 keys 18 / 27 / 46.)
constexpr int64_t kChunkF32 = 64;
struct Plan {
  Part fwd, decode;
  int cols_lo = 0;  // columns that are not the forward kernel's
  size_t cut_bytes = 0, bytes = 0;
};

// Sequences are cut so that a part fills the `t` workgroups (waves) that run at
// a time, once where its uncut units may be fewer; where they are more already,
// into as many units as three rounds, so that uneven lengths even out.  Whole
// call, us, half a round more / two: bf16 H=32 Hkv=8 D=128, t = 1024: B=128
// contexts 10..4000 194 / 181, B=300 10..2000 215 / 209, B=200 100..900 81 / 81;
// fewer uncut units than t, B=64 8000..9000 H=8 338 / 357, 1024..3000 97 / 109.
//
// Decoding stays uncut where a wave is through its sequence before the sums would
// be added: in tables of few keys, or few for the rounds that the uncut units
// take, and (the table may be longer than what is in it) in batches of four rounds
// and of 1024 sequences, whose lengths every wave goes through to find a cut
// unit.  Whole call, us, cut / not, bf16 H=32 Hkv=8 D=128: B=16 up to 160 keys 16.5
// / 11.2, 300 17.5 / 16.9, 600 18.3 / 26.9; B=64 300 25.3 / 19.6, 600 32.0 / 31.1,
// 1200 46 / 56; B=200 300 50 / 37, 1200 121 / 117, 50..4800 318 / 378; B=512 300 105 /
// 75, 50..4000 737 / 726; B=4096 300 2042 / 563.  Hkv=1 H=8: B=1000 50..4000 217 /
// 204, B=3000 642 / 552.  fp32: B=16 300 24.6 / 48.5, B=64 36 / 50, B=128 72 / 54, 600
// 104 / 92.
void cut_part(Part &part, int64_t uncut, int64_t t, int64_t min_chunk, const PagedParams &k, int D, bool decode,
              bool f32) {
  const int64_t few = f32 ? 0 : 320, per_round = f32 ? 500 : 1200;
  part.units = uncut;
  if (k.Tk <= min_chunk || t <= 0) return;
  if (decode && (k.Tk <= few || k.Tk * t <= per_round * uncut || uncut >= 4 * t || k.B >= 1024)) return;
  const int64_t most = uncut * cdiv(k.Tk, min_chunk);
  int64_t extra = uncut >= t ? 2 * t : t - uncut > t / 2 ? t - uncut : t / 2;
  if (extra > most) extra = most;
  part.split_units = (int)extra;
  part.min_chunk = (int)min_chunk;
  part.total_units = (int)(uncut + extra);
  // One more unit per K / V head than the sums say: their rounding.
  part.units = uncut + extra + k.Hkv;
  part.partial_bytes = (size_t)part.units * part.block * D * sizeof(float);
}

Plan make_plan(const sigattn_paged_problem *p, const PagedParams &k, int D) {
  Plan pl;
  const int64_t cols = (int64_t)k.Tq * k.G, all = p->rows_q * k.G, cus = k.ncu;
  // (fp32: no launch for both, so one long sequence takes all to the blocks.)
  const bool f32 = p->dtype == SIGATTN_F32;
  const bool decode = cols <= kDecodeCols || (k.B > 1 && !f32), fwd = cols > kDecodeCols;
  pl.fwd.block = f32 ? sigattn::kPagedBlockF32 : sigattn::paged_block(D), pl.decode.block = kDecodeCols;
  if (decode) {
    const int64_t pairs = (int64_t)k.B * k.Hkv;
    cut_part(pl.decode, pairs, kDecodeWavesPerCu * cus, kDecodeChunk, k, D, true, f32);
  }
  if (fwd) {
    if (decode) pl.cols_lo = kDecodeCols;
    // Blocks: whole ones of all columns, and one that is not whole for each
    // sequence of the kernel's.
    const int64_t seqs = all / (pl.cols_lo + 1) < k.B ? all / (pl.cols_lo + 1) : k.B;
    const int64_t uncut = (all / pl.fwd.block + seqs) * k.Hkv, per_cu = f32 ? 2 : D == 128 ? 1 : (D == 64 ? 3 : 4);
    const int64_t full = cdiv(all, pl.fwd.block) * k.Hkv;
    cut_part(pl.fwd, uncut, full < per_cu * cus ? per_cu * cus : 0, f32 ? kChunkF32 : kChunk, k, D, false, f32);
  }
  const bool cut = pl.fwd.split_units > 0 || pl.decode.split_units > 0;
  pl.cut_bytes = cut ? cdiv((int64_t)k.B * 2 * (int64_t)sizeof(int2), 256) * 256 : 0;
  pl.bytes = pl.cut_bytes + pl.fwd.partial_bytes + pl.decode.partial_bytes;
  return pl;
}

// k's fields for one part of a plan (part.split_units 0: nothing is cut).
PagedParams of_part(const PagedParams &k, const Part &part, int lo, int hi, int2 *cut, float *ws) {
  PagedParams s = k;
  s.cols_lo = lo, s.cols_hi = hi;
  s.split_units = part.split_units, s.total_units = part.total_units, s.min_chunk = part.min_chunk;
  s.max_units = (int)part.units;
  s.cut = cut, s.ws = ws;
  return s;
}

// The learned bias's table as far as the cache's sequences reach.
sigattn::RelTable rel_table_of(const sigattn_paged_problem *p, const sigattn_rel_bias *r) {
  return sigattn::rel_table(r, p->H, p->max_seqlen_q < p->rows_q ? p->max_seqlen_q : p->rows_q,
                            p->max_pages * p->page_size);
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
  Plan pl;
  if (mfma) pl = make_plan(p, k, D);
  if (workspace != nullptr && pl.bytes > 0 && (workspace_bytes < pl.bytes || !aligned16(workspace)))
    return SIGATTN_ERR_WORKSPACE;
  if (workspace == nullptr) {  // nothing is cut
    pl.fwd.split_units = pl.decode.split_units = 0;
  }
  (void)hipGetLastError();
  sigattn::GapAxis gap;
  gap.cu = p->cu_seqlens_q, gap.B = k.B, gap.T = k.Tq, gap.H = k.H, gap.D = (int)p->D;
  gap.rows = p->rows_q, gap.st = p->H * p->D, gap.sh = p->D, gap.out[0] = out;
  if (p->B == 0) {  // no sequence: every row is outside
    sigattn::launch_zero_gaps(gap, sigattn::GapAxis{}, dt == SIGATTN_F32 ? 4 : 2, st);
    return launch_status();
  }
  if (!mfma) {
    sigattn::launch_paged_generic(k, dt, (int)p->D, causal, st);
    return launch_status();
  }
  // The workspace: both parts' cuts, then their partials.
  const auto at = [&](size_t bytes) -> void * { return workspace != nullptr ? (char *)workspace + bytes : nullptr; };
  k.gap[0] = gap;
  // The kernel also zeroes the rows outside every sequence (workgroups in
  // a multiple of 8, so that its items keep their XCDs).
  const int gaps = (int)(cdiv(cdiv(p->rows_q, 64), 8) * 8);
  const PagedParams kf = of_part(k, pl.fwd, pl.cols_lo, INT_MAX, (int2 *)at(0), (float *)at(pl.cut_bytes));
  const PagedParams kd = of_part(k, pl.decode, 0, pl.decode.units > 0 ? kDecodeCols : 0,
                                 (int2 *)at((size_t)p->B * sizeof(int2)),
                                 (float *)at(pl.cut_bytes + pl.fwd.partial_bytes));
  PagedParams first = pl.fwd.units > 0 ? kf : kd;
  first.ngap[0] = gaps;
  if (pl.fwd.units > 0 && pl.decode.units > 0)
    sigattn::launch_paged_mixed(first, (int)pl.fwd.units, kd, (int)pl.decode.units, dt, D, causal, st);
  else if (pl.decode.units > 0 && dt == SIGATTN_F32)
    sigattn::launch_paged_decode_f32(first, (int)pl.decode.units, D, causal, st);
  else if (pl.decode.units > 0) sigattn::launch_paged_decode(first, (int)pl.decode.units, dt, D, causal, st);
  else if (dt == SIGATTN_F32) sigattn::launch_paged_f32(first, (int)pl.fwd.units, D, causal, st);
  else sigattn::launch_paged_fwd(first, (int)pl.fwd.units, dt, D, causal, st);
  if (kf.split_units > 0 || kd.split_units > 0) sigattn::launch_paged_reduce(kf, kd, dt, D, st);
  return launch_status();
}

int sigattn_paged_rel_check(const sigattn_paged_problem *p, const sigattn_rel_bias *r) {
  const int rc = sigattn_paged_check(p);
  if (rc != SIGATTN_OK) return rc;
  if (r == nullptr) return SIGATTN_ERR_NULL_ARG;
  if (r->dtype != SIGATTN_F16 && r->dtype != SIGATTN_BF16 && r->dtype != SIGATTN_F32) return SIGATTN_ERR_DTYPE;
  if (!sigattn::rel_table_ok(r) || p->score_mod != nullptr) return SIGATTN_ERR_REL_BIAS;
  if (p->H > 0 && (r->table == nullptr || r->buckets == nullptr)) return SIGATTN_ERR_NULL_ARG;
  return SIGATTN_OK;
}

size_t sigattn_paged_rel_fwd_workspace_bytes(const sigattn_paged_problem *p, const sigattn_rel_bias *r) {
  if (sigattn_paged_rel_check(p, r) != SIGATTN_OK || p->rows_q == 0 || p->H == 0 || p->B == 0) return 0;
  return (size_t)sigattn::rel_line_bytes(rel_table_of(p, r));
}

int sigattn_paged_rel_fwd(const sigattn_paged_problem *p, const sigattn_rel_bias *r, void *out, void *workspace,
                          size_t workspace_bytes, void *stream) {
  const int rc = sigattn_paged_rel_check(p, r);
  if (rc != SIGATTN_OK) return rc;
  if (p->rows_q == 0 || p->H == 0 || p->B == 0) return sigattn_paged_fwd(p, out, nullptr, 0, stream);
  if (out == nullptr) return SIGATTN_ERR_NULL_ARG;
  const sigattn::RelTable t = rel_table_of(p, r);
  if (workspace == nullptr || !aligned16(workspace) || (int64_t)workspace_bytes < sigattn::rel_line_bytes(t))
    return SIGATTN_ERR_WORKSPACE;
  const hipStream_t st = (hipStream_t)stream;
  sigattn::PagedRelParams k{};
  (PagedParams &)k = make_params(p, out);
  k.line = (const float *)workspace, k.reach = t.reach;
  (void)hipGetLastError();
  sigattn::launch_rel_line(t, (float *)workspace, st);
  sigattn::launch_paged_rel_generic(k, p->dtype, (int)p->D, p->causal != 0, st);
  return launch_status();
}

}  // extern "C"
