// The host's side of a problem (struct sigattn_problem): its kernel parameters and
// what decides its kernels, for the files of the C ABI.
#pragma once

#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>

#include "../../include/sigattn.h"
#include "launch.h"

namespace sigattn {

inline bool is_pow2_head_dim(int64_t D) { return D == 16 || D == 32 || D == 64 || D == 128; }

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline bool aligned16(const void *ptr) { return ((uintptr_t)ptr & 15u) == 0; }

// K / V heads (version 2 of the struct ends before the field).
inline int64_t kv_heads(const sigattn_problem *p) {
  return p->abi_version >= 3 && p->kv_heads != 0 ? p->kv_heads : p->H;
}

// Query heads per K / V head.
inline int64_t head_group(const sigattn_problem *p) { return p->H > 0 ? p->H / kv_heads(p) : 1; }

inline KParams make_params(const sigattn_problem *p) {
  KParams k{};
  k.hgroup = (int)head_group(p);
  k.qgroup = 1;
  k.ncu = device_compute_units();
  k.q = p->q;
  k.k = p->k;
  k.v = p->v;
  k.bias = p->bias;
  k.scale = p->scale;
  k.score_mod = p->score_mod;
  k.seq_q = p->seq_lens_q;
  k.seq_k = p->seq_lens_k;
  k.cu_q = p->cu_seqlens_q;
  k.cu_k = p->cu_seqlens_k;
  k.rows_q = p->rows_q;
  k.rows_k = p->rows_k;
  k.sq_b = p->q_stride_b;
  k.sq_t = p->q_stride_t;
  k.sq_h = p->q_stride_h;
  k.sk_b = p->k_stride_b;
  k.sk_t = p->k_stride_t;
  k.sk_h = p->k_stride_h;
  k.B = (int)p->B;
  k.H = (int)p->H;
  k.Tq = (int)p->Tq;
  k.Tk = (int)p->Tk;
  k.dmem = (int)p->D;
  return k;
}

// T rows of `stride` 16-bit elements span less than 2^31 bytes.
inline bool rows_fit_2g(int64_t T, int64_t stride) {
  return stride == 0 || T <= (((int64_t)1 << 30) - 1) / stride;
}

// Every row start 16-byte aligned (strides in elements of `esize` bytes) and
// every row of a sequence within 2^31 bytes of the sequence's first row (the
// tile copies address rows with a 32-bit byte offset from that row).
inline bool rows_dma_ready(const sigattn_problem *p, const void *const *ptrs, int nptr, int esize) {
  const int64_t per16 = 16 / esize, half_units = esize / 2;
  if (!rows_fit_2g(p->Tq, half_units * p->q_stride_t) || !rows_fit_2g(p->Tk, half_units * p->k_stride_t))
    return false;
  const int64_t strides[6] = {p->q_stride_b, p->q_stride_t, p->q_stride_h,
                              p->k_stride_b, p->k_stride_t, p->k_stride_h};
  for (int64_t s : strides)
    if (s % per16 != 0) return false;
  for (int i = 0; i < nptr; ++i)
    if (ptrs[i] && !aligned16(ptrs[i])) return false;
  return true;
}

// True when the 16-bit MFMA kernels can take the problem: f16 / bf16, D of
// 16, 32, 64 or 128, rows as rows_dma_ready requires.
inline bool use_mfma(const sigattn_problem *p, const void *const *ptrs, int nptr) {
  if (p->dtype == SIGATTN_F32 || !is_pow2_head_dim(p->D)) return false;
  return rows_dma_ready(p, ptrs, nptr, 2);
}

// True when the fp32 MFMA kernels (three-part bf16 splits, see f32.hip) can take
// the problem: fp32, D of 16, 32, 64 or 128, rows as rows_dma_ready requires.
inline bool use_f32_mfma(const sigattn_problem *p, const void *const *ptrs, int nptr) {
  if (p->dtype != SIGATTN_F32 || !is_pow2_head_dim(p->D)) return false;
  return rows_dma_ready(p, ptrs, nptr, 4);
}

// Head dim of the MFMA kernel instance: head_dim 16 runs in the D = 32
// kernels (KParams::dmem = 16).
inline int mfma_head_dim(const sigattn_problem *p) { return p->D == 16 ? 32 : (int)p->D; }

// Head split of grouped dK/dV items (KParams::qsplit).  Items are K / V heads
// times key blocks, a group's queries long each: with few of them the GPU
// waits for the last.  The fewest parts, up to a head each, that make two
// workgroups per CU of them; the parts' fp32 sums are written and read again.
// Forward and backward, us, by workgroups per CU aimed at, none / 1 / 2 / 3 / 6:
// fp16 B=8 T=2048 lengths 512..2048 D=64 H=16 Hkv=2 443 / 264 / 263 / - / 262,
// Hkv=8 236 / 236 / 236 / - / 261; bf16 B=9 T=3001 lengths 67..3001 D=128 H=12
// Hkv=4 664 / 686 / 682 / 771 / -, Hkv=2 - / 793 / 695 / 707 / -, B=2 Hkv=4 - /
// 333 / 305 / 306 / -.  fp32, none / 2: B=1 H=16 Hkv=2 T=2048 D=128 1919 / 625, D=64
// 642 / 336, T=512 D=128 558 / 182; T=4096 H=32 Hkv=8 3919 / 3435; B=8 lengths
// 512..2048 D=64 H=16 Hkv=2 1698 / 1575; B=2 of 6 tokens H=48 Hkv=3 D=128 235 / 103.
constexpr int64_t kHeadSplitPerCu = 2;
struct HeadSplit {
  int n = 1;
  int64_t bytes = 0;
};

inline HeadSplit head_split(const sigattn_problem *p, bool mfma) {
  HeadSplit s;
  const int64_t G = head_group(p), cus = device_compute_units();
  if (!mfma || G <= 1 || p->cu_seqlens_k == nullptr || p->Tq <= 0 || p->Tk <= 0 || cus <= 0) return s;
  // Key blocks: whole ones of all rows, and a part of one for each sequence
  // (half of which are counted).
  const int64_t rows = p->rows_k < p->B * p->Tk ? p->rows_k : p->B * p->Tk;
  const int64_t items = (rows / 128 + (p->B + 1) / 2) * kv_heads(p);
  // (fp32: the nearest number, as its parts cost more.)
  const bool f32 = p->dtype == SIGATTN_F32;
  const int64_t aim = kHeadSplitPerCu * cus, up = f32 ? items / 2 : items - 1;
  int64_t n = items > 0 ? (aim + up) / items : 1;
  if (n > G) n = G;
  // Four tiles of queries a part at least: shorter ones are all start and end
  // (fp32: of D = 128, more of the shorter ones below).
  const int64_t tiles = G * cdiv(p->Tq, 64), least = f32 ? 4 * 128 / p->D : 4;
  if (n > tiles / least) n = tiles / least;
  if (n < 2) return s;
  s.n = (int)n;
  s.bytes = n * 2 * p->rows_k * kv_heads(p) * p->D * (int64_t)sizeof(float);
  return s;
}

// The dK/dV kernels' view of a problem: its items are K / V heads, each of
// which streams the queries of its group (KParams::qgroup), in k.qsplit parts.
inline KParams kv_items(const KParams &k) {
  KParams s = k;
  if (k.hgroup > 1) s.H = k.H / k.hgroup, s.qgroup = k.hgroup, s.hgroup = 1;
  return s;
}

// Packed layout: zeros on the rows of the outputs that no sequence covers
// (rows before cu_seqlens[0], past cu_seqlens[B], past the longest sequence
// Tq / Tk of a longer one), so every row of a packed output is written.
// q_out is the Q-shaped output (O or dQ), k_out0 / k_out1 the K-shaped ones
// (dK, dV); nullptr skips a tensor.  One launch for both axes, on `st`.
// The packed axes whose output rows outside every sequence must be zeroed:
// a for the Q-shaped output, b for the K-shaped ones (rows = 0: none).
inline void gap_axes(const sigattn_problem *p, void *q_out, void *k_out0, void *k_out1, GapAxis &a,
              GapAxis &b) {
  a = b = GapAxis{};
  if (p->H == 0) return;
  if (p->cu_seqlens_q != nullptr && q_out != nullptr && p->rows_q > 0) {
    a.cu = p->cu_seqlens_q;
    a.B = (int)p->B, a.T = (int)p->Tq, a.H = (int)p->H, a.D = (int)p->D;
    a.rows = p->rows_q, a.st = p->q_stride_t, a.sh = p->q_stride_h;
    a.out[0] = q_out;
  }
  if (p->cu_seqlens_k != nullptr && (k_out0 != nullptr || k_out1 != nullptr) && p->rows_k > 0) {
    b.cu = p->cu_seqlens_k;
    b.B = (int)p->B, b.T = (int)p->Tk, b.H = (int)kv_heads(p), b.D = (int)p->D;
    b.rows = p->rows_k, b.st = p->k_stride_t, b.sh = p->k_stride_h;
    b.out[0] = k_out0, b.out[1] = k_out1;
  }
}

// Zeroes those rows with a launch of their own (paths whose kernels do not
// take KParams::gap, and calls that launch no attention kernel).
inline void zero_packed_gaps(const sigattn_problem *p, void *q_out, void *k_out0, void *k_out1, hipStream_t st) {
  GapAxis a, b;
  gap_axes(p, q_out, k_out0, k_out1, a, b);
  launch_zero_gaps(a, b, p->dtype == SIGATTN_F32 ? 4 : 2, st);
}

// Hands axes a and b to the kernel launched with `k` (a forward or dQ
// kernel): its first workgroups, a multiple of 8 per axis, zero the axes'
// gap rows (KParams::gap).
inline void use_gaps(KParams &k, const GapAxis &a, const GapAxis &b) {
  const GapAxis *ax[2] = {&a, &b};
  for (int i = 0; i < 2; ++i) {
    k.gap[i] = *ax[i];
    k.ngap[i] = ax[i]->rows > 0 ? (int)(cdiv(cdiv(ax[i]->rows, 64), 8) * 8) : 0;
  }
}

inline int launch_status() {
  return hipGetLastError() == hipSuccess ? SIGATTN_OK : SIGATTN_ERR_LAUNCH;
}

}  // namespace sigattn
