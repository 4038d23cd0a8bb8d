// The host's side of attention over a paged cache (struct sigattn_paged_problem):
// its kernel parameters and the choice of kernels.
#pragma once

#include "paged.h"
#include "problem.h"

namespace sigattn {

inline PagedParams make_params(const sigattn_paged_problem *p, void *out) {
  PagedParams k{};
  k.ncu = device_compute_units();
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

// The MFMA kernels take rows that start on 16-byte boundaries (and 16 of which
// lie within 2^31 bytes).
inline bool use_mfma(const sigattn_paged_problem *p, const void *out) {
  const int64_t strides[5] = {p->q_stride_t, p->q_stride_h, p->k_stride_p, p->k_stride_t, p->k_stride_h};
  for (int64_t s : strides)
    if (s % (p->dtype == SIGATTN_F32 ? 4 : 8) != 0) return false;
  return p->k_stride_t < (int64_t)1 << 25 && aligned16(p->q) && aligned16(p->k_cache) && aligned16(p->v_cache) &&
         aligned16(out);
}

// Head dim of the kernel instance: head_dim 16 runs in the D = 32 kernels.
inline int kernel_dim(const sigattn_paged_problem *p) { return p->D == 16 ? 32 : (int)p->D; }

// What one kernel runs: its units at most (the device finds out how many there
// are), how it cuts sequences (PagedParams) and the partials that takes.
struct PagedPart {
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
struct PagedPlan {
  PagedPart fwd, decode;
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
inline void cut_part(PagedPart &part, int64_t uncut, int64_t t, int64_t min_chunk, const PagedParams &k, int D, bool decode,
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

inline PagedPlan make_plan(const sigattn_paged_problem *p, const PagedParams &k, int D) {
  PagedPlan pl;
  const int64_t cols = (int64_t)k.Tq * k.G, all = p->rows_q * k.G, cus = k.ncu;
  // (fp32: no launch for both, so one long sequence takes all to the blocks.)
  const bool f32 = p->dtype == SIGATTN_F32;
  const bool decode = cols <= kDecodeCols || (k.B > 1 && !f32), fwd = cols > kDecodeCols;
  pl.fwd.block = f32 ? kPagedBlockF32 : paged_block(D), pl.decode.block = kDecodeCols;
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
template <class P> P of_part(const P &k, const PagedPart &part, int lo, int hi, int2 *cut, float *ws) {
  P s = k;
  s.cols_lo = lo, s.cols_hi = hi;
  s.split_units = part.split_units, s.total_units = part.total_units, s.min_chunk = part.min_chunk;
  s.max_units = (int)part.units;
  s.cut = cut, s.ws = ws;
  return s;
}

// The rows of `out` that no sequence covers.
inline GapAxis paged_gap(const sigattn_paged_problem *p, const PagedParams &k, void *out) {
  GapAxis gap;
  gap.cu = p->cu_seqlens_q, gap.B = k.B, gap.T = k.Tq, gap.H = k.H, gap.D = (int)p->D;
  gap.rows = p->rows_q, gap.st = p->H * p->D, gap.sh = p->D, gap.out[0] = out;
  return gap;
}

// Runs a plan's parts, launch(first part's parameters, blocks, decoding part's
// parameters, decoding units), and the sums of what they cut.  The workspace
// (nullptr: the plan cuts nothing): both parts' cuts, then their partials.  P:
// PagedParams, or with the learned bias.
template <class P, class Launch>
void run_plan(const sigattn_paged_problem *p, P k, const PagedPlan &pl, char *workspace, void *out, hipStream_t st,
              Launch &&launch) {
  const auto at = [&](size_t bytes) -> void * { return workspace != nullptr ? workspace + bytes : nullptr; };
  k.gap[0] = paged_gap(p, k, out);
  const P kf = of_part(k, pl.fwd, pl.cols_lo, INT_MAX, (int2 *)at(0), (float *)at(pl.cut_bytes));
  const P kd = of_part(k, pl.decode, 0, pl.decode.units > 0 ? kDecodeCols : 0, (int2 *)at((size_t)p->B * sizeof(int2)),
                       (float *)at(pl.cut_bytes + pl.fwd.partial_bytes));
  // The kernel also zeroes the rows outside every sequence (workgroups in
  // a multiple of 8, so that its items keep their XCDs).
  P first = pl.fwd.units > 0 ? kf : kd;
  first.ngap[0] = (int)(cdiv(cdiv(p->rows_q, 64), 8) * 8);
  launch(first, (int)pl.fwd.units, kd, (int)pl.decode.units);
  if (kf.split_units > 0 || kd.split_units > 0)
    launch_paged_reduce(kf, kd, p->dtype, p->D == 16 ? 32 : (int)p->D, st);
}

}  // namespace sigattn
