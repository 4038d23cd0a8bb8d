// Bodies of the recompute backward's kernels (see bwd.hip), shared by the plain ones
// and those with a learned bias by relative position.
#pragma once

#include <type_traits>

#include "common.h"
#include "rel.h"

namespace sigattn {

// ---------------------------------------------------------------------------
// dQ: workgroup = 4 waves x 32 queries; walks 64-key tiles of K and V.
//   Sᵀ = K·Qᵀ, dPᵀ = V·dOᵀ (accumulators: lane = query column),
//   dQᵀ += Kᵀ·dSᵀ with dSᵀ taken from the accumulator registers and Kᵀ read
//   from the K tile with ds_read_b64_tr_b16.
// ---------------------------------------------------------------------------
// WK = 2: two pairs of waves of 32 queries; the waves of a pair hold the same
// queries, take one 32-key block of every tile each, and their accumulators
// are added at the end (launch_bwd_dq_mfma says where).
// A learned bias by relative position (P::kRel): WIN places of the head's line are
// staged with each tile, and dS is summed by relative position (PlaceSums).
template <class P, int WK, int NW = 4> constexpr int dq_window() { return P::kRel ? 32 * NW / WK + 64 : 0; }
template <int D, bool SCOREMOD, int WIN = 0> struct DqLds {
  uint16_t k[2][64 * D], v[2][64 * D];
  float c[WIN > 0 ? 2 * WIN : (SCOREMOD ? 2 * 64 : 4)];
};
// (NW waves; eight only with P::kRel at D = 128.)
template <typename T, int D, int WK, bool CAUSAL, bool SCOREMOD, class P = KParams, int NW = 4>
__device__ __forceinline__ void bwd_dq_body(const P &p, const int wg, DqLds<D, SCOREMOD, dq_window<P, WK, NW>()> &lds,
                                            float *near = nullptr) {
  constexpr int NG = NW / WK, BM = 32 * NG, BN = 64;
  constexpr int WIN = dq_window<P, WK, NW>();
  constexpr bool REL = P::kRel;
  constexpr int NKS = D / 16, NDB = D / 32;
  auto &sK = lds.k;
  auto &sV = lds.v;
  auto &sC = lds.c;

  int b, h, qb;
  int ritem = 0, rchunk = 0;  // range split: the item and this workgroup's chunk of its keys
  if (WK == 1 && !CAUSAL && p.rsplit > 1) {
    int bh;
    ritem = wg / p.rsplit, rchunk = wg % p.rsplit;
    dense_item(ritem, p.B * p.H, p.nblk, true, bh, qb);
    b = bh / p.H, h = bh % p.H;
  } else if (p.ragged() && p.B <= 64) {
    const auto lq = [&](int i) SIGATTN_INLINE { return p.len_q(i); };
    const auto lk = [&](int i) SIGATTN_INLINE { return p.len_k(i); };
    const WorkItem it = CAUSAL ? WorkOrder::by_level(wg, p.B, p.H, lq, BM, p.nblk, true, p.ncu,
                                                     D <= 64 ? 3 : 8 / NW)
                               : WorkOrder::by_stream(wg, p.B, p.H, lq, BM, p.nblk, lk);
    b = it.b, h = it.h, qb = it.blk;
  } else {
    const int BH = p.B * p.H;
    int bh;
    dense_item(wg, BH, p.nblk, !CAUSAL, bh, qb);
    if (CAUSAL) qb = p.nblk - 1 - qb;  // heaviest query blocks first
    b = bh / p.H, h = bh % p.H;
  }
  const int Lq = p.len_q(b);
  // Keys of this workgroup: under the range split, its chunk of the item's
  // key tiles, indexed from the chunk's first key.
  int key0 = 0, Lk = p.len_k(b);
  if (WK == 1 && !CAUSAL && p.rsplit > 1) {
    const int ntk = (Lk + BN - 1) / BN;
    key0 = split_tile(rchunk, p.rsplit, ntk) * BN;
    Lk = min(Lk, split_tile(rchunk + 1, p.rsplit, ntk) * BN) - key0;
  }
  const bool half = p.half_head(D);  // head_dim 16 in this D = 32 kernel
  // Padding item: its zero rows as part of one contiguous span (see zero_row_span).
  if (qb * BM >= Lq && p.q_rows_contiguous(half ? 16 : D)) {
    zero_row_span((uint16_t *)p.dq + (int64_t)b * p.sq_b, p.sq_t, qb * BM, min(qb * BM + BM, p.Tq), h, p.H,
                  threadIdx.x, 64 * NW);
    return;
  }

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = WK == 2 ? __builtin_amdgcn_readfirstlane(tid >> 6) : tid >> 6;
  const int l32 = lane & 31, hi = lane >> 5;
  const int wt = w / NG;  // place in the wave's pair (WK = 2)
  const int q0 = qb * BM, qw = q0 + (w % NG) * 32, my_q = qw + l32;

  const int64_t qoff = p.q_base(b, h);
  const int64_t koff = p.k_base(b, h) + (int64_t)key0 * p.sk_t;
  const uint16_t *Qb = (const uint16_t *)p.q + qoff;
  const uint16_t *dOb = (const uint16_t *)p.dout + qoff;
  const uint16_t *Kb = (const uint16_t *)p.k + koff;
  const uint16_t *Vb = (const uint16_t *)p.v + koff;
  uint16_t *dQb = (uint16_t *)p.dq + qoff;

  int nend = Lk;
  if (CAUSAL) nend = min(nend, min(q0 + BM, Lq));
  if (q0 >= Lq) nend = 0;
  const int ntiles = (nend + BN - 1) / BN;

  const float scale = *p.scale;
  const float bias = p.bias[b];
  const float nsl = -scale * kLog2e, nbl = -bias * kLog2e;

  u32x4 qf[NKS], of[NKS];
  {
    const bool ok = my_q < Lq;
    const uint16_t *qr = Qb + (int64_t)my_q * p.sq_t + 8 * hi;
    const uint16_t *orow = dOb + (int64_t)my_q * p.sq_t + 8 * hi;
#pragma unroll
    for (int s = 0; s < NKS; ++s) {
      const bool in = ok && !(half && s > 0);
      qf[s] = in ? *(const u32x4 *)(qr + 16 * s) : zero4();
      of[s] = in ? *(const u32x4 *)(orow + 16 * s) : zero4();
    }
  }
  f32x16 acc[NDB];
#pragma unroll
  for (int d = 0; d < NDB; ++d) acc[d] = zero16();

  TileOffsets<D> to;
  to.init(lane);
  if constexpr (WK == 2) to.advance(32 * wt);  // this wave's half of every tile
  DmaPlan<BN, D, NW> dma;
  dma.init(w, lane, half);
  const int kv_stride_bytes = (int)(p.sk_t * 2);

  [[maybe_unused]] const int win0 = BM - (w % NG) * 32 - l32 + 4 * hi;  // this lane's place of the tile's key 0
  [[maybe_unused]] PlaceSums<NW> sums;
  if constexpr (REL) sums.init(p, near, w, tid);

  // dS of one 32-key block into eight packed words.
  auto ds_block = [&](const f32x16 &s, const f32x16 &dp, int st, int kl, int kbase, uint32_t *out,
                      bool mask) SIGATTN_INLINE {
    float c[16];
    if constexpr (REL) {
#pragma unroll
      for (int i = 0; i < 16; ++i) c[i] = sC[st * WIN + kl + 8 * (i / 4) + i % 4 + win0];
    } else if constexpr (SCOREMOD) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 cv = *(const float4 *)&sC[st * BN + kl + 8 * g + 4 * hi];
        c[4 * g + 0] = cv.x; c[4 * g + 1] = cv.y; c[4 * g + 2] = cv.z; c[4 * g + 3] = cv.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) c[i] = nbl;
    }
    float ds[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float pr = sigmoid_from_neg_log2(__builtin_fmaf(s[i], nsl, c[i]));
      const float t = pr * dp[i];
      ds[i] = __builtin_fmaf(-pr, t, t);
    }
    if (mask) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = kbase + 8 * (i / 4) + 4 * hi + (i % 4);
        if (key >= Lk || (CAUSAL && key > my_q) || (REL && my_q >= Lq)) ds[i] = 0.0f;
      }
    }
    if constexpr (REL) {
      sums.add(ds, kbase - qw, l32, hi);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = Elem<T>::pack(ds[2 * i], ds[2 * i + 1]);
  };

  // dQᵀ[d, q] += Kᵀ[d, key] · dSᵀ[key, q] for the two 16-key steps of block kbi.
  auto dq_block = [&](int st, int kbi, const uint32_t *dsk) SIGATTN_INLINE {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const u32x4 bop = (u32x4){dsk[4 * j], dsk[4 * j + 1], dsk[4 * j + 2], dsk[4 * j + 3]};
#pragma unroll
      for (int db = 0; db < NDB; ++db)
        acc[db] = Elem<T>::mfma(ld_tr<D>(sK[st], to, 2 * kbi + j, db), bop, acc[db]);
    }
  };

  // Per 32-key block: Sᵀ/dPᵀ chains (16 MFMA), dS (VALU), dQ (8 MFMA).  The
  // blocks run one after the other (four 32x32 fp32 accumulators plus the Q
  // and dO operands would not fit next to the dQ accumulators); the second
  // wave on each SIMD supplies the MFMA/VALU overlap.
  auto tile_step = [&](int st, int n0, bool mask) SIGATTN_INLINE {
    const int cl = WK == 2 ? 32 * wt : 0;
#pragma unroll
    for (int kbi = 0; kbi < 2 / WK; ++kbi) {
      f32x16 s = zero16(), dp = zero16();
      uint32_t dk[8];
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        s = Elem<T>::mfma(ld_row<D>(sK[st], to, 32 * kbi, ks), qf[ks], s);
        dp = Elem<T>::mfma(ld_row<D>(sV[st], to, 32 * kbi, ks), of[ks], dp);
      }
      ds_block(s, dp, st, 32 * kbi + cl, n0 + 32 * kbi + cl, dk, mask);
      dq_block(st, kbi, dk);
    }
  };

  float creg = 0.0f;
  auto load_c = [&](int n0) SIGATTN_INLINE {
    if (SCOREMOD && tid < BN) {
      const int key = n0 + tid;
      creg = key < Lk ? -(bias + p.score_mod[p.mod_base(b) + key0 + key]) * kLog2e : 0.0f;
    }
    if constexpr (REL) {
      if (tid < WIN) creg = rel_at(p, h, n0 + tid - q0 - BM);
    }
  };
  auto issue = [&](int st, int n0) SIGATTN_INLINE {
    dma.issue(sK[st], Kb, kv_stride_bytes, n0, Lk);
    dma.issue(sV[st], Vb, kv_stride_bytes, n0, Lk);
  };
  auto iteration = [&](int it, auto stage_tag) SIGATTN_INLINE {
    constexpr int ST = decltype(stage_tag)::value;
    const int n0 = it * BN;
    wait_dma();
    if (SCOREMOD && tid < BN) sC[ST * BN + tid] = creg;
    if constexpr (REL) {
      if (tid < WIN) sC[ST * WIN + tid] = -(bias + creg) * kLog2e;
    }
    __syncthreads();
    if (it + 1 < ntiles) {
      load_c(n0 + BN);
      issue(ST ^ 1, n0 + BN);
    }
    if (!CAUSAL || n0 + (WK == 2 ? 32 * wt : 0) <= qw + 31) {
      // (REL: rows past the last query have dS = 0 too, whatever a key holds: 0 * inf is none.)
      tile_step(ST, n0, (n0 + BN > Lk) || (CAUSAL && n0 + BN - 1 > qw) || (REL && qw + 32 > Lq));
    }
  };

  if (ntiles > 0) {
    load_c(0);
    issue(0, 0);
  }
  for (int it = 0; it < ntiles; it += 2) {
    iteration(it, std::integral_constant<int, 0>{});
    if (it + 1 < ntiles) iteration(it + 1, std::integral_constant<int, 1>{});
  }

  if constexpr (REL) {
    if (q0 < Lq) sums.finish(p, near, b, qb, h, w, tid);  // (no other block: its place may be another's)
  }

  if constexpr (WK == 2) {
    if (!pair_add<NDB, NG>([&](int i) SIGATTN_INLINE -> f32x16 & { return acc[i]; }, (float *)&sK[0][0], w, lane))
      return;
  }
  if (WK == 1 && !CAUSAL && p.rsplit > 1 &&
      !split_combine<NDB, 4>([&](int i) SIGATTN_INLINE -> f32x16 & { return acc[i]; },
                             p.rs_part + (int64_t)ritem * p.rsplit * (BM * D), p.rs_cnt + ritem, rchunk,
                             p.rsplit, w, lane))
    return;

  if (my_q < p.q_rows_out(Lq)) {
    uint16_t *row = dQb + (int64_t)my_q * p.sq_t;
    const bool valid = my_q < Lq;
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (half && g >= 2) break;  // columns 16..31: not in the tensor
        const int d0 = db * 32 + 8 * g + 4 * hi;
        u32x2 o;
        o.x = Elem<T>::pack(acc[db][4 * g] * scale, acc[db][4 * g + 1] * scale);
        o.y = Elem<T>::pack(acc[db][4 * g + 2] * scale, acc[db][4 * g + 3] * scale);
        if (!valid) o = (u32x2){0u, 0u};
        *(u32x2 *)(row + d0) = o;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// dK/dV: workgroup = 4 waves x 32 keys (one wave per SIMD); the
// queries stream through a 4-stage ring of 64-query Q and dO tiles as a
// continuous sequence of 32-query blocks g.  Per block and wave:
//   S = Q·Kᵀ and dP = dO·Vᵀ (A: Q / dO rows from LDS, B: K / V rows held in
//   registers; accumulators: lane = key column, registers = query rows),
//   dVᵀ += dOᵀ·P and dKᵀ += Qᵀ·dS (A: dOᵀ / Qᵀ via ds_read_b64_tr_b16,
//   B: packed P / dS words straight from the accumulator layout).
// Region r runs, as one straight-line sequence, the S / dP MFMAs of block r,
// the gradient MFMAs of block r-2 and the P / dS VALU work of block r-1; every
// MFMA A operand is read from LDS eight MFMAs ahead through a rotating
// register queue, so no MFMA waits on a fresh LDS read.  Element masks
// (causal diagonal, seq_lens_q, pipeline fill) are applied to the packed
// words of the few blocks that need them.
// ---------------------------------------------------------------------------
// The queries that a dK/dV item streams, as tiles t and 32-query blocks g
// counted through: those of one query head, or (GROUPED) of the qgroup heads
// that share the item's K / V head, one head after another without a break in
// the pipeline.  dK and dV of a shared head are the sums over its query heads,
// so they stay in the same accumulators.  Tiles and blocks are visited in
// order, so their places within a head are counters, not divisions.  The rate is
// that of heads with keys of their own where the items fill the GPU (bf16 causal
// B=1 T=8192 H=32 D=128, dK/dV with dS: H_kv = 8 1.16 ms, 32 1.17 + 0.21 ms in the
// two passes that its larger dS takes; B=9 lengths 67..3001 H=12: H_kv = 4 398 us,
// 12 417), and 15 % less at D = 64, split (fp16 B=8 lengths 512..2048 H=16: H_kv =
// 2 126 us and 9 for the parts, 16 110).
template <bool GROUPED> struct HeadStream {
  int nb = 0;                                      // blocks of one head
  int t1 = 0, th = 0;                              // next tile to copy: place in its head, head
  int g[3] = {0, -1, -2}, h[3] = {0, 0, 0};        // blocks r, r - 1, r - 2: the same
  __device__ __forceinline__ explicit HeadStream(int blocks) {
    if constexpr (GROUPED) nb = blocks;
  }
  __device__ __forceinline__ int tile(int t) const { return GROUPED ? t1 : t; }
  __device__ __forceinline__ int64_t head_of_tile(int) const { return GROUPED ? th : 0; }
  __device__ __forceinline__ void next_tile() {
    if constexpr (GROUPED) {
      if (2 * ++t1 == nb) t1 = 0, ++th;
    }
  }
  // Block r - back of region r within its head (negative: pipeline fill).
  __device__ __forceinline__ int block(int r, int back) const { return GROUPED ? g[back] : r - back; }
  __device__ __forceinline__ int head(int back) const { return GROUPED ? h[back] : 0; }
  __device__ __forceinline__ void next_block() {
    if constexpr (GROUPED) {
      g[2] = g[1], h[2] = h[1], g[1] = g[0], h[1] = h[0];
      if (++g[0] == nb) g[0] = 0, ++h[0];
    }
  }
};

// A lane's row of fp32 dK (t = 0) or dV (t = 1) of a head-split item, times `f`.
template <int NDB>
__device__ __forceinline__ void store_part(const KParams &p, int part, int b, int key, int h, const f32x16 (&acc)[NDB],
                                           int t, float f, int hi, bool half) {
  float *row = p.part_row(part, t, packed_first(p.cu_k, p.rows_k, b) + key, h);
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (half && g >= 2) break;  // columns 16..31: not in the tensor
      const f32x16 &a = acc[db];
      *(f32x4 *)(row + db * 32 + 8 * g + 4 * hi) = (f32x4){a[4 * g] * f, a[4 * g + 1] * f, a[4 * g + 2] * f,
                                                           a[4 * g + 3] * f};
    }
}

// WIN: places of the learned bias's line that a tile of 64 queries and the
// workgroup's 128 keys have, staged beside the tile.
template <class P> constexpr int dkdv_window() { return P::kRel ? 128 + 64 : 0; }
template <int D, int WIN = 0> struct DkdvLds {
  uint16_t q[4][64 * D], o[4][64 * D];
};
template <int D> struct DkdvLds<D, 192> {
  uint16_t q[4][64 * D], o[4][64 * D];
  float c[4 * 192];
};
template <typename T, int D, bool CAUSAL, bool SCOREMOD, bool DSOUT, bool GROUPED, class P = KParams>
__device__ __forceinline__ void bwd_dkdv_body(const P &p, const int id, DkdvLds<D, dkdv_window<P>()> &lds) {
  constexpr int WIN = dkdv_window<P>();
  constexpr bool REL = P::kRel;
  constexpr int PB = p_bits<T, P>();
  static_assert(!(DSOUT && GROUPED), "two-pass backward of grouped heads: D = 128 only");
  constexpr int BN = 128;                 // keys per workgroup (32 per wave)
  constexpr int BMQ = 64;                 // queries per LDS tile (two 32-query blocks)
  constexpr int NST = 4;                  // LDS ring stages
  constexpr int NKS = D / 16, NDB = D / 32;
  constexpr int NM = 2 * NKS + 4 * NDB;   // MFMAs per region
  constexpr int LA = D <= 64 ? 4 : 8;     // operand read-ahead, in MFMAs
  constexpr int NWIN = NM / 4;            // VALU windows (four MFMAs each) per region
  constexpr int PPW = 8 / NWIN;           // element pairs per window
  constexpr int BAR = NM - LA;            // MFMA position of the tile barrier in odd regions
  static_assert(NM % LA == 0 && BAR % 4 == 0, "region shape");
  // The region loop unrolls 8 regions (4 tiles); its compile-time stage
  // indices need 4 tiles to be a whole number of ring turns.
  static_assert(4 % NST == 0, "ring stages");

  auto &sQ = lds.q;
  auto &sO = lds.o;

  const int nparts = GROUPED && p.qsplit > 1 ? p.qsplit : 1, wg = GROUPED ? id / nparts : id;
  const int part = GROUPED ? id - wg * nparts : 0;
  int b, h, kblk;
  int ritem = 0, rchunk = 0;  // range split: the item and this workgroup's chunk of its queries
  if (!CAUSAL && !DSOUT && p.rsplit > 1) {
    int bh;
    ritem = wg / p.rsplit, rchunk = wg % p.rsplit;
    dense_item(ritem, p.B * p.H, p.nblk, true, bh, kblk);
    b = bh / p.H, h = bh % p.H;
  } else if (p.ragged() && p.B <= 64) {
    const auto lq = [&](int i) SIGATTN_INLINE { return p.len_q(i); };
    const auto lk = [&](int i) SIGATTN_INLINE { return p.len_k(i); };
    const WorkItem it = CAUSAL ? WorkOrder::by_level(wg, p.B, p.H, lk, BN, p.nblk, false, p.ncu,
                                                     D <= 64 ? 2 : 1)
                               : WorkOrder::by_stream(wg, p.B, p.H, lk, BN, p.nblk, lq);
    b = it.b, h = it.h, kblk = it.blk;
  } else {
    const int BH = p.B * p.H;
    int bh;
    dense_item(wg, BH, p.nblk, !CAUSAL, bh, kblk);  // causal: low key blocks (the most work) first
    b = bh / p.H, h = bh % p.H;
  }
  const int Lq = p.len_q(b);
  const int Lk = p.len_k(b);
  const bool half = p.half_head(D);  // head_dim 16 in this D = 32 kernel
  // Padding item: its zero dK and dV rows as part of contiguous spans (see zero_row_span).
  if (kblk * BN >= Lk && p.k_rows_contiguous(half ? 16 : D)) {
    const int r1 = min(kblk * BN + BN, p.Tk);
    zero_row_span((uint16_t *)p.dk + (int64_t)b * p.sk_b, p.sk_t, kblk * BN, r1, h, p.H, threadIdx.x, 256);
    zero_row_span((uint16_t *)p.dv + (int64_t)b * p.sk_b, p.sk_t, kblk * BN, r1, h, p.H, threadIdx.x, 256);
    return;
  }

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hi = lane >> 5;
  const int k0 = kblk * BN, kw = k0 + w * 32, my_k = kw + l32;

  const int head0 = GROUPED ? p.part_head(part) : 0, nheads = GROUPED ? p.part_head(part + 1) - head0 : 1;
  const int hq = GROUPED ? p.first_q_head(h) + head0 : h;
  const int64_t qoff = p.q_base(b, hq);
  const int64_t koff = p.k_base(b, h);
  const uint16_t *Qb = (const uint16_t *)p.q + qoff;
  const uint16_t *dOb = (const uint16_t *)p.dout + qoff;
  const uint16_t *Kb = (const uint16_t *)p.k + koff;
  const uint16_t *Vb = (const uint16_t *)p.v + koff;
  uint16_t *dKb = (uint16_t *)p.dk + koff;
  uint16_t *dVb = (uint16_t *)p.dv + koff;

  // Causal: queries before the workgroup's first key see none of its keys.
  // Range split: this workgroup's chunk of the item's query tiles.
  int mstart = CAUSAL ? (k0 / BMQ) * BMQ : 0;
  int mend = (k0 >= Lk) ? mstart : Lq;
  if (!CAUSAL && !DSOUT && p.rsplit > 1 && k0 < Lk) {
    const int ntq = (Lq + BMQ - 1) / BMQ;
    mstart = split_tile(rchunk, p.rsplit, ntq) * BMQ;
    mend = min(Lq, split_tile(rchunk + 1, p.rsplit, ntq) * BMQ);
  }
  const int ntiles1 = mend > mstart ? (mend - mstart + BMQ - 1) / BMQ : 0;  // of one query head
  const int ntiles = GROUPED ? nheads * ntiles1 : ntiles1;
  const int NB = 2 * ntiles;
  HeadStream<GROUPED> hs(2 * ntiles1);

  const float scale = *p.scale;
  const float bias = p.bias[b];
  const float nsl = -scale * kLog2e;
  const bool kok = my_k < Lk;
  float nc = -bias * kLog2e;
  if (SCOREMOD) nc = kok ? -(bias + p.score_mod[p.mod_base(b) + my_k]) * kLog2e : 0.0f;

  u32x4 kf[NKS], vf[NKS];
  {
    const uint16_t *kr = Kb + (int64_t)my_k * p.sk_t + 8 * hi;
    const uint16_t *vr = Vb + (int64_t)my_k * p.sk_t + 8 * hi;
#pragma unroll
    for (int s = 0; s < NKS; ++s) {
      const bool in = kok && !(half && s > 0);
      kf[s] = in ? *(const u32x4 *)(kr + 16 * s) : zero4();
      vf[s] = in ? *(const u32x4 *)(vr + 16 * s) : zero4();
    }
  }
  // Consume the K / V loads before the loop, so the compiler's wait for them
  // is not placed at the loop head, where it would also wait for tile copies.
#pragma unroll
  for (int s = 0; s < NKS; ++s) asm volatile("" ::"v"(kf[s]), "v"(vf[s]));

  f32x16 dka[NDB], dva[NDB];
#pragma unroll
  for (int d = 0; d < NDB; ++d) { dka[d] = zero16(); dva[d] = zero16(); }

  TileOffsets<D> to;
  to.init(lane);
  DmaPlan<BMQ, D, 4> dma;
  dma.init(w, lane, half);
  const int q_stride_bytes = (int)(p.sq_t * 2);
  // Place i of a tile's window: query m - key = i - BN from its first ones.
  float creg = 0.0f;
  [[maybe_unused]] const int win0 = BN - w * 32 - l32 + 4 * hi;  // this lane's place of the tile's query 0
  auto store_c = [&](int t) SIGATTN_INLINE {
    if constexpr (REL) {
      if (tid < WIN) lds.c[t % NST * WIN + tid] = -(bias + creg) * kLog2e;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  };
  auto issue = [&](int st, int t) SIGATTN_INLINE {
    if constexpr (REL) {
      if (tid < WIN) creg = rel_at(p, hq + (int)hs.head_of_tile(t), k0 + BN - mstart - hs.tile(t) * BMQ - tid);
    }
    const int64_t at = (int64_t)mstart * p.sq_t + hs.head_of_tile(t) * p.sq_h;
    dma.issue(sQ[st], Qb + at, q_stride_bytes, hs.tile(t) * BMQ, mend - mstart);
    dma.issue(sO[st], dOb + at, q_stride_bytes, hs.tile(t) * BMQ, mend - mstart);
    hs.next_tile();
  };

  f32x16 sacc[2], pacc[2];       // S and dP accumulators, by block parity
  uint32_t pw[2][8], dw[2][8];   // packed P and dS words, by block parity
  u32x4 opq[LA];                 // A operands of the next LA MFMAs (slot = position % LA)
  float ex[PPW][2];              // exp2 terms of the next element pairs

  // A operand of MFMA m of the region whose blocks (S/dP block, gradient
  // block) sit at tile rows kl in ring stages stc / stg.
  auto read_op = [&](int m, int stc, int stg, int kl) SIGATTN_INLINE {
    if (m < 2 * NKS) {
      return (m % 2 == 0) ? ld_row<D>(sQ[stc], to, kl, m / 2) : ld_row<D>(sO[stc], to, kl, m / 2);
    } else {
      const int i = m - 2 * NKS, j = i / (2 * NDB), dbi = (i / 2) % NDB;
      return (i % 2 == 0) ? ld_tr<D>(sO[stg], to, kl / 16 + j, dbi)
                          : ld_tr<D>(sQ[stg], to, kl / 16 + j, dbi);
    }
  };

  // Zeroes the P and dS entries of block g whose query lies before the
  // block range (pipeline fill; as unsigned such queries may also wrap to
  // huge values), at or past seq_lens_q, or (causal) before the lane's key.
  auto mask_words = [&](int slot, int g) SIGATTN_INLINE {
    int qbase = mstart + 32 * g;
    asm volatile("" : "+s"(qbase));  // keeps this rare fix-up in its own branch
    const unsigned lo = CAUSAL ? (unsigned)max(my_k, mstart) : (unsigned)mstart;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = 2 * e;
      const unsigned q0 = (unsigned)(qbase + 8 * (i / 4) + 4 * hi + (i % 4));
      const bool ok0 = q0 >= lo && q0 < (unsigned)Lq;
      const bool ok1 = q0 + 1u >= lo && q0 + 1u < (unsigned)Lq;
      const uint32_t m = (ok0 ? 0x0000ffffu : 0u) | (ok1 ? 0xffff0000u : 0u);
      pw[slot][e] &= m;
      dw[slot][e] &= m;
    }
  };
  auto needs_mask = [&](int g) SIGATTN_INLINE {
    const int qb0 = mstart + 32 * g;
    return g < 0 || qb0 + 32 > Lq || (CAUSAL && qb0 < kw + 31);
  };

  // Two-pass backward: the masked dS words of block g (slot `slot`) become
  // this wave's tile (query block mstart/32 + g, key block kw/32) of the dS
  // workspace (DsLayout).  Tiles of queries past seq_lens_q, of keys past
  // seq_lens_k, or (causal) wholly above the diagonal are not stored; the dQ
  // pass reads none of them.
  const int kbw = kw / 32;
  uint16_t *ds_bh = nullptr;
  if constexpr (DSOUT)
    ds_bh = p.ds + ((int64_t)b * p.H + h) * DsLayout::per_bh(p.ds_nqb, p.ds_nkb, CAUSAL) *
                       DsLayout::kTileElems;
  // Every region issues exactly two store instructions, so the tile
  // barrier can wait for its copies with a fixed vmcnt while the stores are
  // still in flight: a skipped tile is a store through a buffer resource of
  // zero bytes, which the hardware drops.
  auto store_ds = [&](int slot, int g) SIGATTN_INLINE {
    const int qb = mstart / 32 + g;
    const bool ok = g >= 0 && 32 * qb < Lq && kw < Lk && (!CAUSAL || qb >= kbw);
    // Buffer over this wave's tile (or over nothing).
    const uint16_t *tp = ds_bh + (ok ? DsLayout::tile(qb, kbw, p.ds_nqb, CAUSAL) : 0) * DsLayout::kTileElems;
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc((void *)tp, (short)0, ok ? 2048 : 0, kBufferWord3);
    const int off = 16 * lane;
    __builtin_amdgcn_raw_buffer_store_b128((u32x4){dw[slot][0], dw[slot][1], dw[slot][2], dw[slot][3]}, rs,
                                           off, 0, kStoreNT);
    __builtin_amdgcn_raw_buffer_store_b128((u32x4){dw[slot][4], dw[slot][5], dw[slot][6], dw[slot][7]}, rs,
                                           off + 1024, 0, kStoreNT);
  };

  // One region (U = r mod 8, so every slot and ring stage is static).
  auto region = [&](int r, auto u_tag) SIGATTN_INLINE {
    constexpr int U = decltype(u_tag)::value;
    constexpr int SL = U % 2;                     // parity of blocks r and r-2
    constexpr int KL = 32 * (U % 2);              // tile rows of blocks r and r-2
    constexpr int KLn = 32 * ((U + 1) % 2);       // tile rows of blocks r+1 and r-1
    constexpr int STC = (U / 2) % NST;            // stage of block r
    constexpr int STG = ((U + 6) / 2) % NST;      // stage of block r-2
    constexpr int STCn = ((U + 1) / 2) % NST;     // stage of block r+1
    constexpr int STGn = ((U + 7) / 2) % NST;     // stage of block r-1
    float c[16], cn[2 * PPW];                     // exp2 offsets of block r-1, of block r's first pairs
    if constexpr (REL) {
#pragma unroll
      for (int i = 0; i < 16; ++i) c[i] = lds.c[STGn * WIN + KLn + 8 * (i / 4) + i % 4 + win0];
#pragma unroll
      for (int i = 0; i < 2 * PPW; ++i) cn[i] = lds.c[STC * WIN + KL + 8 * (i / 4) + i % 4 + win0];
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) c[i] = nc;
#pragma unroll
      for (int i = 0; i < 2 * PPW; ++i) cn[i] = nc;
    }
#pragma unroll
    for (int win = 0; win < NWIN; ++win) {
      if ((U % 2) == 1 && win * 4 == BAR) {
        // Publish tile (r+1)/2 before the first read of it (the read-ahead of
        // block r+1), then start the copy of the tile after it into the stage
        // of the tile three back, whose last reads were two regions ago.
        const int t1 = (r + 1) / 2;
        if (t1 < ntiles) {
          if constexpr (DSOUT) {
            // Tile t1's copies are older than the dS stores issued since
            // (two per region; region 1 follows only region 0's), which may
            // stay in flight.
            if (r == 1) wait_vm<2>();
            else wait_vm<4>();
          } else {
            wait_dma();
          }
          store_c(t1);
          asm volatile("" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          if (t1 + 1 < ntiles) issue((t1 + 1) % NST, t1 + 1);
        }
      }
      // dS of block r-2 (its words stay intact until the next region's
      // VALU work), stored where the next vmcnt(0) is furthest away: at the
      // start of even regions, after the tile barrier in odd ones.
      if constexpr (DSOUT) {
        if (((U % 2) == 0 && win == 0) || ((U % 2) == 1 && win * 4 == BAR)) store_ds(SL, r - 2);
      }
      // One wait for the window's four operands instead of one per MFMA.
      asm volatile("" ::"v"(opq[(win * 4) % LA]), "v"(opq[(win * 4 + 1) % LA]),
                   "v"(opq[(win * 4 + 2) % LA]), "v"(opq[(win * 4 + 3) % LA]));
#pragma unroll
      for (int mm = 0; mm < 4; ++mm) {
        const int m = win * 4 + mm;
        const u32x4 a = opq[m % LA];
        if (m < 2 * NKS) {
          if (m % 2 == 0) sacc[SL] = Elem<T>::mfma(a, kf[m / 2], m == 0 ? zero16() : sacc[SL]);
          else pacc[SL] = Elem<T>::mfma(a, vf[m / 2], m == 1 ? zero16() : pacc[SL]);
        } else {
          const int i = m - 2 * NKS, j = i / (2 * NDB), dbi = (i / 2) % NDB;
          if (i % 2 == 0) {
            const u32x4 bp = (u32x4){pw[SL][4 * j], pw[SL][4 * j + 1], pw[SL][4 * j + 2], pw[SL][4 * j + 3]};
            dva[dbi] = Elem<T>::mfma(a, bp, dva[dbi]);
          } else {
            const u32x4 bd = (u32x4){dw[SL][4 * j], dw[SL][4 * j + 1], dw[SL][4 * j + 2], dw[SL][4 * j + 3]};
            dka[dbi] = Elem<T>::mfma(a, bd, dka[dbi]);
          }
        }
        // Refill the slot with the operand of MFMA m + LA (next region when
        // it wraps: S/dP block r+1, gradient block r-1).
        if (m + LA < NM) opq[m % LA] = read_op(m + LA, STC, STG, KL);
        else opq[m % LA] = read_op(m + LA - NM, STCn, STGn, KLn);
      }
      // VALU: P / dS of block r-1 (parity 1-SL).  Stage B (reciprocal, dS,
      // packing) for this window's pairs, stage A (exp2) for the next
      // window's pairs -- or, in the last window, the first pairs of block r.
      float nx[PPW][2];
#pragma unroll
      for (int pp = 0; pp < PPW; ++pp) {
        const bool last = win + 1 == NWIN;
        const int e = last ? pp : (win + 1) * PPW + pp;
        const f32x16 &sv = last ? sacc[SL] : sacc[1 - SL];
        nx[pp][0] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc_read(sv[2 * e]), nsl, last ? cn[2 * pp] : c[2 * e]));
        nx[pp][1] = __builtin_amdgcn_exp2f(
            __builtin_fmaf(acc_read(sv[2 * e + 1]), nsl, last ? cn[2 * pp + 1] : c[2 * e + 1]));
      }
#pragma unroll
      for (int pp = 0; pp < PPW; ++pp) {
        const int e = win * PPW + pp;
        // Written stage by stage for both elements, so each transcendental
        // result is not consumed by the very next instruction.
        float pr[2], t[2], ds[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) pr[x] = __builtin_amdgcn_rcpf(1.0f + ex[pp][x]);
#pragma unroll
        for (int x = 0; x < 2; ++x) t[x] = pr[x] * acc_read(pacc[1 - SL][2 * e + x]);
#pragma unroll
        for (int x = 0; x < 2; ++x) ds[x] = __builtin_fmaf(-pr[x], t[x], t[x]);
        if constexpr (PB > 0) pw[1 - SL][e] = Elem<T>::pack(pr[0] * (1 << PB), pr[1] * (1 << PB));
        else pw[1 - SL][e] = Elem<T>::pack(pr[0], pr[1]);
        dw[1 - SL][e] = Elem<T>::pack(ds[0], ds[1]);
        asm volatile("" : "+v"(pw[1 - SL][e]), "+v"(dw[1 - SL][e]));
      }
#pragma unroll
      for (int pp = 0; pp < PPW; ++pp) { ex[pp][0] = nx[pp][0]; ex[pp][1] = nx[pp][1]; }
#pragma unroll
      for (int mm = 0; mm < 4; ++mm) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x402, 4 * PPW, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    const int done = hs.block(r, 1);
    if (r == 0 || needs_mask(done)) mask_words(1 - SL, done);
    hs.next_block();
  };

  // Pipeline fill: blocks -2 and -1 contribute P = dS = 0; their gradient
  // operands come from ring stage 3, zeroed here (tile 3 arrives only after
  // region 3), so 0 * operand stays 0.
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    sacc[x] = zero16();
    pacc[x] = zero16();
#pragma unroll
    for (int e = 0; e < 8; ++e) { pw[x][e] = 0u; dw[x][e] = 0u; }
  }
#pragma unroll
  for (int pp = 0; pp < PPW; ++pp) { ex[pp][0] = 0.0f; ex[pp][1] = 0.0f; }
  for (int i = tid; i < BMQ * D / 8; i += 256) {
    *(u32x4 *)&sQ[NST - 1][8 * i] = zero4();
    *(u32x4 *)&sO[NST - 1][8 * i] = zero4();
  }
  if (ntiles > 0) {
    issue(0, 0);
    wait_dma();
    store_c(0);
  }
  __syncthreads();
  if (ntiles > 1) issue(1, 1);
#pragma unroll
  for (int m = 0; m < LA; ++m) opq[m] = read_op(m, 0, NST - 1, 0);

  for (int r0 = 0; r0 < NB + 2; r0 += 8) {
    region(r0 + 0, std::integral_constant<int, 0>{});
    if (r0 + 1 < NB + 2) region(r0 + 1, std::integral_constant<int, 1>{});
    if (r0 + 2 < NB + 2) region(r0 + 2, std::integral_constant<int, 2>{});
    if (r0 + 3 < NB + 2) region(r0 + 3, std::integral_constant<int, 3>{});
    if (r0 + 4 < NB + 2) region(r0 + 4, std::integral_constant<int, 4>{});
    if (r0 + 5 < NB + 2) region(r0 + 5, std::integral_constant<int, 5>{});
    if (r0 + 6 < NB + 2) region(r0 + 6, std::integral_constant<int, 6>{});
    if (r0 + 7 < NB + 2) region(r0 + 7, std::integral_constant<int, 7>{});
  }

  if (!CAUSAL && !DSOUT && p.rsplit > 1 &&
      !split_combine<2 * NDB, 4>(
          [&](int i) SIGATTN_INLINE -> f32x16 & { return i < NDB ? dka[i] : dva[i - NDB]; },
          p.rs_part + (int64_t)ritem * p.rsplit * (2 * BN * D), p.rs_cnt + ritem, rchunk, p.rsplit, w, lane))
    return;

  if constexpr (PB > 0) {
#pragma unroll
    for (int db = 0; db < NDB; ++db) dva[db] *= 1.0f / (1 << PB);
  }
  if (GROUPED && nparts > 1) {
    if (kok) {
      store_part<NDB>(p, part, b, my_k, h, dka, 0, scale, hi, half);
      store_part<NDB>(p, part, b, my_k, h, dva, 1, 1.0f, hi, half);
    }
    return;
  }
  if (my_k < p.k_rows_out(Lk)) {
    uint16_t *kr = dKb + (int64_t)my_k * p.sk_t;
    uint16_t *vr = dVb + (int64_t)my_k * p.sk_t;
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (half && g >= 2) break;  // columns 16..31: not in the tensor
        const int d0 = db * 32 + 8 * g + 4 * hi;
        u32x2 ok_, ov;
        ok_.x = Elem<T>::pack(dka[db][4 * g] * scale, dka[db][4 * g + 1] * scale);
        ok_.y = Elem<T>::pack(dka[db][4 * g + 2] * scale, dka[db][4 * g + 3] * scale);
        ov.x = Elem<T>::pack(dva[db][4 * g], dva[db][4 * g + 1]);
        ov.y = Elem<T>::pack(dva[db][4 * g + 2], dva[db][4 * g + 3]);
        if (!kok) { ok_ = (u32x2){0u, 0u}; ov = (u32x2){0u, 0u}; }
        *(u32x2 *)(kr + d0) = ok_;
        *(u32x2 *)(vr + d0) = ov;
      }
    }
  }
}

}  // namespace sigattn
