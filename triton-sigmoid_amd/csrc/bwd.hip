// Recompute backward on gfx950 MFMA: dQ kernel (query-stationary) and dK/dV
// kernel (key-stationary).  No atomics: every output element is owned by one
// lane, so results are bitwise deterministic.
//
// Semantics follow the reference's _bwd_dense_dq_kernel / _bwd_dense_dkdv_kernel
// (src/triton_sigmoid/sigmoid_triton_dense.py:162-307, :315-467) and the padded
// variants (src/triton_sigmoid/sigmoid_triton_padded.py:179-339, :342-509):
//   P = sigmoid(S*scale + bias (+ score_mod[key])) recomputed in fp32;
//   dP = dO·Vᵀ; dS = P(1-P)dP computed as fma(P, -P*dP, P*dP); masked dS = 0;
//   dQ = (dS rounded to the I/O dtype)·K · scale;
//   dV = (P rounded)ᵀ·dO;  dK = (dS rounded)ᵀ·Q · scale.
// Padded query rows get dQ = 0 and padded key rows dK = dV = 0.
//
// Both kernels stream their tiles (K, V for dQ; Q, dO for dK/dV) into
// double-buffered swizzled LDS with direct global->LDS DMA one tile ahead,
// and keep the stationary rows as MFMA operands in registers.  The dK/dV
// kernel (one wave per SIMD, accumulators in AGPRs) runs each tile as
// scheduling regions that overlap the P / dS VALU work of one 32-query block
// with the MFMA chains of the next; the dQ kernel (two waves per SIMD) relies
// on the second wave for that overlap.  Rows past seq_lens are fetched as
// copies of the last valid row (in bounds) and masked on boundary tiles.
// Their bodies are in bwd_kernel.h, shared with the learned bias by relative
// position (rel_bwd.hip).
#include <type_traits>

#include "bwd_kernel.h"
#include "common.h"
#include "launch.h"

namespace sigattn {

template <typename T, int D, int WK, bool CAUSAL, bool SCOREMOD>
__global__ __launch_bounds__(256, 2) void bwd_dq_kernel(const KParams p) {
  __shared__ __attribute__((aligned(16))) DqLds<D, SCOREMOD> lds;
  __shared__ unsigned long long gap_lds[2];
  const int wg = gap_prologue<2>(p, gap_lds);  // packed layouts: leading gap-zeroing workgroups
  if (wg >= 0) bwd_dq_body<T, D, WK, CAUSAL, SCOREMOD>(p, wg, lds);
}

// dK and dV of head-split items: the sum of the parts' fp32 rows in their
// order, rounded once.  Rows that no sequence covers are left to the dQ launch,
// which zeroes them.  Eight elements a thread, per_row threads a row, as many
// rows to a workgroup as it has threads for; bound by memory: 45 MB in 9.1 us,
// 5.0 TB/s (four parts of 9945 rows H_kv=2 D=64).
template <typename T> __global__ __launch_bounds__(256) void add_parts_kernel(const KParams p, int per_row) {
  const int rows = per_row < 256 ? 256 / per_row : 1, mine = (int)threadIdx.x / per_row;
  const int64_t row = (int64_t)blockIdx.x * rows + mine;
  if (mine >= rows || row >= p.rows_k) return;
  int lo = 0, hi = p.B - 1;  // the last sequence that begins at or before the row
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (packed_first(p.cu_k, p.rows_k, mid) <= row) lo = mid;
    else hi = mid - 1;
  }
  const int64_t first = packed_first(p.cu_k, p.rows_k, lo);
  if (row < first || row - first >= p.len_k(lo)) return;
  const int64_t tensor = p.rows_k * p.H * p.dmem;
  for (int i = (int)threadIdx.x - mine * per_row; i < per_row; i += 256) {
    const int c = 8 * i, h = c / p.dmem, d = c - h * p.dmem;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x4 v[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
      const float *src = p.kv_part + t * tensor + row * p.H * p.dmem + c;
#pragma unroll 4
      for (int s = 0; s < p.qsplit; ++s) {
        v[0] += *(const f32x4 *)(src + 2 * s * tensor);
        v[1] += *(const f32x4 *)(src + 2 * s * tensor + 4);
      }
      T *to = (T *)(t == 0 ? p.dk : p.dv) + row * p.sk_t + h * p.sk_h + d;
      if constexpr (sizeof(T) == 4) {
        *(f32x4 *)to = v[0], *(f32x4 *)(to + 4) = v[1];
      } else {
        *(u32x4 *)to = (u32x4){Elem<T>::pack(v[0].x, v[0].y), Elem<T>::pack(v[0].z, v[0].w),
                               Elem<T>::pack(v[1].x, v[1].y), Elem<T>::pack(v[1].z, v[1].w)};
      }
    }
  }
}

template <typename T, int D, bool CAUSAL, bool SCOREMOD, bool DSOUT, bool GROUPED>
__global__ __launch_bounds__(256, (D <= 64 ? 2 : 1)) void bwd_dkdv_kernel(const KParams p) {
  __shared__ __attribute__((aligned(16))) DkdvLds<D> lds;
  bwd_dkdv_body<T, D, CAUSAL, SCOREMOD, DSOUT, GROUPED>(p, blockIdx.x, lds);
}

// The recompute backward's two kernels in one launch: the first nkv workgroups
// run dK/dV items, the rest dQ items, WK waves to 32 rows as launch_bwd_dq_mfma
// runs these grids.  On grids within one workgroup per CU the two halves share
// the GPU instead of each leaving half of it idle; on causal ones of several,
// the short dQ items run beside the dK/dV kernel's last ones.  The bodies are
// the kernels' own, so results are bit-identical to the two launches.  They
// share their LDS, and two workgroups fit a CU.
template <typename T, int D, int WK, bool CAUSAL, bool SCOREMOD>
__global__ __launch_bounds__(256, WK) void bwd_fused_kernel(const KParams pq, const KParams pk, int nkv) {
  __shared__ __attribute__((aligned(16))) union {
    DqLds<D, SCOREMOD> dq;
    DkdvLds<D> dkdv;
  } lds;
  if ((int)blockIdx.x < nkv) bwd_dkdv_body<T, D, CAUSAL, SCOREMOD, false, false>(pk, blockIdx.x, lds.dkdv);
  else bwd_dq_body<T, D, WK, CAUSAL, SCOREMOD>(pq, (int)blockIdx.x - nkv, lds.dq);
}

// ---------------------------------------------------------------------------
// dK/dV at D = 128 by wave pairs: workgroup = 8 waves, 128 keys.  Waves w and
// w + 4 own the same 32 keys and share SIMD w (waves are dealt to the four
// SIMDs round-robin), so each SIMD runs one wave of each role:
//   role A (waves 0-3): S = Q·Kᵀ (K rows in registers), P = sigmoid(S),
//     dVᵀ += dOᵀ·P, and every Q / dO tile copy;
//   role B (waves 4-7): dP = dO·Vᵀ (V rows in registers), dS = P·(1-P)·dP,
//     dKᵀ += Qᵀ·dS, and the dS tiles of the two-pass backward.
// The copies and the stores sit in different waves because a wave's memory
// operations complete in issue order: a copy wait behind dS stores would
// also wait for their acknowledgement (measured 3-7 % of the kernel).
// A hands P to B through LDS in fp32, so dS is computed from exactly the
// values bwd_dkdv_kernel uses and dK, dV are bit for bit the same.  Either
// role needs about half that kernel's registers (every accumulator stays in
// VGPRs), and with two waves per SIMD one wave's sigmoid work issues while
// the other wave's MFMAs run.
// The queries stream as in bwd_dkdv_kernel: 64-query tiles of Q and dO in a
// 4-stage ring, processed as 32-query blocks g.  Region r runs
//   A: S of block r, P of block r-1 (packed for the dV product and stored to
//      LDS for B), dV of block r-2;
//   B: dS of block r-2 (P from LDS, dP from its accumulator), dP of block r,
//      dK of block r-2.
// Every region has one barrier, placed before the operand read-ahead reaches
// the next region's first MFMAs: it publishes the tile of the next region
// (A waits for its copies just before) and the P that A stored before it,
// which B reads in the next region (the two P buffers alternate by block
// parity).
// ---------------------------------------------------------------------------
// Dense causal grids in dense_item's XCD-grouped order too: paired key
// blocks make every workgroup's work equal, so grouping costs no balance, and
// each XCD then reads the Q and dO rows of two (batch, head) pairs at a time
// instead of eight.  Measured at B=4 L=4096 H=16 D=128 causal: HBM fetch
// 757 -> 278 MB per launch (the algorithmic 268 MB), 0.661 -> 0.647 ms.
#ifndef SIGATTN_DKDV_GROUPED
#define SIGATTN_DKDV_GROUPED 1
#endif
constexpr bool kDkdvGrouped = SIGATTN_DKDV_GROUPED != 0;

template <typename T, bool CAUSAL, bool SCOREMOD, bool DSOUT, bool GROUPED>
__global__ __launch_bounds__(512, 1) void bwd_dkdv_pair_kernel(const KParams p) {
  constexpr int D = 128;
  constexpr int BN = 128;                 // keys per workgroup (32 per wave pair)
  constexpr int BMQ = 64;                 // queries per LDS tile (two 32-query blocks)
  constexpr int NST = 4;                  // LDS ring stages
  constexpr int NKS = D / 16, NDB = D / 32;
  constexpr int NM = NKS + 2 * NDB;       // MFMAs per region and wave
  constexpr int LA = 4;                   // operand read-ahead, in MFMAs
  constexpr int BAR = NM - LA;            // MFMA position of the region's barrier
  using Dma = DmaPlan<BMQ, D, 4>;
  constexpr int NCP = 2 * Dma::NI;        // copy instructions per tile and A wave
  static_assert(NM % LA == 0 && BAR >= 8, "region shape");
  // The region loop unrolls 8 regions (4 tiles); its compile-time stage
  // indices need 4 tiles to be a whole number of ring turns.
  static_assert(4 % NST == 0, "ring stages");

  __shared__ __attribute__((aligned(16))) uint16_t sQ[NST][BMQ * D];
  __shared__ __attribute__((aligned(16))) uint16_t sO[NST][BMQ * D];
  // P of block g, for pair w: sP[g & 1][w], lane l's elements 4c..4c+3 at 256 c + 4 l.
  __shared__ __attribute__((aligned(16))) float sP[2][4][1024];

  // Work: ragged batches take one key block per workgroup in WorkOrder's
  // order.  Dense problems take key blocks j and nblk-1-j in sequence
  // (grid = ceil(nblk/2) per (batch, head)): under the causal mask the two
  // together cost the same for every j, so all workgroups are equal, and
  // the grid has half as many workgroup starts.  A dense non-causal grid
  // that would not fill the GPU paired runs one key block per workgroup
  // (grid = nblk per (batch, head)).
  const int nparts = GROUPED && p.qsplit > 1 ? p.qsplit : 1, wg = (int)blockIdx.x / nparts;
  const int part = (int)blockIdx.x - wg * nparts;
  int b, h, kblk0, nitems;
  if (p.ragged() && p.B <= 64) {
    const auto lq = [&](int i) SIGATTN_INLINE { return p.len_q(i); };
    const auto lk = [&](int i) SIGATTN_INLINE { return p.len_k(i); };
    const WorkItem it = CAUSAL ? WorkOrder::by_level(wg, p.B, p.H, lk, BN, p.nblk, false, p.ncu, 1)
                               : WorkOrder::by_stream(wg, p.B, p.H, lk, BN, p.nblk, lq);
    b = it.b, h = it.h, kblk0 = it.blk, nitems = 1;
  } else {
    const int BH = p.B * p.H;
    int bh;
    const int nper = (int)(gridDim.x / nparts / BH);
    dense_item(wg, BH, nper, !CAUSAL || kDkdvGrouped, bh, kblk0);
    const bool paired = nper < p.nblk;
    nitems = paired && p.nblk - 1 - kblk0 > kblk0 ? 2 : 1;
    b = bh / p.H, h = bh % p.H;
  }
  for (int item = 0; item < nitems; ++item) {
    const int kblk = item == 0 ? kblk0 : p.nblk - 1 - kblk0;
    // The previous key block's last reads of the ring and of the P buffers
    // precede this block's fills.
    if (item > 0) __syncthreads();
    const int Lq = p.len_q(b);
    const int Lk = p.len_k(b);
    // Padding item (ragged batches, one key block per workgroup): its zero
    // dK and dV rows as part of contiguous spans (see zero_row_span).
    if (nitems == 1 && kblk * BN >= Lk && p.k_rows_contiguous(D)) {
      const int r1 = min(kblk * BN + BN, p.Tk);
      zero_row_span((uint16_t *)p.dk + (int64_t)b * p.sk_b, p.sk_t, kblk * BN, r1, h, p.H, threadIdx.x, 512);
      zero_row_span((uint16_t *)p.dv + (int64_t)b * p.sk_b, p.sk_t, kblk * BN, r1, h, p.H, threadIdx.x, 512);
      return;
    }

    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int pair = wv & 3;
    const bool role_a = wv < 4;
    const int l32 = lane & 31, hi = lane >> 5;
    const int k0 = kblk * BN, kw = k0 + pair * 32, my_k = kw + l32;

    const int head0 = GROUPED ? p.part_head(part) : 0, nheads = GROUPED ? p.part_head(part + 1) - head0 : 1;
    const int hq = GROUPED ? p.first_q_head(h) + head0 : h;
    const int64_t qoff = p.q_base(b, hq);
    const int64_t koff = p.k_base(b, h);
    const uint16_t *Qb = (const uint16_t *)p.q + qoff;
    const uint16_t *dOb = (const uint16_t *)p.dout + qoff;

    // Causal: queries before the workgroup's first key see none of its keys.
    const int mstart = CAUSAL ? (k0 / BMQ) * BMQ : 0;
    const int mend = (k0 >= Lk) ? mstart : Lq;
    const int ntiles1 = mend > mstart ? (mend - mstart + BMQ - 1) / BMQ : 0;  // of one query head
    const int ntiles = GROUPED ? nheads * ntiles1 : ntiles1;
    const int NB = 2 * ntiles;
    HeadStream<GROUPED> hs(2 * ntiles1);

    const float scale = *p.scale;
    const bool kok = my_k < Lk;

    TileOffsets<D> to;
    to.init(lane);
    Dma dma;
    dma.init(pair, lane);
    const int q_stride_bytes = (int)(p.sq_t * 2);
    auto issue = [&](int st, int t) SIGATTN_INLINE {
      const int64_t at = (int64_t)mstart * p.sq_t + hs.head_of_tile(t) * p.sq_h;
      dma.issue(sQ[st], Qb + at, q_stride_bytes, hs.tile(t) * BMQ, mend - mstart);
      dma.issue(sO[st], dOb + at, q_stride_bytes, hs.tile(t) * BMQ, mend - mstart);
      hs.next_tile();
    };

    // Zeroes the packed words of block g whose query lies before the block
    // range (pipeline fill; as unsigned such queries may also wrap to huge
    // values), at or past seq_lens_q, or (causal) before the lane's key.
    auto mask_words = [&](uint32_t(&wds)[8], int g) SIGATTN_INLINE {
      int qbase = mstart + 32 * g;
      asm volatile("" : "+s"(qbase));  // keeps this rare fix-up in its own branch
      const unsigned lo = CAUSAL ? (unsigned)max(my_k, mstart) : (unsigned)mstart;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = 2 * e;
        const unsigned q0 = (unsigned)(qbase + 8 * (i / 4) + 4 * hi + (i % 4));
        const bool ok0 = q0 >= lo && q0 < (unsigned)Lq;
        const bool ok1 = q0 + 1u >= lo && q0 + 1u < (unsigned)Lq;
        wds[e] &= (ok0 ? 0x0000ffffu : 0u) | (ok1 ? 0xffff0000u : 0u);
      }
    };
    auto needs_mask = [&](int g) SIGATTN_INLINE {
      const int qb0 = mstart + 32 * g;
      return g < 0 || qb0 + 32 > Lq || (CAUSAL && qb0 < kw + 31);
    };

    // Pipeline fill: the gradient products of blocks -2 and -1 read ring stage
    // NST-1 (zeroed here; tile NST-1 arrives only in region 2) against zero
    // words, and B's first dS reads the zeroed P buffer 0.
    for (int i = tid; i < BMQ * D / 8; i += 512) {
      *(u32x4 *)&sQ[NST - 1][8 * i] = zero4();
      *(u32x4 *)&sO[NST - 1][8 * i] = zero4();
    }
    for (int i = tid; i < 2 * 4 * 1024 / 4; i += 512) *(u32x4 *)(&sP[0][0][0] + 4 * i) = zero4();
    if (role_a && ntiles > 0) {
      issue(0, 0);
      if (ntiles > 1) {
        issue(1, 1);
        wait_vm<NCP>();
      } else {
        wait_dma();
      }
    }
    __syncthreads();

    const int kmax = p.k_rows_out(Lk);
    if (role_a) {
      // ---------------- role A: S, P, dV ----------------
      const float bias = p.bias[b];
      const float nsl = -scale * kLog2e;
      float nc = -bias * kLog2e;
      if (SCOREMOD) nc = kok ? -(bias + p.score_mod[p.mod_base(b) + my_k]) * kLog2e : 0.0f;
      u32x4 kf[NKS];
      {
        const uint16_t *kr = (const uint16_t *)p.k + koff + (int64_t)my_k * p.sk_t + 8 * hi;
#pragma unroll
        for (int s = 0; s < NKS; ++s) kf[s] = kok ? *(const u32x4 *)(kr + 16 * s) : zero4();
      }
#pragma unroll
      for (int s = 0; s < NKS; ++s) asm volatile("" ::"v"(kf[s]));

      f32x16 dva[NDB], sacc[2];
      uint32_t pw[2][8];
#pragma unroll
      for (int d = 0; d < NDB; ++d) dva[d] = zero16();
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        sacc[x] = zero16();
#pragma unroll
        for (int e = 0; e < 8; ++e) pw[x][e] = 0u;
      }
      float *xb0 = &sP[0][pair][4 * lane];
      float *xb1 = &sP[1][pair][4 * lane];

      // A operand of MFMA m of the region whose blocks (S block, dV block) sit
      // at tile rows kl in ring stages stc / stg.
      auto read_op = [&](int m, int stc, int stg, int kl) SIGATTN_INLINE {
        if (m % 2 == 0) return ld_row<D>(sQ[stc], to, kl, m / 2);
        const int i = m / 2;
        return ld_tr<D>(sO[stg], to, kl / 16 + i / NDB, i % NDB);
      };
      u32x4 opq[LA];
#pragma unroll
      for (int m = 0; m < LA; ++m) opq[m] = read_op(m, 0, NST - 1, 0);

      auto region = [&](int r, auto u_tag) SIGATTN_INLINE {
        constexpr int U = decltype(u_tag)::value;
        constexpr int SL = U % 2;                  // parity of blocks r and r-2
        constexpr int KL = 32 * (U % 2), KLn = 32 * ((U + 1) % 2);
        constexpr int STC = (U / 2) % NST, STG = ((U + 6) / 2) % NST;
        constexpr int STCn = ((U + 1) / 2) % NST, STGn = ((U + 7) / 2) % NST;
        float *xb = SL ? xb0 : xb1;                // P buffer of block r-1
        float keep[2];
#pragma unroll
        for (int m = 0; m < NM; ++m) {
          if (m == BAR) {
            if constexpr (U % 2 == 1) {
              // The next region starts tile t: wait for this wave's copies
              // of it (tile t+1's may stay in flight).
              const int t = (r + 1) / 2;
              if (t < ntiles) {
                if (t + 1 < ntiles) wait_vm<NCP>();
                else wait_dma();
              }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if constexpr (U % 2 == 0) {
              // Every wave has finished region r-1, the last to read the
              // stage of tile r/2 - 2: refill it with tile r/2 + 2.
              const int t = r / 2 + 2;
              if (t < ntiles) issue((U / 2 + 2) % NST, t);
            }
          }
          asm volatile("" ::"v"(opq[m % LA]));
          const u32x4 a = opq[m % LA];
          if (m % 2 == 0) {
            sacc[SL] = Elem<T>::mfma(a, kf[m / 2], m == 0 ? zero16() : sacc[SL]);
          } else {
            const int i = m / 2, j = i / NDB, dbi = i % NDB;
            const u32x4 bp = (u32x4){pw[SL][4 * j], pw[SL][4 * j + 1], pw[SL][4 * j + 2], pw[SL][4 * j + 3]};
            dva[dbi] = Elem<T>::mfma(a, bp, dva[dbi]);
          }
          if (m + LA < NM) opq[m % LA] = read_op(m + LA, STC, STG, KL);
          else opq[m % LA] = read_op(m + LA - NM, STCn, STGn, KLn);
          // P of block r-1: element pair m at MFMA position m, stored to LDS
          // four elements at a time.
          if (m < 8) {
            float pr[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float ex = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[1 - SL][2 * m + x], nsl, nc));
              pr[x] = __builtin_amdgcn_rcpf(1.0f + ex);
            }
            pw[1 - SL][m] = Elem<T>::pack(pr[0], pr[1]);
            if (m % 2 == 0) {
              keep[0] = pr[0];
              keep[1] = pr[1];
            } else {
              *(float4 *)(xb + 256 * (m / 2)) = make_float4(keep[0], keep[1], pr[0], pr[1]);
            }
          }
        }
        const int done = hs.block(r, 1);
        if (r == 0 || needs_mask(done)) mask_words(pw[1 - SL], done);
        hs.next_block();
      };

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

      if (GROUPED && nparts > 1) {
        if (kok) store_part<NDB>(p, part, b, my_k, h, dva, 1, 1.0f, hi, false);
      } else if (my_k < kmax) {
        uint16_t *vr = (uint16_t *)p.dv + koff + (int64_t)my_k * p.sk_t;
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int d0 = db * 32 + 8 * g + 4 * hi;
            u32x2 ov;
            ov.x = Elem<T>::pack(dva[db][4 * g], dva[db][4 * g + 1]);
            ov.y = Elem<T>::pack(dva[db][4 * g + 2], dva[db][4 * g + 3]);
            if (!kok) ov = (u32x2){0u, 0u};
            *(u32x2 *)(vr + d0) = ov;
          }
        }
      }
    } else {
      // ---------------- role B: dP, dS, dK, tile copies ----------------
      u32x4 vf[NKS];
      {
        const uint16_t *vr = (const uint16_t *)p.v + koff + (int64_t)my_k * p.sk_t + 8 * hi;
#pragma unroll
        for (int s = 0; s < NKS; ++s) vf[s] = kok ? *(const u32x4 *)(vr + 16 * s) : zero4();
      }
#pragma unroll
      for (int s = 0; s < NKS; ++s) asm volatile("" ::"v"(vf[s]));

      f32x16 dka[NDB], pacc[2];
      uint32_t dw[8];
#pragma unroll
      for (int d = 0; d < NDB; ++d) dka[d] = zero16();
      pacc[0] = zero16();
      pacc[1] = zero16();
      const float *xb0 = &sP[0][pair][4 * lane];
      const float *xb1 = &sP[1][pair][4 * lane];

      // Two-pass backward: this wave's dS tile of block g (DsLayout), skipped
      // (a store through an empty buffer resource, which the hardware drops)
      // past seq_lens_q / seq_lens_k or wholly above the causal diagonal.
      const int kbw = kw / 32;
      uint16_t *ds_bh = nullptr;
      if constexpr (DSOUT)
        ds_bh = p.ds + ((int64_t)b * p.H * p.q_heads() + hq) * DsLayout::per_bh(p.ds_nqb, p.ds_nkb, CAUSAL) *
                           DsLayout::kTileElems;
      auto store_ds = [&](int g, int head) SIGATTN_INLINE {
        const int qb = mstart / 32 + g;
        const bool ok = g >= 0 && 32 * qb < Lq && kw < Lk && (!CAUSAL || qb >= kbw);
        const int64_t skip = GROUPED ? head * DsLayout::per_bh(p.ds_nqb, p.ds_nkb, CAUSAL) : 0;
        const uint16_t *tp =
            ds_bh + (ok ? skip + DsLayout::tile(qb, kbw, p.ds_nqb, CAUSAL) : 0) * DsLayout::kTileElems;
        const __amdgpu_buffer_rsrc_t rs =
            __builtin_amdgcn_make_buffer_rsrc((void *)tp, (short)0, ok ? 2048 : 0, kBufferWord3);
        const int off = 16 * lane;
        __builtin_amdgcn_raw_buffer_store_b128((u32x4){dw[0], dw[1], dw[2], dw[3]}, rs, off, 0, kStoreNT);
        __builtin_amdgcn_raw_buffer_store_b128((u32x4){dw[4], dw[5], dw[6], dw[7]}, rs, off + 1024, 0, kStoreNT);
      };

      auto read_op = [&](int m, int stc, int stg, int kl) SIGATTN_INLINE {
        if (m % 2 == 0) return ld_row<D>(sO[stc], to, kl, m / 2);
        const int i = m / 2;
        return ld_tr<D>(sQ[stg], to, kl / 16 + i / NDB, i % NDB);
      };
      u32x4 opq[LA];
#pragma unroll
      for (int m = 0; m < LA; ++m) opq[m] = read_op(m, 0, NST - 1, 0);

      auto region = [&](int r, auto u_tag) SIGATTN_INLINE {
        constexpr int U = decltype(u_tag)::value;
        constexpr int SL = U % 2;
        constexpr int KL = 32 * (U % 2), KLn = 32 * ((U + 1) % 2);
        constexpr int STC = (U / 2) % NST, STG = ((U + 6) / 2) % NST;
        constexpr int STCn = ((U + 1) / 2) % NST, STGn = ((U + 7) / 2) % NST;
        // dS of block r-2: P from A (stored in region r-1), dP from the
        // accumulator block r-2 left in pacc[SL].
        {
          const float *xb = SL ? xb1 : xb0;
          float4 pv[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) pv[c] = *(const float4 *)(xb + 256 * c);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float pr0 = (e % 2 == 0) ? pv[e / 2].x : pv[e / 2].z;
            const float pr1 = (e % 2 == 0) ? pv[e / 2].y : pv[e / 2].w;
            const float t0 = pr0 * pacc[SL][2 * e], t1 = pr1 * pacc[SL][2 * e + 1];
            dw[e] = Elem<T>::pack(__builtin_fmaf(-pr0, t0, t0), __builtin_fmaf(-pr1, t1, t1));
          }
          const int done = hs.block(r, 2);
          if (r < 2 || needs_mask(done)) mask_words(dw, done);
          if constexpr (DSOUT) store_ds(done, hs.head(2));
          hs.next_block();
        }
#pragma unroll
        for (int m = 0; m < NM; ++m) {
          if (m == BAR) {
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
          }
          asm volatile("" ::"v"(opq[m % LA]));
          const u32x4 a = opq[m % LA];
          if (m % 2 == 0) {
            pacc[SL] = Elem<T>::mfma(a, vf[m / 2], m == 0 ? zero16() : pacc[SL]);
          } else {
            const int i = m / 2, j = i / NDB, dbi = i % NDB;
            const u32x4 bd = (u32x4){dw[4 * j], dw[4 * j + 1], dw[4 * j + 2], dw[4 * j + 3]};
            dka[dbi] = Elem<T>::mfma(a, bd, dka[dbi]);
          }
          if (m + LA < NM) opq[m % LA] = read_op(m + LA, STC, STG, KL);
          else opq[m % LA] = read_op(m + LA - NM, STCn, STGn, KLn);
        }
      };

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

      if (GROUPED && nparts > 1) {
        if (kok) store_part<NDB>(p, part, b, my_k, h, dka, 0, scale, hi, false);
      } else if (my_k < kmax) {
        uint16_t *kr = (uint16_t *)p.dk + koff + (int64_t)my_k * p.sk_t;
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int d0 = db * 32 + 8 * g + 4 * hi;
            u32x2 ok_;
            ok_.x = Elem<T>::pack(dka[db][4 * g] * scale, dka[db][4 * g + 1] * scale);
            ok_.y = Elem<T>::pack(dka[db][4 * g + 2] * scale, dka[db][4 * g + 3] * scale);
            if (!kok) ok_ = (u32x2){0u, 0u};
            *(u32x2 *)(kr + d0) = ok_;
          }
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// dQ of the two-pass backward: dQ = dS · K · scale from the dS tiles the dK/dV
// kernel stored (DsLayout), with no recomputation of S, P or dP.
// Workgroup = NW waves x 64 queries (two 32-query column blocks per wave);
// keys stream in stages of KB 32-key blocks through an NST-stage LDS ring:
// the K rows (shared by the waves) and each wave's own dS tiles (its two
// query blocks x KB key blocks), all by direct global->LDS copies issued
// NST-1 stages ahead, so about (NST-1) x (32 KB x KB dS + K) per CU is in
// flight against HBM latency.
//   dQᵀ[d, q] += Kᵀ[d, key] · dSᵀ[key, q]
// A = Kᵀ via ds_read_b64_tr_b16 from the row-major K rows; B = dSᵀ via
// ds_read_b64_tr_b16 from the dS tile, which the copy lays out key-major
// (64 bytes per key: its four 16-byte pieces (g-pair c, query half h) at
// slot 2c + h), so lane (query n, k-slot h) receives keys 16ks + 4h + {0..3}
// and 16ks + 8 + 4h + {0..3} -- the same key order as the Kᵀ read.
// Per 32 keys a wave reads 4 KB of dS and runs 16 MFMAs: the kernel is bound
// by HBM bandwidth.
// ---------------------------------------------------------------------------
#ifndef SIGATTN_DQDS_NT
#define SIGATTN_DQDS_NT 1
#endif
constexpr bool kDqDsNT = SIGATTN_DQDS_NT != 0;

// Waves per SIMD of the kernel's resident workgroups (its register budget).
template <int D, int NW, int KB, int NST> constexpr int dq_ds_waves_per_simd() {
  const int occ = 163840 / (NST * (32 * KB * D + NW * 2 * KB * DsLayout::kTileElems) * 2);
  return occ * NW / 4 > 1 ? occ * NW / 4 : 1;
}

template <typename T, int D, bool CAUSAL, int NW, int KB, int NST>
__global__ __launch_bounds__(64 * NW, (dq_ds_waves_per_simd<D, NW, KB, NST>())) void bwd_dq_ds_kernel(
    const KParams p) {
  constexpr int BM = 64 * NW, BN = 32 * KB;
  constexpr int NDB = D / 32;
  constexpr int TE = DsLayout::kTileElems;
  constexpr int KI = BN * D / 8 / 64 / NW;  // K-row copy instructions per wave and stage
  constexpr int NI = KI + 4 * KB;           // copy instructions per wave and stage
  constexpr int PF = NST - 1;               // stages in flight ahead of the one computed
  // Resident workgroups per CU, by the LDS ring's size (160 KB per CU).
  constexpr int OCC = 163840 / (NST * (BN * D + NW * 2 * KB * TE) * 2);
  static_assert(KI >= 1 && (NST - 2) * NI < 64 && OCC >= 1, "stage shape");

  __shared__ __attribute__((aligned(16))) uint16_t sK[NST][BN * D];
  __shared__ __attribute__((aligned(16))) uint16_t sS[NST][NW * 2 * KB * TE];

  const int wg = gap_prologue<2>(p, sK);  // packed layouts: leading gap-zeroing workgroups
  if (wg < 0) return;
  int b, h, qblk;
  if (p.ragged() && p.B <= 64) {
    const auto lq = [&](int i) SIGATTN_INLINE { return p.len_q(i); };
    const auto lk = [&](int i) SIGATTN_INLINE { return p.len_k(i); };
    const WorkItem it = CAUSAL ? WorkOrder::by_level(wg, p.B, p.H, lq, BM, p.nblk, true, p.ncu, OCC)
                               : WorkOrder::by_stream(wg, p.B, p.H, lq, BM, p.nblk, lk);
    b = it.b, h = it.h, qblk = it.blk;
  } else {
    const int BH = p.B * p.H;
    int bh;
    dense_item(wg, BH, p.nblk, !CAUSAL, bh, qblk);
    if (CAUSAL) qblk = p.nblk - 1 - qblk;  // heaviest query blocks first
    b = bh / p.H, h = bh % p.H;
  }
  const int Lq = p.len_q(b);
  const int Lk = p.len_k(b);
  // Padding item: its zero rows as part of one contiguous span (see zero_row_span).
  if (qblk * BM >= Lq && p.q_rows_contiguous(D)) {
    zero_row_span((uint16_t *)p.dq + (int64_t)b * p.sq_b, p.sq_t, qblk * BM, min(qblk * BM + BM, p.Tq), h,
                  p.H, threadIdx.x, 64 * NW);
    return;
  }

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hi = lane >> 5;
  const int q0 = qblk * BM;
  const int qbw = q0 / 32 + 2 * w;  // the wave's two query blocks: qbw, qbw + 1
  const int nqb_valid = (Lq + 31) / 32, nkb_valid = (Lk + 31) / 32;

  const int64_t qoff = p.q_base(b, h);
  const int64_t koff = p.k_base(b, h);
  const uint16_t *Kb = (const uint16_t *)p.k + koff;
  uint16_t *dQb = (uint16_t *)p.dq + qoff;
  const uint16_t *ds_bh = p.ds + ((int64_t)b * p.H + h) * DsLayout::per_bh(p.ds_nqb, p.ds_nkb, CAUSAL) * TE;

  int nend = Lk;
  if (CAUSAL) nend = min(nend, min(q0 + BM, Lq));
  if (q0 >= Lq) nend = 0;
  const int ntiles = (nend + BN - 1) / BN;

  // Tile (query block qb, key block kb) was stored by the dK/dV pass.
  auto tile_ok = [&](int qb, int kb) SIGATTN_INLINE {
    return qb < nqb_valid && kb < nkb_valid && (!CAUSAL || kb <= qb);
  };

  TileOffsets<D> to;
  to.init(lane);
  DmaPlan<BN, D, NW> dma;
  dma.init(w, lane);
  const int kv_stride_bytes = (int)(p.sk_t * 2);

  // Copy of a dS tile: instruction i fills keys 16i .. 16i+15 (1 KB); lane
  // j lands at key 16i + j/4, slot j%4 = (g-pair c, half h) and fetches
  // piece c of the stored lane 32h + key (at 1024 c + 16 (32h + key)).
  uint32_t soff[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int key = 16 * i + lane / 4, s = lane % 4;
    soff[i] = (uint32_t)((s >> 1) * 1024 + 16 * ((s & 1) * 32 + key));
  }
  // dSᵀ operand read: lane (group g16, s = 4e + m) reads key 16ks + 4h + e
  // (+8 for the second half), queries 4M .. 4M+3 with M = 4(g16 & 1) + m.
  int boff;
  {
    const int g16 = lane >> 4, s = lane & 15, e = s >> 2, m = s & 3, hh = g16 >> 1;
    boff = 32 * (4 * hh + e) + 8 * (2 * (g16 & 1) + (m & 1)) + 4 * (m >> 1);
  }
  auto ld_ds = [&](const uint16_t *tile, int ks) SIGATTN_INLINE {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    const uint16_t *base = tile + 512 * ks + boff;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)base);
    const s16x4 c = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4 *)(base + 256));
    const u32x2 lo = __builtin_bit_cast(u32x2, a);
    const u32x2 hv = __builtin_bit_cast(u32x2, c);
    return (u32x4){lo.x, lo.y, hv.x, hv.y};
  };
  // LDS slot of the wave's tile (column block cb, key block kl of the stage).
  auto ds_slot = [&](int st, int cb, int kl) SIGATTN_INLINE {
    return &sS[st][((4 * w + 2 * cb) * KB + 2 * kl) * TE / 2];
  };

  auto issue = [&](int st, int u) SIGATTN_INLINE {
    dma.issue(sK[st], Kb, kv_stride_bytes, u * BN, Lk);
#pragma unroll
    for (int cb = 0; cb < 2; ++cb) {
#pragma unroll
      for (int kl = 0; kl < KB; ++kl) {
        const int qb = qbw + cb, kb = KB * u + kl;
        // Tiles the dK/dV pass did not store are replaced by tile 0 of this
        // (batch, head) (in bounds; their products are skipped).
        const int64_t ti = tile_ok(qb, kb) ? DsLayout::tile(qb, kb, p.ds_nqb, CAUSAL) : 0;
        const uint16_t *src = ds_bh + ti * TE;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint16_t *dst = ds_slot(st, cb, kl) + 512 * i;
          const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)dst);
          // dS is read once: non-temporal loads keep it from displacing the
          // K rows the other workgroups of this (batch, head) re-read.
          if constexpr (kDqDsNT)
            asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt"
                         :
                         : "v"(soff[i]), "s"(src), "{m0}"(m0)
                         : "memory");
          else
            asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                         :
                         : "v"(soff[i]), "s"(src), "{m0}"(m0)
                         : "memory");
        }
      }
    }
  };

  f32x16 acc[2][NDB];
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int d = 0; d < NDB; ++d) acc[c][d] = zero16();

  // Every MFMA runs on every stage: a tile the dK/dV pass did not store
  // enters as a zero operand (the K rows are finite, so it adds exactly 0).
  // Branching around the products instead makes the compiler copy all the
  // accumulators at every join.
  auto compute = [&](int st, int u) SIGATTN_INLINE {
#pragma unroll
    for (int kl = 0; kl < KB; ++kl) {
      const int kb = KB * u + kl;
      const bool ok0 = tile_ok(qbw, kb), ok1 = tile_ok(qbw + 1, kb);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int ks = 2 * kl + j;
        u32x4 b0 = ld_ds(ds_slot(st, 0, kl), j);
        u32x4 b1 = ld_ds(ds_slot(st, 1, kl), j);
        b0 = ok0 ? b0 : zero4();
        b1 = ok1 ? b1 : zero4();
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          const u32x4 a = ld_tr<D>(sK[st], to, ks, db);
          acc[0][db] = Elem<T>::mfma(a, b0, acc[0][db]);
          acc[1][db] = Elem<T>::mfma(a, b1, acc[1][db]);
        }
      }
    }
  };

#pragma unroll
  for (int u = 0; u < PF; ++u)
    if (u < ntiles) issue(u, u);
  for (int u = 0; u < ntiles; ++u) {
    // Wait for this wave's copies of stage u (the later stages' copies may
    // stay in flight), then for every wave's.
    wait_vm_steps<NI, PF - 1>(min(ntiles - 1 - u, PF - 1));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    // The stage the copy fills last held stage u-1, which every wave has
    // finished reading (they all passed the barrier above after computing it).
    if (u + PF < ntiles) issue((u + PF) % NST, u + PF);
    compute(u % NST, u);
  }

  const float scale = *p.scale;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int my_q = q0 + 64 * w + 32 * c + l32;
    if (my_q < p.q_rows_out(Lq)) {
      uint16_t *row = dQb + (int64_t)my_q * p.sq_t;
      const bool valid = my_q < Lq;
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int d0 = db * 32 + 8 * g + 4 * hi;
          u32x2 o;
          o.x = Elem<T>::pack(acc[c][db][4 * g] * scale, acc[c][db][4 * g + 1] * scale);
          o.y = Elem<T>::pack(acc[c][db][4 * g + 2] * scale, acc[c][db][4 * g + 3] * scale);
          if (!valid) o = (u32x2){0u, 0u};
          *(u32x2 *)(row + d0) = o;
        }
      }
    }
  }
}

template <int ROWBLK, typename Launch>
static void launch_rows(const KParams &kp, int rows, Launch &&launch) {
  KParams p = kp;
  p.nblk = (rows + ROWBLK - 1) / ROWBLK;
  launch(p, dim3((unsigned)(p.nblk * p.B * p.H)));
}

template <typename T, int D, int WK>
static void bwd_dq_w(const KParams &kp, bool causal, bool sm, hipStream_t st) {
  launch_rows<128 / WK>(kp, kp.Tq, [&](const KParams &p, dim3 grid) {
    // Range split (dense non-causal): rsplit workgroups per item.
    if (WK == 1 && !causal && p.rsplit > 1) grid.x *= (unsigned)p.rsplit;
    grid.x += (unsigned)(p.ngap[0] + p.ngap[1]);
    if (causal) {
      if (sm) bwd_dq_kernel<T, D, WK, true, true><<<grid, 256, 0, st>>>(p);
      else bwd_dq_kernel<T, D, WK, true, false><<<grid, 256, 0, st>>>(p);
    } else {
      if (sm) bwd_dq_kernel<T, D, WK, false, true><<<grid, 256, 0, st>>>(p);
      else bwd_dq_kernel<T, D, WK, false, false><<<grid, 256, 0, st>>>(p);
    }
  });
}

// Pairs of waves (WK = 2, D <= 64, dq_wave_pairs) halve the longest item's chain
// for twice the tile copies (fp16 causal B=8 Lmax=2048 H=8 D=64, lengths
// 641..2048, 1024 blocks: 50.7 -> 41.5 us; B=4 T=1500 H=16 D=64 non-causal, 768
// blocks, forward + backward: 211 -> 216 us, which keeps one wave).
static bool dq_pairs(const KParams &p, bool causal) {
  return dq_wave_pairs((int64_t)p.B * p.H, p.Tq, p.Tk, causal, p.ragged(), p.ncu);
}

template <typename T, int D>
static void bwd_dq_t(const KParams &kp, bool causal, bool sm, hipStream_t st) {
  if constexpr (D <= 64) {
    if (kp.rsplit <= 1 && dq_pairs(kp, causal)) return bwd_dq_w<T, D, 2>(kp, causal, sm, st);
  }
  bwd_dq_w<T, D, 1>(kp, causal, sm, st);
}

// f(bool constants) of the run-time flags.
template <class F> static void by_flags(bool a, bool b, bool c, F &&f) {
  const auto last = [&](auto x, auto y) {
    if (c) f(x, y, std::true_type{});
    else f(x, y, std::false_type{});
  };
  const auto next = [&](auto x) {
    if (b) last(x, std::true_type{});
    else last(x, std::false_type{});
  };
  if (a) next(std::true_type{});
  else next(std::false_type{});
}

template <typename T, int D, bool DSOUT>
static void bwd_dkdv_t(const KParams &kp, bool causal, bool sm, hipStream_t st) {
  launch_rows<128>(kp, kp.Tk, [&](const KParams &p, dim3 grid) {
    if constexpr (D == 128) {
      // Dense problems: two key blocks per workgroup (see the kernel), or
      // one when a non-causal grid of pairs would not fill the GPU.
      if (!(p.ragged() && p.B <= 64)) {
        const int64_t paired = (int64_t)((p.nblk + 1) / 2) * p.B * p.H;
        const bool one_block = !causal && paired < device_compute_units();
        grid = dim3((unsigned)(one_block ? (int64_t)p.nblk * p.B * p.H : paired));
      }
      if (p.qgroup > 1 && p.qsplit > 1) grid.x *= (unsigned)p.qsplit;
      by_flags(causal, sm, p.qgroup > 1, [&](auto c, auto m, auto g) {
        bwd_dkdv_pair_kernel<T, c.value, m.value, DSOUT, g.value><<<grid, 512, 0, st>>>(p);
      });
      return;
    }
    // Range split (dense non-causal recompute backward): rsplit workgroups per item.
    if (!causal && !DSOUT && p.rsplit > 1) grid.x *= (unsigned)p.rsplit;
    if (p.qgroup > 1 && p.qsplit > 1) grid.x *= (unsigned)p.qsplit;
    by_flags(causal, sm, p.qgroup > 1, [&](auto c, auto m, auto g) {
      // The two-pass backward of grouped heads is D = 128's alone.
      if constexpr (!(DSOUT && g.value)) bwd_dkdv_kernel<T, D, c.value, m.value, DSOUT, g.value><<<grid, 256, 0, st>>>(p);
    });
  });
}

// Waves and ring stages of the D = 128 dQ-from-dS kernel.  Measured at
// B=4 L=4096 H=16 D=128 (causal / non-causal, one run): 8 waves with 4 stages
// (160 KB) 0.254 / 0.414 ms, with 3 stages 0.256 / 0.424 ms, with 2 stages
// 0.284 / 0.478 ms; 4 waves (two workgroups per CU) with 3 or 4 stages
// 0.265 / 0.44-0.45 ms.
#ifndef SIGATTN_DQDS_NW_128
#define SIGATTN_DQDS_NW_128 8
#endif
#ifndef SIGATTN_DQDS_NST_128
#define SIGATTN_DQDS_NST_128 4
#endif

// Grids of the D = 128 kernel with fewer 8-wave workgroups than the GPU has
// compute units (small problems, and long ones whose heads run in groups
// under the workspace cap) take 4-wave workgroups of 256 query rows with a
// 3-stage ring (72 KB, two per CU) instead, twice the workgroups on twice
// the CUs.
#ifndef SIGATTN_DQDS_SMALL_GRID
#define SIGATTN_DQDS_SMALL_GRID 1
#endif

template <typename T, int D>
static void bwd_dq_ds_t(const KParams &kp, bool causal, hipStream_t st) {
  constexpr int NW128 = SIGATTN_DQDS_NW_128, NST128 = SIGATTN_DQDS_NST_128;
  if constexpr (D == 128) {
    const int64_t wide = (int64_t)((kp.Tq + 64 * NW128 - 1) / (64 * NW128)) * kp.B * kp.H;
    if (SIGATTN_DQDS_SMALL_GRID && NW128 == 8 && wide < kp.ncu) {
      launch_rows<256>(kp, kp.Tq, [&](const KParams &p, dim3 grid) {
        grid.x += (unsigned)(p.ngap[0] + p.ngap[1]);
        if (causal) bwd_dq_ds_kernel<T, D, true, 4, 1, 3><<<grid, 256, 0, st>>>(p);
        else bwd_dq_ds_kernel<T, D, false, 4, 1, 3><<<grid, 256, 0, st>>>(p);
      });
      return;
    }
  }
  launch_rows<(D == 128 ? 64 * NW128 : 256)>(kp, kp.Tq, [&](const KParams &p, dim3 grid) {
    // D = 128: 8 waves (512 query rows: each K row read serves twice the dS
    // of a 4-wave workgroup; two waves per SIMD), one 32-key block per stage
    // in a 4-stage ring.  D = 64: 4 waves (the K rows of a 32-key stage do not
    // divide over 8 waves' copies), 6-stage ring.
    grid.x += (unsigned)(p.ngap[0] + p.ngap[1]);
    if constexpr (D == 128) {
      if (causal) bwd_dq_ds_kernel<T, D, true, NW128, 1, NST128><<<grid, 64 * NW128, 0, st>>>(p);
      else bwd_dq_ds_kernel<T, D, false, NW128, 1, NST128><<<grid, 64 * NW128, 0, st>>>(p);
    } else {
      if (causal) bwd_dq_ds_kernel<T, D, true, 4, 1, 6><<<grid, 256, 0, st>>>(p);
      else bwd_dq_ds_kernel<T, D, false, 4, 1, 6><<<grid, 256, 0, st>>>(p);
    }
  });
}

// dtype in {kF16, kBF16}, D in {32, 64, 128} (the two-pass backward's
// dQ-from-dS kernel: 64 and 128 only).
template <bool WITH32 = true, class F>
static void by_type(int dtype, int D, F &&f) {
  const auto d = [&](auto *t) {
    if (D == 128) f(t, std::integral_constant<int, 128>{});
    else if (!WITH32 || D == 64) f(t, std::integral_constant<int, 64>{});
    else if constexpr (WITH32) f(t, std::integral_constant<int, 32>{});
  };
  if (dtype == kBF16) d((__bf16 *)nullptr);
  else d((_Float16 *)nullptr);
}

int bwd_dq_rows_per_workgroup() { return 128; }
int bwd_dkdv_rows_per_workgroup() { return 128; }
// Resident workgroups per CU of the recompute kernels at D = 64 (dQ: 32 KB of
// LDS and at most 168 VGPRs; dK/dV: 64 KB and 128 + 128 registers); D = 32
// the same.
int bwd_dq_workgroups_per_cu(int D) { return D <= 64 ? 3 : 2; }
int bwd_dkdv_workgroups_per_cu(int D) { return D <= 64 ? 2 : 1; }

void launch_bwd_dq_mfma(const KParams &p, int dtype, int D, bool causal, bool sm, hipStream_t st) {
  by_type(dtype, D, [&](auto *t, auto d) {
    bwd_dq_t<std::remove_pointer_t<decltype(t)>, decltype(d)::value>(p, causal, sm, st);
  });
}

void launch_bwd_dkdv_mfma(const KParams &p, int dtype, int D, bool causal, bool sm, bool dsout,
                          hipStream_t st) {
  by_type(dtype, D, [&](auto *t, auto d) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int DD = decltype(d)::value;
    if constexpr (DD > 32) {  // no two-pass form below
      if (dsout) bwd_dkdv_t<T, DD, true>(p, causal, sm, st);
    }
    if (!dsout) bwd_dkdv_t<T, DD, false>(p, causal, sm, st);
  });
  launch_add_parts(p, dtype, st);
}

void launch_add_parts(const KParams &p, int dtype, hipStream_t st) {
  if (p.qgroup <= 1 || p.qsplit <= 1) return;
  const int per_row = p.H * p.dmem / 8, rows = per_row < 256 ? 256 / per_row : 1;
  const dim3 grid((unsigned)((p.rows_k + rows - 1) / rows)), block(256);
  if (dtype == kBF16) add_parts_kernel<__bf16><<<grid, block, 0, st>>>(p, per_row);
  else if (dtype == kF16) add_parts_kernel<_Float16><<<grid, block, 0, st>>>(p, per_row);
  else add_parts_kernel<float><<<grid, block, 0, st>>>(p, per_row);
}

void launch_bwd_fused_mfma(const KParams &kp, int dtype, int D, bool causal, bool sm, hipStream_t st) {
  by_type(dtype, D, [&](auto *t, auto d) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int DD = decltype(d)::value;
    if constexpr (DD <= 64) {
      KParams pq = kp, pk = kp;
      const bool pairs = dq_pairs(kp, causal);
      pq.nblk = pairs ? (kp.Tq + 63) / 64 : (kp.Tq + 127) / 128;
      pk.nblk = (kp.Tk + 127) / 128;
      pq.rsplit = pk.rsplit = 1;
      pq.ngap[0] = pq.ngap[1] = pk.ngap[0] = pk.ngap[1] = 0;  // no packed layouts: no gap rows
      const int nkv = pk.nblk * kp.B * kp.H;
      const dim3 grid((unsigned)(nkv + pq.nblk * kp.B * kp.H));
      const auto launch = [&](auto wk) {
        constexpr int WK = decltype(wk)::value;
        if (causal) {
          if (sm) bwd_fused_kernel<T, DD, WK, true, true><<<grid, 256, 0, st>>>(pq, pk, nkv);
          else bwd_fused_kernel<T, DD, WK, true, false><<<grid, 256, 0, st>>>(pq, pk, nkv);
        } else if constexpr (WK == 1) {  // a workgroup per CU
          if (sm) bwd_fused_kernel<T, DD, WK, false, true><<<grid, 256, 0, st>>>(pq, pk, nkv);
          else bwd_fused_kernel<T, DD, WK, false, false><<<grid, 256, 0, st>>>(pq, pk, nkv);
        }
      };
      if (pairs) launch(std::integral_constant<int, 2>{});
      else launch(std::integral_constant<int, 1>{});
    }
  });
}

void launch_bwd_dq_ds_mfma(const KParams &p, int dtype, int D, bool causal, hipStream_t st) {
  by_type<false>(dtype, D, [&](auto *t, auto d) {
    bwd_dq_ds_t<std::remove_pointer_t<decltype(t)>, decltype(d)::value>(p, causal, st);
  });
}

}  // namespace sigattn
