// Attention over a paged cache for sequences of up to 32 columns (new tokens
// times the query heads of a K / V head): decoding and short chunks.
//
// Bound by the read of K and V: 4·D bytes a key and K / V head against 4·D·32
// matrix operations whatever the columns, a third of what the matrix cores do
// in that time.  The group's query heads are columns of the same product, so a
// K / V head is read once for all of them.  A unit is (sequence, K / V head,
// chunk of keys), chunks so that the GPU is full (PagedUnit); units of
// one chunk write O themselves, the others leave fp32 sums for the reduction.
// Every wave has a unit of its own, the units of one key range in head order,
// so the waves of a workgroup read the rows of neighbouring K / V heads and never
// wait for each other.  A wave streams its 32-key blocks through a private
// two-stage LDS ring with direct, non-temporal global->LDS copies (PagedDma) that
// it waits for with its own vmcnt: Sᵀ = K·Qᵀ, P = sigmoid(Sᵀ) on packed words,
// Oᵀ += Vᵀ·Pᵀ.  bf16 H=32 Hkv=8 D=128: 16 requests of contexts 1024 .. 8191 (250 MB)
// 43 us, 5.8 TB/s; 64 of 8000 .. 9000 6.57 TB/s, of a device copy's 4.9 and a
// fill's 6.9; one of 65535 keys H=16 Hkv=2 (67 MB) 18.5 us, a third of it the
// waves' start (a sequence of one block alone takes 6.5).
#pragma once

#include <type_traits>

#include "paged.h"
#include "rel.h"

namespace sigattn {

// Waves per workgroup.  1 / 2 / 4, us (as the caller's figures): B=16 contexts
// 1024..8191 61 / 48 / 49, B=64 8000..9000 438 / 333 / 338, D=64 35 / 34 / 29.
constexpr int kDecodeWaves = 4;

// Each wave's two stages of K and V blocks, and of their keys' score_mod.
template <int D, int NW> using DecodeTiles = uint16_t[NW][2][32 * D];
template <int NW, bool SCOREMOD> using DecodeTerms = float[SCOREMOD ? NW : 1][2][64];

// The units of workgroup `wg`, on its first NW waves.
template <typename T, int D, int NW, bool CAUSAL, bool SCOREMOD, class P>
__device__ __forceinline__ void paged_decode_body(const P &p, const int wg, DecodeTiles<D, NW> &sK,
                                                  DecodeTiles<D, NW> &sV, DecodeTerms<NW, SCOREMOD> &sM) {
  constexpr int KB = 32;  // keys per block
  constexpr int NKS = D / 16, NDB = D / 32, PB = p_bits<T, P>();
  static_assert(kDecodeCols == 32, "a column a lane");
  using Dma = PagedDma<KB, D, 1, true>;
  constexpr int NI = Dma::NI;                  // copy instructions per block of V
  constexpr int NK = NI + (SCOREMOD ? 1 : 0);  // ... of K, with its keys' score_mod

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hi = lane >> 5;
  if (w >= NW) return;
  const int unit = wg * NW + w;
  const PagedUnit un = paged_unit(p, unit, kDecodeCols);
  if (un.nck == 0) return;
  const bool half = p.half_head(D);
  const int cols = un.Lq * p.G, keys = un.k1 - un.k0;

  const int64_t koff = (int64_t)un.hk * p.sk_h;
  const uint16_t *Kb = (const uint16_t *)p.k + koff, *Vb = (const uint16_t *)p.v + koff;
  const float bias = p.bias_of(un.Lk), nsl = -p.fscale * kLog2e, nbl = -bias * kLog2e;

  // Column l32 as the B operand (k = d = 16s + 8h + j); columns past the unit's are zero.
  u32x4 qf[NKS];
  const int tok = l32 / p.G;
  {
    const bool ok = l32 < cols;
    const uint16_t *qrow = (const uint16_t *)p.q + (packed_first(p.cu_q, p.rows_q, un.b) + tok) * p.sq_t +
                           (int64_t)(un.hk * p.G + l32 - tok * p.G) * p.sq_h + 8 * hi;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) qf[ks] = ok && !(half && ks > 0) ? *(const u32x4 *)(qrow + 16 * ks) : zero4();
  }
  // Keys of the chunk that this lane's token sees, and that every token sees.
  const int lim = CAUSAL ? un.Lk - un.Lq + min(tok, un.Lq - 1) + 1 - un.k0 : keys;
  const int all_see = CAUSAL ? un.Lk - un.Lq + 1 - un.k0 : keys;

  [[maybe_unused]] RelColumn rc;
  if constexpr (P::kRel) {
    const int col = min(l32, cols - 1), t = col / p.G;
    rc.init(p, un.hk * p.G + col - t * p.G, un.Lk - un.Lq + t - un.k0, bias);
  }

  f32x16 acc[1][NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) acc[0][db] = zero16();

  TileOffsets<D> to;
  to.init(lane);
  Dma dma;
  dma.init(p, un.b, un.k0, keys, 0, lane, half);
  const int nb = (keys + KB - 1) / KB;
  const float *mod = SCOREMOD ? p.score_mod + un.b * p.mod_stride + un.k0 : nullptr;
  auto issue_k = [&](int i, const int (&at)[Dma::NE]) SIGATTN_INLINE {
    dma.issue_at(sK[w][i & 1], Kb, KB * i, at);
    if constexpr (SCOREMOD) {
      const uint32_t off = 4u * (uint32_t)min(KB * i + lane, keys - 1);
      const uint32_t dst = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)sM[w][i & 1]);
      asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, %1" : : "v"(off), "s"(mod), "{m0}"(dst) : "memory");
    }
  };
  auto issue_v = [&](int i) SIGATTN_INLINE { dma.issue_last(sV[w][i & 1], Vb, KB * i, KB * (i + 1)); };

  // The first three blocks' pages at once, then one block ahead.
  if (nb > 0) {
    int first[2][Dma::NE];
    dma.entries(0, first[0]);
    dma.entries(KB, first[1]);
    dma.load(2 * KB);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (i < nb) {
        issue_k(i, first[i]);
        dma.issue_at(sV[w][i], Vb, KB * i, first[i]);
      }
  }
  // The wait for Q (which also waits for the copies above) stays out of the loop.
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) asm volatile("" ::"v"(qf[ks]));
  for (int i = 0; i < nb; ++i) {
    // Copies in issue order: K(i) V(i) K(i+1) V(i+1) K(i+2) ...
    if (i + 1 < nb) wait_vm<2 * NI + NK>();
    else wait_vm<NI>();
    const uint16_t *tK = sK[w][i & 1], *tV = sV[w][i & 1];
    f32x16 sc = zero16();
    float c[16];
    if constexpr (P::kRel) rc.block(KB * i, hi, c);
#pragma unroll
    for (int g = 0; g < (P::kRel ? 0 : 4); ++g) {
      f32x4 m = {nbl, nbl, nbl, nbl};
      if (SCOREMOD) {
        const f32x4 x = *(const f32x4 *)&sM[w][i & 1][8 * g + 4 * hi];
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j] = -(bias + x[j]) * kLog2e;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) c[4 * g + j] = m[j];
    }
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) sc = Elem<T>::mfma(ld_row<D>(tK, to, 0, ks), qf[ks], sc);
    if (i + 2 < nb) {
      // Every read of K(i) has returned before the copy that replaces it.
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      issue_k(i + 2, dma.ent);
    }

    // P words: accumulator element e of lane (l32, hi) is key
    // kb + 8(e/4) + 4hi + e%4 of column l32.  Keys past the chunk have zero V rows (but
    // what the learned bias holds there may be NaN).
    const int kb = KB * i;
    uint32_t pk[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      pk[e] = Elem<T>::pack(sigmoid_times_2<PB>(__builtin_fmaf(sc[2 * e], nsl, c[2 * e])),
                            sigmoid_times_2<PB>(__builtin_fmaf(sc[2 * e + 1], nsl, c[2 * e + 1])));
    if ((CAUSAL || P::kRel) && kb + KB > all_see) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int key = kb + 8 * (e / 2) + 4 * hi + 2 * (e % 2);
        pk[e] &= (key < lim ? 0x0000ffffu : 0u) | (key + 1 < lim ? 0xffff0000u : 0u);
      }
    }
    if (i + 2 < nb) wait_vm<NI + 2 * NK>();
    else if (i + 1 < nb) wait_vm<NI + NK>();
    else wait_vm<0>();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const u32x4 bp = (u32x4){pk[4 * j], pk[4 * j + 1], pk[4 * j + 2], pk[4 * j + 3]};
#pragma unroll
      for (int db = 0; db < NDB; ++db) acc[0][db] = Elem<T>::mfma(ld_tr<D>(tV, to, j, db), bp, acc[0][db]);
    }
    if (i + 2 < nb) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      issue_v(i + 2);
    }
  }

  if constexpr (PB > 0) {
#pragma unroll
    for (int db = 0; db < NDB; ++db) acc[0][db] *= 1.0f / (1 << PB);
  }
  paged_store<T, D, 1>(p, un, acc, l32, l32, kDecodeCols, unit, hi, half);
}

}  // namespace sigattn
