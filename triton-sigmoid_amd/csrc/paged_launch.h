// Launches of the matrix kernels over a paged cache (f16 / bf16), plain (PagedParams)
// or with the learned bias by relative position (PagedRelParams).
#pragma once

#include "fwd_kernel.h"
#include "paged_decode.h"

namespace sigattn {

// f(causal, score_mod) as constants; no score_mod beside the learned bias.
template <class P, class F> void by_terms(const P &p, bool causal, F &&f) {
  const auto terms = [&](auto c) {
    if constexpr (!P::kRel) {
      if (p.score_mod) return f(c, std::true_type{});
    }
    f(c, std::false_type{});
  };
  if (causal) terms(std::true_type{});
  else terms(std::false_type{});
}

// D = 128: eight waves, one workgroup per CU; below, four, three and four per
// CU (fwd_kernel.h).
constexpr int waves_of(int D) { return D == 128 ? 8 : 4; }

template <typename T, int D, class P> void fwd_t(const P &p, int units, bool causal, hipStream_t st) {
  constexpr int NWV = waves_of(D);
  const dim3 grid((unsigned)(units + p.ngap[0])), block(64 * NWV);
  by_terms(p, causal, [&](auto c, auto m) {
    fwd_mfma_kernel<T, D, NWV, 1, 1, c.value, m.value, P><<<grid, block, 0, st>>>(p);
  });
}

// Batches with sequences of both kernels: the first nf workgroups (after the gap
// ones) run blocks of columns, the others decode, so that the longer part's
// last workgroups run beside the shorter part's, and a launch less.  The parts
// share their LDS; at D = 64 decoding takes three waves, which fit what three
// workgroups of a CU leave each, and everywhere as many as the LDS holds.
// fp16 H=12 Hkv=4 D=64, 20 requests of a token and 4 of 100 .. 700 on up to 4096
// keys: 38 us (the whole call 41; when it was two launches, one after the other,
// 11 more).
template <int D> constexpr int mixed_waves() { return D == 64 ? 3 : 4; }
template <typename T, int D, bool CAUSAL, bool SCOREMOD, class P>
__global__ __launch_bounds__(64 * waves_of(D), (fwd_occupancy<D, 1, 1>())) void paged_mixed_kernel(
    const P pf, const P pd, const int nf) {
  constexpr int NW = mixed_waves<D>();
  __shared__ __attribute__((aligned(16))) FwdTiles<D, 1> sK, sV;
  __shared__ __attribute__((aligned(16))) FwdTerms<D, 1, SCOREMOD> sC;
  __shared__ __attribute__((aligned(16))) DecodeTerms<NW, SCOREMOD> sM;
  static_assert(sizeof(sK) == sizeof(DecodeTiles<D, NW>), "the parts share their tiles");
  const int wg = gap_prologue<2>(pf, sK);
  if (wg < 0) return;
  if (wg < nf)
    fwd_mfma_body<T, D, waves_of(D), 1, 1, CAUSAL, SCOREMOD, P>(pf, wg, sK, sV, sC);
  else
    paged_decode_body<T, D, NW, CAUSAL, SCOREMOD, P>(pd, wg - nf, reinterpret_cast<DecodeTiles<D, NW> &>(sK),
                                                  reinterpret_cast<DecodeTiles<D, NW> &>(sV), sM);
}

template <typename T, int D, class P>
void mixed_t(const P &pf, int nf, const P &pd, int nd, bool causal, hipStream_t st) {
  constexpr int NW = mixed_waves<D>();
  const dim3 grid((unsigned)(nf + (nd + NW - 1) / NW + pf.ngap[0])), block(64 * waves_of(D));
  by_terms(pf, causal, [&](auto c, auto m) {
    paged_mixed_kernel<T, D, c.value, m.value, P><<<grid, block, 0, st>>>(pf, pd, nf);
  });
}

template <typename T, int D, bool CAUSAL, bool SCOREMOD, class P>
__global__ __launch_bounds__(64 * kDecodeWaves, 1) void paged_decode_kernel(const P p) {
  __shared__ __attribute__((aligned(16))) DecodeTiles<D, kDecodeWaves> sK, sV;
  __shared__ __attribute__((aligned(16))) DecodeTerms<kDecodeWaves, SCOREMOD> sM;
  const int wg = gap_prologue<2>(p, sK);
  if (wg < 0) return;
  paged_decode_body<T, D, kDecodeWaves, CAUSAL, SCOREMOD, P>(p, wg, sK, sV, sM);
}

template <typename T, int D, class P> void decode_t(const P &p, int units, bool causal, hipStream_t st) {
  const dim3 grid((unsigned)((units + kDecodeWaves - 1) / kDecodeWaves + p.ngap[0])), block(64 * kDecodeWaves);
  by_terms(p, causal, [&](auto c, auto m) {
    paged_decode_kernel<T, D, c.value, m.value, P><<<grid, block, 0, st>>>(p);
  });
}

template <class F> void by_type(int dtype, int D, F &&f) {
  const auto d = [&](auto *t) {
    if (D == 128) f(t, std::integral_constant<int, 128>{});
    else if (D == 64) f(t, std::integral_constant<int, 64>{});
    else f(t, std::integral_constant<int, 32>{});
  };
  if (dtype == kBF16) d((__bf16 *)nullptr);
  else if (dtype == kF16) d((_Float16 *)nullptr);
  else d((float *)nullptr);
}

}  // namespace sigattn
