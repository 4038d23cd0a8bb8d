// Launches of the decoding kernel (paged_decode.h).
#include "launch.h"
#include "paged_decode.h"

namespace sigattn {
namespace {

template <typename T, int D, bool CAUSAL, bool SCOREMOD>
__global__ __launch_bounds__(64 * kDecodeWaves, 1) void paged_decode_kernel(const PagedParams p) {
  __shared__ __attribute__((aligned(16))) DecodeTiles<D, kDecodeWaves> sK, sV;
  __shared__ __attribute__((aligned(16))) DecodeTerms<kDecodeWaves, SCOREMOD> sM;
  const int wg = gap_prologue<2>(p, sK);
  if (wg < 0) return;
  paged_decode_body<T, D, kDecodeWaves, CAUSAL, SCOREMOD>(p, wg, sK, sV, sM);
}

template <typename T, int D> void decode_t(const PagedParams &p, int units, bool causal, hipStream_t st) {
  const dim3 grid((unsigned)((units + kDecodeWaves - 1) / kDecodeWaves + p.ngap[0])), block(64 * kDecodeWaves);
  if (causal) {
    if (p.score_mod) paged_decode_kernel<T, D, true, true><<<grid, block, 0, st>>>(p);
    else paged_decode_kernel<T, D, true, false><<<grid, block, 0, st>>>(p);
  } else {
    if (p.score_mod) paged_decode_kernel<T, D, false, true><<<grid, block, 0, st>>>(p);
    else paged_decode_kernel<T, D, false, false><<<grid, block, 0, st>>>(p);
  }
}

template <typename T> void decode_d(const PagedParams &p, int units, int D, bool causal, hipStream_t st) {
  if (D == 128) decode_t<T, 128>(p, units, causal, st);
  else if (D == 64) decode_t<T, 64>(p, units, causal, st);
  else decode_t<T, 32>(p, units, causal, st);
}

}  // namespace

void launch_paged_decode(const PagedParams &p, int units, int dtype, int D, bool causal, hipStream_t st) {
  if (dtype == kBF16) decode_d<__bf16>(p, units, D, causal, st);
  else decode_d<_Float16>(p, units, D, causal, st);
}

}  // namespace sigattn
