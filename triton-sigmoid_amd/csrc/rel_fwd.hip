// The forward kernel (fwd_kernel.h) with the learned bias by relative position:
// sigmoid(q·k·scale + bias + line[k - q]).  A tile of 64 keys meets a block of BM
// queries at BM + 63 relative positions, so BM + 64 values of the line go to LDS with
// each tile, a thread one of them, loaded a tile ahead; a lane (a query) reads the
// sixteen of its accumulator, four in a row at a time.  The scores' fma takes them
// where it takes the bias without the line: the sigmoid's arithmetic bounds D = 64, the
// matrix cores D = 128, as without (us, with / without: bf16 16 sequences of 101 .. 1001
// H=12 D=64 46 / 45; causal, 3 of 1500 .. 4096 H=16 Hkv=4 D=128 201 / 205).
#include "fwd_kernel.h"
#include "launch.h"
#include "rel.h"

namespace sigattn {
namespace {

template <typename T, int D, int NWV, int WK>
void fwd_w(const RelParams &kp, bool causal, hipStream_t st) {
  constexpr int BM = NWV * 32 / WK;
  RelParams p = kp;
  p.nblk = (p.Tq + BM - 1) / BM;
  p.rsplit = 1;
  const dim3 grid((unsigned)(p.nblk * p.B * p.H + p.ngap[0] + p.ngap[1])), block(64 * NWV);
  if (causal) fwd_mfma_kernel<T, D, NWV, 1, WK, true, false, RelParams><<<grid, block, 0, st>>>(p);
  else fwd_mfma_kernel<T, D, NWV, 1, WK, false, false, RelParams><<<grid, block, 0, st>>>(p);
}

// Pairs of waves as without the bias.  Not its 64 queries a wave of large grids at D = 64:
// their windows would be 320 places a tile for 256 threads.  Without that form a wave reads
// each tile for 32 queries; us, with / without the bias, H=16 D=64: one sequence of 8192 353 / 317
// (causal 189 / 169), four 1295 / 1115 (causal 703 / 613), two of 4096 187 / 164.
template <typename T, int D> void fwd_t(const RelParams &p, bool causal, hipStream_t st) {
  if constexpr (D <= 64) {
    if (fwd_wave_pairs(p)) return fwd_w<T, D, 4, 2>(p, causal, st);
  }
  fwd_w<T, D, D <= 64 ? 4 : 8, 1>(p, causal, st);
}

template <typename T> void fwd_d(const RelParams &p, int D, bool causal, hipStream_t st) {
  if (D == 128) fwd_t<T, 128>(p, causal, st);
  else if (D == 64) fwd_t<T, 64>(p, causal, st);
  else fwd_t<T, 32>(p, causal, st);
}

}  // namespace

void launch_rel_fwd_mfma(const RelParams &p, int dtype, int D, bool causal, hipStream_t st) {
  if (dtype == kBF16) fwd_d<__bf16>(p, D, causal, st);
  else fwd_d<_Float16>(p, D, causal, st);
}

}  // namespace sigattn
