// Forward launchers; the kernel is in fwd_kernel.h.
#include "fwd_kernel.h"
#include "launch.h"

namespace sigattn {

// Query column blocks per wave at D = 128: 1 = eight waves of 32 queries (two
// per SIMD, so each SIMD interleaves two waves' VALU and LDS work); 2 = four
// waves of 64 queries (every K / Vᵀ operand read feeds two MFMAs).  Measured at
// B=4 L=4096 H=16 causal: 1 is 2-3% faster.
#ifndef SIGATTN_FWD_NCB
#define SIGATTN_FWD_NCB 1
#endif

template <typename T, int D, int NWV, int WK, int NCB = SIGATTN_FWD_NCB>
static void launch_fwd_w(const KParams &kp, bool causal, bool scoremod, hipStream_t st) {
  constexpr int BM = NWV * 32 * NCB / WK;
  KParams p = kp;
  p.nblk = (p.Tq + BM - 1) / BM;
  // Dense causal problems (the kernel's order when not ragged with B <= 64):
  // two query blocks per workgroup.
  const bool pairs = causal && kFwdCausalPairs && !(p.ragged() && p.B <= 64);
  if (causal || p.rsplit < 1) p.rsplit = 1;
  const dim3 grid((unsigned)((pairs ? (p.nblk + 1) / 2 : p.nblk) * p.B * p.H * p.rsplit + p.ngap[0] + p.ngap[1]));
  const dim3 block(64 * NWV);
  if (causal) {
    if (scoremod) fwd_mfma_kernel<T, D, NWV, NCB, WK, true, true, KParams><<<grid, block, 0, st>>>(p);
    else fwd_mfma_kernel<T, D, NWV, NCB, WK, true, false, KParams><<<grid, block, 0, st>>>(p);
  } else {
    if (scoremod) fwd_mfma_kernel<T, D, NWV, NCB, WK, false, true, KParams><<<grid, block, 0, st>>>(p);
    else fwd_mfma_kernel<T, D, NWV, NCB, WK, false, false, KParams><<<grid, block, 0, st>>>(p);
  }
}

// 64 queries per wave (D = 64, two workgroups of 256 queries per CU): every
// K / Vᵀ operand read from LDS feeds two MFMAs.  With 32 queries the reads take
// as many LDS cycles as the MFMAs take matrix cycles, and their energy lowers
// the power-limited clock.  Same bits.  bf16 us, 32 -> 64: B=8 T=2048 H=32 339
// -> 321 (causal 208 -> 198), B=2 T=8192 H=32 1237 -> 1138 (647 -> 617),
// lengths 1487..8192 B=4 H=12 483 -> 449.  The blocks are twice as long, which
// costs more than that where
//   * a sequence has few of them, or ends in half of one (T=513 to 845 up to 33 %
//     slower, T=1025 23 %, T=1152 3-20 %; from 2048 rows on half a block is 6 %);
//   * the grid is small.  Times of 64 over 32, by 256-query blocks per CU f:
//     dense f = 2.06..2.5 1.06-1.12, 3.06..3.5 1.01-1.04, but 2.0, 2.53..3.0 and
//     3.56..4.0 0.92-0.96 -- the blocks of 128 of an odd round fill CUs that
//     the long blocks leave half empty -- and f > 4 0.92-1.02; causal f = 4..5
//     0.97-1.02, f = 8 0.92-0.97; lengths T/16..T f = 4..5 0.91-1.39, 6..7
//     0.94-1.03 from T = 2000 on (T = 1000 1.09, causal), f = 8 0.93-1.02.
static bool wide_waves(const KParams &p, bool causal) {
  const int64_t n = (p.Tq + 127) / 128, blocks = (int64_t)p.B * p.H * ((p.Tq + 255) / 256), cus = p.ncu;
  if (cus <= 0 || n < 8 || (n % 2 != 0 && n < 16)) return false;
  if (p.ragged()) return blocks >= (n < 16 ? 8 : 6) * cus;
  if (blocks >= 4 * cus) return true;
  return !causal && blocks >= 2 * cus && (2 * blocks + cus - 1) / cus % 2 == 0;
}

// D = 128: one workgroup of eight waves per CU (128 KB of LDS).  D = 64: a
// 3-stage ring of 48 KB, so three workgroups of four waves share a CU (three
// waves per SIMD, at most 168 VGPRs each) in small work units, which balance
// better on small or ragged (padded) batches than two with a 4-stage ring.  Measured
// at 10-20 % dense and 5-13 % padded.
template <typename T, int D>
static void launch_fwd_t(const KParams &kp, bool causal, bool scoremod, hipStream_t st) {
  // Pairs of waves (WK = 2, fwd_wave_pairs): half of every block's chain (fp16
  // B=2 T=1024 H=8 D=64, 128 blocks: call 16.8 -> 12.2 us).  Beyond one block
  // per CU, a tile per region leaves its copy one region of time and the fourth
  // stage the third workgroup (512 blocks 27.6 -> 31.2 us non-causal, 19.8 ->
  // 22.3 causal).
  if constexpr (D <= 64) {
    if (kp.rsplit <= 1 && fwd_wave_pairs(kp)) return launch_fwd_w<T, D, 4, 2>(kp, causal, scoremod, st);
  }
  if constexpr (D == 64) {
    if (kp.rsplit <= 1 && wide_waves(kp, causal)) return launch_fwd_w<T, D, 4, 1, 2>(kp, causal, scoremod, st);
  }
  launch_fwd_w<T, D, (D <= 64 ? 4 : 8) / SIGATTN_FWD_NCB, 1>(kp, causal, scoremod, st);
}

int fwd_rows_per_workgroup(int D) { return (D <= 64 ? 4 : 8) * 32; }
int fwd_workgroups_per_cu(int D) {
  return D == 32 ? fwd_occupancy<32>() : (D == 64 ? fwd_occupancy<64>() : fwd_occupancy<128>());
}

__global__ __launch_bounds__(256) void rs_clear_kernel(int *a, int na, int *b, int nb) {
  for (int i = blockIdx.x * 256 + threadIdx.x; i < na + nb; i += gridDim.x * 256) {
    if (i < na) a[i] = 0;
    else b[i - na] = 0;
  }
}
void launch_rs_clear(int *a, int na, int *b, int nb, hipStream_t st) {
  const int n = na + nb;
  if (n > 0) rs_clear_kernel<<<(unsigned)min((n + 255) / 256, 64), 256, 0, st>>>(a, na, b, nb);
}

void launch_fwd_mfma(const KParams &p, int dtype, int D, bool causal, bool scoremod,
                     hipStream_t st) {
  if (dtype == kBF16) {
    if (D == 128) launch_fwd_t<__bf16, 128>(p, causal, scoremod, st);
    else if (D == 64) launch_fwd_t<__bf16, 64>(p, causal, scoremod, st);
    else launch_fwd_t<__bf16, 32>(p, causal, scoremod, st);
  } else {
    if (D == 128) launch_fwd_t<_Float16, 128>(p, causal, scoremod, st);
    else if (D == 64) launch_fwd_t<_Float16, 64>(p, causal, scoremod, st);
    else launch_fwd_t<_Float16, 32>(p, causal, scoremod, st);
  }
}

}  // namespace sigattn
