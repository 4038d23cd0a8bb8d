// The recompute backward's kernels (bwd_kernel.h) with the learned bias by relative
// position: dQ, which also sums dS by relative position, and dK/dV.
#include "bwd_kernel.h"
#include "launch.h"
#include "rel.h"

namespace sigattn {
namespace {

template <typename T, int D, int WK, bool CAUSAL>
__global__ __launch_bounds__(256, 2) void rel_dq_kernel(const RelParams p) {
  __shared__ __attribute__((aligned(16))) DqLds<D, false, dq_window<RelParams, WK>()> lds;
  __shared__ unsigned long long gap_lds[2];
  extern __shared__ __attribute__((aligned(16))) float near[];  // the four waves' lines and pieces
  const int wg = gap_prologue<2>(p, gap_lds);
  if (wg >= 0) bwd_dq_body<T, D, WK, CAUSAL, false, RelParams>(p, wg, lds, near);
}

template <typename T, int D, bool CAUSAL, bool GROUPED>
__global__ __launch_bounds__(256, (D <= 64 ? 2 : 1)) void rel_dkdv_kernel(const RelParams p) {
  __shared__ __attribute__((aligned(16))) DkdvLds<D, dkdv_window<RelParams>()> lds;
  bwd_dkdv_body<T, D, CAUSAL, false, false, GROUPED, RelParams>(p, blockIdx.x, lds);
}

template <typename T, int D, int WK> void dq_w(const RelParams &kp, bool causal, hipStream_t st) {
  RelParams p = kp;
  p.part_rows = 128 / WK;
  p.nblk = (p.Tq + p.part_rows - 1) / p.part_rows;
  const dim3 grid((unsigned)(p.nblk * p.B * p.H + p.ngap[0] + p.ngap[1]));
  const size_t line = p.part != nullptr ? near_floats(p.reach) * sizeof(float) : 0;
  if (causal) rel_dq_kernel<T, D, WK, true><<<grid, 256, line, st>>>(p);
  else rel_dq_kernel<T, D, WK, false><<<grid, 256, line, st>>>(p);
}

// Pairs of waves as without the bias.
bool dq_pairs(const RelParams &p, int D, bool causal) {
  return D <= 64 && dq_wave_pairs((int64_t)p.B * p.H, p.Tq, p.Tk, causal, p.ragged(), p.ncu);
}

template <typename T, int D> void dkdv_t(const RelParams &kp, bool causal, hipStream_t st) {
  RelParams p = kp;
  p.nblk = (p.Tk + 127) / 128;
  dim3 grid((unsigned)(p.nblk * p.B * p.H));
  if (p.qgroup > 1) {
    if (p.qsplit > 1) grid.x *= (unsigned)p.qsplit;
    if (causal) rel_dkdv_kernel<T, D, true, true><<<grid, 256, 0, st>>>(p);
    else rel_dkdv_kernel<T, D, false, true><<<grid, 256, 0, st>>>(p);
  } else {
    if (causal) rel_dkdv_kernel<T, D, true, false><<<grid, 256, 0, st>>>(p);
    else rel_dkdv_kernel<T, D, false, false><<<grid, 256, 0, st>>>(p);
  }
}

template <class F> void by_type(int dtype, int D, F &&f) {
  const auto d = [&](auto *t) {
    if (D == 128) f(t, std::integral_constant<int, 128>{});
    else if (D == 64) f(t, std::integral_constant<int, 64>{});
    else f(t, std::integral_constant<int, 32>{});
  };
  if (dtype == kBF16) d((__bf16 *)nullptr);
  else d((_Float16 *)nullptr);
}

}  // namespace

int rel_dq_rows(const RelParams &p, int D, bool causal) { return dq_pairs(p, D, causal) ? 64 : 128; }

void launch_rel_dq_mfma(const RelParams &p, int dtype, int D, bool causal, hipStream_t st) {
  by_type(dtype, D, [&](auto *t, auto d) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int DD = decltype(d)::value;
    if constexpr (DD <= 64) {
      if (dq_pairs(p, DD, causal)) return dq_w<T, DD, 2>(p, causal, st);
    }
    dq_w<T, DD, 1>(p, causal, st);
  });
}

void launch_rel_dkdv_mfma(const RelParams &p, int dtype, int D, bool causal, hipStream_t st) {
  by_type(dtype, D, [&](auto *t, auto d) {
    dkdv_t<std::remove_pointer_t<decltype(t)>, decltype(d)::value>(p, causal, st);
  });
  launch_add_parts(p, dtype, st);
}

}  // namespace sigattn
