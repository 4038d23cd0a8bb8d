// The recompute backward's kernels (bwd_kernel.h) with the learned bias by relative
// position: dQ, which also sums dS by relative position, and dK/dV.  The lines' windows
// are staged as in the forward.  bf16, us, with / without the bias: 16 sequences of 101
// .. 1001 H=12 D=64 dK/dV 83 / 78, dQ 73 / 55 (62 without the sums: near the diagonal
// they are a third of a block's arithmetic); causal, 3 of 1500 .. 4096 H=16 Hkv=4
// D=128 dK/dV 419 / 428 (storing dS, in pairs of waves), dQ 327 (300 without the sums) /
// 184 from the stored dS.  No two-pass form: what is stored is rounded, and so would be
// what the table's gradient sums (906 -> 843 us a step, error 1e-6 -> 0.0024).  Calls without
// that gradient take the same kernels, without the sums.
#include <algorithm>

#include "bwd_kernel.h"
#include "launch.h"
#include "rel.h"

namespace sigattn {
namespace {

template <typename T, int D, int WK, bool CAUSAL, int NW>
__global__ __launch_bounds__(64 * NW, 2) void rel_dq_kernel(const RelParams p) {
  __shared__ __attribute__((aligned(16))) DqLds<D, false, dq_window<RelParams, WK, NW>()> lds;
  __shared__ unsigned long long gap_lds[2];
  extern __shared__ __attribute__((aligned(16))) float near[];  // the waves' lines and pieces
  const int wg = gap_prologue<2>(p, gap_lds);
  if (wg >= 0) bwd_dq_body<T, D, WK, CAUSAL, false, RelParams, NW>(p, wg, lds, near);
}

template <typename T, int D, bool CAUSAL, bool GROUPED>
__global__ __launch_bounds__(256, (D <= 64 ? 2 : 1)) void rel_dkdv_kernel(const RelParams p) {
  __shared__ __attribute__((aligned(16))) DkdvLds<D, dkdv_window<RelParams>()> lds;
  bwd_dkdv_body<T, D, CAUSAL, false, false, GROUPED, RelParams>(p, blockIdx.x, lds);
}

template <typename T, int D, int WK, int NW = 4> void dq_w(const RelParams &kp, bool causal, hipStream_t st) {
  RelParams p = kp;
  p.part_rows = 32 * NW / WK;
  p.nblk = (p.Tq + p.part_rows - 1) / p.part_rows;
  const dim3 grid((unsigned)(p.nblk * p.B * p.H + p.ngap[0] + p.ngap[1]));
  const size_t line = p.part != nullptr ? near_floats(p.reach, NW) * sizeof(float) : 0;
  if (causal) rel_dq_kernel<T, D, WK, true, NW><<<grid, 64 * NW, line, st>>>(p);
  else rel_dq_kernel<T, D, WK, false, NW><<<grid, 64 * NW, line, st>>>(p);
}

// At D = 128 two workgroups of four waves share a CU as long as their sums' lines fit
// beside the tiles, up to a reach of 158.  Beyond, one of eight waves holds as many, in
// twice the queries per copied tile (up to 1190, then four alone).  dQ of the causal step of 3
// sequences of 1500 .. 4096 H=16 Hkv=4, us by reach: four waves 140 327, 150 308, 158 306;
// eight 160 327, 300 327, 1100 345, 1190 347; four alone 1200 515.
bool dq_eight_waves(const RelParams &p, int D) {
  constexpr size_t tiles = 4 * 64 * 128 * 2, cu = 163840 - 512;
  const size_t four = tiles + 2 * 192 * 4 + near_floats(p.reach, 4) * 4;
  const size_t eight = tiles + 2 * 320 * 4 + near_floats(p.reach, 8) * 4;
  return D == 128 && p.part != nullptr && 2 * four > cu && eight <= cu;
}

// Both kernels in one launch (D <= 64): the first nkv workgroups (after dQ's gap
// rows) are dK/dV's.
template <typename T, int D, int WK, bool CAUSAL, bool GROUPED>
__global__ __launch_bounds__(256, 2) void rel_bwd_kernel(const RelParams pq, const RelParams pk, int nkv) {
  using Dq = DqLds<D, false, dq_window<RelParams, WK>()>;
  using Dkdv = DkdvLds<D, dkdv_window<RelParams>()>;
  __shared__ unsigned long long gap_lds[2];
  extern __shared__ __attribute__((aligned(16))) float lds[];  // a Dkdv, or a Dq and its sums
  const int wg = gap_prologue<2>(pq, gap_lds);
  if (wg < 0) return;
  if (wg < nkv) bwd_dkdv_body<T, D, CAUSAL, false, false, GROUPED, RelParams>(pk, wg, *(Dkdv *)lds);
  else bwd_dq_body<T, D, WK, CAUSAL, false, RelParams>(pq, wg - nkv, *(Dq *)lds, lds + sizeof(Dq) / 4);
}

// Where that pays: as long as either kernel alone leaves CUs idle for much of its
// time, and two workgroups still fit a CU beside the sums' lines.  Captured steps
// (forward and backward, bf16, reach 128), us, two launches / one, by 128-row workgroups of
// both per CU: H=8 D=64 sequence of 128 0.06, 39.8 / 32.3; four of 512 1, 61 / 51 (causal
// 60 / 48); two of 1001 H=12 1.5, 96 / 85; eight of 512 2, 71 / 72; four of 1024 H=16 4, 150
// / 150 (causal 110 / 107); sixteen of 101 .. 1001 H=12 12, 235 / 233 (D=32 176 / 187;
// causal D=64 171 / 170, D=32 138 / 141); causal, eight of 2048 H=8 8, 266 / 292 (dQ misses
// its third workgroup per CU).
template <int D, int WK> size_t dq_lds(const RelParams &p) {
  return sizeof(DqLds<D, false, dq_window<RelParams, WK>()>) + (p.part != nullptr ? near_floats(p.reach) * 4 : 0);
}
template <int D, int WK> bool one_launch(const RelParams &p, bool causal) {
  const int64_t n = (int64_t)p.B * p.H * ((p.Tq + 127) / 128 + (p.Tk + 127) / 128);
  return n <= (causal ? 4 : 2) * (int64_t)p.ncu && dq_lds<D, WK>(p) <= 79 * 1024;
}

template <typename T, int D, int WK>
void bwd_w(const RelParams &kq, const RelParams &kk, bool causal, hipStream_t st) {
  RelParams pq = kq, pk = kk;
  pq.part_rows = 128 / WK;
  pq.nblk = (pq.Tq + pq.part_rows - 1) / pq.part_rows;
  pk.nblk = (pk.Tk + 127) / 128;
  const bool grouped = pk.qgroup > 1;
  const int nkv = pk.nblk * pk.B * pk.H * (grouped && pk.qsplit > 1 ? pk.qsplit : 1);
  const dim3 grid((unsigned)(nkv + pq.nblk * pq.B * pq.H + pq.ngap[0] + pq.ngap[1]));
  const size_t lds = std::max(dq_lds<D, WK>(pq), sizeof(DkdvLds<D, dkdv_window<RelParams>()>));
  const auto go = [&](auto c, auto g) {
    rel_bwd_kernel<T, D, WK, c.value, g.value><<<grid, 256, lds, st>>>(pq, pk, nkv);
  };
  if (causal) grouped ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
  else grouped ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
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

int rel_dq_rows(const RelParams &p, int D, bool causal) {
  return dq_pairs(p, D, causal) ? 64 : dq_eight_waves(p, D) ? 256 : 128;
}

void launch_rel_dq_mfma(const RelParams &p, int dtype, int D, bool causal, hipStream_t st) {
  by_type(dtype, D, [&](auto *t, auto d) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int DD = decltype(d)::value;
    if constexpr (DD <= 64) {
      if (dq_pairs(p, DD, causal)) return dq_w<T, DD, 2>(p, causal, st);
    } else if (dq_eight_waves(p, DD)) {
      return dq_w<T, DD, 1, 8>(p, causal, st);
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

bool launch_rel_bwd_mfma(const RelParams &pq, const RelParams &pk, int dtype, int D, bool causal, hipStream_t st) {
  bool done = false;
  by_type(dtype, D, [&](auto *t, auto d) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int DD = decltype(d)::value;
    if constexpr (DD <= 64) {
      const auto go = [&](auto wk) {
        if ((done = one_launch<DD, wk.value>(pq, causal))) bwd_w<T, DD, wk.value>(pq, pk, causal, st);
      };
      if (dq_pairs(pq, DD, causal)) go(std::integral_constant<int, 2>{});
      else go(std::integral_constant<int, 1>{});
    }
  });
  if (done) launch_add_parts(pk, dtype, st);
  return done;
}

}  // namespace sigattn
