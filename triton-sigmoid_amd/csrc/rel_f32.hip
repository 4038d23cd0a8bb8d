// The fp32 kernels (f32_kernel.h) with the learned bias by relative position, its
// windows of the lines beside the split tiles in LDS.  us, with / without: five sequences
// of 1 .. 777 H=8 D=32, reach 300, forward 25.5 / 23.6, dK/dV 34 / 31.3, dQ 35.5 / 27.2
// (30.5 without the sums by position); dQ and dK/dV in one launch 50 .. 58.
#include "f32_kernel.h"
#include "rel.h"

namespace sigattn {
namespace {

template <class F> void by_dim(int D, F &&f) {
  if (D == 128) f(std::integral_constant<int, 128>{});
  else if (D == 64) f(std::integral_constant<int, 64>{});
  else f(std::integral_constant<int, 32>{});
}

// Both kernels in one launch: the first nkv workgroups (after dQ's gap rows) are
// dK/dV's.  Captured steps (forward and backward), us, two launches / one: five sequences
// of 1 .. 777 H=8 D=32, reach 300, 110 / 101; one of 128 H=8 D=64 50 / 37; eight of 256 ..
// 1024 H=12 D=64 440 / 390; causal, eight of 512 .. 2048 H=16 Hkv=4 D=64 1266 / 1110; D=128
// H=8 Hkv=2, four of 250 .. 1000 484 / 438, causal, eight of 500 .. 2000 1328 / 1150.
template <int D, bool CAUSAL, int WK>
__global__ __launch_bounds__(64 * FW, (bwd_f32_occupancy<D, WK>())) void rel_bwd_f32_kernel(const RelParams pq,
                                                                                         const RelParams pk, int nkv) {
  __shared__ __attribute__((aligned(16))) float lds[window_floats<D, WK, RelParams>(0)];
  extern __shared__ __attribute__((aligned(16))) float near[];
  const int wg = gap_prologue<4>(pq, lds);
  if (wg < 0) return;
  if (wg < nkv) dkdv_f32_body<D, CAUSAL, false, WK, RelParams>(pk, wg, lds);
  else dq_f32_body<D, CAUSAL, false, WK, RelParams>(pq, wg - nkv, lds, near);
}

}  // namespace

void launch_rel_fwd_f32(const RelParams &p, int D, bool causal, hipStream_t st) {
  by_dim(D, [&](auto d) { fwd_t<d.value>(p, causal, st); });
}

int rel_dq_rows_f32(const RelParams &p, int D, bool causal) {
  int rows = 0;
  by_dim(D, [&](auto d) {
    by_waves<d.value>(p, p.Tq, p.Tk, causal, [&](auto wk, const RelParams &, int64_t) { rows = 32 * FW / wk.value; });
  });
  return rows;
}

void launch_rel_dq_f32(const RelParams &p, int D, bool causal, hipStream_t st) {
  by_dim(D, [&](auto d) { dq_t<d.value>(p, causal, st); });
}

void launch_rel_dkdv_f32(const RelParams &p, int D, bool causal, hipStream_t st) {
  RelParams k = p;
  k.part = nullptr;  // dQ's
  by_dim(D, [&](auto d) { dkdv_t<d.value>(k, causal, st); });
  launch_add_parts(p, kF32, st);
}

bool launch_rel_bwd_f32(const RelParams &kq, const RelParams &kk, int D, bool causal, hipStream_t st) {
  bool done = false;
  RelParams kv = kk;
  kv.part = nullptr;
  by_dim(D, [&](auto d) {
    by_waves<d.value>(kq, kq.Tq, kq.Tk, causal, [&](auto wq, const RelParams &pq, int64_t nq) {
      by_waves<d.value>(kv, kv.Tk, kv.Tq, causal, [&](auto wk, const RelParams &pk, int64_t nk) {
        if constexpr (wq.value == wk.value) {
          constexpr int WK = wk.value;
          const size_t near = rel_near_bytes(pq);
          const size_t tiles = window_floats<d.value, WK, RelParams>(0) * 4;
          if (bwd_f32_occupancy<d.value, WK>() * (tiles + near + 256) > 163840) return;
          const int64_t nkv = nk * (pk.qsplit > 1 ? pk.qsplit : 1);
          done = true;
          const dim3 grid((unsigned)(nq + nkv + pq.ngap[0] + pq.ngap[1])), block(64 * FW);
          if (causal) rel_bwd_f32_kernel<d.value, true, WK><<<grid, block, near, st>>>(pq, pk, (int)nkv);
          else rel_bwd_f32_kernel<d.value, false, WK><<<grid, block, near, st>>>(pq, pk, (int)nkv);
        }
      });
    });
  });
  if (done) launch_add_parts(kv, kF32, st);
  return done;
}

void launch_paged_rel_f32(const PagedRelParams &p, int units, int D, bool causal, hipStream_t st) {
  by_dim(D, [&](auto d) { paged_t<d.value>(p, units, causal, st); });
}

void launch_paged_rel_decode_f32(const PagedRelParams &p, int units, int D, bool causal, hipStream_t st) {
  by_dim(D, [&](auto d) { paged_decode_t<d.value>(p, units, causal, st); });
}

}  // namespace sigattn
