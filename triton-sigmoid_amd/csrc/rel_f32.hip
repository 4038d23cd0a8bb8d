// The fp32 kernels (f32_kernel.h) with the learned bias by relative position.
#include "f32_kernel.h"
#include "rel.h"

namespace sigattn {
namespace {

template <class F> void by_dim(int D, F &&f) {
  if (D == 128) f(std::integral_constant<int, 128>{});
  else if (D == 64) f(std::integral_constant<int, 64>{});
  else f(std::integral_constant<int, 32>{});
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

void launch_paged_rel_f32(const PagedRelParams &p, int units, int D, bool causal, hipStream_t st) {
  by_dim(D, [&](auto d) { paged_t<d.value>(p, units, causal, st); });
}

void launch_paged_rel_decode_f32(const PagedRelParams &p, int units, int D, bool causal, hipStream_t st) {
  by_dim(D, [&](auto d) { paged_decode_t<d.value>(p, units, causal, st); });
}

}  // namespace sigattn
