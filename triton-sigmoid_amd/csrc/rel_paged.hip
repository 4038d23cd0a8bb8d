// The matrix kernels over a paged cache with the learned bias by relative position.
#include "launch.h"
#include "paged_launch.h"
#include "rel.h"

namespace sigattn {
namespace {

template <class F> void by_type16(int dtype, int D, F &&f) {
  by_type(dtype, D, [&](auto *t, auto d) {
    using T = std::remove_pointer_t<decltype(t)>;
    if constexpr (sizeof(T) == 2) f(t, d);
  });
}

}  // namespace

void launch_paged_rel_fwd(const PagedRelParams &p, int units, int dtype, int D, bool causal, hipStream_t st) {
  by_type16(dtype, D, [&](auto *t, auto d) {
    fwd_t<std::remove_pointer_t<decltype(t)>, decltype(d)::value>(p, units, causal, st);
  });
}

void launch_paged_rel_decode(const PagedRelParams &p, int units, int dtype, int D, bool causal, hipStream_t st) {
  by_type16(dtype, D, [&](auto *t, auto d) {
    decode_t<std::remove_pointer_t<decltype(t)>, decltype(d)::value>(p, units, causal, st);
  });
}

void launch_paged_rel_mixed(const PagedRelParams &pf, int nf, const PagedRelParams &pd, int nd, int dtype, int D, bool causal,
                            hipStream_t st) {
  by_type16(dtype, D, [&](auto *t, auto d) {
    mixed_t<std::remove_pointer_t<decltype(t)>, decltype(d)::value>(pf, nf, pd, nd, causal, st);
  });
}

}  // namespace sigattn
