// The matrix kernels over a paged cache with the learned bias by relative position.
// Each lane reads what its column (a query head's token) adds (RelColumn): a
// block's columns are of several heads, whose windows in LDS would be as many.  A block
// of keys beyond the line's end for every column costs a comparison: the kernel, us, with /
// without, 16 requests on 1024 .. 8191 H=32 Hkv=8 D=128 43.3 / 42.4, bound by HBM; 24
// requests, four of them prompts, H=12 Hkv=4 D=64 40.1 / 37.1; the call, two chunks of 1024
// on 5000 .. 12000 H=32 Hkv=8 D=128 351 / 312, where the columns' 32 registers leave the
// products' operands a read-ahead of 8 instead of 16.  (fp32, f32_kernel.h, the same calls: 96 /
// 90, 179 / 175, 2605 / 2578.)
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

void launch_paged_rel_mixed(const PagedRelParams &pf, int nf, const PagedRelParams &pd, int nd, int dtype, int D,
                            bool causal, hipStream_t st) {
  by_type16(dtype, D, [&](auto *t, auto d) {
    mixed_t<std::remove_pointer_t<decltype(t)>, decltype(d)::value>(pf, nf, pd, nd, causal, st);
  });
}

}  // namespace sigattn
