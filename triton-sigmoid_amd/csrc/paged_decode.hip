// Launches of the decoding kernel (paged_decode.h).
#include "launch.h"
#include "paged_launch.h"

namespace sigattn {

void launch_paged_decode(const PagedParams &p, int units, int dtype, int D, bool causal, hipStream_t st) {
  by_type(dtype, D, [&](auto *t, auto d) {
    using T = std::remove_pointer_t<decltype(t)>;
    if constexpr (sizeof(T) == 2) decode_t<T, decltype(d)::value>(p, units, causal, st);
  });
}

}  // namespace sigattn
