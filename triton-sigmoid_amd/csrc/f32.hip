// Launches of the fp32 kernels (f32_kernel.h).
#include "f32_kernel.h"
#include "launch.h"

namespace sigattn {

void launch_paged_decode_f32(const PagedParams &p, int units, int D, bool causal, hipStream_t st) {
  if (D == 128) paged_decode_t<128>(p, units, causal, st);
  else if (D == 64) paged_decode_t<64>(p, units, causal, st);
  else paged_decode_t<32>(p, units, causal, st);
}

void launch_paged_f32(const PagedParams &p, int units, int D, bool causal, hipStream_t st) {
  if (D == 128) paged_t<128>(p, units, causal, st);
  else if (D == 64) paged_t<64>(p, units, causal, st);
  else paged_t<32>(p, units, causal, st);
}

void launch_fwd_f32(const KParams &p, int D, bool causal, bool, hipStream_t st) {
  if (D == 128) fwd_t<128>(p, causal, st);
  else if (D == 64) fwd_t<64>(p, causal, st);
  else fwd_t<32>(p, causal, st);
}

void launch_bwd_dq_f32(const KParams &p, int D, bool causal, bool, hipStream_t st) {
  if (D == 128) dq_t<128>(p, causal, st);
  else if (D == 64) dq_t<64>(p, causal, st);
  else dq_t<32>(p, causal, st);
}

void launch_bwd_dkdv_f32(const KParams &p, int D, bool causal, bool, hipStream_t st) {
  if (D == 128) dkdv_t<128>(p, causal, st);
  else if (D == 64) dkdv_t<64>(p, causal, st);
  else dkdv_t<32>(p, causal, st);
  launch_add_parts(p, kF32, st);
}

}  // namespace sigattn
