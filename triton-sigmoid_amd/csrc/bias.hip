// The default bias of ragged batches, -log(key length of each sequence) in
// fp32 (sigmoid_triton_padded.py:995-996), from the lengths on the device.
// Launch-bound: one launch in place of the conversion, logarithm and negation
// (and the difference of packed offsets) as element-wise operators, each of
// which costs the stream about 4.5 us at these sizes, more than a tenth of a
// decoding step.  Built with -ffp-contract=off: the logarithm's bits are then
// the element-wise operator's (with contraction 38 % of the first million
// lengths differ in the last bit).  The learned bias by relative position takes it
// from the launch that makes its lines.
#include <hip/hip_runtime.h>

#include "../../include/sigattn.h"
#include "launch.h"
#include "rel.h"

namespace {
__device__ __forceinline__ float default_bias(const int32_t *lens, const int32_t *cu, int64_t b) {
  // Offsets differ as the int32 tensors would (modulo 2^32).
  const int32_t n = lens != nullptr ? lens[b] : (int32_t)((uint32_t)cu[b + 1] - (uint32_t)cu[b]);
  return -logf((float)n);
}

__global__ __launch_bounds__(256) void default_bias_kernel(const int32_t *lens, const int32_t *cu, int64_t B,
                                                           float *bias) {
  const int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (b < B) bias[b] = default_bias(lens, cu, b);
}

// One thread per place, then (head 0) one per sequence.  A few KB: bound by its launch,
// 2.5 us, and one launch less is 2.5 us more (forward of 128 tokens H=8 D=64 15.2 us
// with a launch for the default bias).
template <typename T>
__global__ __launch_bounds__(256) void rel_line_kernel(const sigattn::RelTable t, float *line, int blocks,
                                                       const int32_t *cu, int64_t B, float *bias) {
  using namespace sigattn;
  if ((int)blockIdx.x >= blocks) {
    const int64_t b = (int64_t)((int)blockIdx.x - blocks) * 256 + threadIdx.x;
    if (blockIdx.y == 0 && b < B) bias[b] = default_bias(nullptr, cu, b);
    return;
  }
  const int place = blockIdx.x * 256 + threadIdx.x, places = line_places(t.reach), h = blockIdx.y;
  if (place >= places) return;
  const int u = bucket_of(t, min(max(place - kRelPad, 0), 2 * t.reach));
  float x = 0.0f;
  if (u >= 0 && u < t.buckets) {  // (buckets outside the table add nothing and get nothing)
    const int64_t at = (int64_t)u * t.H + h;
    if constexpr (sizeof(T) == 4) x = ((const float *)t.table)[at];
    else x = Elem<T>::to_f32(((const uint16_t *)t.table)[at]);
  }
  line[(int64_t)h * places + place] = x;
}
}  // namespace

namespace sigattn {
void launch_rel_line(const RelTable &t, float *line, const int32_t *cu_k, int64_t B, float *bias, hipStream_t st) {
  if (t.H == 0) return;
  const int blocks = (line_places(t.reach) + 255) / 256;
  const dim3 grid((unsigned)(blocks + (bias != nullptr ? (B + 255) / 256 : 0)), (unsigned)t.H);
  const auto go = [&](auto *x) {
    rel_line_kernel<std::remove_pointer_t<decltype(x)>><<<grid, dim3(256), 0, st>>>(t, line, blocks, cu_k, B, bias);
  };
  if (t.dtype == kF32) go((float *)nullptr);
  else if (t.dtype == kBF16) go((__bf16 *)nullptr);
  else go((_Float16 *)nullptr);
}
}  // namespace sigattn

extern "C" int sigattn_default_bias(const int32_t *seq_lens, const int32_t *cu_seqlens, int64_t B, float *bias,
                                    void *stream) {
  if (B < 0 || (B + 255) / 256 > INT32_MAX) return SIGATTN_ERR_SHAPE;
  if (B == 0) return SIGATTN_OK;
  if (bias == nullptr || (seq_lens == nullptr && cu_seqlens == nullptr)) return SIGATTN_ERR_NULL_ARG;
  if (seq_lens != nullptr && cu_seqlens != nullptr) return SIGATTN_ERR_LAYOUT;
  (void)hipGetLastError();
  default_bias_kernel<<<dim3((unsigned)((B + 255) / 256)), dim3(256), 0, (hipStream_t)stream>>>(seq_lens, cu_seqlens,
                                                                                               B, bias);
  return hipGetLastError() == hipSuccess ? SIGATTN_OK : SIGATTN_ERR_LAUNCH;
}
