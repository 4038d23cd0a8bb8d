// The gradient of the learned bias's table from the dQ kernels' sums by relative
// position (the lines of values that the kernels read: bias.hip).
#include "launch.h"
#include "rel.h"

namespace sigattn {
namespace {

// sums[h][place] of all query blocks: 64 places a workgroup, 16 shares of the
// slots (in turn), added in their order; 5 to 6 us, a few rounds of loads.  Which slots hold a block is found for
// 1024 of them at a time, a thread each, from the batches' first slots in LDS
// (kFirst of them; a larger batch's come from its offsets).
constexpr int kShares = 16, kFirst = 1024;
__global__ __launch_bounds__(64 * kShares) void rel_sums_kernel(const RelParams p, float *sums) {
  __shared__ float got[kShares][64];
  __shared__ bool held[64 * kShares];
  __shared__ int64_t first[kFirst];
  const int h = blockIdx.y, lane = threadIdx.x & 63, share = threadIdx.x >> 6, places = p.places();
  const int place = blockIdx.x * 64 + lane;
  const int64_t slots = p.part != nullptr ? p.part_slots() : 0;
  const bool kept = p.B <= kFirst;
  if (kept && (int)threadIdx.x < p.B) first[threadIdx.x] = p.first_slot(threadIdx.x);
  __syncthreads();
  const auto first_slot = [&](int b) SIGATTN_INLINE { return kept ? first[b] : p.first_slot(b); };
  float x = 0.0f;
  for (int64_t s0 = 0; s0 < slots; s0 += 64 * kShares) {
    const int64_t mine = s0 + threadIdx.x;
    int lo = 0, hi = p.B - 1;  // the last batch that begins at or before the slot
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first_slot(mid) <= mine) lo = mid;
      else hi = mid - 1;
    }
    const int64_t blk = mine - first_slot(lo);
    __syncthreads();
    held[threadIdx.x] = blk >= 0 && blk * p.part_rows < p.len_q(lo);
    __syncthreads();
    const int n = (int)(slots - s0 < 64 * kShares ? slots - s0 : 64 * kShares);
    if (place < places)
#pragma unroll 4
      for (int i = share; i < n; i += kShares)
        if (held[i]) x += p.part[((s0 + i) * p.H + h) * places + place];
  }
  got[share][lane] = x;
  __syncthreads();
  if (share != 0 || place >= places) return;
#pragma unroll
  for (int s = 1; s < kShares; ++s) x += got[s][lane];
  sums[(int64_t)h * places + place] = x;
}

// grad[u][h] = the sum over the places of bucket u.  A workgroup per head keeps the
// sums and their buckets in LDS (5 us; both kernels in one, a workgroup per head,
// took as long as the two); a wave per bucket, its lanes' places added in order
// and the lanes' sums by wave_sum.
constexpr int kGradWaves = 16;
template <typename T>
__global__ __launch_bounds__(64 * kGradWaves) void rel_grad_kernel(const RelTable t, const float *sums, T *grad) {
  extern __shared__ float row[];  // [places] sums, then their buckets
  const int h = blockIdx.x, places = 2 * t.reach + 1, lane = threadIdx.x & 63;
  int *bucket = (int *)row + places;
  for (int i = threadIdx.x; i < places; i += 64 * kGradWaves)
    row[i] = sums[(int64_t)h * places + i], bucket[i] = bucket_of(t, i);
  __syncthreads();
  for (int u = threadIdx.x >> 6; u < t.buckets; u += kGradWaves) {
    float x = 0.0f;
    for (int i = lane; i < places; i += 64) x += bucket[i] == u ? row[i] : 0.0f;
    x = wave_sum(x);
    if (lane != 0) continue;
    if constexpr (sizeof(T) == 4) grad[(int64_t)u * t.H + h] = x;
    else ((uint16_t *)grad)[(int64_t)u * t.H + h] = Elem<T>::from_f32(x);
  }
}

template <class F> void by_type(int dtype, F &&f) {
  if (dtype == kF32) f((float *)nullptr);
  else if (dtype == kBF16) f((__bf16 *)nullptr);
  else f((_Float16 *)nullptr);
}

}  // namespace

void launch_rel_grad(const RelTable &t, const RelParams &p, float *sums, void *grad, hipStream_t st) {
  if (t.H == 0 || t.buckets == 0) return;
  const dim3 grid((unsigned)((p.places() + 63) / 64), (unsigned)t.H);
  rel_sums_kernel<<<grid, dim3(64 * kShares), 0, st>>>(p, sums);
  by_type(t.dtype, [&](auto *x) {
    using T = std::remove_pointer_t<decltype(x)>;
    rel_grad_kernel<T><<<dim3((unsigned)t.H), dim3(64 * kGradWaves), 8 * p.places(), st>>>(t, sums, (T *)grad);
  });
}

}  // namespace sigattn
