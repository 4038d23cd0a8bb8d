// Paged key/value cache: its bookkeeping, its writer, and the portable
// attention kernel (any type; tensors off 16-byte boundaries).
//
// The entry points of include/sigattn.h for the paged cache are here and in
// paged_capi.cpp; none allocates, synchronises the host or throws.
#include <hip/hip_runtime.h>

#include "../../include/sigattn.h"
#include "launch.h"
#include "paged.h"
#include "rel.h"

namespace sigattn {
namespace {

// ---- the plan of a serving step ---------------------------------------------
// need_b = ceil((c_b + n_b) / ps) - ceil(c_b / ps) pages, taken from the free
// list at the exclusive sum of the needs before b; slot of token i of request b
// at position x = c_b + i: page(x / ps) * ps + x % ps.
//
// Every workgroup sums the B lengths itself (LDS prefix arrays, B <=
// kPlanMaxBatch) and then fills its share of the table entries and of the
// slots, each found by a binary search in the sums: one launch, where a scan
// kernel followed by a fill kernel would be two.  Bound by the chain of loads, sums
// and searches of one workgroup: 3.3 us for 64 requests of a token each, 4.9 us
// for 320 with 64 prompts of up to 1999 tokens (7 us a call from the host).
constexpr int kPlanThreads = 256;

// Exclusive sums of a and b over the workgroup's threads; *_total gets the sums.
__device__ __forceinline__ void scan2(int &a, int &b, int &a_total, int &b_total) {
  __shared__ int wa[kPlanThreads / 64], wb[kPlanThreads / 64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int x = a, y = b;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int u = __shfl_up(x, d), v = __shfl_up(y, d);
    if (lane >= d) x += u, y += v;
  }
  if (lane == 63) wa[w] = x, wb[w] = y;
  __syncthreads();
  int xa = 0, yb = 0;
  a_total = b_total = 0;
#pragma unroll
  for (int i = 0; i < kPlanThreads / 64; ++i) {
    if (i < w) xa += wa[i], yb += wb[i];
    a_total += wa[i], b_total += wb[i];
  }
  a = xa + x - a, b = yb + y - b;
}

struct PlanArgs {
  const int32_t *ctx, *add, *free_pages;
  int32_t *table, *slots, *cu, *lens, *needed;
  int64_t table_stride;
  int B, max_pages, num_free, lp, num_tokens;
};

__device__ __forceinline__ int plan_len(const int32_t *p, int b) { return max(p[b], 0); }

__global__ __launch_bounds__(kPlanThreads) void plan_kernel(const PlanArgs a) {
  extern __shared__ int sums[];  // first token, then first free page, of each request and the end
  int *tok = sums, *page = sums + a.B + 1;
  const int tid = threadIdx.x, ps1 = (1 << a.lp) - 1;
  const auto pages = [&](int64_t tokens) { return (int)((tokens + ps1) >> a.lp); };
  // Each thread sums the requests of one contiguous piece.
  const int per = (a.B + kPlanThreads - 1) / kPlanThreads, b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
  int nt = 0, np = 0, all_t, all_p;
  for (int b = b0; b < b1; ++b) {
    const int c = plan_len(a.ctx, b), n = plan_len(a.add, b);
    nt += n, np += pages((int64_t)c + n) - pages(c);
  }
  scan2(nt, np, all_t, all_p);
  for (int b = b0; b < b1; ++b) {
    const int c = plan_len(a.ctx, b), n = plan_len(a.add, b);
    tok[b] = nt, page[b] = np;
    if (blockIdx.x == 0) a.cu[b] = nt, a.lens[b] = c + n;
    nt += n, np += pages((int64_t)c + n) - pages(c);
  }
  if (tid == 0) {
    tok[a.B] = all_t, page[a.B] = all_p;
    if (blockIdx.x == 0) a.cu[a.B] = all_t, *a.needed = all_p;
  }
  __syncthreads();
  // The request that owns item i of the sums s: the last b with s[b] <= i.
  const auto owner = [&](const int *s, int i) {
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  };
  const auto fresh = [&](int64_t i) { return i >= 0 && i < a.num_free ? a.free_pages[i] : -1; };
  // (Positions and the loops' counters in 64 bits: lengths whose sums do not fit
  // 32 give a useless plan, but an end and no access outside the tensors.)
  const int step = gridDim.x * kPlanThreads;
  for (int64_t i = blockIdx.x * kPlanThreads + tid; i < all_p; i += step) {
    const int b = owner(page, (int)i);
    const int64_t j = pages(plan_len(a.ctx, b)) + i - page[b];
    if (j >= 0 && j < a.max_pages) a.table[b * a.table_stride + j] = fresh(i);
  }
  for (int t = blockIdx.x * kPlanThreads + tid; t < a.num_tokens; t += step) {
    int slot = -1;
    if (t < all_t) {
      const int b = owner(tok, t), c = plan_len(a.ctx, b), held = pages(c);
      const int64_t x = (int64_t)c + t - tok[b], j = x >> a.lp;
      if (j >= 0 && j < a.max_pages) {
        // Pages of this step come from the free list itself: their table
        // entries may be another workgroup's to write.
        const int id = j < held ? a.table[b * a.table_stride + j] : fresh(page[b] + j - held);
        if (id >= 0 && id <= INT32_MAX >> a.lp) slot = (id << a.lp) | (int)(x & ps1);
      }
    }
    a.slots[t] = slot;
  }
}

// ---- the writer ---------------------------------------------------------------
// Moves each row in 16-byte pieces (PIECE = 16; 2-byte ones where something
// is not 16-byte aligned), K and V in one launch, a piece a thread: neighbouring
// threads have neighbouring pieces, and the slot is read again from the cache.
// Bound by memory: 16384 rows H_kv=8 D=64 f16 (67 MB) 12 us, 5.5 TB/s; a row for
// each of 64 requests 2.4 us.
struct WriteArgs {
  const char *src[2];
  char *dst[2];
  const int32_t *slots;
  int64_t pieces;  // rows * heads * pieces of a head
  int64_t src_t, src_h, dst_p, dst_t, dst_h;  // bytes
  int64_t num_slots;
  int heads, lp, ld;  // log2 of the pieces of a head's row
};

template <typename Piece>
__global__ __launch_bounds__(256) void write_kernel(const WriteArgs a) {
  const char *src = a.src[blockIdx.y];
  char *dst = a.dst[blockIdx.y];
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.pieces; i += step) {
    const int64_t c = i & ((1 << a.ld) - 1), rh = i >> a.ld;
    const int64_t t = rh / a.heads;
    const int h = (int)(rh - t * a.heads);
    const int32_t slot = a.slots[t];
    if (slot < 0 || slot >= a.num_slots) continue;
    const int64_t at = (int64_t)(slot >> a.lp) * a.dst_p + (slot & ((1 << a.lp) - 1)) * a.dst_t + h * a.dst_h;
    *(Piece *)(dst + at + c * sizeof(Piece)) = *(const Piece *)(src + t * a.src_t + h * a.src_h + c * sizeof(Piece));
  }
}

// ---- portable attention ---------------------------------------------------------
template <typename T> __device__ __forceinline__ float ld_elem(const void *base, int64_t i) {
  if constexpr (sizeof(T) == 4) return ((const float *)base)[i];
  else return Elem<T>::to_f32(((const uint16_t *)base)[i]);
}
template <typename T> __device__ __forceinline__ void st_elem(void *base, int64_t i, float x) {
  if constexpr (sizeof(T) == 4) ((float *)base)[i] = x;
  else ((uint16_t *)base)[i] = Elem<T>::from_f32(x);
}

// One workgroup per packed query row and query head; 256 keys at a time: each
// thread the score of one key, then (column d, share of the keys) per thread
// for P·V.  Any dtype, alignment and strides.  Bound by its scalar loads (each
// thread walks a row of its own): 4 sequences of 2000 keys H=32 Hkv=8 D=128, 1 /
// 16 tokens each, bf16 342 / 631 us, fp32 327 / 547, where aligned rows (the matrix
// kernels) take 16 / 30 and 24 / 53.
template <typename T, int D, bool CAUSAL, class P>
__global__ __launch_bounds__(256) void paged_generic_kernel(const P p) {
  constexpr int PARTS = 256 / D;
  __shared__ float sq[D], sp[256], red[256];
  __shared__ int64_t srow[256];  // element offset of each key's row; -1: no key there
  const int tid = threadIdx.x, h = blockIdx.y;
  const int64_t r = blockIdx.x;
  // The sequence of row r: the last b with cu[b] <= r, if it covers r.
  int lo = 0, hi = p.B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (packed_first(p.cu_q, p.rows_q, mid) <= r) lo = mid;
    else hi = mid - 1;
  }
  const int b = lo;
  const int64_t first = packed_first(p.cu_q, p.rows_q, b);
  const int Lq = packed_len(p.cu_q, p.rows_q, b, p.Tq);
  const bool covered = r >= first && r < first + Lq;
  const int Lk = covered ? p.keys(b) : 0;
  const int end = CAUSAL ? min(Lk, Lk - Lq + (int)(r - first) + 1) : Lk;
  const int64_t qoff = r * p.sq_t + (int64_t)h * p.sq_h;
  if (tid < D) sq[tid] = covered ? ld_elem<T>(p.q, qoff + tid) : 0.0f;
  const float bias = end > 0 ? p.bias_of(Lk) : 0.0f;
  const int64_t head = (int64_t)(h / p.G) * p.sk_h;
  float acc = 0.0f;
  for (int k0 = 0; k0 < end; k0 += 256) {
    __syncthreads();
    const int key = k0 + tid;
    float pr = 0.0f;
    int64_t row = -1;
    if (key < end) {
      const int id = p.table[b * p.table_stride + (key >> p.lp)];
      if (id >= 0 && id < p.num_pages) {
        row = id * p.sk_p + (int64_t)(key & ((1 << p.lp) - 1)) * p.sk_t + head;
        float s = 0.0f;
#pragma unroll 8
        for (int d = 0; d < D; ++d) s = __builtin_fmaf(sq[d], ld_elem<T>(p.k, row + d), s);
        float c = bias + (p.score_mod ? p.score_mod[b * p.mod_stride + key] : 0.0f);
        if constexpr (P::kRel) c = bias + rel_at(p, h, key - (Lk - Lq + (int)(r - first)));
        constexpr int PB = p_bits<T, P>();
        pr = round_to<T>(sigmoid_times_2<PB>(-__builtin_fmaf(s, p.fscale, c) * kLog2e)) * (1.0f / (1 << PB));
      }
    }
    sp[tid] = pr;
    srow[tid] = row;
    __syncthreads();
    const int n = min(256, end - k0), d = tid % D;
#pragma unroll 4
    for (int j = tid / D; j < n; j += PARTS)
      if (srow[j] >= 0) acc = __builtin_fmaf(sp[j], ld_elem<T>(p.v, srow[j] + d), acc);
  }
  __syncthreads();
  red[tid] = acc;
  __syncthreads();
  if (tid < D) {
#pragma unroll
    for (int x = 1; x < PARTS; ++x) acc += red[x * D + tid];
    st_elem<T>(p.out, (r * p.H + h) * D + tid, acc);
  }
}

template <typename T, int D, class P> void generic_t(const P &p, bool causal, hipStream_t st) {
  const dim3 grid((unsigned)p.rows_q, (unsigned)p.H);
  if (causal) paged_generic_kernel<T, D, true, P><<<grid, 256, 0, st>>>(p);
  else paged_generic_kernel<T, D, false, P><<<grid, 256, 0, st>>>(p);
}
template <typename T, class P> void generic_d(const P &p, int D, bool causal, hipStream_t st) {
  switch (D) {
    case 16: return generic_t<T, 16>(p, causal, st);
    case 32: return generic_t<T, 32>(p, causal, st);
    case 64: return generic_t<T, 64>(p, causal, st);
    default: return generic_t<T, 128>(p, causal, st);
  }
}
template <class P> void generic(const P &p, int dtype, int D, bool causal, hipStream_t st) {
  if (dtype == kF32) generic_d<float>(p, D, causal, st);
  else if (dtype == kBF16) generic_d<__bf16>(p, D, causal, st);
  else generic_d<_Float16>(p, D, causal, st);
}

int log2_of(int64_t x) { return 63 - __builtin_clzll((unsigned long long)x); }

int status_of_launch() { return hipGetLastError() == hipSuccess ? SIGATTN_OK : SIGATTN_ERR_LAUNCH; }

bool page_size_ok(int64_t ps) { return ps >= 16 && ps <= (1 << 20) && (ps & (ps - 1)) == 0; }

}  // namespace

void launch_paged_generic(const PagedParams &p, int dtype, int D, bool causal, hipStream_t st) {
  generic(p, dtype, D, causal, st);
}
void launch_paged_rel_generic(const PagedRelParams &p, int dtype, int D, bool causal, hipStream_t st) {
  generic(p, dtype, D, causal, st);
}

}  // namespace sigattn

using namespace sigattn;

extern "C" int sigattn_paged_plan(int64_t B, const int32_t *context_lens, const int32_t *new_lens,
                                  int32_t *block_table, int64_t table_stride, int64_t max_pages,
                                  const int32_t *free_pages, int64_t num_free, int64_t page_size, int64_t num_tokens,
                                  int32_t *slot_mapping, int32_t *cu_seqlens, int32_t *seq_lens,
                                  int32_t *pages_needed, void *stream) {
  if (B < 0 || B > SIGATTN_PLAN_MAX_BATCH || max_pages < 0 || max_pages > INT32_MAX || num_free < 0 ||
      num_free > INT32_MAX || num_tokens < 0 || num_tokens > INT32_MAX / 2 || !page_size_ok(page_size) ||
      (B > 0 && max_pages > INT32_MAX / page_size))
    return SIGATTN_ERR_SHAPE;
  if (table_stride < 0) return SIGATTN_ERR_STRIDE;
  if (cu_seqlens == nullptr || pages_needed == nullptr || (num_tokens > 0 && slot_mapping == nullptr) ||
      (B > 0 && (context_lens == nullptr || new_lens == nullptr || seq_lens == nullptr)) ||
      (B > 0 && max_pages > 0 && block_table == nullptr) || (num_free > 0 && free_pages == nullptr))
    return SIGATTN_ERR_NULL_ARG;
  PlanArgs a{};
  a.ctx = context_lens, a.add = new_lens, a.free_pages = free_pages;
  a.table = block_table, a.slots = slot_mapping, a.cu = cu_seqlens, a.lens = seq_lens, a.needed = pages_needed;
  a.table_stride = table_stride;
  a.B = (int)B, a.max_pages = (int)max_pages, a.num_free = (int)num_free, a.lp = log2_of(page_size);
  a.num_tokens = (int)num_tokens;
  // A workgroup for every 256 tokens, a thread each: every workgroup repeats the
  // sums, and a token costs a search (1024 tokens a workgroup: 7.6 us for 320
  // requests of 65000 tokens).
  const int64_t want = (num_tokens + 255) / 256, grid = want < 1 ? 1 : (want > 1024 ? 1024 : want);
  (void)hipGetLastError();
  plan_kernel<<<dim3((unsigned)grid), dim3(kPlanThreads), 2 * (B + 1) * sizeof(int), (hipStream_t)stream>>>(a);
  return status_of_launch();
}

extern "C" int sigattn_paged_write(const sigattn_paged_rows *r, void *stream) {
  if (r == nullptr) return SIGATTN_ERR_NULL_ARG;
  if (r->esize != 2 && r->esize != 4) return SIGATTN_ERR_DTYPE;
  if (r->D != 16 && r->D != 32 && r->D != 64 && r->D != 128) return SIGATTN_ERR_HEAD_DIM;
  // (rows * kv_heads * pieces of a row fit 63 bits.)
  if (r->rows < 0 || r->kv_heads < 0 || r->num_pages < 0 || r->rows > INT32_MAX / 2 || r->kv_heads > 65535 ||
      !page_size_ok(r->page_size) || r->num_pages > INT32_MAX / r->page_size)
    return SIGATTN_ERR_SHAPE;
  const int64_t strides[5] = {r->src_stride_t, r->src_stride_h, r->cache_stride_p, r->cache_stride_t,
                              r->cache_stride_h};
  for (int64_t s : strides)
    if (s < 0) return SIGATTN_ERR_STRIDE;
  if (r->rows == 0 || r->kv_heads == 0 || r->num_pages == 0) return SIGATTN_OK;
  if (r->k == nullptr || r->v == nullptr || r->k_cache == nullptr || r->v_cache == nullptr ||
      r->slot_mapping == nullptr)
    return SIGATTN_ERR_NULL_ARG;
  WriteArgs a{};
  a.src[0] = (const char *)r->k, a.src[1] = (const char *)r->v;
  a.dst[0] = (char *)r->k_cache, a.dst[1] = (char *)r->v_cache;
  a.slots = r->slot_mapping;
  a.src_t = r->src_stride_t * r->esize, a.src_h = r->src_stride_h * r->esize;
  a.dst_p = r->cache_stride_p * r->esize, a.dst_t = r->cache_stride_t * r->esize;
  a.dst_h = r->cache_stride_h * r->esize;
  a.num_slots = r->num_pages * r->page_size;
  a.heads = (int)r->kv_heads, a.lp = log2_of(r->page_size);
  uint64_t bits = (uintptr_t)r->k | (uintptr_t)r->v | (uintptr_t)r->k_cache | (uintptr_t)r->v_cache;
  bits |= (uint64_t)(a.src_t | a.src_h | a.dst_p | a.dst_t | a.dst_h);
  const bool wide = (bits & 15) == 0;
  a.ld = log2_of(r->D * r->esize / (wide ? 16 : 2));
  a.pieces = (r->rows * r->kv_heads) << a.ld;
  const int64_t groups = (a.pieces + 255) / 256;
  const dim3 grid((unsigned)(groups < (1 << 20) ? groups : 1 << 20), 2);
  (void)hipGetLastError();
  if (wide) write_kernel<u32x4><<<grid, dim3(256), 0, (hipStream_t)stream>>>(a);
  else write_kernel<uint16_t><<<grid, dim3(256), 0, (hipStream_t)stream>>>(a);
  return status_of_launch();
}
