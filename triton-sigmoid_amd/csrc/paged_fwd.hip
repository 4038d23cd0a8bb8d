// Attention over a paged cache: prompts and chunks of them, and the sums of
// sequences whose keys were cut.
//
// The kernel is the forward's (fwd_kernel.h) on PagedParams: its tiles come
// through the block table, its columns are tokens times the query heads of a
// K / V head, and a unit's keys may be a chunk of the sequence's, whose fp32
// sums the reduction adds in chunk order (sigmoid attention has no row
// normalisation, so O is the plain sum over the chunks).
// Bound by its products and sigmoids as the forward is: 2 x 1024 tokens on 5000 ..
// 12000 keys bf16 H=32 Hkv=8 D=128 319 us, 1.02 PFLOP/s (matrix cores busy 48 % of
// the time; HBM 0.36 TB/s, a group's heads and its blocks share what L2 holds).
#include "launch.h"
#include "paged_launch.h"

namespace sigattn {
namespace {

// Output rows (token, query head) of cut sequences: the sum of the chunks'
// partials in chunk order.  CG threads add CG * 4 columns of one row.  Many rows
// (ROWS): CG = D / 4, and every group of a workgroup takes a row of its own.
// Few rows: CG = 8, a workgroup has 32 columns of a row, each of its 32 groups a
// share of the chunks, whose sums are added in group order -- one or two loads
// deep where a sequence has tens of chunks (B=1, 256 chunks, 16 rows D=128: 6.1 us
// with a workgroup per row).  Bound by its start and its chain of loads: 4.4 us
// there, 6.9 us for 512 rows of about 8 parts and for 21120 at D=64 (13 MB).  (Offsets,
// lengths and cuts held by the lanes and found by shuffles: no faster, the first
// 5 % slower.)
struct ReduceArgs {
  PagedParams p;
  const float *ws[2];   // blocks of more than / up to `cols` columns
  const int2 *cut[2];   // nullptr: no sequence was cut there
  int block[2], units[2], cols;
};

template <typename T, int D, bool ROWS>
__global__ __launch_bounds__(256) void paged_reduce_kernel(const ReduceArgs a) {
  constexpr int CG = ROWS ? D / 4 : 8, NG = 256 / CG;
  __shared__ f32x4 part[ROWS ? 1 : NG][CG];
  const PagedParams &p = a.p;
  const int g = threadIdx.x / CG, c = threadIdx.x % CG + (ROWS ? 0 : CG * (int)(blockIdx.x % (D / 32)));
  const int64_t item = ROWS ? (int64_t)blockIdx.x * NG + g : (int64_t)(blockIdx.x / (D / 32));
  const int64_t r = item / p.H;
  const int h = (int)(item - r * p.H);
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  int nck = 0;
  if (r < p.rows_q) {
    int lo = 0, hi = p.B - 1;  // the last sequence that begins at or before row r
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (packed_first(p.cu_q, p.rows_q, mid) <= r) lo = mid;
      else hi = mid - 1;
    }
    const int64_t tok = r - packed_first(p.cu_q, p.rows_q, lo);
    const int Lq = p.len_q(lo), few = Lq * p.G <= a.cols;
    if (tok >= 0 && tok < Lq && a.cut[few] != nullptr) {
      const int2 cut = a.cut[few][lo];
      nck = cut.y;
      if (nck > 1) {
        const int block = a.block[few], hk = h / p.G, col = (int)tok * p.G + h - hk * p.G;
        const int nqb = (Lq * p.G + block - 1) / block, qb = col / block;
        const int64_t unit = (cut.x + (int64_t)(nqb - 1 - qb) * nck) * p.Hkv + hk;
        // (Offsets that are out of order may leave a sequence without units and
        // its cut unwritten: nothing is read past the partials.)
        if (cut.x < 0 || nck > a.units[few] || unit + (int64_t)(nck - 1) * p.Hkv >= a.units[few]) nck = 0;
        const float *src = a.ws[few] + (unit * block + col - qb * block) * D + 4 * c;
        const int64_t step = (int64_t)p.Hkv * block * D;
#pragma unroll 8
        for (int j = ROWS ? 0 : g; j < nck; j += ROWS ? 1 : NG) v += *(const f32x4 *)(src + j * step);
      }
    }
  }
  if constexpr (!ROWS) {
    if (nck <= 1) return;  // the whole workgroup
    part[g][threadIdx.x % CG] = v;
    __syncthreads();
    if (g != 0) return;
#pragma unroll
    for (int x = 1; x < NG; ++x) v += part[x][threadIdx.x];
  }
  if (nck <= 1 || 4 * c >= p.dmem) return;
  const int64_t at = (r * p.H + h) * p.dmem + 4 * c;
  if constexpr (sizeof(T) == 4) *(f32x4 *)((float *)p.out + at) = v;
  else *(u32x2 *)((uint16_t *)p.out + at) = (u32x2){Elem<T>::pack(v.x, v.y), Elem<T>::pack(v.z, v.w)};
}

template <typename T, int D> void reduce_t(const ReduceArgs &a, hipStream_t st) {
  constexpr int NG = 256 / (D / 4);
  const int64_t rows = a.p.rows_q * a.p.H;
  // A workgroup for 32 columns where that is few workgroups a CU.
  const int64_t parts = rows * (D / 32);
  if (parts <= 8 * (int64_t)a.p.ncu) paged_reduce_kernel<T, D, false><<<dim3((unsigned)parts), dim3(256), 0, st>>>(a);
  else paged_reduce_kernel<T, D, true><<<dim3((unsigned)((rows + NG - 1) / NG)), dim3(256), 0, st>>>(a);
}

}  // namespace

static_assert(32 * waves_of(32) > kDecodeCols && kPagedBlockF32 > kDecodeCols, "blocks and decoding units differ");
int paged_block(int D) { return 32 * waves_of(D); }

void launch_paged_fwd(const PagedParams &p, int units, int dtype, int D, bool causal, hipStream_t st) {
  by_type(dtype, D, [&](auto *t, auto d) {
    using T = std::remove_pointer_t<decltype(t)>;
    if constexpr (sizeof(T) == 2) fwd_t<T, decltype(d)::value>(p, units, causal, st);
  });
}

void launch_paged_mixed(const PagedParams &pf, int nf, const PagedParams &pd, int nd, int dtype, int D, bool causal,
                        hipStream_t st) {
  by_type(dtype, D, [&](auto *t, auto d) {
    using T = std::remove_pointer_t<decltype(t)>;
    if constexpr (sizeof(T) == 2) mixed_t<T, decltype(d)::value>(pf, nf, pd, nd, causal, st);
  });
}

void launch_paged_reduce(const PagedParams &fwd, const PagedParams &decode, int dtype, int D, hipStream_t st) {
  ReduceArgs a{};
  a.p = fwd;
  a.ws[0] = fwd.ws, a.ws[1] = decode.ws;
  a.cut[0] = fwd.split_units > 0 ? fwd.cut : nullptr;
  a.cut[1] = decode.split_units > 0 ? decode.cut : nullptr;
  a.units[0] = fwd.max_units, a.units[1] = decode.max_units;
  a.block[0] = dtype == kF32 ? kPagedBlockF32 : paged_block(D), a.block[1] = kDecodeCols, a.cols = decode.cols_hi;
  by_type(dtype, D, [&](auto *t, auto d) {
    reduce_t<std::remove_pointer_t<decltype(t)>, decltype(d)::value>(a, st);
  });
}

}  // namespace sigattn
