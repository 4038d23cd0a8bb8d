// Host-only driver for the address/undefined-behaviour sanitizer build of the
// paged cache's C ABI (csrc/paged_capi.cpp, and the checks and launches of
// csrc/paged.hip).  Launchers of the other files are recorders; kernel launches of
// paged.hip reach the hipLaunchKernel below.  Nothing needs a GPU.  Every valid
// problem of a sweep, its limits among them, is called with the workspace it
// asks for, and what the kernels were given has to stay inside it: they write
// fp32 sums of unit u at u * block * D floats and read max_units of them.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

#include "launch.h"
#include "paged.h"
#include "sigattn.h"

using sigattn::PagedParams;

namespace {
int g_fail = 0, g_cus = 256;
#define EXPECT(cond)                                                        \
  do {                                                                      \
    if (!(cond)) {                                                          \
      std::fprintf(stderr, "%s:%d: expectation failed: %s\n", __FILE__, __LINE__, #cond); \
      ++g_fail;                                                             \
    }                                                                       \
  } while (0)

void *const kFake = reinterpret_cast<void *>(uintptr_t(1) << 20);  // never dereferenced
char *const kWs = reinterpret_cast<char *>(uintptr_t(1) << 40);

struct Launch {
  const char *name;
  PagedParams f, d;  // the forward part's, the decoding part's
  int nf, nd, D;
};
std::vector<Launch> g_calls;
struct Kernel {
  dim3 grid, block;
  size_t lds;
};
std::vector<Kernel> g_kernels;
int g_gaps = 0;
}  // namespace

namespace sigattn {
int device_compute_units() { return g_cus; }
int paged_block(int D) { return D == 128 ? 256 : 128; }
void launch_paged_fwd(const PagedParams &p, int units, int, int D, bool, hipStream_t) {
  g_calls.push_back({"fwd", p, {}, units, 0, D});
}
void launch_paged_decode(const PagedParams &p, int units, int, int D, bool, hipStream_t) {
  g_calls.push_back({"decode", {}, p, 0, units, D});
}
void launch_paged_mixed(const PagedParams &pf, int nf, const PagedParams &pd, int nd, int, int D, bool, hipStream_t) {
  g_calls.push_back({"mixed", pf, pd, nf, nd, D});
}
void launch_paged_decode_f32(const PagedParams &p, int units, int D, bool, hipStream_t) {
  g_calls.push_back({"decode_f32", {}, p, 0, units, D});
}
void launch_paged_f32(const PagedParams &p, int units, int D, bool, hipStream_t) {
  g_calls.push_back({"f32", p, {}, units, 0, D});
}
void launch_paged_reduce(const PagedParams &f, const PagedParams &d, int, int D, hipStream_t) {
  g_calls.push_back({"reduce", f, d, 0, 0, D});
}
void launch_zero_gaps(const GapAxis &, const GapAxis &, int, hipStream_t) { ++g_gaps; }
}  // namespace sigattn

// What the compiler's launches call.
extern "C" {
char __hip_fatbin[16];
void **__hipRegisterFatBinary(const void *) {
  static void *none = nullptr;
  return &none;
}
void __hipUnregisterFatBinary(void **) {}
void __hipRegisterFunction(void **, const void *, char *, const char *, unsigned, void *, void *, void *, void *, int *) {}
void __hipRegisterVar(void **, void *, char *, const char *, int, size_t, int, int) {}
static Kernel g_config;
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, hipStream_t) {
  g_config = {grid, block, lds};
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3 *grid, dim3 *block, size_t *lds, hipStream_t *stream) {
  *grid = g_config.grid, *block = g_config.block, *lds = g_config.lds, *stream = nullptr;
  return hipSuccess;
}
hipError_t hipLaunchKernel(const void *, dim3 grid, dim3 block, void **, size_t lds, hipStream_t) {
  g_kernels.push_back({grid, block, lds});
  return hipSuccess;
}
hipError_t hipGetLastError(void) { return hipSuccess; }
}

namespace {

sigattn_paged_problem problem(int dtype, int64_t B, int64_t Hkv, int64_t G, int64_t D, int64_t rows, int64_t longest,
                              int64_t ps, int64_t max_pages) {
  sigattn_paged_problem p;
  std::memset(&p, 0, sizeof p);
  p.abi_version = SIGATTN_ABI_VERSION, p.dtype = dtype;
  p.B = B, p.H = Hkv * G, p.kv_heads = Hkv, p.D = D, p.rows_q = rows, p.max_seqlen_q = longest;
  p.num_pages = 100, p.page_size = ps, p.max_pages = max_pages;
  p.q_stride_t = p.H * D, p.q_stride_h = D;
  p.k_stride_p = ps * Hkv * D, p.k_stride_t = Hkv * D, p.k_stride_h = D;
  p.table_stride = max_pages;
  p.q = p.k_cache = p.v_cache = kFake;
  p.block_table = p.seq_lens_k = p.cu_seqlens_q = (const int32_t *)kFake;
  p.scale = 0.125f, p.causal = 1;
  return p;
}

// The units that paged_unit makes of a batch: the rule of its comment, in the
// same floats (its sums may be added in another order).
int64_t units_of(const PagedParams &p, int block, const std::vector<int> &tokens, const std::vector<int> &keys) {
  const int B = (int)tokens.size();
  const auto blocks = [&](int b) {
    const int64_t cols = (int64_t)tokens[b] * p.G;
    return (int)(cols > p.cols_lo && cols <= p.cols_hi ? (cols + block - 1) / block : 0);
  };
  if (block == sigattn::kDecodeCols && p.split_units == 0) return (int64_t)B * p.Hkv;
  int C = sigattn::kNoCut;
  if (p.split_units > 0) {
    float work = 0.0f;
    for (int b = 0; b < B; ++b) work += (float)blocks(b) * (float)keys[b];
    work *= (float)p.Hkv;
    const float c = work / (float)p.split_units, least = work / (float)p.total_units;
    C = sigattn::chunk_for(c, p.min_chunk);
    if (B <= 64 && p.Tk < 1 << 23)
      for (int lane = 0; lane < 63; ++lane) {
        const int mine = sigattn::chunk_for(least + (c - least) * lane / 63.0f, p.min_chunk);
        int64_t rows = 0;
        for (int b = 0; b < B; ++b) rows += (int64_t)blocks(b) * std::max((int)std::ceil((float)keys[b] / (float)mine), 1);
        if (rows * p.Hkv <= p.total_units) {
          C = mine;
          break;
        }
      }
  }
  int64_t units = 0;
  for (int b = 0; b < B; ++b) {
    const int64_t L = keys[b], round = block == sigattn::kDecodeCols ? 32 : 64;
    const int64_t most = std::min<int64_t>(std::max<int64_t>((L + C - 1) / C, 1), sigattn::kMostChunks);
    const int64_t len = std::max<int64_t>(((L + most - 1) / most + round - 1) / round * round, round);
    units += blocks(b) * std::max<int64_t>((L + len - 1) / len, 1) * p.Hkv;
  }
  return units;
}

// One part's partials lie in [from, to), and its units hold any lengths'.
void part(const PagedParams &p, int units, int block, int D, const char *from, const char *to, std::mt19937 &rng,
          int64_t rows) {
  EXPECT(units > 0 && p.max_units == units);
  EXPECT((int64_t)units + p.ngap[0] <= INT_MAX);
  if (p.split_units > 0) {
    EXPECT(p.min_chunk > 0 && p.total_units > p.split_units - 1 && p.total_units <= units);
    EXPECT((const char *)p.ws >= from && ((uintptr_t)p.ws & 15) == 0);
    EXPECT((const char *)(p.ws + (int64_t)units * block * D) <= to);
  }
  if (p.B > 3000) return;
  for (int trial = 0; trial < 4; ++trial) {
    std::vector<int> tokens(p.B), keys(p.B);
    int64_t left = rows;
    for (int b = 0; b < p.B; ++b) {
      const int64_t most = std::min<int64_t>(left, p.Tq);
      tokens[b] = trial == 0 ? (int)std::min<int64_t>(most, rows / p.B) : (int)(rng() % (uint64_t)(most + 1));
      if (trial == 1 && b == 0) tokens[b] = (int)most;
      left -= tokens[b];
      keys[b] = trial < 2 ? p.Tk : (int)(rng() % (uint64_t)(p.Tk + 1)) >> (trial == 3 ? rng() % 20 : 0);
    }
    EXPECT(units_of(p, block, tokens, keys) <= units);
  }
}

void sweep() {
  std::mt19937 rng(5);
  const auto pick = [&](std::initializer_list<int64_t> v) { return v.begin()[rng() % v.size()]; };
  int64_t valid = 0, cut = 0, mixed = 0;
  for (int i = 0; i < 40000; ++i) {
    const int dtype = (int)pick({SIGATTN_F16, SIGATTN_BF16, SIGATTN_F32});
    const int64_t ps = pick({16, 32, 64, 128, 1024, 1 << 20});
    const int64_t most = INT_MAX / 2 / ps;
    sigattn_paged_problem p =
        problem(dtype, pick({0, 1, 2, 3, 16, 63, 64, 65, 200, 257, 1023, 1024, 2999, 1 << 20, INT_MAX / 64}),
                pick({1, 2, 3, 8, 16, 64, 1024}), pick({1, 2, 4, 7, 16, 33, 64}), pick({16, 32, 64, 128}),
                pick({0, 1, 2, 33, 64, 500, 4096, 70000, INT_MAX / 64}), pick({0, 1, 2, 8, 33, 300, 5000, INT_MAX}), ps,
                std::min(most, pick({0, 1, 2, 5, 8, 40, 700, 4096, most})));
    g_cus = (int)pick({0, 1, 64, 256, 256, 256});
    const int rc = sigattn_paged_check(&p);
    EXPECT(rc == SIGATTN_OK || rc == SIGATTN_ERR_SHAPE);
    const size_t n = sigattn_paged_fwd_workspace_bytes(&p);
    g_calls.clear(), g_kernels.clear();
    if (rc != SIGATTN_OK) {
      EXPECT(n == 0 && sigattn_paged_fwd(&p, kFake, kWs, n, nullptr) == rc && g_calls.empty());
      continue;
    }
    ++valid;
    g_gaps = 0;
    EXPECT(sigattn_paged_fwd(&p, kFake, n > 0 ? kWs : nullptr, n, nullptr) == SIGATTN_OK);
    if (p.rows_q == 0) {
      EXPECT(n == 0 && g_calls.empty() && g_gaps == 0);
      continue;
    }
    if (p.B == 0) {
      EXPECT(n == 0 && g_calls.empty() && g_gaps == 1);
      continue;
    }
    EXPECT(!g_calls.empty() && g_calls.size() == (n > 0 ? 2 : 1) && g_kernels.empty());
    const Launch c = g_calls[0];
    const PagedParams &first = c.nf > 0 ? c.f : c.d;
    EXPECT(first.ngap[0] % 8 == 0 && (int64_t)first.ngap[0] * 64 >= p.rows_q);
    EXPECT(first.gap[0].rows == p.rows_q && first.gap[0].out[0] == kFake && first.gap[0].st == p.H * p.D);
    const int block = dtype == SIGATTN_F32 ? sigattn::kPagedBlockF32 : sigattn::paged_block(c.D);
    const char *end = kWs + n;
    const bool fs = c.nf > 0 && c.f.split_units > 0, ds = c.nd > 0 && c.d.split_units > 0;
    EXPECT((n > 0) == (fs || ds));
    // Every number of columns is one part's.
    if (c.nf > 0 && c.nd > 0) EXPECT(c.f.cols_lo == c.d.cols_hi && c.d.cols_lo == 0 && c.f.cols_hi == INT_MAX);
    else if (c.nf > 0) EXPECT(c.f.cols_lo == 0 && c.f.cols_hi == INT_MAX);
    else EXPECT(c.d.cols_lo == 0 && (int64_t)c.d.Tq * c.d.G <= c.d.cols_hi);
    if (c.nd > 0) EXPECT(c.d.cols_hi == sigattn::kDecodeCols);
    mixed += c.nf > 0 && c.nd > 0;
    const char *parts = kWs;
    if (n > 0) {
      ++cut;
      EXPECT(std::strcmp(g_calls[1].name, "reduce") == 0);
      parts = kWs + 2 * p.B * (int64_t)sizeof(int2);  // behind both parts' cuts
      if (fs) EXPECT((char *)c.f.cut == kWs);
      if (ds) EXPECT((char *)c.d.cut == kWs + p.B * (int64_t)sizeof(int2));
      if (fs && ds) EXPECT((char *)(c.f.ws + (int64_t)c.nf * block * c.D) <= (char *)c.d.ws);
      // Too little, or off its alignment: refused.  None: nothing is cut.
      g_calls.clear();
      EXPECT(sigattn_paged_fwd(&p, kFake, kWs, n - 1, nullptr) == SIGATTN_ERR_WORKSPACE);
      EXPECT(sigattn_paged_fwd(&p, kFake, kWs + 8, n, nullptr) == SIGATTN_ERR_WORKSPACE && g_calls.empty());
      EXPECT(sigattn_paged_fwd(&p, kFake, nullptr, 0, nullptr) == SIGATTN_OK && g_calls.size() == 1);
      EXPECT(g_calls[0].f.split_units == 0 && g_calls[0].d.split_units == 0);
    }
    if (c.nf > 0) part(c.f, c.nf, block, c.D, parts, end, rng, p.rows_q);
    if (c.nd > 0) part(c.d, c.nd, sigattn::kDecodeCols, c.D, parts, end, rng, p.rows_q);
  }
  EXPECT(valid > 10000 && cut > 2000 && mixed > 1000);
}

// Rows off 16-byte boundaries take the portable kernel: a workgroup a row and head.
void portable() {
  sigattn_paged_problem p = problem(SIGATTN_BF16, 3, 2, 4, 64, 50, 40, 16, 40);
  p.k_stride_t += 4;
  g_calls.clear(), g_kernels.clear();
  EXPECT(sigattn_paged_fwd_workspace_bytes(&p) == 0);
  EXPECT(sigattn_paged_fwd(&p, kFake, nullptr, 0, nullptr) == SIGATTN_OK && g_calls.empty());
  EXPECT(g_kernels.size() == 1 && g_kernels[0].grid.x == 50 && g_kernels[0].grid.y == 8);
  p = problem(SIGATTN_F32, 3, 2, 4, 64, 50, 40, 16, 40);
  EXPECT(sigattn_paged_fwd(&p, (char *)kFake + 4, nullptr, 0, nullptr) == SIGATTN_OK && g_calls.empty());
  EXPECT(g_kernels.size() == 2);
}

void plan_and_writer() {
  int32_t *const i = (int32_t *)kFake;
  const auto plan = [&](int64_t B, int64_t tokens, int64_t max_pages, int64_t ps, int64_t free) {
    return sigattn_paged_plan(B, i, i, i, max_pages, max_pages, i, free, ps, tokens, i, i, i, i, nullptr);
  };
  g_kernels.clear();
  for (int64_t B : {0, 1, 255, 256, SIGATTN_PLAN_MAX_BATCH})
    for (int64_t n : {0, 1, 256, 257, 100000, INT_MAX / 2}) {
      EXPECT(plan(B, n, 4, 16, 100) == SIGATTN_OK && g_kernels.size() == 1);
      EXPECT(g_kernels[0].grid.x >= 1 && g_kernels[0].grid.x <= 1024 && g_kernels[0].block.x == 256);
      EXPECT(g_kernels[0].lds == 2 * (size_t)(B + 1) * 4 && g_kernels[0].lds <= 160 * 1024);
      g_kernels.clear();
    }
  EXPECT(plan(SIGATTN_PLAN_MAX_BATCH + 1, 1, 4, 16, 1) == SIGATTN_ERR_SHAPE);
  EXPECT(plan(1, int64_t(1) << 31, 4, 16, 1) == SIGATTN_ERR_SHAPE);
  EXPECT(plan(1, 1, INT_MAX / 16 + 1, 16, 1) == SIGATTN_ERR_SHAPE);
  EXPECT(plan(1, 1, 4, 16, int64_t(1) << 31) == SIGATTN_ERR_SHAPE);
  sigattn_paged_rows r;
  std::memset(&r, 0, sizeof r);
  r.rows = 1000, r.kv_heads = 8, r.num_pages = 4, r.page_size = 16;
  r.k = r.v = r.k_cache = r.v_cache = kFake, r.slot_mapping = i;
  for (int esize : {2, 4})
    for (int64_t D : {16, 32, 64, 128})
      for (int64_t rows : {int64_t(1), int64_t(1000), int64_t(INT_MAX / 2)})
        for (int64_t heads : {int64_t(8), int64_t(65535)}) {
          r.esize = esize, r.D = D, r.rows = rows, r.kv_heads = heads;
          r.src_stride_t = r.cache_stride_t = heads * D, r.src_stride_h = r.cache_stride_h = D;
          r.cache_stride_p = 16 * heads * D;
          EXPECT(sigattn_paged_write(&r, nullptr) == SIGATTN_OK && g_kernels.size() == 1);
          EXPECT(g_kernels[0].grid.x >= 1 && g_kernels[0].grid.x <= 1 << 20 && g_kernels[0].grid.y == 2);
          g_kernels.clear();
        }
  // More heads than attention takes: refused, their products pass 63 bits.
  for (int64_t heads : {int64_t(65536), int64_t(INT_MAX), int64_t(INT_MAX) + 1}) {
    r.kv_heads = heads;
    EXPECT(sigattn_paged_write(&r, nullptr) == SIGATTN_ERR_SHAPE && g_kernels.empty());
  }
  r.rows = 0, r.kv_heads = 8;
  EXPECT(sigattn_paged_write(&r, nullptr) == SIGATTN_OK && g_kernels.empty());
  EXPECT(sigattn_paged_write(nullptr, nullptr) == SIGATTN_ERR_NULL_ARG);
  EXPECT(sigattn_paged_check(nullptr) == SIGATTN_ERR_NULL_ARG);
  EXPECT(sigattn_paged_fwd_workspace_bytes(nullptr) == 0);
  EXPECT(sigattn_paged_fwd(nullptr, kFake, nullptr, 0, nullptr) == SIGATTN_ERR_NULL_ARG);
}

}  // namespace

int main() {
  sweep();
  portable();
  plan_and_writer();
  if (g_fail == 0) std::puts("all checks passed");
  return g_fail == 0 ? 0 : 1;
}
