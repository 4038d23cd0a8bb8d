// Host-only driver for the address/undefined-behaviour sanitizer build of the learned
// bias by relative position (csrc/rel_capi.cpp, the launches of csrc/rel*.hip,
// bias.hip and generic.hip) and of rotary embedding (csrc/rotary.hip).  Kernel launches
// reach the hipLaunchKernel below with the kernels' own parameters; nothing needs a
// GPU.  Every valid problem of a sweep is called with the workspace that it asks for,
// and what the kernels were given has to stay inside it: lines, sums by position of
// every block of queries, a bucket's sums and the parts of grouped heads, one behind
// the other, grids and LDS within what the hardware takes.
#include <algorithm>
#include <climits>
#include <cstdio>
#include <cstring>
#include <map>
#include <random>
#include <string>
#include <vector>

#include "launch.h"
#include "paged.h"
#include "rel.h"
#include "sigattn.h"

using sigattn::KParams;
using sigattn::PagedParams;
using sigattn::PagedRelParams;
using sigattn::RelParams;
using sigattn::RelTable;

namespace {
int g_fail = 0, g_cus = 256;
#define EXPECT(cond)                                                        \
  do {                                                                      \
    if (!(cond)) {                                                          \
      std::fprintf(stderr, "%s:%d: expectation failed: %s\n", __FILE__, __LINE__, #cond); \
      ++g_fail;                                                             \
    }                                                                       \
  } while (0)

// Addresses that are never dereferenced, far apart.
char *at(int i) { return reinterpret_cast<char *>(uintptr_t(i + 1) << 40); }
char *const kQ = at(0), *const kK = at(1), *const kV = at(2), *const kDo = at(3), *const kDq = at(4),
            *const kDk = at(5), *const kDv = at(6), *const kWs = at(7), *const kO = at(8), *const kTable = at(9),
            *const kLine = at(10);

std::map<const void *, std::string> &names() {
  static std::map<const void *, std::string> m;
  return m;
}
struct Kernel {
  std::string name;
  dim3 grid, block;
  size_t lds;
  RelParams p, pk;       // attention kernels; dK/dV's beside dQ's
  PagedRelParams pp;     // over a paged cache
  RelTable t;            // the line's and the gradient's
  const float *out = nullptr;  // rel_sums_kernel's and rel_line_kernel's
  float *bias = nullptr;
};
std::vector<Kernel> g_kernels;
bool has(const Kernel &k, const char *what) { return k.name.find(what) != std::string::npos; }
int g_parts = 0, g_gaps = 0;
KParams g_part;  // launch_add_parts'
}  // namespace

namespace sigattn {
// What only other sources launch.
void launch_fwd_mfma(const KParams &, int, int, bool, bool, hipStream_t) {}
void launch_bwd_dq_mfma(const KParams &, int, int, bool, bool, hipStream_t) {}
void launch_bwd_dkdv_mfma(const KParams &, int, int, bool, bool, bool, hipStream_t) {}
void launch_bwd_dq_ds_mfma(const KParams &, int, int, bool, hipStream_t) {}
void launch_bwd_fused_mfma(const KParams &, int, int, bool, bool, hipStream_t) {}
void launch_fwd_splitkv(const KParams &, int, int, bool, hipStream_t) {}
void launch_fwd_f32(const KParams &, int, bool, bool, hipStream_t) {}
void launch_bwd_dq_f32(const KParams &, int, bool, bool, hipStream_t) {}
void launch_bwd_dkdv_f32(const KParams &, int, bool, bool, hipStream_t) {}
int fwd_rows_per_workgroup(int D) { return (D == 64 ? 4 : 8) * 32; }
int fwd_workgroups_per_cu(int D) { return D == 64 ? 3 : 1; }
int bwd_dq_rows_per_workgroup() { return 128; }
int bwd_dkdv_rows_per_workgroup() { return 128; }
int bwd_dq_workgroups_per_cu(int D) { return D == 64 ? 3 : 2; }
int bwd_dkdv_workgroups_per_cu(int D) { return D == 64 ? 2 : 1; }
void launch_rs_clear(int *, int, int *, int, hipStream_t) {}
hipError_t splitkv_scratch(float **) { return hipErrorInvalidSymbol; }
int paged_block(int D) { return D == 128 ? 256 : 128; }
void launch_paged_fwd(const PagedParams &, int, int, int, bool, hipStream_t) {}
void launch_paged_decode(const PagedParams &, int, int, int, bool, hipStream_t) {}
void launch_paged_mixed(const PagedParams &, int, const PagedParams &, int, int, int, bool, hipStream_t) {}
void launch_paged_decode_f32(const PagedParams &, int, int, bool, hipStream_t) {}
void launch_paged_f32(const PagedParams &, int, int, bool, hipStream_t) {}
void launch_paged_reduce(const PagedParams &, const PagedParams &, int, int, hipStream_t) {}
// Shared with the kernels without the bias.
void launch_add_parts(const KParams &p, int, hipStream_t) {
  if (p.qgroup > 1 && p.qsplit > 1) g_part = p, ++g_parts;
}
}  // namespace sigattn

extern "C" {
char __hip_fatbin[16];
void **__hipRegisterFatBinary(const void *) {
  static void *none = nullptr;
  return &none;
}
void __hipUnregisterFatBinary(void **) {}
void __hipRegisterFunction(void **, const void *host, char *, const char *name, unsigned, void *, void *, void *,
                           void *, int *) {
  names()[host] = name;
}
void __hipRegisterVar(void **, void *, char *, const char *, int, size_t, int, int) {}
static Kernel g_config;
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, hipStream_t) {
  g_config.grid = grid, g_config.block = block, g_config.lds = lds;
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3 *grid, dim3 *block, size_t *lds, hipStream_t *stream) {
  *grid = g_config.grid, *block = g_config.block, *lds = g_config.lds, *stream = nullptr;
  return hipSuccess;
}
hipError_t hipLaunchKernel(const void *host, dim3 grid, dim3 block, void **args, size_t lds, hipStream_t) {
  Kernel k{names()[host], grid, block, lds, {}, {}, {}, {}};
  EXPECT(!k.name.empty());
  if (has(k, "zero_gaps")) {
    ++g_gaps;
    return hipSuccess;
  }
  if (has(k, "rotary")) {
  } else if (has(k, "rel_line_kernel")) {
    k.t = *(RelTable *)args[0], k.out = *(float **)args[1], k.bias = *(float **)args[5];
  } else if (has(k, "rel_sums_kernel")) {
    k.p = *(RelParams *)args[0], k.out = *(float **)args[1];
  } else if (has(k, "rel_grad_kernel")) {
    k.t = *(RelTable *)args[0], k.out = *(float **)args[1];
  } else if (has(k, "PagedRelParams")) {
    k.pp = *(PagedRelParams *)args[0];
  } else {
    k.p = *(RelParams *)args[0];
    if (has(k, "rel_bwd")) k.pk = *(RelParams *)args[1];
  }
  // What a launch may have.
  EXPECT(grid.x >= 1 && grid.y >= 1 && grid.z == 1 && grid.y <= 65535 && block.x <= 1024);
  EXPECT((uint64_t)grid.x * block.x < uint64_t(1) << 32);
  EXPECT(lds <= 160 * 1024);
  g_kernels.push_back(k);
  return hipSuccess;
}
hipError_t hipGetLastError(void) { return hipSuccess; }
hipError_t hipGetDevice(int *dev) {
  *dev = 0;
  return hipSuccess;
}
hipError_t hipDeviceGetAttribute(int *value, hipDeviceAttribute_t, int) {
  *value = g_cus;
  return hipSuccess;
}
// No second stream: everything on the caller's.
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *status) {
  *status = hipStreamCaptureStatusActive;
  return hipSuccess;
}
hipError_t hipStreamGetDevice(hipStream_t, hipDevice_t *) { return hipErrorUnknown; }
hipError_t hipStreamCreateWithFlags(hipStream_t *, unsigned) { return hipErrorUnknown; }
hipError_t hipEventCreateWithFlags(hipEvent_t *, unsigned) { return hipErrorUnknown; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipErrorUnknown; }
hipError_t hipStreamWaitEvent(hipStream_t, hipEvent_t, unsigned) { return hipErrorUnknown; }
}

namespace {

const Kernel *find(const char *what) {
  const Kernel *k = nullptr;
  for (const Kernel &x : g_kernels)
    if (has(x, what)) {
      EXPECT(k == nullptr);
      k = &x;
    }
  return k;
}

sigattn_problem problem(int dtype, int64_t B, int64_t Hkv, int64_t G, int64_t D, int64_t rows, int64_t longest) {
  sigattn_problem p;
  std::memset(&p, 0, sizeof p);
  p.abi_version = SIGATTN_ABI_VERSION, p.dtype = dtype;
  p.B = B, p.H = Hkv * G, p.kv_heads = Hkv, p.D = D, p.rows_q = p.rows_k = rows, p.Tq = p.Tk = longest;
  p.q_stride_t = p.H * D, p.q_stride_h = D, p.k_stride_t = Hkv * D, p.k_stride_h = D;
  p.q = kQ, p.k = kK, p.v = kV, p.scale = (float *)at(11);
  p.cu_seqlens_q = p.cu_seqlens_k = (const int32_t *)at(12);
  return p;
}

sigattn_rel_bias table(int dtype, int32_t buckets, int64_t reach) {
  sigattn_rel_bias r;
  std::memset(&r, 0, sizeof r);
  r.dtype = dtype, r.num_buckets = buckets, r.max_distance = reach, r.table = kTable, r.buckets = (int32_t *)at(13);
  return r;
}

// Bytes [lo, hi) of the workspace that something takes.
struct Span {
  const char *lo, *hi;
};
void apart(std::vector<Span> spans, const char *ws, size_t bytes) {
  std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.lo < b.lo; });
  const char *at = ws;
  for (const Span &s : spans) {
    EXPECT(s.lo >= at && s.hi >= s.lo);
    at = s.hi;
  }
  EXPECT(at <= ws + bytes);
}
Span line_span(const float *line, int64_t H, int reach) {
  return {(const char *)line, (const char *)(line + H * sigattn::line_places(reach))};
}

void line_of(const Kernel &k, const sigattn_problem &p, int reach, std::vector<Span> &spans) {
  EXPECT(k.t.reach == reach && k.t.H == p.H && k.grid.y == (unsigned)p.H);
  spans.push_back(line_span(k.out, p.H, reach));
  if (p.bias == nullptr) spans.push_back({(char *)k.bias, (char *)(k.bias + p.B)});
  else EXPECT(k.bias == nullptr);
}

// A call of the forward, then backwards with and without the forward's lines.
void training(const sigattn_problem &p, const sigattn_rel_bias &r, bool mfma, bool with_table) {
  const int reach = (int)std::min(r.max_distance, std::max(p.Tq, p.Tk));
  const int es = p.dtype == SIGATTN_F32 ? 4 : 2;
  g_kernels.clear(), g_parts = g_gaps = 0;
  size_t n = sigattn_rel_fwd_workspace_bytes(&p, &r);
  EXPECT(n > 0 && sigattn_rel_fwd(&p, &r, kO, kWs, n, nullptr) == SIGATTN_OK);
  EXPECT(g_kernels.size() == 2 && has(g_kernels[0], "rel_line_kernel"));
  std::vector<Span> spans;
  line_of(g_kernels[0], p, reach, spans);
  apart(spans, kWs, n);
  const Kernel &f = g_kernels[1];
  EXPECT(f.p.line == g_kernels[0].out && f.p.reach == reach && f.p.out == kO);
  EXPECT(f.p.bias == (p.bias != nullptr ? p.bias : g_kernels[0].bias));
  EXPECT(has(f, mfma ? (es == 4 ? "fwd_f32" : "fwd_mfma") : "fwd_generic"));
  EXPECT(g_gaps == (mfma ? 0 : 1));

  for (const bool lines : {false, true}) {
    g_kernels.clear(), g_parts = 0;
    n = (with_table ? sigattn_rel_bwd_workspace_bytes : sigattn_rel_bwd_frozen_workspace_bytes)(&p, &r);
    void *const to = with_table ? kTable : nullptr;
    EXPECT(n > 0 && sigattn_rel_bwd(&p, &r, lines ? kLine : nullptr, kDo, kDq, kDk, kDv, to, kWs, n, nullptr) ==
                        SIGATTN_OK);
    spans.clear();
    const Kernel *made = find("rel_line_kernel"), *one = find("rel_bwd"), *sums = find("rel_sums_kernel"),
                 *grad = find("rel_grad_kernel"), *dq = one != nullptr ? one : find("dq_"),
                 *dkdv = one != nullptr ? one : find("dkdv_");
    EXPECT(dq != nullptr && dkdv != nullptr && (made != nullptr) == !lines);
    if (dq == nullptr || dkdv == nullptr) return;
    if (made != nullptr) line_of(*made, p, reach, spans);
    const RelParams &q = dq->p, &k = one != nullptr ? one->pk : dkdv->p;
    const float *line = lines ? (float *)kLine : made->out;
    EXPECT(q.line == line && k.line == line && q.reach == reach && k.reach == reach);
    const float *theirs = (float *)(kLine + sigattn::rel_line_bytes(sigattn::rel_table(&r, p.H, p.Tq, p.Tk)));
    const float *bias = p.bias != nullptr ? p.bias : lines ? theirs : made->bias;
    EXPECT(q.bias == bias && k.bias == bias);
    EXPECT(q.dq == kDq && k.dk == kDk && k.dv == kDv && q.dout == kDo && k.dout == kDo);
    // Blocks of queries: the launch's and those that have a place for their sums.
    const int waves = mfma ? (int)dq->block.x / 64 : 2;
    EXPECT(mfma || dq->block.x == 64);
    EXPECT((int64_t)q.nblk * q.B * q.H <= dq->grid.x);
    if (with_table) {
      EXPECT(q.part != nullptr && sums != nullptr && grad != nullptr && sums->p.part == q.part);
      EXPECT(q.part_rows > 0 && (q.part_rows % 32) == 0 && sums->p.part_rows == q.part_rows);
      EXPECT((int64_t)q.nblk * q.part_rows >= p.Tq && (int64_t)(q.nblk - 1) * q.part_rows < p.Tq);
      EXPECT(dq->lds >= (mfma ? sigattn::near_floats(reach, waves) : q.places()) * sizeof(float));
      spans.push_back({(char *)q.part, (char *)(q.part + q.part_slots() * q.H * q.places())});
      spans.push_back({(char *)sums->out, (char *)(sums->out + p.H * q.places())});
      EXPECT(grad->out == sums->out && grad->t.buckets == r.num_buckets && grad->t.reach == reach);
      EXPECT(grad->lds >= 8 * (size_t)q.places() && sums->grid.y == (unsigned)p.H);
      EXPECT((int64_t)sums->grid.x * 64 >= q.places());
    } else {
      EXPECT(q.part == nullptr && sums == nullptr && grad == nullptr);
    }
    if (g_parts > 0) {
      EXPECT(k.kv_part == g_part.kv_part && k.qsplit == g_part.qsplit && k.qsplit <= q.hgroup);
      spans.push_back({(char *)k.kv_part, (char *)(k.kv_part + (int64_t)k.qsplit * 2 * p.rows_k * p.kv_heads * p.D)});
    }
    apart(spans, kWs, n);
    // Too little, or off its alignment: refused, and nothing launched.
    g_kernels.clear();
    EXPECT(sigattn_rel_bwd(&p, &r, nullptr, kDo, kDq, kDk, kDv, to, kWs, n - 1, nullptr) == SIGATTN_ERR_WORKSPACE);
    EXPECT(sigattn_rel_bwd(&p, &r, nullptr, kDo, kDq, kDk, kDv, to, kWs + 8, n, nullptr) == SIGATTN_ERR_WORKSPACE);
    EXPECT(g_kernels.empty());
  }
}

void training_sweep() {
  std::mt19937 rng(7);
  const auto pick = [&](int64_t lo, int64_t hi) { return std::uniform_int_distribution<int64_t>(lo, hi)(rng); };
  int valid = 0;
  for (int i = 0; i < 6000; ++i) {
    const int dtype = (int)pick(0, 2);
    const int64_t D = int64_t(16) << pick(0, 3), Hkv = pick(1, 9), G = pick(0, 1) ? pick(1, 8) : 1;
    const int64_t B = pick(0, 5) ? pick(1, 40) : pick(1, 2000), longest = int64_t(1) << pick(0, 13);
    const int64_t rows = pick(1, B * longest);
    sigattn_problem p = problem(dtype, B, Hkv, G, D, rows, std::min(rows, pick(1, longest)));
    const sigattn_rel_bias r = table((int)pick(0, 2), (int32_t)pick(1, SIGATTN_REL_MAX_BUCKETS),
                                     pick(0, SIGATTN_REL_MAX_DISTANCE));
    p.causal = (int)pick(0, 1);
    if (pick(0, 1)) p.bias = (float *)at(14);
    const bool odd = pick(0, 7) == 0;  // rows off 16-byte boundaries
    if (odd) p.k_stride_t += 4 / (dtype == SIGATTN_F32 ? 2 : 1);
    g_cus = pick(0, 3) ? 256 : (int)pick(1, 64);
    if (sigattn_rel_check(&p, &r) != SIGATTN_OK) continue;
    ++valid;
    training(p, r, !odd, pick(0, 3) != 0);
  }
  g_cus = 256;
  EXPECT(valid > 5000);
}

// The rule of D = 128 in f16 and bf16: two workgroups of four waves a CU, one of eight
// where the lines of sums leave room for no second, and one of four where not for eight.
void waves_at_128() {
  const int waves[] = {4, 4, 8, 8, 4, 4}, reaches[] = {0, 158, 159, 1190, 1191, 2048};
  for (int i = 0; i < 6; ++i) {
    sigattn_problem p = problem(SIGATTN_BF16, 3, 2, 2, 128, 9000, 4096);
    const sigattn_rel_bias r = table(SIGATTN_F32, 8, reaches[i]);
    g_kernels.clear();
    EXPECT(sigattn_rel_bwd(&p, &r, kLine, kDo, kDq, kDk, kDv, kTable, kWs, sigattn_rel_bwd_workspace_bytes(&p, &r),
                           nullptr) == SIGATTN_OK);
    const Kernel *dq = find("rel_dq_kernel");
    EXPECT(dq != nullptr && dq->block.x == 64u * waves[i] && dq->p.part_rows == 32 * waves[i]);
  }
}

// Calls that have nothing to do, or less.
void empty_calls() {
  const sigattn_rel_bias r = table(SIGATTN_F32, 8, 20);
  for (const int64_t B : {0, 3})
    for (const int64_t rows : {0, 5})
      for (const int64_t longest : {0, 2}) {
        if (B == 0 && longest > 0) continue;
        sigattn_problem p = problem(SIGATTN_BF16, B, 2, 2, 64, rows, longest);
        if (sigattn_rel_check(&p, &r) != SIGATTN_OK) continue;
        g_kernels.clear();
        EXPECT(sigattn_rel_fwd(&p, &r, kO, kWs, sigattn_rel_fwd_workspace_bytes(&p, &r), nullptr) == SIGATTN_OK);
        const size_t n = sigattn_rel_bwd_workspace_bytes(&p, &r);
        EXPECT(sigattn_rel_bwd(&p, &r, nullptr, kDo, kDq, kDk, kDv, kTable, kWs, n, nullptr) == SIGATTN_OK);
        // (The sums' kernel finds every batch's first slot by dividing by the rows of a block.)
        const Kernel *sums = find("rel_sums_kernel");
        EXPECT(find("rel_grad_kernel") != nullptr && sums != nullptr && sums->p.part_rows > 0);
      }
}

void serving() {
  std::mt19937 rng(8);
  const auto pick = [&](int64_t lo, int64_t hi) { return std::uniform_int_distribution<int64_t>(lo, hi)(rng); };
  int valid = 0;
  for (int i = 0; i < 4000; ++i) {
    sigattn_paged_problem p;
    std::memset(&p, 0, sizeof p);
    const int64_t Hkv = pick(1, 9), G = pick(1, 8), ps = int64_t(16) << pick(0, 5);
    p.abi_version = SIGATTN_ABI_VERSION, p.dtype = (int)pick(0, 2), p.D = int64_t(16) << pick(0, 3);
    p.B = pick(0, 5) ? pick(1, 40) : pick(1, 2000), p.H = Hkv * G, p.kv_heads = Hkv;
    p.rows_q = pick(0, 3) ? pick(1, 4000) : p.B, p.max_seqlen_q = pick(1, p.rows_q);
    p.num_pages = 100, p.page_size = ps, p.max_pages = pick(1, 1 << pick(0, 12));
    p.q_stride_t = p.H * p.D, p.q_stride_h = p.D;
    p.k_stride_p = ps * Hkv * p.D, p.k_stride_t = Hkv * p.D, p.k_stride_h = p.D, p.table_stride = p.max_pages;
    p.q = kQ, p.k_cache = kK, p.v_cache = kV;
    p.block_table = p.seq_lens_k = p.cu_seqlens_q = (const int32_t *)at(12);
    p.scale = 0.125f, p.causal = (int)pick(0, 1);
    const bool odd = pick(0, 7) == 0;
    if (odd) p.k_stride_t += 4 / (p.dtype == SIGATTN_F32 ? 2 : 1);
    const sigattn_rel_bias r = table((int)pick(0, 2), (int32_t)pick(1, SIGATTN_REL_MAX_BUCKETS),
                                     pick(0, SIGATTN_REL_MAX_DISTANCE));
    if (sigattn_paged_rel_check(&p, &r) != SIGATTN_OK) continue;
    ++valid;
    const size_t n = sigattn_paged_rel_fwd_workspace_bytes(&p, &r);
    g_kernels.clear();
    EXPECT(sigattn_paged_rel_fwd(&p, &r, kO, kWs, n, nullptr) == SIGATTN_OK);
    EXPECT(g_kernels.size() == 2 && has(g_kernels[0], "rel_line_kernel") && has(g_kernels[1], "PagedRelParams"));
    if (g_kernels.size() != 2) return;
    const Kernel &line = g_kernels[0], &k = g_kernels[1];
    const int reach = (int)std::min<int64_t>(r.max_distance, std::max(p.max_seqlen_q, p.max_pages * ps));
    EXPECT(line.t.reach == reach && line.bias == nullptr && k.pp.line == line.out && k.pp.reach == reach);
    EXPECT(has(k, "generic") == odd);
    std::vector<Span> spans = {line_span(line.out, p.H, reach)};
    if (k.pp.cut != nullptr && k.pp.split_units > 0) spans.push_back({(char *)k.pp.cut, (char *)(k.pp.cut + p.B)});
    apart(spans, kWs, n);
    g_kernels.clear();
    EXPECT(sigattn_paged_rel_fwd(&p, &r, kO, kWs, n - 1, nullptr) == SIGATTN_ERR_WORKSPACE);
    EXPECT(sigattn_paged_rel_fwd(&p, &r, kO, kWs + 8, n, nullptr) == SIGATTN_ERR_WORKSPACE && g_kernels.empty());
  }
  EXPECT(valid > 3000);
}

void rotary() {
  std::mt19937 rng(9);
  const auto pick = [&](int64_t lo, int64_t hi) { return std::uniform_int_distribution<int64_t>(lo, hi)(rng); };
  for (int i = 0; i < 4000; ++i) {
    sigattn_rotary r;
    std::memset(&r, 0, sizeof r);
    r.dtype = (int)pick(0, 2), r.D = int64_t(16) << pick(0, 3), r.interleaved = (int)pick(0, 1);
    r.rows = pick(1, int64_t(1) << pick(0, 18)), r.q_heads = pick(0, 40), r.kv_heads = pick(0, 16);
    r.rot_dim = 2 * pick(1, r.D / 2), r.num_positions = pick(1, 1 << 20);
    r.q_stride_t = r.q_heads * r.D, r.k_stride_t = r.kv_heads * r.D, r.q_stride_h = r.k_stride_h = r.D;
    if (pick(0, 3) == 0) r.q_stride_t += 1;
    r.num_pages = 100, r.page_size = 16;
    r.cache_stride_p = 16 * r.kv_heads * r.D, r.cache_stride_t = r.kv_heads * r.D, r.cache_stride_h = r.D;
    r.q = kQ, r.k = kK, r.v = kV, r.q_out = kO, r.k_out = kDq, r.k_cache = kDk, r.v_cache = kDv;
    r.positions = (int32_t *)at(12), r.angles = (float *)at(13), r.slot_mapping = (int32_t *)at(14);
    for (const bool cache : {false, true}) {
      g_kernels.clear();
      EXPECT((cache ? sigattn_paged_write_rotary(&r, nullptr) : sigattn_rotary_apply(&r, nullptr)) == SIGATTN_OK);
      EXPECT(g_kernels.size() == (r.q_heads + r.kv_heads > 0 ? 1u : 0u));
    }
  }
  // As many rows as the check lets through, on 16-byte boundaries and off them.
  for (const int dtype : {SIGATTN_BF16, SIGATTN_F32})
    for (const int64_t heads : {1, 40, 65535})
      for (const int64_t D : {16, 128})
        for (const int64_t odd : {0, 1}) {
          sigattn_rotary r;
          std::memset(&r, 0, sizeof r);
          r.dtype = dtype, r.D = r.rot_dim = D, r.q_heads = heads, r.num_positions = 9;
          r.q_stride_t = heads * D + odd, r.q_stride_h = D;
          r.q = kQ, r.q_out = kO, r.positions = (int32_t *)at(12), r.angles = (float *)at(13);
          r.rows = std::min<int64_t>(INT32_MAX / 2, (int64_t(1) << 42) / (heads * D));
          g_kernels.clear();
          EXPECT(sigattn_rotary_apply(&r, nullptr) == SIGATTN_OK && g_kernels.size() == 1);
          const int64_t columns = dtype == SIGATTN_F32 ? 8 : 16;  // of a thread
          const dim3 g = g_kernels[0].grid;
          if (!odd) EXPECT((int64_t)g.x * g.y * 256 >= r.rows * heads * D / columns);
          r.rows = r.rows + 1;
          g_kernels.clear();
          EXPECT(sigattn_rotary_apply(&r, nullptr) == SIGATTN_ERR_SHAPE && g_kernels.empty());
        }
}

}  // namespace

int main() {
  training_sweep();
  waves_at_128();
  empty_calls();
  serving();
  rotary();
  if (g_fail == 0) std::puts("all checks passed");
  return g_fail == 0 ? 0 : 1;
}
