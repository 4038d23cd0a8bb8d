// Host-only driver for the address/undefined-behaviour sanitizer build of
// csrc/capi.cpp: the dispatch of grouped heads.  The launchers are recorders, as
// in capi_driver.cpp; nothing needs a GPU.  For a sweep of packed problems with
// kv_heads < H, every backward entry is called with workspaces of several sizes,
// and what the kernels get has to be whole groups at the right addresses, with dS
// tiles and parts of groups inside the workspace.
#include <algorithm>
#include <climits>
#include <cstdio>
#include <cstring>
#include <random>
#include <string>
#include <vector>

#include "launch.h"
#include "sigattn.h"

using sigattn::GapAxis;
using sigattn::KParams;

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
char *const kQ = at(0), *const kK = at(1), *const kV = at(2), *const kDo = at(3), *const kDq = at(4), *const kDk = at(5),
            *const kDv = at(6), *const kWs = at(7), *const kO = at(8);

struct Launch {
  std::string name;
  KParams p;
};
std::vector<Launch> g_calls;
void record(const char *name, const KParams &p) { g_calls.push_back({name, p}); }
}  // namespace

namespace sigattn {
void launch_fwd_mfma(const KParams &p, int, int, bool, bool, hipStream_t) { record("fwd", p); }
void launch_bwd_dq_mfma(const KParams &p, int, int, bool, bool, hipStream_t) { record("dq", p); }
void launch_bwd_dkdv_mfma(const KParams &p, int, int, bool, bool, bool dsout, hipStream_t) {
  record(dsout ? "dkdv_ds" : "dkdv", p);
}
void launch_bwd_dq_ds_mfma(const KParams &p, int, int, bool, hipStream_t) { record("dq_ds", p); }
void launch_bwd_fused_mfma(const KParams &p, int, int, bool, bool, hipStream_t) { record("fused", p); }
void launch_fwd_splitkv(const KParams &p, int, int, bool, hipStream_t) { record("splitkv", p); }
void launch_fwd_f32(const KParams &p, int, bool, bool, hipStream_t) { record("fwd_f32", p); }
void launch_bwd_dq_f32(const KParams &p, int, bool, bool, hipStream_t) { record("dq_f32", p); }
void launch_bwd_dkdv_f32(const KParams &p, int, bool, bool, hipStream_t) { record("dkdv_f32", p); }
void launch_fwd_generic(const KParams &p, int, int, bool, hipStream_t) { record("fwd_generic", p); }
void launch_bwd_dq_generic(const KParams &p, int, int, bool, hipStream_t) { record("dq_generic", p); }
void launch_bwd_dkdv_generic(const KParams &p, int, int, bool, hipStream_t) { record("dkdv_generic", p); }
int fwd_rows_per_workgroup(int D) { return (D == 64 ? 4 : 8) * 32; }
int fwd_workgroups_per_cu(int D) { return D == 64 ? 3 : 1; }
int bwd_dq_rows_per_workgroup() { return 128; }
int bwd_dkdv_rows_per_workgroup() { return 128; }
int bwd_dq_workgroups_per_cu(int D) { return D == 64 ? 3 : 2; }
int bwd_dkdv_workgroups_per_cu(int D) { return D == 64 ? 2 : 1; }
void launch_rs_clear(int *, int, int *, int, hipStream_t) { EXPECT(!"range split of grouped heads"); }
void launch_zero_gaps(const GapAxis &, const GapAxis &, int, hipStream_t) {}
hipError_t splitkv_scratch(float **) { return hipErrorInvalidSymbol; }
}  // namespace sigattn

extern "C" {
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

struct Case {
  sigattn_problem p;
  int64_t G, esize, ds;  // ds: bytes of a head's dS
};

// The whole problem, on the recompute kernels or the fp32 ones: every item a K / V
// head that streams its group, in parts inside [kWs, kWs + bytes).
void whole(const Case &c, int64_t bytes, bool parts) {
  EXPECT(g_calls.size() == 2);
  for (const Launch &l : g_calls) {
    const KParams &p = l.p;
    EXPECT(p.q == kQ && p.k == kK && p.v == kV);
    if (l.name.compare(0, 4, "dkdv") == 0) {
      EXPECT(p.H == c.p.kv_heads && p.qgroup == c.G && p.hgroup == 1 && p.dk == kDk && p.dv == kDv);
      EXPECT(parts || p.qsplit <= 1);
      if (p.qsplit > 1) {
        EXPECT(p.qsplit <= c.G && (char *)p.kv_part >= kWs && ((uintptr_t)p.kv_part & 15) == 0);
        EXPECT((char *)(p.kv_part + p.qsplit * 2 * p.rows_k * p.H * p.dmem) <= kWs + bytes);
        for (int i = 0; i < p.qsplit; ++i) EXPECT((i + 1) * c.G / p.qsplit > i * c.G / p.qsplit);
      }
    } else {
      EXPECT(p.H == c.p.H && p.hgroup == c.G && p.dq == kDq);
    }
  }
}

// Passes over whole groups: each a dK/dV launch and a dQ launch over the same
// heads, in order, of one size but for the last.
int64_t passes(const Case &c, int64_t bytes) {
  EXPECT(!g_calls.empty() && g_calls.size() % 2 == 0);
  int64_t h0 = 0, n = 0, size = 0;
  for (size_t i = 0; i + 1 < g_calls.size(); i += 2, ++n) {
    const KParams &kv = g_calls[i].p, &dq = g_calls[i + 1].p;
    EXPECT(g_calls[i].name == "dkdv_ds" && g_calls[i + 1].name == "dq_ds");
    EXPECT(dq.H % c.G == 0 && kv.H * c.G == dq.H && kv.qgroup == c.G && kv.hgroup == 1 && dq.hgroup == c.G);
    const int64_t qo = h0 * c.p.q_stride_h * c.esize, ko = h0 / c.G * c.p.k_stride_h * c.esize;
    EXPECT(kv.q == kQ + qo && kv.dout == kDo + qo && dq.dq == kDq + qo && dq.k == kK + ko);
    EXPECT(kv.k == kK + ko && kv.v == kV + ko && kv.dk == kDk + ko && kv.dv == kDv + ko);
    EXPECT((char *)kv.ds == kWs && dq.ds == kv.ds && dq.H * c.ds <= bytes);
    if (kv.qsplit > 1) {
      EXPECT(dq.H == c.p.H && kv.qsplit <= c.G && (char *)kv.kv_part >= kWs + c.p.H * c.ds);
      EXPECT((char *)(kv.kv_part + kv.qsplit * 2 * kv.rows_k * kv.H * kv.dmem) <= kWs + bytes);
    }
    EXPECT(n == 0 || dq.H <= size);
    size = n == 0 ? dq.H : size;
    h0 += dq.H;
  }
  EXPECT(h0 == c.p.H);
  return n;
}

}  // namespace

int main() {
  std::mt19937 rng(3);
  const auto pick = [&](std::initializer_list<int64_t> v) { return v.begin()[rng() % v.size()]; };
  int64_t split = 0, several = 0, recomputed = 0;
  for (int i = 0; i < 30000; ++i) {
    Case c;
    sigattn_problem &p = c.p;
    std::memset(&p, 0, sizeof p);
    p.abi_version = SIGATTN_ABI_VERSION;
    p.dtype = (int)pick({SIGATTN_F16, SIGATTN_BF16, SIGATTN_F32});
    p.causal = (int)pick({0, 1});
    c.G = pick({2, 3, 4, 7, 16}), c.esize = p.dtype == SIGATTN_F32 ? 4 : 2;
    p.kv_heads = pick({1, 2, 3, 4, 5, 8}), p.H = p.kv_heads * c.G, p.D = pick({16, 32, 64, 128, 128});
    p.B = pick({1, 2, 9, 64, 65, 300});
    p.Tq = pick({1, 31, 64, 300, 4096, 60000}), p.Tk = pick({1, 31, 64, 300, 4096, 60000});
    p.rows_q = pick({1, 70, 900, 40000}), p.rows_k = pick({1, 70, 900, 40000});
    p.q_stride_t = p.H * p.D, p.q_stride_h = p.D, p.k_stride_t = p.kv_heads * p.D, p.k_stride_h = p.D;
    p.q = kQ, p.k = kK, p.v = kV, p.bias = p.scale = (const float *)at(9);
    p.cu_seqlens_q = p.cu_seqlens_k = (const int32_t *)at(10);
    g_cus = (int)pick({0, 8, 256, 256});
    const int64_t nq = (p.Tq + 31) / 32, nk = (p.Tk + 31) / 32;
    c.ds = p.B * (p.causal ? nq * (nq + 1) / 2 : nq * nk) * 2048;
    EXPECT(sigattn_check(&p) == SIGATTN_OK);
    const int64_t two = (int64_t)sigattn_bwd_workspace_bytes(&p), parts = (int64_t)sigattn_bwd_split_workspace_bytes(&p);
    const bool two_pass = p.D == 128 && p.dtype != SIGATTN_F32;
    EXPECT(two_pass ? two >= p.H * c.ds && parts == 0 : two == 0);

    const auto ws = [&](int64_t bytes) {
      g_calls.clear();
      EXPECT(sigattn_bwd_ws(&p, kDo, kDq, kDk, kDv, bytes > 0 ? kWs : nullptr, bytes, nullptr) == SIGATTN_OK);
    };
    const auto bwd_split = [&](int64_t bytes) {
      g_calls.clear();
      return sigattn_bwd_split(&p, kDo, kDq, kDk, kDv, bytes > 0 ? kWs : nullptr, bytes, nullptr);
    };
    ws(0);
    whole(c, 0, false);
    if (two_pass) {
      for (int64_t n : {(int64_t)16, c.ds, c.G * c.ds - 16}) {  // less than a group: recomputed
        if (n <= 0) continue;
        ws(n);
        whole(c, n, false);
        ++recomputed;
      }
      for (int64_t groups = 1; groups <= p.kv_heads; ++groups) {
        const int64_t n = groups * c.G * c.ds;
        ws(n);
        const int64_t got = passes(c, n);
        EXPECT(got == (p.kv_heads + groups - 1) / groups);
        several += got > 1;
      }
      ws(two);
      EXPECT(passes(c, two) == 1);
      split += g_calls[0].p.qsplit > 1;
      EXPECT((g_calls[0].p.qsplit > 1) == (two > p.H * c.ds));
      EXPECT(sigattn_bwd_dkdv_ws(&p, kDo, kDk, kDv, kWs, p.H * c.ds - 16, nullptr) == SIGATTN_ERR_WORKSPACE);
    }
    EXPECT(bwd_split(0) == SIGATTN_OK);
    whole(c, 0, false);
    if (parts > 0) {
      EXPECT(bwd_split(parts) == SIGATTN_OK);
      whole(c, parts, true);
      split += std::any_of(g_calls.begin(), g_calls.end(), [](const Launch &l) { return l.p.qsplit > 1; });
      EXPECT(bwd_split(parts - 16) == SIGATTN_ERR_WORKSPACE && g_calls.empty());
    }
    // Forward: short queries the split-KV kernel, else one item per query head.
    g_calls.clear();
    const int64_t fw = (int64_t)sigattn_fwd_decode_workspace_bytes(&p);
    EXPECT(sigattn_fwd_decode(&p, kO, fw > 0 ? kWs : nullptr, fw, nullptr) == SIGATTN_OK && g_calls.size() == 1);
    EXPECT(g_calls[0].p.H == p.H && g_calls[0].p.hgroup == c.G && g_calls[0].p.k == kK);
    if (g_calls[0].name == "splitkv" && g_calls[0].p.nsplit > 1) {
      const KParams &k = g_calls[0].p;
      const int64_t rows = k.rows > 0 ? k.rows : (int64_t)k.nsplit * p.B;
      EXPECT((char *)(k.ws + rows * p.H * p.Tq * p.D) + (k.rows > 0 ? 8 * p.B : 0) <= kWs + fw);
    }
    // Version 2 ends before kv_heads (here the memory does too): each head has its own.
    p.abi_version = 2;
    std::vector<char> old((char *)&p, (char *)&p.kv_heads);
    const sigattn_problem *v2 = (const sigattn_problem *)old.data();
    g_calls.clear();
    EXPECT(sigattn_bwd(v2, kDo, kDq, kDk, kDv, nullptr) == SIGATTN_OK);
    EXPECT(sigattn_fwd(v2, kO, nullptr) == SIGATTN_OK && sigattn_bwd_split_workspace_bytes(v2) == 0);
    for (const Launch &l : g_calls) EXPECT(l.p.H == p.H && l.p.hgroup == 1 && l.p.qgroup == 1);
  }
  EXPECT(split > 1000 && several > 1000 && recomputed > 1000);
  if (g_fail == 0) std::puts("all checks passed");
  return g_fail == 0 ? 0 : 1;
}
