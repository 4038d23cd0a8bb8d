// Eager autograd node of the public APIs (sigmoid_attention,
// sigmoid_attention_padded, sigmoid_attention_varlen), in C++, and the short
// ways of eager calls with canonical arguments into the library.
//
// The reference builds its eager path from torch.autograd.Function-style
// registrations in Python (src/triton_sigmoid/sigmoid_triton_dense.py:696-753,
// sigmoid_triton_padded.py:780-846).  The same node written in Python costs
// tens of microseconds of host time per forward+backward before any kernel
// runs -- more than a small problem's kernels take -- and PyTorch's autograd
// engine runs a CUDA node's backward on its device thread, where a Python
// node must take the GIL.  This module is that node in C++: the forward
// launches the library's forward on the canonical tensors the Python layer
// prepared and saves them; the backward launches the library's backward on
// them.  Launch policy is the Python layer's (_capi._launch_fwd,
// _capi._launch_bwd): the forward is sigattn_fwd_decode with the workspace it
// asks for; the backward takes the range-split
// recompute backward when a small grid splits, else the two-pass kernels at
// the head dims and workspace limit the Python layer configures (in head
// groups when the whole problem's dS does not fit, unless a group's
// dQ-from-dS grid would have fewer workgroups than the GPU has compute
// units), else the recompute backward.  Workspaces come from
// torch's caching allocator; a workspace that cannot be allocated falls back
// to the kernels that need none.
//
// The library's entry points arrive as addresses from the Python layer
// (bind()), so this module calls the very library _capi loaded.  No HIP
// kernels live here.

#include <torch/extension.h>

#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>

#include <atomic>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <map>
#include <mutex>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/sigattn.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;

struct Api {
  decltype(&sigattn_strerror) strerror = nullptr;
  decltype(&sigattn_default_bias) default_bias = nullptr;
  decltype(&sigattn_fwd_workspace_bytes) fwd_workspace_bytes = nullptr;
  decltype(&sigattn_fwd_ws) fwd_ws = nullptr;
  decltype(&sigattn_fwd_decode_workspace_bytes) fwd_decode_workspace_bytes = nullptr;
  decltype(&sigattn_fwd_decode) fwd_decode = nullptr;
  decltype(&sigattn_bwd_workspace_bytes) bwd_workspace_bytes = nullptr;
  decltype(&sigattn_bwd_ws) bwd_ws = nullptr;
  decltype(&sigattn_bwd_split_workspace_bytes) bwd_split_workspace_bytes = nullptr;
  decltype(&sigattn_bwd_split) bwd_split = nullptr;
  decltype(&sigattn_paged_plan) paged_plan = nullptr;
  decltype(&sigattn_paged_write) paged_write = nullptr;
  decltype(&sigattn_paged_fwd_workspace_bytes) paged_fwd_workspace_bytes = nullptr;
  decltype(&sigattn_paged_fwd) paged_fwd = nullptr;
};
Api g_api;
bool g_bound = false;
std::vector<int64_t> g_two_pass_dims;
int64_t g_dq_ds_rows = 0;

void check_rc(int rc, const char *what) {
  TORCH_CHECK(rc == SIGATTN_OK, what, " failed: ", g_api.strerror(rc), " (status ", rc, ")");
}

int32_t dtype_code(const Tensor &t) {
  switch (t.scalar_type()) {
    case at::kHalf: return SIGATTN_F16;
    case at::kBFloat16: return SIGATTN_BF16;
    case at::kFloat: return SIGATTN_F32;
    default: TORCH_CHECK(false, "unsupported dtype ", t.scalar_type());
  }
  return -1;
}

const void *ptr_or_null(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// The sequence layout: seq_lens (padded [B, T, H, D], or undefined for
// dense) or cu_seqlens (packed [rows, H, D], with the longest sequences).
struct Layout {
  Tensor slq, slk, cuq, cuk;
  int64_t max_q = 0, max_k = 0;
  bool packed() const { return cuq.defined(); }
};

// The problem over canonical tensors: Q/K/V contiguous, fp32 bias / scale /
// score_mod and int32 seq_lens / cu_seqlens on Q's device (or undefined).
sigattn_problem make_problem(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &bias,
                             const Tensor &score_mod, const Tensor &scale, const Layout &lay, bool causal) {
  sigattn_problem p;
  std::memset(&p, 0, sizeof(p));
  p.abi_version = SIGATTN_ABI_VERSION;
  p.dtype = dtype_code(q);
  if (lay.packed()) {
    // An axis with no rows has no valid positions whatever max_seqlen says.
    p.B = lay.cuq.numel() - 1;
    p.Tq = q.size(0) > 0 ? lay.max_q : 0;
    p.Tk = k.size(0) > 0 ? lay.max_k : 0;
    p.H = q.size(1);
    p.D = q.size(2);
    p.q_stride_t = q.stride(0);
    p.q_stride_h = q.stride(1);
    p.k_stride_t = k.stride(0);
    p.k_stride_h = k.stride(1);
    p.cu_seqlens_q = static_cast<const int32_t *>(lay.cuq.data_ptr());
    p.cu_seqlens_k = static_cast<const int32_t *>(lay.cuk.data_ptr());
    p.rows_q = q.size(0);
    p.rows_k = k.size(0);
    p.kv_heads = k.size(1);
  } else {
    p.B = q.size(0);
    p.Tq = q.size(1);
    p.Tk = k.size(1);
    p.H = q.size(2);
    p.D = q.size(3);
    p.q_stride_b = q.stride(0);
    p.q_stride_t = q.stride(1);
    p.q_stride_h = q.stride(2);
    p.k_stride_b = k.stride(0);
    p.k_stride_t = k.stride(1);
    p.k_stride_h = k.stride(2);
    p.seq_lens_q = static_cast<const int32_t *>(ptr_or_null(lay.slq));
    p.seq_lens_k = static_cast<const int32_t *>(ptr_or_null(lay.slk));
  }
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.bias = static_cast<const float *>(ptr_or_null(bias));
  p.scale = static_cast<const float *>(ptr_or_null(scale));
  p.score_mod = static_cast<const float *>(ptr_or_null(score_mod));
  p.causal = causal ? 1 : 0;
  return p;
}

int compute_units(int dev) {
  static std::atomic<int> cache[64];
  if (dev < 0 || dev >= 64) return 0;
  int n = cache[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return 0;
    cache[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// A uint8 workspace of `bytes` from the caching allocator, or an undefined
// tensor when none is needed or the device cannot hold it.
Tensor workspace(int64_t bytes, const Tensor &like) {
  if (bytes <= 0) return Tensor();
  try {
    return at::empty({bytes}, like.options().dtype(at::kByte));
  } catch (const c10::OutOfMemoryError &) {
    return Tensor();
  }
}

// Mirror of _capi.bwd_workspace_bytes: the two-pass backward's workspace, 0
// for the recompute backward.
int64_t two_pass_bytes(const sigattn_problem &p, int64_t limit, int dev) {
  bool two_pass = false;
  for (int64_t d : g_two_pass_dims) two_pass |= d == p.D;
  if (!two_pass) return 0;
  const int64_t full = (int64_t)g_api.bwd_workspace_bytes(&p);
  if (full <= limit) return full;
  const int64_t per_head = full / p.H;
  if (p.kv_heads != 0 && p.kv_heads != p.H) {
    const int64_t group = p.H / p.kv_heads, most = limit / per_head / group;
    if (most == 0) return 0;
    const int64_t passes = (p.kv_heads + most - 1) / most, per = (p.kv_heads + passes - 1) / passes;
    return per * (p.rows_k / 128) >= 2 * compute_units(dev) ? per * group * per_head : 0;
  }
  const int64_t heads = limit / per_head;
  const int64_t grid = heads * p.B * ((p.Tq + g_dq_ds_rows - 1) / g_dq_ds_rows);
  if (heads == 0 || grid < compute_units(dev)) return 0;
  return heads * per_head;
}

struct SigattnNode : public torch::autograd::Function<SigattnNode> {
  static Tensor forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v,
                        const Tensor &bias, const std::optional<Tensor> &score_mod, const Tensor &scale,
                        const std::optional<Tensor> &seq_lens_q, const std::optional<Tensor> &seq_lens_k,
                        bool causal, int64_t bwd_limit, const std::optional<Tensor> &cu_seqlens_q,
                        const std::optional<Tensor> &cu_seqlens_k, int64_t max_seqlen_q, int64_t max_seqlen_k) {
    const Tensor sm = score_mod.value_or(Tensor());
    const Layout lay{seq_lens_q.value_or(Tensor()), seq_lens_k.value_or(Tensor()), cu_seqlens_q.value_or(Tensor()),
                     cu_seqlens_k.value_or(Tensor()), max_seqlen_q, max_seqlen_k};
    ctx->save_for_backward({q, k, v, bias, scale, sm, lay.slq, lay.slk, lay.cuq, lay.cuk});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["bwd_limit"] = bwd_limit;
    ctx->saved_data["max_seqlen_q"] = max_seqlen_q;
    ctx->saved_data["max_seqlen_k"] = max_seqlen_k;
    // Packed rows with no sequence at all (B = 0) are zeros.
    if (lay.packed() && lay.cuq.numel() == 1) return at::zeros_like(q);
    Tensor out = at::empty_like(q);
    if (out.numel() == 0) return out;
    const c10::DeviceGuard guard(q.device());
    const sigattn_problem p = make_problem(q, k, v, bias, sm, scale, lay, causal);
    const hipStream_t stream = c10::hip::getCurrentHIPStream(q.device().index()).stream();
    int64_t nbytes = (int64_t)g_api.fwd_decode_workspace_bytes(&p);
    Tensor ws = workspace(nbytes, q);
    if (nbytes == 0 || ws.defined()) {
      check_rc(g_api.fwd_decode(&p, out.data_ptr(), ws.defined() ? ws.data_ptr() : nullptr, nbytes, stream),
               "sigattn_fwd");
      return out;
    }
    nbytes = (int64_t)g_api.fwd_workspace_bytes(&p);
    if (nbytes > 0) ws = at::empty({nbytes}, q.options().dtype(at::kByte));
    check_rc(g_api.fwd_ws(&p, out.data_ptr(), ws.defined() ? ws.data_ptr() : nullptr, nbytes, stream),
             "sigattn_fwd");
    return out;
  }

  static tensor_list backward(AutogradContext *ctx, tensor_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &bias = saved[3], &scale = saved[4],
                 &sm = saved[5];
    const Layout lay{saved[6], saved[7], saved[8], saved[9], ctx->saved_data["max_seqlen_q"].toInt(),
                     ctx->saved_data["max_seqlen_k"].toInt()};
    const bool causal = ctx->saved_data["causal"].toBool();
    const int64_t limit = ctx->saved_data["bwd_limit"].toInt();
    Tensor dout = grads[0];
    if (dout.scalar_type() != q.scalar_type() || dout.device() != q.device() || !dout.is_contiguous())
      dout = dout.to(q.device(), q.scalar_type()).contiguous();
    TORCH_CHECK(dout.sizes() == q.sizes(), "dO shape ", dout.sizes(), " != Q shape ", q.sizes());
    const bool no_seqs = lay.packed() && lay.cuq.numel() == 1;  // B = 0: every packed row is outside
    Tensor dq = no_seqs ? at::zeros_like(q) : at::empty_like(q);
    Tensor dk = no_seqs ? at::zeros_like(k) : at::empty_like(k);
    Tensor dv = no_seqs ? at::zeros_like(v) : at::empty_like(v);
    tensor_list result(14);
    result[0] = dq, result[1] = dk, result[2] = dv;  // none for bias, score_mod, ... (no gradient)
    if ((dq.numel() == 0 && dk.numel() == 0) || no_seqs) return result;
    const c10::DeviceGuard guard(q.device());
    const int dev = q.device().index();
    const sigattn_problem p = make_problem(q, k, v, bias, sm, scale, lay, causal);
    const hipStream_t stream = c10::hip::getCurrentHIPStream(dev).stream();
    bool two_pass = false;
    for (int64_t d : g_two_pass_dims) two_pass |= d == p.D;
    const int64_t split = (int64_t)g_api.bwd_split_workspace_bytes(&p);
    if (split > 0 || !two_pass) {
      const Tensor ws = workspace(split, q);
      check_rc(g_api.bwd_split(&p, dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                               ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? ws.numel() : 0, stream),
               "sigattn_bwd_split");
      return result;
    }
    const Tensor ws = workspace(two_pass_bytes(p, limit, dev), q);
    check_rc(g_api.bwd_ws(&p, dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                          ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? ws.numel() : 0, stream),
             "sigattn_bwd_ws");
    return result;
  }
};

Tensor attention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &bias,
                 const std::optional<Tensor> &score_mod, const Tensor &scale,
                 const std::optional<Tensor> &seq_lens_q, const std::optional<Tensor> &seq_lens_k, bool causal,
                 int64_t bwd_limit, const std::optional<Tensor> &cu_seqlens_q,
                 const std::optional<Tensor> &cu_seqlens_k, int64_t max_seqlen_q, int64_t max_seqlen_k) {
  TORCH_CHECK(g_bound, "_sigattn_autograd: bind() was not called");
  TORCH_CHECK(cu_seqlens_q.has_value() == cu_seqlens_k.has_value(),
              "_sigattn_autograd: cu_seqlens_q and cu_seqlens_k go together");
  return SigattnNode::apply(q, k, v, bias, score_mod, scale, seq_lens_q, seq_lens_k, causal, bwd_limit,
                            cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k);
}

// The eager public APIs' calls with canonical arguments, without the Python
// layer's per-call checks and conversions (about 6 of 12 us of host time, which
// is what a small call takes): exact torch.Tensors, contiguous, one gfx950
// device, matching shapes, plain numbers, no environment overrides, no stream
// capture, no function or dispatch mode or functorch transform (which see the
// Python layer's operators, and would put their own tensors among the kept
// constants).  Everything else -- and so every error -- is None, and the Python
// layer takes the call.
struct Quick {
  // Constants [n] on a device, as _capi.device_constant keeps them: made by a
  // blocking copy, at most kMax, never freed (a queued kernel may read one).
  static constexpr size_t kMax = 256;
  static Tensor constant(int64_t n, double value, at::ScalarType type, const at::Device &dev) {
    if (std::isnan(value)) return Tensor();  // has no place in the map's order: it would match any kept value
    static std::mutex mu;
    static auto *kept = new std::map<std::tuple<int, int64_t, double, int>, Tensor>;  // outlives every thread
    const std::tuple<int, int64_t, double, int> key(dev.index(), n, value, (int)type);
    std::lock_guard<std::mutex> lock(mu);
    const auto it = kept->find(key);
    if (it != kept->end()) return it->second;
    if (kept->size() >= kMax) return Tensor();
    const c10::InferenceMode normal(false);  // kept for calls that save it for backward too
    const auto opt = at::TensorOptions().dtype(type);
    const Tensor t = (n < 0 ? at::full({}, value, opt) : at::full({n}, value, opt)).to(dev);
    kept->emplace(key, t);
    return t;
  }
  static bool gfx950(int dev) {
    static std::atomic<int> known[64];  // 0: not looked at, 1: gfx950, 2: another
    if (dev < 0 || dev >= 64) return false;
    int v = known[dev].load(std::memory_order_relaxed);
    if (v == 0) {
      hipDeviceProp_t prop;
      if (hipGetDeviceProperties(&prop, dev) != hipSuccess) return false;
      v = std::strncmp(prop.gcnArchName, "gfx950", 6) == 0 ? 1 : 2;
      known[dev].store(v, std::memory_order_relaxed);
    }
    return v == 1;
  }
  static bool observed() {
    return at::impl::torch_function_mode_enabled() || c10::impl::dispatch_mode_enabled() ||
           c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
  }
  static bool usable() { return g_bound && !observed() && std::getenv("SIGATTN_EAGER_BINDING") == nullptr; }
  // A tensor of unit stride along its last dim.
  static bool strided(const py::object &o, Tensor &t) {
    if (!THPVariable_CheckExact(o.ptr())) return false;
    t = THPVariable_Unpack(o.ptr());
    return t.layout() == at::kStrided && !t.is_neg() && !t.is_conj() && t.dim() > 0 && t.stride(-1) == 1;
  }
  static bool tensor(const py::object &o, Tensor &t) { return strided(o, t) && t.is_contiguous(); }
  // int32, contiguous, n dims, on `dev`.
  static bool ints(const py::object &o, Tensor &t, int64_t dims, const at::Device &dev) {
    return tensor(o, t) && t.scalar_type() == at::kInt && t.dim() == dims && t.device() == dev;
  }
  static bool integer(const py::object &o, int64_t &v) {
    if (!PyLong_CheckExact(o.ptr())) return false;
    int over = 0;
    v = PyLong_AsLongLongAndOverflow(o.ptr(), &over);
    return over == 0;
  }
  static bool float_type(const Tensor &t) {
    const at::ScalarType type = t.scalar_type();
    return type == at::kHalf || type == at::kBFloat16 || type == at::kFloat;
  }
  // No tensor asks for a gradient or carries a forward-mode tangent (level 0 is
  // the only one; a mode that no_grad leaves on).
  static bool no_grad(std::initializer_list<const Tensor *> tensors) {
    for (const Tensor *t : tensors)
      if (t->defined() && ((at::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(0).defined())) return false;
    return true;
  }
  static bool number(const py::object &o, double &v) {
    if (!PyFloat_CheckExact(o.ptr()) && !PyLong_CheckExact(o.ptr())) return false;
    v = PyFloat_AsDouble(o.ptr());
    if (v == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      return false;
    }
    return true;
  }
};

py::object quick(const py::object &query, const py::object &key, const py::object &value,
                 const py::object &seq_lens_k, const py::object &seq_lens_q, bool padded,
                 const py::object &is_causal, const py::object &scale, const py::object &sigmoid_bias,
                 const py::object &score_mod) {
  constexpr int64_t kBwdLimit = (int64_t)2048 << 20;  // _capi._WS_DEFAULT_MB
  const py::object no = py::none();
  Tensor q, k, v, sm, lq, lk;
  if (!g_bound || Quick::observed() || std::getenv("SIGATTN_EAGER_BINDING") != nullptr ||
      std::getenv("SIGATTN_BWD_WORKSPACE_MB") != nullptr || !Quick::tensor(query, q) || !Quick::tensor(key, k) ||
      !Quick::tensor(value, v) || !PyBool_Check(is_causal.ptr()))
    return no;
  const at::ScalarType type = q.scalar_type();
  const at::Device dev = q.device();
  if (q.dim() != 4 || k.dim() != 4 || k.sizes() != v.sizes() || q.numel() == 0 || k.numel() == 0 ||
      (type != at::kHalf && type != at::kBFloat16 && type != at::kFloat) || k.scalar_type() != type ||
      v.scalar_type() != type || !dev.is_cuda() || k.device() != dev || v.device() != dev || !Quick::gfx950(dev.index()))
    return no;
  const int64_t B = q.size(0), Tq = q.size(1), Tk = k.size(1), D = q.size(3);
  if (k.size(0) != B || k.size(2) != q.size(2) || k.size(3) != D || (!padded && Tq != Tk)) return no;
  if (!score_mod.is_none() &&
      (!Quick::tensor(score_mod, sm) || sm.scalar_type() != at::kFloat || sm.device() != dev || sm.dim() != 2 ||
       sm.size(0) != B || sm.size(1) != Tk))
    return no;
  double s = 1.0 / std::sqrt((double)D), bias_value = -std::log((double)Tk);
  if (!scale.is_none() && !Quick::number(scale, s)) return no;
  const bool own_bias = !sigmoid_bias.is_none();
  if (own_bias && !Quick::number(sigmoid_bias, bias_value)) return no;
  const c10::DeviceGuard guard(dev);
  const hipStream_t stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream, &cs) != hipSuccess || cs != hipStreamCaptureStatusNone) return no;
  const auto lens = [&](const py::object &o, int64_t T, Tensor &t) {
    if (o.is_none()) {
      t = Quick::constant(B, (double)T, at::kInt, dev);
      return t.defined();
    }
    return Quick::tensor(o, t) && t.scalar_type() == at::kInt && t.device() == dev && t.dim() == 1 && t.size(0) == B;
  };
  if (padded && (!lens(seq_lens_k, Tk, lk) || !lens(seq_lens_q, Tq, lq))) return no;
  const Tensor st = Quick::constant(-1, s, at::kFloat, dev);
  if (!st.defined()) return no;
  Tensor bias;
  if (padded && !own_bias) {
    bias = at::empty({B}, q.options().dtype(at::kFloat).requires_grad(false));
    check_rc(g_api.default_bias(static_cast<const int32_t *>(lk.data_ptr()), nullptr, B,
                                static_cast<float *>(bias.data_ptr()), stream),
             "sigattn_default_bias");
  } else {
    bias = Quick::constant(B, bias_value, at::kFloat, dev);
    if (!bias.defined()) return no;
  }
  const auto opt = [](const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
  return py::cast(SigattnNode::apply(q, k, v, bias, opt(sm), st, opt(lq), opt(lk), is_causal.ptr() == Py_True, kBwdLimit,
                                     std::nullopt, std::nullopt, 0, 0));
}

// sigmoid_attention_varlen on canonical arguments, or None.
py::object quick_varlen(const py::object &query, const py::object &key, const py::object &value,
                        const py::object &cu_seqlens_q, const py::object &cu_seqlens_k, const py::object &max_seqlen_q,
                        const py::object &max_seqlen_k, const py::object &is_causal, const py::object &scale,
                        const py::object &sigmoid_bias, const py::object &score_mod) {
  const py::object no = py::none();
  Tensor q, k, v, sm, cq, ck;
  int64_t mq = 0, mk = 0;
  if (!g_bound || Quick::observed() || std::getenv("SIGATTN_EAGER_BINDING") != nullptr ||
      std::getenv("SIGATTN_BWD_WORKSPACE_MB") != nullptr || !Quick::tensor(query, q) || !Quick::tensor(key, k) ||
      !Quick::tensor(value, v) || !PyBool_Check(is_causal.ptr()) || !Quick::integer(max_seqlen_q, mq) ||
      !Quick::integer(max_seqlen_k, mk) || mq < 0 || mk < 0)
    return no;
  const at::Device dev = q.device();
  if (q.dim() != 3 || k.dim() != 3 || k.sizes() != v.sizes() || q.numel() == 0 || k.numel() == 0 ||
      !Quick::float_type(q) || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() ||
      !dev.is_cuda() || k.device() != dev || v.device() != dev || !Quick::gfx950(dev.index()))
    return no;
  const int64_t H = q.size(1), Hkv = k.size(1), D = q.size(2);
  if (k.size(2) != D || H % Hkv != 0 || !Quick::ints(cu_seqlens_q, cq, 1, dev) ||
      !Quick::ints(cu_seqlens_k, ck, 1, dev) || cq.numel() < 2 || ck.numel() != cq.numel())
    return no;
  if (!score_mod.is_none() && (!Quick::tensor(score_mod, sm) || sm.scalar_type() != at::kFloat || sm.device() != dev ||
                               sm.dim() != 1 || sm.size(0) != k.size(0)))
    return no;
  double s = 1.0 / std::sqrt((double)D), bias_value = 0.0;
  if (!scale.is_none() && !Quick::number(scale, s)) return no;
  const bool own_bias = !sigmoid_bias.is_none();
  if (own_bias && !Quick::number(sigmoid_bias, bias_value)) return no;
  const c10::DeviceGuard guard(dev);
  const hipStream_t stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream, &cs) != hipSuccess || cs != hipStreamCaptureStatusNone) return no;
  const int64_t B = cq.numel() - 1;
  const Tensor st = Quick::constant(-1, s, at::kFloat, dev);
  if (!st.defined()) return no;
  Tensor bias;
  if (own_bias) {
    bias = Quick::constant(B, bias_value, at::kFloat, dev);
    if (!bias.defined()) return no;
  } else {
    bias = at::empty({B}, q.options().dtype(at::kFloat).requires_grad(false));
    check_rc(g_api.default_bias(nullptr, static_cast<const int32_t *>(ck.data_ptr()), B,
                                static_cast<float *>(bias.data_ptr()), stream),
             "sigattn_default_bias");
  }
  const int64_t limit = (int64_t)(H == Hkv ? 2048 : 8192) << 20;  // _capi._WS_DEFAULT_MB, _WS_DEFAULT_GROUPED_MB
  return py::cast(SigattnNode::apply(q, k, v, bias, sm.defined() ? std::optional<Tensor>(sm) : std::nullopt, st,
                                     std::nullopt, std::nullopt, is_causal.ptr() == Py_True, limit, cq, ck, mq, mk));
}

// Tells autograd of a tensor that was changed in place.
void changed(const Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

bool page_size_ok(int64_t n) { return n >= 16 && n <= (1 << 20) && (n & (n - 1)) == 0; }

// The paged cache's calls on canonical arguments (int32 tensors of one gfx950
// device, matching shapes, nothing that asks for a gradient), or None where the
// Python layer has to take the call.
py::object quick_plan(const py::object &context_lens, const py::object &new_lens, const py::object &block_table,
                      const py::object &free_pages, const py::object &page_size, const py::object &num_tokens) {
  const py::object no = py::none();
  Tensor ctx, add, table, pages;
  int64_t ps = 0, n = 0;
  if (!Quick::usable() || !Quick::strided(block_table, table) || table.scalar_type() != at::kInt ||
      table.dim() != 2 || !table.is_cuda() || !Quick::integer(page_size, ps) || !Quick::integer(num_tokens, n) ||
      !page_size_ok(ps) || n < 0)
    return no;
  const at::Device dev = table.device();
  const int64_t B = table.size(0);
  if (!Quick::gfx950(dev.index()) || B > SIGATTN_PLAN_MAX_BATCH || (B > 1 && table.stride(0) < table.size(1)) ||
      !Quick::ints(context_lens, ctx, 1, dev) || !Quick::ints(new_lens, add, 1, dev) ||
      !Quick::ints(free_pages, pages, 1, dev) || ctx.size(0) != B || add.size(0) != B)
    return no;
  const c10::DeviceGuard guard(dev);
  const auto opt = table.options();
  const Tensor slots = at::empty({n}, opt), cu = at::empty({B + 1}, opt), lens = at::empty({B}, opt),
               needed = at::empty({}, opt);
  const auto p = [](const Tensor &t) { return static_cast<int32_t *>(t.data_ptr()); };
  check_rc(g_api.paged_plan(B, p(ctx), p(add), p(table), table.stride(0), table.size(1), p(pages), pages.numel(), ps, n,
                            p(slots), p(cu), p(lens), p(needed),
                            c10::hip::getCurrentHIPStream(dev.index()).stream()),
           "sigattn_paged_plan");
  changed(table);
  return py::make_tuple(slots, cu, lens, needed);
}

// The caches: same shape, strides and type, pages the kernels take.
bool quick_caches(const py::object &ko, const py::object &vo, Tensor &k, Tensor &v) {
  return Quick::strided(ko, k) && Quick::strided(vo, v) && k.dim() == 4 && k.sizes() == v.sizes() &&
         k.strides() == v.strides() && Quick::float_type(k) && v.scalar_type() == k.scalar_type() && k.is_cuda() &&
         v.device() == k.device() && page_size_ok(k.size(1)) && Quick::gfx950(k.device().index());
}

bool quick_write(const py::object &key, const py::object &value, const py::object &key_cache,
                 const py::object &value_cache, const py::object &slot_mapping) {
  Tensor k, v, kc, vc, slots;
  if (!Quick::usable() || !quick_caches(key_cache, value_cache, kc, vc) || !Quick::strided(key, k) ||
      !Quick::strided(value, v))
    return false;
  const at::Device dev = kc.device();
  if (k.dim() != 3 || k.sizes() != v.sizes() || k.strides() != v.strides() || k.scalar_type() != kc.scalar_type() ||
      v.scalar_type() != kc.scalar_type() || k.device() != dev || v.device() != dev || k.size(1) != kc.size(2) ||
      k.size(2) != kc.size(3) || !Quick::ints(slot_mapping, slots, 1, dev) || slots.size(0) != k.size(0) ||
      !Quick::no_grad({&k, &v, &kc, &vc}))
    return false;
  for (int i = 0; i < 3; ++i)
    if (kc.size(i) > 1 && kc.stride(i) == 0) return false;
  sigattn_paged_rows r;
  std::memset(&r, 0, sizeof(r));
  r.esize = (int32_t)k.element_size();
  r.rows = k.size(0), r.kv_heads = k.size(1), r.D = k.size(2);
  r.src_stride_t = k.stride(0), r.src_stride_h = k.stride(1);
  r.cache_stride_p = kc.stride(0), r.cache_stride_t = kc.stride(1), r.cache_stride_h = kc.stride(2);
  r.num_pages = kc.size(0), r.page_size = kc.size(1);
  r.k = k.data_ptr(), r.v = v.data_ptr(), r.k_cache = kc.data_ptr(), r.v_cache = vc.data_ptr();
  r.slot_mapping = static_cast<const int32_t *>(slots.data_ptr());
  const c10::DeviceGuard guard(dev);
  check_rc(g_api.paged_write(&r, c10::hip::getCurrentHIPStream(dev.index()).stream()), "sigattn_paged_write");
  changed(kc), changed(vc);
  return true;
}

py::object quick_paged(const py::object &query, const py::object &key_cache, const py::object &value_cache,
                       const py::object &block_table, const py::object &seq_lens_k, const py::object &cu_seqlens_q,
                       const py::object &max_seqlen_q, const py::object &is_causal, const py::object &scale,
                       const py::object &sigmoid_bias, const py::object &score_mod) {
  const py::object no = py::none();
  Tensor q, kc, vc, table, lens, cu, sm;
  if (!Quick::usable() || !Quick::strided(query, q) || !quick_caches(key_cache, value_cache, kc, vc) ||
      !Quick::strided(block_table, table) || !PyBool_Check(is_causal.ptr()))
    return no;
  const at::Device dev = q.device();
  int64_t mq = q.size(0);
  if (q.dim() != 3 || q.scalar_type() != kc.scalar_type() || kc.device() != dev || q.numel() == 0 ||
      q.size(2) != kc.size(3) || kc.size(2) == 0 || q.size(1) % kc.size(2) != 0 || table.dim() != 2 ||
      table.scalar_type() != at::kInt || table.device() != dev)
    return no;
  const int64_t B = table.size(0);
  if (!Quick::ints(seq_lens_k, lens, 1, dev) || lens.size(0) != B || !Quick::ints(cu_seqlens_q, cu, 1, dev) ||
      cu.size(0) != B + 1 || (!max_seqlen_q.is_none() && (!Quick::integer(max_seqlen_q, mq) || mq < 0)))
    return no;
  if (!score_mod.is_none() && (!Quick::tensor(score_mod, sm) || sm.scalar_type() != at::kFloat || sm.device() != dev ||
                               sm.dim() != 2 || sm.size(0) != B || sm.size(1) != table.size(1) * kc.size(1)))
    return no;
  double s = 1.0 / std::sqrt((double)q.size(2)), bias = 0.0;
  if (!scale.is_none() && !Quick::number(scale, s)) return no;
  const bool own_bias = !sigmoid_bias.is_none();
  if (own_bias && !Quick::number(sigmoid_bias, bias)) return no;
  if (!Quick::no_grad({&q, &kc, &vc, &sm})) return no;
  sigattn_paged_problem p;
  std::memset(&p, 0, sizeof(p));
  p.abi_version = SIGATTN_ABI_VERSION;
  p.dtype = dtype_code(q);
  p.B = B, p.H = q.size(1), p.kv_heads = kc.size(2), p.D = q.size(2), p.rows_q = q.size(0), p.max_seqlen_q = mq;
  p.num_pages = kc.size(0), p.page_size = kc.size(1), p.max_pages = table.size(1);
  p.q_stride_t = q.stride(0), p.q_stride_h = q.stride(1);
  p.k_stride_p = kc.stride(0), p.k_stride_t = kc.stride(1), p.k_stride_h = kc.stride(2);
  p.table_stride = table.stride(0);
  p.q = q.data_ptr(), p.k_cache = kc.data_ptr(), p.v_cache = vc.data_ptr();
  p.block_table = static_cast<const int32_t *>(table.data_ptr());
  p.seq_lens_k = static_cast<const int32_t *>(lens.data_ptr());
  p.cu_seqlens_q = static_cast<const int32_t *>(cu.data_ptr());
  if (sm.defined()) p.score_mod = static_cast<const float *>(sm.data_ptr()), p.mod_stride = sm.stride(0);
  p.scale = (float)s, p.bias = (float)bias;
  p.own_bias = own_bias, p.causal = is_causal.ptr() == Py_True;
  const c10::DeviceGuard guard(dev);
  const Tensor out = at::empty(q.sizes(), q.options().requires_grad(false));
  const Tensor ws = workspace((int64_t)g_api.paged_fwd_workspace_bytes(&p), q);  // without it: unsplit
  check_rc(g_api.paged_fwd(&p, out.data_ptr(), ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? ws.numel() : 0,
                           c10::hip::getCurrentHIPStream(dev.index()).stream()),
           "sigattn_paged_fwd");
  return py::cast(out);
}

template <class F> void bind_one(F &dst, const py::dict &fns, const char *name) {
  TORCH_CHECK(fns.contains(name), "_sigattn_autograd.bind: missing ", name);
  dst = reinterpret_cast<F>(fns[name].cast<uintptr_t>());
}

void bind(const py::dict &fns, const std::vector<int64_t> &two_pass_dims, int64_t dq_ds_rows) {
  Api api;
  bind_one(api.strerror, fns, "sigattn_strerror");
  bind_one(api.fwd_workspace_bytes, fns, "sigattn_fwd_workspace_bytes");
  bind_one(api.fwd_ws, fns, "sigattn_fwd_ws");
  bind_one(api.fwd_decode_workspace_bytes, fns, "sigattn_fwd_decode_workspace_bytes");
  bind_one(api.fwd_decode, fns, "sigattn_fwd_decode");
  bind_one(api.bwd_workspace_bytes, fns, "sigattn_bwd_workspace_bytes");
  bind_one(api.bwd_ws, fns, "sigattn_bwd_ws");
  bind_one(api.default_bias, fns, "sigattn_default_bias");
  bind_one(api.bwd_split_workspace_bytes, fns, "sigattn_bwd_split_workspace_bytes");
  bind_one(api.bwd_split, fns, "sigattn_bwd_split");
  bind_one(api.paged_plan, fns, "sigattn_paged_plan");
  bind_one(api.paged_write, fns, "sigattn_paged_write");
  bind_one(api.paged_fwd_workspace_bytes, fns, "sigattn_paged_fwd_workspace_bytes");
  bind_one(api.paged_fwd, fns, "sigattn_paged_fwd");
  TORCH_CHECK(dq_ds_rows > 0, "_sigattn_autograd.bind: dq_ds_rows must be positive");
  g_api = api;
  g_two_pass_dims = two_pass_dims;
  g_dq_ds_rows = dq_ds_rows;
  g_bound = true;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "C++ autograd node of sigmoid_attention / sigmoid_attention_padded over libsigattn";
  m.def("bind", &bind, "Entry point addresses of libsigattn (name -> address), two-pass head dims, "
        "query rows per dQ-from-dS workgroup");
  m.def("quick", &quick,
        "sigmoid_attention (padded False) or sigmoid_attention_padded on canonical arguments, or None where the "
        "Python layer has to take the call",
        py::arg("query"), py::arg("key"), py::arg("value"), py::arg("seq_lens_k"), py::arg("seq_lens_q"),
        py::arg("padded"), py::arg("is_causal"), py::arg("scale"), py::arg("sigmoid_bias"), py::arg("score_mod"));
  m.def("quick_varlen", &quick_varlen, "sigmoid_attention_varlen on canonical arguments, or None");
  m.def("quick_plan", &quick_plan, "paged_plan's new tensors on canonical arguments, or None");
  m.def("quick_write", &quick_write, "paged_cache_write on canonical arguments: whether it took the call");
  m.def("quick_paged", &quick_paged, "sigmoid_attention_paged on canonical arguments, or None");
  m.def("attention", &attention,
        "Forward with autograd; arguments are the canonical tensors of _capi._prepare (and _prepare_packed "
        "for the packed layout, with the longest sequences)",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("bias"), py::arg("score_mod"), py::arg("scale"),
        py::arg("seq_lens_q"), py::arg("seq_lens_k"), py::arg("causal"), py::arg("bwd_limit"),
        py::arg("cu_seqlens_q") = py::none(), py::arg("cu_seqlens_k") = py::none(), py::arg("max_seqlen_q") = 0,
        py::arg("max_seqlen_k") = 0);
}
