// Torch front of the norm, the int8 product and the layer for a few tokens:
// argument checks, outputs, the autograd node and the calls of the C ABI, in
// one native call. These operators are a few microseconds of GPU time on a
// token's rows, and the same steps in Python took longer than that (one row of
// 2048 columns normed: 5.8 us of host time against 10; 1021 rows forward and
// backward through autograd: 42 against 115).
//
// The C ABI's functions are looked up in the library that the package has
// loaded; nothing here is linked against it.
#include <dlfcn.h>

#include <sstream>

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "../../include/megamoe.h"

namespace {

using at::ScalarType;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kMaxHidden = 32768;
constexpr int64_t kMaxK = (int64_t(1) << 17) - 1;
constexpr int64_t kMaxStride = int64_t(1) << 23;

// ------------------------------------------------------------------ the library
struct Abi {
  decltype(&mm_rms_norm) rms_norm = nullptr;
  decltype(&mm_rms_norm_bwd) rms_norm_bwd = nullptr;
  decltype(&mm_rms_norm_bwd_workspace_bytes) rms_norm_bwd_workspace_bytes = nullptr;
  decltype(&mm_quantize_rows) quantize_rows = nullptr;
  decltype(&mm_int8_matmul) int8_matmul = nullptr;
  decltype(&mm_moe_few_scratch_bytes) moe_few_scratch_bytes = nullptr;
  decltype(&mm_moe_few) moe_few = nullptr;
  decltype(&mm_moe_few_int8) moe_few_int8 = nullptr;
  decltype(&mm_last_error) last_error = nullptr;
  PyObject* error = nullptr;  // the package's exception class
};
Abi entry;

template <class F>
void look_up(void* lib, const char* name, F& f) {
  f = reinterpret_cast<F>(dlsym(lib, name));
  if (!f) throw std::runtime_error(std::string("libmegamoe.so does not export ") + name);
}

void bind(const std::string& path, const py::object& error) {
  void* lib = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  if (!lib) throw std::runtime_error(std::string("cannot load ") + path + ": " + dlerror());
  look_up(lib, "mm_rms_norm", entry.rms_norm);
  look_up(lib, "mm_rms_norm_bwd", entry.rms_norm_bwd);
  look_up(lib, "mm_rms_norm_bwd_workspace_bytes", entry.rms_norm_bwd_workspace_bytes);
  look_up(lib, "mm_quantize_rows", entry.quantize_rows);
  look_up(lib, "mm_int8_matmul", entry.int8_matmul);
  look_up(lib, "mm_moe_few_scratch_bytes", entry.moe_few_scratch_bytes);
  look_up(lib, "mm_moe_few", entry.moe_few);
  look_up(lib, "mm_moe_few_int8", entry.moe_few_int8);
  look_up(lib, "mm_last_error", entry.last_error);
  entry.error = error.inc_ref().ptr();  // kept for the life of the process
}

// A failed call raises the package's exception. The backward runs without the
// interpreter's lock, so the message is carried by a C++ exception there.
struct CallError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void check(const char* name, int rc) {
  if (rc == MM_OK) return;
  std::ostringstream s;
  s << name << " failed (" << rc << "): " << entry.last_error();
  throw CallError(s.str());
}

// ------------------------------------------------------------------ checks
template <class E, class... A>
[[noreturn]] void refuse(const A&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw E(s.str());
}
#define CHECK_TYPE(cond, ...) \
  if (!(cond)) refuse<py::type_error>(__VA_ARGS__)
#define CHECK_VALUE(cond, ...) \
  if (!(cond)) refuse<py::value_error>(__VA_ARGS__)

bool is_float(ScalarType t) { return t == at::kBFloat16 || t == at::kHalf || t == at::kFloat; }
bool is_eight_bits(ScalarType t) { return t == at::kChar || t == at::kFloat8_e4m3fn; }

int32_t type_code(ScalarType t) {
  switch (t) {
    case at::kBFloat16: return MM_T_BF16;
    case at::kHalf: return MM_T_FP16;
    case at::kFloat: return MM_T_FP32;
    case at::kChar: return MM_T_INT8;
    case at::kFloat8_e4m3fn: return MM_T_E4M3;
    default: return -1;
  }
}

void check_float(const char* name, const Tensor& t) {
  CHECK_TYPE(is_float(t.scalar_type()), name, " must be bfloat16, float16 or float32, got ", t.scalar_type());
}

void check_device(const char* name, const Tensor& t) {
  CHECK_VALUE(t.is_cuda(), name, " must be a HIP device tensor");
}

// Forward-mode derivatives do not exist here; a tangent would be lost silently.
void check_no_tangent(const char* op, std::initializer_list<const OptTensor*> tensors) {
  for (const OptTensor* t : tensors)
    CHECK_VALUE(!*t || !(*t)->_fw_grad(0).defined(), op, " has no forward-mode derivative");
}

void check_vector(const char* name, const Tensor& t, int64_t n) {
  CHECK_VALUE(t.dim() == 1 && t.size(0) == n && t.is_contiguous(), name, " must be contiguous with shape (", n,
              ",), got ", t.sizes());
}

// [..., columns] as evenly spaced rows.
struct Rows {
  const void* data;
  int64_t ld, rows = 1;
  Rows(const char* name, const Tensor& t) : data(t.const_data_ptr()), ld(t.size(-1)) {
    CHECK_VALUE(ld <= 1 || t.stride(-1) == 1, name, " must have unit column stride");
    bool spaced = false;
    int64_t next = 0;  // the stride that the next axis outwards has to have
    for (int64_t i = t.dim() - 2; i >= 0; --i) {
      rows *= t.size(i);
      if (t.size(i) == 1) continue;
      if (!spaced) ld = t.stride(i);
      CHECK_VALUE(!spaced || t.stride(i) == next || t.numel() == 0, "the rows of ", name,
                  " must be evenly spaced in memory");
      spaced = true;
      next = t.stride(i) * t.size(i);
    }
  }
};

Tensor empty_as(const Tensor& like, ScalarType dtype) {
  return at::empty_like(like, like.options().dtype(dtype), at::MemoryFormat::Contiguous);
}

mm_stream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

const void* data_or_null(const OptTensor& t) { return t ? t->const_data_ptr() : nullptr; }
int32_t type_or_zero(const OptTensor& t) { return t ? type_code(t->scalar_type()) : 0; }

// ------------------------------------------------------------------ norm
struct NormOut {
  Tensor y, scale, h, rstd;
};

NormOut norm_forward(const Tensor& x, const OptTensor& weight, const OptTensor& residual, double eps, ScalarType out,
                     bool keep_rstd) {
  const Rows rx("x", x);
  NormOut o;
  const void* res = nullptr;
  int64_t ldr = 0;
  int32_t h_type = type_code(x.scalar_type());
  if (residual) {
    const Rows rr("residual", *residual);
    res = rr.data;
    ldr = rr.ld;
    h_type = type_code(residual->scalar_type());
    o.h = empty_as(*residual, residual->scalar_type());
  }
  o.y = empty_as(x, out);
  if (is_eight_bits(out)) o.scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  if (keep_rstd) o.rstd = at::empty({rx.rows}, x.options().dtype(at::kFloat));
  if (!rx.rows) return o;
  const c10::DeviceGuard guard(x.device());
  check("mm_rms_norm",
        entry.rms_norm(rx.data, rx.ld, type_code(x.scalar_type()), res, ldr, h_type, data_or_null(weight),
                     type_or_zero(weight), rx.rows, static_cast<int32_t>(x.size(-1)), static_cast<float>(eps),
                     residual ? o.h.data_ptr() : nullptr, o.y.data_ptr(), type_code(out),
                     o.scale.defined() ? o.scale.data_ptr<float>() : nullptr,
                     keep_rstd ? o.rstd.data_ptr<float>() : nullptr, stream_of(x)));
  return o;
}

// The gradients from a second backward on would be silently constant, so they
// raise when one is asked for.
Tensor once_only(Tensor grad) {
  if (!grad.defined() || !at::GradMode::is_enabled()) return grad;
  torch::autograd::DelayedError raise("rms_norm is differentiable once", 1);
  return std::move(raise({grad.detach().requires_grad_(true)})[0]);
}

// The engine hands a gradient over on the stream of the node that takes it. A
// leaf's node keeps the stream of the first graph that used it while that
// graph lives; where this is the default stream, which cannot be captured, the
// hand-over would break a capture, and the process with it.
void check_capture(const torch::autograd::Node& node, const at::Device& device) {
  if (c10::hip::getCurrentHIPStream(device.index()).stream() == nullptr) return;
  for (const torch::autograd::Edge& e : node.next_edges()) {
    if (!e.is_valid()) continue;
    const auto stream = e.function->stream();
    if (stream && stream->id() == 0 && c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
      throw CallError("rms_norm: this backward cannot be captured: a graph that was built on the default stream still "
                      "uses an input; drop that graph, or build it on the stream of the capture");
  }
}

struct RMSNorm : torch::autograd::Function<RMSNorm> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x,
                                                const OptTensor& weight, const OptTensor& residual, double eps) {
    NormOut o = norm_forward(x, weight, residual, eps, x.scalar_type(), true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({residual ? o.h : x, weight ? *weight : Tensor(), o.rstd});
    ctx->saved_data["x_dtype"] = static_cast<int64_t>(x.scalar_type());
    ctx->saved_data["residual"] = residual.has_value();
    if (residual) return {o.y, o.h};
    return {o.y};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &h = saved[0], &rstd = saved[2];
    check_capture(*torch::autograd::get_current_node(), h.device());
    OptTensor weight;
    if (saved[1].defined()) weight = saved[1];
    const bool residual = ctx->saved_data["residual"].toBool();
    const ScalarType x_dtype = static_cast<ScalarType>(ctx->saved_data["x_dtype"].toInt());
    Tensor dy = grads[0], dh = residual ? grads[1] : Tensor();
    if (!dy.defined() && !dh.defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    // a gradient comes in any layout (an expanded scalar, a transposed view)
    dy = dy.defined() ? dy.contiguous() : at::zeros(h.sizes(), h.options().dtype(x_dtype));
    if (dh.defined()) dh = dh.contiguous();
    const bool want_dw = weight && ctx->needs_input_grad(1);
    const bool want_dres = residual && ctx->needs_input_grad(weight ? 2 : 1);
    const Rows rh("h", h);
    const int32_t hidden = static_cast<int32_t>(h.size(-1)), xt = type_code(x_dtype), ht = type_code(h.scalar_type());
    Tensor dx = empty_as(h, x_dtype), dres, dw, workspace;
    if (want_dres) dres = ht == xt ? dx : empty_as(h, h.scalar_type());
    size_t bytes = 0;
    if (want_dw) {
      bytes = entry.rms_norm_bwd_workspace_bytes(rh.rows, hidden);
      dw = empty_as(*weight, weight->scalar_type());
      workspace = at::empty({static_cast<int64_t>(bytes)}, h.options().dtype(at::kByte));
    }
    if (rh.rows || want_dw) {
      const c10::DeviceGuard guard(h.device());
      check("mm_rms_norm_bwd",
            entry.rms_norm_bwd(dy.const_data_ptr(), hidden, dh.defined() ? dh.const_data_ptr() : nullptr, hidden, rh.data,
                             rh.ld, data_or_null(weight), type_or_zero(weight), rstd.const_data_ptr<float>(), xt, ht,
                             rh.rows, hidden, dx.data_ptr(), want_dres && ht != xt ? dres.data_ptr() : nullptr,
                             want_dw ? dw.data_ptr() : nullptr, want_dw ? workspace.data_ptr() : nullptr, bytes,
                             stream_of(h)));
    }
    return {once_only(dx), once_only(dw), once_only(dres), Tensor()};
  }
};

bool wants_grad(std::initializer_list<const OptTensor*> tensors) {
  for (const OptTensor* t : tensors)
    if (*t && (*t)->requires_grad()) return at::GradMode::is_enabled();
  return false;
}

py::object rms_norm(const Tensor& x, const OptTensor& weight, const OptTensor& residual, double eps,
                    std::optional<ScalarType> out_dtype) {
  const ScalarType dtype = x.scalar_type();
  check_float("x", x);
  CHECK_VALUE(x.dim() > 0, "x must have shape [..., hidden]");
  const int64_t hidden = x.size(-1);
  CHECK_VALUE(hidden >= 1 && hidden <= kMaxHidden, "x must have 1 to ", kMaxHidden, " columns, got ", hidden);
  if (weight) {
    check_float("weight", *weight);
    check_vector("weight", *weight, hidden);
    CHECK_VALUE(weight->device() == x.device(), "weight and x must be on the same device");
  }
  if (residual) {
    CHECK_TYPE(residual->scalar_type() == dtype || residual->scalar_type() == at::kFloat, "residual must use ", dtype,
               " or Float, got ", residual->scalar_type());
    CHECK_VALUE(residual->sizes() == x.sizes(), "residual must have shape ", x.sizes(), ", got ", residual->sizes());
    CHECK_VALUE(residual->device() == x.device(), "residual and x must be on the same device");
  }
  CHECK_VALUE(eps >= 0.0, "eps must not be negative, got ", eps);
  const ScalarType out = out_dtype.value_or(dtype);
  CHECK_TYPE(out == dtype || is_eight_bits(out), "out_dtype must be ", dtype, ", int8 or float8_e4m3fn, got ", out);
  const OptTensor ox(x);
  const bool needs_grad = wants_grad({&ox, &weight, &residual}), eight = is_eight_bits(out);
  CHECK_VALUE(!eight || !needs_grad,
              "an 8-bit output carries no gradient; call under torch.no_grad() or on detached inputs");
  check_no_tangent("rms_norm", {&ox, &weight, &residual});
  check_device("x", x);
  if (needs_grad) {
    auto o = RMSNorm::apply(x, weight, residual, eps);
    if (residual) return py::make_tuple(std::move(o[0]), std::move(o[1]));
    return py::cast(std::move(o[0]));
  }
  NormOut o = norm_forward(x, weight, residual, eps, out, false);
  if (!eight && !residual) return py::cast(std::move(o.y));
  if (!eight) return py::make_tuple(std::move(o.y), std::move(o.h));
  if (!residual) return py::make_tuple(std::move(o.y), std::move(o.scale));
  return py::make_tuple(std::move(o.y), std::move(o.scale), std::move(o.h));
}

py::tuple quantize_rows(const Tensor& x, ScalarType dtype) {
  check_float("x", x);
  CHECK_VALUE(x.dim() > 0, "x must have shape [..., columns]");
  CHECK_VALUE(x.size(-1) >= 1 && x.size(-1) <= kMaxHidden, "x must have 1 to ", kMaxHidden, " columns, got ", x.size(-1));
  CHECK_TYPE(is_eight_bits(dtype), "dtype must be int8 or float8_e4m3fn, got ", dtype);
  CHECK_VALUE(!x.requires_grad() || !at::GradMode::is_enabled(),
              "an 8-bit output carries no gradient; call under torch.no_grad() or on a detached input");
  const OptTensor ox(x);
  check_no_tangent("quantize_rows", {&ox});
  check_device("x", x);
  const Rows r("x", x);
  Tensor q = empty_as(x, dtype);
  Tensor scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  if (r.rows) {
    const c10::DeviceGuard guard(x.device());
    check("mm_quantize_rows", entry.quantize_rows(r.data, r.ld, type_code(x.scalar_type()), r.rows,
                                                static_cast<int32_t>(x.size(-1)), q.data_ptr(), type_code(dtype),
                                                scale.data_ptr<float>(), stream_of(x)));
  }
  return py::make_tuple(std::move(q), std::move(scale));
}

// ------------------------------------------------------------------ int8 product
Tensor int8_matmul(const Tensor& a, const Tensor& b, const Tensor& a_scale, const Tensor& b_scale,
                   const OptTensor& bias, ScalarType out_dtype) {
  CHECK_TYPE(a.scalar_type() == at::kChar && b.scalar_type() == at::kChar, "a and b must be int8, got ",
             a.scalar_type(), " and ", b.scalar_type());
  CHECK_VALUE(a.dim() > 0 && b.dim() == 2, "a must have shape [..., K] and b [N, K], got ", a.sizes(), " and ", b.sizes());
  const int64_t n = b.size(0), k = b.size(1), ldb = b.stride(0);
  CHECK_VALUE(a.size(-1) == k, "a has ", a.size(-1), " columns, b has ", k);
  CHECK_VALUE(k >= 1 && k <= kMaxK && n >= 1, "b must have shape [N, K] with N >= 1 and 1 <= K <= ", kMaxK, ", got ",
              b.sizes());
  CHECK_VALUE(k == 1 || b.stride(1) == 1, "b must have unit column stride ([N, K], K contiguous)");
  CHECK_VALUE(n == 1 || (ldb >= k && ldb <= kMaxStride), "the rows of b must be ", k, " to ", kMaxStride,
              " elements apart (no overlap), got ", ldb);
  CHECK_TYPE(a_scale.scalar_type() == at::kFloat && b_scale.scalar_type() == at::kFloat,
             "a_scale and b_scale must be float32, got ", a_scale.scalar_type(), " and ", b_scale.scalar_type());
  CHECK_VALUE(a_scale.sizes() == a.sizes().slice(0, a.dim() - 1) && a_scale.is_contiguous(),
              "a_scale must be contiguous with shape ", a.sizes().slice(0, a.dim() - 1), ", got ", a_scale.sizes());
  check_vector("b_scale", b_scale, n);
  if (bias) {
    check_float("bias", *bias);
    check_vector("bias", *bias, n);
  }
  CHECK_VALUE(b.device() == a.device() && a_scale.device() == a.device() && b_scale.device() == a.device() &&
                  (!bias || bias->device() == a.device()),
              "all operands must be on the device of a");
  CHECK_TYPE(is_float(out_dtype), "out_dtype must be bfloat16, float16 or float32, got ", out_dtype);
  const OptTensor sa(a_scale), sb(b_scale);
  CHECK_VALUE(!wants_grad({&sa, &sb, &bias}),
              "int8_matmul carries no gradient; call under torch.no_grad() or on detached operands");
  check_no_tangent("int8_matmul", {&sa, &sb, &bias});
  check_device("a", a);
  const Rows ra("a", a);
  CHECK_VALUE(ra.rows <= 1 || (ra.ld >= k && ra.ld <= kMaxStride), "the rows of a must be ", k, " to ", kMaxStride,
              " elements apart (no overlap), got ", ra.ld);
  Tensor out;
  if (a.dim() == 2) {
    out = at::empty({ra.rows, n}, a.options().dtype(out_dtype));
  } else {
    auto sizes = a.sizes().vec();
    sizes.back() = n;
    out = at::empty(sizes, a.options().dtype(out_dtype));
  }
  if (ra.rows) {
    const c10::DeviceGuard guard(a.device());
    check("mm_int8_matmul",
          entry.int8_matmul(static_cast<const int8_t*>(ra.data), ra.ld, b.const_data_ptr<int8_t>(), ldb,
                          a_scale.const_data_ptr<float>(), b_scale.const_data_ptr<float>(), data_or_null(bias),
                          type_or_zero(bias), ra.rows, n, k, out.data_ptr(), n, type_code(out_dtype), stream_of(a)));
  }
  return out;
}

// ------------------------------------------------------------------ a few tokens
// The layer of an operator: its sizes and its activation.
struct Layer {
  int64_t most_tokens, top_k, experts, hidden;
  int32_t act_kind;
  float beta, linear_beta, limit;
};

bool is(const Tensor& t, ScalarType dtype, at::IntArrayRef sizes, const Tensor& like) {
  return t.scalar_type() == dtype && t.sizes() == sizes && t.device() == like.device();
}
bool is_whole(const Tensor& t, ScalarType dtype, at::IntArrayRef sizes, const Tensor& like) {
  return is(t, dtype, sizes, like) && t.is_contiguous();
}

// Tokens of operands that fit the layer; -1 where the caller has to say what is
// wrong with them.
int64_t few_tokens(const Layer& l, const Tensor& x, ScalarType x_type, const Tensor& selected, const Tensor& weights,
                   int64_t inter) {
  if (!x.is_cuda() || x.dim() != 2 || l.hidden % 128 || inter <= 0 || inter % 128) return -1;
  const int64_t tokens = x.size(0);
  const bool ok = tokens <= l.most_tokens && is_whole(x, x_type, {tokens, l.hidden}, x) &&
                  is_whole(selected, at::kInt, {tokens, l.top_k}, x) && is_whole(weights, at::kFloat, {tokens, l.top_k}, x);
  return ok ? tokens : -1;
}

// No backward exists: a gradient asked for would be lost silently, and a tangent.
void check_detached(const char* op, std::initializer_list<const Tensor*> tensors) {
  const bool recording = at::GradMode::is_enabled();
  for (const Tensor* t : tensors) {
    CHECK_VALUE(!recording || !t->requires_grad(), op,
                " carries no gradient; call under torch.no_grad() or on detached operands, or use MegaMoEFunction");
    CHECK_VALUE(!t->_fw_grad(0).defined(), op, " has no forward-mode derivative");
  }
}

// [tokens, hidden] of the layer, or None for operands that do not fit it (none
// fit a null layer).
std::optional<Tensor> few_forward(const Layer* layer, const Tensor& x, const Tensor& selected, const Tensor& gate_up,
                                  const Tensor& down, const Tensor& weights) {
  check_detached("forward_few", {&x, &gate_up, &down, &weights});
  if (!layer) return std::nullopt;
  const Layer& l = *layer;
  if (gate_up.dim() != 3 || down.dim() != 3 || gate_up.size(2) % 2) return std::nullopt;
  const int64_t inter = gate_up.size(2) / 2, tokens = few_tokens(l, x, at::kBFloat16, selected, weights, inter);
  if (tokens < 0 || !is_whole(gate_up, at::kBFloat16, {l.experts, l.hidden, 2 * inter}, x) ||
      !is(down, at::kBFloat16, {l.experts, l.hidden, inter}, x) || (down.stride(1) != 1 && down.stride(2) != 1))
    return std::nullopt;
  Tensor out = at::empty({tokens, l.hidden}, x.options());
  if (!tokens) return out;
  const size_t bytes = entry.moe_few_scratch_bytes(tokens, static_cast<int32_t>(l.top_k), static_cast<int32_t>(l.hidden),
                                                   static_cast<int32_t>(inter), 0);
  const Tensor scratch = at::empty({static_cast<int64_t>(bytes)}, x.options().dtype(at::kByte));
  const c10::DeviceGuard guard(x.device());
  check("mm_moe_few",
        entry.moe_few(static_cast<const uint16_t*>(x.const_data_ptr()), selected.const_data_ptr<int32_t>(),
                      weights.const_data_ptr<float>(), static_cast<const uint16_t*>(gate_up.const_data_ptr()),
                      static_cast<const uint16_t*>(down.const_data_ptr()), down.stride(0), down.stride(1), down.stride(2),
                      tokens, static_cast<int32_t>(l.top_k), static_cast<int32_t>(l.experts),
                      static_cast<int32_t>(l.hidden), static_cast<int32_t>(inter), l.act_kind, l.beta, l.linear_beta,
                      l.limit, static_cast<uint16_t*>(out.data_ptr()), scratch.data_ptr(), bytes, stream_of(x)));
  return out;
}

// The same on int8 rows and experts, whose tensors Int8Experts has checked
// against each other.
std::optional<Tensor> few_forward_int8(const Layer* layer, const Tensor& x, const Tensor& x_scale,
                                       const Tensor& selected, const Tensor& gate_up, const Tensor& gate_up_scale,
                                       const Tensor& down, const Tensor& down_scale, const Tensor& weights) {
  check_detached("forward_few_int8", {&x_scale, &gate_up_scale, &down_scale, &weights});
  if (!layer) return std::nullopt;
  const Layer& l = *layer;
  const int64_t inter = down.size(2), tokens = few_tokens(l, x, at::kChar, selected, weights, inter);
  if (tokens < 0 || l.hidden > kMaxK || !is_whole(x_scale, at::kFloat, {tokens}, x) ||
      !is_whole(gate_up, at::kChar, {l.experts, 2 * inter, l.hidden}, x))
    return std::nullopt;
  Tensor out = at::empty({tokens, l.hidden}, x.options().dtype(at::kBFloat16));
  if (!tokens) return out;
  const size_t bytes = entry.moe_few_scratch_bytes(tokens, static_cast<int32_t>(l.top_k), static_cast<int32_t>(l.hidden),
                                                   static_cast<int32_t>(inter), 1);
  const Tensor scratch = at::empty({static_cast<int64_t>(bytes)}, x.options().dtype(at::kByte));
  const c10::DeviceGuard guard(x.device());
  check("mm_moe_few_int8",
        entry.moe_few_int8(x.const_data_ptr<int8_t>(), x_scale.const_data_ptr<float>(), selected.const_data_ptr<int32_t>(),
                           weights.const_data_ptr<float>(), gate_up.const_data_ptr<int8_t>(),
                           gate_up_scale.const_data_ptr<float>(), down.const_data_ptr<int8_t>(),
                           down_scale.const_data_ptr<float>(), tokens, static_cast<int32_t>(l.top_k),
                           static_cast<int32_t>(l.experts), static_cast<int32_t>(l.hidden), static_cast<int32_t>(inter),
                           l.act_kind, l.beta, l.linear_beta, l.limit, static_cast<uint16_t*>(out.data_ptr()),
                           scratch.data_ptr(), bytes, stream_of(x)));
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::register_local_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const CallError& e) {
      PyErr_SetString(entry.error ? entry.error : PyExc_RuntimeError, e.what());
    }
  });
  m.def("bind", &bind);
  m.def("rms_norm", &rms_norm);
  m.def("quantize_rows", &quantize_rows);
  m.def("int8_matmul", &int8_matmul);
  py::class_<Layer>(m, "Layer")
      .def(py::init([](int64_t most_tokens, int64_t top_k, int64_t experts, int64_t hidden, int32_t act_kind, float beta,
                       float linear_beta, float limit) {
        return Layer{most_tokens, top_k, experts, hidden, act_kind, beta, linear_beta, limit};
      }))
      .def(py::pickle(  // an operator that holds one can be copied
          [](const Layer& l) {
            return py::make_tuple(l.most_tokens, l.top_k, l.experts, l.hidden, l.act_kind, l.beta, l.linear_beta, l.limit);
          },
          [](const py::tuple& t) {
            return Layer{t[0].cast<int64_t>(), t[1].cast<int64_t>(), t[2].cast<int64_t>(), t[3].cast<int64_t>(),
                         t[4].cast<int32_t>(), t[5].cast<float>(), t[6].cast<float>(), t[7].cast<float>()};
          }));
  m.def("few_forward", &few_forward);
  m.def("few_forward_int8", &few_forward_int8);
}
