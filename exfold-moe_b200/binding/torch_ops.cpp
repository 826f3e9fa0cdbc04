// The torch side of the norm, the balance loss and the projection with adapters: argument checks, outputs and
// workspaces, autograd nodes, and one call of the C ABI each.  A Python module (exfold_b200._lib loads it; the
// documented functions are exfold_b200.ops').
//
// Compiled, because at small sizes these operators' time is the host's.  us a call from Python, as Python over
// ctypes and so: norm of one token 15.5 and 4.5, 8 bits and back 31 and 9.6, norm of 777 x 1001 fp32 with its
// gradients 130 and 71, balance loss of 512 x 64 with its gradient 109 and 57.  A backward pass runs in
// autograd's own thread, where a Python node takes the interpreter's lock and starts from cold caches.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <pybind11/pybind11.h>

#include "exfold_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// ---- the library ----------------------------------------------------------------------------------
struct Api {
  decltype(&exf_last_error) last_error;
  decltype(&exf_rms_norm) rms_norm;
  decltype(&exf_rms_norm_8bit) rms_norm_8bit;
  decltype(&exf_dequantize_8bit) dequantize_8bit;
  decltype(&exf_rms_norm_backward_workspace_bytes) norm_workspace;
  decltype(&exf_rms_norm_backward) norm_backward;
  decltype(&exf_balance_loss_workspace_bytes) balance_workspace;
  decltype(&exf_balance_loss) balance_loss;
  decltype(&exf_balance_loss_backward) balance_backward;
  decltype(&exf_adapted_linear_workspace_bytes) adapted_workspace;
  decltype(&exf_adapted_linear) adapted_linear;
} api;

template <typename F>
void symbol(void* lib, const char* name, F& f) {
  f = reinterpret_cast<F>(dlsym(lib, name));
  TORCH_CHECK(f, "libexfold_b200 has no ", name);
}

// the library that the Python package has loaded, by its path
void bind(std::string path) {
  void* lib = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(lib, "cannot load ", path, ": ", dlerror());
  symbol(lib, "exf_last_error", api.last_error);
  symbol(lib, "exf_rms_norm", api.rms_norm);
  symbol(lib, "exf_rms_norm_8bit", api.rms_norm_8bit);
  symbol(lib, "exf_dequantize_8bit", api.dequantize_8bit);
  symbol(lib, "exf_rms_norm_backward_workspace_bytes", api.norm_workspace);
  symbol(lib, "exf_rms_norm_backward", api.norm_backward);
  symbol(lib, "exf_balance_loss_workspace_bytes", api.balance_workspace);
  symbol(lib, "exf_balance_loss", api.balance_loss);
  symbol(lib, "exf_balance_loss_backward", api.balance_backward);
  symbol(lib, "exf_adapted_linear_workspace_bytes", api.adapted_workspace);
  symbol(lib, "exf_adapted_linear", api.adapted_linear);
}

void check(int rc) {
  if (rc == EXF_OK) return;
  const std::string message = api.last_error();
  TORCH_CHECK_VALUE(rc != EXF_ERR_INVALID, message);
  TORCH_CHECK_NOT_IMPLEMENTED(rc != EXF_ERR_UNSUPPORTED, message);
  TORCH_CHECK(false, message);
}

// ---- arguments ----------------------------------------------------------------------------------------
bool floating(const Tensor& t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16 ||
         t.scalar_type() == at::kHalf;
}
int code_of(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? EXF_F32 : t.scalar_type() == at::kBFloat16 ? EXF_BF16 : EXF_F16;
}

// (a tensor without memory, a wrapper's, would be a null pointer: an optional one that was not given)
void require_memory(const Tensor& t) {
  TORCH_CHECK_VALUE(t.numel() == 0 || t.const_data_ptr() != nullptr,
                    "ExFold B200 ops require tensors with memory of their own");
}
void require_cuda(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "ExFold B200 ops require CUDA tensors");
  require_memory(t);
}
void require_cuda(const Tensor& first, std::initializer_list<const Tensor*> others) {
  require_cuda(first);
  for (const Tensor* t : others)
    if (t) {
      require_cuda(*t);
      TORCH_CHECK(t->device() == first.device(),
                  "ExFold B200 ops require all tensors on one device");
    }
}
const Tensor* get(const OptTensor& t) { return t.has_value() && t->defined() ? &*t : nullptr; }
void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
exf_stream_t stream_of(const Tensor& t) {
  return static_cast<exf_stream_t>(at::cuda::getCurrentCUDAStream(t.device().index()).stream());
}
Tensor aligned(const Tensor& t) {
  Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}
// a tensor from the caching allocator, by its function itself (through the dispatcher 0.3 us more)
Tensor fresh(at::IntArrayRef shape, const at::TensorOptions& options) {
  return at::detail::empty_cuda(shape, options);
}
Tensor bytes(int64_t n, const Tensor& like) {
  return fresh({n}, like.options().dtype(at::kByte));
}

// t [..., cols] as rows at a constant distance, where they lie if they do
struct Rows {
  Tensor t;
  int64_t n, stride;
};
Rows rows_of(const Tensor& t) {
  const int64_t cols = t.size(-1);
  if (t.is_contiguous()) return {t, t.numel() / cols, cols};
  const Tensor m = t.dim() == 2 ? t : t.reshape({-1, cols});
  if ((m.stride(1) == 1 || cols == 1) && (m.size(0) <= 1 || m.stride(0) >= cols))
    return {m, m.size(0), m.stride(0)};
  return {m.contiguous(), m.size(0), cols};
}

int32_t* status_pointer(const OptTensor& status) {
  const Tensor* s = get(status);
  if (!s) return nullptr;
  TORCH_CHECK_TYPE(s->scalar_type() == at::kInt && s->numel() >= 1,
                   "status must be an int32 tensor of one element");
  return s->data_ptr<int32_t>();
}

// gradients of a recorded backward pass: an error where they are differentiated again, not zero
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list real;
  for (auto& g : grads)
    if (g.defined()) real.push_back(g.detach().requires_grad_(true));
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with once_differentiable",
      static_cast<int64_t>(real.size()));
  variable_list marked = (*error)(std::move(real));
  size_t i = 0;
  for (auto& g : grads)
    if (g.defined()) g = marked[i++];
  return grads;
}

// ---- norm ------------------------------------------------------------------------------------------------
void norm_checks(const char* name, const Tensor& x, const Tensor& weight, double eps,
                 const Tensor* residual) {
  require_cuda(x, {&weight, residual});
  TORCH_CHECK_TYPE(floating(x), name, " needs a float32, bfloat16 or float16 input");
  TORCH_CHECK_TYPE(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat,
                   name, ": the weight must be float32 or of the input's type");
  TORCH_CHECK_TYPE(!residual || residual->scalar_type() == x.scalar_type(), name,
                   ": the residual must be of the input's type");
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 1 && weight.size(0) == x.size(-1) && x.size(-1) > 0,
                    "x ", x.sizes(), " and weight ", weight.sizes(), " must be [..., H] and [H]");
  TORCH_CHECK_VALUE(!residual || residual->sizes() == x.sizes(), "residual ",
                    residual ? residual->sizes() : x.sizes(), " must have x's shape ", x.sizes());
  TORCH_CHECK_VALUE(eps >= 0.0, "eps must not be negative, got ", eps);
}

struct Normed {
  Tensor y, s, x;  // s: undefined without a residual; x: its rows as they were read
  int64_t stride;
};
Normed norm_forward(const Tensor& x, const Tensor* residual, const Tensor& weight, double eps) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Rows rows = rows_of(x);
  Normed out{fresh(x.sizes(), x.options()), Tensor(), rows.t, rows.stride};
  Rows res{Tensor(), 0, 0};
  if (residual) {
    res = rows_of(*residual);
    out.s = fresh(x.sizes(), x.options());
  }
  const Tensor w = weight.contiguous();
  if (rows.n > 0)
    check(api.rms_norm(rows.t.data_ptr(), rows.stride, pointer(res.t), res.stride, w.data_ptr(),
                       code_of(x), code_of(w), rows.n, x.size(-1), static_cast<float>(eps),
                       pointer(out.s), out.y.data_ptr(), stream_of(x)));
  return out;
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                               const OptTensor& residual, double eps) {
    const Tensor* r = get(residual);
    const Normed out = norm_forward(x, r, weight, eps);
    // (the rows read where they lie, or the copy that was made of them)
    const bool copied = out.x.data_ptr() != x.data_ptr();
    ctx->save_for_backward({r ? out.s : copied ? out.x : x, weight});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["residual"] = r != nullptr;
    ctx->set_materialize_grads(false);
    return r ? variable_list{out.y, out.s} : variable_list{out.y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor& x = saved[0];
    const c10::cuda::CUDAGuard guard(x.device());
    const bool residual = ctx->saved_data["residual"].toBool();
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
    const bool want_r = residual && ctx->needs_input_grad(2);
    const Tensor weight = saved[1].contiguous();
    const Rows rows = rows_of(x);
    const int64_t cols = weight.size(0);
    Tensor dx, dw, ws;
    if (want_x || want_r) dx = fresh(shape, x.options());
    if (want_w) dw = fresh({cols}, weight.options());
    // (of s alone, where y was not used)
    const Tensor dy = grads[0].defined() ? grads[0].contiguous() : at::zeros(shape, x.options());
    const Tensor ds = residual && grads[1].defined() ? grads[1].contiguous() : Tensor();
    if (ds.defined()) require_memory(ds);
    const int64_t need = want_w ? api.norm_workspace(rows.n, cols) : 0;
    if (need > 0) ws = bytes(need, x);
    check(api.norm_backward(dy.data_ptr(), pointer(ds), rows.t.data_ptr(), rows.stride,
                            weight.data_ptr(), code_of(x), code_of(weight), rows.n, cols,
                            static_cast<float>(ctx->saved_data["eps"].toDouble()), pointer(dx),
                            pointer(dw), pointer(ws), need, stream_of(x)));
    // (the gradient of the sum is that of both of its terms)
    return once({want_x ? dx : Tensor(), dw, want_r ? dx : Tensor(), Tensor()});
  }
};

variable_list rms_norm(const Tensor& x, const Tensor& weight, double eps, const OptTensor& residual) {
  const Tensor* r = get(residual);
  norm_checks("rms_norm", x, weight, eps, r);
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || weight.requires_grad() || (r && r->requires_grad())))
    return RmsNorm::apply(x, weight, residual, eps);
  const Normed out = norm_forward(x, r, weight, eps);
  return r ? variable_list{out.y, out.s} : variable_list{out.y};
}

int code_kind(at::ScalarType t, const char* message) {
  TORCH_CHECK_TYPE(t == at::kFloat8_e4m3fn || t == at::kChar, message);
  return t == at::kChar ? EXF_I8 : EXF_E4M3;
}
void check_group(int64_t group) {
  TORCH_CHECK_VALUE(group == 0 || group == 32 || group == 64 || group == 128,
                    "group must be 32, 64, 128 or None (a row), got ", group);
}

variable_list rms_norm_8bit(const Tensor& x, const Tensor& weight, double eps,
                            const OptTensor& residual, at::ScalarType dtype, int64_t group) {
  const Tensor* r = get(residual);
  norm_checks("rms_norm_8bit", x, weight, eps, r);
  const int kind = code_kind(dtype, "rms_norm_8bit gives float8_e4m3fn or int8 codes");
  check_group(group);
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t cols = x.size(-1), groups = group ? (cols + group - 1) / group : 1;
  const Rows rows = rows_of(x);
  Rows res{Tensor(), 0, 0};
  Tensor s;
  if (r) {
    res = rows_of(*r);
    s = fresh(x.sizes(), x.options());
  }
  auto shape = x.sizes().vec();
  const Tensor codes = fresh(shape, x.options().dtype(dtype));
  shape.back() = groups;
  const Tensor scales = fresh(shape, x.options().dtype(at::kFloat));
  const Tensor w = weight.contiguous();
  if (rows.n > 0)
    check(api.rms_norm_8bit(rows.t.data_ptr(), rows.stride, pointer(res.t), res.stride, w.data_ptr(),
                            code_of(x), code_of(w), rows.n, cols, static_cast<float>(eps), kind,
                            static_cast<int>(group), pointer(s), codes.data_ptr(),
                            scales.data_ptr<float>(), stream_of(x)));
  return r ? variable_list{codes, scales, s} : variable_list{codes, scales};
}

Tensor dequantize_8bit(const Tensor& codes, const Tensor& scales, int64_t group,
                       at::ScalarType dtype) {
  require_cuda(codes, {&scales});
  const int kind = code_kind(codes.scalar_type(), "dequantize_8bit needs float8_e4m3fn or int8 codes");
  TORCH_CHECK_TYPE(scales.scalar_type() == at::kFloat, "dequantize_8bit needs float32 scales");
  TORCH_CHECK_TYPE(dtype == at::kFloat || dtype == at::kBFloat16 || dtype == at::kHalf,
                   "dequantize_8bit gives float32, bfloat16 or float16");
  check_group(group);
  const int64_t cols = codes.dim() ? codes.size(-1) : 0;
  auto shape = codes.sizes().vec();
  if (cols) shape.back() = group ? (cols + group - 1) / group : 1;
  TORCH_CHECK_VALUE(cols > 0 && scales.sizes() == at::IntArrayRef(shape), "codes ", codes.sizes(),
                    " and scales ", scales.sizes(), " must be [..., H] and [..., groups]");
  const c10::cuda::CUDAGuard guard(codes.device());
  const Tensor c = aligned(codes), s = scales.contiguous();
  const Tensor out = fresh(codes.sizes(), codes.options().dtype(dtype));
  if (out.numel() > 0)
    check(api.dequantize_8bit(c.data_ptr(), kind, s.data_ptr<float>(), out.numel() / cols, cols,
                              static_cast<int>(group), out.data_ptr(), code_of(out), stream_of(out)));
  return out;
}

// ---- balance loss ------------------------------------------------------------------------------------------
int64_t groups_of(const Tensor& logits) {
  int64_t n = 1;
  for (int64_t i = 0; i + 2 < logits.dim(); ++i) n *= logits.size(i);
  return n;
}

// loss, counts and the number of tokens, of contiguous inputs
variable_list balance_forward(const Tensor& logits, const Tensor& ids, const Tensor* mask,
                              int64_t scoring) {
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t groups = groups_of(logits), tokens = logits.size(-2), experts = logits.size(-1);
  TORCH_CHECK_NOT_IMPLEMENTED(experts <= 1024 && groups <= 65535,
                              "exf_balance_loss: at most 1024 experts and 65535 groups");
  auto shape = logits.sizes().vec();
  shape.resize(shape.size() - 2);
  const Tensor loss = fresh(shape, logits.options().dtype(at::kFloat));
  const Tensor valid = fresh(shape, logits.options().dtype(at::kInt));
  shape.push_back(experts);
  const Tensor counts = fresh(shape, logits.options().dtype(at::kInt));
  const int64_t need =
      api.balance_workspace(static_cast<int>(groups), tokens, static_cast<int>(experts));
  Tensor ws;
  if (need > 0) ws = bytes(need, logits);
  check(api.balance_loss(logits.data_ptr(), code_of(logits), ids.data_ptr(),
                         ids.scalar_type() == at::kLong ? EXF_I64 : EXF_I32,
                         mask ? static_cast<const uint8_t*>(mask->data_ptr()) : nullptr,
                         static_cast<int>(groups), tokens, static_cast<int>(experts),
                         static_cast<int>(ids.size(-1)), static_cast<int>(scoring),
                         loss.data_ptr<float>(), counts.data_ptr<int32_t>(),
                         valid.data_ptr<int32_t>(), pointer(ws), need, stream_of(logits)));
  return {loss, counts, valid};
}

struct BalanceLoss : torch::autograd::Function<BalanceLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& ids,
                               const OptTensor& mask, int64_t scoring) {
    const Tensor x = logits.contiguous();
    const Tensor* m = get(mask);
    variable_list out = balance_forward(x, ids, m, scoring);
    ctx->save_for_backward({x, m ? *m : Tensor(), out[1], out[2]});
    ctx->saved_data["scoring"] = scoring;
    ctx->saved_data["top_k"] = ids.size(-1);
    ctx->mark_non_differentiable({out[1]});
    ctx->set_materialize_grads(false);
    return {out[0], out[1]};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &mask = saved[1];
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor dloss = grads[0].contiguous(), out = fresh(x.sizes(), x.options());
    check(api.balance_backward(
        dloss.data_ptr<float>(), x.data_ptr(), code_of(x),
        static_cast<const uint8_t*>(pointer(mask)), saved[2].data_ptr<int32_t>(),
        saved[3].data_ptr<int32_t>(), static_cast<int>(groups_of(x)), x.size(-2),
        static_cast<int>(x.size(-1)), static_cast<int>(ctx->saved_data["top_k"].toInt()),
        static_cast<int>(ctx->saved_data["scoring"].toInt()), out.data_ptr(), stream_of(x)));
    return once({out, Tensor(), Tensor(), Tensor()});
  }
};

variable_list balance_loss(const Tensor& logits, const Tensor& topk_ids, int64_t scoring,
                           const OptTensor& mask) {
  const Tensor* m = get(mask);
  require_cuda(logits, {&topk_ids, m});
  TORCH_CHECK_TYPE(floating(logits), "balance_loss needs float32, bfloat16 or float16 logits");
  TORCH_CHECK_TYPE(!topk_ids.is_floating_point() && !topk_ids.is_complex() &&
                       topk_ids.scalar_type() != at::kBool,
                   "expert ids must be integers, got ", topk_ids.scalar_type());
  TORCH_CHECK_VALUE(logits.dim() >= 2 && topk_ids.dim() == logits.dim() && logits.size(-1) > 0 &&
                        topk_ids.size(-1) > 0 &&
                        topk_ids.sizes().slice(0, logits.dim() - 1) ==
                            logits.sizes().slice(0, logits.dim() - 1),
                    "logits ", logits.sizes(), " and topk_ids ", topk_ids.sizes(),
                    " must be [..., T, E] and [..., T, k]");
  TORCH_CHECK_VALUE(!m || (m->scalar_type() == at::kBool &&
                           m->sizes() == logits.sizes().slice(0, logits.dim() - 1)),
                    "mask must be bool ", logits.sizes().slice(0, logits.dim() - 1));
  TORCH_CHECK_NOT_IMPLEMENTED(topk_ids.size(-1) < (int64_t(1) << 31),
                              "exf_balance_loss: a group's routes must be below 2^31");
  Tensor ids = topk_ids;
  // (narrow and unsigned ids in 64 bits: what lies outside [0, E) stays outside)
  if (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong) ids = ids.to(at::kLong);
  ids = ids.contiguous();
  OptTensor kept = m ? OptTensor(m->contiguous()) : std::nullopt;
  if (at::GradMode::is_enabled() && logits.requires_grad())
    return BalanceLoss::apply(logits, ids, kept, scoring);
  variable_list out = balance_forward(logits.contiguous(), ids, get(kept), scoring);
  out.pop_back();
  return out;
}

// ---- adapters ----------------------------------------------------------------------------------------------
Tensor adapted_linear(const Tensor& x, const Tensor& w, const Tensor& a, const Tensor& b,
                      const Tensor& adapter_ids, const OptTensor& scaling, const OptTensor& status) {
  const Tensor* scale = get(scaling);
  require_cuda(x, {&w, &a, &b, &adapter_ids, scale, get(status)});
  const auto dtype = x.scalar_type();
  TORCH_CHECK_TYPE((dtype == at::kBFloat16 || dtype == at::kHalf) && w.scalar_type() == dtype &&
                       a.scalar_type() == dtype && b.scalar_type() == dtype,
                   "adapted_linear needs x, w, a and b all bfloat16 or all float16");
  TORCH_CHECK_TYPE(!adapter_ids.is_floating_point() && !adapter_ids.is_complex() &&
                       adapter_ids.scalar_type() != at::kBool,
                   "adapter ids must be integers, got ", adapter_ids.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1 && w.dim() == 2 && a.dim() == 3 && b.dim() == 3 &&
                        w.size(1) == x.size(-1) && a.size(2) == w.size(1) && b.size(0) == a.size(0) &&
                        b.size(1) == w.size(0) && b.size(2) == a.size(1) && w.numel() > 0 &&
                        a.size(1) > 0,
                    "x ", x.sizes(), ", w ", w.sizes(), ", a ", a.sizes(), " and b ", b.sizes(),
                    " must be [..., K], [N, K], [R, rank, K] and [R, N, rank]");
  TORCH_CHECK_VALUE(adapter_ids.sizes() == x.sizes().slice(0, x.dim() - 1), "adapter_ids ",
                    adapter_ids.sizes(), " must have x's leading shape ",
                    x.sizes().slice(0, x.dim() - 1));
  const int64_t outer = w.size(0), inner = w.size(1), adapters = a.size(0), rank = a.size(1);
  TORCH_CHECK_VALUE(!scale || (scale->dim() == 1 && scale->size(0) == adapters), "scaling must be [",
                    adapters, "]");
  TORCH_CHECK_NOT_IMPLEMENTED(inner < (1 << 23) && outer < (1 << 23) && adapters < (1 << 24) &&
                                  rank <= 128,
                              "exf_adapted_linear: rank must be at most 128, or shape too large");
  int32_t* flag = status_pointer(status);
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor rows = aligned(x), wc = aligned(w), ac = aligned(a), bc = aligned(b);
  Tensor ids = adapter_ids;
  // (clamped in 64 bits: what lies outside [0, R) stays outside in 32)
  if (ids.scalar_type() != at::kInt) ids = ids.to(at::kLong).clamp(-1, adapters).to(at::kInt);
  ids = ids.contiguous();
  const Tensor factor = scale ? scale->to(at::kFloat).contiguous() : Tensor();
  auto shape = x.sizes().vec();
  shape.back() = outer;
  const Tensor y = fresh(shape, x.options());
  const int64_t tokens = ids.numel();
  const int64_t need = api.adapted_workspace(tokens, static_cast<int>(inner),
                                             static_cast<int>(outer), static_cast<int>(rank));
  const Tensor ws = bytes(need > 32 ? need : 32, x);
  check(api.adapted_linear(rows.data_ptr(), wc.data_ptr(), ac.data_ptr(), bc.data_ptr(),
                           ids.data_ptr<int32_t>(), static_cast<const float*>(pointer(factor)),
                           code_of(x), tokens, static_cast<int>(inner), static_cast<int>(outer),
                           static_cast<int>(adapters), static_cast<int>(rank), y.data_ptr(),
                           ws.data_ptr(), need, flag, stream_of(x)));
  return y;
}

}  // namespace

// ---- the Python module ---------------------------------------------------------------------------------
// Functions of positional arguments, read here: torch's operator calls match a schema and box every argument,
// 3 us of a call's 7.
namespace {

const Tensor& tensor_of(PyObject* o) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), "expected a tensor, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
OptTensor maybe_tensor(PyObject* o) { return o == Py_None ? OptTensor() : OptTensor(tensor_of(o)); }
double number_of(PyObject* o) {
  const double d = PyFloat_AsDouble(o);
  if (d == -1.0 && PyErr_Occurred()) throw python_error();
  return d;
}
int64_t integer_of(PyObject* o) {
  const int64_t i = PyLong_AsLongLong(o);
  if (i == -1 && PyErr_Occurred()) throw python_error();
  return i;
}
at::ScalarType dtype_of(PyObject* o) {
  TORCH_CHECK_TYPE(THPDtype_Check(o), "expected a torch.dtype, got ", Py_TYPE(o)->tp_name);
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}
void no_tangent(const char* name, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t || !t->_fw_grad(0).defined(), name,
                                " has no forward-mode derivative");
}

PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }
PyObject* wrap(const variable_list& l) {
  THPObjectPtr tuple(PyTuple_New(static_cast<Py_ssize_t>(l.size())));
  if (!tuple) throw python_error();
  for (size_t i = 0; i < l.size(); ++i) {
    PyObject* t = wrap(l[i]);
    if (!t) throw python_error();
    PyTuple_SET_ITEM(tuple.get(), static_cast<Py_ssize_t>(i), t);
  }
  return tuple.release();
}

// f(the arguments) -> a tensor or several, without the interpreter's lock where it computes
template <Py_ssize_t N, typename F>
PyObject* call(const char* name, Py_ssize_t n, F f) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == N, name, " takes ", N, " arguments, got ", n);
  return wrap(f());
  END_HANDLE_TH_ERRORS
}
template <typename F>
auto unlocked(F f) {
  pybind11::gil_scoped_release release;
  return f();
}

PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 1 && PyUnicode_Check(a[0]), "bind takes a path");
  const char* path = PyUnicode_AsUTF8(a[0]);
  if (!path) throw python_error();
  bind(path);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
// (x, weight, eps, residual or None) -> y, or (y, s)
PyObject* py_rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 4, "rms_norm takes 4 arguments, got ", n);
  const Tensor &x = tensor_of(a[0]), &weight = tensor_of(a[1]);
  const double eps = number_of(a[2]);
  const OptTensor residual = maybe_tensor(a[3]);
  no_tangent("rms_norm", {&x, &weight, get(residual)});
  const variable_list out = unlocked([&] { return rms_norm(x, weight, eps, residual); });
  return residual ? wrap(out) : wrap(out[0]);
  END_HANDLE_TH_ERRORS
}
// (x, weight, eps, residual or None, dtype, group) -> (codes, scales), or (codes, scales, s)
PyObject* py_rms_norm_8bit(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call<6>("rms_norm_8bit", n, [&] {
    const Tensor &x = tensor_of(a[0]), &weight = tensor_of(a[1]);
    const double eps = number_of(a[2]);
    const OptTensor residual = maybe_tensor(a[3]);
    const at::ScalarType dtype = dtype_of(a[4]);
    const int64_t group = integer_of(a[5]);
    no_tangent("rms_norm_8bit", {&x, &weight, get(residual)});
    return unlocked([&] { return rms_norm_8bit(x, weight, eps, residual, dtype, group); });
  });
}
// (codes, scales, group, dtype) -> values
PyObject* py_dequantize_8bit(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call<4>("dequantize_8bit", n, [&] {
    const Tensor &codes = tensor_of(a[0]), &scales = tensor_of(a[1]);
    const int64_t group = integer_of(a[2]);
    const at::ScalarType dtype = dtype_of(a[3]);
    no_tangent("dequantize_8bit", {&scales});
    return unlocked([&] { return dequantize_8bit(codes, scales, group, dtype); });
  });
}
// (logits, topk_ids, scoring, mask or None) -> (loss, counts)
PyObject* py_balance_loss(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call<4>("balance_loss", n, [&] {
    const Tensor &logits = tensor_of(a[0]), &ids = tensor_of(a[1]);
    const int64_t scoring = integer_of(a[2]);
    const OptTensor mask = maybe_tensor(a[3]);
    no_tangent("balance_loss", {&logits});
    return unlocked([&] { return balance_loss(logits, ids, scoring, mask); });
  });
}
// (x, w, a, b, adapter_ids, scaling or None, status or None) -> y
PyObject* py_adapted_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call<7>("adapted_linear", n, [&] {
    const Tensor &x = tensor_of(a[0]), &w = tensor_of(a[1]), &down = tensor_of(a[2]),
                 &up = tensor_of(a[3]), &ids = tensor_of(a[4]);
    const OptTensor scaling = maybe_tensor(a[5]), status = maybe_tensor(a[6]);
    no_tangent("adapted_linear", {&x, &w, &down, &up, get(scaling)});
    return unlocked([&] { return adapted_linear(x, w, down, up, ids, scaling, status); });
  });
}

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}
PyMethodDef methods[] = {
    {"bind", fast(py_bind), METH_FASTCALL, nullptr},
    {"rms_norm", fast(py_rms_norm), METH_FASTCALL, nullptr},
    {"rms_norm_8bit", fast(py_rms_norm_8bit), METH_FASTCALL, nullptr},
    {"dequantize_8bit", fast(py_dequantize_8bit), METH_FASTCALL, nullptr},
    {"balance_loss", fast(py_balance_loss), METH_FASTCALL, nullptr},
    {"adapted_linear", fast(py_adapted_linear), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "libexfold_b200_torch", nullptr, -1, methods,
                          nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_libexfold_b200_torch() {
  return PyModule_Create(&module_def);
}
