// The layer operators on torch tensors: argument checks, outputs and scratch from torch's caching allocator,
// the current stream, and autograd, over the C entries of include/lwl_layers.h.
//
// These calls are short on the GPU (a layer norm's training step of 8192 x 768 is 36 us of kernels).  Through
// ctypes and Python autograd functions such a step took 130 us of host time, most of it in Python
// operations on autograd's own thread, where each finds its caches cold; autograd nodes in C++ run there
// without Python.  The library is the one that the rest of the package has loaded (bind()).
#include <dlfcn.h>

#include <cmath>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include "lwl_layers.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

// The library's entries (declared in the header; their types are taken from it).
struct Library {
  decltype(&lwl_last_error) last_error = nullptr;
  decltype(&lwl_layer_norm_forward) norm_forward = nullptr;
  decltype(&lwl_layer_norm_backward_workspace_size) norm_backward_workspace = nullptr;
  decltype(&lwl_layer_norm_backward) norm_backward = nullptr;
  decltype(&lwl_gelu8_pitch) gelu8_pitch = nullptr;
  decltype(&lwl_gelu8_forward) gelu8_forward = nullptr;
  decltype(&lwl_gelu8_activation) gelu8_activation = nullptr;
  decltype(&lwl_gelu8_backward_workspace_size) gelu8_backward_workspace = nullptr;
  decltype(&lwl_gelu8_backward) gelu8_backward = nullptr;
  decltype(&lwl_attention_forward_workspace_size) attention_forward_workspace = nullptr;
  decltype(&lwl_attention_forward) attention_forward = nullptr;
  decltype(&lwl_attention_backward_workspace_size) attention_backward_workspace = nullptr;
  decltype(&lwl_attention_backward) attention_backward = nullptr;
} lib;

// An invalid argument: the package's BlockFHTArgumentError (a ValueError and a RuntimeError).
struct ArgumentError : std::runtime_error {
  using std::runtime_error::runtime_error;
};
PyObject* argument_error = nullptr;  // its class, kept for the process

template <class... Parts>
[[noreturn]] void refuse(const Parts&... parts) {
  throw ArgumentError(c10::str(parts...));
}

void check(int rc) {
  if (rc == LWL_OK) return;
  const std::string message = lib.last_error();
  if (rc == LWL_ERR_INVALID) throw ArgumentError(message);
  throw std::runtime_error("latent_weight_lab_amd: " + message);
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return LWL_DTYPE_F32;
    case at::kHalf: return LWL_DTYPE_F16;
    case at::kBFloat16: return LWL_DTYPE_BF16;
    default:
      throw std::runtime_error(c10::str("latent_weight_lab_amd supports float32, float16 and bfloat16, got ", t));
  }
}

// Every tensor on one GPU, none with a forward-mode tangent: outputs are filled through pointers and would have
// none, which is a derivative of zero (and holds without gradient recording too, which does not end this mode).
void on_one_gpu(const Tensor& first) {
  if (!first.is_cuda())
    throw std::runtime_error("latent_weight_lab_amd runs on the GPU only; move the inputs to a cuda device");
  TORCH_CHECK_NOT_IMPLEMENTED(!first._fw_grad(/*level=*/0).defined(),
                              "latent_weight_lab_amd: the layer operators have no forward-mode derivatives");
}
template <class... Rest>
void on_one_gpu(const Tensor& first, const Rest&... rest) {
  on_one_gpu(first);
  const auto same = [&](const auto& t) {
    const Tensor* p = nullptr;
    if constexpr (std::is_same_v<std::decay_t<decltype(t)>, MaybeTensor>) {
      if (!t) return;
      p = &*t;
    } else {
      p = &t;
    }
    on_one_gpu(*p);
    if (p->get_device() != first.get_device())
      throw std::runtime_error(c10::str("latent_weight_lab_amd: tensors on different devices (", first.device(), ", ",
                                        p->device(), ")"));
  };
  (same(rest), ...);
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* ptr(const MaybeTensor& t) { return t ? t->data_ptr() : nullptr; }

Tensor scratch(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}
Tensor typed(const Tensor& t, at::ScalarType dtype) { return t.scalar_type() == dtype ? t : t.to(dtype); }

MaybeTensor vector(const char* name, const MaybeTensor& t, int64_t n, at::ScalarType dtype) {
  if (!t) return t;
  if (t->dim() != 1 || t->size(0) != n || t->scalar_type() != dtype)
    refuse(name, " must be ", n, " values of ", dtype, ", got ", t->sizes(), " of ", t->scalar_type());
  return t->contiguous();
}
int64_t features_of(const char* what, const Tensor& x) {
  if (x.dim() == 0 || x.size(-1) == 0) refuse(what, " needs at least one feature, got ", x.sizes());
  return x.size(-1);
}

// The gradients of a backward that cannot itself be differentiated.  Where a graph of the backward is
// recorded, they lead to an error rather than nowhere.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list ends;
  for (auto& g : grads)
    if (g.defined()) ends.push_back(g.detach().set_requires_grad(true));
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that can be differentiated once only", (int64_t)ends.size());
  auto out = (*error)(std::move(ends));
  size_t i = 0;
  for (auto& g : grads)
    if (g.defined()) g = out[i++];
  return grads;
}
bool records(const Tensor& t) { return t.requires_grad(); }
bool records(const MaybeTensor& t) { return t && t->requires_grad(); }

// ---------------------------------------------------------------- layer norm
struct Normed {
  Tensor h, out, sum, stats;  // h: what was normed, dense; sum: undefined without a residual, stats: unless kept
};

Normed norm_forward(const Tensor& x0, const Tensor& weight0, const MaybeTensor& bias0, double eps,
                    const MaybeTensor& residual0, bool keep_stats) {
  on_one_gpu(x0, weight0, bias0, residual0);
  const int64_t f = features_of("layer norm", x0), rows = x0.numel() / f;
  const int code = dtype_code(x0.scalar_type()), weight_code = dtype_code(weight0.scalar_type());
  const MaybeTensor weight = vector("layer norm's weight", weight0, f, weight0.scalar_type());
  const MaybeTensor bias = vector("layer norm's bias", bias0, f, weight0.scalar_type());
  MaybeTensor residual;
  if (residual0) {
    if (residual0->sizes() != x0.sizes() || residual0->scalar_type() != x0.scalar_type())
      refuse("residual must be ", x0.sizes(), " of ", x0.scalar_type(), ", got ", residual0->sizes(), " of ",
             residual0->scalar_type());
    residual = residual0->contiguous();
  }
  const c10::DeviceGuard guard(x0.device());
  const Tensor x = x0.contiguous();
  Normed r;
  r.out = at::empty(x.sizes(), x.options());
  if (residual) r.sum = at::empty(x.sizes(), x.options());
  r.h = residual ? r.sum : x;
  if (keep_stats) r.stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
  check(lib.norm_forward(x.data_ptr(), ptr(residual), ptr(weight), ptr(bias), code, weight_code, rows, f, eps,
                         r.out.data_ptr(), ptr(r.sum), (float*)ptr(r.stats), stream_of(x)));
  return r;
}

std::tuple<Tensor, Tensor, Tensor> norm_backward(const Tensor& h0, const Tensor& weight0, const Tensor& stats,
                                                 const Tensor& grad_out0, const MaybeTensor& grad_sum0, bool need_x,
                                                 bool need_weight, bool need_bias) {
  on_one_gpu(h0, weight0, stats, grad_out0, grad_sum0);
  const int64_t f = features_of("layer norm", h0), rows = h0.numel() / f;
  // saved tensors come back as a caller's hooks left them
  if (stats.scalar_type() != at::kFloat || !stats.is_contiguous() || stats.sizes() != at::IntArrayRef({2, rows}) ||
      weight0.numel() != f)
    refuse("layer norm backward: statistics ", stats.sizes(), " of ", stats.scalar_type(), " and weight ", weight0.sizes(),
           " are not those of ", h0.sizes());
  const c10::DeviceGuard guard(h0.device());
  const Tensor h = h0.contiguous(), weight = weight0.contiguous(), grad_out = typed(grad_out0, h.scalar_type()).contiguous();
  MaybeTensor grad_sum;
  if (grad_sum0) grad_sum = typed(*grad_sum0, h.scalar_type()).contiguous();
  Tensor gx, gw, gb;
  if (need_x) gx = at::empty(h.sizes(), h.options());
  if (need_weight) gw = at::empty({f}, weight.options());
  if (need_bias) gb = at::empty({f}, weight.options());
  const size_t need = need_weight || need_bias ? lib.norm_backward_workspace(rows, f) : 0;
  const Tensor ws = scratch(need, h);
  check(lib.norm_backward(h.data_ptr(), weight.data_ptr(), (const float*)stats.data_ptr(), grad_out.data_ptr(),
                          ptr(grad_sum), dtype_code(h.scalar_type()), dtype_code(weight.scalar_type()), rows, f, ptr(gx),
                          ptr(gw), ptr(gb), ptr(ws), need, stream_of(h)));
  return {gx, gw, gb};
}

struct NormFn : torch::autograd::Function<NormFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const MaybeTensor& bias,
                               const MaybeTensor& residual, double eps) {
    const Normed r = norm_forward(x, weight, bias, eps, residual, true);
    ctx->save_for_backward({r.h, weight, r.stats});
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["residual"] = residual.has_value();
    ctx->set_materialize_grads(false);
    return residual ? variable_list{r.out, r.sum} : variable_list{r.out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    // numbered over the tensors that were given
    const bool has_b = ctx->saved_data["bias"].toBool(), has_r = ctx->saved_data["residual"].toBool();
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const bool need_b = has_b && ctx->needs_input_grad(2), need_r = has_r && ctx->needs_input_grad(has_b ? 3 : 2);
    const Tensor grad_sum = grads.size() > 1 ? grads[1] : Tensor();
    if (!grads[0].defined())  // only the sum was used
      return {need_x ? grad_sum : Tensor(), Tensor(), Tensor(), need_r ? grad_sum : Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const auto [gx, gw, gb] =
        norm_backward(saved[0], saved[1], saved[2], grads[0], grad_sum.defined() ? MaybeTensor(grad_sum) : MaybeTensor(),
                      need_x || need_r, need_w, need_b);
    return once({need_x ? gx : Tensor(), gw, gb, need_r ? gx : Tensor(), Tensor()});
  }
};

variable_list layer_norm(const Tensor& x, const Tensor& weight, const MaybeTensor& bias, double eps,
                         const MaybeTensor& residual) {
  if (at::GradMode::is_enabled() && (records(x) || records(weight) || records(bias) || records(residual)))
    return NormFn::apply(x, weight, bias, residual, eps);
  const Normed r = norm_forward(x, weight, bias, eps, residual, false);
  return residual ? variable_list{r.out, r.sum} : variable_list{r.out};
}

// ---------------------------------------------------------------- GELU, input kept in 8 bits
std::tuple<Tensor, MaybeTensor, MaybeTensor> gelu8_forward(const Tensor& x0, const MaybeTensor& bias0, bool tanh_form,
                                                           bool keep) {
  on_one_gpu(x0, bias0);
  const int64_t f = features_of("GELU checkpoint", x0), rows = x0.numel() / f;
  const int code = dtype_code(x0.scalar_type());
  const MaybeTensor bias = vector("GELU's bias", bias0, f, x0.scalar_type());
  const c10::DeviceGuard guard(x0.device());
  const Tensor x = x0.contiguous(), out = at::empty(x.sizes(), x.options());
  MaybeTensor codes, scales;
  if (keep) {
    codes = at::empty({rows, lib.gelu8_pitch(f)}, x.options().dtype(at::kChar));
    scales = at::empty({rows, (f + LWL_GELU8_GROUP - 1) / LWL_GELU8_GROUP}, x.options().dtype(at::kFloat));
  }
  check(lib.gelu8_forward(x.data_ptr(), ptr(bias), code, tanh_form, rows, f, out.data_ptr(), (int8_t*)ptr(codes),
                          (float*)ptr(scales), stream_of(x)));
  return {out, codes, scales};
}

// The kernels read both by these shapes alone.
void hold_checkpoint(const Tensor& codes, const Tensor& scales, int64_t rows, int64_t f, at::IntArrayRef shape) {
  const int64_t groups = (f + LWL_GELU8_GROUP - 1) / LWL_GELU8_GROUP;
  if (codes.scalar_type() != at::kChar || scales.scalar_type() != at::kFloat || !codes.is_contiguous() ||
      !scales.is_contiguous() || codes.sizes() != at::IntArrayRef({rows, lib.gelu8_pitch(f)}) ||
      scales.sizes() != at::IntArrayRef({rows, groups}))
    refuse("GELU checkpoint: codes ", codes.sizes(), " of ", codes.scalar_type(), " and scales ", scales.sizes(), " of ",
           scales.scalar_type(), " do not hold ", shape, " as contiguous int8 rows of ", lib.gelu8_pitch(f),
           " and float32 rows of ", groups);
}

Tensor gelu8_activation(const Tensor& codes, const Tensor& scales, std::vector<int64_t> shape, at::ScalarType dtype,
                        bool tanh_form) {
  on_one_gpu(codes, scales);
  const c10::DeviceGuard guard(codes.device());
  const Tensor out = at::empty(shape, codes.options().dtype(dtype));
  const int64_t f = features_of("GELU checkpoint", out);
  hold_checkpoint(codes, scales, out.numel() / f, f, out.sizes());
  check(lib.gelu8_activation((const int8_t*)codes.data_ptr(), (const float*)scales.data_ptr(), dtype_code(dtype), tanh_form,
                             out.numel() / f, f, out.data_ptr(), stream_of(codes)));
  return out;
}

std::tuple<Tensor, MaybeTensor> gelu8_backward(const Tensor& codes, const Tensor& scales, const Tensor& grad_out0,
                                               at::ScalarType dtype, bool tanh_form, bool need_bias) {
  on_one_gpu(codes, scales, grad_out0);
  const c10::DeviceGuard guard(codes.device());
  const int64_t f = features_of("GELU checkpoint", grad_out0), rows = grad_out0.numel() / f;
  hold_checkpoint(codes, scales, rows, f, grad_out0.sizes());
  const Tensor grad_out = typed(grad_out0, dtype).contiguous(), gx = at::empty(grad_out.sizes(), grad_out.options());
  MaybeTensor gb;
  if (need_bias) gb = at::empty({f}, grad_out.options());
  const size_t need = need_bias ? lib.gelu8_backward_workspace(rows, f) : 0;
  const Tensor ws = scratch(need, gx);
  check(lib.gelu8_backward((const int8_t*)codes.data_ptr(), (const float*)scales.data_ptr(), grad_out.data_ptr(),
                           dtype_code(dtype), tanh_form, rows, f, gx.data_ptr(), ptr(gb), ptr(ws), need, stream_of(gx)));
  return {gx, gb};
}

struct Gelu8Fn : torch::autograd::Function<Gelu8Fn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& bias, bool tanh_form) {
    const auto [out, codes, scales] = gelu8_forward(x, bias, tanh_form, true);
    ctx->mark_non_differentiable({*codes, *scales});
    ctx->save_for_backward({*codes, *scales});
    ctx->saved_data["tanh"] = tanh_form;
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["dtype"] = (int64_t)x.scalar_type();
    ctx->set_materialize_grads(false);
    return {out, *codes, *scales};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const auto [gx, gb] =
        gelu8_backward(saved[0], saved[1], grads[0], (at::ScalarType)ctx->saved_data["dtype"].toInt(),
                       ctx->saved_data["tanh"].toBool(), ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(1));
    return once({gx, gb ? *gb : Tensor(), Tensor()});
  }
};

// (activation, codes, scales); the last two are kept where a gradient is recorded or `keep` asks for them.
std::tuple<Tensor, MaybeTensor, MaybeTensor> gelu8(const Tensor& x, const MaybeTensor& bias, bool tanh_form, bool keep) {
  if (at::GradMode::is_enabled() && (records(x) || records(bias))) {
    const variable_list r = Gelu8Fn::apply(x, bias, tanh_form);
    return {r[0], r[1], r[2]};
  }
  return gelu8_forward(x, bias, tanh_form, keep);
}

// ---------------------------------------------------------------- attention
// What a call has beside its tensors.
struct How {
  bool causal;
  std::optional<double> scale;
  std::optional<int64_t> offset;
};

Tensor dense_dim(const Tensor& t) {
  // the kernels take any strides but that of a head's values, which lie one after the other
  return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous();
}
MaybeTensor lengths_of(const MaybeTensor& lengths, int64_t batch) {
  if (!lengths) return lengths;
  if (lengths->dim() != 1 || lengths->size(0) != batch ||
      !at::isIntegralType(lengths->scalar_type(), /*includeBool=*/false))
    refuse("attention: key_lengths must be ", batch, " integers, got ", lengths->sizes(), " of ", lengths->scalar_type());
  return lengths->to(at::kInt).contiguous();
}
lwl_attention_args shape_args(at::ScalarType dtype, const How& how, int64_t batch, int64_t heads, int64_t kv_heads,
                              int64_t queries, int64_t keys, int64_t dim) {
  lwl_attention_args a{};
  a.dtype = dtype_code(dtype);
  a.causal = how.causal;
  a.bottom_right = !how.offset;
  a.causal_offset = how.offset.value_or(0);
  a.batch = batch;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.queries = queries;
  a.keys = keys;
  a.dim = dim;
  a.scale = how.scale ? *how.scale : dim > 0 ? 1.0 / std::sqrt((double)dim) : 0.0;
  return a;
}
void strides(int64_t (&s)[3], const Tensor& t) {
  for (int i = 0; i < 3; ++i) s[i] = t.stride(i);
}
void run(const lwl_attention_args& a, bool forward, const Tensor& like) {
  const size_t need = (forward ? lib.attention_forward_workspace : lib.attention_backward_workspace)(&a);
  const Tensor ws = scratch(need, like);
  check((forward ? lib.attention_forward : lib.attention_backward)(&a, ptr(ws), need, stream_of(like)));
}

lwl_attention_args heads_args(const Tensor& q, const Tensor& k, const Tensor& v, const How& how) {
  if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4)
    refuse("attention: q, k and v must be [batch, heads, tokens, head size], got ", q.sizes(), ", ", k.sizes(), " and ",
           v.sizes());
  if (k.sizes() != v.sizes() || k.size(0) != q.size(0) || k.size(3) != q.size(3))
    refuse("attention: q ", q.sizes(), ", k ", k.sizes(), " and v ", v.sizes(), " do not match");
  if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
    refuse("attention: q, k and v must have one type, got ", q.scalar_type(), ", ", k.scalar_type(), " and ",
           v.scalar_type());
  return shape_args(q.scalar_type(), how, q.size(0), q.size(1), k.size(1), q.size(2), k.size(2), q.size(3));
}
// [batch, heads, tokens, dim] whose tokens lie one after the other, all heads of a token together
Tensor empty_heads(const lwl_attention_args& a, int64_t tokens, int64_t heads, const Tensor& like) {
  const int64_t width = heads * a.dim;
  return at::empty_strided({a.batch, heads, tokens, a.dim}, {tokens * width, a.dim, width, 1}, like.options());
}

std::tuple<Tensor, MaybeTensor> attention_forward(const Tensor& q0, const Tensor& k0, const Tensor& v0, bool causal,
                                                  std::optional<double> scale, const MaybeTensor& lengths0,
                                                  std::optional<int64_t> offset, bool keep_lse) {
  on_one_gpu(q0, k0, v0, lengths0);
  lwl_attention_args a = heads_args(q0, k0, v0, {causal, scale, offset});
  const c10::DeviceGuard guard(q0.device());
  const MaybeTensor lengths = lengths_of(lengths0, a.batch);
  const Tensor q = dense_dim(q0), k = dense_dim(k0), v = dense_dim(v0), out = empty_heads(a, a.queries, a.heads, q);
  MaybeTensor lse;
  if (keep_lse) lse = at::empty({a.batch, a.heads, a.queries}, q.options().dtype(at::kFloat));
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.out = out.data_ptr();
  a.lse = (float*)ptr(lse);
  a.key_lengths = (const int32_t*)ptr(lengths);
  strides(a.q_stride, q);
  strides(a.k_stride, k);
  strides(a.v_stride, v);
  strides(a.out_stride, out);
  run(a, true, q);
  return {out, lse};
}

// What the forward left for the backward: out like q (`shape`), lse float32 for each query of each head.
void check_left(const lwl_attention_args& a, const Tensor& q, at::IntArrayRef shape, const Tensor& out, const Tensor& lse,
                const Tensor& grad_out) {
  if (out.sizes() != shape || grad_out.sizes() != shape || out.scalar_type() != q.scalar_type())
    refuse("attention backward: out ", out.sizes(), " of ", out.scalar_type(), " and grad_out ", grad_out.sizes(),
           " must be ", shape, ", out of ", q.scalar_type());
  if (lse.scalar_type() != at::kFloat || !lse.is_contiguous() || lse.sizes() != at::IntArrayRef({a.batch, a.heads, a.queries}))
    refuse("attention backward: lse must be contiguous float32 [", a.batch, ", ", a.heads, ", ", a.queries, "], got ",
           lse.sizes(), " of ", lse.scalar_type());
}

std::tuple<Tensor, Tensor, Tensor> attention_backward(const Tensor& q0, const Tensor& k0, const Tensor& v0,
                                                      const Tensor& out, const Tensor& lse, const Tensor& grad_out0,
                                                      bool causal, std::optional<double> scale,
                                                      const MaybeTensor& lengths0, std::optional<int64_t> offset) {
  on_one_gpu(q0, k0, v0, out, lse, grad_out0, lengths0);
  lwl_attention_args a = heads_args(q0, k0, v0, {causal, scale, offset});
  check_left(a, q0, q0.sizes(), out, lse, grad_out0);
  const c10::DeviceGuard guard(q0.device());
  const MaybeTensor lengths = lengths_of(lengths0, a.batch);
  const Tensor q = dense_dim(q0), k = dense_dim(k0), v = dense_dim(v0), o = dense_dim(out);
  const Tensor grad_out = dense_dim(typed(grad_out0, q.scalar_type()));
  const Tensor gq = empty_heads(a, a.queries, a.heads, q), gk = empty_heads(a, a.keys, a.kv_heads, q),
               gv = empty_heads(a, a.keys, a.kv_heads, q);
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.out = o.data_ptr();
  a.lse = (float*)lse.data_ptr();
  a.key_lengths = (const int32_t*)ptr(lengths);
  a.grad_out = grad_out.data_ptr();
  a.grad_q = gq.data_ptr();
  a.grad_k = gk.data_ptr();
  a.grad_v = gv.data_ptr();
  strides(a.q_stride, q);
  strides(a.k_stride, k);
  strides(a.v_stride, v);
  strides(a.out_stride, o);
  strides(a.grad_out_stride, grad_out);
  strides(a.grad_q_stride, gq);
  strides(a.grad_k_stride, gk);
  strides(a.grad_v_stride, gv);
  run(a, false, q);
  return {gq, gk, gv};
}

// What autograd keeps of a How.
void keep_how(AutogradContext* ctx, const How& how) {
  ctx->saved_data["causal"] = how.causal;
  ctx->saved_data["scale"] = how.scale ? c10::IValue(*how.scale) : c10::IValue();
  ctx->saved_data["offset"] = how.offset ? c10::IValue(*how.offset) : c10::IValue();
}
How kept_how(AutogradContext* ctx) {
  const auto &scale = ctx->saved_data["scale"], &offset = ctx->saved_data["offset"];
  return {ctx->saved_data["causal"].toBool(), scale.isNone() ? std::nullopt : std::optional<double>(scale.toDouble()),
          offset.isNone() ? std::nullopt : std::optional<int64_t>(offset.toInt())};
}
MaybeTensor kept(const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }

struct AttentionFn : torch::autograd::Function<AttentionFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, bool causal,
                        std::optional<double> scale, const MaybeTensor& lengths, std::optional<int64_t> offset) {
    const auto [out, lse] = attention_forward(q, k, v, causal, scale, lengths, offset, true);
    ctx->save_for_backward({q, k, v, out, *lse, lengths ? *lengths : Tensor()});
    keep_how(ctx, {causal, scale, offset});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const How how = kept_how(ctx);
    const auto [gq, gk, gv] =
        attention_backward(s[0], s[1], s[2], s[3], s[4], grads[0], how.causal, how.scale, kept(s[5]), how.offset);
    return once({gq, gk, gv, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor attention(const Tensor& q, const Tensor& k, const Tensor& v, bool causal, std::optional<double> scale,
                 const MaybeTensor& lengths, std::optional<int64_t> offset) {
  if (at::GradMode::is_enabled() && (records(q) || records(k) || records(v)))
    return AttentionFn::apply(q, k, v, causal, scale, lengths, offset);
  return std::get<0>(attention_forward(q, k, v, causal, scale, lengths, offset, false));
}

// Queries, keys and values side by side in one contiguous [batch, tokens, (heads + 2 kv_heads) * dim].
lwl_attention_args packed_args(const Tensor& qkv, int64_t heads, int64_t kv_heads, const How& how) {
  if (qkv.dim() != 3 || heads <= 0 || kv_heads <= 0 || qkv.size(2) % (heads + 2 * kv_heads))
    refuse("attention_packed: ", qkv.sizes(), " does not hold ", heads, " query and twice ", kv_heads, " key heads");
  const int64_t tokens = qkv.size(1), width = qkv.size(2), dim = width / (heads + 2 * kv_heads);
  // queries and keys are the same tokens, whatever a sequence's length
  const How same{how.causal, how.scale, how.offset.value_or(0)};
  lwl_attention_args a = shape_args(qkv.scalar_type(), same, qkv.size(0), heads, kv_heads, tokens, tokens, dim);
  const int64_t in[3] = {tokens * width, dim, width}, res[3] = {tokens * heads * dim, dim, heads * dim};
  for (int i = 0; i < 3; ++i) {
    a.q_stride[i] = a.k_stride[i] = a.v_stride[i] = a.grad_q_stride[i] = a.grad_k_stride[i] = a.grad_v_stride[i] = in[i];
    a.out_stride[i] = a.grad_out_stride[i] = res[i];
  }
  return a;
}
char* head_of(const Tensor& qkv, const lwl_attention_args& a, int64_t head) {
  return (char*)qkv.data_ptr() + head * a.dim * qkv.element_size();
}

std::tuple<Tensor, MaybeTensor> packed_forward(const Tensor& qkv, int64_t heads, int64_t kv_heads, bool causal,
                                               std::optional<double> scale, const MaybeTensor& lengths0,
                                               std::optional<int64_t> offset, bool keep_lse) {
  on_one_gpu(qkv, lengths0);
  lwl_attention_args a = packed_args(qkv, heads, kv_heads, {causal, scale, offset});
  const c10::DeviceGuard guard(qkv.device());
  const MaybeTensor lengths = lengths_of(lengths0, a.batch);
  const Tensor out = at::empty({a.batch, a.queries, heads * a.dim}, qkv.options());
  MaybeTensor lse;
  if (keep_lse) lse = at::empty({a.batch, heads, a.queries}, qkv.options().dtype(at::kFloat));
  a.q = qkv.data_ptr();
  a.k = head_of(qkv, a, heads);
  a.v = head_of(qkv, a, heads + kv_heads);
  a.out = out.data_ptr();
  a.lse = (float*)ptr(lse);
  a.key_lengths = (const int32_t*)ptr(lengths);
  run(a, true, qkv);
  return {out, lse};
}

struct PackedFn : torch::autograd::Function<PackedFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& qkv, int64_t heads, int64_t kv_heads, bool causal,
                        std::optional<double> scale, const MaybeTensor& lengths, std::optional<int64_t> offset) {
    const auto [out, lse] = packed_forward(qkv, heads, kv_heads, causal, scale, lengths, offset, true);
    ctx->save_for_backward({qkv, out, *lse, lengths ? *lengths : Tensor()});
    keep_how(ctx, {causal, scale, offset});
    ctx->saved_data["heads"] = heads;
    ctx->saved_data["kv_heads"] = kv_heads;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    on_one_gpu(s[0], s[1], s[2], kept(s[3]), grads[0]);
    const Tensor qkv = s[0].contiguous(), out = s[1].contiguous(), lse = s[2];
    const int64_t heads = ctx->saved_data["heads"].toInt(), kv_heads = ctx->saved_data["kv_heads"].toInt();
    lwl_attention_args a = packed_args(qkv, heads, kv_heads, kept_how(ctx));
    check_left(a, qkv, {a.batch, a.queries, heads * a.dim}, out, lse, grads[0]);
    const c10::DeviceGuard guard(qkv.device());
    const MaybeTensor lengths = lengths_of(kept(s[3]), a.batch);
    const Tensor grad_out = typed(grads[0], qkv.scalar_type()).contiguous(), grad = at::empty(qkv.sizes(), qkv.options());
    a.q = qkv.data_ptr();
    a.k = head_of(qkv, a, heads);
    a.v = head_of(qkv, a, heads + kv_heads);
    a.out = out.data_ptr();
    a.lse = (float*)lse.data_ptr();
    a.key_lengths = (const int32_t*)ptr(lengths);
    a.grad_out = grad_out.data_ptr();
    a.grad_q = grad.data_ptr();
    a.grad_k = head_of(grad, a, heads);
    a.grad_v = head_of(grad, a, heads + kv_heads);
    run(a, false, qkv);
    return once({grad, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor attention_packed(const Tensor& qkv0, int64_t heads, int64_t kv_heads, bool causal, std::optional<double> scale,
                        const MaybeTensor& lengths, std::optional<int64_t> offset) {
  const Tensor qkv = qkv0.contiguous();
  if (at::GradMode::is_enabled() && records(qkv))
    return PackedFn::apply(qkv, heads, kv_heads, causal, scale, lengths, offset);
  return std::get<0>(packed_forward(qkv, heads, kv_heads, causal, scale, lengths, offset, false));
}

// Takes the entries from the library at `path`, which the package has loaded, and the class of its
// argument errors.
void bind(const std::string& path, py::object error_class) {
  void* handle = dlopen(path.c_str(), RTLD_NOW | RTLD_NOLOAD);
  if (!handle) throw std::runtime_error("latent_weight_lab_amd: " + path + " is not loaded");
  const auto get = [&](auto& fn, const char* name) {
    fn = reinterpret_cast<std::decay_t<decltype(fn)>>(dlsym(handle, name));
    if (!fn) throw std::runtime_error(std::string("latent_weight_lab_amd: no ") + name + " in the library");
  };
  get(lib.last_error, "lwl_last_error");
  get(lib.norm_forward, "lwl_layer_norm_forward");
  get(lib.norm_backward_workspace, "lwl_layer_norm_backward_workspace_size");
  get(lib.norm_backward, "lwl_layer_norm_backward");
  get(lib.gelu8_pitch, "lwl_gelu8_pitch");
  get(lib.gelu8_forward, "lwl_gelu8_forward");
  get(lib.gelu8_activation, "lwl_gelu8_activation");
  get(lib.gelu8_backward_workspace, "lwl_gelu8_backward_workspace_size");
  get(lib.gelu8_backward, "lwl_gelu8_backward");
  get(lib.attention_forward_workspace, "lwl_attention_forward_workspace_size");
  get(lib.attention_forward, "lwl_attention_forward");
  get(lib.attention_backward_workspace, "lwl_attention_backward_workspace_size");
  get(lib.attention_backward, "lwl_attention_backward");
  argument_error = error_class.release().ptr();
}

}  // namespace

PYBIND11_MODULE(lwl_layers, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const ArgumentError& e) {
      PyErr_SetString(argument_error ? argument_error : PyExc_ValueError, e.what());
    } catch (const c10::NotImplementedError& e) {
      PyErr_SetString(PyExc_NotImplementedError, e.what_without_backtrace());
    }
  });
  using release = py::call_guard<py::gil_scoped_release>;
  m.def("bind", &bind);
  m.def("layer_norm", &layer_norm, release());
  m.def("gelu8", &gelu8, release());
  m.def("gelu8_activation", &gelu8_activation, release());
  m.def("gelu8_backward", &gelu8_backward, release());
  m.def("attention_forward", &attention_forward, release());
  m.def("attention_backward", &attention_backward, release());
  m.def("attention", &attention, release());
  m.def("attention_packed", &attention_packed, release());
}
