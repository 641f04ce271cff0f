// C ABI of the layer operators (declared in include/lwl_layers.h): argument checks, workspace sizes
// and the launches.  Host code only.
#include "../../include/lwl_layers.h"

#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cmath>

#include "layer_launch.h"

namespace {

using lwl::attention_args;
using lwl::check_attention;
using lwl::status_fail;
using lwl::status_hip;
using lwl::status_ok;
using lwl::status_workspace;

constexpr size_t kAlign = 256;
size_t align_up(size_t v) { return (v + kAlign - 1) / kAlign * kAlign; }

bool valid_dtype(int d) { return d == LWL_DTYPE_F32 || d == LWL_DTYPE_F16 || d == LWL_DTYPE_BF16; }

constexpr int64_t kMostFeatures = (int64_t)1 << 24;
// rows x features elements that fit 2^47 (pointers) with room for a workgroup's rounding up
bool fits(int64_t rows, int64_t features) { return rows <= ((int64_t)1 << 46) / features; }

int check_norm(int dtype, int weight_dtype, int64_t rows, int64_t features, double eps) {
  if (!valid_dtype(dtype) || !valid_dtype(weight_dtype))
    return status_fail(LWL_ERR_UNSUPPORTED, "layer norm supports float32, float16 and bfloat16");
  if (weight_dtype != dtype && weight_dtype != LWL_DTYPE_F32)
    return status_fail(LWL_ERR_UNSUPPORTED, "layer norm's weight must be float32 or of the input's type");
  if (rows < 0) return status_fail(LWL_ERR_INVALID, "layer norm: rows must be non-negative");
  if (features <= 0) return status_fail(LWL_ERR_INVALID, "layer norm: features must be positive");
  if (features > kMostFeatures || !fits(rows, features))
    return status_fail(LWL_ERR_UNSUPPORTED, "layer norm: %lld rows of %lld features are too many", (long long)rows,
                       (long long)features);
  if (!(eps >= 0.0) || !std::isfinite(eps))
    return status_fail(LWL_ERR_INVALID, "layer norm: eps must be finite and non-negative");
  return LWL_OK;
}

int check_gelu8(int dtype, int64_t rows, int64_t features) {
  if (!valid_dtype(dtype))
    return status_fail(LWL_ERR_UNSUPPORTED, "GELU checkpoint supports float32, float16 and bfloat16 (dtype code %d)",
                       dtype);
  if (rows < 0) return status_fail(LWL_ERR_INVALID, "GELU checkpoint: rows must be non-negative");
  if (features <= 0) return status_fail(LWL_ERR_INVALID, "GELU checkpoint: features must be positive");
  if (features > kMostFeatures || !fits(rows, features))
    return status_fail(LWL_ERR_UNSUPPORTED, "GELU checkpoint: %lld rows of %lld features are too many",
                       (long long)rows, (long long)features);
  return LWL_OK;
}

int check_kept(const int8_t* codes, const float* scales, int64_t rows) {
  if (rows == 0) return LWL_OK;
  if (!codes || !scales)
    return status_fail(LWL_ERR_INVALID, "GELU checkpoint: codes and scales must be non-null");
  if ((uintptr_t)codes % 8) return status_fail(LWL_ERR_INVALID, "GELU checkpoint: codes must be 8-byte aligned");
  return LWL_OK;
}

lwl::Gelu8Args gelu8_args(int dtype, int tanh_form, int64_t rows, int64_t features, const int8_t* codes,
                          const float* scales) {
  lwl::Gelu8Args g{};
  g.dtype = dtype;
  g.tanh_form = tanh_form != 0;
  g.rows = rows;
  g.features = features;
  g.codes = const_cast<int8_t*>(codes);
  g.scales = const_cast<float*>(scales);
  return g;
}

}  // namespace

namespace lwl {

int check_attention(const lwl_attention_args* a) {
  if (!a) return status_fail(LWL_ERR_INVALID, "attention: args must be non-null");
  if (!valid_dtype(a->dtype))
    return status_fail(LWL_ERR_UNSUPPORTED, "attention supports float32, float16 and bfloat16 (dtype code %d)", a->dtype);
  if (a->reserved != 0) return status_fail(LWL_ERR_INVALID, "attention: reserved must be 0");
  if (a->batch < 0 || a->queries < 0 || a->keys < 0)
    return status_fail(LWL_ERR_INVALID, "attention: batch, queries and keys must be non-negative");
  if (a->heads <= 0 || a->kv_heads <= 0 || a->heads % a->kv_heads)
    return status_fail(LWL_ERR_INVALID, "attention: %lld query heads over %lld key heads: must be a positive multiple",
                       (long long)a->heads, (long long)a->kv_heads);
  if (a->dim <= 0) return status_fail(LWL_ERR_INVALID, "attention: the head size must be positive");
  if (a->dim > LWL_ATTENTION_MAX_DIM)
    return status_fail(LWL_ERR_UNSUPPORTED, "attention supports head sizes up to %d (got %lld)", LWL_ATTENTION_MAX_DIM,
                       (long long)a->dim);
  // the kernels multiply by scale * log2(e) and, in 16-bit types' backward, by its reciprocal times log sums
  if (!(a->scale >= 0x1p-100 && a->scale <= 0x1p100))
    return status_fail(LWL_ERR_INVALID, "attention: scale must be positive, from 2^-100 to 2^100");
  // token indexes are 32 bits in the kernels, workgroups are counted in 32 bits
  const int64_t kTokens = (int64_t)1 << 30, kCount = (int64_t)1 << 31;
  if (a->keys > kTokens || a->queries > kTokens || a->heads > kTokens || a->batch > kTokens)
    return status_fail(LWL_ERR_UNSUPPORTED, "attention: more than 2^30 tokens, heads or sequences");
  const int64_t bh = a->batch * a->heads, blocks = (std::max(a->queries, a->keys) + 15) / 16;
  if (bh >= kCount || bh * blocks >= kCount)
    return status_fail(LWL_ERR_UNSUPPORTED, "attention: too many heads, sequences and tokens in one call");
  if (a->causal && !a->bottom_right && (a->causal_offset > kTokens || a->causal_offset < -kTokens))
    return status_fail(LWL_ERR_UNSUPPORTED, "attention: causal offset beyond 2^30");
  return LWL_OK;
}

int fail_workgroups() {
  return status_fail(LWL_ERR_UNSUPPORTED, "attention: more than %lld workgroups in one call", (long long)kMostWorkgroups);
}

AttnArgs attention_args(const lwl_attention_args* a) {
  AttnArgs t{};
  t.dtype = a->dtype;
  t.causal = a->causal != 0;
  t.bottom_right = a->bottom_right != 0;
  t.causal_offset = a->causal_offset;
  t.batch = a->batch;
  t.heads = a->heads;
  t.kv_heads = a->kv_heads;
  t.queries = a->queries;
  t.keys = a->keys;
  t.dim = a->dim;
  t.scale = (float)a->scale;
  t.q = a->q;
  t.k = a->k;
  t.v = a->v;
  t.out = a->out;
  t.lse = a->lse;
  t.lengths = a->key_lengths;
  t.dout = a->grad_out;
  t.dq = a->grad_q;
  t.dk = a->grad_k;
  t.dv = a->grad_v;
  for (int i = 0; i < 3; ++i) {
    t.qs[i] = a->q_stride[i];
    t.ks[i] = a->k_stride[i];
    t.vs[i] = a->v_stride[i];
    t.os[i] = a->out_stride[i];
    t.dos[i] = a->grad_out_stride[i];
    t.dqs[i] = a->grad_q_stride[i];
    t.dks[i] = a->grad_k_stride[i];
    t.dvs[i] = a->grad_v_stride[i];
  }
  return t;
}

}  // namespace lwl

namespace {

int check_forward(const lwl_attention_args* a) {
  const int rc = check_attention(a);
  return rc || lwl::attention_fwd_fits(attention_args(a)) ? rc : lwl::fail_workgroups();
}
int check_backward(const lwl_attention_args* a) {
  const int rc = check_attention(a);
  return rc || lwl::attention_bwd_fits(attention_args(a)) ? rc : lwl::fail_workgroups();
}

}  // namespace

extern "C" {

int lwl_layer_norm_check(int dtype, int weight_dtype, int64_t rows, int64_t features, double eps) {
  const int rc = check_norm(dtype, weight_dtype, rows, features, eps);
  return rc ? rc : status_ok();
}

int lwl_layer_norm_forward(const void* x, const void* residual, const void* weight, const void* bias, int dtype,
                           int weight_dtype, int64_t rows, int64_t features, double eps, void* out, void* sum,
                           float* stats, void* stream) {
  const int rc = check_norm(dtype, weight_dtype, rows, features, eps);
  if (rc) return rc;
  if (rows == 0) return status_ok();
  if (!x || !weight || !out) return status_fail(LWL_ERR_INVALID, "layer norm: x, weight and out must be non-null");
  if (!residual != !sum) return status_fail(LWL_ERR_INVALID, "layer norm: residual and sum go together");
  lwl::NormArgs n{};
  n.dtype = dtype;
  n.weight_dtype = weight_dtype;
  n.rows = rows;
  n.features = features;
  n.x = x;
  n.residual = residual;
  n.weight = weight;
  n.bias = bias;
  n.out = out;
  n.sum = sum;
  n.stats = stats;
  n.eps = (float)eps;
  return status_hip(lwl::launch_norm_fwd(n, (hipStream_t)stream), "lwl_layer_norm_forward");
}

size_t lwl_layer_norm_backward_workspace_size(int64_t rows, int64_t features) {
  if (rows <= 0 || features <= 0) return 0;
  return align_up((size_t)lwl::norm_bwd_partial_rows(rows, features) * 2 * (size_t)features * sizeof(float));
}

int lwl_layer_norm_backward(const void* h, const void* weight, const float* stats, const void* grad_out,
                            const void* grad_sum, int dtype, int weight_dtype, int64_t rows, int64_t features,
                            void* grad_x, void* grad_weight, void* grad_bias, void* workspace,
                            size_t workspace_bytes, void* stream) {
  int rc = check_norm(dtype, weight_dtype, rows, features, 0.0);
  if (rc) return rc;
  if (rows > 0 && (!h || !weight || !stats || !grad_out))
    return status_fail(LWL_ERR_INVALID, "layer norm backward: h, weight, stats and grad_out must be non-null");
  if (!grad_x && !grad_weight && !grad_bias) return status_ok();
  if (grad_weight || grad_bias) {
    rc = status_workspace(lwl_layer_norm_backward_workspace_size(rows, features), workspace, workspace_bytes);
    if (rc) return rc;
  }
  lwl::NormArgs n{};
  n.dtype = dtype;
  n.weight_dtype = weight_dtype;
  n.rows = rows;
  n.features = features;
  n.x = h;
  n.weight = weight;
  n.stats = const_cast<float*>(stats);
  n.grad_out = grad_out;
  n.grad_sum = grad_sum;
  n.grad_x = grad_x;
  n.grad_weight = grad_weight;
  n.grad_bias = grad_bias;
  n.work = (float*)workspace;
  return status_hip(lwl::launch_norm_bwd(n, (hipStream_t)stream), "lwl_layer_norm_backward");
}

int64_t lwl_gelu8_pitch(int64_t features) { return lwl::gelu8_pitch(features); }

int lwl_gelu8_check(int dtype, int64_t rows, int64_t features) {
  const int rc = check_gelu8(dtype, rows, features);
  return rc ? rc : status_ok();
}

int lwl_gelu8_forward(const void* x, const void* bias, int dtype, int tanh_form, int64_t rows, int64_t features,
                      void* out, int8_t* codes, float* scales, void* stream) {
  int rc = check_gelu8(dtype, rows, features);
  if (rc) return rc;
  if (rows == 0) return status_ok();
  if (!x || !out) return status_fail(LWL_ERR_INVALID, "GELU checkpoint: x and out must be non-null");
  if (codes && (rc = check_kept(codes, scales, rows))) return rc;
  lwl::Gelu8Args g = gelu8_args(dtype, tanh_form, rows, features, codes, scales);
  g.x = x;
  g.bias = bias;
  g.out = out;
  return status_hip(lwl::launch_gelu8_fwd(g, (hipStream_t)stream), "lwl_gelu8_forward");
}

int lwl_gelu8_activation(const int8_t* codes, const float* scales, int dtype, int tanh_form, int64_t rows,
                         int64_t features, void* out, void* stream) {
  int rc = check_gelu8(dtype, rows, features);
  if (rc || (rc = check_kept(codes, scales, rows))) return rc;
  if (rows == 0) return status_ok();
  if (!out) return status_fail(LWL_ERR_INVALID, "GELU checkpoint: out must be non-null");
  lwl::Gelu8Args g = gelu8_args(dtype, tanh_form, rows, features, codes, scales);
  g.out = out;
  return status_hip(lwl::launch_gelu8_activation(g, (hipStream_t)stream), "lwl_gelu8_activation");
}

size_t lwl_gelu8_backward_workspace_size(int64_t rows, int64_t features) {
  if (rows <= 0 || features <= 0) return 0;
  return align_up((size_t)lwl::gelu8_bwd_partial_rows(rows, features) * (size_t)features * sizeof(float));
}

int lwl_gelu8_backward(const int8_t* codes, const float* scales, const void* grad_out, int dtype, int tanh_form,
                       int64_t rows, int64_t features, void* grad_x, void* grad_bias, void* workspace,
                       size_t workspace_bytes, void* stream) {
  int rc = check_gelu8(dtype, rows, features);
  if (rc || (rc = check_kept(codes, scales, rows))) return rc;
  if (rows > 0 && (!grad_out || !grad_x))
    return status_fail(LWL_ERR_INVALID, "GELU checkpoint backward: grad_out and grad_x must be non-null");
  if (grad_bias) {
    rc = status_workspace(lwl_gelu8_backward_workspace_size(rows, features), workspace, workspace_bytes);
    if (rc) return rc;
  }
  lwl::Gelu8Args g = gelu8_args(dtype, tanh_form, rows, features, codes, scales);
  g.grad_out = grad_out;
  g.out = grad_x;
  g.grad_bias = grad_bias;
  g.work = (float*)workspace;
  return status_hip(lwl::launch_gelu8_bwd(g, (hipStream_t)stream), "lwl_gelu8_backward");
}

int lwl_attention_check(const lwl_attention_args* args) {
  const int rc = check_forward(args);
  return rc ? rc : status_ok();
}

size_t lwl_attention_forward_workspace_size(const lwl_attention_args* args) {
  if (check_forward(args)) return 0;
  return align_up((size_t)lwl::attention_fwd_work(attention_args(args)) * sizeof(float));
}

int lwl_attention_forward(const lwl_attention_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_forward(args);
  if (rc) return rc;
  if (args->batch == 0 || args->queries == 0) return status_ok();
  if (!args->q || !args->out || (args->keys > 0 && (!args->k || !args->v)))
    return status_fail(LWL_ERR_INVALID, "attention: q, k, v and out must be non-null");
  rc = status_workspace(lwl_attention_forward_workspace_size(args), workspace, workspace_bytes);
  if (rc) return rc;
  lwl::AttnArgs t = attention_args(args);
  t.work = (float*)workspace;
  return status_hip(lwl::launch_attention_fwd(t, (hipStream_t)stream), "lwl_attention_forward");
}

size_t lwl_attention_backward_workspace_size(const lwl_attention_args* args) {
  if (check_backward(args)) return 0;
  return align_up((size_t)lwl::attention_bwd_work(attention_args(args)) * sizeof(float));
}

int lwl_attention_backward(const lwl_attention_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_backward(args);
  if (rc) return rc;
  if (args->batch == 0 || (args->queries == 0 && args->keys == 0)) return status_ok();
  if ((args->queries > 0 && (!args->q || !args->out || !args->lse || !args->grad_out || !args->grad_q)) ||
      (args->keys > 0 && (!args->k || !args->v || !args->grad_k || !args->grad_v)))
    return status_fail(LWL_ERR_INVALID,
                       "attention backward: q, k, v, out, lse, grad_out, grad_q, grad_k and grad_v must be non-null");
  rc = status_workspace(lwl_attention_backward_workspace_size(args), workspace, workspace_bytes);
  if (rc) return rc;
  lwl::AttnArgs t = attention_args(args);
  t.work = (float*)workspace;
  return status_hip(lwl::launch_attention_bwd(t, (hipStream_t)stream), "lwl_attention_backward");
}

}  // extern "C"
