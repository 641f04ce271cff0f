/*
 * lwl_layers.h — C ABI of the operators between a transformer block's generated linears: layer
 * norm, attention, and GELU whose input is kept in 8 bits for the backward pass.  Part of
 * liblwl_bfht.so; element types, status codes, streams, workspaces and lwl_last_error() as in
 * lwl_bfht.h.  The reference has no counterpart: its model calls torch for these
 * (examples/nanogpt/model.py).
 *
 * Every entry is asynchronous on `stream`, allocates nothing, never synchronizes and may be captured
 * into a HIP graph.  Sums, softmax statistics, means and variances are float32; every result is
 * rounded once to its type.  Results do not depend on the order in which workgroups run (no float
 * atomics).
 */
#ifndef LWL_LAYERS_H
#define LWL_LAYERS_H

#include "lwl_bfht.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------- layer norm
 * Rows of `features` values, row-major and contiguous, x in `dtype`, weight and bias in
 * weight_dtype (float32, or dtype itself):
 *
 *   h = x, or round(x + residual) to dtype;  mu = mean(h);  s = 1 / sqrt(mean((h - mu)^2) + eps)
 *   out = (h - mu) * s * weight + bias
 *
 * residual and bias may be NULL; `sum` receives h and is NULL exactly when residual is.  `stats`
 * (float32 [2][rows]: mu, then s) is what the backward needs and may be NULL.  out and sum may not
 * overlap the inputs.
 */
int lwl_layer_norm_check(int dtype, int weight_dtype, int64_t rows, int64_t features, double eps); /* host only */
int lwl_layer_norm_forward(const void* x, const void* residual, const void* weight, const void* bias, int dtype,
                           int weight_dtype, int64_t rows, int64_t features, double eps, void* out, void* sum,
                           float* stats, void* stream);

/* Backward: h is what was normed (x, or the stored sum), stats as the forward left it.  With
 * n = (h - mu) s, a = grad_out * weight:
 *
 *   grad_x = s (a - mean(a) - n mean(a n)) + grad_sum     (of x, and of residual: the same)
 *   grad_weight = sum over rows of grad_out * n,  grad_bias = sum over rows of grad_out
 *
 * grad_sum (the gradient of h from elsewhere) may be NULL, and each output may be NULL.  The sums
 * over rows run in a fixed order.
 */
size_t lwl_layer_norm_backward_workspace_size(int64_t rows, int64_t features);
int lwl_layer_norm_backward(const void* h, const void* weight, const float* stats, const void* grad_out,
                            const void* grad_sum, int dtype, int weight_dtype, int64_t rows, int64_t features,
                            void* grad_x, void* grad_weight, void* grad_bias, void* workspace,
                            size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------- GELU, input kept in 8 bits
 * z = x + bias (bias may be NULL) over rows of `features` values; out = gelu(z): z Phi(z), or with
 * tanh_form its tanh approximation.  Kept of z: for each row and each group of
 * LWL_GELU8_GROUP consecutive features one float32 scale s = max|z| / 127 and int8 codes
 * c = rint(z / s), standing for c * s.  codes: rows of lwl_gelu8_pitch(features) bytes, 8-byte aligned;
 * scales: float32 rows of ceil(features / LWL_GELU8_GROUP).  In the forward codes == NULL (then scales is
 * not read) keeps nothing.  A group of values below 2^-100 stands for zeros; one with an infinity or a
 * NaN stands for NaN.
 */
#define LWL_GELU8_GROUP 128
int64_t lwl_gelu8_pitch(int64_t features);
int lwl_gelu8_check(int dtype, int64_t rows, int64_t features); /* host only */
int lwl_gelu8_forward(const void* x, const void* bias, int dtype, int tanh_form, int64_t rows, int64_t features,
                      void* out, int8_t* codes, float* scales, void* stream);
/* out = gelu(c * s): the activation again, from the checkpoint. */
int lwl_gelu8_activation(const int8_t* codes, const float* scales, int dtype, int tanh_form, int64_t rows,
                         int64_t features, void* out, void* stream);
/* grad_x = grad_out * gelu'(c * s); grad_bias (may be NULL): its sum over rows, in a fixed order. */
size_t lwl_gelu8_backward_workspace_size(int64_t rows, int64_t features);
int lwl_gelu8_backward(const int8_t* codes, const float* scales, const void* grad_out, int dtype, int tanh_form,
                       int64_t rows, int64_t features, void* grad_x, void* grad_bias, void* workspace,
                       size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------- attention
 * For each sequence b and query head h, whose key head is h / (heads / kv_heads):
 *
 *   out_i = sum_j P_ij v_j,  P_i = softmax over the allowed j of scale * (q_i . k_j)
 *   lse_i = log sum over the allowed j of exp(scale * q_i . k_j)
 *
 * Key j is allowed where j < key_lengths[b] (device int32, values in 0 .. keys; NULL: keys) and, with
 * `causal`, j <= i + offset; offset is causal_offset, or with bottom_right the sequence's length minus
 * queries (the queries are its last tokens).  A query with no allowed key has out = 0, lse = -infinity
 * and no part in any gradient.  What lies past a sequence's length is never multiplied in: it may hold
 * anything.
 *
 * Tensors are [batch, heads, tokens, dim] with the given strides in elements (batch, head, token) and
 * consecutive values along dim; any order, sharing (stride 0 of an input) and alignment of an element.
 * dim is 1 .. LWL_ATTENTION_MAX_DIM, heads a multiple of kv_heads, scale from 2^-100 to 2^100.  lse
 * (float32 [batch][heads][queries], contiguous) may be NULL in the forward.
 *
 * Not finite: a NaN in a key or value that some query may see reaches that query's results, and may reach
 * those of other queries whose `causal` limit hides it (its probability 0 is multiplied by it), as
 * it does where a masked score matrix is multiplied out; in the backward so may one in a query or its gradient
 * reach the gradients of keys hidden from it.  float32 tensors that hold infinities give NaN: their products
 * are those of bfloat16 parts.
 */
#define LWL_ATTENTION_MAX_DIM 128
typedef struct lwl_attention_args {
  int32_t dtype, causal, bottom_right, reserved; /* reserved: 0 */
  int64_t causal_offset;
  int64_t batch, heads, kv_heads, queries, keys, dim;
  double scale;
  const void *q, *k, *v;
  void* out; /* the backward's input */
  float* lse;
  const int32_t* key_lengths;
  int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3];
  /* backward only */
  const void* grad_out;
  void *grad_q, *grad_k, *grad_v;
  int64_t grad_out_stride[3], grad_q_stride[3], grad_k_stride[3], grad_v_stride[3];
} lwl_attention_args;

int lwl_attention_check(const lwl_attention_args* args); /* host only; does not look at pointers */
size_t lwl_attention_forward_workspace_size(const lwl_attention_args* args);
int lwl_attention_forward(const lwl_attention_args* args, void* workspace, size_t workspace_bytes, void* stream);
/* The probabilities are computed again from q, k and lse.  grad_k and grad_v are summed over the query
 * heads that share a key head; all three gradients are overwritten whole (zeros where nothing reaches).
 * float32 divides each row of probabilities by its sum, so that lse's rounding does not count.  16-bit types
 * round probabilities and scores' gradients to the type before their products; float16 holds the latter
 * times powers of two, so that they neither leave its range nor lose digits at its lower end. */
size_t lwl_attention_backward_workspace_size(const lwl_attention_args* args);
int lwl_attention_backward(const lwl_attention_args* args, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LWL_LAYERS_H */
