// C ABI of attention within a window and of a tree, and of tokens' log probabilities (declared in
// include/lwl_tokens.h): argument checks, workspace sizes and the launches.  Host code only.
#include "../../include/lwl_tokens.h"

#include <hip/hip_runtime_api.h>

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

int check_window(const lwl_attention_args* a, int64_t window, int64_t sinks) {
  const int rc = check_attention(a);
  if (rc) return rc;
  if (!a->causal) return status_fail(LWL_ERR_INVALID, "attention: a window needs causal order");
  if (window < 1) return status_fail(LWL_ERR_INVALID, "attention: the window must be positive (got %lld)", (long long)window);
  if (sinks < 0)
    return status_fail(LWL_ERR_INVALID, "attention: sinks must be non-negative (got %lld)", (long long)sinks);
  return LWL_OK;
}
lwl::AttnArgs window_args(const lwl_attention_args* a, int64_t window, int64_t sinks) {
  lwl::AttnArgs t = attention_args(a);
  // the kernels' token numbers have 32 bits; positions reach 2^31, and a window past that hides nothing
  const int64_t most = ((int64_t)1 << 31) - 1, tokens = (int64_t)1 << 30;
  t.window = window < most ? window : most;
  t.sinks = sinks < tokens ? sinks : tokens;
  return t;
}

int check_window_forward(const lwl_attention_args* a, int64_t window, int64_t sinks) {
  const int rc = check_window(a, window, sinks);
  return rc || lwl::attention_window_fwd_fits(window_args(a, window, sinks)) ? rc : lwl::fail_workgroups();
}
int check_window_backward(const lwl_attention_args* a, int64_t window, int64_t sinks) {
  const int rc = check_window(a, window, sinks);
  return rc || lwl::attention_window_bwd_fits(window_args(a, window, sinks)) ? rc : lwl::fail_workgroups();
}

int check_tree(const lwl_attention_args* a) {
  const int rc = check_attention(a);
  if (rc) return rc;
  if (a->causal || a->bottom_right || a->causal_offset)
    return status_fail(LWL_ERR_INVALID, "attention of a tree: causal, bottom_right and causal_offset must be 0");
  if (a->queries > LWL_ATTENTION_MAX_NODES)
    return status_fail(LWL_ERR_UNSUPPORTED, "attention of a tree supports up to %d nodes (got %lld)",
                       LWL_ATTENTION_MAX_NODES, (long long)a->queries);
  // the rows on a key head are counted in 32 bits
  if (a->heads / a->kv_heads * a->queries > (int64_t)1 << 30)
    return status_fail(LWL_ERR_UNSUPPORTED, "attention of a tree: more than 2^30 rows on a key head");
  return lwl::attention_tree_fits(attention_args(a)) ? LWL_OK : lwl::fail_workgroups();
}

int check_log_probs(const lwl_log_probs_args* a) {
  if (!a) return status_fail(LWL_ERR_INVALID, "log probabilities: args must be non-null");
  if (a->dtype != LWL_DTYPE_F32 && a->dtype != LWL_DTYPE_F16 && a->dtype != LWL_DTYPE_BF16)
    return status_fail(LWL_ERR_UNSUPPORTED, "log probabilities support float32, float16 and bfloat16 (dtype code %d)",
                       a->dtype);
  if (a->reserved != 0) return status_fail(LWL_ERR_INVALID, "log probabilities: reserved must be 0");
  if (a->outer < 0 || a->inner < 0)
    return status_fail(LWL_ERR_INVALID, "log probabilities: rows must be non-negative");
  if (a->vocab <= 0) return status_fail(LWL_ERR_INVALID, "log probabilities: the vocabulary must be positive");
  if (a->each < 0 || a->top < 0)
    return status_fail(LWL_ERR_INVALID, "log probabilities: each and top must be non-negative");
  if (a->top > a->vocab)
    return status_fail(LWL_ERR_INVALID, "log probabilities: %d alternatives of %lld tokens", a->top, (long long)a->vocab);
  if (a->each > LWL_LOG_PROBS_MAX_EACH || a->top > LWL_LOG_PROBS_MAX_TOP)
    return status_fail(LWL_ERR_UNSUPPORTED, "log probabilities support up to %d tokens a row and %d alternatives",
                       LWL_LOG_PROBS_MAX_EACH, LWL_LOG_PROBS_MAX_TOP);
  // indexes in a row have 32 bits, a grid's workgroups (of both axes together) are numbered in 32
  const int64_t kVocab = (int64_t)1 << 30, kCount = (int64_t)1 << 31;
  if (a->vocab > kVocab || a->outer >= kCount || a->inner >= kCount || a->outer * a->inner >= kCount ||
      a->outer * a->inner * lwl::log_probs_bwd_ranges(a->vocab) >= kCount)
    return status_fail(LWL_ERR_UNSUPPORTED, "log probabilities: too many rows or tokens in one call");
  return LWL_OK;
}
lwl::LogProbArgs log_prob_args(const lwl_log_probs_args* a) {
  lwl::LogProbArgs t{};
  t.dtype = a->dtype;
  t.each = a->each;
  t.top = a->top;
  t.outer = a->outer;
  t.inner = a->inner;
  t.vocab = a->vocab;
  t.outer_stride = a->outer_stride;
  t.inner_stride = a->inner_stride;
  t.logits = a->logits;
  t.tokens = a->tokens;
  t.log_probs = a->log_probs;
  t.entropy = a->entropy;
  t.top_log_probs = a->top_log_probs;
  t.top_tokens = a->top_tokens;
  t.stats = a->stats;
  t.grad_log_probs = a->grad_log_probs;
  t.grad_entropy = a->grad_entropy;
  t.grad_top = a->grad_top;
  t.grad_logits = a->grad_logits;
  return t;
}

}  // namespace

extern "C" {

int lwl_attention_window_check(const lwl_attention_args* args, int64_t window, int64_t sinks) {
  const int rc = check_window_forward(args, window, sinks);
  return rc ? rc : status_ok();
}

size_t lwl_attention_window_forward_workspace_size(const lwl_attention_args* args, int64_t window, int64_t sinks) {
  if (check_window_forward(args, window, sinks)) return 0;
  return align_up((size_t)lwl::attention_window_fwd_work(window_args(args, window, sinks)) * sizeof(float));
}

int lwl_attention_window_forward(const lwl_attention_args* args, int64_t window, int64_t sinks, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  int rc = check_window_forward(args, window, sinks);
  if (rc) return rc;
  if (args->batch == 0 || args->queries == 0) return status_ok();
  if (!args->q || !args->out || (args->keys > 0 && (!args->k || !args->v)))
    return status_fail(LWL_ERR_INVALID, "attention: q, k, v and out must be non-null");
  rc = status_workspace(lwl_attention_window_forward_workspace_size(args, window, sinks), workspace, workspace_bytes);
  if (rc) return rc;
  lwl::AttnArgs t = window_args(args, window, sinks);
  t.work = (float*)workspace;
  return status_hip(lwl::launch_attention_window_fwd(t, (hipStream_t)stream), "lwl_attention_window_forward");
}

size_t lwl_attention_window_backward_workspace_size(const lwl_attention_args* args, int64_t window, int64_t sinks) {
  if (check_window_backward(args, window, sinks)) return 0;
  return align_up((size_t)lwl::attention_window_bwd_work(window_args(args, window, sinks)) * sizeof(float));
}

int lwl_attention_window_backward(const lwl_attention_args* args, int64_t window, int64_t sinks, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  int rc = check_window_backward(args, window, sinks);
  if (rc) return rc;
  if (args->batch == 0 || (args->queries == 0 && args->keys == 0)) return status_ok();
  if ((args->queries > 0 && (!args->q || !args->out || !args->lse || !args->grad_out || !args->grad_q)) ||
      (args->keys > 0 && (!args->k || !args->v || !args->grad_k || !args->grad_v)))
    return status_fail(LWL_ERR_INVALID,
                       "attention backward: q, k, v, out, lse, grad_out, grad_q, grad_k and grad_v must be non-null");
  rc = status_workspace(lwl_attention_window_backward_workspace_size(args, window, sinks), workspace, workspace_bytes);
  if (rc) return rc;
  lwl::AttnArgs t = window_args(args, window, sinks);
  t.work = (float*)workspace;
  return status_hip(lwl::launch_attention_window_bwd(t, (hipStream_t)stream), "lwl_attention_window_backward");
}

int lwl_attention_tree_check(const lwl_attention_args* args) {
  const int rc = check_tree(args);
  return rc ? rc : status_ok();
}

size_t lwl_attention_tree_workspace_size(const lwl_attention_args* args) {
  if (check_tree(args)) return 0;
  return align_up((size_t)lwl::attention_tree_work(attention_args(args)) * sizeof(float));
}

int lwl_attention_tree_forward(const lwl_attention_args* args, const int32_t* parents, int64_t parents_stride,
                               void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_tree(args);
  if (rc) return rc;
  if (args->batch == 0 || args->queries == 0) return status_ok();
  if (!args->q || !args->out || !parents || (args->keys > 0 && (!args->k || !args->v)))
    return status_fail(LWL_ERR_INVALID, "attention of a tree: q, k, v, out and parents must be non-null");
  rc = status_workspace(lwl_attention_tree_workspace_size(args), workspace, workspace_bytes);
  if (rc) return rc;
  lwl::AttnArgs t = attention_args(args);
  t.parents = parents;
  t.parents_stride = parents_stride;
  t.work = (float*)workspace;
  return status_hip(lwl::launch_attention_tree(t, (hipStream_t)stream), "lwl_attention_tree_forward");
}

int lwl_log_probs_check(const lwl_log_probs_args* args) {
  const int rc = check_log_probs(args);
  return rc ? rc : status_ok();
}

int lwl_log_probs_forward(const lwl_log_probs_args* args, void* stream) {
  const int rc = check_log_probs(args);
  if (rc) return rc;
  if (args->outer == 0 || args->inner == 0) return status_ok();
  if (!args->logits) return status_fail(LWL_ERR_INVALID, "log probabilities: logits must be non-null");
  if ((args->each > 0) != (args->tokens != nullptr) || (args->each > 0) != (args->log_probs != nullptr))
    return status_fail(LWL_ERR_INVALID, "log probabilities: tokens and log_probs go with each");
  if ((args->top > 0) != (args->top_log_probs != nullptr) || (args->top > 0) != (args->top_tokens != nullptr))
    return status_fail(LWL_ERR_INVALID, "log probabilities: top_log_probs and top_tokens go with top");
  return status_hip(lwl::launch_log_probs_fwd(log_prob_args(args), (hipStream_t)stream), "lwl_log_probs_forward");
}

int lwl_log_probs_backward(const lwl_log_probs_args* args, void* stream) {
  const int rc = check_log_probs(args);
  if (rc) return rc;
  if (args->outer == 0 || args->inner == 0) return status_ok();
  if (!args->logits || !args->stats || !args->grad_logits)
    return status_fail(LWL_ERR_INVALID, "log probabilities backward: logits, stats and grad_logits must be non-null");
  if ((args->grad_log_probs && (args->each == 0 || !args->tokens)) || (args->grad_entropy && !args->entropy) ||
      (args->grad_top && (args->top == 0 || !args->top_tokens)))
    return status_fail(LWL_ERR_INVALID, "log probabilities backward: a gradient without what the forward left of its result");
  return status_hip(lwl::launch_log_probs_bwd(log_prob_args(args), (hipStream_t)stream), "lwl_log_probs_backward");
}

}  // extern "C"
