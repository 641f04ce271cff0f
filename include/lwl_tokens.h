/*
 * lwl_tokens.h — C ABI of what answering over long caches and with drafts needs beside lwl_layers.h:
 * attention within a sliding window whose first tokens stay visible, attention of a tree of drafted tokens
 * over a cache, and log probabilities of given tokens with the entropy and the most probable alternatives.
 * Part of liblwl_bfht.so; element types, status codes, streams, workspaces and lwl_last_error() as in
 * lwl_bfht.h.  The reference has no counterpart (its model calls torch's attention and cross entropy,
 * examples/nanogpt/model.py).
 *
 * Every entry is asynchronous on `stream`, allocates nothing, never synchronizes and may be captured
 * into a HIP graph.  Sums and softmax statistics are float32; every result is rounded once to its
 * type.  Results do not depend on the order in which workgroups run.
 */
#ifndef LWL_TOKENS_H
#define LWL_TOKENS_H

#include "lwl_layers.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------- attention within a window
 * lwl_attention_* (lwl_layers.h) where of the keys up to its own position p = i + offset a query sees the
 * last `window` (p among them) and the first `sinks`:
 *
 *   key j is allowed where j < key_lengths[b], j <= p, and j > p - window or j < sinks.
 *
 * args->causal must be 1; window at least 1, sinks from 0.  Only keys that a query of the same block of 128 sees
 * are read, so a long sequence costs its length times the window.  What lwl_layers.h says of values that are
 * not finite holds of keys that the window hides, too.
 */
int lwl_attention_window_check(const lwl_attention_args* args, int64_t window, int64_t sinks); /* host only */
size_t lwl_attention_window_forward_workspace_size(const lwl_attention_args* args, int64_t window, int64_t sinks);
int lwl_attention_window_forward(const lwl_attention_args* args, int64_t window, int64_t sinks, void* workspace,
                                 size_t workspace_bytes, void* stream);
size_t lwl_attention_window_backward_workspace_size(const lwl_attention_args* args, int64_t window, int64_t sinks);
int lwl_attention_window_backward(const lwl_attention_args* args, int64_t window, int64_t sinks, void* workspace,
                                  size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------- attention of a tree over a cache
 * The queries are the nodes of a tree of drafted tokens, whose keys and values are the last `queries` of their
 * sequence: node i's lie at key_lengths[b] - queries + i.  A node sees every key before the tree, its
 * ancestors' and its own.
 *
 * parents (device int32): parents[b * parents_stride + i] is the number of node i's parent, less than i; any other
 * number makes node i a root.  parents_stride 0: one tree for all sequences.  A sequence shorter than the tree
 * lacks the nodes at negative positions; a node that sees nothing gives zeros.
 *
 * A NaN in a node's key or value may reach nodes that do not see it.
 *
 * args as in lwl_attention_forward, with causal, bottom_right and causal_offset 0 and at most
 * LWL_ATTENTION_MAX_NODES queries.  lse may be NULL.  Forward only.
 */
#define LWL_ATTENTION_MAX_NODES 128
int lwl_attention_tree_check(const lwl_attention_args* args); /* host only */
size_t lwl_attention_tree_workspace_size(const lwl_attention_args* args);
int lwl_attention_tree_forward(const lwl_attention_args* args, const int32_t* parents, int64_t parents_stride,
                               void* workspace, size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------- log probabilities of tokens
 * Rows of `vocab` logits z, consecutive values of a row one after the other: row r of outer x inner lies at
 * logits + (r / inner) * outer_stride + (r % inner) * inner_stride (in elements; any strides).  With
 * lse = log sum_j exp(z_j) and p_j = exp(z_j - lse):
 *
 *   log_probs[r][i] = z_t - lse,  t = tokens[r][i], i < each
 *   entropy[r]      = -sum_j p_j log p_j
 *   top_log_probs[r][k], top_tokens[r][k], k < top: the largest log p_j in descending order and their j;
 *                     of equal logits the lowest j first
 *
 * all float32 and contiguous, tokens and top_tokens int64.  A negative token stands for none: its log probability
 * is 0 and has no part in the gradient; one past the vocabulary gives NaN and no gradient.  log_probs and tokens
 * are NULL exactly when each is 0, top_* exactly when top is 0; entropy may be NULL.  stats (float32 [rows][2]: the
 * largest logit and lse less that) is what the backward needs and may be NULL.
 *
 * Logits of minus infinity have probability 0.  A row of nothing else has log probabilities of minus infinity,
 * entropy 0, top_tokens 0 .. top - 1 and gradients of 0.  A NaN or plus infinity in a row makes its results NaN, its
 * top_tokens some tokens of the vocabulary.
 */
#define LWL_LOG_PROBS_MAX_EACH 64
#define LWL_LOG_PROBS_MAX_TOP 64
typedef struct lwl_log_probs_args {
  int32_t dtype, each, top, reserved; /* reserved: 0 */
  int64_t outer, inner, vocab;
  int64_t outer_stride, inner_stride;
  const void* logits;
  const int64_t* tokens;
  float *log_probs, *entropy, *top_log_probs; /* the backward reads entropy, where grad_entropy is given */
  int64_t* top_tokens;
  float* stats;
  /* backward only: the gradients of the forward's results, each may be NULL, and of the logits, contiguous */
  const float *grad_log_probs, *grad_entropy, *grad_top;
  void* grad_logits;
} lwl_log_probs_args;

int lwl_log_probs_check(const lwl_log_probs_args* args); /* host only; does not look at pointers */
int lwl_log_probs_forward(const lwl_log_probs_args* args, void* stream);
/* grad z_j = p_j (-G - grad_entropy (log p_j + entropy)) + sum of the gradients given for token j, G the sum of all
 * of them, in float32 and rounded once to dtype.  A token may be given more than once. */
int lwl_log_probs_backward(const lwl_log_probs_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LWL_TOKENS_H */
