/* ss_hip_serving.h - attention and sampling for serving: long conversations,
 * several answers to one prompt. Part of ss_hip.h.
 *
 * No counterpart in the reference, which serves one sequence. These three
 * allocate nothing and wait for nothing: results stay on the device, and a
 * call may be captured in a HIP graph. Scratch is the caller's: ws_dev of at
 * least the bytes that the _workspace function gives for the same shape
 * (0: NULL will do), 16-byte aligned, its contents of no account before and
 * after. Calls that may run at the same time (two streams, two captured
 * graphs) need workspaces of their own; calls in one stream can share one.
 * Queries, outputs and caches are 16-byte aligned; an output overlaps no
 * input; a cache holds at most 2^30 positions, a call at most 2^24 tokens times
 * heads or 2^22 sequences times heads. The workspace functions return 0 for a
 * shape that the call refuses. */
#ifndef SS_HIP_SERVING_H
#define SS_HIP_SERVING_H

#include "ss_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Attention of the newest n_tokens of a sequence, at positions pos0 ..
 * pos0 + n_tokens - 1, each over a sliding window and the sequence's first
 * positions: token i sees j <= i with i - j < window or j < n_sinks. Cache,
 * q [n_tokens][n_heads * head_dim], out and softmax as ss_hip_attention_rows
 * (n_tokens 1: a decode step), over either cache type (scales as
 * ss_hip_kv_append writes them); the cache already holds the tokens' own K
 * and V. softcap > 0 (a normal float) turns a score s into
 * softcap * tanh(s / softcap) first (Gemma 2); 0: none. Reads only positions
 * that some token sees. A workspace serves every pos0. */
size_t ss_hip_attention_window_workspace(ss_hip_ctx_t *ctx, int32_t n_heads, int32_t n_kv_heads,
                                         int32_t head_dim, int32_t n_tokens, int32_t window,
                                         int32_t n_sinks);
int32_t ss_hip_attention_window(ss_hip_ctx_t *ctx, float *out_dev, const float *q_dev,
                                const void *k_cache, const void *v_cache, const float *k_scale,
                                const float *v_scale, int32_t n_heads, int32_t n_kv_heads,
                                int32_t head_dim, int32_t max_seq, int32_t pos0, int32_t n_tokens,
                                int32_t window, int32_t n_sinks, float softcap, int32_t kv_type,
                                void *ws_dev, size_t ws_bytes, void *stream);

/* One decode step's attention of n_seqs sequences that continue the same
 * prompt. Sequence b (q[b][n_heads * head_dim], out alike) sees the first
 * prefix_len positions of the prefix cache [n_kv_heads][prefix_max][head_dim]
 * and the first own_len_dev[b] positions of its own cache, block b of
 * [n_seqs][n_kv_heads][own_max][head_dim] (so ss_hip_kv_append with max_seq
 * own_max appends to a block; its RoPE position is prefix_len + the index).
 * int8 caches have scales [prefix_max] and [n_seqs][own_max]. The prefix is
 * read once for all sequences. own_len_dev is read on the device when the
 * kernels run, so a captured call follows it; a length below 0 counts as 0, one
 * above own_max as own_max. prefix_len 0 (the prefix pointers may be NULL):
 * sequences of their own only. A sequence that sees nothing gets zeros. */
size_t ss_hip_attention_shared_workspace(ss_hip_ctx_t *ctx, int32_t n_heads, int32_t n_kv_heads,
                                         int32_t head_dim, int32_t n_seqs, int32_t prefix_len,
                                         int32_t own_max);
int32_t ss_hip_attention_shared(ss_hip_ctx_t *ctx, float *out_dev, const float *q_dev,
                                const void *k_prefix, const void *v_prefix,
                                const float *k_prefix_scale, const float *v_prefix_scale,
                                int32_t prefix_max, int32_t prefix_len, const void *k_own,
                                const void *v_own, const float *k_own_scale,
                                const float *v_own_scale, int32_t own_max,
                                const int32_t *own_len_dev, int32_t n_seqs, int32_t n_heads,
                                int32_t n_kv_heads, int32_t head_dim, float softcap,
                                int32_t kv_type, void *ws_dev, size_t ws_bytes, void *stream);

/* The next token of each of n_rows rows of n logits (row r at logits_dev +
 * r * ld, ld >= n, n < 524288) into out_dev[r], from the random number
 * u_dev[r] in [0, 1). Weights e^((x - max) / temperature); what stays are
 * logits of at least the top_k-th largest (0 or >= n: all), of at least the
 * value at which the weights, from the largest down, reach top_p of the sum
 * of all (<= 0 or >= 1: all), and of weight at least min_p (<= 0: all; at most
 * 1); equal logits stay or go together. The token is the first whose running
 * sum of the weights that stay, by index, exceeds u times their sum. top_k and
 * top_p are those of ss_hip_sample_logits, whose sums round to 32 bits where
 * these do not; a weight below 2^-45 of the largest counts as none.
 * temperature <= 0: the first maximum. NaN logits count as
 * -inf; a row without any logit above -inf gives -1. u outside [0, 1) counts
 * as the nearest number inside. */
size_t ss_hip_sample_rows_workspace(ss_hip_ctx_t *ctx, int32_t n_rows, int32_t n);
int32_t ss_hip_sample_rows(ss_hip_ctx_t *ctx, int32_t *out_dev, const float *logits_dev, int32_t n,
                           int32_t n_rows, int64_t ld, float temperature, int32_t top_k,
                           float top_p, float min_p, const float *u_dev, void *ws_dev,
                           size_t ws_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif
