/* moe_spec.h -- from logits to tokens on a B200 (sm_100a), beside the greedy LM head of include/moe_stack.h: the logits
 * of several tokens of one step, their probabilities, and the verification of drafted tokens against them. C ABI, plain
 * pointers and sizes, every call asynchronous on `stream` and on the current device, allocating nothing and returning
 * a cudaError_t as int (0 on success). No reference counterpart: the reference picks the largest logit of one token
 * (qwen.cu:451-456).
 */
#ifndef MOE_SPEC_H
#define MOE_SPEC_H

#include <stddef.h>
#include <stdint.h>

#include "moe_block.h"

#ifdef __cplusplus
extern "C" {
#endif

/* logits fp32 [T][V] = normed bf16 [T][H] . W^T (bf16 [V][H]) for up to 4 tokens, the weights read once; H % 8 == 0,
 * H <= 8192; normed and W 16-byte aligned. */
MOE_API int moe_lm_head_logits(const uint16_t* normed, const uint16_t* lm_head, int V, int H, int T, float* logits,
                               moe_stream_t stream);

/* probs[r][v] = exp((x_v - m) / t_r) / sum_w exp((x_w - m) / t_r), m the row's largest logit, for R rows of V fp32
 * logits; rows lie ld_logits and ld_probs floats apart (at least V; what lies between rows is left alone). temperature
 * fp32 [R] (NULL = 1): a row with t_r = 0 (or negative or NaN) puts everything on its largest logit, the lowest index
 * of a tie, and an infinite one shares equally. NaN logits and -infinity get probability zero (a NaN never wins, as in
 * moe_lm_head_argmax); +infinity takes all (shared by several); a row with no logit above -infinity is all zeros. probs
 * may be logits itself (with the same ld), but not overlap it otherwise. 1 <= V < 2^24, R >= 0. All in fp32: a probability's
 * relative error stays below 2^-20 + 2^-21 (1 + (m - x_v) / t_r). */
MOE_API int moe_softmax_rows(const float* logits, int64_t ld_logits, int R, int V, const float* temperature,
                             float* probs, int64_t ld_probs, moe_stream_t stream);

/* Bytes of caller-owned workspace for moe_spec_verify of up to max_B sequences over V tokens; 0 for unsupported sizes
 * (1 <= max_B <= 65535, 1 <= V < 2^24). Zero it once before its first call; calls that share one must not overlap. */
MOE_API size_t moe_spec_workspace_bytes(int max_B, int V);

/* Verification of drafted tokens by rejection sampling, from given random numbers. Sequence b drafted n_b <= K tokens
 * x_i = drafted[b][i] (n_drafted int32 [B], NULL = K each; values outside [0, K] are taken as the nearer end) from the
 * draft's probabilities q_i = draft[b][i][:] (rows ld_draft floats apart, sequences K ld_draft; NULL: drafts that
 * were not drawn, q_i = 1 at x_i); p_i = target[b][i][:], i <= n_b, are the target's (rows ld_target floats apart,
 * sequences (K + 1) ld_target). u fp32 [B][K + 1] in [0, 1).
 *   Drafts are accepted while u[b][i] q_i(x_i) < p_i(x_i). a = the number accepted.
 *   Then one token is drawn by w = max(p_a - q_a, 0) if a < n_b, and by w = p_a after the last acceptance: the first v
 *   with sum_{j <= v} w_j > u[b][K] sum_j w_j. Where w is zero everywhere, w = p_a.
 * tokens int32 [B][K + 1] = the a accepted tokens, the drawn one, then -1; accepted int32 [B] = a. Products and sums
 * are in fp64. Entries of p and q that are NaN, negative or infinite count as zero; a draft outside [0, V) is rejected;
 * if no entry of p_a is positive, the drawn token is -1. K up to 64, B <= max_B of the workspace. K = 0 (drafted NULL)
 * draws one token a sequence from its probabilities. */
MOE_API int moe_spec_verify(const float* target, int64_t ld_target, const float* draft, int64_t ld_draft,
                            const int32_t* drafted, const int32_t* n_drafted, const float* u, int B, int K, int V,
                            int32_t* tokens, int32_t* accepted, void* workspace, size_t workspace_bytes,
                            moe_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* MOE_SPEC_H */
