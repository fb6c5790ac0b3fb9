/* moe_paged.h -- a paged key-value cache on a B200 (sm_100a) and the attention that reads it: the attention layer of
 * include/moe_stack.h for a batch of sequences, each with any number of cached tokens in pages of one shared pool, and
 * one or a few (drafted) new tokens each. C ABI, plain pointers and sizes, every call asynchronous on `stream` and on
 * the current device, allocating nothing and returning a cudaError_t as int (0 on success). No reference counterpart:
 * the reference decodes one sequence over one contiguous cache (qwen.cu:413-425, kernels.cuh:665-761).
 *
 * Every call takes its lists and lengths from device memory and launches the same grid whatever they hold, so a step
 * can be captured into a CUDA graph once and replayed as the sequences grow. What only the device can see (a page id
 * outside the pool, a list entry outside the table, too few free pages) is recorded in the workspace's error word and
 * the access is left out.
 */
#ifndef MOE_PAGED_H
#define MOE_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "moe_block.h"
#include "moe_stack.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Types of the cached values: bf16 bits, or 8-bit e4m3 (finite range +-448, NaN 0x7F and 0xFF) with an fp32 scale per
 * layer and kv head (value = stored * scale). */
enum { MOE_KV_BF16 = 0, MOE_KV_E4M3 = 1 };

/* A paged cache: caller-owned device memory and its geometry.
 *   k, v     [layers][num_pages][Hkv][page][D] values of kv_type; 16-byte aligned
 *   tables   int32 [max_seqs][max_pages]: the page ids of each sequence, position p in entry p / page; -1 behind the
 *            last page
 *   refs     int32 [num_pages]: how many sequences hold each page; 0 = free
 *   lens     int32 [max_seqs]: tokens of each sequence (the new tokens of a step included)
 *   k_scale, v_scale  fp32 [layers][Hkv], e4m3 only (NULL = 1); positive and finite
 * Supported: D 64, 128 or 256 for bf16, 128 or 256 for e4m3; page a multiple of 16 up to 1024; Hkv up to 64;
 * num_pages up to 2^20; max_seqs up to 65536; max_pages * page below 2^30. */
typedef struct moe_paged_cache {
  void* k;
  void* v;
  int32_t* tables;
  int32_t* refs;
  int32_t* lens;
  const float* k_scale;
  const float* v_scale;
  int32_t layers, num_pages, page, Hkv, D, kv_type, max_seqs, max_pages;
} moe_paged_cache;

/* Bits of the paged workspace's error word (moe_paged_workspace_error). MOE_ERR_TIMEOUT (include/moe_block.h) is set
 * too when a bounded wait of the attention kernel gave up; that call's output is then invalid. */
enum {
  MOE_ERR_PAGE_ID = 1 << 8,   /* a page id outside [0, num_pages): its keys read as zero, its rows are not written */
  MOE_ERR_SEQ_ID = 1 << 9,    /* a list entry outside [0, max_seqs) (-1 marks an unused slot where a call says so), a
                                 length the table cannot hold, the same sequence twice in one list, or a fork onto a
                                 sequence that holds pages: a page call then changes nothing */
  MOE_ERR_NO_PAGES = 1 << 10, /* moe_paged_resize: not enough free pages; nothing is changed */
  MOE_ERR_SHARED = 1 << 11    /* moe_paged_append: a new token falls into a page that another sequence holds too (grow
                                 with moe_paged_resize first); the row is not written */
};

/* 0 if the geometry is supported and every pointer is present and aligned, else cudaErrorInvalidValue. */
MOE_API int moe_paged_check(const moe_paged_cache* c);

/* Bytes of caller-owned workspace for the calls below with Hq query heads, lists of up to max_batch entries
 * (1 .. 4096) and up to max_new new tokens a sequence (1 .. 8 for moe_paged_attend; more for moe_paged_append only); 0
 * for unsupported sizes. One workspace per concurrently running call, on the cache's device. Zero it once before its
 * first call. Calls that share one (two captured graphs of the same stream, say) must not overlap. */
MOE_API size_t moe_paged_workspace_bytes(const moe_paged_cache* c, int Hq, int max_batch, int max_new);

/* Reads and clears the workspace's error word, synchronising the stream; a negative value is -cudaError. */
MOE_API int moe_paged_workspace_error(void* workspace, size_t workspace_bytes, moe_stream_t stream);

/* ---- pages -------------------------------------------------------------------------------------------------------
 * The page calls keep three rules. A free page has refs 0 and is in no table. A sequence of n tokens holds exactly
 * ceil(n / page) pages. After moe_paged_resize the partly filled last page of each listed sequence is held by it
 * alone, so that moe_paged_append may write into it. Which pages are taken depends on the lists and the state alone:
 * the lowest free ids, in list order. A call that finds a fault in its lists, or too few pages, changes nothing. */

/* Sets the length of each of the n listed sequences (distinct): shrinking releases the pages behind the new end (0
 * releases all of them), growing takes free pages, and a partly filled page at the end of what stays that other
 * sequences hold too is replaced by a copy of its filled rows, in every layer, in a page of its own (of k listed
 * sequences that end in one page, all its holders but the last in list order copy). That copy takes a free page, of a
 * sequence that shrinks too; releasing a whole sequence never does. Pages released by a call can be taken by the same
 * call. seqs, new_lens: device int32 [n]. n <= 4096 and at most the workspace's max_batch. */
MOE_API int moe_paged_resize(const moe_paged_cache* c, const int32_t* seqs, const int32_t* new_lens, int n,
                             void* workspace, size_t workspace_bytes, moe_stream_t stream);

/* Makes each dst sequence (distinct, empty, none of them a src) a copy of its src that shares all of its pages. No
 * page is copied: moe_paged_resize copies a shared last page when either side grows. */
MOE_API int moe_paged_fork(const moe_paged_cache* c, const int32_t* src, const int32_t* dst, int n, void* workspace,
                           size_t workspace_bytes, moe_stream_t stream);

/* Moves the live pages to the ids [0, number of live pages): the i-th free id below that bound receives the i-th live
 * page behind it, in every layer, and tables and refs follow. No list; a cache that is compact is left as it is. */
MOE_API int moe_paged_compact(const moe_paged_cache* c, void* workspace, size_t workspace_bytes, moe_stream_t stream);

/* Copies whole pages in every layer: page src[i] to page dst[i], i < n (device int32 [n], any n). The dst pages are
 * distinct and none of them is a src. Tables, refs and lens are not touched. Pairs with an id outside the pool are
 * left out and recorded. */
MOE_API int moe_paged_copy(const moe_paged_cache* c, const int32_t* src, const int32_t* dst, int n, void* workspace,
                           size_t workspace_bytes, moe_stream_t stream);

/* ---- attention ---------------------------------------------------------------------------------------------------
 * A step works on a batch of B slots; slot b is the sequence seqs[b] (device int32 [B], distinct), -1 marks an unused
 * slot. Each has Tq new tokens, the last Tq of its lens tokens: token t of slot b is row b * Tq + t, at position
 * lens - Tq + t. A row whose position is negative (a sequence shorter than Tq) stands for no token. */

/* The per-head norm and rotation of the new tokens and their write into layer `layer` of the cache. qkv bf16
 * [B Tq][(Hq + 2 Hkv) D]: q heads, k heads, v heads (the first GEMV's output in moe_attn_forward). Each q and k head x
 * becomes x rsqrt(mean(x^2) + eps) norm (q_norm, k_norm bf16 [D]; both NULL = no norm), then the pairs
 * (d, d + rope_dim / 2), d < rope_dim / 2, are rotated by the angle position * inv_freq[d] (fp64 [rope_dim / 2], for
 * this model theta^(-2 d / rope_dim); the angle is formed and reduced in fp64, so far positions keep their accuracy;
 * rope_dim 0 with inv_freq NULL = no rotation). q goes to q_out bf16 [B Tq][Hq D]; k and v go into the pages at the
 * tokens' positions, for e4m3 as x / scale rounded to nearest even and saturated. B <= 4096, B * Tq < 2^24, rope_dim
 * even and <= D; qkv, q_out and the norms 16-byte aligned. Rows of unused slots and of no token are left as they were. */
MOE_API int moe_paged_append(const moe_paged_cache* c, int layer, const int32_t* seqs, int B, int Tq,
                             const uint16_t* qkv, int Hq, const uint16_t* q_norm, const uint16_t* k_norm,
                             const double* inv_freq, int rope_dim, float eps, uint16_t* q_out, void* workspace,
                             size_t workspace_bytes, moe_stream_t stream);

/* Causal attention of the new tokens over the cached keys and values of layer `layer`, theirs included: query head h
 * reads kv head h / (Hq / Hkv), softmax(scale q . k) . v, out bf16 [B Tq][Hq D]. Scores, the softmax and all sums are
 * fp32. The weights enter their product with v as two bf16 parts (16 bits of each), over an e4m3 cache as f16 (11
 * bits, or 2^-36 of the row's largest weight where that is more); there the queries are f16 too, scaled by the power
 * of two that brings the largest of a head's to [1, 2): exact down to 2^-17, off by 2^-25 at most below. Sums stay
 * finite over 2^20 keys of the type's largest value. Rows of unused slots, of empty sequences and of no token are
 * zero. What lies in a page behind a sequence's end, and what a token may not see, has no influence, NaN and
 * infinities included. G = Hq / Hkv any whole number with Hq <= 128; Tq <= 8; B <= 4096; B Hkv ceil(G Tq / 64)
 * max_pages page at most 2^34 (the work is counted in 32 bits); q, out 16-byte aligned. The batch's work is shared out
 * over the GPU by keys, whatever the lengths, and the parts of a sequence joined in order: the same call gives the
 * same bits. */
MOE_API int moe_paged_attend(const moe_paged_cache* c, int layer, const int32_t* seqs, int B, int Tq,
                             const uint16_t* q, int Hq, float scale, uint16_t* out, void* workspace,
                             size_t workspace_bytes, moe_stream_t stream);

/* The attention branch of one layer for a batch over the paged cache: moe_attn_forward_rms (include/moe_stack.h) with
 * moe_paged_append and moe_paged_attend in place of its contiguous cache. hidden fp32 [B Tq][H], attn_out bf16
 * [B Tq][H]; w->D and w->Hkv are the cache's; w->rope_dim and w->eps are used, inv_freq replaces w->theta. The two
 * projections run four rows at a time (the weights are read once for every four rows of the batch).
 * moe_attn_paged_workspace_bytes covers the projections' activations and the paged workspace (which leads it, so
 * moe_paged_workspace_error applies). */
MOE_API size_t moe_attn_paged_workspace_bytes(const moe_attn_weights* w, const moe_paged_cache* c, int max_batch,
                                              int max_new);
MOE_API int moe_attn_paged_forward_rms(const moe_attn_weights* w, const uint16_t* rms1, const float* hidden,
                                       const moe_paged_cache* c, int layer, const int32_t* seqs, int B, int Tq,
                                       const double* inv_freq, uint16_t* attn_out, void* workspace,
                                       size_t workspace_bytes, moe_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* MOE_PAGED_H */
