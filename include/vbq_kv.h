/*
 * vbq_kv.h -- C ABI of the 8-bit paged KV cache, the attention over it, the moves of its
 * pages, and the log probabilities taken from the lm_head's output.
 *
 * The reference engine keeps fp32 keys and values per layer and attends to them on the host
 * (cpp/src/fast_model.cpp:690-804); these are the device steps around the matmuls of vbq.h
 * that such an engine needs to decode: store the new keys and values, attend, regroup the
 * sequences of a beam search, and read the distribution over the vocabulary.
 *
 * The cache is two caller-owned device buffers:
 *     codes   int8 [pages][layers][2][kv_heads][page][dim]     (2: keys, then values)
 *     scales  fp32 [pages][layers][2][kv_heads]
 * A stored value is scale * code, scales finite and not negative.  `page` tokens (16, 32, 64 or 128)
 * of one head share a scale; dim is 64, 128 or 256.  A page is one contiguous run over every layer, so moving a
 * page is one copy.  Codes must be 16-byte aligned, scales and every int32 and fp32 array 4-byte aligned.
 *
 * A batch of sequences is described by three device arrays:
 *     tables  int32 [seqs][max_pages]  the page of each run of `page` tokens (-1: none)
 *     lens    int32 [seqs]             tokens of each sequence, the new ones included
 *     q_start int32 [seqs + 1]         rows q_start[s] .. q_start[s + 1] - 1 of the row
 *                                      tensors are the last tokens of sequence s
 * A page that several sequences hold is whole (vbq_kv_fork copies a part-filled one), so an
 * append never writes a shared page.  Entries are checked where they are read: a page number
 * outside 0 .. pages - 1 stands for no tokens.
 *
 * As in vbq.h: device pointers, a stream, no allocation, no synchronisation, status codes
 * with vbq_last_error().
 */
#ifndef VBQ_KV_H
#define VBQ_KV_H

#include "vbq.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Quantise the new tokens' keys and values of one layer into their pages.  k and v are
 * [rows, kv_heads * dim] of `dtype` (VBQ_DTYPE_F32 or VBQ_DTYPE_BF16), rows k_stride and
 * v_stride elements apart (so columns of a packed Q | K | V matmul output can be passed as
 * they are); both 16-byte aligned with row strides of whole 16 bytes.  Per page, head and
 * K / V, with a = the largest finite |x| among its new values:
 *     s1 = max(s0, a / 127), s0 the page's scale where it held earlier tokens of the
 *          sequence, else 0
 *     old codes become rint(code * (s0 / s1)) when s1 > s0
 *     new codes are rint(x / s1) clamped to +-127
 * in fp32 with one rounding an operation, ties to even.  Infinities take the code +-127, NaN
 * takes 0, and neither enters the scale; where s1 is 0 every new code is.  The pages must be in the
 * tables already (vbq_kv_reserve); repeating a call leaves the cache as it is.
 */
int vbq_kv_append(const void* k, int64_t k_stride, const void* v, int64_t v_stride, int32_t dtype,
                  int64_t rows, void* codes, float* scales, int64_t pages, int32_t layers, int32_t layer,
                  int32_t kv_heads, int32_t page, int32_t dim, const int32_t* tables, int32_t max_pages,
                  const int32_t* lens, const int32_t* q_start, int32_t seqs, void* stream);

/*
 * The stored keys and values of the batch's rows: k_out, v_out [rows, kv_heads * dim] of
 * `dtype`, scale * code rounded once.  A token without a page reads as 0.
 */
int vbq_kv_read(const void* codes, const float* scales, int64_t pages, int32_t layers, int32_t layer,
                int32_t kv_heads, int32_t page, int32_t dim, const int32_t* tables, int32_t max_pages,
                const int32_t* lens, const int32_t* q_start, int32_t seqs, int64_t rows, void* k_out,
                void* v_out, int32_t dtype, void* stream);

/* What of an attention workspace has to be zero before its first use: the bytes at its beginning. */
#define VBQ_KV_ATTENTION_ZERO_BYTES 16384

/*
 * Workspace bytes vbq_kv_attention needs on the current device (for any batch); they go by dim.  The first
 * VBQ_KV_ATTENTION_ZERO_BYTES are zeroed before the workspace's first use; see vbq_kv_attention.
 */
int vbq_kv_attention_workspace_bytes(int32_t heads, int32_t kv_heads, int32_t dim, int32_t dtype,
                                     size_t* bytes);

/*
 * Causal attention of the batch's rows over the cache of one layer (the rows' own keys and
 * values appended before):
 *     out[row, h] = sum_j p_j v_j,  p = softmax_j(scale * q[row, h] . k_j)
 * for row i of the n new tokens of a sequence of length L over the tokens
 * L - n + i - window < j <= L - n + i (window 0: from the first).  Query head h reads KV head
 * h / (heads / kv_heads).  q and out are [rows, heads * dim] of `dtype`, rows q_stride and
 * out_stride elements apart, 16-byte aligned with row strides of whole 16 bytes.  lse (fp32
 * [rows, heads], may be NULL) receives the natural log of the row's sum of exponentials.  A
 * row that sees no token, or that no sequence has (before q_start[0], from q_start[seqs] on), gets
 * zeros and -inf.
 *
 * Codes are multiplied exactly and sums are fp32.  Queries enter to 2^-22 of their row's largest
 * value (bf16 prompts of dim 64 or 128: 11 bits of each, so all that bf16 has); softmax weights
 * enter with 22 bits for fp32 and 11 (fp16) for bf16 activations.  Results are
 * deterministic.  max_new: the most new tokens any sequence has, or 0 when unknown; it
 * selects the kernel, never the result's coverage.  workspace: vbq_kv_attention_workspace_bytes() of
 * 16-byte aligned device memory, its first VBQ_KV_ATTENTION_ZERO_BYTES zeroed before its first use; a call
 * leaves what it needs to be zero at zero, and any sizes that fit may follow one another in it.  Calls that
 * may run at the same time must not share it.
 */
int vbq_kv_attention(const void* q, int64_t q_stride, void* out, int64_t out_stride, float* lse,
                     int32_t dtype, int64_t rows, int32_t heads, const void* codes, const float* scales,
                     int64_t pages, int32_t layers, int32_t layer, int32_t kv_heads, int32_t page,
                     int32_t dim, const int32_t* tables, int32_t max_pages, const int32_t* lens,
                     const int32_t* q_start, int32_t seqs, float scale, int32_t window, int32_t max_new,
                     void* workspace, size_t workspace_bytes, void* stream);

/*
 * Workspace bytes the page moves below need for a pool of `pages` pages and `rows` sequences (of
 * vbq_kv_fork the larger of rows and new_rows).  The workspace is 16-byte aligned device memory, zero-filled
 * before its first use and again before it serves a pool of another number of pages (what a fork needs to
 * be zero lies by `pages`); every call leaves that at zero.  Calls that may run at the same time must not
 * share it.
 */
int vbq_kv_pages_workspace_bytes(int64_t pages, int32_t rows, size_t* bytes);

/*
 * Room for new tokens: row s is given pages for lens[s] + new_tokens[s] tokens, the lowest
 * free pages (refs 0) first, rows and positions in order, and lens_out = lens + new_tokens.
 * refs int32 [pages] counts the rows that hold a page.  *missing (device int32) receives how
 * many pages there were not (their entries stay -1).  Each output may be its input.
 */
int vbq_kv_reserve(const int32_t* refs, const int32_t* tables, const int32_t* lens,
                   const int32_t* new_tokens, int64_t pages, int32_t page, int32_t rows,
                   int32_t max_pages, int32_t* refs_out, int32_t* tables_out, int32_t* lens_out,
                   int32_t* missing, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Regroup sequences: new row r continues old row parents[r] (outside 0 .. rows - 1: an empty
 * row).  Whole pages are shared; a part-filled last page stays with the lowest row that
 * continues it and is copied, codes and scales of every layer, to the lowest free page for
 * each later one; pages of rows that nobody continues are let go.  refs_out may be refs;
 * tables_out [new_rows][max_pages] and lens_out must not overlap their inputs.  A row whose copy finds no
 * free page gets -1 there and counts in *missing.  page_bytes = layers * 2 * kv_heads * page * dim (the
 * codes of one page, a multiple of 16), page_scales = layers * 2 * kv_heads.
 */
int vbq_kv_fork(void* codes, float* scales, int64_t pages, int64_t page_bytes, int64_t page_scales,
                int32_t page, const int32_t* refs, const int32_t* tables, const int32_t* lens, int32_t rows,
                int32_t max_pages, const int32_t* parents, int32_t new_rows, int32_t* refs_out,
                int32_t* tables_out, int32_t* lens_out, int32_t* missing, void* workspace,
                size_t workspace_bytes, void* stream);

/*
 * Make the pool dense: with *live pages in use, the pages in use at live and above move, in
 * order, to the free pages below it (lowest first), codes and scales of every layer.
 * refs_out and tables_out hold the new numbers (entries past a row's pages become -1); each
 * may be its input.
 */
int vbq_kv_compact(void* codes, float* scales, int64_t pages, int64_t page_bytes, int64_t page_scales,
                   int32_t page, const int32_t* refs, const int32_t* tables, const int32_t* lens,
                   int32_t rows, int32_t max_pages, int32_t* refs_out, int32_t* tables_out, int32_t* live,
                   void* workspace, size_t workspace_bytes, void* stream);

/*
 * Workspace bytes vbq_token_logprobs needs for these sizes on the current device.  The workspace is 16-byte
 * aligned device memory, zero-filled before its first use; any sizes that fit may follow one another in it.
 * Calls that may run at the same time must not share it.
 */
int vbq_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int32_t top, size_t* bytes);

/*
 * Log probabilities from logits [rows, vocab] (fp32 or bf16, rows `stride` elements apart,
 * element-aligned): with lse = log sum_i e^x_i of a row,
 *     logprob[r]  = x[tokens[r]] - lse           (0 where tokens[r] is outside 0 .. vocab - 1)
 *     entropy[r]  = -sum_i p_i log p_i,  p_i = e^(x_i - lse)
 *     top_logprob / top_token [rows, top]: the `top` (0 .. 32, at most vocab) largest, in
 *     descending order, equal ones by the lower token
 * one pass over the logits, sums in fp32.  -inf logits have probability 0; a row of nothing
 * but -inf has logprob and top_logprob -inf and entropy 0; a row with NaN or +inf has NaN
 * logprob and entropy.  tokens may be NULL (then logprob is not written), entropy may be
 * NULL.
 */
int vbq_token_logprobs(const void* logits, int64_t stride, int32_t dtype, int64_t rows, int64_t vocab,
                       const int32_t* tokens, int32_t top, float* logprob, float* entropy,
                       float* top_logprob, int32_t* top_token, void* workspace, size_t workspace_bytes,
                       void* stream);

#ifdef __cplusplus
}
#endif

#endif /* VBQ_KV_H */
