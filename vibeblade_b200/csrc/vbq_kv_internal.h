// vbq_kv_internal.h -- launchers of the KV cache and log-probability kernels, shared between
// the kernel files and the C-ABI layer.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace vbq {

// One layer of the cache: codes int8 [pages][layers][2][heads][page][dim], scales fp32
// [pages][layers][2][heads].
struct KvCache {
  int8_t* codes;
  float* scales;
  int64_t pages;
  int layers, layer, heads, page, dim;
  int page_log2;
};

// The sequences of a call: page tables, lengths (new tokens included), row ranges.
struct KvBatch {
  const int32_t* tables;
  const int32_t* lens;
  const int32_t* q_start;
  int seqs, max_pages;
};

cudaError_t launch_kv_append(const void* k, int64_t k_stride, const void* v, int64_t v_stride, bool bf16,
                             int64_t rows, const KvCache& c, const KvBatch& b, cudaStream_t st);
cudaError_t launch_kv_read(const KvCache& c, const KvBatch& b, int64_t rows, void* k_out, void* v_out,
                           bool bf16, cudaStream_t st);

struct KvAttention {
  const void* q;
  void* out;
  float* lse;  // may be null
  int64_t q_stride, out_stride;  // elements
  int64_t rows;
  int group;     // query heads per KV head
  float scale;   // log2(e) times the caller's
  int window;    // 0: none
  // a launch takes the sequences whose rows (new tokens times group) are in (rows_above, rows_upto]
  int64_t rows_above, rows_upto;
};
constexpr int kKvMaxSms = 148;
constexpr int kKvMaxResident = 4;  // CTAs an SM of the kernel for few rows
constexpr int kKvCounterBytes = 4 * kKvMaxResident * kKvMaxSms;  // the attention workspace's zeroed head
constexpr int kKvHeadBytes = kKvCounterBytes + 4 * kKvMaxSms;  // with the tile kernel's counters
size_t kv_attn_tile_parts(int dim);  // where in the workspace the tile kernel's parts begin
// Split over the cache's tokens (vbq_kv_attn.cu): any type, any number of new tokens.
size_t kv_attn_workspace(int dim);  // one for both types of activations
cudaError_t launch_kv_attn(const KvAttention& a, const KvCache& c, const KvBatch& b, bool bf16, int max_new,
                           void* workspace, cudaStream_t st);

// Tiles of 256 rows on tcgen05 (vbq_kv_prefill.cu): bf16, dim 64 or 128.
bool kv_prefill_takes(int dim, bool bf16);
size_t kv_prefill_parts_bytes(int dim);
cudaError_t launch_kv_prefill(const KvAttention& a, const KvCache& c, const KvBatch& b, void* workspace, cudaStream_t st);
cudaError_t kv_prefill_status(unsigned* out, bool clear);

// Page moves (vbq_kv_pages.cu).
size_t kv_pages_workspace(int64_t pages, int rows);
struct KvPool {
  uint8_t* codes;
  float* scales;
  int64_t pages, page_bytes, page_scales;
  int page;
};
cudaError_t launch_kv_reserve(const int32_t* refs, const int32_t* tables, const int32_t* lens,
                              const int32_t* add, int64_t pages, int page, int rows, int max_pages,
                              int32_t* refs_out, int32_t* tables_out, int32_t* lens_out, int32_t* missing,
                              void* workspace, cudaStream_t st);
cudaError_t launch_kv_fork(const KvPool& p, const int32_t* refs, const int32_t* tables, const int32_t* lens,
                           int rows, int max_pages, const int32_t* parents, int new_rows, int32_t* refs_out,
                           int32_t* tables_out, int32_t* lens_out, int32_t* missing, void* workspace,
                           cudaStream_t st);
cudaError_t launch_kv_compact(const KvPool& p, const int32_t* refs, const int32_t* tables, const int32_t* lens,
                              int rows, int max_pages, int32_t* refs_out, int32_t* tables_out, int32_t* live,
                              void* workspace, cudaStream_t st);

// Log probabilities (vbq_logprobs.cu).
constexpr int kMaxTop = 32;
size_t logprobs_workspace(int64_t rows, int64_t vocab, int top);
cudaError_t launch_logprobs(const void* logits, int64_t stride, bool bf16, int64_t rows, int64_t vocab,
                            const int32_t* tokens, int top, float* logprob, float* entropy, float* top_logprob,
                            int32_t* top_token, void* workspace, cudaStream_t st);

}  // namespace vbq
