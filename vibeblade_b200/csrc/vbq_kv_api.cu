// vbq_kv_api.cu -- the extern "C" boundary declared in include/vbq_kv.h.
#include <cmath>

#include "vbq_internal.h"
#include "vbq_kv.h"
#include "vbq_kv_internal.h"

namespace {

using vbq::api_status;

static_assert(vbq::kKvHeadBytes <= VBQ_KV_ATTENTION_ZERO_BYTES, "the counters lie in what the caller zeroes");

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// int32 and fp32 arrays; those that may be NULL are aligned then
template <typename... P> bool words(const P*... p) { return (aligned(p, 4) && ...); }
int bad_words(const char* who) { return api_status(VBQ_ERR_ALIGN, "%s: the int32 and fp32 arrays must be 4-byte aligned", who); }

int ok() { return api_status(VBQ_OK, nullptr); }
int launched(const char* who, cudaError_t e) {
  return e == cudaSuccess ? ok() : api_status(VBQ_ERR_CUDA, "%s launch: %s", who, cudaGetErrorString(e));
}

int bad_dtype(const char* who, int32_t dtype) {
  return api_status(VBQ_ERR_SHAPE, "%s: dtype must be VBQ_DTYPE_F32 or VBQ_DTYPE_BF16, got %d", who, dtype);
}
bool dtype_ok(int32_t dtype) { return dtype == VBQ_DTYPE_F32 || dtype == VBQ_DTYPE_BF16; }
bool page_ok(int32_t page) { return page == 16 || page == 32 || page == 64 || page == 128; }
bool dim_ok(int32_t dim) { return dim == 64 || dim == 128 || dim == 256; }

// Sizes of a cache and a batch (pointers are checked once there is something to do).
int sizes(const char* who, int64_t rows, int64_t pages, int32_t layers, int32_t layer, int32_t kv_heads,
          int32_t page, int32_t dim, int32_t max_pages, int32_t seqs) {
  if (rows < 0 || rows > INT32_MAX || seqs < 0)
    return api_status(VBQ_ERR_SHAPE, "%s: rows and seqs must be in 0..2^31-1", who);
  if (pages < 1 || pages > INT32_MAX || layers < 1 || layer < 0 || layer >= layers || kv_heads < 1 || kv_heads > 65535)
    return api_status(VBQ_ERR_SHAPE, "%s: need pages >= 1, 0 <= layer < layers, 1 <= kv_heads <= 65535", who);
  if (!page_ok(page)) return api_status(VBQ_ERR_SHAPE, "%s: page must be 16, 32, 64 or 128 tokens, got %d", who, page);
  if (!dim_ok(dim)) return api_status(VBQ_ERR_SHAPE, "%s: dim must be 64, 128 or 256, got %d", who, dim);
  if (max_pages < 1 || (int64_t)max_pages * page > INT32_MAX)
    return api_status(VBQ_ERR_SHAPE, "%s: max_pages must be at least 1 and max_pages * page below 2^31", who);
  return VBQ_OK;
}
int pointers(const char* who, const void* codes, const float* scales, const int32_t* tables,
             const int32_t* lens, const int32_t* q_start) {
  if (!codes || !scales || !tables || !lens || !q_start) return api_status(VBQ_ERR_NULL, "%s: NULL pointer", who);
  if (!aligned(codes, 16) || !aligned(scales, 4) || !aligned(tables, 4) || !aligned(lens, 4) || !aligned(q_start, 4))
    return api_status(VBQ_ERR_ALIGN, "%s: codes must be 16-byte aligned, scales and the int32 arrays 4-byte", who);
  return VBQ_OK;
}
vbq::KvCache cache(const void* codes, const float* scales, int64_t pages, int32_t layers, int32_t layer,
                   int32_t kv_heads, int32_t page, int32_t dim) {
  vbq::KvCache c;
  c.codes = static_cast<int8_t*>(const_cast<void*>(codes));
  c.scales = const_cast<float*>(scales);
  c.pages = pages;
  c.layers = layers, c.layer = layer, c.heads = kv_heads, c.page = page, c.dim = dim;
  c.page_log2 = page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7;
  return c;
}
// a row tensor: 16-byte aligned, rows of whole 16 bytes, at least as far apart as they are long
int row_tensor(const char* who, const char* name, const void* p, int64_t stride, int64_t width, int32_t dtype) {
  const int64_t size = dtype == VBQ_DTYPE_F32 ? 4 : 2;
  if (!p) return api_status(VBQ_ERR_NULL, "%s: NULL pointer (%s)", who, name);
  if (stride < width) return api_status(VBQ_ERR_SHAPE, "%s: %s's row stride is less than its width", who, name);
  if (!aligned(p, 16) || stride * size % 16 != 0)
    return api_status(VBQ_ERR_ALIGN, "%s: %s must be 16-byte aligned with a row stride of whole 16 bytes", who, name);
  return VBQ_OK;
}
int workspace_ok(const char* who, const void* ws, size_t have, size_t need) {
  if (need == 0) return VBQ_OK;
  if (!ws || have < need)
    return api_status(VBQ_ERR_WORKSPACE, "%s: workspace needs %zu bytes, got %zu", who, need, ws ? have : (size_t)0);
  if (!aligned(ws, 16)) return api_status(VBQ_ERR_ALIGN, "%s: workspace must be 16-byte aligned", who);
  return VBQ_OK;
}

// Page moves: sizes of the pool and the tables.
int pool_sizes(const char* who, int64_t pages, int32_t page, int32_t rows, int32_t max_pages) {
  if (pages < 1 || pages > INT32_MAX / 2)
    return api_status(VBQ_ERR_SHAPE, "%s: pages must be in 1..2^30-1", who);
  if (!page_ok(page)) return api_status(VBQ_ERR_SHAPE, "%s: page must be 16, 32, 64 or 128 tokens, got %d", who, page);
  if (rows < 0 || max_pages < 1 || (int64_t)max_pages * page > INT32_MAX || (int64_t)rows * max_pages > INT32_MAX)
    return api_status(VBQ_ERR_SHAPE, "%s: need rows >= 0, max_pages >= 1, max_pages * page and rows * max_pages below 2^31", who);
  return VBQ_OK;
}
int pool_data(const char* who, const void* codes, const float* scales, int64_t page_bytes, int64_t page_scales) {
  if (!codes || !scales) return api_status(VBQ_ERR_NULL, "%s: NULL pointer", who);
  if (page_bytes < 16 || page_bytes % 16 != 0 || page_scales < 1)
    return api_status(VBQ_ERR_SHAPE, "%s: page_bytes must be a multiple of 16 and page_scales positive", who);
  if (!aligned(codes, 16) || !aligned(scales, 4))
    return api_status(VBQ_ERR_ALIGN, "%s: codes must be 16-byte aligned, scales 4-byte", who);
  return VBQ_OK;
}

}  // namespace

extern "C" {

int vbq_kv_append(const void* k, int64_t k_stride, const void* v, int64_t v_stride, int32_t dtype,
                  int64_t rows, void* codes, float* scales, int64_t pages, int32_t layers, int32_t layer,
                  int32_t kv_heads, int32_t page, int32_t dim, const int32_t* tables, int32_t max_pages,
                  const int32_t* lens, const int32_t* q_start, int32_t seqs, void* stream) {
  const char* who = "vbq_kv_append";
  if (!dtype_ok(dtype)) return bad_dtype(who, dtype);
  if (int rc = sizes(who, rows, pages, layers, layer, kv_heads, page, dim, max_pages, seqs)) return rc;
  if (rows == 0 || seqs == 0) return ok();
  if (int rc = pointers(who, codes, scales, tables, lens, q_start)) return rc;
  const int64_t width = (int64_t)kv_heads * dim;
  if (int rc = row_tensor(who, "k", k, k_stride, width, dtype)) return rc;
  if (int rc = row_tensor(who, "v", v, v_stride, width, dtype)) return rc;
  return launched(who, vbq::launch_kv_append(k, k_stride, v, v_stride, dtype == VBQ_DTYPE_BF16, rows,
                                             cache(codes, scales, pages, layers, layer, kv_heads, page, dim),
                                             vbq::KvBatch{tables, lens, q_start, seqs, max_pages},
                                             static_cast<cudaStream_t>(stream)));
}

int vbq_kv_read(const void* codes, const float* scales, int64_t pages, int32_t layers, int32_t layer,
                int32_t kv_heads, int32_t page, int32_t dim, const int32_t* tables, int32_t max_pages,
                const int32_t* lens, const int32_t* q_start, int32_t seqs, int64_t rows, void* k_out,
                void* v_out, int32_t dtype, void* stream) {
  const char* who = "vbq_kv_read";
  if (!dtype_ok(dtype)) return bad_dtype(who, dtype);
  if (int rc = sizes(who, rows, pages, layers, layer, kv_heads, page, dim, max_pages, seqs)) return rc;
  if (rows == 0) return ok();
  if (seqs == 0) return api_status(VBQ_ERR_SHAPE, "%s: rows without sequences", who);
  if (int rc = pointers(who, codes, scales, tables, lens, q_start)) return rc;
  const int64_t width = (int64_t)kv_heads * dim;
  if (int rc = row_tensor(who, "k_out", k_out, width, width, dtype)) return rc;
  if (int rc = row_tensor(who, "v_out", v_out, width, width, dtype)) return rc;
  return launched(who, vbq::launch_kv_read(cache(codes, scales, pages, layers, layer, kv_heads, page, dim),
                                           vbq::KvBatch{tables, lens, q_start, seqs, max_pages}, rows, k_out, v_out,
                                           dtype == VBQ_DTYPE_BF16, static_cast<cudaStream_t>(stream)));
}

int vbq_kv_attention_workspace_bytes(int32_t heads, int32_t kv_heads, int32_t dim, int32_t dtype,
                                     size_t* bytes) {
  const char* who = "vbq_kv_attention_workspace_bytes";
  if (!bytes) return api_status(VBQ_ERR_NULL, "%s: bytes is NULL", who);
  if (!dtype_ok(dtype)) return bad_dtype(who, dtype);
  if (!dim_ok(dim)) return api_status(VBQ_ERR_SHAPE, "%s: dim must be 64, 128 or 256, got %d", who, dim);
  if (kv_heads < 1 || heads < 1 || heads % kv_heads != 0)
    return api_status(VBQ_ERR_SHAPE, "%s: heads must be a multiple of kv_heads", who);
  *bytes = vbq::kv_attn_workspace(dim);
  return ok();
}

int vbq_kv_attention(const void* q, int64_t q_stride, void* out, int64_t out_stride, float* lse,
                     int32_t dtype, int64_t rows, int32_t heads, const void* codes, const float* scales,
                     int64_t pages, int32_t layers, int32_t layer, int32_t kv_heads, int32_t page,
                     int32_t dim, const int32_t* tables, int32_t max_pages, const int32_t* lens,
                     const int32_t* q_start, int32_t seqs, float scale, int32_t window, int32_t max_new,
                     void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "vbq_kv_attention";
  if (!dtype_ok(dtype)) return bad_dtype(who, dtype);
  if (int rc = sizes(who, rows, pages, layers, layer, kv_heads, page, dim, max_pages, seqs)) return rc;
  if (heads < 1 || heads % kv_heads != 0)
    return api_status(VBQ_ERR_SHAPE, "%s: heads (%d) must be a multiple of kv_heads (%d)", who, heads, kv_heads);
  if (!std::isfinite(scale)) return api_status(VBQ_ERR_SHAPE, "%s: scale must be finite", who);
  if (window < 0 || max_new < 0) return api_status(VBQ_ERR_SHAPE, "%s: window and max_new must not be negative", who);
  if (rows * heads > INT32_MAX) return api_status(VBQ_ERR_SHAPE, "%s: rows * heads above 2^31", who);
  if (rows == 0) return ok();
  if (seqs == 0) return api_status(VBQ_ERR_SHAPE, "%s: rows without sequences", who);
  if (int rc = pointers(who, codes, scales, tables, lens, q_start)) return rc;
  const int64_t width = (int64_t)heads * dim;
  if (int rc = row_tensor(who, "q", q, q_stride, width, dtype)) return rc;
  if (int rc = row_tensor(who, "out", out, out_stride, width, dtype)) return rc;
  if (lse && !aligned(lse, 4)) return api_status(VBQ_ERR_ALIGN, "%s: lse must be 4-byte aligned", who);
  if (int rc = workspace_ok(who, workspace, workspace_bytes, vbq::kv_attn_workspace(dim)))
    return rc;
  vbq::KvAttention a;
  a.q = q, a.out = out, a.lse = lse, a.q_stride = q_stride, a.out_stride = out_stride, a.rows = rows;
  a.group = heads / kv_heads;
  a.scale = scale * 1.4426950408889634f;
  a.window = window;
  return launched(who, vbq::launch_kv_attn(a, cache(codes, scales, pages, layers, layer, kv_heads, page, dim),
                                           vbq::KvBatch{tables, lens, q_start, seqs, max_pages},
                                           dtype == VBQ_DTYPE_BF16, max_new, workspace,
                                           static_cast<cudaStream_t>(stream)));
}

int vbq_kv_pages_workspace_bytes(int64_t pages, int32_t rows, size_t* bytes) {
  const char* who = "vbq_kv_pages_workspace_bytes";
  if (!bytes) return api_status(VBQ_ERR_NULL, "%s: bytes is NULL", who);
  if (pages < 1 || pages > INT32_MAX / 2 || rows < 0)
    return api_status(VBQ_ERR_SHAPE, "%s: need 1 <= pages < 2^30 and rows >= 0", who);
  *bytes = vbq::kv_pages_workspace(pages, rows);
  return ok();
}

int vbq_kv_reserve(const int32_t* refs, const int32_t* tables, const int32_t* lens,
                   const int32_t* new_tokens, int64_t pages, int32_t page, int32_t rows,
                   int32_t max_pages, int32_t* refs_out, int32_t* tables_out, int32_t* lens_out,
                   int32_t* missing, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "vbq_kv_reserve";
  if (int rc = pool_sizes(who, pages, page, rows, max_pages)) return rc;
  if (!refs || !refs_out || !missing || (rows > 0 && (!tables || !lens || !new_tokens || !tables_out || !lens_out)))
    return api_status(VBQ_ERR_NULL, "%s: NULL pointer", who);
  if (!words(refs, tables, lens, new_tokens, refs_out, tables_out, lens_out, missing)) return bad_words(who);
  if (int rc = workspace_ok(who, workspace, workspace_bytes, vbq::kv_pages_workspace(pages, rows))) return rc;
  return launched(who, vbq::launch_kv_reserve(refs, tables, lens, new_tokens, pages, page, rows, max_pages, refs_out,
                                              tables_out, lens_out, missing, workspace,
                                              static_cast<cudaStream_t>(stream)));
}

int vbq_kv_fork(void* codes, float* scales, int64_t pages, int64_t page_bytes, int64_t page_scales,
                int32_t page, const int32_t* refs, const int32_t* tables, const int32_t* lens, int32_t rows,
                int32_t max_pages, const int32_t* parents, int32_t new_rows, int32_t* refs_out,
                int32_t* tables_out, int32_t* lens_out, int32_t* missing, void* workspace,
                size_t workspace_bytes, void* stream) {
  const char* who = "vbq_kv_fork";
  if (int rc = pool_sizes(who, pages, page, rows, max_pages)) return rc;
  if (int rc = pool_sizes(who, pages, page, new_rows, max_pages)) return rc;
  if (int rc = pool_data(who, codes, scales, page_bytes, page_scales)) return rc;
  if (!refs || !refs_out || !missing || (rows > 0 && (!tables || !lens)) ||
      (new_rows > 0 && (!parents || !tables_out || !lens_out)))
    return api_status(VBQ_ERR_NULL, "%s: NULL pointer", who);
  if ((new_rows > 0 && rows > 0) && (tables_out == tables || lens_out == lens))
    return api_status(VBQ_ERR_SHAPE, "%s: tables_out and lens_out must not be tables and lens", who);
  if (!words(refs, tables, lens, parents, refs_out, tables_out, lens_out, missing)) return bad_words(who);
  const int32_t most = rows > new_rows ? rows : new_rows;
  if (int rc = workspace_ok(who, workspace, workspace_bytes, vbq::kv_pages_workspace(pages, most))) return rc;
  const vbq::KvPool pool{static_cast<uint8_t*>(codes), scales, pages, page_bytes, page_scales, page};
  return launched(who, vbq::launch_kv_fork(pool, refs, tables, lens, rows, max_pages, parents, new_rows, refs_out,
                                           tables_out, lens_out, missing, workspace,
                                           static_cast<cudaStream_t>(stream)));
}

int vbq_kv_compact(void* codes, float* scales, int64_t pages, int64_t page_bytes, int64_t page_scales,
                   int32_t page, const int32_t* refs, const int32_t* tables, const int32_t* lens,
                   int32_t rows, int32_t max_pages, int32_t* refs_out, int32_t* tables_out, int32_t* live,
                   void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "vbq_kv_compact";
  if (int rc = pool_sizes(who, pages, page, rows, max_pages)) return rc;
  if (int rc = pool_data(who, codes, scales, page_bytes, page_scales)) return rc;
  if (!refs || !refs_out || !live || (rows > 0 && (!tables || !lens || !tables_out)))
    return api_status(VBQ_ERR_NULL, "%s: NULL pointer", who);
  if (!words(refs, tables, lens, refs_out, tables_out, live)) return bad_words(who);
  if (int rc = workspace_ok(who, workspace, workspace_bytes, vbq::kv_pages_workspace(pages, rows))) return rc;
  const vbq::KvPool pool{static_cast<uint8_t*>(codes), scales, pages, page_bytes, page_scales, page};
  return launched(who, vbq::launch_kv_compact(pool, refs, tables, lens, rows, max_pages, refs_out, tables_out, live,
                                              workspace, static_cast<cudaStream_t>(stream)));
}

static int logprob_sizes(const char* who, int64_t rows, int64_t vocab, int32_t top) {
  if (rows < 0 || rows > INT32_MAX || vocab < 1 || vocab > INT32_MAX - 64)
    return api_status(VBQ_ERR_SHAPE, "%s: need 0 <= rows < 2^31 and 1 <= vocab < 2^31 - 64", who);
  if (top < 0 || top > vbq::kMaxTop || top > vocab)
    return api_status(VBQ_ERR_SHAPE, "%s: top must be in 0..%d and at most vocab, got %d", who, vbq::kMaxTop, top);
  return VBQ_OK;
}

int vbq_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int32_t top, size_t* bytes) {
  const char* who = "vbq_token_logprobs_workspace_bytes";
  if (!bytes) return api_status(VBQ_ERR_NULL, "%s: bytes is NULL", who);
  if (int rc = logprob_sizes(who, rows, vocab, top)) return rc;
  *bytes = vbq::logprobs_workspace(rows, vocab, top);
  return ok();
}

int vbq_token_logprobs(const void* logits, int64_t stride, int32_t dtype, int64_t rows, int64_t vocab,
                       const int32_t* tokens, int32_t top, float* logprob, float* entropy,
                       float* top_logprob, int32_t* top_token, void* workspace, size_t workspace_bytes,
                       void* stream) {
  const char* who = "vbq_token_logprobs";
  if (!dtype_ok(dtype)) return bad_dtype(who, dtype);
  if (int rc = logprob_sizes(who, rows, vocab, top)) return rc;
  if (stride < vocab) return api_status(VBQ_ERR_SHAPE, "%s: the row stride is less than vocab", who);
  if (rows == 0) return ok();
  if (!logits || (tokens && !logprob) || (top > 0 && (!top_logprob || !top_token)))
    return api_status(VBQ_ERR_NULL, "%s: NULL pointer", who);
  if (!aligned(logits, dtype == VBQ_DTYPE_F32 ? 4 : 2))
    return api_status(VBQ_ERR_ALIGN, "%s: logits must be element-aligned", who);
  if (!words(tokens, logprob, entropy, top_logprob, top_token)) return bad_words(who);
  if (int rc = workspace_ok(who, workspace, workspace_bytes, vbq::logprobs_workspace(rows, vocab, top))) return rc;
  return launched(who, vbq::launch_logprobs(logits, stride, dtype == VBQ_DTYPE_BF16, rows, vocab, tokens, top, logprob,
                                            entropy, top_logprob, top_token, workspace,
                                            static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
