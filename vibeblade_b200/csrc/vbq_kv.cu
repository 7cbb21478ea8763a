// vbq_kv.cu -- storing new keys and values in the 8-bit paged cache, and reading them back.
//
// A page holds `page` tokens of every head as int8 codes with one fp32 scale a (layer, keys
// or values, head): value = scale * code.  The new tokens of a sequence touch the pages from
// the one its first new token falls in; per touched block
//     a  = max |x| over the new values (finite ones),   s1 = max(s0, a / 127),
//     old codes: rint(code * (s0 / s1)) where s1 > s0,  new codes: clamp(rint(x / s1), +-127)
// with s0 the block's scale if it already held tokens of the sequence.  Every operation is
// one fp32 rounding, so the stored bytes do not depend on how the work is split.
//
// Bytes bound the long appends: the rows are read once and held on chip between the look for the
// largest value and the rounding.  Measured (device time, append and read back): 6 sequences of up
// to 5001 new tokens, 8 heads of 128, bf16, 150 MB: 39 us, 3.9 TB/s (append 22.5, read 16.5), 70 % of
// its issue slots taken; 64 sequences of one token, fp32: 9 us, which is latency.
#include "vbq_internal.h"
#include "vbq_kv.cuh"

namespace vbq {
namespace kv {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kHold = 8;  // 16-byte vectors of its block a warp's thread keeps between the two looks

template <bool BF16> struct Vec {  // 16 bytes of a row
  static constexpr int kN = BF16 ? 8 : 4;
  __device__ __forceinline__ static uint4 load(const void* p, int64_t at) {
    return __ldg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + at * (BF16 ? 2 : 4)));
  }
  __device__ __forceinline__ static void unpack(const uint4& v, float (&x)[kN]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (BF16) x[2 * i] = bf_lo(w[i]), x[2 * i + 1] = bf_hi(w[i]);
      else x[i] = __uint_as_float(w[i]);
    }
  }
};

// Pages that a sequence's new tokens touch.
__device__ __forceinline__ int touched(const KvCache& c, const KvBatch& b, int s) {
  const int n = seq_new(b, s), len = seq_len(b, s);
  if (n == 0 || len == 0) return 0;
  const int first = max(len - n, 0) >> c.page_log2;
  return ((len - 1) >> c.page_log2) - first + 1;
}

__device__ __forceinline__ int quant1(float x, float s) {
  const float y = rintf(__fdiv_rn(x, s));
  return y != y ? 0 : (int)fminf(fmaxf(y, -127.0f), 127.0f);
}

// One CTA (WARP: one warp, for appends of a token or a few a sequence) a (touched page, head, keys
// or values).
template <bool BF16, bool WARP>
__global__ void __launch_bounds__(kAppendThreads, WARP ? 2 : 5)
append_kernel(const void* __restrict__ k, int64_t k_stride, const void* __restrict__ v, int64_t v_stride,
              int64_t rows, KvCache c, KvBatch b) {
  pdl_wait();
  using V = Vec<BF16>;
  constexpr int kGroup = WARP ? 32 : kAppendThreads;  // threads a block of the cache
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tid = WARP ? lane : threadIdx.x;
  // a page's heads side by side: together they read whole rows
  const uint32_t work = WARP ? blockIdx.x * (kAppendThreads / 32) + warp : blockIdx.x;
  const uint32_t pair = work / (uint32_t)c.heads;
  const int head = (int)(work - pair * c.heads), which = (int)(pair & 1);
  const Unit u = find_unit((int64_t)(pair >> 1), b.seqs, lane, [&](int s) { return touched(c, b, s); });
  if (u.s < 0) return;
  const int n = seq_new(b, u.s), len = seq_len(b, u.s);
  const int start = len - n;
  const int run = (max(start, 0) >> c.page_log2) + (int)u.at;
  const int page = page_of(c, b, u.s, run);
  if (page < 0) return;
  const int p0 = run << c.page_log2;
  const int from = max(start, p0), to = min(len, p0 + c.page);  // the page's new tokens
  const int64_t row0 = (int64_t)__ldg(b.q_start + u.s) + (from - start);
  const int count = (int)min((int64_t)(to - from), rows - row0);
  if (row0 < 0 || count <= 0) return;
  const void* src = which ? v : k;
  const int64_t stride = which ? v_stride : k_stride;
  const int row_log2 = 31 - __clz(c.dim / V::kN);  // threads a row
  const int col = (tid & ((1 << row_log2) - 1)) * V::kN;
  const int step = kGroup >> row_log2, r0 = tid >> row_log2;
  const int64_t base = row0 * stride + (int64_t)head * c.dim + col;

  // the largest |x| as bits (of bf16, two at a time): infinities and NaN are above every number
  uint32_t top = 0;
  auto look = [&](const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (BF16) top = __vmaxu2(top, w[i] & 0x7fff7fffu);
      else top = max(top, w[i] & 0x7fffffffu);
    }
  };
  // between the two looks a warp's values wait in registers, a CTA's in shared memory (each thread's
  // own: it is there for the bytes in flight, 190 KB an SM instead of 96)
  extern __shared__ __align__(16) uint8_t smem[];
  uint4 held[WARP ? kHold : 1];
  uint4* mine = reinterpret_cast<uint4*>(smem) + tid;
  if constexpr (WARP) {
#pragma unroll
    for (int i = 0; i < kHold; ++i)
      if (r0 + i * step < count) held[i] = V::load(src, base + (int64_t)(r0 + i * step) * stride);
#pragma unroll
    for (int i = 0; i < kHold; ++i)
      if (r0 + i * step < count) look(held[i]);
    for (int r = r0 + kHold * step; r < count; r += step) look(V::load(src, base + (int64_t)r * stride));
  } else {
    const uint8_t* from_row = static_cast<const uint8_t*>(src) + base * (BF16 ? 2 : 4);
    for (int r = r0, i = 0; r < count; r += step, ++i)
      cp_async16(mine + i * kGroup, from_row + (int64_t)r * stride * (BF16 ? 2 : 4));
    cp_async_commit();
    cp_async_wait<0>();
    for (int r = r0, i = 0; r < count; r += step, ++i) look(mine[i * kGroup]);
  }
  __shared__ uint32_t part[kAppendThreads / 32];
  auto largest = [&](uint32_t v) {  // of the block's threads
    v = __reduce_max_sync(kFull, v);
    if constexpr (!WARP) {
      __syncthreads();
      if (lane == 0) part[warp] = v;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kAppendThreads / 32; ++w) v = max(v, part[w]);
    }
    return v;
  };
  constexpr uint32_t kInf = 0x7f800000u;
  if constexpr (BF16) top = max(top << 16, top & 0xffff0000u);
  top = largest(top);
  const bool finite = top < kInf;
  if (!finite) {  // once more, passing over what is not finite
    top = 0;
    for (int r = r0; r < count; r += step) {
      float x[V::kN];
      V::unpack(V::load(src, base + (int64_t)r * stride), x);
#pragma unroll
      for (int i = 0; i < V::kN; ++i) {
        const uint32_t m = __float_as_uint(x[i]) & 0x7fffffffu;
        if (m < kInf) top = max(top, m);
      }
    }
    top = largest(top);
  }
  const float a = __uint_as_float(top);

  const int64_t blk = block_index(c, page, which, head);
  int8_t* codes = c.codes + blk * ((int64_t)c.page * c.dim);
  const int old = from - p0;  // tokens of the sequence already in the page
  const float s0 = old > 0 ? c.scales[blk] : 0.0f;
  const float s1 = fmaxf(s0, __fdiv_rn(a, 127.0f));
  if constexpr (WARP) __syncwarp();
  else __syncthreads();
  if (tid == 0)  // every thread has read the scale
     c.scales[blk] = s1;

  if (old > 0 && s1 > s0) {
    const float ratio = __fdiv_rn(s0, s1);
    uint4* oc = reinterpret_cast<uint4*>(codes);
    for (int i = tid; i < old * c.dim / 16; i += kGroup) {
      const uint4 w = oc[i];
      uint32_t in[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t o = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = rintf(__fmul_rn(s8f(in[j] >> (8 * e)), ratio));
          o |= ((uint32_t)(int)y & 0xffu) << (8 * e);
        }
        in[j] = o;
      }
      oc[i] = make_uint4(in[0], in[1], in[2], in[3]);
    }
  }
  // x / s1 to the nearest integer.  y = x (1 / s1) is within 2^-16 of the quotient, so where y is
  // not that near to a half both round to the same integer; the others (and what is not finite)
  // divide.  Adding 1.5 2^23 rounds y to an integer and leaves it in the low byte.
  // (With nothing but numbers in the block |y| is at most 127 and a rounding.)
  const bool quick = finite && s1 > 1e-30f;
  const float inv = quick ? __fdiv_rn(1.0f, s1) : 0.0f;
  auto store = [&](const uint4& v, int r) {
    float x[V::kN];
    V::unpack(v, x);
    uint32_t o[V::kN / 4] = {};
    constexpr float kMagic = 12582912.0f;
    float off[2] = {0.0f, 0.0f};
    uint32_t b[V::kN];
#pragma unroll
    for (int i = 0; i < V::kN; i += 2) {
      const float2 y = __fmul2_rn(make_float2(x[i], x[i + 1]), make_float2(inv, inv));
      const float2 t = __fadd2_rn(y, make_float2(kMagic, kMagic));
      const float2 n = __fadd2_rn(t, make_float2(-kMagic, -kMagic));
      const float2 d = __ffma2_rn(n, make_float2(-1.0f, -1.0f), y);
      off[0] = fmaxf(off[0], fabsf(d.x)), off[1] = fmaxf(off[1], fabsf(d.y));
      b[i] = __float_as_uint(t.x), b[i + 1] = __float_as_uint(t.y);
    }
    if (quick && fmaxf(off[0], off[1]) < 0.49996f) {
#pragma unroll
      for (int i = 0; i < V::kN / 4; ++i)
        o[i] = __byte_perm(__byte_perm(b[4 * i], b[4 * i + 1], 0x0040), __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x0040), 0x5410);
    } else if (s1 > 0.0f) {
#pragma unroll
      for (int i = 0; i < V::kN; ++i) o[i / 4] |= ((uint32_t)quant1(x[i], s1) & 0xffu) << (8 * (i & 3));
    }
    int8_t* dst = codes + (int64_t)(old + r) * c.dim + col;
    if constexpr (BF16) *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
    else *reinterpret_cast<uint32_t*>(dst) = o[0];
  };
  if constexpr (WARP) {
#pragma unroll
    for (int i = 0; i < kHold; ++i)
      if (r0 + i * step < count) store(held[i], r0 + i * step);
    for (int r = r0 + kHold * step; r < count; r += step) store(V::load(src, base + (int64_t)r * stride), r);
  } else {
    for (int r = r0, i = 0; r < count; r += step, ++i) store(mine[i * kGroup], r);
  }
}

// One warp a row: its codes of every head, keys then values.
constexpr int kReadWarps = 8;
template <bool BF16>
__global__ void __launch_bounds__(32 * kReadWarps)
read_kernel(KvCache c, KvBatch b, int64_t rows, void* __restrict__ k_out, void* __restrict__ v_out) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kReadWarps + (threadIdx.x >> 5);
  if (row >= rows) return;
  int s = -1;
  for (int s0 = 0; s0 < b.seqs && s < 0; s0 += 32) {
    const int i = s0 + lane;
    const bool in = i < b.seqs && __ldg(b.q_start + i) <= row && row < __ldg(b.q_start + i + 1);
    const unsigned hit = __ballot_sync(kFull, in);
    if (hit) s = s0 + __ffs(hit) - 1;
  }
  int page = -1, at = 0;
  if (s >= 0) {
    const int pos = seq_len(b, s) - (int)(__ldg(b.q_start + s + 1) - row);
    if (pos >= 0) {
      page = page_of(c, b, s, pos >> c.page_log2);
      at = pos & (c.page - 1);
    }
  }
  // 16 bytes out a lane and step: 4 codes as fp32 or 8 as bf16, adjacent lanes side by side
  const int width = c.heads * c.dim, dim_log2 = 31 - __clz(c.dim);
  constexpr int kCodes = BF16 ? 8 : 4, kAtOnce = 8;
  for (int i0 = lane * kCodes; i0 < 2 * width; i0 += kAtOnce * 32 * kCodes) {
    uint2 w[kAtOnce];
    float sc[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int i = i0 + k * 32 * kCodes;
      w[k] = make_uint2(0x80808080u, 0x80808080u);
      sc[k] = 0.0f;
      if (i < 2 * width && page >= 0) {
        const int which = i >= width, j = which ? i - width : i;
        const int head = j >> dim_log2, col = j & (c.dim - 1);
        const int64_t blk = block_index(c, page, which, head);
        const int8_t* p = c.codes + (blk * c.page + at) * c.dim + col;
        if constexpr (BF16) w[k] = __ldg(reinterpret_cast<const uint2*>(p));
        else w[k].x = __ldg(reinterpret_cast<const uint32_t*>(p));
        sc[k] = __ldg(c.scales + blk);
      }
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int i = i0 + k * 32 * kCodes;
      if (i >= 2 * width) break;
      const int which = i >= width, j = which ? i - width : i;
      float y[kCodes];
#pragma unroll
      for (int e = 0; e < kCodes; ++e)
        y[e] = page >= 0 ? __fmul_rn(sc[k], s8f((e < 4 ? w[k].x : w[k].y) >> (8 * (e & 3)))) : 0.0f;
      const int64_t o = row * width + j;
      if constexpr (BF16)
        __stcs(reinterpret_cast<uint4*>(static_cast<uint16_t*>(which ? v_out : k_out) + o),
               make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7])));
      else
        __stcs(reinterpret_cast<float4*>(static_cast<float*>(which ? v_out : k_out) + o), make_float4(y[0], y[1], y[2], y[3]));
    }
  }
}

}  // namespace
}  // namespace kv

cudaError_t launch_kv_append(const void* k, int64_t k_stride, const void* v, int64_t v_stride, bool bf16,
                             int64_t rows, const KvCache& c, const KvBatch& b, cudaStream_t st) {
  // touched pages: a sequence with n > 0 new tokens touches at most n / page + 2, and at most n
  const int64_t some = rows < b.seqs ? rows : b.seqs;
  int64_t units = rows / c.page + 2 * some;
  if (units > rows) units = rows;
  if (rows <= 4 * (int64_t)b.seqs && c.dim <= (bf16 ? 256 : 128)) {  // a row is at most a warp's 16-byte vectors
    // a few tokens a sequence: a block's work is its latency, so as many blocks at a time as there
    // are warps (64 sequences of one token, 8 heads, with the read back: 17.8 us a CTA a block, 12.9 us
    // a warp a block)
    const int64_t warps = units * 2 * c.heads;
    if (warps > INT32_MAX) return cudaErrorInvalidValue;
    const unsigned grid = (unsigned)((warps + kv::kAppendThreads / 32 - 1) / (kv::kAppendThreads / 32));
    auto kern = bf16 ? kv::append_kernel<true, true> : kv::append_kernel<false, true>;
    return kv::launch_behind(kern, grid, kv::kAppendThreads, 0, st, k, k_stride, v, v_stride, rows, c, b);
  }
  auto kern = bf16 ? kv::append_kernel<true, false> : kv::append_kernel<false, false>;
  const int smem = c.page * c.dim * (bf16 ? 2 : 4);
  static DeviceOnce configured;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!configured.done(dev)) {  // the largest block: 128 tokens of 256 fp32 values
    e = cudaFuncSetAttribute(kv::append_kernel<true, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * 256 * 2);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kv::append_kernel<false, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * 256 * 4);
    if (e != cudaSuccess) return e;
    configured.mark(dev);
  }
  if (units * 2 * c.heads > INT32_MAX) return cudaErrorInvalidValue;
  return kv::launch_behind(kern, (unsigned)(units * 2 * c.heads), kv::kAppendThreads, smem, st, k, k_stride, v, v_stride, rows, c, b);
}

cudaError_t launch_kv_read(const KvCache& c, const KvBatch& b, int64_t rows, void* k_out, void* v_out,
                           bool bf16, cudaStream_t st) {
  const unsigned grid = (unsigned)((rows + kv::kReadWarps - 1) / kv::kReadWarps);
  auto kern = bf16 ? kv::read_kernel<true> : kv::read_kernel<false>;
  return kv::launch_behind(kern, grid, 32 * kv::kReadWarps, 0, st, c, b, rows, k_out, v_out);
}

}  // namespace vbq
