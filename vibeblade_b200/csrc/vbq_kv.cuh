// vbq_kv.cuh -- the 8-bit paged KV cache as the kernels see it.
#pragma once
#include "vbq_common.cuh"
#include "vbq_kv_internal.h"

namespace vbq {
namespace kv {

constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ int seq_new(const KvBatch& b, int s) {
  const int n = __ldg(b.q_start + s + 1) - __ldg(b.q_start + s);
  return n > 0 ? n : 0;
}
__device__ __forceinline__ int seq_len(const KvBatch& b, int s) {
  const int n = __ldg(b.lens + s);
  return n > 0 ? n : 0;
}

// The page that holds token run `j` of sequence s, or -1 where there is none.
__device__ __forceinline__ int page_of(const KvCache& c, const KvBatch& b, int s, int j) {
  if (j < 0 || j >= b.max_pages) return -1;
  const int p = __ldg(b.tables + (int64_t)s * b.max_pages + j);
  return (p >= 0 && p < c.pages) ? p : -1;
}

// Codes [page][dim] and the scale of (page, layer, keys / values, head).
__device__ __forceinline__ int64_t block_index(const KvCache& c, int page, int which, int head) {
  return (((int64_t)page * c.layers + c.layer) * 2 + which) * c.heads + head;
}

// The first key that a row whose last one is `hi` sees; what is before the sequence's first (hi < 0, where the
// row sees nothing) is 0 too, so that no window reaches past int32.
__device__ __forceinline__ int first_key(const KvAttention& a, int hi) {
  return a.window > 0 && hi >= a.window ? hi - a.window + 1 : 0;
}

// A value block's scale as the attention's weights take it.  They carry it, and the sum of exponentials
// takes its reciprocal: a block of zeros, whose scale is 0 and any would do, gets one that leaves the
// sum of 2^24 tokens' weights (2^15 at most) in fp32 and lies below every scale that matters.
__device__ __forceinline__ float value_scale(float vs) { return vs == 0.0f ? 0x1p-60f : fmaxf(vs, 1e-30f); }

// a / b of numbers that are not negative, by the short division where both are short.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return ((a | b) >> 32) ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

template <typename V> __device__ __forceinline__ V warp_scan(V v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V u = __shfl_up_sync(kFull, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Work units laid out sequence after sequence, units(s) of them each: the sequence unit u
// is in and its number there.  Every lane of the warp calls it with the same u; s = -1 past
// the last unit.
struct Unit {
  int s;
  int64_t at;
};
template <typename F>
__device__ __forceinline__ Unit find_unit(int64_t u, int seqs, int lane, F units) {
  int64_t before = 0;
  for (int s0 = 0; s0 < seqs; s0 += 32) {
    const int64_t mine = s0 + lane < seqs ? (int64_t)units(s0 + lane) : 0;
    const int64_t end = before + warp_scan(mine, lane);
    const unsigned past = __ballot_sync(kFull, end > u);
    if (past) {
      const int l = __ffs(past) - 1;
      return {s0 + l, u - __shfl_sync(kFull, end - mine, l)};
    }
    before = __shfl_sync(kFull, end, 31);
  }
  return {-1, 0};
}
template <typename F>
__device__ __forceinline__ int64_t count_units(int seqs, int lane, F units) {
  int64_t n = 0;
  for (int s = lane; s < seqs; s += 32) n += (int64_t)units(s);
#pragma unroll
  for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(kFull, n, o);
  return n;
}

__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// Lets the next kernel of the stream start while this one runs (if it was launched to), and waits
// for the kernel before to have ended.
__device__ __forceinline__ void pdl_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Launches a kernel that begins with pdl_wait(): it is set up while the kernel before it ends.
template <typename... P, typename... A>
cudaError_t launch_behind(void (*kern)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...);
}

// Rows of the call that no sequence has, before q_start's first and from its last on, see no token: zeros
// and -inf.  The grid's CTAs share the rows; there mostly are none.
template <bool F32>
__device__ __forceinline__ void blank_rows(const KvAttention& a, const KvCache& c, const KvBatch& b) {
  const int from = __ldg(b.q_start), to = __ldg(b.q_start + b.seqs);
  const int heads = c.heads * a.group, width = heads * (c.dim * (F32 ? 4 : 2) / 16);  // 16-byte pieces of a row
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    if (row >= from && row < to) continue;
    uint4* out = reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.out) + row * a.out_stride * (F32 ? 4 : 2));
    for (int x = threadIdx.x; x < width; x += blockDim.x) out[x] = make_uint4(0, 0, 0, 0);
    if (a.lse)
      for (int x = threadIdx.x; x < heads; x += blockDim.x) a.lse[row * heads + x] = -INFINITY;
  }
}

constexpr float kLn2 = 0.6931471805599453f;
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t h2(float lo, float hi) {
  const __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ float2 h2f(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }

// 4 codes of a word as fp16 pairs (0, 1) and (2, 3): byte u = code + 128 in the mantissa of
// 1024 is 1024 + u, minus 1152 (both exact).
__device__ __forceinline__ uint32_t sub1152(uint32_t w) {
  const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&w), __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void codes_h2(uint32_t w, uint32_t& a, uint32_t& b) {
  const uint32_t u = w ^ 0x80808080u;
  a = sub1152(__byte_perm(u, 0x64646464u, 0x4140));
  b = sub1152(__byte_perm(u, 0x64646464u, 0x4342));
}

}  // namespace kv
}  // namespace vbq
