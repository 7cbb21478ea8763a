// vbq_logprobs.cu -- log probabilities, entropy and the largest tokens of logit rows.
//
// One pass over a row (or a slice of it) keeps, a thread,
//     Z = sum e^(x - r),  B = sum (x - r) e^(x - r),  the largest x,
// with a reference r that moves only when some x exceeds it by 8.  Then lse = r + log Z and
// entropy = log Z - B / Z: no second pass and no probabilities in memory; the logits' bytes
// bound it.
//
// The `top` largest without a second pass: the top-th largest of 64 lanes' maxima (each warp's
// few largest) is at most the top-th largest logit.  Only lanes whose maximum reaches that bound
// can hold one of the top (not many more than `top`), and only their elements are read again, by
// the whole warp, 32 vectors at a time; the elements that reach the bound are collected in shared
// memory and ranked by counting (value, then lower token).  Where more of them reach it than fit (a mask
// that leaves fewer tokens than are listed: the bound is then the mask's value) the row is read twice
// more: for what lies above the bound, and up to the first of its equals that are wanted.
//
// Few long rows are split over CTAs; the last to arrive joins the slices' sums in slice order
// and ranks their top lists the same way.
//
// Measured (device time of a call among others): 2047 rows of 128256 bf16 logits, top 20, 525 MB: 132 us
// at 1747 MHz, where the power limit holds the SMs in a row of calls, 4.0 TB/s; 117 at 1965 (of its issue
// slots 69 % are taken, of the MUFU's 58 %; the rest is each row's list, under which the other CTAs of the
// SM load).  1023 rows of fp32, as many bytes: 122 us at 1852 MHz.  600 rows of bf16, 154 MB: 47 us; 83
// where a mask leaves three tokens a row.  8 rows of fp32, top 5: 11 us, which is latency: the pass, the
// list's second reads, the join.
#include <climits>
#include <cmath>

#include "vbq_internal.h"
#include "vbq_kv.cuh"

namespace vbq {
namespace lp {
namespace {

using kv::kFull;
constexpr int kCap = 512;           // candidates kept in shared memory
constexpr float kSlack = 8.0f;
constexpr int kSliceThreads = 256;
constexpr int kFew = 4;             // vectors a thread, up to which lanes look at their own
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = 1e30f;       // from here on x - r can leave fp32, or r be a type's lowest value
constexpr int kUnroll = 2;         // vectors on their way a thread (4: 125 us against 114 over 525 MB)
constexpr int kMaxSplits = 128, kMaxSplitRows = 512;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// order of floats as order of ints (no NaN)
__device__ __forceinline__ int key_of(float x) {
  const int b = __float_as_int(x);
  return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float of_key(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }
__device__ __forceinline__ bool better(float x, int i, float y, int j) { return x > y || (x == y && i < j); }

struct Sums {
  float r, z, b;  // reference, sum e^(x - r), sum (x - r) e^(x - r)
};
__device__ __forceinline__ Sums shifted(Sums s, float to) {  // the same sums with the reference `to`
  const float d = s.r - to;
  if (d == 0.0f) return s;
  const float f = ex2(fmaxf(d, -1e4f) * kLog2e);
  return {to, s.z * f, f == 0.0f ? s.z * 0.0f : (s.b + d * s.z) * f};
}
__device__ __forceinline__ Sums joined(Sums a, Sums c) {
  const float to = fmaxf(a.r, c.r);
  a = shifted(a, to), c = shifted(c, to);
  return {to, a.z + c.z, a.b + c.b};
}

// A slice [e0, e1) of a row as aligned 16-byte vectors: whole ones a0 .. a1 - 1, and the elements
// before and after them (less than a vector each).  Vector i holds elements i kN - lead ..
template <bool BF16> struct Row {
  static constexpr int kN = BF16 ? 8 : 4;
  const uint8_t* base;  // 16-byte aligned, lead elements before the row
  int lead, e0, e1, a0, a1;
  __device__ __forceinline__ Row(const void* p, int64_t from, int64_t to) : e0((int)from), e1((int)to) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    base = reinterpret_cast<const uint8_t*>(a & ~uintptr_t(15));
    lead = (int)(a & 15) / (16 / kN);
    a0 = (e0 + lead + kN - 1) / kN;
    a1 = max(a0, (e1 + lead) / kN);
  }
  __device__ __forceinline__ uint4 vec(int i) const { return kv::ld_stream(base + (int64_t)i * 16); }
  __device__ __forceinline__ float one(int e) const {  // element e of the row
    const int64_t i = (int64_t)e + lead;
    if constexpr (BF16) return kv::bf_lo((uint32_t) * (reinterpret_cast<const uint16_t*>(base) + i));
    else return *(reinterpret_cast<const float*>(base) + i);
  }
  // The slice's elements outside its whole vectors, by number 0 .. 2 kN - 1; -1 past the last.
  __device__ __forceinline__ int loose(int k) const {
    const int head = min(e1, a0 * kN - lead);
    if (k < kN) return e0 + k < head ? e0 + k : -1;
    const int tail = max(head, a1 * kN - lead) + k - kN;
    return tail < e1 ? tail : -1;
  }
  __device__ __forceinline__ void unpack(const uint4& w, float (&x)[kN]) const {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (BF16) x[2 * i] = kv::bf_lo(v[i]), x[2 * i + 1] = kv::bf_hi(v[i]);
      else x[i] = __uint_as_float(v[i]);
    }
  }
};

// -inf as the type's lowest value; NaN stays.  Beside a larger reference the weight is 0 either way, and
// 0 times it is 0; a slice that has nothing larger is summed again (kFar).
__device__ __forceinline__ uint32_t floor2(uint32_t w) {
  const __nv_bfloat162 lo = __halves2bfloat162(__ushort_as_bfloat16(0xff7f), __ushort_as_bfloat16(0xff7f));
  const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&w), lo);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

template <int kThreads> struct Shared {
  static constexpr int kWarps = kThreads / 32;
  static constexpr int kTops = 64;    // lane maxima for the bound
  float tops[kTops];
  float cv[kCap];
  int ci[kCap];
  int count;
  float bound_f;
  Sums part[kWarps];
  float lse, shift;
  int last;
  float tv[kMaxTop];
  int ti[kMaxTop];
};

// Ranks sh.cv / ci [0, n) by counting: the top ones to sh.tv / ti (already padded).
template <int kThreads>
__device__ __forceinline__ void rank_candidates(Shared<kThreads>& sh, int n, int top) {
  for (int a = threadIdx.x; a < n; a += kThreads) {
    const float x = sh.cv[a];
    const int i = sh.ci[a];
    int r = 0;
    for (int c = 0; c < n; ++c) r += better(sh.cv[c], sh.ci[c], x, i);
    if (r < top) sh.tv[r] = x, sh.ti[r] = i;
  }
}

// One warp: inserts (x, i) of the lanes for which `want` holds into a list kept one entry a lane.
__device__ __forceinline__ void insert(float x, int i, bool want, int top, int lane, float& lv, int& li) {
  for (;;) {
    const float tv = __shfl_sync(kFull, lv, top - 1);
    const int ti = __shfl_sync(kFull, li, top - 1);
    want = want && better(x, i, tv, ti);
    const unsigned hit = __ballot_sync(kFull, want);
    if (!hit) return;
    const int l = __ffs(hit) - 1;
    const float v = __shfl_sync(kFull, x, l);
    const int j = __shfl_sync(kFull, i, l);
    if (lane == l) want = false;
    const int pos = __popc(__ballot_sync(kFull, better(lv, li, v, j)));
    const float pv = __shfl_up_sync(kFull, lv, 1);
    const int pi = __shfl_up_sync(kFull, li, 1);
    if (lane == pos) lv = v, li = j;
    else if (lane > pos) lv = pv, li = pi;
  }
}

// The list of a slice of which more elements reach the bound than the shared list holds: those above it,
// by rank, then its equals, lowest first.  Too many above it (large logits crowded into few lanes): the
// top-th of as many as fit is a bound too, and a higher one; after kRaises such passes one warp inserts
// the elements one by one.
constexpr int kRaises = 8;
template <bool BF16, int kThreads>
__device__ __forceinline__ void crowded(Shared<kThreads>& sh, const Row<BF16> row, float bound, int top) {
  constexpr int kN = Row<BF16>::kN, kWarps = kThreads / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto above = [&](float x, int e) {
    if (x > bound) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < kCap) sh.cv[at] = x, sh.ci[at] = e;
    }
  };
  int n;
  for (int raise = 0;; ++raise) {
    __syncthreads();
    if (tid == 0) sh.count = 0;
    __syncthreads();
    for (int a = row.a0 + tid; a < row.a1; a += kThreads) {
      float x[kN];
      row.unpack(row.vec(a), x);
#pragma unroll
      for (int j = 0; j < kN; ++j) above(x[j], a * kN - row.lead + j);
    }
    if (tid < 2 * kN && row.loose(tid) >= 0) above(row.one(row.loose(tid)), row.loose(tid));
    __syncthreads();
    n = sh.count;
    if (n <= kCap || raise == kRaises) break;
    for (int a = tid; a < kCap; a += kThreads) {
      int r = 0;
      for (int c = 0; c < kCap; ++c) r += better(sh.cv[c], sh.ci[c], sh.cv[a], sh.ci[a]);
      if (r == top - 1) sh.bound_f = sh.cv[a];
    }
    __syncthreads();
    bound = sh.bound_f;
  }
  if (n > kCap) {
    if (warp == 0) {
      float lv = -INFINITY;
      int li = INT_MAX;
      for (int64_t a = row.e0; a < row.e1; a += 32) {
        const bool in = a + lane < row.e1;
        insert(in ? row.one((int)a + lane) : 0.0f, (int)a + lane, in, top, lane, lv, li);
      }
      if (lane < top) sh.tv[lane] = lv, sh.ti[lane] = li;
    }
    return;
  }
  rank_candidates(sh, n, top);
  // kEach elements a thread, in order
  constexpr int kEach = 8;
  int* counts = reinterpret_cast<int*>(sh.tops);
  for (int64_t e0 = row.e0; e0 < row.e1 && n < top; e0 += kThreads * kEach) {
    const int64_t e = e0 + tid * kEach;
    unsigned equal = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (e + j < row.e1 && row.one((int)(e + j)) == bound) equal |= 1u << j;
    const int upto = kv::warp_scan(__popc(equal), lane);
    if (lane == 31) counts[warp] = upto;
    __syncthreads();
    int r = n + upto - __popc(equal), all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) r += counts[w];
      all += counts[w];
    }
    for (; equal && r < top; ++r, equal &= equal - 1) {
      const int i = (int)e + __ffs(equal) - 1;
      sh.tv[r] = row.one(i), sh.ti[r] = i;
    }
    n += all;
    __syncthreads();
  }
}

// Writes a row's results from its sums (in sh.part[0]) and its top list.
template <int kThreads>
__device__ __forceinline__ void finish(Shared<kThreads>& sh, const Sums& s, float x_token, bool has_token, bool counted, int64_t row,
                                       int top, float* logprob, float* entropy, float* top_logprob,
                                       int32_t* top_token) {
  const bool empty = s.r == -INFINITY && s.z == 0.0f;
  const float lz = logf(s.z);  // lse = s.r + lz
  if (threadIdx.x == 0) {
    if (counted) logprob[row] = !has_token ? 0.0f : empty ? -INFINITY : (x_token - s.r) - lz;
    if (entropy) entropy[row] = empty ? 0.0f : lz - __fdiv_rn(s.b, s.z);
  }
  if ((int)threadIdx.x < top) {
    const float v = sh.tv[threadIdx.x];
    const int i = sh.ti[threadIdx.x];
    top_logprob[row * top + threadIdx.x] = empty ? -INFINITY : i == INT_MAX ? NAN : (v - s.r) - lz;
    top_token[row * top + threadIdx.x] = i == INT_MAX ? -1 : i;
  }
}

// Slice results in the workspace: r, z, b, then top values and tokens.
__host__ __device__ constexpr int slice_words(int top) { return 4 + 2 * top; }

template <bool BF16, int kThreads>
__global__ void __launch_bounds__(kThreads)
logprobs_kernel(const void* __restrict__ logits, int64_t stride, int64_t vocab, int64_t per, int splits,
                const int32_t* __restrict__ tokens, int top, float* logprob, float* entropy, float* top_logprob,
                int32_t* top_token, int* counters, float* slices) {
  kv::pdl_wait();
  using R = Row<BF16>;
  constexpr int kN = R::kN;
  constexpr int kWarps = kThreads / 32;
  __shared__ Shared<kThreads> sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.y;
  const int64_t from = min(vocab, blockIdx.x * per);
  const R x_row(static_cast<const uint8_t*>(logits) + row * stride * (BF16 ? 2 : 4), from, min(vocab, from + per));

  // ---- the pass ----
  float mx = -INFINITY;
  Sums s{-INFINITY, 0.0f, 0.0f};
  float2 z2 = make_float2(0.0f, 0.0f), b2 = make_float2(0.0f, 0.0f);  // s.z and s.b in two lanes
  float ref = 0.0f;  // s.r, or 0 while that is -inf
  auto rise = [&](float cm) {
    if (cm > s.r + kSlack) {
      s.z = z2.x + z2.y, s.b = b2.x + b2.y;
      s = s.r == -INFINITY ? Sums{cm, s.z, s.b} : shifted(s, cm);
      z2 = make_float2(s.z, 0.0f), b2 = make_float2(s.b, 0.0f);
      ref = cm;
    }
  };
  // elements that are not -inf (so the lowest value at least)
  auto add2 = [&](float x0, float x1) {
    const float2 d = __fadd2_rn(make_float2(x0, x1), make_float2(-ref, -ref));
    const float2 t = __fmul2_rn(d, make_float2(kLog2e, kLog2e));
    const float2 e = make_float2(ex2(t.x), ex2(t.y));
    z2 = __fadd2_rn(z2, e);
    b2 = __ffma2_rn(d, e, b2);
  };
  auto take = [&](const uint4& w) {
    if constexpr (BF16) {
      const uint32_t c[4] = {floor2(w.x), floor2(w.y), floor2(w.z), floor2(w.w)};
      const uint32_t m = max2(max2(w.x, w.y), max2(w.z, w.w));
      const float cm = fmaxf(kv::bf_lo(m), kv::bf_hi(m));
      mx = fmaxf(mx, cm);
      rise(cm);
#pragma unroll
      for (int j = 0; j < 4; ++j) add2(kv::bf_lo(c[j]), kv::bf_hi(c[j]));
    } else {
      float x[4];
      x_row.unpack(w, x);
      const float cm = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
      mx = fmaxf(mx, cm);
      rise(cm);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = x[j] == -INFINITY ? -3.402823466e38f : x[j];
      add2(x[0], x[1]);
      add2(x[2], x[3]);
    }
  };
  int i = x_row.a0 + tid;
  if (i + (kUnroll - 1) * kThreads < x_row.a1) {
    uint4 w[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) w[k] = x_row.vec(i + k * kThreads);
    for (;;) {  // the next vectors are on their way while these are added
      const int next = i + kUnroll * kThreads;
      const bool more = next + (kUnroll - 1) * kThreads < x_row.a1;
      uint4 n[kUnroll];
      if (more) {
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) n[k] = x_row.vec(next + k * kThreads);
      }
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) take(w[k]);
      i = next;
      if (!more) break;
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) w[k] = n[k];
    }
  }
  for (; i < x_row.a1; i += kThreads) take(x_row.vec(i));
  if (tid < 2 * kN) {
    const int e = x_row.loose(tid);
    if (e >= 0) {
      const float x = x_row.one(e);
      mx = fmaxf(mx, x);
      rise(x);
      const float d = x - ref, y = ex2(d * kLog2e);
      z2.x += y;
      b2.x = fmaf(fmaxf(d, -1e4f), y, b2.x);
    }
  }
  s.z = z2.x + z2.y, s.b = b2.x + b2.y;
  if (tid == 0) sh.count = 0;
  if (tid < kMaxTop) sh.tv[tid] = -INFINITY, sh.ti[tid] = INT_MAX;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const Sums t{__shfl_xor_sync(kFull, s.r, o), __shfl_xor_sync(kFull, s.z, o), __shfl_xor_sync(kFull, s.b, o)};
    s = joined(s, t);
  }
  if (lane == 0) sh.part[warp] = s;
  __syncthreads();

  // ---- the top list ----
  if (top > 0) {
    // the bound: the top-th largest of each warp's few largest lane maxima (64 in all)
    constexpr int kEach = Shared<kThreads>::kTops / kWarps;
    int key = key_of(mx);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int kth = __reduce_max_sync(kFull, key);
      const unsigned who = __ballot_sync(kFull, key == kth);
      if (lane == __ffs(who) - 1) key = INT_MIN;
      if (lane == j) sh.tops[warp * kEach + j] = of_key(kth);
    }
    __syncthreads();
    if (tid < Shared<kThreads>::kTops) {
      const float x = sh.tops[tid];
      int r = 0;
#pragma unroll 16
      for (int c = 0; c < Shared<kThreads>::kTops; ++c) r += better(sh.tops[c], c, x, tid);
      if (r == top - 1) sh.bound_f = x;
    }
    __syncthreads();
    const float bound = sh.bound_f;
    unsigned flagged = __ballot_sync(kFull, mx >= bound);
    volatile int* found = &sh.count;
    auto candidate = [&](float x, int e) {
      if (*found > kCap) return;
      const int at = atomicAdd(&sh.count, 1);
      if (at < kCap) sh.cv[at] = x, sh.ci[at] = e;
    };
    // a few vectors a thread, as slices have: each such lane looks at its own (the registers for that cost
    // whole rows 136 us against 114)
    const bool few = kThreads == kSliceThreads && x_row.a1 - x_row.a0 <= kFew * kThreads;
    if (few && mx >= bound) {
      uint4 v[kFew];
#pragma unroll
      for (int k = 0; k < kFew; ++k)
        if (x_row.a0 + tid + k * kThreads < x_row.a1) v[k] = x_row.vec(x_row.a0 + tid + k * kThreads);
#pragma unroll
      for (int k = 0; k < kFew; ++k) {
        const int a = x_row.a0 + tid + k * kThreads;
        if (a >= x_row.a1) break;
        float x[kN];
        x_row.unpack(v[k], x);
#pragma unroll
        for (int j = 0; j < kN; ++j)
          if (x[j] >= bound) candidate(x[j], a * kN - x_row.lead + j);
      }
    }
    while (flagged && *found <= kCap) {
      const int l = __ffs(flagged) - 1;
      flagged &= flagged - 1;
      for (int a = few ? x_row.a1 : x_row.a0 + (warp * 32 + l) + lane * kThreads; a < x_row.a1; a += 32 * kThreads) {
        float x[kN];
        x_row.unpack(x_row.vec(a), x);
#pragma unroll
        for (int j = 0; j < kN; ++j)
          if (x[j] >= bound) candidate(x[j], a * kN - x_row.lead + j);
      }
      if (warp == 0 && l < 2 * kN && lane == 0) {
        const int e = x_row.loose(l);
        if (e >= 0 && x_row.one(e) >= bound) candidate(x_row.one(e), e);
      }
    }
    __syncthreads();
    if (sh.count <= kCap) rank_candidates(sh, sh.count, top);
    else crowded<BF16, kThreads>(sh, x_row, bound, top);
    __syncthreads();
  }
  s = sh.part[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) s = joined(s, sh.part[w]);
  // A largest logit this far out, which the pass's shortcuts do not hold for: -inf, read there as the
  // type's lowest value, would weigh as much as that, and x - r may be -inf.  Rows whose every token
  // is masked come here, so the slice is summed once more, element by element.
  if (fabsf(s.r) >= kFar && fabsf(s.r) < INFINITY) {
    Sums t{s.r, 0.0f, 0.0f};
    for (int64_t i = (int64_t)x_row.e0 + tid; i < x_row.e1; i += kThreads) {
      const float d = x_row.one((int)i) - s.r;
      const float y = ex2(d * kLog2e);  // 0 for -inf, NaN for NaN
      t.z += y;
      if (y > 0.0f) t.b = fmaf(d, y, t.b);
    }
    __syncthreads();  // every thread has read the sums of before
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      t.z += __shfl_xor_sync(kFull, t.z, o);
      t.b += __shfl_xor_sync(kFull, t.b, o);
    }
    if (lane == 0) sh.part[warp] = t;
    __syncthreads();
    s = sh.part[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) s.z += sh.part[w].z, s.b += sh.part[w].b;
  }

  if (splits > 1) {
    float* mine = slices + (row * splits + blockIdx.x) * slice_words(top);
    if (tid == 0) __stcg(mine, s.r), __stcg(mine + 1, s.z), __stcg(mine + 2, s.b);
    if (tid < top) __stcg(mine + 4 + tid, sh.tv[tid]), __stcg(mine + 4 + top + tid, __int_as_float(sh.ti[tid]));
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      sh.last = atomicAdd(counters + row, 1) == splits - 1;
      if (sh.last) counters[row] = 0;
      sh.count = 0;
    }
    __syncthreads();
    if (!sh.last) return;
    __threadfence();
    const float* all = slices + row * splits * slice_words(top);
    // each warp joins the slices on its own, in the same order
    Sums t{-INFINITY, 0.0f, 0.0f};
    for (int k = lane; k < splits; k += 32) {
      const float* p = all + k * slice_words(top);
      t = joined(t, Sums{__ldcg(p), __ldcg(p + 1), __ldcg(p + 2)});
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const Sums c{__shfl_xor_sync(kFull, t.r, o), __shfl_xor_sync(kFull, t.z, o), __shfl_xor_sync(kFull, t.b, o)};
      t = joined(t, c);
    }
    s = t;
    if (top > 0) {
      // Where m slices hold an x or more at place j, m j elements reach x: so the m-th largest of the
      // slices' j-th bounds the row's last from below.  (The largest of their last ones leaves so many
      // that the ranking of 33 slices' 32 took 30 us.)
      const int j = (top + splits - 1) / splits, m = (top + j - 1) / j;
      for (int k = tid; k < splits; k += kThreads) sh.cv[k] = __ldcg(all + k * slice_words(top) + 4 + j - 1);
      if (tid < kMaxTop) sh.tv[tid] = -INFINITY, sh.ti[tid] = INT_MAX;
      __syncthreads();
      for (int k = tid; k < splits; k += kThreads) {
        const float x = sh.cv[k];
        int r = 0;
        for (int c = 0; c < splits; ++c) r += better(sh.cv[c], c, x, k);
        if (r == m - 1) sh.bound_f = x;
      }
      __syncthreads();
      const float bound = sh.bound_f;
      for (int a = tid; a < splits * top; a += kThreads) {
        const int k = a / top, j = a - k * top;
        const float* p = all + k * slice_words(top) + 4;
        const float x = __ldcg(p + j);
        const int e = __float_as_int(__ldcg(p + top + j));
        if (x >= bound && e != INT_MAX) {
          const int at = atomicAdd(&sh.count, 1);
          if (at < kCap) sh.cv[at] = x, sh.ci[at] = e;
        }
      }
      __syncthreads();
      if (sh.count <= kCap) {
        rank_candidates(sh, sh.count, top);
      } else if (warp == 0) {
        float lv = -INFINITY;
        int li = INT_MAX;
        for (int a = 0; a < splits * top; a += 32) {
          const int b = a + lane, k = b / top, j = b - k * top;
          const bool in = b < splits * top;
          const float* p = all + k * slice_words(top) + 4;
          const int e = in ? __float_as_int(__ldcg(p + top + j)) : INT_MAX;
          insert(in ? __ldcg(p + j) : 0.0f, e, in && e != INT_MAX, top, lane, lv, li);
        }
        if (lane < top) sh.tv[lane] = lv, sh.ti[lane] = li;
      }
      __syncthreads();
    }
  }
  const int tok = tokens ? __ldg(tokens + row) : -1;
  const bool has = tok >= 0 && tok < vocab;
  finish(sh, s, has ? x_row.one(tok) : 0.0f, has, tokens != nullptr, row, top, logprob, entropy, top_logprob, top_token);
}

// Slices a row: one where the rows alone fill the GPU; else enough for two CTAs an SM, of at
// least four vectors a thread pair (2048 elements).
int64_t splits_of(int64_t rows, int64_t vocab) {
  if (rows <= 0 || rows > kMaxSplitRows) return 1;
  int64_t n = 2 * (int64_t)sm_count() / rows;
  const int64_t most = vocab / 2048;
  if (n > most) n = most;
  if (n > kMaxSplits) n = kMaxSplits;
  return n < 1 ? 1 : n;
}

}  // namespace
}  // namespace lp

size_t logprobs_workspace(int64_t rows, int64_t vocab, int top) {
  const int64_t n = lp::splits_of(rows, vocab);
  if (n <= 1) return 0;
  return 4 * (size_t)lp::kMaxSplitRows + 4 * (size_t)(rows * n * lp::slice_words(top));
}

cudaError_t launch_logprobs(const void* logits, int64_t stride, bool bf16, int64_t rows, int64_t vocab,
                            const int32_t* tokens, int top, float* logprob, float* entropy, float* top_logprob,
                            int32_t* top_token, void* workspace, cudaStream_t st) {
  const int64_t splits = lp::splits_of(rows, vocab);
  const int64_t per = ((vocab + splits - 1) / splits + 7) / 8 * 8;
  int* counters = static_cast<int*>(workspace);
  float* slices = reinterpret_cast<float*>(counters + lp::kMaxSplitRows);
  // rows that fill the GPU by themselves: 512 threads a row (2047 rows of 128256 at 1965 MHz: 114 us,
  // with 256 threads 131, with 1024 194); slices, which are short: 256
  const int threads = splits > 1 ? lp::kSliceThreads : 512;
  auto kern = threads == 512 ? (bf16 ? lp::logprobs_kernel<true, 512> : lp::logprobs_kernel<false, 512>)
                             : (bf16 ? lp::logprobs_kernel<true, lp::kSliceThreads> : lp::logprobs_kernel<false, lp::kSliceThreads>);
  const int64_t elem = bf16 ? 2 : 4;
  for (int64_t r0 = 0; r0 < rows; r0 += 65535) {
    const int64_t n = rows - r0 < 65535 ? rows - r0 : 65535;
    cudaError_t e = kv::launch_behind(
        kern, dim3((unsigned)splits, (unsigned)n), threads, 0, st, static_cast<const uint8_t*>(logits) + r0 * stride * elem,
        stride, vocab, per, (int)splits, tokens ? tokens + r0 : nullptr, top, logprob ? logprob + r0 : nullptr,
        entropy ? entropy + r0 : nullptr, top_logprob ? top_logprob + r0 * top : nullptr,
        top_token ? top_token + r0 * top : nullptr, counters, slices);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace vbq
