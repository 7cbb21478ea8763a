// vbq_kv_attn.cu -- attention over the 8-bit paged cache, split over its tokens (decode).
//
//   out[row] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - max)
//
// with k_j = ks code, v_j = vs code, ks and vs one number a (page, head).  A decode step reads
// every code once and does 2 multiply-adds a code and query head, so the cache's bytes bound
// it as long as the arithmetic hides under the loads.  Both products run on the tensor cores
// with the codes on their 16-wide side, so a tile of 8 rows (a KV head's query heads, for each
// new token) wastes nothing at 8 heads a group.  The k (or m) positions of a fragment are assigned so that
// a thread's are 16-byte pieces of a cache row as it is stored.
//   S^T = K Q^T, integer m16n8k32: 16 tokens x 32 dims of codes as they are (A) times the rows
//     as fixed point in three base-256 digits (B), to 2^-22 of the row's largest value.  Sums
//     are exact.  (Two digits, 2^-14, would do for a bf16 output but put 1e-4 into the log sum,
//     which is fp32.)
//   O^T = V^T P^T, fp16 m16n8k16 with fp32 sums: 16 dims x 16 tokens of codes, exactly fp16
//     numbers, times the weights: rounded to fp16 for bf16 (11 bits, the output keeps 8), an
//     fp16 high part and the fp16 rest for fp32 (22 bits), each block's product then added to
//     the row's sum in fp32 (the tensor core's own accumulation truncates; over thousands of
//     blocks that alone came to 6e-6 of the result).
//
// Softmax: t = log2(e) scale ks (q.code) + e with vs = 2^e f, 1 <= f < 2; w = 2^(t - m + 6)
// and the weight is w f, in fp16's range whatever vs is; the sum takes w 2^-e.  The running
// maximum m moves only when some t exceeds it by 8 (w f < 2^15 then), which after the first
// blocks is rare.
//
// Work split: the (sequence, head, row tile) groups, each a run of chunks of 64 tokens, are
// laid end to end and cut into equal ranges, one a CTA of a resident grid.  A group that lies
// in one range is finished there; otherwise each CTA leaves its part (O, m, l) in the
// workspace and the last to arrive adds them up in range order, so the result does not depend
// on timing.
//
// Measured (device time of a launch among others): 64 sequences of up to 5003 tokens, 32 query heads
// over 8 of 128, bf16, 371 MB of codes: 87 us at 1807 MHz, where the power limit holds the SMs in a long
// row of calls, 80 at 1965; 4.3 and 4.6 TB/s.  4 of up to 131072, 64 over 8 heads, fp32, 762 MB: 173 us
// at 1635 MHz, 143 at 1965; 4.4 and 5.3 TB/s; at 1965 its copies alone, without the arithmetic, take
// 136.  One sequence of 333 tokens: 9.4 us.  What the shorter ones lack is the way to the first block
// (plan, page number, block: 4 to 8 us), the joining of parts (3 to 5 us), and CTAs of one SM that end up
// to a fifth apart; half of the issue slots are taken.  fp32 prompts and those with heads of 256 are this
// kernel's too, in tiles of 16 and 8 rows that each read and turn the codes again: four prompts of 1023
// tokens and less, 73 GFLOP, 785 us in fp32, 746 with heads of 256 in bf16.
#include <cmath>

#include "vbq_internal.h"
#include "vbq_kv.cuh"

namespace vbq {
namespace kv {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kBlockTokens = 16;                   // tokens a warp takes at a time: one page's
constexpr int kChunk = kBlockTokens * kWarps;      // tokens a chunk
constexpr int kMinChunks = 2;                      // a CTA's least share
constexpr float kShift = 6.0f, kSlack = 8.0f;      // w = 2^(t - m + kShift), m moves past kSlack
constexpr float kMagic = 12582912.0f;              // 1.5 2^23: as an integer accumulator's start, it ends as a float
constexpr int kMagicBits = 0x4b400000;
constexpr int kMaxGrid = kKvCounterBytes / 4;      // CTAs the workspace has room for

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// transpose of an 8 x 8 matrix of fp16 spread over the warp as MMA fragments are
__device__ __forceinline__ uint32_t transpose8(uint32_t w) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));
  return r;
}

// The chunks of a sequence's groups: those that hold a key any of its rows sees.
struct Span {
  int n, len, lo, c0, chunks, tiles;
};
__device__ __forceinline__ Span span_of(const KvBatch& b, const KvAttention& a, int s, int tile_rows) {
  Span v;
  v.n = seq_new(b, s), v.len = seq_len(b, s);
  if ((int64_t)v.n * a.group > a.rows_upto) v.n = 0;  // another kernel's
  v.lo = first_key(a, v.len - v.n);
  v.c0 = v.lo / kChunk;
  v.chunks = v.n > 0 ? max(1, (v.len + kChunk - 1) / kChunk - v.c0) : 0;
  v.tiles = (int)(((int64_t)v.n * a.group + tile_rows - 1) / tile_rows);
  return v;
}

template <int D, int NT> struct Part {  // one CTA's part of a group, in the workspace
  static constexpr int kRows = 8 * NT;
  static constexpr int kFloats = kRows * D + 2 * kRows;  // O, m, l
};

constexpr int kDigits = 3;
// Resident CTAs the registers are held to.  Three of dim 128 (166 registers) beat four (128): 142 us
// against 156 over 762 MB.
template <int D, int NT> constexpr int resident_of() { return D == 256 || NT > 1 && D == 128 ? 2 : NT > 1 || D == 128 ? 3 : kKvMaxResident; }

// Shared memory of a CTA: each warp's ring of blocks (16 tokens of K and V and the two scales),
// then the query digits and the warps' maxima and sums.  What the ring is for is loads in flight,
// about 190 KB an SM.  A block's K and its V are one run of bytes each in the pool and are copied
// as such, a warp's 512 bytes at a time (fetching each lane's fragment bytes directly, four rows
// to a quarter of a warp, held the loads alone to 5.1 of 7.0 TB/s); the 16-byte chunks of each
// 128 bytes are permuted on the way so that the fragments' reads meet no bank twice.
template <int D, int NT> struct Smem {
  static constexpr int kRows = 8 * NT;
  static constexpr int kK = kBlockTokens * D;      // bytes of a block's K, and of its V
  static constexpr int kStage = 2 * kK + 16;
  static constexpr int kQ = NT * kDigits * (D / 32) * 256;
  static constexpr int kFixed = kQ + 2 * kWarps * kRows * 4 + 16;
  static constexpr int kFit = (232448 / resident_of<D, NT>() - 1024 - kFixed) / (kWarps * kStage);
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kO = kWarps * kRows * (D + 4) * 4;  // the warps' O, over the ring
  static constexpr int kAlloc = (kRing > kO ? kRing : kO) + kFixed;
  static_assert(kStages >= 2, "ring");
};
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

template <int D, int NT, bool F32>
__global__ void __launch_bounds__(kThreads, resident_of<D, NT>())
attn_kernel(KvAttention a, KvCache c, KvBatch b, float* __restrict__ parts, int* __restrict__ counters) {
  if (a.rows_upto == INT64_MAX) pdl_wait();  // else the tile kernel has, which this one may run beside
  using S = Smem<D, NT>;
  constexpr int kRows = 8 * NT, kWords = D / 16, kParts = F32 ? 2 : 1;
  constexpr int kVec = D / 64;                    // 16-byte loads of a K row a thread makes
  constexpr int kVecV = D >= 128 ? D / 128 : 1;   // and of a V row (8 bytes at D = 64)
  extern __shared__ __align__(16) uint8_t smem[];
  float(*sh_o)[kRows][D + 4] = reinterpret_cast<float(*)[kRows][D + 4]>(smem);
  uint8_t* fixed = smem + (S::kRing > S::kO ? S::kRing : S::kO);
  // the tile's rows as fixed point: digit k of 4 dims a word, in fragment order (every warp's)
  uint32_t(*sh_q)[kDigits][kWords / 2][32][2] = reinterpret_cast<uint32_t(*)[kDigits][kWords / 2][32][2]>(fixed);
  float(*sh_m)[kRows] = reinterpret_cast<float(*)[kRows]>(fixed + S::kQ);
  float(*sh_l)[kRows] = sh_m + kWarps;
  int& sh_last = *reinterpret_cast<int*>(fixed + S::kQ + 2 * kWarps * kRows * 4);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, q4 = lane & 3;

  int longest = 0;  // chunks of this lane's longest group
  auto units = [&](int s) {
    const Span v = span_of(b, a, s, kRows);
    longest = max(longest, v.chunks);
    return (int64_t)v.chunks * v.tiles * c.heads;
  };
  // A CTA's least share: a part more costs the join about a quarter of what a chunk costs its CTA, so
  // n chunks cut into n / m parts of m take least time at m = sqrt(n) / 2 (one sequence of 21391 tokens,
  // 2 heads of 64, 12 rows: 48 us in parts of 2 chunks, 27 in parts of 9)
  auto least = [&]() {
    return (int64_t)max(kMinChunks, (int)sqrtf(0.25f * (float)(int)__reduce_max_sync(kFull, (unsigned)longest)));
  };
  int64_t total, per, u_begin;  // past `total` a CTA has no unit, and its loop no turn
  Unit unit;
  if (b.seqs <= 32) {  // one look at the sequences for both their sum and this CTA's place
    const int64_t mine = lane < b.seqs ? units(lane) : 0;
    const int64_t end = warp_scan(mine, lane);
    total = __shfl_sync(kFull, end, 31);
    per = max(quotient(total + gridDim.x - 1, gridDim.x), least());
    u_begin = blockIdx.x * per;
    const int at = __ffs(__ballot_sync(kFull, end > u_begin)) - 1;
    unit = {at, u_begin - __shfl_sync(kFull, end - mine, at)};
  } else {
    total = count_units(b.seqs, lane, units);
    per = max(quotient(total + gridDim.x - 1, gridDim.x), least());
    u_begin = blockIdx.x * per;
    unit = find_unit(u_begin, b.seqs, lane, units);
  }
  const int64_t u_end = min(total, u_begin + per);
  int64_t u = u_begin;

  while (u < u_end) {
    const int s = unit.s;
    const Span v = span_of(b, a, s, kRows);
    if (v.chunks == 0) {
      unit = {s + 1, 0};
      continue;
    }
    const int64_t gi = quotient(unit.at, v.chunks);  // group within the sequence: head, then tile
    const int head = (int)quotient(gi, v.tiles), tile = (int)(gi - (int64_t)head * v.tiles);
    const int ch0 = (int)(unit.at - gi * v.chunks);
    const int ch1 = (int)min((int64_t)v.chunks, ch0 + (u_end - u));
    const int64_t group_begin = u - ch0, group_end = group_begin + v.chunks;
    const int row_base = tile * kRows;  // flat row: new token * group + query head of the group
    const int64_t first_row = __ldg(b.q_start + s);

    // last and first key of this thread's columns; over the whole tile for the mask-free test
    int hi[NT][2], lo[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = (row_base + 8 * t + 2 * q4 + e) / a.group;
        hi[t][e] = i < v.n ? v.len - v.n + i : -1;
        lo[t][e] = first_key(a, hi[t][e]);
      }
    const int i0 = row_base / a.group, i1 = min(v.n - 1, (row_base + kRows - 1) / a.group);
    const int hi_min = v.len - v.n + i0;  // columns past the last row hold zeros and are never written
    const int hi_max = v.len - v.n + i1;
    const int lo_min = first_key(a, hi_min), lo_max = first_key(a, hi_max);

    // ---- blocks of 16 tokens: each warp a run of them ----
    const int first_tok = max((v.c0 + ch0) * kChunk, lo_min & ~(kBlockTokens - 1));
    const int last_tok = min((v.c0 + ch1) * kChunk, min(v.len, hi_max + 1));
    const int blocks = max(0, last_tok - first_tok + kBlockTokens - 1) / kBlockTokens;
    const int each = (blocks + kWarps - 1) / kWarps;
    const int tok_begin = first_tok + warp * each * kBlockTokens;
    const int tok_end = min(last_tok, tok_begin + each * kBlockTokens);
    const int64_t head_bytes = (int64_t)c.page * D;
    const int64_t v_off = c.heads * head_bytes;  // from K to V
    const int8_t* kp = nullptr;   // the next block to copy: K, this lane's first 16 bytes
    const float* sp = nullptr;    // its K scale
    bool there = false;
    // lane x holds the page of run run0 + x (and ahead: of run0 + 32 + x)
    const int run_end = (tok_end + c.page - 1) >> c.page_log2;
    auto pages_from = [&](int r) { return r + lane < run_end ? page_of(c, b, s, r + lane) : -1; };
    int run = -1, run0 = tok_begin >> c.page_log2;
    int pages = pages_from(run0), ahead = pages_from(run0 + 32);
    const uint32_t ring = smem_u32(smem) + warp * (S::kStages * S::kStage);
    // where this lane's chunk goes within 512 bytes: K with the chunk number's bit 2 flipped in odd
    // rows, V with twice half the token number (mod 8) flipped into it
    const uint32_t kd = D == 64 ? lane * 16 : (lane >> 3) * 128 + (((lane & 7) ^ (D == 128 ? (lane >> 3 & 1) * 4 : (lane >> 4) * 4)) << 4);
    const uint32_t vd0 = (lane >> 3) * 128 + (((lane & 7) ^ (D == 64 ? (lane >> 3) * 2 : D == 128 ? (lane >> 4) * 2 : 0)) << 4);
    auto copy = [&](int tok, uint32_t at) {
      if (tok < tok_end) {
        if ((tok >> c.page_log2) != run) {
          run = tok >> c.page_log2;
          if (run - run0 == 32) {
            run0 = run;
            pages = ahead;
            ahead = pages_from(run0 + 32);
          }
          const int page = __shfl_sync(kFull, pages, run - run0);
          there = page >= 0;
          const int64_t kb = block_index(c, max(page, 0), 0, head);  // no page: any codes will do
          kp = c.codes + kb * head_bytes + (tok & (c.page - 1)) * D + lane * 16;
          sp = c.scales + kb;
        }
#pragma unroll
        for (int e = 0; e < S::kK / 512; ++e) cp16(ring + at + kd + e * 512, kp + e * 512);
#pragma unroll
        for (int e = 0; e < S::kK / 512; ++e) {
          const uint32_t f = D == 64 ? 0 : D == 128 ? (e & 1) * 64 : (e & 3) * 32;
          cp16(ring + at + S::kK + (vd0 ^ f) + e * 512, kp + v_off + e * 512);
        }
        if (lane < 2) {
          if (there) cp4(ring + at + 2 * S::kK + lane * 4, sp + lane * c.heads);
          else asm volatile("st.shared.f32 [%0], %1;" ::"r"(ring + at + 2 * S::kK + lane * 4), "f"(lane ? -INFINITY : 0.0f) : "memory");
        }
        kp += kBlockTokens * D;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // this lane's fragment bytes in a block
    const uint32_t ka = D == 64 ? g * 64 + q4 * 16 : g * D + ((q4 ^ (g & 1) * 4) << 4);
    const uint32_t va = S::kK + (D == 64 ? q4 * 128 + (((g >> 1) ^ q4 * 2) << 4) + (g & 1) * 8 : 2 * q4 * D + ((g ^ q4 * 2) << 4));
    auto word = [](const uint4* r, int w) {
      const uint4& x = r[w >> 2];
      return (w & 3) == 0 ? x.x : (w & 3) == 1 ? x.y : (w & 3) == 2 ? x.z : x.w;
    };
    auto lds16 = [](uint32_t at) {
      uint4 v;
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
      return v;
    };
    auto lds4 = [](uint32_t at) {
      float v;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
      return v;
    };
#pragma unroll
    for (int i = 0; i < S::kStages; ++i) copy(tok_begin + i * kBlockTokens, i * S::kStage);
    // ---- the tile's query rows -> fragments, while the first blocks are on their way; each warp
    // takes a quarter of every row ----
    float qs[NT][2];  // columns 2 (lane % 4), + 1: log2(e) scale / 2^e
    constexpr int kMine = kWords / kWarps;
    float x[NT][kMine][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int fr = row_base + 8 * t + g;
      const int i = fr / a.group;
      const int64_t row = first_row + i;
      const bool live = i < v.n && row >= 0 && row < a.rows;
      const int64_t off = row * a.q_stride + (int64_t)(head * a.group + (fr - i * a.group)) * D + q4 * 16;
      uint32_t top = 0;  // of |x|, as bits: NaN is above infinity
#pragma unroll
      for (int y = 0; y < kMine; ++y) {
        const int w = warp * kMine + y;  // the word's 4 dims
        const int64_t at = off + (w >> 2) * 64 + (w & 3) * 4;
        if constexpr (F32) {
          const float4 z = live ? __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + at)) : make_float4(0, 0, 0, 0);
          x[t][y][0] = z.x, x[t][y][1] = z.y, x[t][y][2] = z.z, x[t][y][3] = z.w;
        } else {
          const uint2 z = live ? __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.q) + at)) : make_uint2(0, 0);
          x[t][y][0] = bf_lo(z.x), x[t][y][1] = bf_hi(z.x), x[t][y][2] = bf_lo(z.y), x[t][y][3] = bf_hi(z.y);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(x[t][y][e]) & 0x7fffffffu);
      }
      top = max(top, __shfl_xor_sync(kFull, top, 1));
      top = max(top, __shfl_xor_sync(kFull, top, 2));
      if (q4 == 0) sh_m[warp][8 * t + g] = __uint_as_float(top);
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      uint32_t top = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = max(top, __float_as_uint(sh_m[w][8 * t + g]));
      // power of two that takes the row's largest value to 2^21 .. 2^22
      const int ex = (int)(top >> 23);
      const int sh = min(max(127 + 21 - ex, -100), 120);
      const float up = __uint_as_float((uint32_t)(127 + sh) << 23);
      // a row with an infinity or NaN: every score NaN
      const float down = ex == 255 ? NAN : a.scale * __uint_as_float((uint32_t)(127 - sh) << 23);
      qs[t][0] = __shfl_sync(kFull, down, 8 * q4);       // of row 2 q4
      qs[t][1] = __shfl_sync(kFull, down, 8 * q4 + 4);   // of row 2 q4 + 1
#pragma unroll
      for (int y = 0; y < kMine; ++y) {
        uint32_t dg[kDigits] = {};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          int n = __float2int_rn(x[t][y][e] * up);
#pragma unroll
          for (int k = 0; k < kDigits; ++k) {
            dg[k] |= ((uint32_t)n & 0xffu) << (8 * e);
            n = (n - (int)(int8_t)n) >> 8;
          }
        }
        const int w = warp * kMine + y;
#pragma unroll
        for (int k = 0; k < kDigits; ++k) sh_q[t][k][w >> 1][lane][w & 1] = dg[k];
      }
    }
    __syncthreads();

    float o[NT][kWords][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int w = 0; w < kWords; ++w)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][w][e] = 0.0f;
#pragma unroll
      for (int e = 0; e < 2; ++e) m[t][e] = -INFINITY, l[t][e] = 0.0f;
    }

    uint32_t at = 0;
#pragma unroll 1
    for (int tok = tok_begin; tok < tok_end; tok += kBlockTokens) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 1) : "memory");
      __syncwarp();  // the other lanes' copies
      uint4 kr[2][kVec], vr[4][kVecV];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < kVec; ++e) kr[h][e] = lds16(ring + at + (ka ^ (e & 1) * 64) + h * 8 * D + (e >> 1) * 128);
      const float ksc = lds4(ring + at + 2 * S::kK), vs = lds4(ring + at + 2 * S::kK + 4);
      // S^T
      int si[NT][kDigits][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < kDigits; ++k) {
#pragma unroll
          for (int e = 0; e < 4; ++e) si[t][k][e] = kMagicBits;
#pragma unroll
          for (int w = 0; w < kWords; w += 2)
            mma16832(si[t][k], word(kr[0], w), word(kr[1], w), word(kr[0], w + 1), word(kr[1], w + 1),
                     sh_q[t][k][w >> 1][lane][0], sh_q[t][k][w >> 1][lane][1]);
        }
      // vs = 2^e f, at least 1e-30 (values below 1.3e-28 are taken as up to that)
      const uint32_t vb = __float_as_uint(value_scale(vs));
      const float vec = vs == -INFINITY ? -INFINITY : (float)((int)(vb >> 23) - 127);  // no page: no weight
      const float vfc = __uint_as_float((vb & 0x7fffffu) | 0x3f800000u);
      const float vdc = __uint_as_float((254u << 23) - (vb & 0x7f800000u));
      const bool mask = tok + kBlockTokens - 1 > hi_min || tok < lo_max;
      uint32_t pb[NT][kParts][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float sc = __int_as_float(si[t][kDigits - 1][e]) - kMagic;
#pragma unroll
          for (int k = kDigits - 2; k >= 0; --k) sc = fmaf(sc, 256.0f, __int_as_float(si[t][k][e]) - kMagic);
          x[e] = fmaf(sc, qs[t][e & 1] * ksc, vec);
          if (mask) {
            const int j = tok + g + 8 * (e >> 1);
            if (j > hi[t][e & 1] || j < lo[t][e & 1]) x[e] = -INFINITY;
          }
        }
        const bool up = x[0] > m[t][0] + kSlack || x[2] > m[t][0] + kSlack || x[1] > m[t][1] + kSlack ||
                        x[3] > m[t][1] + kSlack;
        if (__any_sync(kFull, up)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(x[e], x[e + 2]);
            mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 16));
            mx = fmaxf(mx, m[t][e]);
            const float al = mx == -INFINITY ? 1.0f : ex2(m[t][e] - mx);
            m[t][e] = mx;
            l[t][e] *= al;
#pragma unroll
            for (int w = 0; w < kWords; ++w) o[t][w][e] *= al, o[t][w][e + 2] *= al;
          }
        }
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float mm = m[t][e & 1];
          w[e] = ex2(x[e] - (mm == -INFINITY ? 0.0f : mm - kShift));
          l[t][e & 1] = fmaf(w[e], vdc, l[t][e & 1]);
          w[e] *= vfc;
        }
        const uint32_t h0 = h2(w[0], w[1]), h1 = h2(w[2], w[3]);
        pb[t][0][0] = transpose8(h0);
        pb[t][0][1] = transpose8(h1);
        if constexpr (F32) {
          const float2 r0 = h2f(h0), r1 = h2f(h1);
          pb[t][1][0] = transpose8(h2(w[0] - r0.x, w[1] - r0.y));
          pb[t][1][1] = transpose8(h2(w[2] - r1.x, w[3] - r1.y));
        }
      }
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        if constexpr (D == 64) {
          asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(vr[h][0].x), "=r"(vr[h][0].y)
                       : "r"(ring + at + (va ^ (h & 1) * 64) + (h >> 1) * 512) : "memory");
        } else {
#pragma unroll
          for (int e = 0; e < kVecV; ++e) vr[h][e] = lds16(ring + at + va + ((h & 1) + 8 * (h >> 1)) * D + e * 128);
        }
      }
      // O^T: a word of V holds 4 dims; dims 4 w + 2 i (row g) and + 1 (row g + 8) of MMA 2 w + i
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        const uint32_t t0 = word(vr[0], w) ^ 0x80808080u, t1 = word(vr[1], w) ^ 0x80808080u;
        const uint32_t t2 = word(vr[2], w) ^ 0x80808080u, t3 = word(vr[3], w) ^ 0x80808080u;
        const uint32_t x01 = __byte_perm(t0, t1, 0x5140), y01 = __byte_perm(t0, t1, 0x7362);
        const uint32_t x23 = __byte_perm(t2, t3, 0x5140), y23 = __byte_perm(t2, t3, 0x7362);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t p = i ? y01 : x01, r = i ? y23 : x23;
          const uint32_t a0 = sub1152(__byte_perm(p, 0x64646464u, 0x4140));
          const uint32_t a1 = sub1152(__byte_perm(p, 0x64646464u, 0x4342));
          const uint32_t a2 = sub1152(__byte_perm(r, 0x64646464u, 0x4140));
          const uint32_t a3 = sub1152(__byte_perm(r, 0x64646464u, 0x4342));
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if constexpr (F32) {
              float y[4];
              mma16816_zero(y, a0, a1, a2, a3, pb[t][1][0], pb[t][1][1]);
              mma16816(y, a0, a1, a2, a3, pb[t][0][0], pb[t][0][1]);
#pragma unroll
              for (int e = 0; e < 4; ++e) o[t][2 * w + i][e] += y[e];
            } else {
              mma16816(o[t][2 * w + i], a0, a1, a2, a3, pb[t][0][0], pb[t][0][1]);
            }
          }
        }
      }
      __syncwarp();  // every lane has read the block: its place is free
      copy(tok + S::kStages * kBlockTokens, at);
      at = at + S::kStage == S::kStages * S::kStage ? 0 : at + S::kStage;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // the warps' O goes over the rings

    // ---- the warps' parts add up in shared memory ----
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float y = l[t][e];
        y += __shfl_xor_sync(kFull, y, 4);
        y += __shfl_xor_sync(kFull, y, 8);
        y += __shfl_xor_sync(kFull, y, 16);
        if (g == 0) {
          sh_l[warp][8 * t + 2 * q4 + e] = y;
          sh_m[warp][8 * t + 2 * q4 + e] = m[t][e];
        }
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          // row g of MMA w is this dim, row g + 8 the next
          float2 d = make_float2(o[t][w][e], o[t][w][e + 2]);
          *reinterpret_cast<float2*>(&sh_o[warp][8 * t + 2 * q4 + e][D == 64 ? g * 8 + 2 * w : (w >> 3) * 128 + g * 16 + 2 * (w & 7)]) = d;
        }
      }
    }
    __syncthreads();
    const bool whole = ch0 == 0 && ch1 == v.chunks;
    float* part = parts + ((int64_t)blockIdx.x * 2 + (group_begin < u_begin ? 0 : 1)) * Part<D, NT>::kFloats;
    auto finish = [&](int r, int d, float4 y, float mm, float ll) {
      const int fr = row_base + r, i = fr / a.group;
      const int64_t row = first_row + i;
      if (i >= v.n || row < 0 || row >= a.rows) return;
      const int qh = head * a.group + (fr - i * a.group);
      const float inv = ll == 0.0f ? 0.0f : __fdiv_rn(1.0f, ll);
      y.x *= inv, y.y *= inv, y.z *= inv, y.w *= inv;
      const int64_t off = row * a.out_stride + (int64_t)qh * D + d;
      if constexpr (F32) *reinterpret_cast<float4*>(static_cast<float*>(a.out) + off) = y;
      else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + off) = make_uint2(pack_bf16(y.x, y.y), pack_bf16(y.z, y.w));
      if (a.lse && d == 0)
        a.lse[row * ((int64_t)c.heads * a.group) + qh] = ll == 0.0f ? -INFINITY : (mm - kShift + log2f(ll)) * kLn2;
    };
    for (int x = tid; x < kRows * (D / 4); x += kThreads) {
      const int r = x / (D / 4), d = (x - r * (D / 4)) * 4;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sh_m[w][r]);
      float4 y = make_float4(0, 0, 0, 0);
      float ll = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float al = mm == -INFINITY ? 1.0f : ex2(sh_m[w][r] - mm);
        const float4 z = *reinterpret_cast<const float4*>(&sh_o[w][r][d]);
        y.x = fmaf(z.x, al, y.x), y.y = fmaf(z.y, al, y.y), y.z = fmaf(z.z, al, y.z), y.w = fmaf(z.w, al, y.w);
        ll = fmaf(sh_l[w][r], al, ll);
      }
      if (whole) {
        finish(r, d, y, mm, ll);
      } else {
        __stcg(reinterpret_cast<float4*>(part + r * D + d), y);
        if (d == 0) {
          __stcg(part + kRows * D + r, mm);
          __stcg(part + kRows * D + kRows + r, ll);
        }
      }
    }
    if (!whole) {
      // the group's CTAs are b0 .. b1; the last to arrive adds up their parts
      const int64_t b0 = quotient(group_begin, per), b1 = quotient(group_end - 1, per);
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const int before = atomicAdd(counters + b0, 1);
        sh_last = before == (int)(b1 - b0);
        if (sh_last) counters[b0] = 0;
      }
      __syncthreads();
      if (sh_last) {
        __threadfence();
        // each row's parts: their common maximum and sum, and each part's factor (over the ring);
        // then the parts of O, whose loads depend on nothing
        const int n = (int)(b1 - b0) + 1;
        auto part_of = [&](int k) {
          return parts + ((b0 + k) * 2 + (group_begin < (b0 + k) * per ? 0 : 1)) * Part<D, NT>::kFloats;
        };
        float* fac = reinterpret_cast<float*>(smem);
        constexpr int kAtOnce = S::kRing / (4 * kRows);      // factors the ring has room for, a row
        constexpr int kLanes = kThreads / kRows;             // threads a row: 16 or 8, within a warp
        constexpr int kEach = kRows * D / 4 / kThreads;      // float4 of O a thread
        const int r = tid / kLanes, rl = tid % kLanes;
        float mm = -INFINITY, ll = 0.0f;
        for (int k = rl; k < n; k += kLanes) mm = fmaxf(mm, __ldcg(part_of(k) + kRows * D + r));
#pragma unroll
        for (int o2 = kLanes / 2; o2; o2 >>= 1) mm = fmaxf(mm, __shfl_xor_sync(kFull, mm, o2));
        const float ref = mm == -INFINITY ? 0.0f : mm;
        float4 y[kEach];
#pragma unroll
        for (int x = 0; x < kEach; ++x) y[x] = make_float4(0, 0, 0, 0);
        for (int k0 = 0; k0 < n; k0 += kAtOnce) {
          const int k1 = min(n, k0 + kAtOnce);
          for (int k = k0 + rl; k < k1; k += kLanes) {
            const float* p = part_of(k) + kRows * D;
            const float f = ex2(__ldcg(p + r) - ref);
            fac[(k - k0) * kRows + r] = f;
            ll = fmaf(__ldcg(p + kRows + r), f, ll);
          }
          __syncthreads();
          constexpr int kBatch = 8 / kEach > 0 ? 8 / kEach : 1;  // parts whose loads are made together
#pragma unroll 1
          for (int k = k0; k < k1; k += kBatch) {
            float4 z[kBatch][kEach];
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
#pragma unroll
              for (int x = 0; x < kEach; ++x)
                if (k + i < k1) z[i][x] = __ldcg(reinterpret_cast<const float4*>(part_of(k + i)) + tid + x * kThreads);
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
#pragma unroll
              for (int x = 0; x < kEach; ++x)
                if (k + i < k1) {
                  const float f = fac[(k + i - k0) * kRows + (tid + x * kThreads) / (D / 4)];
                  y[x].x = fmaf(z[i][x].x, f, y[x].x), y[x].y = fmaf(z[i][x].y, f, y[x].y);
                  y[x].z = fmaf(z[i][x].z, f, y[x].z), y[x].w = fmaf(z[i][x].w, f, y[x].w);
                }
          }
          __syncthreads();
        }
#pragma unroll
        for (int o2 = kLanes / 2; o2; o2 >>= 1) ll += __shfl_xor_sync(kFull, ll, o2);
        if (rl == 0) sh_m[0][r] = mm, sh_l[0][r] = ll;
        __syncthreads();
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
          const int at = tid + x * kThreads, row = at / (D / 4), d = (at - row * (D / 4)) * 4;
          finish(row, d, y[x], sh_m[0][row], sh_l[0][row]);
        }
      }
    }
    __syncthreads();  // shared memory is free for the next group
    u += ch1 - ch0;
    unit.at += ch1 - ch0;
    if (unit.at == (int64_t)v.chunks * v.tiles * c.heads) unit = {s + 1, 0};
  }
  if (__ldg(b.q_start) > 0 || __ldg(b.q_start + b.seqs) < a.rows) blank_rows<F32>(a, c, b);
  // Started under the tile kernel, this one needs nothing of it; but the call has ended only when both have.
  pdl_wait();
}

template <int D, int NT, bool F32>
cudaError_t launch(const KvAttention& a, const KvCache& c, const KvBatch& b, void* ws, cudaStream_t st) {
  auto kern = attn_kernel<D, NT, F32>;
  constexpr int smem = Smem<D, NT>::kAlloc;
  static DeviceOnce configured;
  static DeviceSlots resident;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!configured.done(dev)) {
    int n = 0;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, kThreads, smem);
    if (e != cudaSuccess) return e;
    resident.set(dev, n);
    configured.mark(dev);
  }
  int64_t grid = (int64_t)sm_count() * resident.get(dev);
  if (grid > kMaxGrid) grid = kMaxGrid;
  int* counters = static_cast<int*>(ws);
  float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + kKvHeadBytes);
  return launch_behind(kern, (unsigned)grid, kThreads, smem, st, a, c, b, parts, counters);
}

template <int D, bool F32>
cudaError_t pick(const KvAttention& a, const KvCache& c, const KvBatch& b, int max_new, void* ws, cudaStream_t st) {
  const int64_t rows = (int64_t)(max_new > 0 ? max_new : a.rows) * a.group;
  if (rows <= 8) return launch<D, 1, F32>(a, c, b, ws, st);
  // 16 rows of 256 do not fit the registers; 32 of 64 took 28.3 us where 16 take 25.4 (36 to 63 rows
  // a head, windows of 2050 tokens)
  return launch<D, D == 256 ? 1 : 2, F32>(a, c, b, ws, st);
}

}  // namespace
}  // namespace kv

// Counters of this kernel and of the tile kernel, parts of this one, then of the other: the two run
// at the same time.
size_t kv_attn_tile_parts(int dim) { return kKvHeadBytes + sizeof(float) * 2 * (size_t)kv::kMaxGrid * (16 * dim + 32); }
// One workspace serves both types of activations.
size_t kv_attn_workspace(int dim) {
  return kv_attn_tile_parts(dim) + (kv_prefill_takes(dim, true) ? kv_prefill_parts_bytes(dim) : 0);
}

// Rows (new tokens times query heads a KV head) of a sequence above which it takes the tcgen05
// kernel, whose tiles are 256 rows whatever there is in them.  16 sequences of 7001 tokens, 8 heads
// of 128: 36 rows 76 us here and 95 there, 68 rows 117 and 91, 132 rows 196 and 91; 4 heads of 64 in a
// window of 2050: 119 rows 35 and 36, 231 rows 53 and 43; 8 of 38000, one head of 64: 119 rows 48 and
// 68, 231 rows 76 and 69; 16 of 7001, 4 heads of 64 in a window of 2050, 161 rows 42 and 53.  With few rows in all the tiles do not fill the GPU: one sequence of 3000
// tokens, 8 heads of 128: 132 rows 30 us here and 35 there.  (All at 1965 MHz.)
static int64_t tile_rows_from(int dim, int64_t rows) { return dim == 64 ? 192 : rows <= 2048 ? 144 : 64; }

cudaError_t launch_kv_attn(const KvAttention& a0, const KvCache& c, const KvBatch& b, bool bf16, int max_new,
                           void* ws, cudaStream_t st) {
  KvAttention a = a0;
  a.rows_above = -1, a.rows_upto = INT64_MAX;
  const int64_t most = (int64_t)(max_new > 0 ? max_new : a.rows) * a.group;
  const int64_t from = tile_rows_from(c.dim, a.rows * a.group * c.heads);
  if (kv_prefill_takes(c.dim, bf16) && a.rows * a.group > from && (most > from || max_new == 0)) {
    a.rows_above = a.rows_upto = from;
    // One sequence is the tile kernel's whatever rows q_start gives it, which may be fewer than the tensor has.
    if (b.seqs == 1) a.rows_above = -1;
    cudaError_t e = launch_kv_prefill(a, c, b, ws, st);
    if (e != cudaSuccess || b.seqs == 1) return e;
  }
  switch (c.dim) {
    case 64: return bf16 ? kv::pick<64, false>(a, c, b, max_new, ws, st) : kv::pick<64, true>(a, c, b, max_new, ws, st);
    case 128: return bf16 ? kv::pick<128, false>(a, c, b, max_new, ws, st) : kv::pick<128, true>(a, c, b, max_new, ws, st);
    case 256: return bf16 ? kv::pick<256, false>(a, c, b, max_new, ws, st) : kv::pick<256, true>(a, c, b, max_new, ws, st);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace vbq
