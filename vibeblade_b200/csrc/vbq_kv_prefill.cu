// vbq_kv_prefill.cu -- attention of prompt chunks over the 8-bit paged cache, on tcgen05.
//
// The same sums as vbq_kv_attn.cu (log2 weights t = log2(e) scale ks (q.code) + log2(vs), a
// lazily moved reference, codes exact in fp16), for sequences with many new tokens.  A KV
// head's query rows are packed (new token, query head of the group) and cut into tiles of
// 256; a CTA takes two 128-row halves of one tile against 128 cached tokens at a time:
//     S = Q K^T   tcgen05 128 x 128 x dim per half, accumulators in tensor memory
//     P = 2^(t - m), fp16, written over S in tensor memory
//     O += P V    tcgen05 128 x dim x 128, A from tensor memory
// What bounds it: per 128 x 128 tile of S the two products are 4 dim 128 128 flops (1024 cycles
// of the tensor cores at dim 128) against 16384 exponentials (1024 cycles of the SM's MUFU), so
// one half's products run under the other half's softmax.
//
// Warps: 0-3 and 4-7 softmax of the two halves (a thread owns a row); 8-11 turn codes into
// fp16 tiles (global -> registers -> 128-byte-swizzled shared memory, two stages each of K and
// V); 12 issues the MMAs; 13 hands out the work; 14 fetches the scales; 15 brings the next tile's
// queries into L2 (34 prompts of up to 930 tokens: 250 us without, 233 with).  K is the K-major B
// operand of the first product; V, in the same shared-memory layout, the MN-major one of the second.
// Registers are moved from the last two groups to the softmax warps (setmaxnreg), whose threads hold a whole row of S.
//
// Work split as in vbq_kv_attn.cu: all tiles' runs of 128 tokens, laid end to end, cut into
// equal ranges, one a CTA; a tile that spans CTAs is added up, in range order, by the last.
//
// Rounding: codes and products are exact in fp16 and fp32; a query row is scaled by a power of
// two into fp16's range, which keeps all of bf16's digits down to 2^-29 of its largest value (and
// more coarsely 2^-39); weights are rounded to fp16's 11 bits, where the output keeps 8.  The sum of
// exponentials is compensated; O is the tensor core's own fp32 sum, which truncates: rows of equal weights
// come out 0.08 % low over 41000 tokens, 0.16 % over 524288, 0.37 % over a million (a bf16 step is 0.4 %).
//
// Measured (device time of a launch among others, 8 heads of 128): the last 2048 of 32768 tokens of 64
// query heads, 2.13 TFLOP: 2.38 ms at 1627 MHz, where the power limit holds the SMs in a row of calls,
// 0.90 PFLOP/s; a call by itself 2.07 ms, 1.03; four prompts of 1023 tokens and less, 32 query heads, 73
// GFLOP: 112 us at 1965 MHz, 0.65 PFLOP/s.  A run of 128 tokens takes some 4200 cycles where its MMAs
// need 2120 and the exponentials 2048 of the MUFU: a half's softmax is a chain of 3000 (load of S 300,
// largest 300, 64 exponentials 900, P out 250, 64 more 900, P out), after which its second product
// and next scores take 1050, and the halves hide only part of each other.  A tile costs 10000 to
// 15000 cycles more: its queries, the first tiles of K and V, its rows out.  Tried: two threads a row
// (16 softmax warps), 2.36 ms against 2.04; the weights taken before the largest is known, 2.04
// against 2.01; scores in two products of 64 tokens, the first early, 2.15 (an MMA of 64 columns
// takes as long as one of 128); a quarter of the exponentials as polynomials, 2.29.
//
// Every mbarrier wait is bounded in time: the schedule's warp waits for each piece's end by the clock, and
// where it gives up raises the device status word and an abort flag at which every wait returns at once
// and no MMA is issued, so the roles run out of their (finite) schedules, what was issued is waited for,
// and tensor memory is freed.
#include <cmath>

#include "vbq_internal.h"
#include "vbq_kv.cuh"

namespace vbq {

__device__ unsigned g_kv_prefill_status = 0;

namespace kv {
namespace {

constexpr int kTileRows = 256, kHalf = 128, kTok = 128;
constexpr int kPThreads = 512;
constexpr int kScaleRing = 4;
constexpr int kKept = 512;       // sequences whose runs are kept in shared memory
constexpr float kTiny = 1e-30f;  // a block's score factor is at least this: -inf times it is -inf

struct PBars {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t q_full, s_full[2], p_half[2], p_full[2], o_full[2];  // p_half: the first 64 columns of P
  uint64_t scale_full[kScaleRing], scale_empty[kScaleRing];
  uint64_t seg_full[2], seg_empty[2];
  uint64_t part_a, part_b;
  uint64_t drain;  // after an abort: what was issued has ended
  int64_t runs[16];  // of each warp's sequences
  int longest[16];
  uint32_t tmem;
  int abort;
  int first;  // every other part of the tile is there
  int last;
};
// A piece of the CTA's work: runs c0 .. c1 - 1 of the tile's, the tile's first run being `first`.
struct PSeg {
  int s, head, tile, c0, c1, first, n, len;
  int row0;        // q_start of the sequence
  int whole;       // the tile lies in this piece
  int slot;        // else: this CTA's part, and the CTAs b0 .. b1 of the tile
  int b0, b1;
  int stop;        // no piece: the CTA is done
};
// Per 16 tokens of a K / V tile: ks, log2(vs), 1 / vs
struct PScale {
  float ks, lv, iv, pad;
};

template <int D> struct PSmem {
  static constexpr int kTile = kTok * D * 2;        // a 128 x D fp16 tile
  static constexpr int kV = 0;                      // two stages
  static constexpr int kK = kV + 2 * kTile;         // two stages
  static constexpr int kQ = kK + 2 * kTile;         // two halves
  static constexpr int kScale = kQ + 2 * kTile;
  static constexpr int kSeg = kScale + kScaleRing * (kTok / 16) * (int)sizeof(PScale);
  static constexpr int kBar = kSeg + 2 * 64;
  static constexpr int kRuns = kBar + (int)(sizeof(PBars) + 15) / 16 * 16;
  static constexpr int kAlloc = kRuns + kKept * 8 + 1024;
  static_assert(sizeof(PSeg) <= 64 && kAlloc <= 232448, "shared memory per CTA");
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// ---- tcgen05 (one CTA) -----------------------------------------------------------------
// Rows of 128 bytes in 128-byte-swizzled groups of 8 (1024 bytes).  K-major: the next 8 rows
// SBO = 1024 away, LBO unused.  MN-major (V): rows are the K index, the next 8 of them SBO =
// 1024 away, the next 64 columns LBO = one column half away.
// The descriptor's high word is the same for both: SBO, version 1, 128-byte swizzle (2); the
// low word holds the address and LBO, in 16-byte units.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t p_desc(uint32_t saddr, uint32_t lbo) { return ((saddr >> 4) & 0x3fffu) | ((lbo >> 4) << 16); }
// fp32 accumulators, fp16 operands, M = 128
constexpr uint32_t p_idesc(int n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// The whole warp calls these and one lane (`lead`) issues: the operands are then computed once,
// in uniform registers, where an instruction issued under a one-lane branch moves each of them
// there first (the two products of a run took 2000 cycles to issue that way, and 1060 to execute).
__device__ __forceinline__ void p_mma_ss(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHi), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void p_mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 y, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHi), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void p_commit(uint32_t lead, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      ::"r"(bar), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void p_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void p_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void p_ld32(uint32_t taddr, float* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
        "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
        "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
        "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(taddr));
}
// names the registers that the load fills, so that no use of them moves above it
__device__ __forceinline__ void p_wait_ld32(float* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
                 "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15])
               :: "memory");
  asm volatile("" : "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]),
                    "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31]));
}
__device__ __forceinline__ void p_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
__device__ __forceinline__ void p_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};"
               ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void p_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void p_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// volatile: a tile's loads stay together ahead of their uses
__device__ __forceinline__ uint4 ld_q(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// ---- schedule --------------------------------------------------------------------------
// A sequence's rows for this kernel, its tiles, and the 128-token runs a tile looks at.
struct PSeq {
  int n, len, tiles;
};
__device__ __forceinline__ PSeq p_seq(const KvBatch& b, const KvAttention& a, int s) {
  PSeq q;
  q.n = seq_new(b, s), q.len = seq_len(b, s);
  const int64_t rows = (int64_t)q.n * a.group;
  q.tiles = rows > a.rows_above ? (int)((rows + kTileRows - 1) / kTileRows) : 0;
  return q;
}
struct PRun {
  int first, count;  // in runs of 128 tokens
};
__device__ __forceinline__ PRun p_run(const PSeq& q, const KvAttention& a, int tile) {
  const int i0 = (int)quotient((int64_t)tile * kTileRows, a.group);
  const int i1 = min(q.n - 1, (int)quotient((int64_t)tile * kTileRows + kTileRows - 1, a.group));
  const int hi = q.len - q.n + i1;
  const int first = first_key(a, q.len - q.n + i0) / kTok;
  return {first, max(1, hi / kTok + 1 - first)};  // hi < 0: one run, all of it masked
}
// Runs of a sequence over all its tiles, and of its longest; the whole warp.
__device__ __forceinline__ int64_t p_seq_runs(const PSeq& q, const KvAttention& a, int lane, int& longest) {
  int64_t n = 0;
  int most = 0;
  for (int t = lane; t < q.tiles; t += 32) {
    const int c = p_run(q, a, t).count;
    n += c;
    most = max(most, c);
  }
  longest = max(longest, (int)__reduce_max_sync(kFull, (unsigned)most));
#pragma unroll
  for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(kFull, n, o);
  return n;
}

// Walks the CTA's range of units (a unit is a run of 128 tokens of a (sequence, head, tile));
// one warp does, and hands the pieces to the others.
struct PWalk {
  int64_t u, end, per, group_begin;
  int s, head, tile, c0, c1;  // the present piece: runs c0 .. c1 - 1 of the tile's
  PSeq q;
  PRun run;

  // runs: the first kKept sequences' numbers of runs
  __device__ __forceinline__ void init(const KvBatch& b, const KvAttention& a, int heads, int lane, const int64_t* runs,
                                       int64_t total, int longest) {
    total *= heads;
    per = quotient(total + gridDim.x - 1, gridDim.x);
    whole_upto = per < kWholeFew ? kWholeFew : kWhole;
    per = max(per, (int64_t)(longest > whole_upto ? kMinRuns : 1));
    u = blockIdx.x * per;
    end = min(total, u + per);
    if (u >= end) return;
    int64_t before = 0;
    const int kept = min(b.seqs, kKept);
    for (s = 0; s < kept; s += 32) {
      const int64_t mine = s + lane < kept ? runs[s + lane] * heads : 0;
      int64_t to = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(kFull, to, o);
        if (lane >= o) to += x;
      }
      const unsigned past = __ballot_sync(kFull, before + to > u);
      if (past) {
        const int l = __ffs(past) - 1;
        s += l;
        before += __shfl_sync(kFull, to - mine, l);
        break;
      }
      before += __shfl_sync(kFull, to, 31);
    }
    s = min(s, kept);
    for (; s < b.seqs; ++s) {
      q = p_seq(b, a, s);
      const int64_t each = s < kKept ? runs[s] : p_seq_runs(q, a, lane, longest), all = each * heads;
      if (before + all <= u) {
        before += all;
        continue;
      }
      head = (int)quotient(u - before, each);
      int64_t at = u - before - head * each;
      // the longest tiles first: tile numbers go down
      for (int t0 = q.tiles - 1; t0 >= 0; t0 -= 32) {
        const int mine = t0 - lane >= 0 ? p_run(q, a, t0 - lane).count : 0;
        const int to = warp_scan(mine, lane);
        const unsigned past = __ballot_sync(kFull, to > at);
        if (past) {
          const int l = __ffs(past) - 1;
          tile = t0 - l;
          at -= __shfl_sync(kFull, to - mine, l);
          break;
        }
        at -= __shfl_sync(kFull, to, 31);
      }
      run = p_run(q, a, tile);
      if (run.count <= whole_upto && at > 0) {  // the rest of a short tile is the CTA before's
        c0 = (int)at, c1 = run.count;
        next(b, a, heads, runs);
      } else {
        set((int)at);
      }
      return;
    }
  }
  __device__ __forceinline__ bool more() const { return u < end; }
  __device__ __forceinline__ void next(const KvBatch& b, const KvAttention& a, int heads, const int64_t* runs) {
    u += c1 - c0;
    if (u >= end) return;
    if (--tile < 0) {
      if (++head == heads) {
        head = 0;
        do {
          do ++s;
          while (s < kKept && runs[s] == 0);
          q = p_seq(b, a, s);
        } while (q.tiles == 0);
      }
      tile = q.tiles - 1;
    }
    run = p_run(q, a, tile);
    set(0);
  }
  // The piece from run `from` of the present tile, which unit u is.
  __device__ __forceinline__ void set(int from) {
    c0 = from;
    group_begin = u - c0;
    c1 = run.count <= whole_upto ? run.count : (int)min((int64_t)run.count, c0 + (end - u));
  }
  __device__ __forceinline__ bool whole() const { return c0 == 0 && c1 == run.count; }
  // Adding up a tile's parts takes as long as several runs.  So a tile of few runs stays whole, with the
  // CTA that its first run belongs to; one of twice as many too where CTAs have less to do than that; and
  // where longer tiles are split a CTA takes kMinRuns at least.  (16 sequences, 4 heads of 64 in windows
  // of 2050 tokens, 119 rows each: 57 us with 16, 8 and 8 for the three, 36 so; 16 of up to 1138 tokens,
  // 4 heads of 128, 763 rows: 45 us, with 8 for tiles where CTAs have little 53.)
  static constexpr int kWholeFew = 12, kWhole = 6, kMinRuns = 4;
  int whole_upto;
};

// SM clock cycles after which the watch gives up, 1.5 s at 1.965 GHz (of the clock's low word, which comes
// round every 2^32 and is looked at far more often), for every 2^14 runs a CTA's pieces may have.
constexpr uint32_t kWatchCycles = 3000000000u;

template <int D> constexpr int p_part_floats() { return kTileRows * (D + 2); }  // O [D / 4][256][4], m, l

template <int D>
__global__ void __launch_bounds__(kPThreads, 1)
prefill_kernel(KvAttention a, KvCache c, KvBatch b, float* __restrict__ parts, int* __restrict__ counters) {
  pdl_wait();
  using L = PSmem<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  PBars& bars = *reinterpret_cast<PBars*>(smem + L::kBar);
  PScale* ring = reinterpret_cast<PScale*>(smem + L::kScale);
  struct alignas(64) SegSlot : PSeg {};
  SegSlot* segs = reinterpret_cast<SegSlot*>(smem + L::kSeg);
  int64_t* runs = reinterpret_cast<int64_t*>(smem + L::kRuns);
  const int tid = threadIdx.x, warp = __shfl_sync(kFull, tid >> 5, 0), lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars.k_full[i]), 4);
      mbar_init(smem_u32(&bars.v_full[i]), 4);
      mbar_init(smem_u32(&bars.k_empty[i]), 1);
      mbar_init(smem_u32(&bars.v_empty[i]), 1);
      mbar_init(smem_u32(&bars.s_full[i]), 1);
      mbar_init(smem_u32(&bars.p_half[i]), 4);
      mbar_init(smem_u32(&bars.p_full[i]), 4);
      mbar_init(smem_u32(&bars.o_full[i]), 1);
    }
    for (int i = 0; i < kScaleRing; ++i) {
      mbar_init(smem_u32(&bars.scale_full[i]), 1);
      mbar_init(smem_u32(&bars.scale_empty[i]), 8);
    }
    mbar_init(smem_u32(&bars.q_full), 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars.seg_full[i]), 1);
      mbar_init(smem_u32(&bars.seg_empty[i]), 15);  // all warps but the schedule's
    }
    mbar_init(smem_u32(&bars.part_a), 8);
    mbar_init(smem_u32(&bars.part_b), 1);
    mbar_init(smem_u32(&bars.drain), 1);
    bars.abort = 0;
    mbar_fence_init();
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&bars.tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // the kernel for the sequences of few rows may use the SMs that this one leaves free
  if (b.seqs > 1) pdl_release();
  else if (__ldg(b.q_start) > 0 || __ldg(b.q_start + 1) < a.rows) blank_rows<false>(a, c, b);
  // the runs of every sequence, a warp a sequence (by the schedule's warp alone, one after the other,
  // 45 sequences took 60 us)
  {
    int64_t sum = 0;
    int longest = 0;
    constexpr int kW = kPThreads / 32;
    for (int s0 = warp; s0 < b.seqs; s0 += 32 * kW) {  // lane x holds sequence s0 + kW x
      PSeq q = {0, 0, 0};
      if (s0 + kW * lane < b.seqs) q = p_seq(b, a, s0 + kW * lane);
      for (int x = 0; x < 32 && s0 + kW * x < b.seqs; ++x) {
        const PSeq y = {__shfl_sync(kFull, q.n, x), __shfl_sync(kFull, q.len, x), __shfl_sync(kFull, q.tiles, x)};
        const int64_t n = p_seq_runs(y, a, lane, longest);
        if (lane == 0 && s0 + kW * x < kKept) runs[s0 + kW * x] = n;
        sum += n;
      }
    }
    if (lane == 0) bars.runs[warp] = sum, bars.longest[warp] = longest;
  }
  p_fence_before();
  __syncthreads();
  p_fence_after();
  const uint32_t tmem = __shfl_sync(kFull, bars.tmem, 0);
  volatile int* abort_flag = &bars.abort;
  // A wait ends with the abort flag too, which the schedule's warp raises: whatever stalls, a piece does not
  // end, and that warp waits for each piece's end by the clock.  (These waits are many and their code is
  // short for the instruction cache: with a clock in each, short prompts took 122 us instead of 111.)
  auto wait = [&](uint64_t& bar, uint32_t parity) {
    const uint32_t addr = smem_u32(&bar);
#pragma unroll 1
    while (!mbar_try_wait(addr, parity) && !*abort_flag) {
    }
  };
  // the next piece, for a role that has done k pieces; false when there is none
  auto piece = [&](uint32_t k) {
    wait(bars.seg_full[k & 1], (k >> 1) & 1);
    return !__any_sync(kFull, *abort_flag || segs[k & 1].stop);
  };
  auto piece_done = [&](uint32_t k) {
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&bars.seg_empty[k & 1]));
  };
  constexpr int kORow = 256;  // tensor memory: S0 0..127, S1 128..255, O0 256.., O1 256 + D..

  if (warp < 8) {
    // ------------------------------ softmax ------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    const int half = warp >> 2;
    const int r = (warp & 3) * 32 + lane;                 // row of the half
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + half * kTok, to = tmem + lanes + kORow + half * D;
    uint8_t* q_tile = smem + L::kQ + half * L::kTile;
    auto chunk = [&](int y, int e) {  // 16 bytes of the tile's row y
      return reinterpret_cast<uint4*>(q_tile + (e >> 3) * (kHalf * 128) + y * 128 + (((e & 7) ^ (y & 7)) << 4));
    };
    // a warp's 32 rows, kRowsAt at a time, kE lanes a row
    constexpr int kE = D / 8, kRowsAt = 32 / kE;
    auto staged = [&](int e) { return chunk((warp & 3) * 32 + e * kRowsAt + lane / kE, lane % kE); };
    uint32_t s_phase = 0, o_phase = 0, a_phase = 0, b_phase = 0, count = 0;  // count: K / V tiles so far, for the ring
    for (uint32_t k = 0; piece(k); ++k) {
      const PSeg& g = segs[k & 1];
      // this thread's query row -> fp16, scaled by a power of two to 2^14 .. 2^15 at most
      const int fr = g.tile * kTileRows + half * kHalf + r;
      const int i = fr / a.group;
      const bool live = i < g.n;
      const int row = g.row0 + i;
      const int qh = g.head * a.group + (fr - i * a.group);
      const bool inside = live && row >= 0 && row < a.rows;
      // (kE lanes side by side take a row: a lane a row reads 32 lines at a time)
      float qs;
      {
        const int64_t off = inside ? (int64_t)row * a.q_stride + (int64_t)qh * D : -1;
        uint4 x[kE];
        uint32_t there = 0;
#pragma unroll
        for (int e = 0; e < kE; ++e) {  // where there is no row the first one's: every load is on its way at once
          const int64_t o = __shfl_sync(kFull, off, e * kRowsAt + lane / kE);
          there |= (uint32_t)(o >= 0) << e;
          x[e] = ld_q(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + max(o, (int64_t)0)) + lane % kE);
        }
        uint32_t top[kE];  // of each row, over its lanes; the steps of all rows side by side
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const uint32_t keep = 0u - (there >> e & 1);
          x[e] = make_uint4(x[e].x & keep, x[e].y & keep, x[e].z & keep, x[e].w & keep);
          const uint32_t v[4] = {x[e].x, x[e].y, x[e].z, x[e].w};
          top[e] = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) top[e] = max(top[e], max((v[k] << 16) & 0x7fffffffu, v[k] & 0x7fff0000u));
        }
#pragma unroll
        for (int o = kE / 2; o; o >>= 1) {
#pragma unroll
          for (int e = 0; e < kE; ++e) top[e] = max(top[e], __shfl_xor_sync(kFull, top[e], o));
        }
        auto shift = [](uint32_t top) {
          const int ex = (int)(top >> 23);
          return (ex == 0 || ex == 255) ? 0 : min(max(127 + 14 - ex, -100), 100);
        };
        uint32_t mine = 0;
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const uint32_t got = __shfl_sync(kFull, top[e], (lane % kRowsAt) * kE);
          if (lane / kRowsAt == e) mine = got;
        }
        const int sh = shift(mine);
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const uint32_t v[4] = {x[e].x, x[e].y, x[e].z, x[e].w};
          // (a negative scale negates the row: score factors are not negative; an infinity or NaN in the
          // row makes all of it NaN, as scores of -inf alone would pass for masked ones)
          const float up = top[e] >= 0x7f800000u ? NAN : copysignf(__uint_as_float((uint32_t)(127 + shift(top[e])) << 23), a.scale);
          uint32_t h[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) h[k] = h2(bf_lo(v[k]) * up, bf_hi(v[k]) * up);
          *staged(e) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        qs = fabsf(a.scale) * __uint_as_float((uint32_t)(127 - sh) << 23);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bars.q_full));

      // rows past the last hold zeros, are not written, and need no mask
      const int hi = live ? g.len - g.n + i : 0x3fffffff;
      const int lo = live ? first_key(a, hi) : 0;
      float mm = 0.0f, l = 0.0f, rest = 0.0f;  // rest: what l's roundings left out
      bool seen = false;
      const int c0 = g.c0, c1 = g.c1, first = g.first;
      for (int j = c0; j < c1; ++j, ++count) {
        wait(bars.s_full[half], s_phase);
        s_phase ^= 1;
        p_fence_after();
        float t[kTok];
        p_ld32(ts, t);
        wait(bars.scale_full[count % kScaleRing], (count / kScaleRing) & 1);
        const PScale* sc = ring + (count % kScaleRing) * (kTok / 16);
        const int rel_hi = hi - (first + j) * kTok, rel_lo = lo - (first + j) * kTok;
        const bool mask = __any_sync(kFull, rel_hi < kTok - 1 || rel_lo > 0);
        // A block of 16 columns has t = c s + lv - mm with one c > 0, so its largest t is its
        // largest s's; each 32 columns are looked at while the next are on their way.
        float mx = -INFINITY;
#pragma unroll
        for (int h = 0; h < kTok / 32; ++h) {
          p_wait_ld32(t + 32 * h);
          if (h + 1 < kTok / 32) p_ld32(ts + 32 * (h + 1), t + 32 * (h + 1));
          if (mask) {
#pragma unroll
            for (int x = 32 * h; x < 32 * h + 32; ++x) t[x] = (x > rel_hi || x < rel_lo) ? -INFINITY : t[x];
          }
#pragma unroll
          for (int x = 2 * h; x < 2 * h + 2; ++x) {
            float m = max3(t[16 * x], t[16 * x + 1], t[16 * x + 2]), n = max3(t[16 * x + 3], t[16 * x + 4], t[16 * x + 5]);
#pragma unroll
            for (int y = 6; y < 14; y += 4) {
              m = max3(m, t[16 * x + y], t[16 * x + y + 1]);
              n = max3(n, t[16 * x + y + 2], t[16 * x + y + 3]);
            }
            m = max3(m, t[16 * x + 14], t[16 * x + 15]);
            mx = fmaxf(mx, fmaf(fmaxf(m, n), fmaxf(qs * sc[x].ks, kTiny), sc[x].lv - mm));
          }
        }
        // the reference moves when a weight would pass 2^15, and at the row's first token
        const bool move = mx > 15.0f || (!seen && mx > -INFINITY);
        if (__any_sync(kFull, move)) {
          const float d = move ? mx - 7.0f : 0.0f;
          const float f = move && seen ? ex2(-d) : 1.0f;
          mm += d;
          l *= f;
          rest *= f;
          seen = seen || move;
          if (j > c0) {  // S of this run is there, so P V of the one before is done
#pragma unroll 1
            for (int x = 0; x < D / 8; ++x) {
              uint32_t o[8];
              p_ld8(to + 8 * x, o);
              asm volatile("tcgen05.wait::ld.sync.aligned;"
                           : "+r"(o[0]), "+r"(o[1]), "+r"(o[2]), "+r"(o[3]), "+r"(o[4]), "+r"(o[5]), "+r"(o[6]), "+r"(o[7])
                           :: "memory");
#pragma unroll
              for (int y = 0; y < 8; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
              p_st8(to + 8 * x, o);
            }
          }
        }
        float of_run = 0.0f;  // added up by itself first, as its roundings go one way where scores are equal
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          uint32_t pk[16];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const PScale p = sc[2 * h + x];
            const float m1 = fmaxf(qs * p.ks, kTiny), m0 = p.lv - mm;
            float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int y = 0; y < 16; y += 2) {
              const int e = 32 * h + 16 * x + y;
              float2 v = __ffma2_rn(make_float2(t[e], t[e + 1]), make_float2(m1, m1), make_float2(m0, m0));
              v = make_float2(ex2(v.x), ex2(v.y));
              sum = __fadd2_rn(sum, v);
              pk[8 * x + y / 2] = h2(v.x, v.y);
            }
            of_run = fmaf(sum.x + sum.y, p.iv, of_run);
          }
          p_st16(ts + 16 * h, pk);
          if (h == 1) {  // the second product may begin on these
            p_wait_st();
            p_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars.p_half[half]));
          }
        }
        {  // l + rest, to l's own rounding and no more over any number of runs
          const float add = of_run + rest, to_l = l + add;
          rest = add - (to_l - l);
          l = to_l;
        }
        p_wait_st();
        p_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&bars.p_full[half]));
          mbar_arrive(smem_u32(&bars.scale_empty[count % kScaleRing]));
        }
      }

      // ---- the tile's rows out, or this CTA's part of them ----
      const int b0 = g.b0, b1 = g.b1;
      if (!g.whole && tid == 0) {
        bars.first = !*abort_flag && *(volatile int*)(counters + b0) == b1 - b0;
        if (bars.first) counters[b0] = 0;
        mbar_arrive(smem_u32(&bars.part_b));
      }
      __syncwarp();
      wait(bars.o_full[half], o_phase);
      o_phase ^= 1;
      p_fence_after();
      const bool ok = !*abort_flag;
      bool done = g.whole;  // the rows' results are in the place of their queries, which nobody reads any more
      if (g.whole) {
        const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
          float o[32];
          p_ld32(to + 32 * x, o);
          p_wait_ld32(o);
#pragma unroll
          for (int y = 0; y < 4; ++y)
            *chunk(r, 4 * x + y) =
                make_uint4(pack_bf16(o[8 * y] * inv, o[8 * y + 1] * inv), pack_bf16(o[8 * y + 2] * inv, o[8 * y + 3] * inv),
                           pack_bf16(o[8 * y + 4] * inv, o[8 * y + 5] * inv), pack_bf16(o[8 * y + 6] * inv, o[8 * y + 7] * inv));
        }
        if (a.lse && inside && ok)
          a.lse[(int64_t)row * (c.heads * a.group) + qh] = l == 0.0f ? -INFINITY : (mm + log2f(l)) * kLn2;
      } else {
        const int tr = half * kHalf + r;  // row of the tile
        // The last of the tile's CTAs to arrive adds up the parts, in the order of their runs.  It is
        // mostly the one of the tile's beginning, which it does last, long after the others did theirs:
        // then its own part stays where it is.
        wait(bars.part_b, b_phase);
        b_phase ^= 1;
        const bool first = bars.first;
        bool last = first;
        if (!first) {
          float* part = parts + ((int64_t)blockIdx.x * 2 + g.slot) * p_part_floats<D>();
#pragma unroll
          for (int x = 0; x < D / 32; ++x) {
            float o[32];
            p_ld32(to + 32 * x, o);
            p_wait_ld32(o);
#pragma unroll
            for (int y = 0; y < 8; ++y)
              if (live)
                __stcg(reinterpret_cast<float4*>(part) + (8 * x + y) * kTileRows + tr,
                       make_float4(o[4 * y], o[4 * y + 1], o[4 * y + 2], o[4 * y + 3]));
          }
          __stcg(part + kTileRows * D + tr, seen ? mm : -INFINITY);
          __stcg(part + kTileRows * (D + 1) + tr, l);
          __threadfence();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bars.part_a));
          if (tid == 0) {
            wait(bars.part_a, a_phase);
            bars.last = !*abort_flag && atomicAdd(counters + b0, 1) == b1 - b0;
            if (bars.last) counters[b0] = 0;
            mbar_arrive(smem_u32(&bars.part_b));
          }
          __syncwarp();
          wait(bars.part_b, b_phase);
          a_phase ^= 1, b_phase ^= 1;
          last = bars.last;
        }
        if (last) {
          done = true;
          __threadfence();
          // the first CTA holds the tile's beginning as its last piece (slot 1), the others its
          // continuation as their first (slot 0)
          auto at = [&](int n) { return parts + ((int64_t)n * 2 + (n == b0 ? 1 : 0)) * p_part_floats<D>(); };
          const int own = first ? (int)blockIdx.x : -1;
          auto max_of = [&](int n) { return n == own ? (seen ? mm : -INFINITY) : __ldcg(at(n) + kTileRows * D + tr); };
          float top = -INFINITY, sum = 0.0f;
          for (int n = b0; n <= b1; ++n) top = fmaxf(top, max_of(n));
          const float ref = top == -INFINITY ? 0.0f : top;
          for (int n = b0; n <= b1; ++n)
            sum = fmaf(n == own ? l : __ldcg(at(n) + kTileRows * (D + 1) + tr), ex2(max_of(n) - ref), sum);
          const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
#pragma unroll 1
          for (int x = 0; x < (__any_sync(kFull, live) ? D : 0); x += 64) {  // rows past the last have no parts
            float y[64], z[64];
#pragma unroll
            for (int e = 0; e < 64; ++e) y[e] = 0.0f;
#pragma unroll 1
            for (int n = b0; n <= b1; ++n) {
              const float w = ex2(max_of(n) - ref);
              if (n == own) {
                p_ld32(to + x, z);
                p_ld32(to + x + 32, z + 32);
                p_wait_ld32(z);
                p_wait_ld32(z + 32);
              } else {
                const float4* p = reinterpret_cast<const float4*>(at(n)) + (x / 4) * kTileRows + tr;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                  *reinterpret_cast<float4*>(z + 4 * e) = live ? __ldcg(p + e * kTileRows) : make_float4(0, 0, 0, 0);
              }
#pragma unroll
              for (int e = 0; e < 64; ++e) y[e] = fmaf(z[e], w, y[e]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *chunk(r, x / 8 + e) =
                  make_uint4(pack_bf16(y[8 * e] * inv, y[8 * e + 1] * inv), pack_bf16(y[8 * e + 2] * inv, y[8 * e + 3] * inv),
                             pack_bf16(y[8 * e + 4] * inv, y[8 * e + 5] * inv), pack_bf16(y[8 * e + 6] * inv, y[8 * e + 7] * inv));
          }
          if (a.lse && inside && ok)
            a.lse[(int64_t)row * (c.heads * a.group) + qh] = sum == 0.0f ? -INFINITY : (ref + log2f(sum)) * kLn2;
        }
      }
      if (done) {
        const int64_t off = inside && ok ? (int64_t)row * a.out_stride + (int64_t)qh * D : -1;
        __syncwarp();
        uint4 y[kE];
#pragma unroll
        for (int e = 0; e < kE; ++e) y[e] = *staged(e);
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const int64_t o = __shfl_sync(kFull, off, e * kRowsAt + lane / kE);
          if (o >= 0) reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + o)[lane % kE] = y[e];
        }
        __syncwarp();
      }
      p_fence_before();  // O read before the next tile's first product writes it (ordered by p_full)
      piece_done(k);
    }
  } else if (warp < 12) {
    // ------------------------------ codes -> fp16 tiles ------------------------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    constexpr int kPerRow = D / 16;                      // threads (16 codes each) a token
    constexpr int kRowsStep = 128 / kPerRow, kSteps = kTok / kRowsStep;
    // A warp takes 4 (8 at dim 64) tokens a step.  Eight threads that store together write two
    // tokens' chunks of one column half: tokens r and r + 1 sit in opposite parities of the
    // swizzled 16-byte columns, so the eight cover all of them.
    const int wq = warp - 8;
    const int c16 = D == 128 ? (lane >> 3 & 1) * 4 + (lane & 3) : lane & 3;
    const int r0 = D == 128 ? 4 * wq + 2 * (lane >> 4) + (lane >> 2 & 1) : 8 * wq + (lane >> 2);
    uint32_t count = 0;
    uint4 x[kSteps];  // the next tile's codes, each loaded as soon as its register is stored
    const int64_t page_stride = (int64_t)c.layers * 2 * c.heads * c.page * D;
    const int64_t head_bytes = (int64_t)c.page * D;
    // lane y (mod 8) finds tokens 16 y .. 16 y + 15 of a run; where there are none any block's
    // codes will do (their weights are zero: no key, or no page and log2(vs) = -inf)
    auto blocks = [&](int s, int k0, int len) {
      const int tok = k0 + 16 * (lane & 7);
      const int page = tok < len ? page_of(c, b, s, tok >> c.page_log2) : -1;
      return page >= 0 ? page * page_stride + (tok & (c.page - 1)) * D : (int64_t)0;
    };
    auto load = [&](int i, const int8_t* base, int64_t at) {
      const int r = i * kRowsStep + r0;
      x[i] = ld_stream(base + __shfl_sync(kFull, at, r >> 4) + (r & 15) * D);
    };
    for (uint32_t k = 0; piece(k); ++k) {
      const PSeg& g = segs[k & 1];
      const int n = g.c1 - g.c0, s = g.s, len = g.len;
      int k0 = (g.first + g.c0) * kTok;
      const int8_t* kp = c.codes + ((int64_t)c.layer * 2 * c.heads + g.head) * head_bytes + c16 * 16;
      const int8_t* vp = kp + c.heads * head_bytes;
      int64_t at = blocks(s, k0, len), next = 0;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) load(i, kp, at);
      // K and V of a run in turn: step 2 j + which
#pragma unroll 1
      for (int step = 0; step < 2 * n; ++step) {
        const int st = count & 1, which = step & 1;
        const uint32_t parity = ((count >> 1) & 1) ^ 1;
        if (!which) next = step + 2 < 2 * n ? blocks(s, k0 + kTok, len) : at;
        wait(which ? bars.v_empty[st] : bars.k_empty[st], parity);
        uint8_t* tile = smem + (which ? L::kV : L::kK) + st * L::kTile + (c16 >> 2) * (kTok * 128) + r0 * 128;
        const int8_t* from = which ? kp : vp;
        const int64_t to = which ? next : at;
        // token r0 + i kRowsStep: the same swizzle at every step
        uint8_t* d0 = tile + ((((c16 & 3) * 2) ^ (r0 & 7)) << 4);
        uint8_t* d1 = tile + ((((c16 & 3) * 2 + 1) ^ (r0 & 7)) << 4);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const uint32_t v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
          uint32_t h[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) codes_h2(v[e], h[2 * e], h[2 * e + 1]);
          *reinterpret_cast<uint4*>(d0 + i * (kRowsStep * 128)) = make_uint4(h[0], h[1], h[2], h[3]);
          *reinterpret_cast<uint4*>(d1 + i * (kRowsStep * 128)) = make_uint4(h[4], h[5], h[6], h[7]);
          load(i, from, to);  // after the piece's last run: not used
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(which ? &bars.v_full[st] : &bars.k_full[st]));
        if (which) {
          ++count;
          at = next;
          k0 += kTok;
        }
      }
      piece_done(k);
    }
  } else {
    // ------------------------------ MMA issue ------------------------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 12) {
      constexpr uint32_t kIdS = p_idesc(kTok, false), kIdO = p_idesc(D, true);
      const uint32_t lead = lane == 0, base = smem_u32(smem);
      uint32_t count = 0, q_phase = 0, p_phase = 0;
      auto scores = [&](int half, int st) {
        const uint32_t q = p_desc(base + L::kQ + half * L::kTile, 16), k = p_desc(base + L::kK + st * L::kTile, 16);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * (kTok * 128) + (kk & 3) * 32) >> 4;
          p_mma_ss(lead, tmem + half * kTok, q + off, k + off, kIdS, kk > 0);
        }
        p_commit(lead, smem_u32(&bars.s_full[half]));
      };
      auto values = [&](int half, int st, int from, bool acc) {  // 64 tokens from 16 `from`
        const uint32_t v = p_desc(base + L::kV + st * L::kTile, kTok * 128) + from * (2048 >> 4);
#pragma unroll
        for (int kk = 0; kk < kTok / 32; ++kk)
          p_mma_ts(lead, tmem + kORow + half * D, tmem + half * kTok + 8 * (from + kk), v + kk * (2048 >> 4), kIdO, acc || kk > 0);
      };
      auto aborted = [&]() { return __any_sync(kFull, *abort_flag); };
      for (uint32_t k = 0; piece(k); ++k) {
        const int n = __shfl_sync(kFull, segs[k & 1].c1 - segs[k & 1].c0, 0);
        wait(bars.q_full, q_phase);
        q_phase ^= 1;
        wait(bars.k_full[count & 1], (count >> 1) & 1);
        p_fence_after();
        if (!aborted()) {
          scores(0, count & 1);
          scores(1, count & 1);
          p_commit(lead, smem_u32(&bars.k_empty[count & 1]));
        }
#pragma unroll 1
        for (int j = 0; j < n; ++j, ++count) {
          const int st = count & 1, nx = st ^ 1;
          const bool more = j + 1 < n;
          if (more) wait(bars.k_full[nx], ((count + 1) >> 1) & 1);
          wait(bars.v_full[st], (count >> 1) & 1);
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            wait(bars.p_half[half], p_phase);
            p_fence_after();
            if (!aborted()) values(half, st, 0, j > 0);
            wait(bars.p_full[half], p_phase);
            p_fence_after();
            if (aborted()) continue;
            values(half, st, kTok / 32, true);
            if (more) scores(half, nx);
            else p_commit(lead, smem_u32(&bars.o_full[half]));
          }
          p_phase ^= 1;
          if (!aborted()) {
            p_commit(lead, smem_u32(&bars.v_empty[st]));
            if (more) p_commit(lead, smem_u32(&bars.k_empty[nx]));
          }
        }
        piece_done(k);
      }
      // What was issued has ended, and its commits have arrived, before tensor memory is freed and the CTA
      // leaves: after an abort through a commit of its own.  Nobody watches any more: these go by the clock.
      bool ended = true;
      if (aborted()) {
        p_commit(lead, smem_u32(&bars.drain));
        ended = mbar_wait_bounded(smem_u32(&bars.drain), 0, kWaitBudgetCycles);
      } else if (count > 0) {
        for (uint32_t k = count > 2 ? count - 2 : 0; k < count; ++k) {
          ended = mbar_wait_bounded(smem_u32(&bars.k_empty[k & 1]), (k >> 1) & 1, kWaitBudgetCycles) && ended;
          ended = mbar_wait_bounded(smem_u32(&bars.v_empty[k & 1]), (k >> 1) & 1, kWaitBudgetCycles) && ended;
        }
      }
      if (!ended) g_kv_prefill_status = kStatusTimeout;
    } else if (warp == 14) {
      // ------------------------------ scales ------------------------------
      uint32_t count = 0;
      for (uint32_t k = 0; piece(k); ++k) {
        const PSeg& g = segs[k & 1];
        const int n = g.c1 - g.c0, s = g.s, len = g.len;
        const float* base = c.scales + (int64_t)c.layer * 2 * c.heads + g.head;
        int tok = (g.first + g.c0) * kTok + 16 * (lane & 7);
        for (int j = 0; j < n; ++j, ++count, tok += kTok) {
          PScale p{0.0f, -INFINITY, 0.0f, 0.0f};
          const int page = tok < len ? page_of(c, b, s, tok >> c.page_log2) : -1;
          if (page >= 0) {
            const float* q = base + (int64_t)page * c.layers * 2 * c.heads;
            const float v = value_scale(__ldg(q + c.heads));
            p = {__ldg(q), log2f(v), __fdiv_rn(1.0f, v), 0.0f};
          }
          wait(bars.scale_empty[count % kScaleRing], ((count / kScaleRing) & 1) ^ 1);
          if (lane < kTok / 16) ring[(count % kScaleRing) * (kTok / 16) + lane] = p;
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bars.scale_full[count % kScaleRing]));
        }
        piece_done(k);
      }
    } else if (warp == 15) {
      // ------------------------------ the next tile's queries into L2 ------------------------------
      for (uint32_t k = 0; piece(k); ++k) {
        const PSeg& g = segs[k & 1];
        for (int y = lane; y < kTileRows; y += 32) {
          const int fr = g.tile * kTileRows + y, i = fr / a.group, row = g.row0 + i;
          if (i < g.n && row >= 0 && row < a.rows) {
            const uint16_t* p = static_cast<const uint16_t*>(a.q) + (int64_t)row * a.q_stride + (int64_t)(g.head * a.group + fr - i * a.group) * D;
#pragma unroll
            for (int e = 0; e < D; e += 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(p + e));
          }
        }
        piece_done(k);
      }
    } else if (warp == 13) {
      // ------------------------------ schedule ------------------------------
      PWalk w;
      int64_t total = 0;
      int longest = 0;
      for (int i = 0; i < kPThreads / 32; ++i) total += bars.runs[i], longest = max(longest, bars.longest[i]);
      w.init(b, a, c.heads, lane, runs, total, longest);
      // waits for a piece's end; false, and the whole CTA is given up, where that does not come
      auto watch = [&](uint64_t& bar, uint32_t parity) {
        const uint32_t addr = smem_u32(&bar);
        int64_t times = 1 + (w.per >> 14);
        uint32_t since = clock();
#pragma unroll 1
        while (!mbar_try_wait(addr, parity) && !*abort_flag) {
          if ((uint32_t)clock() - since <= kWatchCycles) continue;
          since = clock();
          if (--times > 0) continue;
          *abort_flag = 1;
          g_kv_prefill_status = kStatusTimeout;
        }
        return !__any_sync(kFull, *abort_flag);
      };
      uint32_t k = 0;
      for (; w.more() && watch(bars.seg_empty[k & 1], ((k >> 1) & 1) ^ 1); w.next(b, a, c.heads, runs), ++k) {
        if (lane == 0) {
          PSeg g;
          g.s = w.s, g.head = w.head, g.tile = w.tile, g.c0 = w.c0, g.c1 = w.c1, g.first = w.run.first;
          g.n = w.q.n, g.len = w.q.len, g.row0 = __ldg(b.q_start + w.s), g.whole = w.whole();
          g.slot = w.group_begin < blockIdx.x * w.per ? 0 : 1;
          g.b0 = (int)quotient(w.group_begin, w.per), g.b1 = (int)quotient(w.group_begin + w.run.count - 1, w.per);
          g.stop = 0;
          static_cast<PSeg&>(segs[k & 1]) = g;
          mbar_arrive(smem_u32(&bars.seg_full[k & 1]));
        }
        __syncwarp();
      }
      watch(bars.seg_empty[k & 1], ((k >> 1) & 1) ^ 1);
      if (lane == 0) {
        segs[k & 1].stop = 1;
        mbar_arrive(smem_u32(&bars.seg_full[k & 1]));
      }
      if (k > 0) watch(bars.seg_empty[(k - 1) & 1], ((k - 1) >> 1) & 1);  // the last piece's
    }
  }
  p_fence_before();
  __syncthreads();
  if (warp == 12) {
    p_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

template <int D>
cudaError_t launch_prefill(const KvAttention& a, const KvCache& c, const KvBatch& b, void* ws, cudaStream_t st) {
  auto kern = prefill_kernel<D>;
  static DeviceOnce configured;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!configured.done(dev)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, PSmem<D>::kAlloc);
    if (e != cudaSuccess) return e;
    configured.mark(dev);
  }
  int* counters = reinterpret_cast<int*>(static_cast<uint8_t*>(ws) + kKvCounterBytes);
  float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + kv_attn_tile_parts(D));
  int grid = sm_count();
  if (grid > kKvMaxSms) grid = kKvMaxSms;
  return launch_behind(kern, (unsigned)grid, kPThreads, PSmem<D>::kAlloc, st, a, c, b, parts, counters);
}

}  // namespace
}  // namespace kv

size_t kv_prefill_parts_bytes(int dim) { return sizeof(float) * 2 * (size_t)kKvMaxSms * kv::kTileRows * (dim + 2); }
bool kv_prefill_takes(int dim, bool bf16) { return bf16 && (dim == 64 || dim == 128); }

cudaError_t launch_kv_prefill(const KvAttention& a, const KvCache& c, const KvBatch& b, void* ws, cudaStream_t st) {
  return c.dim == 64 ? kv::launch_prefill<64>(a, c, b, ws, st) : kv::launch_prefill<128>(a, c, b, ws, st);
}

cudaError_t kv_prefill_status(unsigned* out, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(out, g_kv_prefill_status, sizeof(unsigned));
  if (e != cudaSuccess || !clear) return e;
  const unsigned zero = 0;
  return cudaMemcpyToSymbol(g_kv_prefill_status, &zero, sizeof(unsigned));
}

}  // namespace vbq
