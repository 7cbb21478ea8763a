// vbq_kv_pages.cu -- page moves of the KV cache: room for new tokens, regrouping the
// sequences of a beam search, making the pool dense.
//
// The pages in use are those with refs > 0 (refs counts the rows of the page tables that hold
// the page).  "The lowest free pages in order" makes every move a function of its inputs: no
// result depends on the order in which threads run.  Plans are made by one CTA, whose cost is
// the scan over refs; the pages themselves are moved by a grid over 16-byte pieces, which is
// launched under the plan and waits for it.
//
// Measured (device time): a pool made dense, 222 MB moved: 79 us, of which the moves take 70 (6.4 TB/s
// of read and write); a fork of 32 rows with 32 MB of part-filled pages to copy and a reserve: 26 us,
// of which 10 are the plan's chain of dependent reads, 12 the copies and 5 the reserve (7 by itself).  A
// row's fresh pages are listed by one thread: a prompt of 131072 tokens in pages of 16, 472 us.
#include <climits>

#include "vbq_internal.h"
#include "vbq_kv.cuh"

namespace vbq {
namespace kv {
namespace {

constexpr int kPlanThreads = 1024, kPlanWarps = kPlanThreads / 32;

// Sum over the CTA's threads before this one; `total` receives the sum over all.
__device__ __forceinline__ int block_scan(int v, int* sh, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int in = warp_scan(v, lane);
  if (lane == 31) sh[warp] = in;
  __syncthreads();
  const int w = warp_scan(sh[lane], lane);  // kPlanWarps == 32
  total = __shfl_sync(kFull, w, 31);
  const int before = warp ? __shfl_sync(kFull, w, warp - 1) : 0;
  __syncthreads();
  return before + in - v;
}
static_assert(kPlanWarps == 32, "block_scan takes one partial sum a lane");

// Pages of warp w when `pages` are split evenly over the plan's warps, in whole lots of 32.
__device__ __forceinline__ void warp_range(int64_t pages, int warp, int64_t& a, int64_t& z) {
  const int64_t per = ((pages + kPlanWarps - 1) / kPlanWarps + 31) / 32 * 32;
  a = min(pages, warp * per);
  z = min(pages, a + per);
}

// Lists the lowest `need` free pages: calls take(rank, page) for rank 0 .. need - 1 while
// there are any.  refs_at(p) is what page p's count is now.  Returns how many there were.
template <typename R, typename T>
__device__ __forceinline__ int lowest_free(int64_t pages, int need, int* sh, R refs_at, T take) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t a, z;
  warp_range(pages, warp, a, z);
  int mine = 0;
  for (int64_t p = a + lane; p < z; p += 32) mine += refs_at(p) == 0;
#pragma unroll
  for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(kFull, mine, o);
  int total;
  int rank = block_scan(lane == 0 ? mine : 0, sh, total);  // lane 0's: free pages of earlier warps
  rank = __shfl_sync(kFull, rank, 0);
  for (int64_t p0 = a; p0 < z && rank < need; p0 += 32) {
    const bool is = p0 + lane < z && refs_at(p0 + lane) == 0;
    const unsigned hit = __ballot_sync(kFull, is);
    const int r = rank + __popc(hit & ((1u << lane) - 1u));
    if (is && r < need) take(r, (int)(p0 + lane));
    rank += __popc(hit);
  }
  return min(total, need);
}

__device__ __forceinline__ int held_pages(int len, int page) { return len > 0 ? (len + page - 1) / page : 0; }
__device__ __forceinline__ bool valid(int p, int64_t pages) { return p >= 0 && p < pages; }

// ---- reserve ---------------------------------------------------------------------------
// CTA 0 plans; the others copy the table entries that do not change (when not in place).
// Workspace: the list of fresh pages.
__global__ void __launch_bounds__(kPlanThreads)
reserve_kernel(const int32_t* refs, const int32_t* tables, const int32_t* lens,
               const int32_t* __restrict__ add, int64_t pages, int page, int rows, int max_pages,
               int32_t* refs_out, int32_t* tables_out, int32_t* lens_out, int32_t* missing, int32_t* fresh,
               int64_t most) {
  pdl_wait();
  const bool alone = gridDim.x == 1;
  if (blockIdx.x > 0 || alone) {
    if (tables_out != tables) {
      const int first = alone ? 0 : (int)blockIdx.x - 1, by = alone ? 1 : (int)gridDim.x - 1;
      for (int s = first; s < rows; s += by) {
        const int len = lens[s];
        const int64_t want = (int64_t)max(len, 0) + max(add[s], 0);
        const int held = held_pages(len, page);
        const int64_t to = want > 0 ? (want + page - 1) / page : 0;
        for (int j = threadIdx.x; j < max_pages; j += blockDim.x)
          if (j < held || j >= to) tables_out[(int64_t)s * max_pages + j] = tables[(int64_t)s * max_pages + j];
      }
    }
    if (!alone) return;
    __syncthreads();
  }
  __shared__ int sh[kPlanWarps];
  __shared__ int got_sh;
  if (refs_out != refs)
    for (int64_t p = threadIdx.x; p < pages; p += kPlanThreads) refs_out[p] = refs[p];
  // how many each row needs, and in all
  int need = 0;
  for (int s0 = 0; s0 < rows; s0 += kPlanThreads) {
    const int s = s0 + threadIdx.x;
    int mine = 0;
    if (s < rows) {
      const int64_t want = (int64_t)max(lens[s], 0) + max(add[s], 0);
      const int64_t to = min((int64_t)max_pages, want > 0 ? (want + page - 1) / page : 0);
      mine = (int)max((int64_t)0, to - held_pages(lens[s], page));
    }
    int total;
    block_scan(mine, sh, total);
    need += total;
  }
  __syncthreads();
  need = (int)min((int64_t)need, most);
  const int got = lowest_free(pages, need, sh, [&](int64_t p) { return refs[p]; },
                              [&](int r, int p) { fresh[r] = p; });
  if (threadIdx.x == 0) got_sh = got;
  __syncthreads();
  int before = 0, asked = 0;
  for (int s0 = 0; s0 < rows; s0 += kPlanThreads) {
    const int s = s0 + threadIdx.x;
    int mine = 0, held = 0;
    if (s < rows) {
      const int len = max(lens[s], 0), more = max(add[s], 0);
      const int64_t want = (int64_t)len + more;
      held = held_pages(len, page);
      const int64_t to = want > 0 ? (want + page - 1) / page : 0;
      // pages past the table's width are missing too
      mine = (int)max((int64_t)0, min((int64_t)max_pages, to) - held);
      asked += (int)max((int64_t)0, to - held);
    }
    int total;
    const int at = before + block_scan(mine, sh, total);
    for (int i = 0; i < mine; ++i) {
      const int p = at + i < got_sh ? fresh[at + i] : -1;
      tables_out[(int64_t)s * max_pages + held + i] = p;
      if (p >= 0) refs_out[p] = 1;
    }
    before += total;
    if (s < rows) lens_out[s] = max(lens[s], 0) + max(add[s], 0);
  }
  int total;
  block_scan(asked, sh, total);
  if (threadIdx.x == 0) *missing = total - got_sh;
}

// ---- fork ------------------------------------------------------------------------------
// Workspace: delta [pages] (zero between calls: what to add to refs), a counter (zero), then
// the list of copies (destination, source) with its length.
struct ForkSpace {
  int32_t* delta;
  int32_t* arrived;
  int32_t* copies;  // [0]: how many; then pairs from [2]
  int32_t* fresh;
  int32_t* first;   // of each old row, the lowest new row that continues it
};

// CTAs 0 .. rows - 1: what becomes of old row s's pages.  CTAs rows ..: new rows' tables.
// The last CTA to finish plans the copies.
__global__ void __launch_bounds__(kPlanThreads)
fork_kernel(const int32_t* refs, const int32_t* __restrict__ tables,
            const int32_t* __restrict__ lens, const int32_t* __restrict__ parents, int64_t pages, int page,
            int rows, int max_pages, int new_rows, int32_t* refs_out, int32_t* tables_out, int32_t* lens_out,
            int32_t* missing, ForkSpace ws) {
  pdl_wait();
  __shared__ int sh[kPlanWarps];
  __shared__ int flag, lowest;
  __shared__ int near[kPlanThreads];  // the fresh pages, where they fit
  const int tid = threadIdx.x;
  pdl_release();  // only the copying kernel follows, and it waits for this one's end
  if ((int)blockIdx.x < rows) {
    const int s = blockIdx.x;
    if (tid == 0) lowest = INT_MAX;
    __syncthreads();
    int mine = 0;
    for (int r = tid; r < new_rows; r += kPlanThreads)
      if (parents[r] == s) {
        ++mine;
        atomicMin(&lowest, r);
      }
    int children;
    block_scan(mine, sh, children);
    if (tid == 0) ws.first[s] = lowest;
    const int len = max(lens[s], 0), held = min(held_pages(len, page), max_pages), full = len / page;
    for (int j = tid; j < held; j += kPlanThreads) {
      const int p = tables[(int64_t)s * max_pages + j];
      const int d = j < full ? children - 1 : min(children, 1) - 1;
      if (valid(p, pages) && d) atomicAdd(ws.delta + p, d);
    }
  } else if ((int)blockIdx.x - rows < new_rows) {
    const int r = blockIdx.x - rows;
    const int s = parents[r];
    const bool live = s >= 0 && s < rows;
    const int len = live ? max(lens[s], 0) : 0, held = held_pages(len, page);
    for (int j = tid; j < max_pages; j += kPlanThreads) {
      const int p = j < held ? tables[(int64_t)s * max_pages + j] : -1;
      tables_out[(int64_t)r * max_pages + j] = valid(p, pages) ? p : -1;
    }
    if (tid == 0) lens_out[r] = len;
  }
  // what the plan needs of the first rows, asked for before anything is waited for
  int s0 = -1, j0 = 0, src0 = -1;
  if (tid < new_rows) {
    s0 = parents[tid];
    if (s0 >= 0 && s0 < rows) {
      const int len = max(lens[s0], 0);
      j0 = len / page;
      if (len % page != 0 && j0 < max_pages) src0 = tables[(int64_t)s0 * max_pages + j0];
    }
  }
  __threadfence();
  __syncthreads();
  if (tid == 0) flag = atomicAdd(ws.arrived, 1) == (int)gridDim.x - 1;
  __syncthreads();
  if (!flag) return;
  __threadfence();
  // the plan
  for (int64_t p = tid; p < pages; p += kPlanThreads) {
    const int d = __ldcg(ws.delta + p);
    refs_out[p] = max(refs[p] + d, 0);
    if (d) ws.delta[p] = 0;
  }
  // rows that need a copy: their last page is part-filled and a lower row continues the parent
  auto look = [&](int r, int& j) {  // the page to copy, or -1
    int s = s0, src = src0;
    j = j0;
    if (r != tid) {
      s = parents[r], src = -1;
      if (s >= 0 && s < rows) {
        const int len = max(lens[s], 0);
        j = len / page;
        if (len % page != 0 && j < max_pages) src = tables[(int64_t)s * max_pages + j];
      }
    }
    return valid(src, pages) && __ldcg(ws.first + s) != r ? src : -1;
  };
  int need = 0, j;
  const int mine0 = tid < new_rows ? look(tid, j) : -1;
  for (int r0 = 0; r0 < new_rows; r0 += kPlanThreads) {
    const int r = r0 + tid;
    int total;
    block_scan(r < new_rows && (r0 == 0 ? mine0 : look(r, j)) >= 0, sh, total);
    need += total;
  }
  __syncthreads();
  const bool fits = need <= kPlanThreads;
  const int got = lowest_free(pages, need, sh, [&](int64_t p) { return refs_out[p]; },
                              [&](int i, int p) { (fits ? near : ws.fresh)[i] = p; });
  __syncthreads();
  int before = 0;
  for (int r0 = 0; r0 < new_rows; r0 += kPlanThreads) {
    const int r = r0 + tid;
    j = j0;
    const int src = r >= new_rows ? -1 : r0 == 0 ? mine0 : look(r, j);
    int total;
    const int at = before + block_scan(src >= 0, sh, total);
    if (src >= 0) {
      const int p = at < got ? (fits ? near : ws.fresh)[at] : -1;
      if (p >= 0) {
        ws.copies[2 + 2 * at] = p;
        ws.copies[3 + 2 * at] = src;
        refs_out[p] = 1;
      }
      tables_out[(int64_t)r * max_pages + j] = p;
    }
    before += total;
  }
  if (tid == 0) {
    ws.copies[0] = got;
    *missing = need - got;
    *ws.arrived = 0;
  }
}

// ---- compact ---------------------------------------------------------------------------
// Workspace: the list of moves (destination, source), and each page's new number.
__global__ void __launch_bounds__(kPlanThreads)
compact_plan_kernel(const int32_t* refs, int64_t pages, int32_t* refs_out, int32_t* live_out, int32_t* moves,
                    int32_t* to) {
  __shared__ int sh[kPlanWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  pdl_release();  // only the moving kernel follows, and it waits for this one's end
  int64_t a, z;
  warp_range(pages, warp, a, z);
  int used = 0;
  for (int64_t p = a + lane; p < z; p += 32) used += refs[p] > 0;
#pragma unroll
  for (int o = 16; o; o >>= 1) used += __shfl_xor_sync(kFull, used, o);
  int live;
  int before = block_scan(lane == 0 ? used : 0, sh, live);
  before = __shfl_sync(kFull, before, 0);  // pages in use below this warp's
  // holes below `live` and pages in use at or above it, each numbered in order: as many of the
  // one as of the other.  Pages in use below p: u(p).  A hole p is number p - u(p); a page p
  // that moves is number u(p) - u(live), counted here from the other end: live - u(p) pages in
  // use lie at p or above, so it is number (movers - (live - u(p))).
  // movers = live - u(live), found first
  __shared__ int below_live;
  if (threadIdx.x == 0) below_live = 0;
  __syncthreads();
  int mine = 0;
  for (int64_t p = a + lane; p < z && p < live; p += 32) mine += refs[p] > 0;
#pragma unroll
  for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(kFull, mine, o);
  if (lane == 0 && mine) atomicAdd(&below_live, mine);
  __syncthreads();
  const int movers = live - below_live;
  for (int64_t p0 = a; p0 < z; p0 += 32) {
    const int64_t p = p0 + lane;
    const bool in = p < z;
    const bool is = in && refs[p] > 0;
    const unsigned hit = __ballot_sync(kFull, is);
    const int u = before + __popc(hit & ((1u << lane) - 1u));
    if (in && p < live && !is) moves[2 + 2 * ((int)p - u)] = (int)p;
    if (is && p >= live) moves[3 + 2 * (movers - (live - u))] = (int)p;
    before += __popc(hit);
  }
  __syncthreads();
  // refs may be refs_out: every page reads its own count before any is written
  for (int64_t p = threadIdx.x; p < pages; p += kPlanThreads) {
    to[p] = (int)p;
    if (refs_out != refs) refs_out[p] = refs[p];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < movers; i += kPlanThreads) {
    const int d = moves[2 + 2 * i], s = moves[3 + 2 * i];
    to[s] = d;
    refs_out[d] = refs_out[s];  // sources and destinations are disjoint
  }
  __syncthreads();
  for (int i = threadIdx.x; i < movers; i += kPlanThreads) refs_out[moves[3 + 2 * i]] = 0;
  if (threadIdx.x == 0) {
    moves[0] = movers;
    *live_out = live;
  }
}

// Moves pages: list[0] pairs (destination, source) from list[2]; 16-byte pieces of a page over
// the grid.  Sources and destinations are disjoint.  rows > 0: then also the page tables'
// entries through `to`.
constexpr int kMoveThreads = 256, kMoveUnroll = 8;
__global__ void __launch_bounds__(kMoveThreads)
move_kernel(KvPool pool, const int32_t* list, const int32_t* tables,
            const int32_t* __restrict__ lens, int rows, int max_pages, const int32_t* to,
            int32_t* tables_out) {
  pdl_wait();
  const int count = __ldcg(list);
  constexpr int64_t kPiece = (int64_t)kMoveThreads * kMoveUnroll * 16;
  const int64_t per_page = (pool.page_bytes + kPiece - 1) / kPiece;
  for (int64_t u = blockIdx.x; u < count * per_page; u += gridDim.x) {
    const int64_t pair = u / per_page, at = (u - pair * per_page) * kPiece + threadIdx.x * 16;
    const int64_t d = __ldcg(list + 2 + 2 * pair), s = __ldcg(list + 3 + 2 * pair);
    const uint8_t* src = pool.codes + s * pool.page_bytes;
    uint8_t* dst = pool.codes + d * pool.page_bytes;
    uint4 v[kMoveUnroll];
#pragma unroll
    for (int i = 0; i < kMoveUnroll; ++i) {
      const int64_t o = at + (int64_t)i * kMoveThreads * 16;
      if (o < pool.page_bytes) v[i] = ld_stream(src + o);
    }
#pragma unroll
    for (int i = 0; i < kMoveUnroll; ++i) {
      const int64_t o = at + (int64_t)i * kMoveThreads * 16;
      if (o < pool.page_bytes) __stcs(reinterpret_cast<uint4*>(dst + o), v[i]);
    }
    if (u == pair * per_page)
      for (int64_t i = threadIdx.x; i < pool.page_scales; i += kMoveThreads)
        pool.scales[d * pool.page_scales + i] = pool.scales[s * pool.page_scales + i];
  }
  if (rows > 0) {
    const int64_t n = (int64_t)rows * max_pages;
    for (int64_t i = (int64_t)blockIdx.x * kMoveThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kMoveThreads) {
      const int s = (int)(i / max_pages), j = (int)(i - (int64_t)s * max_pages);
      const int p = tables[i];
      tables_out[i] = j < held_pages(lens[s], pool.page) && valid(p, pool.pages) ? __ldcg(to + p) : -1;
    }
  }
}

int64_t pad(int64_t n) { return (n + 3) / 4 * 4; }
// The moves, started under the plan that writes their list.
cudaError_t launch_moves(const KvPool& p, const int32_t* list, const int32_t* tables, const int32_t* lens, int rows,
                         int max_pages, const int32_t* to, int32_t* tables_out, cudaStream_t st) {
  return launch_behind(move_kernel, (unsigned)(sm_count() * 8), kMoveThreads, 0, st, p, list, tables, lens, rows, max_pages,
                       to, tables_out);
}

}  // namespace
}  // namespace kv

// delta [pages] and a counter (kept zero), copies or moves (2 + 2 * entries), fresh pages or
// new numbers, each row's first continuation
size_t kv_pages_workspace(int64_t pages, int rows) {
  const int64_t most = pages > rows ? pages : rows;
  return sizeof(int32_t) * (size_t)(kv::pad(pages + 1) + kv::pad(2 + 2 * most) + 2 * kv::pad(most));
}

cudaError_t launch_kv_reserve(const int32_t* refs, const int32_t* tables, const int32_t* lens,
                              const int32_t* add, int64_t pages, int page, int rows, int max_pages,
                              int32_t* refs_out, int32_t* tables_out, int32_t* lens_out, int32_t* missing,
                              void* workspace, cudaStream_t st) {
  int32_t* fresh = static_cast<int32_t*>(workspace) + kv::pad(pages + 1);
  // the other CTAs read lens while CTA 0 writes lens_out: apart only when they are not the same
  const bool alone = lens_out == lens || tables_out == tables || rows < 4;
  const int sms = sm_count();
  const unsigned grid = alone ? 1u : 1u + (unsigned)(rows < sms - 1 ? rows : sms - 1);
  return kv::launch_behind(kv::reserve_kernel, grid, kv::kPlanThreads, 0, st, refs, tables, lens, add, pages, page, rows,
                           max_pages, refs_out, tables_out, lens_out, missing, fresh, pages);
}

cudaError_t launch_kv_fork(const KvPool& p, const int32_t* refs, const int32_t* tables, const int32_t* lens,
                           int rows, int max_pages, const int32_t* parents, int new_rows, int32_t* refs_out,
                           int32_t* tables_out, int32_t* lens_out, int32_t* missing, void* workspace,
                           cudaStream_t st) {
  int32_t* w = static_cast<int32_t*>(workspace);
  const int64_t wide = rows > new_rows ? rows : new_rows, most = p.pages > wide ? p.pages : wide;
  int32_t* copies = w + kv::pad(p.pages + 1);
  int32_t* fresh = copies + kv::pad(2 + 2 * most);
  const kv::ForkSpace ws{w, w + p.pages, copies, fresh, fresh + kv::pad(most)};
  cudaError_t e = kv::launch_behind(kv::fork_kernel, (unsigned)(rows + new_rows > 0 ? rows + new_rows : 1),
                                    kv::kPlanThreads, 0, st, refs, tables, lens, parents, p.pages, p.page, rows,
                                    max_pages, new_rows, refs_out, tables_out, lens_out, missing, ws);
  if (e != cudaSuccess) return e;
  return kv::launch_moves(p, ws.copies, nullptr, nullptr, 0, 0, nullptr, nullptr, st);
}

cudaError_t launch_kv_compact(const KvPool& p, const int32_t* refs, const int32_t* tables, const int32_t* lens,
                              int rows, int max_pages, int32_t* refs_out, int32_t* tables_out, int32_t* live,
                              void* workspace, cudaStream_t st) {
  int32_t* w = static_cast<int32_t*>(workspace) + kv::pad(p.pages + 1);
  const int64_t most = p.pages > rows ? p.pages : rows;
  int32_t* to = w + kv::pad(2 + 2 * most);
  cudaError_t e = kv::launch_behind(kv::compact_plan_kernel, 1, kv::kPlanThreads, 0, st, refs, p.pages, refs_out, live, w, to);
  if (e != cudaSuccess) return e;
  return kv::launch_moves(p, w, tables, lens, rows, max_pages, to, tables_out, st);
}

}  // namespace vbq
