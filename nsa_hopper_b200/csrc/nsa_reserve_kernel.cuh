// Page tables, packing, positions and slots of a batch, from the tokens that each request gets or gives back.
//
// With p(x) = ceil(x / 64), a sequence that holds h tokens and asks for r more needs p(h + r) - p(h) pages; one that gives -r
// back returns p(h) - p(h + r).  Two sums over the sequences say who gets which page (nsa_reserve_index.h), a third one where
// each row stands; after them every page and every row is found by itself.
//
// What bounds it: latency.  512 sequences of a decode step move 40 KB, 257 prompts with 238000 rows 2.9 MB, 0.4 us at the
// measured copy rate.  So it is one launch of one cluster: each block makes the same three sums from global memory into its shared
// memory (cheaper than passing them on), the cluster meets once, so that lengths and pool may be replaced in place, and its warps
// share out the sequences.  8 sequences 2.8 us, 512 of which 25 have ended 5.3 us, 2999 with drafts 10.5 us (of which their
// 8600 packed rows, each searched for in the sums, take 3).  Many packed rows take a second launch, on all SMs: the prompts
// 8.3 us, and 47 inside the cluster.
#pragma once
#include <stdint.h>

#include "nsa_reserve_index.h"
#include "nsa_programmatic.cuh"
#include "ptx.cuh"

namespace nsa {
namespace reserve {

constexpr int kMaxSeqs = 8192;  // their six sums and lengths fill 192 KB of shared memory
constexpr int kMaxThreads = 1024;
constexpr int kCluster = 8;
constexpr int kRowsInside = 16384;  // packed rows: 8600 take 10.5 us inside the cluster, and 12.9 with a second launch

struct Args {
  int32_t* pages;
  const int32_t* held;
  const int32_t* rows;
  int32_t* pool;
  const int32_t* n_free;
  int32_t* held_out;    // may be held
  int32_t* n_free_out;  // may be n_free
  int32_t* lens;
  int32_t* cu;          // nullptr: row s is sequence s's
  int32_t* positions;   // may be nullptr
  int64_t* slots;       // may be nullptr
  int64_t page_row;
  int32_t n_seqs, width, pool_size, n_rows;
  int32_t rows_apart;   // packed rows are left to rows_kernel
};

__host__ __device__ constexpr int smem_bytes(int n_seqs) { return (6 * n_seqs + 3) * 4; }

struct Sums {
  uint32_t need, give, rows;
};
__device__ __forceinline__ uint32_t add_saturated(uint32_t a, uint32_t b) {
  const uint32_t s = a + b;  // (both at most 2^31 - 1)
  return s < 0x7FFFFFFFu ? s : 0x7FFFFFFFu;
}
__device__ __forceinline__ Sums add(const Sums& a, const Sums& b) {
  return {a.need + b.need, a.give + b.give, add_saturated(a.rows, b.rows)};
}
__device__ __forceinline__ Sums shuffle_up(const Sums& a, int by) {
  return {__shfl_up_sync(0xFFFFFFFFu, a.need, by), __shfl_up_sync(0xFFFFFFFFu, a.give, by),
          __shfl_up_sync(0xFFFFFFFFu, a.rows, by)};
}
// Sum over the threads before this one.
__device__ __forceinline__ Sums sum_before(const Sums& mine, Sums* warps) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  Sums upto = mine;
#pragma unroll
  for (int by = 1; by < 32; by *= 2) {
    const Sums other = shuffle_up(upto, by);
    if (lane >= by) upto = add(upto, other);
  }
  if (lane == 31) warps[warp] = upto;
  __syncthreads();
  if (warp == 0) {
    Sums w = lane < (int)blockDim.x / 32 ? warps[lane] : Sums{0, 0, 0};
#pragma unroll
    for (int by = 1; by < 32; by *= 2) {
      const Sums other = shuffle_up(w, by);
      if (lane >= by) w = add(w, other);
    }
    warps[lane] = w;
  }
  __syncthreads();
  const Sums before = shuffle_up(upto, 1);
  Sums s = lane > 0 ? before : Sums{0, 0, 0};
  if (warp > 0) s = add(warps[warp - 1], s);
  return s;
}

// Moves n pages by a warp, four of a lane on their way at once.
template <class From, class To>
__device__ __forceinline__ void move_pages(uint32_t n, uint32_t lane, From&& from, To&& to) {
  for (uint32_t j0 = lane; j0 - lane < n; j0 += 128) {
    int32_t page[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) page[k] = j0 + 32 * k < n ? from(j0 + 32 * k) : 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (j0 + 32 * k < n) to(j0 + 32 * k, page[k]);
  }
}

__global__ void __launch_bounds__(kMaxThreads) reserve_kernel(const Args a) {
  extern __shared__ uint32_t sm[];
  __shared__ Sums warps[32];
  __shared__ uint32_t s_taken;
  const int n = a.n_seqs, tid = threadIdx.x;
  uint32_t* need = sm;              // [n + 1]
  uint32_t* give = need + n + 1;    // [n + 1]
  uint32_t* cu = give + n + 1;      // [n + 1]
  int32_t* from = reinterpret_cast<int32_t*>(cu + n + 1);
  int32_t* lens = from + n;
  int32_t* held = lens + n;
  start_in_order();
  const int32_t free = clamp_free(a.n_free[0], a.pool_size);
#pragma unroll 4
  for (int s = tid; s < n; s += blockDim.x) lens[s] = a.rows[s], held[s] = a.held[s];
  if (tid == 0) s_taken = 0;
  __syncthreads();
  // the sums, over neighbouring sequences of a thread first
  const int each = (n + blockDim.x - 1) / blockDim.x, s0 = min(n, tid * each), s1 = min(n, s0 + each);
  Sums mine = {0, 0, 0};
  for (int s = s0; s < s1; ++s) {
    const Change c = change_of(held[s], lens[s], a.width);
    mine = add(mine, {(uint32_t)c.need(), (uint32_t)c.give(), (uint32_t)max(lens[s], 0)});
  }
  Sums at = sum_before(mine, warps);
  const Sums all = warps[31];
  const int32_t top = (int32_t)min((uint32_t)a.pool_size, (uint32_t)free + all.give);
  uint32_t taken = 0;
  for (int s = s0; s < s1; ++s) {
    const int32_t rows = lens[s];
    const Change c = change_of(held[s], rows, a.width);
    need[s] = at.need, give[s] = at.give, cu[s] = at.rows;
    at = add(at, {(uint32_t)c.need(), (uint32_t)c.give(), (uint32_t)max(rows, 0)});
    const bool ok = granted(c, at.need, top);
    if (at.need <= (uint32_t)top) taken = at.need;  // (the needs that fit come first)
    from[s] = min(c.before_pages, c.after_pages);
    lens[s] = ok ? c.after : 0;
    held[s] = rows > 0 && !ok ? c.held : c.after;
  }
  if (tid == 0) need[n] = all.need, give[n] = all.give, cu[n] = all.rows;
  taken = __reduce_max_sync(0xFFFFFFFFu, taken);
  if (tid % 32 == 0 && taken > 0) atomicMax(&s_taken, taken);
  ptx::cluster_sync();  // every block has read lengths and n_free, and has its sums
  taken = s_taken;
  Plan p;
  p.pages = a.pages, p.pool = a.pool, p.need = need, p.give = give, p.cu = cu, p.from = from, p.lens = lens;
  p.page_row = a.page_row, p.n_seqs = n, p.width = a.width, p.free = free, p.first = top - (int32_t)taken;

  const uint32_t threads = gridDim.x * blockDim.x, me = blockIdx.x * blockDim.x + tid;
  if (me == 0) a.n_free_out[0] = p.first;
  for (uint32_t s = me; s < (uint32_t)n; s += threads) {
    a.held_out[s] = held[s];
    a.lens[s] = lens[s];
  }
  if (a.cu != nullptr)
    for (uint32_t s = me; s <= (uint32_t)n; s += threads) a.cu[s] = (int32_t)cu[s];
  // Pages that are given back are read from the rows of shrinking sequences and those taken are written to the rows of growing
  // ones; the pool is read below `free` and written from there on.  So nothing that is read here is written here.  A warp has
  // some neighbouring sequences: a lane takes the one page of its sequence, and for more they work together.
  const uint32_t lane = tid % 32, crew = threads / 32;
  uint32_t some = 1;
  while (some < 32 && 4 * some * crew < (uint32_t)n) some *= 2;
  for (uint32_t s0 = me / 32 * some; s0 < (uint32_t)n; s0 += crew * some) {
    const uint32_t s = s0 + lane;
    const bool mine = lane < some && s < (uint32_t)n;
    const uint32_t takes = mine ? min(need[s + 1], taken) - min(need[s], taken) : 0;
    if (takes == 1) a.pages[(int64_t)s * a.page_row + from[s]] = taken_page(p, need[s]);
    uint32_t many = __ballot_sync(0xFFFFFFFFu, takes > 1 || (mine && give[s + 1] > give[s]));
    for (; many != 0; many &= many - 1) {
      const uint32_t x = s0 + __ffs(many) - 1, n0 = need[x], g0 = give[x];
      int32_t* table = a.pages + (int64_t)x * a.page_row + from[x];
      move_pages(min(need[x + 1], taken) - min(n0, taken), lane, [&](uint32_t j) { return taken_page(p, n0 + j); },
                 [&](uint32_t j, int32_t page) { table[j] = page; });
      const int64_t at = free + (int64_t)g0;
      move_pages((uint32_t)max((int64_t)0, min((int64_t)(give[x + 1] - g0), a.pool_size - at)), lane,
                 [&](uint32_t j) { return table[j]; }, [&](uint32_t j, int32_t page) { a.pool[at + j] = page; });
    }
  }
  if (a.cu == nullptr) {
    for (uint32_t s = me; s < (uint32_t)n; s += threads) {
      const int32_t pos = lens[s] - 1;
      if (a.positions != nullptr) a.positions[s] = pos;
      if (a.slots != nullptr) a.slots[s] = pos < 0 ? -1 : slot_of(page_after(p, (int)s, pos / kPage), pos);
    }
  } else if (!a.rows_apart) {
    for (uint32_t r = me; r < (uint32_t)a.n_rows; r += threads) {
      const int s = n > 0 && r < cu[n] ? range_of(cu, n, r) : -1;
      const int32_t pos = s >= 0 && lens[s] > 0 ? lens[s] - (int32_t)(cu[s + 1] - r) : -1;
      if (a.positions != nullptr) a.positions[r] = pos;
      if (a.slots != nullptr) a.slots[r] = pos < 0 ? -1 : slot_of(page_after(p, s, pos / kPage), pos);
    }
  }
}

// Positions and slots of packed rows, a thread each, from what reserve_kernel has written.
__global__ void __launch_bounds__(256) rows_kernel(const Args a) {
  start_in_order();
  const int32_t r = (int32_t)(blockIdx.x * 256u + threadIdx.x);
  if (r >= a.n_rows) return;
  const cache::Batch b = {a.pages, a.lens, a.cu, a.page_row, a.n_seqs, a.width, 0, a.n_rows};
  const int s = cache::sequence_of(b, r);
  const int32_t pos = s >= 0 && a.lens[s] > 0 ? cache::position_of(b, s, r) : -1;
  if (a.positions != nullptr) a.positions[r] = pos;
  if (a.slots != nullptr)  // (a length that the first kernel has written lies in the table)
    a.slots[r] = pos < 0 ? -1 : slot_of(a.pages[(int64_t)s * a.page_row + pos / kPage], pos);
}

}  // namespace reserve
}  // namespace nsa
