// Page tables, packing, positions and slots of a batch, from the tokens that each request gets or gives back.
//
// With p(x) = ceil(x / 64), a sequence that holds h tokens and asks for r more needs p(h + r) - p(h) pages; one that gives -r
// back returns p(h) - p(h + r).  Two sums over the sequences say who gets which page (nsa_reserve_index.h), a third one where
// each row stands; after them every page and every row is found by itself.
//
// What bounds it: latency.  512 sequences move 10 KB, 257 prompts with 218000 rows 2.7 MB (0.4 us at the measured copy
// rate).  So it is one launch of one cluster: each block makes the same three sums from global memory into its shared memory
// (cheaper than passing them on), the cluster meets once, so that lengths and pool may be replaced in place, and its threads
// share out pages and rows.
#pragma once
#include <stdint.h>

#include "nsa_reserve_index.h"
#include "nsa_programmatic.cuh"
#include "ptx.cuh"

namespace nsa {
namespace reserve {

constexpr int kMaxSeqs = 8192;  // their six sums and lengths fill 196 KB of shared memory
constexpr int kMaxThreads = 1024;
constexpr int kCluster = 8;
constexpr int kRows = 4;        // rows of a thread at a time

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

__global__ void __launch_bounds__(kMaxThreads) kernel(const Args a) {
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
  // ones; the pool is read below `free` and written from there on.  So nothing that is read here is written here.
  for (uint32_t j = me; j < taken; j += threads) {
    const int s = range_of(need, n, j);
    a.pages[(int64_t)s * a.page_row + from[s] + (int32_t)(j - need[s])] = taken_page(p, j);
  }
  for (uint32_t j = me; j < all.give && free + (int64_t)j < a.pool_size; j += threads) a.pool[free + (int64_t)j] = given_page(p, j);

  if (a.cu == nullptr) {
    for (uint32_t s = me; s < (uint32_t)n; s += threads) {
      const int32_t pos = lens[s] - 1;
      if (a.positions != nullptr) a.positions[s] = pos;
      if (a.slots != nullptr) a.slots[s] = pos < 0 ? -1 : slot_of(page_after(p, (int)s, pos / kPage), pos);
    }
    return;
  }
  // kRows neighbouring rows of a thread are mostly of one page
  for (uint32_t r0 = me * kRows; r0 < (uint32_t)a.n_rows; r0 += threads * kRows) {
    int s = n > 0 ? range_of(cu, n, r0) : -1;
    int32_t page = -1, page_sub = -1;
    int32_t pos[kRows];
    int64_t slot[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const uint32_t r = r0 + k;
      pos[k] = -1, slot[k] = -1;
      if (s < 0 || r >= cu[n]) continue;
      if (r >= cu[s + 1]) s = range_of(cu, n, r), page_sub = -1;
      if (lens[s] == 0) continue;
      pos[k] = lens[s] - (int32_t)(cu[s + 1] - r);
      if (pos[k] / kPage != page_sub) page_sub = pos[k] / kPage, page = page_after(p, s, page_sub);
      slot[k] = slot_of(page, pos[k]);
    }
    if (r0 + kRows <= (uint32_t)a.n_rows) {
      if (a.positions != nullptr) reinterpret_cast<int4*>(a.positions + r0)[0] = make_int4(pos[0], pos[1], pos[2], pos[3]);
      if (a.slots != nullptr) {
        reinterpret_cast<longlong2*>(a.slots + r0)[0] = make_longlong2(slot[0], slot[1]);
        reinterpret_cast<longlong2*>(a.slots + r0)[1] = make_longlong2(slot[2], slot[3]);
      }
    } else {
      for (int k = 0; k < kRows && r0 + k < (uint32_t)a.n_rows; ++k) {
        if (a.positions != nullptr) a.positions[r0 + k] = pos[k];
        if (a.slots != nullptr) a.slots[r0 + k] = slot[k];
      }
    }
  }
}

}  // namespace reserve
}  // namespace nsa
