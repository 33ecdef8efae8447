// Block selection for single tokens: the best blocks of a row's sequence by the scores of its query against the compressed
// keys of a 4-bit cache,
//     s(block) = sum over the compressed keys i of the block of (sum_g q_g) . k_i,
// the n_sel best, the best first, ties to the lowest block.
//
// Ranks are all that comes out, so where two scores are close a rounding would turn them around.  Hence two kernels:
//   * score_kernel bounds every block's score from both sides, from an approximation on the tensor cores.  A warp has the blocks
//     of about 64 keys; the cache is the A operand (m16n8k16, fp16 in, fp32 out) without its scales.  Each thread takes a
//     quarter of a key's codes, d is permuted to fit, and the eight columns of the B operand are the query's sum in each quarter
//     alone, twice: its fp16 value and what that leaves out.  So the thread that holds a key's quarter, and its scales, gets
//     the two sums of that quarter, and no code has to be multiplied by its scale.
//   * pick_kernel finds a bound that n_sel blocks are certain to reach, and computes the scores of all blocks that may reach
//     it, mostly n_sel and one or two more, in 64 bits from exact parts: codes (doubled) are whole numbers up to 12, the query
//     is cut into whole numbers too (prepare_exact), the 16 products of a group that share a scale are added as integers
//     (dot products of four bytes), and only scale times group sum is rounded, in fp64.  A query whose channels are too far apart
//     for that keeps its sums in fp64, and so are its products.
//
// Error of the approximation, in units of max|k| (six times the largest scale of a unit's keys) times the keys of a block, with
// S = sum over d and heads of |q| and Q = sum over d of |sum of the heads|: the fp32 sum of G heads (G - 1) 2^-24 S; the two
// fp16 parts of the query 2^-22 Q; a group's products, added to the sum so far four at a time, four times (the tensor core cuts
// each term off below 2^-23 of the largest, twice that is allowed for), 20 2^-22 Q; the sums of groups and quarters in fp32
// 8 2^-24 Q; that of up to 258 keys 258 2^-24 Q.  All but the first are less than 90 2^-22 Q, and taken as 2^-15 Q.
//
// What bounds it.  A key costs 9/16 d bytes.  256 sequences of up to 65536 tokens, 4 heads of 128: 156 MB with queries and results,
// which DRAM would deliver in 24 us, take 56.  46 of them are score_kernel's: the ALU pipe, which converts codes (128 of its 400
// instructions for 64 keys), is its busiest unit at 59 %, tensor cores 19 %.  The others are pick_kernel's, 1024 blocks that are
// chains of steps (9000 cycles with 256 threads: reading the bounds 1100, the bin 1450, candidates 650, exact scores 3900, ranks
// 900; 128 threads take longer, but 8 of their blocks fit an SM).  One sequence of 65536 tokens: 9.2 us; 64 of up to 32768: 17 us.
// Where all rows are scored in fp64 these are 63, 12 and 23 us.  Where the bounds tell nothing apart (blocks that are all alike,
// query heads that cancel) every block is summed exactly: 0.77, 0.28 and 0.17 ms.  Tried: exact scores of all blocks with dot
// products of four bytes (the 256 above 102 us); the bin from the threads' largest bounds instead of counts (2000 cycles and half
// as many candidates again).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "nsa_cache_decode.cuh"
#include "nsa_cache_select_index.h"
#include "nsa_programmatic.cuh"
#include "ptx.cuh"

namespace nsa {
namespace cache_select {

constexpr int kStages = 2;        // units of a warp in shared memory: one that is scored and one that is on its way
// Warps of score_kernel, one block of which fills an SM: shared memory holds 14 times two units of d = 192.  (20 warps with
// d = 128 are 2 % faster for long calls and 12 % slower for short ones.)
__host__ __device__ constexpr int warps_of(int d) { return d <= 128 ? 16 : 14; }
constexpr int kLimbs = 6;
constexpr int kMaxRows = 1024;    // of a launch: what is kept of them fills 12 KB of shared memory
constexpr int kUnitKeys = 64;     // keys of a unit, about
constexpr int kUnitBlocks = 31;   // its blocks at most: a lane for each and one for the end
constexpr int kMaxGroup = 256;    // query heads of a KV head
constexpr int kMaxSel = 1024;
__host__ __device__ constexpr int checked(int threads) { return 8 * threads; }  // blocks that pick_kernel looks at at a time
constexpr int kAdded = 512;       // of them, those whose exact scores are compared with the best so far
constexpr int kKeys = 512;        // places of keys that are scored between two meetings
constexpr int kHeldPages = 256;   // first pages of a sequence, looked up beforehand
constexpr float kHuge = 3.0e38f;  // bound of what has none

struct Args {
  Batch b;              // the compressed cache's page table; lens: tokens of the sequences
  const void* q;        // [n_rows, Hq, D], unit stride along D
  int64_t q_row, q_head;
  const uint8_t* cache;
  int64_t page_stride;
  float2* bounds;       // [rows, Hkv, blocks] lower and upper bound of a block's score
  int32_t* sel;         // [n_rows, Hkv, n_sel]
  int32_t hkv, group, n_sel;
  int32_t shift;        // of a block's tokens
  int32_t blocks;       // blocks of a row, at most
  int32_t unit;         // blocks of a unit
  int32_t most;         // tokens of a row, at most
  int32_t cmp_block, cmp_stride;
  int32_t record;       // bytes
  int32_t q_half;
  int32_t bits;         // of a query head's value in the exact sum: its largest is below 2^bits
  int32_t keys;         // of a block, at most
  uint32_t per_key;     // 2^20 / keys, rounded up: exact for the kKeys places
  int32_t at_once;      // blocks that have kKeys places
  int32_t row0, rows;   // rows of this launch
};

// A number that compares like the score: what is no number, or infinite, comes last; -0 is 0.
__device__ __forceinline__ uint64_t rank_of(double x) {
  if (!(fabs(x) < __longlong_as_double(0x7FF0000000000000ll))) return 0;
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | 1ull << 63;
}

__device__ __forceinline__ float query_value(const Args& a, uint32_t bits) {
  return a.q_half ? __half2float(__ushort_as_half((unsigned short)bits)) : __uint_as_float(bits << 16);
}

// ------------------------------------------------------------------ bounds
// A thread's quarter of a key's codes, and their scales.
template <int D>
struct Quarter {
  uint32_t code[D / 32];  // eight codes each
  uint32_t scale;         // D / 64 bytes
};
// Of key t, counted from the quarters of another one.
template <int D>
__device__ __forceinline__ void load_quarter(Quarter<D>& k, const uint8_t* codes, const uint8_t* scales, int t) {
  const uint8_t* code = codes + t * (D / 2);
  const uint8_t* scale = scales + t * (D / 16);
  if constexpr (D == 128) {
    const uint4 v = *reinterpret_cast<const uint4*>(code);
    k.code[0] = v.x, k.code[1] = v.y, k.code[2] = v.z, k.code[3] = v.w;
    k.scale = *reinterpret_cast<const uint16_t*>(scale);
  } else {
    k.scale = 0;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const uint2 v = reinterpret_cast<const uint2*>(code)[i];
      k.code[2 * i] = v.x, k.code[2 * i + 1] = v.y;
      k.scale |= (uint32_t)scale[i] << 8 * i;
    }
  }
}

// The B operand of a (row, head): the sum of its query heads times a power of two, fp16 values (even columns) and what they
// leave out (odd ones), columns 2 q and 2 q + 1 in quarter q alone.  Returns the error of a key's score in units of a scale (not
// finite if a value is not).
template <int D>
__device__ __forceinline__ float load_query(const Args& a, uint32_t (&bq)[D / 8], int row, int head, int lane) {
  constexpr int N = D / 32;  // dims of a lane at first
  const uint16_t* q = static_cast<const uint16_t*>(a.q) + (int64_t)row * a.q_row + (int64_t)head * a.group * a.q_head + lane * N;
  float sum[N] = {}, size = 0.0f;
#pragma unroll 8
  for (int g = 0; g < a.group; ++g) {
    uint32_t two[N / 2];
    if constexpr (N == 4) {
      const uint2 v = *reinterpret_cast<const uint2*>(q + g * a.q_head);
      two[0] = v.x, two[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) two[i] = reinterpret_cast<const uint32_t*>(q + g * a.q_head)[i];
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float x = query_value(a, two[i] & 0xFFFFu), y = query_value(a, two[i] >> 16);
      sum[2 * i] += x, sum[2 * i + 1] += y;
      size += fabsf(x) + fabsf(y);
    }
  }
  size *= (float)(a.group - 1) * 5.9604645e-08f;  // 2^-24
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    top = max(top, __float_as_uint(sum[i]) & 0x7FFFFFFFu);
    size += fabsf(sum[i]) * 3.0517578e-05f;  // 2^-15
  }
  top = __reduce_max_sync(0xFFFFFFFFu, top);
#pragma unroll
  for (int by = 16; by > 0; by /= 2) size += __shfl_xor_sync(0xFFFFFFFFu, size, by);
  // the largest to [2^10, 2^11)
  const int up = min(137 - (int)(top >> 23), 126);
  const float factor = __uint_as_float((uint32_t)(127 + up) << 23);
  uint32_t upper[N / 2], lower[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float x = sum[2 * i] * factor, y = sum[2 * i + 1] * factor;
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    upper[i] = *reinterpret_cast<const uint32_t*>(&h), lower[i] = *reinterpret_cast<const uint32_t*>(&l);
  }
  // pair p of quarter q is dims q D/4 + 2 p, 2 p + 1: pair (p mod N/2) of lane 8 q + p / (N/2)
  const int column = lane / 4, quarter = lane % 4;
#pragma unroll
  for (int p = 0; p < D / 8; ++p) {
    const int from = 8 * quarter + p / (N / 2);
    const uint32_t u = __shfl_sync(0xFFFFFFFFu, upper[p % (N / 2)], from), l = __shfl_sync(0xFFFFFFFFu, lower[p % (N / 2)], from);
    bq[p] = column == 2 * quarter ? u : column == 2 * quarter + 1 ? l : 0u;
  }
  // (sums so small that 2^126 does not bring them there are left to the exact scores)
  return top >> 23 < 11u && size > 0.0f ? __uint_as_float(0x7F800000u) : 6.0f * size * factor;
}

// fp32 of scale bytes 2 I and 2 I + 1 of `s`.
template <int I>
__device__ __forceinline__ float2 scale_values(uint32_t s) {
  const uint32_t two = __byte_perm(s, 0, I == 0 ? 0x4140 : 0x4342) * 128;  // (byte << 7 is the fp16)
  return __half22float2(*reinterpret_cast<const __half2*>(&two));
}

// Keys of a unit as they are in the cache: codes [64][D / 2], scales [64][D / 16].
template <int D>
struct Stage {
  static constexpr int kScaleAt = kUnitKeys * D / 2, kBytes = kUnitKeys * D * 9 / 16;
};
static_assert(kUnitKeys == 64 && kUnitKeys == kPage, "fetch copies, and score_kernel's four tiles read, 64 keys of two pages at most");
template <int D>
struct ScoreWarp {
  uint8_t stage[kStages][Stage<D>::kBytes];
  float part[kUnitKeys * 4];  // score of every quarter of a key
};
__device__ __forceinline__ void copy16(void* to, const void* from, bool there) {  // zeros if it is not there
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ptx::smem_u32(to)), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(void* to, const void* from, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(ptx::smem_u32(to)), "l"(from), "r"(there ? 4 : 0) : "memory");
}
// Starts the copies of keys base to base + 63 of a sequence, zeros for those from `end` on and those of no page.
template <int D>
__device__ __forceinline__ void fetch(const Args& a, uint8_t* stage, int seq, int head, int32_t base, int32_t end, int lane) {
  // (they are of the page of `base` and the next one)
  const int page0 = cache::page_of(a.b, seq, base / kPage), page1 = cache::page_of(a.b, seq, base / kPage + 1);
  const uint8_t* rec = a.cache + (int64_t)head * a.record;
  const int t0 = base % kPage, left = end - base;
  const int here = page0 >= 0 ? left : 0, there = page1 >= 0 ? left : 0, turn = kPage - t0;
  // (where there is no page, an address that is never read)
  const uint8_t* rec0 = rec + (int64_t)max(page0, 0) * a.page_stride;
  const uint8_t* rec1 = rec + (int64_t)max(page1, 0) * a.page_stride;
  const uint8_t *codes0 = rec0 + t0 * (D / 2), *codes1 = rec1 - turn * (D / 2);
  const uint8_t *scales0 = rec0 + cache::k_scale_at(D) + t0 * (D / 16), *scales1 = rec1 + cache::k_scale_at(D) - turn * (D / 16);
  codes0 += 16 * lane, codes1 += 16 * lane, scales0 += 4 * lane, scales1 += 4 * lane;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const int key = (32 * i + lane) / (D / 32);
    const bool first = key < turn;
    copy16(stage + 16 * (32 * i + lane), (first ? codes0 : codes1) + 512 * i, key < (first ? here : there));
  }
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const int key = (32 * i + lane) / (D / 64);
    const bool first = key < turn;
    copy4(stage + Stage<D>::kScaleAt + 4 * (32 * i + lane), (first ? scales0 : scales1) + 128 * i, key < (first ? here : there));
  }
}

// Every unit of `unit` blocks of a row and KV head is a warp's work; the units of all rows stand in one line, head after head,
// that is shared out evenly.  While a warp scores 64 keys in shared memory the next ones are on their way.
template <int D>
__global__ void __launch_bounds__(warps_of(D) * 32) score_kernel(const Args a) {
  constexpr int kWarps = warps_of(D);
  extern __shared__ __align__(16) uint8_t dynamic[];
  __shared__ uint32_t sums[kWarps];
  ScoreWarp<D>* const all_warps = reinterpret_cast<ScoreWarp<D>*>(dynamic);
  int2* const row_of = reinterpret_cast<int2*>(all_warps + kWarps);      // [rows] sequence and tokens
  uint32_t* const line = reinterpret_cast<uint32_t*>(row_of + a.rows);  // [rows + 1] units before every row
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  // (pick_kernel is let go only after this wait, so that it may read what earlier kernels wrote before its own)
  wait_for_earlier();
  allow_next();
  const int each = (a.rows + kWarps * 32 - 1) / (kWarps * 32), r0 = min(a.rows, tid * each), r1 = min(a.rows, r0 + each);
  uint32_t mine = 0;
  for (int r = r0; r < r1; ++r) {
    const int seq = cache::sequence_of(a.b, a.row0 + r);
    row_of[r] = make_int2(seq, tokens_of(a.b, seq, a.row0 + r, a.most));
    line[r] = mine;
    mine += (uint32_t)(blocks_of(row_of[r].y, a.shift) + a.unit - 1) / (uint32_t)a.unit;
  }
  uint32_t upto = mine;
#pragma unroll
  for (int by = 1; by < 32; by *= 2) {
    const uint32_t other = __shfl_up_sync(0xFFFFFFFFu, upto, by);
    if (lane >= by) upto += other;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  uint32_t before = upto - mine, total = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < warp) before += sums[i];
    total += sums[i];
  }
  for (int r = r0; r < r1; ++r) line[r] += before;
  if (tid == 0) line[a.rows] = total;
  __syncthreads();
  if (total == 0) return;

  // (neighbouring shares go to different blocks, so that few units are spread over all SMs)
  const uint32_t all = total * a.hkv, workers = gridDim.x * kWarps, me = warp * gridDim.x + blockIdx.x;
  const uint32_t share = all / workers, more = all % workers;
  uint32_t u = me * share + min(me, more);
  const uint32_t u1 = u + share + (me < more ? 1 : 0);
  if (u >= u1) return;
  ScoreWarp<D>& w = all_warps[warp];
  const int g = lane / 4, quarter = lane % 4;

  // The unit whose keys are fetched: that of `u`, in the row whose units end with `stop`.
  uint32_t stop = u;
  int row = 0, head = 0, seq = 0;
  int32_t first = 0, n_blocks = 0;
  Places p;
  struct Unit {
    float2* bounds;       // of its first block
    int32_t blocks;
    int32_t first, end;   // keys of block `lane`
    int32_t base, last;   // 64 keys from `base` on, of the unit's up to `last`
    int row, head;
  };
  const auto begin = [&]() {
    if (u == stop) {
      head = (int)(u / total);
      const uint32_t place = u - head * total;
      int lo = 0, hi = a.rows;
      while (hi - lo > 1) {
        const int mid = lo + (hi - lo) / 2;
        if (line[mid] <= place) lo = mid;
        else hi = mid;
      }
      stop = u + (line[lo + 1] - place);
      row = a.row0 + lo, seq = row_of[lo].x;
      p = places_of(row_of[lo].y, a.cmp_block, a.cmp_stride, a.shift);
      n_blocks = blocks_of(p.tokens, a.shift);
      first = (int32_t)(place - line[lo]) * a.unit;
    }
    Unit x;
    x.bounds = a.bounds + ((int64_t)(row - a.row0) * a.hkv + head) * a.blocks + first;
    x.blocks = min(a.unit, n_blocks - first);
    x.first = first_key(p, first + min(lane, x.blocks));
    x.end = __shfl_down_sync(0xFFFFFFFFu, x.first, 1);
    x.base = __shfl_sync(0xFFFFFFFFu, x.first, 0), x.last = __shfl_sync(0xFFFFFFFFu, x.first, x.blocks);
    x.row = row, x.head = head;
    ++u, first += a.unit;
    return x;
  };

  Unit now = begin();
  fetch<D>(a, w.stage[0], seq, head, now.base, now.last, lane);
  asm volatile("cp.async.commit_group;" ::: "memory");
  uint32_t bq[D / 8];
  int of_row = -1, of_head = -1, stage = 0;
  float size = 0.0f, score = 0.0f;  // error of a key's score in units of a scale; score of block `lane`
  uint32_t even = 0, odd = 0;
  while (true) {
    const bool whole = now.base + kUnitKeys >= now.last, more = !whole || u < u1;
    Unit next = now;
    if (whole && more) next = begin();
    else next.base += kUnitKeys;
    if (more) fetch<D>(a, w.stage[stage ^ 1], seq, head, next.base, next.last, lane);
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (now.row != of_row || now.head != of_head) {
      size = load_query<D>(a, bq, now.row, now.head, lane);
      of_row = now.row, of_head = now.head;
    }
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    const uint8_t* codes = w.stage[stage] + quarter * (D / 8);
    const uint8_t* scales = w.stage[stage] + Stage<D>::kScaleAt + quarter * (D / 64);
#pragma unroll
    for (int tile = 0; tile < 4; ++tile) {  // keys 16 tile + g and 8 more
      Quarter<D> k[2];
      load_quarter<D>(k[0], codes, scales, 16 * tile + g);
      load_quarter<D>(k[1], codes, scales, 16 * tile + 8 + g);
      float sum[2] = {}, scale[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 x = scale_values<0>(k[h].scale), y = D > 128 ? scale_values<1>(k[h].scale) : make_float2(0.0f, 0.0f);
        scale[h][0] = x.x, scale[h][1] = x.y, scale[h][2] = y.x, scale[h][3] = y.y;
      }
#pragma unroll
      for (int group = 0; group < D / 64; ++group) {
        float c[4] = {};
#pragma unroll
        for (int i = 2 * group; i < 2 * group + 2; ++i) {  // eight codes of both keys: two steps of the tensor core
          const uint32_t x = k[0].code[i], y = k[1].code[i];
          cache::mma(c, cache::decode_byte<0>(x), cache::decode_byte<0>(y), cache::decode_byte<1>(x), cache::decode_byte<1>(y),
                     bq[4 * i], bq[4 * i + 1]);
          cache::mma(c, cache::decode_byte<2>(x), cache::decode_byte<2>(y), cache::decode_byte<3>(x), cache::decode_byte<3>(y),
                     bq[4 * i + 2], bq[4 * i + 3]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          sum[h] = fmaf(scale[h][group], c[2 * h] + c[2 * h + 1], sum[h]);
        }
      }
      // the largest scales: lower bytes of halves, and upper ones (whatever is below them)
      const uint32_t two = __byte_perm(k[0].scale, k[1].scale, 0x5410);
      even = __vmaxu2(even, two & 0x00FF00FFu);
      if (D > 64) odd = __vmaxu2(odd, two);
      if (D > 128) even = __vmaxu2(even, __byte_perm(k[0].scale, k[1].scale, 0x7632));
      w.part[(16 * tile + g) * 4 + quarter] = sum[0];
      w.part[(16 * tile + 8 + g) * 4 + quarter] = sum[1];
    }
    __syncwarp();
    if (lane < now.blocks)
      for (int32_t i = max(now.first, now.base); i < min(now.end, now.base + kUnitKeys); ++i) {
        const float4 x = reinterpret_cast<const float4*>(w.part)[i - now.base];
        score += (x.x + x.y) + (x.z + x.w);
      }
    if (whole) {
      const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, max(max(even & 0xFFFFu, even >> 16), max(odd >> 8 & 0xFFu, odd >> 24)));
      if (lane < now.blocks) {
        const float error = size * (float)(now.end - now.first) * scale_values<0>(top).x;
        const float least = score - error, most = score + error;
        // (what may not be finite has to be looked at)
        const bool fine = top < 0xF8u && fabsf(least) < kHuge && fabsf(most) < kHuge;
        now.bounds[lane] = fine ? make_float2(least, most) : make_float2(-kHuge, kHuge);
      }
      score = 0.0f, even = odd = 0;
    }
    if (!more) break;
    __syncwarp();
    now = next, stage ^= 1;
  }
}

// ------------------------------------------------------------------ exact scores
// What a (row, head)'s exact scores are made from: nothing (a value of the query is no number), whole numbers, fp64.
enum class Query { kNone, kWhole, kWide };
struct alignas(16) Bytes {
  uint32_t x[4];
};
template <int D>
struct Exact {
  Bytes limb[D / 16][kLimbs + 1];  // bytes of the query, the lowest first, of the 16 dims of a group, four to a word (and room
                                  // that puts what the threads of a key read at once into different banks)
  uint2 start[D / 16];             // what the sums of a group begin with: 12 of every code too many, taken off
  union {
    int32_t sum[2][D];            // of the heads: whole parts and fractions
    double wide[D];               // the sum itself, where the bytes do not hold it
  };
  uint32_t top;
  Query query;                    // (here and not in a register, of which the small blocks have none left)
};

// fp64 of an integer, without a conversion: its bits in the mantissa of 2^52 + 2^31 + x.
__device__ __forceinline__ double whole(int32_t x) {
  return __hiloint2double(0x43300000, x ^ 0x80000000) - 4503601774854144.0;
}
// fp64 of a scale byte (NaN for those that stand for no number).
__device__ __forceinline__ double scale_of(uint32_t byte) {
  if (byte < 8) return (double)byte * 7.62939453125e-06;  // (below the smallest normal scale: eighths of 2^-14)
  return __hiloint2double((int)scale_high(byte), 0);
}

// The sum of a (row, head)'s query heads as whole numbers of a power of two, so that the largest stays below 2^46, cut into six
// signed bytes.  With 16 heads that holds all values from 2^-34 of the largest on in bf16 (8 bits of 42), and every fp16 number.
// Where a value does not fit (channels that are further apart), the sum is kept in fp64 instead.  By all threads: kParts of them
// share the heads of two dims; the first kAhead of each are loaded beforehand.
template <int D, int THREADS>
struct Heads {
  static constexpr int kParts = THREADS / (D / 2), kAhead = 1024 / THREADS;
  const uint16_t* q;
  int64_t step;
  int pair, part, n;  // n: heads of this thread
  uint32_t first[kAhead];
  __device__ __forceinline__ Heads(const Args& a, int row, int head) {
    pair = threadIdx.x % (D / 2), part = threadIdx.x / (D / 2);
    q = static_cast<const uint16_t*>(a.q) + (int64_t)row * a.q_row + ((int64_t)head * a.group + part) * a.q_head + 2 * pair;
    step = kParts * a.q_head;
    n = part < kParts && part < a.group ? (a.group - part + kParts - 1) / kParts : 0;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) first[i] = i < n ? __ldcg(reinterpret_cast<const uint32_t*>(q + i * step)) : 0;
  }
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) f(first[i]);  // (zeros behind the last)
#pragma unroll 1
    for (int i = kAhead; i < n; ++i) f(__ldcg(reinterpret_cast<const uint32_t*>(q + i * step)));
  }
};
template <int D, int THREADS>
__device__ __forceinline__ Query prepare_exact(const Args& a, Exact<D>& w, const Heads<D, THREADS>& heads) {
  constexpr int kParts = Heads<D, THREADS>::kParts;
  const int tid = threadIdx.x, pair = heads.pair, part = heads.part;
  uint32_t top = 0;
  heads.each([&](uint32_t two) { top = __vmaxu2(top, two & 0x7FFF7FFFu); });
  if (tid == 0) w.top = 0;
  for (int i = tid; i < 2 * D; i += THREADS) w.sum[0][i] = 0;
  __syncthreads();
  top = __reduce_max_sync(0xFFFFFFFFu, max(top & 0xFFFFu, top >> 16));
  if (tid % 32 == 0) atomicMax(&w.top, top);
  __syncthreads();
  top = w.top;
  if (top >= (a.q_half ? 0x7C00u : 0x7F80u)) return Query::kNone;
  // x 2^up: below 2^(bits - 22), its fraction to 22 bits
  const int up = a.bits - 22 + 126 - max((int)(__float_as_uint(query_value(a, top)) >> 23), 1);
  const float up0 = __uint_as_float((uint32_t)(127 + up / 2) << 23), up1 = __uint_as_float((uint32_t)(127 + up - up / 2) << 23);
  int32_t upper[2] = {}, lower[2] = {};
  // (1.5 2^23: what it is added to, below 2^22, is rounded to a whole number, which the lowest bits then are)
  constexpr float kRound = 12582912.0f;
  bool fits = up >= -16;  // (below that the smallest numbers of bf16 could become 0)
  heads.each([&](uint32_t two) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float value = query_value(a, i == 0 ? two & 0xFFFFu : two >> 16);
      const float x = value * up0 * up1, w0 = __fadd_rn(x, kRound);
      const float rest = __fmul_rn(__fsub_rn(x, __fsub_rn(w0, kRound)), 4194304.0f), w1 = __fadd_rn(rest, kRound);
      upper[i] += __float_as_int(w0) - __float_as_int(kRound);
      lower[i] += __float_as_int(w1) - __float_as_int(kRound);
      fits = fits && __fsub_rn(w1, kRound) == rest;
    }
  });
  if (part < kParts)
#pragma unroll
    for (int i = 0; i < 2; ++i) atomicAdd(&w.sum[0][2 * pair + i], upper[i]), atomicAdd(&w.sum[1][2 * pair + i], lower[i]);
  if (__syncthreads_or(!fits)) {
    if (part == 0) {  // (one thread for two dims, so that the heads are added in their order)
      double sum[2] = {0.0, 0.0};
#pragma unroll 1
      for (int g = 0; g < a.group; ++g) {
        const uint32_t two = __ldcg(reinterpret_cast<const uint32_t*>(heads.q + g * a.q_head));
        sum[0] += (double)query_value(a, two & 0xFFFFu), sum[1] += (double)query_value(a, two >> 16);
      }
      w.wide[2 * pair] = sum[0], w.wide[2 * pair + 1] = sum[1];
    }
    return Query::kWide;
  }
  for (int d = tid; d < D; d += THREADS) {
    int64_t x = (int64_t)w.sum[0][d] * 4194304 + w.sum[1][d];
#pragma unroll
    for (int l = 0; l < kLimbs; ++l) reinterpret_cast<int8_t*>(&w.limb[d / 16][l])[d % 16] = next_byte(x);
  }
  __syncthreads();
  if (tid < D / 16) {
    const auto limb = w.limb[tid];
    w.start[tid] = make_uint2(too_many(limb[0].x, limb[1].x, limb[2].x), too_many(limb[3].x, limb[4].x, limb[5].x));
  }
  return Query::kWhole;  // (the caller meets before the sums are read)
}

// Scores of two keys, by four threads, each with a quarter of both; all of them get them.
template <int D>
__device__ __forceinline__ void dot(const Exact<D>& w, const Quarter<D> (&k)[2], int quarter, double (&x)[2]) {
  double upper[2] = {0.0, 0.0}, lower[2] = {0.0, 0.0};
#pragma unroll
  for (int j = 0; j < D / 64; ++j) {
    const int g = quarter * (D / 64) + j;
    uint32_t c[2][4];
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[y][i] = decode4(k[y].code[2 * j + i / 2] >> i % 2 * 16);
    // (a sum is at most 128 * 12 * 16 in size, so that three of them, a byte apart, fit 32 bits)
    uint32_t up[2] = {}, lo[2] = {};  // (those with 12 of every code too many may wrap around)
#pragma unroll
    for (int l = kLimbs - 1; l >= 0; --l) {
      const Bytes q = w.limb[g][l];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        uint32_t& sum = l >= kLimbs / 2 ? up[y] : lo[y];
        sum = add_group(sum, c[y], q.x);
      }
    }
    const uint2 start = w.start[g];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const double s = scale_of(k[y].scale >> 8 * j & 255u);
      upper[y] = fma(s, whole((int)(up[y] + start.y)), upper[y]);
      lower[y] = fma(s, whole((int)(lo[y] + start.x)), lower[y]);
    }
  }
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    x[y] = fma(upper[y], 16777216.0, lower[y]);
    x[y] += __shfl_xor_sync(0xFFFFFFFFu, x[y], 1);
    x[y] += __shfl_xor_sync(0xFFFFFFFFu, x[y], 2);
  }
}

// The same from the sums in fp64.  (In a loop: unrolled it is seldom run code between that which always is, and took 41
// sequences with drafts 1 % more.)
template <int D>
__device__ __forceinline__ void dot_wide(const Exact<D>& w, const Quarter<D> (&k)[2], int quarter, double (&x)[2]) {
  x[0] = x[1] = 0.0;
#pragma unroll
  for (int j = 0; j < D / 64; ++j) {
    const double* q = w.wide + (quarter * (D / 64) + j) * 16;
    double sum[2] = {0.0, 0.0};
#pragma unroll 1
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const uint32_t four = decode4((i < 2 ? k[y].code[2 * j] : k[y].code[2 * j + 1]) >> i % 2 * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[y] = fma(q[4 * i + e], whole((int)(four >> 8 * e & 255) - kCodeZero), sum[y]);
      }
#pragma unroll
    for (int y = 0; y < 2; ++y) x[y] = fma(scale_of(k[y].scale >> 8 * j & 255u), sum[y], x[y]);
  }
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    x[y] += __shfl_xor_sync(0xFFFFFFFFu, x[y], 1);
    x[y] += __shfl_xor_sync(0xFFFFFFFFu, x[y], 2);
  }
}

// Adds `n` blocks with their scores to a list, by all threads.  Each block has a.keys places, four threads score the keys of two
// places, and one sums those of a block, in their order.
struct List {
  uint64_t* rank;
  uint32_t* index;
};
template <int D, int THREADS>
__device__ __forceinline__ void score_blocks(const Args& a, const Exact<D>& w, const Places& p, int seq, int head,
                                             const int32_t* pages, const uint16_t* blocks, int base, uint32_t n, const List& list,
                                             uint32_t at, double* scores) {
  const int tid = threadIdx.x, quarter = tid % 4;
  for (uint32_t e0 = 0; e0 < n; e0 += a.at_once) {
    const uint32_t some = min(n - e0, (uint32_t)a.at_once), places = some * a.keys;
    for (uint32_t t0 = tid / 4; t0 - tid / 4 < places; t0 += THREADS / 2) {
      Quarter<D> k[2] = {};
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint32_t t = t0 + x * (THREADS / 4), e = t * a.per_key >> 20;  // t / a.keys
        // (two threads find where the block begins, two where it ends)
        const int32_t block = t < places ? base + blocks[e0 + e] : 0;
        const int32_t bound = first_key(p, block + quarter % 2);
        const int32_t i = __shfl_sync(0xFFFFFFFFu, bound, tid % 32 / 4 * 4) + (int32_t)(t - e * a.keys);
        const bool in = i < __shfl_sync(0xFFFFFFFFu, bound, tid % 32 / 4 * 4 + 1) && t < places;
        const int page = !in ? -1 : i / kPage < kHeldPages ? pages[i / kPage] : cache::page_of(a.b, seq, i / kPage);
        const uint8_t* rec = a.cache + (int64_t)page * a.page_stride + (int64_t)head * a.record;
        if (page >= 0)
          load_quarter<D>(k[x], rec + quarter * (D / 8), rec + cache::k_scale_at(D) + quarter * (D / 64), i % kPage);
      }
      double score[2];  // (0 of a place without a key, and of a key of no page)
      if (w.query == Query::kWide) dot_wide<D>(w, k, quarter, score);
      else dot<D>(w, k, quarter, score);
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (quarter == x && t0 + x * (THREADS / 4) < places) scores[t0 + x * (THREADS / 4)] = score[x];
    }
    __syncthreads();
    for (uint32_t e = tid; e < some; e += THREADS) {
      double score = 0.0;
      for (int j = 0; j < a.keys; ++j) score += scores[e * a.keys + j];
      list.rank[at + e0 + e] = rank_of(w.query != Query::kNone ? score : __longlong_as_double(0x7FF8000000000000ll));
      list.index[at + e0 + e] = (uint32_t)(base + blocks[e0 + e]);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ the best of a row
// From the L2: what is read while score_kernel still runs, since an L1 may hold what the kernels before that one have replaced.
struct LoadPastL1 {
  NSA_HD int32_t operator()(const int32_t* p) const {
#ifdef __CUDA_ARCH__
    return __ldcg(p);
#else
    return *p;
#endif
  }
};
__host__ __device__ constexpr int list_size(int n_sel) { return n_sel + kAdded; }
__host__ __device__ constexpr int list_bytes(int n_sel) { return 24 * list_size(n_sel); }  // two lists
// Numbers that compare like fp32, and back.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u >> 31 ? u & 0x7FFFFFFFu : ~u); }
// The bin of a bound: never a lower one for a larger bound.
__device__ __forceinline__ int bin_of(float x, float low, float per, int bins) { return max(0, min(bins - 1, (int)((x - low) * per))); }

template <int D, int THREADS, int PER_SM>
__global__ void __launch_bounds__(THREADS, PER_SM) pick_kernel(const Args a) {
  constexpr int kChecked = checked(THREADS), kBins = 4 * THREADS;
  extern __shared__ __align__(16) uint8_t dynamic[];
  __shared__ Exact<D> w;
  __shared__ double scores[kKeys];
  __shared__ uint16_t found[kChecked];
  __shared__ int32_t pages[kHeldPages];
  __shared__ __align__(16) uint32_t count[kBins];
  __shared__ uint32_t s_least[THREADS / 32], s_most[THREADS / 32], sums[THREADS / 32], s_bin, s_found;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int size = list_size(a.n_sel);
  List list = {reinterpret_cast<uint64_t*>(dynamic), reinterpret_cast<uint32_t*>(dynamic + 16 * size)};
  List other = {list.rank + size, list.index + size};
  allow_next();
  // What earlier kernels wrote is read before score_kernel has ended: it has waited for them before this one could begin.
  const int64_t unit = blockIdx.x;
  const int row = a.row0 + (int)(unit / a.hkv), head = (int)(unit % a.hkv);
  const float2* bounds = a.bounds + unit * a.blocks;
  int32_t* sel = a.sel + ((int64_t)a.row0 * a.hkv + unit) * a.n_sel;
  const Heads<D, THREADS> heads(a, row, head);
  const int seq = cache::sequence_by_32(
      a.b, row,
      [&](int lo, int step, int hi) {
        return __ballot_sync(0xFFFFFFFFu, lane * step < hi - lo && LoadPastL1()(a.b.cu + lo + lane * step) <= row);
      },
      LoadPastL1());
  const int32_t tokens = tokens_of(a.b, seq, row, a.most, LoadPastL1()), n = blocks_of(tokens, a.shift);
  const uint32_t wanted = min((uint32_t)a.n_sel, (uint32_t)n);
  const Places p = places_of(tokens, a.cmp_block, a.cmp_stride, a.shift);
  for (int i = tid; i < min(kHeldPages, (p.n + kPage - 1) / kPage); i += THREADS) pages[i] = cache::page_of(a.b, seq, i, LoadPastL1());
  if (tid == 0) s_found = 0;
  const Query query = prepare_exact<D, THREADS>(a, w, heads);
  if (tid == 0) w.query = query;
  __syncthreads();
  wait_for_earlier();
  // (all of them: in a cu_seqlens out of order score_kernel may have taken the row for another sequence's)
  for (int i = tid; i < a.n_sel; i += THREADS) sel[i] = -1;
  if (n == 0) return;

  uint32_t kept = 0;
  for (int i0 = 0;; i0 += kChecked) {
    // The lower bounds are counted in bins; the n_sel-th largest lies in bin `edge`, so a block whose upper bound is in a bin
    // below that is none of the best.  (256 threads have 1024 bins: mostly one or two blocks too many.)
    constexpr int kEach = kChecked / THREADS;
    const int here = min(n - i0, kChecked);
    float2 x[kEach];
    uint32_t least = 0xFFFFFFFFu, most = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = j * THREADS + tid;
      x[j] = i < here ? bounds[i0 + i] : make_float2(-kHuge, -kHuge);
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (x[j].x > -kHuge) least = min(least, ordered(x[j].x)), most = max(most, ordered(x[j].x));
    float low = 0.0f, per = 0.0f;
    int edge = 0;
    if (here > (int)wanted) {
      least = __reduce_min_sync(0xFFFFFFFFu, least), most = __reduce_max_sync(0xFFFFFFFFu, most);
      if (lane == 0) s_least[warp] = least, s_most[warp] = most;
      reinterpret_cast<uint4*>(count)[tid] = make_uint4(0, 0, 0, 0);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < THREADS / 32; ++i) least = min(least, s_least[i]), most = max(most, s_most[i]);
      if (least < most) {
        low = unordered(least);
        per = (float)kBins / (unordered(most) - low);  // (0 if that is beyond fp32: one bin)
      }
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        if (j * THREADS + tid < here) atomicAdd(&count[bin_of(x[j].x, low, per, kBins)], 1u);
      __syncthreads();
      // four bins of a thread, the largest first
      const uint4 c = reinterpret_cast<const uint4*>(count)[THREADS - 1 - tid];
      const uint32_t mine = c.x + c.y + c.z + c.w;
      uint32_t upto = mine;
#pragma unroll
      for (int by = 1; by < 32; by *= 2) {
        const uint32_t before = __shfl_up_sync(0xFFFFFFFFu, upto, by);
        if (lane >= by) upto += before;
      }
      if (lane == 31) sums[warp] = upto;
      __syncthreads();
      uint32_t at = upto - mine;
#pragma unroll
      for (int i = 0; i < THREADS / 32; ++i) at += i < warp ? sums[i] : 0;
      if (at < wanted && wanted <= at + mine) {
        const int bin = 4 * (THREADS - 1 - tid);
        s_bin = wanted <= at + c.w ? bin + 3 : wanted <= at + c.w + c.z ? bin + 2 : wanted <= at + c.w + c.z + c.y ? bin + 1 : bin;
      }
      __syncthreads();
      edge = (int)s_bin;
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = j * THREADS + tid;
      if (i < here && bin_of(x[j].y, low, per, kBins) >= edge) found[atomicAdd(&s_found, 1u)] = (uint16_t)i;
    }
    __syncthreads();

    // Exact scores of the blocks that are left; where they are many, only the best so far are kept.
    const uint32_t n_found = s_found;
    for (uint32_t f0 = 0;;) {
      const uint32_t some = min(n_found - f0, (uint32_t)kAdded), in = kept + some;
      score_blocks<D, THREADS>(a, w, p, seq, head, pages, found + f0, i0, some, list, kept, scores);
      f0 += some;
      const bool whole = f0 == n_found, last = whole && i0 + kChecked >= n;
      for (uint32_t e0 = tid / 8; e0 - tid / 8 < in; e0 += THREADS / 8) {  // 8 threads for an entry
        const uint32_t e = min(e0, in - 1);
        const uint64_t key = list.rank[e];
        const uint32_t block = list.index[e];
        uint32_t better = 0;
        for (uint32_t j = tid % 8; j < in; j += 8) better += list.rank[j] > key || (list.rank[j] == key && list.index[j] < block);
#pragma unroll
        for (int by = 4; by > 0; by /= 2) better += __shfl_xor_sync(0xFFFFFFFFu, better, by);
        if (tid % 8 != 0 || e0 >= in || better >= wanted) continue;
        if (last) sel[better] = (int32_t)block;
        else other.rank[better] = key, other.index[better] = block;
      }
      if (last) return;
      kept = min(in, wanted);
      const List swap = list;
      list = other, other = swap;
      __syncthreads();
      if (whole) break;
    }
    if (tid == 0) s_found = 0;
    __syncthreads();
  }
}

}  // namespace cache_select
}  // namespace nsa
