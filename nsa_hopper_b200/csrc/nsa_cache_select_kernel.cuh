// Block selection for single tokens: the best blocks of a row's sequence by the scores of its query against the compressed
// keys of a 4-bit cache,
//     s(block) = sum over the compressed keys i of the block of (sum_g q_g) . k_i,
// the n_sel best, the best first, ties to the lowest block.
//
// Ranks are all that comes out, and where two scores are close the wrong sum turns them around.  So the scores are sums in 64
// bits of exact parts: a key's codes (doubled) are whole numbers up to 12, the query becomes whole numbers too (below), and
// the 16 products of a group that share a scale are added in integers; only scale times group sum is added in fp64.  The work
// of that is dot products of four bytes (dp4a), one for each byte of the query and four codes.
//
// The query's heads are added as whole numbers of 2^-k, with k such that the largest head's sum stays below 2^46: values down to
// 2^-33 of the largest are exact in bf16 (2^-30 in fp16), smaller ones off by less than 2^-40 of it at 16 heads.  The sum is cut
// into six signed bytes, of which the lower two are mostly zero in every place; then four are used.
//
// What bounds it: a key costs 9/16 d bytes.  DRAM would deliver a page of 64 keys with d = 128 to an SM in 1.4 thousand
// cycles/148 ... (measured figures: see the launches below).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "nsa_cache_select_index.h"
#include "nsa_programmatic.cuh"

namespace nsa {
namespace cache_select {

constexpr int kWarps = 8;
constexpr int kLimbs = 6;
constexpr int kMaxRows = 8192;    // of a launch: their units' places fill 32 KB of shared memory
constexpr int kUnitKeys = 64;     // keys of a unit, about
constexpr int kUnitBlocks = 31;   // its blocks at most: a lane for each and one for the end
constexpr int kMaxGroup = 256;    // query heads of a KV head
constexpr int kMaxSel = 1024;
constexpr int kPickThreads = 256;

struct Args {
  Batch b;              // the compressed cache's page table; lens: tokens of the sequences
  const void* q;        // [n_rows, Hq, D], unit stride along D
  int64_t q_row, q_head;
  const uint8_t* cache;
  int64_t page_stride;
  uint64_t* score;      // [n_rows, Hkv, blocks], as keys that compare like the scores
  int32_t* sel;         // [n_rows, Hkv, n_sel]
  int32_t hkv, group, n_sel;
  int32_t shift;        // of a block's tokens
  int32_t blocks;       // blocks of a row, at most
  int32_t unit;         // blocks of a unit
  int32_t most;         // tokens of a row, at most
  int32_t cmp_block, cmp_stride;
  int32_t record;       // bytes
  int32_t q_half;
  int32_t bits;         // of a query head's value: its largest is below 2^bits
  int32_t row0, rows;   // rows of this launch
};

// A number that compares like the score; what is no number, or infinite, comes last.
__device__ __forceinline__ uint64_t rank_of(double x) {
  if (!(fabs(x) < __longlong_as_double(0x7FF0000000000000ll))) return 0;
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);  // (-0 is 0)
  return u >> 63 ? ~u : u | 1ull << 63;
}

// fp64 of an integer, without a conversion: its bits in the mantissa of 2^52 + 2^31 + x.
__device__ __forceinline__ double whole(int32_t x) {
  return __hiloint2double(0x43300000, x ^ 0x80000000) - 4503601774854144.0;
}
// fp64 of a scale byte (NaN for those that stand for no number).
__device__ __forceinline__ double scale_of(uint32_t byte) {
  if (byte < 8) return (double)byte * 7.62939453125e-06;  // (below the smallest normal scale: eighths of 2^-14)
  return __hiloint2double(byte < 0xF8 ? (int)((byte << 17) + (1008u << 20)) : 0x7FF80000, 0);
}

template <int D>
struct Warp {
  int4 limb[D / 16][kLimbs];       // of the 16 dims of a group, four to a word
  int32_t start[D / 16][8];        // what the sums of a group begin with: 12 of every code too many, taken off
  double key[kUnitKeys];
};

// Sums the query heads of (row, head) and cuts them into bytes; returns the bytes that are not zero throughout (4 or 6), 0 if a
// value is not finite.
template <int D>
__device__ __forceinline__ int prepare(const Args& a, Warp<D>& w, int row, int head, int lane) {
  constexpr int N = D / 32;  // dims of a lane
  const uint16_t* q = static_cast<const uint16_t*>(a.q) + (int64_t)row * a.q_row + (int64_t)head * a.group * a.q_head + lane * N;
  uint32_t top = 0;
  for (int g = 0; g < a.group; ++g)
#pragma unroll
    for (int i = 0; i < N / 2; ++i) top = __vmaxu2(top, reinterpret_cast<const uint32_t*>(q + g * a.q_head)[i] & 0x7FFF7FFFu);
  top = __reduce_max_sync(0xFFFFFFFFu, max(top & 0xFFFFu, top >> 16));
  if (top >= (a.q_half ? 0x7C00u : 0x7F80u)) return 0;
  const float largest = a.q_half ? __half2float(__ushort_as_half((unsigned short)top)) : __uint_as_float(top << 16);
  // x 2^up: below 2^(bits - 22), its fraction to 22 bits
  const int up = a.bits - 22 + 126 - max((int)(__float_as_uint(largest) >> 23), 1);
  const float up0 = __uint_as_float((uint32_t)(127 + up / 2) << 23), up1 = __uint_as_float((uint32_t)(127 + up - up / 2) << 23);
  int32_t upper[N] = {}, lower[N] = {};
  for (int g = 0; g < a.group; ++g)
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint32_t two = reinterpret_cast<const uint32_t*>(q + g * a.q_head)[i];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t bits = j == 0 ? two & 0xFFFFu : two >> 16;
        const float x = (a.q_half ? __half2float(__ushort_as_half((unsigned short)bits)) : __uint_as_float(bits << 16)) * up0 * up1;
        const float whole_part = rintf(x);
        upper[2 * i + j] += (int)whole_part;
        lower[2 * i + j] += __float2int_rn((x - whole_part) * 4194304.0f);
      }
    }
  uint32_t low = 0;
  int8_t* bytes = reinterpret_cast<int8_t*>(w.limb);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    int64_t x = (int64_t)upper[i] * 4194304 + lower[i];
    const int d = lane * N + i;
#pragma unroll
    for (int l = 0; l < kLimbs; ++l) {  // signed bytes, the lowest first
      const int8_t byte = (int8_t)x;
      x = (x - byte) >> 8;
      bytes[((d / 16) * kLimbs + l) * 16 + d % 16] = byte;
      if (l < 2) low |= (uint8_t)byte;
    }
  }
  __syncwarp();
  for (int i = lane; i < D / 16 * kLimbs; i += 32) {
    const int4 v = w.limb[i / kLimbs][i % kLimbs];
    const int ones = 0x01010101;
    w.start[i / kLimbs][i % kLimbs] = -12 * __dp4a(v.x, ones, __dp4a(v.y, ones, __dp4a(v.z, ones, __dp4a(v.w, ones, 0))));
  }
  const int limbs = __reduce_or_sync(0xFFFFFFFFu, low) != 0 ? 6 : 4;
  __syncwarp();
  return limbs;
}

// Four codes, doubled and 12 more: whole numbers 0 to 24 in four bytes.
__device__ __forceinline__ int decode4(uint32_t codes) {
  // (a selector whose upper bit is set gives the sign of the byte in all its bits, which is 0 for these)
  uint32_t plus, minus;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(plus) : "r"(0x03020100u), "r"(0x0C080604u), "r"(codes));
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(minus) : "r"(0x03020100u), "r"(0x0C080604u), "r"(codes ^ 0x8888u));
  return (int)(0x0C0C0C0Cu + plus - minus);
}

// A key's codes and scales.
template <int D>
struct Key {
  uint4 code[D / 32];
  uint32_t scale[D / 64];
};
template <int D>
__device__ __forceinline__ bool load_key(const Args& a, Key<D>& k, int seq, int head, int i) {
  const int page = cache::page_of(a.b, seq, i / kPage);
  if (page < 0) return false;
  const uint8_t* rec = a.cache + (int64_t)page * a.page_stride + (int64_t)head * a.record;
  const int t = i % kPage;
#pragma unroll
  for (int j = 0; j < D / 32; ++j) k.code[j] = reinterpret_cast<const uint4*>(rec + t * (D / 2))[j];
#pragma unroll
  for (int j = 0; j < D / 64; ++j) k.scale[j] = reinterpret_cast<const uint32_t*>(rec + cache::k_scale_at(D) + t * (D / 16))[j];
  return true;
}

// Scores of two keys.
template <int D, int LIMBS>
__device__ __forceinline__ void dot(const Warp<D>& w, const Key<D> (&k)[2], double (&out)[2]) {
  constexpr int L0 = kLimbs - LIMBS, HALF = LIMBS / 2;
  double upper[2] = {0.0, 0.0}, lower[2] = {0.0, 0.0};
#pragma unroll
  for (int g = 0; g < D / 16; ++g) {
    int sum[2][LIMBS];
#pragma unroll
    for (int l = 0; l < LIMBS; ++l) sum[0][l] = sum[1][l] = w.start[g][L0 + l];
    int c[2][4];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const uint4& v = k[x].code[g / 2];
      const uint32_t w0 = g % 2 == 0 ? v.x : v.z, w1 = g % 2 == 0 ? v.y : v.w;
      c[x][0] = decode4(w0), c[x][1] = decode4(w0 >> 16), c[x][2] = decode4(w1), c[x][3] = decode4(w1 >> 16);
    }
#pragma unroll
    for (int l = 0; l < LIMBS; ++l) {
      const int4 q = w.limb[g][L0 + l];
#pragma unroll
      for (int x = 0; x < 2; ++x)
        sum[x][l] = __dp4a(c[x][0], q.x, __dp4a(c[x][1], q.y, __dp4a(c[x][2], q.z, __dp4a(c[x][3], q.w, sum[x][l]))));
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      // (a sum is at most 128 * 12 * 16 in size, so that three of them, a byte apart, fit 32 bits)
      int up = 0, lo = 0;
#pragma unroll
      for (int l = HALF - 1; l >= 0; --l) up = up * 256 + sum[x][HALF + l], lo = lo * 256 + sum[x][l];
      const double s = scale_of(k[x].scale[g / 4] >> (g % 4 * 8) & 255u);
      upper[x] = fma(s, whole(up), upper[x]);
      lower[x] = fma(s, whole(lo), lower[x]);
    }
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) out[x] = fma(upper[x], (double)(1 << 8 * HALF), lower[x]);
}

// Every unit of `unit` blocks of a row and KV head is a warp's work; the units of all rows stand in one line, head after head,
// that is shared out evenly.
template <int D>
__global__ void __launch_bounds__(kWarps * 32) score_kernel(const Args a) {
  extern __shared__ __align__(16) uint8_t sm[];
  __shared__ uint32_t sums[kWarps];
  Warp<D>* warps = reinterpret_cast<Warp<D>*>(sm);
  uint32_t* line = reinterpret_cast<uint32_t*>(warps + kWarps);  // [rows + 1] units before every row
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  start_in_order();
  // units before every row
  const int each = (a.rows + kWarps * 32 - 1) / (kWarps * 32), r0 = min(a.rows, tid * each), r1 = min(a.rows, r0 + each);
  uint32_t mine = 0;
  for (int r = r0; r < r1; ++r) {
    const int32_t blocks = blocks_of(tokens_of(a.b, a.row0 + r, a.most), a.shift);
    line[r] = mine;
    mine += (uint32_t)(blocks + a.unit - 1) / (uint32_t)a.unit;
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
  for (int i = 0; i < kWarps; ++i) {
    if (i < warp) before += sums[i];
    total += sums[i];
  }
  for (int r = r0; r < r1; ++r) line[r] += before;
  if (tid == 0) line[a.rows] = total;
  __syncthreads();
  if (total == 0) return;

  Warp<D>& w = warps[warp];
  const uint32_t all = total * a.hkv, workers = gridDim.x * kWarps, me = blockIdx.x * kWarps + warp;
  const uint32_t share = all / workers, more = all % workers;
  const uint32_t u0 = me * share + min(me, more), u1 = u0 + share + (me < more ? 1 : 0);
  int last_row = -1, last_head = -1, limbs = 0;
  for (uint32_t u = u0; u < u1; ++u) {
    const int head = (int)(u / total);
    const uint32_t place = u - head * total;
    int lo = 0, hi = a.rows;
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      if (line[mid] <= place) lo = mid;
      else hi = mid;
    }
    const int row = a.row0 + lo;
    if (row != last_row || head != last_head) limbs = prepare<D>(a, w, row, head, lane);
    last_row = row, last_head = head;
    const int seq = cache::sequence_of(a.b, row);
    const int32_t tokens = tokens_of(a.b, row, a.most);
    const int32_t n = completed(tokens, a.cmp_block, a.cmp_stride);
    const int32_t first = (int32_t)(place - line[lo]) * a.unit, blocks = min(a.unit, blocks_of(tokens, a.shift) - first);
    // lane j: the first key of block j of the unit
    const int32_t mine_first = first_key(first + min(lane, blocks), tokens, n, a.shift);
    const int32_t mine_end = __shfl_down_sync(0xFFFFFFFFu, mine_first, 1);
    const int32_t begin = __shfl_sync(0xFFFFFFFFu, mine_first, 0), end = __shfl_sync(0xFFFFFFFFu, mine_first, blocks);
    double score = 0.0;
    for (int32_t base = begin; base < end; base += kUnitKeys) {
      Key<D> k[2] = {};
      bool there[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int32_t i = base + x * 32 + lane;
        there[x] = i < end && load_key<D>(a, k[x], seq, head, i);
      }
      double s[2];
      if (limbs == 4) dot<D, 4>(w, k, s);
      else if (limbs == 6) dot<D, 6>(w, k, s);
      else s[0] = s[1] = __longlong_as_double(0x7FF8000000000000ll);
      __syncwarp();
#pragma unroll
      for (int x = 0; x < 2; ++x) w.key[x * 32 + lane] = there[x] ? s[x] : 0.0;
      __syncwarp();
      if (lane < blocks)
        for (int32_t i = max(mine_first, base); i < min(mine_end, base + kUnitKeys); ++i) score += w.key[i - base];
    }
    if (lane < blocks) a.score[((int64_t)row * a.hkv + head) * a.blocks + first + lane] = rank_of(score);
  }
}

// ------------------------------------------------------------------ the best of a row
// The keys that compare like the scores, and below them the blocks in reverse, are cut into 12 digits of 8 bits; a digit's
// counts say in which of its values the n_sel-th best lies, until all that remain are wanted.
__device__ __forceinline__ uint32_t digit_of(uint64_t key, uint32_t block, int level) {
  return (level < 8 ? (uint32_t)(key >> (56 - 8 * level)) : ~block >> (24 - 8 * (level - 8))) & 255u;
}
// Whether the first `level` digits are those of (prefix, prefix_block).
__device__ __forceinline__ int compare_prefix(uint64_t key, uint32_t block, int level, uint64_t prefix, uint32_t prefix_block) {
  const uint64_t x = level == 0 ? 0 : level < 8 ? key >> (64 - 8 * level) : key;
  if (x != prefix) return x > prefix ? 1 : -1;
  if (level <= 8) return 0;
  const uint32_t y = ~block >> (32 - 8 * (level - 8));
  return y != prefix_block ? (y > prefix_block ? 1 : -1) : 0;
}

__global__ void __launch_bounds__(kPickThreads) pick_kernel(const Args a) {
  __shared__ uint32_t count[256];
  __shared__ uint64_t best[kMaxSel];
  __shared__ uint32_t index[kMaxSel];
  __shared__ uint32_t s_digit, s_above, s_in, s_out;
  const int tid = threadIdx.x, lane = tid % 32;
  start_in_order();
  const int64_t unit = blockIdx.x;
  const int row = a.row0 + (int)(unit / a.hkv);
  const uint64_t* score = a.score + ((int64_t)a.row0 * a.hkv + unit) * a.blocks;
  int32_t* sel = a.sel + ((int64_t)a.row0 * a.hkv + unit) * a.n_sel;
  const int32_t n = blocks_of(tokens_of(a.b, row, a.most), a.shift);
  const uint32_t wanted = min((uint32_t)a.n_sel, (uint32_t)n);

  uint64_t prefix = 0;
  uint32_t prefix_block = 0, above = 0, in = (uint32_t)n;  // entries above the prefix, and with it
  int level = 0;
  while (above + in > wanted) {  // (level 12 would tell all entries apart)
    for (int i = tid; i < 256; i += kPickThreads) count[i] = 0;
    __syncthreads();
    for (int i0 = tid - lane; i0 < n; i0 += kPickThreads) {
      const int i = i0 + lane;
      const uint64_t key = i < n ? score[i] : 0;
      const bool live = i < n && compare_prefix(key, (uint32_t)i, level, prefix, prefix_block) == 0;
      const uint32_t digit = digit_of(key, (uint32_t)i, level);
      const uint32_t same = __match_any_sync(0xFFFFFFFFu, live ? digit : 256u);
      if (live && lane == __ffs(same) - 1) atomicAdd(&count[digit], __popc(same));
    }
    __syncthreads();
    if (tid < 32) {  // the digit in which the last wanted entry lies: 8 values of a lane, the largest first
      uint32_t mine = 0, c[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = count[255 - (lane * 8 + j)], mine += c[j];
      uint32_t upto = mine;
#pragma unroll
      for (int by = 1; by < 32; by *= 2) {
        const uint32_t other = __shfl_up_sync(0xFFFFFFFFu, upto, by);
        if (lane >= by) upto += other;
      }
      uint32_t at = above + upto - mine;
      if (at < wanted && wanted <= at + mine) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (at < wanted && wanted <= at + c[j]) s_digit = 255 - (lane * 8 + j), s_above = at, s_in = c[j];
          at += c[j];
        }
      }
    }
    __syncthreads();
    if (level < 8) prefix = prefix << 8 | s_digit;
    else prefix_block = prefix_block << 8 | s_digit;
    above = s_above, in = s_in;
    ++level;
  }
  if (tid == 0) s_out = 0;
  __syncthreads();
  for (int i = tid; i < n; i += kPickThreads) {
    const uint64_t key = score[i];
    if (compare_prefix(key, (uint32_t)i, level, prefix, prefix_block) < 0) continue;
    const uint32_t at = atomicAdd(&s_out, 1u);
    best[at] = key, index[at] = (uint32_t)i;
  }
  __syncthreads();
  for (uint32_t i = tid; i < (uint32_t)a.n_sel; i += kPickThreads) {
    if (i >= wanted) {
      sel[i] = -1;
      continue;
    }
    const uint64_t key = best[i];
    const uint32_t block = index[i];
    uint32_t rank = 0;
    for (uint32_t j = 0; j < wanted; ++j) rank += best[j] > key || (best[j] == key && index[j] < block);
    sel[rank] = (int32_t)block;
  }
}

}  // namespace cache_select
}  // namespace nsa
