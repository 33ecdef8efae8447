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
//     (dot products of four bytes), and only scale times group sum is rounded, in fp64.
//
// Error of the approximation of a key's score, in units of max|k| (six times the largest scale of the unit's keys), with
// S = sum over d and heads of |q| and Q = sum over d of |sum of the heads|: the fp32 sum of G heads (G - 1) 2^-24 S; the two
// fp16 parts of the query 2^-22 Q; the sums of d products (the tensor core cuts each term off below 2^-23 of the largest, twice
// that is allowed for; a running sum is half of Q on average) and of up to 12 group sums, d 2^-22.9 Q together; taken as
// d 2^-22 Q, with room for the sums over keys.
//
// What bounds it: a key costs 9/16 d bytes, 72 at d = 128, and half as many instructions of a thread: DRAM, for large calls.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "nsa_cache_decode.cuh"
#include "nsa_cache_select_index.h"
#include "nsa_programmatic.cuh"

namespace nsa {
namespace cache_select {

constexpr int kWarps = 8;
// Blocks of an SM: the codes of 64 keys in registers leave room for 24 warps, with d = 192 for 16.
__host__ __device__ constexpr int blocks_per_sm(int d) { return d <= 128 ? 3 : 2; }
constexpr int kLimbs = 6;
constexpr int kMaxRows = 8192;    // of a launch: their units' places fill 32 KB of shared memory
constexpr int kUnitKeys = 64;     // keys of a unit, about
constexpr int kUnitBlocks = 31;   // its blocks at most: a lane for each and one for the end
constexpr int kMaxGroup = 256;    // query heads of a KV head
constexpr int kMaxSel = 1024;
constexpr int kPickThreads = 256;
constexpr int kCandidates = 512;  // blocks whose exact scores are kept beside the n_sel best
constexpr int kHeldBounds = 2048; // bounds that pick_kernel keeps in shared memory
constexpr int kBins = 4 * kPickThreads;
constexpr int kChecked = 8;       // blocks that a thread looks at between two meetings
constexpr float kHuge = 3.0e38f;  // bound of what has none

struct Args {
  Batch b;              // the compressed cache's page table; lens: tokens of the sequences
  const void* q;        // [n_rows, Hq, D], unit stride along D
  int64_t q_row, q_head;
  const uint8_t* cache;
  int64_t page_stride;
  float2* bounds;       // [n_rows, Hkv, blocks] lower and upper bound of a block's score
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
// Place t of a record; its codes and its scales are counted from `codes` and `scales`, the record or as much before it.
template <int D>
__device__ __forceinline__ void load_quarter(Quarter<D>& k, const uint8_t* codes, const uint8_t* scales, int t, int q) {
  const uint8_t* code = codes + t * (D / 2) + q * (D / 8);
  const uint8_t* scale = scales + cache::k_scale_at(D) + t * (D / 16) + q * (D / 64);
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
    size += fabsf(sum[i]) * ((float)D * 2.3841858e-07f);  // 2^-22
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

// fp32 of scale byte I of `s` (a finite one of those that are no numbers: the caller looks for those).
template <int I>
__device__ __forceinline__ float scale_value(uint32_t s) {
  return __uint_as_float(s << (20 - 8 * I) & 0x0FF00000u) * 5.192296858534828e33f;  // 2^112
}

// Every unit of `unit` blocks of a row and KV head is a warp's work; the units of all rows stand in one line, head after head,
// that is shared out evenly.
template <int D>
__global__ void __launch_bounds__(kWarps * 32, blocks_per_sm(D)) score_kernel(const Args a) {
  extern __shared__ uint32_t line[];  // [rows + 1] units before every row
  __shared__ __align__(16) float keys[kWarps][kUnitKeys * 4];  // score of every quarter of a key
  __shared__ uint32_t sums[kWarps];
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  // (pick_kernel is let go only after this wait, so that it may read what earlier kernels wrote without one of its own)
  wait_for_earlier();
  allow_next();
  const int each = (a.rows + kWarps * 32 - 1) / (kWarps * 32), r0 = min(a.rows, tid * each), r1 = min(a.rows, r0 + each);
  uint32_t mine = 0;
  for (int r = r0; r < r1; ++r) {
    line[r] = mine;
    mine += (uint32_t)(blocks_of(tokens_of(a.b, a.row0 + r, a.most), a.shift) + a.unit - 1) / (uint32_t)a.unit;
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
  const int g = lane / 4, quarter = lane % 4;
  while (u < u1) {
    // the units of one (row, head)
    const int head = (int)(u / total);
    const uint32_t place = u - head * total;
    int lo = 0, hi = a.rows;
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      if (line[mid] <= place) lo = mid;
      else hi = mid;
    }
    const uint32_t stop = min(u1, u + (line[lo + 1] - place));
    const int row = a.row0 + lo, seq = cache::sequence_of(a.b, row);
    const Places p = places_of(tokens_of(a.b, row, a.most), a.cmp_block, a.cmp_stride, a.shift);
    const int32_t n_blocks = blocks_of(p.tokens, a.shift);
    float2* bounds = a.bounds + ((int64_t)row * a.hkv + head) * a.blocks;
    uint32_t bq[D / 8];
    const float size = load_query<D>(a, bq, row, head, lane);  // error
    int32_t first = (int32_t)(place - line[lo]) * a.unit;
    for (; u < stop; ++u, first += a.unit) {
      const int32_t blocks = min(a.unit, n_blocks - first);
      // lane j: the first key of block j of the unit
      const int32_t mine_first = first_key(p, first + min(lane, blocks));
      const int32_t mine_end = __shfl_down_sync(0xFFFFFFFFu, mine_first, 1);
      const int32_t begin = __shfl_sync(0xFFFFFFFFu, mine_first, 0), end = __shfl_sync(0xFFFFFFFFu, mine_first, blocks);
      float score = 0.0f;
      uint32_t even = 0, odd = 0;
      for (int32_t base = begin; base < end; base += kUnitKeys) {
        // keys base + 8 j + g (tile j / 2, row g or g + 8), of the page of `base` or the next one
        const int page0 = cache::page_of(a.b, seq, base / kPage), page1 = cache::page_of(a.b, seq, base / kPage + 1);
        const uint8_t* rec0 = a.cache + (int64_t)page0 * a.page_stride + (int64_t)head * a.record;
        const uint8_t* rec1 = a.cache + (int64_t)page1 * a.page_stride + (int64_t)head * a.record;
        const int t = base % kPage + g, left = end - base - g;
        const int here = page0 >= 0 ? left : 0, there = page1 >= 0 ? left : 0;
        Quarter<D> k[8];
        if (end - base >= kUnitKeys && page0 >= 0 && page1 >= 0) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            load_quarter<D>(k[j], t + 8 * j < kPage ? rec0 : rec1 - kPage * (D / 2), t + 8 * j < kPage ? rec0 : rec1 - kPage * (D / 16),
                            t + 8 * j, quarter);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c) k[j].code[c] = 0;
            k[j].scale = 0;
            if (8 * j < (t + 8 * j < kPage ? here : there))
              load_quarter<D>(k[j], t + 8 * j < kPage ? rec0 : rec1 - kPage * (D / 2),
                              t + 8 * j < kPage ? rec0 : rec1 - kPage * (D / 16), t + 8 * j, quarter);
          }
        }
#pragma unroll
        for (int tile = 0; tile < 4; ++tile) {
          float sum[2] = {};
#pragma unroll
          for (int group = 0; group < D / 64; ++group) {
            float c[4] = {};
#pragma unroll
            for (int w = 2 * group; w < 2 * group + 2; ++w) {  // eight codes of both keys: two steps of the tensor core
              const uint32_t u = k[2 * tile].code[w], v = k[2 * tile + 1].code[w];
              cache::mma(c, cache::decode_byte<0>(u), cache::decode_byte<0>(v), cache::decode_byte<1>(u), cache::decode_byte<1>(v),
                         bq[4 * w], bq[4 * w + 1]);
              cache::mma(c, cache::decode_byte<2>(u), cache::decode_byte<2>(v), cache::decode_byte<3>(u), cache::decode_byte<3>(v),
                         bq[4 * w + 2], bq[4 * w + 3]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t s = k[2 * tile + h].scale;
              const float scale = group == 0 ? scale_value<0>(s) : group == 1 ? scale_value<1>(s) : scale_value<2>(s);
              sum[h] = fmaf(scale, c[2 * h] + c[2 * h + 1], sum[h]);
            }
          }
          // the largest scales: lower bytes of halves, and upper ones (whatever is below them)
          const uint32_t two = __byte_perm(k[2 * tile].scale, k[2 * tile + 1].scale, 0x5410);
          even = __vmaxu2(even, two & 0x00FF00FFu);
          if (D > 64) odd = __vmaxu2(odd, two);
          if (D > 128) even = __vmaxu2(even, __byte_perm(k[2 * tile].scale, k[2 * tile + 1].scale, 0x7632));
          keys[warp][(16 * tile + g) * 4 + quarter] = sum[0];
          keys[warp][(16 * tile + 8 + g) * 4 + quarter] = sum[1];
        }
        __syncwarp();
        if (lane < blocks)
          for (int32_t i = max(mine_first, base); i < min(mine_end, base + kUnitKeys); ++i) {
            const float4 x = reinterpret_cast<const float4*>(keys[warp])[i - base];
            score += (x.x + x.y) + (x.z + x.w);
          }
        __syncwarp();
      }
      const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, max(max(even & 0xFFFFu, even >> 16), max(odd >> 8 & 0xFFu, odd >> 24)));
      if (lane < blocks) {
        const float error = size * (float)(mine_end - mine_first) * scale_value<0>(top);
        const float least = score - error, most = score + error;
        // (what may not be finite has to be looked at)
        const bool fine = top < 0xF8u && fabsf(least) < kHuge && fabsf(most) < kHuge;
        bounds[first + lane] = fine ? make_float2(least, most) : make_float2(-kHuge, kHuge);
      }
    }
  }
}

// ------------------------------------------------------------------ exact scores
template <int D>
struct Exact {
  int4 limb[D / 16][kLimbs];   // bytes of the query, the lowest first, of the 16 dims of a group, four to a word
  int32_t start[D / 16][8];    // what the sums of a group begin with: 12 of every code too many, taken off
  uint32_t top, low;
};

// fp64 of an integer, without a conversion: its bits in the mantissa of 2^52 + 2^31 + x.
__device__ __forceinline__ double whole(int32_t x) {
  return __hiloint2double(0x43300000, x ^ 0x80000000) - 4503601774854144.0;
}
// fp64 of a scale byte (NaN for those that stand for no number).
__device__ __forceinline__ double scale_of(uint32_t byte) {
  if (byte < 8) return (double)byte * 7.62939453125e-06;  // (below the smallest normal scale: eighths of 2^-14)
  return __hiloint2double(byte < 0xF8 ? (int)((byte << 17) + (1008u << 20)) : 0x7FF80000, 0);
}
// Four codes, doubled and 12 more: whole numbers 0 to 24 in four bytes.
__device__ __forceinline__ int decode4(uint32_t codes) {
  // (a selector whose upper bit is set gives the sign of the byte in all its bits, which is 0 for these)
  uint32_t plus, minus;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(plus) : "r"(0x03020100u), "r"(0x0C080604u), "r"(codes));
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(minus) : "r"(0x03020100u), "r"(0x0C080604u), "r"(codes ^ 0x8888u));
  return (int)(0x0C0C0C0Cu + plus - minus);
}

// The sum of a (row, head)'s query heads as whole numbers of a power of two, so that the largest stays below 2^46, cut into six
// signed bytes: values down to 2^-33 of the largest are exact in bf16 (2^-30 in fp16) with 16 heads, smaller ones off by less
// than 2^-40 of it.  The lower two bytes are mostly zero in every place.  By all threads; false if a value is not finite.
template <int D>
__device__ __forceinline__ bool prepare_exact(const Args& a, Exact<D>& w, int row, int head) {
  const int d = threadIdx.x;
  const uint16_t* q = static_cast<const uint16_t*>(a.q) + (int64_t)row * a.q_row + (int64_t)head * a.group * a.q_head + d;
  uint32_t top = 0;
  if (d < D) {
#pragma unroll 8
    for (int g = 0; g < a.group; ++g) top = max(top, (uint32_t)q[g * a.q_head] & 0x7FFFu);
  }
  if (d == 0) w.top = w.low = 0;
  __syncthreads();
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  if (d % 32 == 0) atomicMax(&w.top, top);
  __syncthreads();
  top = w.top;
  if (top >= (a.q_half ? 0x7C00u : 0x7F80u)) return false;
  // x 2^up: below 2^(bits - 22), its fraction to 22 bits
  const int up = a.bits - 22 + 126 - max((int)(__float_as_uint(query_value(a, top)) >> 23), 1);
  const float up0 = __uint_as_float((uint32_t)(127 + up / 2) << 23), up1 = __uint_as_float((uint32_t)(127 + up - up / 2) << 23);
  if (d < D) {
    int32_t upper = 0, lower = 0;
#pragma unroll 4
    for (int g = 0; g < a.group; ++g) {
      const float x = query_value(a, q[g * a.q_head]) * up0 * up1, whole_part = rintf(x);
      upper += (int)whole_part;
      lower += __float2int_rn((x - whole_part) * 4194304.0f);
    }
    int64_t x = (int64_t)upper * 4194304 + lower;
    uint32_t low = 0;
#pragma unroll
    for (int l = 0; l < kLimbs; ++l) {
      const int8_t byte = (int8_t)x;
      x = (x - byte) >> 8;
      reinterpret_cast<int8_t*>(&w.limb[d / 16][l])[d % 16] = byte;
      if (l < 2) low |= (uint8_t)byte;
    }
    if (low != 0) w.low = 1;
  }
  __syncthreads();
  if (d < D / 16 * kLimbs) {
    const int4 v = w.limb[d / kLimbs][d % kLimbs];
    const int ones = 0x01010101;
    w.start[d / kLimbs][d % kLimbs] = -12 * __dp4a(v.x, ones, __dp4a(v.y, ones, __dp4a(v.z, ones, __dp4a(v.w, ones, 0))));
  }
  return true;  // (the caller meets before the sums are read)
}

// Score of a key, by four threads, each with a quarter of it; all of them get it.
template <int D, int LIMBS>
__device__ __forceinline__ double dot(const Exact<D>& w, const Quarter<D>& k, int quarter) {
  constexpr int L0 = kLimbs - LIMBS, HALF = LIMBS / 2;
  double upper = 0.0, lower = 0.0;
#pragma unroll
  for (int j = 0; j < D / 64; ++j) {
    const int g = quarter * (D / 64) + j;
    const int c[4] = {decode4(k.code[2 * j]), decode4(k.code[2 * j] >> 16), decode4(k.code[2 * j + 1]),
                      decode4(k.code[2 * j + 1] >> 16)};
    // (a sum is at most 128 * 12 * 16 in size, so that three of them, a byte apart, fit 32 bits)
    int up = 0, lo = 0;
#pragma unroll
    for (int l = LIMBS - 1; l >= 0; --l) {
      const int4 q = w.limb[g][L0 + l];
      const int sum = __dp4a(c[0], q.x, __dp4a(c[1], q.y, __dp4a(c[2], q.z, __dp4a(c[3], q.w, w.start[g][L0 + l]))));
      if (l >= HALF) up = up * 256 + sum;
      else lo = lo * 256 + sum;
    }
    const double s = scale_of(k.scale >> 8 * j & 255u);
    upper = fma(s, whole(up), upper);
    lower = fma(s, whole(lo), lower);
  }
  double x = fma(upper, (double)(1 << 8 * HALF), lower);
  x += __shfl_xor_sync(0xFFFFFFFFu, x, 1);
  return x + __shfl_xor_sync(0xFFFFFFFFu, x, 2);
}

// Scores of entries [from, to) of the list (blocks with the keys of `range`) by all threads: 16 of them for two blocks, four for
// a key, up to 8 keys of either block on their way at once.  `part` is shared.
template <int D>
__device__ __forceinline__ void exact_scores(const Args& a, const Exact<D>& w, int limbs, int seq, int head, const int2* range,
                                             uint64_t* rank, uint32_t from, uint32_t to, double (&part)[kPickThreads / 16][2][8]) {
  constexpr uint32_t kHalves = kPickThreads / 16;
  const int lane = threadIdx.x % 32, quarter = lane % 4, key = lane / 4 % 4, half = threadIdx.x / 16;
  for (uint32_t e0 = from + half; e0 - half < to; e0 += 2 * kHalves) {
    int2 r[2];
    double score = 0.0;  // of block e0 + x kHalves, in lane x of the 16
#pragma unroll
    for (int x = 0; x < 2; ++x) r[x] = e0 + x * kHalves < to ? range[e0 + x * kHalves] : make_int2(0, 0);
    for (int32_t at = 0; __any_sync(0xFFFFFFFFu, at < r[0].y - r[0].x || at < r[1].y - r[1].x); at += 8) {
      Quarter<D> k[4] = {};
      bool there[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int32_t i = r[x / 2].x + at + x % 2 * 4 + key;
        const int page = i < r[x / 2].y ? cache::page_of(a.b, seq, i / kPage) : -1;
        there[x] = page >= 0;
        const uint8_t* rec = a.cache + (int64_t)page * a.page_stride + (int64_t)head * a.record;
        if (there[x]) load_quarter<D>(k[x], rec, rec, i % kPage, quarter);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        double y = 0.0;  // (also of keys that are not there)
        if (__any_sync(0xFFFFFFFFu, there[x])) y = limbs == 4 ? dot<D, 4>(w, k[x], quarter) : dot<D, 6>(w, k[x], quarter);
        if (quarter == 0) part[half][x / 2][x % 2 * 4 + key] = y;
      }
      __syncwarp();
      if (lane % 16 < 2)
#pragma unroll
        for (int j = 0; j < 8; ++j) score += part[half][lane % 16][j];  // (in the order of the keys)
      __syncwarp();
    }
    const uint32_t e = e0 + lane % 16 * kHalves;
    if (lane % 16 < 2 && e < to) rank[e] = rank_of(limbs == 0 ? __longlong_as_double(0x7FF8000000000000ll) : score);
  }
}

// ------------------------------------------------------------------ the best of a row
struct List {
  uint64_t* rank;
  uint32_t* index;
};
// The bin of a bound: never a lower one for a larger bound.
__device__ __forceinline__ int bin_of(float x, float low, float per) { return max(0, min(kBins - 1, (int)((x - low) * per))); }
__host__ __device__ constexpr int list_size(int n_sel) { return n_sel + kCandidates; }
__host__ __device__ constexpr int list_bytes(int n_sel) { return 32 * list_size(n_sel); }  // two lists and the keys of one

// Numbers that compare like fp32, and back.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u >> 31 ? u & 0x7FFFFFFFu : ~u); }

template <int D>
__global__ void __launch_bounds__(kPickThreads) pick_kernel(const Args a) {
  extern __shared__ __align__(16) uint8_t dynamic[];
  __shared__ Exact<D> w;
  __shared__ float2 held[kHeldBounds];
  __shared__ __align__(16) uint32_t count[kBins];
  __shared__ uint32_t sums[kPickThreads / 32];
  __shared__ double part[kPickThreads / 16][2][8];
  __shared__ uint32_t s_least, s_most, s_bin, s_total, s_n;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int size = list_size(a.n_sel);
  List list = {reinterpret_cast<uint64_t*>(dynamic), reinterpret_cast<uint32_t*>(dynamic + 16 * size)};
  List other = {list.rank + size, list.index + size};
  int2* range = reinterpret_cast<int2*>(dynamic + 24 * size);
  allow_next();
  // What earlier kernels wrote is read before score_kernel has ended (see there).
  const int64_t unit = blockIdx.x;
  const int row = a.row0 + (int)(unit / a.hkv), head = (int)(unit % a.hkv);
  const float2* bounds = a.bounds + ((int64_t)a.row0 * a.hkv + unit) * a.blocks;
  int32_t* sel = a.sel + ((int64_t)a.row0 * a.hkv + unit) * a.n_sel;
  const int32_t tokens = tokens_of(a.b, row, a.most), n = blocks_of(tokens, a.shift);
  const uint32_t wanted = min((uint32_t)a.n_sel, (uint32_t)n);
  for (int i = (int)wanted + tid; i < a.n_sel; i += kPickThreads) sel[i] = -1;
  if (n == 0) {
    wait_for_earlier();
    return;
  }
  const int seq = cache::sequence_of(a.b, row);
  const Places p = places_of(tokens, a.cmp_block, a.cmp_stride, a.shift);
  reinterpret_cast<uint4*>(count)[tid] = make_uint4(0, 0, 0, 0);
  if (tid == 0) s_least = 0xFFFFFFFFu, s_most = 0, s_total = 0, s_n = 0;
  int limbs = prepare_exact<D>(a, w, row, head) ? 4 : 0;
  __syncthreads();
  if (limbs != 0 && w.low != 0) limbs = 6;
  wait_for_earlier();

  // The lower bounds are counted in bins; the n_sel-th largest lies in bin `edge`, so a block whose upper bound is in a bin
  // below that is none of the best.
  const bool fits = n <= kHeldBounds;
  uint32_t least = 0xFFFFFFFFu, most = 0;
#pragma unroll 4
  for (int i = tid; i < n; i += kPickThreads) {
    const float2 x = bounds[i];
    if (fits) held[i] = x;
    if (x.x > -kHuge) least = min(least, ordered(x.x)), most = max(most, ordered(x.x));
  }
  const float2* of = fits ? held : bounds;
  least = __reduce_min_sync(0xFFFFFFFFu, least), most = __reduce_max_sync(0xFFFFFFFFu, most);
  if (lane == 0) atomicMin(&s_least, least), atomicMax(&s_most, most);
  __syncthreads();
  float low = 0.0f, per = 0.0f;
  int edge = 0;
  if (n > (int)wanted && s_most > s_least) {
    low = unordered(s_least);
    per = (float)kBins / (unordered(s_most) - low);  // (0 if that is beyond fp32: one bin)
    for (int i = tid; i < n; i += kPickThreads) atomicAdd(&count[bin_of(of[i].x, low, per)], 1u);
    __syncthreads();
    // four bins of a thread, the largest first
    const uint4 c = reinterpret_cast<const uint4*>(count)[kPickThreads - 1 - tid];
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
    for (int i = 0; i < kPickThreads / 32; ++i) at += i < warp ? sums[i] : 0;
    if (at < wanted && wanted <= at + mine) {
      const int bin = 4 * (kPickThreads - 1 - tid);
      s_bin = wanted <= at + c.w ? bin + 3 : wanted <= at + c.w + c.z ? bin + 2 : wanted <= at + c.w + c.z + c.y ? bin + 1 : bin;
    }
    __syncthreads();
    edge = (int)s_bin;
  }

  // Exact scores of the blocks that are left; where they are too many, only the best so far are kept.
  uint32_t scored = 0;
  const auto keep_best = [&](bool last) {
    const uint32_t in = s_n;
    for (uint32_t x = 2 * scored + tid; x < 2 * in; x += kPickThreads)
      (x % 2 == 0 ? range[x / 2].x : range[x / 2].y) = first_key(p, (int32_t)(list.index[x / 2] + x % 2));
    __syncthreads();
    exact_scores<D>(a, w, limbs, seq, head, range, list.rank, scored, in, part);
    __syncthreads();
    for (uint32_t e0 = tid / 8; e0 - tid / 8 < in; e0 += kPickThreads / 8) {  // 8 threads for an entry
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
    scored = min(in, wanted);
    const List swap = list;
    list = other, other = swap;
    __syncthreads();
    if (tid == 0) s_n = scored;
    __syncthreads();
  };
  for (int i0 = 0; i0 < n; i0 += kChecked * kPickThreads) {
    uint32_t mask = 0;
#pragma unroll
    for (int j = 0; j < kChecked; ++j) {
      const int i = i0 + j * kPickThreads + tid;
      if (i < n && bin_of(of[i].y, low, per) >= edge) mask |= 1u << j;
    }
    if (mask != 0) atomicAdd(&s_total, __popc(mask));
    __syncthreads();
    const bool room = s_n + s_total <= (uint32_t)size;
    __syncthreads();
    if (tid == 0) s_total = 0;
    if (room) {
      if (mask != 0) {
        uint32_t at = atomicAdd(&s_n, __popc(mask));
        for (; mask != 0; mask &= mask - 1) list.index[at++] = (uint32_t)(i0 + (__ffs(mask) - 1) * kPickThreads + tid);
      }
    } else {
      for (int j = 0; j < kChecked; ++j) {
        if (mask >> j & 1) list.index[atomicAdd(&s_n, 1u)] = (uint32_t)(i0 + j * kPickThreads + tid);
        __syncthreads();
        const bool full = s_n + kPickThreads > (uint32_t)size;
        __syncthreads();
        if (full) keep_best(false);
      }
    }
    __syncthreads();
  }
  keep_best(true);
}

}  // namespace cache_select
}  // namespace nsa
