// Kernels of the 4-bit paged KV cache: quantising rows as they are written, reading rows back, and
// attention of single tokens over the cache (all keys, a window, or the row's selected blocks).
//
// Number format.  16 neighbouring values x_i of a token share a scale
//     s = round5m3(min(max|x_i| / 6, 10240)),     c_i = round_e2m1(x_i / s),     value = c_i * s,
// both roundings to nearest, ties to even, saturating.  c is sign, two exponent bits and one mantissa bit
// (0, 0.5, 1, 1.5, 2, 3, 4, 6); s has five exponent bits (bias 15) and three mantissa bits, so that
// `byte << 7` is its half-precision pattern and no second, calibrated factor is needed: 4.6e-5 to 61440 is
// covered.  A product has at most 6 significant bits and its sixfold is finite in half precision (10240 * 6 =
// 61440), so reading back is exact in fp16 and bf16, and the attention's operands are the exact values.  A
// group that holds a NaN or an infinity gets the scale 0xFF (NaN), and reads back as NaN.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "nsa_cache_decode.cuh"
#include "nsa_cache_index.h"
#include "nsa_programmatic.cuh"
#include "ptx.cuh"

namespace nsa {
namespace cache {

enum : int { kBf16 = 0, kF32 = 1, kF16 = 2 };

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// ------------------------------------------------------------------ 4-bit conversions
// Codes of eight values, the first in the lowest nibble.
__device__ __forceinline__ uint32_t encode8(const float* y) {
  uint32_t r;
  asm("{.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};}"
      : "=r"(r)
      : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
  return r;
}
__device__ __forceinline__ uint32_t low2(uint32_t x) {  // (an operand's modifier, not an instruction)
  uint32_t r;
  asm("{.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tmov.b32 %0, {l, l};}" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t high2(uint32_t x) {
  uint32_t r;
  asm("{.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tmov.b32 %0, {h, h};}" : "=r"(r) : "r"(x));
  return r;
}
// The scale byte of a group with the largest value amax: the scale nearest to amax / 6, ties to even, at most 10240 (0xE2).
// The product with 1/6 is off by 2^-23 of itself; rounded to 17 bits it is the quotient again where that has few bits (the
// ties), and amax's 8 or 11 bits keep every other quotient 2^-12 of itself away from a tie.
__device__ __forceinline__ uint32_t scale_byte(float amax) {
  const float raw = __uint_as_float((__float_as_uint(amax * 0.16666667f) + 0x40u) & ~0x7Fu);
  if (raw >= 6.103515625e-05f) {  // 2^-14, the smallest normal scale
    const uint32_t b = __float_as_uint(raw);
    return min(((b + 0x7FFFFu + ((b >> 20) & 1u)) >> 20) - 896u, 226u);
  }
  return (uint32_t)__float2int_rn(raw * 131072.0f);  // eighths of 2^-14
}

// ------------------------------------------------------------------ writing
// One thread quantises two neighbouring groups of a row and head: 64 bytes in, 16 bytes of codes and two of scales out, 2.56
// bytes a value, and few enough instructions (with one group a thread the look-up of the row's place took as many as the
// arithmetic, and the kernel 41 us where it now takes 35, for 65536 tokens of 4 heads with d = 128) to be bound by memory.
// x / s must fall on the right side of the borders between codes (0.25, 0.75, ... 5), and exactly on one where it is one, for
// ties to go to the even code.  x (1 / s) has an error of 2^-22 and would miss some of the ties; fma(x, 1 / s, 192) - 192
// rounds the quotient to a multiple of 2^-16 instead.  A border is such a multiple, and with the 8 or 11 significant bits of x
// no other quotient is nearer to a border t than t 2^-11, so the codes are those of a true division.
struct WriteArgs {
  Batch b;
  const void* x[2];               // K, V [n_rows, Hkv, d], unit stride along d
  int64_t row_stride[2], head_stride[2];
  uint8_t* cache;
  int64_t page_stride;
  int32_t hkv, half;              // half: inputs are fp16, else bf16
};

// Codes of 16 values (as they are in memory); `scale`: their byte.
__device__ __forceinline__ uint2 quantise(const uint4& lo, const uint4& hi, bool half, uint32_t& scale) {
  const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  uint32_t top = 0;  // |x| as integers: a NaN is above an infinity, an infinity above every number
#pragma unroll
  for (int j = 0; j < 8; ++j) top = __vmaxu2(top, w[j] & 0x7FFF7FFFu);
  top = max(top & 0xFFFFu, top >> 16);
  const bool fine = top < (half ? 0x7C00u : 0x7F80u);
  scale = fine ? scale_byte(half ? __half2float(__ushort_as_half((unsigned short)top)) : __uint_as_float(top << 16)) : 255u;
  if (!fine || scale == 0) return make_uint2(0, 0);
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(__half2float(__ushort_as_half((unsigned short)(scale << 7)))));
  float y[16];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float2 f = half ? __half22float2(*reinterpret_cast<const __half2*>(&w[j]))
                    : make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
    f = add2(fma2(f, make_float2(inv, inv), make_float2(192.0f, 192.0f)), make_float2(-192.0f, -192.0f));
    y[2 * j] = f.x, y[2 * j + 1] = f.y;
  }
  return make_uint2(encode8(y), encode8(y + 8));
}

template <int DQK, int DV, int WHICH>
__device__ __forceinline__ void write_groups(const WriteArgs& a, uint32_t i) {
  constexpr int D = WHICH == 0 ? DQK : DV, PAIRS = D / 32;
  const uint32_t total = (uint32_t)a.b.n_rows * a.hkv * PAIRS;
  if ((i & ~31u) >= total) return;  // (whole warps)
  const bool in = i < total;
  const uint32_t g = i % PAIRS, rh = (in ? i : total - 1) / PAIRS, row = rh / a.hkv, h = rh - row * a.hkv;
  const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x[WHICH]) + (int64_t)row * a.row_stride[WHICH] +
                                                    (int64_t)h * a.head_stride[WHICH] + g * 32);
  const uint4 x0 = src[0], x1 = src[1], x2 = src[2], x3 = src[3];
  uint32_t s0, s1;
  const uint2 c0 = quantise(x0, x1, a.half, s0), c1 = quantise(x2, x3, a.half, s1);
  // the scales of two neighbouring threads (of one token: PAIRS is even) go out together
  uint32_t scales = s0 | s1 << 8;
  scales |= __shfl_down_sync(0xFFFFFFFFu, scales, 1) << 16;
  const int seq = in ? sequence_of(a.b, row) : -1;
  if (seq < 0) return;
  const int pos = position_of(a.b, seq, row);
  const int page = pos < 0 ? -1 : page_of(a.b, seq, pos / kPage);
  if (page < 0) return;
  uint8_t* rec = a.cache + (int64_t)page * a.page_stride + (int64_t)h * record_bytes(DQK, DV) + (WHICH == 0 ? 0 : v_code_at(DQK));
  const uint32_t at = pos % kPage * PAIRS + g;
  reinterpret_cast<uint4*>(rec)[at] = make_uint4(c0.x, c0.y, c1.x, c1.y);
  if (g % 2 == 0) reinterpret_cast<uint32_t*>(rec + kPage * D / 2)[at / 2] = scales;
}

template <int DQK, int DV>
__global__ void __launch_bounds__(256) write_kernel(const WriteArgs a) {
  start_in_order();
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (blockIdx.y == 0) write_groups<DQK, DV, 0>(a, i);
  else write_groups<DQK, DV, 1>(a, i);
}

// ------------------------------------------------------------------ reading back
// A thread turns ITEMS groups (256 apart: a block's stores are whole lines) of 8 bytes of codes and one of scale into 16 values
// each.  Long inputs take two, for the loads of one to cover the other's (104448 tokens of 4 heads with 192 and 128: 74 us with
// one, 64 with two); where there are few blocks the second only waits for the first's look-up (24700 tokens of one head with
// d = 64: 2.8 us more).
struct ReadArgs {
  Batch b;
  const uint8_t* cache;
  int64_t page_stride;
  void* y[2];  // K, V [Hkv, n_rows, d]
  int32_t hkv, dtype;
};

// 32 bytes at once: a warp's store then fills whole sectors, where two 16-byte stores leave the L2 half ones (65536 tokens of 4
// heads with d = 128: 40 us, and 31 so).
__device__ __forceinline__ void store32(void* to, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

template <int DQK, int DV, int WHICH, int ITEMS>
__device__ __forceinline__ void read_groups(const ReadArgs& a, uint32_t i0) {
  constexpr int D = WHICH == 0 ? DQK : DV, GR = D / kGroup;
  const uint32_t total = (uint32_t)a.b.n_rows * a.hkv * GR;
  uint2 c[ITEMS];
  uint32_t s[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const uint32_t i = i0 + k * 256;
    c[k] = make_uint2(0, 0), s[k] = 0;  // a token that is not there reads as zeros
    if (i >= total) continue;
    const uint32_t g = i % GR, hr = i / GR, h = hr / a.b.n_rows, row = hr - h * a.b.n_rows;
    const int seq = sequence_of(a.b, row);
    const int pos = seq < 0 ? -1 : position_of(a.b, seq, row);
    const int page = pos < 0 ? -1 : page_of(a.b, seq, pos / kPage);
    if (page < 0) continue;
    const uint8_t* rec = a.cache + (int64_t)page * a.page_stride + (int64_t)h * record_bytes(DQK, DV);
    const int t = pos % kPage;
    c[k] = *reinterpret_cast<const uint2*>(rec + (WHICH == 0 ? 0 : v_code_at(DQK)) + t * (D / 2) + g * 8);
    s[k] = rec[(WHICH == 0 ? k_scale_at(DQK) : v_scale_at(DQK, DV)) + t * GR + g];
  }
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const uint32_t i = i0 + k * 256;
    if (i >= total) return;
    const uint32_t z = scale2(s[k]);
    uint32_t v[8] = {mul2(decode_byte<0>(c[k].x), z), mul2(decode_byte<1>(c[k].x), z), mul2(decode_byte<2>(c[k].x), z),
                     mul2(decode_byte<3>(c[k].x), z), mul2(decode_byte<0>(c[k].y), z), mul2(decode_byte<1>(c[k].y), z),
                     mul2(decode_byte<2>(c[k].y), z), mul2(decode_byte<3>(c[k].y), z)};  // fp16 pairs
    if (a.dtype == kF32) {
      float* out = static_cast<float*>(a.y[WHICH]) + (int64_t)i * kGroup;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t w[8];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float2 p = __half22float2(*reinterpret_cast<__half2*>(&v[4 * j + x]));
          w[2 * x] = __float_as_uint(p.x), w[2 * x + 1] = __float_as_uint(p.y);
        }
        store32(out + 8 * j, w);
      }
      continue;
    }
    if (a.dtype == kBf16) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const __nv_bfloat162 p = __float22bfloat162_rn(__half22float2(*reinterpret_cast<__half2*>(&v[j])));
        v[j] = *reinterpret_cast<const uint32_t*>(&p);
      }
    }
    store32(static_cast<uint16_t*>(a.y[WHICH]) + (int64_t)i * kGroup, v);
  }
}

template <int DQK, int DV, int ITEMS>
__global__ void __launch_bounds__(256) read_kernel(const ReadArgs a) {
  start_in_order();
  const uint32_t i = blockIdx.x * (256u * ITEMS) + threadIdx.x;
  if (blockIdx.y == 0) read_groups<DQK, DV, 0, ITEMS>(a, i);
  else read_groups<DQK, DV, 1, ITEMS>(a, i);
}

// ------------------------------------------------------------------ attention
// For a row n, KV head h and its G query heads (8 or 16 at a time: a tile):
//     z_j = scale * q . k_j,   O = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m),   LSE = m + ln sum_j exp(z_j - m)
// over the visible keys j, in one pass with the running maximum m (kept in powers of two).
//
// A key costs 9/16 (d_qk + d_v) bytes and 2 G (d_qk + d_v) operations: at d = 128 and G = 16 57 operations a byte, so the floor
// is the cache's bytes from DRAM, provided that turning 4 bits into tensor-core operands keeps up.  Hence every warp is
// a worker of its own with a ring of page records in shared memory (bulk copies), and codes go from there straight into the
// registers that the tensor core reads (m16n8k16, fp16 in, fp32 out): no dequantised value is ever stored.  (Operands in shared
// memory, as tcgen05 could have them, would cost 64 KB of shared-memory traffic a page beside the 9 KB that are fetched.  The
// decoded operand in tensor memory was not tried.)
// The cache is the A operand, S^T = K Q^T and O^T = V^T P^T, so that 8 query heads cost half the tensor instructions of 16,
// and a decoded fragment serves both halves.  For that
//   * the d axis of QK is permuted so that a thread's K fragments are d_qk / 4 consecutive codes of one key: one
//     wide shared load, one conversion and one product with the scale for each pair, exact in fp16;
//   * a thread's V fragments are d_v / 8 consecutive codes of four keys, which are interleaved two and two; P^T takes
//     its place by transposing 8 x 8 tiles between registers;
//   * the key axis is permuted (rows 2q, 2q + 1 of a tile of 8 are keys q, 4 + (q ^ 1)) so that neither K's nor V's
//     shared loads collide more than two ways on the record as it is.
// Q has up to 8 (bf16) or 11 significant bits, so a power of two per row puts it into fp16 (below 2^-14 of the row's
// largest to within 2^-25 of it).  P is rounded to fp16 for the tensor core (2^-11 of each term, or 2^-32 of the largest where
// that is more: see page()); the sum of its fp32 values is the divisor.  Scores, statistics and O are fp32.
//
// What binds: a page of 64 keys (d = 128) takes a scheduler 1800 cycles with 16 heads and two warps (2090 with one; 1310 and
// 1560 with 8 heads), of which half are the issue of 128 tensor instructions, most of the rest 256 conversions and 256 products;
// DRAM would deliver a page in 1550.  64 rows of up to 32768 keys, 616 MB: 165 us, 3.7 TB/s; 256 rows of 16 selected blocks,
// 155 MB: 47 us, 3.3 TB/s; one row of 16 blocks: 10.2 us.  (In the kernel a warp's page takes 4400 cycles, 3270 of them in
// page(), the rest in finding, copying and waiting for the next ones.)
//
// All (row, page) slots of the call stand in one line that is shared out evenly (split_line): teams of 1 to 8 warps of a
// block take turns at a row's pages and join their (m, sum, O) in shared memory; a row that is cut between teams leaves
// partial results in the workspace, and merge_kernel joins them in the order of the line.  Where rows are few and not
// long, the blocks of a cluster share each and join through one another's shared memory.  Results do not depend on timing.
struct AttendArgs {
  Batch b;
  const void* q;                 // [n_rows, Hq, DQK], bf16 or fp16, unit stride along d
  int64_t q_row, q_head;
  const uint8_t* cache;
  int64_t page_stride;
  const int32_t* sel;            // [n_rows, Hkv, n_sel] or nullptr
  void* o;                       // [n_rows, Hq, DV]
  float* lse;                    // [n_rows, Hq] or nullptr
  const float* weight;
  float* part;                   // partial results, 2 for each team
  uint32_t* starts;              // ragged line: slots before every row's (n_rows + 1), then the share of a team or 0 if no
                                 // row is cut; written by the first block for merge_kernel
  int32_t hq, hkv, group, tiles; // tiles: of a KV head's G query heads
  int32_t n_sel, per, window;    // per: sub-blocks of a selection block
  int32_t slots;                 // slots of every row; 0: as many as it has sub-blocks (the ragged line)
  uint32_t warps;                // of the device
  uint32_t cluster;              // blocks that share each row (1: none do); then rows are whole and a cluster has one
  Split split;                   // (a ragged line's is worked out on the device)
  int32_t q_half, o_dtype, accumulate, fill;  // fill: rows of no sequence get O = 0, LSE = -inf; else they are left
  float scale_log2;
  int32_t* err;                  // optional: NSA_DEVERR_TIMEOUT (1) if a copy did not come
  uint64_t wait_ns;              // bound of every wait for a copy
  int32_t stall;                 // (test) no copy is made, so that the waits run out
};

template <int DQK_, int DV_, int NH_, int STAGES_, int ROUNDS_>
struct AttendCfg {
  static constexpr int DQK = DQK_, DV = DV_, NH = NH_, NW = 8, STAGES = STAGES_, ROUNDS = ROUNDS_;
  static constexpr int kHeads = 8 * NH;       // query heads of a tile
  static constexpr int kRecord = record_bytes(DQK, DV);
  static constexpr int kQueue = 40;           // resolved slots of a warp
  static constexpr int kMaxRagged = 1920;     // rows of a ragged line
  static constexpr int kPart = kHeads * (DV + 2);              // floats of a partial result: O, m, sum
  static constexpr int kJoin = kHeads * (DV / ROUNDS + 4);     // floats of a warp in a team's join: O of a round, m, sum, max
  static constexpr int kWarp = STAGES * (kRecord + 8) + kQueue * 16 + kJoin * 4;
  static constexpr int kSmem = NW * kWarp + (kMaxRagged + 2) * 4;
  static_assert(kSmem + 128 <= 232448, "227 KB of shared memory a block, the static variables included");
};

// Ring depth and rounds of the join for each head dim and tile (NH = 1: up to 8 query heads, 2: 16).  A warp holds O and Q
// of a tile and a page's scores in up to 255 registers, so a block has 8 warps and an SM one block.
template <int DQK, int DV, int NH>
struct CfgFor;
template <int NH>
struct CfgFor<64, 64, NH> : AttendCfg<64, 64, NH, 3, 1> {};
template <int NH>
struct CfgFor<128, 64, NH> : AttendCfg<128, 64, NH, 3, 1> {};
template <int NH>
struct CfgFor<128, 128, NH> : AttendCfg<128, 128, NH, 2, 1> {};
template <int NH>
struct CfgFor<192, 128, NH> : AttendCfg<192, 128, NH, 2, NH> {};

// A record's copy into shared memory, by one thread: the barrier's phase ends when all bytes are there.
__device__ __forceinline__ void copy_record(void* dst, const uint8_t* src, int bytes, uint64_t* bar) {
  ptx::mbar_arrive_expect_tx(bar, bytes);
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   ptx::smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(ptx::smem_u32(bar))
               : "memory");
}
// One lane of a whole warp.  (Known to be one: `lane == 0` makes the compiler provide for a divergent warp, 0.7 % of
// the attention's time.)
__device__ __forceinline__ bool elected() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// Waits for a phase, `ns` at most; false if that runs out.
__device__ __noinline__ bool wait_long(uint64_t* bar, uint32_t parity, uint64_t ns) {
  const uint64_t t0 = ptx::globaltimer();
  while (!ptx::mbar_try_wait(bar, parity))
    if (ptx::globaltimer() - t0 > ns) return false;
  return true;
}
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, uint64_t ns) {
  return ptx::mbar_try_wait(bar, parity) || wait_long(bar, parity, ns);
}
// Waits for the copies that are on their way (a bit of `flying` for each stage), `ns` at most for each: after one that did not
// come in time, and before the ring is used for anything else or the block ends.
__device__ __noinline__ void wait_all(uint64_t* bars, uint32_t phases, uint32_t flying, uint64_t ns) {
  for (int i = 0; flying >> i != 0; ++i)
    if (flying >> i & 1) wait_long(bars + i, phases >> i & 1, ns);
  __syncwarp();
}
__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) { return ptx::ex2(x); }
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// sequence_of by a whole warp.
__device__ __forceinline__ int sequence_of_warp(const Batch& b, int row, int lane) {
  return sequence_by_32(b, row, [&](int lo, int step, int hi) {
    return __ballot_sync(0xFFFFFFFFu, lane * step < hi - lo && b.cu[lo + lane * step] <= row);
  });
}

// 2N consecutive values of one row of Q: as they are in memory, and as fp16 pairs; `factor` undoes the row's power of two.
template <int N>
__device__ __forceinline__ void load_q(uint32_t (&q)[N], const uint16_t* src) {
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    const uint4 x = src ? reinterpret_cast<const uint4*>(src)[i] : make_uint4(0, 0, 0, 0);
    q[4 * i] = x.x, q[4 * i + 1] = x.y, q[4 * i + 2] = x.z, q[4 * i + 3] = x.w;
  }
}
template <int N>
__device__ __forceinline__ void scale_q(uint32_t (&q)[N], bool half, float& factor) {
  auto pair = [&](uint32_t x) {
    return half ? __half22float2(*reinterpret_cast<__half2*>(&x))
                : make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u));
  };
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float2 f = pair(q[i]);
    top = max(top, max(__float_as_uint(f.x) & 0x7FFFFFFFu, __float_as_uint(f.y) & 0x7FFFFFFFu));
  }
  top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
  top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
  // exponent of the row's largest; rows of zeros or subnormals, infinities and NaN stay as they are
  const int e = (int)(top >> 23);
  const bool scaled = e > 1 && e < 254;
  const float down = scaled ? __uint_as_float((uint32_t)(254 - e) << 23) : 1.0f;
  factor = scaled ? __uint_as_float((uint32_t)e << 23) : 1.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float2 f = pair(q[i]);
    q[i] = pack_half(f.x * down, f.y * down);
  }
}

__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool half) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return half ? pack_half(lo, hi) : *reinterpret_cast<const uint32_t*>(&b);
}
// Four neighbouring values of the result of (row, query head) `at`, times k.
template <int DV>
__device__ __forceinline__ void store4(const AttendArgs& a, int64_t at, int d, float4 v, float k) {
  v.x *= k, v.y *= k, v.z *= k, v.w *= k;
  if (a.o_dtype == kF32) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.o) + at * DV + d);
    if (a.accumulate) {
      const float4 x = *p;
      v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
    }
    *p = v;
    return;
  }
  const bool half = a.o_dtype == kF16;
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at * DV + d) = make_uint2(pack16(v.x, v.y, half), pack16(v.z, v.w, half));
}
__device__ __forceinline__ void store_lse(const AttendArgs& a, int64_t at, float m, float l) {
  if (a.lse != nullptr) a.lse[at] = l != 0.0f ? (m + __log2f(l)) * 0.693147180559945309f : -INFINITY;
}

template <class C>
struct Worker {
  static constexpr int DQK = C::DQK, DV = C::DV;
  static constexpr int NH = C::NH;      // 8-wide tiles of query heads
  static constexpr int MT = DV / 16;    // 16-high tiles of O^T
  static constexpr int KS = DQK / 16;   // k steps of QK

  // ---- the producer's side: rows and slots of the team's share, one after the other
  struct Cursor {
    uint32_t next, end;    // slots of the line still to resolve
    int n, hm, j, len;     // row, KV head and tile in it, next slot, slots of the row
    int seq, first, last;  // first and one-past-last visible key
    int entry;             // lane i: entry i of the row's selection (n_sel <= 32)
    unsigned twice;        // bit i: entry i stands before (a selection is a set)
    bool entered;          // seq to twice are those of (n, hm)
  };

  static __device__ __forceinline__ void enter_row(const AttendArgs& a, Cursor& c, const uint32_t* starts, int lane) {
    const int h = c.hm / a.tiles, g0 = c.hm % a.tiles * C::kHeads;
    if (a.sel != nullptr && a.n_sel <= 32)
      c.entry = lane < a.n_sel ? a.sel[((int64_t)c.n * a.hkv + h) * a.n_sel + lane] : -1;
    // the row's queries on their way into L2 (begin() loads them when its turn comes)
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + (int64_t)c.n * a.q_row + (int64_t)(h * a.group + g0) * a.q_head;
    constexpr int kLines = DQK / 64;
#pragma unroll 1
    for (int i = lane; i < min(C::kHeads, a.group - g0) * kLines; i += 32)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(q + i / kLines * a.q_head + i % kLines * 64));
    c.seq = sequence_of_warp(a.b, c.n, lane);
    const int pos = c.seq < 0 ? -1 : position_of(a.b, c.seq, c.n);
    c.last = keys_up_to(a.b, pos);
    c.first = pos < 0 ? 0 : first_key(pos, a.window);
    c.len = a.slots ? a.slots : starts[c.n + 1] - starts[c.n];
    if (a.sel != nullptr && a.n_sel <= 32)
      c.twice = __ballot_sync(0xFFFFFFFFu, (__match_any_sync(0xFFFFFFFFu, c.entry) & ((1u << lane) - 1)) != 0);
    c.entered = true;
  }

  // This warp's part (every team-th, from `turn` on) of the next 32 * team slots of the row into the queue, those that show no
  // key left out but for the warp's last entry of the row's slots here (its owners have to leave the row's result; one
  // without a slot of its own gets an empty entry).  An entry: the record's address (0: none), the first and one past the
  // last visible key of the sub-block (8 bits each), and the row (times 2, + 1 if it is the warp's last entry of it).
  static __device__ __forceinline__ int resolve(const AttendArgs& a, Cursor& c, const uint32_t* starts, int4* queue, int tail,
                                                int team, int turn, int lane) {
    const int rows_h = a.hkv * a.tiles;
    if (!c.entered) enter_row(a, c, starts, lane);
    // (behind the last key of a row that takes its sub-blocks one after the other there is nothing to look for)
    const bool behind = a.sel == nullptr && c.j >= running_slots(c.first, c.last);
    const int left = min((uint32_t)(c.len - c.j), c.end - c.next), count = behind ? left : min(32 * team, left);
    const int own = behind ? 0 : (count - turn + team - 1) / team;  // (0 where count <= turn)
    const int j = c.j + lane * team + turn;
    int sub = -1;
    if (a.sel == nullptr) {
      if (lane < own) sub = running_sub(j, c.first, c.last);
    } else if (a.n_sel <= 32) {
      const int at = min(j / a.per, 31), entry = __shfl_sync(0xFFFFFFFFu, c.entry, at);
      if (lane < own && !(c.twice >> at & 1)) sub = selected_sub(entry, j - at * a.per, a.per, c.first, c.last);
    } else if (lane < own) {
      const int32_t* row = a.sel + ((int64_t)c.n * a.hkv + c.hm / a.tiles) * a.n_sel;
      const int at = j / a.per, entry = row[at];
      sub = selected_sub(entry, j - at * a.per, a.per, c.first, c.last);
#pragma unroll 1
      for (int i = 0; i < at && sub >= 0; ++i)
        if (row[i] == entry) sub = -1;
    }
    const int page = sub < 0 || c.seq < 0 ? -1 : page_of(a.b, c.seq, sub);
    const bool over = c.j + count == c.len || c.next + count == c.end;
    const bool final = over && lane == max(own - 1, 0);
    const bool keep = page >= 0 || final;
    const unsigned kept = __ballot_sync(0xFFFFFFFFu, keep);
    if (keep) {
      const int base = sub * kPage;
      const uint64_t at = page < 0 ? 0 : reinterpret_cast<uint64_t>(a.cache) + (int64_t)page * a.page_stride +
                                             (int64_t)(c.hm / a.tiles) * C::kRecord;
      queue[(tail + __popc(kept & ((1u << lane) - 1))) % C::kQueue] =
          make_int4((int)(uint32_t)at, (int)(uint32_t)(at >> 32),
                    page < 0 ? 0 : max(0, c.first - base) | min(kPage, c.last - base) << 8, (c.n * rows_h + c.hm) * 2 + final);
    }
    __syncwarp();
    c.next += count;
    c.j += count;
    if (c.j == c.len && c.next < c.end) {  // the next row
      c.j = 0;
      if (++c.hm == rows_h) c.hm = 0, ++c.n;
      c.entered = false;
    }
    return tail + __popc(kept);
  }

  static __device__ __forceinline__ const uint8_t* record_of(const int4& e) {
    return reinterpret_cast<const uint8_t*>((uint64_t)(uint32_t)e.y << 32 | (uint32_t)e.x);
  }
  static constexpr float kNone = -3e38f;  // a maximum of no scores

  // ---- the consumer's side.  The thread's heads in tile h are 8 h + 2 c and 8 h + 2 c + 1 (c = lane % 4).
  float o[MT][NH][4];      // O^T: d = (DV / 8) r + 2 j + e / 2 (r = lane / 4) of head 8 h + 2 c + e % 2
  uint32_t q[NH][KS * 2];  // Q of head 8 h + r: d = c * DQK / 4 + 2 i, + 1
  float2 f[NH], m[NH], l[NH];  // of the thread's heads: factor, reference m of the powers of two, the thread's share of the sum

  // A new row: its queries are asked for, then (when the copies of the first pages are under way) made ready.
  __device__ __forceinline__ void ask(const AttendArgs& a, uint32_t row, int lane) {
    const int rows_h = a.hkv * a.tiles, r = lane >> 2, c = lane & 3;
    const int n = row / rows_h, hm = row % rows_h, h = hm / a.tiles, g = hm % a.tiles * C::kHeads + r;
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + (int64_t)n * a.q_row + (int64_t)(h * a.group + g) * a.q_head +
                          c * (DQK / 4);
#pragma unroll
    for (int i = 0; i < NH; ++i) load_q(q[i], g + 8 * i < a.group ? src + 8 * i * a.q_head : nullptr);
  }
  __device__ __forceinline__ void begin(const AttendArgs& a, int lane) {
#pragma unroll
    for (int i = 0; i < NH; ++i) {
      float factor;
      scale_q(q[i], a.q_half, factor);
      // (finite and not 0, so that -inf stays -inf)
      factor = fminf(fmaxf(factor * a.scale_log2, 1e-38f), 3e38f);
      const int from = (lane & 3) * 8;  // row r = 2 c
      f[i] = make_float2(__shfl_sync(0xFFFFFFFFu, factor, from), __shfl_sync(0xFFFFFFFFu, factor, from + 4));
      m[i] = make_float2(kNone, kNone);
      l[i] = make_float2(0.0f, 0.0f);
    }
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int i = 0; i < NH; ++i) o[j][i][0] = o[j][i][1] = o[j][i][2] = o[j][i][3] = 0.0f;
  }

  // One page: keys [lo, lim) of its 64 are visible.
  __device__ __forceinline__ void page(uint8_t* rec, int lim, int lo, int lane) {
    const int r = lane >> 2, c = lane & 3;
    const bool whole = lim >= kPage && lo <= 0;
    const int row = r & 1 ? 4 + (r >> 1 ^ 1) : r >> 1;  // key of the tile's row r
    const uint8_t* krec = rec + row * (DQK / 2) + c * (DQK / 8);
    const uint8_t* kscales = rec + k_scale_at(DQK) + row * (DQK / kGroup) + c * (DQK / 64);
    float s[4][NH][4];  // S^T: element e is key 16 t + row + 8 (e / 2) of head 8 h + 2 c + e % 2
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int h = 0; h < NH; ++h) s[t][h][0] = s[t][h][1] = s[t][h][2] = s[t][h][3] = 0.0f;
      uint32_t w[2][DQK / 32], sc[2][DQK / 64];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint8_t* codes = krec + (16 * t + 8 * x) * (DQK / 2);
        const uint8_t* scales = kscales + (16 * t + 8 * x) * (DQK / kGroup);
        if constexpr (DQK == 128) {
          const uint4 y = *reinterpret_cast<const uint4*>(codes);
          w[x][0] = y.x, w[x][1] = y.y, w[x][2] = y.z, w[x][3] = y.w;
          const uint32_t both = __byte_perm(*reinterpret_cast<const uint16_t*>(scales), 0, 0x4140) << 7;
          sc[x][0] = low2(both), sc[x][1] = high2(both);
        } else {
#pragma unroll
          for (int g = 0; g < DQK / 64; ++g) {
            const uint2 y = *reinterpret_cast<const uint2*>(codes + 8 * g);
            w[x][2 * g] = y.x, w[x][2 * g + 1] = y.y;
            sc[x][g] = scale2(scales[g]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < DQK / 32; ++j) {
        const uint32_t z0 = sc[0][j / 2], z1 = sc[1][j / 2];
        const uint32_t a0 = mul2(decode_byte<0>(w[0][j]), z0), a1 = mul2(decode_byte<0>(w[1][j]), z1);
        const uint32_t a2 = mul2(decode_byte<1>(w[0][j]), z0), a3 = mul2(decode_byte<1>(w[1][j]), z1);
        const uint32_t b0 = mul2(decode_byte<2>(w[0][j]), z0), b1 = mul2(decode_byte<2>(w[1][j]), z1);
        const uint32_t b2 = mul2(decode_byte<3>(w[0][j]), z0), b3 = mul2(decode_byte<3>(w[1][j]), z1);
#pragma unroll
        for (int h = 0; h < NH; ++h) mma(s[t][h], a0, a1, a2, a3, q[h][4 * j], q[h][4 * j + 1]);
#pragma unroll
        for (int h = 0; h < NH; ++h) mma(s[t][h], b0, b1, b2, b3, q[h][4 * j + 2], q[h][4 * j + 3]);
      }
    }
    if (!whole) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int key = 16 * t + 8 * x + row;
          if (key < lo || key >= lim)
#pragma unroll
            for (int h = 0; h < NH; ++h) s[t][h][2 * x] = s[t][h][2 * x + 1] = -INFINITY;
        }
      // what stands in the other keys' places may be anything, NaN too: with a scale of 0 their values are 0
#pragma unroll
      for (int key = lane; key < kPage; key += 32)
        if (key < lo || key >= lim) {
          uint8_t* z = rec + v_scale_at(DQK, DV) + key * (DV / kGroup);
          if constexpr (DV == 128) *reinterpret_cast<uint2*>(z) = make_uint2(0, 0);
          else *reinterpret_cast<uint32_t*>(z) = 0;
        }
      ptx::fence_proxy_async_smem();  // (before the record that is copied here next)
      __syncwarp();
    }
    // Softmax, in powers of two, against m, kBelow less than a maximum of the scores so far.  m is raised, and O and the sums
    // with it, when a score is more than 2^kMost above it, so most pages need no exchange between the threads that share a
    // head.  The largest P is 2^kBelow to 2^kMost: as fp16, a P is off by 2^-11 of itself at most, or, where it is below 2^-14,
    // by 2^-25, which is 2^-32 of the largest or less (with kBelow = 0 it would be 2^-25 of it, and a flat tail of many small
    // weights would be lost from O).  (The first m is so low that every number is above it, and it scales zeros, or NaN, which
    // stays.)
    constexpr float kBelow = 7.0f, kMost = 15.0f;
    uint32_t p[4][NH][2];  // P^T as the tensor core takes it: fp16 pairs of keys (of rows 2c, 2c + 1, and 8 more) of head 8 h + r
    float2 y[4][NH][2];
    float most = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int h = 0; h < NH; ++h) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
          y[t][h][x] = fma2(make_float2(s[t][h][2 * x], s[t][h][2 * x + 1]), f[h], make_float2(-m[h].x, -m[h].y));
        most = max3(max3(most, y[t][h][0].x, y[t][h][0].y), y[t][h][1].x, y[t][h][1].y);
      }
    if (__any_sync(0xFFFFFFFFu, most > kMost)) {
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        float2 top = make_float2(-INFINITY, -INFINITY);
#pragma unroll
        for (int t = 0; t < 4; ++t)
          top.x = max3(top.x, s[t][h][0], s[t][h][2]), top.y = max3(top.y, s[t][h][1], s[t][h][3]);
#pragma unroll
        for (int k = 4; k < 32; k *= 2) {
          top.x = fmaxf(top.x, __shfl_xor_sync(0xFFFFFFFFu, top.x, k));
          top.y = fmaxf(top.y, __shfl_xor_sync(0xFFFFFFFFu, top.y, k));
        }
        // m is the largest score to within its last bit, but the scores below are not rounded before m is taken off: from 2^28
        // on the difference is more than fp16 holds.  So what the largest has over kBelow, or lacks, is taken off as well.
        const float2 was = m[h], z = top;
        top = make_float2(fmaxf(was.x, z.x * f[h].x - kBelow), fmaxf(was.y, z.y * f[h].y - kBelow));
        float2 over = make_float2(fmaf(z.x, f[h].x, -top.x) - kBelow, fmaf(z.y, f[h].y, -top.y) - kBelow);
        over = make_float2(top.x > was.x ? over.x : fmaxf(over.x, 0.0f), top.y > was.y ? over.y : fmaxf(over.y, 0.0f));
        const float2 k = make_float2(exp2_fast(was.x - top.x), exp2_fast(was.y - top.y));
        l[h] = mul2(l[h], k);
#pragma unroll
        for (int j = 0; j < MT; ++j) o[j][h][0] *= k.x, o[j][h][1] *= k.y, o[j][h][2] *= k.x, o[j][h][3] *= k.y;
        m[h] = top;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            y[t][h][x] = add2(fma2(make_float2(s[t][h][2 * x], s[t][h][2 * x + 1]), f[h], make_float2(-top.x, -top.y)),
                              make_float2(-over.x, -over.y));
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float2 e = make_float2(exp2_fast(y[t][h][x].x), exp2_fast(y[t][h][x].y));
          l[h] = add2(l[h], e);
          asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(p[t][h][x]) : "r"(pack_half(e.x, e.y)));
        }
    // PV
    const int odd = 4 + (c ^ 1);  // keys of the tile's rows 2c and 2c + 1: c and odd
    const uint8_t* vrec = rec + v_code_at(DQK) + r * (DV / 16);
    const uint8_t* vscales = rec + v_scale_at(DQK, DV) + (DV == 128 ? r : r >> 1);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      uint32_t w[4][DV / 64], z[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 16 * t + 8 * (i / 2) + (i % 2 ? odd : c);
        const uint8_t* at = vrec + key * (DV / 2);
        if constexpr (DV == 128) {
          const uint2 x = *reinterpret_cast<const uint2*>(at);
          w[i][0] = x.x, w[i][1] = x.y;
        } else {
          w[i][0] = *reinterpret_cast<const uint32_t*>(at);
        }
        z[i] = vscales[key * (DV / kGroup)];
      }
      const uint32_t z0 = z[0] * 128u + (z[1] << 23), z1 = z[2] * 128u + (z[3] << 23);
#pragma unroll
      for (int j = 0; j < DV / 64; ++j) {
        // codes of two keys side by side in every byte: even values of d, then odd ones
        constexpr uint32_t kLow = 0x0F0F0F0Fu;
        const uint32_t x0 = (w[0][j] & kLow) | ((w[1][j] << 4) & ~kLow), x1 = (w[2][j] & kLow) | ((w[3][j] << 4) & ~kLow);
        const uint32_t y0 = ((w[0][j] >> 4) & kLow) | (w[1][j] & ~kLow), y1 = ((w[2][j] >> 4) & kLow) | (w[3][j] & ~kLow);
        pv<0>(o[4 * j + 0], x0, y0, x1, y1, z0, z1, p[t]);
        pv<1>(o[4 * j + 1], x0, y0, x1, y1, z0, z1, p[t]);
        pv<2>(o[4 * j + 2], x0, y0, x1, y1, z0, z1, p[t]);
        pv<3>(o[4 * j + 3], x0, y0, x1, y1, z0, z1, p[t]);
      }
    }
  }
  template <int I>
  static __device__ __forceinline__ void pv(float (&acc)[NH][4], uint32_t x0, uint32_t y0, uint32_t x1, uint32_t y1, uint32_t z0,
                                            uint32_t z1, const uint32_t (&p)[NH][2]) {
    const uint32_t a0 = mul2(decode_byte<I>(x0), z0), a1 = mul2(decode_byte<I>(y0), z0);
    const uint32_t a2 = mul2(decode_byte<I>(x1), z1), a3 = mul2(decode_byte<I>(y1), z1);
#pragma unroll
    for (int h = 0; h < NH; ++h) mma(acc[h], a0, a1, a2, a3, p[h][0], p[h][1]);
  }

  // Four neighbouring values of d (from (DV / 8) r + 4 i on) of the thread's head 8 h + 2 c + e.
  __device__ __forceinline__ float4 piece(int h, int e, int i) const {
    return make_float4(o[2 * i][h][e], o[2 * i][h][2 + e], o[2 * i + 1][h][e], o[2 * i + 1][h][2 + e]);
  }

  // The row's result: whole, or this team's part of it (`part` not null).  `join`: the team's warps' join buffers.
  __device__ __forceinline__ void finish(const AttendArgs& a, uint32_t row, float* part, float* join, int team, int turn,
                                         int barrier, int lane) {
    constexpr int kHeads = C::kHeads, PIECES = DV / 32;  // pieces of a thread and head
    const int rows_h = a.hkv * a.tiles, r = lane >> 2, c = lane & 3;
    const int n = row / rows_h, hm = row % rows_h, g0 = hm % a.tiles * kHeads;
    const int64_t at0 = (int64_t)n * a.hq + hm / a.tiles * a.group + g0;  // the tile's first query head
    const int used = min(kHeads, a.group - g0);
    const bool left = part == nullptr && !a.fill && sequence_of_warp(a.b, n, lane) < 0;  // a row to leave as it was
    const float weight = a.weight != nullptr && part == nullptr ? *a.weight : 1.0f;
    float sum[NH][2], top[NH][2];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      sum[h][0] = l[h].x, sum[h][1] = l[h].y;
      top[h][0] = m[h].x, top[h][1] = m[h].y;
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int k = 4; k < 32; k *= 2) sum[h][e] += __shfl_xor_sync(0xFFFFFFFFu, sum[h][e], k);
    }
    if (team == 1) {
      if (left) return;
      const bool whole = part == nullptr, wide = !whole || a.o_dtype == kF32;
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int x = 8 * h + 2 * c + e;
          if (x >= used) continue;
          if (r == 0) {
            if (whole) store_lse(a, at0 + x, top[h][e], sum[h][e]);
            else part[kHeads * DV + x] = top[h][e], part[kHeads * (DV + 1) + x] = sum[h][e];
          }
          const float k = !whole ? 1.0f : sum[h][e] != 0.0f ? __fdividef(weight, sum[h][e]) : 0.0f;
          if (wide) {
            float4* to = reinterpret_cast<float4*>((whole ? static_cast<float*>(a.o) + at0 * DV : part) + x * DV + r * (DV / 8));
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
              float4 v = whole && a.accumulate ? to[i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              const float4 y = piece(h, e, i);
              v.x += y.x * k, v.y += y.y * k, v.z += y.z * k, v.w += y.w * k;
              to[i] = v;
            }
          } else {  // 16 bytes at once
            uint4* to = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.o) + (at0 + x) * DV + r * (DV / 8));
            const bool half = a.o_dtype == kF16;
#pragma unroll
            for (int i = 0; i < PIECES; i += 2) {
              const float4 y = piece(h, e, i), z = piece(h, e, i + 1);
              to[i / 2] = make_uint4(pack16(y.x * k, y.y * k, half), pack16(y.z * k, y.w * k, half),
                                     pack16(z.x * k, z.y * k, half), pack16(z.z * k, z.w * k, half));
            }
          }
        }
      return;
    }
    // Join: maxima, then every warp's O against the common maximum, some columns a round.  The 16-byte pieces of a row
    // are exchanged so that neither side meets bank conflicts.
    constexpr int CS = PIECES / C::ROUNDS, kMl = kHeads * DV / C::ROUNDS;
    float* mine = join + turn * C::kJoin;
    if (r == 0)
#pragma unroll
      for (int h = 0; h < NH; ++h) mine[kMl + 8 * h + 2 * c] = top[h][0], mine[kMl + 8 * h + 2 * c + 1] = top[h][1];
    named_barrier(barrier, team * 32);
    float k[NH][2];
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int x = 8 * h + 2 * c + e;
        float common = r < team ? join[r * C::kJoin + kMl + x] : kNone;
#pragma unroll
        for (int w = 4; w < 32; w *= 2) common = fmaxf(common, __shfl_xor_sync(0xFFFFFFFFu, common, w));
        k[h][e] = exp2_fast(top[h][e] - common);
        if (r == 0) mine[kMl + kHeads + x] = sum[h][e] * k[h][e], mine[kMl + 2 * kHeads + x] = common;
      }
    const int swap = CS == 4 ? c : (c & 1) | (c & 2) << 1;
#pragma unroll
    for (int t = 0; t < C::ROUNDS; ++t) {
      if (t > 0) named_barrier(barrier, team * 32);
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float4* to = reinterpret_cast<float4*>(mine) + (8 * h + 2 * c + e) * (8 * CS);
#pragma unroll
          for (int i = 0; i < CS; ++i) {
            float4 v = piece(h, e, t * CS + i);
            v.x *= k[h][e], v.y *= k[h][e], v.z *= k[h][e], v.w *= k[h][e];
            to[(r * CS + i) ^ swap] = v;
          }
        }
      named_barrier(barrier, team * 32);
#pragma unroll 1
      for (int i = turn * 32 + lane; i < kHeads * 8 * CS; i += team * 32) {
        const int x = i / (8 * CS), at = i % (8 * CS), d = at / CS * (DV / 8) + (t * CS + at % CS) * 4;
        if (x >= used || left) continue;
        const int q = x >> 1 & 3, place = x * (8 * CS) + (at ^ (CS == 4 ? q : (q & 1) | (q & 2) << 1));
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float all = 0.0f;
#pragma unroll 1
        for (int w = 0; w < team; w += 2) {
          const float *from = join + w * C::kJoin, *next = from + C::kJoin;
          const float4 y = reinterpret_cast<const float4*>(from)[place], z = reinterpret_cast<const float4*>(next)[place];
          v.x += y.x + z.x, v.y += y.y + z.y, v.z += y.z + z.z, v.w += y.w + z.w;
          all += from[kMl + kHeads + x] + next[kMl + kHeads + x];
        }
        const float common = mine[kMl + 2 * kHeads + x];
        if (part != nullptr) {
          *reinterpret_cast<float4*>(part + x * DV + d) = v;
          if (at == 0 && t == 0) part[kHeads * DV + x] = common, part[kHeads * (DV + 1) + x] = all;
        } else {
          store4<DV>(a, at0 + x, d, v, all != 0.0f ? __fdividef(weight, all) : 0.0f);
          if (at == 0 && t == 0) store_lse(a, at0 + x, common, all);
        }
      }
    }
  }
};

// Joins what the blocks of a cluster have of a row (`mine`: this block's part, in shared memory), each of them some columns.
template <class C>
__device__ __forceinline__ void join_cluster(const AttendArgs& a, uint32_t row, const float* mine, uint32_t rank) {
  constexpr int kHeads = C::kHeads, DV = C::DV;
  ptx::cluster_sync();  // all parts are there
  const uint32_t rows_h = a.hkv * a.tiles;
  const int n = row / rows_h, hm = row % rows_h, g0 = hm % a.tiles * kHeads;
  const int64_t at0 = (int64_t)n * a.hq + hm / a.tiles * a.group + g0;
  const int i = rank * (C::NW * 32) + threadIdx.x, x = i / (DV / 4), d = i % (DV / 4) * 4;
  if (x < min(kHeads, a.group - g0) && (a.fill || sequence_of(a.b, n) >= 0)) {
    float m[kCluster], l[kCluster], top = Worker<C>::kNone, sum = 0.0f;
    float4 v[kCluster], acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < (int)kCluster; ++k) {
      m[k] = Worker<C>::kNone, l[k] = 0.0f, v[k] = acc;
      if (k < (int)a.cluster) {
        const float* part = ptx::of_rank(mine, k);
        m[k] = part[kHeads * DV + x], l[k] = part[kHeads * (DV + 1) + x];
        v[k] = *reinterpret_cast<const float4*>(part + x * DV + d);
      }
    }
#pragma unroll
    for (int k = 0; k < (int)kCluster; ++k) top = fmaxf(top, m[k]);
#pragma unroll
    for (int k = 0; k < (int)kCluster; ++k) {
      const float f = exp2_fast(m[k] - top);
      sum += l[k] * f;
      acc.x += v[k].x * f, acc.y += v[k].y * f, acc.z += v[k].z * f, acc.w += v[k].w * f;
    }
    if (d == 0) store_lse(a, at0 + x, top, sum);
    store4<DV>(a, at0 + x, d, acc, sum != 0.0f ? (a.weight ? *a.weight : 1.0f) / sum : 0.0f);
  }
  ptx::cluster_sync();  // nobody leaves while its part is read
}

template <class C>
__global__ void __launch_bounds__(C::NW * 32, 1) attend_kernel(const AttendArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t line[2];  // of a ragged line: slots, the longest row's
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  uint8_t* ring = smem + warp * (C::STAGES * C::kRecord);
  float* join = reinterpret_cast<float*>(smem + C::NW * C::STAGES * C::kRecord);
  int4* queue = reinterpret_cast<int4*>(join + C::NW * C::kJoin) + warp * C::kQueue;
  uint64_t* bars = reinterpret_cast<uint64_t*>(queue + (C::NW - warp) * C::kQueue) + warp * C::STAGES;
  uint32_t* starts = reinterpret_cast<uint32_t*>(smem + C::NW * C::kWarp);
  if (lane < C::STAGES) ptx::mbar_init(bars + lane, 1);
  ptx::fence_mbar_init();
  start_in_order();
  const uint32_t rows_h = a.hkv * a.tiles, rows = a.b.n_rows * rows_h;
  uint32_t total = rows * a.slots;
  Split split = a.split;
  if (a.slots == 0) {
    // the page table on its way into L2 (128 bytes a thread: all of an ordinary one)
    const int64_t line128 = ((int64_t)blockIdx.x * (C::NW * 32) + threadIdx.x) * 32;
    if (line128 < (int64_t)(a.b.n_seqs - 1) * a.b.page_row + a.b.width)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(a.b.pages + line128));
    // the ragged line: every block counts the slots before each row (n_rows <= kMaxRagged)
#pragma unroll 1
    for (int n = threadIdx.x; n < a.b.n_rows; n += C::NW * 32) {
      const int seq = sequence_of(a.b, n), pos = seq < 0 ? -1 : position_of(a.b, seq, n);
      starts[n + 1] = running_slots(pos < 0 ? 0 : first_key(pos, a.window), keys_up_to(a.b, pos));
    }
    __syncthreads();
    if (warp == 0) {
      uint32_t sum = 0, longest = 0;
      if (lane == 0) starts[0] = 0;
#pragma unroll 1
      for (int n0 = 0; n0 < a.b.n_rows; n0 += 32) {
        uint32_t x = n0 + lane < a.b.n_rows ? starts[n0 + lane + 1] : 0;
        longest = max(longest, x);
#pragma unroll
        for (int k = 1; k < 32; k *= 2) {
          const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, x, k);
          if (lane >= k) x += y;
        }
        if (n0 + lane < a.b.n_rows) starts[n0 + lane + 1] = sum + x;
        sum += __shfl_sync(0xFFFFFFFFu, x, 31);
      }
#pragma unroll
      for (int k = 16; k > 0; k /= 2) longest = max(longest, __shfl_xor_sync(0xFFFFFFFFu, longest, k));
      if (lane == 0) line[0] = sum * rows_h, line[1] = longest;
    }
    __syncthreads();
    total = line[0];
    split = split_line(rows, total, line[1], a.warps);
    if (blockIdx.x == 0 && a.part != nullptr) {
#pragma unroll 1
      for (int n = threadIdx.x; n <= a.b.n_rows; n += C::NW * 32) a.starts[n] = starts[n];
      if (threadIdx.x == 0) a.starts[a.b.n_rows + 1] = split.cut ? split.share : 0;
    }
  }
  // neighbouring teams are on different SMs, so that a few of them use many
  const int team = split.team, turn = warp % team, sub_team = warp / team;
  const uint32_t rank = blockIdx.x % a.cluster;
  const uint32_t me = a.cluster > 1 ? blockIdx.x / a.cluster : sub_team * gridDim.x + blockIdx.x;
  const int every = team * a.cluster, first_slot = a.cluster > 1 ? warp * a.cluster + rank : turn;

  typename Worker<C>::Cursor cur;
  auto start_of = [&](uint32_t row) {  // the line's slots before a row
    if (a.slots) return row * a.slots;
    const uint32_t n = row / rows_h, s0 = starts[n];
    return n == a.b.n_rows ? total : s0 * rows_h + row % rows_h * (starts[n + 1] - s0);
  };
  uint32_t row = 0;
  if (split.cut) {
    if ((uint64_t)me * split.share >= total) return;
    cur.next = me * split.share;
    cur.end = total - cur.next < split.share ? total : cur.next + split.share;
    if (a.slots) {
      row = cur.next / a.slots;
    } else {
      int lo = 0, hi = a.b.n_rows;
#pragma unroll 1
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (starts[mid] * rows_h <= cur.next) lo = mid;
        else hi = mid;
      }
      row = lo * rows_h + (cur.next - starts[lo] * rows_h) / (starts[lo + 1] - starts[lo]);
    }
  } else {
    if ((uint64_t)me * split.share >= rows) return;
    row = me * split.share;
    cur.next = start_of(row);
    cur.end = start_of(min(rows - row, split.share) + row);
  }
  cur.n = row / rows_h, cur.hm = row % rows_h, cur.j = cur.next - start_of(row);
  const bool cut_before = cur.j != 0;  // the first row's earlier slots are another team's
  cur.entered = false;

  __syncwarp();
  Worker<C> w;
  int head, tail = 0, issued = 0;
  uint32_t phases = 0, flying = 0;  // each stage's parity of the next phase; copies on their way
  bool lost = false;                // a copy did not come: no more are made, rows from here on are NaN
  bool fresh = true, first_row = true;
  // the ring holds STAGES records: STAGES - 1 on their way (the first of them before the loop's first page) while one is
  // worked on
#pragma unroll 1
  for (head = 1 - C::STAGES;; ++head) {
#pragma unroll 1
    while (tail - issued < C::STAGES && tail - head <= C::kQueue - 32 && cur.next < cur.end)
      tail = Worker<C>::resolve(a, cur, starts, queue, tail, every, first_slot, lane);
    if (head == 1 - C::STAGES) w.ask(a, row, lane);  // (before the pages: they would be ahead of it in the memory's queue)
    if (issued < tail) {
      const uint8_t* src = Worker<C>::record_of(queue[issued % C::kQueue]);
      const int stage = issued++ % C::STAGES;
      if (src != nullptr && !lost && !a.stall) {
        if (elected()) copy_record(ring + stage * C::kRecord, src, C::kRecord, bars + stage);
        flying |= 1u << stage;
      }
    }
    if (head < 0) continue;
    if (head == issued) break;
    const int4 e = queue[head % C::kQueue];
    const int stage = head % C::STAGES;
    if (fresh) {
      if (!first_row) w.ask(a, (uint32_t)e.w >> 1, lane);
      w.begin(a, lane);
    }
    fresh = e.w & 1;
    if (Worker<C>::record_of(e) != nullptr) {
      lost = lost || !__all_sync(0xFFFFFFFFu, wait_for(bars + stage, phases >> stage & 1, a.wait_ns));
      if (!lost) {
        phases ^= 1u << stage, flying &= ~(1u << stage);
        w.page(ring + stage * C::kRecord, e.z >> 8, e.z & 255, lane);
      } else {
        for (int i = 0; i < C::NH; ++i) w.l[i].x = w.l[i].y = __int_as_float(0x7FFFFFFF);
      }
    }
    if (fresh) {
      if (lost) wait_all(bars, phases, flying, a.wait_ns), flying = 0;  // (before a part of the row goes where they end)
      // a row is whole here unless it began before this share, or goes on behind it
      const bool head_cut = first_row && cut_before;
      const bool tail_cut = head + 1 == tail && cur.next == cur.end && cur.j < cur.len;
      float* part = head_cut || tail_cut ? a.part + ((size_t)me * 2 + (head_cut ? 0 : 1)) * C::kPart : nullptr;
      if (a.cluster > 1) part = reinterpret_cast<float*>(smem);  // (the first warp's ring: a cluster has one row)
      w.finish(a, (uint32_t)e.w >> 1, part, join + sub_team * team * C::kJoin, team, turn, 1 + sub_team, lane);
      first_row = false;
    }
    __syncwarp();
  }
  if (a.cluster > 1) join_cluster<C>(a, row, reinterpret_cast<const float*>(smem), rank);
  if (lost && a.err != nullptr && lane == 0) atomicOr(a.err, 1);
}

// Joins the parts of the rows that were cut, in the order of the line.  WPH warps share a row's query head:
// 1 where a row has a few parts, 8 where one row is cut over many teams.
template <class C, int WPH>
__global__ void __launch_bounds__(256) merge_kernel(const AttendArgs a) {
  constexpr int DV = C::DV, V4 = DV / 4;
  __shared__ float shared_o[8][DV];
  __shared__ float shared_ml[8][2];
  start_in_order();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rows_h = a.hkv * a.tiles;
  const int64_t unit = WPH == 1 ? (int64_t)blockIdx.x * 8 + warp : blockIdx.x;  // (row, query head)
  if (unit >= (int64_t)a.b.n_rows * a.hq) return;
  const int n = unit / a.hq, hq = unit % a.hq, h = hq / a.group, g = hq % a.group, x = g % C::kHeads;
  const uint32_t hm = h * a.tiles + g / C::kHeads;
  uint32_t start, len, per = a.split.share;
  if (a.slots) {
    len = a.slots, start = ((uint32_t)n * rows_h + hm) * len;
  } else {
    const uint32_t s0 = a.starts[n];
    len = a.starts[n + 1] - s0, start = s0 * rows_h + hm * len;
    per = a.starts[a.b.n_rows + 1];
  }
  if (per == 0) return;
  const uint32_t w0 = start / per, parts = (start + len - 1) / per - w0 + 1;
  if (parts == 1) return;  // the row was not cut
  if (!a.fill && sequence_of(a.b, n) < 0) return;
  // the first team has the row as its last, the others as their first; this warp has every WPH-th part
  auto part_of = [&](uint32_t i) { return a.part + ((size_t)(w0 + i) * 2 + (i == 0 ? 1 : 0)) * C::kPart; };
  const uint32_t mine = WPH == 1 ? 0 : warp;
  float m = Worker<C>::kNone, l = 0.0f;  // (a maximum is never NaN: fmaxf leaves it out; the NaN is in the sums)
  for (uint32_t i = mine + WPH * lane; i < parts; i += WPH * 32) m = fmaxf(m, part_of(i)[C::kHeads * DV + x]);
#pragma unroll
  for (int k = 16; k > 0; k /= 2) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, k));
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // values 4 lane to 4 lane + 3 (lane < V4)
  for (uint32_t i0 = mine; i0 < parts; i0 += WPH * 32) {
    const uint32_t own = i0 + WPH * lane;
    float factor = 0.0f;
    if (own < parts) {
      const float* p = part_of(own) + C::kHeads * DV + x;
      factor = exp2_fast(p[0] - m);
      l += p[C::kHeads] * factor;
    }
    const int count = min(32u, (parts - i0 + WPH - 1) / WPH);
#pragma unroll 8
    for (int k = 0; k < count; ++k) {
      const float f = __shfl_sync(0xFFFFFFFFu, factor, k);
      if (lane < V4) {
        const float4 v = reinterpret_cast<const float4*>(part_of(i0 + WPH * k) + x * DV)[lane];
        acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
      }
    }
  }
#pragma unroll
  for (int k = 16; k > 0; k /= 2) l += __shfl_xor_sync(0xFFFFFFFFu, l, k);
  if (WPH > 1) {
    if (lane < V4) reinterpret_cast<float4*>(shared_o[warp])[lane] = acc;
    if (lane == 0) shared_ml[warp][0] = m, shared_ml[warp][1] = l;
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int k = 0; k < WPH; ++k) m = fmaxf(m, shared_ml[k][0]);
    l = 0.0f;
    acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < WPH; ++k) {
      const float f = exp2_fast(shared_ml[k][0] - m);
      l += shared_ml[k][1] * f;
      if (lane < V4) {
        const float4 v = reinterpret_cast<const float4*>(shared_o[k])[lane];
        acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
      }
    }
  }
  if (lane == 0) store_lse(a, unit, m, l);
  if (lane < V4) store4<DV>(a, unit, 4 * lane, acc, l != 0.0f ? (a.weight ? *a.weight : 1.0f) / l : 0.0f);
}

}  // namespace cache
}  // namespace nsa
