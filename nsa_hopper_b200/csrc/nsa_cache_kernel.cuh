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

#include "nsa_cache_index.h"
#include "ptx.cuh"

namespace nsa {
namespace cache {

enum : int { kBf16 = 0, kF32 = 1, kF16 = 2 };

// ------------------------------------------------------------------ 4-bit conversions
// Two codes of byte I of `w` as fp16 pair (low nibble in the low half).
template <int I>
__device__ __forceinline__ uint32_t decode_byte(uint32_t w) {
  uint32_t r;
  if constexpr (I == 0)
    asm("{.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b0;}" : "=r"(r) : "r"(w));
  else if constexpr (I == 1)
    asm("{.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b1;}" : "=r"(r) : "r"(w));
  else if constexpr (I == 2)
    asm("{.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b2;}" : "=r"(r) : "r"(w));
  else
    asm("{.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b3;}" : "=r"(r) : "r"(w));
  return r;
}
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
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// A scale byte in both halves of an fp16 pair.
__device__ __forceinline__ uint32_t scale2(uint32_t byte) { return byte * 0x00800080u; }

// The scale byte of a group from max|x| / 6: nearest, ties to even, at most 10240 (0xE2).
__device__ __forceinline__ uint32_t scale_byte(float raw) {
  if (raw >= 6.103515625e-05f) {  // 2^-14, the smallest normal scale
    const uint32_t b = __float_as_uint(raw);
    return min(((b + 0x7FFFFu + ((b >> 20) & 1u)) >> 20) - 896u, 226u);
  }
  return (uint32_t)__float2int_rn(raw * 131072.0f);  // eighths of 2^-14
}

// ------------------------------------------------------------------ writing
// One thread quantises one group: 32 bytes in, 8 bytes of codes and a byte of scale out, so the kernel is
// bound by memory (2.56 bytes a value).  x / s must fall on the right side of the borders between codes (0.25,
// 0.75, ... 5), and exactly on one where it is one, for ties to go to the even code.  x (1 / s) has an error of
// 2^-24 and would miss some of the ties; fma(x, 1 / s, 192) - 192 rounds the quotient to a multiple of 2^-16
// instead.  A border is such a multiple, and with the 8 or 11 significant bits of x no other quotient is nearer
// to a border t than t 2^-11, so the codes are those of a true division.
struct WriteArgs {
  Batch b;
  const void* x[2];               // K, V [n_rows, Hkv, d], unit stride along d
  int64_t row_stride[2], head_stride[2];
  uint8_t* cache;
  int64_t page_stride;
  int32_t hkv, half;              // half: inputs are fp16, else bf16
};

template <int DQK, int DV, int WHICH>
__device__ __forceinline__ void write_group(const WriteArgs& a, uint32_t i) {
  constexpr int D = WHICH == 0 ? DQK : DV, GR = D / kGroup;
  const uint32_t total = (uint32_t)a.b.n_rows * a.hkv * GR;
  if ((i & ~31u) >= total) return;  // (whole warps)
  const bool in = i < total;
  const uint32_t g = i % GR, rh = (in ? i : total - 1) / GR, row = rh / a.hkv, h = rh % a.hkv;
  const uint16_t* src = static_cast<const uint16_t*>(a.x[WHICH]) + (int64_t)row * a.row_stride[WHICH] +
                        (int64_t)h * a.head_stride[WHICH] + g * kGroup;
  const uint4 lo = *reinterpret_cast<const uint4*>(src), hi = *reinterpret_cast<const uint4*>(src + 8);
  const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  uint32_t top = 0;  // |x| as integers: a NaN is above an infinity, an infinity above every number
#pragma unroll
  for (int j = 0; j < 8; ++j) top = __vmaxu2(top, w[j] & 0x7FFF7FFFu);
  top = max(top & 0xFFFFu, top >> 16);
  float amax;
  bool fine;
  if (a.half) {
    fine = top < 0x7C00u;
    amax = __half2float(__ushort_as_half((unsigned short)top));
  } else {
    fine = top < 0x7F80u;
    amax = __uint_as_float(top << 16);
  }
  uint32_t sb = fine ? scale_byte(__fdiv_rn(amax, 6.0f)) : 255u;
  const float s = __half2float(__ushort_as_half((unsigned short)(sb << 7)));
  uint32_t code[2] = {0, 0};
  if (fine && sb != 0) {
    const float inv = __frcp_rn(s);
    float y[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 f = a.half ? __half22float2(*reinterpret_cast<const __half2*>(&w[j]))
                              : make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
      y[2 * j] = __fadd_rn(__fmaf_rn(f.x, inv, 192.0f), -192.0f);
      y[2 * j + 1] = __fadd_rn(__fmaf_rn(f.y, inv, 192.0f), -192.0f);
    }
    code[0] = encode8(y), code[1] = encode8(y + 8);
  }
  // the scales of four neighbouring groups (of one token: GR is a multiple of 4) go out together
  sb |= __shfl_down_sync(0xFFFFFFFFu, sb, 1) << 8;
  sb |= __shfl_down_sync(0xFFFFFFFFu, sb, 2) << 16;
  const int seq = in ? sequence_of(a.b, row) : -1;
  if (seq < 0) return;
  const int pos = position_of(a.b, seq, row);
  const int page = pos < 0 ? -1 : page_of(a.b, seq, pos / kPage);
  if (page < 0) return;
  uint8_t* rec = a.cache + (int64_t)page * a.page_stride + (int64_t)h * record_bytes(DQK, DV);
  const int t = pos % kPage;
  uint8_t* codes = rec + (WHICH == 0 ? 0 : v_code_at(DQK)) + t * (D / 2) + g * 8;
  *reinterpret_cast<uint2*>(codes) = make_uint2(code[0], code[1]);
  if (g % 4 == 0) {
    uint8_t* scales = rec + (WHICH == 0 ? k_scale_at(DQK) : v_scale_at(DQK, DV)) + t * GR + g;
    *reinterpret_cast<uint32_t*>(scales) = sb;
  }
}

template <int DQK, int DV>
__global__ void __launch_bounds__(256) write_kernel(const WriteArgs a) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (blockIdx.y == 0) write_group<DQK, DV, 0>(a, i);
  else write_group<DQK, DV, 1>(a, i);
}

// ------------------------------------------------------------------ reading back
struct ReadArgs {
  Batch b;
  const uint8_t* cache;
  int64_t page_stride;
  void* y[2];  // K, V [Hkv, n_rows, d]
  int32_t hkv, dtype;
};

template <int DQK, int DV, int WHICH>
__device__ __forceinline__ void read_group(const ReadArgs& a, uint32_t i) {
  constexpr int D = WHICH == 0 ? DQK : DV, GR = D / kGroup;
  if (i >= (uint32_t)a.b.n_rows * a.hkv * GR) return;
  const uint32_t g = i % GR, hr = i / GR, h = hr / a.b.n_rows, row = hr % a.b.n_rows;
  const int seq = sequence_of(a.b, row);
  const int pos = seq < 0 ? -1 : position_of(a.b, seq, row);
  const int page = pos < 0 ? -1 : page_of(a.b, seq, pos / kPage);
  uint32_t v[8] = {};  // fp16 pairs; a token that is not there reads as zeros
  if (page >= 0) {
    const uint8_t* rec = a.cache + (int64_t)page * a.page_stride + (int64_t)h * record_bytes(DQK, DV);
    const int t = pos % kPage;
    const uint2 c = *reinterpret_cast<const uint2*>(rec + (WHICH == 0 ? 0 : v_code_at(DQK)) + t * (D / 2) + g * 8);
    const uint32_t s = scale2(rec[(WHICH == 0 ? k_scale_at(DQK) : v_scale_at(DQK, DV)) + t * GR + g]);
    v[0] = mul2(decode_byte<0>(c.x), s), v[1] = mul2(decode_byte<1>(c.x), s);
    v[2] = mul2(decode_byte<2>(c.x), s), v[3] = mul2(decode_byte<3>(c.x), s);
    v[4] = mul2(decode_byte<0>(c.y), s), v[5] = mul2(decode_byte<1>(c.y), s);
    v[6] = mul2(decode_byte<2>(c.y), s), v[7] = mul2(decode_byte<3>(c.y), s);
  }
  const int64_t at = (int64_t)hr * D + g * kGroup;
  if (a.dtype == kF32) {
    float4* out = reinterpret_cast<float4*>(static_cast<float*>(a.y[WHICH]) + at);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 p = __half22float2(*reinterpret_cast<__half2*>(&v[2 * j]));
      const float2 q = __half22float2(*reinterpret_cast<__half2*>(&v[2 * j + 1]));
      out[j] = make_float4(p.x, p.y, q.x, q.y);
    }
    return;
  }
  if (a.dtype == kBf16) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const __nv_bfloat162 p = __float22bfloat162_rn(__half22float2(*reinterpret_cast<__half2*>(&v[j])));
      v[j] = *reinterpret_cast<const uint32_t*>(&p);
    }
  }
  uint4* out = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.y[WHICH]) + at);
  out[0] = make_uint4(v[0], v[1], v[2], v[3]);
  out[1] = make_uint4(v[4], v[5], v[6], v[7]);
}

template <int DQK, int DV>
__global__ void __launch_bounds__(256) read_kernel(const ReadArgs a) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (blockIdx.y == 0) read_group<DQK, DV, 0>(a, i);
  else read_group<DQK, DV, 1>(a, i);
}

// ------------------------------------------------------------------ attention
// For a row n, KV head h and its G query heads (16 at a time, the M of one tensor-core tile):
//     z_j = scale * q . k_j,   O = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m),   LSE = m + ln sum_j exp(z_j - m)
// over the visible keys j, in one pass with the running maximum m (kept in powers of two).
//
// A key costs 9/16 (d_qk + d_v) bytes and 2 G (d_qk + d_v) operations: at d = 128 and G = 16 57 operations a
// byte, so the floor is the cache's bytes from DRAM, provided that turning 4 bits into tensor-core operands keeps
// up.  Hence the layout of the work: every warp is a worker of its own with a ring of page records in shared
// memory (asynchronous copies), and codes go from there straight into the registers that the tensor core
// reads (m16n8k16, fp16 in, fp32 out): no dequantised value is ever stored.  For that
//   * the d axis of QK is permuted so that a thread's K fragments are d_qk / 4 consecutive codes of one key: one
//     wide shared load, one conversion and one product with the scale for each pair, exact in fp16;
//   * a thread's V fragments are d_v / 8 consecutive codes of four keys, which are interleaved two and two; P needs no
//     exchange, its score registers are the A fragment.  The key axis is permuted (k index 2c, 2c + 1 of a tile of 8 is key
//     c, 4 + (c ^ 1)) so that neither K's nor V's shared loads collide more than two ways on the record as it is.
// Q has up to 8 (bf16) or 11 significant bits, so a power of two per row puts it into fp16 (below 2^-14 of the row's
// largest to within 2^-25 of it).  P is rounded to fp16 (at most 2^-11 of each term): the sum of
// its fp32 values is the divisor.  Scores, statistics and O are fp32.
//
// All (row, page) slots of the call stand in one line that is shared out evenly (split_line): teams of 1 to 8 warps of a
// block take turns at a row's pages and join their (m, sum, O) in shared memory; a row that is cut between teams leaves
// partial results in the workspace, and merge_kernel joins them in the order of the line.  Results do not depend on
// timing.
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
  int32_t hq, hkv, group, tiles; // tiles: 16-row tiles of a KV head's G query heads
  int32_t n_sel, per, window;    // per: sub-blocks of a selection block
  int32_t slots;                 // slots of every row; 0: as many as it has sub-blocks (the ragged line)
  uint32_t warps;                // of the device
  Split split;                   // (a ragged line's is worked out on the device)
  int32_t q_half, o_dtype, accumulate, fill;  // fill: rows of no sequence get O = 0, LSE = -inf; else they are left
  float scale_log2;
  int32_t* err;                  // optional: NSA_DEVERR_TIMEOUT (1) if a copy did not come
  uint64_t wait_ns;              // bound of every wait for a copy
  int32_t stall;                 // (test) no copy is made, so that the waits run out
};

template <int DQK_, int DV_, int STAGES_, int ROUNDS_>
struct AttendCfg {
  static constexpr int DQK = DQK_, DV = DV_, NW = 8, STAGES = STAGES_, ROUNDS = ROUNDS_;
  static constexpr int kRecord = record_bytes(DQK, DV);
  static constexpr int kQueue = 40;           // resolved slots of a warp
  static constexpr int kMaxRagged = 512;      // rows of a ragged line
  static constexpr int kPart = 16 * DV + 32;  // floats of a partial result: O, m, sum
  static constexpr int kJoin = 16 * DV / ROUNDS + 64;  // floats of a warp in a team's join: O of a round, m, sum
  static constexpr int kWarp = STAGES * (kRecord + 8) + kQueue * 16 + kJoin * 4;
  static constexpr int kSmem = NW * kWarp + (kMaxRagged + 1) * 4;
  static_assert(kSmem <= 232448, "227 KB of shared memory a block");
};

// Ring depth and rounds of the join for each head dim.  A warp holds O and Q of a 16-row tile and a page's scores in up to
// 255 registers, so a block has 8 warps and an SM one block.
template <int DQK, int DV>
struct CfgFor;
template <>
struct CfgFor<64, 64> : AttendCfg<64, 64, 3, 1> {};
template <>
struct CfgFor<128, 64> : AttendCfg<128, 64, 3, 1> {};
template <>
struct CfgFor<128, 128> : AttendCfg<128, 128, 2, 1> {};
template <>
struct CfgFor<192, 128> : AttendCfg<192, 128, 2, 2> {};

// A record's copy into shared memory, by one thread: the barrier's phase ends when all bytes are there.
__device__ __forceinline__ void copy_record(void* dst, const uint8_t* src, int bytes, uint64_t* bar) {
  ptx::mbar_arrive_expect_tx(bar, bytes);
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   ptx::smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(ptx::smem_u32(bar))
               : "memory");
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
__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) { return ptx::ex2(x); }
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
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// sequence_of by a whole warp: 32 places of cu at a time instead of one.
__device__ __forceinline__ int sequence_of_warp(const Batch& b, int row, int lane) {
  if (b.cu == nullptr) return row < b.n_seqs ? row : -1;
  int lo = 0, hi = b.n_seqs;  // the last s with cu[s] <= row, if there is one, is in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + lane * step;
    const unsigned below = __ballot_sync(0xFFFFFFFFu, at < hi && b.cu[at] <= row);
    // (lane 0 counts as below: lo stays a candidate)
    const int last = 31 - __clz(below | 1u);
    lo += last * step;
    hi = min(hi, lo + step);
  }
  return b.n_seqs > 0 && b.cu[lo] <= row && row < b.cu[lo + 1] ? lo : -1;
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
  uint2 w;
  if (a.o_dtype == kF16) {
    w = make_uint2(pack_half(v.x, v.y), pack_half(v.z, v.w));
  } else {
    const __nv_bfloat162 x = __floats2bfloat162_rn(v.x, v.y), y = __floats2bfloat162_rn(v.z, v.w);
    w = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  }
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at * DV + d) = w;
}
__device__ __forceinline__ void store_lse(const AttendArgs& a, int64_t at, float m, float l) {
  if (a.lse != nullptr) a.lse[at] = l != 0.0f ? (m + log2f(l)) * 0.693147180559945309f : -INFINITY;
}

template <class C>
struct Worker {
  static constexpr int DQK = C::DQK, DV = C::DV;
  static constexpr int NT = DV / 8;     // 8-wide output tiles
  static constexpr int KS = DQK / 16;   // k steps of QK

  // ---- the producer's side: rows and slots of the team's share, one after the other
  struct Cursor {
    uint32_t next, end;    // slots of the line still to resolve
    int n, hm, j, len;     // row, KV head and tile in it, next slot, slots of the row
    int seq, first, last;  // first and one-past-last visible key
    int entry;             // lane i: entry i of the row's selection (n_sel <= 32)
    unsigned twice;        // bit i: entry i stands before (a selection is a set)
  };

  // Called for every KV head and tile of a row; what depends on the row alone is worked out at the first.
  static __device__ __forceinline__ void enter_row(const AttendArgs& a, Cursor& c, const uint32_t* starts, bool same_row,
                                                   int lane) {
    const int h = c.hm / a.tiles, g0 = c.hm % a.tiles * 16;
    if (a.sel != nullptr && a.n_sel <= 32)
      c.entry = lane < a.n_sel ? a.sel[((int64_t)c.n * a.hkv + h) * a.n_sel + lane] : -1;
    // the row's queries on their way into L2 (begin() loads them when its turn comes)
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + (int64_t)c.n * a.q_row + (int64_t)(h * a.group + g0) * a.q_head;
    constexpr int kLines = DQK / 64;
    for (int i = lane; i < min(16, a.group - g0) * kLines; i += 32)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(q + i / kLines * a.q_head + i % kLines * 64));
    if (!same_row) {
      c.seq = sequence_of_warp(a.b, c.n, lane);
      const int pos = c.seq < 0 ? -1 : position_of(a.b, c.seq, c.n);
      c.last = keys_up_to(a.b, pos);
      c.first = pos < 0 ? 0 : first_key(pos, a.window);
      c.len = a.slots ? a.slots : starts[c.n + 1] - starts[c.n];
    }
    if (a.sel != nullptr && a.n_sel <= 32)
      c.twice = __ballot_sync(0xFFFFFFFFu, (__match_any_sync(0xFFFFFFFFu, c.entry) & ((1u << lane) - 1)) != 0);
  }

  // This warp's part (every team-th) of the next 32 * team slots of the row into the queue, those that show no key left out
  // but for the warp's last entry of the row's slots here (its owners have to leave the row's result; one without a slot
  // of its own gets an empty entry).  An entry: the record's address (0: none), the first and one past the last visible key
  // of the sub-block (8 bits each), and the row (times 2, + 1 if it is the warp's last entry of it).
  static __device__ __forceinline__ int resolve(const AttendArgs& a, Cursor& c, const uint32_t* starts, int4* queue, int tail,
                                                int team, int turn, int lane) {
    const int rows_h = a.hkv * a.tiles;
    const int count = min((uint32_t)(32 * team), min((uint32_t)(c.len - c.j), c.end - c.next));
    const int own = (count - turn + team - 1) / team;  // (0 where count <= turn)
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
      if (sub >= 0)
        for (int i = 0; i < at; ++i)
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
      const bool same_row = ++c.hm < rows_h;
      if (!same_row) c.hm = 0, ++c.n;
      enter_row(a, c, starts, same_row, lane);
    }
    return tail + __popc(kept);
  }

  static __device__ __forceinline__ const uint8_t* record_of(const int4& e) {
    return reinterpret_cast<const uint8_t*>((uint64_t)(uint32_t)e.y << 32 | (uint32_t)e.x);
  }
  // ---- the consumer's side
  float o[NT][4];
  uint32_t q0[KS * 2], q1[KS * 2];  // Q of rows r and r + 8: d = c * DQK / 4 + 2i, + 1
  float f0, f1, m0, m1;
  float2 l0, l1;  // each thread's share of the sums

  // A new row: its queries are asked for, then (when the copies of the first pages are under way) made ready.
  __device__ __forceinline__ void ask(const AttendArgs& a, uint32_t row, int lane) {
    const int rows_h = a.hkv * a.tiles, r = lane >> 2, c = lane & 3;
    const int n = row / rows_h, hm = row % rows_h, h = hm / a.tiles, g = hm % a.tiles * 16 + r;
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + (int64_t)n * a.q_row + (int64_t)(h * a.group + g) * a.q_head +
                          c * (DQK / 4);
    load_q(q0, g < a.group ? src : nullptr);
    load_q(q1, g + 8 < a.group ? src + 8 * a.q_head : nullptr);
  }
  __device__ __forceinline__ void begin(const AttendArgs& a) {
    scale_q(q0, a.q_half, f0);
    scale_q(q1, a.q_half, f1);
    // (finite and not 0, so that -inf stays -inf)
    f0 = fminf(fmaxf(f0 * a.scale_log2, 1e-38f), 3e38f), f1 = fminf(fmaxf(f1 * a.scale_log2, 1e-38f), 3e38f);
    m0 = m1 = -INFINITY;
    l0 = l1 = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  }

  // One page: keys [lo, lim) of its 64 are visible.
  __device__ __forceinline__ void page(uint8_t* rec, int lim, int lo, int lane) {
    const int r = lane >> 2, c = lane & 3;
    const bool whole = lim >= kPage && lo <= 0;
    const int odd = 4 + (c ^ 1);                              // keys of this thread's columns in a tile of 8: c and odd
    const int row = r & 1 ? 4 + (r >> 1 ^ 1) : r >> 1;        // key of K's fragment
    const uint8_t* krec = rec + row * (DQK / 2) + c * (DQK / 8);
    const uint8_t* kscales = rec + k_scale_at(DQK) + row * (DQK / kGroup) + c * (DQK / 64);
    float s[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
      const uint8_t* codes = krec + 8 * i * (DQK / 2);
      const uint8_t* scales = kscales + 8 * i * (DQK / kGroup);
      uint32_t w[DQK / 32];
      uint32_t sc[DQK / 64];
      if constexpr (DQK == 128) {
        const uint4 x = *reinterpret_cast<const uint4*>(codes);
        w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
        const uint32_t both = *reinterpret_cast<const uint16_t*>(scales);
        sc[0] = scale2(both & 0xFFu), sc[1] = scale2(both >> 8);
      } else {
#pragma unroll
        for (int g = 0; g < DQK / 64; ++g) {
          const uint2 x = *reinterpret_cast<const uint2*>(codes + 8 * g);
          w[2 * g] = x.x, w[2 * g + 1] = x.y;
          sc[g] = scale2(scales[g]);
        }
      }
#pragma unroll
      for (int j = 0; j < DQK / 32; ++j) {
        const uint32_t z = sc[j / 2];
        const uint32_t b0 = mul2(decode_byte<0>(w[j]), z), b1 = mul2(decode_byte<1>(w[j]), z);
        const uint32_t b2 = mul2(decode_byte<2>(w[j]), z), b3 = mul2(decode_byte<3>(w[j]), z);
        mma(s[i], q0[4 * j], q1[4 * j], q0[4 * j + 1], q1[4 * j + 1], b0, b1);
        mma(s[i], q0[4 * j + 2], q1[4 * j + 2], q0[4 * j + 3], q1[4 * j + 3], b2, b3);
      }
    }
    // score i, element e is key 8 i + (c or odd, by e % 2) of row r + 8 (e / 2)
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = 8 * i + (e ? odd : c);
          if (key < lo || key >= lim) s[i][e] = s[i][e + 2] = -INFINITY;
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
    // softmax: the maximum m of the unscaled scores, f > 0 turns them into powers of two
    float t0 = m0, t1 = m1;
#pragma unroll
    for (int i = 0; i < 8; ++i) t0 = max3(t0, s[i][0], s[i][1]), t1 = max3(t1, s[i][2], s[i][3]);
    t0 = fmaxf(t0, __shfl_xor_sync(0xFFFFFFFFu, t0, 1)), t1 = fmaxf(t1, __shfl_xor_sync(0xFFFFFFFFu, t1, 1));
    t0 = fmaxf(t0, __shfl_xor_sync(0xFFFFFFFFu, t0, 2)), t1 = fmaxf(t1, __shfl_xor_sync(0xFFFFFFFFu, t1, 2));
    const float u0 = t0 == -INFINITY ? 0.0f : t0 * f0, u1 = t1 == -INFINITY ? 0.0f : t1 * f1;
    if (__any_sync(0xFFFFFFFFu, t0 > m0 || t1 > m1)) {
      const float a0 = exp2_fast(m0 * f0 - u0), a1 = exp2_fast(m1 * f1 - u1);
      l0.x *= a0, l0.y *= a0, l1.x *= a1, l1.y *= a1;
#pragma unroll
      for (int i = 0; i < NT; ++i) o[i][0] *= a0, o[i][1] *= a0, o[i][2] *= a1, o[i][3] *= a1;
      m0 = t0, m1 = t1;
    }
    uint32_t p[8][2];  // fp16: rows r and r + 8
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float2 x = fma2(make_float2(s[i][0], s[i][1]), make_float2(f0, f0), make_float2(-u0, -u0));
      float2 y = fma2(make_float2(s[i][2], s[i][3]), make_float2(f1, f1), make_float2(-u1, -u1));
      x = make_float2(exp2_fast(x.x), exp2_fast(x.y)), y = make_float2(exp2_fast(y.x), exp2_fast(y.y));
      l0 = add2(l0, x), l1 = add2(l1, y);
      p[i][0] = pack_half(x.x, x.y), p[i][1] = pack_half(y.x, y.y);
    }
    // PV; output tile j, element e is d = (2c + e % 2) * NT + j of row r + 8 (e / 2)
    const uint8_t* vrec = rec + v_code_at(DQK) + r * (DV / 16);
    const uint8_t* vscales = rec + v_scale_at(DQK, DV) + (DV == 128 ? r : r >> 1);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t a0 = p[2 * t][0], a1 = p[2 * t][1], a2 = p[2 * t + 1][0], a3 = p[2 * t + 1][1];
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
        mma(o[8 * j + 0], a0, a1, a2, a3, mul2(decode_byte<0>(x0), z0), mul2(decode_byte<0>(x1), z1));
        mma(o[8 * j + 1], a0, a1, a2, a3, mul2(decode_byte<0>(y0), z0), mul2(decode_byte<0>(y1), z1));
        mma(o[8 * j + 2], a0, a1, a2, a3, mul2(decode_byte<1>(x0), z0), mul2(decode_byte<1>(x1), z1));
        mma(o[8 * j + 3], a0, a1, a2, a3, mul2(decode_byte<1>(y0), z0), mul2(decode_byte<1>(y1), z1));
        mma(o[8 * j + 4], a0, a1, a2, a3, mul2(decode_byte<2>(x0), z0), mul2(decode_byte<2>(x1), z1));
        mma(o[8 * j + 5], a0, a1, a2, a3, mul2(decode_byte<2>(y0), z0), mul2(decode_byte<2>(y1), z1));
        mma(o[8 * j + 6], a0, a1, a2, a3, mul2(decode_byte<3>(x0), z0), mul2(decode_byte<3>(x1), z1));
        mma(o[8 * j + 7], a0, a1, a2, a3, mul2(decode_byte<3>(y0), z0), mul2(decode_byte<3>(y1), z1));
      }
    }
  }

  // The row's result: whole, or this team's part of it (`part` not null).  `join`: the team's warps' join buffers.
  __device__ __forceinline__ void finish(const AttendArgs& a, uint32_t row, float* part, float* join, int team, int turn,
                                         int barrier, int lane) {
    const int rows_h = a.hkv * a.tiles, r = lane >> 2, c = lane & 3;
    float n0 = l0.x + l0.y, n1 = l1.x + l1.y;
    n0 += __shfl_xor_sync(0xFFFFFFFFu, n0, 1), n1 += __shfl_xor_sync(0xFFFFFFFFu, n1, 1);
    n0 += __shfl_xor_sync(0xFFFFFFFFu, n0, 2), n1 += __shfl_xor_sync(0xFFFFFFFFu, n1, 2);
    float e0 = m0 == -INFINITY ? m0 : m0 * f0, e1 = m1 == -INFINITY ? m1 : m1 * f1;  // as powers of two
    const int n = row / rows_h, hm = row % rows_h, g0 = hm % a.tiles * 16;
    const int64_t at0 = (int64_t)n * a.hq + hm / a.tiles * a.group + g0;  // the tile's first query head
    const int used = min(16, a.group - g0);
    const bool left = part == nullptr && !a.fill && sequence_of_warp(a.b, n, lane) < 0;  // a row to leave as it was
    if (team == 1) {
      if (part != nullptr) {
        if (c == 0) {
          part[16 * DV + r] = e0, part[16 * DV + r + 8] = e1;
          part[16 * DV + 16 + r] = n0, part[16 * DV + 16 + r + 8] = n1;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float4* to = reinterpret_cast<float4*>(part + (r + 8 * (e / 2)) * DV + (2 * c + e % 2) * NT);
#pragma unroll
          for (int j = 0; j < NT / 4; ++j) to[j] = make_float4(o[4 * j][e], o[4 * j + 1][e], o[4 * j + 2][e], o[4 * j + 3][e]);
        }
        return;
      }
      if (left) return;
      const float w = a.weight ? *a.weight : 1.0f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (r + 8 * half >= used) continue;
        const float l = half ? n1 : n0, k = l != 0.0f ? w / l : 0.0f;
        const int64_t at = at0 + r + 8 * half;
        if (c == 0) store_lse(a, at, half ? e1 : e0, l);
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int j = 0; j < NT / 4; ++j)
            store4<DV>(a, at, (2 * c + e) * NT + 4 * j,
                       make_float4(o[4 * j][2 * half + e], o[4 * j + 1][2 * half + e], o[4 * j + 2][2 * half + e],
                                   o[4 * j + 3][2 * half + e]), k);
      }
      return;
    }
    // Join: maxima, then every warp's O against the common maximum, some columns a round.  The 16-byte pieces of a row
    // are exchanged so that neither side meets bank conflicts.
    constexpr int NTR = NT / C::ROUNDS, CS = NTR / 4, kMl = 16 * DV / C::ROUNDS;
    float* mine = join + turn * C::kJoin;
    if (c == 0) mine[kMl + r] = e0, mine[kMl + r + 8] = e1;
    named_barrier(barrier, team * 32);
    float t0 = -INFINITY, t1 = -INFINITY;
    for (int w = 0; w < team; ++w)
      t0 = fmaxf(t0, join[w * C::kJoin + kMl + r]), t1 = fmaxf(t1, join[w * C::kJoin + kMl + r + 8]);
    e0 = exp2_fast(e0 - (t0 == -INFINITY ? 0.0f : t0)), e1 = exp2_fast(e1 - (t1 == -INFINITY ? 0.0f : t1));
    if (c == 0) mine[kMl + 16 + r] = n0 * e0, mine[kMl + 16 + r + 8] = n1 * e1, mine[kMl + 32 + r] = t0, mine[kMl + 40 + r] = t1;
    const float weight = a.weight && part == nullptr ? *a.weight : 1.0f;
#pragma unroll
    for (int q = 0; q < C::ROUNDS; ++q) {
      if (q > 0) named_barrier(barrier, team * 32);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float k = e < 2 ? e0 : e1;
        float4* to = reinterpret_cast<float4*>(mine) + (r + 8 * (e / 2)) * (8 * CS);
#pragma unroll
        for (int j = 0; j < CS; ++j) {
          const int t = q * NTR + 4 * j;
          to[((2 * c + e % 2) * CS + j) ^ (((r & 1) << 2) + c)] =
              make_float4(o[t][e] * k, o[t + 1][e] * k, o[t + 2][e] * k, o[t + 3][e] * k);
        }
      }
      named_barrier(barrier, team * 32);
      for (int i = turn * 32 + lane; i < 16 * 8 * CS; i += team * 32) {
        const int x = i / (8 * CS), k = i % (8 * CS), d = k / CS * NT + q * NTR + k % CS * 4;
        if (x >= used || left) continue;
        const int place = x * (8 * CS) + (k ^ (((x & 1) << 2) + k / (2 * CS)));
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float l = 0.0f;
        for (int w = 0; w < team; ++w) {
          const float* from = join + w * C::kJoin;
          const float4 y = reinterpret_cast<const float4*>(from)[place];
          v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
          l += from[kMl + 16 + x];
        }
        const float m = mine[kMl + 32 + x];
        if (part != nullptr) {
          *reinterpret_cast<float4*>(part + x * DV + d) = v;
          if (k == 0 && q == 0) part[16 * DV + x] = m, part[16 * DV + 16 + x] = l;
        } else {
          store4<DV>(a, at0 + x, d, v, l != 0.0f ? weight / l : 0.0f);
          if (k == 0 && q == 0) store_lse(a, at0 + x, m, l);
        }
      }
    }
  }
};

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
  const uint32_t rows_h = a.hkv * a.tiles, rows = a.b.n_rows * rows_h;
  uint32_t total = rows * a.slots;
  Split split = a.split;
  if (a.slots == 0) {  // the ragged line: every block counts the slots before each row (n_rows <= kMaxRagged)
    for (int n = threadIdx.x; n < a.b.n_rows; n += C::NW * 32) {
      const int seq = sequence_of(a.b, n), pos = seq < 0 ? -1 : position_of(a.b, seq, n);
      starts[n + 1] = running_slots(pos < 0 ? 0 : first_key(pos, a.window), keys_up_to(a.b, pos));
    }
    __syncthreads();
    if (warp == 0) {
      uint32_t sum = 0, longest = 0;
      if (lane == 0) starts[0] = 0;
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
      for (int n = threadIdx.x; n <= a.b.n_rows; n += C::NW * 32) a.starts[n] = starts[n];
      if (threadIdx.x == 0) a.starts[a.b.n_rows + 1] = split.cut ? split.share : 0;
    }
  }
  // neighbouring teams are on different SMs, so that a few of them use many
  const int team = split.team, turn = warp % team, sub_team = warp / team;
  const uint32_t me = sub_team * gridDim.x + blockIdx.x;

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
  Worker<C>::enter_row(a, cur, starts, false, lane);

  if (lane < C::STAGES) ptx::mbar_init(bars + lane, 1);
  ptx::fence_mbar_init();
  __syncwarp();
  Worker<C> w;
  w.ask(a, row, lane);
  int head = 0, tail = 0, issued = 0;
  uint32_t phases = 0, flying = 0;  // each stage's parity of the next phase; copies on their way
  bool lost = false;                // a copy did not come: rows from here on are NaN
  auto issue = [&] {
    while (tail - issued < C::STAGES && tail - head <= C::kQueue - 32 && cur.next < cur.end)
      tail = Worker<C>::resolve(a, cur, starts, queue, tail, team, turn, lane);
    if (issued < tail) {
      const uint8_t* src = Worker<C>::record_of(queue[issued % C::kQueue]);
      const int stage = issued++ % C::STAGES;
      if (src != nullptr && !lost && !a.stall) {
        if (lane == 0) copy_record(ring + stage * C::kRecord, src, C::kRecord, bars + stage);
        flying |= 1u << stage;
      }
    }
  };
  // the ring holds STAGES records: STAGES - 1 on their way while one is worked on
  for (int i = 0; i < C::STAGES - 1; ++i) issue();
  w.begin(a);
  bool fresh = false, first_row = true;
  while (head < issued) {
    issue();
    const int4 e = queue[head % C::kQueue];
    const int stage = head % C::STAGES;
    if (fresh) {
      w.ask(a, (uint32_t)e.w >> 1, lane);
      w.begin(a);
    }
    fresh = e.w & 1;
    if (Worker<C>::record_of(e) != nullptr) {
      lost = lost || !__all_sync(0xFFFFFFFFu, wait_for(bars + stage, phases >> stage & 1, a.wait_ns));
      if (!lost) {
        phases ^= 1u << stage, flying &= ~(1u << stage);
        w.page(ring + stage * C::kRecord, e.z >> 8, e.z & 255, lane);
      } else {
        w.l0.x = w.l1.x = __int_as_float(0x7FFFFFFF);
      }
    }
    if (fresh) {
      // a row is whole here unless it began before this share, or goes on behind it
      const bool head_cut = first_row && cut_before;
      const bool tail_cut = head + 1 == tail && cur.next == cur.end && cur.j < cur.len;
      float* part = head_cut || tail_cut ? a.part + ((size_t)me * 2 + (head_cut ? 0 : 1)) * C::kPart : nullptr;
      w.finish(a, (uint32_t)e.w >> 1, part, join + sub_team * team * C::kJoin, team, turn, 1 + sub_team, lane);
      first_row = false;
    }
    __syncwarp();
    ++head;
  }
  if (lost) {  // the block's memory is not given up under a copy (bounded, too)
    if (a.err != nullptr && lane == 0) atomicOr(a.err, 1);
    for (int i = 0; i < C::STAGES; ++i)
      if (flying >> i & 1) wait_for(bars + i, phases >> i & 1, a.wait_ns);
  }
}

// Joins the parts of the rows that were cut, in the order of the line.  WPH warps share a row's query head:
// 1 where a row has a few parts, 8 where one row is cut over hundreds of workers.
template <class C, int WPH>
__global__ void __launch_bounds__(256) merge_kernel(const AttendArgs a) {
  constexpr int DV = C::DV, V4 = DV / 4;
  __shared__ float shared_o[8][DV];
  __shared__ float shared_ml[8][2];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rows_h = a.hkv * a.tiles;
  const int64_t unit = WPH == 1 ? (int64_t)blockIdx.x * 8 + warp : blockIdx.x;  // (row, query head)
  if (unit >= (int64_t)a.b.n_rows * a.hq) return;
  const int n = unit / a.hq, hq = unit % a.hq, h = hq / a.group, g = hq % a.group;
  const uint32_t hm = h * a.tiles + g / 16;
  uint32_t start, len, per = a.split.share;
  if (a.slots) {
    len = a.slots, start = ((uint32_t)n * rows_h + hm) * len;
  } else {
    const uint32_t s0 = a.starts[n];
    len = a.starts[n + 1] - s0, start = s0 * rows_h + hm * len;
    per = a.starts[a.b.n_rows + 1];
  }
  if (per == 0) return;
  const uint32_t w0 = start / per, w1 = (start + len - 1) / per;
  if (w0 == w1) return;  // the row was not cut
  if (!a.fill && sequence_of(a.b, n) < 0) return;
  // the first team has the row as its last, the others as their first
  auto part_of = [&](uint32_t w) { return a.part + ((size_t)w * 2 + (w == w0 ? 1 : 0)) * C::kPart; };
  const int mine = WPH == 1 ? 0 : warp;
  float m = -INFINITY;
  for (uint32_t w = w0 + mine * 32 + lane; w <= w1; w += 32 * WPH) m = fmaxf(m, part_of(w)[16 * DV + g % 16]);
#pragma unroll
  for (int k = 16; k > 0; k /= 2) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, k));
  const float u = m == -INFINITY ? 0.0f : m;  // (of this warp's parts)
  float l = 0.0f;
  float4 acc[(V4 + 31) / 32];
#pragma unroll
  for (int i = 0; i < (V4 + 31) / 32; ++i) acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (uint32_t w = w0 + mine * 32; w <= w1; w += 32 * WPH)
#pragma unroll 4
    for (uint32_t x = w; x < min(w + 32, w1 + 1); ++x) {
      const float* p = part_of(x);
      const float f = exp2_fast(p[16 * DV + g % 16] - u);
      l += p[16 * DV + 16 + g % 16] * f;
#pragma unroll
      for (int i = 0; i < (V4 + 31) / 32; ++i)
        if (lane + 32 * i < V4) {
          const float4 v = reinterpret_cast<const float4*>(p + g % 16 * DV)[lane + 32 * i];
          acc[i].x += v.x * f, acc[i].y += v.y * f, acc[i].z += v.z * f, acc[i].w += v.w * f;
        }
    }
  float top = m;
  if (WPH > 1) {
#pragma unroll
    for (int i = 0; i < (V4 + 31) / 32; ++i)
      if (lane + 32 * i < V4) reinterpret_cast<float4*>(shared_o[warp])[lane + 32 * i] = acc[i];
    if (lane == 0) shared_ml[warp][0] = m, shared_ml[warp][1] = l;
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int k = 0; k < WPH; ++k) top = fmaxf(top, shared_ml[k][0]);
    const float v = top == -INFINITY ? 0.0f : top;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < (V4 + 31) / 32; ++i) acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < WPH; ++k) {
      // (a maximum is never NaN: fmaxf leaves NaN out; where it is -inf the sums are zeros, or NaN, which stays)
      const float mk = shared_ml[k][0], f = mk == -INFINITY ? 1.0f : exp2_fast(mk - v);
      l += shared_ml[k][1] * f;
#pragma unroll
      for (int i = 0; i < (V4 + 31) / 32; ++i)
        if (lane + 32 * i < V4) {
          const float4 x = reinterpret_cast<const float4*>(shared_o[k])[lane + 32 * i];
          acc[i].x += x.x * f, acc[i].y += x.y * f, acc[i].z += x.z * f, acc[i].w += x.w * f;
        }
    }
  }
  const float k = l != 0.0f ? (a.weight ? *a.weight : 1.0f) / l : 0.0f;
  if (lane == 0) store_lse(a, unit, top, l);
#pragma unroll
  for (int i = 0; i < (V4 + 31) / 32; ++i)
    if (lane + 32 * i < V4) store4<DV>(a, unit, 4 * (lane + 32 * i), acc[i], k);
}

}  // namespace cache
}  // namespace nsa
