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
//   * the key axis is permuted (key 16t + c + 4i is k index 2c, 2c+1, 2c+8, 2c+9 for i = 0..3) so that a thread's V
//     fragments are d_v / 8 consecutive codes of four keys, which are interleaved two and two; P needs no
//     exchange, its score registers are the A fragment.
// Q has up to 8 (bf16) or 11 significant bits, so a power of two per row puts it into fp16 (below 2^-14 of the row's
// largest to within 2^-25 of it).  P is rounded to fp16 (at most 2^-11 of each term): the sum of
// its fp32 values is the divisor.  Scores, statistics and O are fp32.
//
// All (row, page) slots of the call stand in one line that is cut evenly among the workers; a row that is cut
// leaves partial (m, sum, O) in the workspace, and merge_kernel joins them in the order of the line: results do not
// depend on timing.
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
  float* part;                   // partial results, 2 per worker
  uint32_t* starts;              // slots before every row's, n_rows + 1 (ragged line only; the first block writes them)
  int32_t hq, hkv, group, tiles; // tiles: 16-row tiles of a KV head's G query heads
  int32_t n_sel, per, window;    // per: sub-blocks of a selection block
  int32_t slots;                 // slots of every row; 0: as many as it has sub-blocks (the ragged line)
  uint32_t workers, share;       // share: slots of a worker (0: from the line's length, on the device)
  int32_t q_half, o_dtype, accumulate, fill;  // fill: rows of no sequence get O = 0, LSE = -inf; else they are left
  float scale_log2;
};

template <int DQK_, int DV_, int NW_, int STAGES_, int CTAS_>
struct AttendCfg {
  static constexpr int DQK = DQK_, DV = DV_, NW = NW_, STAGES = STAGES_, CTAS = CTAS_;
  static constexpr int kRecord = record_bytes(DQK, DV);
  static constexpr int kQueue = 64;        // resolved slots of a warp
  static constexpr int kMaxRagged = 512;   // rows of a ragged line
  static constexpr int kPart = 16 * DV + 32;  // floats of a partial result: O, m, sum
  static constexpr int kSmem = NW * (STAGES * kRecord + kQueue * 16) + (kMaxRagged + 1) * 4;
};

// Warps of a block, ring depth and blocks of an SM for each head dim: what fits 227 KB of shared memory and the
// registers (a warp holds O and Q of a 16-row tile).
template <int DQK, int DV>
struct CfgFor;
template <>
struct CfgFor<64, 64> : AttendCfg<64, 64, 8, 3, 1> {};
template <>
struct CfgFor<128, 64> : AttendCfg<128, 64, 8, 4, 1> {};
template <>
struct CfgFor<128, 128> : AttendCfg<128, 128, 8, 3, 1> {};
template <>
struct CfgFor<192, 128> : AttendCfg<192, 128, 6, 3, 1> {};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
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

template <int N>
__device__ __forceinline__ void load_q(uint32_t (&q)[N], const uint16_t* src, bool half, float& factor) {
  // N fp16 pairs of consecutive d of one row; `factor` undoes the row's power of two
  uint32_t raw[N];
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    const uint4 x = src ? reinterpret_cast<const uint4*>(src)[i] : make_uint4(0, 0, 0, 0);
    raw[4 * i] = x.x, raw[4 * i + 1] = x.y, raw[4 * i + 2] = x.z, raw[4 * i + 3] = x.w;
  }
  float2 f[N];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    f[i] = half ? __half22float2(*reinterpret_cast<__half2*>(&raw[i]))
                : make_float2(__uint_as_float(raw[i] << 16), __uint_as_float(raw[i] & 0xFFFF0000u));
    top = max(top, max(__float_as_uint(f[i].x) & 0x7FFFFFFFu, __float_as_uint(f[i].y) & 0x7FFFFFFFu));
  }
  top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
  top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
  // exponent of the row's largest; rows of zeros or subnormals, infinities and NaN stay as they are
  const int e = (int)(top >> 23);
  const bool scaled = e > 1 && e < 254;
  const float down = scaled ? __uint_as_float((uint32_t)(254 - e) << 23) : 1.0f;
  factor = scaled ? __uint_as_float((uint32_t)e << 23) : 1.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) q[i] = pack_half(f[i].x * down, f[i].y * down);
}

template <class C>
struct Worker {
  static constexpr int DQK = C::DQK, DV = C::DV;
  static constexpr int NT = DV / 8;     // 8-wide output tiles
  static constexpr int KS = DQK / 16;   // k steps of QK

  // ---- the producer's side: rows and slots of the worker's share, one after the other
  struct Cursor {
    uint32_t next, end;  // slots of the line still to resolve
    int n, hm, j, len;   // row, KV head and tile in it, next slot, slots of the row
    int seq, first, last;  // first and one-past-last visible key
  };

  static __device__ __forceinline__ void enter_row(const AttendArgs& a, Cursor& c, const uint32_t* starts, int lane) {
    c.seq = sequence_of_warp(a.b, c.n, lane);
    const int pos = c.seq < 0 ? -1 : position_of(a.b, c.seq, c.n);
    c.last = keys_up_to(a.b, pos);
    c.first = pos < 0 ? 0 : first_key(pos, a.window);
    c.len = a.slots ? a.slots : starts[c.n + 1] - starts[c.n];
  }

  // Up to 32 more slots into the queue, those that show no key left out but for the last of a row's slots here (its
  // owner has to leave the row's result).  An entry: page (-1: none), one past the last and the first visible key of
  // the sub-block, and the row (times 2, + 1 if it is its last entry here).
  static __device__ __forceinline__ int resolve(const AttendArgs& a, Cursor& c, const uint32_t* starts, int4* queue, int tail,
                                                int lane) {
    const int rows_h = a.hkv * a.tiles;
    const int count = min(32u, min((uint32_t)(c.len - c.j), c.end - c.next));
    const int j = c.j + lane;
    int sub = -1;
    if (lane < count) {
      if (a.sel != nullptr) {
        const int32_t* row = a.sel + ((int64_t)c.n * a.hkv + c.hm / a.tiles) * a.n_sel;
        const int at = j / a.per, entry = row[at];
        sub = selected_sub(entry, j - at * a.per, a.per, c.first, c.last);
        if (sub >= 0)
          for (int i = 0; i < at; ++i)
            if (row[i] == entry) sub = -1;  // a selection is a set
      } else {
        sub = running_sub(j, c.first, c.last);
      }
    }
    const int page = sub < 0 || c.seq < 0 ? -1 : page_of(a.b, c.seq, sub);
    const bool final = lane == count - 1 && (c.j + count == c.len || c.next + count == c.end);
    const bool keep = lane < count && (page >= 0 || final);
    const unsigned kept = __ballot_sync(0xFFFFFFFFu, keep);
    if (keep) {
      const int base = sub * kPage;
      queue[(tail + __popc(kept & ((1u << lane) - 1))) % C::kQueue] =
          make_int4(page, page < 0 ? 0 : min(kPage, c.last - base), page < 0 ? 0 : max(0, c.first - base),
                    (c.n * rows_h + c.hm) * 2 + final);
    }
    __syncwarp();
    c.next += count;
    c.j += count;
    if (c.j == c.len && c.next < c.end) {  // the next row
      c.j = 0;
      if (++c.hm == rows_h) {
        c.hm = 0, ++c.n;
        enter_row(a, c, starts, lane);
      }
    }
    return tail + __popc(kept);
  }

  static __device__ __forceinline__ void copy_record(const AttendArgs& a, const int4& e, uint32_t dst, int lane) {
    if (e.x < 0) return;
    const int h = (e.w >> 1) % (a.hkv * a.tiles) / a.tiles;
    const uint8_t* src = a.cache + (int64_t)e.x * a.page_stride + (int64_t)h * C::kRecord;
    constexpr int KC = DQK / 32, VC = DV / 32;  // 16-byte pieces of a token's codes
#pragma unroll
    for (int i = 0; i < 2 * KC; ++i) {  // K codes; in every 8 tokens, token u stands at place 2 (u % 4) + u / 4
      const int x = lane + 32 * i, row = x / KC, piece = x - row * KC;
      const int place = (row & ~7) | ((row & 3) << 1) | ((row >> 2) & 1);
      cp_async16(dst + place * (DQK / 2) + piece * 16, src + x * 16);
    }
#pragma unroll
    for (int i = 0; i < (DQK / 4 + 31) / 32; ++i)
      if (lane + 32 * i < DQK / 4) cp_async16(dst + k_scale_at(DQK) + (lane + 32 * i) * 16, src + k_scale_at(DQK) + (lane + 32 * i) * 16);
#pragma unroll
    for (int i = 0; i < 2 * VC; ++i) {  // V codes; with 64-byte rows every other pair of tokens has its halves exchanged
      const int x = lane + 32 * i, row = x / VC, piece = x - row * VC;
      const int place = DV == 128 ? piece ^ (((row >> 1) & 1) << 1) : piece;
      cp_async16(dst + v_code_at(DQK) + row * (DV / 2) + place * 16, src + v_code_at(DQK) + x * 16);
    }
#pragma unroll
    for (int i = 0; i < (DV / 4 + 31) / 32; ++i)
      if (lane + 32 * i < DV / 4)
        cp_async16(dst + v_scale_at(DQK, DV) + (lane + 32 * i) * 16, src + v_scale_at(DQK, DV) + (lane + 32 * i) * 16);
  }

  // ---- the consumer's side
  float o[NT][4];
  uint32_t q0[KS * 2], q1[KS * 2];  // Q of rows r and r + 8: d = c * DQK / 4 + 2i, + 1
  float f0, f1, m0, m1, l0, l1;

  __device__ __forceinline__ void begin(const AttendArgs& a, uint32_t row, int lane) {
    const int rows_h = a.hkv * a.tiles, r = lane >> 2, c = lane & 3;
    const int n = row / rows_h, hm = row % rows_h, h = hm / a.tiles, g = hm % a.tiles * 16 + r;
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + (int64_t)n * a.q_row + (int64_t)(h * a.group + g) * a.q_head +
                          c * (DQK / 4);
    load_q(q0, g < a.group ? src : nullptr, a.q_half, f0);
    load_q(q1, g + 8 < a.group ? src + 8 * a.q_head : nullptr, a.q_half, f1);
    f0 *= a.scale_log2, f1 *= a.scale_log2;
    m0 = m1 = -INFINITY;
    l0 = l1 = 0.0f;
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  }

  // One page: keys [lo, lim) of its 64 are visible.
  __device__ __forceinline__ void page(const uint8_t* rec, int lim, int lo, int lane) {
    const int r = lane >> 2, c = lane & 3;
    const bool whole = lim >= kPage && lo <= 0;
    float s[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
      const uint8_t* codes = rec + (8 * i + r) * (DQK / 2) + c * (DQK / 8);
      const uint8_t* scales = rec + k_scale_at(DQK) + (8 * i + (r >> 1) + 4 * (r & 1)) * (DQK / kGroup) + c * (DQK / 64);
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
    // softmax; score i, element e is key 16 (i / 2) + 8 (i % 2) + c + 4 (e % 2) of row r + 8 (e / 2)
    float t0 = m0, t1 = m1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        s[i][e] *= f0, s[i][e + 2] *= f1;
        if (!whole) {
          const int key = 8 * i + c + 4 * e;
          if (key < lo || key >= lim) s[i][e] = s[i][e + 2] = -INFINITY;
        }
        t0 = fmaxf(t0, s[i][e]), t1 = fmaxf(t1, s[i][e + 2]);
      }
    }
    t0 = fmaxf(t0, __shfl_xor_sync(0xFFFFFFFFu, t0, 1)), t1 = fmaxf(t1, __shfl_xor_sync(0xFFFFFFFFu, t1, 1));
    t0 = fmaxf(t0, __shfl_xor_sync(0xFFFFFFFFu, t0, 2)), t1 = fmaxf(t1, __shfl_xor_sync(0xFFFFFFFFu, t1, 2));
    const float u0 = t0 == -INFINITY ? 0.0f : t0, u1 = t1 == -INFINITY ? 0.0f : t1;
    if (__any_sync(0xFFFFFFFFu, t0 > m0 || t1 > m1)) {
      const float a0 = exp2_fast(m0 - u0), a1 = exp2_fast(m1 - u1);
      l0 *= a0, l1 *= a1;
#pragma unroll
      for (int i = 0; i < NT; ++i) o[i][0] *= a0, o[i][1] *= a0, o[i][2] *= a1, o[i][3] *= a1;
      m0 = t0, m1 = t1;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[i][0] = exp2_fast(s[i][0] - u0), s[i][1] = exp2_fast(s[i][1] - u0);
      s[i][2] = exp2_fast(s[i][2] - u1), s[i][3] = exp2_fast(s[i][3] - u1);
      l0 += s[i][0] + s[i][1], l1 += s[i][2] + s[i][3];
    }
    // PV; output tile j, element e is d = (2c + e % 2) * NT + j of row r + 8 (e / 2)
    const uint8_t* vcodes = rec + v_code_at(DQK) + c * (DV / 2) + (DV == 128 ? (r * 8) ^ (((c >> 1) & 1) << 5) : r * 4);
    const uint8_t* vscales = rec + v_scale_at(DQK, DV) + c * (DV / kGroup) + (DV == 128 ? r : r >> 1);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t a0 = pack_half(s[2 * t][0], s[2 * t][1]), a1 = pack_half(s[2 * t][2], s[2 * t][3]);
      const uint32_t a2 = pack_half(s[2 * t + 1][0], s[2 * t + 1][1]), a3 = pack_half(s[2 * t + 1][2], s[2 * t + 1][3]);
      uint32_t w[4][DV / 64], z[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* at = vcodes + (16 * t + 4 * i) * (DV / 2);
        if constexpr (DV == 128) {
          const uint2 x = *reinterpret_cast<const uint2*>(at);
          w[i][0] = x.x, w[i][1] = x.y;
        } else {
          w[i][0] = *reinterpret_cast<const uint32_t*>(at);
        }
        z[i] = vscales[(16 * t + 4 * i) * (DV / kGroup)];
        if (!whole) {  // what stands behind the visible keys may be anything: 0 times a code is 0
          const int key = 16 * t + 4 * i + c;
          if (key < lo || key >= lim) z[i] = 0;
        }
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

  // The row's result: whole, or this worker's part of it (`part` not null).
  __device__ __forceinline__ void finish(const AttendArgs& a, uint32_t row, float* part, int lane) {
    const int rows_h = a.hkv * a.tiles, r = lane >> 2, c = lane & 3;
    l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, 1), l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, 1);
    l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, 2), l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, 2);
    if (part != nullptr) {
      if (c == 0) {
        part[16 * DV + r] = m0, part[16 * DV + r + 8] = m1;
        part[16 * DV + 16 + r] = l0, part[16 * DV + 16 + r + 8] = l1;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float4* to = reinterpret_cast<float4*>(part + (r + 8 * (e / 2)) * DV + (2 * c + e % 2) * NT);
#pragma unroll
        for (int j = 0; j < NT / 4; ++j) to[j] = make_float4(o[4 * j][e], o[4 * j + 1][e], o[4 * j + 2][e], o[4 * j + 3][e]);
      }
      return;
    }
    const int n = row / rows_h, hm = row % rows_h, h = hm / a.tiles, g = hm % a.tiles * 16 + r;
    if (!a.fill && sequence_of_warp(a.b, n, lane) < 0) return;
    const float w = a.weight ? *a.weight : 1.0f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (g + 8 * half >= a.group) continue;
      const float l = half ? l1 : l0, m = half ? m1 : m0, k = l != 0.0f ? w / l : 0.0f;
      const int64_t at = (int64_t)n * a.hq + h * a.group + g + 8 * half;
      if (a.lse != nullptr && c == 0) a.lse[at] = l != 0.0f ? (m + log2f(l)) * 0.693147180559945309f : -INFINITY;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int64_t to = at * DV + (2 * c + e) * NT;
        if (a.o_dtype == kF32) {
          float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.o) + to);
#pragma unroll
          for (int j = 0; j < NT / 4; ++j) {
            float4 v = a.accumulate ? p[j] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            v.x += o[4 * j][2 * half + e] * k, v.y += o[4 * j + 1][2 * half + e] * k;
            v.z += o[4 * j + 2][2 * half + e] * k, v.w += o[4 * j + 3][2 * half + e] * k;
            p[j] = v;
          }
        } else {
          uint32_t v[NT / 2];
#pragma unroll
          for (int j = 0; j < NT / 2; ++j) {
            const float x = o[2 * j][2 * half + e] * k, y = o[2 * j + 1][2 * half + e] * k;
            if (a.o_dtype == kF16) {
              v[j] = pack_half(x, y);
            } else {
              const __nv_bfloat162 p = __floats2bfloat162_rn(x, y);
              v[j] = *reinterpret_cast<const uint32_t*>(&p);
            }
          }
          uint4* p = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.o) + to);
#pragma unroll
          for (int j = 0; j < NT / 8; ++j) p[j] = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        }
      }
    }
  }
};

template <class C>
__global__ void __launch_bounds__(C::NW * 32, C::CTAS) attend_kernel(const AttendArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  uint8_t* ring = smem + warp * (C::STAGES * C::kRecord);
  int4* queue = reinterpret_cast<int4*>(smem + C::NW * C::STAGES * C::kRecord) + warp * C::kQueue;
  uint32_t* starts = reinterpret_cast<uint32_t*>(smem + C::NW * (C::STAGES * C::kRecord + C::kQueue * 16));
  const uint32_t rows_h = a.hkv * a.tiles;
  uint32_t total = (uint32_t)a.b.n_rows * rows_h * a.slots;
  if (a.slots == 0) {  // the ragged line: every block counts the slots before each row (n_rows <= kMaxRagged)
    for (int n = threadIdx.x; n < a.b.n_rows; n += C::NW * 32) {
      const int seq = sequence_of(a.b, n), pos = seq < 0 ? -1 : position_of(a.b, seq, n);
      starts[n + 1] = running_slots(pos < 0 ? 0 : first_key(pos, a.window), keys_up_to(a.b, pos));
    }
    __syncthreads();
    if (warp == 0) {
      uint32_t sum = 0;
      if (lane == 0) starts[0] = 0;
      for (int n0 = 0; n0 < a.b.n_rows; n0 += 32) {
        uint32_t x = n0 + lane < a.b.n_rows ? starts[n0 + lane + 1] : 0;
#pragma unroll
        for (int k = 1; k < 32; k *= 2) {
          const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, x, k);
          if (lane >= k) x += y;
        }
        if (n0 + lane < a.b.n_rows) starts[n0 + lane + 1] = sum + x;
        sum += __shfl_sync(0xFFFFFFFFu, x, 31);
      }
    }
    __syncthreads();
    if (blockIdx.x == 0 && a.part != nullptr)
      for (int n = threadIdx.x; n <= a.b.n_rows; n += C::NW * 32) a.starts[n] = starts[n];
    total = starts[a.b.n_rows] * rows_h;
  }
  const uint32_t per = a.share ? a.share : share(total, a.workers);
  // neighbouring shares are on different SMs, so that a short line uses many of them
  const uint32_t me = warp * gridDim.x + blockIdx.x;
  if (me >= a.workers || (uint64_t)me * per >= total) return;

  typename Worker<C>::Cursor cur;
  cur.next = me * per;
  cur.end = min(total, cur.next + per);
  uint32_t before;  // the line's slots before the row
  if (a.slots) {
    const uint32_t row = cur.next / a.slots;
    cur.n = row / rows_h, cur.hm = row % rows_h, cur.j = cur.next % a.slots;
    before = row * a.slots;
  } else {
    int lo = 0, hi = a.b.n_rows;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (starts[mid] * rows_h <= cur.next) lo = mid;
      else hi = mid;
    }
    const uint32_t len = starts[lo + 1] - starts[lo], into = cur.next - starts[lo] * rows_h;
    cur.n = lo, cur.hm = into / len, cur.j = into % len;
    before = cur.next - cur.j;
  }
  const bool cut_before = before < cur.next;  // the first row's earlier slots are another worker's
  Worker<C>::enter_row(a, cur, starts, lane);

  Worker<C> w;
  int head = 0, tail = 0, issued = 0;
  bool fresh = true, first_row = true;
  // the ring holds STAGES records: STAGES - 1 in flight while one is worked on; one (maybe empty) copy group each
  auto issue = [&] {
    while (tail - issued < C::STAGES && tail - head <= C::kQueue - 32 && cur.next < cur.end)
      tail = Worker<C>::resolve(a, cur, starts, queue, tail, lane);
    if (issued < tail) {
      const int4 e = queue[issued % C::kQueue];
      Worker<C>::copy_record(a, e, (uint32_t)__cvta_generic_to_shared(ring + (issued % C::STAGES) * C::kRecord), lane);
      ++issued;
    }
    cp_commit();
  };
  for (int i = 0; i < C::STAGES - 1; ++i) issue();
  while (head < issued) {
    const int4 e = queue[head % C::kQueue];
    cp_wait<C::STAGES - 2>();
    __syncwarp();
    const uint32_t row = (uint32_t)e.w >> 1;
    if (fresh) w.begin(a, row, lane);
    fresh = e.w & 1;
    if (e.x >= 0) w.page(ring + (head % C::STAGES) * C::kRecord, e.y, e.z, lane);
    if (fresh) {
      // a row is whole here unless it began before this share, or goes on behind it
      const bool head_cut = first_row && cut_before;
      const bool tail_cut = head + 1 == tail && cur.next == cur.end && cur.j < cur.len;
      float* part = head_cut || tail_cut ? a.part + ((size_t)me * 2 + (head_cut ? 0 : 1)) * C::kPart : nullptr;
      w.finish(a, row, part, lane);
      first_row = false;
    }
    __syncwarp();
    ++head;
    issue();
  }
  cp_wait<0>();
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
  uint32_t start, len, total;
  if (a.slots) {
    len = a.slots, start = ((uint32_t)n * rows_h + hm) * len, total = (uint32_t)a.b.n_rows * rows_h * a.slots;
  } else {
    const uint32_t s0 = a.starts[n];
    len = a.starts[n + 1] - s0, start = s0 * rows_h + hm * len, total = a.starts[a.b.n_rows] * rows_h;
  }
  const uint32_t per = a.share ? a.share : share(total, a.workers);
  const uint32_t w0 = start / per, w1 = (start + len - 1) / per;
  if (w0 == w1) return;  // the row was not cut
  if (!a.fill && sequence_of(a.b, n) < 0) return;
  // the first worker has the row as its last, the others as their first
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
  if (a.lse != nullptr && lane == 0) a.lse[unit] = l != 0.0f ? (top + log2f(l)) * 0.693147180559945309f : -INFINITY;
#pragma unroll
  for (int i = 0; i < (V4 + 31) / 32; ++i) {
    if (lane + 32 * i >= V4) continue;
    float4 v = make_float4(acc[i].x * k, acc[i].y * k, acc[i].z * k, acc[i].w * k);
    const int64_t at = unit * V4 + lane + 32 * i;
    if (a.o_dtype == kF32) {
      float4* p = static_cast<float4*>(a.o) + at;
      if (a.accumulate) {
        const float4 x = *p;
        v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
      }
      *p = v;
    } else if (a.o_dtype == kF16) {
      static_cast<uint2*>(a.o)[at] = make_uint2(pack_half(v.x, v.y), pack_half(v.z, v.w));
    } else {
      const __nv_bfloat162 x = __floats2bfloat162_rn(v.x, v.y), y = __floats2bfloat162_rn(v.z, v.w);
      static_cast<uint2*>(a.o)[at] = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
    }
  }
}

}  // namespace cache
}  // namespace nsa
