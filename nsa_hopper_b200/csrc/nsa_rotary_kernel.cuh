// Rotary positions of one or several axes: pairs of a head's values turned by angles that grow with the token's position.
//
//     (a_i, b_i) -> (a_i cos w_i - b_i sin w_i, b_i cos w_i + a_i sin w_i),   w_i = position[axis(i)] * inv_freq(i)
//
// for the pairs i of the rotary part of a head (values i and i + pairs, or 2 i and 2 i + 1), the rest is copied; the gradient is
// the same with -w.  Angles are kept in turns, as 64-bit fixed point: position * round(inv_freq / 2 pi * 2^64) wraps around
// at whole turns by itself, so far positions cost no bits (an fp32 product would be off by 0.06 radians at a position of a
// million).  Its upper 32 bits give the quadrant and the rest of it, at most an eighth of a turn, whose sine and cosine are
// taken in fp32.  Products and sums are fp32, rounded once to the output's type.
//
// What bounds it: DRAM, 2 bytes in and 2 out a value of 16 bits.  A block has a token with all its heads, Q's and K's in one
// launch: its angles are computed once, in shared memory, where all heads read them; of few heads, which have no work for a block,
// it has several tokens.  Any strides come in and go out, so that [B, T, H, d], as projections write it, becomes the
// [B, H, T, d] that the attention reads on the way.  65536 tokens of 64 + 4 heads of 128 in bf16: 347 us, 6.6 TB/s, the measured
// copy rate.  What brought it there was few registers: with four words a thread in flight and 127 registers it took 574 us,
// with two and 64 430, with one and 32 (8 blocks an SM) 358, and with the outgoing address computed before the words are loaded
// 347.  There tokens together in a block (2, 4, 8, 16) gave nothing, streaming loads took 398, streaming stores 379.
//
// Two forms are far from the copy rate.  Rotary parts that no words of 8 bytes fit are bound by instructions (36 of 128 values in
// bf16, 16384 tokens of 68 heads: 171 us for 88 us of copying, issue slots 75 %; two or four words of an item at once took 163
// and 153 in a kernel whose wide words they made 2 % slower, and have not been built for narrow words alone).  Few heads, several
// tokens a block, are bound by latency (65536 tokens of 2 heads of 128: 28 us for 10): a thread loads a position, makes an
// angle, meets the others, and only then loads the one item that it has.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "nsa_programmatic.cuh"
#include "nsa_rotary_index.h"

namespace nsa {
namespace rotary {

constexpr int kMaxPairs = 128;  // of a head of 256 values
constexpr int kThreads = 256;   // of a block, at most
constexpr int kAngles = 1024;   // of a block of several tokens, at most: they fill 8 KB of shared memory

struct Tensor {
  const void* x;
  void* y;
  int64_t xs[3], ys[3];  // strides of batch, head, token
};
struct Args {
  Tensor t[2];
  const int32_t* pos;
  int64_t ps[3];                 // strides of axis, batch, token
  int32_t heads, first;          // of both tensors together, of the first one
  int32_t batch, tokens;         // tokens of a batch entry
  int32_t offset, pairs, rest;   // first value and pairs of the rotary part; values beside it
  int32_t total;                 // tokens of all batch entries
  int32_t heads_block;           // heads of a block
  int32_t tokens_block;          // tokens of a block
  int32_t interleaved;
  uint32_t flip;                 // sign bit of the sines
  uint64_t turn[kMaxPairs];      // inv_freq / 2 pi in units of 2^-64
  uint8_t axis[kMaxPairs];
};

// VEC neighbouring values as one word.
template <int BYTES>
struct Word;
template <>
struct Word<16> { using type = uint4; };
template <>
struct Word<8> { using type = uint2; };
template <>
struct Word<4> { using type = uint32_t; };
template <>
struct Word<2> { using type = uint16_t; };

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Cosine and sine of an angle of `turns` 2^-64.
__device__ __forceinline__ float2 cos_sin(uint64_t turns, uint32_t flip) {
  const uint32_t t = (uint32_t)(turns >> 32);
  const uint32_t quadrant = (t + 0x20000000u) >> 30;
  const float half_turns = (float)(int32_t)(t - (quadrant << 30)) * 4.656612873077393e-10f;  // (2^-31) in [-1/4, 1/4]
  float s, c;
  sincospif(half_turns, &s, &c);
  const float x = quadrant & 1 ? -s : c, y = quadrant & 1 ? c : s;
  const uint32_t turned = (quadrant & 2) << 30;
  return make_float2(__uint_as_float(__float_as_uint(x) ^ turned), __uint_as_float(__float_as_uint(y) ^ turned ^ flip));
}

// (The same roundings in every instance, so that results do not depend on strides and alignment.)
template <class T>
__device__ __forceinline__ void turn(T& a, T& b, float2 cs) {
  const float u = to_float(a), v = to_float(b);
  a = from_float<T>(__fmaf_rn(u, cs.x, -__fmul_rn(v, cs.y)));
  b = from_float<T>(__fmaf_rn(v, cs.x, __fmul_rn(u, cs.y)));
}

// Places of the angles in shared memory: those that neighbouring items of a warp read at once lie side by side.
template <int VEC>
__device__ __forceinline__ int place(int pair, int items) {
  if (VEC == 1) return pair;
  const int k = pair / VEC, e = pair % VEC;
  return ((e / 2) * items + k) * 2 + e % 2;
}

// What lies in the parameters, as memory: the constant cache serves one address of a warp at a time.
template <class T>
__device__ __forceinline__ const T* as_memory(const T* p) {
  asm("mov.b64 %0, %0;" : "+l"(p));
  return p;
}

// A block turns a.heads_block heads of one token, or (SEVERAL) all heads of a.tokens_block tokens, an item each thread.
template <class T, int VEC, bool SEVERAL>
__global__ void __launch_bounds__(kThreads, SEVERAL ? 6 : 8) rotary_kernel(const __grid_constant__ Args a) {
  using W = typename Word<VEC * (int)sizeof(T)>::type;
  extern __shared__ __align__(16) float2 angles[];  // [a.tokens_block, a.pairs]
  const int tid = threadIdx.x;
  const int h0 = SEVERAL ? 0 : blockIdx.y * a.heads_block, h1 = SEVERAL ? a.heads : min(h0 + a.heads_block, a.heads);
  const int turning = a.pairs / VEC;                                // items of a head that turn 2 VEC values
  const int items = turning + (a.rest + 2 * VEC - 1) / (2 * VEC);   // and those that copy as many
  const int first = first_token(blockIdx.x, SEVERAL ? a.tokens_block : 1);
  if constexpr (!SEVERAL) {
    const uint64_t turn = tid < a.pairs ? a.turn[tid] : 0;
    start_in_order();
    if (tid < a.pairs) {
      const int b = first / a.tokens, t = first - b * a.tokens;
      const int64_t pos = a.pos[a.axis[tid] * a.ps[0] + b * a.ps[1] + t * a.ps[2]];
      angles[place<VEC>(tid, turning)] = cos_sin((uint64_t)pos * turn, a.flip);
    }
  } else {
    // (a thread keeps its pair; q and k of one head, 65536 tokens: 28 us, and 35 with the pairs from the constant cache)
    const int at_once = blockDim.x / a.pairs, pair = tid % a.pairs;
    const uint64_t turn = as_memory(a.turn)[pair];
    const int axis = as_memory(a.axis)[pair];
    start_in_order();
    for (int token = tid / a.pairs; token < a.tokens_block && tid < at_once * a.pairs; token += at_once) {
      const int g = token_or_last(first, token, a.total), b = g / a.tokens, t = g - b * a.tokens;
      const int64_t pos = a.pos[axis * a.ps[0] + b * a.ps[1] + t * a.ps[2]];
      angles[token * a.pairs + place<VEC>(pair, turning)] = cos_sin((uint64_t)pos * turn, a.flip);
    }
  }
  __syncthreads();

  // item and head of a thread's next item, stepped without divisions
  const int token = SEVERAL ? tid / (items * a.heads) : 0;
  if (SEVERAL && !has_token(first, token, a.tokens_block, a.total)) return;
  const int of_token = SEVERAL ? tid - token * (items * a.heads) : tid;
  const int b = (first + token) / a.tokens, t = first + token - b * a.tokens;
  int item = of_token % items, head = h0 + of_token / items;
  const int step = SEVERAL ? 0 : blockDim.x % items, steps = SEVERAL ? a.heads : blockDim.x / items;
  for (; head < h1; item += step, head += steps) {
    if (item >= items) {
      item -= items;
      if (++head >= h1) break;
    }
    // two words, `second` values apart
    int at, second;
    if (item < turning) {
      at = a.offset + item * VEC * (a.interleaved ? 2 : 1);
      second = a.interleaved ? VEC : a.pairs;
    } else {
      // (the values beside the rotary part stand in one line; a last half item has no second word)
      const int c = (item - turning) * 2 * VEC, d = c + VEC;
      at = c < a.offset ? c : c + 2 * a.pairs;
      second = d >= a.rest ? 0 : (d < a.offset ? d : d + 2 * a.pairs) - at;
    }
    const bool q = head < a.first;
    const Tensor& x = a.t[q ? 0 : 1];
    const int h = q ? head : head - a.first;
    const T* src = static_cast<const T*>(x.x) + (b * x.xs[0] + h * x.xs[1] + t * x.xs[2]) + at;
    T* dst = static_cast<T*>(x.y) + (b * x.ys[0] + h * x.ys[1] + t * x.ys[2]) + at;
    W lo = *reinterpret_cast<const W*>(src), hi = *reinterpret_cast<const W*>(src + second);
    if (item < turning) {
      alignas(16) T v[2 * VEC];
      *reinterpret_cast<W*>(v) = lo;
      *reinterpret_cast<W*>(v + VEC) = hi;
      float2 cs[VEC];
      const float2* mine = angles + token * a.pairs + (VEC == 1 ? 1 : 2) * item;
      if constexpr (VEC == 1) {
        cs[0] = mine[0];
      } else {
#pragma unroll
        for (int e = 0; e < VEC; e += 2) {
          const float4 two = *reinterpret_cast<const float4*>(mine + e * turning);
          cs[e] = make_float2(two.x, two.y), cs[e + 1] = make_float2(two.z, two.w);
        }
      }
      if (a.interleaved) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) turn(v[2 * e], v[2 * e + 1], cs[e]);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) turn(v[e], v[e + VEC], cs[e]);
      }
      lo = *reinterpret_cast<const W*>(v);
      hi = *reinterpret_cast<const W*>(v + VEC);
    }
    *reinterpret_cast<W*>(dst) = lo;
    if (second != 0) *reinterpret_cast<W*>(dst + second) = hi;
  }
}

}  // namespace rotary
}  // namespace nsa
