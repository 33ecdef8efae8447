// Where the compressed keys of a 4-bit cache stand among the selection blocks, for the block selection of single tokens, and the
// whole numbers of its exact scores.  Plain C++, which the CPU tests compile.  A
// row at position t sees the first T = t + 1 tokens of its sequence as block selection sees a prompt of T: n compressed keys,
// key i in the block of the float32 linspace(0, T - 1, n)[i] (see nsa_linspace.cuh).
#pragma once
#include "nsa_cache_index.h"
#include "nsa_linspace.cuh"

namespace nsa {
namespace cache_select {

using cache::Batch;
using cache::kGroup;
using cache::kPage;

// Longest sequence: positions are whole numbers in float32, so that the places of keys never run backwards.
constexpr int32_t kMaxTokens = 1 << 24;

NSA_HD int32_t completed(int32_t tokens, int32_t block, int32_t stride) {
  return tokens >= block ? (tokens - block) / stride + 1 : 0;
}
// Tokens of the longest sequence whose compressed keys a table of `width` pages holds.
NSA_HD int32_t most_tokens(int32_t width, int32_t block, int32_t stride) {
  const int64_t keys = (int64_t)width * kPage, t = (keys < kMaxTokens ? keys : kMaxTokens) * stride + block - 1;
  return t < kMaxTokens ? (int32_t)t : kMaxTokens;
}
// Tokens that a row of sequence `seq` (from sequence_of) sees, 0 where it selects nothing (no such token, or more of them than the table or float32 can place).
template <class L = cache::Load>
NSA_HD int32_t tokens_of(const Batch& b, int seq, int row, int32_t most, L load = L()) {
  const int pos = seq < 0 ? -1 : cache::position_of(b, seq, row, load);
  return pos >= 0 && pos < most ? pos + 1 : 0;
}
NSA_HD int32_t blocks_of(int32_t tokens, int32_t shift) { return (int32_t)(((int64_t)tokens + (1 << shift) - 1) >> shift); }

// The compressed keys of a row's tokens among the blocks.
struct Places {
  int32_t tokens, n;  // n: compressed keys
  int32_t shift;      // of a block's tokens
  float step;         // tokens from one key to the next
  float per;          // and the reverse, about
};
NSA_LINSPACE Places places_of(int32_t tokens, int32_t block, int32_t stride, int32_t shift) {
  Places p;
  p.tokens = tokens, p.n = completed(tokens, block, stride), p.shift = shift;
  p.step = p.n > 1 ? linspace_step(tokens, p.n) : 1.f;
  p.per = 1.f / p.step;
  return p;
}
// linspace_at with one rounding.  It has one too: a key and a position are below 2^24 and the step is at least 1, so that
// products and differences have at most 48 bits and are exact in fp64 (the CPU tests compare the two).
NSA_LINSPACE float place_of(const Places& p, int32_t i) {
#ifdef __CUDA_ARCH__
  return i < p.n / 2 ? __fmul_rn(p.step, (float)i) : __fmaf_rn(-p.step, (float)(p.n - 1 - i), (float)(p.tokens - 1));
#else
  return i < p.n / 2 ? p.step * (float)i : fmaf(-p.step, (float)(p.n - 1 - i), (float)(p.tokens - 1));
#endif
}
// The block of key i of more than one.  (A place is at most that of the last token, so no block is behind the last one.)
NSA_LINSPACE int32_t block_of(const Places& p, int32_t i) { return (int32_t)place_of(p, i) >> p.shift; }
// The first key that is not in a block before `block`; n if there is none.
NSA_LINSPACE int32_t first_key(const Places& p, int32_t block) {
  if (block <= 0) return 0;
  if (p.n <= 1) return p.n;
  const float guess = ceilf((float)((int64_t)block << p.shift) * p.per);
  int32_t i = guess < (float)p.n ? (int32_t)guess : p.n;
  const bool down = i > 0 && block_of(p, i - 1) >= block, up = i < p.n && block_of(p, i) < block;
  if (down || up) {  // (the guess is off by a key where a block begins at one, about)
    while (i > 0 && block_of(p, i - 1) >= block) --i;
    while (i < p.n && block_of(p, i) < block) ++i;
  }
  return i;
}

// ------------------------------------------------------------------ whole numbers
// Four bytes of a and b (places 4 to 7), by the lower three bits of the nibbles of `select`; with the fourth bit the sign of that
// byte in all its bits.
NSA_HD uint32_t pick_bytes(uint32_t a, uint32_t b, uint32_t select) {
#ifdef __CUDA_ARCH__
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(select));
  return r;
#else
  uint32_t r = 0;
  for (int i = 0; i < 4; ++i) {
    const uint32_t s = select >> 4 * i & 15, at = s & 7, byte = (at < 4 ? a >> 8 * at : b >> 8 * (at - 4)) & 255;
    r |= (s < 8 ? byte : byte >> 7 != 0 ? 255u : 0u) << 8 * i;
  }
  return r;
#endif
}
// sum + the four products of signed bytes, modulo 2^32.
NSA_HD uint32_t add_products(uint32_t a, uint32_t b, uint32_t sum) {
#ifdef __CUDA_ARCH__
  return (uint32_t)__dp4a((int)a, (int)b, (int)sum);
#else
  for (int i = 0; i < 4; ++i) sum += (uint32_t)((int32_t)(int8_t)(a >> 8 * i & 255) * (int8_t)(b >> 8 * i & 255));
  return sum;
#endif
}
constexpr int kCodeZero = 12;  // of decode4
// Four codes, doubled and 12 more: whole numbers 0 to 24 in four bytes.
NSA_HD uint32_t decode4(uint32_t codes) {
  // (for negative codes the first gives the sign, 0, of a byte of the table; for the others the second does)
  const uint32_t plus = pick_bytes(0x03020100u, 0x0C080604u, codes), minus = pick_bytes(0x03020100u, 0x0C080604u, codes ^ 0x8888u);
  return 0x0C0C0C0Cu + plus - minus;
}
// The lowest signed byte of x, which is taken off; the next ones follow.
NSA_HD int8_t next_byte(int64_t& x) {
  const int8_t byte = (int8_t)(x & 255);
  x = (x - byte) >> 8;
  return byte;
}
// Adds 16 codes (from decode4) times 16 bytes of the query to the sum of the higher bytes.
NSA_HD uint32_t add_group(uint32_t higher, const uint32_t (&codes)[4], const uint32_t (&bytes)[4]) {
  return add_products(codes[0], bytes[0],
                      add_products(codes[1], bytes[1], add_products(codes[2], bytes[2], add_products(codes[3], bytes[3], higher * 256))));
}
// What three bytes' sums are too large by, negative: 12 of every code.
NSA_HD uint32_t too_many(const uint32_t (&low)[4], const uint32_t (&middle)[4], const uint32_t (&high)[4]) {
  const uint32_t twelve[4] = {0x0C0C0C0Cu, 0x0C0C0C0Cu, 0x0C0C0C0Cu, 0x0C0C0C0Cu};
  return 0u - add_group(add_group(add_group(0, twelve, high), twelve, middle), twelve, low);
}
// Upper half of the fp64 of a scale byte of at least 8 (a quiet NaN's for those that stand for no number); its lower half is 0.
NSA_HD uint32_t scale_high(uint32_t byte) { return byte < 0xF8 ? (byte << 17) + (1008u << 20) : 0x7FF80000u; }

}  // namespace cache_select
}  // namespace nsa
