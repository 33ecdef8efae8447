// Where the compressed keys of a 4-bit cache stand among the selection blocks, for the block selection of single tokens.  A
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

}  // namespace cache_select
}  // namespace nsa
