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
  const int64_t t = (int64_t)width * kPage * stride + block - 1;
  return t < kMaxTokens ? (int32_t)t : kMaxTokens;
}
// Tokens that a row sees, 0 where it selects nothing (no such token, or more of them than the table or float32 can place).
NSA_HD int32_t tokens_of(const Batch& b, int row, int32_t most) {
  const int seq = cache::sequence_of(b, row);
  const int pos = seq < 0 ? -1 : cache::position_of(b, seq, row);
  return pos >= 0 && pos < most ? pos + 1 : 0;
}
NSA_HD int32_t blocks_of(int32_t tokens, int32_t shift) { return (int32_t)(((int64_t)tokens + (1 << shift) - 1) >> shift); }

// The block of compressed key i of n.
NSA_LINSPACE int32_t block_of(int i, int32_t tokens, int32_t n, int32_t shift) {
  const int32_t block = (int32_t)linspace_f32(i, tokens, n) >> shift, last = blocks_of(tokens, shift) - 1;
  return block < last ? block : last;
}
// The first compressed key that is not in a block before `block`; n if there is none.
NSA_LINSPACE int32_t first_key(int32_t block, int32_t tokens, int32_t n, int32_t shift) {
  if (block <= 0 || n <= 1) return block <= 0 ? 0 : n;
  int64_t i = (int64_t)((double)((int64_t)block << shift) * (double)(n - 1) / (double)(tokens - 1));
  if (i > n) i = n;
  while (i > 0 && block_of((int)i - 1, tokens, n, shift) >= block) --i;
  while (i < n && block_of((int)i, tokens, n, shift) < block) ++i;
  return (int32_t)i;
}

}  // namespace cache_select
}  // namespace nsa
