// The tokens of a block of the rotary kernel.  Plain C++, so that the CPU tests compile it: with all tokens that a call may
// have, a last block of several tokens ends behind 2^31 - 1.
#pragma once
#include "nsa_cache_index.h"

namespace nsa {
namespace rotary {

// First token of a block (below 2^31 - 1, the most that a call has).
NSA_HD int32_t first_token(uint32_t block, int32_t tokens_block) { return (int32_t)(block * (uint32_t)tokens_block); }
// Whether the block that begins at `first` has a token `i`.
NSA_HD bool has_token(int32_t first, int32_t i, int32_t tokens_block, int32_t total) { return i < tokens_block && i < total - first; }
// Token `i` of the block, the last one of all where it has none.
NSA_HD int32_t token_or_last(int32_t first, int32_t i, int32_t total) { return i < total - first ? first + i : total - 1; }

}  // namespace rotary
}  // namespace nsa
