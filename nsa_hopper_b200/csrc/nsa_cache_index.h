// Where things are in the 4-bit paged KV cache: the record's layout, a row's sequence and position, a
// token's page, and the share of one worker of the attention kernel.  Every index that the cache kernels
// take from the caller's device tensors (page table, lengths, cu_seqlens, selection) is turned into an
// address here and nowhere else, and each is checked against its range first: the host cannot see those
// values, so a value out of range makes the token absent, never an access out of bounds.  Plain C++ on
// purpose: the CPU tests compile this header and feed it broken tables.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define NSA_HD __host__ __device__ __forceinline__
#else
#define NSA_HD inline
#endif

namespace nsa {
namespace cache {

constexpr int kPage = 64;   // tokens of a page
constexpr int kGroup = 16;  // neighbouring values that share a scale

// A record (one page of one KV head): K codes, K scales, V codes, V scales, token after token.
NSA_HD constexpr int record_bytes(int d_qk, int d_v) { return kPage * (d_qk + d_v) * 9 / 16; }
NSA_HD constexpr int k_scale_at(int d_qk) { return kPage * d_qk / 2; }
NSA_HD constexpr int v_code_at(int d_qk) { return kPage * d_qk * 9 / 16; }
NSA_HD constexpr int v_scale_at(int d_qk, int d_v) { return v_code_at(d_qk) + kPage * d_v / 2; }

// Of a number that is not 0.
NSA_HD int highest_bit(uint32_t x) {
#ifdef __CUDA_ARCH__
  return 31 - __clz(x);
#else
  return 31 - __builtin_clz(x);
#endif
}

// The batch that all three calls describe: page table [n_seqs, width], lengths, packed rows.
struct Batch {
  const int32_t* pages;
  const int32_t* lens;
  const int32_t* cu;      // nullptr: row r is the last token of sequence r
  int64_t page_row;       // entries between two sequences' rows of `pages`
  int32_t n_seqs, width;  // width: pages a sequence can have
  int32_t num_pages;      // pages of the cache
  int32_t n_rows;
};

// The sequence of a row, -1 for a row of none (before cu[0] or behind cu[n_seqs]).  In a cu_seqlens that is out of order it is
// one of those whose range holds the row, or -1, and the two forms need not agree.
NSA_HD int sequence_of(const Batch& b, int row) {
  if (b.cu == nullptr) return row < b.n_seqs ? row : -1;
  if (b.n_seqs <= 0 || row < b.cu[0]) return -1;
  int lo = 0, hi = b.n_seqs;  // the last s with cu[s] <= row is in [lo, hi)
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (b.cu[mid] <= row) lo = mid;
    else hi = mid;
  }
  return row < b.cu[lo + 1] ? lo : -1;
}
// The same, 32 places of cu at a time: `below(lo, step, hi)` has bit i set where place lo + i * step is before hi and its cu not
// above the row.  (A thread that searches by itself is faster with the form above: the reading kernel takes 64 us for 104448
// tokens of 16 sequences, and 71 with this one's steps.)
template <class Below>
NSA_HD int sequence_by_32(const Batch& b, int row, Below&& below) {
  if (b.cu == nullptr) return row < b.n_seqs ? row : -1;
  int lo = 0, hi = b.n_seqs;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int last = highest_bit(below(lo, step, hi) | 1);  // (lo stays a candidate)
    lo += last * step;
    hi = hi - lo > step ? lo + step : hi;
  }
  return b.n_seqs > 0 && b.cu[lo] <= row && row < b.cu[lo + 1] ? lo : -1;
}

// Position of a row in its sequence (from sequence_of, >= 0): the sequence's last rows are the call's.
// Negative where the sequence has no such token.
NSA_HD int position_of(const Batch& b, int seq, int row) {
  const int len = b.lens[seq] > 0 ? b.lens[seq] : 0;
  const int behind = b.cu == nullptr ? 1 : b.cu[seq + 1] - row;  // >= 1
  return len - behind;
}

// Keys of a sequence that a row at `pos` may see at most: those up to itself that the page table can hold.
NSA_HD int keys_up_to(const Batch& b, int pos) {
  if (pos < 0) return 0;
  const int64_t held = (int64_t)b.width * kPage;
  return pos < held ? pos + 1 : (int)held;
}

// The cache page of 64-key sub-block `sub` of a sequence, -1 where there is none.
NSA_HD int page_of(const Batch& b, int seq, int sub) {
  if (sub < 0 || sub >= b.width) return -1;
  const int p = b.pages[(int64_t)seq * b.page_row + sub];
  return p >= 0 && p < b.num_pages ? p : -1;
}

// First and one-past-last visible key of a row (window <= 0: no window).
NSA_HD int first_key(int pos, int window) { return window > 0 && pos + 1 > window ? pos + 1 - window : 0; }

// The sub-block that slot j of a row stands for, -1 if it shows no key: entry j / per of the row's
// selection (per = l' / 64), or the j-th sub-block from the window's first.
NSA_HD int selected_sub(int entry, int part, int per, int first, int end) {
  if (entry < 0 || end <= 0 || entry > (end - 1) / (per * kPage)) return -1;  // (before the product can overflow)
  const int sub = entry * per + part;
  return sub <= (end - 1) / kPage && sub >= first / kPage ? sub : -1;  // (the last one's end may be 2^31)
}
NSA_HD int running_sub(int j, int first, int end) {
  const int sub = first / kPage + j;
  return end > first && sub * (int64_t)kPage < end ? sub : -1;
}
// Slots of a row that takes its sub-blocks one after the other; at least one, so that every row has an owner.
NSA_HD int running_slots(int first, int end) { return end > first ? (end - 1) / kPage - first / kPage + 1 : 1; }

NSA_HD uint32_t ceil_div(uint32_t a, uint32_t b) { return a / b + (a % b != 0); }

// How the slots of a call (rows x slots, standing in one line) are shared out among the device's warps.  `team` warps (a
// power of two, neighbours of a block) take turns at a row's slots and join their results; a team has `share` whole rows, or,
// where rows are cut, `share` slots, whose parts a second kernel joins.
struct Split {
  uint32_t team, share, cut;
};
constexpr uint32_t kTeam = 8;     // largest team: a block
constexpr uint32_t kCluster = 8;  // largest cluster of blocks
constexpr uint32_t kLong = 16;    // slots of a warp from which on warps of their own are better than teams where rows are cut
// What things take, in quarters of the time that a warp needs for a slot while it has its quarter of the SM for itself
// (2000 cycles): a slot beside another warp, a team's join, the second kernel.
constexpr uint32_t kSlotAlone = 4, kSlotShared = 7, kJoin = 5, kMerge = 18;

// Time of whole rows of at most `longest` slots with teams of `team` warps.
NSA_HD uint64_t whole_rows(uint32_t rows, uint32_t longest, uint32_t warps, uint32_t team) {
  const uint32_t slot = (uint64_t)rows * team * 2 > warps ? kSlotShared : kSlotAlone;
  return (uint64_t)ceil_div(rows, warps / team) * ((uint64_t)ceil_div(longest, team) * slot + (team > 1 ? kJoin : 0));
}
NSA_HD uint32_t best_team(uint32_t rows, uint32_t longest, uint32_t warps) {
  uint32_t best = 1;
  for (uint32_t team = 2; team <= kTeam; team *= 2)
    if (whole_rows(rows, longest, warps, team) < whole_rows(rows, longest, warps, best)) best = team;
  return best;
}

// `longest`: slots of the longest row (>= 1), `total` < 2^31: of all rows; `warps`: a multiple of kTeam.
NSA_HD Split split_line(uint32_t rows, uint32_t total, uint32_t longest, uint32_t warps) {
  Split s;
  s.team = best_team(rows, longest, warps);
  const uint32_t cutting = total / warps >= kLong ? 1 : kTeam, share = ceil_div(total, warps / cutting);
  const uint64_t cut = (uint64_t)ceil_div(share, cutting) * kSlotShared + (cutting > 1 ? kJoin : 0) + kMerge;
  s.cut = cut < whole_rows(rows, longest, warps, s.team);
  if (s.cut) s.team = cutting;
  s.share = s.cut ? share : ceil_div(rows, warps / s.team);
  return s;
}
// Whether split_line can cut rows of at most `longest` slots at all.
NSA_HD bool may_cut(uint32_t rows, uint32_t longest, uint32_t warps) {
  return whole_rows(rows, longest, warps, best_team(rows, longest, warps)) > kSlotShared + kMerge;
}
// Blocks that share each row, in a cluster, where rows are so few that most SMs would have none: at most as many as leave
// each a slot for every second warp, and only where no warp gets many.  1: no clusters.
NSA_HD uint32_t cluster_of(uint32_t rows, uint32_t longest, uint32_t warps) {
  uint32_t n = kCluster;
  while (n > 1 && ((uint64_t)rows * kTeam * n > warps || longest < kTeam * n / 2)) n /= 2;
  return ceil_div(longest, kTeam * n) <= 5 ? n : 1;
}

}  // namespace cache
}  // namespace nsa
