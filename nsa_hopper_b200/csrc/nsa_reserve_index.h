// The arithmetic of nsa_cache_reserve: which pages a batch of sequences takes from the pool and gives back, and where each row
// of the call then lies.  As in nsa_cache_index.h every index that comes from the caller's device tensors is checked here and
// nowhere else, and the CPU tests compile this header and feed it broken tables.
#pragma once
#include "nsa_cache_index.h"

namespace nsa {
namespace reserve {

using cache::kPage;

NSA_HD int32_t pages_of(int32_t tokens) { return tokens / kPage + (tokens % kPage != 0); }

// What `rows` does to a sequence that holds `held` tokens, before it is known whether the pool has the pages.
struct Change {
  int32_t held;           // tokens before, inside the table
  int32_t after;          // tokens after (as before if they do not fit)
  int32_t before_pages, after_pages;
  bool grows;             // it asks for rows that the table can hold
  NSA_HD int32_t need() const { return after_pages > before_pages ? after_pages - before_pages : 0; }
  NSA_HD int32_t give() const { return before_pages > after_pages ? before_pages - after_pages : 0; }
};
NSA_HD Change change_of(int32_t held, int32_t rows, int32_t width) {
  const int64_t table = (int64_t)width * kPage, most = table < 0x7FFFFFFF ? table : 0x7FFFFFFF;
  Change c;
  c.held = held < 0 ? 0 : held > most ? (int32_t)most : held;
  const int64_t want = (int64_t)c.held + rows;
  c.grows = rows > 0 && want <= most;
  c.after = c.grows ? (int32_t)want : rows >= 0 ? c.held : want > 0 ? (int32_t)want : 0;
  c.before_pages = pages_of(c.held);
  c.after_pages = pages_of(c.after);
  return c;
}

// The batch after the sums over its sequences: sequence s takes the pages need[s] .. need[s + 1] - 1 of those that are
// wanted, gives the pages give[s] .. give[s + 1] - 1 of those that come back, and has the rows cu[s] .. cu[s + 1] - 1.
struct Plan {
  const int32_t* pages;    // [n_seqs, width]
  const int32_t* pool;     // [pool_size]
  const uint32_t* need;    // [n_seqs + 1] each
  const uint32_t* give;
  const uint32_t* cu;
  const int32_t* from;     // [n_seqs] first page of a sequence's row of the table that is taken or given back
  const int32_t* lens;     // [n_seqs] tokens after the call of a sequence that has rows, 0 where it has none
  int64_t page_row;
  int32_t n_seqs, width;
  int32_t free;            // pages of the pool before the call, in [0, pool_size]
  int32_t first;           // place of the first page that is taken in the pool to which the pages given back are added
};

NSA_HD int32_t clamp_free(int32_t free, int32_t pool_size) { return free < 0 ? 0 : free > pool_size ? pool_size : free; }
// Whether sequence s, with the sum `end` of the needs up to its own, gets its pages: `top` are there.
NSA_HD bool granted(const Change& c, uint32_t end, int32_t top) { return c.grows && (c.need() == 0 || end <= (uint32_t)top); }

// The last s in [0, n) with at[s] <= i (at[0] = 0): the one whose range holds i, if i < at[n].
NSA_HD int range_of(const uint32_t* at, int n, uint32_t i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (at[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}
// Page j of those that are given back (j < give[n_seqs]).
NSA_HD int32_t given_page(const Plan& p, uint32_t j) {
  const int s = range_of(p.give, p.n_seqs, j);
  return p.pages[(int64_t)s * p.page_row + p.from[s] + (int32_t)(j - p.give[s])];
}
// Page j of those that are taken (j below the sum of the granted needs): the topmost of the pool, in its order.  The pages
// given back may not be there yet, so they come from the table, where no call that gives them back changes them.
NSA_HD int32_t taken_page(const Plan& p, uint32_t j) {
  const int64_t at = (int64_t)p.first + j;
  return at < p.free ? p.pool[at] : given_page(p, (uint32_t)(at - p.free));
}
// The page of sub-block `sub` of a sequence that has rows, after the call.
NSA_HD int32_t page_after(const Plan& p, int s, int32_t sub) {
  return sub < p.from[s] ? p.pages[(int64_t)s * p.page_row + sub] : taken_page(p, p.need[s] + (uint32_t)(sub - p.from[s]));
}
NSA_HD int64_t slot_of(int32_t page, int32_t pos) { return page < 0 ? -1 : (int64_t)page * kPage + pos % kPage; }

}  // namespace reserve
}  // namespace nsa
