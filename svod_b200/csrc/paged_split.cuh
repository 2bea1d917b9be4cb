// How the CTAs of the paged attention (attention_paged_tc.cu) share its work out: arithmetic on
// the rows' lengths alone, compiled for the kernel and, without CUDA, for the host.
//
// An item is the query tokens of two tiles of a row and KV head. It weighs its blocks of visible
// keys and a fixed cost. The items of all rows lie one after the other, rows, KV heads, query
// tokens; CTA c takes the units [c * quota, (c + 1) * quota) of their weight. The first units of an
// item stand for its fixed cost, so a CTA whose run touches those alone has nothing of the item.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define SVODB_SPLIT __host__ __device__ __forceinline__
#else
#define SVODB_SPLIT inline
#endif

namespace svodb {
namespace paged {

constexpr int kBlockKeys = 64;  // keys of a block
constexpr int kItemCost = 2;    // what an item costs beside its blocks, in blocks
// Blocks (and items' costs) a CTA takes at least, where there are few. 16 heads on 8 KV heads
// with 2, 4 and 8: 150 tokens from the start on 15, 18 and 20 us; 2 x 64 tokens behind up to
// 1000 held ones, where a share of 2 is a part of one block, 22, 20 and 21. Neither is best for
// both; 4 is within a fifth of either's best.
constexpr int kLeastShare = 4;

// What a row of the batch holds: its first `n` chunk tokens are real and stand at positions
// `start` and on, the last key at start + n - 1.
struct Row {
  int64_t start;
  int n;
  bool bad;  // a start below zero or keys past the table: the row is taken as empty and the status word says so
};

// Keys [first, last) that the query token at position `pos` sees in a row of `end` keys; both
// grow with the position. A: causal, has_window, win_left, win_right.
template <typename A>
SVODB_SPLIT int first_key(const A& a, int64_t pos) {
  const int64_t x = a.has_window ? pos - a.win_left : 0;
  return (int)(x > 0 ? x : 0);
}
template <typename A>
SVODB_SPLIT int last_key(const A& a, int64_t pos, int64_t end) {
  int64_t x = end;
  if (a.causal && pos + 1 < x) x = pos + 1;
  if (a.has_window && pos + a.win_right + 1 < x) x = pos + a.win_right + 1;
  return (int)x;
}

// The keys of item q of a row. P: a, and the tokens of a tile.
template <typename P>
SVODB_SPLIT void item_keys(const P& p, const Row& r, int q, int& lo, int& hi) {
  const int t = q * 2 * p.tile_tokens, end = t + 2 * p.tile_tokens, t_last = (end < r.n ? end : r.n) - 1;
  lo = first_key(p.a, r.start + t);
  hi = last_key(p.a, r.start + t_last, r.start + r.n);
}
template <typename P>
SVODB_SPLIT int item_blocks(const P& p, const Row& r, int q) {
  int lo, hi;
  item_keys(p, r, q, lo, hi);
  return (hi + kBlockKeys - 1) / kBlockKeys - lo / kBlockKeys;
}
template <typename P>
SVODB_SPLIT int live_items(const P& p, const Row& r) {
  return (r.n + 2 * p.tile_tokens - 1) / (2 * p.tile_tokens);
}
// What a row's items weigh, for one KV head.
template <typename P>
SVODB_SPLIT int64_t row_weight(const P& p, const Row& r) {
  int64_t w = 0;
  for (int q = 0; q < live_items(p, r); ++q) w += item_blocks(p, r, q) + kItemCost;
  return w;
}

// A CTA's equal run of the work, units [c0, c1) of `total`.
struct Run {
  int64_t quota, c0, c1;
};
SVODB_SPLIT Run run_of(int64_t total, uint32_t cta, uint32_t ctas) {
  int64_t quota = (total + ctas - 1) / ctas;
  if (quota < kLeastShare) quota = kLeastShare;
  const int64_t c0 = quota * cta;
  return Run{quota, c0, c0 + quota < total ? c0 + quota : total};
}

// Where a run begins in a row whose work begins at `x` and weighs `weight` a KV head: the KV head
// and the item, and where that item's work begins.
template <typename P>
SVODB_SPLIT void find_item(const P& p, const Run& run, const Row& row, int64_t weight, int64_t& x, int& hk, int& q) {
  hk = (int)((run.c0 - x) / weight);
  x += hk * weight;
  q = 0;
  for (int64_t w = item_blocks(p, row, 0) + kItemCost; x + w <= run.c0; w = item_blocks(p, row, q) + kItemCost) x += w, ++q;
}

// A run's share of an item that weighs `weight` from `x` on: its blocks [from, to), none where the
// run has units of the fixed cost alone. (As scalars: a struct of them in the kernel's walk makes
// windowed e4m3 chunks 1.5 % slower.)
SVODB_SPLIT int share_from(int64_t c0, int64_t x) {
  const int64_t u = (c0 > x ? c0 - x : 0) - kItemCost;
  return u > 0 ? (int)u : 0;
}
SVODB_SPLIT int share_to(int64_t c1, int64_t x, int64_t weight) {
  const int64_t u = (c1 < x + weight ? c1 - x : weight) - kItemCost;
  return u > 0 ? (int)u : 0;
}
// Where a share's state goes: nowhere where it is the whole item (-1), else 1 for the item's first
// part and 0 for another.
SVODB_SPLIT int part_of(int from, int to, int blocks) { return from == 0 && to == blocks ? -1 : from == 0 ? 1 : 0; }
// The CTA that has the item's last part.
SVODB_SPLIT int last_cta(int64_t x, int64_t weight, int64_t quota) { return (int)((x + weight - 1) / quota); }

}  // namespace paged
}  // namespace svodb
