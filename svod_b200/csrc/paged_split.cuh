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
SVODB_SPLIT Run run_of(int64_t total, int cta, int ctas) {
  int64_t quota = (total + ctas - 1) / ctas;
  if (quota < kLeastShare) quota = kLeastShare;
  const int64_t c0 = quota * cta;
  return Run{quota, c0, c0 + quota < total ? c0 + quota : total};
}

// A run's share of an item: its blocks [from, to).
struct Share {
  int b, hk, q;
  int from, to, blocks;  // of the item's blocks
  int part;              // -1: the whole item; else where its state goes: 1 the item's first part, 0 another
  int last_cta;          // the CTA that has the item's last part
};

// Walks a run that is not empty, share by share, until it ends or `take` returns false. Row b is the
// row in which it begins; that row's work begins at `x` and is `weight` a KV head.
template <typename P, typename RowAt, typename Take>
SVODB_SPLIT void walk_run(const P& p, const Run& run, int batch, int kv_heads, int b, int64_t x, int64_t weight, RowAt&& row_at,
                          Take&& take) {
  Row row = row_at(b);
  int hk = (int)((run.c0 - x) / weight), q = 0;
  x += hk * weight;
  for (int64_t w = item_blocks(p, row, 0) + kItemCost; x + w <= run.c0; w = item_blocks(p, row, q) + kItemCost) x += w, ++q;
  while (x < run.c1) {
    const int blocks = item_blocks(p, row, q);
    const int64_t w = blocks + kItemCost;
    const int64_t u0 = (run.c0 > x ? run.c0 - x : 0) - kItemCost, u1 = (run.c1 < x + w ? run.c1 - x : w) - kItemCost;
    const int from = u0 > 0 ? (int)u0 : 0, to = u1 > 0 ? (int)u1 : 0;
    if (to > from) {
      const int part = from == 0 && to == blocks ? -1 : from == 0 ? 1 : 0;
      if (!take(row, Share{b, hk, q, from, to, blocks, part, (int)((x + w - 1) / run.quota)})) return;
    }
    x += w;
    if (++q < live_items(p, row)) continue;
    q = 0;
    if (++hk < kv_heads) continue;
    hk = 0;
    // (rows without tokens have no items)
    do {
      if (++b >= batch) return;
      row = row_at(b);
    } while (row.n == 0);
  }
}

}  // namespace paged
}  // namespace svodb
