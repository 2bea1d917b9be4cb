// Attention of a chunk of new tokens over a paged cache on tcgen05: many query rows a KV head.
//
// The arithmetic is attention_tc.cu's and the pipeline attention_tc_p.cu's: base-2 online
// softmax in f32 with the lazy rescale, weights rounded to the stream type before P.V while
// their sum is taken in f32, scores one block of 64 keys ahead of the softmax, two 128-row
// tiles whose softmax warps take turns on the MUFU unit, one CTA an SM that walks its items
// behind a two-slot ring of `Work`. What differs:
//
// Rows: the query heads that share a KV head lie in one tile, 128 / group tokens x group heads
// (one TMA box [tokens, group, 64 columns]), so that a KV head's keys are fetched once for all
// of them and a causal edge crosses fewer rows' blocks.
//
// Pages: a block of 64 keys is 64 / box boxes of box = gcd(page_size, 64) keys, one page each,
// issued by as many lanes; a box outside the item's visible keys is fetched past the last page,
// where a copy reads zeros and no table entry is looked at. What the first and last block's
// pages hold beside visible keys may be NaN: the issuers clear those rows of V before they
// take them (K needs none of it, hidden scores are replaced).
//
// Work split: the batch's lengths are device memory, so the CTAs share the work out themselves.
// Every one adds up the blocks of all items (a fixed cost of kItemCost blocks each) and takes
// its equal run of them, in the order rows, KV heads, tiles. A run may begin and end inside an
// item: such a part leaves its f32 state in the workspace and a second kernel merges an item's
// parts. Rows of 0 to 6000 held keys and 128 to 512 new ones then take what their sum takes,
// not what the longest does. No atomics, the same parts in every run.
//
// 8-bit pages: a fourth warpgroup widens each block from a ring of raw e4m3 blocks into the
// 16-bit rings, value * 2^e, exact in bf16 (a value is 4 bits) and rounded once in f16's
// subnormals and at its top (`in_range`; weights rounded to f16 could carry an average of its
// largest values past it, so such results are kept in range too). A thread moves a key's row:
// the e4m3 fields are shifted to where the 16-bit type has them and one packed multiply puts
// exponent bias and scale right, 5 instructions a pair of values (a conversion through f32 is 6,
// on slower pipes).
//
// Every mbarrier wait is bounded; a warp that gave up walks on as in attention_tc_p.cu.
#include <cuda.h>
#include <math.h>
#include <stdio.h>

#include "attention_parts.cuh"
#include "common.cuh"
#include "kernels.h"
#include "launch.h"
#include "paged.cuh"
#include "svodb.h"
#include "tensormap.h"

namespace svodb {

namespace {

using namespace fa_parts;
using namespace paged;

static_assert(kBlockKeys == kBKV, "the work is shared out in the blocks that the tiles take");

template <bool Q8, int D>
struct PagedTcCfg {
  static constexpr int kThreads = Q8 ? 512 : 384;
  static constexpr int kStages = 4;
  static constexpr int kRawStages = 4;
  static constexpr int kRawBytes = kBKV * 128;      // one block of e4m3 rows, 128 bytes a key
  static constexpr int kQTile = 128 * D * 2;
  static constexpr int kKv = kBKV * D * 2;
  static constexpr size_t kSmem = 1024 + (size_t)2 * kQTile + (size_t)2 * kStages * kKv + (Q8 ? kRawStages * kRawBytes : 0) +
                                  768;  // the barriers and the items
  static_assert(kSmem <= 232448, "beyond the 227 KiB a CTA may hold");
};

struct PagedTcParams {
  PagedAttnArgs a;
  int group, tile_tokens;  // tokens of a 128-row tile: 128 / group
  int box;
  Divider page_size;
  float scale_log2;
  int* heads_of_split;     // [grid][kSplitInts]: the split item whose first part a CTA has
  float* parts;            // [grid][2][part floats]
};

// What a CTA says about the item it has the first part of, where others have the rest.
constexpr int kSplitInts = 8;
struct SplitItem {
  int valid, b, hk, t0, n_live, last_cta;
};
// A part's state: O [D][256] by columns, then m and l of its 256 rows.
template <int D>
constexpr int64_t kPartFloats = (int64_t)D * 256 + 512;

struct PagedWork {
  int valid, b, hk, t0, n_live, start;
  int key_lo, key_hi;  // of the item
  Range r0, r1;        // this part's blocks, per tile
  int u_lo, u_hi;
  int part;            // -1: the whole item, else the slot that the state goes to
};

__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// Two e4m3 values, bytes 0 and 1 (or 2 and 3) of `w`, as a 16-bit pair whose exponent bias is
// still e4m3's; the multiply by `up` (2^120 or 2^8 times the row's scale) puts it right.
template <typename T>
__device__ __forceinline__ uint32_t widen_pair(uint32_t w, int upper, uint32_t up) {
  const uint32_t t = __byte_perm(w, 0, upper ? 0x3424 : 0x1404);  // each value in the upper byte of a half
  if constexpr (std::is_same<T, __half>::value) {
    const uint32_t u = (t & 0x80008000u) | ((t >> 1) & 0x3f803f80u);
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&u), *reinterpret_cast<const __half2*>(&up));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const uint32_t u = (t & 0x80008000u) | ((t >> 4) & 0x07f007f0u);
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&u), *reinterpret_cast<const __nv_bfloat162*>(&up));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}
// The multiplier of `widen_pair` for a row's scale code as a 16-bit pair; 0 where the type has
// no normal number for it (then the row goes through f32).
template <typename T>
__device__ __forceinline__ uint32_t widen_factor(uint32_t code) {
  uint32_t h;
  if constexpr (std::is_same<T, __half>::value) {
    const int e = (int)code - 127 + 8 + 15;  // f16's exponent field of 2^(code - 127 + 8)
    h = e >= 1 && e <= 30 ? (uint32_t)e << 10 : 0u;
  } else {
    const int e = (int)code + 120;
    h = e <= 254 ? (uint32_t)e << 7 : 0u;
  }
  return h | (h << 16);
}

// A softmax warp that no item came to within the limit, which the status word says: the loader's
// next wait ends, but what it published until then the warp's partner may have caught, and both
// have to walk the same turns. So it takes what has come after a while longer.
__device__ __noinline__ void walk_late_items(uint64_t* item_full, uint64_t* item_empty, const PagedWork* ring, uint32_t n_it, int i,
                                             uint32_t turns, int my_turn, int other_turn) {
  for (; mbar_arrives(&item_full[n_it & 1], (n_it >> 1) & 1, kWaitLimit / 64); ++n_it) {
    const int n_paired = ring[n_it & 1].valid ? paired_blocks(ring[n_it & 1].r0, ring[n_it & 1].r1) : -1;
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&item_empty[n_it & 1]);
    if (n_paired < 0) break;
    for (int m = 0; m < n_paired; ++m, ++turns) {
      if (i == 1 || turns > 0) named_barrier(my_turn, 64);
      named_barrier_arrive(other_turn, 64);
    }
  }
}

template <typename T, bool Q8, int D>
__global__ void __launch_bounds__((PagedTcCfg<Q8, D>::kThreads), 1)
    attention_paged_tc_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                              const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ PagedTcParams p) {
  using C = PagedTcCfg<Q8, D>;
  constexpr int S = C::kStages, R = C::kRawStages;
  constexpr int QB = C::kQTile, KB = C::kKv;
  constexpr int KBOX = kBKV * 128;  // bytes of one 64-column box of a K/V block
  const PagedAttnArgs& a = p.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = smem;               // [2][QB]
  uint8_t* k_s = q_s + 2 * QB;       // [S][KB]
  uint8_t* v_s = k_s + S * KB;       // [S][KB]
  uint8_t* raw_s = v_s + S * KB;     // [R][kRawBytes] (8-bit pages)
  uint64_t* bars = reinterpret_cast<uint64_t*>(raw_s + (Q8 ? R * C::kRawBytes : 0));
  uint64_t* q_full = bars;            // [2]
  uint64_t* q_empty = bars + 2;       // [2]
  uint64_t* k_full = bars + 4;        // [S]
  uint64_t* k_empty = k_full + S;
  uint64_t* v_full = k_empty + S;
  uint64_t* v_empty = v_full + S;
  uint64_t* s_full = v_empty + S;     // [2 tiles][2 buffers]
  uint64_t* p_full = s_full + 4;      // [2 tiles][2 buffers]
  uint64_t* tail_done = p_full + 4;   // [2 tiles]: the last two P.V of a tile
  uint64_t* o_empty = tail_done + 2;  // [2 tiles]
  uint64_t* item_full = o_empty + 2;  // [2 slots]
  uint64_t* item_empty = item_full + 2;
  uint64_t* raw_full = item_empty + 2;  // [R]
  uint64_t* raw_empty = raw_full + R;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(raw_empty + R);
  PagedWork* item_ring = reinterpret_cast<PagedWork*>(tmem_slot + 2);  // [2]
  static_assert((4 + 4 * S + 18 + 2 * R) * 8 + 8 + 2 * sizeof(PagedWork) <= 768, "the barriers and the items fit");

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&tail_done[i], 1);
      mbar_init(&o_empty[i], 4);                // the tile's four softmax warps
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], Q8 ? 15 : 11);  // value loader, two issuers, eight softmax warps, four widening ones
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);  // one arrival per softmax warp
    }
    for (int i = 0; i < S; ++i) {
      mbar_init(&k_full[i], Q8 ? 2 : 1);  // widening warps, or the loader's copies
      mbar_init(&k_empty[i], 2);          // released by both tiles' issuers
      mbar_init(&v_full[i], Q8 ? 2 : 1);
      mbar_init(&v_empty[i], 2);
    }
    for (int i = 0; i < R; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], 2);
    }
    mbar_fence_init();
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (warp == 2) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  pdl_wait();
  const uint32_t tmem_base = *tmem_slot;
  const int64_t capacity = a.c.width * a.c.page_size;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    const int nb = kBKV / p.box;
    constexpr int kCols = Q8 ? 1 : D / 64;
    const int my_box = lane % nb, my_col = lane / nb;
    const bool mine = my_col < kCols;
    // Lane 0's bounded wait, for the warp.
    auto wait_by_lane0 = [&](uint64_t* bar, uint32_t parity) {
      bool done = true;
      if (lane == 0) done = mbar_wait(bar, parity, a.status);
      return __shfl_sync(0xffffffffu, (int)done, 0) != 0;
    };
    // A part's blocks of keys (or values), the lanes issuing a block's boxes side by side; `pos`
    // counts the blocks of all parts. A copy per lane is a trip through the warp's uniform
    // registers each: keys and values go by a warp of their own (pages of 16 tokens: 16 copies a
    // block, 1.5 us by one warp where the block's arithmetic takes 1.2).
    auto load_blocks = [&](const PagedWork& w, int kv, uint32_t& pos) {
      const int32_t* table = a.c.table + (int64_t)w.b * a.c.table_sb;
      auto look_up = [&](int blk, int& at) -> int {
        const int j = blk * kBKV + my_box * p.box;
        at = 0;
        if (!mine || blk >= w.u_hi || j + p.box <= w.key_lo || j >= w.key_hi) return (int)a.c.pages;
        const uint32_t page = p.page_size.div((uint32_t)j);
        at = j - (int)(page * p.page_size.d);
        const int id = table[page];
        if (id < 0 || id >= a.c.pages) {
          report_bad_index(a.bad_index);
          return (int)a.c.pages;
        }
        return id;
      };
      const CUtensorMap* map = kv ? &tmap_v : &tmap_k;
      int next_at;
      int next_id = look_up(w.u_lo, next_at);
      for (int j = w.u_lo; j < w.u_hi; ++j, ++pos) {
        const int id = next_id, at = next_at;
        next_id = look_up(j + 1, next_at);
        uint64_t *full, *empty;
        uint8_t* to;
        uint32_t round;
        if constexpr (Q8) {  // the raw ring's stages: K V K V
          static_assert(R == 4);
          const int st = (int)((pos & 1) << 1) | kv;
          full = raw_full + st, empty = raw_empty + st, to = raw_s + st * C::kRawBytes, round = pos >> 1;
        } else {
          const int st = (int)(pos % S);
          full = (kv ? v_full : k_full) + st, empty = (kv ? v_empty : k_empty) + st, to = (kv ? v_s : k_s) + st * KB, round = pos / S;
        }
        if (!wait_by_lane0(empty, (round & 1) ^ 1)) return false;
        if (lane == 0) mbar_expect_tx(full, Q8 ? C::kRawBytes : KB);
        __syncwarp();
        if (mine) tma_load_4d(to + my_col * KBOX + my_box * p.box * 128, map, full, my_col * 64, w.hk, at, id);
      }
      return true;
    };
    if (warp == 0) {
      // ---------------- the CTA's run of the work, and its keys ----------------
      auto row_at = [&](int b) { return row_of(a.start, a.lens, b, a.t, capacity); };
      const int batch = (int)a.batch;
      // lane l keeps row l: a batch of up to 32 rows is read and weighed once
      const Row my_row = lane < batch ? row_at(lane) : Row{0, 0, false};
      const int64_t my_weight = row_weight(p, my_row);
      if (my_row.bad && blockIdx.x == 0) report_bad_index(a.bad_index);
      int64_t total = my_weight;
      for (int b = lane + 32; b < batch; b += 32) {
        const Row r = row_at(b);
        if (r.bad && blockIdx.x == 0) report_bad_index(a.bad_index);
        total += row_weight(p, r);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      total *= a.c.kv_heads;
      const Run run = run_of(total, blockIdx.x, gridDim.x);
      const int64_t c0 = run.c0, c1 = run.c1;
      // Row b for the whole warp.
      auto fetch_row = [&](int b) {
        if (b >= 32) return row_at(b);
        Row r;
        r.start = __shfl_sync(0xffffffffu, my_row.start, b);
        r.n = __shfl_sync(0xffffffffu, my_row.n, b);
        r.bad = false;
        return r;
      };
      // Where the run begins: row b, KV head hk, item q, whose weight lies at [x, x + weight).
      int b = 0, hk = 0, q = 0;
      int64_t x = 0;
      Row row{0, 0, false};
      int64_t weight_of_row = 0;
      if (c0 < c1) {
        int64_t base = 0;
        for (int b0 = 0; b0 < batch; b0 += 32) {
          const int64_t w = (b0 == 0 ? my_weight : b0 + lane < batch ? row_weight(p, row_at(b0 + lane)) : 0) * a.c.kv_heads;
          int64_t upto = w;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
          }
          const uint32_t past = __ballot_sync(0xffffffffu, base + upto > c0);
          if (past != 0u) {
            const int l = __ffs((int)past) - 1;
            b = b0 + l;
            weight_of_row = __shfl_sync(0xffffffffu, w, l) / a.c.kv_heads;
            x = base + __shfl_sync(0xffffffffu, upto - w, l);
            break;
          }
          base += __shfl_sync(0xffffffffu, upto, 31);
        }
        row = fetch_row(b);
        find_item(p, run, row, weight_of_row, x, hk, q);
      }
      SplitItem split{0, 0, 0, 0, 0, 0};
      uint32_t pos = 0;
      bool ok = true;
      uint32_t n_it = 0;
      // (a CTA whose run would begin behind the last item has none)
      while (c0 < c1 && x < c1 && ok) {
        PagedWork w;
        w.valid = 1, w.b = b, w.hk = hk, w.t0 = q * 2 * p.tile_tokens, w.n_live = row.n, w.start = (int)row.start;
        item_keys(p, row, q, w.key_lo, w.key_hi);
        const int blk_lo = w.key_lo / kBKV, blk_n = (w.key_hi + kBKV - 1) / kBKV - blk_lo;
        const int64_t weight = blk_n + kItemCost;
        // this run's part of the item's blocks: its first kItemCost units stand for the fixed cost
        const int from = share_from(c0, x), to = share_to(c1, x, weight);
        if (to > from) {
          w.part = part_of(from, to, blk_n);
          if (w.part == 1) split = SplitItem{1, b, hk, w.t0, row.n, last_cta(x, weight, run.quota)};
          auto range = [&](int t) {
            Range r{0, 0};
            if (t >= row.n) return r;
            const int t_last = min(t + p.tile_tokens, row.n) - 1;
            const int lo = first_key(a, row.start + t) / kBKV;
            const int hi = (last_key(a, row.start + t_last, row.start + row.n) + kBKV - 1) / kBKV;
            const int y = max(lo, blk_lo + from), z = min(hi, blk_lo + to);
            if (z > y) r.lo = y, r.hi = z;
            return r;
          };
          w.r0 = range(w.t0);
          w.r1 = range(w.t0 + p.tile_tokens);
          const bool live0 = w.r0.hi > w.r0.lo, live1 = w.r1.hi > w.r1.lo;
          w.u_lo = w.u_hi = 0;
          if (live0 && live1) {
            w.u_lo = w.r0.lo < w.r1.lo ? w.r0.lo : w.r1.lo;
            w.u_hi = w.r0.hi > w.r1.hi ? w.r0.hi : w.r1.hi;
          } else if (live0) {
            w.u_lo = w.r0.lo, w.u_hi = w.r0.hi;
          } else if (live1) {
            w.u_lo = w.r1.lo, w.u_hi = w.r1.hi;
          }
          const int slot = (int)(n_it & 1);
          ok = wait_by_lane0(&item_empty[slot], ((n_it >> 1) & 1) ^ 1);
          if (!ok) break;
          if (lane == 0) {
            item_ring[slot] = w;
            __threadfence_block();
            mbar_arrive(&item_full[slot]);
          }
          ++n_it;
          ok = load_blocks(w, 0, pos);
        }
        // the next item
        x += weight;
        if (++q == live_items(p, row)) {
          q = 0;
          if (++hk == a.c.kv_heads) {
            hk = 0;
            do row = ++b < batch ? fetch_row(b) : Row{0, 0, false};
            while (b < batch && row.n == 0);
            if (b >= batch) break;
          }
        }
      }
      if (lane == 0) {
        int* h = p.heads_of_split + (int64_t)blockIdx.x * kSplitInts;
        h[0] = split.valid, h[1] = split.b, h[2] = split.hk, h[3] = split.t0, h[4] = split.n_live, h[5] = split.last_cta;
      }
      const int slot = (int)(n_it & 1);
      if (ok && wait_by_lane0(&item_empty[slot], ((n_it >> 1) & 1) ^ 1) && lane == 0) {
        item_ring[slot].valid = 0;
        __threadfence_block();
        mbar_arrive(&item_full[slot]);
      }
      if (!ok)
        for (int i = 0; i < 64; ++i) __nanosleep(1000);  // copies in flight land before the CTA's memory goes
    } else if (warp == 2) {
      // ---------------- query tiles and values ----------------
      uint32_t q_items[2] = {0, 0};  // live items so far, per tile
      uint32_t pos = 0;
      bool ok = true;
      for (uint32_t n_it = 0; ok; ++n_it) {
        const int slot = (int)(n_it & 1);
        if (!wait_by_lane0(&item_full[slot], (n_it >> 1) & 1)) break;
        const PagedWork w = item_ring[slot];
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[slot]);
        if (!w.valid) break;
        for (int i = 0; i < 2 && ok; ++i) {
          if (i == 0 ? w.r0.hi <= w.r0.lo : w.r1.hi <= w.r1.lo) continue;
          // the issuer's last QK of the tile's previous live item has read this Q tile
          ok = wait_by_lane0(&q_empty[i], (q_items[i] & 1) ^ 1);
          ++q_items[i];
          if (ok && lane == 0) {
            mbar_expect_tx(&q_full[i], (uint32_t)(p.tile_tokens * p.group * 128 * (D / 64)));
            for (int c = 0; c < D / 64; ++c)
              tma_load_4d(q_s + i * QB + c * (128 * 128), &tmap_q, &q_full[i], c * 64, w.hk * p.group,
                          w.t0 + i * p.tile_tokens, w.b);
          }
        }
        if (ok) ok = load_blocks(w, 1, pos);
      }
      if (!ok)
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    } else {
      // ---------------- MMA issuers: warp 1 drives tile 0, warp 3 tile 1 (attention_tc_p.cu) ----------------
      const int i = warp == 1 ? 0 : 1;
      const bool leader = elect_one();
      constexpr uint32_t idesc_qk = umma_idesc(Elem<T>::kUmmaFormat, 128, kBKV, 0, 0);
      constexpr uint32_t idesc_pv = umma_idesc(Elem<T>::kUmmaFormat, 128, D, 0, 1);
      const uint64_t qa = umma_desc_sw128(smem_u32(q_s) + i * QB, 16, 1024);
      const uint64_t k_desc0 = umma_desc_sw128(smem_u32(k_s), 16, 1024);
      const uint64_t v_desc0 = umma_desc_sw128(smem_u32(v_s), KBOX, 1024);
      uint32_t kv_blocks = 0;  // K/V blocks of all earlier items (ring position)
      uint32_t my_blocks = 0;  // blocks of this tile in all earlier items (S/P buffer and phase)
      uint32_t my_items = 0;   // live items of this tile so far
      bool ok = true;
      for (uint32_t n_it = 0; ok; ++n_it) {
        const int slot = (int)(n_it & 1);
        if (!mbar_wait(&item_full[slot], (n_it >> 1) & 1, a.status)) break;
        const PagedWork w = item_ring[slot];
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[slot]);
        if (!w.valid) break;
        const Range r = i == 0 ? w.r0 : w.r1;
        const int nblk = r.hi - r.lo;
        const bool live = nblk > 0;
        // blocks that hold slots beside the item's keys
        const int edge_lo = w.key_lo % kBKV != 0 ? w.key_lo / kBKV : -1;
        const int edge_hi = w.key_hi % kBKV != 0 ? w.key_hi / kBKV : -1;
        bool q_ready = false;
        for (int t = w.u_lo - 1; t <= w.u_hi && ok; ++t) {
          const int jq = t + 1;  // block whose scores are issued this step
          const int jp = t - 1;  // block whose P.V is issued this step
          const bool have_k = jq >= w.u_lo && jq < w.u_hi;
          const bool have_v = jp >= w.u_lo && jp < w.u_hi;
          const uint32_t kpos = kv_blocks + (uint32_t)(have_k ? jq - w.u_lo : 0);
          const uint32_t vpos = kv_blocks + (uint32_t)(have_v ? jp - w.u_lo : 0);
          const int ks_slot = (int)(kpos % S), vs_slot = (int)(vpos % S);
          const bool do_pv = have_v && jp >= r.lo && jp < r.hi;
          const bool do_qk = have_k && jq >= r.lo && jq < r.hi;
          // Every slot is waited for and released by both issuers, used or not.
          if ((have_k && !mbar_wait(&k_full[ks_slot], (kpos / S) & 1, a.status)) ||
              (have_v && !mbar_wait(&v_full[vs_slot], (vpos / S) & 1, a.status))) {
            ok = false;
            break;
          }
          if (do_pv) {
            const uint32_t n = (uint32_t)(jp - r.lo);
            const uint32_t N = my_blocks + n;  // this tile's running block counter
            if (n == 0 && !mbar_wait(&o_empty[i], (my_items & 1) ^ 1, a.status)) {
              ok = false;  // the previous item's O has not been read out
              break;
            }
            if (!mbar_wait(&p_full[i * 2 + (N & 1)], (N >> 1) & 1, a.status)) {
              ok = false;
              break;
            }
            if constexpr (!Q8) {
              // Rows beside the item's keys hold whatever the pages hold there: 0 * NaN must not
              // enter the sum. Both issuers clear them, to the same zeros, before either lets go.
              if (jp == edge_lo || jp == edge_hi) {
                for (int y = lane; y < kBKV * (D / 8); y += 32) {
                  const int row = y / (D / 8), c = y % (D / 8), key = jp * kBKV + row;
                  if (key < w.key_lo || key >= w.key_hi)
                    *reinterpret_cast<uint4*>(v_s + vs_slot * KB + (c >> 3) * KBOX + row * 128 + (c & 7) * 16) =
                        make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
                __syncwarp();
              }
            }
            tc_fence_after();
            const uint32_t d_tmem = tmem_base + 256 + i * D;
            const uint32_t a_tmem = tmem_base + (uint32_t)((i * 2 + (N & 1)) * kBKV);
            const uint64_t vb = v_desc0 + (uint64_t)((vs_slot * KB) >> 4);
            const uint32_t first = n != 0 ? 1u : 0u;
#pragma unroll
            for (int ks = 0; ks < kBKV / 16; ++ks)  // 16 keys per step = 2 KiB of V, 8 packed P columns
              if (leader)
                umma_ts(d_tmem, a_tmem + ks * 8, vb + (uint64_t)(ks * (2048 >> 4)), idesc_pv,
                        (first | (uint32_t)ks) != 0 ? 1u : 0u);
            if (leader && (int)n + 2 >= nblk) tc_commit(&tail_done[i]);
          }
          if (do_qk) {
            if (!q_ready) {
              if (!mbar_wait(&q_full[i], my_items & 1, a.status)) {
                ok = false;
                break;
              }
              q_ready = true;
            }
            tc_fence_after();
            const uint32_t N = my_blocks + (uint32_t)(jq - r.lo);
            const uint32_t d_tmem = tmem_base + (uint32_t)((i * 2 + (N & 1)) * kBKV);
            const uint64_t kb = k_desc0 + (uint64_t)((ks_slot * KB) >> 4);
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
              const uint64_t qoff = (uint64_t)((ks >> 2) * ((128 * 128) >> 4) + (ks & 3) * 2);
              const uint64_t koff = (uint64_t)((ks >> 2) * (KBOX >> 4) + (ks & 3) * 2);
              if (leader) umma_ss(d_tmem, qa + qoff, kb + koff, idesc_qk, ks != 0 ? 1u : 0u);
            }
            if (leader) tc_commit(&s_full[i * 2 + (N & 1)]);
            // the item's last QK has read the Q tile: the loader may bring the next one
            if (leader && jq == r.hi - 1) tc_commit(&q_empty[i]);
          }
          if (leader && have_v) tc_commit(&v_empty[vs_slot]);
          if (leader && have_k) tc_commit(&k_empty[ks_slot]);
          __syncwarp();
        }
        kv_blocks += (uint32_t)(w.u_hi - w.u_lo);
        if (live) {
          my_blocks += (uint32_t)nblk;
          ++my_items;
        }
      }
    }
  } else if (Q8 && warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    // ---------------- widening: raw e4m3 blocks into the 16-bit rings ----------------
    if constexpr (Q8) {
      // two warps the keys, two the values: a thread a key's row
      const int tid = threadIdx.x - 384, r = tid & 63, kv = tid >> 6;
      constexpr int kPieces = D / 16;  // 16-byte pieces of a raw row
      const int page_size = a.c.page_size;
      const int pages_on = kBKV / page_size, slots_on = kBKV % page_size;  // from a block to the next
      uint64_t* const full = kv ? v_full : k_full;
      uint64_t* const empty = kv ? v_empty : k_empty;
      // 16-byte piece c of a 128-byte row r lies at (c ^ r) mod 8
      const uint32_t src0 = smem_u32(raw_s) + kv * C::kRawBytes + r * 128 + ((r & 7) << 4);
      const uint32_t dst0 = smem_u32(kv ? v_s : k_s) + r * 128 + ((r & 7) << 4);
      uint32_t pos = 0;  // K/V blocks so far (ring position)
      bool ok = true;
      for (uint32_t n_it = 0; ok; ++n_it) {
        const int islot = (int)(n_it & 1);
        if (!mbar_wait(&item_full[islot], (n_it >> 1) & 1, a.status)) break;
        const PagedWork w = item_ring[islot];
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[islot]);
        if (!w.valid) break;
        const int32_t* table = a.c.table + (int64_t)w.b * a.c.table_sb;
        const uint8_t* scales = kv ? a.c.v_scale + (int64_t)w.hk * a.c.vs_sh : a.c.k_scale + (int64_t)w.hk * a.c.ks_sh;
        const int64_t scales_sp = kv ? a.c.vs_sp : a.c.ks_sp;
        // my key's page and slot walk a block at a time; its page id is looked up two blocks
        // ahead, its scale code one
        int key = w.u_lo * kBKV + r;
        int page = key / page_size, slot = key - page * page_size;
        auto id_of = [&](int k) -> int { return k >= w.key_lo && k < w.key_hi && k < w.u_hi * kBKV ? table[page] : -1; };
        auto code_of = [&](int id) -> uint32_t { return id >= 0 && id < a.c.pages ? scales[id * scales_sp + slot] : 0u; };
        auto step = [&]() {
          page += pages_on, slot += slots_on;
          if (slot >= page_size) slot -= page_size, ++page;
        };
        uint32_t code = code_of(id_of(key));
        step();
        int id_next = id_of(key + kBKV);
        // The rare path rolled up: the roles' code has to stay in the instruction cache. (With
        // both paths unrolled, for keys and for values, these warps waited for every line of
        // theirs: 1100 cycles for 180 instructions.)
        for (int j = w.u_lo; j < w.u_hi; ++j, ++pos, key += kBKV) {
          const uint32_t code_next = code_of(id_next);
          step();
          id_next = id_of(key + 2 * kBKV);
          const int s = (int)(pos % S), st = (int)((pos & 1) << 1);
          const bool real = key >= w.key_lo && key < w.key_hi;
          if (!mbar_wait(&raw_full[st | kv], (pos >> 1) & 1, a.status) || !mbar_wait(&empty[s], ((pos / S) & 1) ^ 1, a.status)) {
            ok = false;
            break;
          }
          const uint32_t src = src0 + st * C::kRawBytes, dst = dst0 + s * KB;
          // a slot beside the item's keys becomes zeros, whatever it holds: every pattern is finite here
          const uint32_t factor = widen_factor<T>(code), up = real ? factor : 0u;
          if (!real || factor != 0u) {
#pragma unroll 1
            for (int h = 0; h < kPieces / 4; ++h) {
              // four pieces of 16 values: a 64-column box of the 16-bit row
              uint4 in[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) in[i] = lds128(src ^ (uint32_t)((4 * h + i) << 4));
              const uint32_t to = dst + h * KBOX;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                sts128(to ^ (uint32_t)((2 * i) << 4), widen_pair<T>(in[i].x, 0, up), widen_pair<T>(in[i].x, 1, up),
                       widen_pair<T>(in[i].y, 0, up), widen_pair<T>(in[i].y, 1, up));
                sts128(to ^ (uint32_t)((2 * i + 1) << 4), widen_pair<T>(in[i].z, 0, up), widen_pair<T>(in[i].z, 1, up),
                       widen_pair<T>(in[i].w, 0, up), widen_pair<T>(in[i].w, 1, up));
              }
            }
          } else {
            // a scale beyond the type's normal numbers, or NaN: through f32
            const float scale = scale_value(code);
#pragma unroll 1
            for (int i = 0; i < 2 * kPieces; ++i) {
              const uint4 in = lds128(src ^ (uint32_t)((i >> 1) << 4));
              const uint32_t wa = i & 1 ? in.z : in.x, wb = i & 1 ? in.w : in.y;
              const float2 x = from_e4m3x2(wa & 0xffffu), y = from_e4m3x2(wa >> 16);
              const float2 z = from_e4m3x2(wb & 0xffffu), u = from_e4m3x2(wb >> 16);
              auto pair = [&](float2 v) { return pack_in_range<T>(v.x * scale, v.y * scale); };
              sts128((dst + (i >> 3) * KBOX) ^ (uint32_t)((i & 7) << 4), pair(x), pair(y), pair(z), pair(u));
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&full[s]);
            mbar_arrive(&raw_empty[st | kv]);
          }
          code = code_next;
        }
      }
    }
  } else {
    // (8-bit pages: 4 x 72 + 4 x 72 + 8 x 184 registers a lane are the 512 x 128 of the launch)
    if constexpr (Q8) asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ---------------- softmax + epilogue (attention_tc_p.cu) ----------------
    // Rows behind a chunk's real tokens that no item has: zeros. An equal run of the batch's
    // tokens a CTA and warp, while the first scores are on their way (one warp that clears an
    // item's 128 tokens x 16 heads alone takes 150 us).
    {
      const int step = 2 * p.tile_tokens, pieces = a.c.d / 8;
      const int64_t tokens = a.batch * a.t, runs = (int64_t)gridDim.x * 8, run = (tokens + runs - 1) / runs;
      const int64_t me = (int64_t)blockIdx.x * 8 + warp - 4;
      const int64_t last = run * (me + 1) < tokens ? run * (me + 1) : tokens;
      for (int64_t u = run * me; u < last;) {
        const int64_t b = u / a.t, row_lo = b * a.t, row_hi = row_lo + a.t < last ? row_lo + a.t : last;
        const Row r = row_of(a.start, a.lens, b, a.t, capacity);
        const int64_t dead = row_lo + (int64_t)live_items(p, r) * step;  // the row's first token without an item
        for (u = u < dead ? dead : u; u < row_hi; ++u) {
          T* o = (T*)a.o + b * a.o_sb + (u - row_lo) * a.o_st;
          for (int x = lane; x < a.heads * pieces; x += 32)
            stg128(o + (int64_t)(x / pieces) * a.o_sh + (x % pieces) * 8, make_uint4(0, 0, 0, 0));
          if (a.lse != nullptr)
            for (int h = lane; h < a.heads; h += 32) a.lse[(b * a.heads + h) * a.t + u - row_lo] = -INFINITY;
        }
        u = row_hi;
      }
    }
    const int i = (warp - 4) >> 2;  // query tile
    const int quarter = warp & 3;   // TMEM lane quarter
    const int tile_row = quarter * 32 + lane;
    const int row_token = tile_row / p.group, row_head = tile_row % p.group;
    const bool in_tile = tile_row < p.tile_tokens * p.group;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const uint32_t o_tmem = tmem_base + 256 + i * D + lane_addr;
    const float sl2 = p.scale_log2;
    const int my_turn = 1 + i * 4 + quarter;
    const int other_turn = 1 + (1 - i) * 4 + quarter;
    uint32_t my_blocks = 0;   // blocks of this tile in all earlier items
    uint32_t tail_count = 0;  // tail commits of this tile in all earlier items
    // Turns on the MUFU unit (attention_tc.cu): tile 0 takes its n-th block that both tiles have,
    // then tile 1 its own, and so on from item to item. A named barrier counts arrivals and does
    // not know their turn: were a warp to arrive twice before its partner has waited once, the
    // two arrivals would complete the barrier between them and the partner would wait for good
    // (short items, where tile 0 finds its next item before tile 1 has begun this one's last
    // block). So each side waits for the other's last turn before every one of its own, the
    // CTA's first excepted, and a warp whose bounded wait ran out walks all turns on.
    uint32_t turns = 0;       // of all earlier items and this one
    bool ok = true;           // false once a bounded wait ran out: nothing is computed from then on
    bool late = false;        // no item came within the limit
    uint32_t n_it = 0;
    for (;; ++n_it) {
      const int slot = (int)(n_it & 1);
      if (!mbar_wait_patient(&item_full[slot], (n_it >> 1) & 1, a.status)) {
        late = true;
        break;
      }
      const PagedWork w = item_ring[slot];
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[slot]);
      if (!w.valid) break;
      const int n_paired = paired_blocks(w.r0, w.r1);
      int turns_done = 0;     // of this item
      bool my_turn_now = false;
      auto take_turn = [&]() {
        if (i == 1 || turns > 0) named_barrier(my_turn, 64);
        my_turn_now = true;
      };
      auto pass_turn = [&]() {
        named_barrier_arrive(other_turn, 64);
        ++turns, ++turns_done;
        my_turn_now = false;
      };
      auto walk_turns = [&]() {
        while (turns_done < n_paired) {
          if (!my_turn_now) take_turn();
          pass_turn();
        }
      };
      if (!ok) {
        walk_turns();
        continue;
      }
      const Range r = i == 0 ? w.r0 : w.r1;
      const int nblk = r.hi - r.lo;
      const int t_first = w.t0 + i * p.tile_tokens, t_row = t_first + row_token;
      const bool row_ok = in_tile && t_row < a.t;  // a row of the output
      const bool row_real = row_ok && t_row < w.n_live;
      const int64_t end = (int64_t)w.start + w.n_live;
      const int vis_lo = row_real ? first_key(a, (int64_t)w.start + t_row) : 0;
      const int vis_hi = row_real ? last_key(a, (int64_t)w.start + t_row, end) : 0;
      // keys that every live token of the tile sees
      const int t_last = min(t_first + p.tile_tokens, w.n_live) - 1;
      const int all_lo = first_key(a, (int64_t)w.start + t_last), all_hi = last_key(a, (int64_t)w.start + t_first, end);
      auto vis_word = [&](int base) -> uint32_t {
        int x = vis_lo - base, y = vis_hi - base;
        x = x < 0 ? 0 : x;
        y = y > 32 ? 32 : y;
        uint32_t word = 0;
        if (y > x) word = (y == 32 ? 0xffffffffu : ((1u << y) - 1u)) & ~((1u << x) - 1u);
        return word;
      };
      float m_run = -INFINITY;  // running maximum, scaled log2 units
      float l_run = 0.f;
      uint32_t sr[2][32];
      bool requested = false;
      for (int j = r.lo; j < r.hi && ok; ++j) {
        const int n = j - r.lo;
        const uint32_t N = my_blocks + (uint32_t)n;
        const int buf = (int)(N & 1);
        const uint32_t s_tmem = tmem_base + (uint32_t)((i * 2 + buf) * kBKV) + lane_addr;
        if (!requested) {
          if (!mbar_wait(&s_full[i * 2 + buf], (N >> 1) & 1, a.status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          tmem_ld32(s_tmem, sr[0]);
          tmem_ld32(s_tmem + 32, sr[1]);
        }
        const int j0 = j * kBKV;
        const bool need_mask = j0 < all_lo || j0 + kBKV > all_hi;
        tmem_ld_wait_for(sr[0]);
        tmem_ld_wait_for(sr[1]);
        if (need_mask) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t vw = vis_word(j0 + 32 * c);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (((vw >> e) & 1u) == 0) sr[c][e] = 0xff800000u;
          }
        }
        float mx;
        {
          float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              m0 = max3(m0, __uint_as_float(sr[c][e]), __uint_as_float(sr[c][e + 1]));
              m1 = max3(m1, __uint_as_float(sr[c][e + 2]), __uint_as_float(sr[c][e + 3]));
              m2 = max3(m2, __uint_as_float(sr[c][e + 4]), __uint_as_float(sr[c][e + 5]));
              m3 = max3(m3, __uint_as_float(sr[c][e + 6]), __uint_as_float(sr[c][e + 7]));
            }
          }
          mx = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
        }
        const float mx_t = mx * sl2;  // scale > 0 on this path
        float m_new = m_run;
        if (mx_t > m_run + kRescaleAbove || m_run == -INFINITY) m_new = fmaxf(m_run, mx_t);
        bool tail0_seen = false;
        const bool moved = m_new != m_run && m_run != -INFINITY;
        const float corr = moved ? ex2_approx(m_run - m_new) : 1.0f;
        if (__any_sync(0xffffffffu, moved)) {
          const uint32_t Nn = N + 1;
          const bool landed = n + 1 < nblk ? mbar_wait(&s_full[i * 2 + (int)(Nn & 1)], (Nn >> 1) & 1, a.status)
                                           : mbar_wait(&tail_done[i], tail_count & 1, a.status);
          if (!landed) {
            ok = false;
            break;
          }
          tail0_seen = n + 1 == nblk;
          tc_fence_after();
          l_run *= corr;
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t orr[32];
            tmem_ld32(o_tmem + c, orr);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) orr[e] = __float_as_uint(__uint_as_float(orr[e]) * corr);
            tmem_st32(o_tmem + c, orr);
          }
          tmem_st_wait();
        }
        m_run = m_new;
        float m_use = m_run == -INFINITY ? 0.f : m_run;
        if (n < n_paired) {
          take_turn();
          asm volatile("" : "+f"(m_use));  // keeps the exponentials below the barrier
        }
        const float2 sl2_2 = make_float2(sl2, sl2), nm_2 = make_float2(-m_use, -m_use);
        float2 la = make_float2(0.f, 0.f), lb = make_float2(0.f, 0.f);
        uint32_t pk[32];
        constexpr int kLag = 6;
        float2 xs[32];
#pragma unroll
        for (int k = 0; k < 32; ++k)
          xs[k] = __ffma2_rn(make_float2(__uint_as_float(sr[k >> 4][2 * (k & 15)]),
                                         __uint_as_float(sr[k >> 4][2 * (k & 15) + 1])),
                             sl2_2, nm_2);
#pragma unroll
        for (int k = 0; k < 32 + kLag; ++k) {
          if (k < 32) {
            xs[k].x = ex2_approx(xs[k].x);
            xs[k].y = ex2_approx(xs[k].y);
          }
          if (k >= kLag) {
            const int d = k - kLag;
            if (d & 1) lb = __fadd2_rn(lb, xs[d]);
            else la = __fadd2_rn(la, xs[d]);
            pk[d] = Elem<T>::pack(xs[d].x, xs[d].y);
          }
        }
        tmem_st32(s_tmem, pk);
        if (n < n_paired) pass_turn();
        l_run += (la.x + la.y) + (lb.x + lb.y);
        requested = false;
        if (n + 1 < nblk) {
          const uint32_t Nn = N + 1;
          if (mbar_test_wait(&s_full[i * 2 + (int)(Nn & 1)], (Nn >> 1) & 1)) {
            tc_fence_after();
            const uint32_t next_tmem = tmem_base + (uint32_t)((i * 2 + (int)(Nn & 1)) * kBKV) + lane_addr;
            tmem_ld32(next_tmem, sr[0]);
            tmem_ld32(next_tmem + 32, sr[1]);
            requested = true;
          }
        }
        tmem_st_wait();
        if (n + 1 == nblk && nblk >= 2 && !tail0_seen && !mbar_wait(&tail_done[i], tail_count & 1, a.status)) {
          ok = false;
          break;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[i * 2 + buf]);
      }
      if (!ok) {
        walk_turns();
        continue;
      }
      // ---- epilogue: O / l, zeros in rows without a key; or a part's state ----
      const int head = w.hk * p.group + row_head;
      float* part = w.part < 0 ? nullptr : p.parts + ((int64_t)blockIdx.x * 2 + w.part) * kPartFloats<D>;
      const int row = i * 128 + tile_row;
      if (!row_real) l_run = 0.f;
      const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;
      T* orow = (T*)a.o + (int64_t)w.b * a.o_sb + (int64_t)t_row * a.o_st + (int64_t)head * a.o_sh;
      if (nblk > 0) {
        // the last P.V: the item's second tail commit (its only one for a one-block tile)
        const uint32_t last = tail_count + (nblk >= 2 ? 1u : 0u);
        if (!mbar_wait(&tail_done[i], last & 1, a.status)) {
          ok = false;  // the item's hand-over sequence is complete: drain from the next item on
          continue;
        }
        tc_fence_after();
        if (part != nullptr) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t orr[32];
            tmem_ld32(o_tmem + c, orr);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) part[(c + e) * 256 + row] = __uint_as_float(orr[e]);
          }
        } else {
          // A small rolled body: this code runs once an item, and what the block loop's did not
          // leave in the instruction cache comes at the price of its fetches (a whole prompt of 4 x
          // 4096 tokens: 32 columns unrolled, a row a lane, 288 us; 16 so, 279.5).
          const unsigned long long mine = row_ok ? (unsigned long long)orow : 0ull;
          T* const row_even = (T*)__shfl_sync(0xffffffffu, mine, lane & 30);
          T* const row_odd = (T*)__shfl_sync(0xffffffffu, mine, lane | 1);
          auto pair = [](float x, float y) {
            if constexpr (Q8 && std::is_same<T, __half>::value) return pack_in_range<T>(x, y);
            else return Elem<T>::pack(x, y);
          };
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t orr[16], o[8];
            tmem_ld16(o_tmem + c, orr);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 8; ++e)
              o[e] = l_run == 0.f ? 0u : pair(__uint_as_float(orr[2 * e]) * inv, __uint_as_float(orr[2 * e + 1]) * inv);
            // two lanes change halves and write 32 bytes of either row side by side, whole sectors
            const bool odd = (lane & 1) != 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t give = __shfl_xor_sync(0xffffffffu, odd ? o[e] : o[4 + e], 1);
              if (odd) o[e] = give;
              else o[4 + e] = give;
            }
            const int col = c + (odd ? 8 : 0);
            if (row_even != nullptr && col < a.c.d) stg128(row_even + col, make_uint4(o[0], o[1], o[2], o[3]));
            if (row_odd != nullptr && col < a.c.d) stg128(row_odd + col, make_uint4(o[4], o[5], o[6], o[7]));
          }
        }
        // O is read out: the next live item's first P.V may overwrite it
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_empty[i]);
        my_blocks += (uint32_t)nblk;
        tail_count += nblk >= 2 ? 2u : 1u;
      } else if (part == nullptr && row_ok) {
        for (int c = 0; c < a.c.d; c += 8) stg128(orow + c, make_uint4(0, 0, 0, 0));
      }
      if (part != nullptr) {
        part[D * 256 + row] = m_run;
        part[D * 256 + 256 + row] = l_run;
      } else if (a.lse != nullptr && row_ok) {
        a.lse[((int64_t)w.b * a.heads + head) * a.t + t_row] = l_run == 0.f ? -INFINITY : kLn2F * (m_run + log2f(l_run));
      }
    }
    if (late) walk_late_items(item_full, item_empty, item_ring, n_it, i, turns, my_turn, other_turn);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// The parts of the items that more than one CTA had: block (CTA, kMergeCols columns), a thread a
// row. Bound by the parts' way through L2 (up to 38 MB) and the trips to memory one after another,
// hence two parts' 34 loads at a time, the first two beside the table that says whether they are
// there (24 x 512 tokens: 80.1 us with the table first, 78.6 so; a merge of nothing takes 1.7).
constexpr int kMergeCols = 16;
template <typename T, int D>
__global__ void __launch_bounds__(256) attention_paged_merge_kernel(const __grid_constant__ PagedTcParams p) {
  pdl_trigger();
  pdl_wait();
  const PagedAttnArgs& a = p.a;
  const int first = blockIdx.x, row = threadIdx.x, d0 = blockIdx.y * kMergeCols;
  // the first part lies in its CTA's second slot, the others in their CTAs' first
  auto part_of = [&](int k) { return p.parts + ((int64_t)k * 2 + (k == first ? 1 : 0)) * kPartFloats<D>; };
  // Two parts at a time; the first two are asked for beside the table that says whether there are any.
  float mr[2], lr[2], x[2][kMergeCols];
  auto fetch = [&](int u, int k) {
    const float* part = part_of(k);
    mr[u] = part[D * 256 + row];
    lr[u] = part[D * 256 + 256 + row];
#pragma unroll
    for (int e = 0; e < kMergeCols; ++e) x[u][e] = part[(d0 + e) * 256 + row];
  };
  const int4* h = reinterpret_cast<const int4*>(p.heads_of_split + (int64_t)first * kSplitInts);
  const int4 h0 = h[0], h1 = h[1];
  fetch(0, first);
  fetch(1, first + 1 < (int)gridDim.x ? first + 1 : first);
  if (h0.x == 0) return;
  const int b = h0.y, hk = h0.z, t0 = h0.w, n_live = h1.x, last = h1.y;
  const int in_tile = row & 127;
  const int t_row = t0 + (row >> 7) * p.tile_tokens + in_tile / p.group;
  const int head = hk * p.group + in_tile % p.group;
  if (in_tile >= p.tile_tokens * p.group || t_row >= a.t) return;
  float m = -INFINITY, l = 0.f, acc[kMergeCols];
#pragma unroll
  for (int e = 0; e < kMergeCols; ++e) acc[e] = 0.f;
  if (t_row < n_live) {
    for (int k0 = first;;) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        // no key of this row there (NaN scores leave the maximum at -inf, the sum says so), or no such part
        if (k0 + u > last || lr[u] == 0.f) continue;
        const float m_new = fmaxf(m, mr[u]);
        const float f0 = m == -INFINITY ? 1.f : ex2_approx(m - m_new), f1 = mr[u] == -INFINITY ? 1.f : ex2_approx(mr[u] - m_new);
        l = fmaf(l, f0, f1 * lr[u]);
#pragma unroll
        for (int e = 0; e < kMergeCols; ++e) acc[e] = fmaf(acc[e], f0, f1 * x[u][e]);
        m = m_new;
      }
      k0 += 2;
      if (k0 > last) break;
      fetch(0, k0);
      fetch(1, k0 < last ? k0 + 1 : k0);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const bool q8 = a.c.dtype == SVODB_E4M3;
  auto pair = [&](float x, float y) { return std::is_same<T, __half>::value && q8 ? pack_in_range<T>(x, y) : Elem<T>::pack(x, y); };
  T* o = (T*)a.o + (int64_t)b * a.o_sb + (int64_t)t_row * a.o_st + (int64_t)head * a.o_sh + d0;
#pragma unroll
  for (int v = 0; v < kMergeCols / 8; ++v) {
    if (d0 + v * 8 >= a.c.d) break;  // padded head dim
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = pair(acc[v * 8 + 2 * e] * inv, acc[v * 8 + 2 * e + 1] * inv);
    stg128(o + v * 8, make_uint4(w[0], w[1], w[2], w[3]));
  }
  if (a.lse != nullptr && d0 == 0)
    a.lse[((int64_t)b * a.heads + head) * a.t + t_row] = l == 0.f ? -INFINITY : kLn2F * (m + log2f(l));
}

// One CTA an SM.
int grid_of(const PagedAttnArgs&) {
  static int n[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  int& sms = n[dev & 63];
  if (sms == 0) {
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) {
      cudaGetLastError();
      sms = 148;
    }
  }
  return sms;
}

template <typename T, bool Q8, int D>
int run(const PagedAttnArgs& a, cudaStream_t s, char* cfg, size_t cfg_len) {
  using C = PagedTcCfg<Q8, D>;
  PagedTcParams p{};
  p.a = a;
  p.group = a.heads / a.c.kv_heads;
  p.tile_tokens = 128 / p.group;
  p.box = page_box(a.c.page_size, kBKV);
  p.scale_log2 = a.scale * kLog2eF;
  p.page_size = divider((uint32_t)a.c.page_size);
  const int grid = grid_of(a);
  p.parts = (float*)a.workspace;
  p.heads_of_split = (int*)(p.parts + (int64_t)grid * 2 * kPartFloats<D>);
  CUtensorMap tq, tk, tv;
  {
    const uint64_t dims[4] = {(uint64_t)a.c.d, (uint64_t)a.heads, (uint64_t)a.t, (uint64_t)a.batch};
    const uint64_t any = 128;  // a dim of one element has no stride of its own
    const uint64_t st[3] = {a.heads == 1 ? any : (uint64_t)a.q_sh, a.t == 1 ? any : (uint64_t)a.q_st,
                            a.batch == 1 ? any : (uint64_t)a.q_sb};
    const uint32_t box[4] = {64, (uint32_t)p.group, (uint32_t)p.tile_tokens, 1};
    if (!make_tmap(&tq, a.q, a.dtype, 4, dims, st, box)) return -1;
  }
  if (!page_map(&tk, a.c, false, Q8 ? 128 : 64, p.box) || !page_map(&tv, a.c, true, Q8 ? 128 : 64, p.box)) return -1;
  static bool attr_seen[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr_seen[dev & 63]) {
    if (cudaFuncSetAttribute(attention_paged_tc_kernel<T, Q8, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)C::kSmem) != cudaSuccess)
      return -1;
    attr_seen[dev & 63] = true;
  }
  if (launch_pdl(attention_paged_tc_kernel<T, Q8, D>, dim3((unsigned)grid), dim3(C::kThreads), C::kSmem, s, 1,
                 a.batch * a.t, tq, tk, tv, p) != cudaSuccess)
    return -1;
  if (launch_pdl(attention_paged_merge_kernel<T, D>, dim3((unsigned)grid, (unsigned)((a.c.d + kMergeCols - 1) / kMergeCols)),
                 dim3(256), 0, s, 1, 0, p) != cudaSuccess)
    return -1;
  snprintf(cfg, cfg_len, "{bq:%d,bkv:%d,d:%d,box:%d,grid:%d%s}", 2 * kBQ, kBKV, a.c.d, p.box, grid, Q8 ? ",e4m3" : "");
  return 0;
}

template <typename T>
int run_type(const PagedAttnArgs& a, cudaStream_t s, char* cfg, size_t cfg_len) {
  const bool q8 = a.c.dtype == SVODB_E4M3;
  if (a.c.d > 64) return q8 ? run<T, true, 128>(a, s, cfg, cfg_len) : run<T, false, 128>(a, s, cfg, cfg_len);
  return q8 ? run<T, true, 64>(a, s, cfg, cfg_len) : run<T, false, 64>(a, s, cfg, cfg_len);
}

}  // namespace

bool attention_paged_tc_covers(const PagedAttnArgs& a) {
  if (!attention_paged_tiles(a)) return false;
  const int64_t group = a.heads / a.c.kv_heads;
  if (group > 128 || a.batch > 0x7fffff00LL || a.t > 0x7fffff00LL) return false;
  // the query rows come by a tensor map, which has no stride of zero (an expanded view)
  return !((a.heads > 1 && a.q_sh == 0) || (a.t > 1 && a.q_st == 0) || (a.batch > 1 && a.q_sb == 0));
}

size_t attention_paged_tc_workspace(const PagedAttnArgs& a) {
  const int64_t part = a.c.d > 64 ? kPartFloats<128> : kPartFloats<64>;
  return (size_t)grid_of(a) * (2 * (size_t)part * sizeof(float) + kSplitInts * sizeof(int));
}

int launch_attention_paged_tc(const PagedAttnArgs& a, cudaStream_t s, char* cfg, size_t cfg_len) {
  return a.dtype == SVODB_BF16 ? run_type<__nv_bfloat16>(a, s, cfg, cfg_len) : run_type<__half>(a, s, cfg, cfg_len);
}

}  // namespace svodb
