// Attention of a chunk of new tokens over a paged cache on tcgen05: many query rows a KV head.
//
// The arithmetic is attention_tc.cu's: base-2 online softmax in f32 with the lazy rescale,
// weights rounded to the stream type before P.V while their sum is taken in f32, scores one
// block of 64 keys ahead of the softmax, two 128-row tiles a CTA whose softmax warps take
// turns on the MUFU unit. What differs:
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
// 8-bit pages: a fourth warpgroup widens each block from a ring of raw e4m3 blocks into the
// 16-bit rings, value * 2^e, exact in bf16 (a value is 4 bits) and rounded once in f16's
// subnormals. A thread moves half a key's row: the e4m3 fields are shifted to where the 16-bit
// type has them and one packed multiply puts exponent bias and scale right, 5 instructions a
// pair of values (a conversion through f32 is 6, on slower pipes). A block costs its warps 360
// issue slots beside the two softmax warps' 700 on the same scheduler.
//
// Keys split over a cluster: where there are fewer items than SMs, C CTAs take equal shares of
// an item's blocks and merge their f32 states through distributed shared memory: one launch,
// no workspace.
//
// Every mbarrier wait is bounded; a warp that gave up walks on as in attention_tc.cu.
#include <cuda.h>
#include <math.h>
#include <stdio.h>

#include "attention_decode_parts.cuh"
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
using dec_parts::cluster_at;
using dec_parts::ld_cluster_f32;

template <bool Q8, int D>
struct PagedTcCfg {
  static constexpr int kThreads = Q8 ? 512 : 384;
  static constexpr int kStages = 4;
  static constexpr int kRawStages = 4;
  static constexpr int kRawBytes = kBKV * 128;      // one block of e4m3 rows, 128 bytes a key
  static constexpr int kQTile = 128 * D * 2;
  static constexpr int kKv = kBKV * D * 2;
  static constexpr size_t kSmem = 1024 + (size_t)2 * kQTile + (size_t)2 * kStages * kKv + (Q8 ? kRawStages * kRawBytes : 0) +
                                  512;  // the barriers
  static_assert(kSmem <= 232448, "beyond the 227 KiB a CTA may hold");
  static_assert(256 * D * 4 <= 2 * kQTile + kStages * kKv, "a share's output is laid over the tiles of q and k");
  static_assert(2 * 256 * 4 <= kStages * kKv, "and its m and l over those of v");
};

struct PagedTcParams {
  PagedAttnArgs a;
  int group, tile_tokens;  // tokens of a 128-row tile: 128 / group
  int box;
  float scale_log2;
};

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
  float* ml_s = reinterpret_cast<float*>(v_s);  // [2][256]: m and l of a share, once its blocks are done
  uint64_t* bars = reinterpret_cast<uint64_t*>(raw_s + (Q8 ? R * C::kRawBytes : 0));
  uint64_t* q_full = bars;           // [2]
  uint64_t* k_full = bars + 2;       // [S]
  uint64_t* k_empty = k_full + S;
  uint64_t* v_full = k_empty + S;
  uint64_t* v_empty = v_full + S;
  uint64_t* s_full = v_empty + S;    // [2 tiles][2 buffers]
  uint64_t* p_full = s_full + 4;     // [2 tiles][2 buffers]
  uint64_t* tail_done = p_full + 4;  // [2 tiles]: the last two P.V of a tile
  uint64_t* raw_full = tail_done + 2;  // [R]
  uint64_t* raw_empty = raw_full + R;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(raw_empty + R);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  uint32_t rank, csize;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(csize));
  // Later query tiles, heavier under a causal mask, come first for every row and head.
  const int qt = (int)gridDim.y - 1 - (int)blockIdx.y;
  const int pair = blockIdx.x / csize;
  const int b = pair / a.c.kv_heads, hk = pair % a.c.kv_heads;
  const int t0 = qt * 2 * p.tile_tokens;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&tail_done[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);  // one arrival per softmax warp
    }
    for (int i = 0; i < S; ++i) {
      mbar_init(&k_full[i], Q8 ? 4 : 1);  // widening warps, or the loader's copies
      mbar_init(&k_empty[i], 2);          // released by both tiles' issuers
      mbar_init(&v_full[i], Q8 ? 4 : 1);
      mbar_init(&v_empty[i], 2);
    }
    for (int i = 0; i < R; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], 4);
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
  __syncthreads();
  pdl_trigger();
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  const Row row_b = row_of(a.start, a.lens, b, a.t, a.c.width * a.c.page_size);
  if (row_b.bad && threadIdx.x == 0 && qt == 0 && hk == 0 && rank == 0) atomicExch(a.status, (uint32_t)kStatusBadIndex);
  const int64_t end = row_b.start + row_b.n;
  // Keys [first, last) that query token t sees; both grow with t.
  auto first_of = [&](int t) {
    const int64_t x = a.has_window ? row_b.start + t - a.win_left : 0;
    return (int)(x > 0 ? x : 0);
  };
  auto last_of = [&](int t) {
    int64_t x = end;
    if (a.causal && row_b.start + t + 1 < x) x = row_b.start + t + 1;
    if (a.has_window && row_b.start + t + a.win_right + 1 < x) x = row_b.start + t + a.win_right + 1;
    return (int)x;
  };
  // What the live tokens [t, t + tile_tokens) of a tile see: all its keys, and those that every token sees.
  const int n_live = row_b.n;
  const int ta = t0, tb = t0 + p.tile_tokens;
  auto last_token = [&](int t) { return min(t + p.tile_tokens, n_live) - 1; };
  const bool has0 = ta < n_live, has1 = tb < n_live;
  const int lo0 = has0 ? first_of(ta) : 0, hi0 = has0 ? last_of(last_token(ta)) : 0;
  const int lo1 = has1 ? first_of(tb) : lo0, hi1 = has1 ? last_of(last_token(tb)) : hi0;
  const int key_lo = lo0, key_hi = hi1 > hi0 ? hi1 : hi0;  // of the item
  const int blk_lo = key_lo / kBKV, blk_n = key_hi > key_lo ? (key_hi + kBKV - 1) / kBKV - blk_lo : 0;
  // this CTA's share of the item's blocks
  const int per = (blk_n + (int)csize - 1) / (int)csize;
  const int sh_lo = blk_lo + min((int)rank * per, blk_n), sh_hi = min(sh_lo + per, blk_lo + blk_n);
  auto range = [&](bool has, int lo, int hi) {
    Range r{0, 0};
    if (!has || hi <= lo) return r;
    const int x = max(lo / kBKV, sh_lo), y = min((hi + kBKV - 1) / kBKV, sh_hi);
    if (y > x) r.lo = x, r.hi = y;
    return r;
  };
  const Range r0 = range(has0, lo0, hi0), r1 = range(has1, lo1, hi1);
  const bool live0 = r0.hi > r0.lo, live1 = r1.hi > r1.lo;
  int u_lo = 0, u_hi = 0;
  if (live0 && live1) {
    u_lo = r0.lo < r1.lo ? r0.lo : r1.lo;
    u_hi = r0.hi > r1.hi ? r0.hi : r1.hi;
  } else if (live0) {
    u_lo = r0.lo, u_hi = r0.hi;
  } else if (live1) {
    u_lo = r1.lo, u_hi = r1.hi;
  }
  // the first and the last block hold slots beside the item's keys
  const bool ragged_lo = key_lo % kBKV != 0, ragged_hi = key_hi % kBKV != 0;
  const int32_t* table = a.c.table + (int64_t)b * a.c.table_sb;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 0) {
      // ---------------- TMA loader: the lanes issue a block's boxes side by side ----------------
      if (u_hi > u_lo) {
        const int nb = kBKV / p.box;
        constexpr int kCols = Q8 ? 1 : D / 64;
        const int my_box = lane % nb, my_col = lane / nb;
        const bool mine = my_col < kCols;
        if (lane == 0) {
          const uint32_t bytes = (uint32_t)(p.tile_tokens * p.group * 128 * (D / 64));
          for (int i = 0; i < 2; ++i) {
            if (i == 0 ? live0 : live1) {
              mbar_expect_tx(&q_full[i], bytes);
              for (int c = 0; c < D / 64; ++c)
                tma_load_4d(q_s + i * QB + c * (128 * 128), &tmap_q, &q_full[i], c * 64, hk * p.group,
                            t0 + i * p.tile_tokens, b);
            }
          }
        }
        auto look_up = [&](int blk, int& slot) -> int {
          const int j = blk * kBKV + my_box * p.box;
          slot = 0;
          if (!mine || j + p.box <= key_lo || j >= key_hi) return (int)a.c.pages;
          const int page = j / a.c.page_size;
          slot = j - page * a.c.page_size;
          const int id = table[page];
          if (id < 0 || id >= a.c.pages) {
            atomicExch(a.status, (uint32_t)kStatusBadIndex);
            return (int)a.c.pages;
          }
          return id;
        };
        int slot, next_slot;
        int next_id = look_up(u_lo, next_slot);
        bool ok = true;
        auto wait_free = [&](uint64_t* bar, uint32_t parity) {
          bool free = true;
          if (lane == 0) free = mbar_wait(bar, parity, a.status);
          ok = __shfl_sync(0xffffffffu, (int)free, 0) != 0;
          return ok;
        };
        int s = 0;       // ring slot of the next block (16-bit pages), or copy count of the raw ring
        uint32_t ph = 0;
        for (int j = u_lo; j < u_hi; ++j) {
          const int id = next_id;
          slot = next_slot;
          if (j + 1 < u_hi) next_id = look_up(j + 1, next_slot);
          for (int kv = 0; kv < 2; ++kv) {
            const CUtensorMap* map = kv ? &tmap_v : &tmap_k;
            if constexpr (Q8) {
              if (!wait_free(&raw_empty[s], ph ^ 1)) break;
              if (lane == 0) mbar_expect_tx(&raw_full[s], C::kRawBytes);
              __syncwarp();
              if (mine) tma_load_4d(raw_s + s * C::kRawBytes + my_box * p.box * 128, map, &raw_full[s], 0, hk, slot, id);
              if (++s == R) s = 0, ph ^= 1;
            } else {
              uint64_t* full = kv ? v_full : k_full;
              if (!wait_free(kv ? &v_empty[s] : &k_empty[s], ph ^ 1)) break;
              if (lane == 0) mbar_expect_tx(&full[s], KB);
              __syncwarp();
              if (mine)
                tma_load_4d((kv ? v_s : k_s) + s * KB + my_col * KBOX + my_box * p.box * 128, map, &full[s], my_col * 64, hk,
                            slot, id);
            }
          }
          if (!ok) break;
          if (!Q8 && ++s == S) s = 0, ph ^= 1;
        }
        if (!ok)
          for (int i = 0; i < 64; ++i) __nanosleep(1000);  // copies in flight land before the CTA's memory goes
      }
    } else if (warp == 1 || warp == 3) {
      // ---------------- MMA issuers: warp 1 drives tile 0, warp 3 tile 1 (attention_tc.cu) ----------------
      const int i = warp == 1 ? 0 : 1;
      const Range r = i == 0 ? r0 : r1;
      const bool leader = elect_one();
      if (u_hi > u_lo) {
        constexpr uint32_t idesc_qk = umma_idesc(Elem<T>::kUmmaFormat, 128, kBKV, 0, 0);
        constexpr uint32_t idesc_pv = umma_idesc(Elem<T>::kUmmaFormat, 128, D, 0, 1);
        const uint64_t qa = umma_desc_sw128(smem_u32(q_s) + i * QB, 16, 1024);
        const uint64_t k_desc0 = umma_desc_sw128(smem_u32(k_s), 16, 1024);
        const uint64_t v_desc0 = umma_desc_sw128(smem_u32(v_s), KBOX, 1024);
        const int nblk = r.hi - r.lo;
        bool ok = true;
        bool q_ready = false;
        for (int t = u_lo - 1; t <= u_hi && ok; ++t) {
          const int jq = t + 1;  // block whose scores are issued this step
          const int jp = t - 1;  // block whose P.V is issued this step
          const bool have_k = jq >= u_lo && jq < u_hi;
          const bool have_v = jp >= u_lo && jp < u_hi;
          const int ks_slot = have_k ? (jq - u_lo) % S : 0;
          const int vs_slot = have_v ? (jp - u_lo) % S : 0;
          const bool do_pv = have_v && jp >= r.lo && jp < r.hi;
          const bool do_qk = have_k && jq >= r.lo && jq < r.hi;
          // Every slot is waited for and released by both issuers, used or not.
          if ((have_k && !mbar_wait(&k_full[ks_slot], (uint32_t)(((jq - u_lo) / S) & 1), a.status)) ||
              (have_v && !mbar_wait(&v_full[vs_slot], (uint32_t)(((jp - u_lo) / S) & 1), a.status))) {
            ok = false;
            break;
          }
          if (do_pv) {
            const int n = jp - r.lo;  // this tile's block counter
            if (!mbar_wait(&p_full[i * 2 + (n & 1)], (uint32_t)((n >> 1) & 1), a.status)) {
              ok = false;
              break;
            }
            if constexpr (!Q8) {
              // Rows beside the item's keys hold whatever the pages hold there: 0 * NaN must not
              // enter the sum. Both issuers clear them, to the same zeros, before either lets go.
              if ((ragged_lo && jp == blk_lo) || (ragged_hi && jp == blk_lo + blk_n - 1)) {
                for (int x = lane; x < kBKV * (D / 8); x += 32) {
                  const int row = x / (D / 8), c = x % (D / 8), key = jp * kBKV + row;
                  if (key < key_lo || key >= key_hi)
                    *reinterpret_cast<uint4*>(v_s + vs_slot * KB + (c >> 3) * KBOX + row * 128 + (c & 7) * 16) =
                        make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
                __syncwarp();
              }
            }
            tc_fence_after();
            const uint32_t d_tmem = tmem_base + 256 + i * D;
            const uint32_t a_tmem = tmem_base + (uint32_t)((i * 2 + (n & 1)) * kBKV);
            const uint64_t vb = v_desc0 + (uint64_t)((vs_slot * KB) >> 4);
            const uint32_t first = n != 0 ? 1u : 0u;
#pragma unroll
            for (int ks = 0; ks < kBKV / 16; ++ks)  // 16 keys per step = 2 KiB of V, 8 packed P columns
              if (leader)
                umma_ts(d_tmem, a_tmem + ks * 8, vb + (uint64_t)(ks * (2048 >> 4)), idesc_pv,
                        (first | (uint32_t)ks) != 0 ? 1u : 0u);
            if (leader && n + 2 >= nblk) tc_commit(&tail_done[i]);
          }
          if (do_qk) {
            if (!q_ready) {
              if (!mbar_wait(&q_full[i], 0, a.status)) {
                ok = false;
                break;
              }
              q_ready = true;
            }
            tc_fence_after();
            const int n = jq - r.lo;
            const uint32_t d_tmem = tmem_base + (uint32_t)((i * 2 + (n & 1)) * kBKV);
            const uint64_t kb = k_desc0 + (uint64_t)((ks_slot * KB) >> 4);
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
              const uint64_t qoff = (uint64_t)((ks >> 2) * ((128 * 128) >> 4) + (ks & 3) * 2);
              const uint64_t koff = (uint64_t)((ks >> 2) * (KBOX >> 4) + (ks & 3) * 2);
              if (leader) umma_ss(d_tmem, qa + qoff, kb + koff, idesc_qk, ks != 0 ? 1u : 0u);
            }
            if (leader) tc_commit(&s_full[i * 2 + (n & 1)]);
          }
          if (leader && have_v) tc_commit(&v_empty[vs_slot]);
          if (leader && have_k) tc_commit(&k_empty[ks_slot]);
          __syncwarp();
        }
      }
    }
  } else if (Q8 && warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    // ---------------- widening: raw e4m3 blocks into the 16-bit rings ----------------
    if constexpr (Q8) {
      const int tid = threadIdx.x - 384;
      const int r = tid & 63, half = tid >> 6;  // a key of the block, half of its row
      constexpr int kPieces = D / 32;           // 16-byte pieces of half a row
      // my key's scale codes, its page looked up a block ahead
      auto key_page = [&](int j) -> int {
        const int key = j * kBKV + r;
        return j < u_hi && key >= key_lo && key < key_hi ? table[key / a.c.page_size] : -1;
      };
      auto key_codes = [&](int j, int page, uint32_t& kc, uint32_t& vc) {
        kc = vc = 0u;
        if (page >= 0 && page < a.c.pages) {
          const int64_t slot = (j * kBKV + r) % a.c.page_size;
          kc = a.c.k_scale[page * a.c.ks_sp + hk * a.c.ks_sh + slot];
          vc = a.c.v_scale[page * a.c.vs_sp + hk * a.c.vs_sh + slot];
        }
      };
      uint32_t codes[2], next_codes[2];
      key_codes(u_lo, key_page(u_lo), codes[0], codes[1]);
      int page_next = key_page(u_lo + 1);
      int rs = 0;
      uint32_t rph = 0;
      bool ok = true;
      for (int j = u_lo; j < u_hi && ok; ++j) {
        key_codes(j + 1, page_next, next_codes[0], next_codes[1]);
        page_next = key_page(j + 2);
        const int s = (j - u_lo) % S;
        const uint32_t ph = (uint32_t)(((j - u_lo) / S) & 1);
        const int key = j * kBKV + r;
        const bool real = key >= key_lo && key < key_hi;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          if (!mbar_wait(&raw_full[rs], rph, a.status) || !mbar_wait(kv ? &v_empty[s] : &k_empty[s], ph ^ 1, a.status)) {
            ok = false;
            break;
          }
          const uint8_t* src = raw_s + rs * C::kRawBytes + r * 128;
          uint8_t* dst = (kv ? v_s : k_s) + s * KB + r * 128;
          const uint32_t up = widen_factor<T>(codes[kv]);
          const bool plain = up != 0u;
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            const int c = half * kPieces + i;  // 16 columns from 16 c
            const uint4 u = *reinterpret_cast<const uint4*>(src + ((c ^ (r & 7)) << 4));
            const uint32_t in[4] = {u.x, u.y, u.z, u.w};
            uint32_t w[8];
            if (plain) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                w[2 * e] = widen_pair<T>(in[e], 0, up);
                w[2 * e + 1] = widen_pair<T>(in[e], 1, up);
              }
            } else {
              const float scale = scale_value(codes[kv]);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 x = from_e4m3x2(in[e] & 0xffffu), y = from_e4m3x2(in[e] >> 16);
                w[2 * e] = Elem<T>::pack(x.x * scale, x.y * scale);
                w[2 * e + 1] = Elem<T>::pack(y.x * scale, y.y * scale);
              }
            }
            if (!real) {
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] = 0u;
            }
            const int c0 = 2 * c;  // two 16-byte pieces of the 16-bit row
            uint8_t* box = dst + (c0 >> 3) * KBOX;
            *reinterpret_cast<uint4*>(box + (((c0 & 7) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4*>(box + ((((c0 & 7) + 1) ^ (r & 7)) << 4)) = make_uint4(w[4], w[5], w[6], w[7]);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(kv ? &v_full[s] : &k_full[s]);
            mbar_arrive(&raw_empty[rs]);
          }
          if (++rs == R) rs = 0, rph ^= 1;
        }
        codes[0] = next_codes[0], codes[1] = next_codes[1];
      }
    }
  } else {
    if constexpr (Q8) asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ---------------- softmax + epilogue (attention_tc.cu) ----------------
    const int i = (warp - 4) >> 2;  // query tile
    const int quarter = warp & 3;   // TMEM lane quarter
    const Range r = i == 0 ? r0 : r1;
    const int tile_row = quarter * 32 + lane;
    const int t_first = t0 + i * p.tile_tokens;
    const int t_row = t_first + tile_row / p.group;
    const int head = hk * p.group + tile_row % p.group;
    const bool row_ok = tile_row < p.tile_tokens * p.group && t_row < a.t;  // a row of the output
    const bool row_real = row_ok && t_row < n_live;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const uint32_t o_tmem = tmem_base + 256 + i * D + lane_addr;
    const float sl2 = p.scale_log2;
    const int vis_lo = row_real ? first_of(t_row) : 0, vis_hi = row_real ? last_of(t_row) : 0;
    // keys that every live token of the tile sees
    const bool has = i == 0 ? has0 : has1;
    const int all_lo = has ? first_of(last_token(t_first)) : 0, all_hi = has ? last_of(t_first) : 0;
    auto vis_word = [&](int base) -> uint32_t {
      int x = vis_lo - base, y = vis_hi - base;
      x = x < 0 ? 0 : x;
      y = y > 32 ? 32 : y;
      uint32_t w = 0;
      if (y > x) w = (y == 32 ? 0xffffffffu : ((1u << y) - 1u)) & ~((1u << x) - 1u);
      return w;
    };
    float m_run = -INFINITY;  // running maximum, scaled log2 units
    float l_run = 0.f;
    bool ok = true;
    const int nblk = r.hi - r.lo;
    // turns on the MUFU unit, as in attention_tc.cu
    const int n_paired = paired_blocks(r0, r1);
    const int my_turn = 1 + i * 4 + quarter;
    const int other_turn = 1 + (1 - i) * 4 + quarter;
    int turns_done = 0;
    uint32_t sr[2][32];
    bool requested = false;
    for (int j = r.lo; j < r.hi; ++j) {
      const int n = j - r.lo;
      const int buf = n & 1;
      turns_done = n;
      const uint32_t s_tmem = tmem_base + (uint32_t)((i * 2 + buf) * kBKV) + lane_addr;
      if (!requested) {
        if (!mbar_wait(&s_full[i * 2 + buf], (uint32_t)((n >> 1) & 1), a.status)) {
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
        const bool landed = n + 1 < nblk
                                ? mbar_wait(&s_full[i * 2 + ((n + 1) & 1)], (uint32_t)(((n + 1) >> 1) & 1), a.status)
                                : mbar_wait(&tail_done[i], 0, a.status);
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
      if (n < n_paired && (i == 1 || n > 0)) {
        named_barrier(my_turn, 64);
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
      if (n < n_paired && (i == 0 || n + 1 < n_paired)) named_barrier_arrive(other_turn, 64);
      turns_done = n + 1;
      l_run += (la.x + la.y) + (lb.x + lb.y);
      requested = false;
      if (n + 1 < nblk && mbar_test_wait(&s_full[i * 2 + (buf ^ 1)], (uint32_t)(((n + 1) >> 1) & 1))) {
        tc_fence_after();
        const uint32_t next_tmem = tmem_base + (uint32_t)((i * 2 + (buf ^ 1)) * kBKV) + lane_addr;
        tmem_ld32(next_tmem, sr[0]);
        tmem_ld32(next_tmem + 32, sr[1]);
        requested = true;
      }
      tmem_st_wait();
      if (n + 1 == nblk && nblk >= 2 && !tail0_seen && !mbar_wait(&tail_done[i], 0, a.status)) {
        ok = false;
        break;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[i * 2 + buf]);
    }
    if (!ok) {
      for (int m = turns_done; m < n_paired; ++m)
        if (i == 0 || m + 1 < n_paired) named_barrier_arrive(other_turn, 64);
    }
    // the last P.V: the tail barrier's second phase (its only one for a one-block tile)
    if (r.hi > r.lo && ok) ok = mbar_wait(&tail_done[i], nblk >= 2 ? 1u : 0u, a.status);
    tc_fence_after();
    if (csize == 1) {
      // ---- epilogue: O / l; zeros where no key reaches a row ----
      if (!row_real) l_run = 0.f;
      const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;
      T* orow = (T*)a.o + (int64_t)b * a.o_sb + (int64_t)t_row * a.o_st + (int64_t)head * a.o_sh;
      const bool any = r.hi > r.lo;
      if (ok) {
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t orr[32];
          if (any) {
            tmem_ld32(o_tmem + c, orr);
            tmem_ld_wait();
          }
          if (row_ok) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              if (c + v * 8 >= a.c.d) break;  // padded head dim: nothing past the real columns
              uint32_t w[4] = {0u, 0u, 0u, 0u};
              if (any && l_run != 0.f) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  w[e] = Elem<T>::pack(__uint_as_float(orr[v * 8 + 2 * e]) * inv, __uint_as_float(orr[v * 8 + 2 * e + 1]) * inv);
              }
              stg128(orow + c + v * 8, make_uint4(w[0], w[1], w[2], w[3]));
            }
          }
        }
      }
      if (a.lse != nullptr && row_ok && ok)
        a.lse[((int64_t)b * a.heads + head) * a.t + t_row] = l_run == 0.f ? -INFINITY : kLn2F * (m_run + log2f(l_run));
    } else {
      // ---- this share's state into shared memory, [column][row]: every MMA of both tiles is done ----
      named_barrier(9, 256);
      float* op = reinterpret_cast<float*>(smem);
      const int row = i * 128 + tile_row;
      if (r.hi > r.lo) {
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t orr[32];
          tmem_ld32(o_tmem + c, orr);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) op[(c + e) * 256 + row] = __uint_as_float(orr[e]);
        }
      }
      ml_s[row] = m_run;
      ml_s[256 + row] = r.hi > r.lo ? l_run : 0.f;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
  if (csize > 1) {
    cluster_sync_all();
    if (warp >= 4 && warp < 12) {
      const int tid = threadIdx.x - 128;
      const uint32_t op_addr = smem_u32(smem), ml_addr = smem_u32(ml_s);
      // a thread: eight columns of a row; a warp 32 rows, so that its reads are whole lines
      for (int w = (int)rank * 256 + tid; w < 256 * (a.c.d / 8); w += (int)csize * 256) {
        const int row = w & 255, d0 = (w >> 8) * 8;
        const int in_tile = row & 127;
        const int t_row = t0 + (row >> 7) * p.tile_tokens + in_tile / p.group;
        const int head = hk * p.group + in_tile % p.group;
        if (in_tile >= p.tile_tokens * p.group || t_row >= a.t) continue;
        float m = -INFINITY, l = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (t_row < n_live) {
          for (uint32_t k = 0; k < csize; ++k) m = fmaxf(m, ld_cluster_f32(cluster_at(ml_addr + row * 4, k)));
          for (uint32_t k = 0; k < csize; ++k) {
            const float mr = ld_cluster_f32(cluster_at(ml_addr + row * 4, k));
            const float lr = ld_cluster_f32(cluster_at(ml_addr + (256 + row) * 4, k));
            if (lr == 0.f) continue;  // the share saw no key of this row
            const float f = mr == -INFINITY ? 1.f : ex2_approx(mr - m);
            l = fmaf(f, lr, l);
            const uint32_t src = cluster_at(op_addr + (uint32_t)(d0 * 256 + row) * 4, k);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = fmaf(f, ld_cluster_f32(src + e * 1024), acc[e]);
          }
        }
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        stg128((T*)a.o + (int64_t)b * a.o_sb + (int64_t)t_row * a.o_st + (int64_t)head * a.o_sh + d0,
               make_uint4(Elem<T>::pack(acc[0] * inv, acc[1] * inv), Elem<T>::pack(acc[2] * inv, acc[3] * inv),
                          Elem<T>::pack(acc[4] * inv, acc[5] * inv), Elem<T>::pack(acc[6] * inv, acc[7] * inv)));
        if (a.lse != nullptr && d0 == 0)
          a.lse[((int64_t)b * a.heads + head) * a.t + t_row] = l == 0.f ? -INFINITY : kLn2F * (m + log2f(l));
      }
    }
    cluster_sync_all();  // no CTA leaves while a peer still reads its state
  }
}

int sm_count_paged() {
  static int n = 0;
  if (n == 0) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (n <= 0) n = 148;
  }
  return n;
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
  const int64_t n_qt = (a.t + 2 * p.tile_tokens - 1) / (2 * p.tile_tokens);
  const int64_t pairs = a.batch * a.c.kv_heads, items = pairs * n_qt;
  int64_t keys = a.c.width * a.c.page_size;
  if (a.has_window) {
    const int64_t w = a.win_left + 2 * p.tile_tokens + (a.causal ? 0 : a.win_right) + kBKV;
    keys = w < keys ? w : keys;
  }
  const int64_t blocks = (keys + kBKV - 1) / kBKV;
  int csize = 1;
  while (csize < 8 && items * csize * 2 <= sm_count_paged() && blocks >= 4 * csize * 2) csize *= 2;
  if (launch_pdl(attention_paged_tc_kernel<T, Q8, D>, dim3((unsigned)(pairs * csize), (unsigned)n_qt), dim3(C::kThreads),
                 C::kSmem, s, (unsigned)csize, a.batch * a.t, tq, tk, tv, p) != cudaSuccess)
    return -1;
  snprintf(cfg, cfg_len, "{bq:%d,bkv:%d,d:%d,box:%d,cluster:%d%s}", 2 * kBQ, kBKV, a.c.d, p.box, csize, Q8 ? ",e4m3" : "");
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
  if (group > 128 || a.batch * a.c.kv_heads > (1 << 26) || a.t > 0x7fffff00LL) return false;
  // the query rows come by a tensor map, which has no stride of zero (an expanded view)
  if ((a.heads > 1 && a.q_sh == 0) || (a.t > 1 && a.q_st == 0) || (a.batch > 1 && a.q_sb == 0)) return false;
  const int64_t tokens = 2 * (128 / group);
  return (a.t + tokens - 1) / tokens <= 65535;
}

int launch_attention_paged_tc(const PagedAttnArgs& a, cudaStream_t s, char* cfg, size_t cfg_len) {
  return a.dtype == SVODB_BF16 ? run_type<__nv_bfloat16>(a, s, cfg, cfg_len) : run_type<__half>(a, s, cfg, cfg_len);
}

}  // namespace svodb
