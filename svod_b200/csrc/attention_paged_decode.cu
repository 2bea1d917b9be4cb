// Attention of few query rows (a token, a handful of drafted ones) over a paged cache: the
// keys and values of a KV head are read once from HBM for all the query rows that share it.
//
// What bounds it: the cache's bytes. The layout is attention_decode.cu's: keys are the M of
// both contractions, so a block of 128 keys costs two small MMAs whatever the number of rows,
//     S^T [128 keys x 16]  = K [128 x D] . Q^T            O^T [D x 16] += V^T [D x 128] . P^T
// a softmax thread owns one key, a cluster of C CTAs takes one (row, KV head) and merges its
// C partial states through distributed shared memory: one launch, no workspace.
//
// Pages: a block of 128 keys is 128 / box boxes of box = gcd(page_size, 128) keys, none of
// which straddles two pages; the lanes of the loader warp look up their boxes' pages a block
// ahead and issue the copies side by side. Boxes outside the keys that any query row sees are
// fetched past the last page, where a copy reads zeros: their table entries are not looked at.
//
// 8-bit pages go into the MMAs as they are (kind::f8f6f4): nothing widens them. The other
// operand is split into 8-bit pieces instead, which cost M = 128 MMAs of 16 columns more and
// no bytes of the cache: a query row, scaled to 448 by a power of two, is the exact sum of two
// (bf16) or three (f16) e4m3 values, down to 2^-18 of its largest. A weight w <= 4, times its
// key's V scale over the CTA's largest, is one e4m3 value (4 bits) and three (f16: four) e5m2
// remainders (3 bits each) at 2^17 times their size, in an accumulator of their own: within
// 2^-9 (f16: 2^-12) of a weight too small for the first, 2^-13 (2^-16) of a larger one, and
// within 2^-34 of any. Scales are powers of two: K's multiply the scores, V's the weights,
// and neither rounds.
//
// CTA roles (192 threads), barriers and the ring are attention_decode.cu's: warps 0-3 softmax,
// warp 4 TMA loader, warp 5 MMA issuer. Every mbarrier wait is bounded.
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
using namespace dec_parts;
using namespace paged;

// Pieces of a query row and of a weight in 8 bits.
template <typename T>
constexpr int kQueryPieces = std::is_same<T, __half>::value ? 3 : 2;
template <typename T>
constexpr int kWeightPieces = std::is_same<T, __half>::value ? 5 : 4;
constexpr float kRemainderUp = 131072.f;  // 2^17: the remainder of a weight of 4 is at most 2^-2, and e5m2 ends at 57344
// A row adopts a new maximum when it grew by more than this, in log2 units. With 8-bit pieces
// what a weight may grow to is taken from what small ones keep.
template <bool Q8>
constexpr float kAdoptAbove = Q8 ? 2.f : kRescaleAbove;

constexpr int kRows = 16;  // query rows of a KV head: the N of both MMAs

template <typename T, bool Q8, int D>
struct PagedDecCfg {
  static_assert(!Q8 || D == 128, "8-bit rows are a 128-byte tile, zero-filled behind the head");
  static constexpr int kBoxes = Q8 ? 1 : D / 64;  // 128-byte boxes of a row
  static constexpr int kSlotBytes = kKeys * 128 * kBoxes;
  static constexpr int kSlots = 3;
  static constexpr int kPerSm = !Q8 && D == 128 ? 2 : 3;
  static constexpr int kRing = kSlots * kSlotBytes;
  static constexpr int kQBytes = Q8 ? kQueryPieces<T> * kRows * 128 : kRows * D * 2;
  static constexpr int kPBytes = Q8 ? kWeightPieces<T> * kRows * 128 : 2 * 2 * kRows * 128;
  // A second buffer of weights lets a block's exponentials run under the previous block's P.V.
  static constexpr int kPBufs = D == 128 && (!Q8 || kWeightPieces<T> > 4) ? 1 : 2;
  static constexpr int kRedBytes = kRows * 4 * 4;
  static constexpr int kTail = kQBytes + kPBufs * kPBytes + kRedBytes + 7 * kRows * 4 + 32 + 256;
  static constexpr size_t kSmem = 1024 + (size_t)kRing + (kTail > kBox ? kTail : kBox);
  static constexpr int kTmemCols = 4 * kRows;
  static_assert(kPerSm * (kSmem + 1024) <= 233472, "the CTAs of an SM fit its shared memory");
  static_assert(kPBufs * kPBytes >= 2 * 1024, "the order of the rows is found over the weights");
  static_assert(kRows * D * 4 <= kRing, "the partial outputs are laid over the ring");
};

// Rows of a batch that are taken in order, longest first, so that short rows fill the places
// that long ones leave: a class of length a byte for each has to fit the smallest weights'
// buffer beside the classes' counts. The order pays where the CTAs are a few times what the chip
// holds at once; beyond that its places fill themselves, and every wave of CTAs pays the 1 to
// 2.5 us of the order. In order | as they lie, 8 KV heads, us: 64..4095 keys in bf16, 64 rows
// (1.7 times) 90 | 126, 112 rows (3.0) 156 | 174, 160 rows (4.3) 220 | 230; in e4m3 64 rows (1.2)
// 57 | 68, 128 rows (2.3) 104 | 111, 192 rows (3.5) 155 | 155, 256 rows (4.6) 204 | 192;
// 64..16000 keys, 80 rows in bf16 (2.2) 384 | 505, 120 in e4m3 (2.2) 300 | 378; 100..1000 keys in
// bf16, 64 rows 37.5 | 41.1, 96 rows (2.6) 54.7 | 55.6, 128 rows (3.5) 71 | 67, 512 rows (14) 264 |
// 220, 1024 rows (28) 543 | 428; in e4m3 128 rows 48 | 46; 64 rows of 4095 each 167 | 164.
constexpr int kOrderedWaves = 3;
constexpr int kSortedRows = 1024;
constexpr int kClasses = 256;

struct PagedDecParams {
  PagedAttnArgs a;
  int group, rows;  // rows = t * group query rows per KV head
  int box;          // keys of a box
  Divider page_size;
  int longest_first;  // rows in the order of their visible keys (kOrderedWaves)
  float scale_log2;
};

// Keys [lo, hi) that query token t of a row sees; both ends grow with t.
__device__ __forceinline__ int first_seen(const PagedAttnArgs& a, const Row& r, int t) {
  const int64_t x = a.has_window ? r.start + t - a.win_left : 0;
  return (int)(x > 0 ? x : 0);
}
__device__ __forceinline__ int last_seen(const PagedAttnArgs& a, const Row& r, int t) {
  int64_t x = r.start + r.n;
  if (a.causal && r.start + t + 1 < x) x = r.start + t + 1;
  if (a.has_window && r.start + t + a.win_right + 1 < x) x = r.start + t + a.win_right + 1;
  return (int)x;
}

// A row's visible keys in blocks of `unit`; and the class of a number of blocks, 0 to 254: itself
// where they are few, from 16 on to four bits behind the first, so rows of one class differ by a
// sixteenth at most.
__device__ __forceinline__ int row_keys(const PagedAttnArgs& a, int64_t b, int64_t capacity, int unit) {
  const Row r = row_of(a.start, a.lens, b, a.t, capacity);
  if (r.n <= 0) return 0;
  const int n = (last_seen(a, r, r.n - 1) + unit - 1) / unit - first_seen(a, r, 0) / unit;
  return n < 0 ? 0 : n;
}
__device__ __forceinline__ int length_class(int blocks) {
  return blocks < 16 ? blocks : min((int)(__float_as_uint((float)blocks) >> 19) - (131 << 4) + 16, kClasses - 2);
}

// The row that comes `at`-th when the batch is put in order, longest first and rows of one length
// (or class) as they lie: the chip takes the long rows first, the short ones fill its last places.
// Up to kRankedRows rows are compared with each other. More would take work that grows with the
// square of the batch in each of its CTAs (1024 rows of 100..1000 keys x 8 KV heads: 3317 us, 543
// by classes); by classes it is in proportion: every row's class is counted, every warp finds from
// the counts which class holds the place and from the classes which of its rows that is. By
// comparison | by classes, 8 KV heads, us: 16 rows of 8000..32767 keys in e4m3 118.8 | 120.4, 64
// of 64..4095 56.9 | 57.6, 128 of them 104.9 | 104.0; 96 in bf16 137.8 | 137.2; 300 rows of
// 16..200 x 2 KV heads 45 | 29. `mem` (2 KB) is free again when the call returns.
constexpr int kRankedRows = 64;
__device__ __forceinline__ int longest_first_row(const PagedAttnArgs& a, int at, int64_t capacity, uint8_t* mem) {
  const int tid = threadIdx.x, lane = tid & 31, batch = (int)a.batch;
  if (batch <= kRankedRows) {
    int* keys = reinterpret_cast<int*>(mem);  // [padded], then the row
    const int padded = (batch + 3) & ~3;
    if (tid < padded) keys[tid] = tid < batch ? row_keys(a, tid, capacity, 1) : -1;
    __syncthreads();
    if (tid < batch) {
      const int mine = keys[tid];
      int rank = 0;
      for (int o = 0; o < padded; o += 4) {
        const int4 n = *reinterpret_cast<const int4*>(keys + o);
        rank += (n.x > mine || (n.x == mine && o < tid)) + (n.y > mine || (n.y == mine && o + 1 < tid)) +
                (n.z > mine || (n.z == mine && o + 2 < tid)) + (n.w > mine || (n.w == mine && o + 3 < tid));
      }
      if (rank == at) keys[padded] = tid;
    }
    __syncthreads();
    const int row = keys[padded];
    __syncthreads();  // before anything is written over it
    return row;
  }
  int* counts = reinterpret_cast<int*>(mem);  // [kClasses]
  uint8_t* classes = mem + kClasses * 4;      // [32 lanes][per]
  const int per = (batch + 127) / 128 * 4;    // rows that a lane looks through
  for (int k = tid; k < kClasses; k += kThreadsDec) counts[k] = 0;
  __syncthreads();
  for (int k = tid; k < 32 * per; k += kThreadsDec) {
    int c = kClasses - 1;  // no row's
    if (k < batch) {
      c = length_class(row_keys(a, k, capacity, kKeys));
      atomicAdd(&counts[c], 1);
    }
    classes[k] = (uint8_t)c;
  }
  __syncthreads();
  // lane l has the classes 255 - 8 l down to 248 - 8 l
  int mine[8], sum = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) mine[e] = counts[kClasses - 1 - 8 * lane - e], sum += mine[e];
  int upto = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  int left = at - (upto - sum), cls = 0;  // rows of my classes before the place
  bool here = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (here) continue;
    if (left >= 0 && left < mine[e]) here = true, cls = kClasses - 1 - 8 * lane - e;
    else left -= mine[e];
  }
  const int who = __ffs((int)__ballot_sync(0xffffffffu, here)) - 1;
  cls = __shfl_sync(0xffffffffu, cls, who), left = __shfl_sync(0xffffffffu, left, who);
  // the row that has `left` of its class before it
  const uint32_t* words = reinterpret_cast<const uint32_t*>(classes + lane * per);
  const uint32_t want = (uint32_t)cls * 0x01010101u;
  int found = 0;
  for (int w = 0; w < per / 4; ++w) found += __popc(__vcmpeq4(words[w], want)) >> 3;
  upto = found;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  left -= upto - found;
  here = left >= 0 && left < found;
  int row = 0;
  if (here) {
    for (row = lane * per;; ++row)
      if (classes[row] == cls && left-- == 0) break;
  }
  const int owner = __ffs((int)__ballot_sync(0xffffffffu, here)) - 1;
  row = __shfl_sync(0xffffffffu, row, owner);
  __syncthreads();  // before anything is written over the counts
  return row;
}

__device__ __forceinline__ uint32_t to_e5m2x2(float lo, float hi) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E5M2);
}
__device__ __forceinline__ float2 from_e5m2x2(uint32_t u) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)u, __NV_E5M2);
  return __half22float2(__half2(h));
}

// 2^e, e <= 0; zero where that is no normal number.
__device__ __forceinline__ float power_below(int e) { return e < -126 ? 0.f : __uint_as_float((uint32_t)(127 + e) << 23); }

// D[tmem] (+)= A[smem] . B[smem] over 8-bit operands.
__device__ __forceinline__ void umma_ss_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor of kind::f8f6f4 with an f32 accumulator: as kind::f16's, formats
// 0 = e4m3, 1 = e5m2, each operand its own.
__host__ __device__ constexpr uint32_t umma_idesc_f8(int a_fmt, int b_fmt, int m, int n, int a_mn_major) {
  return (1u << 4) | (uint32_t(a_fmt) << 7) | (uint32_t(b_fmt) << 10) | (uint32_t(a_mn_major) << 15) |
         (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

// W columns of 32-bit accumulators, in registers when the call returns.
template <int W>
__device__ __forceinline__ void tmem_ld_w(uint32_t at, uint32_t (&r)[W]) {
  if constexpr (W == 4) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
  } else if constexpr (W == 8) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(at)
                 : "memory");
  } else {
    tmem_ld16(at, r);
  }
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < W; ++i) asm volatile("" : "+r"(r[i]));  // no use moves above the wait
}
template <int W>
__device__ __forceinline__ void tmem_st_w(uint32_t at, const uint32_t (&r)[W]) {
  if constexpr (W == 4) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3])
                 : "memory");
  } else if constexpr (W == 8) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  } else {
    tmem_st16(at, r);
  }
}

// W: the columns (query rows) that softmax threads keep in registers, the least of 4, 8 and 16
// that holds them (a register each for scores and sums, and three CTAs an SM leave 96; 16 rows
// x 8000..32767 e4m3 keys, two query rows a KV head: 145 us with 16 columns, 118 with 4).
template <typename T, bool Q8, int D, int W>
__global__ void __launch_bounds__(kThreadsDec, (PagedDecCfg<T, Q8, D>::kPerSm))
    attention_paged_decode_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                                  const __grid_constant__ PagedDecParams p) {
  using C = PagedDecCfg<T, Q8, D>;
  constexpr int S = C::kSlots;
  constexpr int QP = kQueryPieces<T>, WP = kWeightPieces<T>;
  const PagedAttnArgs& a = p.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = ring + C::kRing;
  uint8_t* p_s = q_s + C::kQBytes;
  float* red = reinterpret_cast<float*>(p_s + C::kPBufs * C::kPBytes);  // [kRows][4 warps]
  float* mc = red + kRows * 4;                                       // [2][kRows]: the maximum in use, the rescale factor
  float* ml = mc + 2 * kRows;                                        // [2][kRows]: this CTA's m (as it runs) and l
  float* fc = ml + 2 * kRows;                                        // [kRows]: log2 units a raw score
  int* lim = reinterpret_cast<int*>(fc + kRows);                     // [2][kRows]: a column's keys [lo, hi)
  int* vred = lim + 2 * kRows;                                       // [4] (8 words kept): per-warp largest V scale code
  uint64_t* bars = reinterpret_cast<uint64_t*>(vred + 8);
  uint64_t* full = bars;
  uint64_t* empty = full + S;
  uint64_t* s_full = empty + S;   // [2]
  uint64_t* p_full = s_full + 2;  // [2]
  uint64_t* pv_done = p_full + 2; // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pv_done + 2);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 128) {
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  uint32_t rank, csize;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(csize));
  const int pair = blockIdx.x / csize, hk = pair % a.c.kv_heads;
  int b = pair / a.c.kv_heads;

  pdl_wait();
  const int64_t capacity = a.c.width * a.c.page_size;
  if (p.longest_first) b = longest_first_row(a, b, capacity, p_s);
  const Row r = row_of(a.start, a.lens, b, a.t, capacity);
  if (r.bad && tid == 0 && rank == 0 && hk == 0) report_bad_index(a.bad_index);
  auto first_of = [&](int t) { return first_seen(a, r, t); };
  auto last_of = [&](int t) { return last_seen(a, r, t); };
  const int lo = r.n > 0 ? first_of(0) : 0, hi = r.n > 0 ? last_of(r.n - 1) : 0;
  // keys that every live query token sees
  const int all_lo = r.n > 0 ? first_of(r.n - 1) : 0, all_hi = r.n > 0 ? last_of(0) : 0;
  const int blk0 = lo / kKeys;
  const int total = hi > lo ? (hi + kKeys - 1) / kKeys - blk0 : 0;
  const int per = (total + (int)csize - 1) / (int)csize;
  const int g_lo = blk0 + min((int)rank * per, total);
  const int n = min(per, blk0 + total - g_lo);  // blocks of this CTA (0: an empty share)
  const int32_t* table = a.c.table + (int64_t)b * a.c.table_sb;

  // ---- loader: copies in the ring's order, a warp's lanes side by side ----
  const int nb = kKeys / p.box;  // boxes a block and 128-byte column
  const int my_box = lane % nb, my_col = lane / nb;
  const bool mine = my_col < C::kBoxes;
  int id0 = 0, slot0 = 0;  // my box's page and slot in the block of keys loaded last,
  int id1 = 0, slot1 = 0;  // and in the one before (its V follows)
  int slot_in_page = 0;
  bool ok = true;
  int at = 0;  // copies issued so far, in the ring's order
  auto look_up = [&](int g) -> int {
    // positions [j, j + box) of one page; outside [lo, hi) nothing is looked at
    const int j = g * kKeys + my_box * p.box;
    slot_in_page = 0;
    if (!mine || j + p.box <= lo || j >= hi) return (int)a.c.pages;
    const uint32_t page = p.page_size.div((uint32_t)j);
    slot_in_page = j - (int)(page * p.page_size.d);
    const int id = table[page];
    if (id < 0 || id >= a.c.pages) {
      report_bad_index(a.bad_index);
      return (int)a.c.pages;
    }
    return id;
  };
  int next_id = 0, next_slot = 0;  // of the next block of keys
  auto load = [&]() {
    const int s = at % S;
    const bool is_v = at == 2 * n - 1 || (at > 0 && (at & 1) == 0);
    if (at >= S) {
      bool free = true;
      if (lane == 0) free = mbar_wait(&empty[s], (at / S - 1) & 1, a.status);
      ok = __shfl_sync(0xffffffffu, (int)free, 0) != 0;
      if (!ok) return;
    }
    if (lane == 0) mbar_expect_tx(&full[s], C::kSlotBytes);
    int id, slot;
    if (is_v) {
      // V(j) follows K(j + 1), the last V its own K
      const bool last = at == 2 * n - 1;
      id = last ? id0 : id1, slot = last ? slot0 : slot1;
    } else {
      id1 = id0, slot1 = slot0;
      id = id0 = next_id, slot = slot0 = next_slot;
    }
    __syncwarp();
    if (mine)
      tma_load_4d(ring + s * C::kSlotBytes + my_col * kBox + my_box * p.box * 128, is_v ? &tmap_v : &tmap_k, &full[s],
                  my_col * 64, hk, slot, id);
    ++at;
    if (!is_v) {
      const int g = g_lo + (at == 1 ? 1 : at / 2 + 1);  // K(j) was copy 2j - 1 (0 for j = 0)
      if (g < g_lo + n) next_id = look_up(g), next_slot = slot_in_page;
    }
  };
  if (warp == 4) {
    if (n > 0) next_id = look_up(g_lo), next_slot = slot_in_page;
    if (lane == 0) {
      for (int i = 0; i < S; ++i) {
        mbar_init(&full[i], 1);
        mbar_init(&empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_full[i], 1);
        mbar_init(&p_full[i], 4);
        mbar_init(&pv_done[i], 1);
      }
      mbar_fence_init();
    }
    __syncwarp();
    while (ok && at < 2 * n && at < S) load();
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  // Query rows (zero past `rows`, past the chunk's real tokens and past the head's width) and
  // zeroed weights: the columns of dead rows stay zero throughout.
  if (tid < 128) {
    const T* qb = (const T*)a.q + (int64_t)b * a.q_sb;
    auto query = [&](int row, int col) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (row < p.rows && row / p.group < r.n && col < a.c.d)
        u = ldg128(qb + (int64_t)(row / p.group) * a.q_st + (int64_t)(hk * p.group + row % p.group) * a.q_sh + col);
      return u;
    };
    if constexpr (!Q8) {
      for (int i = tid; i < kRows * (D / 8); i += 128) {
        const int row = i / (D / 8), c = i % (D / 8);
        *reinterpret_cast<uint4*>(q_s + (c >> 3) * (kRows * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = query(row, c * 8);
      }
    } else {
      for (int i = tid; i < kRows * 16; i += 128) {  // 16 lanes a row, 8 values each
        const int row = i >> 4, c = i & 15;
        const uint4 u = query(row, c * 8);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        float f[8];
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x = Elem<T>::unpack(w[e]);
          f[2 * e] = x.x, f[2 * e + 1] = x.y;
          top = max(top, max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu));
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const uint32_t code = scale_code(__uint_as_float(top));  // NaN and infinity: every score of the row is NaN
        const float inv = code == 255u ? 0.f : scale_inverse(code);
        if (c == 0) {
          // a factor too small for 32 bits is their least one: zero would make NaN of hidden scores
          const float f = p.scale_log2 * scale_value(code);
          fc[row] = f == 0.f ? __uint_as_float(1u) : f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = code == 255u ? 0.f : f[e] * inv;
#pragma unroll
        for (int k = 0; k < QP; ++k) {
          uint32_t piece[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            piece[e] = to_e4m3x2(f[2 * e], f[2 * e + 1]);
            const float2 x = from_e4m3x2(piece[e]);
            f[2 * e] -= x.x, f[2 * e + 1] -= x.y;
          }
          *reinterpret_cast<uint2*>(q_s + k * (kRows * 128) + row * 128 + (((c >> 1) ^ (row & 7)) << 4) + (c & 1) * 8) =
              make_uint2(piece[0] | (piece[1] << 16), piece[2] | (piece[3] << 16));
        }
      }
    }
    for (int i = tid; i < C::kPBufs * C::kPBytes / 16; i += 128) reinterpret_cast<uint4*>(p_s)[i] = make_uint4(0, 0, 0, 0);
    if (tid < kRows) {
      const int t = tid / p.group;
      const bool live = tid < p.rows && t < r.n;
      lim[tid] = live ? first_of(t) : 0;
      lim[kRows + tid] = live ? last_of(t) : 0;
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 4) {
    // the rest of the ring's copies
    while (ok && at < 2 * n) load();
    if (!ok)
      for (int i = 0; i < 64; ++i) __nanosleep(1000);  // copies in flight land before the CTA's memory goes
  } else if (warp == 5) {
    // ---------------- MMA issuer ----------------
    const bool leader = elect_one();
    const uint64_t k_desc = umma_desc_sw128(smem_u32(ring), 16, 1024);
    const uint64_t v_desc = umma_desc_sw128(smem_u32(ring), kBox, 1024);
    const uint64_t q_desc = umma_desc_sw128(smem_u32(q_s), 16, 1024);
    const uint64_t p_desc = umma_desc_sw128(smem_u32(p_s), 16, 1024);
    bool ok = true;
    auto scores = [&](int j) {
      const uint32_t pos = pos_k(j);
      const int s = (int)(pos % S);
      if (!mbar_wait(&full[s], (pos / S) & 1, a.status)) {
        ok = false;
        return;
      }
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + (uint32_t)((j & 1) * kRows);
      if constexpr (!Q8) {
        constexpr uint32_t idesc = umma_idesc(Elem<T>::kUmmaFormat, 128, kRows, 0, 0);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          if (leader)
            umma_ss(d_tmem, k_desc + (uint64_t)((s * C::kSlotBytes + (ks >> 2) * kBox) >> 4) + (uint64_t)((ks & 3) * 2),
                    q_desc + (uint64_t)(((ks >> 2) * (kRows * 128)) >> 4) + (uint64_t)((ks & 3) * 2), idesc, ks != 0 ? 1u : 0u);
      } else {
        constexpr uint32_t idesc = umma_idesc_f8(0, 0, 128, kRows, 0);
#pragma unroll
        for (int k = 0; k < QP; ++k)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)  // 32 columns = 32 bytes a step
            if (leader)
              umma_ss_f8(d_tmem, k_desc + (uint64_t)((s * C::kSlotBytes) >> 4) + (uint64_t)(ks * 2),
                         q_desc + (uint64_t)((k * kRows * 128) >> 4) + (uint64_t)(ks * 2), idesc, (k | ks) != 0 ? 1u : 0u);
      }
      if (leader) {
        tc_commit(&empty[s]);
        tc_commit(&s_full[j & 1]);
      }
    };
    if (n > 0) scores(0);
    for (int j = 0; j < n && ok; ++j) {
      if (j + 1 < n) scores(j + 1);
      if (!ok || !mbar_wait(&p_full[j & 1], (j >> 1) & 1, a.status)) break;
      const uint32_t pos = pos_v(j, n);
      const int s = (int)(pos % S);
      if (!mbar_wait(&full[s], (pos / S) & 1, a.status)) break;
      tc_fence_after();
      const uint64_t vb = v_desc + (uint64_t)((s * C::kSlotBytes) >> 4);
      const uint64_t pb = p_desc + (uint64_t)(((j % C::kPBufs) * C::kPBytes) >> 4);
      if constexpr (!Q8) {
        constexpr uint32_t idesc = umma_idesc(Elem<T>::kUmmaFormat, 128, 2 * kRows, 1, 0);
#pragma unroll
        for (int ks = 0; ks < kKeys / 16; ++ks)
          if (leader)
            umma_ss(tmem_base + 2 * kRows, vb + (uint64_t)(ks * (2048 >> 4)),
                    pb + (uint64_t)(((ks >> 2) * (2 * kRows * 128)) >> 4) + (uint64_t)((ks & 3) * 2), idesc,
                    (j | ks) != 0 ? 1u : 0u);
      } else {
#pragma unroll
        for (int k = 0; k < WP; ++k) {
          const uint32_t idesc = k == 0 ? umma_idesc_f8(0, 0, 128, kRows, 1) : umma_idesc_f8(0, 1, 128, kRows, 1);
#pragma unroll
          for (int ks = 0; ks < kKeys / 32; ++ks)  // 32 keys = 4 KiB of V, 32 bytes of a weight row
            if (leader)
              umma_ss_f8(tmem_base + (uint32_t)((k == 0 ? 2 : 3) * kRows), vb + (uint64_t)(ks * (4096 >> 4)),
                         pb + (uint64_t)((k * kRows * 128) >> 4) + (uint64_t)(ks * 2), idesc,
                         (j | ks) != 0 || k > 1 ? 1u : 0u);
        }
      }
      if (leader) {
        tc_commit(&empty[s]);
        tc_commit(&pv_done[j & 1]);
      }
      __syncwarp();
    }
  } else {
    // ---------------- softmax: thread = key ----------------
    const uint32_t lane_addr = (uint32_t)(warp * 32) << 16;
    const uint32_t o_tmem = tmem_base + 2 * kRows + lane_addr;
    float m_run = -INFINITY;  // of column `tid`: thread c keeps the running maximum of column c
    float l_lane[W];
#pragma unroll
    for (int c = 0; c < W; ++c) l_lane[c] = 0.f;
    if (tid < 2 * kRows) mc[tid] = 0.f;
    // the maxima as they are compared with: nothing is above those of columns that are not there
    if (tid < kRows) ml[tid] = tid < p.rows ? -INFINITY : INFINITY;
    const float my_fc = Q8 ? (tid < kRows ? fc[tid] : 0.f) : p.scale_log2;
    bool live = true;  // false once a bounded wait ran out: barriers are still walked, nothing is waited for
    uint32_t sr[W];
    // 8-bit pages: my key's scale codes, its page looked up a block ahead
    uint32_t k_code = 127, v_code = 127;
    int v_top = -1;  // the largest V scale code so far: weights are taken relative to it
    int page_next = -1, slot_next = 0;
    auto key_page = [&](int j, int& slot) -> int {
      const int key = (g_lo + j) * kKeys + tid;
      slot = 0;
      if (j >= n || key < lo || key >= hi) return -1;
      const uint32_t page = p.page_size.div((uint32_t)key);
      slot = key - (int)(page * p.page_size.d);
      return table[page];
    };
    auto key_codes = [&](int page, int slot, uint32_t& kc, uint32_t& vc) {
      kc = vc = 127u;
      if (page >= 0 && page < a.c.pages) {
        kc = a.c.k_scale[page * a.c.ks_sp + hk * a.c.ks_sh + slot];
        vc = a.c.v_scale[page * a.c.vs_sp + hk * a.c.vs_sh + slot];
      }
    };
    if constexpr (Q8) {
      const int page = key_page(0, slot_next);
      key_codes(page, slot_next, k_code, v_code);
      page_next = key_page(1, slot_next);
    }
    for (int j = 0; j < n; ++j) {
      uint32_t k_code_next = 127, v_code_next = 127;
      if constexpr (Q8) {
        key_codes(page_next, slot_next, k_code_next, v_code_next);
        page_next = key_page(j + 2, slot_next);
      }
      if (live && !mbar_wait(&s_full[j & 1], (j >> 1) & 1, a.status)) live = false;
      tc_fence_after();
      const uint32_t s_tmem = tmem_base + (uint32_t)((j & 1) * kRows) + lane_addr;
      const int base = (g_lo + j) * kKeys;
      const int key = base + tid;
      const bool real = key >= lo && key < hi;
      // whether some query token of the row does not see some key of the block
      const bool edge = base < all_lo || base + kKeys > all_hi;
      const float ks = Q8 ? scale_value(k_code) : 1.f;
      tmem_ld_w<W>(s_tmem, sr);
      if (Q8) {
#pragma unroll
        for (int c = 0; c < W; ++c) sr[c] = __float_as_uint(__uint_as_float(sr[c]) * ks);
      }
      if (edge) {
#pragma unroll
        for (int c = 0; c < W; ++c)
          if (key < lim[c] || key >= lim[kRows + c]) sr[c] = 0xff800000u;
      }
      // Most blocks bring no score (and no V scale) above what the running maxima allow: one
      // barrier says so, and the maxima and the reference stay. The first block sets them.
      bool over = j == 0;
#pragma unroll
      for (int c = 0; c < W; ++c)
        over = over || __uint_as_float(sr[c]) * (Q8 ? fc[c] : p.scale_log2) > ml[c] + kAdoptAbove<Q8>;
      if constexpr (Q8) over = over || (real && v_code != 255u && (int)v_code > v_top);
      bool moved = false;
      float v_corr = 1.f;  // 2^(old - new) of the V scales' reference
      if (barrier_or(2, over)) {
        float mine_max = 0.f;
#pragma unroll
        for (int c = 0; c < W; ++c) {
          const float wm = redux_max(__uint_as_float(sr[c]));
          if (lane == c) mine_max = wm;
        }
        if (lane < p.rows) red[lane * 4 + warp] = mine_max;
        if constexpr (Q8) {
          const int wv = __reduce_max_sync(0xffffffffu, real && v_code != 255u ? (int)v_code : -1);
          if (lane == 0) vred[warp] = wv;
        }
        named_barrier(1, 128);
        if constexpr (Q8) {
          const int v_new = max(v_top, max(max(vred[0], vred[1]), max(vred[2], vred[3])));
          if (v_new != v_top && v_top >= 0) {
            v_corr = power_below(v_top - v_new);
            moved = true;
          }
          v_top = v_new;
        }
        if (tid < p.rows) {
          const float4 w4 = *reinterpret_cast<const float4*>(red + tid * 4);
          const float mx = fmaxf(fmaxf(w4.x, w4.y), fmaxf(w4.z, w4.w)) * my_fc;
          float corr = 1.f;
          if (mx > m_run + kAdoptAbove<Q8> || m_run == -INFINITY) {
            const float m_new = fmaxf(m_run, mx);
            if (m_new != m_run && m_run != -INFINITY) {
              corr = ex2_approx(m_run - m_new);
              moved = true;
            }
            m_run = m_new;
          }
          mc[tid] = m_run == -INFINITY ? 0.f : m_run;
          mc[kRows + tid] = corr;
          ml[tid] = m_run;
        }
        moved = barrier_or(2, moved);
      }
      if (moved && j > 0) {
        // O holds the blocks before this one: rescale it once the last P.V is complete
        if (live && !mbar_wait(&pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1, a.status)) live = false;
        tc_fence_after();
        float f[W];
#pragma unroll
        for (int c = 0; c < W; ++c) f[c] = mc[kRows + c];
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          uint32_t orr[W];
          tmem_ld_w<W>(o_tmem + half * kRows, orr);
#pragma unroll
          for (int c = 0; c < W; ++c) orr[c] = __float_as_uint(__uint_as_float(orr[c]) * (f[c] * v_corr));
          tmem_st_w<W>(o_tmem + half * kRows, orr);
        }
#pragma unroll
        for (int c = 0; c < W; ++c) l_lane[c] *= f[c];
        tmem_st_wait();
      }
      // the block that last used this buffer of weights has been multiplied
      if (j >= C::kPBufs && live &&
          !mbar_wait(&pv_done[(j - C::kPBufs) & 1], ((j - C::kPBufs) >> 1) & 1, a.status))
        live = false;
      // this key's V scale over the largest; a NaN row's is NaN
      float vs = 1.f;
      if constexpr (Q8) vs = !real ? 0.f : v_code == 255u ? __uint_as_float(0x7fffffffu) : power_below((int)v_code - v_top);
      // All loads, then the arithmetic, then all stores: the compiler may not move a load of a
      // maximum above a store of a weight.
      float mu[W], sc[W];
#pragma unroll
      for (int c = 0; c < W; ++c) mu[c] = mc[c], sc[c] = Q8 ? fc[c] : p.scale_log2;
      if constexpr (!Q8) {
        uint8_t* pbox = p_s + (j % C::kPBufs) * C::kPBytes + (tid >> 6) * (2 * kRows * 128) + (tid & 7) * 2;
        const int chunk = (tid & 63) >> 3;
        T high[W], low[W];
#pragma unroll
        for (int c = 0; c < W; ++c) {
          const float pr = ex2_approx(fmaf(__uint_as_float(sr[c]), sc[c], -mu[c]));
          l_lane[c] += pr;
          const float up = pr * kValueUp<T>;
          high[c] = Elem<T>::from_f(up);
          low[c] = Elem<T>::from_f((up - Elem<T>::to_f(high[c])) * kRestUp<T>);
        }
#pragma unroll
        for (int c = 0; c < W; ++c) {
          uint8_t* dst = pbox + c * 128 + ((chunk ^ (c & 7)) << 4);
          *reinterpret_cast<T*>(dst) = high[c];
          *reinterpret_cast<T*>(dst + kRows * 128) = low[c];
        }
      } else {
        uint8_t* pbox = p_s + (j % C::kPBufs) * C::kPBytes + (tid & 15);
        const int chunk = tid >> 4;
        uint32_t piece[WP][W / 2];  // two columns each
#pragma unroll
        for (int c = 0; c < W; c += 2) {
          const float p0 = ex2_approx(fmaf(__uint_as_float(sr[c]), sc[c], -mu[c]));
          const float p1 = ex2_approx(fmaf(__uint_as_float(sr[c + 1]), sc[c + 1], -mu[c + 1]));
          l_lane[c] += p0, l_lane[c + 1] += p1;
          float w0 = real ? p0 * vs : 0.f, w1 = real ? p1 * vs : 0.f;
          piece[0][c / 2] = to_e4m3x2(w0, w1);
          const float2 x = from_e4m3x2(piece[0][c / 2]);
          w0 = (w0 - x.x) * kRemainderUp, w1 = (w1 - x.y) * kRemainderUp;
#pragma unroll
          for (int k = 1; k < WP; ++k) {
            piece[k][c / 2] = to_e5m2x2(w0, w1);
            if (k + 1 < WP) {
              const float2 y = from_e5m2x2(piece[k][c / 2]);
              w0 -= y.x, w1 -= y.y;
            }
          }
        }
#pragma unroll
        for (int c = 0; c < W; ++c)
#pragma unroll
          for (int k = 0; k < WP; ++k)
            pbox[k * (kRows * 128) + c * 128 + ((chunk ^ (c & 7)) << 4)] = (uint8_t)(piece[k][c / 2] >> ((c & 1) * 8));
      }
      if (base < lo || base + kKeys > hi) {
        // The block's rows outside the visible keys hold whatever the pages hold there:
        // their weights are zero, and zero values keep 0 * NaN out of the sum.
        const uint32_t pos = pos_v(j, n);
        if (live && !mbar_wait(&full[pos % S], (pos / S) & 1, a.status)) live = false;
        if (!real) {
          uint8_t* vr = ring + (pos % S) * C::kSlotBytes + tid * 128;
#pragma unroll
          for (int c = 0; c < C::kBoxes * 8; ++c)
            *reinterpret_cast<uint4*>(vr + (c >> 3) * kBox + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
      }
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[j & 1]);
      k_code = k_code_next, v_code = v_code_next;
    }
    // ---- this CTA's state: m, l, O (f32) into shared memory ----
    if (n > 0) {
      if (live && !mbar_wait(&pv_done[(n - 1) & 1], ((n - 1) >> 1) & 1, a.status)) live = false;
      tc_fence_after();
      float* op = reinterpret_cast<float*>(ring);
      const float low_down = Q8 ? 1.f / kRemainderUp : 1.f / kRestUp<T>;
      const float o_up = Q8 ? scale_value(v_top < 0 ? 127u : (uint32_t)v_top) : 1.f / kValueUp<T>;
      float mine_sum = 0.f;
#pragma unroll
      for (int c = 0; c < W; ++c) {
        const float x = warp_sum(l_lane[c]);
        if (lane == c) mine_sum = x;
      }
      if (lane < p.rows) red[lane * 4 + warp] = mine_sum;
      if (warp * 32 < D) {
        uint32_t low[W];
        tmem_ld_w<W>(o_tmem, sr);
        tmem_ld_w<W>(o_tmem + kRows, low);
#pragma unroll
        for (int c = 0; c < W; ++c)
          if (c < p.rows) op[c * D + tid] = fmaf(__uint_as_float(low[c]), low_down, __uint_as_float(sr[c])) * o_up;
      }
      named_barrier(1, 128);
    }
    if (tid < p.rows) {
      float l = 0.f;
      if (n > 0) {
        const float4 w4 = *reinterpret_cast<const float4*>(red + tid * 4);
        l = (w4.x + w4.y) + (w4.z + w4.w);
      }
      ml[tid] = n > 0 ? m_run : -INFINITY;
      ml[kRows + tid] = l;
    }
    tc_fence_before();
  }
  __syncwarp();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
  // ---- merge the cluster's partial states: CTA `rank` takes every csize-th run of columns ----
  cluster_sync_all();
  {
    const int per_row = a.c.d / 8;
    const uint32_t op_addr = smem_u32(ring), ml_addr = smem_u32(ml);
    for (int i = (int)rank * kThreadsDec + tid; i < p.rows * per_row; i += (int)csize * kThreadsDec) {
      const int c = i / per_row, d0 = (i % per_row) * 8;
      const int64_t tq = c / p.group;
      const int h = hk * p.group + c % p.group;
      float m = -INFINITY, l = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (tq < r.n) {
        // four CTAs' states at a time: one after the other, each is a trip across the cluster
        for (uint32_t k0 = 0; k0 < csize; k0 += 4) {
          float mr[4], lr[4];
          float4 x[4], y[4];
#pragma unroll
          for (uint32_t u = 0; u < 4; ++u) {
            const uint32_t k = k0 + u < csize ? k0 + u : k0;
            mr[u] = ld_cluster_f32(cluster_at(ml_addr + c * 4, k));
            lr[u] = ld_cluster_f32(cluster_at(ml_addr + (kRows + c) * 4, k));
            const uint32_t src = cluster_at(op_addr + (c * D + d0) * 4, k);
            x[u] = ld_cluster_f32x4(src), y[u] = ld_cluster_f32x4(src + 16);
          }
#pragma unroll
          for (uint32_t u = 0; u < 4; ++u) {
            // a share that saw no key (its sum says so: NaN scores leave the maximum at -inf too), or none at all
            if (k0 + u >= csize || lr[u] == 0.f) continue;
            const float m_new = fmaxf(m, mr[u]);
            const float f0 = m == -INFINITY ? 1.f : ex2_approx(m - m_new), f1 = mr[u] == -INFINITY ? 1.f : ex2_approx(mr[u] - m_new);
            m = m_new;
            l = fmaf(l, f0, f1 * lr[u]);
            acc[0] = fmaf(acc[0], f0, f1 * x[u].x), acc[1] = fmaf(acc[1], f0, f1 * x[u].y);
            acc[2] = fmaf(acc[2], f0, f1 * x[u].z), acc[3] = fmaf(acc[3], f0, f1 * x[u].w);
            acc[4] = fmaf(acc[4], f0, f1 * y[u].x), acc[5] = fmaf(acc[5], f0, f1 * y[u].y);
            acc[6] = fmaf(acc[6], f0, f1 * y[u].z), acc[7] = fmaf(acc[7], f0, f1 * y[u].w);
          }
        }
      }
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      // (65504 in f16 is 65536 as the pages hold it)
      auto pair = [&](float x, float y) {
        if constexpr (Q8 && std::is_same<T, __half>::value) return pack_in_range<T>(x * inv, y * inv);
        else return Elem<T>::pack(x * inv, y * inv);
      };
      stg128((T*)a.o + (int64_t)b * a.o_sb + tq * a.o_st + (int64_t)h * a.o_sh + d0,
             make_uint4(pair(acc[0], acc[1]), pair(acc[2], acc[3]), pair(acc[4], acc[5]), pair(acc[6], acc[7])));
      if (a.lse != nullptr && d0 == 0)
        a.lse[((int64_t)b * a.heads + h) * a.t + tq] = l == 0.f ? -INFINITY : kLn2F * (m + log2f(l));
    }
  }
  cluster_sync_all();  // no CTA leaves while a peer still reads its partial state
}

int sms() {
  static int n = 0;
  if (n == 0) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (n <= 0) n = 148;
  }
  return n;
}

// The most blocks of keys a row may see: what its table reaches, or its window.
int64_t most_blocks(const PagedAttnArgs& a) {
  int64_t keys = a.c.width * a.c.page_size;
  if (a.has_window) {
    const int64_t w = a.win_left + a.t + (a.causal ? 0 : a.win_right) + kKeys;
    keys = w < keys ? w : keys;
  }
  return (keys + kKeys - 1) / kKeys;
}

// Shares per (row, KV head): doubled while the grid stays within the CTAs that the chip holds
// at once, and once beyond that while a share keeps 32 blocks: the rows' lengths are not known
// here, and shares of ragged rows fill the chip's last places better, while each costs its
// start and a merge. 8 KV heads throughout, this rule, no share beyond the chip, shares
// up to four times the chip: 24 rows of 64..16000 keys in bf16 133, 168, 134 us; in e4m3 16
// rows of 8000..32767 116, 169, 130 and 40 such rows 268, 397, 310; where all rows are equally
// long the last two win (16 rows of 32767 220, 184, 199). Clusters have to find their CTAs'
// places in one GPC, hence the limits of attention_decode.cu.
int cluster_of(int64_t pairs, int64_t blocks, int per_sm) {
  const int64_t room = (int64_t)sms() * per_sm;
  int csize = 1;
  while (csize < 16 && csize * 2 <= blocks &&
         (pairs * csize * 2 <= room || (pairs * csize <= room && blocks >= 32 * csize * 2))) {
    if (csize == 8 && pairs > 6 * per_sm) break;
    csize *= 2;
  }
  return csize;
}

template <typename T, bool Q8, int D, int W>
int run_rows(const PagedAttnArgs& a, cudaStream_t s, char* cfg, size_t cfg_len) {
  using C = PagedDecCfg<T, Q8, D>;
  CUtensorMap tk, tv;
  PagedDecParams p{};
  p.box = page_box(a.c.page_size, kKeys);
  p.page_size = divider((uint32_t)a.c.page_size);
  if (!page_map(&tk, a.c, false, Q8 ? 128 : 64, p.box) || !page_map(&tv, a.c, true, Q8 ? 128 : 64, p.box)) return -1;
  static bool attr_seen[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr_seen[dev & 63]) {
    if (cudaFuncSetAttribute(attention_paged_decode_kernel<T, Q8, D, W>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)C::kSmem) != cudaSuccess ||
        cudaFuncSetAttribute(attention_paged_decode_kernel<T, Q8, D, W>, cudaFuncAttributeNonPortableClusterSizeAllowed,
                             1) != cudaSuccess)
      return -1;
    attr_seen[dev & 63] = true;
  }
  p.a = a;
  p.group = a.heads / a.c.kv_heads;
  p.rows = (int)a.t * p.group;
  p.scale_log2 = a.scale * kLog2eF;
  const int64_t pairs = a.batch * a.c.kv_heads;
  const int csize = cluster_of(pairs, most_blocks(a), C::kPerSm);
  const int64_t room = (int64_t)sms() * C::kPerSm;
  p.longest_first = a.batch > 1 && a.batch <= kSortedRows && pairs * csize > room && pairs * csize <= kOrderedWaves * room;
  if (launch_pdl(attention_paged_decode_kernel<T, Q8, D, W>, dim3((unsigned)(pairs * csize)), dim3(kThreadsDec), C::kSmem,
                 s, (unsigned)csize, a.batch * a.t, tk, tv, p) != cudaSuccess)
    return -1;
  snprintf(cfg, cfg_len, "{rows:%d,bkv:%d,d:%d,box:%d,cluster:%d%s%s}", W, kKeys, a.c.d, p.box, csize, Q8 ? ",e4m3" : "",
           p.longest_first ? ",longest_first" : "");
  return 0;
}

template <typename T, bool Q8, int D>
int run_width(const PagedAttnArgs& a, cudaStream_t s, char* cfg, size_t cfg_len) {
  const int64_t rows = a.t * (a.heads / a.c.kv_heads);
  if (rows <= 4) return run_rows<T, Q8, D, 4>(a, s, cfg, cfg_len);
  if (rows <= 8) return run_rows<T, Q8, D, 8>(a, s, cfg, cfg_len);
  return run_rows<T, Q8, D, 16>(a, s, cfg, cfg_len);
}

template <typename T>
int run_type(const PagedAttnArgs& a, cudaStream_t s, char* cfg, size_t cfg_len) {
  if (a.c.dtype == SVODB_E4M3) return run_width<T, true, 128>(a, s, cfg, cfg_len);
  return a.c.d > 64 ? run_width<T, false, 128>(a, s, cfg, cfg_len) : run_width<T, false, 64>(a, s, cfg, cfg_len);
}

}  // namespace

int page_box(int page_size, int most) {
  int x = page_size, y = most;
  while (y != 0) {
    const int z = x % y;
    x = y, y = z;
  }
  return x;
}

bool page_map(CUtensorMap* map, const PagedCache& c, bool values, uint32_t cols, uint32_t rows) {
  const uint64_t dims[4] = {(uint64_t)c.d, (uint64_t)c.kv_heads, (uint64_t)c.page_size, (uint64_t)c.pages};
  // a dim of one element has no stride of its own: any that the map takes will do
  const uint64_t any = 128;
  const uint64_t st[3] = {c.kv_heads == 1 ? any : (uint64_t)(values ? c.v_sh : c.k_sh),
                          c.page_size == 1 ? any : (uint64_t)(values ? c.v_ss : c.k_ss),
                          c.pages == 1 ? any : (uint64_t)(values ? c.v_sp : c.k_sp)};
  const uint32_t box[4] = {cols, 1, rows, 1};
  return make_tmap(map, values ? c.v : c.k, c.dtype, 4, dims, st, box);
}

// What the tensor-core kernels over pages take: 16-bit streams, pages of them or of e4m3 on
// the 16-byte grid, head widths that are whole 16-byte pieces, pages of whole 8-row groups (a
// box starts on a 1 KiB boundary of its tile), a positive scale (maxima are of raw scores).
bool attention_paged_tiles(const PagedAttnArgs& a) {
  if (a.dtype != SVODB_BF16 && a.dtype != SVODB_F16) return false;
  const int64_t size = a.c.dtype == SVODB_E4M3 ? 1 : 2;
  if (a.c.d < 8 || a.c.d > 128 || a.c.d * size % 16 != 0) return false;
  if (a.c.page_size % 8 != 0 || a.c.pages == 0 || a.c.width == 0) return false;
  if (!(a.scale > 0.f) || !isfinite(a.scale)) return false;
  if (!aligned16(a.c.k) || !aligned16(a.c.v) || !aligned16(a.q) || !aligned16(a.o)) return false;
  const int64_t pages[6] = {a.c.kv_heads > 1 ? a.c.k_sh : 0, a.c.k_ss, a.c.pages > 1 ? a.c.k_sp : 0,
                            a.c.kv_heads > 1 ? a.c.v_sh : 0, a.c.v_ss, a.c.pages > 1 ? a.c.v_sp : 0};
  for (int64_t st : pages)
    if (st * size % 16 != 0 || st * size >= (int64_t)1 << 40) return false;
  // a tensor map has no stride of zero (an expanded view)
  if (a.c.k_ss == 0 || a.c.v_ss == 0 || (a.c.kv_heads > 1 && (a.c.k_sh == 0 || a.c.v_sh == 0)) ||
      (a.c.pages > 1 && (a.c.k_sp == 0 || a.c.v_sp == 0)))
    return false;
  for (int64_t st : {a.q_sb, a.q_st, a.q_sh, a.o_sb, a.o_st, a.o_sh})
    if (st % 8 != 0) return false;
  return true;
}

// Up to 16 query rows a KV head, whatever the keys. With more of them this form loses to the
// 128-row tiles, which share the keys out evenly and take 64 rows for what they take for one
// (measured here with 32 and 64 columns against there: 24 rows x 100..2500 keys x 27 query rows
// 66 us | 27; 64 x 64..4095 x 24 196 | 173; 16 x 8000..32767 in e4m3 x 24 516 | 386; 1 x 30000 x
// 60 148 | 62; 1 x 776 x 24 20 | 19). Where it takes the call, the other way round: 24 rows x 15
// query rows 20 | 27, 64 x 12 110 | 174, 16 in e4m3 x 12 215 | 386, 1 x 776 x 12 12 | 19.
bool attention_paged_few_rows(const PagedAttnArgs& a) {
  return a.t * (a.heads / a.c.kv_heads) <= kRows && a.batch * a.c.kv_heads <= (1 << 26);
}

bool attention_paged_decode_covers(const PagedAttnArgs& a) { return attention_paged_tiles(a) && attention_paged_few_rows(a); }

int launch_attention_paged_decode(const PagedAttnArgs& a, cudaStream_t s, char* cfg, size_t cfg_len) {
  return a.dtype == SVODB_BF16 ? run_type<__nv_bfloat16>(a, s, cfg, cfg_len) : run_type<__half>(a, s, cfg, cfg_len);
}

}  // namespace svodb
