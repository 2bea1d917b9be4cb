// A paged key/value cache: new tokens written into its pages (as they are or in 8 bits),
// pages read back into rows, and attention over the pages for every type, width and page
// size (`attention_paged_exact`; the tensor-core kernels are in their own files).
//
// Write and read move every byte once and are bound by HBM, or by the chain
// start -> table -> page of dependent loads where there is little to move. Reading, and writing
// 16 bits, a lane owns 8 elements of a head row, 16 bytes on the 16-bit side and 8 on the 8-bit
// side, so that a warp's accesses are whole lines (with 16 elements a lane every other 16 bytes:
// 113 us against 103 for reading six rows of 3000 to 16384 e4m3 tokens, 117 against 100 in bf16,
// which is 6.4 TB/s); writing 8 bits it owns 16 (kPerLane), and a row's lanes find its largest
// value among themselves.
#include <math.h>

#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "launch.h"
#include "paged.cuh"
#include "svodb.h"

namespace svodb {

namespace {

using namespace paged;

constexpr int kThreadsPaged = 256;

// The slot of position `pos` of row b: {page, slot}; page < 0 when the table's entry is none.
__device__ __forceinline__ int64_t page_of(const PagedCache& c, int64_t b, int64_t page, uint32_t* bad_index) {
  const int32_t id = c.table[b * c.table_sb + page];
  if (id < 0 || id >= c.pages) {
    report_bad_index(bad_index);
    return -1;
  }
  return id;
}

template <typename T>
__device__ __forceinline__ void widen8(uint4 u, float* f) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = Elem<T>::unpack(w[i]);
    f[2 * i] = v.x, f[2 * i + 1] = v.y;
  }
}

// Head rows a thread has a part of at once, their look-ups and loads on their way together. A
// row on its way into 8 bits holds 16 values in registers: there more threads an SM do more
// (10240 tokens x 8 heads x 128: 20.9 us with four, 17.5 with two, 18.9 with one).
template <bool Q8Write>
constexpr int kRowsAtOnce = Q8Write ? 2 : 4;

// Values of a head row that a lane has: whole lines go out and in with 8 of them (16 bytes on
// the 16-bit side); into 8 bits 16, whose e4m3 values are one 16-byte store and whose row
// needs a shuffle less (10240 tokens x 8 heads x 128: 21 us against 25).
template <bool Q8>
constexpr int kPerLane = Q8 ? 16 : 8;

// A token's head row a group of LPR lanes; block (run of a row's head rows, keys or values,
// row). One head row a thread, with its row and head from 64-bit divisions, took 26 us for
// 10240 tokens x 8 heads x 128 into e4m3.
template <typename T, bool Q8, int LPR>
__global__ void __launch_bounds__(kThreadsPaged) cache_write_kernel(const CacheWriteArgs a, const Divider heads, const Divider page_size) {
  constexpr int E = kPerLane<Q8>, N = kRowsAtOnce<Q8>;
  pdl_trigger();
  pdl_wait();
  const bool is_v = blockIdx.y != 0;
  const int b = blockIdx.z, sub = threadIdx.x % LPR;
  const Row r = row_of(a.start, a.lens, b, a.t, a.c.width * a.c.page_size);
  if (r.bad && blockIdx.x == 0 && threadIdx.x == 0) report_bad_index(a.bad_index);
  const uint32_t rows = (uint32_t)r.n * a.c.kv_heads;  // of this sequence's chunk
  const uint32_t row0 = blockIdx.x * (kThreadsPaged / LPR * N) + threadIdx.x / LPR;
  if (blockIdx.x * (kThreadsPaged / LPR * N) >= rows) return;  // the whole block: shuffles stay whole
  const T* src = is_v ? (const T*)a.v + b * a.v_sb : (const T*)a.k + b * a.k_sb;
  const int64_t src_t = is_v ? a.v_st : a.k_st, src_h = is_v ? a.v_sh : a.k_sh;
  const int64_t sp = is_v ? a.c.v_sp : a.c.k_sp, ss = is_v ? a.c.v_ss : a.c.k_ss, sh = is_v ? a.c.v_sh : a.c.k_sh;
  uint4 u[N][E / 8];
  int64_t page[N];
  uint32_t slot[N], head[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const uint32_t row = row0 + k * (kThreadsPaged / LPR);
    page[k] = -1;
    const uint32_t i = heads.div(row);
    head[k] = row - i * heads.d;
#pragma unroll
    for (int e = 0; e < E / 8; ++e) u[k][e] = make_uint4(0, 0, 0, 0);
    if (row < rows) {
#pragma unroll
      for (int e = 0; e < E / 8; ++e) u[k][e] = ldg128(src + i * src_t + head[k] * src_h + sub * E + e * 8);
      const uint32_t pos = (uint32_t)r.start + i, at = page_size.div(pos);
      slot[k] = pos - at * page_size.d;
      page[k] = page_of(a.c, b, at, a.bad_index);
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int64_t to = page[k] * sp + slot[k] * ss + head[k] * sh + sub * E;
    if constexpr (!Q8) {
      if (page[k] >= 0) stg128((T*)(is_v ? a.c.v : a.c.k) + to, u[k][0]);
    } else {
      float f[E];
#pragma unroll
      for (int e = 0; e < E / 8; ++e) widen8<T>(u[k][e], f + 8 * e);
      // the largest as an integer: a NaN's bits are above every number's, and stay so
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (page[k] < 0) continue;
      const uint32_t code = scale_code(__uint_as_float(top));
      const float inv = code == 255u ? 0.f : scale_inverse(code);
      uint32_t w[E / 4];
#pragma unroll
      for (int e = 0; e < E / 4; ++e) {
        const uint32_t lo = to_e4m3x2(f[4 * e] * inv, f[4 * e + 1] * inv), hi = to_e4m3x2(f[4 * e + 2] * inv, f[4 * e + 3] * inv);
        w[e] = code == 255u ? 0u : lo | (hi << 16);
      }
      stg128((uint8_t*)(is_v ? a.c.v : a.c.k) + to, make_uint4(w[0], w[1], w[2], w[3]));
      if (sub == 0) {
        if (is_v) a.c.v_scale[page[k] * a.c.vs_sp + head[k] * a.c.vs_sh + slot[k]] = (uint8_t)code;
        else a.c.k_scale[page[k] * a.c.ks_sp + head[k] * a.c.ks_sh + slot[k]] = (uint8_t)code;
      }
    }
  }
}

// The same for every width and alignment: a warp a head row.
template <typename T, bool Q8>
__global__ void __launch_bounds__(kThreadsPaged) cache_write_any_kernel(const CacheWriteArgs a) {
  pdl_trigger();
  pdl_wait();
  const bool is_v = blockIdx.y != 0;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * (kThreadsPaged / 32) + (threadIdx.x >> 5);
  if (row >= a.batch * a.t * a.c.kv_heads) return;
  const int64_t token = row / a.c.kv_heads;
  const int h = (int)(row % a.c.kv_heads);
  const int64_t b = token / a.t, i = token % a.t;
  const Row r = row_of(a.start, a.lens, b, a.t, a.c.width * a.c.page_size);
  if (r.bad && i == 0 && lane == 0) report_bad_index(a.bad_index);
  if (i >= r.n) return;
  const int64_t pos = r.start + i, at = pos / a.c.page_size;
  const int slot = (int)(pos - at * a.c.page_size);
  const int64_t page = page_of(a.c, b, at, a.bad_index);
  if (page < 0) return;
  const T* src = is_v ? (const T*)a.v + b * a.v_sb + i * a.v_st + h * a.v_sh : (const T*)a.k + b * a.k_sb + i * a.k_st + h * a.k_sh;
  const int64_t to = is_v ? page * a.c.v_sp + slot * a.c.v_ss + h * a.c.v_sh : page * a.c.k_sp + slot * a.c.k_ss + h * a.c.k_sh;
  void* base = is_v ? a.c.v : a.c.k;
  if constexpr (!Q8) {
    for (int e = lane; e < a.c.d; e += 32) ((T*)base)[to + e] = src[e];
  } else {
    uint32_t top = 0;
    for (int e = lane; e < a.c.d; e += 32) top = max(top, __float_as_uint(Elem<T>::to_f(src[e])) & 0x7fffffffu);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const uint32_t code = scale_code(__uint_as_float(top));
    const float inv = code == 255u ? 0.f : scale_inverse(code);
    for (int e = lane; e < a.c.d; e += 32)
      ((uint8_t*)base)[to + e] = code == 255u ? 0 : (uint8_t)(to_e4m3x2(Elem<T>::to_f(src[e]) * inv, 0.f) & 0xffu);
    if (lane == 0) {
      if (is_v) a.c.v_scale[page * a.c.vs_sp + h * a.c.vs_sh + slot] = (uint8_t)code;
      else a.c.k_scale[page * a.c.ks_sp + h * a.c.ks_sh + slot] = (uint8_t)code;
    }
  }
}

// Eight e4m3 values times their scale, rounded to the stream type and kept in its range.
template <typename T>
__device__ __forceinline__ uint4 widen_e4m3(uint2 u, float scale) {
  const float2 a = from_e4m3x2(u.x & 0xffffu), b = from_e4m3x2(u.x >> 16), c = from_e4m3x2(u.y & 0xffffu), d = from_e4m3x2(u.y >> 16);
  return make_uint4(pack_in_range<T>(a.x * scale, a.y * scale), pack_in_range<T>(b.x * scale, b.y * scale),
                    pack_in_range<T>(c.x * scale, c.y * scale), pack_in_range<T>(d.x * scale, d.y * scale));
}

__device__ __forceinline__ uint2 ldg64(const void* p) {
  uint2 v;
  asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

// As cache_write_kernel is laid out; rows behind a sequence's end are zeros.
template <typename T, bool Q8, int LPR>
__global__ void __launch_bounds__(kThreadsPaged) cache_read_kernel(const CacheReadArgs a, const Divider heads, const Divider page_size) {
  constexpr int N = kRowsAtOnce<false>;
  pdl_trigger();
  pdl_wait();
  const bool is_v = blockIdx.y != 0;
  const int b = blockIdx.z, sub = threadIdx.x % LPR;
  const Row r = row_of(nullptr, a.lens, b, a.len, a.c.width * a.c.page_size);
  if (r.bad && blockIdx.x == 0 && threadIdx.x == 0) report_bad_index(a.bad_index);
  const uint32_t rows = (uint32_t)a.len * a.c.kv_heads;
  const uint32_t row0 = blockIdx.x * (kThreadsPaged / LPR * N) + threadIdx.x / LPR;
  const int64_t sp = is_v ? a.c.v_sp : a.c.k_sp, ss = is_v ? a.c.v_ss : a.c.k_ss, sh = is_v ? a.c.v_sh : a.c.k_sh;
  T* out = is_v ? (T*)a.v + b * a.v_sb : (T*)a.k + b * a.k_sb;
  const int64_t out_t = is_v ? a.v_st : a.k_st, out_h = is_v ? a.v_sh : a.k_sh;
  std::conditional_t<Q8, uint2, uint4> u[N];
  uint32_t code[N], head[N], token[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const uint32_t row = row0 + k * (kThreadsPaged / LPR);
    token[k] = heads.div(row);
    head[k] = row - token[k] * heads.d;
    code[k] = 0u;
    u[k] = {};
    if (row < rows && token[k] < (uint32_t)r.n) {
      const uint32_t at = page_size.div(token[k]), slot = token[k] - at * page_size.d;
      const int64_t page = page_of(a.c, b, at, a.bad_index);
      if (page >= 0) {
        const int64_t from = page * sp + slot * ss + head[k] * sh + sub * 8;
        if constexpr (Q8) {
          u[k] = ldg64((const uint8_t*)(is_v ? a.c.v : a.c.k) + from);
          code[k] = is_v ? a.c.v_scale[page * a.c.vs_sp + head[k] * a.c.vs_sh + slot]
                         : a.c.k_scale[page * a.c.ks_sp + head[k] * a.c.ks_sh + slot];
        } else {
          u[k] = ldg128((const T*)(is_v ? a.c.v : a.c.k) + from);
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    if (row0 + k * (kThreadsPaged / LPR) >= rows) continue;
    T* dst = out + token[k] * out_t + head[k] * out_h + sub * 8;
    if constexpr (Q8) stg128(dst, widen_e4m3<T>(u[k], scale_value(code[k])));
    else stg128(dst, u[k]);
  }
}

template <typename T, bool Q8>
__global__ void __launch_bounds__(kThreadsPaged) cache_read_any_kernel(const CacheReadArgs a) {
  pdl_trigger();
  pdl_wait();
  const bool is_v = blockIdx.y != 0;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * (kThreadsPaged / 32) + (threadIdx.x >> 5);
  if (row >= a.batch * a.len * a.c.kv_heads) return;
  const int64_t token = row / a.c.kv_heads;
  const int h = (int)(row % a.c.kv_heads);
  const int64_t b = token / a.len, pos = token % a.len;
  const Row r = row_of(nullptr, a.lens, b, a.len, a.c.width * a.c.page_size);
  if (r.bad && pos == 0 && lane == 0) report_bad_index(a.bad_index);
  int64_t page = -1, from = 0;
  float scale = 0.f;
  if (pos < r.n) {
    const int64_t at = pos / a.c.page_size;
    const int slot = (int)(pos - at * a.c.page_size);
    page = page_of(a.c, b, at, a.bad_index);
    if (page >= 0) {
      from = is_v ? page * a.c.v_sp + slot * a.c.v_ss + h * a.c.v_sh : page * a.c.k_sp + slot * a.c.k_ss + h * a.c.k_sh;
      if constexpr (Q8) scale = scale_value(is_v ? a.c.v_scale[page * a.c.vs_sp + h * a.c.vs_sh + slot] : a.c.k_scale[page * a.c.ks_sp + h * a.c.ks_sh + slot]);
    }
  }
  T* dst = is_v ? (T*)a.v + b * a.v_sb + pos * a.v_st + h * a.v_sh : (T*)a.k + b * a.k_sb + pos * a.k_st + h * a.k_sh;
  const void* base = is_v ? a.c.v : a.c.k;
  for (int e = lane; e < a.c.d; e += 32) {
    if (page < 0) dst[e] = Elem<T>::from_f(0.f);
    else if constexpr (Q8) dst[e] = Elem<T>::from_f(in_range<T>(from_e4m3x2(((const uint8_t*)base)[from + e]).x * scale));
    else dst[e] = ((const T*)base)[from + e];
  }
}

// ---- exact attention -------------------------------------------------------------
// A block a query row and head; its four warps take every fourth visible key, lanes hold
// the head's elements d = lane + 32 i, and the four running states meet in shared memory.
template <typename T, bool Q8>
__global__ void __launch_bounds__(128) attention_paged_exact_kernel(const PagedAttnArgs a) {
  constexpr int kMaxD = 256, kPer = kMaxD / 32, kWarps = 4;
  __shared__ float o_s[kWarps][kMaxD];
  __shared__ float m_s[kWarps], l_s[kWarps];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t item = blockIdx.x;
  const int h = (int)(item % a.heads);
  const int64_t i = item / a.heads % a.t, b = item / a.heads / a.t;
  const int hk = h / (a.heads / a.c.kv_heads), d = a.c.d;
  const Row r = row_of(a.start, a.lens, b, a.t, a.c.width * a.c.page_size);
  if (r.bad && i == 0 && h == 0 && threadIdx.x == 0) report_bad_index(a.bad_index);
  const int64_t pos = r.start + i;
  int64_t lo = 0, hi = r.start + r.n;
  if (a.causal && pos + 1 < hi) hi = pos + 1;
  if (a.has_window) {
    if (pos - a.win_left > lo) lo = pos - a.win_left;
    if (pos + a.win_right + 1 < hi) hi = pos + a.win_right + 1;
  }
  if (i >= r.n) hi = lo;
  float q[kPer], o[kPer];
  const T* qp = (const T*)a.q + b * a.q_sb + i * a.q_st + h * a.q_sh;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    q[e] = lane + 32 * e < d ? Elem<T>::to_f(qp[lane + 32 * e]) : 0.f;
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t j = lo + warp; j < hi; j += kWarps) {
    const int64_t at = j / a.c.page_size;
    const int slot = (int)(j - at * a.c.page_size);
    const int64_t page = page_of(a.c, b, at, a.bad_index);
    const bool there = page >= 0;  // where no page is, a key and a value of zeros, as reading gives
    const int64_t fk = page * a.c.k_sp + slot * a.c.k_ss + hk * a.c.k_sh, fv = page * a.c.v_sp + slot * a.c.v_ss + hk * a.c.v_sh;
    float ks = 1.f, vs = 1.f;
    if (Q8 && there) {
      ks = scale_value(a.c.k_scale[page * a.c.ks_sp + hk * a.c.ks_sh + slot]);
      vs = scale_value(a.c.v_scale[page * a.c.vs_sp + hk * a.c.vs_sh + slot]);
    }
    float s = 0.f, v[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int c = lane + 32 * e;
      v[e] = 0.f;
      if (c < d && there) {
        if constexpr (Q8) {
          s = fmaf(q[e], in_range<T>(from_e4m3x2(((const uint8_t*)a.c.k)[fk + c]).x * ks), s);
          v[e] = in_range<T>(from_e4m3x2(((const uint8_t*)a.c.v)[fv + c]).x * vs);
        } else {
          s = fmaf(q[e], Elem<T>::to_f(((const T*)a.c.k)[fk + c]), s);
          v[e] = Elem<T>::to_f(((const T*)a.c.v)[fv + c]);
        }
      }
    }
    s = warp_sum(s) * a.scale;
    const float m_new = fmaxf(m, s), m_use = m_new == -INFINITY ? 0.f : m_new;
    const float corr = m == -INFINITY ? 0.f : expf(m - m_use), p = expf(s - m_use);
    l = fmaf(l, m == -INFINITY ? 1.f : corr, p);
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] = fmaf(o[e], m == -INFINITY ? 1.f : corr, p * v[e]);
    m = m_new;
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) o_s[warp][lane + 32 * e] = o[e];
  if (lane == 0) m_s[warp] = m, l_s[warp] = l;
  __syncthreads();
  float top = -INFINITY, total = 0.f, w[kWarps];
#pragma unroll
  for (int k = 0; k < kWarps; ++k) top = fmaxf(top, m_s[k]);
#pragma unroll
  for (int k = 0; k < kWarps; ++k) {
    w[k] = l_s[k] == 0.f ? 0.f : m_s[k] == -INFINITY ? 1.f : expf(m_s[k] - top);
    total = fmaf(w[k], l_s[k], total);
  }
  T* op = (T*)a.o + b * a.o_sb + i * a.o_st + h * a.o_sh;
  const float inv = total == 0.f ? 0.f : 1.0f / total;
  for (int c = threadIdx.x; c < d; c += 128) {
    float x = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k)
      if (l_s[k] != 0.f) x = fmaf(w[k], o_s[k][c], x);
    op[c] = Elem<T>::from_f(x * inv);
  }
  if (a.lse != nullptr && threadIdx.x == 0) a.lse[(b * a.heads + h) * a.t + i] = total == 0.f ? -INFINITY : top + logf(total);
}

// Lanes a row of d values takes at `per` a lane: a power of two, a warp's at most; 0 = no such.
int lanes_a_row(int d, int per) {
  if (d % per != 0 || d > 32 * per) return 0;
  const int l = d / per;
  return (l & (l - 1)) == 0 ? l : 0;
}
bool on_grid(const void* p, std::initializer_list<int64_t> strides, int64_t size) {
  if (!aligned16(p)) return false;
  for (int64_t s : strides)
    if (s * size % 16 != 0) return false;
  return true;
}
bool pages_on_grid(const PagedCache& c) {
  const int64_t size = c.dtype == SVODB_E4M3 ? 1 : c.dtype == SVODB_F32 ? 4 : 2;
  return on_grid(c.k, {c.k_sp, c.k_ss, c.k_sh}, size) && on_grid(c.v, {c.v_sp, c.v_ss, c.v_sh}, size);
}

unsigned blocks_of(int64_t n, int64_t per) { return (unsigned)((n + per - 1) / per); }

// Whether a vector kernel's block and row numbers hold the call: 31 bits of head rows a sequence.
bool within(const PagedCache& c, int64_t batch, int64_t tokens) {
  return batch <= 65535 && tokens * c.kv_heads < (int64_t)1 << 31;
}

template <typename T, bool Q8>
int run_write(const CacheWriteArgs& a, cudaStream_t s) {
  const int64_t rows = a.batch * a.t * a.c.kv_heads;
  const int lpr = lanes_a_row(a.c.d, kPerLane<Q8>);
  if constexpr (!std::is_same<T, float>::value) {
    if (lpr != 0 && within(a.c, a.batch, a.t) && pages_on_grid(a.c) && on_grid(a.k, {a.k_sb, a.k_st, a.k_sh}, 2) && on_grid(a.v, {a.v_sb, a.v_st, a.v_sh}, 2)) {
      const dim3 grid(blocks_of(a.t * a.c.kv_heads * lpr, kThreadsPaged * kRowsAtOnce<Q8>), 2, (unsigned)a.batch), block(kThreadsPaged);
      const Divider heads = divider((uint32_t)a.c.kv_heads), page = divider((uint32_t)a.c.page_size);
      const int64_t pdl = a.batch * a.t;
      switch (lpr) {
        case 1: launch_pdl(cache_write_kernel<T, Q8, 1>, grid, block, 0, s, 1, pdl, a, heads, page); return 1;
        case 2: launch_pdl(cache_write_kernel<T, Q8, 2>, grid, block, 0, s, 1, pdl, a, heads, page); return 1;
        case 4: launch_pdl(cache_write_kernel<T, Q8, 4>, grid, block, 0, s, 1, pdl, a, heads, page); return 1;
        case 8: launch_pdl(cache_write_kernel<T, Q8, 8>, grid, block, 0, s, 1, pdl, a, heads, page); return 1;
        case 16: launch_pdl(cache_write_kernel<T, Q8, 16>, grid, block, 0, s, 1, pdl, a, heads, page); return 1;
        case 32: launch_pdl(cache_write_kernel<T, Q8, 32>, grid, block, 0, s, 1, pdl, a, heads, page); return 1;
      }
    }
  }
  launch_pdl(cache_write_any_kernel<T, Q8>, dim3(blocks_of(rows, kThreadsPaged / 32), 2), dim3(kThreadsPaged), 0, s, 1, a.batch * a.t, a);
  return 0;
}

template <typename T, bool Q8>
int run_read(const CacheReadArgs& a, cudaStream_t s) {
  const int64_t rows = a.batch * a.len * a.c.kv_heads;
  const int lpr = lanes_a_row(a.c.d, 8);
  if constexpr (!std::is_same<T, float>::value) {
    if (lpr != 0 && within(a.c, a.batch, a.len) && pages_on_grid(a.c) && on_grid(a.k, {a.k_sb, a.k_st, a.k_sh}, 2) && on_grid(a.v, {a.v_sb, a.v_st, a.v_sh}, 2)) {
      const dim3 grid(blocks_of(a.len * a.c.kv_heads * lpr, kThreadsPaged * kRowsAtOnce<false>), 2, (unsigned)a.batch), block(kThreadsPaged);
      const Divider heads = divider((uint32_t)a.c.kv_heads), page = divider((uint32_t)a.c.page_size);
      const int64_t pdl = a.batch * a.len;
      switch (lpr) {
        case 1: launch_pdl(cache_read_kernel<T, Q8, 1>, grid, block, 0, s, 1, pdl, a, heads, page); return 1;
        case 2: launch_pdl(cache_read_kernel<T, Q8, 2>, grid, block, 0, s, 1, pdl, a, heads, page); return 1;
        case 4: launch_pdl(cache_read_kernel<T, Q8, 4>, grid, block, 0, s, 1, pdl, a, heads, page); return 1;
        case 8: launch_pdl(cache_read_kernel<T, Q8, 8>, grid, block, 0, s, 1, pdl, a, heads, page); return 1;
        case 16: launch_pdl(cache_read_kernel<T, Q8, 16>, grid, block, 0, s, 1, pdl, a, heads, page); return 1;
        case 32: launch_pdl(cache_read_kernel<T, Q8, 32>, grid, block, 0, s, 1, pdl, a, heads, page); return 1;
      }
    }
  }
  launch_pdl(cache_read_any_kernel<T, Q8>, dim3(blocks_of(rows, kThreadsPaged / 32), 2), dim3(kThreadsPaged), 0, s, 1, a.batch * a.len, a);
  return 0;
}

// `f` with the stream type and whether the pages hold 8 bits.
template <typename F>
int by_type(int dtype, bool q8, F&& f) {
  switch (dtype) {
    case SVODB_BF16: return q8 ? f(__nv_bfloat16{}, std::true_type{}) : f(__nv_bfloat16{}, std::false_type{});
    case SVODB_F16: return q8 ? f(__half{}, std::true_type{}) : f(__half{}, std::false_type{});
    default: return q8 ? f(float{}, std::true_type{}) : f(float{}, std::false_type{});
  }
}

}  // namespace

int launch_cache_write(const CacheWriteArgs& a, cudaStream_t s) {
  return by_type(a.dtype, a.c.dtype == SVODB_E4M3,
                 [&](auto t, auto q8) { return run_write<decltype(t), decltype(q8)::value>(a, s); });
}

int launch_cache_read(const CacheReadArgs& a, cudaStream_t s) {
  return by_type(a.dtype, a.c.dtype == SVODB_E4M3,
                 [&](auto t, auto q8) { return run_read<decltype(t), decltype(q8)::value>(a, s); });
}

int launch_attention_paged_exact(const PagedAttnArgs& a, cudaStream_t s) {
  return by_type(a.dtype, a.c.dtype == SVODB_E4M3, [&](auto t, auto q8) {
    launch_pdl(attention_paged_exact_kernel<decltype(t), decltype(q8)::value>, dim3((unsigned)(a.batch * a.t * a.heads)),
               dim3(128), 0, s, 1, a.batch * a.t, a);
    return 0;
  });
}

}  // namespace svodb
