// Pieces shared by the attention kernels that take the keys as the M of both contractions
// (attention_decode.cu over rows of keys, attention_paged_decode.cu over pages).
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace svodb {
namespace dec_parts {

constexpr int kKeys = 128;  // keys per block: the M of both MMAs
constexpr int kThreadsDec = 192;
constexpr int kBox = kKeys * 128;  // bytes of one 64-column box of 128 rows

// Powers of two the halves of a weight are scaled by: value, and the remainder once more.
template <typename T>
constexpr float kValueUp = std::is_same<T, __half>::value ? 128.f : 1.f;
template <typename T>
constexpr float kRestUp = std::is_same<T, __half>::value ? 2048.f : 1.f;

__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[16]) {
  tmem_ld16(taddr, r);
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(r[i]));  // no use moves above the wait
}

__device__ __forceinline__ float redux_max(float x) {
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

// Named barrier over the 128 softmax threads that also ORs a predicate over them.
__device__ __forceinline__ bool barrier_or(int id, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred P, Q;\n\t"
      "setp.ne.u32 P, %1, 0;\n\t"
      "barrier.cta.red.or.pred Q, %2, 128, P;\n\t"
      "selp.u32 %0, 1, 0, Q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v), "r"(id)
      : "memory");
  return r != 0;
}

// The shared::cluster address of `addr` in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_at(uint32_t addr, uint32_t rank) {
  uint32_t out;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(addr), "r"(rank));
  return out;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Position of block j's K and V in the ring's order K0 K1 V0 K2 V1 ... K(n-1) V(n-2) V(n-1).
__device__ __forceinline__ uint32_t pos_k(int j) { return j == 0 ? 0u : (uint32_t)(2 * j - 1); }
__device__ __forceinline__ uint32_t pos_v(int j, int n) { return j == n - 1 ? (uint32_t)(2 * n - 1) : (uint32_t)(2 * j + 2); }

// Runs `f` on the first 4, 8 or 16 columns of a chunk: the least that holds `live` of them.
// The columns between are zero query rows: whatever is computed for them is never stored.
template <typename F>
__device__ __forceinline__ void by_width(int live, F&& f) {
  if (live <= 4) f(std::integral_constant<int, 4>{});
  else if (live <= 8) f(std::integral_constant<int, 8>{});
  else f(std::integral_constant<int, 16>{});
}

}  // namespace dec_parts
}  // namespace svodb
