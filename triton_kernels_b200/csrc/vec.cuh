// 16-byte vector access for fp32 / bf16 rows, presented to the math as fp32 lanes.
#pragma once

#include "common.cuh"

namespace fluxb {

template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  float v[4];
  __device__ __forceinline__ void unpack(const uint4& t) {
    v[0] = __uint_as_float(t.x); v[1] = __uint_as_float(t.y);
    v[2] = __uint_as_float(t.z); v[3] = __uint_as_float(t.w);
  }
  __device__ __forceinline__ void load(const float* p) {
    float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
  }
  __device__ __forceinline__ void load_nc(const float* p) {
    float4 t = __ldg(reinterpret_cast<const float4*>(p));
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
  }
  __device__ __forceinline__ void store(float* p) const {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  float v[8];
  __device__ __forceinline__ void unpack(const uint4& t) {
    v[0] = bf16_lo(t.x); v[1] = bf16_hi(t.x); v[2] = bf16_lo(t.y); v[3] = bf16_hi(t.y);
    v[4] = bf16_lo(t.z); v[5] = bf16_hi(t.z); v[6] = bf16_lo(t.w); v[7] = bf16_hi(t.w);
  }
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    unpack(*reinterpret_cast<const uint4*>(p));
  }
  __device__ __forceinline__ void load_nc(const __nv_bfloat16* p) {
    unpack(__ldg(reinterpret_cast<const uint4*>(p)));
  }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const {
    uint4 t;
    t.x = pack_bf16(v[0], v[1]); t.y = pack_bf16(v[2], v[3]);
    t.z = pack_bf16(v[4], v[5]); t.w = pack_bf16(v[6], v[7]);
    *reinterpret_cast<uint4*>(p) = t;
  }
};

// Makes the compiler forget what it knows about a packed vector, so the fp32 widening is redone
// at each use instead of being kept live (which doubles the registers of a bf16 row).
__device__ __forceinline__ void forget(uint4& t) {
  asm volatile("" : "+r"(t.x), "+r"(t.y), "+r"(t.z), "+r"(t.w));
}

__device__ __forceinline__ uint4 ld_nc_u4(const void* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
// The same for kernels that may start before the one in front has ended: what they read is not constant for their whole
// life, and a load by the read-only path might be moved in front of the wait.  (As a volatile instruction it stays behind
// the wait, but may pass the stores of other elements, which a plain load may not.)
__device__ __forceinline__ uint4 ld_u4(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// One row from global into shared memory by an asynchronous bulk copy (16-byte multiples and alignment).
__device__ __forceinline__ void bulk_load_row(void* smem_dst, const void* gsrc, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
      :
      : "r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(gsrc)), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

}  // namespace fluxb
