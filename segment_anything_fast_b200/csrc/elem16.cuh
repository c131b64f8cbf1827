// The two 16-bit element types behind one name: eight of them (16 bytes) to and from fp32.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "rowquant.cuh"

namespace samb {

struct Bf16 {
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) { unpack8(u, f); }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) { return pack8(f); }
  static __device__ __forceinline__ float to_float(uint16_t v) { return __uint_as_float(uint32_t(v) << 16); }
  static __device__ __forceinline__ uint16_t from_float(float f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f)); }
  static __device__ __forceinline__ uint32_t pack2f(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static __device__ __forceinline__ float2 unpack2f(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
};

struct F16 {
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = unpack2f(w[j]);
      f[2 * j] = t.x;
      f[2 * j + 1] = t.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    return make_uint4(pack2f(f[0], f[1]), pack2f(f[2], f[3]), pack2f(f[4], f[5]), pack2f(f[6], f[7]));
  }
  static __device__ __forceinline__ float to_float(uint16_t v) { return __half2float(__ushort_as_half(v)); }
  static __device__ __forceinline__ uint16_t from_float(float f) { return __half_as_ushort(__float2half_rn(f)); }
  static __device__ __forceinline__ uint32_t pack2f(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack2f(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
};

}  // namespace samb
