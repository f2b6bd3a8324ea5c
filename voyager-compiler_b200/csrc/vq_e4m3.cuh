// E4M3 bytes to and from float, and the small reductions shared by the
// float32-scaled E4M3 kernels (norm, linear, key / value cache).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace vq {
namespace e4 {

constexpr uint32_t FULL = 0xFFFFFFFFu;
constexpr float QMAX = 448.0f;  // the largest E4M3 value, 1.75 * 2^8

// Two floats rounded to nearest-even E4M3, saturating at +-448 (NaN -> 0x7F):
// the byte of `lo` in bits 0-7, of `hi` in bits 8-15.
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint16_t b;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b) : "f"(hi), "f"(lo));
  return b;
}
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  return pack2(a, b) | (pack2(c, d) << 16);
}
// The two E4M3 bytes in bits 0-15 of `w` as an f16 pair (exact).
__device__ __forceinline__ uint32_t unpack2(uint32_t w) {
  uint32_t h;
  asm("{\n\t.reg .b16 t, u;\n\tmov.b32 {t, u}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}"
      : "=r"(h) : "r"(w));
  return h;
}
// ... and the two in bits 16-31.
__device__ __forceinline__ uint32_t unpack2_hi(uint32_t w) {
  uint32_t h;
  asm("{\n\t.reg .b16 t, u;\n\tmov.b32 {t, u}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, u;\n\t}"
      : "=r"(h) : "r"(w));
  return h;
}
__device__ __forceinline__ float2 half2f(uint32_t h) {
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}

__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t bf_pack(float lo, float hi) {
  __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&b);
}

// Element types of the kernels' float tensors: VEC elements of 16-byte
// loads, 8 elements as floats.
struct BF16 {
  using type = uint16_t;
  static __device__ __forceinline__ float load(const uint16_t* p) {
    return __uint_as_float((uint32_t)*p << 16);
  }
  static __device__ __forceinline__ void store(uint16_t* p, float v) {
    __nv_bfloat16 b = __float2bfloat16_rn(v);
    *p = *reinterpret_cast<uint16_t*>(&b);
  }
  // 8 elements as they lie in memory (to be held while the loads of others
  // are used) and as floats
  struct Raw {
    uint4 a;
  };
  static __device__ __forceinline__ Raw fetch8(const uint16_t* p) {
    return {__ldg(reinterpret_cast<const uint4*>(p))};
  }
  static __device__ __forceinline__ void widen8(const Raw& r, float (&v)[8]) {
    const uint4 u = r.a;
    v[0] = bf_lo(u.x), v[1] = bf_hi(u.x), v[2] = bf_lo(u.y), v[3] = bf_hi(u.y);
    v[4] = bf_lo(u.z), v[5] = bf_hi(u.z), v[6] = bf_lo(u.w), v[7] = bf_hi(u.w);
  }
  static __device__ __forceinline__ void load8(const uint16_t* p, float (&v)[8]) { widen8(fetch8(p), v); }
  static __device__ __forceinline__ void store8(uint16_t* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(bf_pack(v[0], v[1]), bf_pack(v[2], v[3]),
                                              bf_pack(v[4], v[5]), bf_pack(v[6], v[7]));
  }
};
struct F32 {
  using type = float;
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
  struct Raw {
    float4 a, b;
  };
  static __device__ __forceinline__ Raw fetch8(const float* p) {
    return {__ldg(reinterpret_cast<const float4*>(p)), __ldg(reinterpret_cast<const float4*>(p) + 1)};
  }
  static __device__ __forceinline__ void widen8(const Raw& r, float (&v)[8]) {
    v[0] = r.a.x, v[1] = r.a.y, v[2] = r.a.z, v[3] = r.a.w;
    v[4] = r.b.x, v[5] = r.b.y, v[6] = r.b.z, v[7] = r.b.w;
  }
  static __device__ __forceinline__ void load8(const float* p, float (&v)[8]) { widen8(fetch8(p), v); }
  static __device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
};

}  // namespace e4
}  // namespace vq
