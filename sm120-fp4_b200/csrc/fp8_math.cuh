// Shared pieces of the FP8 and router operators: element types, 16-byte loads as floats, maxima that keep NaN, E4M3 conversion.
#pragma once
#include "ptx.cuh"

namespace b200 {

enum { DT_BF16 = 0, DT_F32 = 1, DT_F16 = 2 };   // dtype codes of the C ABI

template <typename T> struct Elem;
template <> struct Elem<__nv_bfloat16> {
  static constexpr int kSize = 2;
  static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ __nv_bfloat16 make(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ void unpack(uint32_t w, float& a, float& b) { a = __uint_as_float(w << 16), b = __uint_as_float(w & 0xffff0000u); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
    return d;
  }
};
template <> struct Elem<__half> {
  static constexpr int kSize = 2;
  static __device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ __half make(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ void unpack(uint32_t w, float& a, float& b) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    a = f.x, b = f.y;
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
    return d;
  }
};
template <> struct Elem<float> {
  static constexpr int kSize = 4;
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ float make(float v) { return v; }
};

// 16 bytes of T as floats: eight of 16 bits, four of 32
template <typename T> __device__ __forceinline__ void unpack16(uint4 w, float* v) {
  if constexpr (Elem<T>::kSize == 2) {
    Elem<T>::unpack(w.x, v[0], v[1]), Elem<T>::unpack(w.y, v[2], v[3]), Elem<T>::unpack(w.z, v[4], v[5]), Elem<T>::unpack(w.w, v[6], v[7]);
  } else {
    v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
  }
}

// the larger of two, NaN where one is NaN (fmaxf drops it)
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// the largest of a warp's values, NaN where a lane has one; all lanes have to be here, so it stays where it is called
__device__ __forceinline__ float warp_max(float v) {
  float m;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
// four floats -> four E4M3 bytes, element order kept; to nearest, ties to even, saturating at 448, NaN kept
__device__ __forceinline__ uint32_t cvt_e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// Scale and factor of values whose largest magnitude is amax: scale = fl(amax / 448) is kept, factor = fl(448 / amax) is what values are
// multiplied by. The floor keeps a group of zeros finite. A NaN goes to both; an infinity gives scale inf and codes 0 (finite) and NaN (infinite).
struct Fp8Scale { float scale, factor; };
__device__ __forceinline__ Fp8Scale fp8_scale(float amax) {
  const float a = max_nan(amax, 1e-12f);
  return {__fdiv_rn(a, 448.f), __fdiv_rn(448.f, a)};
}

}  // namespace b200
