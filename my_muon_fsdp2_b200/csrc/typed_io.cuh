// Vector loads and stores of VEC values of one type (bf16, fp16 or fp32) through one access of
// VEC * sizeof(T) bytes (2, 4, 8 or 16), held raw in registers and widened to fp32 for the
// arithmetic.  Rounding back is to nearest even, once for each stored value.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace mmf {

template <int BYTES>
struct RawBytes;
template <>
struct RawBytes<2> {
  using type = uint16_t;
};
template <>
struct RawBytes<4> {
  using type = uint32_t;
};
template <>
struct RawBytes<8> {
  using type = uint2;
};
template <>
struct RawBytes<16> {
  using type = uint4;
};
template <typename T, int VEC>
using Raw = typename RawBytes<VEC * static_cast<int>(sizeof(T))>::type;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}

__device__ __forceinline__ float2 widen2(uint32_t w, __nv_bfloat16) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
__device__ __forceinline__ float2 widen2(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ uint32_t narrow2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t narrow2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Raw<T, VEC>& r, float* v) {
  if constexpr (sizeof(T) == 4) {
    const float* f = reinterpret_cast<const float*>(&r);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = f[e];
  } else if constexpr (VEC == 1) {
    v[0] = to_f32(*reinterpret_cast<const T*>(&r));
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) {
      const float2 f = widen2(w[e], T());
      v[2 * e] = f.x;
      v[2 * e + 1] = f.y;
    }
  }
}

template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> pack(const float* v) {
  Raw<T, VEC> r;
  if constexpr (sizeof(T) == 4) {
    float* f = reinterpret_cast<float*>(&r);
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = v[e];
  } else if constexpr (VEC == 1) {
    const T t = from_f32<T>(v[0]);
    r = *reinterpret_cast<const uint16_t*>(&t);
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) w[e] = narrow2(v[2 * e], v[2 * e + 1], T());
  }
  return r;
}

template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> ld_raw(const T* p) {
  return *reinterpret_cast<const Raw<T, VEC>*>(p);
}
template <typename T, int VEC>
__device__ __forceinline__ void st_raw(T* p, const Raw<T, VEC>& r) {
  *reinterpret_cast<Raw<T, VEC>*>(p) = r;
}

}  // namespace mmf
