// N neighbouring elements of type T as one load or store, and as fp32 values.
#pragma once
#include "common.cuh"

namespace llsa {

template <typename T, int N>
struct Vec;
template <>
struct Vec<__nv_bfloat16, 8> {
  using type = uint4;
  static __device__ __forceinline__ void unpack(const uint4& x, float* v) {
    v[0] = bf16_lo(x.x); v[1] = bf16_hi(x.x); v[2] = bf16_lo(x.y); v[3] = bf16_hi(x.y);
    v[4] = bf16_lo(x.z); v[5] = bf16_hi(x.z); v[6] = bf16_lo(x.w); v[7] = bf16_hi(x.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* v) {
    return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
  }
};
template <>
struct Vec<__nv_bfloat16, 4> {
  using type = uint2;
  static __device__ __forceinline__ void unpack(const uint2& x, float* v) {
    v[0] = bf16_lo(x.x); v[1] = bf16_hi(x.x); v[2] = bf16_lo(x.y); v[3] = bf16_hi(x.y);
  }
  static __device__ __forceinline__ uint2 pack(const float* v) { return make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])); }
};
template <>
struct Vec<float, 4> {
  using type = float4;
  static __device__ __forceinline__ void unpack(const float4& x, float* v) { v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; }
  static __device__ __forceinline__ float4 pack(const float* v) { return make_float4(v[0], v[1], v[2], v[3]); }
};
// element by element: rows on no particular boundary
template <typename T>
struct Two {
  T a, b;
};
template <typename T>
struct Vec<T, 2> {
  using type = Two<T>;
  static __device__ __forceinline__ void unpack(const Two<T>& x, float* v) { v[0] = to_f32<T>(x.a); v[1] = to_f32<T>(x.b); }
  static __device__ __forceinline__ Two<T> pack(const float* v) { return Two<T>{from_f32<T>(v[0]), from_f32<T>(v[1])}; }
};
template <typename T>
struct Vec<T, 1> {
  using type = T;
  static __device__ __forceinline__ void unpack(const T& x, float* v) { v[0] = to_f32<T>(x); }
  static __device__ __forceinline__ T pack(const float* v) { return from_f32<T>(v[0]); }
};

}  // namespace llsa
