// Values held as float, bfloat16 or IEEE half (enum scn_type), read and written as float.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "scn_common.cuh"

namespace scn {

inline bool type_known(int type) { return type == SCN_F32 || type == SCN_BF16 || type == SCN_F16; }
inline int type_bytes(int type) { return type == SCN_F32 ? 4 : 2; }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_float(float v); // rounded to nearest, ties to even
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// W consecutive values as one access of W * sizeof(T) bytes (at most 16), which their address has to be a multiple of.
template <int BYTES> struct Raw;
template <> struct Raw<2> { using type = unsigned short; };
template <> struct Raw<4> { using type = unsigned; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<16> { using type = uint4; };
template <class T, int W> union Pack {
  typename Raw<W * (int)sizeof(T)>::type raw;
  T v[W];
  __device__ Pack() {}
};
template <class T, int W> __device__ __forceinline__ Pack<T, W> load_pack(const T *p) {
  Pack<T, W> r;
  r.raw = __ldg((const typename Raw<W * (int)sizeof(T)>::type *)p);
  return r;
}

// Values 2 i and 2 i + 1 of a pack as floats.
template <int W> __device__ __forceinline__ float2 pair_of(const Pack<float, W> &p, int i) { return make_float2(p.v[2 * i], p.v[2 * i + 1]); }
template <int W> __device__ __forceinline__ float2 pair_of(const Pack<__half, W> &p, int i) { return __half22float2(((const __half2 *)p.v)[i]); }
template <int W> __device__ __forceinline__ float2 pair_of(const Pack<__nv_bfloat16, W> &p, int i) {
  const unsigned x = ((const unsigned *)p.v)[i];
  return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}

// Eight consecutive values, 32-byte (float), 16-byte (16-bit) aligned, as one access.
__device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
  asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]) : "l"(p) : "memory");
}
__device__ __forceinline__ void store8(float *p, const float (&x)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]),
               "f"(x[6]), "f"(x[7]) : "memory");
}
template <class T> __device__ __forceinline__ void load8_16(const T *p, float (&x)[8]) {
  Pack<T, 8> r;
  r.raw = *(const uint4 *)p;
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = to_float(r.v[k]);
}
template <class T> __device__ __forceinline__ void store8_16(T *p, const float (&x)[8]) {
  Pack<T, 8> r;
#pragma unroll
  for (int k = 0; k < 8; ++k) r.v[k] = from_float<T>(x[k]);
  *(uint4 *)p = r.raw;
}

// The statements with T naming the C++ type of a run-time scn_type.
#define SCN_DISPATCH_TYPE(type, T, ...)                                                     \
  switch (type) {                                                                           \
  case SCN_BF16: { using T = __nv_bfloat16; __VA_ARGS__; } break;                                  \
  case SCN_F16: { using T = __half; __VA_ARGS__; } break;                                          \
  default: { using T = float; __VA_ARGS__; } break;                                                \
  }

} // namespace scn
