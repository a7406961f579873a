// Loads, stores and reductions shared by the row kernels around the attention (rotate.cu,
// norm.cu): eight consecutive values of a row per thread, held in fp32.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace recap {

// Two 16-bit values of a 32-bit word <-> fp32 (bf16 widens by a shift; fp16 converts).
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  return pack_bf16(a, b);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Eight values of type T as loaded, not yet widened: 4 or 8 registers.
template <typename T>
struct Raw8 {
  uint32_t w[2 * sizeof(T)];
};

// 8 and 16 bytes without a cache hint (plain loads: the inputs may be the outputs).
__device__ __forceinline__ uint4 ld_v4(const void* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ uint2 ld_v2(const void* p) { return *reinterpret_cast<const uint2*>(p); }

// Values p[0 .. 8).
template <typename T>
__device__ __forceinline__ void load8(Raw8<T>& r, const T* p) {
  const uint4 a = ld_v4(p);
  r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w;
  if constexpr (sizeof(T) == 4) {
    const uint4 b = ld_v4(p + 4);
    r.w[4] = b.x, r.w[5] = b.y, r.w[6] = b.z, r.w[7] = b.w;
  }
}
// Values p[0 .. 4) and q[0 .. 4).
template <typename T>
__device__ __forceinline__ void load4x2(Raw8<T>& r, const T* p, const T* q) {
  if constexpr (sizeof(T) == 4) {
    const uint4 a = ld_v4(p), b = ld_v4(q);
    r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w;
    r.w[4] = b.x, r.w[5] = b.y, r.w[6] = b.z, r.w[7] = b.w;
  } else {
    const uint2 a = ld_v2(p), b = ld_v2(q);
    r.w[0] = a.x, r.w[1] = a.y, r.w[2] = b.x, r.w[3] = b.y;
  }
}
template <typename T>
__device__ __forceinline__ void widen8(float (&x)[8], const Raw8<T>& r) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(r.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<T>(r.w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
  }
}
template <typename T>
__device__ __forceinline__ void store4x2(T* p, T* q, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(q) = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
    *reinterpret_cast<uint2*>(q) = make_uint2(pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
  }
}

// Values p[at .. at + n) of a small parameter vector whose type is known at run time (norm
// weights and biases, modulations): n is 4 or 8, the address aligned to n values.
template <int N>
__device__ __forceinline__ void load_param(float* x, const void* p, int64_t at, int type) {
  if (type == kTypeF32) {
    const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float4 v = s[i];
      x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
    }
    return;
  }
  uint32_t w[N / 2];
  const uint16_t* s = static_cast<const uint16_t*>(p) + at;
  if constexpr (N == 8) {
    const uint4 v = ld_v4(s);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else {
    const uint2 v = ld_v2(s);
    w[0] = v.x, w[1] = v.y;
  }
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float2 f = type == kTypeBf16 ? unpack2<__nv_bfloat16>(w[i]) : unpack2<__half>(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

// Sum over aligned groups of N lanes, in every lane.
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace recap
