// Loads, stores and reductions shared by the row kernels around the attention (rotate.cu,
// norm.cu): eight consecutive values of a row per thread, held in fp32.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace recap {

// Programmatic launch: a kernel launched by launch_after() is set up while the one before it on the stream
// ends, and every thread waits in grid_wait() until that one is complete and its writes visible, before it
// touches global memory.  It takes the gap out of calls that follow one another (device times from the stream,
// us: 69 MB rotation 16.4 -> 14.4, 32760 x 1536 norm 53.2 -> 51.4, 4680 x 1536 gate and norm 20.5 -> 18.1);
// releasing the next kernel earlier, from inside the running one, gained nothing more.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename Args>
int launch_after(void (*kernel)(Args), dim3 grid, int threads, int smem, cudaStream_t s, const Args& a) {
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = s;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  if (cudaLaunchKernelEx(&config, kernel, a) == cudaSuccess) return kOk;
  cudaGetLastError();  // the error goes back as a code, not to a later call
  return kErrLaunch;
}

// Lets a kernel's blocks have `bytes` of dynamic shared memory.
template <typename Args>
bool allow_shared(void (*kernel)(Args), int bytes) {
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess) return true;
  cudaGetLastError();  // as above
  return false;
}

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

// The same for what all blocks read: it stays in L1 while rows stream past (gate and norm of 32760 x 5120, fp32
// modulations: 304 us, without the hint 306; at the power limit 326 and 330).
__device__ __forceinline__ uint4 ld_v4_keep(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::evict_last.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ uint2 ld_v2_keep(const void* p) {
  uint2 v;
  asm volatile("ld.global.L1::evict_last.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

// Asynchronous copies from global to shared memory, in groups that the issuing thread waits for.
__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy8(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the last n committed groups of this thread have landed.
template <int n>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory");
}

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
// Values p[0 .. 4) as the first four.
template <typename T>
__device__ __forceinline__ void load4(Raw8<T>& r, const T* p) {
  if constexpr (sizeof(T) == 4) {
    const uint4 a = ld_v4(p);
    r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w;
  } else {
    const uint2 a = ld_v2(p);
    r.w[0] = a.x, r.w[1] = a.y;
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
__device__ __forceinline__ void store4(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4)
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  else
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
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

template <typename T>
__device__ __forceinline__ void zero8(Raw8<T>& r) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(2 * sizeof(T)); ++i) r.w[i] = 0;
}

// Eight values at p[at] of a parameter vector whose type is known at run time (norm weights
// and biases, modulations), as loaded and widened; the address is aligned to 16 bytes.
struct RawParam8 {
  uint32_t w[8];
};
// kSplit: two runs of four values at at0 and at1, else eight values at at0.
template <bool kSplit>
__device__ __forceinline__ void load_param_raw(RawParam8& r, const void* p, int64_t at0, int64_t at1, int type) {
  if (type == kTypeF32) {
    const float* f = static_cast<const float*>(p);
    const uint4 a = ld_v4_keep(f + at0), b = ld_v4_keep(f + (kSplit ? at1 : at0 + 4));
    r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w, r.w[4] = b.x, r.w[5] = b.y, r.w[6] = b.z, r.w[7] = b.w;
  } else if (kSplit) {
    const uint16_t* h = static_cast<const uint16_t*>(p);
    const uint2 a = ld_v2_keep(h + at0), b = ld_v2_keep(h + at1);
    r.w[0] = a.x, r.w[1] = a.y, r.w[2] = b.x, r.w[3] = b.y;
  } else {
    const uint4 a = ld_v4_keep(static_cast<const uint16_t*>(p) + at0);
    r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w;
  }
}
__device__ __forceinline__ void widen_param8(float (&x)[8], const RawParam8& r, int type) {
  if (type == kTypeF32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(r.w[i]);
  } else if (type == kTypeBf16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<__nv_bfloat16>(r.w[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<__half>(r.w[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
}
// Eight values of kBytes (2 or 4) each at a byte address, as loaded.
template <bool kSplit, int kBytes>
__device__ __forceinline__ void load_own(uint32_t (&w)[2 * kBytes], const void* row, int c0, int c1) {
  const char* p = static_cast<const char*>(row);
  if constexpr (kBytes == 4) {
    const uint4 a = ld_v4(p + c0 * 4), b = ld_v4(p + c1 * 4);
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
  } else if constexpr (kSplit) {
    const uint2 a = ld_v2(p + c0 * 2), b = ld_v2(p + c1 * 2);
    w[0] = a.x, w[1] = a.y, w[2] = b.x, w[3] = b.y;
  } else {
    const uint4 a = ld_v4(p + c0 * 2);
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
  }
}
template <bool kSplit>
__device__ __forceinline__ void load_param(float (&x)[8], const void* p, int64_t at0, int64_t at1, int type) {
  RawParam8 r;
  load_param_raw<kSplit>(r, p, at0, at1, type);
  widen_param8(x, r, type);
}

// Sum over aligned groups of N lanes, in every lane.
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace recap
