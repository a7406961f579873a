// The norms, gates and residual sums before and after a transformer block, in one pass.
//
// For each token, with x and branch rows of C values:
//   norm:  h = (norm(x) w + b) (1 + scale) + shift
//   gate:  x' = residual + gate norm_b(branch),  and of that x' the same h on the way
// where norm is layer norm or root mean square over the C values, and scale, shift and gate are
// vectors of C values that a batch shares, or one of its samples, or that belong to one token.
//
// Bound by memory: every row is read once and written once and lies in registers between.  A
// row lies on one block of W warps, kVec times eight values per thread; the sums go over lanes
// and then over the warps through shared memory.  Modulations that many rows share come from
// L1 and L2 after the first.  h is formed from the fp32 x', not from its rounded copy: one
// rounding instead of two.
#include "elements.cuh"

namespace recap {
namespace {

constexpr int kMaxVec = 4;     // vectors of eight values a thread holds of a row
constexpr int kMaxWarps = 16;  // warps of a row

// Sum over the block, in every thread.  `buf` holds one float per warp; two calls in a row use
// different buffers, so that one barrier each is enough.
__device__ __forceinline__ float block_sum(float v, float* buf, int warps) {
  v = lanes_sum<32>(v);
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < warps; ++i) s += buf[i];
  return s;
}

// norm(x) in place: the row mean (layer norm), then the mean square, in two sums.
template <int kVec>
__device__ __forceinline__ void norm_rows(float (&x)[kVec][8], int layer, int C, float eps, float* buf, int warps) {
  const float inv = 1.f / static_cast<float>(C);
  if (layer) {
    float m = 0.f;
#pragma unroll
    for (int v = 0; v < kVec; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) m += x[v][j];
    m = block_sum(m, buf, warps) * inv;
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      const bool in = (v * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * 8 < C;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[v][j] = in ? x[v][j] - m : 0.f;
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int v = 0; v < kVec; ++v)
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(x[v][j], x[v][j], ss);
  const float r = rsqrtf(block_sum(ss, buf + kMaxWarps, warps) * inv + eps);
#pragma unroll
  for (int v = 0; v < kVec; ++v)
#pragma unroll
    for (int j = 0; j < 8; ++j) x[v][j] *= r;
}

// x = x * weight + bias with weight and bias optional parameter vectors
__device__ __forceinline__ void affine8(float (&x)[8], const void* w, const void* b, int64_t at, int type) {
  float p[8];
  if (w != nullptr) {
    load_param<8>(p, w, at, type);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= p[j];
  }
  if (b != nullptr) {
    load_param<8>(p, b, at, type);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] += p[j];
  }
}

// Values [at, at + 8) of modulation m (0 scale, 1 shift, 2 gate) for sample b, token s.
__device__ __forceinline__ void modulation8(float (&p)[8], const NormArgs& a, int m, int b, int s, int at) {
  load_param<8>(p, a.mod[m], b * a.mod_stride[m][0] + s * a.mod_stride[m][1] + at, a.mod_type);
}

template <typename TX, typename TH, int kVec, bool kGate>
__global__ void __launch_bounds__(kMaxWarps * 32) norm_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float buf[4 * kMaxWarps];
  const int warps = blockDim.x >> 5;
  const int b = blockIdx.x / a.S;
  const int s = blockIdx.x - b * a.S;
  const int C = a.C;
  const TX* xr = static_cast<const TX*>(a.x) + b * a.x_stride[0] + s * a.x_stride[1];
  float x[kVec][8];
  Raw8<TX> rx[kVec];
  Raw8<TH> ry[kGate ? kVec : 1];
#pragma unroll
  for (int v = 0; v < kVec; ++v) {
    const int at = (v * blockDim.x + threadIdx.x) * 8;
    if (at < C) {
      load8(rx[v], xr + at);
      if constexpr (kGate)
        load8(ry[v], static_cast<const TH*>(a.branch) + b * a.branch_stride[0] + s * a.branch_stride[1] + at);
    }
  }
  if constexpr (kGate) {
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[v][j] = 0.f;
      if (static_cast<int>(v * blockDim.x + threadIdx.x) * 8 < C) widen8(x[v], ry[v]);
    }
    if (a.branch_norm != kNormNone) norm_rows(x, a.branch_norm == kNormLayer, C, a.branch_eps, buf, warps);
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      const int at = (v * blockDim.x + threadIdx.x) * 8;
      if (at < C) {
        affine8(x[v], a.branch_weight, a.branch_bias, at, a.branch_weight_type);
        float p[8];
        if (a.mod[2] != nullptr) {
          modulation8(p, a, 2, b, s, at);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[v][j] *= p[j];
        }
        widen8(p, rx[v]);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[v][j] += p[j];
        store8(static_cast<TX*>(a.x_out) + b * a.x_out_stride[0] + s * a.x_out_stride[1] + at, x[v]);
      }
    }
    if (a.norm == kNormNone) return;
  } else {
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[v][j] = 0.f;
      if (static_cast<int>(v * blockDim.x + threadIdx.x) * 8 < C) widen8(x[v], rx[v]);
    }
  }
  norm_rows(x, a.norm == kNormLayer, C, a.eps, buf + 2 * kMaxWarps, warps);
#pragma unroll
  for (int v = 0; v < kVec; ++v) {
    const int at = (v * blockDim.x + threadIdx.x) * 8;
    if (at < C) {
      affine8(x[v], a.weight, a.bias, at, a.weight_type);
      float p[8];
      if (a.mod[0] != nullptr) {
        modulation8(p, a, 0, b, s, at);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[v][j] = fmaf(x[v][j], p[j], x[v][j]);
      }
      if (a.mod[1] != nullptr) {
        modulation8(p, a, 1, b, s, at);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[v][j] += p[j];
      }
      store8(static_cast<TH*>(a.h) + b * a.h_stride[0] + s * a.h_stride[1] + at, x[v]);
    }
  }
}



template <typename TX, typename TH, int kVec>
int launch_gate(const NormArgs& a, int threads, cudaStream_t s) {
  const unsigned rows = static_cast<unsigned>(static_cast<int64_t>(a.batch) * a.S);
  if (a.branch != nullptr)
    norm_kernel<TX, TH, kVec, true><<<rows, threads, 0, s>>>(a);
  else
    norm_kernel<TX, TH, kVec, false><<<rows, threads, 0, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

template <typename TX, typename TH>
int launch_vec(const NormArgs& a, cudaStream_t s) {
  // the fewest warps that hold a row at kMaxVec vectors a thread, then the fewest vectors
  const int vecs = a.C / 8;
  int warps = 1;
  while (warps * 32 * kMaxVec < vecs) warps *= 2;
  const int per = (vecs + warps * 32 - 1) / (warps * 32);
  const int threads = warps * 32;
  if (per == 1) return launch_gate<TX, TH, 1>(a, threads, s);
  if (per == 2) return launch_gate<TX, TH, 2>(a, threads, s);
  if (per == 3) return launch_gate<TX, TH, 3>(a, threads, s);
  return launch_gate<TX, TH, 4>(a, threads, s);
}

}  // namespace

int norm_max_channels() { return kMaxWarps * 32 * kMaxVec * 8; }

int launch_norm_rows(const NormArgs& a, cudaStream_t s) {
  if (a.x_type == kTypeBf16 && a.h_type == kTypeBf16) return launch_vec<__nv_bfloat16, __nv_bfloat16>(a, s);
  if (a.x_type == kTypeF16 && a.h_type == kTypeF16) return launch_vec<__half, __half>(a, s);
  if (a.x_type == kTypeF32 && a.h_type == kTypeF32) return launch_vec<float, float>(a, s);
  if (a.x_type == kTypeF32 && a.h_type == kTypeBf16) return launch_vec<float, __nv_bfloat16>(a, s);
  if (a.x_type == kTypeF32 && a.h_type == kTypeF16) return launch_vec<float, __half>(a, s);
  return kErrUnsupported;
}

}  // namespace recap
