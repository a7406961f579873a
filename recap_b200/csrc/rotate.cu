// Query/key norm and rotary positions of several axes, in one pass over q and k.
//
// For token n and head h the row x [D] of q or k becomes
//   y = norm(x)                        none, root mean square or layer norm over the D values
//                                      (weight, bias [D]), or root mean square over all heads
//                                      of the token (weight [heads D]);
//   (y_a, y_b) -> (y_a c - y_b s, y_a s + y_b c)   for every pair p of turned values,
// with c, s = cos, sin of 2 pi (position[axis p](n) turns_p + phase_p).  The angle is kept in
// turns as a 64-bit fixed-point fraction: position * turns_p wraps modulo one turn by itself,
// so a position of any size has an angle exact to 2^-32 of a turn, with no table and no
// reduction of a large float.  Values past the turned ones, and tokens outside the grid (text),
// are only normalised.
//
// Bound by memory: each row is read once and written once, everything between stays in
// registers.  A row lies on kLanes lanes (8, 16 or 32 for head dims up to 64, 128 and 256), 16
// bytes of bf16 each; those lanes form a group.  A token's cosines depend on the token and the
// pair only, so a group computes its lane's four once and then walks the heads of its token,
// kBatch rows in flight at a time.  `split` groups share the heads of one token: more of them
// where tokens are few.
#include "elements.cuh"

namespace recap {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 4;       // rows of a group in flight
constexpr int kAcrossRows = 8;  // rows a group holds in registers for a norm across heads

// cos and sin of the lane's four pairs of the token; returns a bit for each turned pair.
__device__ __forceinline__ uint32_t token_angles(const RotateArgs& a, const uint64_t* turns, const uint64_t* phase,
                                                 const uint8_t* axis, int b, int s, int pair0, float (&c)[4],
                                                 float (&sn)[4]) {
  if (pair0 >= a.pairs) return 0;
  int64_t pos[kMaxAxes];
  if (a.position_bits == 0) {
    const int64_t v = a.first_token + s - a.video_offset;
    if (v < 0 || v >= a.video_tokens) return 0;
    int rest = static_cast<int>(v);
#pragma unroll
    for (int i = kMaxAxes - 1; i >= 0; --i) {
      pos[i] = 0;
      if (i < a.axes) {
        const int q = rest / a.grid[i];
        pos[i] = rest - q * a.grid[i];
        rest = q;
      }
    }
  } else {
    const int64_t at = b * a.position_stride[0] + s * a.position_stride[1];
#pragma unroll
    for (int i = 0; i < kMaxAxes; ++i) {
      pos[i] = 0;
      if (i < a.axes)
        pos[i] = a.position_bits == 64 ? static_cast<const int64_t*>(a.positions)[at + i * a.position_stride[2]]
                                       : static_cast<const int32_t*>(a.positions)[at + i * a.position_stride[2]];
    }
  }
  uint32_t turned = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int p = pair0 + j;
    c[j] = 1.f;
    sn[j] = 0.f;
    if (p >= a.pairs) continue;
    const int ax = axis[p];
    uint64_t n = static_cast<uint64_t>(pos[0]);
#pragma unroll
    for (int i = 1; i < kMaxAxes; ++i)
      if (ax == i) n = static_cast<uint64_t>(pos[i]);
    const uint64_t t = n * turns[p] + phase[p];
    // the top 32 bits as a signed fraction of half a turn: the angle is pi times it
    sincospif(static_cast<float>(static_cast<int32_t>(t >> 32)) * 0x1p-31f, &sn[j], &c[j]);
    turned |= 1u << j;
  }
  return turned;
}

template <typename TI, typename TO, int kLanes, int kNorm, bool kHalves>
__global__ void __launch_bounds__(kThreads) rotate_kernel(const __grid_constant__ RotateArgs a) {
  constexpr int kGroups = kThreads / kLanes;
  constexpr int kRows = kNorm == kNormRmsAcross ? kAcrossRows : kBatch;
  __shared__ uint64_t s_turns[kMaxPairs], s_phase[kMaxPairs];
  __shared__ uint8_t s_axis[kMaxPairs];
  __shared__ float s_sum[kGroups];

  const int t = blockIdx.y;  // 0: q, 1: k
  const int tid = threadIdx.x;
  const int lane = tid % kLanes;
  const int group = tid / kLanes;
  const int split = 1 << a.split_log2[t];
  const int tokens = kGroups >> a.split_log2[t];  // tokens of this block
  // neighbouring groups take neighbouring tokens of a head, or neighbouring heads of a token,
  // whichever lie closer in memory
  const int slot = a.token_fast[t] ? group / tokens : group % split;
  const int token = a.token_fast[t] ? group % tokens : group / split;
  const int64_t flat = static_cast<int64_t>(blockIdx.x) * tokens + token;
  const bool live = flat < static_cast<int64_t>(a.batch) * a.S;
  const int b = live ? static_cast<int>(flat / a.S) : 0;
  const int s = live ? static_cast<int>(flat - static_cast<int64_t>(b) * a.S) : 0;

  // The lane's eight values of a row: two runs of four.  Halves pair value i with value
  // pairs + i, so turned lanes take four of each half; values past the turned ones follow.
  int d0 = lane * 8, d1 = d0 + 4;
  int pair0 = lane * 4;
  if (kHalves && lane * 4 < a.pairs) {
    d0 = lane * 4;
    d1 = a.pairs + d0;
  }
  const bool in_row = lane * 8 < a.D;
  const int heads = a.heads[t];
  const TI* src = static_cast<const TI*>(a.x[t]) + b * a.x_stride[t][0] + s * a.x_stride[t][2];
  TO* dst = static_cast<TO*>(a.out[t]) + b * a.out_stride[t][0] + s * a.out_stride[t][2];

  Raw8<TI> raw[kRows];
  auto load_rows = [&](int h0) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int h = h0 + i * split;
      if (live && in_row && h < heads) {
        const TI* row = src + h * a.x_stride[t][1];
        if constexpr (kHalves)
          load4x2(raw[i], row + d0, row + d1);
        else
          load8(raw[i], row + d0);
      } else {
#pragma unroll
        for (int j = 0; j < static_cast<int>(2 * sizeof(TI)); ++j) raw[i].w[j] = 0;
      }
    }
  };
  load_rows(slot);

  for (int i = tid; i < a.pairs; i += kThreads) {
    s_turns[i] = a.turns[i];
    s_phase[i] = a.phase[i];
    s_axis[i] = a.axis[i];
  }
  __syncthreads();

  float c[4], sn[4];
  uint32_t turned = 0;
  if (live && in_row) turned = token_angles(a, s_turns, s_phase, s_axis, b, s, pair0, c, sn);

  constexpr bool kPerHead = kNorm == kNormRms || kNorm == kNormLayer;
  float w[8], bias[8];
  if (kPerHead) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = 1.f;
      bias[i] = 0.f;
    }
    if (in_row && a.weight[t] != nullptr) {
      load_param<4>(w, a.weight[t], d0, a.weight_type);
      load_param<4>(w + 4, a.weight[t], d1, a.weight_type);
    }
    if (in_row && kNorm == kNormLayer && a.bias[t] != nullptr) {
      load_param<4>(bias, a.bias[t], d0, a.weight_type);
      load_param<4>(bias + 4, a.bias[t], d1, a.weight_type);
    }
  }

  auto finish = [&](float (&x)[8], int h) {
    if (turned != 0) {
      float y[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i0 = kHalves ? j : 2 * j, i1 = kHalves ? j + 4 : 2 * j + 1;
        y[i0] = x[i0] * c[j] - x[i1] * sn[j];
        y[i1] = x[i0] * sn[j] + x[i1] * c[j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i0 = kHalves ? j : 2 * j, i1 = kHalves ? j + 4 : 2 * j + 1;
        // an unturned value is passed on as it is, an infinity beside it included
        if ((turned >> j) & 1) x[i0] = y[i0], x[i1] = y[i1];
      }
    }
    TO* row = dst + h * a.out_stride[t][1];
    if constexpr (kHalves)
      store4x2(row + d0, row + d1, x);
    else
      store8(row + d0, x);
  };

  if constexpr (kNorm == kNormRmsAcross) {
    // every row of the token is in registers: the sum of squares over the groups' rows, then
    // the rows again
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      float x[8];
      widen8(x, raw[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
    }
    ss = lanes_sum<kLanes>(ss);
    if (lane == 0) s_sum[group] = ss;
    __syncthreads();
    ss = 0.f;
    for (int i = 0; i < split; ++i) ss += s_sum[a.token_fast[t] ? i * tokens + token : token * split + i];
    const float r = rsqrtf(ss / (static_cast<float>(heads) * a.D) + a.eps[t]);
    if (!live || !in_row) return;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int h = slot + i * split;
      if (h < heads) {
        float x[8], wr[8];
        widen8(x, raw[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) wr[j] = 1.f;
        if (a.weight[t] != nullptr) {
          load_param<4>(wr, a.weight[t], static_cast<int64_t>(h) * a.D + d0, a.weight_type);
          load_param<4>(wr + 4, a.weight[t], static_cast<int64_t>(h) * a.D + d1, a.weight_type);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= r * wr[j];
        finish(x, h);
      }
    }
  } else {
    const float inv_d = 1.f / static_cast<float>(a.D);
    // every group of a warp takes the same number of turns, so that the sums over lanes meet
    for (int h0 = slot; h0 - slot < heads; h0 += kRows * split) {
      if (h0 != slot) load_rows(h0);
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int h = h0 + i * split;
        float x[8];
        widen8(x, raw[i]);
        if constexpr (kPerHead) {
          if constexpr (kNorm == kNormLayer) {
            float m = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) m += x[j];
            m = lanes_sum<kLanes>(m) * inv_d;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = in_row ? x[j] - m : 0.f;
          }
          float ss = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
          const float r = rsqrtf(lanes_sum<kLanes>(ss) * inv_d + a.eps[t]);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = kNorm == kNormLayer ? fmaf(x[j] * r, w[j], bias[j]) : x[j] * r * w[j];
        }
        if (live && in_row && h < heads) finish(x, h);
      }
    }
  }
}

template <typename TI, typename TO, int kLanes, int kNorm>
int launch_pairs(const RotateArgs& a, dim3 grid, cudaStream_t s) {
  if (a.halves)
    rotate_kernel<TI, TO, kLanes, kNorm, true><<<grid, kThreads, 0, s>>>(a);
  else
    rotate_kernel<TI, TO, kLanes, kNorm, false><<<grid, kThreads, 0, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

template <typename TI, typename TO, int kLanes>
int launch_norm(const RotateArgs& a, dim3 grid, cudaStream_t s) {
  switch (a.norm) {
    case kNormNone: return launch_pairs<TI, TO, kLanes, kNormNone>(a, grid, s);
    case kNormRms: return launch_pairs<TI, TO, kLanes, kNormRms>(a, grid, s);
    case kNormLayer: return launch_pairs<TI, TO, kLanes, kNormLayer>(a, grid, s);
    case kNormRmsAcross: return launch_pairs<TI, TO, kLanes, kNormRmsAcross>(a, grid, s);
  }
  return kErrUnsupported;
}

template <typename TI, typename TO>
int launch_lanes(const RotateArgs& a, int lanes, dim3 grid, cudaStream_t s) {
  if (lanes == 8) return launch_norm<TI, TO, 8>(a, grid, s);
  if (lanes == 16) return launch_norm<TI, TO, 16>(a, grid, s);
  return launch_norm<TI, TO, 32>(a, grid, s);
}

}  // namespace

int rotate_max_heads_across(int D) { return kThreads / (D <= 64 ? 8 : D <= 128 ? 16 : 32) * kAcrossRows; }

int launch_rotate(RotateArgs& a, cudaStream_t s) {
  const int lanes = a.D <= 64 ? 8 : a.D <= 128 ? 16 : 32;
  const int groups = kThreads / lanes;
  const int64_t tokens = static_cast<int64_t>(a.batch) * a.S;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  int64_t blocks = 0;
  for (int t = 0; t < 2; ++t) {
    int log2 = 0;
    // share a token's heads among more groups while a group would still have a row of its own
    // and the blocks do not fill the device, or while a norm across heads does not fit
    while ((1 << log2) < groups && (1 << log2) < a.heads[t] &&
           ((a.norm == kNormRmsAcross && (a.heads[t] + (1 << log2) - 1) >> log2 > kAcrossRows) ||
            2 * ((tokens << log2) + groups - 1) / groups < 4 * sms))
      ++log2;
    a.split_log2[t] = log2;
    const int64_t n = ((tokens << log2) + groups - 1) / groups;
    blocks = n > blocks ? n : blocks;
    a.token_fast[t] = a.x_stride[t][2] < a.x_stride[t][1];
  }
  const dim3 grid(static_cast<unsigned>(blocks), a.heads[1] > 0 ? 2 : 1);
  if (a.in_type == kTypeBf16 && a.out_type == kTypeBf16)
    return launch_lanes<__nv_bfloat16, __nv_bfloat16>(a, lanes, grid, s);
  if (a.in_type == kTypeF16 && a.out_type == kTypeF16) return launch_lanes<__half, __half>(a, lanes, grid, s);
  if (a.in_type == kTypeF32 && a.out_type == kTypeF32) return launch_lanes<float, float>(a, lanes, grid, s);
  if (a.in_type == kTypeF16 && a.out_type == kTypeBf16) return launch_lanes<__half, __nv_bfloat16>(a, lanes, grid, s);
  if (a.in_type == kTypeF32 && a.out_type == kTypeBf16) return launch_lanes<float, __nv_bfloat16>(a, lanes, grid, s);
  return kErrUnsupported;
}

}  // namespace recap
