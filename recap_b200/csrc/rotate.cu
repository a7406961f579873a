// Query/key norm and rotary positions of several axes, in one pass over q and k.
//
// For token n and head h the row x [D] of q or k becomes
//   y = norm(x)                        none, root mean square or layer norm over the D values
//                                      (weight, bias [D]), or root mean square over all heads
//                                      of the token (weight [heads D]);
//   (y_a, y_b) -> (y_a c - y_b s, y_a s + y_b c)   for every pair p of turned values,
// with c, s = cos, sin of 2 pi (position[axis p](n) turns_p + phase_p).  The angle is kept in
// turns as a 64-bit fixed-point fraction: position * turns_p wraps modulo one turn by itself,
// so the angle of a position of any size is that of turns_p to 2^-32 of a turn, with no table and no
// reduction of a large float.  (turns_p is as good as its maker's: block.py rounds frequencies to 53 bits.)
// Values past the turned ones, and tokens outside the grid (text), are only normalised.
//
// Bound by memory: each row is read once and written once.  A row lies on kLanes lanes (8, 16 or
// 32 for head dims up to 64, 128 and 256), 16 bytes of bf16 each; those lanes form a group.  A
// token's cosines depend on the token and the pair only, so a group computes its lane's four
// once, folds the norm's weight into them, and then walks the heads of its token.  `split` groups
// share the heads of one token: more of them where tokens are few.  Next to memory the issue
// slots count: the arithmetic is packed two values an instruction, and the rows of a warp
// stay together without branches.  Measured on B200 (bf16): 24 heads of 128, 119056 tokens, rms
// norm: 441 us, 6.6 TB/s, the rate of a copy; 12 heads, 32760 tokens, rms across heads: 66 us, 6.1
// TB/s.  Under load for a tenth of a second the card reaches its power limit, the SM clock falls from 1.96
// to 1.6 GHz, and they take 452 and 71 us.
#include <type_traits>

#include "elements.cuh"

namespace recap {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 4;       // rows of a group in flight
// Most rows a group takes for a norm across heads: 16 rows of bf16 for all groups of a block are 64 KB,
// three blocks an SM.  (B200, 12 heads of 128, 32760 tokens, bf16: 68 us; at most 8, so two groups a
// token and their sum between: 78 us.)
constexpr int kAcrossRows = 16;
constexpr int kAcrossHeads = 8;  // limit of the heads: this many for each group of a block

__device__ __forceinline__ uint32_t divide(uint32_t n, const Divisor& d) {
  return static_cast<uint32_t>((static_cast<uint64_t>(n) * d.mul) >> d.shift);
}

// What a thread of either kernel works on.
template <int kLanes, bool kHalves>
struct Place {
  int lane, group, log2, split, slot, token, b, s, d0, d1, pair0;
  bool in_row, active;
  __device__ __forceinline__ explicit Place(const RotateArgs& a) {
    constexpr int kGroupsLog2 = kThreads / kLanes == 32 ? 5 : kThreads / kLanes == 16 ? 4 : 3;
    lane = threadIdx.x % kLanes;
    group = threadIdx.x / kLanes;
    log2 = a.split_log2;
    split = 1 << log2;
    const int tokens_log2 = kGroupsLog2 - log2;  // of the tokens of a block
    // neighbouring groups take neighbouring tokens of a head, or neighbouring heads of a token,
    // whichever lie closer in memory
    slot = a.token_fast ? group >> tokens_log2 : group & (split - 1);
    token = a.token_fast ? group & ((1 << tokens_log2) - 1) : group >> log2;
    const uint32_t flat = (blockIdx.x << tokens_log2) + token;
    const bool live = flat < a.tokens;
    b = live ? divide(flat, a.s_div) : 0;
    s = live ? flat - b * a.S : 0;
    // The lane's eight values of a row: two runs of four.  Halves pair value i with value
    // pairs + i, so turned lanes take four of each half; values past the turned ones follow.
    // A lane past the row reads its start and stores nothing.
    pair0 = lane * 4;
    in_row = lane * 8 < a.D;
    d0 = in_row ? lane * 8 : 0;
    d1 = d0 + 4;
    if (kHalves && pair0 < a.pairs) {
      d0 = pair0;
      d1 = a.pairs + d0;
    }
    active = live && in_row;
  }
};

// The turns of the pairs in shared memory: fraction of a turn per position (64 bits), phase
// (the top 32 bits), axis.
__device__ __forceinline__ void stage_pairs(const RotateArgs& a, uint4* s_pair) {
  for (int i = threadIdx.x; i < a.pairs; i += kThreads)
    s_pair[i] = make_uint4(static_cast<uint32_t>(a.turns[i]), static_cast<uint32_t>(a.turns[i] >> 32),
                           static_cast<uint32_t>(a.phase[i] >> 32), a.axis[i]);
}

// cos and sin of the lane's four pairs of the token; returns a bit for each turned pair, the others
// getting 1 and 0.
template <bool kFast>
__device__ __forceinline__ uint32_t token_angles(const RotateArgs& a, const uint4* s_pair, int b, int s, int pair0,
                                                 float (&c)[4], float (&sn)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c[j] = 1.f, sn[j] = 0.f;
  if (pair0 >= a.pairs) return 0;
  uint32_t lo[kMaxAxes], hi[kMaxAxes];  // the position, 64 bits
#pragma unroll
  for (int i = 0; i < kMaxAxes; ++i) lo[i] = hi[i] = 0;
  if (a.position_bits == 0) {
    const int64_t v = a.first_token + s - a.video_offset;
    if (v < 0 || v >= a.video_tokens) return 0;
    uint32_t rest = static_cast<uint32_t>(v);
#pragma unroll
    for (int i = kMaxAxes - 1; i >= 0; --i) {
      if (i < a.axes) {
        const uint32_t q = divide(rest, a.grid_div[i]);
        lo[i] = rest - q * a.grid[i];
        rest = q;
      }
    }
  } else {
    const int64_t at = b * a.position_stride[0] + s * a.position_stride[1];
#pragma unroll
    for (int i = 0; i < kMaxAxes; ++i) {
      if (i < a.axes) {
        const int64_t n = a.position_bits == 64 ? static_cast<const int64_t*>(a.positions)[at + i * a.position_stride[2]]
                                                : static_cast<const int32_t*>(a.positions)[at + i * a.position_stride[2]];
        lo[i] = static_cast<uint32_t>(n);
        hi[i] = static_cast<uint32_t>(n >> 32);
      }
    }
  }
  uint32_t turned = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (pair0 + j >= a.pairs) break;
    const uint4 f = s_pair[pair0 + j];
    uint32_t n = lo[0], nh = hi[0];
#pragma unroll
    for (int i = 1; i < kMaxAxes; ++i)
      if (i < a.axes && f.w == i) n = lo[i], nh = hi[i];
    // bits 32 .. 63 of the 64-bit product and the phase: a signed fraction of half a turn
    uint32_t t = __umulhi(n, f.x) + n * f.y + f.z;
    if (a.position_bits != 0) t += nh * f.x;
    const float half_turns = static_cast<float>(static_cast<int32_t>(t)) * 0x1p-31f;
    if constexpr (kFast) {
      // 16-bit outputs: sin.approx and cos.approx on [-pi, pi] are within 2^-21.1 of one, against the
      // 2^-9 and 2^-12 of the outputs' half step, for a seventh of the instructions
      __sincosf(half_turns * 3.14159265358979f, &sn[j], &c[j]);
    } else {
      sincospif(half_turns, &sn[j], &c[j]);
    }
    turned |= 1u << j;
  }
  return turned;
}

// A lane's eight values of a row as four pairs, first and second values apart.
template <typename T, bool kHalves>
__device__ __forceinline__ void widen_pairs(float (&xa)[4], float (&xb)[4], const Raw8<T>& r) {
  float x[8];
  widen8(x, r);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    xa[j] = kHalves ? x[j] : x[2 * j];
    xb[j] = kHalves ? x[j + 4] : x[2 * j + 1];
  }
}
template <bool kHalves>
__device__ __forceinline__ void load_param_pairs(float (&xa)[4], float (&xb)[4], const void* p, int64_t at0, int64_t at1,
                                                 int type) {
  float x[8];
  load_param<kHalves>(x, p, at0, at1, type);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    xa[j] = kHalves ? x[j] : x[2 * j];
    xb[j] = kHalves ? x[j + 4] : x[2 * j + 1];
  }
}
template <typename T, bool kHalves>
__device__ __forceinline__ void load_row(Raw8<T>& r, const T* row, int d0, int d1) {
  if constexpr (kHalves)
    load4x2(r, row + d0, row + d1);
  else
    load8(r, row + d0);
}
template <typename T, bool kHalves>
__device__ __forceinline__ void store_row(T* row, int d0, int d1, const float (&ya)[4], const float (&yb)[4]) {
  float y[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    y[kHalves ? j : 2 * j] = ya[j];
    y[kHalves ? j + 4 : 2 * j + 1] = yb[j];
  }
  if constexpr (kHalves)
    store4x2(row + d0, row + d1, y);
  else
    store8(row + d0, y);
}

__device__ __forceinline__ float square_sum(const float (&xa)[4], const float (&xb)[4]) {
  float s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int j = 0; j < 4; j += 2) {
    fma2(s0, s1, xa[j], xa[j + 1], xa[j], xa[j + 1], s0, s1);
    fma2(s0, s1, xb[j], xb[j + 1], xb[j], xb[j + 1], s0, s1);
  }
  return s0 + s1;
}

// (u, v) -> (u ca + v nsb, u sa + v cb) for the four pairs.  kFull: all of them turn in every lane of
// the warp; else an unturned value goes on without its neighbour, so that an infinity there stays there.
template <bool kFull>
__device__ __forceinline__ void turn(float (&xa)[4], float (&xb)[4], const float (&ca)[4], const float (&nsb)[4],
                                     const float (&sa)[4], const float (&cb)[4], uint32_t turned) {
  float ya[4], yb[4];
#pragma unroll
  for (int j = 0; j < 4; j += 2) {
    ya[j] = xa[j], ya[j + 1] = xa[j + 1], yb[j] = xb[j], yb[j + 1] = xb[j + 1];
    mul2(ya[j], ya[j + 1], ca[j], ca[j + 1]);
    mul2(yb[j], yb[j + 1], cb[j], cb[j + 1]);
    float za[2] = {ya[j], ya[j + 1]}, zb[2] = {yb[j], yb[j + 1]};
    fma2(ya[j], ya[j + 1], xb[j], xb[j + 1], nsb[j], nsb[j + 1], ya[j], ya[j + 1]);
    fma2(yb[j], yb[j + 1], xa[j], xa[j + 1], sa[j], sa[j + 1], yb[j], yb[j + 1]);
    if constexpr (!kFull) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (!((turned >> (j + k)) & 1)) ya[j + k] = za[k], yb[j + k] = zb[k];
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) xa[j] = ya[j], xb[j] = yb[j];
}

// No norm, or one within each head.  One tensor a block (blockIdx.y: q, k).  Four blocks an SM (three
// for fp32): the layer norm spills some registers for it and is faster all the same (48 heads of 64, two
// samples of 45106 tokens, fp16: 354 us, 0.96 of the copy rate; three blocks without spills 388 us).
template <typename TI, typename TO, int kLanes, int kNorm, bool kHalves>
__global__ void __launch_bounds__(kThreads, sizeof(TI) == 4 ? 3 : 4)
    rotate_kernel(const __grid_constant__ RotateArgs a) {
  __shared__ uint4 s_pair[kMaxPairs];
  const Place<kLanes, kHalves> me(a);
  const int d0 = me.d0, d1 = me.d1;
  const int t = blockIdx.y;
  // the group's rows are heads slot, slot + split, ...: `mine` of them (none for a lane past the row or a
  // group past the tokens), `most` in any group
  const int heads = a.heads[t];
  const int most = (heads + me.split - 1) >> me.log2;
  const int mine = me.active ? (heads - me.slot + me.split - 1) >> me.log2 : 0;
  const TI* src = static_cast<const TI*>(a.x[t]) + me.b * a.x_stride[t][0] + me.s * a.x_stride[t][2] +
                  (me.slot < heads ? me.slot : 0) * a.x_stride[t][1];
  // Every group has the same rows, in whole batches: nothing to ask for row by row, in the layer norm of 16-bit rows,
  // where issue slots count most.  (48 heads of 64, two samples of 45106 tokens, fp16: 354 us, asked 356; at the
  // card's power limit 377 and 387.  Root mean square: 24 heads of 128 447 and 452, but in halves of 64 42.8 and
  // 42.1, and fp32 rows 78 and 76 us.)
  constexpr bool kTryEven = kNorm == kNormLayer && sizeof(TI) == 2;
  const bool even = kTryEven && heads == (most << me.log2) && most % kBatch == 0;
  const int64_t x_step = me.active || !even ? a.x_stride[t][1] << me.log2 : 0;
  Raw8<TI> raw[kBatch];
  // A lane without a row of its own loads its last one again: no value has to be made up, and the
  // warp stays together.
  auto load_rows = [&](int i0, bool whole) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (!whole && i0 + i >= most) break;
      load_row<TI, kHalves>(raw[i], src, d0, d1);
      if (whole || i0 + i + 1 < mine) src += x_step;
    }
  };
  stage_pairs(a, s_pair);
  grid_wait();
  load_rows(0, even);
  __syncthreads();

  // a pair (u, v) of normalised values before weight and bias becomes
  //   (u ca + v nsb + ba, u sa + v cb + bb),   cb = ca where no weight is in them
  constexpr bool kWeights = kNorm != kNormNone;
  float ca[4], sa[4], nsb[4], cb_[4], ba[4], bb[4];
  uint32_t turned = 0;
  if (me.active) {
    turned = token_angles<sizeof(TO) == 2>(a, s_pair, me.b, me.s, me.pair0, ca, sa);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) ca[j] = 1.f, sa[j] = 0.f;
  }
  const bool full = __all_sync(0xffffffffu, turned == 0xf || !me.active);
  float(&cb)[4] = kWeights ? cb_ : ca;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    cb[j] = ca[j];
    nsb[j] = -sa[j];
    ba[j] = bb[j] = 0.f;
  }
  if constexpr (kWeights) {
    float wa[4], wb[4];
    if (kNorm == kNormLayer && a.bias[t] != nullptr) {
      load_param_pairs<kHalves>(wa, wb, a.bias[t], d0, d1, a.weight_type);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ba[j] = wa[j] * ca[j] - wb[j] * sa[j];
        bb[j] = wa[j] * sa[j] + wb[j] * ca[j];
      }
    }
    if (a.weight[t] != nullptr) {
      load_param_pairs<kHalves>(wa, wb, a.weight[t], d0, d1, a.weight_type);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ca[j] *= wa[j];
        sa[j] *= wa[j];
        nsb[j] *= wb[j];
        cb[j] *= wb[j];
      }
    }
  }

  TO* dst = static_cast<TO*>(a.out[t]) + me.b * a.out_stride[t][0] + me.s * a.out_stride[t][2] + me.slot * a.out_stride[t][1];
  const int64_t out_step = a.out_stride[t][1] << me.log2;
  const float inv_d = 1.f / static_cast<float>(a.D);
  const float eps = a.eps[t];
  auto walk = [&](auto full_tag, auto even_tag) {
    constexpr bool kEven = decltype(even_tag)::value;
    for (int i0 = 0; i0 < most; i0 += kBatch) {
      if (i0 != 0) load_rows(i0, kEven);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (!kEven && i0 + i >= most) break;
        float xa[4], xb[4];
        widen_pairs<TI, kHalves>(xa, xb, raw[i]);
        [[maybe_unused]] float r = 1.f;
        if constexpr (kNorm == kNormLayer) {
          float m0 = 0.f, m1 = 0.f;
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            add2(m0, m1, xa[j], xa[j + 1]);
            add2(m0, m1, xb[j], xb[j + 1]);
          }
          const float m = lanes_sum<kLanes>(me.in_row ? m0 + m1 : 0.f) * -inv_d;
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            add2(xa[j], xa[j + 1], m, m);
            add2(xb[j], xb[j + 1], m, m);
          }
        }
        if constexpr (kNorm != kNormNone) {
          const float ss = square_sum(xa, xb);
          r = rsqrtf(fmaf(lanes_sum<kLanes>(me.in_row ? ss : 0.f), inv_d, eps));
        }
        turn<decltype(full_tag)::value>(xa, xb, ca, nsb, sa, cb, turned);
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          if constexpr (kNorm == kNormLayer) {
            fma2(xa[j], xa[j + 1], xa[j], xa[j + 1], r, r, ba[j], ba[j + 1]);
            fma2(xb[j], xb[j + 1], xb[j], xb[j + 1], r, r, bb[j], bb[j + 1]);
          } else if constexpr (kNorm == kNormRms) {
            mul2(xa[j], xa[j + 1], r, r);
            mul2(xb[j], xb[j + 1], r, r);
          }
        }
        if (kEven ? me.active : i0 + i < mine) store_row<TO, kHalves>(dst, d0, d1, xa, xb);
        dst += out_step;
      }
    }
  };
  if (full && even)
    walk(std::true_type{}, std::bool_constant<kTryEven>{});
  else if (full)
    walk(std::true_type{}, std::false_type{});
  else
    walk(std::false_type{}, std::false_type{});
}

// Root mean square over all heads of a token.  One tensor a block, whose rows go to shared memory by
// asynchronous copies, each thread copying and reading its own values only: all of them are in flight
// at once, and registers hold one row at a time.  The sum of squares takes the first walk over the rows,
// its 1 / root goes into the cosines, and the second walk turns and stores.  Shared memory: the
// weights as fp32 (first and second values of the pairs apart, a lane's four beside the next
// lane's), then the rows.
template <typename TI, typename TO, int kLanes, bool kHalves>
__global__ void __launch_bounds__(kThreads, 4) rotate_across_kernel(const __grid_constant__ RotateArgs a) {
  constexpr int kVec = sizeof(TI) / 2;  // 16-byte slots of a lane's values
  __shared__ uint4 s_pair[kMaxPairs];
  __shared__ double s_sum[kThreads / kLanes];
  extern __shared__ uint4 s_dynamic[];
  const Place<kLanes, kHalves> me(a);
  const int d0 = me.d0, d1 = me.d1;
  const int t = blockIdx.y;
  const int heads = a.heads[t];
  const int mine = me.active ? (heads - me.slot + me.split - 1) >> me.log2 : 0;
  const bool weighted = a.weight[t] != nullptr;
  float4* weights = reinterpret_cast<float4*>(s_dynamic) + me.lane;
  uint4* rows = s_dynamic + (weighted ? heads * (2 * kLanes) : 0) + threadIdx.x;
  stage_pairs(a, s_pair);
  grid_wait();
  {
    const TI* src = static_cast<const TI*>(a.x[t]) + me.b * a.x_stride[t][0] + me.s * a.x_stride[t][2] + me.slot * a.x_stride[t][1];
    const int64_t x_step = a.x_stride[t][1] << me.log2;
    uint4* to = rows;
    for (int i = 0; i < mine; ++i) {
      if constexpr (kVec == 2) {
        copy16(to, src + d0);
        copy16(to + kThreads, src + d1);
      } else if constexpr (kHalves) {
        copy8(to, src + d0);
        copy8(reinterpret_cast<uint2*>(to) + 1, src + d1);
      } else {
        copy16(to, src + d0);
      }
      src += x_step;
      to += kVec * kThreads;
    }
    copies_commit();
  }
  if (weighted) {
    for (int h = me.group; h < heads; h += kThreads / kLanes) {
      float wa[4], wb[4];
      load_param_pairs<kHalves>(wa, wb, a.weight[t], h * a.D + d0, h * a.D + d1, a.weight_type);
      weights[h * (2 * kLanes)] = make_float4(wa[0], wa[1], wa[2], wa[3]);
      weights[h * (2 * kLanes) + kLanes] = make_float4(wb[0], wb[1], wb[2], wb[3]);
    }
  }
  __syncthreads();

  float ca[4], sa[4], nsb[4];
  uint32_t turned = 0;
  if (me.active) {
    turned = token_angles<sizeof(TO) == 2>(a, s_pair, me.b, me.s, me.pair0, ca, sa);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) ca[j] = 1.f, sa[j] = 0.f;
  }
  const bool full = __all_sync(0xffffffffu, turned == 0xf || !me.active);

  copies_wait<0>();
  auto read = [&](int i, float(&xa)[4], float(&xb)[4]) {
    Raw8<TI> raw;
    const uint4 v = rows[i * (kVec * kThreads)];
    raw.w[0] = v.x, raw.w[1] = v.y, raw.w[2] = v.z, raw.w[3] = v.w;
    if constexpr (kVec == 2) {
      const uint4 u = rows[i * (kVec * kThreads) + kThreads];
      raw.w[4] = u.x, raw.w[5] = u.y, raw.w[6] = u.z, raw.w[7] = u.w;
    }
    widen_pairs<TI, kHalves>(xa, xb, raw);
  };
  // The rows' sums are added in 64 bits, where sums of fp32 values of like size are exact: the result does not
  // depend on how many groups share a token, so a shard or a chunk of a sequence gives the bits of the whole.
  double sum = 0.;
#pragma unroll 2
  for (int i = 0; i < mine; ++i) {
    float xa[4], xb[4];
    read(i, xa, xb);
    sum += square_sum(xa, xb);
  }
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (!a.token_fast && me.split * kLanes <= 32) {
    for (int o = kLanes; o < me.split * kLanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  } else if (me.split > 1) {
    if (me.lane == 0) s_sum[me.token * me.split + me.slot] = sum;
    __syncthreads();
    sum = 0.;
    for (int i = 0; i < me.split; ++i) sum += s_sum[me.token * me.split + i];
  }
  const float total = static_cast<float>(sum);
  const float r = rsqrtf(total / (static_cast<float>(heads) * a.D) + a.eps[t]);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    ca[j] *= r;
    sa[j] *= r;
    nsb[j] = -sa[j];
  }
  TO* dst = static_cast<TO*>(a.out[t]) + me.b * a.out_stride[t][0] + me.s * a.out_stride[t][2] + me.slot * a.out_stride[t][1];
  const int64_t out_step = a.out_stride[t][1] << me.log2;
  const float4* wr = weights + me.slot * (2 * kLanes);
  auto walk = [&](auto full_tag) {
#pragma unroll 2
    for (int i = 0; i < mine; ++i) {
      float xa[4], xb[4];
      read(i, xa, xb);
      if (weighted) {
        const float4 wa = wr[0], wb = wr[kLanes];
        mul2(xa[0], xa[1], wa.x, wa.y);
        mul2(xa[2], xa[3], wa.z, wa.w);
        mul2(xb[0], xb[1], wb.x, wb.y);
        mul2(xb[2], xb[3], wb.z, wb.w);
        wr += (2 * kLanes) << me.log2;
      }
      turn<decltype(full_tag)::value>(xa, xb, ca, nsb, sa, ca, turned);
      store_row<TO, kHalves>(dst, d0, d1, xa, xb);
      dst += out_step;
    }
  };
  if (full)
    walk(std::true_type{});
  else
    walk(std::false_type{});
}

template <typename TI, typename TO, int kLanes, int kNorm, bool kHalves>
int launch_kernel(const RotateArgs& a, dim3 grid, int smem, cudaStream_t s) {
  if constexpr (kNorm == kNormRmsAcross) {
    auto* kernel = rotate_across_kernel<TI, TO, kLanes, kHalves>;
    // the most of any call, so that calls of two host threads set the same: rows of a group and the weights of all heads
    constexpr int kMost = kAcrossRows * kThreads * (sizeof(TI) == 4 ? 32 : 16) + kThreads / kLanes * kAcrossHeads * 2 * kLanes * 16;
    if (smem > 40 * 1024 && !allow_shared(kernel, kMost)) return kErrLaunch;
    return launch_after(kernel, grid, kThreads, smem, s, a);
  } else {
    return launch_after(rotate_kernel<TI, TO, kLanes, kNorm, kHalves>, grid, kThreads, 0, s, a);
  }
}

template <typename TI, typename TO, int kLanes, int kNorm>
int launch_pairs(const RotateArgs& a, dim3 grid, int smem, cudaStream_t s) {
  return a.halves ? launch_kernel<TI, TO, kLanes, kNorm, true>(a, grid, smem, s)
                  : launch_kernel<TI, TO, kLanes, kNorm, false>(a, grid, smem, s);
}

template <typename TI, typename TO, int kLanes>
int launch_norm(const RotateArgs& a, dim3 grid, int smem, cudaStream_t s) {
  switch (a.norm) {
    case kNormNone: return launch_pairs<TI, TO, kLanes, kNormNone>(a, grid, smem, s);
    case kNormRms: return launch_pairs<TI, TO, kLanes, kNormRms>(a, grid, smem, s);
    case kNormLayer: return launch_pairs<TI, TO, kLanes, kNormLayer>(a, grid, smem, s);
    case kNormRmsAcross: return launch_pairs<TI, TO, kLanes, kNormRmsAcross>(a, grid, smem, s);
  }
  return kErrUnsupported;
}

template <typename TI, typename TO>
int launch_lanes(const RotateArgs& a, int lanes, dim3 grid, int smem, cudaStream_t s) {
  if (lanes == 8) return launch_norm<TI, TO, 8>(a, grid, smem, s);
  if (lanes == 16) return launch_norm<TI, TO, 16>(a, grid, smem, s);
  return launch_norm<TI, TO, 32>(a, grid, smem, s);
}

// Division of numbers below 2^31 by d as a product: with l = ceil(log2 d) and m = ceil(2^(31 + l) /
// d) < 2^32, n m / 2^(31 + l) exceeds n / d by less than 1 / d (m d - 2^(31 + l) < d <= 2^l).
Divisor divisor(uint32_t d) {
  int l = 0;
  while ((1ull << l) < d) ++l;
  return {static_cast<uint32_t>(((1ull << (31 + l)) + d - 1) / d), 31 + l};
}

}  // namespace

// Heads and a group's split less one are added in 32 bits.
int rotate_max_heads() { return 0x7fffffff - (kThreads / 8 - 1); }

int rotate_max_heads_across(int D) { return kThreads / (D <= 64 ? 8 : D <= 128 ? 16 : 32) * kAcrossHeads; }

int launch_rotate(RotateArgs& a, cudaStream_t s) {
  const int lanes = a.D <= 64 ? 8 : a.D <= 128 ? 16 : 32;
  const int groups = kThreads / lanes;
  const int64_t tokens = static_cast<int64_t>(a.batch) * a.S;
  if (tokens > 0x7fffffff) return kErrShape;
  a.tokens = static_cast<uint32_t>(tokens);
  a.s_div = divisor(a.S);
  for (int i = 0; i < a.axes; ++i) a.grid_div[i] = divisor(a.grid[i] > 0 ? a.grid[i] : 1);
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const bool across = a.norm == kNormRmsAcross;
  const int most = a.heads[0] > a.heads[1] ? a.heads[0] : a.heads[1];
  // Groups that share a token's heads: the power of two with the least (turns of the device's blocks) *
  // (instructions of a block: about 80 a row of a group and 330 for a token's cosines, weights and places).  Few tokens
  // share more; blocks of many rows share where they would need a second turn for a few of them.  (us, not
  // shared / shared by two / by four / chosen: 40 heads of 128, 600 tokens 11.5 / 8.6 / 7.4 / by four; 5000 tokens
  // 46.3 / 39.5 / 39.0 / by four; 24 heads, 9400 tokens 39.6 / 39.8 / 46.3 / not; 8 heads, 30000 tokens 44.8 / 52.6 / 81.5 / not.)
  const int64_t resident = static_cast<int64_t>(sms) * (across || a.in_type == kTypeF32 ? 3 : 4);
  const int tensors = a.heads[1] > 0 ? 2 : 1;
  const auto blocks = [&](int l) { return ((tokens << l) + groups - 1) / groups; };
  int log2 = 0;
  int64_t least = -1;
  for (int l = 0; (1 << l) <= groups && (l == 0 || (1 << (l - 1)) < most); ++l) {
    const int rows = ((most - 1) >> l) + 1;
    if (across && rows > kAcrossRows && (2 << l) <= groups) continue;
    const int64_t cost = (blocks(l) * tensors + resident - 1) / resident * (80LL * rows + 330);
    if (least < 0 || cost < least) {
      least = cost;
      log2 = l;
    }
  }
  a.split_log2 = log2;
  a.token_fast = a.x_stride[0][2] < a.x_stride[0][1];
  const dim3 grid(static_cast<unsigned>(blocks(log2)), tensors);
  int smem = 0;
  if (across) {
    const bool weighted = a.weight[0] != nullptr || a.weight[1] != nullptr;
    const int rows = ((most - 1) >> log2) + 1;
    smem = rows * kThreads * (a.in_type == kTypeF32 ? 32 : 16) + (weighted ? most * 2 * lanes * 16 : 0);
  }
  if (a.in_type == kTypeBf16 && a.out_type == kTypeBf16)
    return launch_lanes<__nv_bfloat16, __nv_bfloat16>(a, lanes, grid, smem, s);
  if (a.in_type == kTypeF16 && a.out_type == kTypeF16) return launch_lanes<__half, __half>(a, lanes, grid, smem, s);
  if (a.in_type == kTypeF32 && a.out_type == kTypeF32) return launch_lanes<float, float>(a, lanes, grid, smem, s);
  if (a.in_type == kTypeF16 && a.out_type == kTypeBf16)
    return launch_lanes<__half, __nv_bfloat16>(a, lanes, grid, smem, s);
  if (a.in_type == kTypeF32 && a.out_type == kTypeBf16)
    return launch_lanes<float, __nv_bfloat16>(a, lanes, grid, smem, s);
  return kErrUnsupported;
}

}  // namespace recap
