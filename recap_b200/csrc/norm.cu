// The norms, gates and residual sums before and after a transformer block, in one pass.
//
// For each token, with x and branch rows of C values:
//   norm:  h = (norm(x) w + b) (1 + scale) + shift
//   gate:  x' = residual + gate norm_b(branch),  and of that x' the same h on the way
// where norm is layer norm or root mean square over the C values, and scale, shift and gate are
// vectors of C values that a batch shares, or one of its samples, or that belong to one token.
//
// Bound by memory: every row is read once and written once and lies in registers between.  A
// row lies on one block, kVec times eight values per thread; a block takes kRows tokens of a
// sample at once, so that their loads are in flight together, their sums share shuffles and
// barriers, and modulations that tokens share are read once for them.  Modulations of single
// tokens are loaded with the rows, ahead of the sums.  Rows of more than eight values a thread wait in
// shared memory until they are summed (asynchronous copies, each thread of its own values): in
// registers they left two blocks on an SM (5120 values, fp32 and bf16: 344 us, in shared memory 315 us).
// A 16-bit branch beside an fp32 residual waits in registers instead, which leaves room in L1 for the modulations
// that blocks share (304 us); beside a 16-bit residual it is staged too (16384 x 5120: 122 us, in registers 139 us).
// fp32 rows are read in runs of four values, the next lane's run following: 16 bytes a lane side by
// side.  h is formed from the fp32 x', not from its rounded copy: one rounding instead of two.
// Measured on B200: 32760 tokens of 5120, fp32 residual, bf16 branch and norm: 304 us, 6.6 TB/s; layer norm of
// 32760 fp32 rows of 1536 to bf16: 46 us, 6.6 TB/s; both norms, gate and modulations of every token, 17777 rows
// of 2304 in bf16: 87 us, 6.6 TB/s: the rate of a copy.  These are from rest.  After a tenth of a second at this
// rate the card is at its power limit, the SM clock falls from 1.96 to 1.6 GHz, and the same calls take 326, 47
// and 92 us (a copy of as many bytes 309, 53 and 94): instructions that are saved are time then.
#include "elements.cuh"

namespace recap {
namespace {

constexpr int kMaxVec = 4;     // vectors of eight values a thread holds of a row
constexpr int kMaxWarps = 16;  // warps of a row
constexpr int kTeams = 4;      // warps of a block whose rows take one warp each (15000 rows of 144: 4.6 -> 3.5 us)

// Sums of kRows (1, 2, 4) values over the warp.  Two values share the steps of one: each half of
// the lanes keeps one value and hands the other over, then goes on with its own.  On return
// v[0] of lane l is the sum of value l / (32 / kRows).
template <int kRows>
__device__ __forceinline__ float warp_sums(float (&v)[kRows]) {
  const int lane = threadIdx.x & 31;
  if constexpr (kRows == 4) {
    const bool up = lane & 16;
    const float k0 = up ? v[2] : v[0], k1 = up ? v[3] : v[1];
    const float o0 = up ? v[0] : v[2], o1 = up ? v[1] : v[3];
    v[0] = k0 + __shfl_xor_sync(0xffffffffu, o0, 16);
    v[1] = k1 + __shfl_xor_sync(0xffffffffu, o1, 16);
  }
  if constexpr (kRows >= 2) {
    constexpr int o = kRows == 4 ? 8 : 16;
    const bool up = lane & o;
    const float keep = up ? v[1] : v[0], other = up ? v[0] : v[1];
    v[0] = keep + __shfl_xor_sync(0xffffffffu, other, o);
  }
  return lanes_sum<32 / kRows>(v[0]);
}

// Sums of kRows values over the block, in every thread.  `buf` holds kRows * kMaxWarps floats; calls
// take two buffers in turn, so that one barrier each is enough: a buffer is written again only after
// the next call's barrier, which every thread reaches after it has read it.
template <int kRows>
__device__ __forceinline__ void block_sum(float (&v)[kRows], float* buf, int warps) {
  constexpr int kPer = 32 / kRows;  // lanes of a value
  constexpr int kUse = kPer < kMaxWarps ? kPer : kMaxWarps;
  const int lane = threadIdx.x & 31;
  float s = warp_sums<kRows>(v);
  if (warps > 1) {
    if (lane % kPer == 0) buf[(lane / kPer) * kMaxWarps + (threadIdx.x >> 5)] = s;
    __syncthreads();
    const float* mine = buf + (lane / kPer) * kMaxWarps;
    s = 0.f;
#pragma unroll
    for (int w = 0; w < kMaxWarps; w += kUse) {
      const int at = w + lane % kUse;
      if (at < warps) s += mine[at];
    }
    s = lanes_sum<kUse>(s);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) v[r] = kRows == 1 ? s : __shfl_sync(0xffffffffu, s, r * kPer);
}

// The threads of a row: the block's, or, where one warp holds a row, each warp with rows of its own.
template <bool kWarps>
struct Team {
  __device__ __forceinline__ static int threads() { return kWarps ? 32 : blockDim.x; }
  __device__ __forceinline__ static int me() { return kWarps ? threadIdx.x & 31 : threadIdx.x; }
  __device__ __forceinline__ static int index() { return kWarps ? threadIdx.x >> 5 : 0; }
};

// The columns of a thread's vector v: two runs of four values, apart (kSplit) or one after the other.
// kWhole: no thread has columns past the row, which takes the selects out of the sums (32760 x 1536, fp32 to bf16:
// 46 us, with them 47; at the power limit 47 and 49).
template <bool kSplit, bool kWarps, bool kWhole>
struct Columns {
  int c0, c1;
  bool in0, in1;
  __device__ __forceinline__ Columns(int v, int C) {
    const int threads = Team<kWarps>::threads(), me = Team<kWarps>::me();
    if (kSplit) {
      c0 = (2 * v * threads + me) * 4;
      c1 = c0 + 4 * threads;
      in0 = kWhole || c0 < C;
      in1 = kWhole || c1 < C;
    } else {
      c0 = (v * threads + me) * 8;
      c1 = c0 + 4;
      in0 = in1 = kWhole || c0 < C;
    }
  }
};

// A row's values of those columns, zero past its end.
template <bool kSplit, typename T, typename C>
__device__ __forceinline__ void load_columns(Raw8<T>& r, const T* row, const C& c, bool live) {
  if (live && c.in1) {
    if constexpr (kSplit)
      load4x2(r, row + c.c0, row + c.c1);
    else
      load8(r, row + c.c0);
  } else {
    zero8(r);
    if (kSplit && live && c.in0) load4(r, row + c.c0);
  }
}
// The same by way of the thread's own 16-byte slots of shared memory, `slot` and, for fp32, the one
// blockDim.x on: copied without waiting, then read.
constexpr int slots_of(int value_bytes) { return value_bytes / 2; }
template <bool kSplit, typename T, typename C>
__device__ __forceinline__ void fetch_columns(uint4* slot, const T* row, const C& c) {
  if constexpr (sizeof(T) == 4) {
    if (c.in0) copy16(slot, row + c.c0);
    if (c.in1) copy16(slot + blockDim.x, row + c.c1);
  } else if constexpr (kSplit) {
    if (c.in0) copy8(slot, row + c.c0);
    if (c.in1) copy8(reinterpret_cast<uint2*>(slot) + 1, row + c.c1);
  } else {
    if (c.in0) copy16(slot, row + c.c0);
  }
}
template <bool kSplit, typename T, typename C>
__device__ __forceinline__ void read_columns(float (&x)[8], const uint4* slot, const C& c) {
  Raw8<T> r;
  const uint4 a = *slot;
  r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w;
  if constexpr (sizeof(T) == 4) {
    const uint4 b = slot[blockDim.x];
    r.w[4] = b.x, r.w[5] = b.y, r.w[6] = b.z, r.w[7] = b.w;
  }
  widen8(x, r);
  if (!c.in1) {  // never copied
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = c.in0 ? x[j] : 0.f;
      x[j + 4] = 0.f;
    }
  }
}
template <bool kSplit, typename T, typename C>
__device__ __forceinline__ void store_columns(T* row, const C& c, const float (&x)[8]) {
  if (c.in1) {
    if constexpr (kSplit)
      store4x2(row + c.c0, row + c.c1, x);
    else
      store8(row + c.c0, x);
  } else if (kSplit && c.in0) {
    store4(row + c.c0, x);
  }
}

// norm(x) in place: the row mean (layer norm), then the mean square, in two sums.
template <int kRows, int kVec, bool kSplit, bool kWarps, bool kWhole>
__device__ __forceinline__ void norm_rows(float (&x)[kRows][kVec][8], int layer, int C, float eps, float* buf,
                                          int& turn) {
  const int warps = Team<kWarps>::threads() >> 5;
  const float inv = 1.f / static_cast<float>(C);
  float t[kRows];
  if (layer) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      float m0 = 0.f, m1 = 0.f;
#pragma unroll
      for (int v = 0; v < kVec; ++v)
#pragma unroll
        for (int j = 0; j < 8; j += 2) add2(m0, m1, x[r][v][j], x[r][v][j + 1]);
      t[r] = m0 + m1;
    }
    block_sum(t, buf + (turn ^= kRows * kMaxWarps), warps);
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      const Columns<kSplit, kWarps, kWhole> c(v, C);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const float m = -t[r] * inv;
        const float m0 = c.in0 ? m : 0.f, m1 = c.in1 ? m : 0.f;
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          add2(x[r][v][j], x[r][v][j + 1], m0, m0);
          add2(x[r][v][j + 4], x[r][v][j + 5], m1, m1);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int v = 0; v < kVec; ++v)
#pragma unroll
      for (int j = 0; j < 8; j += 2)
        fma2(s0, s1, x[r][v][j], x[r][v][j + 1], x[r][v][j], x[r][v][j + 1], s0, s1);
    t[r] = s0 + s1;
  }
  block_sum(t, buf + (turn ^= kRows * kMaxWarps), warps);
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const float q = rsqrtf(fmaf(t[r], inv, eps));
#pragma unroll
    for (int v = 0; v < kVec; ++v)
#pragma unroll
      for (int j = 0; j < 8; j += 2) mul2(x[r][v][j], x[r][v][j + 1], q, q);
  }
}

// x = x * p or x + p, eight values
__device__ __forceinline__ void mul8(float (&x)[8], const float (&p)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) mul2(x[j], x[j + 1], p[j], p[j + 1]);
}
__device__ __forceinline__ void add8(float (&x)[8], const float (&p)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) add2(x[j], x[j + 1], p[j], p[j + 1]);
}

// Most threads of a block with eight values each.  The split of a row over threads depends on its length and type
// only, so a token's sums, and its result, do not depend on how many tokens a call or a block has.
constexpr int one_vector_threads(int x_bytes) { return x_bytes == 4 ? 384 : 512; }

// How a block comes by its modulations: read when needed, one vector for its tokens (or its one
// token); or each token's own, of 16 or 32 bits a value, loaded with the rows.
enum : int { kModsLate = 0, kMods16 = 2, kMods32 = 4 };

// Which rows wait in shared memory: wide ones, and four fp32 residuals a block, which registers do not hold.
template <typename TX, int kVec, int kRows, bool kGate>
constexpr bool stages() {
  return kVec > 1 || (kGate && kRows == 4 && sizeof(TX) == 4);
}

template <typename TX, typename TH, int kVec, int kRows, bool kGate, int kMods, int kThreads, bool kWarps, bool kWhole>
__global__ void __launch_bounds__(kThreads, 2) norm_kernel(const __grid_constant__ NormArgs a) {
  constexpr bool kSplit = sizeof(TX) == 4;
  constexpr bool kStaged = stages<TX, kVec, kRows, kGate>();
  constexpr bool kStagedBranch = kGate && kStaged && sizeof(TH) == sizeof(TX);
  extern __shared__ uint4 staged[];
  constexpr bool kOwn = kMods != kModsLate;
  __shared__ float buf[2 * kRows * kMaxWarps];
  int turn = 0;
  grid_wait();
  const int C = a.C;
  const int b = a.batch == 1 ? 0 : blockIdx.x / a.blocks;
  const int s0 = ((blockIdx.x - b * a.blocks) * (kWarps ? kTeams : 1) + Team<kWarps>::index()) * kRows;
  const int rows = kRows == 1 && !kWarps ? 1 : min(kRows, a.S - s0);
  if (kWarps && rows <= 0) return;  // a warp past the last token; it has no barrier to keep

  Raw8<TX> rx[kStaged ? 1 : kRows][kStaged ? 1 : kVec];
  Raw8<TH> ry[kStagedBranch || !kGate ? 1 : kRows][kStagedBranch ? 1 : kVec];
  constexpr int kXSlots = slots_of(sizeof(TX)), kSlots = kXSlots + (kStagedBranch ? slots_of(sizeof(TH)) : 0);
  auto slot = [&](int r, int v) { return staged + (r * kVec + v) * kSlots * blockDim.x + threadIdx.x; };
  {
    const TX* xr = static_cast<const TX*>(a.x) + b * a.x_stride[0] + s0 * a.x_stride[1];
    const TH* yr = nullptr;
    if constexpr (kGate) yr = static_cast<const TH*>(a.branch) + b * a.branch_stride[0] + s0 * a.branch_stride[1];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
#pragma unroll
      for (int v = 0; v < kVec; ++v) {
        const Columns<kSplit, kWarps, kWhole> c(v, C);
        if constexpr (kStaged) {
          if (r < rows) {
            fetch_columns<kSplit>(slot(r, v), xr, c);
            if constexpr (kStagedBranch) fetch_columns<kSplit>(slot(r, v) + kXSlots * blockDim.x, yr, c);
          }
        } else {
          load_columns<kSplit>(rx[r][v], xr, c, r < rows);
        }
        if constexpr (kGate && !kStagedBranch) load_columns<kSplit>(ry[r][v], yr, c, r < rows);
      }
      xr += a.x_stride[1];
      if constexpr (kGate) yr += a.branch_stride[1];
    }
  }
  if constexpr (kStaged) copies_commit();
  auto row_values = [&](float (&x)[8], int r, int v) {
    if constexpr (kStaged)
      read_columns<kSplit, TX>(x, slot(r, v), Columns<kSplit, kWarps, kWhole>(v, C));
    else
      widen8(x, rx[r][v]);
  };
  auto branch_values = [&](float (&x)[8], int r, int v) {
    if constexpr (kStagedBranch)
      read_columns<kSplit, TH>(x, slot(r, v) + kXSlots * blockDim.x, Columns<kSplit, kWarps, kWhole>(v, C));
    else
      widen8(x, ry[r][v]);
  };
  // modulations of single tokens are as far away as the rows: ask for them now
  uint32_t own[kOwn ? 3 : 1][kOwn ? kRows : 1][kOwn ? kVec : 1][kOwn ? 2 * kMods : 1];
  if constexpr (kOwn) {
#pragma unroll
    for (int m = 0; m < (kGate ? 3 : 2); ++m) {
      if (a.mod[m] == nullptr) continue;
      const char* row = static_cast<const char*>(a.mod[m]) + (b * a.mod_stride[m][0] + s0 * a.mod_stride[m][1]) * kMods;
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
          const Columns<kSplit, kWarps, kWhole> c(v, C);
          if (r < rows && c.in0) load_own<kSplit, kMods>(own[m][r][v], row, c.c0, c.in1 ? c.c1 : c.c0);
        }
        row += a.mod_stride[m][1] * kMods;
      }
    }
  }
  // modulation m of the block's row r; late ones are read for the first row and stay
  auto modulation = [&](float (&p)[8], int m, int r, int v, int c0, int c1) {
    if constexpr (kOwn) {
      RawParam8 w;
#pragma unroll
      for (int j = 0; j < 2 * kMods; ++j) w.w[j] = own[m][r][v][j];
      widen_param8(p, w, kMods == kMods32 ? kTypeF32 : a.mod_type);
    } else if (r == 0) {
      const int64_t at = b * a.mod_stride[m][0] + (kRows == 1 ? s0 * a.mod_stride[m][1] : 0);
      load_param<kSplit>(p, a.mod[m], at + c0, at + c1, a.mod_type);
    }
  };

  float x[kRows][kVec][8];
  float p[8];
  if constexpr (kStaged && (!kGate || kStagedBranch)) copies_wait<0>();
  if constexpr (kGate) {
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int v = 0; v < kVec; ++v) branch_values(x[r][v], r, v);
    if constexpr (kStaged && !kStagedBranch) copies_wait<0>();
    if (a.branch_norm != kNormNone)
      norm_rows<kRows, kVec, kSplit, kWarps, kWhole>(x, a.branch_norm == kNormLayer, C, a.branch_eps, buf, turn);
    TX* out = static_cast<TX*>(a.x_out) + b * a.x_out_stride[0] + s0 * a.x_out_stride[1];
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      const Columns<kSplit, kWarps, kWhole> c(v, C);
      if (!c.in0) continue;
      const int c1 = c.in1 ? c.c1 : c.c0;  // a run past the row reads the one before it and is not stored
      if (a.branch_weight != nullptr) {
        load_param<kSplit>(p, a.branch_weight, c.c0, c1, a.branch_weight_type);
#pragma unroll
        for (int r = 0; r < kRows; ++r) mul8(x[r][v], p);
      }
      if (a.branch_bias != nullptr) {
        load_param<kSplit>(p, a.branch_bias, c.c0, c1, a.branch_weight_type);
#pragma unroll
        for (int r = 0; r < kRows; ++r) add8(x[r][v], p);
      }
      if (a.mod[2] != nullptr) {
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          modulation(p, 2, r, v, c.c0, c1);
          mul8(x[r][v], p);
        }
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        float res[8];
        row_values(res, r, v);
        add8(x[r][v], res);
        if (r < rows) store_columns<kSplit>(out + r * a.x_out_stride[1], c, x[r][v]);
        if (kSplit && !c.in1) x[r][v][4] = x[r][v][5] = x[r][v][6] = x[r][v][7] = 0.f;  // out of the sums
      }
    }
    if (a.norm == kNormNone) return;
  } else {
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int v = 0; v < kVec; ++v) row_values(x[r][v], r, v);
  }
  norm_rows<kRows, kVec, kSplit, kWarps, kWhole>(x, a.norm == kNormLayer, C, a.eps, buf, turn);
  TH* out = static_cast<TH*>(a.h) + b * a.h_stride[0] + s0 * a.h_stride[1];
#pragma unroll
  for (int v = 0; v < kVec; ++v) {
    const Columns<kSplit, kWarps, kWhole> c(v, C);
    if (!c.in0) continue;
    const int c1 = c.in1 ? c.c1 : c.c0;
    if (a.weight != nullptr) {
      load_param<kSplit>(p, a.weight, c.c0, c1, a.weight_type);
#pragma unroll
      for (int r = 0; r < kRows; ++r) mul8(x[r][v], p);
    }
    if (a.bias != nullptr) {
      load_param<kSplit>(p, a.bias, c.c0, c1, a.weight_type);
#pragma unroll
      for (int r = 0; r < kRows; ++r) add8(x[r][v], p);
    }
    if (a.mod[0] != nullptr) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        modulation(p, 0, r, v, c.c0, c1);
#pragma unroll
        for (int j = 0; j < 8; j += 2)
          fma2(x[r][v][j], x[r][v][j + 1], x[r][v][j], x[r][v][j + 1], p[j], p[j + 1], x[r][v][j], x[r][v][j + 1]);
      }
    }
    if (a.mod[1] != nullptr) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        modulation(p, 1, r, v, c.c0, c1);
        add8(x[r][v], p);
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (r < rows) store_columns<kSplit>(out + r * a.h_stride[1], c, x[r][v]);
  }
}

template <typename TX, typename TH, int kVec, int kRows, bool kGate, int kMods, int kThreads, bool kWarps, bool kWhole>
int launch_kernel(NormArgs& a, int threads, cudaStream_t s) {
  auto* kernel = norm_kernel<TX, TH, kVec, kRows, kGate, kMods, kThreads, kWarps, kWhole>;
  constexpr int kTokens = kRows * (kWarps ? kTeams : 1);  // of a block
  a.blocks = (a.S - 1) / kTokens + 1;  // S up to 2^31 - 1
  const unsigned blocks = static_cast<unsigned>(a.batch) * static_cast<unsigned>(a.blocks);
  const int block = kWarps ? 32 * kTeams : threads;
  int smem = 0;
  if constexpr (stages<TX, kVec, kRows, kGate>()) {
    constexpr int kPerThread = kRows * kVec * (slots_of(sizeof(TX)) + (kGate && sizeof(TH) == sizeof(TX) ? slots_of(sizeof(TH)) : 0)) * 16;
    smem = kPerThread * block;
    // the most of any call, so that calls of two host threads set the same
    if (smem > 46 * 1024 && !allow_shared(kernel, kPerThread * kThreads)) return kErrLaunch;
  }
  return launch_after(kernel, dim3(blocks), block, smem, s, a);
}

// kOneWarp: rows of 32 threads come here too.
template <typename TX, typename TH, int kVec, int kRows, bool kGate, int kMods, int kThreads, bool kOneWarp = kVec == 1>
int launch_team(NormArgs& a, int threads, cudaStream_t s) {
  // a row of one warp leaves a block room for others'
  if constexpr (kOneWarp)
    if (threads == 32) return launch_kernel<TX, TH, kVec, kRows, kGate, kMods, 32 * kTeams, true, false>(a, threads, s);
  if (a.C == 8 * kVec * threads) return launch_kernel<TX, TH, kVec, kRows, kGate, kMods, kThreads, false, true>(a, threads, s);
  return launch_kernel<TX, TH, kVec, kRows, kGate, kMods, kThreads, false, false>(a, threads, s);
}

// Four tokens a block, but two of an fp32 residual and its branch, which 64 registers a thread hold; four of them
// wait in shared memory where an SM takes only two blocks of so many threads, and the branch is of 16 bits.  (Gate,
// layer norm, fp32 residual, bf16 branch: 16384 x 2560 two tokens 79 us, four staged 80; 16384 x 2568 two tokens 99 us,
// four staged 89; with an fp32 branch 16384 x 2560 two 100 us, four 101, at the power limit 101 and 105.  Gate and
// norms of bf16, 16384 x 1536: four tokens 36 us, two 38 us.)
template <typename TX, typename TH, int kVec, int kRows, int kMods, int kThreads = 512>
int launch_gate(NormArgs& a, int threads, cudaStream_t s) {
  if (a.branch == nullptr) return launch_team<TX, TH, kVec, kRows, false, kMods, kThreads>(a, threads, s);
  if constexpr (kRows == 4 && sizeof(TX) == 4 && sizeof(TH) == 4) {
    return launch_team<TX, TH, kVec, 2, true, kMods, kThreads>(a, threads, s);
  } else if constexpr (kRows == 4 && sizeof(TX) == 4) {
    if (threads <= 320) return launch_team<TX, TH, kVec, 2, true, kMods, kThreads>(a, threads, s);
    return launch_team<TX, TH, kVec, kRows, true, kMods, kThreads, false>(a, threads, s);
  } else {
    return launch_team<TX, TH, kVec, kRows, true, kMods, kThreads>(a, threads, s);
  }
}

template <typename TX, typename TH>
int launch_vec(NormArgs& a, cudaStream_t s) {
  bool shared = true;
  for (int m = 0; m < 3; ++m) shared = shared && (a.mod[m] == nullptr || a.mod_stride[m][1] == 0);
  // Eight values a thread as far as that goes, sixteen up to 8192 values, else 32: the narrower, the more rows
  // a block takes and the more blocks are resident.  (B200, bf16 norm with scale and shift, 16384 tokens: 4096
  // values as 512 threads of eight, four rows a block 51 us, as 256 threads of sixteen, two rows 56 us; bf16
  // gate and norms of 8192 values as 512 threads of sixteen 215 us, as 256 of 32 287 us.)
  const int vecs = a.C / 8;
  const int per = vecs <= one_vector_threads(sizeof(TX)) ? 1 : vecs <= 1024 ? 2 : 4;
  const int threads = ((vecs + per - 1) / per + 31) / 32 * 32;
  const bool narrow = a.mod_type != kTypeF32;
  // tokens by the block only where blocks of one token would be more than the device holds, and a sample
  // fills a block
  const bool many = static_cast<int64_t>(a.batch) * a.S >= 2048 && a.S >= 4;
  if (per == 1) {
    if (shared) return many ? launch_gate<TX, TH, 1, 4, kModsLate>(a, threads, s) : launch_gate<TX, TH, 1, 1, kModsLate>(a, threads, s);
    if (!narrow) return launch_gate<TX, TH, 1, 1, kMods32>(a, threads, s);
    if (!many) return launch_gate<TX, TH, 1, 1, kMods16>(a, threads, s);
    // two tokens and their modulations in 80 registers rather than 64 as long as blocks are small enough
    // (2304 values, both norms, bf16: 87 us, in 64 registers 90 us)
    if constexpr (one_vector_threads(sizeof(TX)) > 384) {
      if (threads > 384) return launch_gate<TX, TH, 1, 2, kMods16>(a, threads, s);
    }
    return launch_gate<TX, TH, 1, 2, kMods16, 384>(a, threads, s);
  }
  if (per == 2) {
    if constexpr (sizeof(TX) == 2) {
      // four rows in 96 registers as long as two blocks of that fit (16384 x 5120 bf16: 64 us, two rows 75 us)
      if (shared && many && a.branch == nullptr && threads <= 320) return launch_team<TX, TH, 2, 4, false, kModsLate, 320>(a, threads, s);
    }
    if (shared && many) return launch_gate<TX, TH, 2, 2, kModsLate>(a, threads, s);
    if (!shared && narrow) return launch_gate<TX, TH, 2, 1, kMods16>(a, threads, s);
    return launch_gate<TX, TH, 2, 1, kModsLate>(a, threads, s);
  }
  return launch_gate<TX, TH, 4, 1, kModsLate>(a, threads, s);
}

}  // namespace

int norm_max_channels() { return kMaxWarps * 32 * kMaxVec * 8; }

int launch_norm_rows(NormArgs& a, cudaStream_t s) {
  if (a.x_type == kTypeBf16 && a.h_type == kTypeBf16) return launch_vec<__nv_bfloat16, __nv_bfloat16>(a, s);
  if (a.x_type == kTypeF16 && a.h_type == kTypeF16) return launch_vec<__half, __half>(a, s);
  if (a.x_type == kTypeF32 && a.h_type == kTypeF32) return launch_vec<float, float>(a, s);
  if (a.x_type == kTypeF32 && a.h_type == kTypeBf16) return launch_vec<float, __nv_bfloat16>(a, s);
  if (a.x_type == kTypeF32 && a.h_type == kTypeF16) return launch_vec<float, __half>(a, s);
  return kErrUnsupported;
}

}  // namespace recap
