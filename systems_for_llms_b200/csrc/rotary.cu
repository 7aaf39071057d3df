// Rotary position embedding of attention heads, alone or behind a per-head RMS norm.
//
//   u = x / sqrt(mean(x^2) + eps) * w        (or u = x without a weight)
//   y_a = u_a cos - u_b sin,  y_b = u_a sin + u_b cos   for each rotated pair (a, b)
//   y_e = u_e                                           for lanes beyond the rotated ones
//
// Pairs are (2i, 2i+1) in the interleaved layout and (i, i + R/2) in the half layout, R being
// the number of rotated lanes.  Backward, with v the gradient turned by the opposite angle:
//   dw = sum over rows of v * xhat,   dx = rstd (v w - xhat mean(v w xhat)),  xhat = x rstd
//
// The reference norms whole residual rows and rotates in separate eager kernels
// (src/llmlab/model/layers.py:133-141, src/llmlab/model/attention.py:44-58); this is one pass
// that reads each head once.  It is bound by memory, so everything is arranged around 16-byte
// accesses in flight: a lane owns eight consecutive elements of a head, a group of 4 to 32
// lanes owns a head (so the norm is a few shuffles and the statistics never leave registers),
// and a warp issues the loads of several head groups of one token before it uses the first.
// The table row of the token is read once for all of them.  The backward pass recomputes the
// statistics from x, which it has to read anyway, instead of storing them.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "launch.cuh"
#include "ptx.cuh"
#include "sfl.h"

namespace sfl {
namespace {

constexpr int kVec = 8;        // elements of a head that one lane holds
constexpr int kWarps = 8;      // warps per block
constexpr int kMaxDim = 256;   // 32 lanes of eight elements

// How a lane finds the other element of a pair.
enum Pairing : int {
  kInterleaved = 0,  // in its own registers
  kHalfShuffle = 1,  // R/2 a multiple of 8: the same register of another lane
  kHalfShared = 2,   // any other R: through a strip of shared memory
};

struct Side {
  const void* x;
  void* y;            // forward: result; backward: dx
  const void* dy;     // backward only
  const float* weight;
  long x_b, x_h, x_t, y_b, y_h, y_t, dy_b, dy_h, dy_t;
  int heads;
  int vec;            // every row of x, y (and dy) starts on a 16-byte boundary
};

struct RotaryParams {
  Side side[2];
  int blocks0;        // blocks [0, blocks0) serve side 0, the others side 1
  const float* cos;
  const float* sin;
  const int64_t* positions;  // NULL: the token's own index
  long pos_b, pos_t;
  int table_rows, rotated, table_vec;
  int B, T, D;
  int group;          // lanes per head (power of two)
  float eps, sign;    // sign -1 turns by the opposite angle
  float* partial;     // backward with norm: [blocks, D]
};

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

// The eight elements as they lie in memory; converted to fp32 only when they are used, so that
// loads in flight hold 16 bytes (32 for fp32) of registers per lane.
template <typename T> struct Raw { T v[kVec]; };

template <typename T>
__device__ __forceinline__ void load_raw(Raw<T>& r, const T* row, int e0, int D, bool vec,
                                         bool live) {
  if (live && vec) {
    const uint4* src = reinterpret_cast<const uint4*>(row + e0);
    uint4* dst = reinterpret_cast<uint4*>(r.v);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(Raw<T>) / 16); ++i) dst[i] = src[i];
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      r.v[i] = live && e0 + i < D ? row[e0 + i] : from_f32<T>(0.f);
  }
}

template <typename T>
__device__ __forceinline__ void store_raw(T* row, const float (&f)[kVec], int e0, int D, bool vec) {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < kVec; ++i) r.v[i] = from_f32<T>(f[i]);
  if (vec) {
    uint4* dst = reinterpret_cast<uint4*>(row + e0);
    const uint4* src = reinterpret_cast<const uint4*>(r.v);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(Raw<T>) / 16); ++i) dst[i] = src[i];
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (e0 + i < D) row[e0 + i] = r.v[i];
  }
}

// y_e = u_e C_e + u_partner S_e for the eight elements from e0; S carries the pair's sign.
// A position outside the table turns its rotated lanes into NaN instead of reading past it.
template <int PAIR>
__device__ __forceinline__ void load_angles(const RotaryParams& p, int b, int t, int e0,
                                            float (&C)[kVec], float (&S)[kVec]) {
  long pos = t;
  if (p.positions != nullptr) pos = p.positions[b * p.pos_b + t * p.pos_t];
  const bool known = pos >= 0 && pos < p.table_rows;
  const int half = p.rotated >> 1;
  const float* cr = p.cos + (known ? pos : 0) * static_cast<long>(half);
  const float* sr = p.sin + (known ? pos : 0) * static_cast<long>(half);
  const float bad = known ? 0.f : NAN;
  if (p.table_vec && e0 + kVec <= p.rotated) {
    if constexpr (PAIR == kInterleaved) {
      const float4 c = *reinterpret_cast<const float4*>(cr + (e0 >> 1));
      const float4 s = *reinterpret_cast<const float4*>(sr + (e0 >> 1));
      const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        C[i] = cc[i >> 1] + bad;
        S[i] = (i & 1) ? p.sign * ss[i >> 1] : -p.sign * ss[i >> 1];
      }
      return;
    } else if constexpr (PAIR == kHalfShuffle) {
      const bool second = e0 >= half;
      const int at = second ? e0 - half : e0;
      const float flip = second ? p.sign : -p.sign;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 c = *reinterpret_cast<const float4*>(cr + at + 4 * j);
        const float4 s = *reinterpret_cast<const float4*>(sr + at + 4 * j);
        C[4 * j] = c.x + bad; C[4 * j + 1] = c.y + bad; C[4 * j + 2] = c.z + bad;
        C[4 * j + 3] = c.w + bad;
        S[4 * j] = flip * s.x; S[4 * j + 1] = flip * s.y; S[4 * j + 2] = flip * s.z;
        S[4 * j + 3] = flip * s.w;
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int e = e0 + i;
    C[i] = 1.f;
    S[i] = 0.f;
    if (e < p.rotated) {
      const bool second = PAIR == kInterleaved ? (e & 1) : e >= half;
      const int at = PAIR == kInterleaved ? e >> 1 : (second ? e - half : e);
      C[i] = cr[at] + bad;
      S[i] = second ? p.sign * sr[at] : -p.sign * sr[at];
    }
  }
}

// Turns the pairs of u in place.  All lanes of the warp take part.  Lanes beyond the rotated
// ones keep their value untouched: multiplying by S = 0 would make NaN of an infinity.
template <int PAIR>
__device__ __forceinline__ void turn(const RotaryParams& p, float (&u)[kVec], const float (&C)[kVec],
                                     const float (&S)[kVec], int e0, int lane, float* strip) {
  if constexpr (PAIR == kInterleaved) {
#pragma unroll
    for (int i = 0; i < kVec; i += 2) {
      if (e0 + i < p.rotated) {
        const float a = u[i], b = u[i + 1];
        u[i] = fmaf(a, C[i], b * S[i]);
        u[i + 1] = fmaf(b, C[i + 1], a * S[i + 1]);
      }
    }
  } else if constexpr (PAIR == kHalfShuffle) {
    const int half = p.rotated >> 1;
    const int apart = half / kVec;
    const int src = e0 < half ? lane + apart : (e0 < p.rotated ? lane - apart : lane);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const float other = __shfl_sync(0xffffffffu, u[i], src);
      if (e0 < p.rotated) u[i] = fmaf(u[i], C[i], other * S[i]);
    }
  } else {
    const int half = p.rotated >> 1;
    float* mine = strip + (lane - e0 / kVec) * kVec;  // the head's first element
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kVec; ++i) strip[lane * kVec + i] = u[i];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int e = e0 + i;
      if (e < p.rotated) u[i] = fmaf(u[i], C[i], mine[e < half ? e + half : e - half] * S[i]);
    }
  }
}

__device__ __forceinline__ float group_sum(float v, int group) {
  for (int o = group >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Where {
  int lane, e0, sub;   // lane, its first element, head within the warp's group of heads
  bool live;           // the lane holds elements of a head
};

__device__ __forceinline__ Where where(const RotaryParams& p) {
  Where w;
  w.lane = threadIdx.x & 31;
  const int in = w.lane & (p.group - 1);
  w.e0 = in * kVec;
  w.sub = w.lane / p.group;
  w.live = w.e0 < p.D;
  return w;
}

// One warp takes PER head groups of one token.  Measured on B200 (training microbatches,
// L2-cold): PER = 4 keeps enough bytes in flight; PER = 1 is for calls with few tokens, which
// are over sooner when every head group has a warp of its own.
template <typename T, int PAIR, bool NORM, int PER>
__global__ void __launch_bounds__(32 * kWarps)
rotary_kernel(const __grid_constant__ RotaryParams p) {
  __shared__ float strips[PAIR == kHalfShared ? kWarps * 32 * kVec : 1];
  pdl_launch_dependents();
  pdl_wait();
  const bool first = static_cast<int>(blockIdx.x) < p.blocks0;
  const Side& s = p.side[first ? 0 : 1];
  const int block = first ? blockIdx.x : blockIdx.x - p.blocks0;
  const int warp = threadIdx.x >> 5;
  const Where w = where(p);
  float* strip = strips + (PAIR == kHalfShared ? warp * 32 * kVec : 0);
  const int heads_per = 32 / p.group;
  const int chunks = (s.heads + heads_per * PER - 1) / (heads_per * PER);
  const long item = static_cast<long>(block) * kWarps + warp;
  const long token = item / chunks;
  if (token >= static_cast<long>(p.B) * p.T) return;  // warp-uniform
  const int h0 = static_cast<int>(item - token * chunks) * heads_per * PER + w.sub;
  const int b = static_cast<int>(token / p.T), t = static_cast<int>(token - static_cast<long>(b) * p.T);
  const T* x = static_cast<const T*>(s.x) + b * s.x_b + t * s.x_t;
  T* y = static_cast<T*>(s.y) + b * s.y_b + t * s.y_t;

  Raw<T> raw[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int h = h0 + j * heads_per;
    load_raw(raw[j], x + static_cast<long>(h) * s.x_h, w.e0, p.D, s.vec, w.live && h < s.heads);
  }
  float C[kVec], S[kVec], weight[kVec];
  load_angles<PAIR>(p, b, t, w.e0, C, S);
  if constexpr (NORM) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) weight[i] = w.e0 + i < p.D ? s.weight[w.e0 + i] : 0.f;
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int h = h0 + j * heads_per;
    float u[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) u[i] = to_f32(raw[j].v[i]);
    if constexpr (NORM) {
      float sq = 0.f;
#pragma unroll
      for (int i = 0; i < kVec; ++i) sq = fmaf(u[i], u[i], sq);
      sq = group_sum(sq, p.group);
      const float rstd = 1.0f / sqrtf(sq / p.D + p.eps);
#pragma unroll
      for (int i = 0; i < kVec; ++i) u[i] = u[i] * rstd * weight[i];
    }
    turn<PAIR>(p, u, C, S, w.e0, w.lane, strip);
    if (w.live && h < s.heads) store_raw(y + static_cast<long>(h) * s.y_h, u, w.e0, p.D, s.vec);
  }
}

// Backward with the norm.  A persistent grid: every warp keeps the weight gradient of its
// eight elements in registers over all its tokens; the block folds its warps in a fixed order
// and leaves one row of partial sums (deterministic, no atomics).
template <typename T, int PAIR, int PER>
__global__ void __launch_bounds__(32 * kWarps)
rotary_bwd_kernel(const __grid_constant__ RotaryParams p) {
  __shared__ float strips[PAIR == kHalfShared ? kWarps * 32 * kVec : 1];
  __shared__ float fold[kWarps][kMaxDim];
  pdl_launch_dependents();
  pdl_wait();
  const bool first = static_cast<int>(blockIdx.x) < p.blocks0;
  const Side& s = p.side[first ? 0 : 1];
  const int block = first ? blockIdx.x : blockIdx.x - p.blocks0;
  const int blocks = first ? p.blocks0 : gridDim.x - p.blocks0;
  const int warp = threadIdx.x >> 5;
  const Where w = where(p);
  float* strip = strips + (PAIR == kHalfShared ? warp * 32 * kVec : 0);
  const int heads_per = 32 / p.group;
  const int chunks = (s.heads + heads_per * PER - 1) / (heads_per * PER);
  const long items = static_cast<long>(p.B) * p.T * chunks;

  float weight[kVec], acc[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    weight[i] = w.e0 + i < p.D ? s.weight[w.e0 + i] : 0.f;
    acc[i] = 0.f;
  }
  for (long item = static_cast<long>(block) * kWarps + warp; item < items;
       item += static_cast<long>(blocks) * kWarps) {
    const long token = item / chunks;
    const int h0 = static_cast<int>(item - token * chunks) * heads_per * PER + w.sub;
    const int b = static_cast<int>(token / p.T), t = static_cast<int>(token - static_cast<long>(b) * p.T);
    const T* x = static_cast<const T*>(s.x) + b * s.x_b + t * s.x_t;
    const T* dy = static_cast<const T*>(s.dy) + b * s.dy_b + t * s.dy_t;
    T* dx = static_cast<T*>(s.y) + b * s.y_b + t * s.y_t;
    Raw<T> rx[PER], rg[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int h = h0 + j * heads_per;
      const bool live = w.live && h < s.heads;
      load_raw(rx[j], x + static_cast<long>(h) * s.x_h, w.e0, p.D, s.vec, live);
      load_raw(rg[j], dy + static_cast<long>(h) * s.dy_h, w.e0, p.D, s.vec, live);
    }
    float C[kVec], S[kVec];
    load_angles<PAIR>(p, b, t, w.e0, C, S);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int h = h0 + j * heads_per;
      float v[kVec], u[kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        v[i] = to_f32(rg[j].v[i]);
        u[i] = to_f32(rx[j].v[i]);
      }
      turn<PAIR>(p, v, C, S, w.e0, w.lane, strip);
      float sq = 0.f, dot = 0.f;
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        sq = fmaf(u[i], u[i], sq);
        dot = fmaf(v[i] * weight[i], u[i], dot);
      }
      sq = group_sum(sq, p.group);
      dot = group_sum(dot, p.group);
      const float rstd = 1.0f / sqrtf(sq / p.D + p.eps);
      const float mean = dot * rstd / p.D;
      if (w.live && h < s.heads) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const float unit = u[i] * rstd;
          acc[i] = fmaf(v[i], unit, acc[i]);
          v[i] = rstd * (v[i] * weight[i] - unit * mean);
        }
        store_raw(dx + static_cast<long>(h) * s.y_h, v, w.e0, p.D, s.vec);
      }
    }
  }
  // heads of the warp, then warps of the block
#pragma unroll
  for (int i = 0; i < kVec; ++i)
    for (int o = p.group; o < 32; o <<= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
  if (w.sub == 0 && w.live) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) fold[warp][w.e0 + i] = acc[i];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.D; e += blockDim.x) {
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) sum += fold[k][e];
    p.partial[static_cast<long>(blockIdx.x) * p.D + e] = sum;
  }
}

// dw of both sides from the blocks' rows: one block per 32 elements, 32 warps over the rows.
__global__ void __launch_bounds__(1024)
rotary_dw_kernel(const float* __restrict__ partial, int blocks0, int blocks1, int D,
                 float* __restrict__ dw0, float* __restrict__ dw1) {
  __shared__ float sums[32][33];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int e = blockIdx.x * 32 + lane;
  const bool second = blockIdx.y == 1;
  const int rows = second ? blocks1 : blocks0;
  const float* src = partial + (second ? static_cast<long>(blocks0) * D : 0);
  float sum = 0.f;
  if (e < D)
    for (int r = warp; r < rows; r += 32) sum += src[static_cast<long>(r) * D + e];
  sums[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && e < D) {
    float total = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) total += sums[k][lane];
    (second ? dw1 : dw0)[e] = total;
  }
}

// ------------------------------------------------------------------ host ----
bool aligned(const void* base, long b, long h, long t, int size) {
  return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && (b * size) % 16 == 0 &&
         (h * size) % 16 == 0 && (t * size) % 16 == 0;
}

int sm_count_here() {
  int device = 0, count = 0;
  if (cudaGetDevice(&device) != cudaSuccess ||
      cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
    return 0;
  return count;
}

int fill(RotaryParams& p, const SflRotaryTensor* tensors, int count, const SflRotaryTable* table,
         int B, int T, int D, float eps, int inverse, int dtype, bool backward) {
  if (tensors == nullptr || table == nullptr || count < 1 || count > 2 || B < 0 || T < 0 || D < 1 ||
      D > kMaxDim || dtype < 0 || dtype > 2)
    return -2;
  if (table->rotated < 0 || table->rotated > D || (table->rotated & 1) || table->rows < 1) return -2;
  if (table->rotated > 0 && (table->cos == nullptr || table->sin == nullptr)) return -2;
  const int size = dtype == 2 ? 4 : 2;
  const bool norm = tensors[0].weight != nullptr;
  for (int i = 0; i < count; ++i) {
    const SflRotaryTensor& q = tensors[i];
    if (q.heads < 1 || q.x == nullptr || q.y == nullptr || (q.weight != nullptr) != norm) return -2;
    if (backward && (q.dy == nullptr || !norm)) return -2;
    Side& s = p.side[i];
    s = Side{q.x, q.y, q.dy, q.weight, q.x_b, q.x_h, q.x_t, q.y_b, q.y_h, q.y_t, q.dy_b, q.dy_h,
             q.dy_t, q.heads, 0};
    s.vec = D % kVec == 0 && aligned(q.x, q.x_b, q.x_h, q.x_t, size) &&
            aligned(q.y, q.y_b, q.y_h, q.y_t, size) &&
            (!backward || aligned(q.dy, q.dy_b, q.dy_h, q.dy_t, size));
  }
  if (count == 1) p.side[1] = p.side[0];
  p.cos = table->cos;
  p.sin = table->sin;
  p.positions = table->positions;
  p.pos_b = table->pos_b;
  p.pos_t = table->pos_t;
  p.table_rows = table->rows;
  p.rotated = table->rotated;
  p.table_vec = (table->rotated / 2) % 4 == 0 && (reinterpret_cast<uintptr_t>(table->cos) & 15) == 0 &&
                (reinterpret_cast<uintptr_t>(table->sin) & 15) == 0;
  p.B = B;
  p.T = T;
  p.D = D;
  p.group = 1;
  while (p.group * kVec < D) p.group *= 2;
  p.eps = eps;
  p.sign = inverse ? -1.f : 1.f;
  p.partial = nullptr;
  return 0;
}

long blocks_for(const RotaryParams& p, const Side& s, int per) {
  const int each = 32 / p.group * per;
  const long items = static_cast<long>(p.B) * p.T * ((s.heads + each - 1) / each);
  return (items + kWarps - 1) / kWarps;
}

int pairing(int half_layout, int rotated) {
  if (!half_layout) return kInterleaved;
  return (rotated / 2) % kVec == 0 ? kHalfShuffle : kHalfShared;
}

template <typename T, int PAIR, bool NORM>
int launch_forward(RotaryParams p, int count, int sms, cudaStream_t stream) {
  auto go = [&](auto kernel, int per) -> int {
    const long b0 = blocks_for(p, p.side[0], per);
    const long b1 = count == 2 ? blocks_for(p, p.side[1], per) : 0;
    if (b0 + b1 > 0x7fffffffL) return -2;
    p.blocks0 = static_cast<int>(b0);
    return launch_pdl(kernel, dim3(static_cast<unsigned>(b0 + b1)), dim3(32 * kWarps), 0, stream, p);
  };
  long few = blocks_for(p, p.side[0], 4) + (count == 2 ? blocks_for(p, p.side[1], 4) : 0);
  if (few >= 2L * sms) return go(rotary_kernel<T, PAIR, NORM, 4>, 4);
  return go(rotary_kernel<T, PAIR, NORM, 1>, 1);
}

template <typename T>
int forward_of(const RotaryParams& p, int count, int pair, bool norm, int sms, cudaStream_t stream) {
  switch (pair * 2 + (norm ? 1 : 0)) {
    case 0: return launch_forward<T, kInterleaved, false>(p, count, sms, stream);
    case 1: return launch_forward<T, kInterleaved, true>(p, count, sms, stream);
    case 2: return launch_forward<T, kHalfShuffle, false>(p, count, sms, stream);
    case 3: return launch_forward<T, kHalfShuffle, true>(p, count, sms, stream);
    case 4: return launch_forward<T, kHalfShared, false>(p, count, sms, stream);
    default: return launch_forward<T, kHalfShared, true>(p, count, sms, stream);
  }
}

// Warps of the persistent backward grid share the tokens; each side gets blocks in proportion
// to its heads, and no more than it has work for.
constexpr int kBwdPer = 2;
constexpr int kBwdBlocksPerSm = 3;

void backward_blocks(const RotaryParams& p, int count, int sms, int* b0, int* b1) {
  const long total = static_cast<long>(sms) * kBwdBlocksPerSm;
  const long heads = p.side[0].heads + (count == 2 ? p.side[1].heads : 0);
  auto share = [&](const Side& s) {
    long want = total * s.heads / heads;
    const long most = blocks_for(p, s, kBwdPer);
    if (want > most) want = most;
    return static_cast<int>(want < 1 ? 1 : want);
  };
  *b0 = share(p.side[0]);
  *b1 = count == 2 ? share(p.side[1]) : 0;
}

template <typename T>
int backward_of(const RotaryParams& p, int pair, int grid, cudaStream_t stream) {
  auto go = [&](auto kernel) {
    return launch_pdl(kernel, dim3(grid), dim3(32 * kWarps), 0, stream, p);
  };
  if (pair == kInterleaved) return go(rotary_bwd_kernel<T, kInterleaved, kBwdPer>);
  if (pair == kHalfShuffle) return go(rotary_bwd_kernel<T, kHalfShuffle, kBwdPer>);
  return go(rotary_bwd_kernel<T, kHalfShared, kBwdPer>);
}

}  // namespace
}  // namespace sfl

extern "C" int sfl_rotary(const SflRotaryTensor* tensors, int count, const SflRotaryTable* table,
                          int B, int T, int D, float eps, int half_layout, int inverse, int dtype,
                          void* stream) {
  using namespace sfl;
  RotaryParams p{};
  const int bad = fill(p, tensors, count, table, B, T, D, eps, inverse, dtype, false);
  if (bad != 0) return bad;
  if (B == 0 || T == 0) return 0;
  const int sms = sm_count_here();
  if (sms == 0) return -1;
  const int pair = pairing(half_layout, p.rotated);
  const bool norm = tensors[0].weight != nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == 0) return forward_of<__nv_bfloat16>(p, count, pair, norm, sms, st);
  if (dtype == 1) return forward_of<__half>(p, count, pair, norm, sms, st);
  return forward_of<float>(p, count, pair, norm, sms, st);
}

extern "C" long sfl_rotary_bwd_partial_bytes(int heads0, int heads1, int B, int T, int D) {
  using namespace sfl;
  if (heads0 < 1 || heads1 < 0 || B < 1 || T < 1 || D < 1 || D > kMaxDim) return -1;
  const int sms = sm_count_here();
  if (sms == 0) return -1;
  // an upper bound that does not depend on the pairing: every block of the grid leaves a row
  return (static_cast<long>(sms) * kBwdBlocksPerSm + 2) * D * static_cast<long>(sizeof(float));
}

extern "C" int sfl_rotary_bwd(const SflRotaryTensor* tensors, int count,
                              const SflRotaryTable* table, int B, int T, int D, float eps,
                              int half_layout, int dtype, float* partial, long partial_bytes,
                              float* dw0, float* dw1, void* stream) {
  using namespace sfl;
  RotaryParams p{};
  const int bad = fill(p, tensors, count, table, B, T, D, eps, 1, dtype, true);
  if (bad != 0) return bad;
  if (partial == nullptr || dw0 == nullptr || (count == 2 && dw1 == nullptr)) return -2;
  if (B == 0 || T == 0) return -2;
  const int sms = sm_count_here();
  if (sms == 0) return -1;
  int b0, b1;
  backward_blocks(p, count, sms, &b0, &b1);
  if (static_cast<long>(b0 + b1) * D * static_cast<long>(sizeof(float)) > partial_bytes) return -2;
  p.blocks0 = b0;
  p.partial = partial;
  const int pair = pairing(half_layout, p.rotated);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int code;
  if (dtype == 0) code = backward_of<__nv_bfloat16>(p, pair, b0 + b1, st);
  else if (dtype == 1) code = backward_of<__half>(p, pair, b0 + b1, st);
  else code = backward_of<float>(p, pair, b0 + b1, st);
  if (code != 0) return code;
  return launch_pdl(rotary_dw_kernel, dim3((D + 31) / 32, count), dim3(1024), 0, st,
                    static_cast<const float*>(partial), b0, b1, D, dw0, dw1);
}
