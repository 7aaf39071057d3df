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
// The table row of the token is read once for all of them and multiplied by the weights, so that
// a head costs two products per element; partners of the half layout travel between lanes as the
// 16-bit pairs they were loaded as, and arithmetic is done on two fp32 numbers per instruction.
// (A first form with a product per weight, fp32 exchanges, IEEE division and 64-bit index
// arithmetic issued 255 instructions per head group and was bound by them.)  The backward pass
// recomputes the statistics from x, which it has to read anyway, instead of storing them.
//
// Measured at 2 x 32768 tokens of 32 + 8 heads of 128, bf16: forward 247 us for 1.34 GB (5.4 TB/s),
// backward 475 us for 2.0 GB (4.2 TB/s; 40 registers of operands in flight per lane leave it five
// blocks per SM, and a ring of asynchronous copies through shared memory took 598 us).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <type_traits>

#include "launch.cuh"
#include "ptx.cuh"
#include "sfl.h"

namespace sfl {
namespace {

constexpr int kVec = 8;        // elements of a head that one lane holds
constexpr int kWarps = 4;      // warps per block
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
  float inv_dim;
  int chunks0, chunks1;  // warp items per token on each side
  int rounds0, rounds1;  // rounds of PER head groups that one warp item walks
  int tokens;
  float* partial;     // backward with norm: [blocks, D]
};

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

// Two fp32 numbers in one register pair, and the instructions that work on both: these kernels
// are bound by instruction issue as much as by memory.
struct Two { unsigned long long v; };
__device__ __forceinline__ Two two(float lo, float hi) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split(Two a, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v));
}
__device__ __forceinline__ Two mul(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float sum(Two a) {
  float lo, hi;
  split(a, lo, hi);
  return lo + hi;
}
__device__ __forceinline__ Two swapped(Two a) {
  float lo, hi;
  split(a, lo, hi);
  return two(hi, lo);
}
constexpr int kTwos = kVec / 2;

// Two values in one conversion instruction.
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  return pack_bf16(lo, hi);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// The eight elements as they lie in memory, in 32-bit words; converted to fp32 only when they are
// used, so that loads in flight hold 16 bytes (32 for fp32) of registers per lane.  Conversions
// work on words: one shift or mask per bf16 number instead of an extraction and a shift.
template <typename T> struct Raw { uint32_t w[kVec * sizeof(T) / 4]; };

template <typename T>
__device__ __forceinline__ void unpack(const Raw<T>& r, Two (&f)[kTwos]) {
#pragma unroll
  for (int i = 0; i < kTwos; ++i) {
    if constexpr (sizeof(T) == 4) {
      f[i] = two(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
    } else if constexpr (std::is_same<T, __half>::value) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
      f[i] = two(v.x, v.y);
    } else {
      f[i] = two(__uint_as_float(r.w[i] << 16), __uint_as_float(r.w[i] & 0xffff0000u));
    }
  }
}

template <bool VEC, typename T>
__device__ __forceinline__ void load_raw(Raw<T>& r, const T* row, int e0, int D, bool live) {
  constexpr int kQuads = static_cast<int>(sizeof(r.w) / 16);
  if constexpr (VEC) {
    const uint4* src = reinterpret_cast<const uint4*>(row + e0);
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const uint4 q = live ? src[i] : make_uint4(0, 0, 0, 0);
      r.w[4 * i] = q.x; r.w[4 * i + 1] = q.y; r.w[4 * i + 2] = q.z; r.w[4 * i + 3] = q.w;
    }
  } else {
    T v[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      v[i] = live && e0 + i < D ? row[e0 + i] : from_f32<T>(0.f);
    memcpy(r.w, v, sizeof(v));
  }
}

template <bool VEC, typename T>
__device__ __forceinline__ void store_raw(T* row, const Two (&g)[kTwos], int e0, int D) {
  float f[kVec];
#pragma unroll
  for (int i = 0; i < kTwos; ++i) split(g[i], f[2 * i], f[2 * i + 1]);
  if constexpr (VEC && sizeof(T) == 4) {
    float4* dst = reinterpret_cast<float4*>(row + e0);
    dst[0] = make_float4(f[0], f[1], f[2], f[3]);
    dst[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else if constexpr (VEC) {
    *reinterpret_cast<uint4*>(row + e0) = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]),
                                                     pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (e0 + i < D) row[e0 + i] = from_f32<T>(f[i]);
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

// The other element of each pair, as loaded.  All lanes of the warp take part.  Lanes beyond the
// rotated ones get zeros: S is zero there, and an infinity times zero would be NaN.
template <typename T, int PAIR>
__device__ __forceinline__ void partners(const RotaryParams& p, const Raw<T>& mine, Raw<T>& other,
                                         int e0, int lane, T* strip) {
  if constexpr (PAIR == kHalfShuffle) {
    const int half = p.rotated >> 1;
    const bool turns = e0 < p.rotated;
    const int src = turns ? (e0 < half ? lane + half / kVec : lane - half / kVec) : lane;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(mine.w) / 4); ++i) {
      const uint32_t got = __shfl_sync(0xffffffffu, mine.w[i], src);
      other.w[i] = turns ? got : 0u;
    }
  } else if constexpr (PAIR == kHalfShared) {
    const int half = p.rotated >> 1;
    const T* head = strip + (lane * kVec - e0);  // the head's first element
    __syncwarp();
    memcpy(strip + lane * kVec, mine.w, sizeof(mine.w));
    __syncwarp();
    T v[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int e = e0 + i;
      v[i] = e < p.rotated ? head[e < half ? e + half : e - half] : from_f32<T>(0.f);
    }
    memcpy(other.w, v, sizeof(v));
  }
}

__device__ __forceinline__ void pair_up(const float (&f)[kVec], Two (&g)[kTwos]) {
#pragma unroll
  for (int i = 0; i < kTwos; ++i) g[i] = two(f[2 * i], f[2 * i + 1]);
}

// f_e = own_e C_e + partner_e S_e
template <typename T, int PAIR>
__device__ __forceinline__ void combine(const RotaryParams& p, const Two (&own)[kTwos],
                                        const Raw<T>& other, const Two (&C)[kTwos],
                                        const Two (&S)[kTwos], int e0, Two (&f)[kTwos]) {
  if constexpr (PAIR == kInterleaved) {
#pragma unroll
    for (int i = 0; i < kTwos; ++i) {
      f[i] = mul(own[i], C[i]);
      if (e0 + 2 * i < p.rotated) f[i] = fma(swapped(own[i]), S[i], f[i]);
    }
  } else {
    Two partner[kTwos];
    unpack(other, partner);
#pragma unroll
    for (int i = 0; i < kTwos; ++i) f[i] = fma(partner[i], S[i], mul(own[i], C[i]));
  }
}

// Eight weights from element e, zero beyond the head.
template <bool VEC>
__device__ __forceinline__ void load_weights(const float* weight, int e, int D, float (&w)[kVec]) {
  if constexpr (VEC) {
    const float4* src = reinterpret_cast<const float4*>(weight + (e < D ? e : 0));
    const float4 a = src[0], b = src[1];
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) w[i] = e + i < D ? weight[e + i] : 0.f;
  }
}

// Half layout: the element whose weight multiplies the partner of element e.
__device__ __forceinline__ int partner_of(const RotaryParams& p, int e) {
  if (e >= p.rotated) return e;
  const int half = p.rotated >> 1;
  return e < half ? e + half : e - half;
}

__device__ __forceinline__ float group_sum(float v, int group) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < group) v += __shfl_xor_sync(0xffffffffu, v, o);  // group is uniform
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

// One warp takes PER head groups of one token.  PER = 4 keeps 2 KB of loads in flight per warp;
// PER = 1 is for calls with few tokens, which are over sooner when every head group has a warp
// of its own.  Kernel time at 40 heads of 128, PER 1 against 4: one token 2.1 and 2.7 us, 16
// tokens 2.2 and 2.8; at 512 tokens of 32 heads of 64, 256 blocks of PER 4, 3.3 and 3.0.
template <typename T, int PAIR, bool VEC, bool NORM, int PER>
__global__ void __launch_bounds__(32 * kWarps, PER == 4 && VEC && sizeof(T) == 2 ? 8 : 4)
rotary_kernel(const __grid_constant__ RotaryParams p) {
  __shared__ __align__(16) T strips[PAIR == kHalfShared ? kWarps * 32 * kVec : 1];
  // Only the short form lets its successor in early: waiting CTAs would take the slots of this
  // kernel's later ones (measured on the long form: 1150 us against 845 us, run by itself).
  if constexpr (PER == 1) pdl_launch_dependents();
  pdl_wait();
  const unsigned chunks = p.chunks0 + p.chunks1;
  const unsigned block_token = blockIdx.x / chunks;
  int chunk = blockIdx.x - block_token * chunks;
  const bool first = chunk < p.chunks0;
  if (!first) chunk -= p.chunks0;
  const Side& s = p.side[first ? 0 : 1];
  const int warp = threadIdx.x >> 5;
  const Where w = where(p);
  T* strip = strips + (PAIR == kHalfShared ? warp * 32 * kVec : 0);
  const int heads_per = 32 / p.group;
  const unsigned token = block_token * kWarps + warp;
  if (token >= static_cast<unsigned>(p.tokens)) return;  // warp-uniform
  const int b = token / static_cast<unsigned>(p.T), t = token - b * p.T;
  const int rounds = first ? p.rounds0 : p.rounds1;
  int h0 = chunk * rounds * heads_per * PER + w.sub;
  const T* x = static_cast<const T*>(s.x) + b * s.x_b + t * s.x_t + h0 * s.x_h;
  T* y = static_cast<T*>(s.y) + b * s.y_b + t * s.y_t + h0 * s.y_h;
  Raw<T> raw[PER];
  const long x_step = heads_per * s.x_h, y_step = heads_per * s.y_h;
  auto load = [&] {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      load_raw<VEC>(raw[j], x + j * x_step, w.e0, p.D,
                    w.live && h0 + j * heads_per < s.heads);
  };
  load();
  float C[kVec], S[kVec];
  load_angles<PAIR>(p, b, t, w.e0, C, S);
  if constexpr (NORM) {
    float own[kVec];
    load_weights<VEC>(s.weight, w.e0, p.D, own);
#pragma unroll
    for (int i = 0; i < kVec; ++i) C[i] *= own[i];
    if constexpr (PAIR == kInterleaved) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) S[i] *= own[i ^ 1];
    } else if constexpr (PAIR == kHalfShuffle) {
      load_weights<VEC>(s.weight, partner_of(p, w.e0), p.D, own);
#pragma unroll
      for (int i = 0; i < kVec; ++i) S[i] *= own[i];
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        S[i] *= w.e0 + i < p.D ? s.weight[partner_of(p, w.e0 + i)] : 0.f;
    }
  }
  Two C2[kTwos], S2[kTwos];
  pair_up(C, C2);
  pair_up(S, S2);
  for (int round = 0;;) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      Two own[kTwos], f[kTwos];
      unpack(raw[j], own);
      Two scale;
      if constexpr (NORM) {
        Two sq = mul(own[0], own[0]);
#pragma unroll
        for (int i = 1; i < kTwos; ++i) sq = fma(own[i], own[i], sq);
        const float rstd = rsqrtf(fmaf(group_sum(sum(sq), p.group), p.inv_dim, p.eps));
        scale = two(rstd, rstd);
      }
      Raw<T> other;
      partners<T, PAIR>(p, raw[j], other, w.e0, w.lane, strip);
      combine<T, PAIR>(p, own, other, C2, S2, w.e0, f);
      if constexpr (NORM) {
#pragma unroll
        for (int i = 0; i < kTwos; ++i) f[i] = mul(f[i], scale);
      }
      if (w.live && h0 + j * heads_per < s.heads)
        store_raw<VEC>(y + j * y_step, f, w.e0, p.D);
    }
    if (++round == rounds) break;
    h0 += heads_per * PER;
    if (h0 - w.sub >= s.heads) break;  // warp-uniform
    x += PER * x_step;
    y += PER * y_step;
    load();
  }
}

// Backward with the norm.  A persistent grid: every warp keeps the weight gradient of its
// eight elements in registers over all its tokens; the block folds its warps in a fixed order
// and leaves one row of partial sums (deterministic, no atomics).  Two head groups per round and
// five blocks per SM: 2 x 32768 tokens of 40 heads take 475 us, 16 x 512 tokens of 32 heads of 64
// 16.6; six blocks 463 and 17.8, seven 541 and 17.6, one group and eight blocks 581 and 24.9.
constexpr int kBwdBlocksPerSm = 5;

template <typename T, int PAIR, bool VEC, int PER>
__global__ void __launch_bounds__(32 * kWarps, VEC && sizeof(T) == 2 ? kBwdBlocksPerSm : 4)
rotary_bwd_kernel(const __grid_constant__ RotaryParams p) {
  __shared__ __align__(16) T strips[PAIR == kHalfShared ? kWarps * 32 * kVec : 1];
  __shared__ float fold[kWarps][kMaxDim];
  __shared__ __align__(16) float weights[kMaxDim];  // eight registers per lane fewer than held there
  pdl_wait();
  const bool first = static_cast<int>(blockIdx.x) < p.blocks0;
  const Side& s = p.side[first ? 0 : 1];
  const unsigned block = first ? blockIdx.x : blockIdx.x - p.blocks0;
  const unsigned blocks = first ? p.blocks0 : gridDim.x - p.blocks0;
  const int warp = threadIdx.x >> 5;
  const Where w = where(p);
  T* strip = strips + (PAIR == kHalfShared ? warp * 32 * kVec : 0);
  const int heads_per = 32 / p.group;
  const unsigned chunks = first ? p.chunks0 : p.chunks1;
  const int rounds = first ? p.rounds0 : p.rounds1;
  const unsigned items = static_cast<unsigned>(p.tokens) * chunks;  // below 2^31

  for (int e = threadIdx.x; e < kMaxDim; e += blockDim.x) weights[e] = e < p.D ? s.weight[e] : 0.f;
  __syncthreads();
  const float4* my_weights = reinterpret_cast<const float4*>(weights + w.e0);
  Two acc[kTwos];
#pragma unroll
  for (int i = 0; i < kTwos; ++i) acc[i] = two(0.f, 0.f);
  for (unsigned item = block * kWarps + warp; item < items; item += blocks * kWarps) {
    const unsigned token = item / chunks;
    int h0 = static_cast<int>(item - token * chunks) * rounds * heads_per * PER + w.sub;
    const int b = token / static_cast<unsigned>(p.T), t = token - b * p.T;
    const T* x = static_cast<const T*>(s.x) + b * s.x_b + t * s.x_t + h0 * s.x_h;
    const T* dy = static_cast<const T*>(s.dy) + b * s.dy_b + t * s.dy_t + h0 * s.dy_h;
    T* dx = static_cast<T*>(s.y) + b * s.y_b + t * s.y_t + h0 * s.y_h;
    Raw<T> rx[PER], rg[PER];
    auto load = [&] {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const bool live = w.live && h0 + j * heads_per < s.heads;
        load_raw<VEC>(rx[j], x + j * heads_per * s.x_h, w.e0, p.D, live);
        load_raw<VEC>(rg[j], dy + j * heads_per * s.dy_h, w.e0, p.D, live);
      }
    };
    load();
    Two C2[kTwos], S2[kTwos];
    {
      float C[kVec], S[kVec];
      load_angles<PAIR>(p, b, t, w.e0, C, S);
      pair_up(C, C2);
      pair_up(S, S2);
    }
    for (int round = 0;;) {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        Raw<T> other;
        partners<T, PAIR>(p, rg[j], other, w.e0, w.lane, strip);
        Two v[kTwos], u[kTwos];
        unpack(rg[j], u);
        combine<T, PAIR>(p, u, other, C2, S2, w.e0, v);
        unpack(rx[j], u);
        const float4 w0 = my_weights[0], w1 = my_weights[1];
        const Two weight[kTwos] = {two(w0.x, w0.y), two(w0.z, w0.w), two(w1.x, w1.y), two(w1.z, w1.w)};
        Two sq2 = mul(u[0], u[0]), dot2 = mul(mul(v[0], weight[0]), u[0]);
#pragma unroll
        for (int i = 1; i < kTwos; ++i) {
          sq2 = fma(u[i], u[i], sq2);
          dot2 = fma(mul(v[i], weight[i]), u[i], dot2);
        }
        const float sq = group_sum(sum(sq2), p.group);
        const float dot = group_sum(sum(dot2), p.group);
        const float rstd = rsqrtf(fmaf(sq, p.inv_dim, p.eps));
        const float pull = -dot * p.inv_dim * rstd * rstd * rstd;  // -mean(v w xhat) / mean square
        if (w.live && h0 + j * heads_per < s.heads) {
          const Two scale = two(rstd, rstd), back = two(pull, pull);
#pragma unroll
          for (int i = 0; i < kTwos; ++i) {
            const Two vs = mul(v[i], scale);
            acc[i] = fma(vs, u[i], acc[i]);
            v[i] = fma(u[i], back, mul(vs, weight[i]));
          }
          store_raw<VEC>(dx + j * heads_per * s.y_h, v, w.e0, p.D);
        }
      }
      if (++round == rounds) break;
      h0 += heads_per * PER;
      if (h0 - w.sub >= s.heads) break;  // warp-uniform
      x += heads_per * PER * s.x_h;
      dy += heads_per * PER * s.dy_h;
      dx += heads_per * PER * s.y_h;
      load();
    }
  }
  // heads of the warp, then warps of the block
#pragma unroll
  for (int i = 0; i < kTwos; ++i) {
    float each[2];
    split(acc[i], each[0], each[1]);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      for (int o = p.group; o < 32; o <<= 1) each[k] += __shfl_xor_sync(0xffffffffu, each[k], o);
      if (w.sub == 0 && w.live) fold[warp][w.e0 + 2 * i + k] = each[k];
    }
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
  if (e < D) {
#pragma unroll 8
    for (int r = warp; r < rows; r += 32) sum += src[static_cast<long>(r) * D + e];
  }
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
         int B, int T, int D, float eps, int inverse, int dtype, bool backward, bool* vec) {
  *vec = true;
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
             q.dy_t, q.heads};
    // 16-byte accesses need every head row of x, y (and dy) to start on a 16-byte boundary
    *vec = *vec && D % kVec == 0 && aligned(q.x, q.x_b, q.x_h, q.x_t, size) &&
           aligned(q.y, q.y_b, q.y_h, q.y_t, size) &&
           (!backward || aligned(q.dy, q.dy_b, q.dy_h, q.dy_t, size)) &&
           (reinterpret_cast<uintptr_t>(q.weight) & 15) == 0;
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
  if (static_cast<long>(B) * T > 0x7fffffffL) return -2;
  p.B = B;
  p.T = T;
  p.D = D;
  p.tokens = B * T;
  p.inv_dim = 1.0f / static_cast<float>(D);
  p.group = 1;
  while (p.group * kVec < D) p.group *= 2;
  p.eps = eps;
  p.sign = inverse ? -1.f : 1.f;
  p.partial = nullptr;
  return 0;
}

// Warp items per token.  A warp that walks all heads of its token reads the angles and weights
// once for them (237 -> 172 instructions per head group at 16 heads of 64); with fewer tokens
// than keep the SMs busy that way, the heads are spread over more warps.
void set_chunks(RotaryParams& p, int count, int per, long warps_wanted) {
  const int each = 32 / p.group * per;
  const int all0 = (p.side[0].heads + each - 1) / each;
  const int all1 = count == 2 ? (p.side[1].heads + each - 1) / each : 0;
  int rounds = all0 > all1 ? all0 : all1;
  auto items = [&](int r) { return static_cast<long>(p.tokens) * ((all0 + r - 1) / r + (all1 + r - 1) / r); };
  while (rounds > 1 && items(rounds) < warps_wanted) rounds = (rounds + 1) / 2;
  p.rounds0 = p.rounds1 = rounds;
  p.chunks0 = (all0 + rounds - 1) / rounds;
  p.chunks1 = (all1 + rounds - 1) / rounds;
}

// Unaligned rows are read element by element; of the half layout's forms only the one through
// shared memory exists for them.
int pairing(int half_layout, int rotated, bool vec) {
  if (!half_layout) return kInterleaved;
  return vec && (rotated / 2) % kVec == 0 ? kHalfShuffle : kHalfShared;
}

template <typename T, int PAIR, bool VEC, bool NORM>
int launch_forward(RotaryParams p, int count, int sms, cudaStream_t stream) {
  const long token_blocks = (p.tokens + kWarps - 1L) / kWarps;
  auto go = [&](auto kernel) -> int {
    const long blocks = token_blocks * (p.chunks0 + p.chunks1);
    if (blocks > 0x7fffffffL) return -2;
    return launch_pdl(kernel, dim3(static_cast<unsigned>(blocks)), dim3(32 * kWarps), 0, stream, p);
  };
  set_chunks(p, count, 4, 64L * sms);  // two rounds of 32 resident warps per SM
  if (token_blocks * (p.chunks0 + p.chunks1) >= sms)
    return go(rotary_kernel<T, PAIR, VEC, NORM, 4>);
  set_chunks(p, count, 1, 64L * sms);
  return go(rotary_kernel<T, PAIR, VEC, NORM, 1>);
}

template <typename T, bool NORM>
int forward_of(const RotaryParams& p, int count, int pair, bool vec, int sms, cudaStream_t stream) {
  if (vec) {
    if (pair == kInterleaved) return launch_forward<T, kInterleaved, true, NORM>(p, count, sms, stream);
    if (pair == kHalfShuffle) return launch_forward<T, kHalfShuffle, true, NORM>(p, count, sms, stream);
    return launch_forward<T, kHalfShared, true, NORM>(p, count, sms, stream);
  }
  if (pair == kInterleaved) return launch_forward<T, kInterleaved, false, NORM>(p, count, sms, stream);
  return launch_forward<T, kHalfShared, false, NORM>(p, count, sms, stream);
}

// Warps of the persistent backward grid share the tokens; each side gets blocks in proportion
// to its heads, and no more than it has work for.  Returns false beyond 32-bit item counts.
constexpr int kBwdPer = 2;

bool backward_blocks(RotaryParams& p, int count, int sms, int* b0, int* b1) {
  set_chunks(p, count, kBwdPer, 4L * kBwdBlocksPerSm * kWarps * sms);
  const long total = static_cast<long>(sms) * kBwdBlocksPerSm;
  const long heads = p.side[0].heads + (count == 2 ? p.side[1].heads : 0);
  auto share = [&](const Side& s, int chunks) {
    long want = total * s.heads / heads;
    const long most = (static_cast<long>(p.tokens) * chunks + kWarps - 1) / kWarps;
    if (want > most) want = most;
    return static_cast<int>(want < 1 ? 1 : want);
  };
  *b0 = share(p.side[0], p.chunks0);
  *b1 = count == 2 ? share(p.side[1], p.chunks1) : 0;
  // the grid's stride past the last item must not wrap either
  const long most = p.chunks0 > p.chunks1 ? p.chunks0 : p.chunks1;
  return p.tokens * most + total * kWarps <= 0x7fffffffL;
}

template <typename T>
int backward_of(const RotaryParams& p, int pair, bool vec, int grid, cudaStream_t stream) {
  auto go = [&](auto kernel) {
    return launch_pdl(kernel, dim3(grid), dim3(32 * kWarps), 0, stream, p);
  };
  if (vec) {
    if (pair == kInterleaved) return go(rotary_bwd_kernel<T, kInterleaved, true, kBwdPer>);
    if (pair == kHalfShuffle) return go(rotary_bwd_kernel<T, kHalfShuffle, true, kBwdPer>);
    return go(rotary_bwd_kernel<T, kHalfShared, true, kBwdPer>);
  }
  if (pair == kInterleaved) return go(rotary_bwd_kernel<T, kInterleaved, false, kBwdPer>);
  return go(rotary_bwd_kernel<T, kHalfShared, false, kBwdPer>);
}

}  // namespace
}  // namespace sfl

extern "C" int sfl_rotary(const SflRotaryTensor* tensors, int count, const SflRotaryTable* table,
                          int B, int T, int D, float eps, int half_layout, int inverse, int dtype,
                          void* stream) {
  using namespace sfl;
  RotaryParams p{};
  bool vec;
  const int bad = fill(p, tensors, count, table, B, T, D, eps, inverse, dtype, false, &vec);
  if (bad != 0) return bad;
  if (B == 0 || T == 0) return 0;
  const int sms = sm_count_here();
  if (sms == 0) return -1;
  const int pair = pairing(half_layout, p.rotated, vec);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto of = [&](auto zero) -> int {
    using T = decltype(zero);
    return tensors[0].weight != nullptr ? forward_of<T, true>(p, count, pair, vec, sms, st)
                                        : forward_of<T, false>(p, count, pair, vec, sms, st);
  };
  if (dtype == 0) return of(__nv_bfloat16{});
  if (dtype == 1) return of(__half{});
  return of(0.f);
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
  bool vec;
  const int bad = fill(p, tensors, count, table, B, T, D, eps, 1, dtype, true, &vec);
  if (bad != 0) return bad;
  if (partial == nullptr || dw0 == nullptr || (count == 2 && dw1 == nullptr)) return -2;
  if (B == 0 || T == 0) return -2;
  const int sms = sm_count_here();
  if (sms == 0) return -1;
  int b0, b1;
  if (!backward_blocks(p, count, sms, &b0, &b1)) return -2;
  if (static_cast<long>(b0 + b1) * D * static_cast<long>(sizeof(float)) > partial_bytes) return -2;
  p.blocks0 = b0;
  p.partial = partial;
  const int pair = pairing(half_layout, p.rotated, vec);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int code;
  if (dtype == 0) code = backward_of<__nv_bfloat16>(p, pair, vec, b0 + b1, st);
  else if (dtype == 1) code = backward_of<__half>(p, pair, vec, b0 + b1, st);
  else code = backward_of<float>(p, pair, vec, b0 + b1, st);
  if (code != 0) return code;
  return launch_pdl(rotary_dw_kernel, dim3((D + 31) / 32, count), dim3(1024), 0, st,
                    static_cast<const float*>(partial), b0, b1, D, dw0, dw1);
}
