// Orthogonalised updates: Newton-Schulz products over a stack of matrices.
//
//   X = U / (|U|_F + eps);   repeat:  G = X X^T,  X <- a X + (b G + c G G) X
//
// (the Gram matrix of the shorter side: X^T X on the right for tall matrices, so nothing is
// transposed).  Singular vectors stay, singular values go through the odd quintic
// a s + b s^3 + c s^5 each time.  The reference trains with AdamW only (src/llmlab/train.py:169);
// the operator serves optim.FusedMuon.
//
// All products run on CTA-pair tensor-core tiles (pair_gemm.cuh), one launch per product for the
// whole stack.  The two Gram-sized products are symmetric: only tiles on and above the diagonal
// are computed and stored.  Where a later product needs a tile below it, it loads the stored one
// as an MN-major operand - the tensor cores read either orientation, step by step.  A tile on the
// diagonal has the same rows as both operands and loads them once.
//
// Precision.  The quintic multiplies small singular values by 3.4 a step, and with them whatever
// was rounded away: five steps in bf16 are off by 1 to 5 percent.  Operands are therefore fp16,
// times 2^12: entries of X, G and b G + c G G are at most 1.2, 1.5 and 2.8 (X's singular values
// never exceed 1.2), far below 65504 / 4096, and their small entries stay normal numbers down to
// 2^-26.  X itself is carried as hi + lo, two fp16 numbers with 22 bits between them, of which hi
// is what the tensor cores multiply: a X is then exact to fp32 and the rounding of hi does not
// compound.  In the last two steps singular values are spread less and most are near 1, where a X
// and P X nearly cancel; there lo is dropped and X <- (P + a I) hi, one product whose factors are
// smaller than the terms they replace.  Sums are fp32, the norm is accumulated in 64 bits.
// Measured against 64 bits: 1.8e-3 to 2.3e-3 of the result's norm, of which its rounding to bf16 is
// 1.7e-3 (hi alone throughout: up to 1e-2; a X apart in every step: up to 2.7e-3).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "pair_gemm.cuh"
#include "sfl.h"

namespace sfl {
namespace {

using pair::EpiContext;
using pair::Tile;

constexpr float kScale = 4096.0f;

// ------------------------------------------------------------- norm and split ----
struct Stack {
  const void* base;
  long stride0, stride1, row;  // matrix z starts at (z / inner) * stride0 + (z % inner) * stride1
  int inner;
};
template <typename T>
__device__ __forceinline__ const T* matrix(const Stack& s, int z) {
  return static_cast<const T*>(s.base) + (z / s.inner) * s.stride0 + (z % s.inner) * s.stride1;
}
__device__ __forceinline__ float wide(float v) { return v; }
__device__ __forceinline__ float wide(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float wide(__half v) { return __half2float(v); }

constexpr int kChunks = 64;       // blocks per matrix, and partial sums of its norm
constexpr int kNormThreads = 256;

// Four elements of a row from column c (a multiple of 4), zero beyond the row.
template <typename T>
__device__ __forceinline__ void load4(const T* row, int c, int n, bool vec, float (&v)[4]) {
  if (vec && c + 4 <= n) {
    if constexpr (sizeof(T) == 4) {
      const float4 q = *reinterpret_cast<const float4*>(row + c);
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
      const uint2 q = *reinterpret_cast<const uint2*>(row + c);
      const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = wide(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = c + i < n ? wide(row[c + i]) : 0.f;
  }
}

// A block's share of a matrix: its threads lie side by side along a row (or along several short
// rows), and each visits kDepth rows at a time so that as many loads are in flight.
constexpr int kDepth = 4;
template <class F>
__device__ __forceinline__ void walk(int m, int quads, F&& visit) {
  const unsigned across = quads < kNormThreads ? quads : kNormThreads;
  const unsigned down = kNormThreads / across;
  const unsigned r_in = threadIdx.x / across, c_in = threadIdx.x - r_in * across;
  if (r_in >= down) return;
  const long step = static_cast<long>(gridDim.x) * down;
  for (int q = c_in; q < quads; q += across)
    for (long r = blockIdx.x * static_cast<long>(down) + r_in; r < m; r += step * kDepth)
      visit(r, step, q);
}

// Sum of squares of each block's share of a matrix.  64-bit sums: squares of fp32 entries neither
// overflow nor vanish in them.
template <typename T>
__global__ void __launch_bounds__(kNormThreads)
ns_norm_kernel(Stack s, int m, int n, int vec, double* __restrict__ partial) {
  __shared__ double sums[kNormThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const T* src = matrix<T>(s, blockIdx.y);
  const int quads = (n + 3) >> 2;
  double sum = 0.0;
  walk(m, quads, [&](long r, long step, int q) {
    float v[kDepth][4];
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const bool in = r + d * step < m;
      load4(src + (in ? r + d * step : r) * s.row, in ? q * 4 : n, n, vec, v[d]);
    }
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double x = v[d][j];
        sum = fma(x, x, sum);
      }
    }
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = 0.0;
#pragma unroll
    for (int k = 0; k < kNormThreads / 32; ++k) all += sums[k];
    partial[static_cast<long>(blockIdx.y) * gridDim.x + blockIdx.x] = all;
  }
}

// hi + lo = 2^12 U / (|U| + eps), rows padded to a pitch of ld (a multiple of 8) with zeros.
template <typename T>
__global__ void __launch_bounds__(kNormThreads)
ns_split_kernel(Stack s, int m, int n, int ld, int vec, const double* __restrict__ partial,
                float eps, __half* __restrict__ hi, __half* __restrict__ lo /* may be NULL */) {
  __shared__ float inv_sh;
  pdl_launch_dependents();
  pdl_wait();
  const int z = blockIdx.y;
  if (threadIdx.x < 32) {  // lanes add pairs of the partial sums, then each other
    static_assert(kChunks <= 64, "two partial sums per lane");
    const double* mine = partial + static_cast<long>(z) * gridDim.x;
    double sum = threadIdx.x < gridDim.x ? mine[threadIdx.x] : 0.0;
    if (threadIdx.x + 32 < gridDim.x) sum += mine[threadIdx.x + 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (threadIdx.x == 0) inv_sh = static_cast<float>(kScale / (sqrt(sum) + static_cast<double>(eps)));
  }
  __syncthreads();
  const float inv = inv_sh;
  const T* src = matrix<T>(s, z);
  const long out0 = static_cast<long>(z) * m * ld;
  const int quads = ld >> 2;
  walk(m, quads, [&](long r, long step, int q) {
    float v[kDepth][4];
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const bool in = r + d * step < m;
      load4(src + (in ? r + d * step : r) * s.row, in ? q * 4 : n, n, vec, v[d]);
    }
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      if (r + d * step >= m) break;
      const long at = out0 + (r + d * step) * ld + q * 4;
      __half h[4], l[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = v[d][j] * inv;
        h[j] = __float2half_rn(x);
        l[j] = __float2half_rn(x - __half2float(h[j]));
      }
      *reinterpret_cast<uint2*>(hi + at) = *reinterpret_cast<const uint2*>(h);
      if (lo != nullptr) *reinterpret_cast<uint2*>(lo + at) = *reinterpret_cast<const uint2*>(l);
    }
  });
}

// ------------------------------------------------------------- Muon around it ----
// Rows are layers: `len` consecutive elements (a multiple of 4) of a parameter, `stride` apart in
// the flat buffers and packed in u / o.
//   v <- momentum v + coef g,   u = coef g + momentum v   (or u = v without Nesterov's look-ahead)
__global__ void __launch_bounds__(256)
muon_momentum_kernel(const float* __restrict__ g, float* __restrict__ v, float* __restrict__ u,
                     long quads, long stride, float momentum, int nesterov,
                     const float* __restrict__ coef, const float* __restrict__ ok) {
  pdl_launch_dependents();
  pdl_wait();
  const float c = coef == nullptr ? 1.f : *coef;
  const bool keep = ok != nullptr && *ok == 0.f;  // non-finite gradients: the momentum stays
  const long row = blockIdx.y * stride;
  float4* out = reinterpret_cast<float4*>(u) + blockIdx.y * quads;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < quads; i += gridDim.x * 256L) {
    const float4 a = reinterpret_cast<const float4*>(g + row)[i];
    float4 b = reinterpret_cast<const float4*>(v + row)[i];
    const float4 s = make_float4(a.x * c, a.y * c, a.z * c, a.w * c);
    b = make_float4(fmaf(momentum, b.x, s.x), fmaf(momentum, b.y, s.y), fmaf(momentum, b.z, s.z),
                    fmaf(momentum, b.w, s.w));
    if (!keep) reinterpret_cast<float4*>(v + row)[i] = b;
    out[i] = nesterov ? make_float4(fmaf(momentum, b.x, s.x), fmaf(momentum, b.y, s.y),
                                    fmaf(momentum, b.z, s.z), fmaf(momentum, b.w, s.w))
                      : b;
  }
}

// p <- decay p - rate o, and its bf16 copy
__global__ void __launch_bounds__(256)
muon_apply_kernel(float* __restrict__ p, __nv_bfloat16* __restrict__ shadow,
                  const __nv_bfloat16* __restrict__ o, long quads, long stride, float decay,
                  float rate, const float* __restrict__ ok) {
  pdl_launch_dependents();
  pdl_wait();
  if (ok != nullptr && *ok == 0.f) return;
  const long row = blockIdx.y * stride;
  const uint2* src = reinterpret_cast<const uint2*>(o) + blockIdx.y * quads;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < quads; i += gridDim.x * 256L) {
    float4 a = reinterpret_cast<const float4*>(p + row)[i];
    const uint2 q = src[i];
    const float2 x = unpack_bf16(q.x), y = unpack_bf16(q.y);
    a = make_float4(fmaf(-rate, x.x, a.x * decay), fmaf(-rate, x.y, a.y * decay),
                    fmaf(-rate, y.x, a.z * decay), fmaf(-rate, y.y, a.w * decay));
    reinterpret_cast<float4*>(p + row)[i] = a;
    if (shadow != nullptr)
      reinterpret_cast<uint2*>(shadow + row)[i] = make_uint2(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w));
  }
}

bool rows_ok(const void* p, int rows, long len, long stride, int align) {
  return p != nullptr && (reinterpret_cast<uintptr_t>(p) % align) == 0 && rows >= 1 &&
         rows <= 65535 && len >= 4 && len % 4 == 0 && (rows == 1 || (stride >= len && stride % 4 == 0));
}
dim3 rows_grid(int rows, long len) {
  const long blocks = (len / 4 + 1023) / 1024;  // four steps per thread
  return dim3(static_cast<unsigned>(blocks < 1 ? 1 : (blocks > 65535 ? 65535 : blocks)), rows);
}

// ------------------------------------------------- symmetric products: G, b G + c G G ----
// Of a symmetric matrix the 256 x 256 tiles on and above the diagonal are stored.  As an operand
// with rows of tile i, the steps before turn(i) lie below the diagonal and are read transposed.
__device__ __forceinline__ int turn(int i) { return i * (pair::kTileN / pair::kBK); }

// out = alpha aux + beta A B^T (+ shift I) on and above the diagonal.  Gram matrix: A = B = X;
// polynomial: A = B = G, aux = G.
struct SymOp : pair::NoMaps, pair::RoundRobin {
  static constexpr int kEpiTiles = 2;
  struct Params {
    CUtensorMap k_major, mn_major;  // the operand (X in one orientation, G in both)
    CUtensorMap aux, out;           // 64-column lines of 32 rows
    int total, num_kb;
    bool fp16;
    int* status;
    int nt, per;                    // tiles along a side, tiles per matrix
    int size;                       // rows and columns of the result
    int mn;                         // X is read MN-major
    int gram;                       // 1: Gram matrix, 0: polynomial
    float alpha, beta;
    float shift;                    // added to the diagonal
  };
  static __device__ __forceinline__ Tile tile(const Params& p, int w) {
    const int z = w / p.per;
    int in = w - z * p.per, i = 0;
    while (in >= p.nt - i) {  // row i of the upper triangle has nt - i tiles
      in -= p.nt - i;
      ++i;
    }
    const int j = i + in;
    return Tile{i * pair::kTileM, j * pair::kTileN, z, p.num_kb, 0, 0,
                p.gram ? p.mn * p.num_kb : turn(i), p.gram ? p.mn * p.num_kb : turn(j), in == 0};
  }
  static constexpr int kForms =
      pair::kFormKK | pair::kFormMM | pair::kFormKM | pair::kFormMK | pair::kFormSame;
  static __device__ __forceinline__ const CUtensorMap* map_a_k(const Params& p, const Tile&) {
    return &p.k_major;
  }
  static __device__ __forceinline__ const CUtensorMap* map_b_k(const Params& p, const Tile&) {
    return &p.k_major;
  }
  static __device__ __forceinline__ const CUtensorMap* map_a_mn(const Params& p, const Tile&) {
    return &p.mn_major;
  }
  static __device__ __forceinline__ const CUtensorMap* map_b_mn(const Params& p, const Tile&) {
    return &p.mn_major;
  }
  // The warp's two 64-column chunks have a staging tile each: aux arrives in it, the result
  // replaces it.
  static __device__ __forceinline__ void begin(const Params& p, const Tile& t, EpiContext& c) {
    const int col0 = t.n0 + c.part * 128;
    if (p.gram || c.row0 >= p.size || col0 >= p.size || c.lane != 0) return;
    const bool two = col0 + 64 < p.size;
    tma_store_wait_read<0>();  // the tiles' last stores have read them
    mbar_expect_tx(c.aux_bar, (two ? 2 : 1) * pair::kEpiTileBytes);
    tma_load_3d(c.smem, &p.aux, c.aux_bar, col0, c.row0, t.z);
    if (two) tma_load_3d(c.smem + pair::kEpiTileBytes, &p.aux, c.aux_bar, col0 + 64, c.row0, t.z);
  }
  static __device__ __forceinline__ void epilogue(const Params& p, const Tile& t, EpiContext& c) {
    const int col0 = t.n0 + c.part * 128;
    if (c.row0 >= p.size || col0 >= p.size) return;  // warp-uniform
    if (!p.gram) pair::wait_aux(c);
#pragma unroll 1
    for (int ch = 0; ch < 2; ++ch) {
      const int begin = col0 + ch * 64;
      if (begin >= p.size) break;  // warp-uniform
      uint8_t* tile = c.smem + ch * pair::kEpiTileBytes;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[32];
        pair::load_acc(c.acc + c.part * 128 + ch * 64 + h * 32, v);
        if (p.gram) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] *= p.beta;
          if (h == 0) {  // this tile's store is the one before the last
            if (c.lane == 0) tma_store_wait_read<1>();
            __syncwarp();
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 q = *reinterpret_cast<const uint4*>(pair::tile_chunk(tile, c.lane, 4 * h + j));
            const __half2* e = reinterpret_cast<const __half2*>(&q);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 f = __half22float2(e[k]);
              v[8 * j + 2 * k] = fmaf(v[8 * j + 2 * k], p.beta, p.alpha * f.x);
              v[8 * j + 2 * k + 1] = fmaf(v[8 * j + 2 * k + 1], p.beta, p.alpha * f.y);
            }
          }
          const int diagonal = c.row0 + c.lane - begin - h * 32;
          if (p.shift != 0.f && __any_sync(0xffffffffu, diagonal >= 0 && diagonal < 32)) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (diagonal == j) v[j] += p.shift;
          }
        }
        pair::stage_16(tile, c.lane, h, v, true);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (c.lane == 0) {
        pair::store_3d(&p.out, tile, begin, c.row0, t.z);
        tma_store_commit();
      }
    }
  }
};

// ------------------------------------------------------------ X <- a X + P X ----
struct ApplyOp : pair::NoMaps, pair::RoundRobin {
  static constexpr int kEpiTiles = 2;
  struct Params {
    CUtensorMap x;                 // X: B read MN-major (wide) or A read K-major (tall)
    CUtensorMap p_k, p_mn;         // P, symmetric, in both orientations
    CUtensorMap hi, lo;        // X as it was: 64-column lines of 32 rows; lo is rewritten in place
    CUtensorMap hi_out, out;   // the next hi, or the bf16 result
    int total, num_kb;
    bool fp16;
    int* status;
    int mt, per;
    int m, n;
    int band;                  // row tiles that are walked before the next column tile
    int nt;
    int wide;                  // A = P and B = X (MN-major), else A = X and B = P
    int folded;                // 1: P holds a X as well; hi + lo of X are not read
    int keep_lo;               // 1: write lo of the next X
    int last;                  // 0: next X, 1: result through TMA, 2: result element by element
    float alpha, beta;
    __nv_bfloat16* result;     // [batch, m, n]
  };
  static __device__ __forceinline__ Tile tile(const Params& p, int w) {
    const int z = w / p.per;
    int in = w - z * p.per;
    const int b = in / (p.band * p.nt);
    in -= b * p.band * p.nt;
    const int width = p.mt - b * p.band < p.band ? p.mt - b * p.band : p.band;
    const int n = in / width;
    const int m = b * p.band + in - n * width;
    return Tile{m * pair::kTileM, n * pair::kTileN, z, p.num_kb, 0, p.wide,
                p.wide ? turn(m) : 0, p.wide ? p.num_kb : turn(n), false};
  }
  // wide: A = P in either orientation, B = X MN-major; tall: A = X K-major, B = P in either
  static constexpr int kForms = pair::kFormKK | pair::kFormMM | pair::kFormKM;
  static __device__ __forceinline__ const CUtensorMap* map_a_k(const Params& p, const Tile& t) {
    return t.kind != 0 ? &p.p_k : &p.x;
  }
  static __device__ __forceinline__ const CUtensorMap* map_a_mn(const Params& p, const Tile&) {
    return &p.p_mn;
  }
  static __device__ __forceinline__ const CUtensorMap* map_b_k(const Params& p, const Tile&) {
    return &p.p_k;
  }
  static __device__ __forceinline__ const CUtensorMap* map_b_mn(const Params& p, const Tile& t) {
    return t.kind != 0 ? &p.x : &p.p_mn;
  }
  static __device__ __forceinline__ void load_aux(const Params& p, const Tile& t, EpiContext& c,
                                                  int begin) {
    if (c.lane == 0) {
      tma_store_wait_read<0>();
      mbar_expect_tx(c.aux_bar, 2 * pair::kEpiTileBytes);
      tma_load_3d(c.smem, &p.hi, c.aux_bar, begin, c.row0, t.z);
      tma_load_3d(c.smem + pair::kEpiTileBytes, &p.lo, c.aux_bar, begin, c.row0, t.z);
    }
  }
  static __device__ __forceinline__ void begin(const Params& p, const Tile& t, EpiContext& c) {
    const int col0 = t.n0 + c.part * 128;
    if (!p.folded && c.row0 < p.m && col0 < p.n) load_aux(p, t, c, col0);
  }
  static __device__ __forceinline__ void epilogue(const Params& p, const Tile& t, EpiContext& c) {
    const int col0 = t.n0 + c.part * 128;
    if (c.row0 >= p.m) return;  // warp-uniform
    const int row = c.row0 + c.lane;
#pragma unroll 1
    for (int ch = 0; ch < 2; ++ch) {
      const int begin = col0 + ch * 64;
      if (begin >= p.n) break;  // warp-uniform
      // hi and lo of a chunk take both staging tiles; without them the chunks alternate
      uint8_t* tile = p.folded ? c.smem + ch * pair::kEpiTileBytes : c.smem;
      uint8_t* low = c.smem + pair::kEpiTileBytes;
      if (p.folded) {
        if (c.lane == 0) tma_store_wait_read<1>();
        __syncwarp();
      } else {
        pair::wait_aux(c);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[32];
        pair::load_acc(c.acc + c.part * 128 + ch * 64 + h * 32, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // each lane rewrites exactly the bytes it read
          uint4* qh = reinterpret_cast<uint4*>(pair::tile_chunk(tile, c.lane, 4 * h + j));
          uint4* ql = reinterpret_cast<uint4*>(pair::tile_chunk(low, c.lane, 4 * h + j));
          uint4 a = make_uint4(0, 0, 0, 0), b = a;
          if (!p.folded) {
            a = *qh;
            b = *ql;
          }
          __half2* eh = reinterpret_cast<__half2*>(&a);
          __half2* el = reinterpret_cast<__half2*>(&b);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 fh = __half22float2(eh[k]), fl = __half22float2(el[k]);
            const float x = fmaf(v[8 * j + 2 * k], p.beta, p.alpha * (fh.x + fl.x));
            const float y = fmaf(v[8 * j + 2 * k + 1], p.beta, p.alpha * (fh.y + fl.y));
            if (p.last == 0) {
              eh[k] = __floats2half2_rn(x, y);
              if (p.keep_lo) {
                const float2 r = __half22float2(eh[k]);
                el[k] = __floats2half2_rn(x - r.x, y - r.y);
              }
            } else {
              const uint32_t packed = pack_bf16(x, y);
              eh[k] = *reinterpret_cast<const __half2*>(&packed);
            }
          }
          *qh = a;
          if (p.keep_lo) *ql = b;
          if (p.last == 2 && row < p.m) {
            const __nv_bfloat16* e = reinterpret_cast<const __nv_bfloat16*>(&a);
            const int col = begin + h * 32 + 8 * j;
            __nv_bfloat16* dst = p.result + (static_cast<long>(t.z) * p.m + row) * p.n + col;
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (col + k < p.n) dst[k] = e[k];
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (c.lane == 0 && p.last != 2) {
        if (p.last == 0) {
          pair::store_3d(&p.hi_out, tile, begin, c.row0, t.z);
          if (p.keep_lo) pair::store_3d(&p.lo, low, begin, c.row0, t.z);
        } else {
          pair::store_3d(&p.out, tile, begin, c.row0, t.z);
        }
        tma_store_commit();
      }
      if (!p.folded && ch == 0 && begin + 64 < p.n) load_aux(p, t, c, begin + 64);
    }
  }
};

// ------------------------------------------------------------------- host ----
long round_up(long v, long to) { return (v + to - 1) / to * to; }

int tiles_of(long n, int size) { return static_cast<int>((n + size - 1) / size); }

struct Sizes {
  long ld, gram_ld, x_bytes, gram_bytes, norm_bytes, total;
};

Sizes sizes_of(int batch, int m, int n) {
  Sizes s;
  const long side = m < n ? m : n;
  s.ld = round_up(n, 8);
  s.gram_ld = round_up(side, 8);
  s.x_bytes = round_up(2L * batch * m * s.ld, 256);
  s.gram_bytes = round_up(2L * batch * side * s.gram_ld, 256);
  s.norm_bytes = round_up(8L * batch * kChunks, 256);
  s.total = 3 * s.x_bytes + 2 * s.gram_bytes + s.norm_bytes;  // two hi, lo, G, P, norms
  return s;
}

template <typename T>
int normalise(const Stack& s, int batch, int m, int n, int ld, float eps, double* partial,
              __half* hi, __half* lo, cudaStream_t stream) {
  const int size = sizeof(T);
  const int bytes = 4 * size;  // four elements at a time
  const int vec = (reinterpret_cast<uintptr_t>(s.base) % bytes) == 0 && (s.row * size) % bytes == 0 &&
                  (s.stride0 * size) % bytes == 0 && (s.stride1 * size) % bytes == 0;
  const long quads = static_cast<long>(m) * (ld / 4);
  const long want = (quads + 4L * kNormThreads - 1) / (4L * kNormThreads);
  const int chunks = static_cast<int>(want < 1 ? 1 : (want > kChunks ? kChunks : want));
  int rc = launch_pdl(ns_norm_kernel<T>, dim3(chunks, batch), dim3(kNormThreads), 0, stream, s, m, n,
                      vec, partial);
  if (rc != 0) return rc;
  return launch_pdl(ns_split_kernel<T>, dim3(chunks, batch), dim3(kNormThreads), 0, stream, s, m, n,
                    ld, vec, static_cast<const double*>(partial), eps, hi, lo);
}

}  // namespace
}  // namespace sfl

extern "C" int sfl_muon_momentum(const float* grad, float* momentum_buffer, float* update, int rows,
                                 long len, long stride, float momentum, int nesterov,
                                 const float* grad_coef, const float* ok_flag, void* stream) {
  using namespace sfl;
  if (!rows_ok(grad, rows, len, stride, 16) || !rows_ok(momentum_buffer, rows, len, stride, 16) ||
      !rows_ok(update, rows, len, stride, 16))
    return -2;
  return launch_pdl(muon_momentum_kernel, rows_grid(rows, len), dim3(256), 0,
                    static_cast<cudaStream_t>(stream), grad, momentum_buffer, update, len / 4, stride,
                    momentum, nesterov, grad_coef, ok_flag);
}

extern "C" int sfl_muon_apply(float* param, void* bf16_shadow, const void* update_bf16, int rows,
                              long len, long stride, float decay, float rate, const float* ok_flag,
                              void* stream) {
  using namespace sfl;
  if (!rows_ok(param, rows, len, stride, 16) || !rows_ok(update_bf16, rows, len, stride, 8) ||
      (bf16_shadow != nullptr && !rows_ok(bf16_shadow, rows, len, stride, 8)))
    return -2;
  return launch_pdl(muon_apply_kernel, rows_grid(rows, len), dim3(256), 0,
                    static_cast<cudaStream_t>(stream), param,
                    static_cast<__nv_bfloat16*>(bf16_shadow),
                    static_cast<const __nv_bfloat16*>(update_bf16), len / 4, stride, decay, rate,
                    ok_flag);
}

extern "C" long sfl_newton_schulz_bytes(int batch, int m, int n) {
  using namespace sfl;
  if (batch < 1 || m < 1 || n < 1 || batch > 65535) return -1;
  return sizes_of(batch, m, n).total;
}

extern "C" int sfl_newton_schulz(const SflNewtonSchulz* a, void* stream_) {
  using namespace sfl;
  if (a == nullptr || a->batch < 1 || a->batch > 65535 || a->m < 1 || a->n < 1 || a->inner < 1 ||
      a->steps < 1 || a->steps > 64 || a->dtype < 0 || a->dtype > 2 || a->update == nullptr ||
      a->out == nullptr || a->work == nullptr || (reinterpret_cast<uintptr_t>(a->work) & 255))
    return -2;
  const int batch = a->batch, m = a->m, n = a->n;
  const Sizes z = sizes_of(batch, m, n);
  if (a->work_bytes < z.total) return -2;
  const int side = m < n ? m : n, longer = m < n ? n : m;
  const bool wide = m <= n;
  const int mt = tiles_of(m, pair::kTileM), nt = tiles_of(n, pair::kTileN);
  if (static_cast<long>(batch) * mt * nt > 0x7fffffffL) return -2;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);

  uint8_t* at = static_cast<uint8_t*>(a->work);
  __half* hi[2] = {reinterpret_cast<__half*>(at), reinterpret_cast<__half*>(at + z.x_bytes)};
  __half* lo = reinterpret_cast<__half*>(at + 2 * z.x_bytes);
  __half* gram = reinterpret_cast<__half*>(at + 3 * z.x_bytes);
  __half* poly = reinterpret_cast<__half*>(at + 3 * z.x_bytes + z.gram_bytes);
  double* norms = reinterpret_cast<double*>(at + 3 * z.x_bytes + 2 * z.gram_bytes);

  const Stack s{a->update, a->stride0, a->stride1, a->row, a->inner};
  int rc;
  const int ld = static_cast<int>(z.ld);
  __half* first_lo = a->steps > 2 ? lo : nullptr;  // folded steps read hi alone
  if (a->dtype == 0) rc = normalise<__nv_bfloat16>(s, batch, m, n, ld, a->eps, norms, hi[0], first_lo, stream);
  else if (a->dtype == 1) rc = normalise<__half>(s, batch, m, n, ld, a->eps, norms, hi[0], first_lo, stream);
  else rc = normalise<float>(s, batch, m, n, ld, a->eps, norms, hi[0], first_lo, stream);
  if (rc != 0) return rc;

  const uint64_t x_stride = static_cast<uint64_t>(m) * z.ld;
  const uint64_t g_stride = static_cast<uint64_t>(side) * z.gram_ld;
  const int gt = tiles_of(side, pair::kTileN);

  SymOp::Params q{};
  q.fp16 = true;
  q.status = a->status;
  q.nt = gt;
  q.per = gt * (gt + 1) / 2;
  q.total = batch * q.per;
  q.size = side;
  ApplyOp::Params x{};
  x.fp16 = true;
  x.status = a->status;
  x.mt = mt;
  x.per = mt * nt;
  x.total = batch * x.per;
  x.num_kb = tiles_of(side, pair::kBK);
  x.nt = nt;
  x.band = mt < 8 ? mt : 8;
  x.m = m;
  x.n = n;
  x.wide = wide;
  x.result = static_cast<__nv_bfloat16*>(a->out);
  const bool out_tma = (static_cast<long>(n) * 2) % 16 == 0 &&
                       (reinterpret_cast<uintptr_t>(a->out) & 15) == 0;

  auto gram_map = [&](CUtensorMap* map, __half* g) {
    return pair::map_3d(map, g, 2, side, side, z.gram_ld, batch, g_stride, 64, 32);
  };
  // G and P as operands, in both orientations
  auto symmetric = [&](CUtensorMap* k_major, CUtensorMap* mn_major, __half* g) {
    const int bad = pair::map_operand(k_major, g, false, side, side, z.gram_ld, batch, g_stride);
    return bad != 0 ? bad
                    : pair::map_operand(mn_major, g, true, side, side, z.gram_ld, batch, g_stride);
  };
  auto x_map = [&](CUtensorMap* map, __half* v) {
    return pair::map_3d(map, v, 2, n, m, z.ld, batch, x_stride, 64, 32);
  };

  for (int step = 0; step < a->steps; ++step) {
    __half* now = hi[step & 1];
    __half* next = hi[(step + 1) & 1];
    // G = X X^T (wide: X is K-major) or X^T X (tall: X read MN-major)
    q.gram = 1;
    q.mn = !wide;
    q.num_kb = tiles_of(longer, pair::kBK);
    q.alpha = 0.f;
    q.beta = 1.0f / kScale;
    q.shift = 0.f;
    rc = pair::map_operand(wide ? &q.k_major : &q.mn_major, now, !wide, side, longer, z.ld, batch,
                           x_stride);
    if (rc == 0) rc = gram_map(&q.out, gram);
    if (rc != 0) return 1000 + rc;
    rc = pair::launch_pair<SymOp>(q, stream);
    if (rc != 0) return rc;
    // P = b G + c G G (+ a I)
    const bool folded = step + 2 >= a->steps;
    const float k = folded ? a->a : 0.f;
    q.gram = 0;
    q.num_kb = tiles_of(side, pair::kBK);
    q.alpha = a->b;
    q.beta = a->c / kScale;
    q.shift = k * kScale;
    q.aux = q.out;
    rc = symmetric(&q.k_major, &q.mn_major, gram);
    if (rc == 0) rc = gram_map(&q.out, poly);
    if (rc != 0) return 1000 + rc;
    rc = pair::launch_pair<SymOp>(q, stream);
    if (rc != 0) return rc;
    // X <- a X + P X (wide) or a X + X P (tall; P is symmetric)
    const bool last = step + 1 == a->steps;
    x.last = !last ? 0 : (out_tma ? 1 : 2);
    const float unscale = last ? 1.0f / kScale : 1.0f;
    x.folded = folded;
    x.keep_lo = step + 3 < a->steps;  // the next step is not folded either
    x.alpha = (a->a - k) * unscale;
    x.beta = unscale / kScale;
    rc = symmetric(&x.p_k, &x.p_mn, poly);
    if (rc == 0)
      rc = wide ? pair::map_operand(&x.x, now, true, n, m, z.ld, batch, x_stride)
                : pair::map_operand(&x.x, now, false, m, n, z.ld, batch, x_stride);
    if (rc == 0) rc = x_map(&x.hi, now);
    if (rc == 0) rc = x_map(&x.lo, lo);
    if (rc == 0) rc = x_map(&x.hi_out, next);
    if (rc == 0 && x.last == 1)
      rc = pair::map_3d(&x.out, a->out, 2, n, m, n, batch, static_cast<uint64_t>(m) * n, 64, 32);
    if (rc != 0) return 1000 + rc;
    rc = pair::launch_pair<ApplyOp>(x, stream);
    if (rc != 0) return rc;
  }
  return 0;
}
