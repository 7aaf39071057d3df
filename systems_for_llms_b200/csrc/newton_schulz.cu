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
// 1.7e-3 (in a simulation, hi alone throughout: up to 2e-2; a X apart in every step: up to 2.7e-3).
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

// kScale / (norm + eps) as a power of two and the rest, neither of which leaves the fp32 range: the
// norm of fp32 entries spans 2^-149 to 2^140.
__device__ __forceinline__ float2 inverse_norm(double square_sum, float eps) {
  const double inv = kScale / (sqrt(square_sum) + static_cast<double>(eps));
  const double power = inv > 1e30 ? 0x1p100 : (inv < 1e-30 ? 0x1p-40 : 1.0);
  return make_float2(static_cast<float>(power), static_cast<float>(inv / power));
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
  __shared__ float2 inv_sh;
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
    if (threadIdx.x == 0) inv_sh = inverse_norm(sum, eps);
  }
  __syncthreads();
  const float2 inv = inv_sh;
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
        const float x = v[d][j] * inv.x * inv.y;
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
// Two staging tiles take turns: chunk 0 may be written once everything has left them (the tile
// before may have had no chunk 1), chunk 1 once all but chunk 0's store has.
__device__ __forceinline__ void reuse(const EpiContext& c, int chunk) {
  if (c.lane == 0) {
    if (chunk == 0) tma_store_wait_read<0>();
    else tma_store_wait_read<1>();
  }
  __syncwarp();
}

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
          if (h == 0) reuse(c, ch);
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
// What the epilogue of the product needs to know.
struct ApplyView {
  const CUtensorMap *hi, *lo;       // X as it was: 64-column lines of 32 rows; lo is rewritten in place
  const CUtensorMap *hi_out, *out;  // the next hi, or the bf16 result
  int m, n;
  int folded;                       // 1: P holds a X as well; hi + lo of X are not read
  int keep_lo;                      // 1: write lo of the next X
  int last;                         // 0: next X, 1: result through TMA, 2: result element by element
  float alpha, beta;
  __nv_bfloat16* result;            // [batch, m, n]
};

__device__ __forceinline__ void apply_load(const ApplyView& p, const Tile& t, EpiContext& c,
                                           int begin) {
  if (c.lane == 0) {
    tma_store_wait_read<0>();
    mbar_expect_tx(c.aux_bar, 2 * pair::kEpiTileBytes);
    tma_load_3d(c.smem, p.hi, c.aux_bar, begin, c.row0, t.z);
    tma_load_3d(c.smem + pair::kEpiTileBytes, p.lo, c.aux_bar, begin, c.row0, t.z);
  }
}
__device__ __forceinline__ void apply_begin(const ApplyView& p, const Tile& t, EpiContext& c) {
  const int col0 = t.n0 + c.part * 128;
  if (!p.folded && c.row0 < p.m && col0 < p.n) apply_load(p, t, c, col0);
}
__device__ __forceinline__ void apply_epilogue(const ApplyView& p, const Tile& t, EpiContext& c) {
  const int col0 = t.n0 + c.part * 128;
  if (c.row0 >= p.m) return;  // warp-uniform
#pragma unroll 1
  for (int ch = 0; ch < 2; ++ch) {
    const int begin = col0 + ch * 64;
    if (begin >= p.n) break;  // warp-uniform
    // hi and lo of a chunk take both staging tiles; without them the chunks alternate
    uint8_t* tile = p.folded ? c.smem + ch * pair::kEpiTileBytes : c.smem;
    uint8_t* low = c.smem + pair::kEpiTileBytes;
    if (p.folded) {
      reuse(c, ch);
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
      }
    }
    if (p.last == 2) {  // rows that TMA cannot address: written by the whole warp, row after row
      __syncwarp();
      const int rows = p.m - c.row0 < 32 ? p.m - c.row0 : 32, col = begin + c.lane;
      uint16_t* dst = reinterpret_cast<uint16_t*>(p.result) +
                      (static_cast<long>(t.z) * p.m + c.row0) * p.n + col;
#pragma unroll 4
      for (int r = 0; r < rows; ++r, dst += p.n) {
        const int at = (c.lane & 7) * 2;
        if (col < p.n)
          dst[0] = *reinterpret_cast<const uint16_t*>(pair::tile_chunk(tile, r, c.lane >> 3) + at);
        if (col + 32 < p.n)
          dst[32] = *reinterpret_cast<const uint16_t*>(pair::tile_chunk(tile, r, 4 + (c.lane >> 3)) + at);
      }
      __syncwarp();
      continue;
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (c.lane == 0) {
      if (p.last == 0) {
        pair::store_3d(p.hi_out, tile, begin, c.row0, t.z);
        if (p.keep_lo) pair::store_3d(p.lo, low, begin, c.row0, t.z);
      } else {
        pair::store_3d(p.out, tile, begin, c.row0, t.z);
      }
      tma_store_commit();
    }
    if (!p.folded && ch == 0 && begin + 64 < p.n) apply_load(p, t, c, begin + 64);
  }
}

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
    int wide;                  // A = P and B = X (MN-major), else A = X and B = P
    int folded;                // 1: P holds a X as well; hi + lo of X are not read
    int keep_lo;               // 1: write lo of the next X
    int last;                  // 0: next X, 1: result through TMA, 2: result element by element
    float alpha, beta;
    __nv_bfloat16* result;     // [batch, m, n]
  };
  static __device__ __forceinline__ Tile tile(const Params& p, int w) {
    const int z = w / p.per;
    const int in = w - z * p.per;
    const int n = in / p.mt, m = in - n * p.mt;
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
  static __device__ __forceinline__ ApplyView view(const Params& p) {
    return ApplyView{&p.hi, &p.lo, &p.hi_out, &p.out, p.m, p.n, p.folded, p.keep_lo, p.last, p.alpha,
                     p.beta, p.result};
  }
  static __device__ __forceinline__ void begin(const Params& p, const Tile& t, EpiContext& c) {
    apply_begin(view(p), t, c);
  }
  static __device__ __forceinline__ void epilogue(const Params& p, const Tile& t, EpiContext& c) {
    apply_epilogue(view(p), t, c);
  }
};

// 32 of the 64 fp16 numbers of a row in an operand block (see pair::stage_16).
__device__ __forceinline__ void kept(uint8_t* block, int row, int half, float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint4 q = *reinterpret_cast<const uint4*>(pair::tile_chunk(block, row, 4 * half + j));
    const __half2* e = reinterpret_cast<const __half2*>(&q);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = __half22float2(e[k]);
      v[8 * j + 2 * k] = f.x;
      v[8 * j + 2 * k + 1] = f.y;
    }
  }
}

// ------------------------------------------- G and P of a short side in one kernel ----
// Where the shorter side is at most 256 the Gram matrix is one tile: a cluster keeps it in the
// shared memory of its two CTAs, squares it there and stores P alone.  Two dependent launches per
// step instead of three (256 x 512: 123 -> 105 us for five steps), and G never leaves the SM.
//
// Roles as in pair_kernel.  A ring stage holds 128 rows x 64 of X, both operands of the Gram
// product.  G lies as four 64-column blocks of 128 rows per CTA - a CTA's rows as A, both CTAs' as
// the 256 rows of B.  op_ready (leader's): all sixteen epilogue warps have written G.
constexpr int kPolyStages = 6;
constexpr int kPolyStageBytes = pair::kABytes;
constexpr int kPolyWarpBytes = 2 * pair::kEpiTileBytes;
constexpr int kPolySmem = 1024 + kPolyStages * kPolyStageBytes + 4 * pair::kABytes +
                          pair::kEpiWarps * kPolyWarpBytes + 512;
static_assert(kPolySmem <= 232448, "more than a CTA's shared memory");

struct PolyParams {
  CUtensorMap x;            // X as the Gram product's operand
  CUtensorMap out;          // P in 64-column lines of 32 rows
  int batch, size, wide;
  int side_kb, long_kb;     // 64-deep steps of the shorter and the longer side
  float b, c, shift;
  int* status;
};

struct __align__(8) PolyBarriers {
  uint64_t full[kPolyStages];
  uint64_t empty[kPolyStages];
  uint64_t acc_full[2];     // G, G G
  uint64_t acc_empty;       // both have been read
  uint64_t op_ready;
  uint32_t tmem_base;
  int abort;
};

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pair::kThreads, 1)
ns_poly_kernel(const __grid_constant__ PolyParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint8_t* op = smem + kPolyStages * kPolyStageBytes;  // G
  uint8_t* epi_smem = op + 4 * pair::kABytes;
  PolyBarriers* bars = reinterpret_cast<PolyBarriers*>(epi_smem + pair::kEpiWarps * kPolyWarpBytes);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = pair::cluster_rank();
  const int clusters = gridDim.x >> 1;
  const int cluster = blockIdx.x >> 1;
  volatile int* abort = &bars->abort;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPolyStages; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    mbar_init(&bars->acc_full[0], 1);
    mbar_init(&bars->acc_full[1], 1);
    mbar_init(&bars->acc_empty, 2 * pair::kEpiWarps);
    mbar_init(&bars->op_ready, 2 * pair::kEpiWarps);
    bars->abort = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&bars->tmem_base)),
                 "r"(pair::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  pair::cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  pdl_launch_dependents();
  pdl_wait();

  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    if (pair::wait_or_leave(bar, parity, abort)) return true;
    if (lane == 0) report_status(p.status, code);
    *abort = 1;
    return false;
  };

  if (warp == 0) {
    // ------------------------------------------------------ TMA producer ----
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t full0 = pair::in_leader(smem_u32(&bars->full[0]));
    const int rows0 = rank * pair::kCtaM;
    for (int z = cluster; z < p.batch && ok; z += clusters) {
      for (int kb = 0; kb < p.long_kb; ++kb) {
        ok = wait(&bars->empty[stage], phase ^ 1, kStatusTimeoutEmpty);
        if (!ok) break;
        uint8_t* at = smem + stage * kPolyStageBytes;
        const uint32_t bar = full0 + stage * static_cast<uint32_t>(sizeof(uint64_t));
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(&bars->full[stage], 2 * kPolyStageBytes);
          if (p.wide) {
            pair::load_3d(at, &p.x, bar, kb * pair::kBK, rows0, z);
          } else {
            pair::load_3d(at, &p.x, bar, rows0, kb * pair::kBK, z);
            pair::load_3d(at + pair::kBK * 128, &p.x, bar, rows0 + 64, kb * pair::kBK, z);
          }
        }
        __syncwarp();
        if (++stage == kPolyStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    for (int s = 0; s < kPolyStages; ++s) {  // as in pair_kernel
      if (!mbar_wait(&bars->empty[stage], phase ^ 1)) break;
      if (++stage == kPolyStages) {
        stage = 0;
        phase ^= 1;
      }
    }
  } else if (warp == 1) {
    // -------------------------------------------------------- MMA issuer ----
    if (rank == 0) {
      const uint64_t k0 = umma_smem_desc(smem_u32(smem), 16, 1024);
      const uint64_t mn0 = umma_smem_desc(smem_u32(smem), pair::kBK * 128, 1024);
      const uint64_t op0 = umma_smem_desc(smem_u32(op), 16, 1024);
      int stage = 0;
      uint32_t phase = 0, round = 0;
      bool ok = true;
      auto square = [&](auto mn, uint64_t at, uint32_t d, bool more) {
        constexpr bool kMn = decltype(mn)::value;
        const uint32_t idesc = pair::instruction_descriptor(true, kMn, kMn);
#pragma unroll
        for (int k = 0; k < pair::kBK / 16; ++k) {
          const uint64_t both = umma_desc_advance(at, k * (kMn ? 2048 : 32));
          pair::mma_pair(d, both, both, idesc, more || k != 0);
        }
      };
      for (int z = cluster; z < p.batch && ok; z += clusters, ++round) {
        if (round > 0) {
          ok = wait(&bars->acc_empty, (round - 1) & 1, kStatusTimeoutTmemEmpty);
          tc_fence_after();
        }
        for (int kb = 0; kb < p.long_kb && ok; ++kb) {
          ok = wait(&bars->full[stage], phase, kStatusTimeoutFull);
          if (!ok) break;
          tc_fence_after();
          const uint64_t at = umma_desc_advance(p.wide ? k0 : mn0, stage * kPolyStageBytes);
          if (elect_one()) {
            if (p.wide) square(std::false_type(), at, tmem_base, kb != 0);
            else square(std::true_type(), at, tmem_base, kb != 0);
            pair::commit_pair(&bars->empty[stage]);
            if (kb + 1 == p.long_kb) pair::commit_pair(&bars->acc_full[0]);
          }
          __syncwarp();
          if (++stage == kPolyStages) {
            stage = 0;
            phase ^= 1;
          }
        }
        ok = ok && wait(&bars->op_ready, round & 1, kStatusTimeoutTmemEmpty);
        if (!ok) break;
        asm volatile("fence.acq_rel.cluster;" ::: "memory");
        tc_fence_after();
        if (elect_one()) {
          for (int kb = 0; kb < p.side_kb; ++kb)
            square(std::false_type(), umma_desc_advance(op0, kb * pair::kABytes),
                   tmem_base + pair::kTileN, kb != 0);
          pair::commit_pair(&bars->acc_full[1]);
        }
        __syncwarp();
      }
    }
  } else {
    // ---------------------------------------------------------- epilogue ----
    const int quarter = warp & 3, part = (warp - 2) >> 2;
    uint8_t* staging = epi_smem + (warp - 2) * kPolyWarpBytes;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t op_ready = pair::in_leader(smem_u32(&bars->op_ready));
    const int row = quarter * 32 + lane;            // of this CTA's 128 rows
    const int row0 = rank * pair::kCtaM + quarter * 32;
    const int cols = p.side_kb * pair::kBK;         // columns of G that are multiplied
    uint32_t phase = 0;
    for (int z = cluster; z < p.batch; z += clusters, phase ^= 1) {
      if (!wait(&bars->acc_full[0], phase, kStatusTimeoutTmemFull)) break;
      tc_fence_after();
#pragma unroll 1
      for (int ch = 0; ch < 4; ++ch) {
        const int col = part * 128 + ch * 32;
        if (col >= cols) break;  // warp-uniform
        float v[32];
        pair::load_acc(tmem_base + lanes + col, v);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] *= 1.0f / kScale;
        pair::stage_16(op + (col >> 6) * pair::kABytes, row, (col >> 5) & 1, v, true);
      }
      // both CTAs' shared memory is read by the products that the leader issues
      fence_proxy_async();
      tc_fence_before();
      __syncwarp();
      if (lane == 0)
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(op_ready)
                     : "memory");
      if (!wait(&bars->acc_full[1], phase, kStatusTimeoutTmemFull)) break;
      tc_fence_after();
#pragma unroll 1
      for (int ch = 0; ch < 2; ++ch) {
        const int begin = part * 128 + ch * 64;
        if (begin >= p.size || row0 >= p.size) break;  // warp-uniform
        uint8_t* tile = staging + ch * pair::kEpiTileBytes;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int col = begin + h * 32;
          float v[32], g[32];
          // the rounded G that was multiplied: b and c must see the same matrix, or its rounding
          // enters with the slope of c G G alone
          kept(op + (col >> 6) * pair::kABytes, row, h, g);
          pair::load_acc(tmem_base + pair::kTileN + lanes + col, v);
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            v[j] = fmaf(v[j], p.c / kScale, g[j] * p.b);
            if (col + j == row0 + lane) v[j] += p.shift;
          }
          if (h == 0) {
            if (lane == 0) {
              if (ch == 0) tma_store_wait_read<0>();
              else tma_store_wait_read<1>();
            }
            __syncwarp();
          }
          pair::stage_16(tile, lane, h, v, true);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          pair::store_3d(&p.out, tile, begin, row0, z);
          tma_store_commit();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) pair::arrive_leader(&bars->acc_empty);
    }
    if (lane == 0) tma_store_wait<0>();
  }

  tc_fence_before();
  __syncthreads();
  pair::cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                 "r"(pair::kTmemCols)
                 : "memory");
  }
}

// ------------------------------------------- a short-sided matrix that stays on chip ----
// A matrix of at most 128 x 384 (either way round) fits on one SM and stays there from its norm to
// its result: X as fp16 operand in shared memory, (a - k) X as fp32 in tensor memory, where the
// product P X is added to it.  Nothing is rounded but the operands.  The block of 128 rows x 64
// columns of X is at once the K-major operand of X X^T (rows are rows) and the MN-major operand of
// P X (rows are steps of the reduction): the swizzled layouts are the same bytes.  Tall matrices
// are taken transposed, X = U^T.  In the last two steps k = -(b + c), which makes P + k I vanish
// where singular values are 1.
//
// Up to eight times longer matrices are shared by a cluster, 384 columns or fewer to each CTA.
// Only the norm and G need the others: every CTA leaves its share of X X^T in shared memory, adds
// the shares of some rows in a fixed order and stores the sum into all (96 KB a step and CTA);
// polynomial and update are its own.
//
// One launch instead of twelve or more; its time is the latency of three products and three passes
// through registers per step and, in a cluster, of two barriers and the exchange.  Five steps of
// 128 x 384 take 38 us a call, where a launch per product took 114; 128 x 2000 65 us (128 with a
// launch for G and P and one for X), 96 matrices of 100 x 2000 330 us (491).
constexpr int kBlockRows = 128;
constexpr int kBlockCols = 384;          // 512 columns of tensor memory less 128 of G
constexpr int kBlockEpiWarps = 8;
constexpr int kBlockThreads = 32 * (kBlockEpiWarps + 1);
constexpr int kBlockBytes = kBlockRows * 128;  // 128 rows x 64 fp16
constexpr int kMaxCluster = 8;                 // CTAs that share a matrix
constexpr int kPartPitch = kBlockRows + 4;     // of a CTA's share of G: rows start four banks apart
constexpr int kPartBytes = kBlockRows * kPartPitch * static_cast<int>(sizeof(float));

// The same shared-memory offset in another CTA of the cluster, and accesses to it.
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 load_far(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ double load_far_double(uint32_t addr) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void store_far(uint32_t addr, uint32_t a, uint32_t b) {
  asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}

struct BlockParams {
  Stack u;
  int m, n, wide, steps;
  int cluster, share;       // CTAs per matrix, 64-column blocks of the longer side in each
  float a, b, c, eps;
  int vec_in, vec_out;      // rows may be read / written 16 bytes at a time (wide)
  __nv_bfloat16* out;
  int* status;
};

// 32 columns of the warp's rows of the result, back in the orientation of the matrix.  `block` is
// the operand block that held them, free by now.
__device__ __forceinline__ void block_store(const BlockParams& p, float (&v)[32], int z, int row0,
                                            int side, int col0, int longer, uint8_t* block, int half) {
  const int lane = threadIdx.x & 31, row = row0 + lane;
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] *= 1.0f / (kScale * kScale);
  __nv_bfloat16* out = p.out + static_cast<long>(z) * p.m * p.n;
  if (!p.wide) {  // a warp's lanes are neighbours in memory
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (row < side && col0 + j < longer)
        out[static_cast<long>(col0 + j) * p.n + row] = __float2bfloat16_rn(v[j]);
    return;
  }
  if (p.vec_out) {  // rows are whole groups of eight
    __nv_bfloat16* dst = out + static_cast<long>(row) * p.n + col0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (row < side && col0 + 8 * j < longer)
        *reinterpret_cast<uint4*>(dst + 8 * j) =
            make_uint4(pack_bf16(v[8 * j], v[8 * j + 1]), pack_bf16(v[8 * j + 2], v[8 * j + 3]),
                       pack_bf16(v[8 * j + 4], v[8 * j + 5]), pack_bf16(v[8 * j + 6], v[8 * j + 7]));
    return;
  }
  pair::stage_16(block, row, half, v, false);  // row after row, lanes along the row
  __syncwarp();
  uint16_t* dst = reinterpret_cast<uint16_t*>(out) + static_cast<long>(row0) * p.n + col0 + lane;
  const int rows = side - row0 < 32 ? side - row0 : 32;
  if (col0 + lane < longer) {
#pragma unroll 8
    for (int r = 0; r < rows; ++r, dst += p.n)
      *dst = *reinterpret_cast<const uint16_t*>(
          pair::tile_chunk(block, row0 + r, 4 * half + (lane >> 3)) + (lane & 7) * 2);
  }
  __syncwarp();
}

template <typename T, bool SHARED>
__global__ void __launch_bounds__(kBlockThreads, 1)
ns_block_kernel(const __grid_constant__ BlockParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t done_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ double sums[kBlockEpiWarps];
  __shared__ double cta_sum;
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* op = smem_raw + (((raw + 1023u) & ~1023u) - raw);  // G, then P: two blocks
  uint8_t* xs = op + 2 * kBlockBytes;                         // X: up to six blocks
  float* parts = reinterpret_cast<float*>(xs + p.share * kBlockBytes);  // this CTA's share of G
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int quarter = warp & 3, part = warp >> 2;
  const int row = quarter * 32 + lane;
  const int side = p.wide ? p.m : p.n, longer = p.wide ? p.n : p.m;
  const int cluster = SHARED ? p.cluster : 1;
  const int rank = SHARED ? static_cast<int>(pair::cluster_rank()) : 0;
  const int z = SHARED ? blockIdx.x / cluster : blockIdx.x;
  const int first = rank * p.share * 64;     // column of the longer side
  const int left = longer - first;
  const int blocks = left >= p.share * 64 ? p.share : (left + 63) >> 6;  // of X
  const int chunks = 2 * blocks;             // of 32 columns; a warp takes every other one
  const uint32_t columns = blocks <= 2 ? 256 : 512;  // of tensor memory: 128 of G, 64 per block
  const int side_blocks = (side + 63) >> 6;  // of G and P
  volatile int* abort = &abort_flag;

  if (threadIdx.x == 0) {
    mbar_init(&done_bar, 1);
    abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == kBlockEpiWarps) {
    tmem_alloc(&tmem_slot, columns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const uint32_t mine = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  const uint32_t x_acc = 128;  // columns of X in tensor memory
  pdl_launch_dependents();
  pdl_wait();

  uint32_t phase = 0;
  // Everyone waits for the products that the last warp has just issued.  A wait that runs out is
  // reported once; the block then runs to its end without waiting again.
  auto products_done = [&] {
    if (!*abort && !mbar_wait(&done_bar, phase)) {
      if (lane == 0) report_status(p.status, kStatusTimeoutTmemFull);
      *abort = 1;
    }
    phase ^= 1;
    tc_fence_after();
  };
  auto operands_written = [&] {
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  };
  auto to_tmem = [&](uint32_t at, const float (&v)[32]) {
    uint32_t q[16];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < 16; ++j) q[j] = __float_as_uint(v[16 * h + j]);
      tmem_st_32x16(at + 16 * h, q);
    }
  };
  auto held = [&](int step) { return step + 2 >= p.steps && p.b + p.c < 0.f ? -(p.b + p.c) : 0.f; };

  // ---- the matrix into tensor memory, its norm, then both forms of X
  const T* u = matrix<T>(p.u, z);
  double sum = 0.0;
  if (warp < kBlockEpiWarps) {
    for (int ch = part; ch < chunks; ch += 2) {
      float v[32];
      if (p.wide) {
        const T* src = u + static_cast<long>(row < side ? row : 0) * p.u.row + first + ch * 32;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float q[4];
          load4(src, 4 * j, row < side ? left - ch * 32 : 0, p.vec_in, q);
#pragma unroll
          for (int k = 0; k < 4; ++k) v[4 * j + k] = q[k];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const int l = first + ch * 32 + j;
          v[j] = row < side && l < longer ? wide(u[static_cast<long>(l) * p.u.row + row]) : 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) sum = fma(static_cast<double>(v[j]), static_cast<double>(v[j]), sum);
      to_tmem(mine + x_acc + ch * 32, v);
    }
    tmem_st_wait();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sums[warp] = sum;
  }
  __syncthreads();
  if constexpr (SHARED) {
    if (threadIdx.x == 0) {
      sum = 0.0;
#pragma unroll
      for (int k = 0; k < kBlockEpiWarps; ++k) sum += sums[k];
      cta_sum = sum;
    }
    __syncwarp();
    pair::cluster_sync();
  }
  if (warp < kBlockEpiWarps) {
    sum = 0.0;
    if constexpr (SHARED) {
      for (int k = 0; k < cluster; ++k) sum += load_far_double(in_cta(smem_u32(&cta_sum), k));
    } else {
#pragma unroll
      for (int k = 0; k < kBlockEpiWarps; ++k) sum += sums[k];
    }
    const float2 inv = inverse_norm(sum, p.eps);
    const float ahead = (p.a - held(0)) * kScale;
    for (int ch = part; ch < chunks; ch += 2) {
      float v[32];
      pair::load_acc(mine + x_acc + ch * 32, v);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = v[j] * inv.x * inv.y;
      pair::stage_16(xs + (ch >> 1) * kBlockBytes, row, ch & 1, v, true);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] *= ahead;
      to_tmem(mine + x_acc + ch * 32, v);
    }
    tmem_st_wait();
  }
  operands_written();

  const uint64_t op_k = umma_smem_desc(smem_u32(op), 16, 1024);
  const uint64_t x_k = umma_smem_desc(smem_u32(xs), 16, 1024);
  const uint64_t x_mn = umma_smem_desc(smem_u32(xs), kBlockBytes, 1024);
  auto idesc = [](int cols, bool b_mn) {
    return umma_idesc_bf16(kBlockRows, cols, false, b_mn) & ~((1u << 7) | (1u << 10));  // fp16
  };
  auto square = [&](uint64_t operand, int count) {  // G = X X^T or G G, into columns 0 .. 127
    if (warp != kBlockEpiWarps) return;
    if (elect_one()) {
      for (int kb = 0; kb < count; ++kb) {
        const uint64_t at = umma_desc_advance(operand, kb * kBlockBytes);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_bf16_ss(tmem, umma_desc_advance(at, k * 32), umma_desc_advance(at, k * 32),
                       idesc(kBlockRows, false), (kb | k) != 0);
      }
      umma_commit(&done_bar);
    }
    __syncwarp();
  };

  for (int step = 0; step < p.steps; ++step) {
    const bool last = step + 1 == p.steps;
    const float k = held(step);
    square(x_k, blocks);
    products_done();
    if (warp < kBlockEpiWarps && part < side_blocks) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[32];
        pair::load_acc(mine + part * 64 + h * 32, v);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] *= 1.0f / kScale;
        if constexpr (SHARED) {
          float4* dst = reinterpret_cast<float4*>(parts + row * kPartPitch + part * 64 + h * 32);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            dst[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        } else {
          pair::stage_16(op + part * kBlockBytes, row, h, v, true);
        }
      }
    }
    if constexpr (SHARED) {
      // Every CTA adds the shares of its rows of G, in order, and leaves the sum with all.  The
      // others' products read G only after the second barrier, and nobody rewrites a share before it.
      pair::cluster_sync();
      const int col = 4 * lane;
      if (warp < kBlockEpiWarps && col < side_blocks * 64) {
        const uint32_t from = smem_u32(parts + col);
#pragma unroll 2
        for (int r = rank + cluster * warp; r < kBlockRows; r += cluster * kBlockEpiWarps) {
          float4 g = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int k = 0; k < kMaxCluster; ++k) {
            if (k >= cluster) break;
            const float4 q = load_far(in_cta(from + r * kPartPitch * static_cast<int>(sizeof(float)), k));
            g = make_float4(g.x + q.x, g.y + q.y, g.z + q.z, g.w + q.w);
          }
          const uint32_t lo = pair::pack_16(true, g.x, g.y), hi = pair::pack_16(true, g.z, g.w);
          const uint32_t to = smem_u32(pair::tile_chunk(op + (col >> 6) * kBlockBytes, r, (col & 63) >> 3)) +
                              (col & 7) * 2;
          for (int k = 0; k < cluster; ++k) store_far(in_cta(to, k), lo, hi);
        }
        fence_proxy_async();
      }
      __syncwarp();
      pair::cluster_sync();
    }
    operands_written();
    square(op_k, side_blocks);
    products_done();
    if (warp < kBlockEpiWarps && part < side_blocks) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[32], g[32];
        kept(op + part * kBlockBytes, row, h, g);
        pair::load_acc(mine + part * 64 + h * 32, v);
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          v[j] = fmaf(v[j], p.c / kScale, g[j] * p.b);
          if (part * 64 + h * 32 + j == row) v[j] += k * kScale;
        }
        pair::stage_16(op + part * kBlockBytes, row, h, v, true);
      }
    }
    operands_written();
    if (warp == kBlockEpiWarps) {
      if (elect_one()) {  // (a - k) X + P X, 256 columns at a time
        for (int n0 = 0; n0 < blocks * 64; n0 += 256) {
          const int cols = blocks * 64 - n0 < 256 ? blocks * 64 - n0 : 256;
          const uint64_t b0 = umma_desc_advance(x_mn, (n0 >> 6) * kBlockBytes);
          for (int kk = 0; kk < side_blocks * 4; ++kk)
            umma_bf16_ss(tmem + x_acc + n0,
                         umma_desc_advance(op_k, (kk >> 2) * kBlockBytes + (kk & 3) * 32),
                         umma_desc_advance(b0, kk * 2048), idesc(cols, true), 1);
        }
        umma_commit(&done_bar);
      }
      __syncwarp();
    }
    products_done();
    if (warp < kBlockEpiWarps) {
      const float ahead = last ? 0.f : p.a - held(step + 1);
      for (int ch = part; ch < chunks; ch += 2) {
        float v[32];
        pair::load_acc(mine + x_acc + ch * 32, v);
        if (!last) {
          float h[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            h[j] = v[j] * (1.0f / kScale);
            v[j] *= ahead;
          }
          pair::stage_16(xs + (ch >> 1) * kBlockBytes, row, ch & 1, h, true);
          to_tmem(mine + x_acc + ch * 32, v);
        } else {
          block_store(p, v, z, quarter * 32, side, first + ch * 32, longer,
                      xs + (ch >> 1) * kBlockBytes, ch & 1);
        }
        __syncwarp();  // tensor memory is read by whole warps
      }
      if (!last) tmem_st_wait();
    }
    if (!last) operands_written();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kBlockEpiWarps) {
    tc_fence_after();
    tmem_dealloc(tmem, columns);
  }
}

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

// Every row starts where four elements can be read at once.
template <typename T>
int rows_of_four(const Stack& s) {
  const long bytes = 4 * sizeof(T);
  return (reinterpret_cast<uintptr_t>(s.base) % bytes) == 0 && s.row % 4 == 0 && s.stride0 % 4 == 0 &&
         s.stride1 % 4 == 0;
}

template <typename T>
int normalise(const Stack& s, int batch, int m, int n, int ld, float eps, double* partial,
              __half* hi, __half* lo, cudaStream_t stream) {
  const int vec = rows_of_four<T>(s);
  const long quads = static_cast<long>(m) * (ld / 4);
  const long want = (quads + 4L * kNormThreads - 1) / (4L * kNormThreads);
  const int chunks = static_cast<int>(want < 1 ? 1 : (want > kChunks ? kChunks : want));
  int rc = launch_pdl(ns_norm_kernel<T>, dim3(chunks, batch), dim3(kNormThreads), 0, stream, s, m, n,
                      vec, partial);
  if (rc != 0) return rc;
  return launch_pdl(ns_split_kernel<T>, dim3(chunks, batch), dim3(kNormThreads), 0, stream, s, m, n,
                    ld, vec, static_cast<const double*>(partial), eps, hi, lo);
}

// A matrix stays on chip up to 128 x 384 for each of at most eight CTAs.  It takes as few as hold
// it, whatever the stack: the order of G's sum, and with it the last bits of the result, then do not
// depend on its neighbours.  (More CTAs are sooner done with one matrix and later with many: 128 x
// 1000 in three takes 60 us and 32 of them 63, in eight 48 and 144.)
bool fits_blocks(int m, int n) {
  const int side = m < n ? m : n, longer = m < n ? n : m;
  return side <= kBlockRows && longer <= kMaxCluster * kBlockCols;
}

template <typename T>
int launch_block(const SflNewtonSchulz& a, const Stack& s, cudaStream_t stream) {
  const int blocks = tiles_of(a.m < a.n ? a.n : a.m, 64);
  const int cluster = tiles_of(blocks, kBlockCols / 64);
  BlockParams p{};
  p.u = s;
  p.m = a.m;
  p.n = a.n;
  p.wide = a.m <= a.n;
  p.steps = a.steps;
  p.a = a.a;
  p.b = a.b;
  p.c = a.c;
  p.eps = a.eps;
  p.vec_in = rows_of_four<T>(s);
  p.vec_out = a.n % 8 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
  p.out = static_cast<__nv_bfloat16*>(a.out);
  p.status = a.status;
  p.cluster = cluster;  // every CTA has a block: share (cluster - 1) < blocks
  p.share = tiles_of(blocks, cluster);
  auto go = [&](auto kernel, int extra) -> int {
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             1024 + (2 + kBlockCols / 64) * kBlockBytes + extra);
    if (e != cudaSuccess) return static_cast<int>(e);
    return launch_pdl_clusters(extra > 0 ? cluster : 0, kernel, dim3(a.batch * cluster), dim3(kBlockThreads),
                               1024 + (2 + p.share) * kBlockBytes + extra, stream, p);
  };
  return cluster == 1 ? go(ns_block_kernel<T, false>, 0) : go(ns_block_kernel<T, true>, kPartBytes);
}

int launch_poly(const PolyParams& p, cudaStream_t stream) {
  int device = 0;
  const int pairs = pair::sm_count_here(&device) / 2;
  if (pairs < 1) return -1;
  static bool configured[64] = {};
  if (device >= 64 || !configured[device]) {
    const cudaError_t e = cudaFuncSetAttribute(
        ns_poly_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPolySmem);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (device < 64) configured[device] = true;
  }
  const int clusters = p.batch < pairs ? p.batch : pairs;
  return launch_pdl(ns_poly_kernel, dim3(2 * clusters), dim3(pair::kThreads), kPolySmem, stream, p);
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

extern "C" int sfl_newton_schulz_kernels(int m, int n, int steps) {
  using namespace sfl;
  if (fits_blocks(m, n)) return 1;
  return 2 + steps * ((m < n ? m : n) <= pair::kTileN ? 2 : 3);
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

  const Stack s{a->update, a->stride0, a->stride1, a->row, a->inner};
  if (fits_blocks(m, n)) {
    if (a->dtype == 0) return launch_block<__nv_bfloat16>(*a, s, stream);
    if (a->dtype == 1) return launch_block<__half>(*a, s, stream);
    return launch_block<float>(*a, s, stream);
  }

  uint8_t* at = static_cast<uint8_t*>(a->work);
  __half* hi[2] = {reinterpret_cast<__half*>(at), reinterpret_cast<__half*>(at + z.x_bytes)};
  __half* lo = reinterpret_cast<__half*>(at + 2 * z.x_bytes);
  __half* gram = reinterpret_cast<__half*>(at + 3 * z.x_bytes);
  __half* poly = reinterpret_cast<__half*>(at + 3 * z.x_bytes + z.gram_bytes);
  double* norms = reinterpret_cast<double*>(at + 3 * z.x_bytes + 2 * z.gram_bytes);

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

  // Encoding a map takes the host as long as a product takes a small matrix: each is made once.
  struct {
    CUtensorMap gram_x[2], apply_x[2], x[2], lo, gram, gram_k, gram_mn, poly, poly_k, poly_mn, out;
  } maps;
  const bool fused_poly = side <= pair::kTileN;
  rc = 0;
  for (int i = 0; i < 2 && rc == 0; ++i) {
    rc = pair::map_operand(&maps.gram_x[i], hi[i], !wide, side, longer, z.ld, batch, x_stride);
    if (rc == 0)
      rc = wide ? pair::map_operand(&maps.apply_x[i], hi[i], true, n, m, z.ld, batch, x_stride)
                : pair::map_operand(&maps.apply_x[i], hi[i], false, m, n, z.ld, batch, x_stride);
    if (rc == 0) rc = x_map(&maps.x[i], hi[i]);
  }
  if (rc == 0) rc = x_map(&maps.lo, lo);
  if (rc == 0 && !fused_poly) rc = gram_map(&maps.gram, gram);
  if (rc == 0 && !fused_poly) rc = symmetric(&maps.gram_k, &maps.gram_mn, gram);
  if (rc == 0) rc = gram_map(&maps.poly, poly);
  if (rc == 0) rc = symmetric(&maps.poly_k, &maps.poly_mn, poly);
  if (rc == 0 && out_tma)
    rc = pair::map_3d(&maps.out, a->out, 2, n, m, n, batch, static_cast<uint64_t>(m) * n, 64, 32);
  if (rc != 0) return 1000 + rc;
  x.lo = maps.lo;
  x.p_k = maps.poly_k;
  x.p_mn = maps.poly_mn;
  if (out_tma) x.out = maps.out;

  for (int step = 0; step < a->steps; ++step) {
    const int now = step & 1;
    const bool folded = step + 2 >= a->steps;
    const float k = folded ? a->a : 0.f;
    if (fused_poly) {
      PolyParams g{};
      g.x = maps.gram_x[now];
      g.out = maps.poly;
      g.batch = batch;
      g.size = side;
      g.wide = wide;
      g.side_kb = tiles_of(side, pair::kBK);
      g.long_kb = tiles_of(longer, pair::kBK);
      g.b = a->b;
      g.c = a->c;
      g.shift = k * kScale;
      g.status = a->status;
      rc = launch_poly(g, stream);
      if (rc != 0) return rc;
    } else {
      // G = X X^T (wide: X is K-major) or X^T X (tall: X read MN-major)
      q.gram = 1;
      q.mn = !wide;
      q.num_kb = tiles_of(longer, pair::kBK);
      q.alpha = 0.f;
      q.beta = 1.0f / kScale;
      q.shift = 0.f;
      (wide ? q.k_major : q.mn_major) = maps.gram_x[now];
      q.out = maps.gram;
      rc = pair::launch_pair<SymOp>(q, stream);
      if (rc != 0) return rc;
      // P = b G + c G G (+ a I)
      q.gram = 0;
      q.num_kb = tiles_of(side, pair::kBK);
      q.alpha = a->b;
      q.beta = a->c / kScale;
      q.shift = k * kScale;
      q.k_major = maps.gram_k;
      q.mn_major = maps.gram_mn;
      q.aux = maps.gram;
      q.out = maps.poly;
      rc = pair::launch_pair<SymOp>(q, stream);
      if (rc != 0) return rc;
    }
    // X <- a X + P X (wide) or a X + X P (tall; P is symmetric)
    const bool last = step + 1 == a->steps;
    x.last = !last ? 0 : (out_tma ? 1 : 2);
    const float unscale = last ? 1.0f / kScale : 1.0f;
    x.folded = folded;
    x.keep_lo = step + 3 < a->steps;  // the next step is not folded either
    x.alpha = (a->a - k) * unscale;
    x.beta = unscale / kScale;
    x.x = maps.apply_x[now];
    x.hi = maps.x[now];
    x.hi_out = maps.x[now ^ 1];
    rc = pair::launch_pair<ApplyOp>(x, stream);
    if (rc != 0) return rc;
  }
  return 0;
}
