// Softmax cross entropy of a vocabulary projection that keeps no logits.
//
//   loss_i = log(sum_v exp(h_i . w_v)) - h_i . w_t(i)
//   dl_iv  = softmax_iv - [v = t(i)]          (zero rows where the target is ignored)
//   dh     = g dl W,   dW = g dl^T h          g = incoming gradient (over the count, for a mean)
//
// The reference materialises the logits, their fp32 copy and its softmax
// (src/llmlab/training/loss.py:4-22), and this library's other head keeps them in bf16
// (elementwise.cu).  Here the projection's accumulators go from tensor memory straight into the
// running maximum and sum of exponentials of their row: forward writes one (max, sum) pair per
// row and 128 columns.  Backward walks the vocabulary in pieces: the piece's logits are computed
// again, leave the epilogue as 16-bit dl, and two products consume them (dW of the piece, whose
// rows are then final, and the piece's share of dh).  Pieces bound the memory:
// dl of one piece is all that exists of the logits.  The price is the second projection: 8 N D V
// operations for forward and backward where keeping the logits takes 6.  Both products of a piece
// run in one launch.
//
// Measured, bf16, forward and backward: 4096 rows x 1024 x 10000 in 212 us (334 GFLOP of 8 N D V:
// 1.58 PFLOP/s), 8192 x 2048 x 131072 in 12.4 ms (17.6 TFLOP: 1.42 PFLOP/s, at the power limit).
// The operand traffic between L2 and the SMs bounds the small case's products, power the large one.
//
// Logits are never rounded: statistics and losses see fp32 accumulators.  dl is rounded once to
// the operands' type, which is what the tensor cores multiply; fp16 holds dl times 2^12, so
// probabilities down to 2^-26 keep full precision and 1 becomes 4096, far below the largest fp16.
// The tensor cores add in fp32 and drop what lies below the sum's last bit: losses are off by 1.2e-7
// of their value at dim 768 and 5.6e-7 at 4096, where a product of fp32 FMAs is 4 to 7 times closer.
// All sums have a fixed order; there are no atomics.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <functional>
#include <utility>

#include "pair_gemm.cuh"
#include "sfl.h"

namespace sfl {
namespace {

using pair::EpiContext;
using pair::Tile;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kFp16Shift = 12;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Tiles of an mt x nt grid with m fastest inside bands of `band` row tiles: a band's rows stay in
// the L2 cache while the vocabulary streams past them once.
struct Grid {
  int mt, nt, band;
};
__device__ __forceinline__ void grid_tile(const Grid& g, int w, int* m, int* n) {
  const int per_band = g.band * g.nt;
  const int b = w / per_band;
  const int in = w - b * per_band;
  const int left = g.mt - b * g.band;
  const int width = left < g.band ? left : g.band;
  *n = in / width;
  *m = b * g.band + (in - *n * width);
}

// ---------------------------------------------------- row statistics (forward) ----
struct StatsOp : pair::NoMaps, pair::Plain, pair::RoundRobin {
  struct Params {
    CUtensorMap a, b;
    Grid grid;
    int total, num_kb;
    bool fp16;
    int* status;
    const int64_t* targets;
    float2* part;      // [2 * nt][rows]
    float* picked;     // [rows]: the target's logit
    int rows, vocab;
  };
  static constexpr int kForms = pair::kFormKK;
  static __device__ __forceinline__ const CUtensorMap* map_a_k(const Params& p, const Tile&) {
    return &p.a;
  }
  static __device__ __forceinline__ const CUtensorMap* map_b_k(const Params& p, const Tile&) {
    return &p.b;
  }
  static __device__ __forceinline__ Tile tile(const Params& p, int w) {
    int m, n;
    grid_tile(p.grid, w, &m, &n);
    return Tile{m * pair::kTileM, n * pair::kTileN, 0, p.num_kb, 0, 0, 0, 0, false};
  }
  static __device__ __forceinline__ void epilogue(const Params& p, const Tile& t, EpiContext& c) {
    const int row = c.row0 + c.lane;
    const int col0 = t.n0 + c.part * 128;
    int64_t target = row < p.rows ? p.targets[row] : -1;
    if (target < col0 || target >= col0 + 128 || target >= p.vocab) target = -1;
    const int at = target < 0 ? -1 : static_cast<int>(target) - col0;  // column of this warp's 128
    float mx = -INFINITY, sum = 0.f, mine = 0.f;
#pragma unroll 1
    for (int ch = 0; ch < 2; ++ch) {
      const int begin = col0 + ch * 64;
      if (begin >= p.vocab) break;  // warp-uniform
      float v[64];
      {
        uint32_t r0[32], r1[32];
        tmem_ld_32x32(c.acc + c.part * 128 + ch * 64, r0);
        tmem_ld_32x32(c.acc + c.part * 128 + ch * 64 + 32, r1);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          v[j] = __uint_as_float(r0[j]);
          v[32 + j] = __uint_as_float(r1[j]);
        }
      }
      if (begin + 64 > p.vocab) {
#pragma unroll
        for (int j = 0; j < 64; ++j)
          if (begin + j >= p.vocab) v[j] = -INFINITY;
      }
      const int in = at - ch * 64;
      if (__any_sync(0xffffffffu, in >= 0 && in < 64)) {
#pragma unroll
        for (int j = 0; j < 64; ++j)
          if (in == j) mine = v[j];
      }
      float m[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
      for (int j = 4; j < 64; ++j) m[j & 3] = fmaxf(m[j & 3], v[j]);
      const float next = fmaxf(mx, fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
      const float base = next == -INFINITY ? 0.f : next * kLog2e;  // -inf - -inf is NaN
      float s[4] = {sum * exp2_fast(fmaf(mx, kLog2e, -base)), 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 64; ++j) s[j & 3] += exp2_fast(fmaf(v[j], kLog2e, -base));
      sum = (s[0] + s[1]) + (s[2] + s[3]);
      mx = next;
    }
    if (row < p.rows) {
      const long strip = 2L * (t.n0 / pair::kTileN) + c.part;
      p.part[strip * p.rows + row] = make_float2(mx, sum);
      if (at >= 0) p.picked[row] = mine;
    }
  }
};

// Joins a row's strips.  A block has eight rows (whole sectors of a strip) and 32 groups of
// threads that share the strips and meet in shuffles and shared memory; a few hundred rows thus
// occupy more than a few SMs.  173 rows x 394 strips: 5.7 us (10.9 with 32 rows and eight groups),
// 8192 x 1024: 24 us (50).
constexpr int kJoinWarps = 8;
constexpr int kJoinRows = 8;
constexpr int kJoinGroups = 32 * kJoinWarps / kJoinRows;
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float next = fmaxf(m, m2);
  const float base = next == -INFINITY ? 0.f : next;
  s = s * exp2_fast((m - base) * kLog2e) + s2 * exp2_fast((m2 - base) * kLog2e);
  m = next;
}

__global__ void __launch_bounds__(32 * kJoinWarps)
ce_join_kernel(const float2* __restrict__ part, int strips, const float* __restrict__ picked,
               const int64_t* __restrict__ targets, int64_t ignore, int rows, int vocab,
               float shift, float* __restrict__ row_loss, float* __restrict__ lse2) {
  __shared__ float2 sh[kJoinWarps][kJoinRows];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int mine = threadIdx.x % kJoinRows;
  const int row = blockIdx.x * kJoinRows + mine;
  float m = -INFINITY, s = 0.f;
  if (row < rows) {
#pragma unroll 4
    for (int k = threadIdx.x / kJoinRows; k < strips; k += kJoinGroups) {
      const float2 q = part[static_cast<long>(k) * rows + row];
      join(m, s, q.x, q.y);
    }
  }
#pragma unroll
  for (int o = kJoinRows; o < 32; o <<= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    join(m, s, m2, s2);
  }
  if (lane < kJoinRows) sh[warp][mine] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x >= kJoinRows || row >= rows) return;
#pragma unroll
  for (int k = 1; k < kJoinWarps; ++k) join(m, s, sh[k][mine].x, sh[k][mine].y);
  const int64_t t = targets[row];
  const float lse = m + logf(s);
  float loss, out;
  if (t == ignore) {
    loss = 0.f;
    out = INFINITY;  // every probability of the row becomes zero
  } else if (t < 0 || t >= vocab) {
    loss = out = NAN;  // a target that is no entry of the vocabulary spoils the result visibly
  } else {
    loss = lse - picked[row];
    out = fmaf(lse, kLog2e, -shift);
  }
  row_loss[row] = loss;
  lse2[row] = out;
}

// totals = {sum of the rows' losses, rows that count}; out = their quotient or the sum.
__global__ void __launch_bounds__(1024)
ce_total_kernel(const float* __restrict__ row_loss, const int64_t* __restrict__ targets,
                int64_t ignore, int rows, int mean, float* __restrict__ totals,
                float* __restrict__ out) {
  __shared__ double sums[32];
  __shared__ int counts[32];
  pdl_launch_dependents();
  pdl_wait();
  double sum = 0.0;
  int count = 0;
  for (int i = threadIdx.x; i < rows; i += blockDim.x) {
    sum += row_loss[i];
    count += targets[i] != ignore;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    count += __shfl_xor_sync(0xffffffffu, count, o);
  }
  if ((threadIdx.x & 31) == 0) {
    sums[threadIdx.x >> 5] = sum;
    counts[threadIdx.x >> 5] = count;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    sum = sums[threadIdx.x];
    count = counts[threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      count += __shfl_xor_sync(0xffffffffu, count, o);
    }
    if (threadIdx.x == 0) {
      totals[0] = static_cast<float>(sum);
      totals[1] = static_cast<float>(count);
      out[0] = static_cast<float>(mean ? sum / count : sum);  // no counted row: 0 / 0
    }
  }
}

// --------------------------------------------- dl of a piece of the vocabulary ----
struct DlogitsOp : pair::NoMaps, pair::Plain, pair::RoundRobin {
  struct Params {
    CUtensorMap a, b, out;
    Grid grid;
    int total, num_kb;
    bool fp16;
    int* status;
    const int64_t* targets;
    const float* lse2;   // log-sum-exp in powers of two, less the shift
    float one;           // 1, or 2^12 for fp16
    int rows, vocab_begin, width;
  };
  static constexpr int kForms = pair::kFormKK;
  static __device__ __forceinline__ const CUtensorMap* map_a_k(const Params& p, const Tile&) {
    return &p.a;
  }
  static __device__ __forceinline__ const CUtensorMap* map_b_k(const Params& p, const Tile&) {
    return &p.b;
  }
  static __device__ __forceinline__ Tile tile(const Params& p, int w) {
    int m, n;
    grid_tile(p.grid, w, &m, &n);
    return Tile{m * pair::kTileM, n * pair::kTileN, 0, p.num_kb, 0, 0, 0, 0, false};
  }
  static __device__ __forceinline__ void epilogue(const Params& p, const Tile& t, EpiContext& c) {
    const int row = c.row0 + c.lane;
    const int col0 = t.n0 + c.part * 128;
    float lse2 = INFINITY;
    int at = -1;
    if (row < p.rows) {
      lse2 = p.lse2[row];
      const int64_t target = p.targets[row] - p.vocab_begin;
      if (target >= col0 && target < col0 + 128) at = static_cast<int>(target) - col0;
    }
    if (lse2 == INFINITY) at = -1;  // ignored
#pragma unroll 1
    for (int ch = 0; ch < 2; ++ch) {
      const int begin = col0 + ch * 64;
      if (begin >= p.width || c.row0 >= p.rows) break;  // warp-uniform
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[32];
        pair::load_acc(c.acc + c.part * 128 + ch * 64 + h * 32, v);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = exp2_fast(fmaf(v[j], kLog2e, -lse2));
        const int in = at - ch * 64 - h * 32;
        if (__any_sync(0xffffffffu, in >= 0 && in < 32)) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (in == j) v[j] -= p.one;
        }
        if (h == 0) pair::stage_reuse(c.lane);
        pair::stage_16(c.smem, c.lane, h, v, p.fp16);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (c.lane == 0) {
        pair::store_3d(&p.out, c.smem, begin, c.row0, 0);
        tma_store_commit();
      }
    }
  }
};

// --------------------------------------------------- products that consume dl ----
enum OutKind : int { kOut16 = 0, kOutF32 = 1, kOutF32Add = 2, kOutNone = 3 };

struct GradScale {
  const float* grad;     // incoming gradient, a device scalar (NULL: 1)
  const float* totals;   // {sum, count}: divide by the count (NULL: do not)
  float factor;
};
__device__ __forceinline__ float grad_scale(const GradScale& g) {
  float s = g.factor;
  if (g.grad != nullptr) s *= g.grad[0];
  if (g.totals != nullptr) {
    const float count = g.totals[1];
    s = count > 0.f ? s / count : 0.f;
  }
  return s;
}

// Both products of a piece in one launch: dW = dl^T h (A = dl read MN-major) and dh = dl W, whose
// reduction runs over the piece and may be split into parts that each leave their own fp32 sum.
// One product after the other leaves the pairs idle at the end of each (dh of 4096 x 1024 has 64
// tiles for 74 pairs); dealt together, the longest tiles first, only the end of both is ragged
// (4096 x 1024 x 10000: 132 -> 105 us).  begin[c] .. begin[c + 1] are the tiles of cluster c.
constexpr int kMaxClusters = 96;
enum Product : int { kDw = 0, kDh = 1 };

struct GradOp : pair::NoMaps, pair::Plain {
  struct Params {
    CUtensorMap dl_mn, dl_k, h, w, dw, dh;
    int total, dh_tiles;         // dh's tiles are the first of each cluster's range
    bool fp16;
    int* status;
    GradScale scale;             // of dw, and of dh when it is final
    int dw_mt, dh_mt, dh_nt;
    int dw_kb, dh_kb, dh_part_kb;  // steps of the two reductions, and of a part of dh's
    int rows, width, dim;
    int dw_kind, dh_kind;
    int dh_begin[kMaxClusters + 1], dw_begin[kMaxClusters + 1];
  };
  // A tile's number: dh tiles come first, then dw tiles.
  static __device__ __forceinline__ int first(const Params& p, int c) {
    if (p.dh_begin[c] < p.dh_begin[c + 1]) return p.dh_begin[c];
    return p.dw_begin[c] < p.dw_begin[c + 1] ? p.dh_tiles + p.dw_begin[c] : p.total;
  }
  static __device__ __forceinline__ int next(const Params& p, int w, int c, int) {
    if (w < p.dh_tiles) {
      if (w + 1 < p.dh_begin[c + 1]) return w + 1;
      return p.dw_begin[c] < p.dw_begin[c + 1] ? p.dh_tiles + p.dw_begin[c] : p.total;
    }
    return w + 1 < p.dh_tiles + p.dw_begin[c + 1] ? w + 1 : p.total;
  }
  static __device__ __forceinline__ Tile tile(const Params& p, int w) {
    if (w >= p.dh_tiles) {
      w -= p.dh_tiles;
      return Tile{w % p.dw_mt * pair::kTileM, w / p.dw_mt * pair::kTileN, 0, p.dw_kb, 0, kDw,
                  p.dw_kb, p.dw_kb, false};
    }
    const int per_part = p.dh_mt * p.dh_nt;
    const int part = w / per_part;
    w -= part * per_part;
    const int kb0 = part * p.dh_part_kb;
    const int left = p.dh_kb - kb0;
    return Tile{w % p.dh_mt * pair::kTileM, w / p.dh_mt * pair::kTileN, 0,
                left < p.dh_part_kb ? left : p.dh_part_kb, kb0, kDh + 2 * part, 0, p.dh_part_kb,
                false};
  }
  static constexpr int kForms = pair::kFormMM | pair::kFormKM;
  static __device__ __forceinline__ const CUtensorMap* map_a_mn(const Params& p, const Tile&) {
    return &p.dl_mn;
  }
  static __device__ __forceinline__ const CUtensorMap* map_a_k(const Params& p, const Tile&) {
    return &p.dl_k;
  }
  static __device__ __forceinline__ const CUtensorMap* map_b_mn(const Params& p, const Tile& t) {
    return t.kind == kDw ? &p.h : &p.w;
  }
  static __device__ __forceinline__ void epilogue(const Params& p, const Tile& t, EpiContext& c) {
    const bool dw = t.kind == kDw;
    const int rows = dw ? p.width : p.rows, part = t.kind >> 1;
    if (c.row0 >= rows) return;  // warp-uniform
    const int kind = dw ? p.dw_kind : p.dh_kind;
    const CUtensorMap* out = dw ? &p.dw : &p.dh;
    const float scale = dw || kind == kOut16 ? grad_scale(p.scale) : 1.0f;
    const int col0 = t.n0 + c.part * 128;
#pragma unroll 1
    for (int ch = 0; ch < 4; ++ch) {
      const int begin = col0 + ch * 32;
      if (begin >= p.dim) break;  // warp-uniform
      float v[32];
      pair::load_acc(c.acc + c.part * 128 + ch * 32, v);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] *= scale;
      if (kind == kOut16) {
        // two 32-column steps share a 64-column line
        if ((ch & 1) == 0) pair::stage_reuse(c.lane);
        pair::stage_16(c.smem, c.lane, ch & 1, v, p.fp16);
        if ((ch & 1) == 0 && begin + 32 < p.dim) continue;
        fence_proxy_async_smem();
        __syncwarp();
        if (c.lane == 0) {
          pair::store_3d(out, c.smem, begin & ~63, c.row0, part);
          tma_store_commit();
        }
      } else {
        pair::stage_reuse(c.lane);
        pair::stage_32(c.smem, c.lane, v);
        fence_proxy_async_smem();
        __syncwarp();
        if (c.lane == 0) {
          if (kind == kOutF32Add) pair::reduce_add_3d(out, c.smem, begin, c.row0, part);
          else pair::store_3d(out, c.smem, begin, c.row0, part);
          tma_store_commit();
        }
      }
    }
  }
};

// dh in the operands' type from its fp32 parts [parts][rows][dim], added in order.
__global__ void __launch_bounds__(256)
ce_dh_kernel(const float* __restrict__ sums, int parts, long vecs, int vecs_per_row,
             void* __restrict__ out, long ld_out, GradScale g, int fp16) {
  pdl_launch_dependents();
  pdl_wait();
  const float scale = grad_scale(g);
  for (long i = blockIdx.x * static_cast<long>(blockDim.x) + threadIdx.x; i < vecs;
       i += static_cast<long>(gridDim.x) * blockDim.x) {
    float4 a = make_float4(0, 0, 0, 0), b = a;
    for (int k = 0; k < parts; ++k) {
      const float4* src = reinterpret_cast<const float4*>(sums) + 2 * (k * vecs + i);
      const float4 c = src[0], d = src[1];
      a.x += c.x; a.y += c.y; a.z += c.z; a.w += c.w;
      b.x += d.x; b.y += d.y; b.z += d.z; b.w += d.w;
    }
    const long row = i / vecs_per_row;
    const long col = (i - row * vecs_per_row) * 8;
    uint4 q;
    q.x = pair::pack_16(fp16, a.x * scale, a.y * scale);
    q.y = pair::pack_16(fp16, a.z * scale, a.w * scale);
    q.z = pair::pack_16(fp16, b.x * scale, b.y * scale);
    q.w = pair::pack_16(fp16, b.z * scale, b.w * scale);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + row * ld_out + col) = q;
  }
}

// ------------------------------------------------------------------- host ----
bool aligned16(const void* ptr, long ld, int elem) {
  return ptr != nullptr && (reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && ld > 0 &&
         (ld * elem) % 16 == 0;
}

int tiles_of(long n, int size) { return static_cast<int>((n + size - 1) / size); }

// Row tiles of a band: at most 32 MB of rows, at least four (statistics of 16384 x 4096 x 32000: 2.5
// ms, in bands of 64 MB 2.6, of four tiles 2.7, without bands 3.0).
int band_of(int mt, int dim) {
  const long rows = (32L << 20) / (2L * dim);
  const int band = static_cast<int>(rows / pair::kTileM);
  return band < 4 ? (mt < 4 ? mt : 4) : (band < mt ? band : mt);
}

// Steps of overhead that a tile adds to its reduction (filling the ring, draining the accumulator).
constexpr int kTileOverheadKb = 4;

// Parts of dh's reduction over `width` entries: as few as keep one of its tiles within the average
// load of a pair, so that few rows do not leave most pairs idle (1024 x 512 x 10000 has 8 tiles of
// 157 steps: 51 us in one part; dh and dW together take 21 us split).  Only a vocabulary walked in
// one piece is split.
int dh_parts(int rows, int dim, int width, int pairs, bool with_dw) {
  const long tiles = static_cast<long>(tiles_of(rows, pair::kTileM)) * tiles_of(dim, pair::kTileN);
  const long kb = tiles_of(width, pair::kBK);
  const long dw = !with_dw ? 0
                           : static_cast<long>(tiles_of(width, pair::kTileM)) *
                                 tiles_of(dim, pair::kTileN) *
                                 (tiles_of(rows, pair::kBK) + kTileOverheadKb);
  const long average = (dw + tiles * (kb + kTileOverheadKb)) / pairs + 1;
  long parts = (kb + average - 1) / average;
  if (parts > 16) parts = 16;
  // every part has work
  const long part_kb = (kb + parts - 1) / parts;
  return static_cast<int>((kb + part_kb - 1) / part_kb);
}

// Deals dh's tiles, then dw's, each to the cluster with the least work so far; every cluster's
// tiles of a kind are consecutive.
void deal(GradOp::Params& p, int dh_tiles, int dw_tiles, int clusters) {
  int dh_count[kMaxClusters] = {}, dw_count[kMaxClusters] = {};
  using Load = std::pair<long, int>;  // work so far, cluster
  Load heap[kMaxClusters];            // the least loaded cluster on top
  for (int c = 0; c < clusters; ++c) heap[c] = Load(0, c);
  auto give = [&](int tiles, int kb, int* count) {
    for (int k = 0; k < tiles; ++k) {
      std::pop_heap(heap, heap + clusters, std::greater<Load>());
      heap[clusters - 1].first += kb + kTileOverheadKb;
      ++count[heap[clusters - 1].second];
      std::push_heap(heap, heap + clusters, std::greater<Load>());
    }
  };
  give(dh_tiles, p.dh_part_kb, dh_count);
  give(dw_tiles, p.dw_kb, dw_count);
  p.dh_begin[0] = p.dw_begin[0] = 0;
  for (int c = 0; c < kMaxClusters; ++c) {
    p.dh_begin[c + 1] = p.dh_begin[c] + (c < clusters ? dh_count[c] : 0);
    p.dw_begin[c + 1] = p.dw_begin[c] + (c < clusters ? dw_count[c] : 0);
  }
}

int check(const SflLinearCe* a) {
  if (a == nullptr || a->rows < 1 || a->dim < 8 || a->dim % 8 != 0 || a->vocab < 1) return -2;
  if (!aligned16(a->hidden, a->ld_hidden, 2) || !aligned16(a->weight, a->ld_weight, 2)) return -2;
  if (a->ld_hidden < a->dim || a->ld_weight < a->dim) return -2;
  if (a->targets == nullptr || a->lse2 == nullptr) return -2;
  // tile counts are 32-bit
  if (static_cast<long>(tiles_of(a->rows, pair::kTileM)) * tiles_of(a->vocab, pair::kTileN) > 0x7fffffffL)
    return -2;
  return 0;
}

}  // namespace
}  // namespace sfl

// Sizes of the argument records of rotary.cu, this file and newton_schulz.cu, for bindings to compare with.
extern "C" int sfl_operator_struct_sizes(int* sizes, int capacity) {
  const int all[] = {sizeof(SflRotaryTensor), sizeof(SflRotaryTable), sizeof(SflLinearCe),
                     sizeof(SflLinearCeGrad), sizeof(SflNewtonSchulz)};
  const int count = static_cast<int>(sizeof(all) / sizeof(all[0]));
  for (int i = 0; i < count && i < capacity; ++i) sizes[i] = all[i];
  return count;
}

extern "C" long sfl_linear_ce_part_bytes(int rows, int vocab) {
  using namespace sfl;
  if (rows < 1 || vocab < 1) return -1;
  // (max, sum) per row and 128 columns, and the target's logit
  return static_cast<long>(rows) * (2L * tiles_of(vocab, pair::kTileN) * 8 + 4);
}

extern "C" int sfl_linear_ce_fwd(const SflLinearCe* a, void* part, long part_bytes, float* row_loss,
                                 int mean, float* totals, float* loss, void* stream_) {
  using namespace sfl;
  const int bad = check(a);
  if (bad != 0) return bad;
  if (part == nullptr || row_loss == nullptr || (totals == nullptr) != (loss == nullptr) ||
      part_bytes < sfl_linear_ce_part_bytes(a->rows, a->vocab))
    return -2;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  StatsOp::Params p{};
  int rc = pair::map_operand(&p.a, a->hidden, false, a->rows, a->dim, a->ld_hidden, 1,
                             static_cast<uint64_t>(a->rows) * a->ld_hidden);
  if (rc == 0)
    rc = pair::map_operand(&p.b, a->weight, false, a->vocab, a->dim, a->ld_weight, 1,
                           static_cast<uint64_t>(a->vocab) * a->ld_weight);
  if (rc != 0) return 1000 + rc;
  p.grid.mt = tiles_of(a->rows, pair::kTileM);
  p.grid.nt = tiles_of(a->vocab, pair::kTileN);
  p.grid.band = band_of(p.grid.mt, a->dim);
  p.total = p.grid.mt * p.grid.nt;
  p.num_kb = tiles_of(a->dim, pair::kBK);
  p.fp16 = a->fp16 != 0;
  p.status = a->status;
  p.targets = a->targets;
  p.part = static_cast<float2*>(part);
  p.picked = reinterpret_cast<float*>(p.part + 2L * p.grid.nt * a->rows);
  p.rows = a->rows;
  p.vocab = a->vocab;
  rc = pair::launch_pair<StatsOp>(p, stream);
  if (rc != 0) return rc;
  rc = launch_pdl(ce_join_kernel, dim3(tiles_of(a->rows, kJoinRows)), dim3(32 * kJoinWarps), 0, stream,
                  static_cast<const float2*>(p.part), 2 * p.grid.nt,
                  static_cast<const float*>(p.picked), a->targets, a->ignore_index, a->rows,
                  a->vocab, a->fp16 ? static_cast<float>(kFp16Shift) : 0.f, row_loss, a->lse2);
  if (rc != 0 || loss == nullptr) return rc;
  return launch_pdl(ce_total_kernel, dim3(1), dim3(1024), 0, stream,
                    static_cast<const float*>(row_loss), a->targets, a->ignore_index, a->rows, mean,
                    totals, loss);
}

extern "C" long sfl_linear_ce_dh_sum_bytes(int rows, int dim, int vocab, int piece, int with_dw) {
  using namespace sfl;
  if (rows < 1 || dim < 1 || vocab < 1 || piece < 1) return -1;
  const int pairs = pair::pairs_here();
  if (pairs < 1) return -1;
  const int parts = piece < vocab ? 1 : dh_parts(rows, dim, vocab, pairs, with_dw != 0);
  return piece < vocab || parts > 1 ? 4L * parts * rows * dim : 0;
}

extern "C" int sfl_linear_ce_bwd(const SflLinearCe* a, const SflLinearCeGrad* g, void* stream_) {
  using namespace sfl;
  const int bad = check(a);
  if (bad != 0) return bad;
  if (g == nullptr || g->piece < pair::kTileN || g->piece % pair::kTileN != 0 ||
      g->dw_kind < kOut16 || g->dw_kind > kOutNone || (g->dw_kind == kOutNone) != (g->dw == nullptr))
    return -2;
  const int dw_elem = g->dw_kind == kOut16 ? 2 : 4;
  const bool with_dh = g->dh != nullptr, with_dw = g->dw != nullptr;
  if (!aligned16(g->dlogits, g->piece, 2) || (!with_dh && !with_dw) ||
      (with_dh && (!aligned16(g->dh, g->ld_dh, 2) || g->ld_dh < a->dim)) ||
      (with_dw && (!aligned16(g->dw, g->ld_dw, dw_elem) || g->ld_dw < a->dim)))
    return -2;
  const int pieces = tiles_of(a->vocab, g->piece);
  if (pieces > 1 && with_dh && g->dh_sum == nullptr) return -2;
  const int pairs = pair::pairs_here();
  if (pairs < 1 || pairs > kMaxClusters) return -1;
  const int parts = pieces > 1 || !with_dh ? 1 : dh_parts(a->rows, a->dim, a->vocab, pairs, with_dw);
  const bool summed = with_dh && (pieces > 1 || parts > 1);  // dh is the sum of fp32 parts
  if (summed && (!aligned16(g->dh_sum, a->dim, 4) ||
                 g->dh_sum_bytes < 4L * parts * a->rows * a->dim))
    return -2;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const uint64_t rows = a->rows, dim = a->dim;
  const float factor = a->fp16 ? 1.0f / (1 << kFp16Shift) : 1.0f;
  const GradScale scale{g->grad, g->totals, factor};

  for (int i = 0; i < pieces; ++i) {
    const long begin = static_cast<long>(i) * g->piece;
    const int width = static_cast<int>(a->vocab - begin < g->piece ? a->vocab - begin : g->piece);
    const uint16_t* w = static_cast<const uint16_t*>(a->weight) + begin * a->ld_weight;
    const uint64_t dl_size = rows * g->piece;

    DlogitsOp::Params d{};
    int rc = pair::map_operand(&d.a, a->hidden, false, rows, dim, a->ld_hidden, 1,
                               rows * a->ld_hidden);
    if (rc == 0)
      rc = pair::map_operand(&d.b, w, false, width, dim, a->ld_weight, 1,
                             static_cast<uint64_t>(width) * a->ld_weight);
    if (rc == 0)
      rc = pair::map_3d(&d.out, g->dlogits, 2, width, rows, g->piece, 1, dl_size, 64, 32);
    if (rc != 0) return 1000 + rc;
    d.grid = Grid{tiles_of(rows, pair::kTileM), tiles_of(width, pair::kTileN), 0};
    d.grid.band = band_of(d.grid.mt, a->dim);
    d.total = d.grid.mt * d.grid.nt;
    d.num_kb = tiles_of(dim, pair::kBK);
    d.fp16 = a->fp16 != 0;
    d.status = a->status;
    d.targets = a->targets;
    d.lse2 = a->lse2;
    d.one = a->fp16 ? static_cast<float>(1 << kFp16Shift) : 1.0f;
    d.rows = a->rows;
    d.vocab_begin = static_cast<int>(begin);
    d.width = width;
    rc = pair::launch_pair<DlogitsOp>(d, stream);
    if (rc != 0) return rc;

    GradOp::Params q{};
    rc = pair::map_operand(&q.dl_mn, g->dlogits, true, width, rows, g->piece, 1, dl_size);
    if (rc == 0)
      rc = pair::map_operand(&q.dl_k, g->dlogits, false, rows, width, g->piece, 1, dl_size);
    if (rc == 0)
      rc = pair::map_operand(&q.h, a->hidden, true, dim, rows, a->ld_hidden, 1,
                             rows * a->ld_hidden);
    if (rc == 0)
      rc = pair::map_operand(&q.w, w, true, dim, width, a->ld_weight, 1,
                             static_cast<uint64_t>(width) * a->ld_weight);
    if (rc == 0 && with_dw)
      rc = pair::map_3d(&q.dw, static_cast<uint8_t*>(g->dw) + begin * g->ld_dw * dw_elem, dw_elem,
                        dim, width, g->ld_dw, 1, static_cast<uint64_t>(width) * g->ld_dw,
                        128 / dw_elem, 32);
    if (rc == 0 && summed)
      rc = pair::map_3d(&q.dh, g->dh_sum, 4, dim, rows, dim, parts, rows * dim, 32, 32);
    else if (rc == 0 && with_dh)
      rc = pair::map_3d(&q.dh, g->dh, 2, dim, rows, g->ld_dh, 1, rows * g->ld_dh, 64, 32);
    if (rc != 0) return 1000 + rc;
    q.fp16 = a->fp16 != 0;
    q.status = a->status;
    q.scale = scale;
    q.dw_mt = tiles_of(width, pair::kTileM);
    q.dh_mt = tiles_of(rows, pair::kTileM);
    q.dh_nt = tiles_of(dim, pair::kTileN);
    q.dw_kb = tiles_of(rows, pair::kBK);
    q.dh_kb = tiles_of(width, pair::kBK);
    q.dh_part_kb = tiles_of(q.dh_kb, parts);
    const int dw_tiles = with_dw ? q.dw_mt * q.dh_nt : 0;
    q.dh_tiles = with_dh ? q.dh_mt * q.dh_nt * parts : 0;
    q.total = q.dh_tiles + dw_tiles;
    q.rows = a->rows;
    q.width = width;
    q.dim = a->dim;
    q.dw_kind = g->dw_kind;
    q.dh_kind = !summed ? kOut16 : (i == 0 ? kOutF32 : kOutF32Add);
    deal(q, q.dh_tiles, dw_tiles, q.total < pairs ? q.total : pairs);
    rc = pair::launch_pair<GradOp>(q, stream);
    if (rc != 0) return rc;
  }
  if (!summed) return 0;
  const long vecs = static_cast<long>(a->rows) * a->dim / 8;
  const long blocks = (vecs + 255) / 256;
  return launch_pdl(ce_dh_kernel, dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096)),
                    dim3(256), 0, stream, static_cast<const float*>(g->dh_sum), parts, vecs, a->dim / 8,
                    g->dh, g->ld_dh, scale, a->fp16);
}
