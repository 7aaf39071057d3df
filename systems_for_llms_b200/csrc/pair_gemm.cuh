// Matrix products by pairs of CTAs: the main loop shared by the projection cross entropy
// (linear_ce.cu) and the Newton-Schulz products (newton_schulz.cu).
//
//   D[256, 256] += A[256, 64] * B[256, 64]^T   per stage, fp32 accumulation in tensor memory
//
// A cluster of two CTAs computes one 256 x 256 tile with tcgen05.mma.cta_group::2: each CTA
// brings its own 128 rows of A and half of the columns of B (16 + 16 KB per 64-deep step against
// 16 + 32 KB for a CTA that works alone on 128 x 256), so a step needs a third less operand
// traffic and shared memory holds six steps instead of four.  Per CTA: warp 0 streams its operand
// halves with TMA (no multicast), warp 1 of the leading CTA issues the products for both, and
// warps 2-9 drain one of two 128 x 256 accumulators through the epilogue while the other fills.
// Persistent: a cluster walks tiles cluster_id, cluster_id + clusters, ...
//
// Barriers.  full[s] exists in the leader only: it expects the bytes of both CTAs' loads, which
// both CTAs' TMA units report to it.  empty[s] and acc_full[a] are signalled in both CTAs by one
// multicast commit.  acc_empty[a] is the leader's; all sixteen epilogue warps arrive on it.  Every
// wait is bounded; one that runs out sets the status word and the CTA's abort flag, and both CTAs
// then leave through the common exit (copies in flight are waited for, tensor memory is freed).
//
// Op supplies the tile order, the tensor maps and the epilogue:
//   struct Op::Params { ...; int total; bool fp16; int* status; }
//   static int  Op::first(p, cluster), Op::next(p, w, cluster, clusters)
//                                  the cluster's first tile and the one after w (>= total: none)
//   static Tile Op::tile(p, w)     where the tile lies
//   static constexpr int Op::kForms  the combinations of orientations that occur
//   static const CUtensorMap* Op::map_a_k(p, t), map_a_mn, map_b_k, map_b_mn   rank-3 maps
//                                    {inner, rows, batch} of the orientations that occur
//   static constexpr int Op::kEpiTiles           staging tiles per epilogue warp, 1 or 2
//   static void Op::begin(p, t, EpiContext&)     before the accumulator is ready (prefetches)
//   static void Op::epilogue(p, t, EpiContext&)  one warp's share of the tile
#pragma once
#include <cuda_fp16.h>

#include <type_traits>

#include "launch.cuh"
#include "ptx.cuh"
#include "tensormap.cuh"

namespace sfl {
namespace pair {

constexpr int kCtaM = 128;               // rows of A (and of the accumulator) per CTA
constexpr int kTileM = 2 * kCtaM;        // rows of a pair's tile
constexpr int kTileN = 256;
constexpr int kHalfN = kTileN / 2;       // columns of B that each CTA brings
constexpr int kBK = 64;
constexpr int kABytes = kCtaM * kBK * 2;
constexpr int kStageBytes = kABytes + kHalfN * kBK * 2;
constexpr int kMaxStages = 6;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kEpiTileBytes = 32 * 128;  // a staging tile: 32 rows of 128 bytes
constexpr int kTmemCols = 512;           // two accumulators of 256 columns

// Shared memory of an Op whose epilogue warps own one or two staging tiles each.
template <class Op>
struct Config {
  static constexpr int kStages = Op::kEpiTiles == 1 ? 6 : 5;
  static constexpr int kWarpBytes = Op::kEpiTiles * kEpiTileBytes;
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kEpiWarps * kWarpBytes + 512;
  static_assert(kSmemBytes <= 232448 && kStages <= kMaxStages, "more than a CTA's shared memory");
};

struct Tile {
  int m0, n0, z;  // first row, first column, batch index
  int num_kb;     // 64-deep steps
  int kb0;        // first step of the reduction
  int kind;       // for Ops that mix products
  int a_mn, b_mn; // steps before this one read A / B MN-major (see gemm.cu), the others K-major
  bool same;      // B's rows are A's: one copy serves as both operands
};

struct __align__(8) Barriers {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t aux_full[kEpiWarps];
  uint32_t tmem_base;
  int abort;
};

struct EpiContext {
  uint32_t acc;      // tensor-memory address of this warp's lanes, column 0 of the accumulator
  int row0;          // global row of lane 0
  int part;          // columns [128 * part, 128 * part + 128) of the tile belong to this warp
  int lane;
  uint8_t* smem;     // the warp's staging tiles
  uint64_t* aux_bar; // the warp's barrier for loads of its own
  uint32_t aux_phase;
  volatile int* abort;
  int* status;
};

// ------------------------------------------------------------- primitives ----
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile(
      "barrier.cluster.arrive.release.aligned;\n\t"
      "barrier.cluster.wait.acquire.aligned;" ::
          : "memory");
}
// The same shared-memory offset in the pair's leading CTA.
__device__ __forceinline__ uint32_t in_leader(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void arrive_leader(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(in_leader(smem_u32(bar)))
               : "memory");
}
// A load into this CTA's shared memory whose bytes are reported to the leader's barrier.
__device__ __forceinline__ void load_3d(void* dst, const CUtensorMap* map, uint32_t leader_bar,
                                        int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(leader_bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void store_3d(const CUtensorMap* map, const void* src, int x, int y,
                                         int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void reduce_add_3d(const CUtensorMap* map, const void* src, int x, int y,
                                              int z) {
  asm volatile(
      "cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], "
      "[%1];" ::"l"(reinterpret_cast<uint64_t>(map)),
      "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                         uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives on the barrier at this offset in both CTAs once the products issued so far are done.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %1;" ::"r"(smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

// As mbar_wait, but also gives up when the CTA is already leaving.
__device__ __forceinline__ bool wait_or_leave(uint64_t* bar, uint32_t parity, volatile int* abort) {
  unsigned long long started = 0;
  for (uint32_t spin = 0; spin < (1u << 26); ++spin) {
    if (mbar_try_wait(bar, parity)) return true;
    if (spin > 2048) {
      __nanosleep(256);
      if (*abort) return false;
      if ((spin & 1023) == 0) {
        unsigned long long now;
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
        if (started == 0) started = now;
        if (now - started > 2000000000ull) return false;
      }
    }
  }
  return false;
}

// Instruction descriptor of the pair's 256 x 256 x 16 product; both operands have one type.
__device__ __forceinline__ uint32_t instruction_descriptor(bool fp16, bool a_mn, bool b_mn) {
  const uint32_t d = umma_idesc_bf16(kTileM, kTileN, a_mn, b_mn);
  return fp16 ? d & ~((1u << 7) | (1u << 10)) : d;  // operand format 0: fp16
}

// The warp's own loads (the bytes it announced on aux_bar) have landed.  A wait that runs out
// makes the CTA leave; the tile's results are then incomplete and the status word says so.
__device__ __forceinline__ void wait_aux(EpiContext& c) {
  if (!wait_or_leave(c.aux_bar, c.aux_phase, c.abort)) {
    report_status(c.status, kStatusTimeoutFull);
    *c.abort = 1;
  }
  c.aux_phase ^= 1;
}

// Names for the orientations that an Op does not use.
struct NoMaps {
  template <class P> static __device__ const CUtensorMap* map_a_k(const P&, const Tile&) { return nullptr; }
  template <class P> static __device__ const CUtensorMap* map_a_mn(const P&, const Tile&) { return nullptr; }
  template <class P> static __device__ const CUtensorMap* map_b_k(const P&, const Tile&) { return nullptr; }
  template <class P> static __device__ const CUtensorMap* map_b_mn(const P&, const Tile&) { return nullptr; }
};

// Bases for Ops whose epilogue loads nothing of its own, and whose tiles are dealt round robin.
struct Plain {
  static constexpr int kEpiTiles = 1;
  template <class P, class C>
  static __device__ __forceinline__ void begin(const P&, const Tile&, C&) {}
};
struct RoundRobin {
  template <class P> static __device__ __forceinline__ int first(const P&, int cluster) {
    return cluster;
  }
  template <class P>
  static __device__ __forceinline__ int next(const P&, int w, int, int clusters) {
    return w + clusters;
  }
};

// ------------------------------------------------------- epilogue helpers ----
// A staging tile is 32 rows of 128 bytes in the 128-byte swizzle of its tensor map.
__device__ __forceinline__ uint8_t* tile_chunk(uint8_t* tile, int row, int chunk) {
  return tile + row * 128 + ((chunk ^ (row & 7)) << 4);
}
__device__ __forceinline__ uint32_t pack_16(bool fp16, float lo, float hi) {
  if (fp16) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  return pack_bf16(lo, hi);
}
// 32 values of one row into half `half` (0 or 1) of its 128-byte line.
__device__ __forceinline__ void stage_16(uint8_t* tile, int row, int half, const float (&v)[32],
                                         bool fp16) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint4 q;
    q.x = pack_16(fp16, v[8 * j + 0], v[8 * j + 1]);
    q.y = pack_16(fp16, v[8 * j + 2], v[8 * j + 3]);
    q.z = pack_16(fp16, v[8 * j + 4], v[8 * j + 5]);
    q.w = pack_16(fp16, v[8 * j + 6], v[8 * j + 7]);
    *reinterpret_cast<uint4*>(tile_chunk(tile, row, 4 * half + j)) = q;
  }
}
__device__ __forceinline__ void stage_32(uint8_t* tile, int row, const float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    *reinterpret_cast<float4*>(tile_chunk(tile, row, j)) =
        make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
}
// The staging tile may be rewritten once its last store has read it.
__device__ __forceinline__ void stage_reuse(int lane) {
  if (lane == 0) tma_store_wait_read<0>();
  __syncwarp();
}
__device__ __forceinline__ void load_acc(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  tmem_ld_32x32(addr, r);
  tmem_ld_wait();
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
}

// Calls f(a_mn, b_mn, only_a) with constants for the step's orientations; only the combinations
// that Op::kForms names are compiled.
enum Form : int {
  kFormKK = 1, kFormMM = 2, kFormKM = 4, kFormMK = 8,  // A and B K-major / MN-major
  kFormSame = 16,                                      // KK and MM also with one copy for both
};
template <class Op, class F>
__device__ __forceinline__ void by_orientation(const Tile& t, int kb, F&& f) {
  const std::true_type yes;
  const std::false_type no;
  constexpr int kForms = Op::kForms;
  if constexpr ((kForms & kFormSame) != 0) {
    if (t.same) {
      if ((kForms & kFormMM) != 0 && kb < t.a_mn) f(yes, yes, yes);
      else f(no, no, yes);
      return;
    }
  }
  if constexpr (kForms == kFormKK) {
    f(no, no, no);
  } else if constexpr (kForms == kFormMM) {
    f(yes, yes, no);
  } else {
    const bool a = kb < t.a_mn, b = kb < t.b_mn;
    if constexpr ((kForms & kFormKK) != 0) {
      if (!a && !b) f(no, no, no);
    }
    if constexpr ((kForms & kFormMM) != 0) {
      if (a && b) f(yes, yes, no);
    }
    if constexpr ((kForms & kFormKM) != 0) {
      if (!a && b) f(no, yes, no);
    }
    if constexpr ((kForms & kFormMK) != 0) {
      if (a && !b) f(yes, no, no);
    }
  }
}

// ----------------------------------------------------------------- kernel ----
template <class Op>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
pair_kernel(const __grid_constant__ typename Op::Params p) {
  constexpr int kStages = Config<Op>::kStages;
  extern __shared__ uint8_t smem_raw[];
  // The dynamic segment starts at the same offset in both CTAs, so this does too.
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint8_t* epi_smem = smem + kStages * kStageBytes;
  Barriers* bars = reinterpret_cast<Barriers*>(epi_smem + kEpiWarps * Config<Op>::kWarpBytes);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int clusters = gridDim.x >> 1;
  const int cluster = blockIdx.x >> 1;
  volatile int* abort = &bars->abort;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars->acc_full[s], 1);
      mbar_init(&bars->acc_empty[s], 2 * kEpiWarps);
    }
    for (int s = 0; s < kEpiWarps; ++s) mbar_init(&bars->aux_full[s], 1);
    bars->abort = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&bars->tmem_base)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  pdl_launch_dependents();
  pdl_wait();

  if (warp == 0) {
    // ------------------------------------------------------ TMA producer ----
    // The whole warp walks the loops and one elected lane issues, with code of its own for each
    // orientation, for the reason given at the MMA issuer: the operands of a TMA instruction are
    // uniform registers too, and a lane that has to move coordinates and map addresses there takes
    // 770 cycles per step where the products take 512.
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t full0 = in_leader(smem_u32(&bars->full[0]));
    for (int w = Op::first(p, cluster); w < p.total && ok; w = Op::next(p, w, cluster, clusters)) {
      const Tile t = Op::tile(p, w);
      const int m0 = t.m0 + rank * kCtaM;
      const int n0 = t.n0 + rank * kHalfN;
      for (int kb = 0; kb < t.num_kb; ++kb) {
        if (!wait_or_leave(&bars->empty[stage], phase ^ 1, abort)) {
          if (lane == 0) report_status(p.status, kStatusTimeoutEmpty);
          *abort = 1;
          ok = false;
          break;
        }
        uint8_t* sa = smem + stage * kStageBytes;
        const uint32_t bar = full0 + stage * static_cast<uint32_t>(sizeof(uint64_t));
        const int k0 = (t.kb0 + kb) * kBK;
        auto bring = [&](auto a_mn, auto b_mn, auto only_a) {
          if (elect_one()) {
            if (rank == 0)
              mbar_expect_tx(&bars->full[stage],
                             2 * (decltype(only_a)::value ? kABytes : kStageBytes));
            if constexpr (decltype(a_mn)::value) {
              load_3d(sa, Op::map_a_mn(p, t), bar, m0, k0, t.z);
              load_3d(sa + kBK * 128, Op::map_a_mn(p, t), bar, m0 + 64, k0, t.z);
            } else {
              load_3d(sa, Op::map_a_k(p, t), bar, k0, m0, t.z);
            }
            if constexpr (!decltype(only_a)::value) {
              if constexpr (decltype(b_mn)::value) {
                load_3d(sa + kABytes, Op::map_b_mn(p, t), bar, n0, k0, t.z);
                load_3d(sa + kABytes + kBK * 128, Op::map_b_mn(p, t), bar, n0 + 64, k0, t.z);
              } else {
                load_3d(sa + kABytes, Op::map_b_k(p, t), bar, k0, n0, t.z);
              }
            }
          }
          __syncwarp();
        };
        by_orientation<Op>(t, kb, bring);
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    // Leave only when every stage has been handed back: no commit from the leader and no copy
    // is then still on its way into this CTA's shared memory.
    for (int s = 0; s < kStages; ++s) {
      if (!mbar_wait(&bars->empty[stage], phase ^ 1)) break;
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
  } else if (warp == 1) {
    // -------------------------------------------------------- MMA issuer ----
    // The leader's warp walks converged; one elected lane issues (see gemm.cu).
    if (rank == 0) {
      const uint64_t k0 = umma_smem_desc(smem_u32(smem), 16, 1024);           // K-major
      const uint64_t mn0 = umma_smem_desc(smem_u32(smem), kBK * 128, 1024);   // MN-major
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int w = Op::first(p, cluster); w < p.total && ok; w = Op::next(p, w, cluster, clusters)) {
        const Tile t = Op::tile(p, w);
        if (!wait_or_leave(&bars->acc_empty[acc], acc_phase ^ 1, abort)) {
          report_status(p.status, kStatusTimeoutTmemEmpty);
          *abort = 1;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + acc * kTileN;
        for (int kb = 0; kb < t.num_kb; ++kb) {
          if (!wait_or_leave(&bars->full[stage], phase, abort)) {
            report_status(p.status, kStatusTimeoutFull);
            *abort = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          // Each orientation has code of its own: descriptors are then the sum of warp-uniform
          // values and stay in uniform registers.  Chosen by arithmetic on the tile they would be
          // moved there for every product, which the issuing lane has no time for.
          auto issue = [&](auto a_mn, auto b_mn, auto only_a) {
            constexpr bool kA = decltype(a_mn)::value, kB = decltype(b_mn)::value;
            constexpr uint32_t b_at = decltype(only_a)::value ? 0 : kABytes;
            const uint64_t a = umma_desc_advance(kA ? mn0 : k0, stage * kStageBytes);
            const uint64_t b = umma_desc_advance(kB ? mn0 : k0, stage * kStageBytes + b_at);
            const uint32_t idesc = instruction_descriptor(p.fp16, kA, kB);
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < kBK / 16; ++k)
                mma_pair(d, umma_desc_advance(a, k * (kA ? 2048 : 32)),
                         umma_desc_advance(b, k * (kB ? 2048 : 32)), idesc, (kb | k) != 0);
              commit_pair(&bars->empty[stage]);
            }
          };
          by_orientation<Op>(t, kb, issue);
          if (kb == t.num_kb - 1 && elect_one()) commit_pair(&bars->acc_full[acc]);
          __syncwarp();
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
    }
  } else {
    // ---------------------------------------------------------- epilogue ----
    const int quarter = warp & 3;  // tensor-memory lanes this warp may read
    EpiContext c;
    c.part = (warp - 2) >> 2;
    c.lane = lane;
    c.smem = epi_smem + (warp - 2) * Config<Op>::kWarpBytes;
    c.aux_bar = &bars->aux_full[warp - 2];
    c.aux_phase = 0;
    c.abort = abort;
    c.status = p.status;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int w = Op::first(p, cluster); w < p.total; w = Op::next(p, w, cluster, clusters)) {
      const Tile t = Op::tile(p, w);
      c.acc = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * kTileN;
      c.row0 = t.m0 + rank * kCtaM + quarter * 32;
      Op::begin(p, t, c);
      if (!wait_or_leave(&bars->acc_full[acc], acc_phase, abort)) {
        report_status(p.status, kStatusTimeoutTmemFull);
        *abort = 1;
        break;
      }
      tc_fence_after();
      Op::epilogue(p, t, c);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_leader(&bars->acc_empty[acc]);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    if (lane == 0) tma_store_wait<0>();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                 "r"(kTmemCols)
                 : "memory");
  }
}

// ------------------------------------------------------------------- host ----
// Rank-3 operand or output map: {inner, rows, batch} of 2-byte (or fp32) elements.
inline int map_3d(CUtensorMap* out, const void* base, int elem, uint64_t inner, uint64_t rows,
                  uint64_t ld, uint64_t batch, uint64_t batch_stride, uint32_t box_inner,
                  uint32_t box_rows) {
  const uint64_t dims[3] = {inner, rows, batch};
  const uint64_t strides[3] = {0, ld * elem, batch_stride * elem};
  const uint32_t box[3] = {box_inner, box_rows, 1};
  return make_tensormap_nd(out, base, elem, 3, dims, strides, box, 3);
}
// K-major operand [rows, k] (box 64 k x 128 rows) or MN-major operand [k, rows] (box 64 x 64).
inline int map_operand(CUtensorMap* out, const void* base, bool mn, uint64_t rows, uint64_t k,
                       uint64_t ld, uint64_t batch, uint64_t batch_stride) {
  return mn ? map_3d(out, base, 2, rows, k, ld, batch, batch_stride, 64, kBK)
            : map_3d(out, base, 2, k, rows, ld, batch, batch_stride, kBK, kCtaM);
}

inline int sm_count_here(int* device_out = nullptr) {
  int device = 0, count = 0;
  if (cudaGetDevice(&device) != cudaSuccess ||
      cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
    return 0;
  if (device_out != nullptr) *device_out = device;
  return count;
}

inline int pairs_here() { return sm_count_here() / 2; }

template <class Op>
int launch_pair(const typename Op::Params& p, cudaStream_t stream) {
  if (p.total <= 0) return 0;
  int device = 0;
  const int sms = sm_count_here(&device);
  if (sms < 2) return -1;
  // The attribute belongs to the kernel on one device.
  static bool configured[64] = {};
  if (device >= 64 || !configured[device]) {
    const cudaError_t e = cudaFuncSetAttribute(
        pair_kernel<Op>, cudaFuncAttributeMaxDynamicSharedMemorySize, Config<Op>::kSmemBytes);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (device < 64) configured[device] = true;
  }
  const int pairs = sms / 2;
  const int clusters = p.total < pairs ? p.total : pairs;
  return launch_pdl(pair_kernel<Op>, dim3(2 * clusters), dim3(kThreads), Config<Op>::kSmemBytes, stream, p);
}

}  // namespace pair
}  // namespace sfl
