// Product of two matrices held in 4 bits (formats and layouts: fp4.cuh):
//
//   D[m, n] = out((sum_k A[m, k] B[n, k]) * scale_b[n] * scale_a[m] (+ bias[n]))
//
// with A and B the codes times their block scales.  The block scales enter the tensor
// cores' product itself: tcgen05.mma.kind::mxf4nvf4.block_scale multiplies each run of
// 16 (or 32) products by the two scales, which it reads from tensor memory, and sums in
// fp32; the row scales and the bias are applied in the epilogue.
//
// Both kernels stream K in blocks of 128 bytes (256 elements, one 128-byte swizzle row)
// through a ring of mbarrier stages: codes by 2-D TMA, scale tiles (512 bytes per 128
// rows x 4 blocks, as they lie) by 3-D TMA, then tcgen05.cp (32 lanes x 128 bits, to all
// four lane quadrants) of each scale tile and four products of K = 64.  One thread issues
// both; the tensor-core pipe runs them in order, so nothing waits in between.  The issuing
// warp stays converged and elects the thread at each stage: its addresses are then
// warp-uniform values, which the instructions' operands need anyway.  Rows and
// blocks past the end arrive as zero from the TMA.
//
//   fp4_gemm_pair_kernel   256 x 256 tiles on CTA pairs (cta_group::2)
//   fp4_gemm_rows_kernel   for few rows of A: 128 rows of B x up to 128 rows of A, K split
//                          over a cluster
//
// Bound and measured (B200).  Large products: 38 KB per stage and CTA (35 with blocks of 32)
// come in at 88 GB/s per SM, 13 TB/s in all: the loads alone take 109 us of the 10800 x 9216 x
// 3072 product, the tensor cores alone 104; together 139 us (4.4 PFLOP/s) in a short run and
// 161-165 (3.7) once the power cap lowers the clock.  From 233 us on: an issuing warp that
// stays converged 169 (a lone lane took 40 cycles per scale copy and more per product),
// results by TMA 140.  Walking the tiles in bands of 4, 8 or 16 rows, four stages instead of
// five, and evict-first stores changed nothing.  1350 x 3072 x 12288 (blocks of 32): 24 us.
// Few rows: the weight's bytes, and a fixed 4 us: one row x 9216 x 3072 5.1 us, 6.6 with the
// quantisation of the row, which each CTA does for itself while the weight comes in (7.9 with
// a kernel before); 128 rows 10.7.
//
// Every mbarrier wait is bounded (pipeline.cuh), as in the FP8 product.
#include "fp4_quant.cuh"
#include "tcgen05.cuh"

namespace jo {
namespace {

constexpr int kKBytes = 128;                // of K per stage
constexpr int kKElems = 2 * kKBytes;        // 256
constexpr int kSteps = 4;                   // products of K = 64 per stage
constexpr int kChunk = 512;                 // bytes of a scale tile

template <bool kMx>
struct Fmt {
  static constexpr int kTiles = kMx ? 2 : 4;  // scale tiles per 128 rows and stage
  static constexpr int kScale = kTiles * kChunk;
  static constexpr int kCols = kTiles * 4;  // tensor-memory columns of 128 rows' scales of a stage
};

// Instruction descriptor, block-scaled: e2m1 x e2m1, both K-major; the scale ids pick the
// byte pair of each 32-bit tensor-memory cell that a K = 64 product of blocks of 32 uses.
template <bool kMx>
__device__ __forceinline__ constexpr uint32_t fp4_idesc(int m, int n, int id) {
  return ((uint32_t)id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)kMx << 23) |
         ((uint32_t)(m >> 4) << 24) | ((uint32_t)id << 29);
}
// Scale tile in shared memory: 32 rows of 16 bytes, no swizzle, 8-row groups 128 B apart.
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}
template <bool kPair>
__device__ __forceinline__ void scale_copy(uint32_t taddr, uint64_t desc) {
  if constexpr (kPair)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
#define JO_FP4_MMA(GROUP, VEC)                                                                              \
  asm volatile(                                                                                             \
      "{\n\t.reg .pred p;\n\t"                                                                              \
      "setp.ne.b32 p, %6, 0;\n\t"                                                                           \
      "tcgen05.mma.cta_group::" GROUP ".kind::mxf4nvf4.block_scale.scale_vec::" VEC                         \
      " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),                                                    \
      "l"(ad), "l"(bd), "r"(idesc), "r"(sfa), "r"(sfb), "r"((uint32_t)accumulate)                           \
      : "memory")
template <bool kPair, bool kMx>
__device__ __forceinline__ void fp4_mma(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t sfa,
                                        uint32_t sfb, bool accumulate) {
  if constexpr (kPair && kMx)
    JO_FP4_MMA("2", "2X");
  else if constexpr (kPair)
    JO_FP4_MMA("2", "4X");
  else if constexpr (kMx)
    JO_FP4_MMA("1", "2X");
  else
    JO_FP4_MMA("1", "4X");
}
#undef JO_FP4_MMA

// One stage: scales to tensor memory at `sf` (A's, then B's), then its products.  ad, bd:
// descriptors of the stage's codes; sad, sbd: of its scales; kGroups: 128-row groups of B's
// scales.  `steps` < 4 only in the last stage.
template <bool kPair, bool kMx, int kM, int kN, int kGroups>
__device__ __forceinline__ void stage_products(uint32_t acc, uint64_t ad, uint64_t bd, uint64_t sad, uint64_t sbd,
                                               uint32_t sf, int steps, bool first) {
  using F = Fmt<kMx>;
#pragma unroll
  for (int j = 0; j < F::kTiles; ++j) {
    scale_copy<kPair>(sf + j * 4, sad + j * (kChunk >> 4));
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
      scale_copy<kPair>(sf + F::kCols + (j * kGroups + g) * 4, sbd + ((g * F::kScale + j * kChunk) >> 4));
  }
#pragma unroll
  for (int kk = 0; kk < kSteps; ++kk) {
    const int j = kMx ? kk >> 1 : kk;
    if (kk < steps)
      fp4_mma<kPair, kMx>(acc, ad + 2 * kk, bd + 2 * kk, fp4_idesc<kMx>(kM, kN, kMx ? 2 * (kk & 1) : 0), sf + j * 4,
                          sf + F::kCols + j * 4 * kGroups, !(first && kk == 0));
  }
}

struct Fp4GemmArgs {
  void* d;
  int64_t ldd;
  const float* sa;  // null: 1
  const float* sb;
  const void* bias;
  int m, n, k;
  int tiles_m, tiles_n;
  bool b_ready;  // B was complete before the previous kernel of the stream began
  const void* x;  // rows that the product's kernel quantises itself (null: A is given in 4 bits)
  int64_t ldx;
  int x_align;  // bytes that every run's address is a multiple of (Run::load)
  unsigned int* fault;
};

__device__ __forceinline__ int steps_of(int k, int kb) { return min(kSteps, (k - kb * kKElems + 63) / 64); }

// ------------------------------------------------------------------ CTA pairs
// As the FP8 product's pair kernel (CTA rank r of a (2,1,1) cluster loads A rows and B rows
// [128 r, 128 r + 128) of a 256 x 256 tile, the leader issues for both), with, per stage, the
// scales of the CTA's own 128 rows of A and of all 256 rows of B, which each CTA's half of
// the product needs whole.
//
// Tensor memory: two accumulators of 256 columns and two stages of scales (2 x 48 columns)
// are more than the 512 there are, so the accumulators overlap by 96 columns, at 0 and 160,
// the scales at 416.  An epilogue first takes its accumulator's overlapped columns into
// registers; the next tile's products start then, while it works on the other 160.
// Results leave by TMA, 32 rows x 64 columns at a time from a staging box per warp.
constexpr int kAccStep = 160, kScaleCol = 416;
constexpr int kPairM = 256, kPairN = 256;
constexpr int kEpiWarps = 8;
constexpr int kPairThreads = 64 + 32 * kEpiWarps;

template <bool kMx>
struct PairSmem {
  using F = Fmt<kMx>;
  static constexpr int kStages = 5;
  static constexpr int kOp = 128 * kKBytes;  // 16 KB of codes
  static constexpr int kStage = 2 * kOp + 3 * F::kScale;
  static constexpr int kA = 0, kB = kStages * kOp;
  static constexpr int kSA = 2 * kStages * kOp, kSB = kSA + kStages * F::kScale;
  static constexpr int kBox = 32 * 128;  // an epilogue warp's staging box: 32 rows x 64 columns
  static constexpr int kOut = (kSB + kStages * 2 * F::kScale + 1023) / 1024 * 1024;
  static constexpr int kBars = kOut + kEpiWarps * kBox;
  static constexpr int kBytes = kBars + 256 + 1024 /*align*/;
};

// 32 accumulator columns of this lane's row: scales, bias, rounding, four 16-byte chunks into
// the warp's staging box (row = lane, 128-byte swizzle) from chunk `c0` on.
template <typename OutT>
__device__ __forceinline__ void stage32(const Fp4GemmArgs& g, const uint32_t* r, int n0, float s_a, uint8_t* box,
                                        int lane, int c0) {
  const OutT* bias = reinterpret_cast<const OutT*>(g.bias);
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const int n = n0 + 8 * h;
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = __uint_as_float(r[8 * h + e]);
    if (n < g.n) {  // N is a multiple of 8; columns past it are not stored
      if (g.sb) {
        const float4 s0 = __ldg(reinterpret_cast<const float4*>(g.sb + n));
        const float4 s1 = __ldg(reinterpret_cast<const float4*>(g.sb + n + 4));
        const float s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] *= s[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] *= s_a;
      if (bias) {
        float b[8];
        Elt<OutT>::unpack(__ldg(reinterpret_cast<const uint4*>(bias + n)), b);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] += b[e];
      }
    }
    *reinterpret_cast<uint4*>(box + lane * 128 + (((c0 + h) ^ (lane & 7)) << 4)) = Elt<OutT>::pack(o);
  }
}
// The warp's staging box, filled by all lanes, to rows [m0, m0 + 32) x columns [n0, n0 + 64)
// of D (what lies outside D is clipped by the TMA).
__device__ __forceinline__ void store_box(const CUtensorMap* map, const Fp4GemmArgs& g, uint32_t box, int n0, int m0,
                                          int lane) {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if (lane == 0 && n0 < g.n && m0 < g.m) {
    tma_store_2d(map, box, n0, m0);
    bulk_commit();
  }
}

template <typename OutT, bool kMx>
__global__ void __launch_bounds__(kPairThreads, 1)
    fp4_gemm_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                         const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb,
                         const __grid_constant__ CUtensorMap map_d, const Fp4GemmArgs args) {
  using S = PairSmem<kMx>;
  using F = Fmt<kMx>;
  constexpr int kStages = S::kStages;
  unsigned int* const fault = args.fault;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t base = (raw_base + 1023u) & ~1023u;  // identical offsets in both CTAs
  uint8_t* gbase = smem_raw + (base - raw_base);
  const uint32_t bars = base + S::kBars;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (kStages + s); };
  const uint32_t tfull = bars + 8u * (2 * kStages), drained = tfull + 8, done = tfull + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbase + (tfull + 24 - base));

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  const int cluster = (int)(blockIdx.x >> 1), nclusters = (int)(gridDim.x >> 1);
  const int num_tiles = args.tiles_m * args.tiles_n;
  const int kblocks = (args.k + kKElems - 1) / kKElems;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(tfull, 1);
    mbar_init(drained, 2 * kEpiWarps);  // the epilogue warps of both CTAs
    mbar_init(done, 1);
    mbar_init_fence();
  }
  if (warp == 1) {  // same warp in both CTAs: the pair allocation is collective
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  __syncthreads();
  cluster_sync();  // both CTAs' barriers initialised before any cross-CTA signal
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- TMA producer (both CTAs)
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      int issued = 0;
      for (int tile = cluster; tile < num_tiles && ok; tile += nclusters) {
        const int tm = tile / args.tiles_n, tn = tile - tm * args.tiles_n;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, fault)) {
            ok = false;
            break;
          }
          const uint32_t fb = cluster_addr(full_bar(stage), 0);
          if (leader) mbar_expect_tx(full_bar(stage), 2 * S::kStage);
          tma_load_2d_pair(base + S::kA + stage * S::kOp, &map_a, kb * kKBytes, tm * kPairM + (int)rank * 128, fb);
          tma_load_2d_pair(base + S::kB + stage * S::kOp, &map_b, kb * kKBytes, tn * kPairN + (int)rank * 128, fb);
          tma_load_3d_pair(base + S::kSA + stage * F::kScale, &map_sa, 0, kb * F::kTiles, tm * 2 + (int)rank, fb);
          tma_load_3d_pair(base + S::kSB + stage * 2 * F::kScale, &map_sb, 0, kb * F::kTiles, tn * 2, fb);
          ++issued;
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // drain (leader): the pair's copies into every issued stage must have landed (the
      // leader's full barriers count both CTAs' bytes); the peer is held by the final
      // cluster barrier until then
      if (leader)
        for (int j = max(0, issued - kStages); j < issued; ++j)
          mbar_wait(full_bar(j % kStages), (j / kStages) & 1, fault);
    }
  } else if (warp == 1) {
    if (leader) {
      // ---------------- MMA issuer (leader CTA only)
      const uint64_t ad = sw128_desc(base + S::kA), bd = sw128_desc(base + S::kB);
      const uint64_t sad = scale_desc(base + S::kSA), sbd = scale_desc(base + S::kSB);
      int stage = 0;
      uint32_t phase = 0;
      int count = 0;  // stages so far: scales alternate between two column sets
      bool ok = true;
      int i = 0;
      for (int tile = cluster; tile < num_tiles && ok; tile += nclusters, ++i) {
        if (i > 0 && !(ok = __all_sync(0xffffffffu, mbar_wait(drained, (i - 1) & 1, fault)))) break;
        tc_fence_after();
        const uint32_t acc = tmem + (i & 1) * kAccStep;
        for (int kb = 0; kb < kblocks; ++kb, ++count) {
          if (!(ok = __all_sync(0xffffffffu, mbar_wait(full_bar(stage), phase, fault)))) break;
          tc_fence_after();
          if (elect_one()) {
            stage_products<true, kMx, kPairM, kPairN, 2>(
                acc, ad + stage * (S::kOp >> 4), bd + stage * (S::kOp >> 4), sad + stage * (F::kScale >> 4),
                sbd + stage * (2 * F::kScale >> 4), tmem + kScaleCol + (count & 1) * 3 * F::kCols,
                steps_of(args.k, kb), kb == 0);
            // the stage is reusable in both CTAs once these products have read it
            tc_commit_pair(empty_bar(stage));
            tc_commit_pair(cluster_addr(empty_bar(stage), 1));
            if (kb == kblocks - 1) {  // accumulator complete, in both CTAs
              tc_commit_pair(tfull);
              tc_commit_pair(cluster_addr(tfull, 1));
            }
          }
          __syncwarp();
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // TMEM is freed below and the peer's shared memory is read by these products: wait
      // until every one of them has retired
      if (elect_one()) tc_commit_pair(done);
      __syncwarp();
      mbar_wait(done, 0, fault);
    }
  } else {
    // ---------------- epilogue: warps 2..9 of both CTAs; warp w: lanes 32*(w%4).., and the
    // half (w-2)/4 of the accumulator's columns, as two boxes of 64
    const int q = warp & 3, half = (warp - 2) >> 2;
    uint8_t* const box = gbase + S::kOut + (warp - 2) * S::kBox;
    const uint32_t box_addr = base + S::kOut + (warp - 2) * S::kBox;
    auto refill = [&]() {  // the last box has left the staging buffer
      if (lane == 0) bulk_wait_read_all();
      __syncwarp();
    };
    auto drained_by_us = [&]() {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (leader)
          mbar_arrive(drained);
        else
          mbar_arrive_cluster(cluster_addr(drained, 0));
      }
    };
    int i = 0;
    for (int tile = cluster; tile < num_tiles; tile += nclusters, ++i) {
      const int tm = tile / args.tiles_n, tn = tile - tm * args.tiles_n;
      if (!__all_sync(0xffffffffu, mbar_wait(tfull, i & 1, fault))) break;
      tc_fence_after();
      const int m0 = tm * kPairM + (int)rank * 128 + q * 32, row = m0 + lane;
      const float s_a = row < args.m && args.sa ? __ldg(args.sa + row) : 1.f;
      const int odd = i & 1;
      const uint32_t t_acc = tmem + ((uint32_t)(q * 32) << 16) + odd * kAccStep;
      const int n0 = tn * kPairN;
      if (half == odd) {
        // none of this half's columns is the other accumulator's
        drained_by_us();
#pragma unroll 1
        for (int c = half * 128; c < half * 128 + 128; c += 64) {
          uint32_t r[64];
          tmem_ld64(t_acc + c, r);
          refill();
          stage32<OutT>(args, r, n0 + c, s_a, box, lane, 0);
          stage32<OutT>(args, r + 32, n0 + c + 32, s_a, box, lane, 4);
          store_box(&map_d, args, box_addr, n0 + c, m0, lane);
        }
      } else {
        // of [160, 256) (even) or [0, 96) (odd): 64 columns that are a box, 32 of the other box
        const int whole = odd ? 0 : 192, part = odd ? 64 : 160, rest = odd ? 96 : 128;
        uint32_t r[64], p[32];
        tmem_ld32(t_acc + part, p);
        tmem_ld64(t_acc + whole, r);
        drained_by_us();
        refill();
        stage32<OutT>(args, r, n0 + whole, s_a, box, lane, 0);
        stage32<OutT>(args, r + 32, n0 + whole + 32, s_a, box, lane, 4);
        store_box(&map_d, args, box_addr, n0 + whole, m0, lane);
        uint32_t o[32];
        tmem_ld32(t_acc + rest, o);
        refill();
        stage32<OutT>(args, p, n0 + part, s_a, box, lane, odd ? 0 : 4);
        stage32<OutT>(args, o, n0 + rest, s_a, box, lane, odd ? 4 : 0);
        store_box(&map_d, args, box_addr, n0 + (odd ? part : rest), m0, lane);
      }
      tc_fence_before();
    }
    refill();
  }
  __syncthreads();
  // neither CTA leaves while the other may still signal its barriers or have its shared
  // memory read by the pair's products
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ------------------------------------------------------------------ few rows
// B (the weight) takes the tensor cores' 128 rows and A's rows their columns, kCols of them,
// so a single token costs 16 columns and not 128 rows (kCols < 128 serves one tile of at
// most kCols rows: a tile's scales start at a 128-row group).  The CTAs of a cluster take
// contiguous parts of K of one tile; each then receives, from every CTA of the cluster by
// distributed shared memory, its share of the columns, and adds the parts in the CTAs'
// order: one result whatever the timing.
constexpr int kRowsThreads = 192;
constexpr int kMaxSplit = 8;

// kFused: A's part of K lies beside the ring, which then holds the weight alone.
template <bool kMx, int kCols, bool kFused>
struct RowsSmem {
  using F = Fmt<kMx>;
  static constexpr int kB = 128 * kKBytes;    // the weight's codes
  static constexpr int kA = kCols * kKBytes;  // kCols rows of A
  static constexpr int kStage = kFused ? kB + F::kScale : kB + kA + 2 * F::kScale;
  static constexpr int kPart = 128 * kCols * 4;  // received parts
  static constexpr int kRoom = 227 * 1024 - 2048 - kPart;
  static constexpr int kStages = kFused ? 6 : kRoom / kStage < 8 ? kRoom / kStage : 8;
  static constexpr int kAStages = kFused ? (kRoom - kStages * kStage) / (kA + F::kScale) : kStages;
  static constexpr int kOffB = 0, kOffA = kStages * kB, kOffSB = kOffA + kAStages * kA;
  static constexpr int kOffSA = kOffSB + kStages * F::kScale;
  static constexpr int kOffPart = kOffSA + kAStages * F::kScale;
  static constexpr int kBars = kOffPart + kPart;
  static constexpr int kRowScale = kBars + 256;        // kFused: per epilogue warp, 16 row scales
  static constexpr int kRowMax = kRowScale + 4 * 64;   // and of each row the four warps' maxima
  static constexpr int kBytes = kRowMax + 4 * 64 + 1024;
  static_assert(kBytes <= 227 * 1024, "shared memory");
  static_assert(kCols / kMaxSplit >= 2, "every CTA of a cluster has columns to add up");
  static constexpr int kTmem = kCols + 64 <= 128 ? 128 : 256;  // accumulator, two stages of scales
};

// `count` consecutive rows of A at column n of D: a warp writes 64 contiguous bytes per row.
// row_scale: A's in shared memory, or null.
template <typename OutT, int kCount>
__device__ __forceinline__ void store_column(const Fp4GemmArgs& g, const float* row_scale, const float* v, int m0,
                                             int n, float s_b, float bias) {
  float s_a[kCount];
#pragma unroll
  for (int e = 0; e < kCount; ++e)
    s_a[e] = m0 + e >= g.m ? 1.f : row_scale ? row_scale[m0 + e] : g.sa ? __ldg(g.sa + m0 + e) : 1.f;
  OutT* d = reinterpret_cast<OutT*>(g.d) + (int64_t)m0 * g.ldd + n;
#pragma unroll
  for (int e = 0; e < kCount; ++e)
    if (m0 + e < g.m) d[e * g.ldd] = Elt<OutT>::from_f(v[e] * s_b * s_a[e] + bias);
}

// quant_fp4 of this CTA's part of K of x, into the place of A's codes and scales, by the epilogue's
// warps; each CTA finds the maxima of whole rows for itself (a row of 3072 is 6 KB out of L2).
// Rows past the last stay as they are: they reach only their own columns of the accumulator.
// Loads go out in batches of four runs: a row at a time costs its latency, 1.1 us, per row.
template <typename T, bool kMx, typename S>
__device__ __forceinline__ void quantise_part(const Fp4GemmArgs& g, uint8_t* gbase, int kb0, int kb1) {
  constexpr int kThreads = 128, kBatch = 4, kRuns = kKElems / 16;  // runs of a stage
  const int t = threadIdx.x - (kRowsThreads - kThreads), w = t >> 5, lane = t & 31, runs = g.k / 16;
  const T* const x = reinterpret_cast<const T*>(g.x);
  float* const row_scale = reinterpret_cast<float*>(gbase + S::kRowScale) + w * 16;
  uint32_t top_row = 0;  // of row `lane`
  float rs_row = 0.f;
  if constexpr (!kMx) {
    uint32_t* const row_max = reinterpret_cast<uint32_t*>(gbase + S::kRowMax);
    const int share = g.m == 1 ? 4 : g.m == 2 ? 2 : 1;  // warps to a row
    for (int m = w / share; m < g.m; m += 4 / share) {
      uint32_t top = 0;
      for (int u0 = (w % share) * 32 + lane; u0 < runs; u0 += 32 * share * kBatch) {
        Run<T> run[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int u = u0 + i * 32 * share;
          if (u < runs)
            run[i].load(x + m * g.ldx + (int64_t)u * 16, g.x_align);
          else
            run[i].clear();
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) top = max(top, run[i].amax_bits());
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0) row_max[m * 4 + w % share] = top;
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (lane < g.m) {
      for (int i = 0; i < share; ++i) top_row = max(top_row, row_max[lane * 4 + i]);
      rs_row = fp4_row_scale(top_row);
      row_scale[lane] = top_row >= 0x7f800000u ? __int_as_float(0x7fffffff) : rs_row;
    }
  }
  const int part = (kb1 - kb0) * kRuns, all = g.m * part;
  for (int i0 = t; i0 - t < all; i0 += kThreads * kBatch) {
    Run<T> run[kBatch];
    int row[kBatch], at[kBatch];  // row (g.m: none) and run of this CTA's part
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      row[i] = min(i0 + i * kThreads, all) / max(part, 1);
      at[i] = i0 + i * kThreads - row[i] * part;
      if (row[i] < g.m && kb0 * kRuns + at[i] < runs)
        run[i].load(x + row[i] * g.ldx + (int64_t)(kb0 * kRuns + at[i]) * 16, g.x_align);
      else
        run[i].clear();
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (i0 - t + i * kThreads >= all) break;  // the same for all threads
      uint32_t top = run[i].amax_bits(), code;
      float rs = 0.f, rc = 0.f;
      bool bad = false;
      if constexpr (kMx) {
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      } else {
        const int from = min(row[i], g.m - 1);
        bad = __shfl_sync(0xffffffffu, top_row, from) >= 0x7f800000u;
        rs = __shfl_sync(0xffffffffu, rs_row, from);
        rc = __frcp_rn(rs);
      }
      const uint2 c = run_to_fp4<T, kMx>(run[i], top, bad, rs, rc, code);
      if (row[i] < g.m) {
        // 128-byte swizzle; scales: the tile's order (fp4.cuh), the row being one of the first 32
        const int stage = at[i] / kRuns, j = at[i] % kRuns, b = kMx ? j >> 1 : j;
        *reinterpret_cast<uint2*>(gbase + S::kOffA + stage * S::kA + row[i] * kKBytes +
                                  (((j >> 1) ^ (row[i] & 7)) << 4) + (j & 1) * 8) = c;
        if (!kMx || (j & 1) == 0)
          gbase[S::kOffSA + stage * S::F::kScale + (b >> 2) * kChunk + row[i] * 16 + (b & 3)] = (uint8_t)code;
      }
    }
  }
}

// kFused: A's rows come in 16 bits and are quantised here; K's parts fit into kAStages.
template <typename OutT, bool kMx, int kCols, bool kFused>
__global__ void __launch_bounds__(kRowsThreads, 1)
    fp4_gemm_rows_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                         const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb,
                         const Fp4GemmArgs args, const int split) {
  using S = RowsSmem<kMx, kCols, kFused>;
  using F = Fmt<kMx>;
  constexpr int kStages = S::kStages;
  static_assert(kStages >= 3, "ring too short");
  static_assert(!kFused || kCols == 16, "row scales for 16 rows");
  unsigned int* const fault = args.fault;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t base = (raw_base + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw_base);
  const uint32_t bars = base + S::kBars;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (kStages + s); };
  const uint32_t tfull = bars + 8u * (2 * kStages);
  const uint32_t tmem_slot = tfull + 8, a_ready = tfull + 16;

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int rank = split > 1 ? (int)cluster_rank() : 0;
  const int tn = (int)blockIdx.x / split, tm = (int)blockIdx.y;
  const int kblocks = (args.k + kKElems - 1) / kKElems;
  const int kb0 = kblocks * rank / split, kb1 = kblocks * (rank + 1) / split;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(tfull, 1);
    if constexpr (kFused) mbar_init(a_ready, 4);  // one arrival per quantising warp
    mbar_init_fence();
  }
  if (warp == 1) tmem_alloc(tmem_slot, S::kTmem);
  __syncthreads();
  if (split > 1) cluster_sync();  // every CTA of the cluster runs before any part is sent
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<uint32_t*>(gbase + (tmem_slot - base));
  auto load_b = [&](int stage, int kb) {
    mbar_expect_tx(full_bar(stage), S::kStage);
    tma_load_2d(base + S::kOffB + stage * S::kB, &map_b, kb * kKBytes, tn * 128, full_bar(stage));
    tma_load_3d(base + S::kOffSB + stage * F::kScale, &map_sb, 0, kb * F::kTiles, tn, full_bar(stage));
  };
  // a layer's weight streams in while the kernel before still quantises its input
  const int early = args.b_ready ? min(kStages, kb1 - kb0) : 0;
  if (warp == 0 && lane == 0)
    for (int s = 0; s < early; ++s) load_b(s, kb0 + s);
  pdl_wait();
  pdl_trigger();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (issued >= early) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, fault)) break;
          load_b(stage, kb);
        }
        if constexpr (!kFused) {
          tma_load_2d(base + S::kOffA + stage * S::kA, &map_a, kb * kKBytes, tm * kCols, full_bar(stage));
          tma_load_3d(base + S::kOffSA + stage * F::kScale, &map_sa, 0, kb * F::kTiles, tm, full_bar(stage));
        }
        ++issued;
        if (++stage == kStages) stage = 0, phase ^= 1u;
      }
      for (int j = max(0, issued - kStages); j < issued; ++j)
        mbar_wait(full_bar(j % kStages), (j / kStages) & 1, fault);
    }
  } else if (warp == 1) {
    const uint64_t bd = sw128_desc(base + S::kOffB), ad = sw128_desc(base + S::kOffA);
    const uint64_t sbd = scale_desc(base + S::kOffSB), sad = scale_desc(base + S::kOffSA);
    int stage = 0;
    uint32_t phase = 0;
    const bool ready = !kFused || __all_sync(0xffffffffu, mbar_wait(a_ready, 0, fault));
    for (int kb = kb0; kb < kb1 && ready; ++kb) {
      if (!__all_sync(0xffffffffu, mbar_wait(full_bar(stage), phase, fault))) break;
      tc_fence_after();
      if (elect_one()) {
        const int at = kFused ? kb - kb0 : stage;
        stage_products<false, kMx, 128, kCols, 1>(
            tmem, bd + stage * (S::kB >> 4), ad + at * (S::kA >> 4), sbd + stage * (F::kScale >> 4),
            sad + at * (F::kScale >> 4), tmem + kCols + ((kb - kb0) & 1) * 2 * F::kCols, steps_of(args.k, kb),
            kb == kb0);
        tc_commit(empty_bar(stage));
      }
      __syncwarp();
      if (++stage == kStages) stage = 0, phase ^= 1u;
    }
    if (elect_one()) tc_commit(tfull);  // also after a failed wait: everything issued has retired
    __syncwarp();
    mbar_wait(tfull, 0, fault);
  } else {
    // ---------------- epilogue: thread = row of B (tensor-memory lane), columns = rows of A
    const int q = warp & 3, nl = q * 32 + lane, n = tn * 128 + nl;
    const uint32_t t_row = tmem + ((uint32_t)(q * 32) << 16);
    const bool live = n < args.n;
    const float s_b = live && args.sb ? __ldg(args.sb + n) : 1.f;
    const float bias = live && args.bias ? Elt<OutT>::to_f(reinterpret_cast<const OutT*>(args.bias)[n]) : 0.f;
    const float* row_scale = nullptr;
    if constexpr (kFused) {
      quantise_part<OutT, kMx, S>(args, gbase, kb0, kb1);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(a_ready);
      if (!kMx) row_scale = reinterpret_cast<const float*>(gbase + S::kRowScale) + (warp - 2) * 16;
    }
    const bool ok = __all_sync(0xffffffffu, mbar_wait(tfull, 0, fault));
    tc_fence_after();
    // each CTA of the cluster adds up kCols / split of the columns (both powers of two)
    const int shift = 31 - __clz(kCols / split), share = 1 << shift;
    const uint32_t part = base + S::kOffPart + (uint32_t)(rank * share * 128 + nl) * 4;
#pragma unroll 1
    for (int c = 0; c < kCols && ok; c += 16) {
      uint32_t r[16];
      if (kb1 > kb0) {
        tmem_ld16(t_row + c, r);
        tmem_ld_wait(r);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) r[e] = 0;
      }
      if (split == 1) {
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = __uint_as_float(r[e]);
        if (live) store_column<OutT, 16>(args, row_scale, v, tm * kCols + c, n, s_b, bias);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int to = (c + e) >> shift, at = (c + e) & (share - 1);
          asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(part + at * 512, to)), "r"(r[e])
                       : "memory");
        }
      }
    }
    tc_fence_before();
    if (split > 1) {
      cluster_sync();  // every part has arrived, and nothing reaches another CTA any more
      const float* from = reinterpret_cast<const float*>(gbase + S::kOffPart) + nl;
      auto sums = [&](auto count, int c) {
        constexpr int kCount = decltype(count)::value;
        float v[kCount] = {};
        for (int r = 0; r < split; ++r)
#pragma unroll
          for (int e = 0; e < kCount; ++e) v[e] += from[((r << shift) + c + e) * 128];
        if (live) store_column<OutT, kCount>(args, row_scale, v, tm * kCols + rank * share + c, n, s_b, bias);
      };
      if (share >= 8)
        for (int c = 0; c < share; c += 8) sums(std::integral_constant<int, 8>{}, c);
      else
        for (int c = 0; c < share; c += 2) sums(std::integral_constant<int, 2>{}, c);
    }
  }
  __syncwarp();
  if (split > 1 && warp < 2) cluster_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_free(tmem, S::kTmem);
  }
}

// ------------------------------------------------------------------ host side
int make_code_map(CUtensorMap* map, const void* ptr, int64_t rows, int64_t kbytes, int64_t ld, int box_rows) {
  auto fn = tensor_map_encoder();
  if (!fn) return fail(JO_ERR_CUDA, "fp4_scaled_mm: cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {(cuuint64_t)kbytes, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {(cuuint32_t)kKBytes, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(JO_ERR_CUDA, "fp4_scaled_mm: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return JO_OK;
}
// Scale tiles [groups of 128 rows][tiles along K][512 bytes].
int make_scale_map(CUtensorMap* map, const void* ptr, int64_t groups, int64_t tiles_k, int box_tiles, int box_groups) {
  auto fn = tensor_map_encoder();
  if (!fn) return fail(JO_ERR_CUDA, "fp4_scaled_mm: cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[3] = {kChunk / 4, (cuuint64_t)tiles_k, (cuuint64_t)groups};
  cuuint64_t strides[2] = {kChunk, (cuuint64_t)tiles_k * kChunk};
  cuuint32_t box[3] = {kChunk / 4, (cuuint32_t)box_tiles, (cuuint32_t)box_groups};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(ptr), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(JO_ERR_CUDA, "fp4_scaled_mm: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return JO_OK;
}

// D [m, n], stored in boxes of 32 rows x 64 columns.
int make_out_map(CUtensorMap* map, const Fp4GemmArgs& g, bool bf16) {
  auto fn = tensor_map_encoder();
  if (!fn) return fail(JO_ERR_CUDA, "fp4_scaled_mm: cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {(cuuint64_t)g.n, (cuuint64_t)g.m};
  cuuint64_t strides[1] = {(cuuint64_t)g.ldd * 2};
  cuuint32_t box[2] = {64, 32};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, g.d, dims,
                        strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(JO_ERR_CUDA, "fp4_scaled_mm: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return JO_OK;
}

struct Operands {
  const void* a;
  const void* b;
  const void* block_a;
  const void* block_b;
  int64_t lda, ldb;
};

template <bool kMx>
int make_maps(CUtensorMap* maps, const Operands& o, const Fp4GemmArgs& g, int rows_a, int rows_b, int groups_b) {
  using F = Fmt<kMx>;
  const int64_t tk = fp4_tiles_k(g.k, kMx ? JO_FP4_MX : JO_FP4_NV);
  if (g.x == nullptr) {  // else A is not read
    if (int s = make_code_map(&maps[0], o.a, g.m, g.k / 2, o.lda, rows_a)) return s;
    if (int s = make_scale_map(&maps[2], o.block_a, cdiv(g.m, 128), tk, F::kTiles, 1)) return s;
  }
  if (int s = make_code_map(&maps[1], o.b, g.n, g.k / 2, o.ldb, rows_b)) return s;
  return make_scale_map(&maps[3], o.block_b, cdiv(g.n, 128), tk, F::kTiles, groups_b);
}

template <typename OutT, bool kMx>
int launch_pair(const Operands& o, Fp4GemmArgs g, cudaStream_t st, const DeviceInfo* di) {
  const char* op = "fp4_scaled_mm";
  using S = PairSmem<kMx>;
  auto kern = fp4_gemm_pair_kernel<OutT, kMx>;
  static std::atomic<uint64_t> reserved{0};
  if (int s = reserve_smem((const void*)kern, S::kBytes, reserved, di, op)) return s;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kPairThreads, 1, 1);
  cfg.dynamicSmemBytes = S::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // see launch_pdl
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  static std::atomic<int> resident[64];  // CTA pairs held at once, per device (0 = not asked yet)
  int pairs = resident[di->ordinal].load(std::memory_order_relaxed);
  if (!pairs) {
    cfg.gridDim = dim3(2, 1, 1);
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&pairs, (const void*)kern, &cfg) != cudaSuccess || pairs < 1) {
      cudaGetLastError();
      return fail(JO_ERR_CUDA, "%s: no resident CTA pair", op);
    }
    resident[di->ordinal].store(pairs, std::memory_order_relaxed);
  }
  g.tiles_m = (int)cdiv(g.m, kPairM);
  g.tiles_n = (int)cdiv(g.n, kPairN);
  if ((int64_t)g.tiles_m * g.tiles_n > INT32_MAX) return fail(JO_ERR_SHAPE, "%s: too many tiles", op);
  CUtensorMap maps[5];
  if (int s = make_maps<kMx>(maps, o, g, 128, 128, 2)) return s;
  if (int s = make_out_map(&maps[4], g, std::is_same<OutT, __nv_bfloat16>::value)) return s;
  const int tiles = g.tiles_m * g.tiles_n;
  cfg.gridDim = dim3(2 * (unsigned)(tiles < pairs ? tiles : pairs), 1, 1);
  cfg.numAttrs = 2;
  if (cudaError_t e = cudaLaunchKernelEx(&cfg, kern, maps[0], maps[1], maps[2], maps[3], maps[4], g))
    return launch_failed(e, op);
  return after_launch("fp4_gemm_pair_kernel");
}

// K in as many parts as still leave two stages each, until every SM has a CTA.
int rows_split(int64_t tiles, int64_t k, int sm_count) {
  const int64_t kblocks = cdiv(k, kKElems);
  int split = 1;
  while (split < kMaxSplit && tiles * split * 2 <= sm_count && kblocks >= split * 4) split *= 2;
  return split;
}

template <typename OutT, bool kMx, int kCols, bool kFused>
int launch_rows(const Operands& o, Fp4GemmArgs g, cudaStream_t st, const DeviceInfo* di) {
  const char* op = "fp4_scaled_mm";
  using S = RowsSmem<kMx, kCols, kFused>;
  auto kern = fp4_gemm_rows_kernel<OutT, kMx, kCols, kFused>;
  static std::atomic<uint64_t> reserved{0};
  if (int s = reserve_smem((const void*)kern, S::kBytes, reserved, di, op)) return s;
  g.tiles_m = (int)cdiv(g.m, kCols);
  g.tiles_n = (int)cdiv(g.n, 128);
  if (kCols < 128 && g.tiles_m > 1) return fail(JO_ERR_SHAPE, "%s: %d rows in a tile of %d", op, g.m, kCols);
  if (g.tiles_m > 65535 || (int64_t)g.tiles_n * kMaxSplit > INT32_MAX)
    return fail(JO_ERR_SHAPE, "%s: too many tiles", op);
  const int split = rows_split((int64_t)g.tiles_m * g.tiles_n, g.k, di->sm_count);
  CUtensorMap maps[4] = {};
  if (int s = make_maps<kMx>(maps, o, g, kCols, 128, 1)) return s;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(g.tiles_n * split), (unsigned)g.tiles_m, 1);
  cfg.blockDim = dim3(kRowsThreads, 1, 1);
  cfg.dynamicSmemBytes = S::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)split;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  if (cudaError_t e = cudaLaunchKernelEx(&cfg, kern, maps[0], maps[1], maps[2], maps[3], g, split))
    return launch_failed(e, op);
  return after_launch("fp4_gemm_rows_kernel");
}

template <typename OutT, bool kMx>
int dispatch(const Operands& o, const Fp4GemmArgs& g, cudaStream_t st, const DeviceInfo* di) {
  // CTA pairs where their 256 x 256 tiles occupy at least half of the SMs; below that the rows
  // kernel's 128 x 128 tiles take one round of the SMs, above it two. Pairs / rows, microseconds,
  // M x N x K, pair tiles of the 74 that the GPU holds: JO_FP4_NV 200 x 1024 x 1024 (4) 8.8 / 8.8;
  // 512 x 3072 x 3072 (24) 11.5 / 10.4; 768 x 3072 x 3072 (36) 11.8 / 10.5; 1024 x 2560 x 3072
  // (40) 12.1 / 19.8; 512 x 4864 x 1024 (38) 9.3 / 15.3; 1350 x 3072 x 3072 (72) 12.3 / 20.9.
  // JO_FP4_MX 768 x 3072 x 3072 9.0 / 9.3; 1024 x 2560 x 3072 9.5 / 17.4.
  const int64_t pair_tiles = cdiv(g.m, kPairM) * cdiv(g.n, kPairN);
  if (g.m > 128 && pair_tiles * 2 * 2 >= di->sm_count) return launch_pair<OutT, kMx>(o, g, st, di);
  if (g.x) return launch_rows<OutT, kMx, 16, true>(o, g, st, di);
  if (g.m <= 16) return launch_rows<OutT, kMx, 16, false>(o, g, st, di);
  if (g.m <= 32) return launch_rows<OutT, kMx, 32, false>(o, g, st, di);
  if (g.m <= 64) return launch_rows<OutT, kMx, 64, false>(o, g, st, di);
  return launch_rows<OutT, kMx, 128, false>(o, g, st, di);
}

}  // namespace
}  // namespace jo

namespace jo {
namespace {

int fp4_mm(const char* op, void* d, int64_t ldd, const Operands& o, const float* scale_a, const float* scale_b,
           const void* bias, int64_t m, int64_t n, int64_t k, int format, int out_dtype, bool b_ready,
           const void* x, int64_t ldx, cudaStream_t st) {
  const DeviceInfo* di;
  if (int s = device_info(&di)) return s;
  if (format != JO_FP4_NV && format != JO_FP4_MX)
    return fail(JO_ERR_INVALID, "%s: unknown 4-bit format %d", op, format);
  if (m < 0 || n < 0 || k < 0) return fail(JO_ERR_SHAPE, "%s: negative size", op);
  if (out_dtype != JO_BF16 && out_dtype != JO_F16) return fail(JO_ERR_DTYPE, "%s: out dtype must be bf16/fp16", op);
  if (m == 0 || n == 0) return JO_OK;
  if (k == 0 || k % 32) return fail(JO_ERR_SHAPE, "%s: K must be a positive multiple of 32", op);
  const int64_t most = INT32_MAX - 512;
  if (m > most || n > most || k > most) return fail(JO_ERR_SHAPE, "%s: size too large", op);
  if (!d || !o.a || !o.b || !o.block_a || !o.block_b) return fail(JO_ERR_INVALID, "%s: null operand", op);
  if (o.lda < k / 2 || o.ldb < k / 2 || ldd < n)
    return fail(JO_ERR_SHAPE, "%s: leading dimension smaller than the row", op);
  if (o.lda % 16 || o.ldb % 16 || n % 8 || ldd % 8)
    return fail(JO_ERR_ALIGN, "%s: lda and ldb must be multiples of 16 bytes, N and ldd of 8", op);
  if (!aligned16(d) || !aligned16(o.a) || !aligned16(o.b) || !aligned16(o.block_a) || !aligned16(o.block_b) ||
      (scale_b && !aligned16(scale_b)) || (bias && !aligned16(bias)))
    return fail(JO_ERR_ALIGN, "%s: operands must be 16-byte aligned", op);
  Fp4GemmArgs g{};
  g.d = d;
  g.ldd = ldd;
  g.sa = scale_a;
  g.sb = scale_b;
  g.bias = bias;
  g.m = (int)m;
  g.n = (int)n;
  g.k = (int)k;
  g.b_ready = b_ready;
  g.x = x;
  g.ldx = ldx;
  const uint64_t at = reinterpret_cast<uintptr_t>(x) | (uint64_t)(m > 1 ? ldx * 2 : 0);
  g.x_align = at % 32 == 0 ? 32 : at % 16 == 0 ? 16 : 2;
  g.fault = di->fault;
  const bool mx = format == JO_FP4_MX;
  if (out_dtype == JO_BF16)
    return mx ? dispatch<__nv_bfloat16, true>(o, g, st, di) : dispatch<__nv_bfloat16, false>(o, g, st, di);
  return mx ? dispatch<__half, true>(o, g, st, di) : dispatch<__half, false>(o, g, st, di);
}

// Whether the product's kernel quantises x itself: where each part of K fits beside the ring,
// and the runs of 16 that each of a CTA's 128 threads goes through are few: m K / 2048 over
// the parts of K, and for the maxima of whole rows (JO_FP4_NV) as many as a third of m K /
// 2048, once for every tile of the SM.  us per call (and on the GPU), one kernel / two:
//   JO_FP4_NV  9216 x 3072   1 row (1.2) 8.2 / 9.4 (6.7 / 7.8), 4 rows (4.8) 8.5 / 9.4 (8.3 / 7.7),
//                            8 rows (9.6) 10.5 / 9.3 (10.4 / 8.0)
//              12288 x 3072  2 rows (3.9) 8.9 / 9.2 (8.1 / 8.6), 4 rows (7.8) 10.7 / 9.3 (10.2 / 8.7)
//   JO_FP4_MX  9216 x 3072   1 row (0.8) 7.1 / 9.3 (5.8 / 7.8), 8 rows (6) 7.2 / 9.3 (6.9 / 8.0),
//                            16 rows (12) 8.6 / 9.4 (8.6 / 8.0)
//              28672 x 4096  2 rows (8) 16.1 / 18.5 (15.7 / 18.3), 4 rows (16) 18.7 / 18.6 (18.4 / 17.7)
constexpr int64_t kMostFused = 16;  // rows
bool quantises_itself(int64_t m, int64_t n, int64_t k, int format, int sm_count) {
  const bool mx = format == JO_FP4_MX;
  const int64_t tiles = cdiv(n, 128);
  const int split = rows_split(tiles, k, sm_count);
  if (cdiv(cdiv(k, kKElems), split) > (mx ? RowsSmem<true, 16, true>::kAStages : RowsSmem<false, 16, true>::kAStages))
    return false;
  const double runs = (double)(cdiv(tiles * split, sm_count) * m * k) / 2048.;
  return m <= kMostFused && (mx ? runs / split <= 8. : runs * (0.3 + 1. / split) <= 5.);
}

// fp4_linear's workspace: codes, block scales and row scales of x, each from 512 bytes on.
struct LinearWork {
  int64_t scales, rows, bytes;
};
LinearWork linear_work(int64_t m, int64_t k, int format) {
  LinearWork w;
  w.scales = cdiv(m * (k / 2), 512) * 512;
  w.rows = w.scales + jo_fp4_scale_bytes(m, k, format);
  w.bytes = w.rows + cdiv(4 * m, 512) * 512;
  return w;
}

}  // namespace
}  // namespace jo

using namespace jo;

extern "C" {

int jo_fp4_scaled_mm(void* d, int64_t ldd, const void* a, int64_t lda, const void* b, int64_t ldb,
                     const void* block_a, const void* block_b, const float* scale_a, const float* scale_b,
                     const void* bias, int64_t m, int64_t n, int64_t k, int format, int out_dtype, void* stream) {
  return fp4_mm("fp4_scaled_mm", d, ldd, Operands{a, b, block_a, block_b, lda, ldb}, scale_a, scale_b, bias, m, n, k,
                format, out_dtype, false, nullptr, 0, (cudaStream_t)stream);
}

int64_t jo_fp4_linear_workspace(int64_t m, int64_t k, int format) {
  if (m < 0 || m > INT32_MAX || k <= 0 || k % 32 || (m > 0 && k > fp4_longest_row(JO_BF16)) ||
      (format != JO_FP4_NV && format != JO_FP4_MX))
    return -1;
  return linear_work(m, k, format).bytes;
}

int jo_fp4_linear(void* d, int64_t ldd, const void* x, int64_t x_row_stride, const void* b, int64_t ldb,
                  const void* block_b, const float* scale_b, const void* bias, int64_t m, int64_t n, int64_t k,
                  int format, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* op = "fp4_linear";
  if (dtype != JO_BF16 && dtype != JO_F16) return fail(JO_ERR_DTYPE, "%s: x must be bf16 or fp16", op);
  if (m < 0 || n < 0) return fail(JO_ERR_SHAPE, "%s: negative size", op);
  const int64_t bytes = jo_fp4_linear_workspace(m, k, format);
  if (bytes < 0)
    return fail(JO_ERR_SHAPE, "%s: K must be a positive multiple of 32 and at most %lld, in a 4-bit format", op,
                (long long)fp4_longest_row(dtype));
  if (m == 0 || n == 0) return JO_OK;
  if (!workspace || !aligned16(workspace) || workspace_bytes < bytes)
    return fail(JO_ERR_INVALID, "%s: a 16-byte aligned workspace of %lld bytes is needed", op, (long long)bytes);
  const LinearWork w = linear_work(m, k, format);
  uint8_t* const q = (uint8_t*)workspace;
  float* const rows = format == JO_FP4_NV ? reinterpret_cast<float*>(q + w.rows) : nullptr;
  const DeviceInfo* di = nullptr;
  if (m <= kMostFused)
    if (int s = device_info(&di)) return s;
  if (di && quantises_itself(m, n, k, format, di->sm_count)) {
    if (!x) return fail(JO_ERR_INVALID, "%s: null operand", op);
    if (m > 1 && x_row_stride < k) return fail(JO_ERR_SHAPE, "%s: row stride smaller than the row", op);
    if (reinterpret_cast<uintptr_t>(x) % 2) return fail(JO_ERR_ALIGN, "%s: x must be aligned to its elements", op);
    return fp4_mm(op, d, ldd, Operands{q, b, q + w.scales, block_b, k / 2, ldb}, nullptr, scale_b, bias, m, n, k,
                  format, dtype, false, x, x_row_stride, (cudaStream_t)stream);
  }
  if (int s = jo_quant_fp4(q, k / 2, q + w.scales, rows, x, x_row_stride, m, k, format, dtype, stream)) return s;
  // the quantisation releases the product's launch only once everything before it is complete
  return fp4_mm(op, d, ldd, Operands{q, b, q + w.scales, block_b, k / 2, ldb}, rows, scale_b, bias, m, n, k, format,
                dtype, true, nullptr, 0, (cudaStream_t)stream);
}

}  // extern "C"
