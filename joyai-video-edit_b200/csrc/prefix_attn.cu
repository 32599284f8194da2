// Attention of a batch of requests over a prefix that all of them share and, per
// request, its own cache rows.
//
// Query i of request b (of its Lq, which are the last Lq of its own rows when causal)
// attends over the P prefix rows and over its request's own rows j < n(b, i):
//
//   n(b, i) = len[b], or, causal, min(len[b], len[b] - Lq + i + 1) (none when negative)
//   out = sum_j softmax_j(scale q.k_j) v_j,  lse = log sum_j exp(scale q.k_j)
//
// A query that sees no row at all gives 0 and -inf.  With the running maximum m and
// sum l of a row over its tiles of 128 keys, in powers of two,
//
//   p_j = 2^(s_j c - m),  c = scale log2(e),  l = sum p_j,  O = sum p_j v_j,
//   out = O / l,  log2-sum-exp = m + log2(l),
//
// m is raised (and O and l scaled down) only when a tile's maximum exceeds it by more
// than 8: until then p <= 2^8, which neither format nor the fp32 sums mind, and the
// quotient O / l does not depend on m.  Parts over disjoint keys are joined by their
// log2-sum-exps.
//
// Rows and keys.  All queries that read one k/v head can share its keys whatever request
// they belong to: a row of a tensor-core tile is any (request, query, q head of the k/v
// head's group), up to 256 of them to a work unit, and the unit's keys are a walk over tiles
// of 128: first the prefix's, read once for all of the unit's rows, then the own rows of
// each request that has a row in the unit, which only that request's rows see (for the
// others their p is 0).  For single tokens the tensor cores have time for that: a tile costs
// its bytes.  Row tiles run across requests or stay within one, whichever costs fewer tiles
// (plan_attention).  Where the units do not fill the GPU evenly, the last ones' walks are
// split and joined: by a second kernel, or, where all units are parts and few rows are to be
// joined, by the CTAs of a cluster from each other's shared memory (one launch and no
// workspace: one token over 777 rows 11.3 -> 8.3 us per call, 8.2 -> 7.2 on the GPU).
//
// One CTA per SM goes through its units with two streams, each with its own S, P and O in
// tensor memory, so that one stream's softmax runs while the other's products do:
//   a unit of more than 128 rows: the streams take its two halves, and share every K and
//   V tile (64 KB per tile of 128 keys would otherwise exceed what an SM can take in);
//   a unit of up to 128 rows (single tokens): the streams take alternate key tiles of the
//   same rows and are joined at the end.
// Warps 0-3 and 4-7: softmax of stream 0 and 1, one row per thread (tensor-memory lane):
//   S from tensor memory, the running maximum and sum, P back in place of S in two halves
//   (the product may start on the first), O rescaled in place; Q and the results.
// Warp 8: TMA producer of K and V tiles of 128 rows (128-byte swizzle) into one ring, in
//   the order of their first use; it runs ahead across units.
// Warp 9: tcgen05.mma issuer: S = Q K^T (both operands in shared memory), O += P V with P
//   from tensor memory and V as it lies ([keys, D], the MN-major operand).
//
// P is rounded to q's 16-bit type for the tensor cores, whose errors average out over the keys; l
// sums the unrounded p.  bf16: a relative 2^-8 at most, as the output's own rounding.  fp16:
// 2^-11, but below 2^-14 an absolute 2^-25, and p under that vanishes, which does not
// average out (43200 keys 26 bits below one more would lose their 6e-4 of the weight).  So
// fp16 has p = 2^(s_j c - m + 7): at most 2^15 with m raised as above (the format ends at
// 65504), and n keys lose less than n 2^-32 of a weight whose sum is at least 1.  l carries
// the same 2^7, and the log-sum-exp takes it back.
//
// Bound and measured (B200; us per call, calls in a row).  Many queries: the chain of one
// stream, S -> softmax -> P V -> S, whose softmax (S in 300 cycles, maximum 150-300,
// exponentials 1300 at 16 per clock and SM, P 150) is longer than the other stream's products
// (1024): 2 x 900 queries x 24 heads of 128 over 43200 + 900 rows 890 us = 1.08 PFLOP/s (1050
// us once the power cap lowers the clock), tensor cores busy 57 %.  Single tokens: bytes, and
// the start and end of the one unit that each SM has: 32 tokens x 8 k/v heads over 10800
// shared and 512 own rows 32 us (the first tile arrives 5 us after the launch, the tiles take
// 15, storing and joining the parts 8), one token over 777 rows 7.2 us.
//
// Tried and slower, same 2 x 900 queries: a quarter / half of the exponentials as a polynomial
// on the FMA units 943 / 1056 us (938 without), two threads per row and 16 softmax warps 1021
// (928), one tile of 128 rows per CTA and two CTAs per SM 1535; spinning instead of suspended
// barrier waits and a longer ring for single tokens changed nothing.
#include "quant.cuh"
#include "tcgen05.cuh"

namespace jo {
namespace {

constexpr int kTileRows = 128;           // rows per stream (UMMA M)
constexpr int kUnitRows = 2 * kTileRows;  // rows per unit at most
constexpr int kTileKeys = 128;           // keys per tile (UMMA N of S, K of P V)
constexpr int kSoftmaxThreads = 256;
constexpr int kAttnThreads = 384;  // two softmax warpgroups; producer, issuer and two idle warps
// The launch gives each of the 384 threads 168 registers, 64,512 in all; the softmax threads
// hold a row of S (128 values) and take 224 each, the others keep 56: 64,512.
constexpr int kSoftmaxRegs = 224, kOtherRegs = 56;
constexpr int kColO = 256;  // tensor memory: S / P of the streams at 0 and 128, O at 256 and 384
constexpr float kRaise = 8.f;
template <typename T>
constexpr float kBias = std::is_same<T, __half>::value ? 7.f : 0.f;  // of p's exponent
constexpr int kMaxCluster = 8;  // parts that a cluster joins at most (the portable cluster size)

// From a CTA of the cluster (cluster address).
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float r;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(r) : "r"(addr) : "memory");
  return r;
}
__device__ __forceinline__ void ld_cluster2(uint32_t addr, float* v) {
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(addr) : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// n / d for 0 <= n < 2^31 by a multiplication: with s = ceil(log2 d) and m =
// ceil(2^(31+s) / d) < 2^32, the error m d - 2^(31+s) < d <= 2^s keeps floor(n m / 2^(31+s))
// exact.  A unit's place takes half a dozen divisions in a row, each some 200 cycles otherwise.
struct FastDiv {
  uint32_t mul = 1u << 31, shift = 31;
  FastDiv() = default;
  explicit FastDiv(int64_t d) {
    int s = 0;
    while (((int64_t)1 << s) < d) ++s;
    shift = 31 + s;
    mul = (uint32_t)((((uint64_t)1 << shift) + (uint64_t)d - 1) / (uint64_t)d);
  }
  __device__ __forceinline__ int operator()(int n) const { return (int)(((uint64_t)(uint32_t)n * mul) >> shift); }
};

struct AttnArgs {
  void* out;
  float* lse;
  const void* q;
  int64_t q_b, q_t, q_h;  // element strides
  const int32_t* lens;
  int prefix;
  int batch, lq, heads, group, own;  // heads: of k and v; group: q heads per k/v head; own: rows of the own caches
  int causal;
  float scale_log2;
  // plan: items 0..items-1 are the row tiles (of `tile_rows` rows) of `groups` groups (k/v
  // heads, or within_request: (head, request) pairs), every group's last tile after all
  // others; the walks of those from `whole` on are split in `splits`
  int within_request;
  int tile_rows, groups, row_tiles;
  int items, whole, splits;
  int units;   // whole + (items - whole) * splits
  int rows;    // queries per k/v head
  // by lq * group, group, batch, row_tiles - 1, the number of full and of last row tiles that are
  // split, and splits
  FastDiv by_request, by_group, by_batch, by_full, by_tail, by_last, by_splits;
  float* part_o;        // [slots, D]
  float* part_lse;
  unsigned int* fault;
};

// One work unit: rows [row0, row0 + rows) of k/v head h (row: (b * Lq + i) * G + g), which
// belong to requests b0..b1, and tiles [first, last) of its walk.
struct Unit {
  int h, row0, rows, b0, b1;
  int first, last;
  int64_t slot;  // partial slot of row0 (-1: final output)
};

__device__ __forceinline__ int own_visible(const AttnArgs& a, int len, int i) {
  return a.causal ? min(len, max(0, len - a.lq + i + 1)) : len;
}
__device__ __forceinline__ int own_len(const AttnArgs& a, int b) { return min(max(__ldg(a.lens + b), 0), a.own); }
__device__ __forceinline__ int prefix_tiles(const AttnArgs& a) { return (a.prefix + kTileKeys - 1) / kTileKeys; }
// Tiles of request b's own rows that the unit's rows see: its last row there sees the most.
__device__ __forceinline__ int own_tiles(const AttnArgs& a, const Unit& u, int b) {
  const int per_request = a.lq * a.group;
  const int last = min(u.row0 + u.rows, (b + 1) * per_request) - 1 - b * per_request;
  return (own_visible(a, own_len(a, b), a.by_group(last)) + kTileKeys - 1) / kTileKeys;
}

// Group and row tile of an item.
__device__ __forceinline__ void tile_of(const AttnArgs& a, int item, int& grp, int& t) {
  const int full = a.groups * (a.row_tiles - 1);
  if (item < full) {
    grp = a.by_full(item);
    t = item - grp * (a.row_tiles - 1);
  } else {
    grp = item - full;
    t = a.row_tiles - 1;
  }
}

// Work unit `index`; by a converged warp.  kCluster: a cluster's CTAs take an item's parts.
template <bool kCluster>
__device__ __forceinline__ Unit unit_of(const AttnArgs& a, int index) {
  Unit u;
  const int per_request = a.lq * a.group, lane = threadIdx.x & 31;
  int piece = 0, pieces = 1, item = index, grp, t;
  if (kCluster) {
    pieces = a.splits;
    item = a.by_splits(index);
    piece = index - item * pieces;
  } else if (index >= a.whole) {
    // the parts of full row tiles first, then those of the groups' last tiles
    const int full = a.groups * (a.row_tiles - 1), cut = max(a.whole, full);
    const int j = index - a.whole, tail = cut - a.whole, last = j - tail * a.splits;
    if (last < 0) {
      piece = a.by_tail(j);
      item = a.whole + j - piece * tail;
    } else {
      piece = a.by_last(last);
      item = cut + last - piece * (a.items - cut);
    }
    pieces = a.splits;
  }
  tile_of(a, item, grp, t);
  if (a.within_request) {
    u.h = a.by_batch(grp);
    u.b0 = u.b1 = grp - u.h * a.batch;
    u.row0 = u.b0 * per_request + t * a.tile_rows;
    u.rows = min(a.tile_rows, per_request - t * a.tile_rows);
  } else {
    u.h = grp;
    u.row0 = t * a.tile_rows;
    u.rows = min(a.tile_rows, a.rows - u.row0);
    u.b0 = a.by_request(u.row0);
    u.b1 = a.by_request(u.row0 + u.rows - 1);
  }
  u.slot = !kCluster && pieces > 1 ? ((int64_t)(item - a.whole) * pieces + piece) * a.tile_rows : -1;
  int own = 0;
  if (a.own > 0)
    for (int b = u.b0 + lane; b <= u.b1; b += 32) own += own_tiles(a, u, b);
  const int tiles = prefix_tiles(a) + __reduce_add_sync(0xffffffffu, own);
  u.first = pieces > 1 ? a.by_splits(tiles * piece) : 0;
  u.last = pieces > 1 ? a.by_splits(tiles * (piece + 1)) : tiles;
  return u;
}

// A place in a unit's walk: tile t of the prefix (b < 0) or of request b's own rows.
struct Walk {
  int b, t, count;  // count: tiles of this part of the walk
  // place `at`; by a converged warp
  __device__ __forceinline__ Walk(const AttnArgs& a, const Unit& u, int at) {
    b = -1;
    t = at;
    count = prefix_tiles(a);
    if (at < count) return;
    at -= count;
    const int lane = threadIdx.x & 31;
    for (int first = u.b0; first <= u.b1; first += 32) {
      const int mine = first + lane <= u.b1 ? own_tiles(a, u, first + lane) : 0;
      int upto = mine;  // inclusive sum over the lanes
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, upto > at);
      if (past) {
        const int l = __ffs(past) - 1;
        b = first + l;
        count = __shfl_sync(0xffffffffu, mine, l);
        t = at - (__shfl_sync(0xffffffffu, upto, l) - count);
        return;
      }
      at -= __shfl_sync(0xffffffffu, upto, 31);
    }
    b = u.b1 + 1;  // the end
    t = count = 0;
  }
  __device__ __forceinline__ void next(const AttnArgs& a, const Unit& u) {
    if (++t < count) return;
    t = 0;
    b = b < 0 ? u.b0 : b + 1;
    for (; b <= u.b1; ++b)
      if ((count = a.own > 0 ? own_tiles(a, u, b) : 0) > 0) return;
  }
};

template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  return pack_bf16x2(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
  return pack_f16x2(lo, hi);
}

// kAlone: every unit has at most 128 rows, so one Q tile does, and the other's place is one
// more of the ring's: such units hold four tiles at work (two streams' K and V) and are bound
// by the bytes that are under way beside them.
template <int D, bool kAlone>
struct AttnSmem {
  static constexpr int kTile = kTileKeys * D * 2;  // bytes of a K, V or Q tile
  static constexpr int kRing = (D == 64 ? 11 : 5) + kAlone;
  static constexpr int kQ = 0;
  static constexpr int kKV = (kAlone ? 1 : 2) * kTile;
  static constexpr int kBars = kKV + kRing * kTile;
  static constexpr int kGuard = kBars + 320;  // first non-finite value row of a tile, per warp
  static constexpr int kBytes = kGuard + 64 + 1024 /*align*/;
};

// The ring's order of loads for n tiles, which is the order of their first use.
//   shared by both streams:  K0 V0 K1 V1 ...
//   alternate tiles:         K0 K1 V0 K2 V1 K3 ... V(n-2) V(n-1)
__device__ __forceinline__ int v_index(bool alternate, int tile, int n) {
  return alternate ? (tile == n - 1 ? 2 * n - 1 : 2 * tile + 2) : 2 * tile + 1;
}
// A place in the ring: slot, and the parity of its full barrier.
template <int kRing>
struct Ring {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void advance(int by) {  // by <= kRing
    slot += by;
    if (slot >= kRing) {
      slot -= kRing;
      phase ^= 1u;
    }
  }
};
// Whether load `idx` is a V tile.
__device__ __forceinline__ bool value_at(bool alternate, int idx, int n) {
  if (!alternate) return idx & 1;
  return idx == 2 * n - 1 || (idx >= 2 && !(idx & 1));
}

// 16-bit operands, fp32 accumulator, M = 128.
template <typename T>
constexpr uint32_t attn_idesc(int n, bool b_mn_major) {
  const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kTileRows >> 4) << 24);
}

__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// Where a row's result goes, and its log-sum-exp there.
template <typename T, int D>
struct RowOut {
  T* out = nullptr;
  float* part = nullptr;
  __device__ __forceinline__ RowOut(const AttnArgs& a, const Unit& u, int r, bool live, bool lse, float m, float l) {
    if (!live) return;
    const float lse2 = l == 0.f ? -INFINITY : m + __log2f(l);
    if (u.slot >= 0) {
      part = a.part_o + (u.slot + r) * D;
      if (lse) a.part_lse[u.slot + r] = lse2;
    } else {
      const int per_request = a.lq * a.group, row = u.row0 + r;
      const int b = a.by_request(row), in = row - b * per_request, i = a.by_group(in), g = in - i * a.group;
      const int64_t hq = (int64_t)a.heads * a.group, h = (int64_t)u.h * a.group + g;
      out = reinterpret_cast<T*>(a.out) + (((int64_t)b * a.lq + i) * hq + h) * D;
      if (lse) a.lse[(b * hq + h) * a.lq + i] = lse2 * 0.6931471805599453f;
    }
  }
  __device__ __forceinline__ void store32(int c, const float* f) const {
    if (part != nullptr) {
#pragma unroll
      for (int e = 0; e < 32; e += 8) st_global32(part + c + e, Elt<float>::pack(f + e), Elt<float>::pack(f + e + 4));
    } else if (out != nullptr) {
#pragma unroll
      for (int e = 0; e < 32; e += 16) st_global32(out + c + e, Elt<T>::pack(f + e), Elt<T>::pack(f + e + 8));
    }
  }
};

// Result of a row (of the batch) of k/v head h, whose parts' results (weighted, o: elements
// lane * D/32 on) add up to o and their weights, relative to 2^top, to sum; by a warp.
template <typename T, int D>
__device__ __forceinline__ void store_joined(const AttnArgs& a, int h, int row, const float* o, float sum, float top) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31, per_request = a.lq * a.group;
  const int64_t hq = (int64_t)a.heads * a.group;
  const int b = a.by_request(row), in = row - b * per_request, i = a.by_group(in), g = in - i * a.group;
  const int64_t hh = (int64_t)h * a.group + g;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* const at = reinterpret_cast<T*>(a.out) + (((int64_t)b * a.lq + i) * hq + hh) * D + lane * E;
  uint32_t* const out = reinterpret_cast<uint32_t*>(at);
#pragma unroll
  for (int e = 0; e < E; e += 2) out[e / 2] = pack16<T>(o[e] * inv, o[e + 1] * inv);
  if (lane == 0)
    a.lse[(b * hq + hh) * a.lq + i] = sum == 0.f ? -INFINITY : (top + __log2f(sum)) * 0.6931471805599453f;
}

// kCluster: every unit is a part of a walk, each CTA has one, and a cluster's CTAs join
// theirs through distributed shared memory.
template <typename T, int D, bool kAlone, bool kCluster>
__global__ void __launch_bounds__(kAttnThreads, 1)
    prefix_attn_kernel(const __grid_constant__ CUtensorMap map_kp, const __grid_constant__ CUtensorMap map_vp,
                       const __grid_constant__ CUtensorMap map_ko, const __grid_constant__ CUtensorMap map_vo,
                       const AttnArgs a) {
  static_assert(kAlone || !kCluster, "the parts of a cluster have at most 128 rows");
  using S = AttnSmem<D, kAlone>;
  constexpr int kRing = S::kRing;
  constexpr int kBox = kTileKeys * 128;  // bytes of one 64-element-wide box
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const uint32_t bars = base + S::kBars;
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (kRing + s); };
  const uint32_t q_full = bars + 8u * (2 * kRing);
  auto s_full = [&](int s) { return q_full + 8u + 8u * s; };
  auto p_full = [&](int s, int half) { return q_full + 24u + 16u * half + 8u * s; };
  auto o_full = [&](int s) { return q_full + 56u + 8u * s; };
  const uint32_t done = q_full + 72u, tmem_slot = q_full + 80u;
  auto guarded_by_0 = [&](int i) { return q_full + 88u + 8u * i; };
  const int warp = warp_index(), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kRing; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(q_full, kSoftmaxThreads / 32);
    mbar_init(done, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(s_full(s), 1);
      mbar_init(p_full(s, 0), kTileRows / 32);  // one arrival per warp
      mbar_init(p_full(s, 1), kTileRows / 32);
      mbar_init(o_full(s), 1);
      mbar_init(guarded_by_0(s), kTileRows / 32);
    }
    mbar_init_fence();
  }
  if (warp == 9) tmem_alloc(tmem_slot, 512);
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<uint32_t*>(gbase + (tmem_slot - base));
  pdl_wait();  // lens, q, k and v may be the previous kernel's
  pdl_trigger();

  // kCluster: this CTA's part, in place of the K and V that it is done with; rows are padded by
  // 16 bytes, so that the threads of a warp, a row each, store to different banks
  constexpr int kPartRow = D + 4;
  static_assert(kTileRows * (kPartRow + 1) * 4 <= kRing * S::kTile, "a part fits into the ring");
  float* const part = reinterpret_cast<float*>(gbase + S::kKV);
  float* const part_lse = part + kTileRows * kPartRow;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 8) {
      // ---------------- TMA producer (lane 0; the warp finds the units together)
      int at = 0;  // loads so far
      bool ok = true, first_unit = true;
      for (int unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
        const Unit u = unit_of<kCluster>(a, unit);
        const int n = u.last - u.first;
        if (n == 0) continue;
        const bool alternate = kAlone || u.rows <= kTileRows;
        Walk wk(a, u, u.first), wv(wk);  // of K, of V
        // The first unit's Q is asked for before any K and V: behind a ring's worth of them on
        // every SM (24 MB) it would take 4 us.
        if (first_unit) asm volatile("bar.sync 5, 288;" ::: "memory");
        first_unit = false;
        for (int j = 0; j < 2 * n && lane == 0 && ok; ++j, ++at) {
          const int slot = at % kRing;
          if (!(ok = mbar_wait(empty(slot), ((at / kRing) & 1) ^ 1u, a.fault))) break;
          auto load = [&](const CUtensorMap* prefix, const CUtensorMap* own, Walk& w) {
            mbar_expect_tx(full(slot), S::kTile);
#pragma unroll
            for (int x = 0; x < D; x += 64)
              tma_load_4d(base + S::kKV + slot * S::kTile + (x / 64) * kBox, w.b < 0 ? prefix : own, x, u.h,
                          w.t * kTileKeys, max(w.b, 0), full(slot));
            w.next(a, u);
          };
          if (value_at(alternate, j, n))
            load(&map_vp, &map_vo, wv);
          else
            load(&map_kp, &map_ko, wk);
        }
        __syncwarp();
      }
      // every copy issued has landed before the CTA may exit
      if (lane == 0)
        for (int j = max(0, at - kRing); j < at; ++j) mbar_wait(full(j % kRing), (j / kRing) & 1, a.fault);
    } else if (warp == 9) {
      // ---------------- MMA issuer: the warp stays converged and elects one thread per step
      constexpr uint32_t idesc_s = attn_idesc<T>(kTileKeys, false), idesc_o = attn_idesc<T>(D, true);
      const uint64_t qd0 = sw128_desc(base + S::kQ), kd0 = sw128_desc(base + S::kKV);
      const uint64_t vd0 = sw128_desc_mn(base + S::kKV, kBox);
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t phase) {
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar, phase, a.fault));
        tc_fence_after();
      };
      Ring<kRing> k, v;  // the next K and V tiles
      uint32_t p_phase[2] = {0, 0}, q_phase = 0;
      // S of stream s; `last`: no other stream uses the K tile
      auto products_s = [&](int s, const Ring<kRing>& at, bool alternate, bool last) {
        if (ok && elect_one()) {
          const uint64_t kd = kd0 + at.slot * (S::kTile >> 4), qd = qd0 + (alternate ? 0 : s * (S::kTile >> 4));
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const int off = ((kk / 4) * kBox + (kk % 4) * 32) >> 4;
            tc_mma_f16_ss(tmem + s * kTileKeys, qd + off, kd + off, idesc_s, kk != 0);
          }
          tc_commit(s_full(s));
          if (last) tc_commit(empty(at.slot));
        }
        __syncwarp();
      };
      // O of stream s
      auto products_o = [&](int s, const Ring<kRing>& at, bool first, bool last, bool end) {
        const uint64_t vd = vd0 + at.slot * (S::kTile >> 4);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          wait(p_full(s, half), p_phase[s]);
          if (ok && elect_one()) {
#pragma unroll
            for (int kk = 4 * half; kk < 4 * half + 4; ++kk)
              tc_mma_f16_ts(tmem + kColO + s * kTileKeys, tmem + s * kTileKeys + kk * 8, vd + kk * (2048 >> 4), idesc_o,
                            !first || kk != 0);
            if (half == 1) {
              if (last) tc_commit(empty(at.slot));
              if (end) tc_commit(o_full(s));
            }
          }
          __syncwarp();
        }
        p_phase[s] ^= 1u;
      };
      for (int unit = blockIdx.x; unit < a.units && ok; unit += gridDim.x) {
        const Unit u = unit_of<kCluster>(a, unit);
        const int n = u.last - u.first;
        if (n == 0) continue;
        wait(q_full, q_phase);
        q_phase ^= 1u;
        if (!kAlone && u.rows > kTileRows) {
          // both streams use every tile: K0 V0 K1 V1 ...
          v = k;
          v.advance(1);
          wait(full(k.slot), k.phase);
          products_s(0, k, false, false);
          products_s(1, k, false, true);
          for (int t = 0; t < n && ok; ++t) {
            const bool end = t == n - 1;
            k.advance(2);
            wait(full(v.slot), v.phase);
            products_o(0, v, t == 0, false, end);
            if (!end) {
              wait(full(k.slot), k.phase);
              products_s(0, k, false, false);
            }
            products_o(1, v, t == 0, true, end);
            if (!end) products_s(1, k, false, true);
            v.advance(2);
          }
        } else {
          // alternate tiles: every load is used once, in the order of the loads
          for (int s = 0; s < 2 && s < n; ++s) {
            wait(full(k.slot), k.phase);
            if (s == 0)
              products_s(0, k, true, true);
            else
              products_s(1, k, true, true);
            k.advance(1);
          }
          for (int t = 0; t < n && ok; t += 2) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              if (t + s >= n) continue;
              wait(full(k.slot), k.phase);
              products_o(s, k, t == 0, true, t + s + 2 >= n);
              k.advance(1);
              if (t + s + 2 < n) {
                wait(full(k.slot), k.phase);
                products_s(s, k, true, true);
                k.advance(1);
              }
            }
          }
        }
      }
      // tensor memory is freed below: everything issued has retired, also after a failed wait
      if (elect_one()) tc_commit(done);
      __syncwarp();
      mbar_wait(done, 0, a.fault);
    }
    if constexpr (kCluster) {
      __syncwarp();
      cluster_sync();
      cluster_sync();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ---------------- softmax: stream s, thread r owns a row (tensor-memory lane r)
    const int s = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + s * kTileKeys, t_o = tmem + lanes + kColO + s * kTileKeys;
    const int per_request = a.lq * a.group;
    bool ok = true;
    auto wait = [&](uint32_t bar, int phase) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar, phase & 1, a.fault));
      return ok;
    };
    auto arrive_warp = [&](uint32_t bar) {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    bool first_unit = true;
    int part_h = 0, part_row0 = 0, part_rows = 0;  // kCluster: of the one unit
    int count = 0, at = 0, o_count[2] = {0, 0};
    int guards = 0, shared_guards = 0;  // guarded tiles so far: a stream's own, and those that both use
    for (int unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
      const Unit u = unit_of<kCluster>(a, unit);
      const int n = u.last - u.first;
      const bool alternate = kAlone || u.rows <= kTileRows;
      const int row = alternate ? r : s * kTileRows + r;  // of the unit
      const bool live = row < u.rows;
      if constexpr (kCluster) part_h = u.h, part_row0 = u.row0, part_rows = u.rows;
      if (n == 0) {  // nothing to see: an empty part
        if constexpr (kCluster) {
          if (s == 0) {
            part_lse[r] = -INFINITY;
            for (int c = 0; c < D; ++c) part[r * kPartRow + c] = 0.f;
          }
        } else if (!alternate || s == 0) {
          const RowOut<T, D> dst(a, u, row, live, true, 0.f, 0.f);
          const float zero[32] = {};
          for (int c = 0; c < D; c += 32) dst.store32(c, zero);
        }
        continue;
      }
      // this row's request, query and head
      const int flat = u.row0 + min(row, u.rows - 1), my_b = a.by_request(flat);
      const int in = flat - my_b * per_request, my_i = a.by_group(in), my_g = in - my_i * a.group;
      {
        // Q: a thread loads its row (of a row that both streams use, one half), 32 bytes at a
        // time, all of it before the streams meet; 128-byte swizzle; rows past the last are zero
        constexpr int kVecs = D / 16;
        const T* q = reinterpret_cast<const T*>(a.q) + my_b * a.q_b + my_i * a.q_t + (int64_t)(u.h * a.group + my_g) * a.q_h;
        const int first = alternate ? s * (kVecs / 2) : 0, last = alternate ? first + kVecs / 2 : kVecs;
        uint4 v[kVecs][2];
#pragma unroll
        for (int c = 0; c < kVecs; ++c) {
          v[c][0] = v[c][1] = make_uint4(0, 0, 0, 0);
          if (live && c >= first && c < last) {
            v[c][0] = ld_stream(q + c * 16);
            v[c][1] = ld_stream(q + c * 16 + 8);
          }
        }
        if (first_unit) asm volatile("bar.arrive 5, 288;" ::: "memory");  // Q is on its way: K and V may follow
        first_unit = false;
        softmax_sync();  // both streams are done with the last unit's Q and O
        uint8_t* const dst = gbase + S::kQ + (alternate ? 0 : s * S::kTile) + r * 128;
#pragma unroll
        for (int c = 0; c < kVecs; ++c)
          if (c >= first && c < last) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int g = 2 * c + e;  // 16-byte vector of the row
              *reinterpret_cast<uint4*>(dst + (g / 8) * kBox + (((g ^ r) & 7) << 4)) = v[c][e];
            }
          }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        arrive_warp(q_full);
      }
      const int visible = a.own > 0 ? own_visible(a, own_len(a, my_b), my_i) : 0;  // own rows that this row sees
      const bool warp_live = (alternate ? 0 : s * kTileRows) + ((warp & 3) << 5) < u.rows;
      const int steps = alternate ? (n + 1 - s) / 2 : n;
      // of a unit within one request: own rows that all of its rows see
      const int seen_by_all =
          a.own > 0 ? own_visible(a, own_len(a, u.b0), a.by_group(u.row0 - u.b0 * per_request)) : 0;
      bool poisoned = false;
      Walk w(a, u, u.first);
      if (alternate && s == 1) w.next(a, u);
      float m = -INFINITY, l = 0.f;
      for (int t = 0; t < steps; ++t, ++count) {
        const bool own = w.b >= 0;
        const int key0 = w.t * kTileKeys;
        const int limit = min(kTileKeys, (own ? (my_b == w.b ? visible : 0) : a.prefix) - key0);
        wait(s_full(s), count);
        tc_fence_after();
        // Value rows that not every row here sees must not reach the others' products, where p is 0
        // but 0 * inf is not: cache rows past the request's length, which hold anything, and rows
        // with an infinity or a NaN where requests or causal limits differ.  They are zeroed (a tile
        // that both streams use: by stream 0, whose product comes first); a row that does see such a
        // value gives NaN.  Every other tile ends before seen_by_all, which is at most the length.
        if (own && (u.b0 != u.b1 || key0 + kTileKeys > seen_by_all)) {
          const int len = own_len(a, w.b);
          const int turn = alternate ? guards & 1 : shared_guards & 1;
          int* const first_bad = reinterpret_cast<int*>(gbase + S::kGuard) + turn * 8 + (alternate ? s * 4 : 0);
          if (alternate || s == 0) {
            const int idx = at + v_index(alternate, alternate ? 2 * t + s : t, n), slot = idx % kRing;
            wait(full(slot), idx / kRing);
            uint8_t* const vrow = gbase + S::kKV + slot * S::kTile + r * 128;
            bool zero = ok && key0 + r >= len, bad = false;
            if (ok && !zero) {
              uint32_t mag = 0;
#pragma unroll
              for (int c = 0; c < D / 8; ++c) {
                const uint4 x = *reinterpret_cast<const uint4*>(vrow + (c / 8) * kBox + (((c ^ r) & 7) << 4));
                mag = absmax16x2<T>(absmax16x2<T>(absmax16x2<T>(absmax16x2<T>(mag, x.x), x.y), x.z), x.w);
              }
              zero = bad = !isfinite(bits16_to_f<T>(amax16_bits(mag)));
            }
            if (zero) {
#pragma unroll
              for (int c = 0; c < D / 8; ++c)
                *reinterpret_cast<uint4*>(vrow + (c / 8) * kBox + (((c ^ r) & 7) << 4)) = make_uint4(0, 0, 0, 0);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            const int low = __reduce_min_sync(0xffffffffu, bad ? r : kTileKeys);
            if (lane == 0) first_bad[warp & 3] = low;
          }
          // Stream 1 takes what stream 0 found in a tile that both use.  Stream 0 goes on without
          // waiting for it and may be one such tile ahead, not two: S(t + 2) of stream 0 is issued
          // after O += P V of stream 1's tile t, whose P comes after this.  So two barriers in turn
          // do, and waits that are bounded as all others.
          if (alternate) {
            if (s == 0)
              asm volatile("bar.sync 2, 128;" ::: "memory");
            else
              asm volatile("bar.sync 3, 128;" ::: "memory");
            ++guards;
          } else {
            if (s == 0) {
              arrive_warp(guarded_by_0(turn));
              asm volatile("bar.sync 2, 128;" ::: "memory");
            } else {
              wait(guarded_by_0(turn), shared_guards >> 1);
            }
            ++shared_guards;
          }
          const int low = min(min(first_bad[0], first_bad[1]), min(first_bad[2], first_bad[3]));
          poisoned = poisoned || low < limit;
        }
        if (!ok) {
          // a wait ran out: the rest of the walk is only gone through, for the barriers in it
        } else if (warp_live && !__any_sync(0xffffffffu, limit > 0)) {
          // a request's own rows, none of whose queries is here
          const uint32_t p[32] = {};
          tmem_st32(t_s, p);
          tmem_st32(t_s + 32, p);
          tmem_st_wait();
          tc_fence_before();
          arrive_warp(p_full(s, 0));
          arrive_warp(p_full(s, 1));
        } else if (warp_live) {
          const bool masked = __any_sync(0xffffffffu, limit < kTileKeys);
          // S in two halves, the second under way while the first's maximum is found
          uint32_t v[128];
          tmem_ld64_async(t_s, v);
          tmem_ld_wait64(v);
          tmem_ld64_async(t_s + 64, v + 64);
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (half == 1) tmem_ld_wait64(v + 64);
            if (masked) {
#pragma unroll
              for (int e = half * 64; e < half * 64 + 64; ++e) v[e] = e < limit ? v[e] : 0xff800000u;
            }
#pragma unroll
            for (int e = half * 64; e < half * 64 + 64; e += 8)
#pragma unroll
              for (int j = 0; j < 4; ++j) mx[j] = max3(mx[j], __uint_as_float(v[e + j]), __uint_as_float(v[e + 4 + j]));
          }
          const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * a.scale_log2;
          const bool raise = top > m + kRaise;
          float fac = 1.f;
          if (raise) {
            fac = ex2_approx(m - top);
            m = top;
          }
          if (t > 0 && __any_sync(0xffffffffu, raise)) {
            // O so far: its last product finished before this tile's S did
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16];
              tmem_ld16(t_o + c, o);
              tmem_ld_wait(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fac);
              tmem_st16(t_o + c, o);
            }
          }
          const float shift = m == -INFINITY ? 0.f : m - kBias<T>;
          const float2 scale2 = make_float2(a.scale_log2, a.scale_log2), shift2 = make_float2(-shift, -shift);
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int c = half * 64; c < half * 64 + 64; c += 32) {
              uint32_t p[16];
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float2 x = __ffma2_rn(make_float2(__uint_as_float(v[c + e]), __uint_as_float(v[c + e + 1])),
                                            scale2, shift2);
                const float2 y = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                sum[(e >> 1) & 1] = __fadd2_rn(sum[(e >> 1) & 1], y);
                p[e / 2] = pack16<T>(y.x, y.y);
              }
              tmem_st16(t_s + c / 2, p);
            }
            tmem_st_wait();
            tc_fence_before();
            arrive_warp(p_full(s, half));
          }
          l = l * fac + ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
        } else {
          tc_fence_before();
          arrive_warp(p_full(s, 0));
          arrive_warp(p_full(s, 1));
        }
        w.next(a, u);
        if (alternate) w.next(a, u);
      }
      m -= kBias<T>;  // l and O are in these units
      if (steps > 0) wait(o_full(s), o_count[s]);
      if (!alternate) {
        tc_fence_after();
        const RowOut<T, D> dst(a, u, row, live && ok, true, m, l);
        const float inv = poisoned ? __int_as_float(0x7fffffff) : l == 0.f ? 0.f : rcp_approx(l);
        if (warp_live && ok) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld32(t_o + c, o);
            float f[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) f[e] = l == 0.f ? 0.f : __uint_as_float(o[e]) * inv;
            dst.store32(c, f);
          }
        }
      } else {
        // join the streams: each one's warps read both O and store half of the columns.  (m, l)
        // go through Q's place: both streams' products are done with it.
        if (s == 1 || n > 1) wait(o_full(s ^ 1), o_count[s ^ 1]);
        float2* const join = reinterpret_cast<float2*>(gbase + S::kQ);
        join[s * kTileRows + r] = make_float2(m, poisoned ? -l : l);  // l >= 0: the sign bit is free
        softmax_sync();
        float2 other = join[(s ^ 1) * kTileRows + r];
        tc_fence_after();
        poisoned = poisoned || signbit(other.y);
        other.y = fabsf(other.y);
        const float top = fmaxf(m, other.x), shift = top == -INFINITY ? 0.f : top;
        float mine = ex2_approx(m - shift), theirs = ex2_approx(other.x - shift);
        const float sum = mine * l + theirs * other.y;
        const RowOut<T, D> dst(a, u, row, !kCluster && live && ok, s == 0, shift, sum);
        if (kCluster && s == 0 && ok) part_lse[r] = sum == 0.f ? -INFINITY : shift + __log2f(sum);
        const float inv = poisoned ? __int_as_float(0x7fffffff) : sum == 0.f ? 0.f : rcp_approx(sum);
        const float f0 = (s == 0 ? mine : theirs) * inv, f1 = (s == 0 ? theirs : mine) * inv;
        if (warp_live && ok) {
          const uint32_t t_0 = tmem + lanes + kColO;
#pragma unroll 1
          for (int c = s * (D / 2); c < (s + 1) * (D / 2); c += 32) {
            uint32_t o[32];
            tmem_ld32(t_0 + c, o);
            float f[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) f[e] = sum == 0.f ? 0.f : __uint_as_float(o[e]) * f0;
            if (n > 1) {
              tmem_ld32(t_0 + kTileKeys + c, o);
#pragma unroll
              for (int e = 0; e < 32; ++e) f[e] = sum == 0.f ? 0.f : fmaf(__uint_as_float(o[e]), f1, f[e]);
            }
            if constexpr (kCluster) {
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                *reinterpret_cast<float4*>(part + r * kPartRow + c + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
            } else {
              dst.store32(c, f);
            }
          }
        }
      }
      tc_fence_before();
      at += 2 * n;
      ++o_count[0];
      if (!alternate || n > 1) ++o_count[1];
    }
    if constexpr (kCluster) {
      __syncwarp();
      cluster_sync();  // every part is there
      // the cluster's warps take the rows in turn; parts are added in their order
      constexpr int E = D / 32;
      const uint32_t from = smem_u32(part), lse_from = smem_u32(part_lse);
      for (int row = (int)cluster_rank() + a.splits * warp; row < part_rows; row += a.splits * (kSoftmaxThreads / 32)) {
        const float lse = lane < a.splits ? ld_cluster(cluster_addr(lse_from + 4u * row, lane)) : -INFINITY;
        float v[kMaxCluster][E];
#pragma unroll
        for (int p = 0; p < kMaxCluster; ++p)
          if (p < a.splits) {
            const uint32_t at = cluster_addr(from + 4u * (row * kPartRow + lane * E), p);
#pragma unroll
            for (int e = 0; e < E; e += 2) ld_cluster2(at + 4u * e, v[p] + e);
          }
        const float top = warp_max(lse), shift = top == -INFINITY ? 0.f : top;
        const float wgt = ex2_approx(lse - shift);
        float o[E] = {}, sum = 0.f;
#pragma unroll
        for (int p = 0; p < kMaxCluster; ++p)
          if (p < a.splits) {
            const float w = __shfl_sync(0xffffffffu, wgt, p);
            sum += w;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fmaf(w, v[p][e], o[e]);
          }
        store_joined<T, D>(a, part_h, part_row0 + row, o, sum, top);
      }
      __syncwarp();
      cluster_sync();  // no CTA leaves while another reads its part
    }
  }
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_free(tmem, 512);
  }
}

// Joins the parts of each row of the split units by their log2-sum-exps.  One CTA per row,
// its warps taking every fourth part, so that a row of many parts (single tokens: as many as
// fill the GPU) costs a few loads in a row and not one per part; the warps' sums are added in
// their order.
constexpr int kJoinWarps = 4;
template <typename T, int D>
__global__ void __launch_bounds__(32 * kJoinWarps) prefix_attn_join_kernel(const AttnArgs a) {
  constexpr int E = D / 32;
  __shared__ float sums[kJoinWarps][D + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per_request = a.lq * a.group;
  const int j = (int)(blockIdx.x / (unsigned)a.tile_rows), r = (int)(blockIdx.x - (unsigned)j * a.tile_rows);
  int grp, t;
  tile_of(a, a.whole + j, grp, t);
  const int h = a.within_request ? a.by_batch(grp) : grp, b0 = a.within_request ? grp - h * a.batch : 0;
  pdl_wait();
  pdl_trigger();
  if (t * a.tile_rows + r >= (a.within_request ? per_request : a.rows)) return;
  const int row = b0 * per_request + t * a.tile_rows + r, all = a.splits;
  const int64_t slot0 = (int64_t)j * all * a.tile_rows + r;
  auto slot_of = [&](int s) { return slot0 + (int64_t)s * a.tile_rows; };
  float top = -INFINITY;
  for (int s = lane; s < all; s += 32) top = fmaxf(top, a.part_lse[slot_of(s)]);
  top = warp_max(top);
  const float shift = top == -INFINITY ? 0.f : top;
  float o[E] = {}, sum = 0.f;
#pragma unroll 4
  for (int s = warp; s < all; s += kJoinWarps) {
    const int64_t slot = slot_of(s);
    const float wgt = ex2_approx(a.part_lse[slot] - shift);
    const float* p = a.part_o + slot * D + lane * E;
    sum += wgt;
    if constexpr (E == 4) {
      const float4 v = *reinterpret_cast<const float4*>(p);
      o[0] = fmaf(wgt, v.x, o[0]), o[1] = fmaf(wgt, v.y, o[1]), o[2] = fmaf(wgt, v.z, o[2]), o[3] = fmaf(wgt, v.w, o[3]);
    } else {
      const float2 v = *reinterpret_cast<const float2*>(p);
      o[0] = fmaf(wgt, v.x, o[0]), o[1] = fmaf(wgt, v.y, o[1]);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) sums[warp][lane * E + e] = o[e];
  if (lane == 0) sums[warp][D] = sum;
  __syncthreads();
  if (warp != 0) return;
#pragma unroll
  for (int w = 1; w < kJoinWarps; ++w) {
    sum += sums[w][D];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] += sums[w][lane * E + e];
  }
  store_joined<T, D>(a, h, row, o, sum, top);
}

// ------------------------------------------------------------------ host side
struct Plan {
  bool within_request;
  int64_t tile_rows, groups, row_tiles, items, whole, splits, units, rows, slots;
  bool clustered;  // the parts of an item are the CTAs of a cluster
  double cost;  // key tiles that the longest-working SM walks, and what joining costs
};

// What a unit costs beside its tiles (finding it, Q, the pipeline's ends, the results) and
// what joining costs, in steps of 128 keys and 256 rows.
constexpr double kUnitTiles = 2.0, kJoinTiles = 1.0, kClusterTiles = 0.7;
// Rows that a cluster joins at most.  Its CTAs read each other's parts at a few bytes a cycle, where the
// second kernel has a CTA for every row: with 32 rows 10.9 us per call in clusters and 13.1
// without, with 64 12.9 and 12.7, with 128 16.0 and 14.9.
constexpr int64_t kClusterRows = 32;
// A step of a unit of up to 128 rows takes two tiles, which is as much to load as two steps.
constexpr double kHalfStep = 0.6;

// Clusters of 2..kMaxCluster CTAs of this kernel that the GPU holds at once: the SMs come in
// groups that a cluster may not straddle, so a second round can start long before every SM has
// a CTA (24 clusters of 6: 25 us, where 6 parts and the second kernel take 17).
struct ClusterRoom {
  int clusters[kMaxCluster + 1];
};
int cluster_room(const DeviceInfo* di, ClusterRoom* room) {
  static std::atomic<uint64_t> known{0}, reserved{0};
  static std::atomic<int> held[64][kMaxCluster + 1];
  const uint64_t bit = 1ull << di->ordinal;
  if (!(known.load(std::memory_order_acquire) & bit)) {
    const auto kern = prefix_attn_kernel<__nv_bfloat16, 128, true, true>;
    constexpr int smem = AttnSmem<128, true>::kBytes;
    if (int s = reserve_smem((const void*)kern, smem, reserved, di, "shared_prefix_attention")) return s;
    for (int n = 2; n <= kMaxCluster; ++n) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)n, 1, 1);
      cfg.blockDim = dim3(kAttnThreads, 1, 1);
      cfg.dynamicSmemBytes = smem;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = (unsigned)n;
      at[0].val.clusterDim.y = 1;
      at[0].val.clusterDim.z = 1;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      int count = 0;
      if (cudaOccupancyMaxActiveClusters(&count, kern, &cfg) != cudaSuccess) {
        cudaGetLastError();
        count = 0;
      }
      held[di->ordinal][n].store(count, std::memory_order_relaxed);
    }
    known.fetch_or(bit, std::memory_order_acq_rel);
  }
  room->clusters[0] = room->clusters[1] = 0;
  for (int n = 2; n <= kMaxCluster; ++n) room->clusters[n] = held[di->ordinal][n].load(std::memory_order_relaxed);
  return JO_OK;
}

Plan make_plan(bool within_request, int64_t tile_rows, int64_t batch, int64_t lq, int64_t heads, int64_t group,
               int64_t prefix, int64_t own, int64_t hold, const ClusterRoom& room) {
  Plan p{};
  const int64_t per_request = lq * group;
  p.within_request = within_request;
  p.rows = batch * per_request;
  p.tile_rows = tile_rows;
  p.groups = within_request ? heads * batch : heads;
  p.row_tiles = cdiv(within_request ? per_request : p.rows, tile_rows);
  p.items = p.groups * p.row_tiles;
  // requests that a row tile meets
  int64_t met = within_request ? 1 : tile_rows / per_request + (tile_rows % per_request ? 2 : 0);
  if (met > batch) met = batch;
  const int64_t tiles = cdiv(prefix, kTileKeys) + met * cdiv(own, kTileKeys);
  const int64_t full = p.groups * (p.row_tiles - 1);  // items before the groups' last row tiles
  const int64_t last_rows = (within_request ? per_request : p.rows) - (p.row_tiles - 1) * tile_rows;
  auto step = [](int64_t rows) { return rows <= kTileRows ? kHalfStep : 1.0; };
  // The units go round the SMs in order, the longest first: the first SM's are the most work.
  // Every whole round of items is left whole, or all but the last; the rest is split in the
  // number of parts that ends first.
  const int64_t most = tiles / 2 < 1 ? 1 : tiles / 2 < hold ? tiles / 2 : hold;
  const int64_t rounds = p.items / hold;
  const int64_t limit = INT32_MAX / (tiles + 1);  // tiles * splits stays within 31 bits
  bool any = false;
  for (int64_t whole = rounds * hold; whole >= 0 && whole >= (rounds - 1) * hold; whole -= hold)
    for (int trial = 1; trial <= 19; ++trial) {
      // up to 16 parts, and the numbers that fill one, two and three rounds
      const int64_t s = trial <= 16 ? trial : whole < p.items ? (trial - 16) * hold / (p.items - whole) : 1;
      if (s > most || s < 1 || (s > 1 && s > limit) || (s > 1 && whole == p.items)) continue;
      const int64_t cut = whole > full ? whole : full;
      // one unit of few rows to a CTA, in as many parts as a cluster may have CTAs
      const bool clustered = (p.row_tiles > 1 ? tile_rows : last_rows) <= kClusterRows && tile_rows <= kTileRows &&
                             whole == 0 && s > 1 && s <= kMaxCluster && p.items <= room.clusters[s];
      double cost = clustered ? kClusterTiles : s > 1 ? kJoinTiles + 0.05 * (double)s : 0.;
      int64_t at = 0;
      auto add = [&](int64_t units, double tiles_each, double per_tile) {
        cost += (double)(cdiv(at + units, hold) - cdiv(at, hold)) * (tiles_each * per_tile + kUnitTiles);
        at += units;
      };
      const int64_t whole_full = whole < full ? whole : full;
      add(whole_full, (double)tiles, step(tile_rows));
      add(whole - whole_full, (double)tiles, step(last_rows));
      add((cut - whole) * s, (double)cdiv(tiles, s), step(tile_rows));
      add((p.items - cut) * s, (double)cdiv(tiles, s), step(last_rows));
      if (!any || cost < p.cost) {
        p.cost = cost;
        p.whole = whole;
        p.splits = s;
        p.clustered = clustered;
        any = true;
      }
    }
  if (p.splits == 1) p.whole = p.items;
  p.units = p.whole + (p.items - p.whole) * p.splits;
  p.slots = p.clustered ? 0 : (p.items - p.whole) * p.splits * tile_rows;
  return p;
}

// `hold`: CTAs that the GPU holds at once (one per SM).
Plan plan_attention(int64_t batch, int64_t lq, int64_t heads, int64_t group, int64_t prefix, int64_t own,
                    int64_t hold, const ClusterRoom& room) {
  Plan best{};
  for (int64_t tile_rows : {(int64_t)kTileRows, (int64_t)kUnitRows})
    for (bool within : {true, false}) {
      if (!within && batch == 1) continue;
      const Plan p = make_plan(within, tile_rows, batch, lq, heads, group, prefix, own, hold, room);
      if (best.units == 0 || p.cost < best.cost) best = p;
    }
  return best;
}

int check_sizes(const char* op, int64_t batch, int64_t lq, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                int64_t prefix, int64_t own) {
  if (batch < 0 || lq < 0 || prefix < 0 || own < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads)
    return fail(JO_ERR_SHAPE, "%s: bad sizes (q heads must be a multiple of the k/v heads)", op);
  if (head_dim != 64 && head_dim != 128) return fail(JO_ERR_SHAPE, "%s: head_dim must be 64 or 128", op);
  const int64_t most = INT32_MAX / 2;
  if (batch > most || lq > most || prefix > most || own > most || q_heads > most || lq * (q_heads / kv_heads) > most ||
      batch * q_heads > most || batch * lq > most || batch * lq * (q_heads / kv_heads) > most ||
      batch * lq * q_heads > (int64_t)1 << 38)
    return fail(JO_ERR_SHAPE, "%s: size too large", op);
  return JO_OK;
}

// [batch, rows, heads, D] with element strides; dimensions of size 1 get any valid stride.
int make_kv_map(const char* op, CUtensorMap* map, const void* ptr, int64_t d, int64_t heads, int64_t rows,
                int64_t batch, int64_t st_h, int64_t st_t, int64_t st_b, int dtype) {
  auto fn = tensor_map_encoder();
  if (!fn) return fail(JO_ERR_CUDA, "%s: cuTensorMapEncodeTiled unavailable", op);
  cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)rows, (cuuint64_t)batch};
  cuuint64_t strides[3] = {(cuuint64_t)(heads > 1 ? st_h : d) * 2, (cuuint64_t)(rows > 1 ? st_t : d) * 2,
                           (cuuint64_t)(batch > 1 ? st_b : d) * 2};
  cuuint32_t box[4] = {64, 1, (cuuint32_t)kTileKeys, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = fn(map, dtype == JO_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                        const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(JO_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed (%d)", op, (int)r);
  return JO_OK;
}

template <typename T, int D, bool kAlone, bool kCluster>
int launch_units(const CUtensorMap* maps, const AttnArgs& a, cudaStream_t st, const DeviceInfo* di) {
  const char* op = "shared_prefix_attention";
  auto kern = prefix_attn_kernel<T, D, kAlone, kCluster>;
  constexpr int smem = AttnSmem<D, kAlone>::kBytes;
  static std::atomic<uint64_t> reserved{0};
  if (int s = reserve_smem((const void*)kern, smem, reserved, di, op)) return s;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.units < di->sm_count ? a.units : di->sm_count), 1, 1);
  cfg.blockDim = dim3(kAttnThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)a.splits;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = kCluster ? 2 : 1;
  if (cudaError_t e = cudaLaunchKernelEx(&cfg, kern, maps[0], maps[1], maps[2], maps[3], a))
    return launch_failed(e, op);
  return after_launch("prefix_attn_kernel");
}

template <typename T, int D>
int launch_attention(const CUtensorMap* maps, const AttnArgs& a, const Plan& p, cudaStream_t st, const DeviceInfo* di) {
  if (p.clustered) return launch_units<T, D, true, true>(maps, a, st, di);
  if (int s = p.tile_rows <= kTileRows ? launch_units<T, D, true, false>(maps, a, st, di)
                                       : launch_units<T, D, false, false>(maps, a, st, di))
    return s;
  if (const int64_t joined = (p.items - p.whole) * p.tile_rows) {
    if (cudaError_t e = launch_pdl(prefix_attn_join_kernel<T, D>, dim3((unsigned)joined), dim3(32 * kJoinWarps), 0, st, a))
      return launch_failed(e, "shared_prefix_attention");
    return after_launch("prefix_attn_join_kernel");
  }
  return JO_OK;
}

}  // namespace
}  // namespace jo

using namespace jo;

extern "C" {

int64_t jo_shared_prefix_attention_workspace(int64_t batch, int64_t q_len, int64_t q_heads, int64_t kv_heads,
                                             int64_t head_dim, int64_t prefix_len, int64_t own_len) {
  const DeviceInfo* di;
  if (device_info(&di)) return -1;
  if (check_sizes("shared_prefix_attention", batch, q_len, q_heads, kv_heads, head_dim, prefix_len, own_len)) return -1;
  if (batch == 0 || q_len == 0) return 0;
  ClusterRoom room;
  if (cluster_room(di, &room)) return -1;
  const Plan p = plan_attention(batch, q_len, kv_heads, q_heads / kv_heads, prefix_len, own_len, di->sm_count, room);
  return p.slots * (head_dim + 1) * 4;
}

int jo_shared_prefix_attention(void* out, float* lse, const void* q, int64_t q_stride_b, int64_t q_stride_t,
                               int64_t q_stride_h, const void* k_prefix, int64_t kp_stride_t, int64_t kp_stride_h,
                               const void* v_prefix, int64_t vp_stride_t, int64_t vp_stride_h, const void* k_own,
                               int64_t ko_stride_b, int64_t ko_stride_t, int64_t ko_stride_h, const void* v_own,
                               int64_t vo_stride_b, int64_t vo_stride_t, int64_t vo_stride_h, const int32_t* lens,
                               int64_t batch, int64_t q_len, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                               int64_t prefix_len, int64_t own_len, int causal, float scale, void* workspace,
                               int64_t workspace_bytes, int dtype, void* stream) {
  const char* op = "shared_prefix_attention";
  const DeviceInfo* di;
  if (int s = device_info(&di)) return s;
  if (dtype != JO_BF16 && dtype != JO_F16) return fail(JO_ERR_DTYPE, "%s: q, k and v must be bf16 or fp16", op);
  if (int s = check_sizes(op, batch, q_len, q_heads, kv_heads, head_dim, prefix_len, own_len)) return s;
  if (!(scale > 0.f && scale <= 3.4e38f)) return fail(JO_ERR_INVALID, "%s: scale must be positive and finite", op);
  if (batch == 0 || q_len == 0) return JO_OK;
  if (!out || !lse || !q || !lens || (prefix_len && (!k_prefix || !v_prefix)) || (own_len && (!k_own || !v_own)))
    return fail(JO_ERR_INVALID, "%s: null operand", op);
  if ((reinterpret_cast<uintptr_t>(out) & 31) || !aligned16(q) || !aligned16(k_prefix) || !aligned16(v_prefix) ||
      !aligned16(k_own) || !aligned16(v_own))
    return fail(JO_ERR_ALIGN, "%s: operands must be 16-byte aligned (out: 32)", op);
  // a stride of a dimension of size 1 is never used
  const struct {
    int64_t size, stride;
  } used[] = {{batch, q_stride_b},        {q_len, q_stride_t},        {q_heads, q_stride_h},
              {prefix_len, kp_stride_t},  {prefix_len, vp_stride_t},  {prefix_len ? kv_heads : 0, kp_stride_h},
              {prefix_len ? kv_heads : 0, vp_stride_h},               {own_len ? batch : 0, ko_stride_b},
              {own_len ? batch : 0, vo_stride_b},                     {own_len, ko_stride_t},
              {own_len, vo_stride_t},     {own_len ? kv_heads : 0, ko_stride_h},
              {own_len ? kv_heads : 0, vo_stride_h}};
  for (const auto& u : used)
    if (u.size > 1 && (u.stride % 8 || u.stride < 0))
      return fail(JO_ERR_ALIGN, "%s: strides must be multiples of 16 bytes and not negative", op);
  ClusterRoom room;
  if (int s = cluster_room(di, &room)) return s;
  const Plan p = plan_attention(batch, q_len, kv_heads, q_heads / kv_heads, prefix_len, own_len, di->sm_count, room);
  if (p.units > INT32_MAX / 2 || (p.items - p.whole) * p.tile_rows > INT32_MAX)
    return fail(JO_ERR_SHAPE, "%s: size too large", op);
  if (p.slots && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 31) ||
                  workspace_bytes < p.slots * (head_dim + 1) * 4))
    return fail(JO_ERR_INVALID, "%s: a 32-byte aligned workspace of %lld bytes is needed", op,
                (long long)(p.slots * (head_dim + 1) * 4));
  AttnArgs a{};
  a.out = out;
  a.lse = lse;
  a.q = q;
  a.q_b = q_stride_b;
  a.q_t = q_stride_t;
  a.q_h = q_stride_h;
  a.lens = lens;
  a.prefix = (int)prefix_len;
  a.batch = (int)batch;
  a.lq = (int)q_len;
  a.heads = (int)kv_heads;
  a.group = (int)(q_heads / kv_heads);
  a.own = (int)own_len;
  a.causal = causal;
  a.scale_log2 = scale * kLog2E;
  a.within_request = p.within_request;
  a.tile_rows = (int)p.tile_rows;
  a.groups = (int)p.groups;
  a.row_tiles = (int)p.row_tiles;
  a.items = (int)p.items;
  a.whole = (int)p.whole;
  a.splits = (int)p.splits;
  a.units = (int)p.units;
  a.rows = (int)p.rows;
  const int64_t full = p.groups * (p.row_tiles - 1), cut = p.whole > full ? p.whole : full;
  auto at_least_1 = [](int64_t d) { return FastDiv(d > 1 ? d : 1); };
  a.by_request = FastDiv(q_len * a.group);
  a.by_group = FastDiv(a.group);
  a.by_batch = FastDiv(batch);
  a.by_full = at_least_1(p.row_tiles - 1);
  a.by_tail = at_least_1(cut - p.whole);
  a.by_last = at_least_1(p.items - cut);
  a.by_splits = FastDiv(p.splits);
  a.part_o = (float*)workspace;
  a.part_lse = (float*)workspace + p.slots * head_dim;
  a.fault = di->fault;
  CUtensorMap maps[4] = {};
  if (prefix_len) {
    if (int s = make_kv_map(op, &maps[0], k_prefix, head_dim, kv_heads, prefix_len, 1, kp_stride_h, kp_stride_t, 0, dtype))
      return s;
    if (int s = make_kv_map(op, &maps[1], v_prefix, head_dim, kv_heads, prefix_len, 1, vp_stride_h, vp_stride_t, 0, dtype))
      return s;
  }
  if (own_len) {
    if (int s = make_kv_map(op, &maps[2], k_own, head_dim, kv_heads, own_len, batch, ko_stride_h, ko_stride_t,
                            ko_stride_b, dtype))
      return s;
    if (int s = make_kv_map(op, &maps[3], v_own, head_dim, kv_heads, own_len, batch, vo_stride_h, vo_stride_t,
                            vo_stride_b, dtype))
      return s;
  }
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == JO_BF16)
    return head_dim == 64 ? launch_attention<__nv_bfloat16, 64>(maps, a, p, st, di)
                          : launch_attention<__nv_bfloat16, 128>(maps, a, p, st, di);
  return head_dim == 64 ? launch_attention<__half, 64>(maps, a, p, st, di)
                        : launch_attention<__half, 128>(maps, a, p, st, di);
}

}  // extern "C"
