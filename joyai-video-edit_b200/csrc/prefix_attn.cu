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
// Rows.  All queries that read one k/v head can share its keys whatever request they
// belong to, so over the prefix a row of a tensor-core tile is any (request, query, q head
// of the k/v head's group): the prefix is read once for up to 256 such rows, not once per
// request.  Two plans (plan_attention):
//   packed  row tiles run across requests; the prefix and each request's own rows are
//           separate work items, joined afterwards;
//   fused   row tiles stay within a request and walk the prefix, then its own rows.
// Where the items do not fill the GPU evenly, the last ones' keys are split and joined.
//
// One CTA per SM walks over the items with two streams, each with its own S, P and O in
// tensor memory, so that one stream's softmax runs while the other's products do:
//   an item of more than 128 rows: the streams take its two halves, and share every K and
//   V tile (64 KB per tile of 128 keys would otherwise exceed what an SM can take in);
//   an item of up to 128 rows (single tokens): the streams take alternate key tiles of the
//   same rows and are joined at the end.
// Warps 0-3 and 4-7: softmax of stream 0 and 1, one row per thread (tensor-memory lane):
//   S from tensor memory, the running maximum and sum, P back in place of S in two halves
//   (the product may start on the first), O rescaled in place; Q and the results.
// Warp 8: TMA producer of K and V tiles of 128 rows (128-byte swizzle) into one ring, in
//   the order of their first use; it runs ahead across items.
// Warp 9: tcgen05.mma issuer: S = Q K^T (both operands in shared memory), O += P V with P
//   from tensor memory and V as it lies ([keys, D], the MN-major operand).
//
// P is rounded to q's 16-bit type for the tensor cores (its error averages out over the
// keys: 2^-9 relative for bf16, like the output's own rounding); l sums the unrounded p.
#include "tcgen05.cuh"

namespace jo {
namespace {

constexpr int kTileRows = 128;           // rows per stream (UMMA M)
constexpr int kItemRows = 2 * kTileRows;  // rows per item at most
constexpr int kTileKeys = 128;           // keys per tile (UMMA N of S, K of P V)
constexpr int kSoftmaxThreads = 256;
constexpr int kAttnThreads = 320;
constexpr int kColO = 256;  // tensor memory: S / P of the streams at 0 and 128, O at 256 and 384
constexpr float kRaise = 8.f;

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
  // plan: items 0..items-1 are the row tiles of `groups` groups (packed: k/v heads, fused:
  // (head, request) pairs), every group's last tile after all others; those from `whole` on
  // are split in `splits`; then, packed, the own rows of each (request, head)
  int fused;
  int groups, row_tiles;
  int items, whole, splits;
  int own_tiles, own_splits;
  int blocks;           // work units in all
  int64_t rows;         // queries per k/v head
  int64_t slot_tail;    // first slot of the split items' parts
  int64_t slot_own;     // and of the own rows'; whole items' parts (packed): from 0
  float* part_o;        // [slots, D]
  float* part_lse;
  unsigned int* fault;
};

// One work unit: rows [row0, row0 + rows) of k/v head h (row: (b * Lq + i) * G + g) and tiles
// [first, last) of the prefix's, then the request's own, keys.
struct Item {
  int h, b;  // b: the request of the own rows (-1: none)
  int row0, rows;
  int prefix_tiles;  // tiles of the walk that belong to the prefix
  int first, last;
  int len;       // own rows of b
  int64_t slot;  // partial slot of row0 (-1: final output)
};

__device__ __forceinline__ int own_visible(const AttnArgs& a, int len, int i) {
  return a.causal ? min(len, max(0, len - a.lq + i + 1)) : len;
}

// Group and row tile of an item.
__device__ __forceinline__ void tile_of(const AttnArgs& a, int item, int& grp, int& t) {
  const int full = a.groups * (a.row_tiles - 1);
  if (item < full) {
    grp = item / (a.row_tiles - 1);
    t = item - grp * (a.row_tiles - 1);
  } else {
    grp = item - full;
    t = a.row_tiles - 1;
  }
}

__device__ Item item_of(const AttnArgs& a, int block) {
  Item it;
  const int per_request = a.lq * a.group;
  const int ptiles = (a.prefix + kTileKeys - 1) / kTileKeys;
  int piece = 0, pieces = 1, t;
  it.slot = -1;
  const int first_kind = a.whole + (a.items - a.whole) * a.splits;
  if (block < first_kind) {
    int item = block;
    if (block >= a.whole) {
      const int tail = a.items - a.whole, j = block - a.whole;
      piece = j / tail;
      item = a.whole + j - piece * tail;
      pieces = a.splits;
    }
    int grp;
    tile_of(a, item, grp, t);
    if (a.fused) {
      it.h = grp / a.batch;
      it.b = grp - it.h * a.batch;
      it.row0 = it.b * per_request + t * kItemRows;
      it.rows = min(kItemRows, per_request - t * kItemRows);
    } else {
      it.h = grp;
      it.b = -1;
      it.row0 = t * kItemRows;
      it.rows = (int)min((int64_t)kItemRows, a.rows - it.row0);
    }
    it.prefix_tiles = ptiles;
    if (item >= a.whole && (pieces > 1 || a.own_splits > 0))
      it.slot = a.slot_tail + ((int64_t)(item - a.whole) * pieces + piece) * kItemRows;
    else if (a.own_splits > 0)
      it.slot = (int64_t)it.h * a.rows + it.row0;
  } else {
    int j = block - first_kind;
    pieces = a.own_splits;
    const int rest = j / pieces;
    piece = j - rest * pieces;
    j = rest / a.own_tiles;
    t = rest - j * a.own_tiles;
    it.b = j / a.heads;
    it.h = j - it.b * a.heads;
    it.row0 = it.b * per_request + t * kItemRows;
    it.rows = min(kItemRows, per_request - t * kItemRows);
    it.prefix_tiles = 0;
    it.slot = a.slot_own + ((int64_t)piece * a.heads + it.h) * a.rows + it.row0;
  }
  int tiles = it.prefix_tiles;
  it.len = 0;
  if (it.b >= 0) {
    it.len = min(max(__ldg(a.lens + it.b), 0), a.own);
    // the last of the tile's queries sees the most
    tiles += (own_visible(a, it.len, (it.row0 - it.b * per_request + it.rows - 1) / a.group) + kTileKeys - 1) / kTileKeys;
  }
  it.first = (int)((int64_t)tiles * piece / pieces);
  it.last = (int)((int64_t)tiles * (piece + 1) / pieces);
  return it;
}

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

template <int D>
struct AttnSmem {
  static constexpr int kTile = kTileKeys * D * 2;  // bytes of a K, V or Q tile
  static constexpr int kRing = D == 64 ? 8 : 5;
  static constexpr int kQ = 0;  // two tiles
  static constexpr int kKV = 2 * kTile;
  static constexpr int kJoin = kKV + kRing * kTile;  // (m, l) of stream 1
  static constexpr int kBars = kJoin + kTileRows * 8;
  static constexpr int kBytes = kBars + 256 + 1024 /*align*/;
};

// The ring's order of loads for n tiles, which is the order of their first use.
//   shared by both streams:  K0 V0 K1 V1 ...
//   alternate tiles:         K0 K1 V0 K2 V1 K3 ... V(n-2) V(n-1)
__device__ __forceinline__ int k_index(bool alternate, int tile) {
  return alternate ? (tile < 2 ? tile : 2 * tile - 1) : 2 * tile;
}
__device__ __forceinline__ int v_index(bool alternate, int tile, int n) {
  return alternate ? (tile == n - 1 ? 2 * n - 1 : 2 * tile + 2) : 2 * tile + 1;
}
__device__ __forceinline__ void load_at(bool alternate, int idx, int n, int& tile, bool& value) {
  if (!alternate) {
    tile = idx >> 1;
    value = idx & 1;
  } else if (idx == 2 * n - 1) {
    tile = n - 1;
    value = true;
  } else if (idx < 2) {
    tile = idx;
    value = false;
  } else {
    value = !(idx & 1);
    tile = value ? (idx - 2) >> 1 : (idx + 1) >> 1;
  }
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
  __device__ __forceinline__ RowOut(const AttnArgs& a, const Item& it, int r, bool live, float m, float l) {
    if (!live) return;
    const float lse2 = l == 0.f ? -INFINITY : m + __log2f(l);
    if (it.slot >= 0) {
      part = a.part_o + (it.slot + r) * D;
      a.part_lse[it.slot + r] = lse2;
    } else {
      const int per_request = a.lq * a.group, row = it.row0 + r;
      const int b = row / per_request, in = row - b * per_request, i = in / a.group, g = in - i * a.group;
      const int64_t hq = (int64_t)a.heads * a.group, h = (int64_t)it.h * a.group + g;
      out = reinterpret_cast<T*>(a.out) + (((int64_t)b * a.lq + i) * hq + h) * D;
      a.lse[(b * hq + h) * a.lq + i] = lse2 * 0.6931471805599453f;
    }
  }
  __device__ __forceinline__ void store32(int c, const float* f) const {
    if (part != nullptr) {
#pragma unroll
      for (int e = 0; e < 32; e += 4) st_global(part + c + e, Elt<float>::pack(f + e));
    } else if (out != nullptr) {
#pragma unroll
      for (int e = 0; e < 32; e += 8) st_global(out + c + e, Elt<T>::pack(f + e));
    }
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kAttnThreads, 1)
    prefix_attn_kernel(const __grid_constant__ CUtensorMap map_kp, const __grid_constant__ CUtensorMap map_vp,
                       const __grid_constant__ CUtensorMap map_ko, const __grid_constant__ CUtensorMap map_vo,
                       const AttnArgs a) {
  using S = AttnSmem<D>;
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
  const int warp = warp_index(), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kRing; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(q_full, kSoftmaxThreads);
    mbar_init(done, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(s_full(s), 1);
      mbar_init(p_full(s, 0), kTileRows);
      mbar_init(p_full(s, 1), kTileRows);
      mbar_init(o_full(s), 1);
    }
    mbar_init_fence();
  }
  if (warp == 9) tmem_alloc(tmem_slot, 512);
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<uint32_t*>(gbase + (tmem_slot - base));
  pdl_wait();  // lens, q, k and v may be the previous kernel's
  pdl_trigger();

  if (warp == 8) {
    if (lane == 0) {
      // ---------------- TMA producer
      int at = 0;  // loads so far
      bool ok = true;
      for (int block = blockIdx.x; block < a.blocks && ok; block += gridDim.x) {
        const Item it = item_of(a, block);
        const int n = it.last - it.first;
        const bool alternate = it.rows <= kTileRows;
        for (int j = 0; j < 2 * n; ++j, ++at) {
          const int slot = at % kRing;
          if (!(ok = mbar_wait(empty(slot), ((at / kRing) & 1) ^ 1u, a.fault))) break;
          int tile;
          bool value;
          load_at(alternate, j, n, tile, value);
          tile += it.first;
          const bool own = tile >= it.prefix_tiles;
          const CUtensorMap* map = value ? (own ? &map_vo : &map_vp) : (own ? &map_ko : &map_kp);
          const int row = (own ? tile - it.prefix_tiles : tile) * kTileKeys;
          mbar_expect_tx(full(slot), S::kTile);
#pragma unroll
          for (int x = 0; x < D; x += 64)
            tma_load_4d(base + S::kKV + slot * S::kTile + (x / 64) * kBox, map, x, it.h, row, own ? it.b : 0, full(slot));
        }
      }
      // every copy issued has landed before the CTA may exit
      for (int j = max(0, at - kRing); j < at; ++j) mbar_wait(full(j % kRing), (j / kRing) & 1, a.fault);
    }
  } else if (warp == 9) {
    // ---------------- MMA issuer: the warp stays converged and elects one thread per step
    constexpr uint32_t idesc_s = attn_idesc<T>(kTileKeys, false), idesc_o = attn_idesc<T>(D, true);
    const uint64_t qd = sw128_desc(base + S::kQ), kd0 = sw128_desc(base + S::kKV);
    const uint64_t vd0 = sw128_desc_mn(base + S::kKV, kBox);
    int at = 0, count[2] = {0, 0}, items = 0;
    bool ok = true;
    auto wait = [&](uint32_t bar, int phase) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar, phase & 1, a.fault));
      return ok;
    };
    for (int block = blockIdx.x; block < a.blocks && ok; block += gridDim.x) {
      const Item it = item_of(a, block);
      const int n = it.last - it.first;
      if (n == 0) continue;
      const bool alternate = it.rows <= kTileRows;
      const int steps[2] = {alternate ? (n + 1) / 2 : n, alternate ? n / 2 : n};
      auto products_s = [&](int s, int t) {  // S of stream s, step t
        const int idx = at + k_index(alternate, alternate ? 2 * t + s : t), slot = idx % kRing;
        if (!wait(full(slot), idx / kRing)) return;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t kd = kd0 + slot * (S::kTile >> 4), q = qd + (alternate ? 0 : s * (S::kTile >> 4));
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const int off = ((kk / 4) * kBox + (kk % 4) * 32) >> 4;
            tc_mma_f16_ss(tmem + s * kTileKeys, q + off, kd + off, idesc_s, kk != 0);
          }
          if (alternate || s == 1) tc_commit(empty(slot));
          tc_commit(s_full(s));
        }
        __syncwarp();
      };
      auto products_o = [&](int s, int t) {  // O of stream s, step t
        const int idx = at + v_index(alternate, alternate ? 2 * t + s : t, n), slot = idx % kRing;
        if (!wait(full(slot), idx / kRing)) return;
        const uint64_t vd = vd0 + slot * (S::kTile >> 4);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (!wait(p_full(s, half), count[s])) return;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int kk = 4 * half; kk < 4 * half + 4; ++kk)
              tc_mma_f16_ts(tmem + kColO + s * kTileKeys, tmem + s * kTileKeys + kk * 8, vd + kk * (2048 >> 4), idesc_o,
                            t != 0 || kk != 0);
            if (half == 1) {
              if (alternate || s == 1) tc_commit(empty(slot));
              if (t == steps[s] - 1) tc_commit(o_full(s));
            }
          }
          __syncwarp();
        }
        ++count[s];
      };
      if (!wait(q_full, items++)) break;
      products_s(0, 0);
      if (steps[1] > 0) products_s(1, 0);
      for (int t = 0; t < steps[0] && ok; ++t) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (t >= steps[s]) continue;
          products_o(s, t);
          if (t + 1 < steps[s]) products_s(s, t + 1);
        }
      }
      at += 2 * n;
    }
    // tensor memory is freed below: everything issued has retired, also after a failed wait
    if (elect_one()) tc_commit(done);
    __syncwarp();
    mbar_wait(done, 0, a.fault);
  } else {
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
    int count = 0, at = 0, o_count[2] = {0, 0};
    for (int block = blockIdx.x; block < a.blocks; block += gridDim.x) {
      const Item it = item_of(a, block);
      const int n = it.last - it.first;
      const bool alternate = it.rows <= kTileRows;
      const int row = alternate ? r : s * kTileRows + r;  // of the item
      const bool live = row < it.rows;
      if (n == 0) {  // nothing to see: an empty part
        if (!alternate || s == 0) {
          const RowOut<T, D> dst(a, it, row, live, 0.f, 0.f);
          const float zero[32] = {};
          for (int c = 0; c < D; c += 32) dst.store32(c, zero);
        }
        continue;
      }
      softmax_sync();  // both streams are done with the last item's Q and O
      {
        // Q, 16 bytes per step, 128-byte swizzle; rows past the last are zero
        constexpr int kVecs = D / 8, kStep = kSoftmaxThreads / kVecs;
        const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)it.h * a.group * a.q_h;
        const int c = threadIdx.x % kVecs, rows = alternate ? kTileRows : kItemRows;
#pragma unroll 4
        for (int j = threadIdx.x / kVecs; j < rows; j += kStep) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (j < it.rows) {
            const int flat = it.row0 + j, b = flat / per_request;
            const int in = flat - b * per_request, i = in / a.group, g = in - i * a.group;
            v = ld_stream(q + b * a.q_b + i * a.q_t + g * a.q_h + c * 8);
          }
          const uint32_t off = (j / kTileRows) * S::kTile + (c / 8) * kBox + (j % kTileRows) * 128 + (((c & 7) ^ (j & 7)) << 4);
          *reinterpret_cast<uint4*>(gbase + S::kQ + off) = v;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(q_full);
      }
      // own rows that this query sees
      int visible = 0;
      if (it.b >= 0) visible = own_visible(a, it.len, (it.row0 - it.b * per_request + min(row, it.rows - 1)) / a.group);
      const bool warp_live = (alternate ? 0 : s * kTileRows) + ((warp & 3) << 5) < it.rows;
      const int steps = alternate ? (n + 1 - s) / 2 : n;
      float m = -INFINITY, l = 0.f;
      for (int t = 0; t < steps; ++t, ++count) {
        const int local = alternate ? 2 * t + s : t, tile = it.first + local;
        const bool own = tile >= it.prefix_tiles;
        const int key0 = (own ? tile - it.prefix_tiles : tile) * kTileKeys;
        const int limit = min(kTileKeys, (own ? visible : a.prefix) - key0);
        if (!wait(s_full(s), count)) break;
        tc_fence_after();
        if (own && key0 + kTileKeys > it.len && it.len < a.own && (alternate || s == 0)) {
          // cache rows past the request's length hold anything: their p is 0, but 0 * inf is
          // not (a tile that both streams use: stream 0's product comes first)
          const int idx = at + v_index(alternate, local, n), slot = idx % kRing;
          if (!wait(full(slot), idx / kRing)) break;
          if (key0 + r >= it.len) {
#pragma unroll
            for (int x = 0; x < D / 64; ++x)
#pragma unroll
              for (int c = 0; c < 8; ++c)
                *reinterpret_cast<uint4*>(gbase + S::kKV + slot * S::kTile + x * kBox + r * 128 + c * 16) =
                    make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        if (warp_live) {
          const bool masked = __any_sync(0xffffffffu, limit < kTileKeys);
          uint32_t v[128];
          tmem_ld128(t_s, v);
          if (masked) {
#pragma unroll
            for (int e = 0; e < 128; ++e) v[e] = e < limit ? v[e] : 0xff800000u;
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < 128; e += 8)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              mx[j] = fmaxf(fmaxf(mx[j], __uint_as_float(v[e + j])), __uint_as_float(v[e + 4 + j]));
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2;
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
          const float shift = m == -INFINITY ? 0.f : m;
          const float2 scale2 = make_float2(a.scale_log2, a.scale_log2), shift2 = make_float2(-shift, -shift);
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t p[32];
#pragma unroll
            for (int e = 0; e < 64; e += 2) {
              const float2 x = __ffma2_rn(make_float2(__uint_as_float(v[half * 64 + e]), __uint_as_float(v[half * 64 + e + 1])),
                                          scale2, shift2);
              const float2 y = make_float2(ex2_approx(x.x), ex2_approx(x.y));
              sum[(e >> 1) & 1] = __fadd2_rn(sum[(e >> 1) & 1], y);
              p[e / 2] = pack16<T>(y.x, y.y);
            }
            tmem_st32(t_s + half * 32, p);
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(p_full(s, half));
          }
          l = l * fac + ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
        } else {
          tc_fence_before();
          mbar_arrive(p_full(s, 0));
          mbar_arrive(p_full(s, 1));
        }
      }
      if (steps > 0) wait(o_full(s), o_count[s]);
      if (!alternate) {
        tc_fence_after();
        const RowOut<T, D> dst(a, it, row, live && ok, m, l);
        const float inv = l == 0.f ? 0.f : 1.f / l;
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
        // join the streams: stream 0's warps read both O
        float2* const join = reinterpret_cast<float2*>(gbase + S::kJoin);
        if (s == 1) join[r] = make_float2(m, l);
        softmax_sync();
        if (s == 0) {
          if (n > 1) wait(o_full(1), o_count[1]);
          tc_fence_after();
          const float2 other = n > 1 ? join[r] : make_float2(-INFINITY, 0.f);
          const float top = fmaxf(m, other.x), shift = top == -INFINITY ? 0.f : top;
          float f0 = ex2_approx(m - shift), f1 = ex2_approx(other.x - shift);
          const float sum = f0 * l + f1 * other.y;
          const RowOut<T, D> dst(a, it, row, live && ok, shift, sum);
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          f0 *= inv;
          f1 *= inv;
          if (warp_live && ok) {
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              tmem_ld32(t_o + c, o);
              float f[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) f[e] = sum == 0.f ? 0.f : __uint_as_float(o[e]) * f0;
              if (n > 1) {
                tmem_ld32(t_o + kTileKeys + c, o);
#pragma unroll
                for (int e = 0; e < 32; ++e) f[e] = sum == 0.f ? 0.f : fmaf(__uint_as_float(o[e]), f1, f[e]);
              }
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
  }
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_free(tmem, 512);
  }
}

// Joins the parts of each row by their log2-sum-exps: one warp per row.  With own parts,
// every row has them and one part (whole items) or `splits` over the prefix; without, only
// the split items' rows are here.
template <typename T, int D>
__global__ void __launch_bounds__(256) prefix_attn_join_kernel(const AttnArgs a, int64_t total) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  pdl_wait();
  pdl_trigger();
  if (w >= total) return;
  const int per_request = a.lq * a.group;
  int h, row, parts;
  int64_t slot0, step;
  if (a.own_splits == 0) {
    const int item = a.whole + (int)(w / kItemRows), r = (int)(w % kItemRows);
    int grp, t;
    tile_of(a, item, grp, t);
    h = a.fused ? grp / a.batch : grp;
    const int b = a.fused ? grp - h * a.batch : 0;
    if (t * kItemRows + r >= (a.fused ? (int64_t)per_request : a.rows)) return;
    row = b * per_request + t * kItemRows + r;
    parts = a.splits;
    slot0 = a.slot_tail + (w / kItemRows) * parts * kItemRows + r;
    step = kItemRows;
  } else {
    h = (int)(w / a.rows);
    row = (int)(w - h * a.rows);
    const int t = row / kItemRows, full = a.row_tiles - 1;
    const int item = t < full ? h * full + t : a.heads * full + h;
    if (item < a.whole) {
      parts = 1;
      slot0 = h * a.rows + row;
      step = 0;
    } else {
      parts = a.splits;
      slot0 = a.slot_tail + (int64_t)(item - a.whole) * parts * kItemRows + row - t * kItemRows;
      step = kItemRows;
    }
  }
  const int64_t own0 = a.slot_own + (int64_t)h * a.rows + row, own_step = a.heads * a.rows;
  const int all = parts + a.own_splits;
  auto slot_of = [&](int s) { return s < parts ? slot0 + s * step : own0 + (s - parts) * own_step; };
  float top = -INFINITY;
  for (int s = lane; s < all; s += 32) top = fmaxf(top, a.part_lse[slot_of(s)]);
  top = warp_max(top);
  const float shift = top == -INFINITY ? 0.f : top;
  float o[E] = {}, sum = 0.f;
#pragma unroll 4
  for (int s = 0; s < all; ++s) {
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
  const int64_t hq = (int64_t)a.heads * a.group;
  const int b = row / per_request, in = row - b * per_request, i = in / a.group, g = in - i * a.group;
  const int64_t hh = (int64_t)h * a.group + g;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint32_t* out = reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(a.out) + (((int64_t)b * a.lq + i) * hq + hh) * D + lane * E);
#pragma unroll
  for (int e = 0; e < E; e += 2) out[e / 2] = pack16<T>(o[e] * inv, o[e + 1] * inv);
  if (lane == 0)
    a.lse[(b * hq + hh) * a.lq + i] = sum == 0.f ? -INFINITY : (top + __log2f(sum)) * 0.6931471805599453f;
}

// ------------------------------------------------------------------ host side
struct Plan {
  bool fused;
  int64_t groups, row_tiles, items, whole, splits, own_tiles, own_splits, blocks, rows;
  int64_t slot_tail, slot_own, slots, joined;
  double cost;  // key tiles that the longest-working SM walks, and what joining costs
};

// What a unit costs beside its tiles (Q, the results, the pipeline's ends) and what its rows'
// parts cost to join, in key tiles; measured on single tokens (about 1 us each).
constexpr double kUnitTiles = 2.0, kJoinTiles = 1.0;

// How many parts the items that do not fill the last round over `hold` CTAs are split in, and
// the time of all of them in tiles.
int64_t best_split(int64_t tail, int64_t tiles, int64_t hold, double per_tile, double* cost) {
  int64_t best = 1;
  const int64_t most = tiles / 2 < 1 ? 1 : tiles / 2 < hold ? tiles / 2 : hold;
  for (int64_t s = 1; s <= most; ++s) {
    const double c = (double)cdiv(tail * s, hold) * ((double)cdiv(tiles, s) * per_tile + kUnitTiles) +
                     (s > 1 ? kJoinTiles + 0.05 * (double)s : 0.);
    if (s == 1 || c < *cost) {
      *cost = c;
      best = s;
    }
  }
  return best;
}

Plan make_plan(bool fused, int64_t batch, int64_t lq, int64_t heads, int64_t group, int64_t prefix, int64_t own,
               int64_t hold) {
  Plan p{};
  const int64_t per_request = lq * group;
  const int64_t ptiles = cdiv(prefix, kTileKeys), otiles = cdiv(own, kTileKeys);
  p.fused = fused;
  p.rows = batch * per_request;
  const int64_t tile_rows = fused ? per_request : p.rows;
  p.groups = fused ? heads * batch : heads;
  p.row_tiles = cdiv(tile_rows, kItemRows);
  p.items = fused || prefix > 0 ? p.groups * p.row_tiles : 0;
  p.splits = 1;
  const int64_t tiles = fused ? ptiles + otiles : ptiles;
  // up to 128 rows: two tiles per step
  const double per_tile = tile_rows <= kTileRows ? 0.5 : 1.0;
  p.whole = p.items / hold * hold;
  p.cost = (double)(p.whole / hold) * ((double)tiles * per_tile + kUnitTiles);
  if (p.items > p.whole) {
    double c;
    p.splits = best_split(p.items - p.whole, tiles, hold, per_tile, &c);
    p.cost += c;
  }
  if (p.splits == 1) p.whole = p.items;
  p.blocks = p.whole + (p.items - p.whole) * p.splits;
  if (!fused && own > 0) {
    p.own_tiles = cdiv(per_request, kItemRows);
    const int64_t units = heads * batch * p.own_tiles;
    const double per = per_request <= kTileRows ? 0.5 : 1.0;
    double c;
    p.own_splits = units < hold ? best_split(units, otiles, hold, per, &c) : 1;
    if (units >= hold) c = (double)units / (double)hold * ((double)otiles * per + kUnitTiles);
    p.cost += c + kJoinTiles;
    p.blocks += units * p.own_splits;
  }
  const bool keep = p.own_splits > 0;
  p.slot_tail = keep && p.whole > 0 ? heads * p.rows : 0;
  p.slot_own = p.slot_tail + (p.items - p.whole) * p.splits * kItemRows;
  p.slots = p.slot_own + p.own_splits * heads * p.rows;
  p.joined = keep ? heads * p.rows : (p.items - p.whole) * kItemRows;
  return p;
}

// `hold`: CTAs that the GPU holds at once (one per SM).
Plan plan_attention(int64_t batch, int64_t lq, int64_t heads, int64_t group, int64_t prefix, int64_t own,
                    int64_t hold) {
  const Plan fused = make_plan(true, batch, lq, heads, group, prefix, own, hold);
  if (prefix == 0 || batch == 1) return fused;
  const Plan packed = make_plan(false, batch, lq, heads, group, prefix, own, hold);
  return packed.cost < fused.cost ? packed : fused;
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

template <typename T, int D>
int launch_attention(const CUtensorMap* maps, const AttnArgs& a, const Plan& p, cudaStream_t st, const DeviceInfo* di) {
  const char* op = "shared_prefix_attention";
  auto kern = prefix_attn_kernel<T, D>;
  constexpr int smem = AttnSmem<D>::kBytes;
  static std::atomic<uint64_t> reserved{0};
  if (int s = reserve_smem((const void*)kern, smem, reserved, di, op)) return s;
  if (cudaError_t e = launch_pdl(kern, dim3((unsigned)(p.blocks < di->sm_count ? p.blocks : di->sm_count)), dim3(kAttnThreads), smem, st, maps[0], maps[1],
                                 maps[2], maps[3], a))
    return launch_failed(e, op);
  if (int s = after_launch("prefix_attn_kernel")) return s;
  if (p.joined) {
    if (cudaError_t e = launch_pdl(prefix_attn_join_kernel<T, D>, dim3((unsigned)cdiv(p.joined, 8)), dim3(256), 0, st,
                                   a, p.joined))
      return launch_failed(e, op);
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
  const Plan p = plan_attention(batch, q_len, kv_heads, q_heads / kv_heads, prefix_len, own_len, di->sm_count);
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
  if (!aligned16(out) || !aligned16(q) || !aligned16(k_prefix) || !aligned16(v_prefix) || !aligned16(k_own) ||
      !aligned16(v_own))
    return fail(JO_ERR_ALIGN, "%s: operands must be 16-byte aligned", op);
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
  const Plan p = plan_attention(batch, q_len, kv_heads, q_heads / kv_heads, prefix_len, own_len, di->sm_count);
  if (p.blocks > INT32_MAX || cdiv(p.joined, 8) > INT32_MAX) return fail(JO_ERR_SHAPE, "%s: size too large", op);
  if (p.slots && (!workspace || !aligned16(workspace) || workspace_bytes < p.slots * (head_dim + 1) * 4))
    return fail(JO_ERR_INVALID, "%s: a 16-byte aligned workspace of %lld bytes is needed", op,
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
  a.fused = p.fused;
  a.groups = (int)p.groups;
  a.row_tiles = (int)p.row_tiles;
  a.items = (int)p.items;
  a.whole = (int)p.whole;
  a.splits = (int)p.splits;
  a.own_tiles = (int)p.own_tiles;
  a.own_splits = (int)p.own_splits;
  a.blocks = (int)p.blocks;
  a.rows = p.rows;
  a.slot_tail = p.slot_tail;
  a.slot_own = p.slot_own;
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
