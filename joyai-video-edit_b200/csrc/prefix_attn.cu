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
// belong to, so over the prefix a row of the 128-row tensor-core tile is any (request,
// query, q head of the k/v head's group): the prefix is read once per 128 such rows,
// not once per request.  Two plans (plan_attention):
//   packed  row tiles run across requests; the prefix and each request's own rows are
//           separate work items, joined afterwards;
//   fused   row tiles stay within a request and walk the prefix, then its own rows;
//           taken when that costs hardly more tiles (many queries per request).
// Where there are fewer items than the GPU holds, their keys are split and joined.
//
// One item = one CTA of 6 warps, two CTAs per SM so that one's softmax runs while the
// other's products do:
//   warp 4  TMA producer: K and V tiles of 128 rows (128-byte swizzle);
//   warp 5  tcgen05.mma issuer: S = Q K^T (128 x 128, both operands in shared memory),
//           then O += P V with P from tensor memory and V as it lies ([keys, D], the
//           MN-major operand); owns the 256 tensor-memory columns (S and, in its place,
//           P as 16-bit pairs; O);
//   warps 0-3  load Q, then per tile: S from tensor memory (one row per thread), the
//           running maximum and sum, P back to tensor memory, O rescaled in place.
//
// P is rounded to q's 16-bit type for the tensor cores (its error averages out over the
// keys: 2^-9 relative for bf16, like the output's own rounding); l sums the unrounded p.
#include "tcgen05.cuh"

namespace jo {
namespace {

constexpr int kTileRows = 128;  // queries per tile (UMMA M)
constexpr int kTileKeys = 128;  // keys per tile (UMMA N of S, K of P V)
constexpr int kSoftmaxThreads = 128;
constexpr int kAttnThreads = 192;
constexpr int kTmemColsAttn = 256;  // S / P: 0..127, O: 128..128+D-1
constexpr float kRaise = 8.f;

struct AttnArgs {
  void* out;
  float* lse;
  const void* q;
  int64_t q_b, q_t, q_h;  // element strides
  const int32_t* lens;
  int64_t prefix;
  int batch, lq, heads, group, own;  // heads: of k and v; group: q heads per k/v head; own: rows of the own caches
  int causal;
  float scale_log2;
  // plan
  int fused;
  int row_tiles;   // per k/v head over all requests (packed) or per request (fused)
  int own_tiles;   // packed: row tiles per request
  int whole;       // fused: items that are not split
  int items;       // first kind: packed prefix items, or fused items
  int splits;      // of the items after the first `whole`
  int own_splits;  // packed: of a request's own rows
  float* part_o;   // [slots, D]
  float* part_lse;
  unsigned int* fault;
};

// One CTA's share: rows [row0, row0 + rows) of k/v head h (flat row: (b * Lq + i) * G + g),
// and tiles [first, last) of the prefix's, then the request's own, keys.
struct Item {
  int h, b;  // b: the request of the own rows (-1: none)
  int64_t row0;
  int rows;
  int prefix_tiles;  // tiles of the walk that belong to the prefix
  int first, last;
  int len;       // own rows of b
  int64_t slot;  // partial slot of row0 (-1: final output)
};

__device__ __forceinline__ int own_visible(const AttnArgs& a, int len, int i) {
  return a.causal ? min(len, max(0, len - a.lq + i + 1)) : len;
}

__device__ Item item_of(const AttnArgs& a, int block) {
  Item it;
  const int per_request = a.lq * a.group;
  const int ptiles = (int)((a.prefix + kTileKeys - 1) / kTileKeys);
  int piece = 0, pieces = 1;
  it.slot = -1;
  int t;
  bool own;
  if (a.fused) {
    int item = block;
    if (block >= a.whole) {
      const int tail = a.items - a.whole, j = block - a.whole;
      item = a.whole + j % tail;
      piece = j / tail;
      pieces = a.splits;
      if (pieces > 1) it.slot = ((int64_t)(item - a.whole) * pieces + piece) * kTileRows;
    }
    it.h = item / (a.batch * a.row_tiles);
    const int rest = item - it.h * (a.batch * a.row_tiles);
    it.b = rest / a.row_tiles;
    t = rest - it.b * a.row_tiles;
    it.prefix_tiles = ptiles;
    own = true;
  } else {
    const int64_t rows = (int64_t)a.batch * per_request;
    const int first_kind = a.items * a.splits;
    int slot;
    if (block < first_kind) {
      const int item = block % a.items;
      slot = piece = block / a.items;
      pieces = a.splits;
      it.h = item / a.row_tiles;
      it.b = -1;
      t = item - it.h * a.row_tiles;
      it.row0 = (int64_t)t * kTileRows;
      it.rows = (int)min((int64_t)kTileRows, rows - it.row0);
      it.prefix_tiles = ptiles;
      own = false;
    } else {
      int j = block - first_kind;
      piece = j % a.own_splits;
      pieces = a.own_splits;
      slot = a.splits + piece;
      j /= a.own_splits;
      t = j % a.own_tiles;
      j /= a.own_tiles;
      it.h = j % a.heads;
      it.b = j / a.heads;
      it.prefix_tiles = 0;
      own = true;
    }
    if (own) it.row0 = (int64_t)it.b * per_request + t * kTileRows;
    if (a.splits + a.own_splits > 1) it.slot = ((int64_t)slot * a.heads + it.h) * rows + it.row0;
  }
  int tiles = it.prefix_tiles;
  it.len = 0;
  if (own) {
    it.row0 = (int64_t)it.b * per_request + t * kTileRows;
    it.rows = min(kTileRows, per_request - t * kTileRows);
    it.len = min(max(a.lens[it.b], 0), a.own);
    // the last of the tile's queries sees the most
    tiles += (own_visible(a, it.len, (t * kTileRows + it.rows - 1) / a.group) + kTileKeys - 1) / kTileKeys;
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

template <typename T, int D>
struct AttnSmem {
  static constexpr int kStages = D == 64 ? 2 : 1;  // two CTAs per SM in 227 KB
  static constexpr int kTile = kTileKeys * D * 2;  // bytes of a K or V tile, and of Q
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + kTile;
  static constexpr int kV = kK + kStages * kTile;
  static constexpr int kBars = kV + kStages * kTile;
  static constexpr int kBytes = kBars + 256 + 1024 /*align*/;
};

// 16-bit operands, fp32 accumulator, M = 128.
template <typename T>
constexpr uint32_t attn_idesc(int n, bool b_mn_major) {
  const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kTileRows >> 4) << 24);
}

// Final result or partial of one row: O (this thread's lane) times inv.
template <typename T, int D>
__device__ __forceinline__ void store_row(const AttnArgs& a, const Item& it, int r, uint32_t o_tmem, bool any,
                                          float m, float l) {
  const bool live = r < it.rows;
  const int64_t row = it.row0 + r;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const float lse2 = l == 0.f ? -INFINITY : m + __log2f(l);
  T* out = nullptr;
  float* po = nullptr;
  if (it.slot >= 0) {
    po = a.part_o + (it.slot + r) * D;
    if (live) a.part_lse[it.slot + r] = lse2;
  } else {
    const int per_request = a.lq * a.group;
    const int64_t b = row / per_request;
    const int in = (int)(row - b * per_request), i = in / a.group, g = in - i * a.group;
    const int64_t hq = (int64_t)a.heads * a.group, h = (int64_t)it.h * a.group + g;
    out = reinterpret_cast<T*>(a.out) + ((b * a.lq + i) * hq + h) * D;
    if (live) a.lse[(b * hq + h) * a.lq + i] = lse2 * 0.6931471805599453f;
  }
#pragma unroll 1
  for (int c = 0; c < D / 32; ++c) {
    uint32_t o[32];
    if (any) {
      tmem_ld32(o_tmem + (uint32_t)(c * 32), o);
    } else {
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = 0;
    }
    if (!live) continue;
    float f[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) f[e] = l == 0.f ? 0.f : __uint_as_float(o[e]) * inv;
    if (po != nullptr) {
#pragma unroll
      for (int e = 0; e < 32; e += 4) st_global(po + c * 32 + e, Elt<float>::pack(f + e));
    } else {
#pragma unroll
      for (int e = 0; e < 32; e += 8) st_global(out + c * 32 + e, Elt<T>::pack(f + e));
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kAttnThreads, 2)
    prefix_attn_kernel(const __grid_constant__ CUtensorMap map_kp, const __grid_constant__ CUtensorMap map_vp,
                       const __grid_constant__ CUtensorMap map_ko, const __grid_constant__ CUtensorMap map_vo,
                       const AttnArgs a) {
  using S = AttnSmem<T, D>;
  constexpr int kStages = S::kStages;
  constexpr int kBox = kTileKeys * 128;  // bytes of one 64-element-wide box
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const uint32_t bars = base + S::kBars;
  const uint32_t q_full = bars, s_full = bars + 8, p_full = bars + 16, o_full = bars + 24;
  auto k_full = [&](int s) { return bars + 32 + 8u * s; };
  auto k_empty = [&](int s) { return bars + 32 + 8u * (kStages + s); };
  auto v_full = [&](int s) { return bars + 32 + 8u * (2 * kStages + s); };
  auto v_empty = [&](int s) { return bars + 32 + 8u * (3 * kStages + s); };
  const uint32_t tmem_slot = bars + 32 + 8u * (4 * kStages);
  const int warp = warp_index(), lane = threadIdx.x & 31;

  pdl_wait();  // lens, q, k and v may be the previous kernel's
  pdl_trigger();
  const Item it = item_of(a, blockIdx.x);
  const int n = it.last - it.first;
  if (n == 0) {  // nothing to see: an empty part
    if (threadIdx.x < kSoftmaxThreads) store_row<T, D>(a, it, threadIdx.x, 0, false, 0.f, 0.f);
    return;
  }
  if (threadIdx.x == 0) {
    mbar_init(q_full, kSoftmaxThreads);
    mbar_init(s_full, 1);
    mbar_init(p_full, kSoftmaxThreads);
    mbar_init(o_full, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(k_full(s), 1);
      mbar_init(k_empty(s), 1);
      mbar_init(v_full(s), 1);
      mbar_init(v_empty(s), 1);
    }
    mbar_init_fence();
  }
  if (warp == 5) tmem_alloc(tmem_slot, kTmemColsAttn);
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<uint32_t*>(gbase + (tmem_slot - base));
  const uint32_t tmem_o = tmem + kTileKeys;

  if (warp == 4) {
    if (lane == 0) {
      // ---------------- TMA producer
      auto load = [&](uint32_t dst, bool value, int tile, uint32_t bar) {
        const bool own = tile >= it.prefix_tiles;
        const CUtensorMap* map = value ? (own ? &map_vo : &map_vp) : (own ? &map_ko : &map_kp);
        const int row = (own ? tile - it.prefix_tiles : tile) * kTileKeys;
        mbar_expect_tx(bar, S::kTile);
#pragma unroll
        for (int x = 0; x < D; x += 64) tma_load_4d(dst + (x / 64) * kBox, map, x, it.h, row, own ? it.b : 0, bar);
      };
      int s = 0;
      uint32_t phase = 0;
      int kn = 0, vn = 0;  // tiles issued
      for (int t = 0; t < n; ++t) {
        if (!mbar_wait(k_empty(s), phase ^ 1u, a.fault)) break;
        load(base + S::kK + s * S::kTile, false, it.first + t, k_full(s));
        ++kn;
        if (!mbar_wait(v_empty(s), phase ^ 1u, a.fault)) break;
        load(base + S::kV + s * S::kTile, true, it.first + t, v_full(s));
        ++vn;
        if (++s == kStages) s = 0, phase ^= 1u;
      }
      // every copy issued has landed before the CTA may exit
      for (int j = max(0, kn - kStages); j < kn; ++j) mbar_wait(k_full(j % kStages), (j / kStages) & 1, a.fault);
      for (int j = max(0, vn - kStages); j < vn; ++j) mbar_wait(v_full(j % kStages), (j / kStages) & 1, a.fault);
    }
  } else if (warp == 5) {
    // ---------------- MMA issuer: the warp stays converged and elects one thread per tile
    constexpr uint32_t idesc_s = attn_idesc<T>(kTileKeys, false), idesc_o = attn_idesc<T>(D, true);
    const uint64_t qd = sw128_desc(base + S::kQ), kd0 = sw128_desc(base + S::kK);
    const uint64_t vd0 = sw128_desc_mn(base + S::kV, kBox);
    bool ok = __all_sync(0xffffffffu, mbar_wait(q_full, 0, a.fault));
    int s = 0;
    uint32_t phase = 0;
    for (int t = 0; t < n && ok; ++t) {
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(k_full(s), phase, a.fault)))) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t kd = kd0 + s * (S::kTile >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const int off = ((kk / 4) * kBox + (kk % 4) * 32) >> 4;
          tc_mma_f16_ss(tmem, qd + off, kd + off, idesc_s, kk != 0);
        }
        tc_commit(k_empty(s));
        tc_commit(s_full);
      }
      __syncwarp();
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(v_full(s), phase, a.fault)))) break;
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(p_full, t & 1, a.fault)))) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t vd = vd0 + s * (S::kTile >> 4);
#pragma unroll
        for (int kk = 0; kk < kTileKeys / 16; ++kk)
          tc_mma_f16_ts(tmem_o, tmem + kk * 8, vd + kk * (2048 >> 4), idesc_o, t != 0 || kk != 0);
        tc_commit(v_empty(s));
      }
      __syncwarp();
      if (++s == kStages) s = 0, phase ^= 1u;
    }
    if (elect_one()) tc_commit(o_full);  // also after a failed wait: everything issued has retired
    __syncwarp();
    mbar_wait(o_full, 0, a.fault);
  } else {
    // ---------------- softmax: thread r owns query row r (tensor-memory lane r)
    const int r = threadIdx.x;
    {
      // Q, 16 bytes per step, 128-byte swizzle; rows past the last are zero
      constexpr int kVecs = D / 8;
      const T* q = reinterpret_cast<const T*>(a.q);
      const int per_request = a.lq * a.group;
#pragma unroll 4
      for (int j = r; j < kTileRows * kVecs; j += kSoftmaxThreads) {
        const int row = j / kVecs, c = j - row * kVecs;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row < it.rows) {
          const int64_t flat = it.row0 + row, b = flat / per_request;
          const int in = (int)(flat - b * per_request), i = in / a.group, g = in - i * a.group;
          v = ld_stream(q + b * a.q_b + i * a.q_t + (int64_t)(it.h * a.group + g) * a.q_h + c * 8);
        }
        const uint32_t off = (c / 8) * kBox + row * 128 + (((c & 7) ^ (row & 7)) << 4);
        *reinterpret_cast<uint4*>(gbase + S::kQ + off) = v;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(q_full);
    }
    const bool warp_live = (warp << 5) < it.rows;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    // own rows that this query sees
    int visible = 0;
    if (it.b >= 0) visible = own_visible(a, it.len, (int)((it.row0 + min(r, it.rows - 1)) % (a.lq * a.group)) / a.group);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int t = 0; t < n; ++t) {
      const int tile = it.first + t;
      const bool own = tile >= it.prefix_tiles;
      const int key0 = (own ? tile - it.prefix_tiles : tile) * kTileKeys;
      const int limit = (int)min((int64_t)kTileKeys, (own ? (int64_t)visible : a.prefix) - key0);
      if (!(ok = mbar_wait(s_full, t & 1, a.fault))) break;
      tc_fence_after();
      if (own && key0 + kTileKeys > it.len && it.len < a.own) {
        // cache rows past the request's length hold anything: their p is 0, but 0 * inf is not
        const int st = t % kStages;
        if (!(ok = mbar_wait(v_full(st), (t / kStages) & 1, a.fault))) break;
        if (key0 + r >= it.len) {
#pragma unroll
          for (int x = 0; x < D / 64; ++x)
#pragma unroll
            for (int c = 0; c < 8; ++c)
              *reinterpret_cast<uint4*>(gbase + S::kV + st * S::kTile + x * kBox + r * 128 + c * 16) =
                  make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      if (warp_live) {
        const bool masked = __any_sync(0xffffffffu, limit < kTileKeys);
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t v[64];
          tmem_ld64(tmem + lanes + c * 64, v);
          if (masked) {
#pragma unroll
            for (int e = 0; e < 64; ++e) mx = fmaxf(mx, c * 64 + e < limit ? __uint_as_float(v[e]) : -INFINITY);
          } else {
#pragma unroll
            for (int e = 0; e < 64; ++e) mx = fmaxf(mx, __uint_as_float(v[e]));
          }
        }
        mx *= a.scale_log2;
        const bool raise = mx > m + kRaise;
        float fac = 1.f;
        if (raise) {
          fac = ex2_approx(m - mx);
          m = mx;
        }
        if (t > 0 && __any_sync(0xffffffffu, raise)) {
          // O so far: its last product finished before this tile's S did
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(tmem_o + lanes + c * 32, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fac);
            tmem_st32(tmem_o + lanes + c * 32, o);
          }
        }
        const float shift = m == -INFINITY ? 0.f : m;
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t v[64];
          tmem_ld64(tmem + lanes + c * 64, v);
          uint32_t p[32];
#pragma unroll
          for (int e = 0; e < 64; e += 2) {
            float s0 = __uint_as_float(v[e]), s1 = __uint_as_float(v[e + 1]);
            if (masked) {
              s0 = c * 64 + e < limit ? s0 : -INFINITY;
              s1 = c * 64 + e + 1 < limit ? s1 : -INFINITY;
            }
            const float p0 = ex2_approx(fmaf(s0, a.scale_log2, -shift));
            const float p1 = ex2_approx(fmaf(s1, a.scale_log2, -shift));
            sum += p0 + p1;
            p[e / 2] = pack16<T>(p0, p1);
          }
          tmem_st32(tmem + lanes + c * 32, p);  // over columns of S that have been read
        }
        l = l * fac + sum;
        tmem_st_wait();
      }
      tc_fence_before();
      mbar_arrive(p_full);
    }
    if (ok) ok = mbar_wait(o_full, 0, a.fault);
    tc_fence_after();
    if (ok) store_row<T, D>(a, it, r, tmem_o + lanes, true, m, l);
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_free(tmem, kTmemColsAttn);
  }
}

// Joins the parts of each row by their log2-sum-exps: one warp per row.
template <typename T, int D>
__global__ void __launch_bounds__(256) prefix_attn_join_kernel(const AttnArgs a, int64_t total) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  pdl_wait();
  pdl_trigger();
  if (w >= total) return;
  const int per_request = a.lq * a.group;
  int64_t slot0, step, row;
  int h, parts;
  if (a.fused) {
    const int64_t item = a.whole + w / kTileRows;
    const int r = (int)(w % kTileRows);
    h = (int)(item / (a.batch * a.row_tiles));
    const int rest = (int)(item - (int64_t)h * a.batch * a.row_tiles), b = rest / a.row_tiles, t = rest - b * a.row_tiles;
    if (t * kTileRows + r >= per_request) return;
    row = (int64_t)b * per_request + t * kTileRows + r;
    parts = a.splits;
    slot0 = (w / kTileRows) * parts * kTileRows + r;
    step = kTileRows;
  } else {
    const int64_t rows = (int64_t)a.batch * per_request;
    h = (int)(w / rows);
    row = w - h * rows;
    parts = a.splits + a.own_splits;
    slot0 = w;
    step = a.heads * rows;
  }
  float top = -INFINITY;
  for (int s = lane; s < parts; s += 32) top = fmaxf(top, a.part_lse[slot0 + s * step]);
  top = warp_max(top);
  const float shift = top == -INFINITY ? 0.f : top;
  float o[E] = {}, sum = 0.f;
#pragma unroll 4
  for (int s = 0; s < parts; ++s) {
    const float wgt = ex2_approx(a.part_lse[slot0 + s * step] - shift);
    const float* p = a.part_o + (slot0 + s * step) * D + lane * E;
    sum += wgt;
    if constexpr (E == 4) {
      const float4 v = *reinterpret_cast<const float4*>(p);
      o[0] = fmaf(wgt, v.x, o[0]), o[1] = fmaf(wgt, v.y, o[1]), o[2] = fmaf(wgt, v.z, o[2]), o[3] = fmaf(wgt, v.w, o[3]);
    } else {
      const float2 v = *reinterpret_cast<const float2*>(p);
      o[0] = fmaf(wgt, v.x, o[0]), o[1] = fmaf(wgt, v.y, o[1]);
    }
  }
  const int64_t b = row / per_request, hq = (int64_t)a.heads * a.group;
  const int in = (int)(row - b * per_request), i = in / a.group, g = in - i * a.group;
  const int64_t hh = (int64_t)h * a.group + g;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint32_t* out = reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(a.out) + ((b * a.lq + i) * hq + hh) * D + lane * E);
#pragma unroll
  for (int e = 0; e < E; e += 2) out[e / 2] = pack16<T>(o[e] * inv, o[e + 1] * inv);
  if (lane == 0)
    a.lse[(b * hq + hh) * a.lq + i] = sum == 0.f ? -INFINITY : (top + __log2f(sum)) * 0.6931471805599453f;
}

// ------------------------------------------------------------------ host side
struct Plan {
  bool fused;
  int64_t row_tiles, own_tiles, whole, items, splits, own_splits, blocks, slots, joined;
};

// Which tiles there are, how they are split, and what has to be joined.  `hold`: CTAs
// that the GPU holds at once (two per SM).
Plan plan_attention(int64_t batch, int64_t lq, int64_t heads, int64_t group, int64_t prefix, int64_t own,
                    int64_t hold) {
  Plan p{};
  const int64_t per_request = lq * group, rows = batch * per_request;
  const int64_t ptiles = cdiv(prefix, kTileKeys), otiles = cdiv(own, kTileKeys);
  const int64_t packed = cdiv(rows, kTileRows), split_rows = cdiv(per_request, kTileRows);
  // Tiles of work: packed, and with row tiles that stay within a request.  The packed plan
  // also writes and reads every row's parts, which costs about as much as two tiles.
  const int64_t cost_packed = packed * (ptiles + 2) + batch * split_rows * (otiles + 2);
  const int64_t cost_fused = batch * split_rows * (ptiles + otiles);
  p.fused = cost_fused <= cost_packed;
  if (prefix == 0) p.fused = true;  // one kind of key: no parts unless split
  if (prefix > 0 && own == 0) p.fused = batch == 1;
  if (p.fused) {
    p.row_tiles = split_rows;
    p.items = heads * batch * split_rows;
    p.whole = p.items / hold * hold;
    const int64_t tail = p.items - p.whole;
    p.splits = 1;
    if (tail) {
      p.splits = hold / tail;
      const int64_t most = cdiv(ptiles + otiles, 2);  // two tiles per part at least
      if (p.splits > most) p.splits = most > 0 ? most : 1;
    }
    if (p.splits <= 1) {
      p.splits = 1;
      p.whole = p.items;
    }
    p.blocks = p.whole + (p.items - p.whole) * p.splits;
    p.slots = p.splits > 1 ? (p.items - p.whole) * p.splits * kTileRows : 0;
    p.joined = p.splits > 1 ? (p.items - p.whole) * kTileRows : 0;
  } else {
    p.row_tiles = packed;
    p.own_tiles = split_rows;
    p.items = prefix > 0 ? heads * packed : 0;
    p.splits = 0;
    if (p.items) {
      const int64_t most = cdiv(ptiles, 2);
      p.splits = hold / p.items;
      if (p.splits > most) p.splits = most;
      if (p.splits < 1) p.splits = 1;
    }
    const int64_t own_items = own > 0 ? heads * batch * split_rows : 0;
    p.own_splits = 0;
    if (own_items) {
      const int64_t most = cdiv(otiles, 4);
      p.own_splits = hold / own_items;
      if (p.own_splits > most) p.own_splits = most;
      if (p.own_splits < 1) p.own_splits = 1;
    }
    p.blocks = p.items * p.splits + own_items * p.own_splits;
    const bool parts = p.splits + p.own_splits > 1;
    p.slots = parts ? (p.splits + p.own_splits) * heads * rows : 0;
    p.joined = parts ? heads * rows : 0;
  }
  return p;
}

int check_sizes(const char* op, int64_t batch, int64_t lq, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                int64_t prefix, int64_t own) {
  if (batch < 0 || lq < 0 || prefix < 0 || own < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads)
    return fail(JO_ERR_SHAPE, "%s: bad sizes (q heads must be a multiple of the k/v heads)", op);
  if (head_dim != 64 && head_dim != 128) return fail(JO_ERR_SHAPE, "%s: head_dim must be 64 or 128", op);
  const int64_t most = INT32_MAX / 2;
  if (batch > most || lq > most || prefix > most || own > most || q_heads > most || lq * (q_heads / kv_heads) > most ||
      batch * q_heads > most || batch * lq > most || batch * lq * q_heads > (int64_t)1 << 38)
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
  constexpr int smem = AttnSmem<T, D>::kBytes;
  static std::atomic<uint64_t> reserved{0};
  if (int s = reserve_smem((const void*)kern, smem, reserved, di, op)) return s;
  if (cudaError_t e = launch_pdl(kern, dim3((unsigned)p.blocks), dim3(kAttnThreads), smem, st, maps[0], maps[1],
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
  const Plan p = plan_attention(batch, q_len, kv_heads, q_heads / kv_heads, prefix_len, own_len, 2 * di->sm_count);
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
  const Plan p = plan_attention(batch, q_len, kv_heads, q_heads / kv_heads, prefix_len, own_len, 2 * di->sm_count);
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
  a.prefix = prefix_len;
  a.batch = (int)batch;
  a.lq = (int)q_len;
  a.heads = (int)kv_heads;
  a.group = (int)(q_heads / kv_heads);
  a.own = (int)own_len;
  a.causal = causal;
  a.scale_log2 = scale * kLog2E;
  a.fused = p.fused;
  a.row_tiles = (int)p.row_tiles;
  a.own_tiles = (int)p.own_tiles;
  a.whole = (int)p.whole;
  a.items = (int)p.items;
  a.splits = (int)p.splits;
  a.own_splits = (int)p.own_splits;
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
