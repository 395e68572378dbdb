// Attention of single tokens of rows whose first slots lie in the same pages (b200p_paged_attn_shared); part of paged_attn.cu.
//
//   o = sum_j p_j v_j over a group's shared slots and the row's own ones: either part leaves its maximum m, sum l and unnormalised output, and
//   o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i,  m = max m_i
//
// The shared slots are read once for a tile of up to PS_ROWS query heads of the group's tokens, instead of once for every token: products of many rows,
// which the matrix instructions bound and not the memory.  The own slots go through paged_attn_kernel behind the shared ones, and a third launch joins the
// parts of both.
#pragma once
#include "rowgroups.cuh"

namespace b200p {

constexpr int PS_HEAD = 8;                       // floats before a part's outputs: maximum, sum (whole sectors of 32 bytes behind them)
constexpr int PS_ROWS = 256;                     // query rows of a tile: tokens x query heads of a key head
constexpr int PS_HALF = 128, PS_WARPS = 8;       // of which paged_prefix_kernel takes 128 at a time, 16 to a warp

struct PagedPrefix {
  const void *q, *k, *v;
  PageTable pt;
  const int32_t *t_row, *t_slot, *index, *prefix;
  RowGroups plan;
  int M, H, G, groups;
  float scale_log2e;
  uint64_t inv_tpp;
  int tpp;
  // [M H + CTAs * rows of an item, PS_HEAD + D] parts: of a query row of an item in CTA c at the row's place among all (row0 and its place in the item)
  // + c * rows of an item.  (Items lie on a line and every CTA has a run of it: a part begins behind the last row of the one before.)
  float* rec;
  int4* info;            // [M] the tile's first place in the plan's order, the token's place in it (in the upper half the tile's tokens), the tile's first unit,
                         // units of an item (0: the token reads by itself)
  unsigned* total;       // units of all
  int* wait_word;
  int box;               // keys that one copy brings: they lie in one page
  int few;               // half of the GPU's SMs
  int64_t rec_rows;      // that rec has room for
};

// The units (KT shared keys of an item: the rows of a tile, or of a half of it, and a key head) lie end to end and every CTA has an equal part of them, as in
// paged_attn_kernel.
struct PrefixShares {
  unsigned n, q, r;
  // A CTA has some 8 us to set up and to leave its part, a unit takes 1.6: four units each, unless half of the GPU is enough for fewer.  What is left of
  // the GPU begins with the own slots.
  __device__ PrefixShares(unsigned U, unsigned ctas, unsigned few) : n(min(ctas, max(U / 4, min(U, few)))) {
    q = n ? U / n : 1;
    r = U - q * n;
  }
  __device__ unsigned begin(unsigned c) const { return c < n ? c * q + min(c, r) : q * n + r; }
  __device__ unsigned of(unsigned u) const { return u < r * (q + 1) ? u / (q + 1) : r + (u - r * (q + 1)) / q; }
};

// The slots that a token has in common with its group (of those that the table has).  0: it belongs to none, or stands before their end and reads what it
// sees by itself.
__device__ __forceinline__ int shared_slots(const int32_t* index, const int32_t* prefix, int groups, const PageTable& pt, int t, int seen) {
  const int g = index[t];
  if ((unsigned)g >= (unsigned)groups) return 0;
  const int n = min(max(prefix[g], 0), table_slots(pt));
  return seen < n ? 0 : n;
}

// A run of an item's units.
struct PrefixRun {
  int4 tile;
  int ti, n, common, table_row;        // the tile, units of an item, shared slots, the table row that has their pages
  int g, half, first, last, rows;      // key head, half, units [first, last), query rows of the tile
  int64_t row0;                        // the item's first query row among those of all items
};

// SPLIT: an item has half of a tile's rows (where it has more than that), else all of them.
template <int KT, bool SPLIT>
struct PrefixCursor {
  unsigned u, end, base;
  int ti;
  static __device__ __forceinline__ void look(const PagedPrefix& a, int i, PrefixRun& r) {
    r.tile = a.plan.tile(i);
    r.ti = i;
    r.common = min(max(a.prefix[r.tile.x], 0), table_slots(a.pt));
    r.table_row = -1;                                               // that of the first member that holds the shared slots
    for (int k = 0; k < r.tile.z && r.table_row < 0; ++k) {
      const int t = a.plan.order()[r.tile.y + k], row = a.t_row[t];
      if (row >= 0 && row < a.pt.rows && slots_seen(a.pt, a.t_slot[t]) >= r.common) r.table_row = row;
    }
    r.n = r.table_row < 0 ? 0 : (r.common + KT - 1) / KT;
    r.rows = r.tile.z * (a.H / a.G);
  }
  static __device__ __forceinline__ int halves(const PrefixRun& r) { return SPLIT && r.rows > PS_HALF ? 2 : 1; }
  static __device__ __forceinline__ unsigned units(const PagedPrefix& a, const PrefixRun& r) { return (unsigned)r.n * a.G * halves(r); }
  __device__ bool next(const PagedPrefix& a, PrefixRun& r) {
    if (u >= end) return false;
    if (r.ti != ti) look(a, ti, r);                                 // (the plan has looked at the first)
    while (u - base >= units(a, r)) {
      base += units(a, r);
      look(a, ++ti, r);
    }
    const int at = (int)((u - base) / (unsigned)r.n), h = halves(r);
    r.g = at / h, r.half = at - r.g * h;
    r.first = (int)(u - base) - at * r.n, r.last = min(r.n, r.first + (int)(end - u));
    r.row0 = (int64_t)r.tile.y * a.H + (int64_t)r.g * r.rows + PS_HALF * r.half;
    u += r.last - r.first;
    return true;
  }
  // what the join has to know of the tile's tokens, by the threads of the CTA that begins its first item
  __device__ __forceinline__ void tell(const PagedPrefix& a, const PrefixRun& r, int thread) const {
    if (r.g == 0 && r.half == 0 && r.first == 0 && thread < r.tile.z) {
      const int t = a.plan.order()[r.tile.y + thread];
      const bool shares = slots_seen(a.pt, a.t_slot[t]) >= r.common;
      a.info[t] = make_int4(r.tile.y, thread | r.tile.z << 16, (int)base, shares ? r.n : 0);
    }
  }
};

// By the whole CTA: units of all tiles and this CTA's part.
struct PrefixPlan {
  unsigned sum[16], base;
  PrefixRun first;
};
template <int THREADS, int KT, bool SPLIT>
__device__ __forceinline__ PrefixCursor<KT, SPLIT> prefix_plan(const PagedPrefix& a, PrefixPlan& s, PrefixRun& first) {
  using C = PrefixCursor<KT, SPLIT>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = a.plan.tiles(), chunk = (tiles + THREADS - 1) / THREADS;
  const int i0 = min(tiles, (int)threadIdx.x * chunk), i1 = min(tiles, i0 + chunk);
  PrefixRun r;
  unsigned mine = 0;
  for (int i = i0; i < i1; ++i) {
    C::look(a, i, r);
    mine += C::units(a, r);
  }
  unsigned before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned x = __shfl_up_sync(~0u, before, o);
    if (lane >= o) before += x;
  }
  if (lane == 31) s.sum[warp] = before;
  __syncthreads();
  before -= mine;
  unsigned U = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += s.sum[w];
    U += s.sum[w];
  }
  const PrefixShares sh(U, gridDim.x, a.few);
  C c;
  c.u = sh.begin(blockIdx.x), c.end = sh.begin(blockIdx.x + 1);
  for (int i = i0; i < i1; ++i) {
    if (i0 + 1 < i1) C::look(a, i, r);
    const unsigned n = C::units(a, r);
    if (c.u - before < n) s.first = r, s.base = before;
    if (n == 0 && blockIdx.x == 0)                                  // nobody will go through this tile
      for (int k = 0; k < r.tile.z; ++k) a.info[a.plan.order()[r.tile.y + k]] = make_int4(0, 0, 0, 0);
    before += n;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.total = U;
  __syncthreads();
  first = s.first;                                                  // (where there is nothing to do nobody looks at it)
  c.ti = first.ti, c.base = s.base;
  return c;
}

template <typename T, int D>
struct PrefixTile {
  static constexpr int KT = D > 128 ? 32 : 64, STAGES = 3, CHUNKS = D / 8, PIECES = CHUNKS % 8 ? (CHUNKS | 1) : CHUNKS, LINE = PIECES * 16;
  static constexpr int KV_BYTES = KT * LINE, STAGE = 2 * KV_BYTES, Q_BYTES = PS_HALF * LINE, SMEM = Q_BYTES + STAGES * STAGE;
  static __device__ __forceinline__ uint32_t at(int line, int c) { return (uint32_t)(line * LINE + ((CHUNKS % 8 ? c : c ^ (line & 7)) << 4)); }
};

template <typename T, int D>
__global__ void __launch_bounds__(PS_WARPS * 32, 1)
paged_prefix_kernel(const __grid_constant__ PagedPrefix a) {
  using P = PrefixTile<T, D>;
  constexpr int KT = P::KT, THREADS = PS_WARPS * 32, CHUNKS = P::CHUNKS, NP = KT / 16;
  // f16: weights up to 2^14 and not 1, so that small ones keep their bits
  constexpr float SHIFT = std::is_same<T, __half>::value ? 14.f : 0.f;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ PrefixPlan s_plan;
  __shared__ int s_token[PS_HALF];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, qr = lane >> 2, qc = lane & 3, mat = lane >> 3, r8 = lane & 7;
  const int per = a.H / a.G;
  pdl_wait();
  pdl_launch_dependents();
  PrefixRun run;
  PrefixCursor<KT, true> cursor = prefix_plan<THREADS, KT, true>(a, s_plan, run);
  const uint32_t qs = (uint32_t)__cvta_generic_to_shared(smem), ring = qs + P::Q_BYTES;
  while (cursor.next(a, run)) {
    const int first = run.first, last = run.last, g = run.g, common = run.common, rows = run.rows - PS_HALF * run.half, r0 = PS_HALF * run.half;
    const int32_t* table = a.pt.table + (int64_t)run.table_row * a.pt.width;
    cursor.tell(a, run, threadIdx.x);
    __syncthreads();                                                // the item before this one is done with shared memory
    if ((int)threadIdx.x < PS_HALF) {
      const int k = (r0 + (int)threadIdx.x) / per;
      s_token[threadIdx.x] = k < run.tile.z ? a.plan.order()[run.tile.y + k] : -1;
    }
    __syncthreads();
    for (int x = threadIdx.x; x < PS_HALF * CHUNKS; x += THREADS) {
      const int r = x / CHUNKS, c = x - r * CHUNKS, token = s_token[r];
      const uint4* src = reinterpret_cast<const uint4*>(a.q) + ((int64_t)(token < 0 ? 0 : token) * a.H + (int64_t)g * per + (r0 + r) % per) * CHUNKS + c;
      cp_async16(qs + P::at(r, c), src, token >= 0);
    }
    // 16 keys at a time lie in one page; their page is looked up a tile ahead
    int id[NP];
    unsigned paged = 0;                                             // of every stage's 16 keys each: whether they have a page
    auto seek = [&](int tile_u) {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int kt = tile_u * NP + i, index = (int)((uint64_t)(unsigned)kt * a.inv_tpp >> 36);
        id[i] = tile_u < last && kt * 16 < common ? table[index] : -1;
      }
    };
    auto issue = [&](int tile_u) {
      if (tile_u < last) {
        const int stage = tile_u % P::STAGES;
        const uint32_t ks = ring + (uint32_t)stage * P::STAGE;
        paged &= ~(((1u << NP) - 1u) << (NP * stage));
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int kt = tile_u * NP + i, index = (int)((uint64_t)(unsigned)kt * a.inv_tpp >> 36);
          const bool page = (unsigned)id[i] < (unsigned)a.pt.P;
          const int64_t line = (((int64_t)(page ? id[i] : 0) * a.G + g) * a.tpp + (page ? kt - index * a.tpp : 0)) * 16;
          paged |= (page ? 1u : 0u) << (NP * stage + i);
          if (!page && kt * 16 < common && threadIdx.x == 0) atomicAdd(&g_paged_attn_fault, 1u);
#pragma unroll
          for (int x = threadIdx.x; x < 16 * CHUNKS; x += THREADS) {
            const int key = x / CHUNKS, c = x - key * CHUNKS;
            const bool ok = page && kt * 16 + key < common;
            const int64_t from = line * CHUNKS + (ok ? x : 0);
            cp_async16(ks + P::at(16 * i + key, c), reinterpret_cast<const uint4*>(a.k) + from, ok);
            cp_async16(ks + P::KV_BYTES + P::at(16 * i + key, c), reinterpret_cast<const uint4*>(a.v) + from, ok);
          }
        }
        seek(tile_u + 1);
      }
      cp_async_commit();
    };
    seek(first);
    for (int s = 0; s < P::STAGES - 1; ++s) issue(first + s);

    float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    const bool works = 16 * warp < rows;
#pragma unroll 1
    for (int v = first; v < last; ++v) {
      cp_async_wait<P::STAGES - 2>();
      __syncthreads();
      const unsigned paged_now = paged >> (NP * (v % P::STAGES)) & ((1u << NP) - 1u);
      issue(v + P::STAGES - 1);                                     // (into the stage that all were done with at this barrier)
      if (!works) continue;
      const uint32_t ks = ring + (uint32_t)(v % P::STAGES) * P::STAGE, vs = ks + P::KV_BYTES;
      float s[KT / 8][4];
#pragma unroll
      for (int j = 0; j < KT / 8; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t qf[4];
        ldsm_x4(qs + P::at(16 * warp + r8 + 8 * (mat & 1), 2 * k + (mat >> 1)), qf);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          uint32_t kf[4];
          ldsm_x4(ks + P::at(16 * j + r8 + 8 * (mat >> 1), 2 * k + (mat & 1)), kf);
          mma16816<T>(s[2 * j], qf, kf[0], kf[1]);
          mma16816<T>(s[2 * j + 1], qf, kf[2], kf[3]);
        }
      }
      const unsigned pages = paged_now;
      const bool whole = (v + 1) * KT <= common && pages == (1u << NP) - 1u;
      float f[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float t = -INFINITY;
#pragma unroll
        for (int j = 0; j < KT / 8; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = s[j][2 * h + e] * a.scale_log2e;
            if (!whole && (v * KT + 8 * j + 2 * qc + e >= common || !(pages >> (j / 2) & 1u))) x = -INFINITY;
            s[j][2 * h + e] = x;
            t = fmaxf(t, x);
          }
        t = fmaxf(t, __shfl_xor_sync(~0u, t, 1));
        t = fmaxf(t, __shfl_xor_sync(~0u, t, 2));
        t = fmaxf(t - SHIFT, m[h]);
        const float ref = t == -INFINITY ? 0.f : t;
        f[h] = raise2(m[h] - ref);
        m[h] = t;
        l[h] *= f[h];
#pragma unroll
        for (int j = 0; j < KT / 8; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) s[j][2 * h + e] = raise2(s[j][2 * h + e] - ref);
      }
      if (__any_sync(~0u, f[0] != 1.f || f[1] != 1.f)) {            // a maximum grew (or is not a number)
#pragma unroll
        for (int j = 0; j < D / 8; ++j) o[j][0] *= f[0], o[j][1] *= f[0], o[j][2] *= f[1], o[j][3] *= f[1];
      }
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        // The weights multiply the values as two 16-bit numbers each, the rounded weight and what it lost, as in paged_attn_kernel, so that the output
        // carries its own rounding only.  (As one number a weight is off by half a step of its type: 1.3 times the output's rounding alone in bf16.)
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = s[2 * j + (e >> 1)][2 * (e & 1)], y = s[2 * j + (e >> 1)][2 * (e & 1) + 1];
          l[e & 1] += x + y;
          hi[e] = pack2<T>(x, y);
          const T* p = reinterpret_cast<const T*>(&hi[e]);
          lo[e] = pack2<T>(x - Tr<T>::to_f(p[0]), y - Tr<T>::to_f(p[1]));
        }
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          uint32_t vf[4];
          ldsm_x4_trans(vs + P::at(16 * j + r8 + 8 * (mat & 1), 2 * k + (mat >> 1)), vf);
          mma16816<T>(o[2 * k], hi, vf[0], vf[1]);
          mma16816<T>(o[2 * k + 1], hi, vf[2], vf[3]);
          mma16816<T>(o[2 * k], lo, vf[0], vf[1]);
          mma16816<T>(o[2 * k + 1], lo, vf[2], vf[3]);
        }
      }
    }
    cp_async_wait<0>();
    // ---- the part ---------------------------------------------------------------------------------------------------------------
    if (works) {
      float* rec = a.rec + (run.row0 + (int64_t)blockIdx.x * PS_HALF) * (D + PS_HEAD);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float sum = l[h];
        sum += __shfl_xor_sync(~0u, sum, 1);
        sum += __shfl_xor_sync(~0u, sum, 2);
        float* row = rec + (16 * warp + 8 * h + qr) * (D + PS_HEAD);
        if (16 * warp + 8 * h + qr >= rows) continue;               // (another item's place)
        if (qc == 0) *reinterpret_cast<float2*>(row) = make_float2(m[h], sum);
#pragma unroll
        for (int j = 0; j < D / 8; ++j) *reinterpret_cast<float2*>(row + PS_HEAD + 8 * j + 2 * qc) = make_float2(o[j][2 * h], o[j][2 * h + 1]);
      }
    }
  }
}

// The parts of the shared slots and of the own ones become a token's outputs: W warps per query head, a CTA of 8.
template <typename T, int NQ, int ROWS, int W>
__global__ void __launch_bounds__(256)
paged_shared_join_kernel(const __grid_constant__ PagedAttn a, const __grid_constant__ PagedPrefix p, int prefix_ctas, int item_rows) {
  __shared__ float2 s_ml[8];
  __shared__ float4 s_o[W > 1 ? 8 : 1][32 * NQ];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = a.D, per = a.H / a.G, blocks = (per + ROWS - 1) / ROWS, t = blockIdx.y;
  const int head = (int)blockIdx.x * (8 / W) + warp / W, g = head / per, r = head - g * per;
  pdl_wait();
  const bool here = head < a.H;
  const int64_t line = ((int64_t)t * a.G + (here ? g : 0)) * blocks + (here ? r / ROWS : 0);
  const int row = a.t_row[t], group = p.index[t];
  const uint2 parts = a.parts[line];
  const int4 info = p.info[t];                                      // (written for tokens of groups)
  const unsigned total = *p.total;
  if (row < 0 || row >= a.pt.rows) return;
  int heads = 0, c0 = 0;                                            // parts of the shared slots
  int64_t row0 = 0;                                                 // its row in the first of them
  if ((unsigned)group < (unsigned)p.groups && info.w > 0) {
    const PrefixShares sh(total, prefix_ctas, p.few);
    const int rows = (info.y >> 16) * per, halves = item_rows == PS_HALF && rows > PS_HALF ? 2 : 1;
    const int at = (info.y & 0xffff) * per + r, half = halves > 1 && at >= PS_HALF ? 1 : 0;
    const unsigned u = (unsigned)info.z + (unsigned)((g * halves + half) * info.w);
    c0 = (int)sh.of(u);
    heads = (int)sh.of(u + info.w - 1) - c0 + 1;
    row0 = (int64_t)info.x * a.H + (int64_t)g * rows + at + (int64_t)c0 * item_rows;
    // (a plan that is not the index's leaves what it likes here: wrong, but nothing behind the workspace is read)
    if (heads > prefix_ctas || row0 < 0 || row0 + (int64_t)(heads - 1) * item_rows >= p.rec_rows) heads = 0;
  }
  const int all = here ? heads + (int)parts.y : 0;
  auto at = [&](int i) -> const float* {                            // its outputs; maximum and sum stand before them
    if (i < heads) return p.rec + (row0 + (int64_t)i * item_rows) * (D + PS_HEAD) + PS_HEAD;
    if (parts.y == 1) return a.whole + ((int64_t)t * a.H + head) * (D + 4) + 4;
    return part_at(a, parts.x, i - heads, ROWS, r % ROWS) + 4;
  };
  constexpr int AHEAD = 4;
  float M = -INFINITY, L = 0.f;
  float4 acc[NQ];
#pragma unroll
  for (int x = 0; x < NQ; ++x) acc[x] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int i0 = warp % W; i0 < all; i0 += AHEAD * W) {
    float2 ml[AHEAD];
    float4 y[AHEAD][NQ];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = i0 + k * W;
      const bool in = i < all;
      const float* from = at(in ? i : i0);
      ml[k] = in ? *reinterpret_cast<const float2*>(from - (i < heads ? PS_HEAD : 4)) : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int x = 0; x < NQ; ++x)
        y[k][x] = in && 4 * lane + 128 * x < D ? *reinterpret_cast<const float4*>(from + 4 * lane + 128 * x) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float top = M;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) top = fmaxf(top, ml[k].x);
    const float ref = top == -INFINITY ? 0.f : top, f = raise2(M - ref);
    M = top;
    L *= f;
#pragma unroll
    for (int x = 0; x < NQ; ++x) acc[x].x *= f, acc[x].y *= f, acc[x].z *= f, acc[x].w *= f;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const float w = raise2(ml[k].x - ref);
      L += ml[k].y * w;
#pragma unroll
      for (int x = 0; x < NQ; ++x) acc[x].x += y[k][x].x * w, acc[x].y += y[k][x].y * w, acc[x].z += y[k][x].z * w, acc[x].w += y[k][x].w * w;
    }
  }
  if constexpr (W > 1) {
    if (lane == 0) s_ml[warp] = make_float2(M, L);
#pragma unroll
    for (int x = 0; x < NQ; ++x) s_o[warp][lane + 32 * x] = acc[x];
    __syncthreads();
    if (warp % W) return;                                           // the first warp of a head goes on
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, s_ml[warp + w].x);
    const float ref = top == -INFINITY ? 0.f : top;
    L = 0.f;
#pragma unroll
    for (int x = 0; x < NQ; ++x) acc[x] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = raise2(s_ml[warp + w].x - ref);
      L += s_ml[warp + w].y * f;
#pragma unroll
      for (int x = 0; x < NQ; ++x) {
        const float4 y = s_o[warp + w][lane + 32 * x];
        acc[x].x += y.x * f, acc[x].y += y.y * f, acc[x].z += y.z * f, acc[x].w += y.w * f;
      }
    }
  }
  if (!here) return;
  const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
  for (int x = 0; x < NQ; ++x) {
    const int d = 4 * lane + 128 * x;
    if (d < D)
      store_row4<T>(reinterpret_cast<T*>(a.out) + ((int64_t)t * a.H + head) * D, d, make_float4(acc[x].x * inv, acc[x].y * inv, acc[x].z * inv, acc[x].w * inv),
                    a.out_perm);
  }
}

}  // namespace b200p
