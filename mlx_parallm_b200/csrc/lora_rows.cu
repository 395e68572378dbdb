// Low-rank updates with an adapter of its own for every row (b200p_row_groups, b200p_lora_rows): requests under many adapters in one batch.
//
//   y[m, columns of target t] += s_i ((x_m A_{i,t}^T) B_{i,t}^T),   i = the row's adapter; rows without one stay as they are
//
// The rows are put in the order of their adapters once per batch (row_groups_kernel); the layers then go by tiles of 16 or 128 rows of one adapter.
// A cluster of CTAs has a tile: every CTA takes a part of K for z = x A^T, the parts meet through distributed shared memory, and every CTA has all of
// z for its part of the columns.  So both products are one launch, an adapter is read once for a tile, and even a single row has eight SMs.
// z is fp32; for the second product its rows are scaled by a power of two and split into 16-bit numbers: two of f16, which carry 22 bits of a z that is not below
// 2^-17 of its row's largest (2^-39 of that below), or three of bf16, 24 bits of any, two and 16 where y is bf16 itself.  So the update is as exact as its sums
// (for bf16 y as y's rounding asks for); it is added to y in fp32 and rounded once where y is 16-bit.
#include <cooperative_groups.h>

#include <atomic>

#include "attn_tc.cuh"
#include "mma_util.cuh"
#include "rowgroups.cuh"

namespace cg = cooperative_groups;

namespace b200p {

int sm_count();

// ------------------------------------------------------------------------------------------------ the plan
constexpr int RG_WARPS = 16;

// A stable counting sort by one CTA: every warp counts its run of rows by group, the counts become places, and the warps go over their rows again.
// (8000 rows of 7 groups: a launch per batch, not per layer.)
__global__ void __launch_bounds__(RG_WARPS * 32)
row_groups_kernel(const int32_t* index, int32_t* plan, int M, int groups, int tile) {
  extern __shared__ int s_count[];               // [RG_WARPS][groups]
  __shared__ int s_begin[RG_GROUPS], s_tile[RG_GROUPS], s_size[RG_GROUPS], s_bad;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  for (int i = threadIdx.x; i < RG_WARPS * groups; i += RG_WARPS * 32) s_count[i] = 0;
  if (threadIdx.x == 0) s_bad = 0;
  __syncthreads();
  const int run = (M + RG_WARPS * 32 - 1) / (RG_WARPS * 32) * 32, r0 = min(M, warp * run), r1 = min(M, r0 + run);
  int* count = s_count + warp * groups;
  for (int base = r0; base < r1; base += 32) {
    const int i = base + lane, g = i < r1 ? index[i] : -1;
    const unsigned same = __match_any_sync(~0u, g), bad = __ballot_sync(~0u, g >= groups);
    if (g >= 0 && g < groups && lane == __ffs(same) - 1) count[g] += __popc(same);
    if (bad && lane == 0) atomicAdd(&s_bad, __popc(bad));
    __syncwarp();
  }
  __syncthreads();
  for (int g = threadIdx.x; g < groups; g += RG_WARPS * 32) {
    int sum = 0;
    for (int w = 0; w < RG_WARPS; ++w) {
      const int n = s_count[w * groups + g];
      s_count[w * groups + g] = sum;
      sum += n;
    }
    s_size[g] = sum;
  }
  __syncthreads();
  if (warp == 0) {
    int rows = 0, tiles = 0;
    for (int base = 0; base < groups; base += 32) {
      const int g = base + lane, n = g < groups ? s_size[g] : 0, k = (n + tile - 1) / tile;
      int a = n, b = k;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(~0u, a, o), y = __shfl_up_sync(~0u, b, o);
        if (lane >= o) a += x, b += y;
      }
      if (g < groups) s_begin[g] = rows + a - n, s_tile[g] = tiles + b - k;
      rows += __shfl_sync(~0u, a, 31), tiles += __shfl_sync(~0u, b, 31);
    }
    if (lane == 0) plan[0] = tiles, plan[1] = rows, plan[2] = s_bad, plan[3] = tile;
  }
  __syncthreads();
  int32_t* order = plan + RG_HEAD;
  int4* tiles = reinterpret_cast<int4*>(order + (M + 3) / 4 * 4);
  for (int g = threadIdx.x; g < groups; g += RG_WARPS * 32)
    for (int k = 0; k * tile < s_size[g]; ++k) tiles[s_tile[g] + k] = make_int4(g, s_begin[g] + k * tile, min(tile, s_size[g] - k * tile), s_begin[g]);
  for (int base = r0; base < r1; base += 32) {
    const int i = base + lane, g = i < r1 ? index[i] : -1;
    const bool in = g >= 0 && g < groups;
    const unsigned same = __match_any_sync(~0u, g);
    if (in) order[s_begin[g] + count[g] + __popc(same & ((1u << lane) - 1u))] = i;
    __syncwarp();
    if (in && lane == __ffs(same) - 1) count[g] += __popc(same);
    __syncwarp();
  }
}

// ------------------------------------------------------------------------------------------------ the update
constexpr int LW_WARPS = 8, LW_THREADS = LW_WARPS * 32;
// targets, CTAs of a tile, ranks of a target at most
constexpr int LW_TARGETS = 4, LW_CLUSTER = 8, LW_RANK = 64, LW_RANKS = LW_RANK * LW_TARGETS;

struct LoraRows {
  const void *x, *a, *b;
  const float* scales;
  void* y;
  RowGroups plan;
  int64_t ldx, ldy;
  int K, R, N, targets, steps;                   // rank of a target, columns of all targets, 32 of K each
  int sub;                                       // 16-row tiles of a tile of the plan
  int* wait_word;
  int col0[LW_TARGETS], start[LW_TARGETS + 1], tile0[LW_TARGETS + 1];      // first column of y, of b; first run of 16 columns
};

// (two bf16 numbers where y is rounded to bf16: 16 bits of z against y's 8)
template <typename T, typename YT> struct LwParts { static constexpr int N = std::is_same<T, __nv_bfloat16>::value && sizeof(YT) == 4 ? 3 : 2; };
// Shared floats of a row: the warps' parts of z, of which the first becomes this CTA's, and the split z behind that.
template <typename T, typename YT>
__host__ __device__ constexpr int lw_row_floats(int ranks) {
  const int split = LwParts<T, YT>::N * (ranks + 8) / 2 + ranks;
  return split > LW_WARPS * 32 ? split : LW_WARPS * 32;
}

// up = 2^e, down = 2^-e with top * down in [1, 2), for f16 in [2^14, 2^15): what is much smaller than the row's largest keeps its bits too, above the smallest
// numbers of f16.  1 for a row of zeros or one that is not finite.
template <typename T>
__device__ __forceinline__ void lw_scale(float top, float& up, float& down) {
  constexpr uint32_t LIFT = std::is_same<T, __half>::value ? 14 : 0;
  const uint32_t e = __float_as_uint(top) >> 23;
  const bool plain = e < LIFT + 1 || e > 252;
  down = plain ? 1.f : __uint_as_float((254u + LIFT - e) << 23), up = plain ? 1.f : __uint_as_float((e - LIFT) << 23);
}

__device__ __forceinline__ void red_add4(float* p, float a, float b, float c, float d) {
  asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}

// A run of 16 columns: a lane's four are neighbours, as the two products' column j is 4 (j / 2) + j % 2 and two further.
struct LwRun {
  int target, c0, width;
  __device__ __forceinline__ LwRun(const LoraRows& p, int run) : target(0) {
#pragma unroll
    for (int k = 1; k < LW_TARGETS; ++k)
      if (k < p.targets && run >= p.tile0[k]) target = k;
    width = p.start[target + 1] - p.start[target];
    c0 = (run - p.tile0[target]) * 16;
  }
};
template <typename T, int KS>
__device__ __forceinline__ void lw_load(const LoraRows& p, const T* b, int run, int run1, uint2 (&w)[KS][2]) {
  if (run >= run1) return;
  const LwRun r(p, run);
  const int lane = threadIdx.x & 31, g = lane >> 2, n0 = r.c0 + 4 * (g >> 1) + (g & 1);
  const T* at = b + (int64_t)(p.start[r.target] + n0) * p.R + 4 * (lane & 3);
#pragma unroll
  for (int k = 0; k < KS; ++k)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      w[k][h] = n0 + 2 * h < r.width && 16 * k < p.R ? *reinterpret_cast<const uint2*>(at + 2 * h * p.R + 16 * k) : make_uint2(0, 0);
}

// Tiles of 16 rows: decode batches, bound by memory where adapters are many (64 rows of 64 adapters of rank 16, 4096 to 5120: 12.5 us
// for 29 MB, three sets of them in turn, 11.8 with one that stays in L2; a floor of 4.6) and by the chain of two products, the parts' meeting and two round trips
// where they are few (1 row 7.6 us).  Four steps of K and eight runs of 16 columns are under way (two and four: 14.1 us for the 64).  YT: y's type; KS: 16 ranks each (R or more).  Eight warps: 32 ranks each (of all targets) side by side, the rest of the warps splits
// this CTA's part of K.  Operands come straight from memory, 16 bytes a lane: the order of k within a product is free as long as both operands have the same.
template <typename T, typename YT, int KS>
__global__ void __launch_bounds__(LW_THREADS, 2)
lora_rows_kernel(const __grid_constant__ LoraRows p) {
  constexpr int ROWS = 16, PARTS = LwParts<T, YT>::N, NZ = (16 * KS + 31) / 32;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int s_row[ROWS];
  __shared__ float s_factor[ROWS][LW_TARGETS];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), C = (int)cluster.num_blocks();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int TR = p.targets * p.R, wn = TR > 128 ? 8 : TR > 64 ? 4 : TR > 32 ? 2 : 1, wk = LW_WARPS / wn, ranks = wn * 32, ld = ranks + 8;
  float* s_part = reinterpret_cast<float*>(smem);                 // [wk][ROWS][ranks]
  T* s_split = reinterpret_cast<T*>(s_part + ROWS * ranks);      // [PARTS][ROWS][ld]
  pdl_wait();
  const int tile_index = blockIdx.x / C / p.sub, from = 16 * (blockIdx.x / C - tile_index * p.sub), tiles = p.plan.tiles();
  int4 tile = p.plan.tile(tile_index);                            // (the plan has room for every tile of the grid)
  if (tile_index >= tiles || from >= tile.z) return;              // (the whole cluster)
  tile.y += from, tile.z = min(16, tile.z - from);
  const T* b = reinterpret_cast<const T*>(p.b) + (int64_t)tile.x * p.N * p.R;
  const int runs = p.tile0[p.targets], run0 = (int)((int64_t)runs * rank / C), run1 = (int)((int64_t)runs * (rank + 1) / C);
  if ((int)threadIdx.x < ROWS) s_row[threadIdx.x] = (int)threadIdx.x < tile.z ? p.plan.order()[tile.y + threadIdx.x] : -1;
  __syncthreads();

  // ---- this CTA's part of z ---------------------------------------------------------------------------------------------------
  float acc[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  const int my_n = warp % wn * 32, my_k = warp / wn;
  if (my_n < TR) {
    const T* xr[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = s_row[8 * h + g];
      xr[h] = row < 0 ? nullptr : reinterpret_cast<const T*>(p.x) + (int64_t)row * p.ldx + 8 * t;
    }
    const T* ar[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = my_n + 8 * j + g;
      ar[j] = n < TR ? reinterpret_cast<const T*>(p.a) + ((int64_t)tile.x * TR + n) * p.K + 8 * t : nullptr;
    }
    const int s0 = (int)((int64_t)p.steps * rank / C), s1 = (int)((int64_t)p.steps * (rank + 1) / C);
    const uint4 zero = make_uint4(0, 0, 0, 0);
    constexpr int DEEP = 4;                         // steps whose loads are under way together
#pragma unroll 1
    for (int s = s0 + my_k; s < s1; s += DEEP * wk) {
      uint4 av[DEEP][4], xv[DEEP][2];
#pragma unroll
      for (int u = 0; u < DEEP; ++u) {
        const int k = (s + u * wk) * 32;
        const bool in = s + u * wk < s1 && k + 8 * t < p.K;
#pragma unroll
        for (int j = 0; j < 4; ++j) av[u][j] = in && ar[j] ? *reinterpret_cast<const uint4*>(ar[j] + k) : zero;
#pragma unroll
        for (int h = 0; h < 2; ++h) xv[u][h] = in && xr[h] ? *reinterpret_cast<const uint4*>(xr[h] + k) : zero;
      }
#pragma unroll
      for (int u = 0; u < DEEP; ++u) {
        const uint32_t lo[4] = {xv[u][0].x, xv[u][1].x, xv[u][0].y, xv[u][1].y};
        const uint32_t hi[4] = {xv[u][0].z, xv[u][1].z, xv[u][0].w, xv[u][1].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          mma16816<T>(acc[j], lo, av[u][j].x, av[u][j].y);
          mma16816<T>(acc[j], hi, av[u][j].z, av[u][j].w);
        }
      }
    }
  }
  constexpr int AHEAD = 8 / KS;                      // runs whose b is under way
  uint2 w[AHEAD][KS][2];
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) lw_load<T, KS>(p, b, run0 + warp + u * LW_WARPS, run1, w[u]);
  {
    float* part = s_part + my_k * ROWS * ranks + my_n;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      *reinterpret_cast<float2*>(part + g * ranks + 8 * j + 2 * t) = make_float2(acc[j][0], acc[j][1]);
      *reinterpret_cast<float2*>(part + (8 + g) * ranks + 8 * j + 2 * t) = make_float2(acc[j][2], acc[j][3]);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < tile.z * ranks; i += LW_THREADS) {
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < LW_WARPS; ++k)
      if (k < wk) sum += s_part[k * ROWS * ranks + i];
    s_part[i] = sum;                                              // (nobody else looks at place i of the first part)
  }
  if (C > 1) cluster.sync();
  else __syncthreads();

  // ---- z of all CTAs, as 16-bit numbers: a warp per row and target ---------------------------------------------------------------
  auto whole = [&](int i, float (&z)[NZ]) {
    const int row = i / p.targets, at = row * ranks + (i - row * p.targets) * p.R;
#pragma unroll
    for (int k = 0; k < NZ; ++k) {
      z[k] = 0.f;
      if (32 * k >= p.R) continue;
      float v[LW_CLUSTER];
#pragma unroll
      for (int r = 0; r < LW_CLUSTER; ++r) v[r] = r < C && 32 * k + lane < p.R ? cluster.map_shared_rank(s_part, r)[at + 32 * k + lane] : 0.f;
#pragma unroll
      for (int r = 0; r < LW_CLUSTER; ++r) z[k] += v[r];           // in one order everywhere
    }
  };
  auto split = [&](int i, const float (&z)[NZ]) {
    const int row = i / p.targets, target = i - row * p.targets;
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < NZ; ++k) top = fmaxf(top, fabsf(z[k]));
    top = warp_max(top);
    float up, down;
    lw_scale<T>(top, up, down);
    if (lane == 0) s_factor[row][target] = up * p.scales[tile.x];
#pragma unroll
    for (int k = 0; k < NZ; ++k) {
      if (32 * k + lane >= p.R) continue;
      float v = z[k] * down;
#pragma unroll
      for (int part = 0; part < PARTS; ++part) {
        const T h = Tr<T>::from_f(v);
        s_split[(part * ROWS + row) * ld + target * p.R + 32 * k + lane] = h;
        v -= Tr<T>::to_f(h);
      }
    }
  };
  for (int i = warp; i < tile.z * p.targets; i += LW_WARPS) {
    float z[NZ];
    whole(i, z);
    split(i, z);
  }
  if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  __syncthreads();
  pdl_launch_dependents();

  // ---- this CTA's columns: 16 at a time, of which a lane has four neighbours -----------------------------------------------------
#pragma unroll 1
  for (int first = run0 + warp; first < run1; first += AHEAD * LW_WARPS) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int run = first + u * LW_WARPS;
      if (run >= run1) break;
      const LwRun r(p, run);
      const bool in = r.c0 + 4 * t < r.width;
      const int64_t col = p.col0[r.target] + r.c0 + 4 * t;
      uint2 old[2];                                               // 16-bit y, on its way beside the products (fp32 is added in memory)
      if constexpr (sizeof(YT) == 2) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = s_row[8 * h + g];
          old[h] = row >= 0 && in ? *reinterpret_cast<const uint2*>(reinterpret_cast<const YT*>(p.y) + (int64_t)row * p.ldy + col) : make_uint2(0, 0);
        }
      }
      float d[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) d[h][0] = d[h][1] = d[h][2] = d[h][3] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        if (16 * k >= p.R) break;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          const T* z = s_split + (part * ROWS + g) * ld + r.target * p.R + 16 * k + 4 * t;
          const uint2 lo = *reinterpret_cast<const uint2*>(z), hi = *reinterpret_cast<const uint2*>(z + 8 * ld);
          const uint32_t f[4] = {lo.x, hi.x, lo.y, hi.y};
          mma16816<T>(d[0], f, w[u][k][0].x, w[u][k][0].y);
          mma16816<T>(d[1], f, w[u][k][1].x, w[u][k][1].y);
        }
      }
      lw_load<T, KS>(p, b, run + AHEAD * LW_WARPS, run1, w[u]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = 8 * h + g, row = s_row[at];
        if (row < 0 || !in) continue;
        const float f = s_factor[at][r.target];
        YT* y = reinterpret_cast<YT*>(p.y) + (int64_t)row * p.ldy + col;
        if constexpr (sizeof(YT) == 4) {
          red_add4(y, f * d[0][2 * h], f * d[0][2 * h + 1], f * d[1][2 * h], f * d[1][2 * h + 1]);
        } else {
          const YT* e = reinterpret_cast<const YT*>(&old[h]);
          *reinterpret_cast<uint2*>(y) = make_uint2(pack2<YT>(fmaf(f, d[0][2 * h], Tr<YT>::to_f(e[0])), fmaf(f, d[0][2 * h + 1], Tr<YT>::to_f(e[1]))),
                                                    pack2<YT>(fmaf(f, d[1][2 * h], Tr<YT>::to_f(e[2])), fmaf(f, d[1][2 * h + 1], Tr<YT>::to_f(e[3]))));
        }
      }
    }
  }
  if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");      // nobody leaves before all have read
}

// Tiles of 128 rows on tcgen05: prompts with 16-bit y and up to three targets.  The same steps, one CTA per SM: rows of x (wherever they lie) and of A come by
// 16-byte copies into tiles of 64 of K, z = x A^T grows in TMEM, meets the other CTAs' and becomes the operand of the second product, whose blocks of 64 or
// 128 columns take b along with the old y; y grows in its place in shared memory and leaves by whole lines while the next block's product runs.
// RK: ranks of all targets, filled up to 32, 64, 128 or 256.  8000 rows of rank 64, 4096 to 5120: 56 us of 31.
constexpr int LT_ROWS = 128, LT_TARGETS = 3, LT_CLUSTER = 8, LT_THREADS = LW_THREADS + 128;
template <int RK, int COLS>
struct LtShape {
  static constexpr int STAGES_B = COLS == 128 ? 3 : 4, STAGES_Y = COLS == 128 ? 3 : 5;
  static constexpr int STAGE_A = (LT_ROWS + RK) * 128, STAGES_A = RK == 256 ? 4 : 6, TMEM = RK == 256 || COLS == 128 ? 256 : 128;
  static constexpr int B_BYTES = COLS * 128, Y_PITCH = COLS * 2 + 16, Y_BYTES = LT_ROWS * Y_PITCH;
  static constexpr int Z_TILE = LT_ROWS * 128;                    // of one part of a target's z: 64 ranks a line
  static __host__ __device__ constexpr int z_pitch(int TR) { return TR + 4; }      // floats; a row per thread without conflicts
  static __host__ __device__ constexpr int front(int TR) {
    const int z = LT_ROWS * z_pitch(TR) * 4, c = STAGES_B * B_BYTES + STAGES_Y * Y_BYTES;
    return ((z > c ? z : c) + 1023) / 1024 * 1024;
  }
  static __host__ __device__ constexpr int bytes(int TR, int targets) {
    const int a = STAGES_A * STAGE_A, c = front(TR) + 2 * targets * Z_TILE;
    return 1024 + (a > c ? a : c);
  }
  static_assert(B_BYTES % 1024 == 0 && STAGE_A % 1024 == 0, "tiles at whole swizzles");
};

struct LtBarriers {
  uint64_t step[6], block[2], read[2];                            // a stage's products, a block's; its results are read
  uint32_t tmem;
  volatile int abort;
};

// A wait that gives up is reported and everything goes on (the other waits then give up at once): the threads keep meeting at the CTA's and the cluster's
// barriers, and only the numbers are wrong.
template <typename T, int RK, int COLS>
__global__ void __launch_bounds__(LT_THREADS, 1)
lora_prompt_kernel(const __grid_constant__ LoraRows p) {
  using S = LtShape<RK, COLS>;
  constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  constexpr uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((128u >> 4) << 24);      // D fp32, 128 rows, K-major operands; N below
  constexpr uint32_t idesc_z = idesc | ((uint32_t)(RK >> 3) << 17), idesc_y = idesc | ((uint32_t)(COLS >> 3) << 17);
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int s_row[LT_ROWS];
  __shared__ float s_factor[LT_TARGETS][LT_ROWS];
  __shared__ LtBarriers s_bar;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), C = (int)cluster.num_blocks();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int TR = p.targets * p.R, zp = S::z_pitch(TR);
  const uint32_t raw = smem_u32(smem), s0 = (raw + 1023u) & ~1023u;
  uint8_t* base = smem + (s0 - raw);                              // (the same offset in every CTA of the cluster)
  float* s_z = reinterpret_cast<float*>(base);                    // [128][zp], over the first stages
  const uint32_t zop = s0 + S::front(TR);                         // [part][target] tiles of z
  pdl_wait();
  const int tile_index = blockIdx.x / C, tiles = p.plan.tiles();
  const int4 tile = p.plan.tile(tile_index);                      // (the plan has room for every tile of the grid)
  if (tile_index >= tiles) return;                                // (the whole cluster)
  if ((int)threadIdx.x < LT_ROWS) s_row[threadIdx.x] = (int)threadIdx.x < tile.z ? p.plan.order()[tile.y + threadIdx.x] : -1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 6; ++i) mbar_init(smem_u32(&s_bar.step[i]), 1);
    for (int i = 0; i < 2; ++i) { mbar_init(smem_u32(&s_bar.block[i]), 1); mbar_init(smem_u32(&s_bar.read[i]), LW_WARPS); }
    s_bar.abort = 0;
    fence_barrier_init();
  }
  // (behind the wait: an older launch on this SM takes its TMEM first)
  if (warp == LW_WARPS) tmem_alloc(smem_u32(&s_bar.tmem), S::TMEM);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_bar.tmem;
  auto wait = [&](uint64_t& bar, uint32_t parity, int role) { mbar_wait_warp(smem_u32(&bar), parity, &s_bar.abort, p.wait_word, role); };

  // ---- this CTA's part of z ---------------------------------------------------------------------------------------------------
  const int steps = (int)((p.K + 63) / 64), k0 = (int)((int64_t)steps * rank / C), k1 = (int)((int64_t)steps * (rank + 1) / C);
  {
    const int c = threadIdx.x & 7, line = threadIdx.x >> 3;       // this thread's 16 bytes of a line of 64, and its first line
    const bool copies = warp < LW_WARPS;                          // the warp behind them issues the products
    const T* xr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = copies ? s_row[line + 32 * i] : -1;
      xr[i] = row < 0 ? nullptr : reinterpret_cast<const T*>(p.x) + (int64_t)row * p.ldx + 8 * c;
    }
    const T* ar = reinterpret_cast<const T*>(p.a) + ((int64_t)tile.x * TR + line) * p.K + 8 * c;
    auto issue = [&](int s) {
      if (copies && s < k1) {
        const uint32_t at = s0 + (uint32_t)((s - k0) % S::STAGES_A) * S::STAGE_A + ((c ^ (line & 7)) << 4);
        const bool in = s * 64 + 8 * c < p.K;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool ok = in && xr[i];
          cp_async16(at + (line + 32 * i) * 128, ok ? xr[i] + s * 64 : reinterpret_cast<const T*>(p.x), ok);
        }
#pragma unroll
        for (int i = 0; i < RK / 32; ++i) {
          const bool ok = in && line + 32 * i < TR;
          cp_async16(at + (LT_ROWS + line + 32 * i) * 128, ok ? ar + (int64_t)32 * i * p.K + s * 64 : reinterpret_cast<const T*>(p.a), ok);
        }
      }
      cp_async_commit();
    };
    for (int s = 0; s < S::STAGES_A - 1; ++s) issue(k0 + s);
#pragma unroll 1
    for (int s = k0; s < k1; ++s) {
      const int n = s - k0;
      cp_async_wait<S::STAGES_A - 2>();
      fence_proxy_async_smem();                                   // this thread's copies, for the products
      __syncthreads();
      if (warp == LW_WARPS && elect_one()) {
        const uint32_t xs = s0 + (uint32_t)(n % S::STAGES_A) * S::STAGE_A;
        const uint64_t ad = make_desc_sw128(xs), bd = make_desc_sw128(xs + LT_ROWS * 128);
#pragma unroll
        for (int k = 0; k < 4; ++k) ft_mma_ss(tmem, ad + 2 * k, bd + 2 * k, idesc_z, n || k ? 1u : 0u);
        umma_commit(smem_u32(&s_bar.step[n % S::STAGES_A]));
      }
      __syncwarp();
      if (n > 0) wait(s_bar.step[(n - 1) % S::STAGES_A], (uint32_t)((n - 1) / S::STAGES_A) & 1u, 8);      // its stage is the one that is filled now
      issue(s + S::STAGES_A - 1);
    }
    cp_async_wait<0>();
    if (k1 > k0) wait(s_bar.step[(k1 - k0 - 1) % S::STAGES_A], (uint32_t)((k1 - k0 - 1) / S::STAGES_A) & 1u, 8);
    tc_fence_after();
    __syncthreads();                                              // the stages are nobody's any more
    // a thread per row and every other 32 ranks
    const int row = 32 * (warp & 3) + lane;
    for (int r = 32 * (warp >> 2); copies && r < TR; r += 64) {
      float z[32];
      if (k1 > k0) {
        tmem_ld32(tmem + ((uint32_t)(32 * (warp & 3)) << 16) + r, z);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) z[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 32; i += 4)
        if (r + i < TR) *reinterpret_cast<float4*>(s_z + row * zp + r + i) = make_float4(z[i], z[i + 1], z[i + 2], z[i + 3]);
    }
    tc_fence_before();                                            // (the blocks' products write there again)
  }
  if (C > 1) cluster.sync();
  else __syncthreads();

  // ---- z of all CTAs, as two 16-bit numbers: a CTA adds up and splits 1 / C of the rows for all of them, 16 lanes a row and target, four ranks each.  (Each
  // all rows: every CTA would read the z of eight, 512 KB.) --------------------------------------------------------------------------
  auto meet = [&](auto most) {                                    // of up to `most` CTAs
    constexpr int CTAS = decltype(most)::value;
    const int l = threadIdx.x & 15, k = 4 * l, rows = LT_ROWS / C;
#pragma unroll(CTAS > 4 ? 2 : 4)
    for (int i = threadIdx.x >> 4; i < rows * p.targets; i += LW_THREADS / 16) {
      const int target = i / rows, row = rank * rows + i - target * rows, at = row * zp + target * p.R + k;
      float4 z = make_float4(0.f, 0.f, 0.f, 0.f), v[CTAS];
#pragma unroll
      for (int r = 0; r < CTAS; ++r)
        v[r] = r < C && k < p.R ? *reinterpret_cast<const float4*>((r == rank ? s_z : cluster.map_shared_rank(s_z, r)) + at) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int r = 0; r < CTAS; ++r) z.x += v[r].x, z.y += v[r].y, z.z += v[r].z, z.w += v[r].w;      // in one order
      float top = fmaxf(fmaxf(fabsf(z.x), fabsf(z.y)), fmaxf(fabsf(z.z), fabsf(z.w))), up, down;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
      lw_scale<T>(top, up, down);
      z.x *= down, z.y *= down, z.z *= down, z.w *= down;
      auto rest = [](float x) { return x - Tr<T>::to_f(Tr<T>::from_f(x)); };
      const uint2 high = make_uint2(pack2<T>(z.x, z.y), pack2<T>(z.z, z.w)), low = make_uint2(pack2<T>(rest(z.x), rest(z.y)), pack2<T>(rest(z.z), rest(z.w)));
      uint8_t* to = base + S::front(TR) + (size_t)target * S::Z_TILE + row * 128 + (((k >> 3) ^ (row & 7)) << 4) + (k & 4) * 2;
      const float factor = up * p.scales[tile.x];
      for (int r = 0; r < C; ++r) {
        if (l == 0) (r == rank ? s_factor : cluster.map_shared_rank(s_factor, r))[target][row] = factor;
        if (k >= p.R) continue;
        uint8_t* there = r == rank ? to : cluster.map_shared_rank(to, r);
        *reinterpret_cast<uint2*>(there) = high;
        *reinterpret_cast<uint2*>(there + (size_t)p.targets * S::Z_TILE) = low;
      }
    }
  };
  if (warp < LW_WARPS) {
    if (C == 1) meet(std::integral_constant<int, 1>());
    else if (C <= 4) meet(std::integral_constant<int, 4>());
    else meet(std::integral_constant<int, LT_CLUSTER>());
  }
  fence_proxy_async_smem();
  if (C > 1) cluster.sync();                                      // all have read and written: the stages may lie there again
  else __syncthreads();
  fence_proxy_async_smem();                                       // (the others' writes, for the products)
  tc_fence_after();
  pdl_launch_dependents();

  // ---- this CTA's columns -------------------------------------------------------------------------------------------------------
  const T* b = reinterpret_cast<const T*>(p.b) + (int64_t)tile.x * p.N * p.R;
  int blocks = 0;
  for (int k = 0; k < p.targets; ++k) blocks += (p.start[k + 1] - p.start[k] + COLS - 1) / COLS;
  const int b0 = (int)((int64_t)blocks * rank / C), b1 = (int)((int64_t)blocks * (rank + 1) / C);
  struct Place {                                                  // of a block: its target and first column in it
    int target, col, width;
  };
  auto step = [&](Place& x) {
    x.col += COLS;
    if (x.col >= x.width && x.target + 1 < p.targets) ++x.target, x.col = 0, x.width = p.start[x.target + 1] - p.start[x.target];
  };
  Place ahead{0, 0, p.start[1]};                                  // the next block to fetch
  for (int k = 0; k < b0; ++k) step(ahead);
  Place here = ahead;
  if (warp >= LW_WARPS) {
    // b, by four warps (one alone took 1500 cycles a block for its copies), and the products, by one of their threads
    constexpr int BP = COLS * LW_RANK / 8 / 128;
    const int per = p.R / 8, pieces = COLS * per;              // 16-byte pieces of a line of b, and of a block: they lie in a row
    uint32_t to[BP];                                              // where this thread's go
#pragma unroll
    for (int k = 0; k < BP; ++k) {
      const int x = (int)threadIdx.x - LW_THREADS + 128 * k, n = x / per, c = x - n * per;
      to[k] = (uint32_t)(n * 128 + ((c ^ (n & 7)) << 4));
    }
    auto issue = [&](int block) {
      if (block < b1) {
        const uint32_t bs = s0 + (uint32_t)((block - b0) % S::STAGES_B) * S::B_BYTES;
        const T* from = b + (int64_t)(p.start[ahead.target] + ahead.col) * p.R;
        const int some = min(pieces, (ahead.width - ahead.col) * per);
#pragma unroll
        for (int k = 0; k < BP; ++k) {
          const int x = (int)threadIdx.x - LW_THREADS + 128 * k;
          if (x < pieces) cp_async16(bs + to[k], from + (x < some ? 8 * x : 0), x < some);
        }
        step(ahead);
      }
      cp_async_commit();
    };
    for (int s = 0; s < S::STAGES_B - 1; ++s) issue(b0 + s);
#pragma unroll 1
    for (int block = b0; block < b1; ++block) {
      const int n = block - b0;
      cp_async_wait<S::STAGES_B - 2>();
      fence_proxy_async_smem();                                   // this thread's copies, for the products
      named_bar_sync(3, 128);
      if (warp == LW_WARPS) {
        if (n >= 2) wait(s_bar.read[n & 1], (uint32_t)((n >> 1) - 1) & 1u, 9);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t bd = make_desc_sw128(s0 + (uint32_t)(n % S::STAGES_B) * S::B_BYTES);
          for (int part = 0; part < 2; ++part) {
            const uint64_t ad = make_desc_sw128(zop + (uint32_t)(part * p.targets + here.target) * S::Z_TILE);
#pragma unroll
            for (int k = 0; k < LW_RANK / 16; ++k)
              if (16 * k < p.R) ft_mma_ss(tmem + COLS * (n & 1), ad + 2 * k, bd + 2 * k, idesc_y, part || k ? 1u : 0u);
          }
          umma_commit(smem_u32(&s_bar.block[n & 1]));
        }
        __syncwarp();
      }
      step(here);
      if (n >= 1) wait(s_bar.block[(n - 1) & 1], (uint32_t)((n - 1) >> 1) & 1u, 9);      // its stage is the one that is filled now
      issue(block + S::STAGES_B - 1);
    }
  } else {
    // y.  A warp has 32 rows and half of a block's columns all by itself: copies, adds and stores them, and meets nobody.
    constexpr int CL = COLS / 16, RL = 32 / CL;                   // lanes of a row (eight columns each), rows at a time
    const uint32_t y0 = s0 + S::STAGES_B * S::B_BYTES;
    const int r0 = 32 * (warp & 3), c0 = COLS / 2 * (warp >> 2), c8 = c0 + 8 * (lane % CL);
    const int at = (r0 + lane / CL) * S::Y_PITCH + c8 * 2;
    T* y_row[CL];
#pragma unroll
    for (int k = 0; k < CL; ++k) {
      const int row = s_row[r0 + lane / CL + RL * k];
      y_row[k] = row < 0 ? nullptr : reinterpret_cast<T*>(p.y) + (int64_t)row * p.ldy + c8;
    }
    auto issue = [&](int block, int stage) {
      if (block < b1) {
        const int64_t col = p.col0[ahead.target] + ahead.col;
        const bool in = ahead.col + c8 < ahead.width;
#pragma unroll
        for (int k = 0; k < CL; ++k) {
          const bool ok = in && y_row[k];
          cp_async16(y0 + stage * S::Y_BYTES + at + RL * k * S::Y_PITCH, ok ? y_row[k] + col : reinterpret_cast<const T*>(p.y), ok);
        }
        step(ahead);
      }
      cp_async_commit();
    };
    for (int s = 0; s < S::STAGES_Y; ++s) issue(b0 + s, s);
    int stage = 0;
#pragma unroll 1
    for (int block = b0; block < b1; ++block) {
      const int n = block - b0;
      wait(s_bar.block[n & 1], (uint32_t)(n >> 1) & 1u, 9);
      tc_fence_after();
      float d[COLS / 2];
#pragma unroll
      for (int k = 0; k < COLS / 2; k += 32) tmem_ld32(tmem + ((uint32_t)r0 << 16) + COLS * (n & 1) + c0 + k, d + k);
      cp_async_wait<S::STAGES_Y - 1>();
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&s_bar.read[n & 1]));
      uint8_t* ys = base + S::STAGES_B * S::B_BYTES + (size_t)stage * S::Y_BYTES;
      const float f = s_factor[here.target][r0 + lane];
      uint4* mine = reinterpret_cast<uint4*>(ys + (r0 + lane) * S::Y_PITCH + c0 * 2);
#pragma unroll
      for (int k = 0; k < CL; ++k) {
        const uint4 v = mine[k];
        const T* e = reinterpret_cast<const T*>(&v);
        const float* x = d + 8 * k;
        mine[k] = make_uint4(pack2<T>(fmaf(f, x[0], Tr<T>::to_f(e[0])), fmaf(f, x[1], Tr<T>::to_f(e[1]))),
                             pack2<T>(fmaf(f, x[2], Tr<T>::to_f(e[2])), fmaf(f, x[3], Tr<T>::to_f(e[3]))),
                             pack2<T>(fmaf(f, x[4], Tr<T>::to_f(e[4])), fmaf(f, x[5], Tr<T>::to_f(e[5]))),
                             pack2<T>(fmaf(f, x[6], Tr<T>::to_f(e[6])), fmaf(f, x[7], Tr<T>::to_f(e[7]))));
      }
      __syncwarp();
      if (here.col + c8 < here.width) {
        const int64_t col = p.col0[here.target] + here.col;
#pragma unroll
        for (int k = 0; k < CL; ++k)
          if (y_row[k]) *reinterpret_cast<uint4*>(y_row[k] + col) = *reinterpret_cast<const uint4*>(ys + at + RL * k * S::Y_PITCH);
      }
      step(here);
      issue(block + S::STAGES_Y, stage);                          // (a lane fills what it has stored itself)
      stage = stage + 1 == S::STAGES_Y ? 0 : stage + 1;
    }
  }
  cp_async_wait<0>();
  if (s_bar.abort) wait_settle();
  tc_fence_before();
  __syncthreads();
  if (warp == LW_WARPS) {
    tc_fence_after();
    tmem_dealloc(tmem, S::TMEM);
  }
}

// Clusters of up to C CTAs, as many as fit the GPU.  (us, 64 rows of 64 adapters in clusters of 1 / 2 / 4 / 8: 31.1 / 18.4 / 12.5 / 19.3, three sets of adapters in turn;
// 1 row 20.9 / 13.6 / 9.3 / 7.6.)
static int launch_lora(void (*kern)(LoraRows), int threads, int most_bytes, int bytes, int C, int per_sm, std::atomic<uint64_t>& ready, const LoraRows& p, int64_t tiles,
                       cudaStream_t st) {
  int dev = 0;
  cudaError_t ae = cudaGetDevice(&dev);
  if (ae == cudaSuccess && (dev > 63 || !(ready.load(std::memory_order_relaxed) >> dev & 1))) {      // ready: devices whose copy of the kernel has its shared memory
    ae = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most_bytes);
    if (ae == cudaSuccess && dev < 64) ready.fetch_or(1ull << dev);
  }
  if (ae != cudaSuccess) return cuda_fail(ae, "cudaFuncSetAttribute(lora kernels)");
  // (clusters of eight with an SM for each CTA fill three quarters of the GPU at most, as their SMs are of one GPC: 2000 rows of 2 adapters of rank 64 in 16
  // of them 42.7, in fours 31.1)
  while (C > 1 && tiles * C > (int64_t)per_sm * sm_count() * (C > 4 && per_sm == 1 ? 3 : 4) / 4) C >>= 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * C));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  return e == cudaSuccess ? B200P_OK : cuda_fail(e, "lora kernels");
}

template <typename T, typename YT, int KS>
static int launch_lora_rows(const LoraRows& p, int64_t tiles, cudaStream_t st) {
  static std::atomic<uint64_t> ready{0};
  const int TR = p.targets * p.R, ranks = TR > 128 ? 256 : TR > 64 ? 128 : TR > 32 ? 64 : 32;
  return launch_lora(lora_rows_kernel<T, YT, KS>, LW_THREADS, lw_row_floats<T, YT>(LW_RANKS) * 16 * 4, lw_row_floats<T, YT>(ranks) * 16 * 4, LW_CLUSTER, 2, ready, p,
                     tiles * p.sub, st);
}

template <typename T, int RK, int COLS>
static int launch_lora_prompt_of(LoraRows p, int64_t tiles, cudaStream_t st) {
  static std::atomic<uint64_t> ready{0};
  using S = LtShape<RK, COLS>;
  constexpr int TARGETS = COLS == 128 ? 2 : LT_TARGETS, MOST = RK < LW_RANK * TARGETS ? RK : LW_RANK * TARGETS;
  static_assert(S::bytes(MOST, TARGETS) <= 224 * 1024, "beside the static shared memory");
  return launch_lora(lora_prompt_kernel<T, RK, COLS>, LT_THREADS, S::bytes(MOST, TARGETS), S::bytes(p.targets * p.R, p.targets), LT_CLUSTER, 1, ready, p, tiles, st);
}
// Blocks of 128 columns, whose products take the tensor core as long as those of 64 do; of 64 where three targets' z take their room.
template <typename T, int RK>
static int launch_lora_prompt(LoraRows p, int64_t tiles, cudaStream_t st) {
  if (const int rc = wait_word(WAIT_GEMM_TC, &p.wait_word)) return rc;
  if constexpr (RK <= 2 * LW_RANK) {
    if (p.targets <= 2) return launch_lora_prompt_of<T, RK, 128>(p, tiles, st);
  }
  return launch_lora_prompt_of<T, RK, 64>(p, tiles, st);
}

template <typename T, typename YT>
static int launch_lora_tiles(LoraRows p, int tile, int64_t tiles, cudaStream_t st) {
  const int TR = p.targets * p.R;
  if constexpr (sizeof(YT) == 2) {
    bool whole = aligned(p.y, 16) && p.ldy % 8 == 0;                // y by 16 bytes
    for (int k = 0; k < p.targets; ++k) whole = whole && p.col0[k] % 8 == 0;
    if (tile == LT_ROWS && p.targets <= LT_TARGETS && whole) {
      if (TR > 128) return launch_lora_prompt<T, 256>(p, tiles, st);
      if (TR > 64) return launch_lora_prompt<T, 128>(p, tiles, st);
      if (TR > 32) return launch_lora_prompt<T, 64>(p, tiles, st);
      return launch_lora_prompt<T, 32>(p, tiles, st);
    }
  }
  p.sub = tile / 16;                                                // (fp32 y, four targets, y by 8 bytes: tiles of 16 rows of the plan's)
  if (p.R == 16) return launch_lora_rows<T, YT, 1>(p, tiles, st);
  if (p.R == 32) return launch_lora_rows<T, YT, 2>(p, tiles, st);
  return launch_lora_rows<T, YT, 4>(p, tiles, st);
}

}  // namespace b200p

using namespace b200p;

extern "C" int64_t b200p_row_groups_ints(int64_t M, int64_t groups, int64_t tile) {
  if (M < 0 || M > RG_ROWS || groups <= 0 || groups > RG_GROUPS || tile <= 0) return 0;
  return row_group_ints(M, groups, tile);
}

extern "C" int b200p_row_groups(const int32_t* index, int32_t* plan, int64_t M, int groups, int tile, int64_t plan_ints, void* stream) {
  PdlClass pdl_cls(64);
  B200P_REQUIRE(M >= 0 && M <= RG_ROWS, B200P_ERR_ARG, "bad shape: %lld rows, at most 2^20", (long long)M);
  B200P_REQUIRE(groups > 0 && groups <= RG_GROUPS, B200P_ERR_ARG, "%d groups: 1 to %d", groups, RG_GROUPS);
  B200P_REQUIRE(tile > 0 && tile <= RG_ROWS, B200P_ERR_ARG, "%d rows of a tile", tile);
  B200P_REQUIRE(plan && (index || M == 0), B200P_ERR_ARG, "null pointer");
  B200P_REQUIRE(plan_ints >= row_group_ints(M, groups, tile), B200P_ERR_ARG, "a plan of %lld rows in %d groups has %lld integers, got room for %lld", (long long)M,
                groups, (long long)row_group_ints(M, groups, tile), (long long)plan_ints);
  B200P_REQUIRE(aligned(plan, 16) && aligned(index, 4), B200P_ERR_ALIGN, "the plan must be 16-byte aligned, the index to its type");
  if (groups > 512) {                                             // (more than every launch may have)
    const cudaError_t e = cudaFuncSetAttribute(row_groups_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RG_WARPS * RG_GROUPS * 4);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(row_groups_kernel)");
  }
  launch_pdl(row_groups_kernel, 1u, RG_WARPS * 32, (size_t)RG_WARPS * groups * 4, (cudaStream_t)stream, index, plan, (int)M, groups, tile);
  B200P_LAUNCH_CHECK("row_groups_kernel");
  return B200P_OK;
}

// Tiles of 128 rows read an adapter an eighth as often as tiles of 16 and put it on the tensor core, and have more to set up for few rows.  us, tiles of
// 16 / 128, 4096 to 5120 columns, ranks 16 and 64: 2 adapters, 500 rows 13.6 / 19.4 and 23.8 / 22.0, 1000 16.4 / 19.5 and 32.6 / 22.1, 1500 32.0 / 20.1 and
// 60.7 / 23.2, 8000 116 / 53 and 234 / 56; 16 adapters, 500 rows 13.5 / 25.8 and 25.1 / 27.7, 1000 21.8 / 26.1 and 54.3 / 28.0; 64 adapters, 500 rows
// 19.9 / 40.9 and 56.9 / 46.7, 1500 51 / 67 and 102 / 74, 8000 118 / 80 and 226 / 88.  (A plan is laid out once for layers of every rank.)
extern "C" int b200p_lora_rows_tile(int64_t M, int groups) { return M >= 1000 && M >= 16ll * groups ? LT_ROWS : 16; }

extern "C" int b200p_lora_rows(const void* x, const int32_t* plan, const void* a, const void* b, const float* scales, void* y, const int32_t* host_columns,
                               int64_t M, int adapters, int tile, int targets, int R, int64_t K, int64_t ldx, int64_t ldy, int dtype, int y_f32,
                               void* stream) {
  PdlClass pdl_cls(64);
  B200P_REQUIRE(dtype == B200P_F16 || dtype == B200P_BF16, B200P_ERR_ARG, "adapters and their inputs are 16-bit");
  B200P_REQUIRE(M >= 0 && M <= RG_ROWS && adapters > 0 && adapters <= RG_GROUPS, B200P_ERR_ARG, "bad shape: %lld rows, %d adapters", (long long)M, adapters);
  B200P_REQUIRE(tile == 16 || tile == LT_ROWS, B200P_ERR_ARG, "the plan's tiles have 16 or 128 rows, not %d", tile);
  B200P_REQUIRE(targets > 0 && targets <= LW_TARGETS, B200P_ERR_ARG, "%d targets: 1 to %d", targets, LW_TARGETS);
  B200P_REQUIRE(R > 0 && R % 16 == 0 && R <= LW_RANK, B200P_ERR_ARG, "rank %d: a multiple of 16, %d at most", R, LW_RANK);
  B200P_REQUIRE(K > 0 && K % 8 == 0 && K < (1ll << 24) && ldx >= K, B200P_ERR_ARG, "bad K %lld: a multiple of 8, not above ldx", (long long)K);
  B200P_REQUIRE(host_columns, B200P_ERR_ARG, "null pointer");
  LoraRows p{};
  for (int t = 0; t < targets; ++t) {
    const int64_t col = host_columns[2 * t], width = host_columns[2 * t + 1];
    B200P_REQUIRE(col >= 0 && width > 0 && width % 8 == 0 && col + width <= ldy, B200P_ERR_ARG, "target %d: columns %lld to %lld of %lld, a multiple of 8", t,
                  (long long)col, (long long)(col + width), (long long)ldy);
    B200P_REQUIRE(col % 4 == 0, B200P_ERR_ALIGN, "a target's first column is a multiple of 4");
    for (int u = 0; u < t; ++u)
      B200P_REQUIRE(col + width <= host_columns[2 * u] || col >= (int64_t)host_columns[2 * u] + host_columns[2 * u + 1], B200P_ERR_ARG, "targets overlap");
    p.col0[t] = (int)col, p.start[t + 1] = p.start[t] + (int)width, p.tile0[t + 1] = p.tile0[t] + (int)((width + 15) / 16);
  }
  if (M == 0) return B200P_OK;
  B200P_REQUIRE(x && plan && a && b && scales && y, B200P_ERR_ARG, "null pointer");
  B200P_REQUIRE(aligned(x, 16) && aligned(a, 16) && aligned(b, 16) && aligned(plan, 16) && ldx % 8 == 0, B200P_ERR_ALIGN,
                "x, its rows, the adapters and the plan must be 16-byte aligned");
  B200P_REQUIRE(aligned(y, y_f32 ? 16 : 8) && ldy % 4 == 0, B200P_ERR_ALIGN, "four neighbours of y must be aligned");
  p.x = x, p.a = a, p.b = b, p.scales = scales, p.y = y, p.plan = RowGroups{plan, (int)M}, p.ldx = ldx, p.ldy = ldy;
  p.K = (int)K, p.R = R, p.N = p.start[targets], p.targets = targets, p.steps = (int)((K + 31) / 32);
  const int64_t tiles = row_group_tiles(M, adapters, tile);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == B200P_F16) return y_f32 ? launch_lora_tiles<__half, float>(p, tile, tiles, st) : launch_lora_tiles<__half, __half>(p, tile, tiles, st);
  return y_f32 ? launch_lora_tiles<__nv_bfloat16, float>(p, tile, tiles, st) : launch_lora_tiles<__nv_bfloat16, __nv_bfloat16>(p, tile, tiles, st);
}
