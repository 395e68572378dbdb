// Attention of single tokens over a paged key-value cache, with a window behind which the first tokens stay visible, and the weight that
// every cached token receives added up.
//
//   token t of row r at slot s sees the slots j < n = s + 1 with j < first or j >= n - window (window 0: all j < n)
//   o = sum_j p_j v_j,  p = softmax_j(scale q . k_j)  per query head;  mass[j] += sum of p_j over the query heads of j's key head
//
// Scores, their maximum and sum, the outputs and the weights are fp32 throughout; the output is rounded once.
#include <stdlib.h>

#include "mma_util.cuh"
#include "paged.cuh"

namespace b200p {

int sm_count();

// tiles of keys that met an id that names no page (b200p_paged_fault_count); such keys count as masked
__device__ unsigned int g_paged_attn_fault = 0;

int paged_attn_faults(unsigned int* count, int reset, cudaStream_t st) {
  cudaError_t e = cudaMemcpyFromSymbolAsync(count, g_paged_attn_fault, sizeof(*count), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && reset) {
    const unsigned int zero = 0;
    e = cudaMemcpyToSymbolAsync(g_paged_attn_fault, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  }
  return e == cudaSuccess ? B200P_OK : cuda_fail(e, "paged_attn_faults");
}

constexpr int PA_TILE = 16;      // keys of a tile: never across a page

// The tiles a token reads: those that hold first slots, then those from the window's beginning on.
struct Span {
  int n, lo, first;              // slots; the window's beginning (0: everything is visible)
  int t0, skip, tiles;           // tiles before the gap, the tile behind it, tiles in all
  __host__ __device__ Span(int n_, int first_, int window) : n(n_), first(first_) {
    lo = window > 0 && n > window ? n - window : 0;
    const int f = first < lo ? first : lo;
    t0 = (f + PA_TILE - 1) / PA_TILE;
    skip = lo / PA_TILE > t0 ? lo / PA_TILE : t0;
    tiles = n > 0 ? t0 + (n + PA_TILE - 1) / PA_TILE - skip : 0;
  }
  __device__ int key0(int v) const { return (v < t0 ? v : v - t0 + skip) * PA_TILE; }
  __device__ bool visible(int j) const { return j < n && (j < first || j >= lo); }
};

struct PagedAttn {
  const void *q, *k, *v;
  void* out;
  float *mass, *ws;
  PageTable pt;
  const int32_t *t_row, *t_slot;
  int H, G, D, first, window, cap, out_perm;      // cap: visible slots a token can have, in whole tiles
  float scale_log2e;
};

// ------------------------------------------------------------------------------------------------ any type and size
// One CTA per (block of 8 query heads of a key head, token); its warps take the tiles in turn.  A warp stages a tile of keys and values in
// shared memory (rows padded to an odd number of 16-byte pieces); two lanes share a key for the scores, for the outputs a lane owns 4 (D
// > 128: 8) dimensions of every head.
constexpr int PG_WARPS = 4, PG_ROWS = 8;

template <typename T, int NG>
__global__ void __launch_bounds__(PG_WARPS * 32)
paged_attn_any_kernel(const PagedAttn a) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = a.H / a.G, blocks = (per + PG_ROWS - 1) / PG_ROWS;
  const int g = blockIdx.x / blocks, r0 = (blockIdx.x % blocks) * PG_ROWS, t = blockIdx.y;
  const int rows = min(PG_ROWS, per - r0), D = a.D;
  const int row = a.t_row[t];
  if (row < 0 || row >= a.pt.rows) return;
  const Span span(slots_seen(a.pt, a.t_slot[t]), a.first, a.window);
  const int chunks = D * (int)sizeof(T) / 16, stride = (chunks | 1) * 16;
  float* qs = reinterpret_cast<float*>(smem);                       // [PG_ROWS][D]
  float* ps = qs + PG_ROWS * D + warp * PG_ROWS * PA_TILE;          // [PG_WARPS][PG_ROWS][16]
  float* ms = qs + PG_ROWS * D + PG_WARPS * PG_ROWS * PA_TILE;      // [PG_WARPS][PG_ROWS][2 + D]
  uint8_t* ks = reinterpret_cast<uint8_t*>(ms + PG_WARPS * PG_ROWS * (2 + D)) + warp * 2 * PA_TILE * stride;
  uint8_t* vs = ks + PA_TILE * stride;
  const T* q = reinterpret_cast<const T*>(a.q) + ((int64_t)t * a.H + (int64_t)g * per + r0) * D;
  for (int i = threadIdx.x; i < rows * D; i += blockDim.x) qs[i] = Tr<T>::to_f(q[i]) * a.scale_log2e;
  __syncthreads();
  float o[PG_ROWS][NG][4], m[PG_ROWS], l[PG_ROWS];
#pragma unroll
  for (int r = 0; r < PG_ROWS; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int x = 0; x < NG; ++x) o[r][x][0] = o[r][x][1] = o[r][x][2] = o[r][x][3] = 0.f;
  }
  float* scores = a.ws + ((int64_t)t * a.H + (int64_t)g * per + r0) * a.cap;
  for (int v = warp; v < span.tiles; v += PG_WARPS) {
    const int j0 = span.key0(v);
    const int64_t id = page_id(a.pt, row, j0 / a.pt.page);
    const int64_t base = ((id < 0 ? 0 : id) * a.G + g) * a.pt.page + j0 % a.pt.page;
    if (id < 0 && lane == 0) atomicAdd(&g_paged_attn_fault, 1u);
    const uint8_t* kg = reinterpret_cast<const uint8_t*>(a.k) + base * D * (int)sizeof(T);
    const uint8_t* vg = reinterpret_cast<const uint8_t*>(a.v) + base * D * (int)sizeof(T);
    for (int x = lane; x < PA_TILE * chunks; x += 32) {
      const int key = x / chunks, c = x - key * chunks;
      const bool ok = id >= 0 && span.visible(j0 + key);
      cp_async16((uint32_t)__cvta_generic_to_shared(ks + key * stride + c * 16), kg + (ok ? x : 0) * 16, ok);
      cp_async16((uint32_t)__cvta_generic_to_shared(vs + key * stride + c * 16), vg + (ok ? x : 0) * 16, ok);
    }
    cp_async_commit();
    cp_async_wait<0>();
    __syncwarp();
    const int key = lane & 15, half = lane >> 4;
    float s[PG_ROWS];
#pragma unroll
    for (int r = 0; r < PG_ROWS; ++r) s[r] = 0.f;
    constexpr int E = 16 / sizeof(T);
    for (int c = half; c < chunks; c += 2) {
      T kv[E];
      *reinterpret_cast<uint4*>(kv) = *reinterpret_cast<const uint4*>(ks + key * stride + c * 16);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float x = Tr<T>::to_f(kv[e]);
#pragma unroll
        for (int r = 0; r < PG_ROWS; ++r)
          if (r < rows) s[r] = fmaf(x, qs[r * D + c * E + e], s[r]);
      }
    }
    const bool seen = id >= 0 && span.visible(j0 + key);
#pragma unroll
    for (int r = 0; r < PG_ROWS; ++r) {
      if (r >= rows) break;
      float x = s[r] + __shfl_xor_sync(0xffffffffu, s[r], 16);
      x = seen ? x : -INFINITY;
      if (a.mass && half == 0) scores[(int64_t)r * a.cap + v * PA_TILE + key] = x;
      const float mx = fmaxf(m[r], warp_max(x));
      const float ref = mx == -INFINITY ? 0.f : mx;              // nothing seen yet
      const float f = exp2f(m[r] - ref), p = exp2f(x - ref);
      m[r] = mx;
      l[r] = l[r] * f + warp_sum(half == 0 ? p : 0.f);
      if (half == 0) ps[r * PA_TILE + key] = p;
#pragma unroll
      for (int x2 = 0; x2 < NG; ++x2)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[r][x2][e] *= f;
    }
    __syncwarp();
    for (int k = 0; k < PA_TILE; ++k)
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        const int d = (lane + 32 * x) * 4;
        if (d >= D) break;
        T vv[4];
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(vv) = *reinterpret_cast<const uint4*>(vs + k * stride + d * 4);
        else *reinterpret_cast<uint2*>(vv) = *reinterpret_cast<const uint2*>(vs + k * stride + d * 2);
#pragma unroll
        for (int r = 0; r < PG_ROWS; ++r)
          if (r < rows)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[r][x][e] = fmaf(ps[r * PA_TILE + k], Tr<T>::to_f(vv[e]), o[r][x][e]);
      }
    __syncwarp();
  }
#pragma unroll
  for (int r = 0; r < PG_ROWS; ++r) {
    float* p = ms + (warp * PG_ROWS + r) * (2 + D);
    if (lane == 0) { p[0] = m[r]; p[1] = l[r]; }
#pragma unroll
    for (int x = 0; x < NG; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if ((lane + 32 * x) * 4 < D) p[2 + (lane + 32 * x) * 4 + e] = o[r][x][e];
  }
  __syncthreads();
  T* out = reinterpret_cast<T*>(a.out) + ((int64_t)t * a.H + (int64_t)g * per + r0) * D;
  for (int i = threadIdx.x; i < rows * D; i += blockDim.x) {
    const int r = i / D, d = i - r * D;
    float M = -INFINITY, L = 0.f, acc = 0.f;
    for (int w = 0; w < PG_WARPS; ++w) M = fmaxf(M, ms[(w * PG_ROWS + r) * (2 + D)]);
    const float ref = M == -INFINITY ? 0.f : M;
    for (int w = 0; w < PG_WARPS; ++w) {
      const float* p = ms + (w * PG_ROWS + r) * (2 + D);
      const float f = exp2f(p[0] - ref);
      L += p[1] * f;
      acc += p[2 + d] * f;
    }
    out[(int64_t)r * D + (a.out_perm ? perm8_pos(d) : d)] = Tr<T>::from_f(L == 0.f ? 0.f : acc / L);
  }
  if (!a.mass) return;
  __syncthreads();
  if (threadIdx.x < rows) {                                        // maximum and 1 / sum of every head, into the first warp's record
    const int r = threadIdx.x;
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < PG_WARPS; ++w) M = fmaxf(M, ms[(w * PG_ROWS + r) * (2 + D)]);
    const float ref = M == -INFINITY ? 0.f : M;
    for (int w = 0; w < PG_WARPS; ++w) L += ms[(w * PG_ROWS + r) * (2 + D) + 1] * exp2f(ms[(w * PG_ROWS + r) * (2 + D)] - ref);
    qs[2 * r] = ref;
    qs[2 * r + 1] = L == 0.f ? 0.f : 1.f / L;
  }
  __syncthreads();
  for (int x = threadIdx.x; x < span.tiles * PA_TILE; x += blockDim.x) {
    const int j = span.key0(x / PA_TILE) + x % PA_TILE;
    if (!span.visible(j)) continue;
    const int64_t id = page_id(a.pt, row, j / a.pt.page);
    if (id < 0) continue;
    float w = 0.f;
    for (int r = 0; r < rows; ++r) w += exp2f(scores[(int64_t)r * a.cap + x] - qs[2 * r]) * qs[2 * r + 1];
    atomicAdd(&a.mass[(id * a.G + g) * a.pt.page + j % a.pt.page], w);
  }
}

template <typename T, int NG>
static int launch_any(const PagedAttn& a, int64_t M, cudaStream_t st) {
  const int chunks = a.D * (int)sizeof(T) / 16, stride = (chunks | 1) * 16;
  const size_t smem = 4 * (size_t)(PG_ROWS * a.D + PG_WARPS * PG_ROWS * PA_TILE + PG_WARPS * PG_ROWS * (2 + a.D)) + (size_t)PG_WARPS * 2 * PA_TILE * stride;
  auto kern = paged_attn_any_kernel<T, NG>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(paged_attn_any_kernel)");
  const int per = a.H / a.G, blocks = (per + PG_ROWS - 1) / PG_ROWS;
  kern<<<dim3((unsigned)(blocks * a.G), (unsigned)M), PG_WARPS * 32, smem, st>>>(a);
  B200P_LAUNCH_CHECK("paged_attn_any_kernel");
  return B200P_OK;
}

// visible slots a token can have, in whole tiles
static int64_t visible_cap(int64_t slots, int64_t first, int64_t window) {
  const int64_t seen = window > 0 ? first + window + 2 * PA_TILE : slots;
  return ((seen < slots ? seen : slots) + PA_TILE - 1) / PA_TILE * PA_TILE;
}

}  // namespace b200p

using namespace b200p;

extern "C" size_t b200p_paged_attn_workspace_bytes(int64_t M, int H, int D, int64_t keys) {
  (void)D;
  return M > 0 && H > 0 && keys > 0 ? (size_t)M * H * ((keys + PA_TILE - 1) / PA_TILE * PA_TILE) * sizeof(float) : 0;
}

extern "C" int b200p_paged_attn(const void* q, const void* kpages, const void* vpages, float* mass, const int32_t* table, const int32_t* t_row,
                                const int32_t* t_slot, void* out, int64_t M, int H, int G, int D, int64_t P, int page, int rows, int width, float scale,
                                int64_t first, int64_t window, int dtype, int flags, void* workspace, size_t workspace_bytes, void* stream) {
  PdlClass pdl_cls(8);
  const PageTable pt{table, P, rows, width, page};
  const int rc = check_pages(kpages, vpages, pt, G, D, dtype);
  if (rc) return rc;
  B200P_REQUIRE(M == 0 || (q && out && t_row && t_slot), B200P_ERR_ARG, "null pointer");
  B200P_REQUIRE(H > 0 && H % G == 0, B200P_ERR_ARG, "bad head counts %d/%d", H, G);
  B200P_REQUIRE(M >= 0 && M < 65536, B200P_ERR_ARG, "bad shape: %lld tokens", (long long)M);
  B200P_REQUIRE(first >= 0 && window >= 0, B200P_ERR_ARG, "first and window are counts");
  B200P_REQUIRE((flags & ~B200P_OUT_PERM8) == 0, B200P_ERR_ARG, "unknown flags 0x%x", flags);
  B200P_REQUIRE(aligned(q, 16) && aligned(out, 16), B200P_ERR_ALIGN, "q and out must be 16-byte aligned");
  if (M == 0) return B200P_OK;
  const int64_t slots = (int64_t)width * page, cap = visible_cap(slots, first, window);
  B200P_REQUIRE(!mass || (workspace && workspace_bytes >= b200p_paged_attn_workspace_bytes(M, H, D, cap) && aligned(workspace, 16)), B200P_ERR_ARG,
                "paged attention workspace too small");
  const PagedAttn a{q,     kpages, vpages, out, mass, (float*)workspace, pt, t_row, t_slot, H, G, D, (int)(first < slots ? first : slots),
                    (int)(window < slots ? window : slots), (int)cap, (flags & B200P_OUT_PERM8) ? 1 : 0, scale * 1.4426950408889634f};
  if (D <= 128) B200P_DISPATCH_DTYPE(dtype, T, return (launch_any<T, 1>(a, M, (cudaStream_t)stream)));
  B200P_DISPATCH_DTYPE(dtype, T, return (launch_any<T, 2>(a, M, (cudaStream_t)stream)));
  return B200P_OK;
}
