// Attention of single tokens over a paged key-value cache, with a window behind which the first tokens stay visible, and the weight that
// every cached token receives added up.
//
//   token t of row r at slot s sees the slots j < n = s + 1 with j < first or j >= n - window (window 0: all j < n)
//   o = sum_j p_j v_j,  p = softmax_j(scale q . k_j)  per query head;  mass[j] += sum of p_j over the query heads of j's key head
//
// Scores, their maximum and sum, the outputs and the weights are fp32 throughout; the output is rounded once.
#include <stdlib.h>

#include <atomic>

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

__device__ __forceinline__ float raise2(float x) {                // 2^x, to 2 steps of fp32; results below 2^-126 become 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

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
  __device__ int key_tile(int v) const { return v < t0 ? v : v - t0 + skip; }
  __device__ int key0(int v) const { return key_tile(v) * PA_TILE; }
  __device__ bool visible(int j) const { return j < n && (j < first || j >= lo); }
  __device__ bool whole(int j0) const { return j0 + PA_TILE <= n && (j0 >= lo || j0 + PA_TILE <= first); }
};

struct PagedAttn {
  const void *q, *k, *v;
  void* out;
  float* mass;
  PageTable pt;
  const int32_t *t_row, *t_slot;
  int M, H, G, D, first, window, out_perm;
  float scale_log2e;
  // workspace
  unsigned* arrived;   // [CTAs] parts that are in, of the item that is cut first in this CTA: zero between calls
  float* rec;          // [CTAs, 2, rows of a block, D + 4] parts: maximum, sum, -, -, outputs
  float* stat;         // [M, H, 2] maximum and 1 / sum of every head (with a mass)
  float* scores;       // [M, items, cap, pitch] log2-scaled scores (with a mass)
  uint64_t inv_tpp;    // 2^40 / (tiles of a page), rounded up: tile * inv_tpp >> 40 is the page's index for any tile below 2^26
  int tpp;
  int cap, pitch;      // visible slots a token can have, in whole tiles; heads of a line of scores, a power of two
};

// The work is cut evenly however unequal the rows are: every token's visible tiles are counted in units of one tile per warp, the units of all
// (token, key head, block of query heads) items are laid end to end, and each of C CTAs takes the same number of them.  An item that lies in one
// CTA's share is finished there; of one that is cut every CTA leaves a part, and the CTA that comes last joins them, in their order (it reads
// what the others left: nobody waits).  (One CTA per item left the GPU idle behind the longest rows: 64 rows of 130 to 500 tokens took 108 us,
// 16 of 8192 940.  Joining in a second launch: one row of 1000 tokens 11.6 us.)
struct Token {
  int row, units;
  Span span;
  __device__ Token() : row(-1), units(0), span(0, 0, 0) {}
  __device__ Token(const PagedAttn& a, int t, int warps) : row(a.t_row[t]), units(0), span(0, 0, 0) {
    if (row >= 0 && row < a.pt.rows) {
      span = Span(slots_seen(a.pt, a.t_slot[t]), a.first, a.window);
      units = span.tiles > warps ? (span.tiles + warps - 1) / warps : 1;      // a token that sees nothing: one, for its zeros
    }
  }
};
// CTAs that share U units of n items; a join reads a part per CTA, one after the other, so that 64 of them are enough for an item
__device__ __forceinline__ int64_t shares(int64_t U, int64_t n, int most) { return min(min(U, 64 * n), (int64_t)most); }
__device__ __forceinline__ int64_t share_begin(int64_t U, int64_t C, int64_t c) { return U * c / C; }
__device__ __forceinline__ int64_t share_of(int64_t U, int64_t C, int64_t u) {
  int64_t c = u * C / U;
  while (share_begin(U, C, c + 1) <= u) ++c;
  return c;
}

// A position in a CTA's share: the token, and of its units the run [a, b) of one item.
struct Cursor {
  int64_t u, end, base;
  int t, item, a, b;
  Token tok;
  __device__ Cursor(const PagedAttn& p, int64_t u_, int64_t end_, int t_, int64_t base_, int warps)
      : u(u_), end(end_), base(base_), t(t_), item(0), a(0), b(0), tok(p, t_, warps) {}
  __device__ bool next(const PagedAttn& p, int items, int warps) {
    if (u >= end) return false;
    while (u >= base + (int64_t)tok.units * items) {
      base += (int64_t)tok.units * items;
      tok = Token(p, ++t, warps);
    }
    const unsigned at = (unsigned)(u - base);
    item = at / (unsigned)tok.units;
    a = at - item * tok.units;
    b = (int)min((int64_t)tok.units, a + (end - u));
    u += b - a;
    return true;
  }
};

// ------------------------------------------------------------------------------------------------ engines
// What a warp does with a staged tile of 16 keys.  ROWS query heads of one key head share it, so keys and values are read once.

// 16-bit types, D a multiple of 16: mma.sync m16n8k16 with the 16 keys as its rows and the query heads as its columns, 8 (or, NB 2, 16) of them, so
// that hardly a product is wasted on absent heads: S^T = K Q^T, O^T = V^T P^T.  (With the heads as the 16 rows the products and the registers
// were twice as many.)  The weights multiply the values as two 16-bit numbers each (the rounded weight and what it lost), so that the output carries
// its own rounding only.
template <typename T_, int D_, int NB>
struct TcEngine {
  using T = T_;
  static constexpr int D = D_, ROWS = 8 * NB, WARPS = 4, STAGES = D_ > 128 ? 2 : 3, CTAS = D_ > 128 ? 1 : 2;
  static constexpr int CHUNKS = D / 8, PIECES = CHUNKS % 8 ? (CHUNKS | 1) : CHUNKS;    // 16-byte pieces of a staged line
  static constexpr int Q_STRIDE = D * 2 + 16, Q_BYTES = ROWS * Q_STRIDE;
  static constexpr int NQ = (ROWS * CHUNKS + WARPS * 32 - 1) / (WARPS * 32);
  // f16: the largest weight of a tile is 2^14 and not 1 (m is the maximum less 14), so that small weights keep their bits
  static constexpr float SHIFT = std::is_same<T_, __half>::value ? 14.f : 0.f;
  float o[NB][D / 16][4], m[NB][2], l[NB][2];                    // of the heads 8 nb + 2 qc and the next
  uint32_t qf[NB][D / 16][2];

  static __device__ __forceinline__ int dim(const PagedAttn&) { return D; }
  static __host__ __device__ __forceinline__ int tile_bytes(int) { return 2 * PA_TILE * PIECES * 16; }
  static __device__ __forceinline__ uint32_t at(int key, int c) {
    return (uint32_t)(key * PIECES * 16 + ((CHUNKS % 8 ? c : c ^ (key & 7)) << 4));
  }
  static __device__ __forceinline__ void put_q(uint8_t* qs, int r, int c, const uint4& x, int) {
    *reinterpret_cast<uint4*>(qs + r * Q_STRIDE + c * 16) = x;
  }
  __device__ __forceinline__ void begin(uint32_t qs) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int j = 0; j < D / 16; ++j) o[nb][j][0] = o[nb][j][1] = o[nb][j][2] = o[nb][j][3] = 0.f;
      m[nb][0] = m[nb][1] = -INFINITY;
      l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t p = qs + (8 * nb + (lane >> 2)) * Q_STRIDE + k * 32 + (lane & 3) * 4;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(qf[nb][k][0]) : "r"(p));
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(qf[nb][k][1]) : "r"(p + 16));
      }
    }
  }
  __device__ __forceinline__ void tile(const PagedAttn& a, uint32_t, uint32_t ks, int j0, const Span& sp, bool all, bool page, float* sc, int rows,
                                       uint8_t*) {
    const int lane = threadIdx.x & 31, qr = lane >> 2, qc = lane & 3, mat = lane >> 3, r8 = lane & 7;
    const uint32_t vs = ks + PA_TILE * PIECES * 16;
    float s[NB][4];                                              // keys qr and qr + 8 of two heads
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.f;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      uint32_t kf[4];
      ldsm_x4(ks + at(r8 + 8 * (mat & 1), 2 * k + (mat >> 1)), kf);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) mma16816<T>(s[nb], kf, qf[nb][k][0], qf[nb][k][1]);
    }
    const bool seen0 = all || (page && sp.visible(j0 + qr)), seen1 = all || (page && sp.visible(j0 + qr + 8));
    uint32_t hi[NB][2], lo[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float f[2], p[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x = seen0 ? s[nb][h] * a.scale_log2e : -INFINITY, y = seen1 ? s[nb][2 + h] * a.scale_log2e : -INFINITY;
        s[nb][h] = x;
        s[nb][2 + h] = y;
        float t = fmaxf(x, y);
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
        t = fmaxf(t - SHIFT, m[nb][h]);
        const float ref = t == -INFINITY ? 0.f : t;              // nothing seen yet
        f[h] = raise2(m[nb][h] - ref);
        p[h] = raise2(x - ref);
        p[2 + h] = raise2(y - ref);
        m[nb][h] = t;
        l[nb][h] = l[nb][h] * f[h] + (p[h] + p[2 + h]);
      }
      if (sc) {                                                  // lines of a.pitch heads, one per key
        const int head = 8 * nb + 2 * qc;
        if (head + 1 < a.pitch) {
          *reinterpret_cast<float2*>(sc + qr * a.pitch + head) = make_float2(s[nb][0], s[nb][1]);
          *reinterpret_cast<float2*>(sc + (qr + 8) * a.pitch + head) = make_float2(s[nb][2], s[nb][3]);
        } else if (head < a.pitch) {
          sc[qr * a.pitch] = s[nb][0];
          sc[(qr + 8) * a.pitch] = s[nb][2];
        }
      }
      if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {  // a maximum grew (or is not a number)
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          o[nb][j][0] *= f[0]; o[nb][j][1] *= f[1]; o[nb][j][2] *= f[0]; o[nb][j][3] *= f[1];
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {                              // 8 keys x 8 heads, turned to the operand's order
        const float a0 = p[2 * i], a1 = p[2 * i + 1];
        hi[nb][i] = transpose8(pack2<T>(a0, a1));
        lo[nb][i] = transpose8(pack2<T>(a0 - Tr<T>::to_f(Tr<T>::from_f(a0)), a1 - Tr<T>::to_f(Tr<T>::from_f(a1))));
      }
    }
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      uint32_t vf[4];
      ldsm_x4_trans(vs + at(r8 + 8 * (mat >> 1), 2 * j + (mat & 1)), vf);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        mma16816<T>(o[nb][j], vf, hi[nb][0], hi[nb][1]);
        mma16816<T>(o[nb][j], vf, lo[nb][0], lo[nb][1]);
      }
    }
  }
  static __device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
  }
  // heads [8 pass, 8 pass + 8) of this warp's part to p [8][D + 4]
  __device__ __forceinline__ void publish(float* p, int pass, int) {
    const int lane = threadIdx.x & 31, qr = lane >> 2, qc = lane & 3;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      if (nb == pass) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float* row = p + (2 * qc + h) * (D + 4);
          float sum = l[nb][h];
          sum += __shfl_xor_sync(0xffffffffu, sum, 4);
          sum += __shfl_xor_sync(0xffffffffu, sum, 8);
          sum += __shfl_xor_sync(0xffffffffu, sum, 16);
          if (qr == 0) { row[0] = m[nb][h]; row[1] = sum; }
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            row[4 + 16 * j + qr] = o[nb][j][h];
            row[4 + 16 * j + 8 + qr] = o[nb][j][2 + h];
          }
        }
      }
  }
};

// Every type and size, in fp32 FMAs: two lanes share a key for the scores, for the outputs a lane owns 4 (NG 2: 8) dimensions of 8 query heads.
template <typename T_, int NG>
struct FmaEngine {
  using T = T_;
  static constexpr int ROWS = 8, WARPS = sizeof(T_) == 4 && NG == 2 ? 2 : 4, STAGES = 2, CTAS = 1;
  static constexpr int E = 16 / (int)sizeof(T_);
  static constexpr int Q_BYTES = (ROWS * NG * 128 + WARPS * ROWS * PA_TILE) * 4;     // queries and every warp's weights, fp32
  static constexpr int NQ = (ROWS * NG * 128 / E + WARPS * 32 - 1) / (WARPS * 32);
  float o[ROWS][NG][4], m[ROWS], l[ROWS];

  static __device__ __forceinline__ int dim(const PagedAttn& a) { return a.D; }
  static __host__ __device__ __forceinline__ int line(int D) { return (D / E | 1) * 16; }
  static __host__ __device__ __forceinline__ int tile_bytes(int D) { return 2 * PA_TILE * line(D); }
  static __device__ __forceinline__ void put_q(uint8_t* qs, int r, int c, const uint4& x, int D) {
    const T* v = reinterpret_cast<const T*>(&x);
#pragma unroll
    for (int e = 0; e < E; ++e) reinterpret_cast<float*>(qs)[r * D + c * E + e] = Tr<T>::to_f(v[e]);
  }
  __device__ __forceinline__ void begin(uint32_t) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int x = 0; x < NG; ++x) o[r][x][0] = o[r][x][1] = o[r][x][2] = o[r][x][3] = 0.f;
    }
  }
  __device__ __forceinline__ void tile(const PagedAttn& a, uint32_t qs_, uint32_t, int j0, const Span& sp, bool all, bool page, float* sc, int rows,
                                       uint8_t* ks) {
    const int lane = threadIdx.x & 31, key = lane & 15, half = lane >> 4, D = a.D, chunks = D / E, stride = line(D);
    const uint8_t* vs = ks + PA_TILE * stride;
    extern __shared__ __align__(16) uint8_t smem[];
    const float* qs = reinterpret_cast<const float*>(smem);
    float* ps = reinterpret_cast<float*>(smem) + ROWS * NG * 128 + (threadIdx.x >> 5) * ROWS * PA_TILE;
    float s[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) s[r] = 0.f;
    for (int c = half; c < chunks; c += 2) {
      T kv[E];
      *reinterpret_cast<uint4*>(kv) = *reinterpret_cast<const uint4*>(ks + key * stride + c * 16);
#pragma unroll
      for (int e = 0; e < E; e += 4) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
          if (r < rows) {
            const float4 q = *reinterpret_cast<const float4*>(qs + r * D + c * E + e);
            s[r] = fmaf(Tr<T>::to_f(kv[e]), q.x, s[r]);
            s[r] = fmaf(Tr<T>::to_f(kv[e + 1]), q.y, s[r]);
            s[r] = fmaf(Tr<T>::to_f(kv[e + 2]), q.z, s[r]);
            s[r] = fmaf(Tr<T>::to_f(kv[e + 3]), q.w, s[r]);
          }
      }
    }
    const bool seen = all || (page && sp.visible(j0 + key));
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (r >= rows) break;
      float x = (s[r] + __shfl_xor_sync(0xffffffffu, s[r], 16)) * a.scale_log2e;
      x = seen ? x : -INFINITY;
      if (sc && half == 0) sc[key * a.pitch + r] = x;
      const float t = fmaxf(m[r], warp_max(x));
      const float ref = t == -INFINITY ? 0.f : t;
      const float f = raise2(m[r] - ref), p = raise2(x - ref);
      m[r] = t;
      l[r] = l[r] * f + warp_sum(half == 0 ? p : 0.f);
      if (half == 0) ps[r * PA_TILE + key] = p;
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[r][g][e] *= f;
    }
    __syncwarp();
    for (int k = 0; k < PA_TILE; ++k)
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const int d = (lane + 32 * g) * 4;
        if (d >= D) break;
        T vv[4];
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(vv) = *reinterpret_cast<const uint4*>(vs + k * stride + d * 4);
        else *reinterpret_cast<uint2*>(vv) = *reinterpret_cast<const uint2*>(vs + k * stride + d * 2);
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
          if (r < rows)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[r][g][e] = fmaf(ps[r * PA_TILE + k], Tr<T>::to_f(vv[e]), o[r][g][e]);
      }
  }
  static __device__ __forceinline__ uint32_t at(int key, int c, int D) { return (uint32_t)(key * line(D) + c * 16); }
  __device__ __forceinline__ void publish(float* p, int, int D) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float* row = p + r * (D + 4);
      if (lane == 0) { row[0] = m[r]; row[1] = l[r]; }
#pragma unroll
      for (int g = 0; g < NG; ++g)
        if ((lane + 32 * g) * 4 < D) *reinterpret_cast<float4*>(row + 4 + (lane + 32 * g) * 4) = make_float4(o[r][g][0], o[r][g][1], o[r][g][2], o[r][g][3]);
    }
  }
};

template <typename E> struct IsTc { static constexpr bool value = false; };
template <typename T, int D, int NB> struct IsTc<TcEngine<T, D, NB>> { static constexpr bool value = true; };

template <typename T>
__device__ __forceinline__ void store_row4(T* out, int d, float4 v, int perm) {
  if (perm) {
    out[perm8_pos(d)] = Tr<T>::from_f(v.x);
    out[perm8_pos(d + 1)] = Tr<T>::from_f(v.y);
    out[perm8_pos(d + 2)] = Tr<T>::from_f(v.z);
    out[perm8_pos(d + 3)] = Tr<T>::from_f(v.w);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(out + d) = v;
  } else {
    *reinterpret_cast<uint2*>(out + d) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
  }
}

// ------------------------------------------------------------------------------------------------ the kernel
template <typename E>
__global__ void __launch_bounds__(E::WARPS * 32, E::CTAS)
paged_attn_kernel(const PagedAttn a) {
  using T = typename E::T;
  constexpr int W = E::WARPS, THREADS = W * 32;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t s_sum[W], s_base;
  __shared__ int s_t, s_part[W], s_live[W];
  __shared__ bool s_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int D = E::dim(a), chunks = D * (int)sizeof(T) / 16;
  const int per = a.H / a.G, blocks = (per + E::ROWS - 1) / E::ROWS, items = a.G * blocks;
  uint8_t* ring = smem + E::Q_BYTES + warp * E::STAGES * E::tile_bytes(D);
  const uint32_t qs = (uint32_t)__cvta_generic_to_shared(smem), ring32 = (uint32_t)__cvta_generic_to_shared(ring);
  pdl_wait();

  // ---- the plan: units of all tokens, this CTA's share, the token in which it begins -------------------------------------
  const int chunk = (a.M + THREADS - 1) / THREADS;
  const int t0 = min(a.M, (int)threadIdx.x * chunk), t1 = min(a.M, t0 + chunk);
  int64_t mine = 0;
  int live = 0;
  for (int t = t0; t < t1; ++t) {
    const int n = Token(a, t, W).units;
    mine += (int64_t)n * items;
    live += n > 0;
  }
  int64_t before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += x;
  }
  live = __reduce_add_sync(0xffffffffu, live);
  if (lane == 31) {
    s_sum[warp] = before;
    s_live[warp] = live;
  }
  __syncthreads();
  before -= mine;
  int64_t U = 0, n_items = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < warp) before += s_sum[w];
    U += s_sum[w];
    n_items += (int64_t)s_live[w] * items;
  }
  const int64_t C = shares(U, n_items, (int)gridDim.x);
  if ((int64_t)blockIdx.x >= C) return;
  const int64_t ub = share_begin(U, C, blockIdx.x), ue = share_begin(U, C, blockIdx.x + 1);
  if (ub >= before && ub < before + mine) {
    int64_t x = before;
    for (int t = t0; t < t1; ++t) {
      const int64_t n = (int64_t)Token(a, t, W).units * items;
      if (ub < x + n) {
        s_t = t;
        s_base = x;
        break;
      }
      x += n;
    }
  }
  __syncthreads();

  // ---- loads run ahead of the products, across items --------------------------------------------------------------------
  Cursor ld(a, ub, ue, s_t, s_base, W), cu = ld;
  bool more = ld.next(a, items, W);
  int tile = ld.a * W + warp, tile_end = min(ld.b * W, ld.tok.span.tiles);
  unsigned paged = 0;                                             // stages whose keys have a page
  int id = -1, off = 0;                                           // the next tile's page, looked up a tile ahead, and its tile in it
  auto seek = [&]() {                                             // the next tile this warp loads
    while (more && tile >= tile_end) {
      more = ld.next(a, items, W);
      tile = ld.a * W + warp;
      tile_end = min(ld.b * W, ld.tok.span.tiles);
    }
    if (more) {
      const int kt = ld.tok.span.key_tile(tile), index = (int)((uint64_t)(unsigned)kt * a.inv_tpp >> 40);
      off = kt - index * a.tpp;
      id = __ldg(a.pt.table + (int64_t)ld.tok.row * a.pt.width + index);
    }
  };
  auto issue = [&](int stage) {
    if (more) {
      const Span& sp = ld.tok.span;
      const int j0 = sp.key0(tile);
      const bool page = (unsigned)id < (unsigned)a.pt.P, all = page && sp.whole(j0);
      const int64_t line = (((int64_t)(page ? id : 0) * a.G + ld.item / blocks) * a.tpp + off) * PA_TILE;
      const uint4* kg = reinterpret_cast<const uint4*>(a.k) + line * chunks + lane;
      const uint4* vg = reinterpret_cast<const uint4*>(a.v) + line * chunks + lane;
      const uint32_t ks = ring32 + stage * E::tile_bytes(D), vs = ks + E::tile_bytes(D) / 2;
      paged = (paged & ~(1u << stage)) | ((page ? 1u : 0u) << stage);
      if (!page && lane == 0) atomicAdd(&g_paged_attn_fault, 1u);
      if constexpr (IsTc<E>::value) {
        constexpr int N = PA_TILE * E::CHUNKS;
        if (all) {
#pragma unroll
          for (int i = 0; i < N / 32; ++i) {
            const uint32_t at = E::at((i * 32 + lane) / E::CHUNKS, (i * 32 + lane) % E::CHUNKS);
            copy16(ks + at, kg + i * 32);
            copy16(vs + at, vg + i * 32);
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < N / 32; ++i) {
            const int key = (i * 32 + lane) / E::CHUNKS;
            const uint32_t at = E::at(key, (i * 32 + lane) % E::CHUNKS);
            const bool ok = page && sp.visible(j0 + key);
            cp_async16(ks + at, ok ? kg + i * 32 : kg, ok);
            cp_async16(vs + at, ok ? vg + i * 32 : vg, ok);
          }
        }
      } else {
        for (int x = lane; x < PA_TILE * chunks; x += 32) {
          const int key = x / chunks, c = x - key * chunks;
          const bool ok = all || (page && sp.visible(j0 + key));
          cp_async16(ks + E::at(key, c, D), kg + (ok ? x - lane : 0), ok);
          cp_async16(vs + E::at(key, c, D), vg + (ok ? x - lane : 0), ok);
        }
      }
      tile += W;
      seek();
    }
    cp_async_commit();
  };
  // the queries of an item, a few 16-byte pieces per thread: those of the next one are fetched while this one's keys pass
  uint4 qn[E::NQ];
  auto fetch_q = [&](const Cursor& c) {
    const int g = c.item / blocks, r0 = (c.item - g * blocks) * E::ROWS, rows = min(E::ROWS, per - r0);
    const uint4* q = reinterpret_cast<const uint4*>(a.q) + ((int64_t)c.t * a.H + (int64_t)g * per + r0) * chunks;
#pragma unroll
    for (int i = 0; i < E::NQ; ++i) {
      const int x = i * THREADS + (int)threadIdx.x;
      qn[i] = x < rows * chunks ? q[x] : make_uint4(0, 0, 0, 0);
    }
  };
  auto put_q = [&]() {
#pragma unroll
    for (int i = 0; i < E::NQ; ++i) {
      const int x = i * THREADS + (int)threadIdx.x;
      if (x < E::ROWS * chunks) E::put_q(smem, x / chunks, x % chunks, qn[i], D);
    }
  };
  bool work = cu.next(a, items, W);
  fetch_q(cu);
  seek();
#pragma unroll
  for (int s = 0; s < E::STAGES - 1; ++s) issue(s);
  put_q();
  __syncthreads();

  E e;
  int stage = 0;                                                  // of the next tile
  while (work) {
    const Cursor me = cu;
    work = cu.next(a, items, W);
    if (work) fetch_q(cu);
    const int g = me.item / blocks, r0 = (me.item - g * blocks) * E::ROWS, rows = min(E::ROWS, per - r0);
    const int64_t head = (int64_t)me.t * a.H + (int64_t)g * per + r0;
    const Span sp = me.tok.span;
    float* scores = a.scores + ((int64_t)me.t * items + me.item) * a.cap * a.pitch;
    e.begin(qs);
    const int end = min(me.b * W, sp.tiles);
    for (int v = me.a * W + warp; v < end; v += W) {
      issue(stage == 0 ? E::STAGES - 1 : stage - 1);
      cp_async_wait<E::STAGES - 1>();
      __syncwarp();
      const int j0 = sp.key0(v);
      const bool page = (paged >> stage) & 1u;
      const bool all = page && sp.whole(j0);
      e.tile(a, qs, ring32 + stage * E::tile_bytes(D), j0, sp, all, page, a.mass ? scores + (int64_t)v * PA_TILE * a.pitch : nullptr, rows,
             ring + stage * E::tile_bytes(D));
      __syncwarp();                                               // the stage is refilled by the next issue
      stage = stage + 1 == E::STAGES ? 0 : stage + 1;
    }
    // ---- the warps' parts become one: each in the one stage of its ring that waits for nothing ------------------------------
    const int part = (warp * E::STAGES + (stage == 0 ? E::STAGES - 1 : stage - 1)) * E::tile_bytes(D);
    if (lane == 0) s_part[warp] = part;
    const bool whole = me.a == 0 && me.b == me.tok.units;
    const int64_t part_size = (int64_t)E::ROWS * (D + 4);
    float* rec = a.rec + ((int64_t)blockIdx.x * 2 + (me.a == 0 ? 1 : 0)) * part_size;
    for (int pass = 0; pass * 8 < rows; ++pass) {
      e.publish(reinterpret_cast<float*>(smem + E::Q_BYTES + part), pass, D);
      __syncthreads();
      if (pass == 0 && work) put_q();
      const int here = min(8, rows - pass * 8), quads = D / 4;
      for (int x = threadIdx.x; x < here * quads; x += THREADS) {
        const int r = x / quads, d = (x - r * quads) * 4;
        float M = -INFINITY, L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) M = fmaxf(M, reinterpret_cast<const float*>(smem + E::Q_BYTES + s_part[w])[r * (D + 4)]);
        const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float* p = reinterpret_cast<const float*>(smem + E::Q_BYTES + s_part[w]) + r * (D + 4);
          const float f = raise2(p[0] - ref);
          const float4 y = *reinterpret_cast<const float4*>(p + 4 + d);
          L += p[1] * f;
          acc.x += y.x * f; acc.y += y.y * f; acc.z += y.z * f; acc.w += y.w * f;
        }
        const int row = pass * 8 + r;
        if (whole) {
          const float inv = L == 0.f ? 0.f : 1.f / L;
          store_row4<T>(reinterpret_cast<T*>(a.out) + (head + row) * D, d, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv), a.out_perm);
          if (a.mass && d == 0) *reinterpret_cast<float2*>(a.stat + (head + row) * 2) = make_float2(ref, inv);
        } else {
          float* p = rec + row * (D + 4);
          *reinterpret_cast<float4*>(p + 4 + d) = acc;
          if (d == 0) *reinterpret_cast<float2*>(p) = make_float2(M, L);
        }
      }
      __syncthreads();
    }
    if (whole) continue;
    // ---- an item that is cut: the last of its CTAs joins the parts ----------------------------------------------------------
    const int64_t u0 = me.base + (int64_t)me.item * me.tok.units, c0 = share_of(U, C, u0), c1 = share_of(U, C, u0 + me.tok.units - 1);
    const int parts = (int)(c1 - c0) + 1;
    if (threadIdx.x == 0) {
      __threadfence();                                            // (the barrier before: every thread's part of the record)
      const bool last = atomicAdd(a.arrived + c0, 1u) == (unsigned)(parts - 1);
      if (last) {
        a.arrived[c0] = 0;                                        // as it was found
        __threadfence();
      }
      s_last = last;
    }
    __syncthreads();
    if (!s_last) continue;
    const float* first = a.rec + (c0 * 2 + 1) * part_size;
    const float* other = a.rec + (c0 + 1) * 2 * part_size;       // of part i > 0: + (i - 1) * 2 * part_size
    const int quads = D / 4;
    for (int x = threadIdx.x; x < rows * quads; x += THREADS) {
      const int r = x / quads, d = (x - r * quads) * 4;
      float M = -INFINITY, L = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      constexpr int AHEAD = 8;
      for (int i0 = 0; i0 < parts; i0 += AHEAD) {
        float2 ml[AHEAD];
        float4 y[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          const float* p = (i0 + i == 0 ? first : other + (int64_t)(i0 + i - 1) * 2 * part_size) + r * (D + 4);
          ml[i] = i0 + i < parts ? __ldcg(reinterpret_cast<const float2*>(p)) : make_float2(-INFINITY, 0.f);
          y[i] = i0 + i < parts ? __ldcg(reinterpret_cast<const float4*>(p + 4 + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float top = M;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) top = fmaxf(top, ml[i].x);
        const float ref = top == -INFINITY ? 0.f : top, f = raise2(M - ref);
        M = top;
        L *= f;
        acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          const float w = raise2(ml[i].x - ref);
          L += ml[i].y * w;
          acc.x += y[i].x * w; acc.y += y[i].y * w; acc.z += y[i].z * w; acc.w += y[i].w * w;
        }
      }
      const float inv = L == 0.f ? 0.f : 1.f / L;
      store_row4<T>(reinterpret_cast<T*>(a.out) + (head + r) * D, d, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv), a.out_perm);
      if (a.mass && d == 0) *reinterpret_cast<float2*>(a.stat + (head + r) * 2) = make_float2(M == -INFINITY ? 0.f : M, inv);
    }
  }
  cp_async_wait<0>();
}

// The weights that every visible slot received: a CTA per item (x) and slice of its visible slots (y), a thread per slot.
constexpr int PM_THREADS = 256;

template <int ROWS>
__global__ void __launch_bounds__(PM_THREADS)
paged_attn_mass_kernel(const PagedAttn a, int warps) {
  const int per = a.H / a.G, blocks = (per + ROWS - 1) / ROWS, items = a.G * blocks;
  const int t = blockIdx.x / items, item = blockIdx.x - t * items;
  const int g = item / blocks, r0 = (item - g * blocks) * ROWS, rows = min(ROWS, per - r0);
  pdl_wait();
  const Token tok(a, t, warps);
  const int seen = tok.span.tiles * PA_TILE;
  if ((int)blockIdx.y * PM_THREADS >= seen) return;
  const float2* stat = reinterpret_cast<const float2*>(a.stat) + (int64_t)t * a.H + (int64_t)g * per + r0;
  const float* sc = a.scores + (int64_t)blockIdx.x * a.cap * a.pitch;
  float2 st[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) st[r] = r < rows ? stat[r] : make_float2(0.f, 0.f);
  for (int x = blockIdx.y * PM_THREADS + threadIdx.x; x < seen; x += gridDim.y * PM_THREADS) {
    const int j = tok.span.key0(x / PA_TILE) + x % PA_TILE;
    if (!tok.span.visible(j)) continue;
    const int64_t id = page_id(a.pt, tok.row, j / a.pt.page);
    if (id < 0) continue;
    const float* s = sc + (int64_t)x * a.pitch;
    float w = 0.f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (r < rows) w += raise2(s[r] - st[r].x) * st[r].y;
    atomicAdd(&a.mass[(id * a.G + g) * a.pt.page + j % a.pt.page], w);    // slots that several tokens see
  }
}

// ------------------------------------------------------------------------------------------------ host
constexpr int PA_CTAS = 2;            // per SM: one's join beside the other's stream

// visible slots a token can have, in whole tiles
static int64_t visible_cap(int64_t slots, int64_t first, int64_t window) {
  const int64_t seen = window > 0 ? first + window + 2 * PA_TILE : slots;
  return ((seen < slots ? seen : slots) + PA_TILE - 1) / PA_TILE * PA_TILE;
}

static size_t round256(size_t n) { return (n + 255) / 256 * 256; }
constexpr size_t PA_ARRIVED = 4096;                               // bytes
static size_t rec_bytes(int D) { return round256((size_t)sm_count() * PA_CTAS * 2 * 16 * (D + 4) * 4); }
static size_t stat_bytes(int64_t M, int H) { return round256((size_t)M * H * 8); }

template <typename E>
static int launch_paged(PagedAttn a, cudaStream_t st) {
  const int smem = E::Q_BYTES + E::WARPS * E::STAGES * E::tile_bytes(a.D);
  const int blocks = (a.H / a.G + E::ROWS - 1) / E::ROWS, items = a.G * blocks;
  B200P_REQUIRE((int64_t)items * (a.cap / PA_TILE / E::WARPS + 1) < (1ll << 31) && (int64_t)a.M * items < (1ll << 31), B200P_ERR_ARG,
                "%d tokens of %d key heads over %d slots: too many for one call", a.M, a.G, a.cap);
  auto kern = paged_attn_kernel<E>;
  static std::atomic<uint64_t> ready{0};                          // devices whose copy of the kernel has its shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev > 63 || !(ready.load(std::memory_order_relaxed) >> dev & 1))) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024);
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(paged_attn_kernel)");
  const int ctas = sm_count() * (2 * (smem + 1024 + 256) <= 228 * 1024 ? 2 : 1);
  const int64_t most = (int64_t)a.M * items * ((a.cap / PA_TILE + E::WARPS - 1) / E::WARPS);
  const int grid = (int)(most < ctas ? most : ctas);
  B200P_REQUIRE(grid <= (int)(PA_ARRIVED / 4), B200P_ERR_ARCH, "%d SMs", sm_count());
  a.tpp = a.pt.page / PA_TILE;
  a.inv_tpp = ((1ull << 40) + a.tpp - 1) / a.tpp;
  a.pitch = 1;
  while (a.pitch < E::ROWS && a.pitch < a.H / a.G) a.pitch *= 2;
  launch_pdl(kern, (unsigned)grid, E::WARPS * 32, smem, st, a);
  B200P_LAUNCH_CHECK("paged_attn_kernel");
  if (!a.mass) return B200P_OK;
  // slices: as many as there are, but no more CTAs than fill the GPU
  const int64_t slices = (a.cap + PM_THREADS - 1) / PM_THREADS, fill = 8ll * sm_count() / ((int64_t)a.M * items) + 1;
  launch_pdl(paged_attn_mass_kernel<E::ROWS>, dim3((unsigned)(a.M * items), (unsigned)(slices < fill ? slices : fill)), PM_THREADS, 0, st, a, (int)E::WARPS);
  B200P_LAUNCH_CHECK("paged_attn_mass_kernel");
  return B200P_OK;
}

template <typename T>
static int launch_paged_type(const PagedAttn& a, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    const bool few = a.H / a.G <= 8;
    switch (a.D) {
      case 64: return few ? launch_paged<TcEngine<T, 64, 1>>(a, st) : launch_paged<TcEngine<T, 64, 2>>(a, st);
      case 80: return few ? launch_paged<TcEngine<T, 80, 1>>(a, st) : launch_paged<TcEngine<T, 80, 2>>(a, st);
      case 96: return few ? launch_paged<TcEngine<T, 96, 1>>(a, st) : launch_paged<TcEngine<T, 96, 2>>(a, st);
      case 128: return few ? launch_paged<TcEngine<T, 128, 1>>(a, st) : launch_paged<TcEngine<T, 128, 2>>(a, st);
      case 256: return launch_paged<TcEngine<T, 256, 1>>(a, st);     // (16 heads do not fit the registers)
    }
  }
  return a.D <= 128 ? launch_paged<FmaEngine<T, 1>>(a, st) : launch_paged<FmaEngine<T, 2>>(a, st);
}

}  // namespace b200p

using namespace b200p;

extern "C" size_t b200p_paged_attn_workspace_bytes(int64_t M, int H, int D, int64_t keys) {
  if (M <= 0 || H <= 0 || D <= 0) return 0;
  size_t n = PA_ARRIVED + rec_bytes(D);
  if (keys > 0) n += stat_bytes(M, H) + (size_t)M * H * 2 * ((keys + PA_TILE - 1) / PA_TILE * PA_TILE) * 4;     // (pitch < 2 x heads)
  return n;
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
  const int64_t slots = (int64_t)width * page;
  first = first < slots ? first : slots;
  window = window < slots ? window : slots;
  const int64_t cap = visible_cap(slots, first, window);
  B200P_REQUIRE(workspace && workspace_bytes >= b200p_paged_attn_workspace_bytes(M, H, D, mass ? cap : 0) && aligned(workspace, 256), B200P_ERR_ARG,
                "paged attention workspace too small or not aligned to 256 bytes");
  PagedAttn a{};
  a.q = q, a.k = kpages, a.v = vpages, a.out = out, a.mass = mass, a.pt = pt, a.t_row = t_row, a.t_slot = t_slot;
  a.M = (int)M, a.H = H, a.G = G, a.D = D, a.first = (int)first, a.window = (int)window, a.out_perm = (flags & B200P_OUT_PERM8) ? 1 : 0;
  a.scale_log2e = scale * 1.4426950408889634f, a.cap = (int)cap;
  uint8_t* ws = (uint8_t*)workspace;
  a.arrived = (unsigned*)ws;
  a.rec = (float*)(ws += PA_ARRIVED);
  a.stat = (float*)(ws += rec_bytes(D));
  a.scores = (float*)(ws + stat_bytes(M, H));
  B200P_DISPATCH_DTYPE(dtype, T, return (launch_paged_type<T>(a, (cudaStream_t)stream)));
  return B200P_OK;
}
