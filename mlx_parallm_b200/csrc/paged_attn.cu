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

// tiles of keys that met an id that names no page (b200p_paged_fault_count; such keys count as masked), and tokens of rows or at slots behind the table
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
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// The tiles a token reads: those that hold first slots, then those from the window's beginning on.
struct Span {
  int n, lo, first;              // slots; the window's beginning (0: everything is visible)
  int t0, skip, tiles;           // tiles before the gap, the tile behind it, tiles in all
  Span() = default;
  __host__ __device__ Span(int n_, int first_, int window) : n(n_), first(first_) {
    lo = window > 0 && n > window ? n - window : 0;
    const int f = first < lo ? first : lo;
    t0 = (f + PA_TILE - 1) / PA_TILE;
    skip = lo / PA_TILE > t0 ? lo / PA_TILE : t0;
    tiles = n > 0 ? t0 + (n + PA_TILE - 1) / PA_TILE - skip : 0;
  }
  __device__ int key_tile(int v) const { return v < t0 ? v : v - t0 + skip; }
  __device__ int tile_of(int kt) const { return kt < t0 ? kt : kt - skip + t0; }
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
  uint2* parts;        // [M, items] the first of the shares an item lies in and their number (idle tokens': not written)
  float* rec;          // [shares, 2, rows of a block, D + 4] parts: maximum, sum, -, -, outputs
  float* stat;         // [M, H, 2] maximum and 1 / sum of the heads that lie in one share (with a mass)
  float* scores;       // [M, items, cap, pitch] log2-scaled scores (with a mass)
  uint64_t inv_tpp;    // 2^36 / (tiles of a page, 256 at most), rounded up: tile * inv_tpp >> 36 is the page's index for any tile below 2^26
  int tpp, last;       // tiles of a page; CTAs for small shares at the line's end
  int cap, pitch;      // visible slots a token can have, in whole tiles; heads of a line of scores, a power of two
  // behind shared slots (paged_shared.cuh): a token's group, the groups' shared slots, the parts of items that lie in one share
  const int32_t *index, *prefix;
  int groups;
  float* whole;        // [M, H, D + 4]
};

__device__ __forceinline__ int shared_slots(const int32_t* index, const int32_t* prefix, int groups, const PageTable& pt, int t, int seen);

// The work is cut evenly however unequal the rows are: every token's visible tiles are counted in units of one tile per warp, the units of all
// (token, key head, block of query heads) items are laid end to end, and each resident CTA takes an equal share of that line.  An item in one share is
// finished there; of one that is cut every share leaves a part, and a second launch joins them.  (One CTA per item left the GPU idle behind the longest
// rows: 64 rows of 128 to 500 tokens took 108 us, 16 of 8192 940.  Joining in the CTA whose part comes last, by counters, cost a row of 1000 tokens 3.7 us
// of fences and atomics in a row; the second launch costs it less.  SMs differ by a quarter in what they get of the memory's bandwidth, so that of 16 rows of
// 8192 tokens the first CTAs are done after 63 us and the last after 90; a counter of small shares for whoever comes first evened that out but cost more than
// it gave: 106 us in all against 95.)
struct Token {
  int row, units;
  Span span;
  __device__ Token() : row(-1), units(0), span(0, 0, 0) {}
  // from > 0: only the slots from there on
  __device__ Token(const PagedAttn& a, int row_, int slots, int from, int warps) : row(row_), units(0), span(0, 0, 0) {
    if (row >= 0) {
      span = from == 0 ? Span(slots, a.first, a.window) : slots > from ? Span(slots, 0, slots - from) : Span(0, 0, 0);
      units = span.tiles > warps ? (span.tiles + warps - 1) / warps : 1;      // a token that sees nothing: one, for its zeros
    }
  }
  template <bool TAIL>
  static __device__ Token of(const PagedAttn& a, int t, int warps, int* begins = nullptr) {
    const int r = a.t_row[t];
    if (r < 0 || r >= a.pt.rows) return Token();
    const int n = slots_seen(a.pt, a.t_slot[t]), from = TAIL ? shared_slots(a.index, a.prefix, a.groups, a.pt, t, n) : 0;
    if (TAIL && begins) *begins = from;
    return Token(a, r, n, from, warps);
  }
};

constexpr int PA_TOKENS = 512;         // up to so many tokens a CTA keeps all of them in shared memory

// Where every CTA's share is long (PA_LAST_UNITS units, some 50 us in all) it gives a part away: PA_LAST_PERCENT of the line, its end, is cut into small
// shares for 3/4 as many more CTAs, which the hardware starts where the first ones have ended.  (16 rows of 8192 tokens 95.1 -> 90.0 us, 128 of 1000
// 96.1 -> 90.9, 64 of 1000 52.4 -> 51.8 in a captured graph; launched one by one 16 of 8192 96.0 -> 94.2.  64 of 500, below the bound, 31.3, and 33.5 with it.
// CTAs that find no share, where the table has room for long rows and the rows are short: 0.3 us at most.)
constexpr int PA_LAST_UNITS = 24, PA_LAST_PERCENT = 12;
__host__ __device__ inline int last_ctas(int ctas) { return ctas * 3 / 4; }

struct Shares {
  unsigned n, n1, u1, q, r, q2, r2;    // how many; the first n1 lie in [0, u1): r of q + 1 units, then of q; the small ones alike behind it
  // of U units that belong to so many items: a warp of the join reads its parts one after the other, 128 of an item are enough
  __device__ Shares(unsigned U, unsigned items, unsigned ctas, unsigned last)
      : n(min(min(U, ctas), items < 65536 ? 128 * items : ctas)), n1(n), u1(U), q2(1), r2(0) {
    if (last && n == ctas && U >= PA_LAST_UNITS * ctas) {
      u1 = U - U / 100 * PA_LAST_PERCENT;
      n += last;
      q2 = (U - u1) / last;
      r2 = U - u1 - q2 * last;
    }
    q = n1 ? u1 / n1 : 1;
    r = u1 - q * n1;
  }
  __device__ unsigned begin(unsigned c) const { return c <= n1 ? c * q + min(c, r) : u1 + (c - n1) * q2 + min(c - n1, r2); }
  __device__ unsigned of(unsigned u) const {
    const bool small = u >= u1;
    const unsigned v = small ? u - u1 : u, size = small ? q2 : q, more = small ? r2 : r;
    return (small ? n1 : 0) + (v < more * (size + 1) ? v / (size + 1) : more + (v - more * (size + 1)) / size);
  }
};

// The tokens of a call of up to PA_TOKENS: their rows and where their slots end.  (Under a full stream of keys a look at global memory
// takes 2 to 3 us, L2 hit or not.)
template <bool TAIL>
struct Tokens {
  int row[PA_TOKENS], slots[PA_TOKENS], from[TAIL ? PA_TOKENS : 1];
};

// A position in a share: the token, and of its units the run [a, b) of one item.
template <bool TAIL>
struct Cursor {
  unsigned u, end, base;
  int t, item, a, b;
  Token tok;
  __device__ void load(const PagedAttn& p, const Tokens<TAIL>& ts, int warps) {
    tok = p.M <= PA_TOKENS ? Token(p, ts.row[t], ts.slots[t], TAIL ? ts.from[t] : 0, warps) : Token::of<TAIL>(p, t, warps);
  }
  __device__ bool next(const PagedAttn& p, const Tokens<TAIL>& ts, int items, int warps) {
    if (u >= end) return false;
    while (u - base >= (unsigned)(tok.units * items)) {
      base += tok.units * items;
      ++t;
      load(p, ts, warps);
    }
    const unsigned at = u - base;
    item = at / (unsigned)tok.units;
    a = at - item * tok.units;
    b = min(tok.units, (int)(a + (end - u)));
    u += b - a;
    return true;
  }
};

// What the streaming warps need to know of a run of one item's tiles.
struct Run {
  int tile, tile_end;                  // of the item's visible tiles; tile < 0: there is no run any more
  Span span;
  int row, g, head, rows, line;        // table row, key head, first query head of all, heads, item of all
  int part;                            // where it goes; -1: it is the whole item
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
  static constexpr int D = D_, MAX_D = D_, ROWS = 8 * NB, WARPS = 4, STAGES = D_ > 128 ? 2 : D_ > 64 ? 3 : 4, CTAS = D_ > 128 ? 1 : 2;
  static constexpr int CHUNKS = D / 8, PIECES = CHUNKS % 8 ? (CHUNKS | 1) : CHUNKS;    // 16-byte pieces of a staged line
  static constexpr int Q_STRIDE = D * 2 + 16, Q_BYTES = ROWS * Q_STRIDE;
  static constexpr int NQ = (ROWS * CHUNKS + WARPS * 32 - 1) / (WARPS * 32);
  // f16: the largest weight of a tile is 2^14 and not 1 (m is the maximum less 14), so that small weights keep their bits
  static constexpr float SHIFT = std::is_same<T_, __half>::value ? 14.f : 0.f;
  float o[NB][D / 16][4], m[NB][2], l[NB][2];                    // of the heads 8 nb + 2 qc and the next
  // 16 heads' queries do not fit the registers beside the outputs: read again with every tile (32 rows of 4000 tokens, 64 / 4 heads of 128: 56.4 -> 45.0 us)
  static constexpr bool KEEP_Q = NB == 1;
  uint32_t qf[KEEP_Q ? NB : 1][KEEP_Q ? D / 16 : 1][2];

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
      for (int k = 0; k < (KEEP_Q ? D / 16 : 0); ++k) {
        const uint32_t p = qs + (8 * nb + (lane >> 2)) * Q_STRIDE + k * 32 + (lane & 3) * 4;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(qf[nb][k][0]) : "r"(p));
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(qf[nb][k][1]) : "r"(p + 16));
      }
    }
  }
  __device__ __forceinline__ void tile(const PagedAttn& a, uint32_t qs, uint32_t ks, int j0, const Span& sp, bool all, bool page, float* sc, int rows,
                                       uint8_t*) {
    const int lane = threadIdx.x & 31, qr = lane >> 2, qc = lane & 3, mat = lane >> 3, r8 = lane & 7;
    const uint32_t vs = ks + PA_TILE * PIECES * 16;
    float s[NB][4];                                              // keys qr and qr + 8 of two heads
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.f;
    uint32_t q4[KEEP_Q ? 1 : NB][4];                             // of two steps
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      uint32_t kf[4];
      ldsm_x4(ks + at(r8 + 8 * (mat & 1), 2 * k + (mat >> 1)), kf);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        if constexpr (KEEP_Q) {
          mma16816<T>(s[nb], kf, qf[nb][k][0], qf[nb][k][1]);
        } else {
          if (k % 2 == 0) ldsm_x4(qs + (8 * nb + r8) * Q_STRIDE + (2 * k + (k + 1 < D / 16 ? mat : mat & 1)) * 16, q4[nb]);
          mma16816<T>(s[nb], kf, q4[nb][2 * (k & 1)], q4[nb][2 * (k & 1) + 1]);
        }
      }
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

// Every type and size, in fp32 FMAs, R query heads at a time: four lanes share two keys for the scores, for the outputs a lane owns 4 (NG 2: 8)
// dimensions of every head, so that a 16-byte piece of queries or weights read from shared memory serves 8 or 16 products.
template <typename T_, int NG, int R>
struct FmaEngine {
  using T = T_;
  static constexpr int MAX_D = 128 * NG, ROWS = R, STAGES = 2, CTAS = 1;
  static constexpr int WARPS = sizeof(T_) * NG == 8 ? 3 : 6;
  static constexpr int E = 16 / (int)sizeof(T_);
  static constexpr int Q_BYTES = (ROWS * NG * 128 + WARPS * ROWS * PA_TILE) * 4;     // queries and every warp's weights, fp32
  static constexpr int NQ = (ROWS * NG * 128 / E + WARPS * 32 - 1) / (WARPS * 32);
  float o[ROWS][NG][4], m[ROWS], l[ROWS];                         // l: this lane's two keys' share

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
  __device__ __forceinline__ void tile(const PagedAttn& a, uint32_t, uint32_t, int j0, const Span& sp, bool all, bool page, float* sc, int rows,
                                       uint8_t* ks) {
    const int lane = threadIdx.x & 31, key = lane & 7, quarter = lane >> 3, D = a.D, chunks = D / E, stride = line(D);
    const uint8_t* vs = ks + PA_TILE * stride;
    extern __shared__ __align__(16) uint8_t smem[];
    const float* qs = reinterpret_cast<const float*>(smem);
    float* ps = reinterpret_cast<float*>(smem) + ROWS * NG * 128 + (threadIdx.x >> 5) * ROWS * PA_TILE;
    float s[ROWS][2];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) s[r][0] = s[r][1] = 0.f;
#pragma unroll 1
    for (int c = quarter; c < chunks; c += 4) {
      T k0[E], k1[E];
      *reinterpret_cast<uint4*>(k0) = *reinterpret_cast<const uint4*>(ks + key * stride + c * 16);
      *reinterpret_cast<uint4*>(k1) = *reinterpret_cast<const uint4*>(ks + (key + 8) * stride + c * 16);
#pragma unroll
      for (int e = 0; e < E; e += 4)
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {                          // (queries of absent heads are zeros)
          const float4 q = *reinterpret_cast<const float4*>(qs + r * D + c * E + e);
          s[r][0] = fmaf(Tr<T>::to_f(k0[e]), q.x, s[r][0]);
          s[r][1] = fmaf(Tr<T>::to_f(k1[e]), q.x, s[r][1]);
          s[r][0] = fmaf(Tr<T>::to_f(k0[e + 1]), q.y, s[r][0]);
          s[r][1] = fmaf(Tr<T>::to_f(k1[e + 1]), q.y, s[r][1]);
          s[r][0] = fmaf(Tr<T>::to_f(k0[e + 2]), q.z, s[r][0]);
          s[r][1] = fmaf(Tr<T>::to_f(k1[e + 2]), q.z, s[r][1]);
          s[r][0] = fmaf(Tr<T>::to_f(k0[e + 3]), q.w, s[r][0]);
          s[r][1] = fmaf(Tr<T>::to_f(k1[e + 3]), q.w, s[r][1]);
        }
    }
    const bool seen0 = all || (page && sp.visible(j0 + key)), seen1 = all || (page && sp.visible(j0 + key + 8));
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float x = s[r][0], y = s[r][1];
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      y += __shfl_xor_sync(0xffffffffu, y, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      y += __shfl_xor_sync(0xffffffffu, y, 16);
      x = seen0 ? x * a.scale_log2e : -INFINITY;
      y = seen1 ? y * a.scale_log2e : -INFINITY;
      if (sc && quarter == 0 && r < rows) {
        sc[key * a.pitch + r] = x;
        sc[(key + 8) * a.pitch + r] = y;
      }
      float t = fmaxf(x, y);
      t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
      t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
      t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
      t = fmaxf(t, m[r]);
      const float ref = t == -INFINITY ? 0.f : t;
      const float f = raise2(m[r] - ref), p0 = raise2(x - ref), p1 = raise2(y - ref);
      m[r] = t;
      l[r] = l[r] * f + (p0 + p1);
      if (quarter == 0) {
        ps[r * PA_TILE + key] = p0;
        ps[r * PA_TILE + key + 8] = p1;
      }
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[r][g][e] *= f;
    }
    __syncwarp();
#pragma unroll 1
    for (int k = 0; k < PA_TILE; k += 4) {
      float4 w[ROWS];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) w[r] = *reinterpret_cast<const float4*>(ps + r * PA_TILE + k);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const int d = (lane + 32 * g) * 4;
        if (d >= D) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          T vv[4];
          if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(vv) = *reinterpret_cast<const uint4*>(vs + (k + i) * stride + d * 4);
          else *reinterpret_cast<uint2*>(vv) = *reinterpret_cast<const uint2*>(vs + (k + i) * stride + d * 2);
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            const float p = i == 0 ? w[r].x : i == 1 ? w[r].y : i == 2 ? w[r].z : w[r].w;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[r][g][e] = fmaf(p, Tr<T>::to_f(vv[e]), o[r][g][e]);
          }
        }
      }
    }
  }
  static __device__ __forceinline__ uint32_t at(int key, int c, int D) { return (uint32_t)(key * line(D) + c * 16); }
  __device__ __forceinline__ void publish(float* p, int, int D) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float* row = p + r * (D + 4);
      float sum = l[r];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      if (lane == 0) { row[0] = m[r]; row[1] = sum; }
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
template <int W, bool TAIL>
struct Plan {
  unsigned sum[W], live[W], base;
  int t, part[W];
  Tokens<TAIL> tok;
  Run run[4];
};

template <int THREADS>
__device__ __forceinline__ void meet(int barrier) { asm volatile("barrier.cta.sync %0, %1;" ::"r"(barrier), "n"(THREADS) : "memory"); }

// W warps that stream and multiply, and one that works out what they do next.  They meet at the end of every run.
// The code has to stay small: it is fetched through the memory that streams the keys, and when it had 90 KB every seldom taken path took microseconds.
// TAIL: only the slots behind the shared ones; every item leaves parts for the launch that joins them with those of the shared slots.  The launch before
// this one (paged_prefix_kernel) waits for everything older before it lets this one begin, and writes nothing that is read here, so this one waits
// for it at its end.
template <typename E, bool TAIL>
__global__ void __launch_bounds__(E::WARPS * 32 + 32, E::CTAS)
paged_attn_kernel(const __grid_constant__ PagedAttn a) {
  using T = typename E::T;
  constexpr int W = E::WARPS, THREADS = W * 32;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Plan<W, TAIL> s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int D = E::dim(a), chunks = D * (int)sizeof(T) / 16;
  const int per = a.H / a.G, blocks = (per + E::ROWS - 1) / E::ROWS, items = a.G * blocks;
  {                                                               // the first look at them is a wait for DRAM: all of it at once, beside the plan
    const int64_t line = (int64_t)blockIdx.x * (THREADS + 32) + threadIdx.x, tables = ((int64_t)a.pt.rows * a.pt.width * 4 + 127) / 128,
                  queries = ((int64_t)a.M * a.H * D * (int)sizeof(T) + 127) / 128;
    if (line < tables) prefetch_l2(reinterpret_cast<const uint8_t*>(a.pt.table) + line * 128);
    else if (line - tables < queries) prefetch_l2(reinterpret_cast<const uint8_t*>(a.q) + (line - tables) * 128);
  }
  if (!TAIL) pdl_wait();

  // ---- the plan: units of all tokens, the shares, the token in which this CTA's begins -------------------------------------
  const int chunk = (a.M + THREADS - 1) / THREADS;
  const int t0 = min(a.M, (int)threadIdx.x * chunk), t1 = min(a.M, t0 + chunk);        // (none for the last warp)
  unsigned mine = 0, live = 0;
#pragma unroll 1
  for (int t = t0; t < t1; ++t) {
    int from = 0;
    const Token tok = Token::of<TAIL>(a, t, W, &from);
    mine += tok.units * items;
    live += tok.units > 0;
    if (blockIdx.x == 0 && (a.t_row[t] >= a.pt.rows || (a.t_row[t] >= 0 && a.t_slot[t] >= table_slots(a.pt)))) atomicAdd(&g_paged_attn_fault, 1u);
    if (a.M <= PA_TOKENS) {
      s.tok.row[t] = tok.row;
      s.tok.slots[t] = TAIL && tok.row >= 0 ? slots_seen(a.pt, a.t_slot[t]) : tok.span.n;
      if (TAIL) s.tok.from[t] = from;
    }
  }
  unsigned before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned x = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += x;
  }
  live = __reduce_add_sync(0xffffffffu, live);
  if (lane == 31 && warp < W) {
    s.sum[warp] = before;
    s.live[warp] = live;
  }
  __syncthreads();
  before -= mine;
  unsigned U = 0, n_items = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < warp) before += s.sum[w];
    U += s.sum[w];
    n_items += s.live[w] * items;
  }
  pdl_launch_dependents();                                        // (the join waits for this launch's end; until then it has no room anyway)
  const Shares sh(U, n_items, gridDim.x - a.last, a.last);
  if (blockIdx.x >= sh.n) {
    if (TAIL) pdl_wait();
    return;
  }
  const unsigned ub = sh.begin(blockIdx.x);
#pragma unroll 1
  for (int t = t0; t < t1; ++t) {
    const unsigned n = (a.M <= PA_TOKENS ? Token(a, s.tok.row[t], s.tok.slots[t], TAIL ? s.tok.from[t] : 0, W) : Token::of<TAIL>(a, t, W)).units * items;
    if (ub - before < n) {
      s.t = t;
      s.base = before;
    }
    before += n;
  }
  __syncthreads();

  // ---- the warp for the runs and the parts ----------------------------------------------------------------------------------
  if (warp == W) {
    Cursor<TAIL> c;
    c.u = ub, c.end = sh.begin(blockIdx.x + 1), c.base = s.base, c.t = s.t;
    c.load(a, s.tok, W);
    // runs 0 to 2 before the others start, then run n + 3 when run n has ended
#pragma unroll 1
    for (int n = 0;; ++n) {
      Run r;
      r.tile = -1;
      if (c.next(a, s.tok, items, W)) {
        r.g = c.item / blocks;
        const int r0 = (c.item - r.g * blocks) * E::ROWS;
        r.tile = c.a * W, r.tile_end = min(c.b * W, c.tok.span.tiles);
        r.span = c.tok.span;
        r.row = c.tok.row, r.head = c.t * a.H + r.g * per + r0, r.rows = min(E::ROWS, per - r0), r.line = c.t * items + c.item;
        const bool cut = c.b - c.a < c.tok.units;
        r.part = cut ? (int)blockIdx.x * 2 + (c.a == 0 ? 1 : 0) : -1;
        if (c.a == 0 && lane == 0)                                // for the join
          a.parts[r.line] = make_uint2(blockIdx.x, cut ? sh.of(c.base + (c.item + 1) * c.tok.units - 1) - blockIdx.x + 1 : 1u);
      }
      if (lane == 0) s.run[n & 3] = r;
      if (n < 2) continue;
      if (n == 2) __syncthreads();
      meet<THREADS + 32>(2);                                      // the end of run n - 2
      if (s.run[(n - 1) & 3].tile < 0) {
        if (TAIL) pdl_wait();
        return;
      }
    }
  }

  // ---- loads run ahead of the products, across runs -------------------------------------------------------------------------
  uint8_t* ring = smem + E::Q_BYTES + warp * E::STAGES * E::tile_bytes(D);
  const uint32_t qs = (uint32_t)__cvta_generic_to_shared(smem), ring32 = (uint32_t)__cvta_generic_to_shared(ring);
  int tile = 0, tile_end = 0, ld_run = -1, id = -1, off = 0;      // the next tile to load: its run, its page, its place in it
  int inflight = 0, ld_stage = 0, stage = 0;                      // tiles on their way or here; where the next one goes; where the next one lies
  unsigned paged = 0;                                             // stages whose keys have a page
  Span ls(0, 0, 0);
  const int32_t* table = nullptr;
  int64_t kv_head = 0;
  uint4 qn[E::NQ];
  auto fetch_q = [&](const Run& r) {
    const uint4* q = reinterpret_cast<const uint4*>(a.q) + (int64_t)r.head * chunks;
    const int n = r.rows * chunks;
#pragma unroll
    for (int i = 0; i < E::NQ; ++i) {
      const int x = i * THREADS + (int)threadIdx.x;
      qn[i] = x < n ? q[x] : make_uint4(0, 0, 0, 0);
    }
  };
  auto put_q = [&]() {
#pragma unroll
    for (int i = 0; i < E::NQ; ++i) {
      const int x = i * THREADS + (int)threadIdx.x;
      if (x < E::ROWS * chunks) E::put_q(smem, x / chunks, x % chunks, qn[i], D);
    }
  };
  __syncthreads();
  fetch_q(s.run[0]);

  E e;
#pragma unroll 1
  for (int n = 0;; ++n) {
    const Run& r = s.run[n & 3];
    const bool more = s.run[(n + 1) & 3].tile >= 0;
    const int rows = r.rows, end = r.tile_end;
    const Span sp = r.span;
    float* scores = a.mass ? a.scores + (int64_t)r.line * a.cap * a.pitch : nullptr;
    bool begun = false;
#pragma unroll 1
    for (int v = r.tile + warp;; v += W) {
      // as many loads as there are stages (but one stage stays free at a run's end)
#pragma unroll 1
      while (inflight < (v < end ? E::STAGES : E::STAGES - 1)) {
        bool turned = false;
#pragma unroll 1
        while (tile >= tile_end && ld_run <= n) {                 // (no further than the run behind this one)
          const Run& l = s.run[(ld_run + 1) & 3];
          if (l.tile < 0) break;
          ++ld_run;
          tile = l.tile + warp, tile_end = l.tile_end;
          ls = l.span;
          table = a.pt.table + (int64_t)l.row * a.pt.width;
          kv_head = l.g;
          turned = true;
        }
        if (tile >= tile_end) break;
        auto seek = [&]() {
          const int kt = ls.key_tile(tile), index = (int)((uint64_t)(unsigned)kt * a.inv_tpp >> 36);
          off = kt - index * a.tpp;
          id = table[index];
        };
        if (turned) seek();
        const int j0 = ls.key0(tile);
        const bool page = (unsigned)id < (unsigned)a.pt.P, all = page && ls.whole(j0);
        const int64_t line = (((int64_t)(page ? id : 0) * a.G + kv_head) * a.tpp + off) * PA_TILE;
        const uint4* kg = reinterpret_cast<const uint4*>(a.k) + line * chunks + lane;
        const uint4* vg = reinterpret_cast<const uint4*>(a.v) + line * chunks + lane;
        const uint32_t ks = ring32 + ld_stage * E::tile_bytes(D), vs = ks + E::tile_bytes(D) / 2;
        paged = (paged & ~(1u << ld_stage)) | ((page ? 1u : 0u) << ld_stage);
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
              const bool ok = page && ls.visible(j0 + key);
              cp_async16(ks + at, ok ? kg + i * 32 : kg, ok);
              cp_async16(vs + at, ok ? vg + i * 32 : vg, ok);
            }
          }
        } else {
#pragma unroll 1
          for (int x = lane; x < PA_TILE * chunks; x += 32) {
            const int key = x / chunks, c = x - key * chunks;
            const bool ok = all || (page && ls.visible(j0 + key));
            cp_async16(ks + E::at(key, c, D), kg + (ok ? x - lane : 0), ok);
            cp_async16(vs + E::at(key, c, D), vg + (ok ? x - lane : 0), ok);
          }
        }
        cp_async_commit();
        ld_stage = ld_stage + 1 == E::STAGES ? 0 : ld_stage + 1;
        ++inflight;
        tile += W;
        if (tile < tile_end) seek();                              // a tile ahead
      }
      if (!begun) {
        begun = true;
        if (n == 0) {
          put_q();
          meet<THREADS>(1);
        }
        e.begin(qs);
        if (more) fetch_q(s.run[(n + 1) & 3]);                    // for the end of this run
      }
      if (v >= end) break;
      if (inflight >= 4) cp_async_wait<3>();
      else if (inflight == 3) cp_async_wait<2>();
      else if (inflight == 2) cp_async_wait<1>();
      else cp_async_wait<0>();
      __syncwarp();
      const int j0 = sp.key0(v);
      const bool page = (paged >> stage) & 1u;
      const bool all = page && sp.whole(j0);
      e.tile(a, qs, ring32 + stage * E::tile_bytes(D), j0, sp, all, page, scores ? scores + (int64_t)v * PA_TILE * a.pitch : nullptr, rows,
             ring + stage * E::tile_bytes(D));
      __syncwarp();                                               // the stage is refilled by the next load
      stage = stage + 1 == E::STAGES ? 0 : stage + 1;
      --inflight;
    }
    // ---- the warps' parts become one: each in the one stage of its ring that waits for nothing; a warp per head -------------
    const int part = (warp * E::STAGES + ld_stage) * E::tile_bytes(D);
    if (lane == 0) s.part[warp] = part;
    const int head = r.head;
    const bool cut = TAIL || r.part >= 0;
    float* rec = (TAIL && r.part < 0 ? a.whole + (int64_t)head * (D + 4) : a.rec + (int64_t)r.part * E::ROWS * (D + 4));
#pragma unroll 1
    for (int pass = 0; pass * 8 < rows; ++pass) {
      e.publish(reinterpret_cast<float*>(smem + E::Q_BYTES + part), pass, D);
      meet<THREADS>(1);
      if (pass == 0 && more) put_q();
#pragma unroll 1
      for (int row = warp; row < rows; row += W) {
        if (row >> 3 != pass) continue;
        float M = -INFINITY, L = 0.f, f[W];
        const float* p[W];
#pragma unroll
        for (int w = 0; w < W; ++w) {
          p[w] = reinterpret_cast<const float*>(smem + E::Q_BYTES + s.part[w]) + (row & 7) * (D + 4);
          f[w] = p[w][0];
          M = fmaxf(M, f[w]);
        }
        const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          f[w] = raise2(f[w] - ref);
          L += p[w][1] * f[w];
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll 1
        for (int d = 4 * lane; d < D; d += 128) {
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < W; ++w) {
            const float4 y = *reinterpret_cast<const float4*>(p[w] + 4 + d);
            acc.x += y.x * f[w]; acc.y += y.y * f[w]; acc.z += y.z * f[w]; acc.w += y.w * f[w];
          }
          if (!cut)
            store_row4<T>(reinterpret_cast<T*>(a.out) + ((int64_t)head + row) * D, d, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv),
                          a.out_perm);
          else
            *reinterpret_cast<float4*>(rec + row * (D + 4) + 4 + d) = acc;
        }
        if (lane == 0) {
          if (cut) *reinterpret_cast<float2*>(rec + row * (D + 4)) = make_float2(M, L);
          else if (a.mass) *reinterpret_cast<float2*>(a.stat + ((int64_t)head + row) * 2) = make_float2(ref, inv);
        }
      }
      if (pass * 8 + 8 < rows) meet<THREADS>(1);
    }
    meet<THREADS + 32>(2);
    if (!more) {
      if (TAIL) pdl_wait();
      return;
    }
  }
}

// Part i of an item that lies in the shares from c0 on: the first is its share's second, the others are their shares' first.
__device__ __forceinline__ const float* part_at(const PagedAttn& a, unsigned c0, unsigned i, int rows, int row) {
  return a.rec + (((int64_t)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * rows + row) * (a.D + 4);
}

// A warp's share of an item's parts, from i_first on: their maximum, sum and outputs, 128 dimensions of its lanes NQ times.
template <int NQ, int PJ_AHEAD>
__device__ __forceinline__ void sum_parts(const PagedAttn& a, uint2 parts, int row, int block_rows, unsigned i_first, unsigned i_step, float& M, float& L,
                                          float4 (&acc)[NQ]) {
  const int lane = threadIdx.x & 31;
  M = -INFINITY, L = 0.f;
#pragma unroll
  for (int x = 0; x < NQ; ++x) acc[x] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (unsigned i0 = i_first; i0 < parts.y; i0 += PJ_AHEAD * i_step) {
    float2 ml[PJ_AHEAD];
    float4 y[PJ_AHEAD][NQ];
#pragma unroll
    for (int u = 0; u < PJ_AHEAD; ++u) {
      const unsigned i = i0 + u * i_step;
      const bool in = i < parts.y;
      const float* p = part_at(a, parts.x, i, block_rows, row);
      ml[u] = in ? *reinterpret_cast<const float2*>(p) : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int x = 0; x < NQ; ++x)
        y[u][x] = in && 4 * lane + 128 * x < a.D ? *reinterpret_cast<const float4*>(p + 4 + 4 * lane + 128 * x) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float top = M;
#pragma unroll
    for (int u = 0; u < PJ_AHEAD; ++u) top = fmaxf(top, ml[u].x);
    const float ref = top == -INFINITY ? 0.f : top, f = raise2(M - ref);
    M = top;
    L *= f;
#pragma unroll
    for (int x = 0; x < NQ; ++x) acc[x].x *= f, acc[x].y *= f, acc[x].z *= f, acc[x].w *= f;
#pragma unroll
    for (int u = 0; u < PJ_AHEAD; ++u) {
      const float w = raise2(ml[u].x - ref);
      L += ml[u].y * w;
#pragma unroll
      for (int x = 0; x < NQ; ++x) acc[x].x += y[u][x].x * w, acc[x].y += y[u][x].y * w, acc[x].z += y[u][x].z * w, acc[x].w += y[u][x].w * w;
    }
  }
}

// A CTA per token and query head joins the parts where the item was cut: its warps take them in turn, then become one.  Few instructions: a launch
// this short waits for its code more than for its data.  Eight warps where the CTAs are few (one row of 1000 tokens of 32 heads, both launches, us, four /
// eight warps: 7.8 / 7.4), four where they are many (64 rows of 40 heads 25.2 / 26.4).  PJ_AHEAD parts of a warp on their way at once: four for the few,
// which have long lists (one key head over 60000 tokens 20.0 with one, 17.9 with three, 17.2 with four, 16.5 with eight, but one row of 1000 then 7.3 ->
// 7.5), one for the many (64 rows of 40 heads 25.2, with four 26.1).
template <typename T, int NQ, int PJ_WARPS, int PJ_AHEAD>
__device__ __forceinline__ void join_parts(const PagedAttn& a, int t, int64_t line, int row, int64_t head, int block_rows) {
  __shared__ float2 s_ml[PJ_WARPS];
  __shared__ float4 s_o[PJ_WARPS][32 * NQ];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int token_row = a.t_row[t];
  const uint2 parts = a.parts[line];
  if (token_row < 0 || token_row >= a.pt.rows || parts.y < 2) return;
  float M, L;
  float4 acc[NQ];
  sum_parts<NQ, PJ_AHEAD>(a, parts, row, block_rows, warp, PJ_WARPS, M, L, acc);
  if (lane == 0) s_ml[warp] = make_float2(M, L);
#pragma unroll
  for (int x = 0; x < NQ; ++x) s_o[warp][lane + 32 * x] = acc[x];
  __syncthreads();
  const int d = 4 * threadIdx.x;
  if (d >= a.D) return;
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < PJ_WARPS; ++w) top = fmaxf(top, s_ml[w].x);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int w = 0; w < PJ_WARPS; ++w) {
    const float f = raise2(s_ml[w].x - ref);
    const float4 y = s_o[w][threadIdx.x];
    sum += s_ml[w].y * f;
    o.x += y.x * f, o.y += y.y * f, o.z += y.z * f, o.w += y.w * f;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  store_row4<T>(reinterpret_cast<T*>(a.out) + head * a.D, d, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv), a.out_perm);
}

// The same by one warp.
template <typename T, int NQ>
__device__ __forceinline__ void join_alone(const PagedAttn& a, int t, int64_t line, int row, int64_t head, int block_rows) {
  const int token_row = a.t_row[t], lane = threadIdx.x & 31;
  const uint2 parts = a.parts[line];
  if (token_row < 0 || token_row >= a.pt.rows || parts.y < 2) return;
  float M, L;
  float4 acc[NQ];
  sum_parts<NQ, 4>(a, parts, row, block_rows, 0, 1, M, L, acc);
  const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
  for (int x = 0; x < NQ; ++x) {
    const int d = 4 * lane + 128 * x;
    if (d < a.D)
      store_row4<T>(reinterpret_cast<T*>(a.out) + head * a.D, d, make_float4(acc[x].x * inv, acc[x].y * inv, acc[x].z * inv, acc[x].w * inv), a.out_perm);
  }
}

template <typename T, int NQ, int PJ_WARPS>
__global__ void __launch_bounds__(PJ_WARPS * 32)
paged_attn_join_kernel(const __grid_constant__ PagedAttn a, int rows_log2) {
  const int r = blockIdx.x, g = blockIdx.y, t = blockIdx.z, rows = 1 << rows_log2, blocks = (gridDim.x + rows - 1) >> rows_log2;
  pdl_wait();
  const int64_t tg = (int64_t)t * a.G + g;
  join_parts<T, NQ, PJ_WARPS, PJ_WARPS == 8 ? 4 : 1>(a, t, tg * blocks + (r >> rows_log2), r & (rows - 1), tg * gridDim.x + r, rows);
}

// With a mass, one launch for both: the first CTAs (x) of an item (y) of a token (z) join its heads, a CTA each where the items are few, else one with
// a warp per head; the others are slices of the row's visible slots, a thread per slot, and add up the weights that it received.  The heads' maxima and
// sums come from the parts again (a warp per head, a lane per part), which needs no word from the join.  The slices of a row's first token in the call do so
// for all of the row's tokens and all of their heads in turn, the others leave, so that a slot's weights are added by one thread in one order (unless rows
// share its page).
// 12 rows of 972 to 3333 tokens, 64 heads: 26.1 us for the launch before, 5.8 for this one (9.0 with a CTA for every head).  (Atomics of all tokens at once took 1.4
// less there, and 50 for the last 32 of 2048 tokens instead of 115; four tokens of a row at a time 88 there, but 2 more for the 12 rows.)
template <typename T, int NQ, int ROWS>
__global__ void __launch_bounds__(256)
paged_attn_mass_kernel(const __grid_constant__ PagedAttn a, int per, int blocks, int joiners) {
  __shared__ float2 s_stat[2][ROWS];
  __shared__ int s_from[8];
  __shared__ int2 s_seen[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, items = a.G * blocks;
  const int t = blockIdx.z, item = blockIdx.y, g = blocks == 1 ? item : item / blocks, block = item - g * blocks;
  if ((int)blockIdx.x < joiners) {
    const int r0 = block * ROWS;
    pdl_wait();
    if (joiners == 1) {
#pragma unroll 1
      for (int r = warp; r < min(ROWS, per - r0); r += 8)
        join_alone<T, NQ>(a, t, (int64_t)t * items + item, r, (int64_t)t * a.H + (int64_t)g * per + r0 + r, ROWS);
    } else if (r0 + (int)blockIdx.x < per)
      join_parts<T, NQ, 8, 1>(a, t, (int64_t)t * items + item, blockIdx.x, (int64_t)t * a.H + (int64_t)g * per + r0 + blockIdx.x, ROWS);
    return;
  }
  if (block) return;
  // The tokens' rows and slots are older than the launch before this one, which let this one begin behind its own wait.
  const int slice = blockIdx.x - joiners, slices = gridDim.x - joiners, row = a.t_row[t];
  if (row < 0 || row >= a.pt.rows) return;
  bool before = false;                                            // a token of this row stands before this one: most often close by
  unsigned first32 = 0;                                           // which of the next tokens, this warp's 32 of 256, are of this row
  int lo = INT_MAX, hi = 0;                                       // the fewest and the most slots that one of them sees
#pragma unroll 1
  for (int i0 = 0; i0 < a.M; i0 += 256) {
    const int i = i0 + threadIdx.x;
    const bool mine = i < a.M - t && a.t_row[t + i] == row;
    if (i < t) before |= a.t_row[t - 1 - i] == row;
    if (mine) {
      const int n = slots_seen(a.pt, a.t_slot[t + i]);
      lo = min(lo, n), hi = max(hi, n);
    }
    const unsigned found = __ballot_sync(~0u, mine);
    if (i0 == 0) {
      first32 = found;
      if (a.M > 256 && __syncthreads_or(before)) return;
    }
  }
  lo = __reduce_min_sync(~0u, lo), hi = __reduce_max_sync(~0u, hi), before = __any_sync(~0u, before);
  if (lane == 0) s_from[warp] = (int)first32, s_seen[warp] = make_int2(lo, before ? -1 : hi);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    if (s_seen[w].y < 0) return;
    lo = min(lo, s_seen[w].x), hi = max(hi, s_seen[w].y);
  }
  const Span all(hi, a.first, lo < a.window || !a.window ? 0 : a.window + hi - lo);      // what any of them sees
  const int seen = all.tiles * PA_TILE;
  if (slice * 256 >= seen) return;
  int buffer = 0;
  bool waited = false;
#pragma unroll 1
  for (int base = t; base < a.M; base += 256) {
    // the row's tokens among the next 256, in their order
    unsigned found;
    if (base > t) {
      found = __ballot_sync(~0u, base + threadIdx.x < a.M && a.t_row[base + threadIdx.x] == row);
      __syncthreads();
      if (lane == 0) s_from[warp] = (int)found;
      __syncthreads();
    }
#pragma unroll 1
    for (int w = 0; w < 8; ++w)
#pragma unroll 1
      for (found = (unsigned)s_from[w]; found; found &= found - 1) {
        const int tt = base + 32 * w + __ffs(found) - 1;
        const Span span(slots_seen(a.pt, a.t_slot[tt]), a.first, a.window);
        if (!waited) pdl_wait(), waited = true;
#pragma unroll 1
        for (int blk = 0; blk < blocks; ++blk, buffer ^= 1) {
          const int rows = min(ROWS, per - blk * ROWS);
          const int64_t line = (int64_t)tt * items + g * blocks + blk, head = (int64_t)tt * a.H + (int64_t)g * per + blk * ROWS;
          const uint2 parts = a.parts[line];
          float w8[ROWS];
          int64_t place = -1;
          auto look = [&](int x) {                                // a slot's place and what its heads scored
            place = -1;
            if (x >= seen) return;
            const int kt = all.key_tile(x / PA_TILE), j = kt * PA_TILE + x % PA_TILE, index = (int)((uint64_t)(unsigned)kt * a.inv_tpp >> 36);
            if (!span.visible(j)) return;
            const int64_t id = page_id(a.pt, row, index);
            if (id < 0) return;
            place = (id * a.G + g) * a.pt.page + (kt - index * a.tpp) * PA_TILE + x % PA_TILE;
            const float* p = a.scores + (line * a.cap + span.tile_of(kt) * PA_TILE + x % PA_TILE) * a.pitch;
            if (a.pitch >= 4) {
#pragma unroll
              for (int r = 0; r < ROWS; r += 4)
                if (r < a.pitch) *reinterpret_cast<float4*>(w8 + r) = *reinterpret_cast<const float4*>(p + r);
            } else {
              w8[0] = p[0];
              if (a.pitch > 1) w8[1] = p[1];
            }
          };
          const int x0 = slice * 256 + threadIdx.x;
          look(x0);                                               // on its way beside the parts
#pragma unroll 1
          for (int r = warp; r < rows; r += 8) {
            float2 st;
            if (parts.y < 2) {
              st = reinterpret_cast<const float2*>(a.stat)[head + r];
            } else {
              float M = -INFINITY, L = 0.f;
#pragma unroll 1
              for (unsigned i = lane; i < parts.y; i += 32) {
                const float2 ml = *reinterpret_cast<const float2*>(part_at(a, parts.x, i, ROWS, r));
                const float top = fmaxf(M, ml.x), ref = top == -INFINITY ? 0.f : top;
                L = L * raise2(M - ref) + ml.y * raise2(ml.x - ref);
                M = top;
              }
              const float top = warp_max(M), ref = top == -INFINITY ? 0.f : top, sum = warp_sum(L * raise2(M - ref));
              st = make_float2(ref, sum == 0.f ? 0.f : 1.f / sum);
            }
            if (lane == 0) s_stat[buffer][r] = st;
          }
          __syncthreads();
#pragma unroll 1
          for (int x = x0; x < seen; x += slices * 256) {
            if (x != x0) look(x);
            if (place < 0) continue;
            float w = 0.f;
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
              if (r < rows) w += raise2(w8[r] - s_stat[buffer][r].x) * s_stat[buffer][r].y;
            atomicAdd(a.mass + place, w);                         // (rows may share the page)
          }
        }
      }
  }
}

}  // namespace b200p

#include "paged_shared.cuh"
#include "paged_prefix_tc.cuh"

namespace b200p {

// ------------------------------------------------------------------------------------------------ host
// visible slots a token can have, in whole tiles
static int64_t visible_cap(int64_t slots, int64_t first, int64_t window) {
  const int64_t seen = window > 0 ? first + window + 2 * PA_TILE : slots;
  return ((seen < slots ? seen : slots) + PA_TILE - 1) / PA_TILE * PA_TILE;
}

static size_t round256(size_t n) { return (n + 255) / 256 * 256; }
static size_t parts_bytes(int64_t M, int H) { return round256((size_t)M * H * 8); }      // (no more items than heads)
// two CTAs per SM at most and those for small shares: two parts of 16 heads each
static size_t rec_bytes(int D) { return round256((size_t)(2 * sm_count() + last_ctas(2 * sm_count())) * 2 * 16 * (D + 4) * 4); }
static size_t stat_bytes(int64_t M, int H) { return round256((size_t)M * H * 8); }

// The streaming launch; its grid and what it needs to know are written into a.
template <typename E, bool TAIL>
static int launch_stream(PagedAttn& a, cudaStream_t st) {
  const int smem = E::Q_BYTES + E::WARPS * E::STAGES * E::tile_bytes(a.D);
  const int blocks = (a.H / a.G + E::ROWS - 1) / E::ROWS, items = a.G * blocks;
  B200P_REQUIRE((int64_t)a.M * items * (a.cap / PA_TILE / E::WARPS + 1) < (1ll << 31) && (int64_t)a.M * a.H < (1ll << 31) && items < 65536, B200P_ERR_ARG,
                "%d tokens of %d key heads over %d slots: too many for one call", a.M, a.G, a.cap);
  auto kern = paged_attn_kernel<E, TAIL>;
  static std::atomic<uint64_t> ready{0};                          // devices whose copy of the kernel has its shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev > 63 || !(ready.load(std::memory_order_relaxed) >> dev & 1))) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 216 * 1024);
    if (e == cudaSuccess && dev < 64) ready.fetch_or(1ull << dev);
  }
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(paged_attn_kernel)");
  const int ctas = sm_count() * E::CTAS;
  const int64_t most = (int64_t)a.M * items * ((a.cap / PA_TILE + E::WARPS - 1) / E::WARPS);
  a.last = most >= (int64_t)PA_LAST_UNITS * ctas ? last_ctas(ctas) : 0;
  const int grid = (int)(most < ctas ? most : ctas) + a.last;
  a.tpp = a.pt.page / PA_TILE;
  a.inv_tpp = ((1ull << 36) + a.tpp - 1) / a.tpp;
  a.pitch = 1;
  while (a.pitch < E::ROWS && a.pitch < a.H / a.G) a.pitch *= 2;
  launch_pdl(kern, (unsigned)grid, E::WARPS * 32 + 32, smem, st, a);
  B200P_LAUNCH_CHECK("paged_attn_kernel");
  return B200P_OK;
}

template <typename E>
static int launch_paged(PagedAttn a, cudaStream_t st) {
  const int rc = launch_stream<E, false>(a, st);
  if (rc) return rc;
  using T = typename E::T;
  const int per = a.H / a.G, blocks = (per + E::ROWS - 1) / E::ROWS, items = a.G * blocks, rows_log2 = E::ROWS == 4 ? 2 : E::ROWS == 8 ? 3 : 4;
  const dim3 heads((unsigned)per, (unsigned)a.G, (unsigned)a.M);
  const bool few = (int64_t)a.M * a.H <= 4 * sm_count();             // CTAs of the join
  if (a.mass) {
    // slices of the visible slots: as many as there are, but no more CTAs than fill the GPU (each row's first token has some that stay)
    const int64_t stay = (int64_t)(a.M < a.pt.rows ? a.M : a.pt.rows) * items, slices = (a.cap + 255) / 256, fill = (6ll * sm_count() + stay - 1) / stay;
    const int joiners = few ? E::ROWS : 1;
    const dim3 rest((unsigned)(joiners + (slices < fill ? slices : fill)), (unsigned)items, (unsigned)a.M);
    launch_pdl(a.D <= 128 ? paged_attn_mass_kernel<T, 1, E::ROWS> : paged_attn_mass_kernel<T, 2, E::ROWS>, rest, 256, 0, st, a, per, blocks, joiners);
    B200P_LAUNCH_CHECK("paged_attn_mass_kernel");
    return B200P_OK;
  }
  if (few)
    launch_pdl(a.D <= 128 ? paged_attn_join_kernel<T, 1, 8> : paged_attn_join_kernel<T, 2, 8>, heads, 8 * 32, 0, st, a, rows_log2);
  else
    launch_pdl(a.D <= 128 ? paged_attn_join_kernel<T, 1, 4> : paged_attn_join_kernel<T, 2, 4>, heads, 4 * 32, 0, st, a, rows_log2);
  B200P_LAUNCH_CHECK("paged_attn_join_kernel");
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
  const bool four = a.H / a.G <= 4;
  if (a.D <= 128) return four ? launch_paged<FmaEngine<T, 1, 4>>(a, st) : launch_paged<FmaEngine<T, 1, 8>>(a, st);
  return four ? launch_paged<FmaEngine<T, 2, 4>>(a, st) : launch_paged<FmaEngine<T, 2, 8>>(a, st);
}

// ---- behind shared slots ------------------------------------------------------------------------------------------------------
// Which calls go by groups: those that the matrix instructions serve (fp32 and other sizes are bound by their FMAs, of which sharing saves none), and in
// which the tokens' rows could have keys and values of 64 MiB in common.  Below, the third launch costs more than the reading: us by token / by group, 32 / 8
// heads of 128, 16 rows behind 512 slots (30 MiB) 13.9 / 14.6, 32 behind 256 (31 MiB) 14.2 / 18.8, 8 behind 2000 (54 MiB) 16.9 / 16.6, 2 behind 16000 (63 MiB)
// 23.5 / 27.6, 64 behind 256 (63 MiB) 21.1 / 24.9, 4 behind 8000 (94 MiB) 23.4 / 22.8, 16 behind 2000 (116 MiB) 24.7 / 20.4, 64 behind 1000 48.1 / 31.3, 64
// behind 4000 134 / 43.  (Only the table's room is known here: what rows do have in common is on the device.)
static std::atomic<int> g_shared_path{0};                           // 1: by groups wherever it is served, 2: never
static bool shared_served(int64_t M, int H, int G, int D, int64_t slots, int dtype) {
  const int path = g_shared_path.load(std::memory_order_relaxed);
  if (path == 2 || dtype == B200P_F32 || H / G > PS_ROWS || !(D == 64 || D == 80 || D == 96 || D == 128 || D == 256)) return false;
  return path == 1 || (M - 1) * slots * G * D * 4 >= 64ll << 20;
}
static int shared_tile(int H, int G) { return H / G < PS_ROWS ? PS_ROWS / (H / G) : 1; }
static size_t whole_bytes(int64_t M, int H, int D) { return round256((size_t)M * H * (D + 4) * 4); }
static size_t prefix_bytes(int64_t M, int H, int D) { return round256(((size_t)M * H + (size_t)sm_count() * PS_ROWS) * (D + PS_HEAD) * 4); }
static size_t info_bytes(int64_t M) { return round256((size_t)M * 16 + 16); }

template <typename K>
static int shared_memory_of(K kern, int bytes, std::atomic<uint64_t>& ready, const char* what) {      // ready: devices whose copy of the kernel has it
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev > 63 || !(ready.load(std::memory_order_relaxed) >> dev & 1))) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) ready.fetch_or(1ull << dev);
  }
  return e == cudaSuccess ? B200P_OK : cuda_fail(e, what);
}

// tcgen05: copies of whole boxes of keys by 32-bit lines, and a scale that keeps the scores' order
template <typename T>
static int launch_prefix_tc(const PagedPrefix& p, unsigned ctas, cudaStream_t st) {
  static std::atomic<uint64_t> ready{0};
  auto kern = paged_prefix_tc_kernel<T>;
  if (const int rc = shared_memory_of(kern, FT_SMEM, ready, "cudaFuncSetAttribute(paged_prefix_tc_kernel)")) return rc;
  TcEncodeFn enc = tc_get_encode();
  B200P_REQUIRE(enc != nullptr, B200P_ERR_CUDA, "cuTensorMapEncodeTiled entry point not available");
  const CUtensorMapDataType dt = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  PagedPrefix q = p;
  if (const int rc = wait_word(WAIT_ATTN_TC, &q.wait_word)) return rc;
  q.box = q.pt.page % 128 == 0 ? 128 : q.pt.page % 64 == 0 ? 64 : q.pt.page % 32 == 0 ? 32 : 16;
  CUtensorMap tm[2];
  for (int i = 0; i < 2; ++i)
    if (const int rc = tc_encode_2d(enc, &tm[i], dt, i ? q.v : q.k, FT_D, (uint64_t)q.pt.P * q.G * q.pt.page, FT_D * 2, 64, (uint32_t)q.box,
                                    CU_TENSOR_MAP_SWIZZLE_128B, "cuTensorMapEncodeTiled(pages)"))
      return rc;
  launch_pdl(kern, ctas, FT_THREADS, FT_SMEM, st, tm[0], tm[1], q);
  B200P_LAUNCH_CHECK("paged_prefix_tc_kernel");
  return B200P_OK;
}

template <typename T, int D, int NB>
static int launch_shared(PagedAttn a, PagedPrefix p, int64_t tiles, cudaStream_t st) {
  using E = TcEngine<T, D, NB>;
  const bool tc = D == FT_D && p.scale_log2e >= 1e-30f && p.scale_log2e <= 1e30f && a.pt.P * a.G * a.pt.page < (1ll << 31) - FT_KEYS;
  const int64_t slots = (int64_t)a.pt.width * a.pt.page, kt = tc ? FT_KEYS : PrefixTile<T, D>::KT, units = tiles * a.G * (tc ? 1 : 2) * ((slots + kt - 1) / kt);
  B200P_REQUIRE(units < (1ll << 31), B200P_ERR_ARG, "%lld tiles of %d key heads over %lld slots: too many for one call", (long long)tiles, a.G, (long long)slots);
  const unsigned ctas = (unsigned)(units < sm_count() ? units : sm_count());
  p.tpp = a.pt.page / PA_TILE;
  p.inv_tpp = ((1ull << 36) + p.tpp - 1) / p.tpp;
  p.few = sm_count() / 2;
  int rc;
  if (tc) {
    if constexpr (D == FT_D) {
      if ((rc = launch_prefix_tc<T>(p, ctas, st))) return rc;
    }
  } else {
    static std::atomic<uint64_t> ready{0};
    auto kern = paged_prefix_kernel<T, D>;
    if ((rc = shared_memory_of(kern, PrefixTile<T, D>::SMEM, ready, "cudaFuncSetAttribute(paged_prefix_kernel)"))) return rc;
    launch_pdl(kern, ctas, PS_WARPS * 32, PrefixTile<T, D>::SMEM, st, p);
    B200P_LAUNCH_CHECK("paged_prefix_kernel");
  }
  if ((rc = launch_stream<E, true>(a, st))) return rc;
  // warps per query head: eight where the heads are few, one where they are many
  constexpr int NQ = D <= 128 ? 1 : 2;
  const int W = (int64_t)a.M * a.H <= 4 * sm_count() ? 8 : (int64_t)a.M * a.H <= 32 * sm_count() ? 2 : 1, rows = tc ? PS_ROWS : PS_HALF;
  const dim3 grid((unsigned)((a.H * W + 7) / 8), (unsigned)a.M);
  launch_pdl(W == 8 ? paged_shared_join_kernel<T, NQ, E::ROWS, 8> : W == 2 ? paged_shared_join_kernel<T, NQ, E::ROWS, 2> : paged_shared_join_kernel<T, NQ, E::ROWS, 1>, grid, 256, 0, st, a, p, (int)ctas, rows);
  B200P_LAUNCH_CHECK("paged_shared_join_kernel");
  return B200P_OK;
}

template <typename T>
static int launch_shared_type(const PagedAttn& a, const PagedPrefix& p, int64_t tiles, cudaStream_t st) {
  const bool few = a.H / a.G <= 8;
  switch (a.D) {
    case 64: return few ? launch_shared<T, 64, 1>(a, p, tiles, st) : launch_shared<T, 64, 2>(a, p, tiles, st);
    case 80: return few ? launch_shared<T, 80, 1>(a, p, tiles, st) : launch_shared<T, 80, 2>(a, p, tiles, st);
    case 96: return few ? launch_shared<T, 96, 1>(a, p, tiles, st) : launch_shared<T, 96, 2>(a, p, tiles, st);
    case 128: return few ? launch_shared<T, 128, 1>(a, p, tiles, st) : launch_shared<T, 128, 2>(a, p, tiles, st);
    default: return launch_shared<T, 256, 1>(a, p, tiles, st);
  }
}

}  // namespace b200p

using namespace b200p;

static size_t workspace_bytes(int64_t M, int H, int D, int64_t keys, int64_t lines) {
  if (M <= 0 || H <= 0 || D <= 0) return 0;
  size_t n = parts_bytes(M, H) + rec_bytes(D);
  if (keys > 0) n += stat_bytes(M, H) + (size_t)M * lines * ((keys + PA_TILE - 1) / PA_TILE * PA_TILE) * 4;
  return n;
}

extern "C" size_t b200p_paged_attn_workspace_bytes(int64_t M, int H, int D, int64_t keys) {
  return workspace_bytes(M, H, D, keys, 2 * (int64_t)H);          // (a line of scores is less than twice its heads, whatever G)
}

extern "C" size_t b200p_paged_attn_workspace_bytes_of(int64_t M, int H, int G, int D, int64_t keys) {
  if (G <= 0 || H < G || H % G) return 0;
  // a key head's scores of a slot: a power of two up to 16 heads, whole blocks of 16 behind that (blocks of 4 or 8 take no more)
  const int per = H / G;
  int64_t line = 1;
  while (line < 16 && line < per) line *= 2;
  if (per > 16) line = (per + 15) / 16 * 16;
  return workspace_bytes(M, H, D, keys, G * line);
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
  B200P_REQUIRE(workspace && workspace_bytes >= b200p_paged_attn_workspace_bytes_of(M, H, G, D, mass ? cap : 0) && aligned(workspace, 256), B200P_ERR_ARG,
                "paged attention workspace too small or not aligned to 256 bytes");
  PagedAttn a{};
  a.q = q, a.k = kpages, a.v = vpages, a.out = out, a.mass = mass, a.pt = pt, a.t_row = t_row, a.t_slot = t_slot;
  a.M = (int)M, a.H = H, a.G = G, a.D = D, a.first = (int)first, a.window = (int)window, a.out_perm = (flags & B200P_OUT_PERM8) ? 1 : 0;
  a.scale_log2e = scale * 1.4426950408889634f, a.cap = (int)cap;
  uint8_t* ws = (uint8_t*)workspace;
  a.parts = (uint2*)ws;
  a.rec = (float*)(ws += parts_bytes(M, H));
  a.stat = (float*)(ws += rec_bytes(D));
  a.scores = (float*)(ws + stat_bytes(M, H));
  B200P_DISPATCH_DTYPE(dtype, T, return (launch_paged_type<T>(a, (cudaStream_t)stream)));
  return B200P_OK;
}

extern "C" int b200p_paged_attn_shared_set_path(int path) {
  B200P_REQUIRE(path >= 0 && path <= 2, B200P_ERR_ARG, "path %d: 0 by the rule, 1 by groups, 2 by tokens", path);
  g_shared_path.store(path, std::memory_order_relaxed);
  return B200P_OK;
}

extern "C" int b200p_paged_attn_shared_tile(int H, int G) { return G > 0 && H >= G && H % G == 0 ? shared_tile(H, G) : 0; }

extern "C" size_t b200p_paged_attn_shared_workspace_bytes(int64_t M, int H, int G, int D, int groups) {
  if (M <= 0 || G <= 0 || H < G || H % G || D <= 0 || groups <= 0 || groups > RG_GROUPS) return 0;
  return workspace_bytes(M, H, D, 0, 0) + whole_bytes(M, H, D) + prefix_bytes(M, H, D) + info_bytes(M);
}

extern "C" int b200p_paged_attn_shared(const void* q, const void* kpages, const void* vpages, const int32_t* table, const int32_t* t_row,
                                       const int32_t* t_slot, void* out, const int32_t* index, const int32_t* prefix, const int32_t* plan, int64_t M, int H,
                                       int G, int D, int groups, int tile, int64_t P, int page, int rows, int width, float scale, int dtype, int flags,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  B200P_REQUIRE(M == 0 || (index && prefix && plan), B200P_ERR_ARG, "null pointer");
  B200P_REQUIRE(groups > 0 && groups <= RG_GROUPS, B200P_ERR_ARG, "%d groups: 1 to %d", groups, RG_GROUPS);
  B200P_REQUIRE(G > 0 && H > 0 && H % G == 0, B200P_ERR_ARG, "bad head counts %d/%d", H, G);
  B200P_REQUIRE(tile == shared_tile(H, G), B200P_ERR_ARG, "the plan's tiles have %d rows for these heads, not %d", shared_tile(H, G), tile);
  B200P_REQUIRE(aligned(plan, 16), B200P_ERR_ALIGN, "the plan must be 16-byte aligned");
  B200P_REQUIRE(M <= 0 || (workspace && workspace_bytes >= b200p_paged_attn_shared_workspace_bytes(M, H, G, D, groups)), B200P_ERR_ARG,
                "workspace of paged attention behind shared slots too small");
  if (M <= 0 || !shared_served(M, H, G, D, (int64_t)width * page, dtype))                     // (the other checks are paged attention's)
    return b200p_paged_attn(q, kpages, vpages, nullptr, table, t_row, t_slot, out, M, H, G, D, P, page, rows, width, scale, 0, 0, dtype, flags, workspace,
                            workspace_bytes, stream);
  PdlClass pdl_cls(8);
  const PageTable pt{table, P, rows, width, page};
  const int rc = check_pages(kpages, vpages, pt, G, D, dtype);
  if (rc) return rc;
  B200P_REQUIRE(q && out && t_row && t_slot, B200P_ERR_ARG, "null pointer");
  B200P_REQUIRE(M < 65536, B200P_ERR_ARG, "bad shape: %lld tokens", (long long)M);
  B200P_REQUIRE((flags & ~B200P_OUT_PERM8) == 0, B200P_ERR_ARG, "unknown flags 0x%x", flags);
  B200P_REQUIRE(aligned(q, 16) && aligned(out, 16), B200P_ERR_ALIGN, "q and out must be 16-byte aligned");
  B200P_REQUIRE(aligned(workspace, 256), B200P_ERR_ARG, "workspace not aligned to 256 bytes");
  PagedAttn a{};
  a.q = q, a.k = kpages, a.v = vpages, a.out = out, a.pt = pt, a.t_row = t_row, a.t_slot = t_slot;
  a.M = (int)M, a.H = H, a.G = G, a.D = D, a.out_perm = (flags & B200P_OUT_PERM8) ? 1 : 0;
  a.scale_log2e = scale * 1.4426950408889634f, a.cap = (int)visible_cap((int64_t)width * page, 0, 0);
  a.index = index, a.prefix = prefix, a.groups = groups;
  uint8_t* ws = (uint8_t*)workspace;
  a.parts = (uint2*)ws;
  a.rec = (float*)(ws += parts_bytes(M, H));
  a.whole = (float*)(ws += rec_bytes(D));
  PagedPrefix p{};
  p.q = q, p.k = kpages, p.v = vpages, p.pt = pt, p.t_row = t_row, p.t_slot = t_slot, p.index = index, p.prefix = prefix;
  p.plan = RowGroups{plan, (int)M}, p.M = (int)M, p.H = H, p.G = G, p.groups = groups, p.scale_log2e = a.scale_log2e;
  p.rec = (float*)(ws += whole_bytes(M, H, D));
  p.rec_rows = (int64_t)(prefix_bytes(M, H, D) / ((D + PS_HEAD) * 4));
  p.info = (int4*)(ws += prefix_bytes(M, H, D));
  p.total = (unsigned*)(p.info + M);
  const int64_t tiles = row_group_tiles(M, groups, tile);
  return dtype == B200P_F16 ? launch_shared_type<__half>(a, p, tiles, (cudaStream_t)stream) : launch_shared_type<__nv_bfloat16>(a, p, tiles, (cudaStream_t)stream);
}
