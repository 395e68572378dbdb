// Paged key-value cache: append (norms, rotation, write), eviction by received attention weight (selection, closing up), dense view.
#include <cooperative_groups.h>
#include <stdlib.h>

#include <atomic>

#include "mma_util.cuh"
#include "paged.cuh"

namespace b200p {

namespace cg = cooperative_groups;
int sm_count();

// How often the append, the eviction and the dense view met an id that names no page where they needed one, or a row longer than the table
// (b200p_paged_fault_count).
__device__ unsigned int g_paged_fault = 0;

int paged_attn_faults(unsigned int* count, int reset, cudaStream_t st);

// ------------------------------------------------------------------------------------------------ append
// Sine and cosine of position * rate: the product in double precision, reduced to a turn there (positions of 10^6 times a rate of one leave fp32 with
// an error of 0.06 rad).
__device__ __forceinline__ float2 turn(int pos, float rate) {
  const double turns = (double)pos * (double)rate * 0.15915494309189535;
  float2 sc;
  sincospif((float)((turns - rint(turns)) * 2.0), &sc.x, &sc.y);
  return sc;
}

// Every head is split over 2^width_log2 lanes (the power of two that holds D / 8), 8 neighbouring values a lane: one to two 16-byte loads and stores (8
// bytes at a time, four values and the four that they turn with, took 102 us), a rotation partner from the lane that has it (pairs of halves) or from
// this one (neighbours).  A lane keeps its angles and the norms' weights and walks over heads: without norms one after the other, four on their way (two where
// the tokens are few); with them two at once, their mean squares by shuffles side by side.  A CTA holds 2^tpc_log2 tokens, each with (256 >> width_log2) >>
// tpc_log2 walkers, and where the tokens are few gridDim.y CTAs share a token's heads.  fp32 from the read to the one rounding.
// Bound by HBM from some hundred tokens on, with norms by the instructions: 6004 tokens of 64 + 16 heads of 128, 246 MB, 47.5 us (two ahead 52.5), with
// norms 62.5 (four at once 66, one after the other 84); one token 2.6.  (A CTA per token, a warp per head and an element per lane took 114 us;
// CTAs that take their tokens one after the other, so that what is read lies closer together, 73.)
template <typename T, typename TIN, int AHEAD, bool PAIRS, bool NORM>
__global__ void __launch_bounds__(256, 3)
paged_append_rows_kernel(TIN* qkv, int64_t ldq, T* q_out, T* kp, T* vp, float* mass, PageTable pt, const int32_t* t_row, const int32_t* t_slot,
                         const int32_t* t_pos, const T* qw, const T* kw, const float* rates, int n_rot, float eps, int M, int H, int G, int D,
                         int width_log2, int tpc_log2) {
  constexpr bool ACC_IN = !std::is_same<TIN, T>::value;
  constexpr int IN = sizeof(TIN) * 8 / 16, OUT = sizeof(T) * 8 / 16, TURNS = PAIRS ? 4 : 8;      // 16-byte pieces of 8 values; angles
  constexpr int GROUP = NORM ? AHEAD : 1;                         // heads worked on at once
  __shared__ float2 s_turn[8][128];
  const int tpc = 1 << tpc_log2, width = 1 << width_log2, token0 = blockIdx.x << tpc_log2;
  const int c = threadIdx.x & (width - 1), slot = threadIdx.x >> width_log2;
  const int k = slot & (tpc - 1), t = min(token0 + k, M - 1), step = (256 >> width_log2) >> tpc_log2;
  const bool mine = token0 + k < M && c < D / 8;
  pdl_wait();
  const int row = t_row[t], place = t_slot[t], heads = H + 2 * G;
  const bool live = row >= 0 && row < pt.rows;
  TIN* src = qkv + (int64_t)t * ldq + 8 * c;
  const int first = (int)blockIdx.y * step + (slot >> tpc_log2), stride = step * gridDim.y;
  uint4 in[AHEAD][IN];
  auto fetch = [&](uint4 (&into)[IN], int head) {
    if (mine && (live || ACC_IN) && head < heads) {
      uint4* p = reinterpret_cast<uint4*>(src + (int64_t)head * D);
#pragma unroll
      for (int i = 0; i < IN; ++i) {
        into[i] = p[i];
        if (ACC_IN) p[i] = make_uint4(0, 0, 0, 0);
      }
    }
  };
#pragma unroll
  for (int a = 0; a < AHEAD; ++a) fetch(in[a], first + a * stride);      // on their way while the angles are worked out
  for (int i = threadIdx.x; i < n_rot << tpc_log2; i += 256) {
    const int kk = i & (tpc - 1), pair = i >> tpc_log2;
    if (token0 + kk < M) s_turn[kk][pair] = turn(t_pos[token0 + kk], rates[pair]);
  }
  int64_t id = -1;
  if (live && place >= 0 && place < table_slots(pt)) id = page_id(pt, row, place / pt.page);
  if (mine && c == 0 && slot < tpc && blockIdx.y == 0 && (row >= pt.rows || (live && id < 0))) atomicAdd(&g_paged_fault, 1u);
  const int off = id < 0 ? 0 : place % pt.page;
  uint4 weight[2][OUT];                                           // of queries and keys
  if constexpr (NORM)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const T* w = i ? kw : qw;
#pragma unroll
      for (int n = 0; n < OUT; ++n)
        if (w && c < D / 8) weight[i][n] = reinterpret_cast<const uint4*>(w + 8 * c)[n];
    }
  __syncthreads();
  const float inv_D = 1.f / (float)D;
  float cs[TURNS], sn[TURNS];                                     // halves: out = x * cs + partner * sn
  const int partner = (threadIdx.x & 31) + (PAIRS || 8 * c >= 2 * n_rot ? 0 : 8 * c < n_rot ? n_rot / 8 : -(n_rot / 8));
#pragma unroll
  for (int j = 0; j < TURNS; ++j) {
    const int e = TURNS * c + j;
    const bool turns = e < (PAIRS ? n_rot : 2 * n_rot), second = !PAIRS && e >= n_rot;
    const float2 sc = turns ? s_turn[k][second ? e - n_rot : e] : make_float2(0.f, 1.f);
    cs[j] = sc.y, sn[j] = PAIRS || second ? sc.x : -sc.x;
  }
#pragma unroll 1
  for (int base = first; base - first < heads; base += AHEAD * stride) {      // the same number of turns for every lane of a warp
#pragma unroll
    for (int a0 = 0; a0 < AHEAD; a0 += GROUP) {
      float x[GROUP][8];
#pragma unroll
      for (int a = 0; a < GROUP; ++a) {
        const int head = base + (a0 + a) * stride;
        const bool ok = mine && live && head < heads;
        const TIN* v = reinterpret_cast<const TIN*>(in[a0 + a]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[a][j] = ok ? Tr<TIN>::to_f(v[j]) : 0.f;
          if (ACC_IN) x[a][j] = Tr<T>::to_f(Tr<T>::from_f(x[a][j]));
        }
        fetch(in[a0 + a], head + AHEAD * stride);
      }
      if constexpr (NORM) {
        float ss[GROUP];
#pragma unroll
        for (int a = 0; a < GROUP; ++a) {
          ss[a] = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) ss[a] += x[a][j] * x[a][j];
        }
        for (int o = 1; o < width; o <<= 1)
#pragma unroll
          for (int a = 0; a < GROUP; ++a) ss[a] += __shfl_xor_sync(0xffffffffu, ss[a], o);
#pragma unroll
        for (int a = 0; a < GROUP; ++a) {
          const int head = base + (a0 + a) * stride;
          const bool queries = head < H;
          if (head < H + G && (queries ? qw : kw)) {
            const float inv = rsqrtf(fmaf(ss[a], inv_D, eps));
            uint4 w8[OUT];
#pragma unroll
            for (int n = 0; n < OUT; ++n) w8[n] = queries ? weight[0][n] : weight[1][n];
            const T* w = reinterpret_cast<const T*>(w8);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[a][j] *= inv * Tr<T>::to_f(w[j]);
          }
        }
      }
#pragma unroll
      for (int a = 0; a < GROUP; ++a) {
        const int head = base + (a0 + a) * stride;
        if (n_rot) {
          const bool turned = head < H + G && 8 * c < 2 * n_rot;
          if constexpr (PAIRS) {
            if (turned)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (4 * c + j < n_rot) {
                  const float y0 = x[a][2 * j], y1 = x[a][2 * j + 1];
                  x[a][2 * j] = y0 * cs[j] - y1 * sn[j];
                  x[a][2 * j + 1] = y0 * sn[j] + y1 * cs[j];
                }
          } else {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = __shfl_sync(0xffffffffu, x[a][j], partner);
            if (turned)
#pragma unroll
              for (int j = 0; j < 8; ++j) x[a][j] = x[a][j] * cs[j] + y[j] * sn[j];
          }
        }
        if (!(mine && live && head < heads)) continue;
        T* dst;
        if (head < H) {
          dst = q_out + ((int64_t)t * H + head) * D;
        } else {
          if (id < 0) continue;
          const int64_t at = (id * G + (head < H + G ? head - H : head - H - G)) * pt.page + off;
          dst = (head < H + G ? kp : vp) + at * D;
          if (mass && head < H + G && c == 0) mass[at] = 0.f;
        }
        uint4* to = reinterpret_cast<uint4*>(dst + 8 * c);
        if constexpr (sizeof(T) == 2) {
          *to = make_uint4(pack2<T>(x[a][0], x[a][1]), pack2<T>(x[a][2], x[a][3]), pack2<T>(x[a][4], x[a][5]), pack2<T>(x[a][6], x[a][7]));
        } else {
          *reinterpret_cast<float4*>(to) = make_float4(x[a][0], x[a][1], x[a][2], x[a][3]);
          *reinterpret_cast<float4*>(to + 1) = make_float4(x[a][4], x[a][5], x[a][6], x[a][7]);
        }
      }
    }
  }
}

// The same for what the lanes above do not hold (halves that are no multiple of 8 values apart, rows that are not 16-byte aligned): one CTA per token, a
// warp per head.
template <typename T, typename TIN>
__global__ void __launch_bounds__(256)
paged_append_kernel(TIN* qkv, int64_t ldq, T* q_out, T* kp, T* vp, float* mass, PageTable pt, const int32_t* t_row, const int32_t* t_slot,
                    const int32_t* t_pos, const T* qw, const T* kw, const float* rates, int n_rot, int pairs, float eps, int H, int G, int D) {
  __shared__ float sn[128], cs[128];
  __shared__ float buf[8][256];
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = t_row[t], slot = t_slot[t];
  TIN* src0 = qkv + (int64_t)t * ldq;
  constexpr bool ACC_IN = !std::is_same<TIN, T>::value;
  const bool live = row >= 0 && row < pt.rows;
  int64_t id = -1;
  if (live) {
    if (slot >= 0 && slot < table_slots(pt)) id = page_id(pt, row, slot / pt.page);
    for (int i = threadIdx.x; i < n_rot; i += blockDim.x) {
      const float2 sc = turn(t_pos[t], rates[i]);
      sn[i] = sc.x;
      cs[i] = sc.y;
    }
  }
  if (threadIdx.x == 0 && (row >= pt.rows || (live && id < 0))) atomicAdd(&g_paged_fault, 1u);
  __syncthreads();
  const int off = slot % pt.page;
  for (int h = warp; h < H + 2 * G; h += 8) {
    TIN* src = src0 + (int64_t)h * D;
    float ss = 0.f;
    for (int i = lane; i < D; i += 32) {
      float x = Tr<TIN>::to_f(src[i]);
      if constexpr (ACC_IN) {
        x = Tr<T>::to_f(Tr<T>::from_f(x));
        src[i] = TIN(0.f);
      }
      buf[warp][i] = x;
      ss += x * x;
    }
    if (!live) continue;
    const T* w = h < H ? qw : (h < H + G ? kw : nullptr);
    if (w) {
      const float inv = 1.f / sqrtf(warp_sum(ss) / (float)D + eps);
      for (int i = lane; i < D; i += 32) buf[warp][i] *= inv * Tr<T>::to_f(w[i]);
    }
    __syncwarp();
    if (h < H + G) {
      for (int i = lane; i < n_rot; i += 32) {
        const int a = pairs ? 2 * i : i, b = pairs ? 2 * i + 1 : i + n_rot;
        const float x = buf[warp][a], y = buf[warp][b];
        buf[warp][a] = x * cs[i] - y * sn[i];
        buf[warp][b] = x * sn[i] + y * cs[i];
      }
      __syncwarp();
    }
    T* dst;
    if (h < H) {
      dst = q_out + ((int64_t)t * H + h) * D;
    } else {
      if (id < 0) continue;
      const int g = h < H + G ? h - H : h - H - G;
      const int64_t at = (id * G + g) * pt.page + off;
      dst = (h < H + G ? kp : vp) + at * D;
      if (mass && h < H + G && lane == 0) mass[at] = 0.f;
    }
    for (int i = lane; i < D; i += 32) dst[i] = Tr<T>::from_f(buf[warp][i]);
    __syncwarp();
  }
}

// ------------------------------------------------------------------------------------------------ eviction
// Order of the weights as integers: larger weight, larger number; NaN and places without a page lowest, both zeros equal.
__device__ __forceinline__ uint32_t weight_key(float x) {
  if (!(x == x)) return 0u;
  if (x == 0.f) return 0x80000000u;
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// A cluster of CTAs per row and key head, each with a run of the row's slots whose keys it keeps in shared memory (rows too long for that: it reads the
// weights anew in every pass).  The need-th largest key of the candidates [first, n - recent) in three passes over 11, 11 and 10 bits: every CTA counts
// its keys' digits, then adds up all CTAs' counts of its share of the digits through distributed shared memory and hands the sums to the others' copies;
// the digit in which the need-th lies is found from the sums.  Then each warp counts what it keeps of its slots, and with the counts before it (of the keys
// equal to the last one the lowest slots are kept) it writes them in order.  Bound by its few barriers: the weights are 4 bytes a slot.
// (One CTA, 8 bits at a time from global memory: 40001 slots of 8 heads took 230 us, now 21.)  Whether the keys are held goes by the table's width,
// which the host knows, not by the rows' lengths: 64 rows of 4096 of 8 heads take 31.8 us, and 63.6 in a table of 65536 slots.
constexpr int SEL_MAX_CLUSTER = 8, SEL_BINS = 2048;

struct SelShared {
  unsigned hist[SEL_BINS], sums[SEL_BINS];
  unsigned warp_sum[32];
  unsigned digit, left;
  bool all;
  unsigned take[32], eq[32];
  unsigned all_above, all_eq;          // this CTA's, for the others
};

template <int SEL_THREADS>
__global__ void __launch_bounds__(SEL_THREADS)
paged_select_kernel(const float* mass, PageTable pt, const int32_t* lengths, int32_t* kept, int G, int keep, int first, int recent, int room) {
  constexpr int SEL_WARPS = SEL_THREADS / 32, EACH = SEL_BINS / SEL_THREADS;
  extern __shared__ uint32_t keys[];
  __shared__ SelShared s;
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned S = cluster.num_blocks(), rank = cluster.block_rank();
  const int g = blockIdx.y, r = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  int n = lengths[r];
  if (n > table_slots(pt) && g == 0 && rank == 0 && tid == 0) atomicAdd(&g_paged_fault, 1u);
  n = n < 0 ? 0 : (n > table_slots(pt) ? table_slots(pt) : n);
  int32_t* out = kept + ((int64_t)r * G + g) * keep;
  if (n <= keep) {                                                // the same for the whole cluster
    for (int i = rank * SEL_THREADS + tid; i < keep; i += S * SEL_THREADS) out[i] = i < n ? i : -1;
    return;
  }
  // this CTA's slots [j0, j1): whole tiles, and in each warp a run of 32 at a time
  const int per = ((n + (int)S - 1) / (int)S + 31) / 32 * 32, j0 = min(n, (int)rank * per), j1 = min(n, j0 + per);
  const int lo = first, hi = n - recent;
  const bool held = per <= room;
  auto look = [&](int j) -> uint32_t {
    const int64_t id = page_id(pt, r, j / pt.page);
    return id < 0 ? 0u : weight_key(mass[(id * G + g) * pt.page + j % pt.page]);
  };
  for (int i = tid; i < SEL_BINS; i += SEL_THREADS) s.hist[i] = 0;
  if (held) {
#pragma unroll 4
    for (int j = j0 + tid; j < j1; j += SEL_THREADS) keys[j - j0] = look(j);      // (a thread looks at its own slots again below)
  }
  __syncthreads();
  unsigned need = (unsigned)(keep - first - recent), prefix = 0, mask = 0;
  const bool picks = need > 0;
  constexpr int BITS[3] = {11, 11, 10};
  int shift = 32;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    if (!picks && pass > 0) break;
    const int bits = BITS[pass], bins = 1 << bits;
    shift -= bits;
    for (int b = j0 + warp * 32; b < j1; b += SEL_THREADS) {
      const int j = b + lane;
      uint32_t u = 0;
      if (j < j1) u = held ? keys[j - j0] : look(j);
      // tokens that nobody looked at have equal weights: one count for a warp whose keys share a digit
      const bool counts = picks && j < j1 && j >= lo && j < hi && (u & mask) == prefix;
      const unsigned d = (u >> shift) & (bins - 1), who = __ballot_sync(0xffffffffu, counts);
      if (!who) continue;
      const int leader = __ffs(who) - 1;
      const unsigned common = __shfl_sync(0xffffffffu, d, leader);
      if (__all_sync(0xffffffffu, !counts || d == common)) {
        if (lane == leader) atomicAdd(&s.hist[d], (unsigned)__popc(who));
      } else if (counts) {
        atomicAdd(&s.hist[d], 1u);
      }
    }
    if (!picks) break;
    const unsigned* sums = s.hist;
    if (S == 1) {
      __syncthreads();
    } else {                                                      // all CTAs' counts of this CTA's share of the digits, into every CTA
      sums = s.sums;
      cluster.sync();
      const int part = bins / (int)S;
      for (int i = tid; i < part; i += SEL_THREADS) {
        const int d = rank * part + i;
        unsigned sum = 0;
        for (unsigned c = 0; c < S; ++c) sum += cluster.map_shared_rank(s.hist, c)[d];
        for (unsigned c = 0; c < S; ++c) cluster.map_shared_rank(s.sums, c)[d] = sum;
      }
      cluster.sync();
    }
    // the digit: the largest with at least `need` keys from it up.  Thread i holds the digits [i w, (i + 1) w) counted from the top
    const int w = bins / SEL_THREADS, top = bins - 1 - tid * w;
    unsigned c[EACH], mine = 0;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      c[k] = k < w ? sums[top - k] : 0;
      mine += c[k];
    }
    unsigned before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned x = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += x;
    }
    if (lane == 31) s.warp_sum[warp] = before;
    __syncthreads();
    for (int i = tid; i < SEL_BINS; i += SEL_THREADS) s.hist[i] = 0;
    unsigned others = lane < warp ? s.warp_sum[lane] : 0;      // (warp: below 32)
    others = __reduce_add_sync(0xffffffffu, others);
    before += others - mine;
    if (before < need && before + mine >= need) {
#pragma unroll
      for (int k = 0; k < EACH; ++k) {
        if (before < need && before + c[k] >= need) {
          s.digit = top - k;
          s.left = need - before;
          s.all = c[k] == need - before;
        }
        before += c[k];
      }
    }
    __syncthreads();
    prefix |= s.digit << shift;
    need = s.left;
    mask |= (unsigned)(bins - 1) << shift;
    if (s.all && prefix) {                                        // every key of this digit is kept: no need to look at the others' bits
      --prefix;
      need = 0;
      break;
    }
  }
  __syncthreads();
  // ---- counts of what is kept for certain and of the keys equal to the last one, by warp and by CTA ------------------------
  const int run = (per / 32 + SEL_WARPS - 1) / SEL_WARPS * 32, w0 = min(j1, j0 + warp * run), w1 = min(j1, w0 + run);
  auto key_at = [&](int j) -> uint32_t { return held ? keys[j - j0] : look(j); };
  unsigned above = 0, equal = 0;
  for (int b = w0; b < w1; b += 32) {
    const int j = b + lane;
    const bool always = j < w1 && (j < lo || j >= hi), cand = picks && j < w1 && !always;
    const uint32_t u = cand ? key_at(j) : 0u;
    above += __popc(__ballot_sync(0xffffffffu, always || (cand && u > prefix)));
    equal += __popc(__ballot_sync(0xffffffffu, cand && u == prefix));
  }
  if (lane == 0) {
    s.take[warp] = above;
    s.eq[warp] = equal;
  }
  __syncthreads();
  unsigned a = lane < SEL_WARPS ? s.take[lane] : 0, e = lane < SEL_WARPS ? s.eq[lane] : 0, sum_a = a, sum_e = e;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned x = __shfl_up_sync(0xffffffffu, sum_a, o), y = __shfl_up_sync(0xffffffffu, sum_e, o);
    if (lane >= o) sum_a += x, sum_e += y;
  }
  if (tid == 31) {
    s.all_above = sum_a;
    s.all_eq = sum_e;
  }
  unsigned at = __shfl_sync(0xffffffffu, sum_a - a, warp), rank_e = __shfl_sync(0xffffffffu, sum_e - e, warp);      // before this warp
  cluster.sync();
  for (unsigned c = 0; c < rank; ++c) {
    at += *cluster.map_shared_rank(&s.all_above, c);
    rank_e += *cluster.map_shared_rank(&s.all_eq, c);
  }
  at += min(rank_e, need);
  for (int b = w0; b < w1; b += 32) {
    const int j = b + lane;
    const bool always = j < w1 && (j < lo || j >= hi), cand = picks && j < w1 && !always;
    const uint32_t u = cand ? key_at(j) : 0u;
    const bool eq = cand && u == prefix;
    const unsigned be = __ballot_sync(0xffffffffu, eq), below = (1u << lane) - 1;
    const bool take = always || (cand && u > prefix) || (eq && rank_e + __popc(be & below) < need);
    const unsigned bt = __ballot_sync(0xffffffffu, take);
    if (take) out[at + __popc(bt & below)] = j;
    at += __popc(bt);
    rank_e += __popc(be);
  }
  cluster.sync();                                                 // a CTA's shared memory lives until the others have read it
}

// A CTA or a cluster of them per row, key head and kind (keys or values; the weights go with the keys) closes the kept slots up in rounds: a round's lines
// go to shared memory, then (everybody has read that round) to their places.  One CTA keeps four rounds of 16 KB under way; a cluster, whose barriers cost 2
// us, takes rounds of 80 KB (one row of 8 heads cut from 40001 to 5000 tokens, selection and all, in rounds of 16 KB 43 us, 80 KB 39, 160 KB and half the
// CTAs per SM 46).  A slot never moves up and the kept ones ascend, so no later round reads a place that an earlier one wrote.  Where lines come from and
// go to is looked up for MOVE_LINES of them at once: a look at the list, then the table, then the line, round by round, made every round wait 5 us (16 rows
// of 8 heads cut from 4096 to 2048 tokens: 160 us, now 70).  Bound by HBM where rows and heads are many.
constexpr int MOVE_THREADS = 256, MOVE_STAGES = 4, MOVE_LINES = 2048, MOVE_MAX_CLUSTER = 8;
constexpr int MOVE_UNITS_ONE = 4, MOVE_UNITS_CLUSTER = 20;        // 16-byte pieces of a thread in a round
// shared memory of a CTA's share: the ring's stages that its rounds use, and the lists of its lines
__host__ __device__ inline int move_ring(int stages, int units, int rounds) { return min(stages, rounds) * units * MOVE_THREADS * 16; }
__host__ __device__ inline int move_lists(int rounds, int lines) { return min(MOVE_LINES, rounds * lines); }

template <int STAGES, int UNITS>
__global__ void __launch_bounds__(MOVE_THREADS)
paged_compact_kernel(uint4* kp, uint4* vp, float* mass, PageTable pt, const int32_t* lengths, const int32_t* kept, int G, int chunks, unsigned inv_chunks,
                     int keep) {
  extern __shared__ __align__(16) uint8_t smem[];
  uint4* ring = reinterpret_cast<uint4*>(smem);
  cg::cluster_group cluster = cg::this_cluster();
  const int S = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), tid = threadIdx.x;
  const int g = blockIdx.y >> 1, r = blockIdx.z;
  const bool values = blockIdx.y & 1;
  uint4* pages = values ? vp : kp;
  pdl_wait();
  int n = lengths[r];
  if (n > table_slots(pt) && blockIdx.y == 0 && rank == 0 && tid == 0) atomicAdd(&g_paged_fault, 1u);
  n = n > table_slots(pt) ? table_slots(pt) : n;
  const int32_t* list = kept + ((int64_t)r * G + g) * keep;
  if (n <= 1) return;                                             // nothing can move: the same for the whole cluster
  auto meet = [&]() {
    if (S > 1) cluster.sync();
    else __syncthreads();
  };
  auto place = [&](int j) -> int64_t {
    const int index = j / pt.page;
    const int64_t id = page_id(pt, r, index);
    return id < 0 ? -1 : (id * G + g) * pt.page + (j - index * pt.page);
  };
  // in round m this CTA takes the kept slots from (m S + rank) lines on
  const int lines = min(MOVE_THREADS * UNITS / chunks, MOVE_LINES), rounds = (keep + S * lines - 1) / (S * lines), ahead = MOVE_LINES / lines;
  const int listed = move_lists(rounds, lines);
  int64_t* from = reinterpret_cast<int64_t*>(smem + move_ring(STAGES, UNITS, rounds));
  int64_t* to = from + listed;
  for (int m0 = 0; m0 < rounds; m0 += ahead) {
    const int m1 = min(rounds, m0 + ahead);
    constexpr int EACH = MOVE_LINES / MOVE_THREADS;
    float weight[EACH];
    int64_t weight_to[EACH];
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const int q = k * MOVE_THREADS + tid, m = m0 + q / lines, i = (m * S + rank) * lines + q % lines;
      int64_t src = -1, dst = -1;
      if (m < m1 && i < keep) {
        const int j = list[i];
        if (j > i && j < n) {
          src = place(j), dst = place(i);
          if ((src < 0 || dst < 0) && !values) atomicAdd(&g_paged_fault, 1u);
        }
      }
      if (src < 0 || dst < 0) src = dst = -1;
      if (q < listed) {
        from[q] = src;
        to[q] = dst;
      }
      weight_to[k] = mass && !values ? dst : -1;
      weight[k] = weight_to[k] >= 0 ? mass[src] : 0.f;
    }
    meet();                                                       // everybody has read its weights
#pragma unroll
    for (int k = 0; k < EACH; ++k)
      if (weight_to[k] >= 0) mass[weight_to[k]] = weight[k];
    // a thread's units of a round: x = u MOVE_THREADS + tid of lines * chunks
    auto read = [&](int m) {
      if (m < m1) {
        uint4* at = ring + (m % STAGES) * UNITS * MOVE_THREADS;
#pragma unroll 4
        for (int u = 0; u < UNITS; ++u) {
          const int x = u * MOVE_THREADS + tid, line = chunks == 1 ? x : (int)__umulhi((unsigned)x, inv_chunks);
          if (line >= lines) break;
          const int64_t src = from[(m - m0) * lines + line];
          if (src >= 0) cp_async16((uint32_t)__cvta_generic_to_shared(at + x), pages + src * chunks + (x - line * chunks), true);
        }
      }
      cp_async_commit();
    };
    for (int m = m0; m < m0 + STAGES - 1; ++m) read(m);
    for (int m = m0; m < m1; ++m) {
      read(m + STAGES - 1);
      cp_async_wait<STAGES - 1>();
      meet();                                                     // everybody has read round m
      const uint4* at = ring + (m % STAGES) * UNITS * MOVE_THREADS;
#pragma unroll 4
      for (int u = 0; u < UNITS; ++u) {
        const int x = u * MOVE_THREADS + tid, line = chunks == 1 ? x : (int)__umulhi((unsigned)x, inv_chunks);
        if (line >= lines) break;
        const int64_t dst = to[(m - m0) * lines + line];
        if (dst >= 0) pages[dst * chunks + (x - line * chunks)] = at[x];
      }
    }
    meet();                                                       // the lists are written anew
  }
}

// grid (cluster, y, z) of clusters along x
template <typename... KArgs, typename... Args>
static cudaError_t launch_clusters(void (*kern)(KArgs...), int S, int y, int z, int threads, size_t smem, cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)S, (unsigned)y, (unsigned)z);
  cfg.blockDim = threads;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)S;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}
// CTAs of a cluster: as many as still find an SM each, at most `most`
static int cluster_of(int64_t clusters, int most, int per_sm) {
  int S = 1;
  while (S < most && clusters * S * 2 <= (int64_t)sm_count() * per_sm) S *= 2;
  return S;
}

// ------------------------------------------------------------------------------------------------ dense view
// A CTA copies GATHER_BYTES' worth of slots of one key head's keys and values, whatever the pages: a thread asks for four pieces of either before it
// stores the first: 12.7 us for 7777 tokens of 8 heads, 64 MB moved.  (A CTA per page and one piece at a time: 18.4.)
constexpr int GATHER_THREADS = 256, GATHER_AHEAD = 4;

__global__ void __launch_bounds__(GATHER_THREADS)
paged_gather_kernel(const uint4* kp, const uint4* vp, PageTable pt, const int32_t* rows, const int32_t* lengths, uint4* kc, uint4* vc, int extra, int G,
                    int chunks, unsigned inv_chunks, int slots, int64_t Tcap) {
  const int g = blockIdx.y, i = blockIdx.z;
  pdl_wait();
  const int r = rows[i];
  if (r < 0) return;
  if (r >= pt.rows) {
    if (threadIdx.x == 0 && blockIdx.x == 0 && g == 0) atomicAdd(&g_paged_fault, 1u);
    return;
  }
  if (lengths[r] > table_slots(pt) && threadIdx.x == 0 && blockIdx.x == 0 && g == 0) atomicAdd(&g_paged_fault, 1u);
  int64_t n = (int64_t)lengths[r] + extra;
  if (n > table_slots(pt)) n = table_slots(pt);
  if (n > Tcap) n = Tcap;
  const int j0 = blockIdx.x * slots;
  if (j0 >= n) return;
  const int count = (int)(n - j0 < slots ? n - j0 : slots) * chunks;
  const int64_t dst = (((int64_t)i * G + g) * Tcap + j0) * chunks;
  bool missing = false;
  for (int x0 = threadIdx.x; x0 < count; x0 += GATHER_AHEAD * GATHER_THREADS) {
    uint4 a[GATHER_AHEAD], b[GATHER_AHEAD];
    bool here[GATHER_AHEAD];
#pragma unroll
    for (int u = 0; u < GATHER_AHEAD; ++u) {
      const int x = x0 + u * GATHER_THREADS;
      here[u] = false;
      if (x < count) {
        const int line = chunks == 1 ? x : (int)__umulhi((unsigned)x, inv_chunks), j = j0 + line, index = j / pt.page;      // (x / chunks: x is at most 1024)
        const int64_t id = page_id(pt, r, index);
        here[u] = id >= 0;
        missing |= id < 0;
        const int64_t src = ((id < 0 ? 0 : id * G + g) * pt.page + (j - index * pt.page)) * chunks + (x - line * chunks);
        if (id >= 0) {
          a[u] = ldg_stream(kp + src);
          b[u] = ldg_stream(vp + src);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < GATHER_AHEAD; ++u)
      if (here[u]) {
        kc[dst + x0 + u * GATHER_THREADS] = a[u];
        vc[dst + x0 + u * GATHER_THREADS] = b[u];
      }
  }
  if (missing) atomicAdd(&g_paged_fault, 1u);
}

// ------------------------------------------------------------------------------------------------ counters
__global__ void paged_advance_kernel(int32_t* lengths, int32_t* positions, const int32_t* rows, int64_t count, int32_t delta) {
  pdl_wait();
  const int64_t r = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= count || rows[r] < 0) return;
  lengths[r] += delta;
  positions[r] += delta;
}

}  // namespace b200p

using namespace b200p;

extern "C" int b200p_paged_append(void* qkv, int64_t ldq, void* q_out, void* kpages, void* vpages, float* mass, const int32_t* table,
                                  const int32_t* t_row, const int32_t* t_slot, const int32_t* t_pos, const void* q_norm_w, const void* k_norm_w,
                                  const float* rates, int n_rot, int pairs, float eps, int64_t M, int H, int G, int D, int64_t P, int page, int rows,
                                  int width, int dtype, int qkv_f32, void* stream) {
  PdlClass pdl_cls(4);
  const PageTable pt{table, P, rows, width, page};
  const int rc = check_pages(kpages, vpages, pt, G, D, dtype);
  if (rc) return rc;
  B200P_REQUIRE(M == 0 || (qkv && q_out && t_row && t_slot && t_pos), B200P_ERR_ARG, "null pointer");
  B200P_REQUIRE(!qkv_f32 || dtype != B200P_F32, B200P_ERR_ARG, "qkv_f32 is the accumulation-buffer input of 16-bit models");
  B200P_REQUIRE(H > 0 && H % G == 0 && H + 2 * G < 65536, B200P_ERR_ARG, "bad head counts %d/%d", H, G);
  B200P_REQUIRE(n_rot >= 0 && 2 * n_rot <= D && (n_rot == 0 || rates), B200P_ERR_ARG, "%d rotated pairs of %d dimensions", n_rot, D);
  B200P_REQUIRE(pairs == 0 || pairs == 1, B200P_ERR_ARG, "pairs is 0 (halves) or 1 (neighbours)");
  B200P_REQUIRE(M >= 0 && M < (1ll << 31) && ldq >= (int64_t)(H + 2 * G) * D, B200P_ERR_ARG, "bad shape: %lld tokens, rows of %lld", (long long)M,
                (long long)ldq);
  if (M == 0) return B200P_OK;
  const cudaStream_t st = (cudaStream_t)stream;
  const size_t in = qkv_f32 || dtype == B200P_F32 ? 4 : 2;
  if ((pairs || n_rot % 8 == 0) && aligned(qkv, 16) && ldq * in % 16 == 0 && aligned(q_out, 16) && aligned(q_norm_w, 16) && aligned(k_norm_w, 16)) {
    int width_log2 = 0, lg = 3;
    while ((8 << width_log2) < D) ++width_log2;
    const int walkers = 256 >> width_log2, sms = sm_count();
    while (lg > 0 && ((M >> lg) < 4 * sms || (1 << lg) > walkers)) --lg;
    // two CTAs per SM at least, by sharing a token's heads
    int64_t split = 2 * sms / M, most = (H + 2 * G + walkers - 1) / walkers;
    if (split < 1 || lg > 0) split = 1;
    const dim3 grid((unsigned)((M + (1 << lg) - 1) >> lg), (unsigned)(split < most ? split : most));
    auto go = [&](auto t, auto in) {
      using T = decltype(t);
      using TIN = decltype(in);
      auto pick = [&](auto pairs) {
        constexpr bool PAIRS = decltype(pairs)::value;
        return q_norm_w || k_norm_w ? paged_append_rows_kernel<T, TIN, 2, PAIRS, true>
               : lg > 0             ? paged_append_rows_kernel<T, TIN, 4, PAIRS, false>
                                    : paged_append_rows_kernel<T, TIN, 2, PAIRS, false>;
      };
      auto kern = pairs ? pick(std::true_type()) : pick(std::false_type());
      launch_pdl(kern, grid, 256, 0, st, (TIN*)qkv, ldq, (T*)q_out, (T*)kpages, (T*)vpages, mass, pt, t_row, t_slot, t_pos, (const T*)q_norm_w,
                 (const T*)k_norm_w, rates, n_rot, eps, (int)M, H, G, D, width_log2, lg);
    };
    if (qkv_f32) {
      B200P_DISPATCH_DTYPE(dtype, T, (go(T(), float())));
    } else {
      B200P_DISPATCH_DTYPE(dtype, T, (go(T(), T())));
    }
    B200P_LAUNCH_CHECK("paged_append_rows_kernel");
    return B200P_OK;
  }
  if (qkv_f32) {
    B200P_DISPATCH_DTYPE(dtype, T, (paged_append_kernel<T, float><<<(unsigned)M, 256, 0, st>>>((float*)qkv, ldq, (T*)q_out, (T*)kpages, (T*)vpages, mass, pt,
                                       t_row, t_slot, t_pos, (const T*)q_norm_w, (const T*)k_norm_w, rates, n_rot, pairs, eps, H, G, D)));
  } else {
    B200P_DISPATCH_DTYPE(dtype, T, (paged_append_kernel<T, T><<<(unsigned)M, 256, 0, st>>>((T*)qkv, ldq, (T*)q_out, (T*)kpages, (T*)vpages, mass, pt,
                                       t_row, t_slot, t_pos, (const T*)q_norm_w, (const T*)k_norm_w, rates, n_rot, pairs, eps, H, G, D)));
  }
  B200P_LAUNCH_CHECK("paged_append_kernel");
  return B200P_OK;
}

extern "C" int b200p_paged_select(const float* mass, const int32_t* table, const int32_t* lengths, int32_t* kept, int64_t P, int G, int page, int rows,
                                  int width, int keep, int first, int recent, void* stream) {
  const PageTable pt{table, P, rows, width, page};
  const int rc = check_pages(mass, mass, pt, G, 8, B200P_F32);
  if (rc) return rc;
  B200P_REQUIRE(lengths && kept, B200P_ERR_ARG, "null pointer");
  B200P_REQUIRE(keep > 0 && first >= 0 && recent >= 0 && (int64_t)first + recent <= keep, B200P_ERR_ARG, "%d first and %d recent of %d kept tokens", first,
                recent, keep);
  B200P_REQUIRE(keep <= 1 << 30, B200P_ERR_ARG, "%d kept tokens: a row has at most 2^30", keep);
  B200P_REQUIRE(rows < 65536, B200P_ERR_ARG, "too many rows");
  B200P_REQUIRE(G < 32768, B200P_ERR_ARG, "too many key heads");
  constexpr int SEL_ROOM = 48 * 1024;                             // keys: 192 KB
  auto large = paged_select_kernel<1024>;
  auto small = paged_select_kernel<256>;
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev > 63 || !(ready.load(std::memory_order_relaxed) >> dev & 1))) {
    e = cudaFuncSetAttribute(large, cudaFuncAttributeMaxDynamicSharedMemorySize, SEL_ROOM * 4);
    if (e == cudaSuccess && dev < 64) ready.fetch_or(1ull << dev);
  }
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(paged_select_kernel)");
  const int64_t slots = (int64_t)width * page;
  // more CTAs for a row where SMs are free and a CTA's passes are long (4096 slots: 4 per thread)
  int S = cluster_of((int64_t)G * rows, SEL_MAX_CLUSTER, 1);
  while (S > 1 && slots / S < 2048) S /= 2;
  int64_t room = ((slots + S - 1) / S + 31) / 32 * 32;
  if (room > SEL_ROOM) room = 0;                                  // (a shorter row of such a table is read three times all the same)
  // short rows in numbers: a CTA of 256 threads has less to set up, and more of them fit an SM
  const bool many = slots <= 4096 && (int64_t)G * rows > 2 * sm_count();
  e = launch_clusters(many ? small : large, S, G, rows, many ? 256 : 1024, (size_t)room * 4, (cudaStream_t)stream, mass, pt, lengths, kept, G, keep, first,
                      recent, (int)room);
  if (e != cudaSuccess) return cuda_fail(e, "paged_select_kernel");
  B200P_LAUNCH_CHECK("paged_select_kernel");
  return B200P_OK;
}

extern "C" int b200p_paged_compact(void* kpages, void* vpages, float* mass, const int32_t* table, const int32_t* lengths, const int32_t* kept, int64_t P,
                                   int G, int D, int page, int rows, int width, int keep, int dtype, void* stream) {
  const PageTable pt{table, P, rows, width, page};
  const int rc = check_pages(kpages, vpages, pt, G, D, dtype);
  if (rc) return rc;
  B200P_REQUIRE(lengths && kept && keep > 0, B200P_ERR_ARG, "null pointer or nothing to keep");
  B200P_REQUIRE(keep <= 1 << 30, B200P_ERR_ARG, "%d kept tokens: a row has at most 2^30", keep);
  B200P_REQUIRE(rows < 65536, B200P_ERR_ARG, "too many rows");
  const int chunks = D * (dtype == B200P_F32 ? 4 : 2) / 16;
  B200P_REQUIRE(G < 32768, B200P_ERR_ARG, "too many key heads");
  auto one = paged_compact_kernel<MOVE_STAGES, MOVE_UNITS_ONE>;
  auto many = paged_compact_kernel<1, MOVE_UNITS_CLUSTER>;
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev > 63 || !(ready.load(std::memory_order_relaxed) >> dev & 1))) {
    e = cudaFuncSetAttribute(one, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             move_ring(MOVE_STAGES, MOVE_UNITS_ONE, MOVE_STAGES) + MOVE_LINES * 16);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(many, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                       move_ring(1, MOVE_UNITS_CLUSTER, 1) + MOVE_LINES * 16);
    if (e == cudaSuccess && dev < 64) ready.fetch_or(1ull << dev);
  }
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(paged_compact_kernel)");
  int S = cluster_of((int64_t)2 * G * rows, MOVE_MAX_CLUSTER, 2);
  while (S > 1 && (int64_t)keep * chunks <= S * 1024) S /= 2;               // (at least 16 KB of lines each)
  const unsigned inv = (unsigned)(((1ull << 32) + chunks - 1) / chunks);
  const int stages = S > 1 ? 1 : MOVE_STAGES, units = S > 1 ? MOVE_UNITS_CLUSTER : MOVE_UNITS_ONE, lines = min(MOVE_THREADS * units / chunks, MOVE_LINES);
  const int rounds = (int)(((int64_t)keep + S * lines - 1) / (S * lines)), smem = move_ring(stages, units, rounds) + move_lists(rounds, lines) * 16;
  e = launch_clusters(S > 1 ? many : one, S, 2 * G, rows, MOVE_THREADS, smem, (cudaStream_t)stream, (uint4*)kpages, (uint4*)vpages, mass, pt,
                      lengths, kept, G, chunks, inv, keep);
  if (e != cudaSuccess) return cuda_fail(e, "paged_compact_kernel");
  B200P_LAUNCH_CHECK("paged_compact_kernel");
  return B200P_OK;
}

extern "C" int b200p_paged_gather(const void* kpages, const void* vpages, const int32_t* table, const int32_t* row_of, const int32_t* lengths, void* kcache,
                                  void* vcache, int extra, int64_t count, int G, int D, int64_t P, int page, int rows, int width, int64_t Tcap, int dtype,
                                  void* stream) {
  const PageTable pt{table, P, rows, width, page};
  const int rc = check_pages(kpages, vpages, pt, G, D, dtype);
  if (rc) return rc;
  B200P_REQUIRE(count == 0 || (row_of && lengths && kcache && vcache), B200P_ERR_ARG, "null pointer");
  B200P_REQUIRE(count >= 0 && count < 65536 && Tcap > 0, B200P_ERR_ARG, "bad shape: %lld rows of %lld", (long long)count, (long long)Tcap);
  B200P_REQUIRE(aligned(kcache, 16) && aligned(vcache, 16), B200P_ERR_ALIGN, "caches must be 16-byte aligned");
  if (count == 0) return B200P_OK;
  const int chunks = D * (dtype == B200P_F32 ? 4 : 2) / 16;
  const int64_t longest = Tcap < (int64_t)width * page ? Tcap : (int64_t)width * page;
  // 16 KB of keys and of values per CTA, 4 where that leaves SMs without one
  int slots = 16384 / (16 * chunks);
  while (slots > 64 / chunks + 1 && (longest + slots - 1) / slots * G * count < 2 * sm_count()) slots = (slots + 1) / 2;
  const unsigned inv = (unsigned)(((1ull << 32) + chunks - 1) / chunks);
  PdlClass pdl_cls(32);
  launch_pdl(paged_gather_kernel, dim3((unsigned)((longest + slots - 1) / slots), (unsigned)G, (unsigned)count), GATHER_THREADS, 0, (cudaStream_t)stream,
             (const uint4*)kpages, (const uint4*)vpages, pt, row_of, lengths, (uint4*)kcache, (uint4*)vcache, extra, G, chunks, inv, slots, Tcap);
  B200P_LAUNCH_CHECK("paged_gather_kernel");
  return B200P_OK;
}

extern "C" int b200p_paged_advance(int32_t* lengths, int32_t* positions, const int32_t* rows, int64_t count, int32_t delta, void* stream) {
  PdlClass pdl_cls(32);
  B200P_REQUIRE(lengths && positions && rows, B200P_ERR_ARG, "null pointer");
  B200P_REQUIRE(count >= 0 && count < (1ll << 31), B200P_ERR_ARG, "bad number of rows %lld", (long long)count);
  if (count == 0) return B200P_OK;
  launch_pdl(paged_advance_kernel, (unsigned)((count + 255) / 256), 256, 0, (cudaStream_t)stream, lengths, positions, rows, count, delta);
  B200P_LAUNCH_CHECK("paged_advance_kernel");
  return B200P_OK;
}

extern "C" int b200p_paged_fault_count(unsigned int* count, int reset, void* stream) {
  B200P_REQUIRE(count, B200P_ERR_ARG, "null pointer");
  const cudaStream_t st = (cudaStream_t)stream;
  unsigned int a = 0, b = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&a, g_paged_fault, sizeof(a), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return cuda_fail(e, "b200p_paged_fault_count");
  const int rc = paged_attn_faults(&b, reset, st);
  if (rc) return rc;
  if (reset) {
    const unsigned int zero = 0;
    e = cudaMemcpyToSymbolAsync(g_paged_fault, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e != cudaSuccess) return cuda_fail(e, "b200p_paged_fault_count(reset)");
  }
  *count = a + b;
  return B200P_OK;
}
