// Log probabilities of given tokens, the entropy of every row and its most likely tokens, from logits (b200p_token_logprobs).
//
//   p_i = exp(x_i / T) / sum_j exp(x_j / T);   log p_t,   H = -sum_i p_i log p_i,   the largest x_i, lowest index first among equals
//
// One pass over a row: with m the largest value so far, u_i = x_i - m and e_i = exp(u_i / T), every thread keeps s = sum e_i and
// t = sum e_i u_i, which become f s and f (t + d s) when m grows by -d and f = exp(d / T).  Then log p_i = (x_i - m) / T - log s and
// H = log s - t / (T s).  All of it is fp32; nothing of the row is written.
//
// The alternatives come out of the same pass: the k-th largest of the maxima of 64 groups of threads is no larger than the row's k-th largest
// value, and only few values are as large (some 24 for k = 20).  A thread whose maximum reaches it has its values read again, a lane per vector; what reaches
// the bound goes into a list, which is ranked by counting.  Rows in which too many do (equal values) are selected from digit by digit.
//
// A row is split over the CTAs of a cluster where the rows are few, as in sampler.cu.
#include <cooperative_groups.h>
#include <float.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace b200p {

int sm_count();

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32;
constexpr int LP_TOP = 32;             // alternatives at most: half of the groups, so that their k-th largest maximum is a bound
constexpr int LP_CLUSTER = 8;
constexpr int LP_GROUPS = 64;
static_assert(LP_WARPS * LP_CLUSTER == LP_GROUPS, "a warp is a group in the largest cluster");
constexpr int LP_LIST = 1024;          // values that reach the bound; more are selected from digit by digit

__device__ __forceinline__ float lp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// the larger one, NaN if either is: u of a logit that is not a number stays that and reaches the sums
__device__ __forceinline__ float lp_max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// Differences are held above -1e30, so that a weight of 0 times the difference of a logit of minus infinity is 0.  (It is 0 as long as 1e30 / T is more than
// the 88 behind which 2^x ends: temperatures up to 1e27.)
__device__ __forceinline__ float lp_diff(float x, float m) { return lp_max_nan(x - m, -1e30f); }

// an order of all floats as unsigned numbers: -0 like 0, NaN like minus infinity
__device__ __forceinline__ uint32_t lp_key(float x) {
  if (!(x > -INFINITY)) return 0x007fffffu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float lp_value(uint32_t key) { return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu)); }

struct LogProbs {
  const void* logits;
  const int32_t* tokens;
  float *logprob, *entropy, *top_logprobs;
  int32_t* top_ids;
  int64_t ld;
  int V, top;
  float inv_t, c;                      // 1 / T, log2(e) / T
};

// A row as 16-byte vectors, and the loose elements before and behind them.
template <typename T>
struct RowParts {
  static constexpr int E = 16 / (int)sizeof(T);
  const T* row;
  int head, vectors, tail, loose;
  __device__ RowParts(const T* r, int V) : row(r) {
    const int off = (int)((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
    head = min(V, off ? E - off : 0);
    vectors = (V - head) / E;
    tail = head + vectors * E;
    loose = head + V - tail;
  }
  __device__ __forceinline__ uint4 load(int v) const { return *(reinterpret_cast<const uint4*>(row + head) + v); }
  __device__ __forceinline__ int index(int v) const { return head + v * E; }
  __device__ __forceinline__ int loose_index(int i) const { return i < head ? i : tail + i - head; }
};

template <typename T> __device__ __forceinline__ uint4 lp_nothing();
template <> __device__ __forceinline__ uint4 lp_nothing<float>() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
template <> __device__ __forceinline__ uint4 lp_nothing<__half>() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }
template <> __device__ __forceinline__ uint4 lp_nothing<__nv_bfloat16>() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }

// Two values at a time where an instruction takes two.
struct LpPair {
  float2 s, t;
  __device__ LpPair() : s(make_float2(0.f, 0.f)), t(s) {}
  __device__ __forceinline__ void add(float x, float y, float m, float c) {
    float2 u = __fadd2_rn(make_float2(x, y), make_float2(-m, -m));
    u.x = lp_max_nan(u.x, -1e30f), u.y = lp_max_nan(u.y, -1e30f);
    const float2 d = __fmul2_rn(u, make_float2(c, c)), e = make_float2(lp_exp2(d.x), lp_exp2(d.y));
    s = __fadd2_rn(s, e);
    t = __ffma2_rn(e, u, t);
  }
};

struct LpSums {
  float m, s, t;
  // (m starts at the lowest number, not at minus infinity: a difference to it is a number or minus infinity)
  __device__ LpSums() : m(-FLT_MAX), s(0.f), t(0.f) {}
  __device__ __forceinline__ void raise(float to, float c) {
    const float d = lp_diff(m, to), f = lp_exp2(d * c);
    t = f * fmaf(d, s, t);
    s *= f;
    m = to;
  }
  __device__ __forceinline__ void add(float x, float c) {
    const float u = lp_diff(x, m), e = lp_exp2(u * c);
    s += e;
    t = fmaf(e, u, t);
  }
};

struct LpShared {
  float4 part[LP_WARPS], cta[LP_CLUSTER];      // m, s, t of the warps, and (in the first CTA) of the cluster's CTAs
  alignas(16) float group[LP_GROUPS];
  float bound, m, log_s;
  int count;
  uint2 list[LP_LIST];                 // key and index
  int hist[256], warp_count[LP_WARPS];
  uint32_t prefix;
  int need;
};

template <typename T, typename F>
__device__ __forceinline__ void lp_visit(const RowParts<T>& p, F&& f) {
  for (int v = threadIdx.x; v < p.vectors; v += LP_THREADS) {
    const uint4 x = p.load(v);
    const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
    for (int i = 0; i < RowParts<T>::E; ++i) f(Tr<T>::to_f(e[i]), p.index(v) + i);
  }
  if ((int)threadIdx.x < p.loose) f(Tr<T>::to_f(p.row[p.loose_index(threadIdx.x)]), p.loose_index(threadIdx.x));
}

// The k-th largest key of the row, and of the values that have it how many belong to the k (in s.prefix, s.need).  Seldom run: kept small.
template <typename T>
__device__ __noinline__ void lp_select(const RowParts<T>& p, LpShared& s, int k) {
  if (threadIdx.x == 0) s.prefix = 0u, s.need = k;
#pragma unroll 1
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += LP_THREADS) s.hist[i] = 0;
    __syncthreads();
    const uint32_t prefix = s.prefix;
    auto count = [&](float x, bool here) {                          // by whole warps
      const uint32_t key = lp_key(x);
      const bool in = here && (shift == 24 || key >> (shift + 8) == prefix);
      const unsigned digit = key >> shift & 255u;
      int same;
      __match_all_sync(~0u, in ? digit : 256u, &same);              // (rows that get here are full of equal values)
      if (in && (!same || (threadIdx.x & 31) == 0)) atomicAdd(&s.hist[digit], same ? 32 : 1);
    };
    for (int base = 0; base < p.vectors; base += LP_THREADS) {
      const int v = base + (int)threadIdx.x;
      const uint4 raw = v < p.vectors ? p.load(v) : lp_nothing<T>();
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < RowParts<T>::E; ++i) count(Tr<T>::to_f(e[i]), v < p.vectors);
    }
    const bool loose = (int)threadIdx.x < p.loose;
    count(loose ? Tr<T>::to_f(p.row[p.loose_index(threadIdx.x)]) : 0.f, loose);
    __syncthreads();
    if (threadIdx.x < 32) {                                         // a lane has 8 digits, the first lane the largest
      const int top = 255 - 8 * (int)threadIdx.x, need = s.need;
      int sum = 0;
      for (int i = 0; i < 8; ++i) sum += s.hist[top - i];
      int before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(~0u, before, o);
        if ((int)threadIdx.x >= o) before += x;
      }
      before -= sum;
      if (before < need && need <= before + sum) {
        int d = top;
        while (before + s.hist[d] < need) before += s.hist[d--];
        s.prefix = prefix << 8 | (uint32_t)d;
        s.need = need - before;
      }
    }
    __syncthreads();
  }
}

// The first `need` elements whose key is `key`, in the row's order, behind the `have` first ones of the list.
template <typename T>
__device__ __noinline__ void lp_first_equal(const RowParts<T>& p, LpShared& s, int V, uint32_t key, int have, int need) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll 1
  for (int base = 0; need > 0 && base < V; base += LP_THREADS) {
    const int i = base + (int)threadIdx.x;
    const bool eq = i < V && lp_key(Tr<T>::to_f(p.row[i])) == key;
    const unsigned found = __ballot_sync(~0u, eq);
    if (lane == 0) s.warp_count[warp] = __popc(found);
    __syncthreads();
    int at = __popc(found & ((1u << lane) - 1u)), all = 0;
#pragma unroll
    for (int w = 0; w < LP_WARPS; ++w) {
      if (w < warp) at += s.warp_count[w];
      all += s.warp_count[w];
    }
    if (eq && at < need) s.list[have + at] = make_uint2(key, (uint32_t)i);
    have += min(all, need);
    need -= all;
    __syncthreads();
  }
}

// grid (S * rows), clusters of S: as many CTAs to a row as fit the GPU side by side, four per SM, with two vectors or more for a thread (us, device: 1 row of
// 128256 in 1 / 2 / 4 / 8 CTAs, 20 alternatives 20.6 / 13.2 / 8.4 / 6.7; 64 rows of 32000 bf16 without 4.9 / 4.0 / 3.8 / 5.2; 333 rows of 50257 bf16
// 13.4 / 14.2 / 15.8 / 20.3).  Four CTAs of 256 threads and not two of 512: 333 rows with 8 alternatives 22.0 -> 17.1 (16.6 with values in pairs), 1500 rows
// of 151936 144.6 -> 139.9, 99 % of the copy's bandwidth.  (Eight vectors of a thread under way through shared memory instead of four through registers gave nothing.)
template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_THREADS, 4)
token_logprobs_kernel(const __grid_constant__ LogProbs a) {
  __shared__ LpShared s;
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned rank = cluster.block_rank(), S = cluster.num_blocks();
  const int64_t r = blockIdx.x / S;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int E = RowParts<T>::E, AHEAD = 4;
  if (S > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");     // this CTA runs: the others may write into it
  pdl_wait();
  const RowParts<T> p(reinterpret_cast<const T*>(a.logits) + r * a.ld, a.V);
  const int per = (p.vectors + (int)S - 1) / (int)S, v0 = min(p.vectors, (int)rank * per), v1 = min(p.vectors, v0 + per);
  const float c = a.c;
  int token = -1;
  float given = 0.f;
  if (rank == 0 && threadIdx.x == 0 && a.tokens) {
    token = a.tokens[r];
    if (token >= 0 && token < a.V) given = Tr<T>::to_f(p.row[token]);
  }

  LpSums sum;
#pragma unroll 1
  for (int v = v0 + (int)threadIdx.x; v < v1; v += AHEAD * LP_THREADS) {
    uint4 raw[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) raw[k] = k == 0 || v + k * LP_THREADS < v1 ? p.load(v + k * LP_THREADS) : lp_nothing<T>();
    float top = -FLT_MAX;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const T* e = reinterpret_cast<const T*>(&raw[k]);
#pragma unroll
      for (int i = 0; i < E; ++i) top = fmaxf(top, Tr<T>::to_f(e[i]));       // (drops NaN)
    }
    if (top > sum.m) sum.raise(top, c);
    LpPair pair;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const T* e = reinterpret_cast<const T*>(&raw[k]);
#pragma unroll
      for (int i = 0; i < E; i += 2) pair.add(Tr<T>::to_f(e[i]), Tr<T>::to_f(e[i + 1]), sum.m, c);
    }
    sum.s += pair.s.x + pair.s.y;
    sum.t += pair.t.x + pair.t.y;
  }
  if (rank == 0 && (int)threadIdx.x < p.loose) {
    const float x = Tr<T>::to_f(p.row[p.loose_index(threadIdx.x)]);
    if (x > sum.m) sum.raise(x, c);
    sum.add(x, c);
  }

  // ---- the threads' maxima and sums become the row's ------------------------------------------------------------------------
  const float mine = sum.m;
  float high = mine;
  const int lanes = 32 / LP_CLUSTER * (int)S;                       // of a group
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    if (TOP && o == lanes && (lane & (lanes - 1)) == 0) s.group[rank * (LP_THREADS / lanes) + threadIdx.x / lanes] = high;
    high = fmaxf(high, __shfl_xor_sync(~0u, high, o));
  }
  if (TOP && lanes == 32 && lane == 0) s.group[rank * LP_WARPS + warp] = high;
  sum.raise(high, c);
  sum.s = warp_sum(sum.s), sum.t = warp_sum(sum.t);
  if (lane == 0) s.part[warp] = make_float4(sum.m, sum.s, sum.t, 0.f);
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();
  if (S > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  auto merge = [&](const float4* from, int n) {                     // by one warp
    LpSums q;
    if (lane < n) q.m = from[lane].x, q.s = from[lane].y, q.t = from[lane].z;
    q.raise(warp_max(q.m), c);
    q.s = warp_sum(q.s), q.t = warp_sum(q.t);
    return q;
  };
  if (warp == 0) {
    const LpSums q = merge(s.part, LP_WARPS);
    if (lane == 0) *cluster.map_shared_rank(&s.cta[rank], 0) = make_float4(q.m, q.s, q.t, 0.f);
  }
  const int groups = LP_THREADS / lanes;
  if (TOP && S > 1) {
    for (int i = threadIdx.x; i < groups * (int)S; i += LP_THREADS) {
      const int g = rank * groups + i % groups, to = i / groups;
      if (to != (int)rank) *cluster.map_shared_rank(&s.group[g], to) = s.group[g];
    }
  }
  if (S > 1) cluster.sync();
  else __syncthreads();
  if (rank == 0 && warp == 0) {
    const LpSums q = merge(s.cta, (int)S);
    if (lane == 0) {
      const float log_s = logf(q.s);
      s.m = q.m, s.log_s = log_s;
      if (a.logprob) a.logprob[r] = token < 0 ? 0.f : token < a.V ? (given - q.m) * a.inv_t - log_s : __int_as_float(0x7fc00000);
      if (a.entropy) a.entropy[r] = log_s - q.t * a.inv_t / q.s;
    }
  }
  if (!TOP) return;

  // ---- the bound, and what reaches it ----------------------------------------------------------------------------------------
  if (threadIdx.x < LP_GROUPS) {
    const float x = s.group[threadIdx.x];
    int above = 0;
#pragma unroll
    for (int j = 0; j < LP_GROUPS; j += 4) {
      const float4 y = *reinterpret_cast<const float4*>(s.group + j);
      above += (y.x > x || (y.x == x && j < (int)threadIdx.x)) + (y.y > x || (y.y == x && j + 1 < (int)threadIdx.x)) +
               (y.z > x || (y.z == x && j + 2 < (int)threadIdx.x)) + (y.w > x || (y.w == x && j + 3 < (int)threadIdx.x));
    }
    if (above == a.top - 1) s.bound = x;
  }
  __syncthreads();
  const float bound = s.bound;
  int* count = cluster.map_shared_rank(&s.count, 0);
  uint2* list = cluster.map_shared_rank(s.list, 0);
  auto push = [&](float x, int i) {
    if (x >= bound) {
      const int at = atomicAdd(count, 1);
      if (at < LP_LIST) list[at] = make_uint2(lp_key(x), (uint32_t)i);
    }
  };
  for (unsigned left = __ballot_sync(~0u, mine >= bound); left; left &= left - 1) {
    const int thread = warp * 32 + __ffs(left) - 1;
    for (int v = v0 + thread + lane * LP_THREADS; v < v1; v += 32 * LP_THREADS) {
      const uint4 raw = p.load(v);
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < E; ++i) push(Tr<T>::to_f(e[i]), p.index(v) + i);
    }
    if (rank == 0 && lane == 0 && thread < p.loose) push(Tr<T>::to_f(p.row[p.loose_index(thread)]), p.loose_index(thread));
  }
  if (S > 1) cluster.sync();                                        // (nobody looks into another CTA behind this)
  else __syncthreads();
  if (rank != 0) return;
  int have = s.count;
  if (have > LP_LIST) {
    lp_select(p, s, a.top);
    const uint32_t key = s.prefix;
    const int need = s.need;
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
    lp_visit(p, [&](float x, int i) {
      const uint32_t k = lp_key(x);
      if (k > key) s.list[atomicAdd(&s.count, 1)] = make_uint2(k, (uint32_t)i);
    });
    __syncthreads();
    lp_first_equal(p, s, a.V, key, a.top - need, need);
    have = a.top;
  } else if (have < a.top) {                                        // all that is more than minus infinity is in the list
    lp_first_equal(p, s, a.V, lp_key(-INFINITY), have, a.top - have);
    have = a.top;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < have; i += LP_THREADS) {
    const uint2 x = s.list[i];
    int above = 0;
    for (int j = 0; j < have; ++j) {
      const uint2 y = s.list[j];
      above += y.x > x.x || (y.x == x.x && y.y < x.y);
    }
    if (above < a.top) {
      a.top_ids[r * a.top + above] = (int32_t)x.y;
      a.top_logprobs[r * a.top + above] = (lp_value(x.x) - s.m) * a.inv_t - s.log_s;
    }
  }
}

template <typename T>
static int launch_logprobs(const LogProbs& a, int64_t M, cudaStream_t st) {
  int S = LP_CLUSTER;
  const int64_t vectors = a.V / RowParts<T>::E;
  while (S > 1 && (M * S > 4 * sm_count() || vectors < 2 * S * LP_THREADS)) S >>= 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(M * S));
  cfg.blockDim = dim3(LP_THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)S;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, a.top ? token_logprobs_kernel<T, true> : token_logprobs_kernel<T, false>, a);
  return e == cudaSuccess ? B200P_OK : cuda_fail(e, "token_logprobs_kernel");
}

}  // namespace b200p

using namespace b200p;

extern "C" int b200p_token_logprobs(const void* logits, const int32_t* tokens, float* logprob, float* entropy, int32_t* top_ids, float* top_logprobs,
                                    int64_t M, int64_t V, int64_t ldl, int top, float temperature, int dtype, void* stream) {
  PdlClass pdl_cls(32);
  B200P_REQUIRE(M >= 0 && M < (1ll << 27) && V > 0 && V < (1ll << 30) && ldl >= V, B200P_ERR_ARG, "bad shape: %lld rows of %lld logits, stride %lld",
                (long long)M, (long long)V, (long long)ldl);
  B200P_REQUIRE(top >= 0 && top <= LP_TOP && top <= V, B200P_ERR_ARG, "%d alternatives of %lld: at most %d", top, (long long)V, LP_TOP);
  B200P_REQUIRE(temperature >= 1e-30f && temperature <= 1e27f, B200P_ERR_ARG, "temperature must be between 1e-30 and 1e27");
  B200P_REQUIRE(dtype == B200P_F32 || dtype == B200P_F16 || dtype == B200P_BF16, B200P_ERR_ARG, "bad dtype %d", dtype);
  if (M == 0) return B200P_OK;
  B200P_REQUIRE(logits && (!logprob || tokens) && (!top || (top_ids && top_logprobs)), B200P_ERR_ARG, "null pointer");
  B200P_REQUIRE(aligned(logits, dtype == B200P_F32 ? 4 : 2), B200P_ERR_ALIGN, "logits are aligned to their type");
  LogProbs a{};
  a.logits = logits, a.tokens = logprob ? tokens : nullptr, a.logprob = logprob, a.entropy = entropy, a.top_ids = top_ids, a.top_logprobs = top_logprobs;
  a.ld = ldl, a.V = (int)V, a.top = top, a.inv_t = 1.f / temperature, a.c = 1.4426950408889634f / temperature;
  B200P_DISPATCH_DTYPE(dtype, T, return (launch_logprobs<T>(a, M, (cudaStream_t)stream)));
  return B200P_OK;
}
