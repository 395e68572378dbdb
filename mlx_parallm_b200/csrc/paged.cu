// Paged key-value cache: append (norms, rotation, write), eviction by received attention weight (selection, closing up), dense view.
#include <stdlib.h>

#include "paged.cuh"

namespace b200p {

int sm_count();

// Calls of the append and the eviction that met an id that names no page where they needed one (b200p_paged_fault_count).
__device__ unsigned int g_paged_fault = 0;

int paged_attn_faults(unsigned int* count, int reset, cudaStream_t st);

// ------------------------------------------------------------------------------------------------ append
// One CTA per token.  Angles: position * rate in double precision, reduced to a turn there (positions of 10^6 times a rate of one leave fp32
// with an error of 0.06 rad); sine and cosine once per pair, shared by all heads.  A warp per head: mean square, weights and rotation in
// fp32, one rounding at the end.
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
      const double turns = (double)t_pos[t] * (double)rates[i] * 0.15915494309189535;
      sincospif((float)((turns - rint(turns)) * 2.0), &sn[i], &cs[i]);
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

// One CTA per row and key head: the need-th largest key of the candidates [first, n - recent) by four passes over 8 bits each, then the
// kept slots in order (of the keys equal to it the lowest slots).
constexpr int SEL_THREADS = 1024;
__global__ void __launch_bounds__(SEL_THREADS)
paged_select_kernel(const float* mass, PageTable pt, const int32_t* lengths, int32_t* kept, int G, int keep, int first, int recent) {
  __shared__ unsigned hist[256];
  __shared__ unsigned s_prefix, s_need;
  __shared__ unsigned w_take[32], w_eq[32];
  const int g = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int n = lengths[r];
  n = n < 0 ? 0 : (n > table_slots(pt) ? table_slots(pt) : n);
  int32_t* out = kept + ((int64_t)r * G + g) * keep;
  if (n <= keep) {
    for (int i = tid; i < keep; i += SEL_THREADS) out[i] = i < n ? i : -1;
    return;
  }
  const int lo = first, hi = n - recent;
  auto key_at = [&](int j) -> uint32_t {
    const int64_t id = page_id(pt, r, j / pt.page);
    return id < 0 ? 0u : weight_key(mass[(id * G + g) * pt.page + j % pt.page]);
  };
  unsigned need = (unsigned)(keep - first - recent), prefix = 0, mask = 0;
  if (need > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += SEL_THREADS) hist[i] = 0;
      __syncthreads();
      for (int j = lo + tid; j < hi; j += SEL_THREADS) {
        const uint32_t u = key_at(j);
        if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift) & 255], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        unsigned left = need;
        int b = 255;
        while (b > 0 && hist[b] < left) left -= hist[b--];
        s_prefix = prefix | ((unsigned)b << shift);
        s_need = left;
      }
      __syncthreads();
      prefix = s_prefix;
      need = s_need;
      mask |= 255u << shift;
      __syncthreads();
    }
  }
  int base = 0;
  unsigned eq_base = 0;
  for (int j0 = 0; j0 < n; j0 += SEL_THREADS) {
    const int j = j0 + tid;
    const bool always = j < n && (j < lo || j >= hi);
    const uint32_t u = j < n && !always ? key_at(j) : 0u;
    const bool cand = j < n && !always && keep > first + recent;
    const bool eq = cand && u == prefix;
    const unsigned be = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) w_eq[warp] = __popc(be);
    __syncthreads();
    unsigned rank = eq_base + __popc(be & ((1u << lane) - 1)), all_eq = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) rank += w_eq[w];
      all_eq += w_eq[w];
    }
    const bool take = always || (cand && u > prefix) || (eq && rank < need);
    const unsigned bt = __ballot_sync(0xffffffffu, take);
    if (lane == 0) w_take[warp] = __popc(bt);
    __syncthreads();
    int at = base + __popc(bt & ((1u << lane) - 1)), all = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) at += w_take[w];
      all += w_take[w];
    }
    if (take && at < keep) out[at] = j;
    base += all;
    eq_base += all_eq;
    __syncthreads();
  }
}

// One CTA per row and key head closes the kept slots up in rounds: a round's lines go to registers, then (all of them read) to their places.
// A slot never moves up and the kept ones ascend, so no later round reads a place that an earlier one wrote.
constexpr int MOVE_THREADS = 512, MOVE_UNITS = 4;
__global__ void __launch_bounds__(MOVE_THREADS)
paged_compact_kernel(uint4* kp, uint4* vp, float* mass, PageTable pt, const int32_t* lengths, const int32_t* kept, int G, int chunks, int keep) {
  const int g = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
  int n = lengths[r];
  n = n > table_slots(pt) ? table_slots(pt) : n;
  const int32_t* from = kept + ((int64_t)r * G + g) * keep;
  auto place = [&](int j) -> int64_t {
    const int64_t id = page_id(pt, r, j / pt.page);
    return id < 0 ? -1 : (id * G + g) * pt.page + j % pt.page;
  };
  const int lines = min(MOVE_THREADS * MOVE_UNITS / chunks, MOVE_THREADS);     // per round; one weight per thread
  for (int i0 = 0; i0 < keep; i0 += lines) {
    uint4 a[MOVE_UNITS], b[MOVE_UNITS];
    float m = 0.f;
    int64_t to[MOVE_UNITS], to_m = -1;
#pragma unroll
    for (int u = 0; u < MOVE_UNITS; ++u) {
      const int x = u * MOVE_THREADS + tid, line = x / chunks, c = x - line * chunks, i = i0 + line;
      to[u] = -1;
      if (line < lines && i < keep) {
        const int j = from[i];
        if (j > i && j < n) {
          const int64_t src = place(j), dst = place(i);
          if (src >= 0 && dst >= 0) {
            a[u] = kp[src * chunks + c];
            b[u] = vp[src * chunks + c];
            to[u] = dst * chunks + c;
          } else if (c == 0) {
            atomicAdd(&g_paged_fault, 1u);
          }
        }
      }
    }
    if (mass && tid < lines && i0 + tid < keep) {
      const int i = i0 + tid, j = from[i];
      if (j > i && j < n) {
        const int64_t src = place(j), dst = place(i);
        if (src >= 0 && dst >= 0) { m = mass[src]; to_m = dst; }
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < MOVE_UNITS; ++u)
      if (to[u] >= 0) { kp[to[u]] = a[u]; vp[to[u]] = b[u]; }
    if (to_m >= 0) mass[to_m] = m;
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ dense view
// A page of a head is one run in the pages and one run of the dense cache: CTAs copy runs.
__global__ void __launch_bounds__(256)
paged_gather_kernel(const uint4* kp, const uint4* vp, PageTable pt, const int32_t* rows, const int32_t* lengths, uint4* kc, uint4* vc, int extra, int G,
                    int chunks, int64_t Tcap) {
  const int g = blockIdx.y, i = blockIdx.z, r = rows[i];
  if (r < 0) return;
  if (r >= pt.rows) {
    if (threadIdx.x == 0) atomicAdd(&g_paged_fault, 1u);
    return;
  }
  int64_t n = (int64_t)lengths[r] + extra;
  if (n > table_slots(pt)) n = table_slots(pt);
  if (n > Tcap) n = Tcap;
  const int64_t j0 = (int64_t)blockIdx.x * pt.page;
  if (j0 >= n) return;
  const int64_t id = page_id(pt, r, blockIdx.x);
  if (id < 0) {
    if (threadIdx.x == 0) atomicAdd(&g_paged_fault, 1u);
    return;
  }
  const int64_t left = n - j0, count = (left < pt.page ? left : pt.page) * chunks;
  const int64_t src = (id * G + g) * pt.page * chunks, dst = (((int64_t)i * G + g) * Tcap + j0) * chunks;
  for (int64_t x = threadIdx.x; x < count; x += blockDim.x) {
    kc[dst + x] = kp[src + x];
    vc[dst + x] = vp[src + x];
  }
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
  B200P_REQUIRE(rows < 65536, B200P_ERR_ARG, "too many rows");
  paged_select_kernel<<<dim3((unsigned)G, (unsigned)rows), SEL_THREADS, 0, (cudaStream_t)stream>>>(mass, pt, lengths, kept, G, keep, first, recent);
  B200P_LAUNCH_CHECK("paged_select_kernel");
  return B200P_OK;
}

extern "C" int b200p_paged_compact(void* kpages, void* vpages, float* mass, const int32_t* table, const int32_t* lengths, const int32_t* kept, int64_t P,
                                   int G, int D, int page, int rows, int width, int keep, int dtype, void* stream) {
  const PageTable pt{table, P, rows, width, page};
  const int rc = check_pages(kpages, vpages, pt, G, D, dtype);
  if (rc) return rc;
  B200P_REQUIRE(lengths && kept && keep > 0, B200P_ERR_ARG, "null pointer or nothing to keep");
  B200P_REQUIRE(rows < 65536, B200P_ERR_ARG, "too many rows");
  const int chunks = D * (dtype == B200P_F32 ? 4 : 2) / 16;
  paged_compact_kernel<<<dim3((unsigned)G, (unsigned)rows), MOVE_THREADS, 0, (cudaStream_t)stream>>>((uint4*)kpages, (uint4*)vpages, mass, pt, lengths, kept,
                                                                                                     G, chunks, keep);
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
  const int64_t most = (Tcap + page - 1) / page;
  paged_gather_kernel<<<dim3((unsigned)(most < width ? most : width), (unsigned)G, (unsigned)count), 256, 0, (cudaStream_t)stream>>>(
      (const uint4*)kpages, (const uint4*)vpages, pt, row_of, lengths, (uint4*)kcache, (uint4*)vcache, extra, G, chunks, Tcap);
  B200P_LAUNCH_CHECK("paged_gather_kernel");
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
