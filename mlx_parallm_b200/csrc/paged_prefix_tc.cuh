// The shared slots of b200p_paged_attn_shared on tcgen05, 16-bit caches, head_dim 128 (part of paged_attn.cu): attn_prefill_tc.cu's two tiles of 128 rows that
// take turns, here the two halves of a tile of query heads of a group's tokens, over keys in pages and without a mask but for the last.
//
// The 128 keys of a step come as boxes of 16 to 128 keys that lie in one page each; their ids are looked up a step ahead, a lane per box, and a box without
// a page is fetched from behind the pages, where the copy brings zeros.  A CTA's part of the work is runs of steps of one item after the other, each of
// which leaves a part.  Products, softmax and roles are those of the prompt kernel, but the maximum may lag by 2^6 before outputs are rescaled (a part is few
// steps, in most of which one of a warp's rows finds a new one: 114 -> 104 thousand cycles for 30 steps), and for f16 it is held 8 lower, so that weights reach
// 2^14 and small ones keep their bits.  A weight is two 16-bit numbers, the rounded one and what it lost, which multiply the same values one after the other, so
// that an output carries its own rounding only, as it does where nothing is shared.  (As one number, with the sum of the rounded ones,
// the error was 1.3 times that, and 128 rows behind 16000 slots took 106.0 us instead of 119.6, 64 behind 4000 44.5 instead of 46.2.)
//
// The weights of a step's first 64 keys are multiplied while those of the last 64 are made (128 rows behind 16000 slots, one number a weight, 109.4 -> 106.1 us).
//
// 128 rows in two groups behind 16000 and 12032 slots, 64 / 8 heads (60 GFLOP, 90 with the weights' second numbers): CTAs end after 72 to 91 us, 81 in the median;
// 4250 cycles a step of 256 rows, against 3072 of the tensor core's and 2048 of its exponentials.  Of 64 rows behind 4000 slots a CTA has 3.5 steps, and the plan (4000 cycles), queries
// (5000), first copy (1500) and the part (5000) are most of its time.
#pragma once
#include "attn_tc.cuh"

namespace b200p {

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
               "r"(r[15])
               : "memory");
}

template <typename T>
__global__ void __launch_bounds__(FT_THREADS, 1)
paged_prefix_tc_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const __grid_constant__ PagedPrefix a) {
  constexpr float SHIFT = std::is_same<T, __half>::value ? 8.f : 0.f, LAG = 6.f;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ PrefixPlan s_plan;
  __shared__ uint64_t s_rest[2];                            // the weights of a step's last 64 keys (sh->p_full: of its first)
  __shared__ struct { PrefixCursor<FT_KEYS, false> cursor; PrefixRun run; } s_kept[8];      // the steps' loop has no registers for them
  const uint32_t raw = smem_u32(smem);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t ring = base + 2 * FT_TILE_BYTES;
  AttnTcShared* sh = reinterpret_cast<AttnTcShared*>(smem + (base - raw) + (2 + FT_RING) * FT_TILE_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&sh->q_full), 8);
    for (int s = 0; s < FT_RING; ++s) { mbar_init(smem_u32(&sh->kv_full[s]), 1); mbar_init(smem_u32(&sh->kv_empty[s]), 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(smem_u32(&sh->s_full[i]), 1); mbar_init(smem_u32(&sh->p_full[i]), 4); mbar_init(smem_u32(&s_rest[i]), 4); mbar_init(smem_u32(&sh->o_full[i]), 1); }
    sh->abort = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmk);
    tma_prefetch_desc(&tmv);
  }
  if (warp == 8) tmem_alloc(smem_u32(&sh->tmem_base), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;                     // S of half i at 128 i (P over its first 64, what P lost over the others), O of half i at 256 + 128 i
  pdl_wait();
  pdl_launch_dependents();
  PrefixRun run;
  PrefixCursor<FT_KEYS, false> cursor = prefix_plan<FT_THREADS, FT_KEYS, false>(a, s_plan, run);
  auto wait = [&](uint64_t& bar, uint32_t parity, int role) { return mbar_wait_warp(smem_u32(&bar), parity, &sh->abort, a.wait_word, role); };
  bool ok = true;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(ft_regs_other(true)));
    if (warp == 9) {
      // ===================================== TMA producer =====================================
      const int boxes = FT_KEYS / a.box, page = a.pt.page;
      int slot = 0;
      uint32_t ph = 0;
      while (ok && cursor.next(a, run)) {
        const int32_t* table = a.pt.table + (int64_t)run.table_row * a.pt.width;
        const int nowhere = (int)(a.pt.P * a.G * page);    // behind the pages: zeros (the host has checked that it fits)
        auto seek = [&](int u) {                           // the line of this lane's box
          const int key = u * FT_KEYS + lane * a.box;
          if (lane >= boxes || u >= run.last || key >= run.common) return nowhere;
          const int index = key / page, id = table[index];
          if ((unsigned)id >= (unsigned)a.pt.P) {
            atomicAdd(&g_paged_attn_fault, 1u);
            return nowhere;
          }
          return (id * a.G + run.g) * page + key - index * page;
        };
        int line = seek(run.first);
        for (int u = run.first; ok && u < run.last; ++u) {
          const int ahead = seek(u + 1);
#pragma unroll 1
          for (int kv = 0; kv < 2; ++kv) {
            if (!(ok = wait(sh->kv_empty[slot], ph ^ 1u, 0))) break;
            const uint32_t bar = smem_u32(&sh->kv_full[slot]), dst = ring + slot * FT_TILE_BYTES;
            const CUtensorMap* m = kv ? &tmv : &tmk;
            if (lane == 0) mbar_arrive_expect_tx(bar, FT_TILE_BYTES);
#pragma unroll 1
            for (int b = 0; b < boxes; ++b) {
              const int at = __shfl_sync(~0u, line, b);
              if (lane == 0) {
                tma_load_2d(dst + b * a.box * 128, m, 0, at, bar);
                tma_load_2d(dst + FT_HALF + b * a.box * 128, m, 64, at, bar);
              }
            }
            __syncwarp();
            if (++slot == FT_RING) { slot = 0; ph ^= 1u; }
          }
          line = ahead;
        }
      }
    } else if (warp == 8) {
      // ===================================== MMA issuer =======================================
      constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      constexpr uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
      constexpr uint32_t idesc_pv = idesc | (1u << 16);    // B is N-major
      auto qk = [&](int i, int slot) {
        const uint64_t ad = make_desc_sw128(base + i * FT_TILE_BYTES), bd = make_desc_sw128(ring + slot * FT_TILE_BYTES);
#pragma unroll
        for (int k = 0; k < 8; ++k) {                      // 16 k = 32 bytes of a 128-byte row; k 4..7 in the other half of the operand
          const uint64_t off = (uint64_t)((k & 3) * 2 + (k >> 2) * (FT_HALF >> 4));
          ft_mma_ss(tmem + 128 * i, ad + off, bd + off, idesc, k ? 1u : 0u);
        }
      };
      auto pv = [&](int i, int slot, int from, uint32_t acc) {
        const uint64_t bd = ft_desc_n_major(ring + slot * FT_TILE_BYTES);
#pragma unroll
        for (int k = from; k < from + 4; ++k) {            // 16 keys = 2048 bytes; P: 8 columns, and what it lost 64 columns further
          umma_f16_ts(tmem + 256 + 128 * i, tmem + 128 * i + 8 * k, bd + (uint64_t)(k * (2048 >> 4)), idesc_pv, (k || acc) ? 1u : 0u);
          umma_f16_ts(tmem + 256 + 128 * i, tmem + 128 * i + 64 + 8 * k, bd + (uint64_t)(k * (2048 >> 4)), idesc_pv, 1u);
        }
      };
      int slot = 0, round = 0;
      uint32_t ph = 0, pph[2] = {0, 0};                    // phases of `slot` and of the probabilities' barriers
      while (ok && cursor.next(a, run)) {
        const int both = run.rows > PS_HALF ? 2 : 1, steps = run.last - run.first;
        const int k0 = slot;
        if (!(ok = wait(sh->q_full, (uint32_t)(round & 1), 1) && wait(sh->kv_full[k0], ph, 1))) break;
        ++round;
        if (++slot == FT_RING) { slot = 0; ph ^= 1u; }
        tc_fence_after();
        if (elect_one()) {
          for (int i = 0; i < both; ++i) {
            qk(i, k0);
            umma_commit(smem_u32(&sh->s_full[i]));
          }
          umma_commit(smem_u32(&sh->kv_empty[k0]));
        }
        __syncwarp();
        for (int j = 0; j < steps && ok; ++j) {
          const int vslot = slot;
          if (!(ok = wait(sh->kv_full[vslot], ph, 1))) break;
          if (++slot == FT_RING) { slot = 0; ph ^= 1u; }
          const int left = run.common - (run.first + j) * FT_KEYS;
          if (left < FT_KEYS) {
            // the weights of keys behind the shared ones are zero, but what lies there may not be finite: zero those rows of V
            for (int c = lane; c < (FT_KEYS - left) * 16; c += 32) {
              const int row = left + (c >> 4), hf = (c >> 3) & 1, ch = c & 7;
              asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(ring + vslot * FT_TILE_BYTES + hf * FT_HALF + row * 128 + ch * 16), "r"(0) : "memory");
            }
            fence_proxy_async_smem();
            __syncwarp();
          }
          const bool more = j + 1 < steps;
          const int kslot = slot;
          if (more) {
            if (!(ok = wait(sh->kv_full[kslot], ph, 1))) break;
            if (++slot == FT_RING) { slot = 0; ph ^= 1u; }
          }
          for (int i = 0; i < both; ++i) {
            if (!(ok = wait(sh->p_full[i], pph[i], 1))) break;
            tc_fence_after();
            if (elect_one()) pv(i, vslot, 0, j > 0 ? 1u : 0u);
            __syncwarp();
            if (!(ok = wait(s_rest[i], pph[i], 1))) break;
            pph[i] ^= 1u;
            tc_fence_after();
            if (elect_one()) {
              pv(i, vslot, 4, 1u);
              if (i == both - 1) umma_commit(smem_u32(&sh->kv_empty[vslot]));
              if (more) {
                qk(i, kslot);
                umma_commit(smem_u32(&sh->s_full[i]));
                if (i == both - 1) umma_commit(smem_u32(&sh->kv_empty[kslot]));
              } else {
                umma_commit(smem_u32(&sh->o_full[i]));
              }
            }
            __syncwarp();
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(ft_regs_softmax(true)));
    // ===================================== softmax and parts ================================
    const int i = warp >> 2, q = warp & 3, per = a.H / a.G;
    const int r = q * 32 + lane;                           // row of the half = TMEM lane
    const uint32_t s_addr = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(128 * i), o_addr = s_addr + 256;
    const float2 sc2 = make_float2(a.scale_log2e, a.scale_log2e);
    uint32_t sph = 0, oph = 0, round = 0;
    while (ok && cursor.next(a, run)) {
      // (all products of the run before have been waited for by the half that both runs have, or were not made: the queries' place is free)
      const bool mine = i == 0 || run.rows > PS_HALF;
      const int at = PS_HALF * i + r;
      cursor.tell(a, run, at);
      if (mine) {
        // 16 lanes have a row, so that a load is two whole rows (a row per lane, 32 lines a load: 9100 cycles up to the arrival instead of 5000)
        const int64_t line = at < run.rows ? ((int64_t)a.plan.order()[run.tile.y + at / per] * a.H + (int64_t)run.g * per + at % per) * 16 : -1;
        const int c = lane & 15;
        uint4 x[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const int64_t from = __shfl_sync(~0u, line, 2 * k + (lane >> 4));
          x[k] = from >= 0 ? reinterpret_cast<const uint4*>(a.q)[from + c] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const int row = q * 32 + 2 * k + (lane >> 4);
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(base + i * FT_TILE_BYTES + (c >> 3) * FT_HALF + row * 128 + (((c & 7) ^ (row & 7)) << 4)),
                       "r"(x[k].x), "r"(x[k].y), "r"(x[k].z), "r"(x[k].w)
                       : "memory");
        }
        fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh->q_full));
      // whether every key of the run has a page: seldom not, and then the scores look theirs up
      const int32_t* table = a.pt.table + (int64_t)run.table_row * a.pt.width;
      bool bad = false;
      for (int p = run.first * FT_KEYS / a.pt.page + lane; p <= (min(run.common, run.last * FT_KEYS) - 1) / a.pt.page; p += 32)
        bad |= (unsigned)table[p] >= (unsigned)a.pt.P;
      bad = __any_sync(~0u, bad);
      if (!mine) {                                         // (an arrival for the next run would count for this one until all of its are in)
        ok = wait(sh->q_full, round & 1u, 2 + i);
        ++round;
        continue;
      }
      ++round;
      if (lane == 0) s_kept[warp].cursor = cursor, s_kept[warp].run = run;
      __syncwarp();
      const int common = run.common, first = run.first, last = run.last;
      float m = -INFINITY, sum = 0.f;
      for (int u = first; u < last; ++u) {
        if (!(ok = wait(sh->s_full[i], sph, 2 + i))) break;
        sph ^= 1u;
        tc_fence_after();
        float s[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + 32 * c, s + 32 * c);
        tmem_ld_wait();
        const int n = common - u * FT_KEYS;            // shared keys from this step's first on
        if (n < FT_KEYS || bad) {
          unsigned pages = 0xffu;                          // which 16 keys have a page
          if (bad) {
            pages = 0;
#pragma unroll 1
            for (int c = 0; c < 8; ++c)
              if (16 * c < n) pages |= ((unsigned)table[(u * FT_KEYS + 16 * c) / a.pt.page] < (unsigned)a.pt.P ? 1u : 0u) << c;
          }
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c] = c < n && (pages >> (c / 16) & 1u) ? s[c] : -INFINITY;
        }
        float t0 = max3(s[0], s[1], s[2]), t1 = max3(s[3], s[4], s[5]), t2 = max3(s[6], s[7], s[8]), t3 = max3(s[9], s[10], s[11]);
#pragma unroll
        for (int c = 12; c + 8 <= 128; c += 8) {
          t0 = max3(t0, s[c], s[c + 1]);
          t1 = max3(t1, s[c + 2], s[c + 3]);
          t2 = max3(t2, s[c + 4], s[c + 5]);
          t3 = max3(t3, s[c + 6], s[c + 7]);
        }
        t0 = max3(t0, s[124], s[125]);
        t1 = max3(t1, s[126], s[127]);
        const float mt = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3)) * a.scale_log2e - SHIFT;      // (the host sends positive scales here)
        const float mn = mt > m + LAG ? mt : m, ref = mn == -INFINITY ? 0.f : mn, f = ex2(m - ref);
        const bool rescale = u > first && __any_sync(~0u, mn > m);
        m = mn;
        const float2 nm2 = make_float2(-ref, -ref);
        if (rescale) {                                     // (beside 128 scores in registers: 16 columns at a time)
#pragma unroll 1
          for (int c = 0; c < FT_D; c += 16) {
            float o[16];
            uint32_t w[16];
            tmem_ld16(o_addr + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 16; ++k) w[k] = __float_as_uint(o[k] * f);
            tmem_st16(o_addr + c, w);
          }
        }
        float2 a0 = make_float2(0.f, 0.f), a1 = a0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int part = 4 * h; part < 4 * h + 4; part += 2) {      // 32 keys at a time: what the weights lost has no registers beside all of them
            uint32_t w[16], rest[16];
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const int key = 16 * part + 2 * c;
              const float2 x = __ffma2_rn(make_float2(s[key], s[key + 1]), sc2, nm2), e = make_float2(ex2(x.x), ex2(x.y));
              w[c] = ft_pack<T>(e.x, e.y);
              const float2 lost = __ffma2_rn(ft_unpack<T>(w[c]), make_float2(-1.f, -1.f), e);
              rest[c] = ft_pack<T>(lost.x, lost.y);
              if (c & 1) a1 = __fadd2_rn(a1, e); else a0 = __fadd2_rn(a0, e);
            }
            tmem_st16(s_addr + 8 * part, w);
            tmem_st16(s_addr + 64 + 8 * part, rest);
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(h ? &s_rest[i] : &sh->p_full[i]));
        }
        sum = sum * f + ((a0.x + a0.y) + (a1.x + a1.y));
      }
      if (ok) ok = wait(sh->o_full[i], oph, 2 + i);
      oph ^= 1u;
      cursor = s_kept[warp].cursor, run = s_kept[warp].run;
      if (ok) {
        tc_fence_after();
        // A row's outputs are in a lane: 32 columns at a time go through the warp's own place among the queries, which nobody reads any more, so that
        // lines are written whole.
        float* part = a.rec + (run.row0 + (int64_t)blockIdx.x * PS_ROWS + PS_HALF * i + 32 * q) * (FT_D + PS_HEAD);
        const int rows = min(32, run.rows - PS_HALF * i - 32 * q);
        if (lane < rows) *reinterpret_cast<float2*>(part + lane * (FT_D + PS_HEAD)) = make_float2(m, sum);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t own = base + i * FT_TILE_BYTES + (c & 1) * FT_HALF + q * 4096;
          float o[32];
          tmem_ld32(o_addr + 32 * c, o);
          tmem_ld_wait();
          if (rows <= 0) continue;
#pragma unroll
          for (int k = 0; k < 8; ++k)
            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(own + lane * 128 + ((k ^ (lane & 7)) << 4)), "f"(o[4 * k]), "f"(o[4 * k + 1]),
                         "f"(o[4 * k + 2]), "f"(o[4 * k + 3])
                         : "memory");
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int row = 4 * k + (lane >> 3), ch = lane & 7;
            const uint4 y = lds128(own + row * 128 + ((ch ^ (row & 7)) << 4));
            if (row < rows) *reinterpret_cast<uint4*>(part + row * (FT_D + PS_HEAD) + PS_HEAD + 32 * c + 4 * ch) = y;
          }
          __syncwarp();
        }
        tc_fence_before();                                 // (the next run's first products write there again)
      }
    }
  }
  if (sh->abort) wait_settle();
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace b200p
