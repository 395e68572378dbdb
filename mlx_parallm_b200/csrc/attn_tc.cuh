// What the tcgen05 attention kernels share (attn_prefill_tc.cu, paged_prefix_tc.cuh): the shape of their tiles, barriers, operands and arithmetic.
#pragma once
#include <type_traits>

#include "common.cuh"
#include "tc_ptx.cuh"

namespace b200p {

constexpr int FT_D = 128, FT_ROWS = 128, FT_KEYS = 128;
constexpr int FT_TILE_BYTES = 128 * FT_D * 2;              // 32 KB: a Q, K or V tile, two halves of [128 rows x 128 bytes]
constexpr int FT_HALF = FT_TILE_BYTES / 2;
constexpr int FT_RING = 5;
constexpr int FT_THREADS = 384;
// registers of 384 threads at launch: 384 x 168 = 64512 = 256 x 216 + 128 x 72, with several items per CTA 256 x 200 + 128 x 104
constexpr int ft_regs_softmax(bool many) { return many ? 200 : 216; }
constexpr int ft_regs_other(bool many) { return many ? 104 : 72; }
constexpr int FT_SMEM = 1024 + (2 + FT_RING) * FT_TILE_BYTES + 256;

struct AttnTcShared {
  uint64_t q_full, q_empty, kv_full[FT_RING], kv_empty[FT_RING], s_full[2], p_full[2], o_full[2];
  uint32_t tmem_base;
  volatile int abort;
};

__device__ __forceinline__ void ft_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// N-major (rows of the tile = k, 64 n per 128-byte row) SWIZZLE_128B operand: 8-k groups 1024 bytes apart, the next 64 n one half
// tile further
__device__ __forceinline__ uint64_t ft_desc_n_major(uint32_t smem_addr) {
  return (uint64_t)((smem_addr >> 4) & 0x3FFFu) | ((uint64_t)(FT_HALF >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
      "%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <typename T> __device__ __forceinline__ uint32_t ft_pack(float a, float b);
template <> __device__ __forceinline__ uint32_t ft_pack<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t ft_pack<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T> __device__ __forceinline__ float2 ft_unpack(uint32_t u);
template <> __device__ __forceinline__ float2 ft_unpack<__half>(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
template <> __device__ __forceinline__ float2 ft_unpack<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

}  // namespace b200p
