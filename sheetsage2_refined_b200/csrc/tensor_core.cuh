// tcgen05 and TMA helpers of the 16-bit attention tiles (sm_100a), beside
// those of gemm_tc.cuh: both operand types, 3-D loads, operands from tensor
// memory and operands whose M/N axis is contiguous.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>

#include "gemm_tc.cuh"
#include "mbarrier.cuh"
#include "prefill_attn.cuh"

namespace s2r {

// mbar_wait whose first tries come without a look at the timer, for waits in
// the chain of a tile (reading the timer costs hundreds of cycles).
__device__ __forceinline__ bool mbar_wait_fast(uint64_t* bar, unsigned parity) {
  const uint32_t addr = smem_u32(bar);
#pragma unroll 1
  for (int i = 0; i < 128; ++i)
    if (mbar_try(addr, parity)) return true;
  return mbar_wait(bar, parity);
}

// One lane of a converged warp (the same one each time).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// 3-D tiled TMA load of the box at (x, y, z); x in elements, a multiple of 64 here.
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// Instruction descriptor of kind::f16 with a float32 accumulator: `format` 0
// f16, 1 bf16 (the same for A and B); A K-major, B K-major or, with
// `b_mn_major` (bit 16), with its N axis contiguous.
__host__ __device__ constexpr uint32_t umma_idesc(uint32_t format, int m, int n, bool b_mn_major) {
  return (1u << 4) | (format << 7) | (format << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}

// Shared-memory matrix descriptor of an operand whose M/N axis is contiguous,
// 128-byte swizzle: rows of 64 M/N elements (128 bytes) per K index, 8 K
// indices to a 1024-byte group (stride byte offset: the next group), `next`
// bytes to the next 64 M/N elements (leading byte offset).
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(const void* smem, uint32_t next) {
  const uint64_t addr = smem_u32(smem);
  return ((addr >> 4) & 0x3FFFull) | ((uint64_t)(next >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
         (2ull << 61);
}

// D (tensor memory) = or += A B, A from shared memory.
__device__ __forceinline__ void umma_f16(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, bool accumulate) {
  umma_bf16(d, a_desc, b_desc, idesc, accumulate ? 1u : 0u);
}

// The same with A from tensor memory (two 16-bit K elements a column).
__device__ __forceinline__ void umma_f16_ta(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b_desc), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(0), "r"(0), "r"(0), "r"(0)
      : "memory");
}

// 32 columns of this thread's tensor-memory lane; visible after tmem_wait_st().
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// Two floats as one 64-bit operand of the packed float32 instructions.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t y;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
  return y;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t y;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
  return y;
}

__device__ __forceinline__ uint32_t pack_pair(bf16, float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_pair(__half, float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

}  // namespace s2r
