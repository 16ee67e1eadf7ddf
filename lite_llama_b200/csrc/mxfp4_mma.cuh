// Block-scaled tensor core products of microscaled 4-bit operands (mxfp4.cuh): tcgen05.mma kind::mxf4, scales in tensor memory.
//
// One MMA multiplies 64 elements of k (32 bytes of a row) and takes two scales per row of either operand.  A scale tile (128 rows x 128
// elements, 512 bytes: 32 rows of 16) fills 4 columns: lane r of every quarter, column c holds the four scales of row 32 c + r, two
// MMAs' worth; the scale ids of the instruction descriptor choose the half.  tcgen05.cp brings a tile in ahead of the MMAs that read
// it, issued by the same thread (the pair is ordered by itself).  Columns are reused a whole ring of stages later, when the
// barrier that freed the stage has said that its MMAs are done.
#pragma once
#include "mxfp4.cuh"

namespace mx4 {

constexpr int kStageK = 256;           // elements of k per pipeline stage: 128 bytes of a row, one swizzle atom, four MMAs
constexpr int kSfBytes = 2 * kTileBytes;   // scales of 128 rows per stage

#ifdef __CUDACC__

// M x N of the MMA (M = 128, a pair 256); e2m1 operands, power-of-two scales, `half` the pair of scales within a column
__host__ __device__ constexpr uint32_t idesc(uint32_t M, uint32_t N, uint32_t half) {
  return ((2u * half) << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | (1u << 23) | ((M >> 4) << 24) | ((2u * half) << 29);
}

constexpr uint32_t kSecondHalf = (2u << 4) | (2u << 29);      // idesc(M, N, 1) is idesc(M, N, 0) with these bits
static_assert(idesc(256, 256, 1) == (idesc(256, 256, 0) | kSecondHalf), "scale ids");

// 32 rows of 16 bytes, rows in groups of eight one after another
__device__ __forceinline__ uint64_t scale_desc(uint32_t smem_addr) {
  return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | ((uint64_t)(128u >> 4) << 16) | ((uint64_t)(128u >> 4) << 32) | ((uint64_t)1 << 46);
}

template <int CTAS> __device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t desc) {
  if (CTAS == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}

template <int CTAS>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if (CTAS == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}

// silu(g) * u in 32 bits
__device__ __forceinline__ float gated(float g, float u) { return __fdividef(g, 1.f + expf(-g)) * u; }

#endif  // __CUDACC__

}  // namespace mx4
