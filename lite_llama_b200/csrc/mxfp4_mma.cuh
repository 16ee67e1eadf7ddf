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

// ---- silu(g) * u of two sums, quantised ----
// Computed in 32 bits, to within 11 x 2^-24 of itself: expf and the quotient two units of the last place each, two roundings, and one of the
// scaled value.  What lies within 2^-20 of a border, or a largest magnitude that near to a power of two, is computed again in 64 bits from the
// same sums, so the codes are those of exact arithmetic on the sums (one value in 10^6 was off by a step without it, by a quarter of
// itself: 2.5e-3 of the result where it stood in a strong token).  A bias is added in 32 bits, which the exponential
// takes up to |g| times, and exactly in the second computation: 2^-17.  1000 x 28672 x 4096: 49.3 us, 47.0
// without the second look.
__device__ __forceinline__ float gated(float g, float u) { return __fdividef(g, 1.f + expf(-g)) * u; }      // 0 where the divisor is above 2^126
static __device__ __noinline__ double gated_64(double g, double u) { return g / (1.0 + exp(-g)) * u; }

struct Near { float below, above; uint32_t steps; };      // the interval's ends as factors, and in units of 2^-24
__device__ __forceinline__ Near near_of(bool biased) { return biased ? Near{1.f - 0x1p-17f, 1.f + 0x1p-17f, 128u} : Near{1.f - 0x1p-20f, 1.f + 0x1p-20f, 16u}; }
// A block all of which is below 2^-60 is always computed again: there are gates of less than -80 in it, where 32 bits lose digits.
__device__ __forceinline__ bool near_power(uint32_t top, uint32_t steps) { return top < 0x21800000u || ((top - steps) ^ (top + steps)) >> 23 != 0u; }

// Blocks again in 64 bits, those that a lane of `asked` has a share of: a block at a time, a value to each lane (a value takes some 2000 cycles,
// nearly all of them latency: a thread with a whole block by itself made 1000 x 28672 x 4096 twice as slow).
template <int N, typename T>
__device__ __forceinline__ void unit_again(const float (&g)[N], const float (&u)[N], const T* bias, uint32_t asked, uint32_t (&codes)[(N + 7) / 8],
                                           uint32_t& byte) {
  constexpr int kLanes = 32 / N;
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  while (asked) {
    const int first = (__ffs(asked) - 1) & ~(kLanes - 1), from = first + lane / N, at = lane % N;
    asked &= ~(((1u << kLanes) - 1u) << first);
    float gate = 0.f, up = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float a = __shfl_sync(0xffffffffu, g[j], from), b = __shfl_sync(0xffffffffu, u[j], from);
      if (at == j) { gate = a; up = b; }
    }
    double a = gate, b = up;
    if (bias) {                        // of the whole warp or of none
      const T* rows = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, (unsigned long long)bias, from)) + at;
      a += (double)to_f32(rows[0]);
      b += (double)to_f32(rows[64]);
    }
    const double v = gated_64(a, b);
    double top = fabs(v);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    const uint32_t scale = scale_byte(top);
    uint32_t word = (scale == 255u ? 0u : code_of(v * inverse_scale_64(scale))) << (4 * (lane & 7));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
    const int share = lane - first;    // of the block
    const bool mine = share >= 0 && share < kLanes;
#pragma unroll
    for (int q = 0; q < (N + 7) / 8; ++q) {
      const uint32_t w = __shfl_sync(0xffffffffu, word, (share * N + 8 * q) & 31);
      if (mine) codes[q] = N == 4 ? w >> (16 * (share & 1)) & 0xffffu : w;
    }
    if (mine) byte = scale;
  }
}

// A lane's N of a block's 32 activations from their sums (32 / N neighbouring lanes; the whole warp takes part): the codes, and the block's scale
// byte.  bias: of these gate rows, the up rows' 64 further on, or null.  in: of an output; others are as it comes.
template <int N, typename T>
__device__ __forceinline__ void quantise_unit(const float (&g)[N], const float (&u)[N], const T* bias, bool in, uint32_t (&codes)[(N + 7) / 8],
                                              uint32_t& byte) {
  const Near near = near_of(bias != nullptr);
  float v[N], m = 0.f;
  if (bias) {                          // a branch of its own: without a bias nothing of it is issued
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = gated(g[j] + to_f32(bias[j]), u[j] + to_f32(bias[64 + j]));
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = gated(g[j], u[j]);
  }
#pragma unroll
  for (int j = 0; j < N; j += 2) m = max_abs(m, v[j], v[j + 1]);
#pragma unroll
  for (int o = 1; o < 32 / N; o <<= 1) m = max_abs(m, __shfl_xor_sync(0xffffffffu, m, o), 0.f);
  const uint32_t top = abs_bits(m);
  byte = scale_byte(top);
  const float inv = inverse_scale(byte);
  const f32x2 low = pair_of(inv * near.below, inv * near.below), high = pair_of(inv * near.above, inv * near.above);
  bool unsure = near_power(top, near.steps);
#pragma unroll
  for (int q = 0; q < (N + 7) / 8; ++q) {
    f32x2 a[4], b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = 8 * q + 2 * j;
      const f32x2 x = i < N ? pair_of(v[i < N ? i : 0], v[i < N ? i + 1 : 0]) : 0ull;
      a[j] = mul2(x, low);
      b[j] = mul2(x, high);
    }
    codes[q] = codes8(a);
    unsure = unsure || codes[q] != codes8(b);
    if (byte == 255u) codes[q] = 0u;
  }
  if (top == 0u) {                     // zeros, or too small for 32 bits
    unsure = false;
#pragma unroll
    for (int j = 0; j < N; ++j)
      unsure = unsure || (bias ? g[j] + to_f32(bias[j]) != 0.f && u[j] + to_f32(bias[64 + j]) != 0.f : g[j] != 0.f && u[j] != 0.f);
  }
  const uint32_t asked = __ballot_sync(0xffffffffu, unsure && in && byte != 255u);
  if (asked) unit_again<N, T>(g, u, bias, asked, codes, byte);
}

#endif  // __CUDACC__

}  // namespace mx4
