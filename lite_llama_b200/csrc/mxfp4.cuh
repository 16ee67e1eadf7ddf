// Microscaled 4-bit floating point: rows of e2m1 elements (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), 32 consecutive
// ones of which share a power of two (the OCP microscaling format MXFP4).
//
//   scale byte   b = max(exponent field of the block's largest magnitude - 2, 0), the scale is 2^(b - 127): the largest power of
//                two not above that magnitude, over 4 (the largest power of two of an element).  255: the block is NaN, which is
//                what a block with an infinity or a NaN becomes.
//   element      the value over the scale, rounded to the nearest element (ties to the even code), at most 6 in magnitude
//   codes        uint8 [rows, k / 2], element 2i in the low half of byte i
//   scales       uint8 [ceil(rows / 128)][ceil(k / 128)][32][4][4], indices row % 32, row % 128 / 32, block % 4: tiles of 512 bytes
//                for 128 rows x 128 elements.  It is the order in which the tensor cores want their scales (a tile fills 32
//                lanes x 4 columns of tensor memory by one tcgen05.cp), so no product rearranges them.  Blocks behind k are 0;
//                rows behind the last one hold anything.
//
// Scaling by a power of two is exact, so an element depends on its value alone: what is quantised from 16 bits is the same
// bits wherever it is quantised.  Kernels that quantise what they computed in 32 bits (the norm, the gated unit) look whether the value lies
// so near a border that its own error could decide, and compute those blocks again in 64 bits.
#pragma once
#include "common.cuh"
#include <type_traits>

namespace mx4 {

constexpr int kBlock = 32;             // elements that share a scale
constexpr int kTileBytes = 512;        // scales of 128 rows x 128 elements

static inline int64_t k_tiles(int64_t k) { return cdiv64(k, 128); }

#ifdef __CUDACC__

// byte offset of the scale word (4 blocks = 128 elements) `kt` of a row
__device__ __forceinline__ int64_t scale_word(int64_t row, int kt, int64_t ktiles) {
  return ((row >> 7) * ktiles + kt) * kTileBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// bits of a magnitude -> scale byte (monotonic: infinities and NaN have the exponent field 255)
__device__ __forceinline__ uint32_t scale_byte(uint32_t abs_bits) {
  const uint32_t field = abs_bits >> 23;
  return field == 255u ? 255u : (field > 2u ? field - 2u : 0u);
}
// 2^(127 - byte), exactly representable for every byte of a finite block (at most 252)
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float((254u - (byte > 253u ? 253u : byte)) << 23); }
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __uint_as_float(byte == 0u ? 0x00400000u : (byte == 255u ? 0x7fc00000u : byte << 23));
}

// eight scaled values -> eight codes, the first in the lowest half byte
__device__ __forceinline__ uint32_t codes8(const float (&t)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r) : "f"(t[0]), "f"(t[1]), "f"(t[2]), "f"(t[3]), "f"(t[4]), "f"(t[5]), "f"(t[6]), "f"(t[7]));
  return r;
}
// eight codes -> eight elements (exact)
__device__ __forceinline__ void elements8(uint32_t c, float (&t)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(c));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    t[2 * i] = f.x;
    t[2 * i + 1] = f.y;
  }
}
// scale byte of a block by its largest magnitude in 64 bits, 2^(127 - byte), and the code of a scaled value
__device__ __forceinline__ uint32_t scale_byte(double top) {
  const int field = (int)((__double_as_longlong(top) >> 52) & 2047) - 1023 + 127;
  return field > 254 ? 255u : (field > 2 ? (uint32_t)(field - 2) : 0u);
}
__device__ __forceinline__ double inverse_scale_64(uint32_t byte) { return __longlong_as_double((long long)(1023 + 127 - (int)byte) << 52); }
__device__ __forceinline__ uint32_t code_of(double t) {
  const double m = fabs(t);
  const uint32_t c = (m > 0.25) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0);
  return c | (signbit(t) ? 8u : 0u);
}

// Four neighbouring lanes hold a block.  All lanes of the warp take part; `abs_bits` is the lane's largest magnitude.
__device__ __forceinline__ uint32_t block_max(uint32_t abs_bits) {
  uint32_t m = abs_bits;
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  return max(m, __shfl_xor_sync(0xffffffffu, m, 2));
}
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// the largest magnitude; NaN if one of them is
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// pairs of 32-bit values (one instruction for both)
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair_of(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float first_of(f32x2 p) { return __uint_as_float((uint32_t)p); }
__device__ __forceinline__ float second_of(f32x2 p) { return __uint_as_float((uint32_t)(p >> 32)); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// two 16-bit values in 32 bits
template <typename T> __device__ __forceinline__ f32x2 widen(uint32_t w);
template <> __device__ __forceinline__ f32x2 widen<__nv_bfloat16>(uint32_t w) { return pair_of(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
template <> __device__ __forceinline__ f32x2 widen<__half>(uint32_t w) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return pair_of(f.x, f.y);
}
__device__ __forceinline__ uint32_t codes8(const f32x2 (&t)[4]) {
  const float v[8] = {first_of(t[0]), second_of(t[0]), first_of(t[1]), second_of(t[1]), first_of(t[2]), second_of(t[2]), first_of(t[3]), second_of(t[3])};
  return codes8(v);
}

// A lane's eight of a block's 32 values (four neighbouring lanes; the whole warp takes part): the codes, and the block's scale byte.
__device__ __forceinline__ uint32_t quantise8(float (&v)[8], uint32_t& byte) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[j]));
  byte = scale_byte(block_max(m));
  const float inv = inverse_scale(byte);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] *= inv;
  const uint32_t c = codes8(v);
  return byte == 255u ? 0u : c;
}

// The same of a lane's eight values as they lie in memory.  16 bits: magnitudes are compared two at a time as the whole numbers that their bits are,
// bf16 is scaled in pairs (exact but for what is far below the smallest element): 6 instructions an element, 14 by way of 32 bits.
template <typename T> struct Raw8 { uint4 q; };
template <> struct Raw8<float> { uint4 q, r; };
template <typename T> __device__ __forceinline__ uint32_t quantise_raw(const Raw8<T>& x, uint32_t& byte) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&x.q);
  uint32_t m = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
  m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 2));
  m = max(m & 0xffffu, m >> 16);
  f32x2 t[4];
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    byte = scale_byte(m << 16);
    const uint32_t f = (254u - (byte > 253u ? 253u : byte)) * 0x00800080u;
    const __nv_bfloat162 factor = *reinterpret_cast<const __nv_bfloat162*>(&f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 s = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), factor);
      t[i] = widen<__nv_bfloat16>(*reinterpret_cast<const uint32_t*>(&s));
    }
  } else {
    byte = scale_byte(__float_as_uint(__half2float(__ushort_as_half((unsigned short)m))));
    const float inv = inverse_scale(byte);
    const f32x2 inv2 = pair_of(inv, inv);
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = mul2(widen<__half>(w[i]), inv2);
  }
  const uint32_t c = codes8(t);
  return byte == 255u ? 0u : c;
}
template <> __device__ __forceinline__ uint32_t quantise_raw<float>(const Raw8<float>& x, uint32_t& byte) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = __uint_as_float(reinterpret_cast<const uint32_t*>(&x.q)[i]);
    v[4 + i] = __uint_as_float(reinterpret_cast<const uint32_t*>(&x.r)[i]);
  }
  return quantise8(v, byte);
}
template <typename T> __device__ __forceinline__ void load_raw(const T* p, Raw8<T>& x) { x.q = ldg_stream_128(p); }
template <> __device__ __forceinline__ void load_raw<float>(const float* p, Raw8<float>& x) {
  x.q = ldg_stream_128(p);
  x.r = ldg_stream_128(p + 4);
}
template <typename T> __device__ __forceinline__ void zero_raw(Raw8<T>& x) {
  x.q = make_uint4(0u, 0u, 0u, 0u);
  if constexpr (sizeof(T) == 4) x.r = x.q;
}

__device__ __forceinline__ uint32_t ld_once(const uint8_t* p) {
  uint32_t v;
  asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}

#endif  // __CUDACC__

}  // namespace mx4
