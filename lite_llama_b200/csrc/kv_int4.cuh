// Cache rows of K and V in 4 bits: layout and host checks shared by the writer, the reader and the attention kernels.
//
// One row of bytes per token.  For every kv head in turn:
//   K codes   head_dim / 2 bytes, element 2i in the low four bits of byte i
//   V codes   head_dim / 2 bytes
//   K groups  (scale, minimum) per group of `group` elements, both in the activations' type
//   V groups  the same
// and the row filled up to a multiple of 16 bytes.  An element is minimum + scale * code.  A token's heads lie side by side, so that
// one copy brings a block of heads, and a head's scales lie behind its codes, so that no second table has to be walked.
#pragma once
#include "common.cuh"

namespace kv4 {

constexpr int head_bytes(int d, int group) { return d + 8 * (d / group); }
inline int64_t row_bytes(int kv_heads, int d, int group) { return ((int64_t)kv_heads * head_bytes(d, group) + 15) / 16 * 16; }

// supported pairs of head size and group
constexpr bool shape_ok(int d, int group) {
  return (d == 32 || d == 64 || d == 128) && (group == 32 || group == 64 || group == 128) && group <= d;
}

#ifdef __CUDACC__
// (scale, minimum) as stored
template <typename T> __device__ __forceinline__ float2 scale_min(uint32_t w);
template <> __device__ __forceinline__ float2 scale_min<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
template <> __device__ __forceinline__ float2 scale_min<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
#endif

}  // namespace kv4

// Run `body` with `D` and `GS` bound to the head size and the group (host side, inside an int-returning function).
#define KV4_DISPATCH_SHAPE(d, group, ...)                                     \
  do {                                                                        \
    if ((d) == 128 && (group) == 64) { constexpr int D = 128, GS = 64; __VA_ARGS__ }        \
    else if ((d) == 128 && (group) == 32) { constexpr int D = 128, GS = 32; __VA_ARGS__ }   \
    else if ((d) == 128 && (group) == 128) { constexpr int D = 128, GS = 128; __VA_ARGS__ } \
    else if ((d) == 64 && (group) == 64) { constexpr int D = 64, GS = 64; __VA_ARGS__ }     \
    else if ((d) == 64 && (group) == 32) { constexpr int D = 64, GS = 32; __VA_ARGS__ }     \
    else { constexpr int D = 32, GS = 32; __VA_ARGS__ }                       \
  } while (0)
