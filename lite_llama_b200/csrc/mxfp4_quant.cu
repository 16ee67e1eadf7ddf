// 16-bit (or 32-bit) rows to microscaled 4-bit floating point and back, by themselves and behind a residual add and RMS norm.
// Format and layout: mxfp4.cuh.  All three are bound by memory on large inputs and by launch latency on a decode step.
#include "mxfp4.cuh"

namespace mx4 {

constexpr int kWarps = 8;

// A warp takes 256 consecutive elements of a row: 16 bytes a lane (512 a warp) in, four bytes a lane out, one scale word per 16 lanes.
// Rows are `per` to a matrix; a matrix starts on a tile of scales of its own.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
quantize_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, const T* __restrict__ x, int64_t rows, int64_t per,
                int64_t k, int64_t x_stride, int64_t ktiles, int units) {
  pdl_prologue();
  const int lane = threadIdx.x & 31;
  const int64_t u = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int64_t row = u / units;
  if (row >= rows) return;                             // whole warps
  const int64_t c = (u - row * units) * 32 + lane;     // chunk of eight elements
  const bool in = c * 8 < k;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (in) load8(x + row * x_stride + c * 8, v);
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[j]));
  const uint32_t byte = scale_byte(block_max(m));
  const float inv = inverse_scale(byte);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] *= inv;
  const uint32_t word = word_of(in ? byte : 0u, lane);
  if (in) *reinterpret_cast<uint32_t*>(codes + row * (k / 2) + c * 4) = byte == 255u ? 0u : codes8(v);
  if (in && (lane & 15) == 0) {
    const int64_t matrix = row / per;
    const int64_t padded = matrix * ((per + 127) / 128 * 128) + (row - matrix * per);
    *reinterpret_cast<uint32_t*>(scales + scale_word(padded, (int)(c >> 4), ktiles)) = word;
  }
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
dequantize_kernel(T* __restrict__ y, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows,
                  int64_t per, int64_t k, int64_t codes_stride, int64_t ktiles, int units) {
  pdl_prologue();
  const int lane = threadIdx.x & 31;
  const int64_t u = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int64_t row = u / units;
  const int64_t c = (u - row * units) * 32 + lane;
  if (row >= rows || c * 8 >= k) return;
  const int64_t matrix = row / per;
  const int64_t padded = matrix * ((per + 127) / 128 * 128) + (row - matrix * per);
  const uint32_t word = *reinterpret_cast<const uint32_t*>(scales + scale_word(padded, (int)(c >> 4), ktiles));
  const uint32_t q = *reinterpret_cast<const uint32_t*>(codes + row * codes_stride + c * 4);
  const float s = scale_value((word >> (8 * ((c >> 2) & 3))) & 255u);
  float t[8];
  elements8(q, t);
  T* out = y + row * k + c * 8;
  if constexpr (sizeof(T) == 4) {
    stg_128(out, make_uint4(__float_as_uint(t[0] * s), __float_as_uint(t[1] * s), __float_as_uint(t[2] * s), __float_as_uint(t[3] * s)));
    stg_128(out + 4, make_uint4(__float_as_uint(t[4] * s), __float_as_uint(t[5] * s), __float_as_uint(t[6] * s), __float_as_uint(t[7] * s)));
  } else {
    stg_128(out, make_uint4(pack2<T>(t[0] * s, t[1] * s), pack2<T>(t[2] * s, t[3] * s), pack2<T>(t[4] * s, t[5] * s),
                            pack2<T>(t[6] * s, t[7] * s)));
  }
}

// ---------------------------------------------------------------------------------------------------------------
// s = x + r (stored over r, or to `sum`, in the activations' type), y = s / sqrt(mean s^2 + eps) * w, quantised.
//
// y is not rounded to 16 bits on the way: the 16-bit norm would round it twice (before and behind the weight), and elements that
// lie next to a border would then go by those roundings.  It is computed in 32 bits, at most 2^-21.5 off; where that could change an
// element or the scale (values within 2^-20 of a border, one element in 10^5), the warp computes its blocks again in 64 bits, so
// the codes are those of exact arithmetic.  The sum of squares is in 64 bits for them from the start.
// ---------------------------------------------------------------------------------------------------------------
template <typename T, int VPT>
__global__ void __launch_bounds__(512)
norm_quantize_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, T* __restrict__ sum, const T* __restrict__ x,
                     const T* __restrict__ res, const T* __restrict__ w, int64_t n, int64_t x_stride, int64_t r_stride,
                     int64_t s_stride, int64_t ktiles, float eps) {
  pdl_prologue();
  const int64_t row = blockIdx.x;
  const int chunks = (int)(n / 8), lane = threadIdx.x & 31;
  uint4 xv[VPT], rv[VPT];
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    xv[i] = rv[i] = make_uint4(0u, 0u, 0u, 0u);
    if (c < chunks) {
      xv[i] = ldg_128(x + row * x_stride + c * 8);
      if (res) rv[i] = ldg_128(res + row * r_stride + c * 8);
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    const T *xe = reinterpret_cast<const T*>(&xv[i]), *re = reinterpret_cast<const T*>(&rv[i]);
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float a = to_f32(xe[j]), b = to_f32(xe[j + 1]), d = to_f32(re[j]), e = to_f32(re[j + 1]);
      o[j / 2] = pack2<T>(a + d, b + e);
      const double p = (double)a + (double)d, q = (double)b + (double)e;
      ss = fma(p, p, ss);
      ss = fma(q, q, ss);
    }
    if (res && c < chunks) stg_128(sum + row * s_stride + c * 8, make_uint4(o[0], o[1], o[2], o[3]));
  }
  __shared__ double red[16];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (lane == 0) red[threadIdx.x >> 5] = ss;
  __syncthreads();
  double tot = 0.0;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) tot += red[i];
  const double rrms = 1.0 / sqrt(tot / (double)n + (double)eps);
  const float r32 = (float)rrms;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (c - lane >= chunks) break;                     // whole warps
    const bool in = c < chunks;
    uint4 wv = make_uint4(0u, 0u, 0u, 0u);
    if (in) wv = ldg_128(w + c * 8);
    const T *xe = reinterpret_cast<const T*>(&xv[i]), *re = reinterpret_cast<const T*>(&rv[i]), *we = reinterpret_cast<const T*>(&wv);
    float v[8];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = (to_f32(xe[j]) + to_f32(re[j])) * r32 * to_f32(we[j]);
      m = max(m, abs_bits(v[j]));
    }
    m = block_max(m);
    uint32_t byte = scale_byte(m);
    const float inv = inverse_scale(byte);
    float lo[8], hi[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float t = v[j] * inv;
      lo[j] = fmaf(t, -0x1p-20f, t);
      hi[j] = fmaf(t, 0x1p-20f, t);
    }
    uint32_t code = codes8(lo);
    // a value next to a border, a maximum next to a power of two (8 steps of 2^-23), or so small that 32 bits lose digits
    const bool near = m != 0u && byte != 255u && (code != codes8(hi) || ((m - 8u) >> 23) != ((m + 8u) >> 23) || m < 0x0d000000u);
    if (__any_sync(0xffffffffu, near)) {
      double d[8], top = 0.0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        d[j] = ((double)to_f32(xe[j]) + (double)to_f32(re[j])) * rrms * (double)to_f32(we[j]);
        top = fmax(top, fabs(d[j]));
      }
      top = fmax(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmax(top, __shfl_xor_sync(0xffffffffu, top, 2));
      if (byte != 255u) {                              // infinities and NaN are those of 32 bits
        const int field = (int)((__double_as_longlong(top) >> 52) & 2047) - 1023 + 127;
        byte = field > 254 ? 255u : (field > 2 ? (uint32_t)(field - 2) : 0u);
        const double scale = __longlong_as_double((long long)(1023 + 127 - (int)byte) << 52);
        code = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) code |= code_of(d[j] * scale) << (4 * j);
      }
    }
    const uint32_t word = word_of(in ? byte : 0u, lane);
    if (in) *reinterpret_cast<uint32_t*>(codes + row * (n / 2) + (int64_t)c * 4) = byte == 255u ? 0u : code;
    if (in && (lane & 15) == 0) *reinterpret_cast<uint32_t*>(scales + scale_word(row, c >> 4, ktiles)) = word;
  }
}

template <typename T>
static int launch_norm(void* codes, void* scales, void* sum, const void* x, const void* res, const void* w, int64_t rows,
                       int64_t n, int64_t xs, int64_t rs, int64_t ss, float eps, cudaStream_t st) {
  const int64_t chunks = n / 8;
#define NORM(V)                                                                                                                \
  {                                                                                                                            \
    const int threads = (int)(cdiv64(cdiv64(chunks, V), 32) * 32);                                                             \
    b2l_launch(norm_quantize_kernel<T, V>, dim3((unsigned)rows), dim3(threads), (size_t)0, st, (uint8_t*)codes, (uint8_t*)scales, \
               (T*)sum, (const T*)x, (const T*)res, (const T*)w, n, xs, rs, ss, k_tiles(n), eps);                               \
  }
  if (chunks <= 512) NORM(1)
  else if (chunks <= 1024) NORM(2)
  else NORM(4)
#undef NORM
  B2L_LAUNCH_CHECK();
  return B2L_OK;
}

}  // namespace mx4

extern "C" int64_t b2l_mxfp4_scale_bytes(int64_t rows, int64_t k) {
  return rows <= 0 || k <= 0 ? 0 : cdiv64(rows, 128) * mx4::k_tiles(k) * mx4::kTileBytes;
}

extern "C" int b2l_mxfp4_quantize(void* codes, void* scales, const void* x, int64_t matrices, int64_t rows, int64_t k,
                                  int64_t x_row_stride, int dtype, void* stream) {
  B2L_REQUIRE(matrices >= 0 && rows >= 0 && k > 0 && k % 32 == 0 && k < (1ll << 31), "mxfp4_quantize: %lld rows of %lld (a multiple of 32)",
              (long long)rows, (long long)k);
  const int64_t all = matrices * rows;
  if (all == 0) return B2L_OK;
  B2L_REQUIRE(codes && scales && x, "mxfp4_quantize: null pointer");
  const int esz = dtype == B2L_F32 ? 4 : 2;
  B2L_REQUIRE((uintptr_t)x % 16 == 0 && x_row_stride * esz % 16 == 0 && (uintptr_t)codes % 4 == 0 && (uintptr_t)scales % 4 == 0,
              "mxfp4_quantize: rows must start on 16 bytes");
  const int units = (int)cdiv64(k, 256);
  const int64_t grid = cdiv64(all * units, mx4::kWarps);
  B2L_REQUIRE(grid < (1ll << 31), "mxfp4_quantize: too many rows");
  B2L_DISPATCH_FLOAT(dtype, "mxfp4_quantize", {
    b2l_launch(mx4::quantize_kernel<T>, dim3((unsigned)grid), dim3(mx4::kWarps * 32), (size_t)0, (cudaStream_t)stream,
               (uint8_t*)codes, (uint8_t*)scales, (const T*)x, all, rows, k, x_row_stride, mx4::k_tiles(k), units);
  });
  B2L_LAUNCH_CHECK();
  return B2L_OK;
}

extern "C" int b2l_mxfp4_dequantize(void* y, const void* codes, const void* scales, int64_t matrices, int64_t rows, int64_t k,
                                    int64_t codes_row_stride, int dtype, void* stream) {
  B2L_REQUIRE(matrices >= 0 && rows >= 0 && k > 0 && k % 32 == 0 && k < (1ll << 31), "mxfp4_dequantize: %lld rows of %lld (a multiple of 32)",
              (long long)rows, (long long)k);
  const int64_t all = matrices * rows;
  if (all == 0) return B2L_OK;
  B2L_REQUIRE(y && codes && scales, "mxfp4_dequantize: null pointer");
  B2L_REQUIRE((uintptr_t)y % 16 == 0 && (uintptr_t)codes % 4 == 0 && codes_row_stride % 4 == 0 && (uintptr_t)scales % 4 == 0,
              "mxfp4_dequantize: misaligned rows");
  const int units = (int)cdiv64(k, 256);
  const int64_t grid = cdiv64(all * units, mx4::kWarps);
  B2L_REQUIRE(grid < (1ll << 31), "mxfp4_dequantize: too many rows");
  B2L_DISPATCH_FLOAT(dtype, "mxfp4_dequantize", {
    b2l_launch(mx4::dequantize_kernel<T>, dim3((unsigned)grid), dim3(mx4::kWarps * 32), (size_t)0, (cudaStream_t)stream, (T*)y,
               (const uint8_t*)codes, (const uint8_t*)scales, all, rows, k, codes_row_stride, mx4::k_tiles(k), units);
  });
  B2L_LAUNCH_CHECK();
  return B2L_OK;
}

extern "C" int b2l_skip_rmsnorm_mxfp4(void* codes, void* scales, void* sum, const void* x, const void* residual,
                                      const void* weight, int64_t rows, int64_t n, int64_t x_row_stride, int64_t r_row_stride,
                                      int64_t s_row_stride, float eps, int dtype, void* stream) {
  B2L_REQUIRE(rows >= 0 && rows < (1ll << 31) && n > 0 && n % 32 == 0 && n <= 16384,
              "skip_rmsnorm_mxfp4: %lld rows of %lld (a multiple of 32, at most 16384)", (long long)rows, (long long)n);
  if (rows == 0) return B2L_OK;
  B2L_REQUIRE(codes && scales && x && weight && (!residual || sum), "skip_rmsnorm_mxfp4: null pointer");
  B2L_REQUIRE(((uintptr_t)x | (uintptr_t)residual | (uintptr_t)sum | (uintptr_t)weight) % 16 == 0 &&
                  (x_row_stride | r_row_stride | s_row_stride) % 8 == 0 && (uintptr_t)codes % 4 == 0 && (uintptr_t)scales % 4 == 0,
              "skip_rmsnorm_mxfp4: rows must start on 16 bytes");
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == B2L_F16)
    return mx4::launch_norm<__half>(codes, scales, sum, x, residual, weight, rows, n, x_row_stride, r_row_stride, s_row_stride, eps, st);
  if (dtype == B2L_BF16)
    return mx4::launch_norm<__nv_bfloat16>(codes, scales, sum, x, residual, weight, rows, n, x_row_stride, r_row_stride, s_row_stride, eps, st);
  B2L_UNSUPPORTED("skip_rmsnorm_mxfp4: dtype %d", dtype);
}
