// 16-bit (or 32-bit) rows to microscaled 4-bit floating point and back, by themselves and behind a residual add and RMS norm.
// Format and layout: mxfp4.cuh.  All three are bound by memory on large inputs and by launch latency on a decode step.
#include "mxfp4.cuh"

namespace mx4 {

constexpr int kWarps = 8;

// A warp takes U x 256 consecutive elements of a row and asks for all of them before it uses the first: 16 bytes a lane (512 a warp) in,
// four bytes a lane out, and a scale byte per four lanes.  Rows are `per` to a matrix; a matrix starts on a tile of scales of its own.
template <typename T, int U>
__global__ void __launch_bounds__(kWarps * 32)
quantize_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, const T* __restrict__ x, uint32_t rows, uint32_t per,
                uint32_t k, int64_t x_stride, int64_t ktiles, uint32_t units) {
  pdl_prologue();
  const int lane = threadIdx.x & 31;
  const uint32_t u = blockIdx.x * kWarps + (threadIdx.x >> 5), row = u / units;
  if (row >= rows) return;                             // whole warps
  const uint32_t first = (u - row * units) * (32 * U) + lane, chunks = k / 8;      // chunks of eight elements
  const T* src = x + row * x_stride + (int64_t)first * 8;
  Raw8<T> v[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    zero_raw(v[i]);
    if (first + 32 * i < chunks) load_raw(src + 256 * i, v[i]);
  }
  const uint32_t matrix = row / per;
  const int64_t padded = (int64_t)matrix * ((per + 127) / 128 * 128) + (row - matrix * per);
  uint8_t* out = codes + (int64_t)row * (k / 2) + first * 4;
  uint8_t* scale = scales + scale_word(padded, (int)(first >> 4), ktiles) + ((first >> 2) & 3);
  const uint32_t behind = (chunks + 15) & ~15u;        // blocks up to here are filled up with zeros
#pragma unroll
  for (int i = 0; i < U; ++i) {
    uint32_t byte;                                     // of a block behind the end: 0
    const uint32_t code = quantise_raw(v[i], byte);
    if (first + 32 * i < chunks) *reinterpret_cast<uint32_t*>(out + 128 * i) = code;
    if ((lane & 3) == 0 && first + 32 * i < behind) scale[2 * kTileBytes * i] = (uint8_t)byte;
  }
}

// Eight codes and their block's scale byte -> eight values, rounded once
template <typename T> __device__ __forceinline__ uint4 values8(uint32_t c, uint32_t byte) {
  uint32_t o[4];
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    // The elements' bf16 bits from two tables of eight bytes; the scale is a bf16 for every byte.
    const uint32_t s = byte == 0u ? 0x00400040u : (byte == 255u ? 0x7fc07fc0u : byte * 0x00800080u);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t q = (c >> (16 * h)) & 0xffffu, index = q & 0x7777u;
      const uint32_t high = __byte_perm(0x3f3f3f00u, 0x40404040u, index), low = __byte_perm(0xc0800000u, 0xc0804000u, index);
      const uint32_t a = __byte_perm(low, high, 0x5140) | ((q << 12) & 0x8000u) | ((q << 24) & 0x80000000u);
      const uint32_t b = __byte_perm(low, high, 0x7362) | ((q << 4) & 0x8000u) | ((q << 16) & 0x80000000u);
      const __nv_bfloat162 s2 = *reinterpret_cast<const __nv_bfloat162*>(&s);
      const __nv_bfloat162 y0 = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), s2), y1 = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&b), s2);
      o[2 * h] = *reinterpret_cast<const uint32_t*>(&y0);
      o[2 * h + 1] = *reinterpret_cast<const uint32_t*>(&y1);
    }
  } else {
    float t[8];
    elements8(c, t);
    const float s = scale_value(byte);
    const f32x2 s2 = pair_of(s, s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 y = mul2(pair_of(t[2 * i], t[2 * i + 1]), s2);
      o[i] = pack2<__half>(first_of(y), second_of(y));
    }
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// The same cut; a lane reads four bytes of codes and its block's byte and writes eight values.
template <typename T, int U>
__global__ void __launch_bounds__(kWarps * 32)
dequantize_kernel(T* __restrict__ y, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, uint32_t rows, uint32_t per,
                  uint32_t k, int64_t codes_stride, int64_t ktiles, uint32_t units) {
  pdl_prologue();
  const int lane = threadIdx.x & 31;
  const uint32_t u = blockIdx.x * kWarps + (threadIdx.x >> 5), row = u / units;
  if (row >= rows) return;
  const uint32_t first = (u - row * units) * (32 * U) + lane, chunks = k / 8;
  const uint32_t matrix = row / per;
  const int64_t padded = (int64_t)matrix * ((per + 127) / 128 * 128) + (row - matrix * per);
  const uint8_t* src = codes + row * codes_stride + first * 4;
  const uint8_t* scale = scales + scale_word(padded, (int)(first >> 4), ktiles) + ((first >> 2) & 3);
  T* out = y + (int64_t)row * k + (int64_t)first * 8;
  uint32_t q[U], b[U];
#pragma unroll
  for (int i = 0; i < U; ++i)
    if (first + 32 * i < chunks) {
      q[i] = ld_once(src + 128 * i);
      b[i] = scale[2 * kTileBytes * i];
    }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if (first + 32 * i >= chunks) break;
    if constexpr (sizeof(T) == 4) {
      float t[8];
      elements8(q[i], t);
      const float s = scale_value(b[i]);
#pragma unroll
      for (int j = 0; j < 8; j += 4)
        stg_128(out + 256 * i + j, make_uint4(__float_as_uint(t[j] * s), __float_as_uint(t[j + 1] * s), __float_as_uint(t[j + 2] * s),
                                              __float_as_uint(t[j + 3] * s)));
    } else {
      stg_128(out + 256 * i, values8<T>(q[i], b[i]));
    }
  }
}

// Units of 256 elements to a warp: one where there are few, for latency, else four (quantiser / reader, one -> four, us: 32 x 4096 1.31 / 1.33 ->
// 1.70 / 1.59; 256 x 4096 2.1 / 2.1 -> 2.0 / 1.7; 1000 x 4096 3.7 / 3.5 -> 3.4 / 3.2; 4000 x 4096 12.2 / 10.6 -> 7.8 / 6.6).
static int units_of(int64_t rows, int64_t k) { return rows * cdiv64(k, 256) < 24LL * b2l_num_sms() ? 1 : 4; }

// ---------------------------------------------------------------------------------------------------------------
// s = x + r (stored over r, or to `sum`, in the activations' type), y = s / sqrt(mean s^2 + eps) * w, quantised.
//
// y is not rounded to 16 bits on the way: the 16-bit norm would round it twice (before and behind the weight), and elements that
// lie next to a border would then go by those roundings.  The sum of squares is in 64 bits, y in 32, four roundings of 2^-24.  A value that
// lies within 2^-21 of a border, or a largest magnitude that near to a power of two, is decided in 64 bits: the warp computes the blocks
// in question again (one element in 10^5), so the codes are those of exact arithmetic.
// Bound: latency; counters at 1999 x 3584: issue 54 %, resident warps 38 % (64 registers), DRAM 22 %, and all of a block waits at the row's sum.
// eps comes in 32 bits.  1999 x 3584, us with the reader behind it: 25.8 with all in 64 bits and integer maxima, 20.8 with the sum in 32 bits,
// wider margins and rows with a doubtful block added up again by their CTA, 18.5 so; 17.8 without any decision in 64 bits.
// Two chunks a thread 18.5, four 19.0, one 22.3.
// ---------------------------------------------------------------------------------------------------------------
template <typename T, int VPT>
__global__ void __launch_bounds__(512, 2)
norm_quantize_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, T* sum, const T* x, const T* res,      // sum: may be x or res
                     const T* __restrict__ w, int n, int64_t x_stride, int64_t r_stride, int64_t s_stride, int64_t ktiles, double inv_n,
                     float eps) {
  pdl_prologue();
  const int64_t row = blockIdx.x;
  const int chunks = n / 8, lane = threadIdx.x & 31;
  x += row * x_stride;
  res = res ? res + row * r_stride : nullptr;
  f32x2 s[VPT][4];
  double sq = 0.0;
  uint4 xv[VPT], rv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    xv[i] = rv[i] = make_uint4(0u, 0u, 0u, 0u);
    if (c < chunks) {
      xv[i] = ldg_128(x + c * 8);
      if (res) rv[i] = ldg_128(res + c * 8);
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x2 a = widen<T>(reinterpret_cast<const uint32_t*>(&xv[i])[j]), b = widen<T>(reinterpret_cast<const uint32_t*>(&rv[i])[j]);
      s[i][j] = add2(a, b);
      const double p = (double)first_of(a) + (double)first_of(b), q = (double)second_of(a) + (double)second_of(b);
      sq = fma(q, q, fma(p, p, sq));
    }
  __shared__ double wide[16];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
  if (lane == 0) wide[threadIdx.x >> 5] = sq;
  __syncthreads();
  double all = 0.0;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) all += wide[i];
  const double root = rsqrt(fma(all, inv_n, (double)eps));
  const float rrms = (float)root;
  const f32x2 r2 = pair_of(rrms, rrms), below = pair_of(-0x1p-21f, -0x1p-21f), above = pair_of(0x1p-21f, 0x1p-21f);
  const uint32_t behind = ((uint32_t)chunks + 15u) & ~15u;
  uint32_t near = 0;                   // chunks that 64 bits decide
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (c - lane >= chunks) break;                     // whole warps
    const bool in = c < chunks;
    uint4 wv = make_uint4(0u, 0u, 0u, 0u);
    if (in) wv = ldg_128(w + c * 8);
    f32x2 v[4];
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = mul2(mul2(s[i][j], r2), widen<T>(reinterpret_cast<const uint32_t*>(&wv)[j]));
      m = max_abs(m, first_of(v[j]), second_of(v[j]));
    }
    m = max_abs(m, __shfl_xor_sync(0xffffffffu, m, 1), 0.f);
    m = max_abs(m, __shfl_xor_sync(0xffffffffu, m, 2), 0.f);
    const uint32_t top = __float_as_uint(m) & 0x7fffffffu, byte = scale_byte(top);
    const float inv = inverse_scale(byte);
    const f32x2 inv2 = pair_of(inv, inv);
    f32x2 end[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = mul2(v[j], inv2);
      end[j] = fma2(v[j], below, v[j]);
    }
    const uint32_t code = codes8(end);
#pragma unroll
    for (int j = 0; j < 4; ++j) end[j] = fma2(v[j], above, v[j]);
    // next to a border, the largest next to a power of two (4 steps of 2^-23), or so small that 32 bits lose digits
    const bool unsure = byte != 255u && (code != codes8(end) || ((top - 4u) ^ (top + 4u)) >> 23 != 0u || top < 0x0d000000u) && top != 0u;
    const uint32_t group = __ballot_sync(0xffffffffu, unsure) >> (lane & 28) & 15u;      // of the block's four lanes
    near |= (group != 0u ? 1u : 0u) << i;
    if (in) *reinterpret_cast<uint32_t*>(codes + row * (n / 2) + c * 4) = byte == 255u ? 0u : code;
    if ((lane & 3) == 0 && (uint32_t)c < behind) scales[scale_word(row, c >> 4, ktiles) + ((c >> 2) & 3)] = (uint8_t)byte;
  }
  if (__any_sync(0xffffffffu, (int)near)) {
    __syncwarp();                      // behind the stores above
    // again in 64 bits, from memory (a thread's own chunks, whose sums are stored below); blocks that were sure keep their codes
#pragma unroll 1
    for (int i = 0; i < VPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c - lane >= chunks || __ballot_sync(0xffffffffu, (near >> i) & 1u) == 0u) continue;      // whole warps
      auto exact = [&](int j) {
        return c >= chunks ? 0.0 : ((double)to_f32(x[c * 8 + j]) + (res ? (double)to_f32(res[c * 8 + j]) : 0.0)) * root * (double)to_f32(w[c * 8 + j]);
      };
      double top = 0.0;
      for (int j = 0; j < 8; ++j) top = fmax(top, fabs(exact(j)));
      top = fmax(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmax(top, __shfl_xor_sync(0xffffffffu, top, 2));
      if ((near >> i) & 1u) {
        const uint32_t byte = scale_byte(top);
        const double scale = inverse_scale_64(byte);
        uint32_t code = 0;
        if (byte != 255u)
          for (int j = 0; j < 8; ++j) code |= code_of(exact(j) * scale) << (4 * j);
        *reinterpret_cast<uint32_t*>(codes + row * (n / 2) + c * 4) = code;
        if ((lane & 3) == 0) scales[scale_word(row, c >> 4, ktiles) + ((c >> 2) & 3)] = (uint8_t)byte;
      }
    }
  }
  if (res) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < chunks)
        stg_128(sum + row * s_stride + c * 8, make_uint4(pack2<T>(first_of(s[i][0]), second_of(s[i][0])), pack2<T>(first_of(s[i][1]), second_of(s[i][1])),
                                                         pack2<T>(first_of(s[i][2]), second_of(s[i][2])), pack2<T>(first_of(s[i][3]), second_of(s[i][3]))));
    }
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
               (T*)sum, (const T*)x, (const T*)res, (const T*)w, (int)n, xs, rs, ss, k_tiles(n), 1.0 / (double)n, eps);               \
  }
  // many rows are read by fewer threads each, so that more of them are in flight (one -> two chunks a thread, us: 32 x 4096 2.6 -> 2.9, 400 x
  // 4096 4.9 -> 5.2, 800 x 4096 7.7 -> 7.0, 1999 x 3584 with the reader 22.3 -> 18.5)
  const bool many = rows > 4LL * b2l_num_sms();
  if (chunks <= 512 && !many) NORM(1)
  else if (chunks <= 1024) NORM(2)
  else NORM(4)
#undef NORM
  B2L_LAUNCH_CHECK();
  return B2L_OK;
}

// Whether sums may be written while rows of `in` are read: each over its own row, or where no row lies.  Strides in bytes, rows of `bytes`.
static bool writable(const void* sum, int64_t s_stride, const void* in, int64_t stride, int64_t rows, int64_t bytes) {
  if (!in || rows == 0) return true;
  if (rows == 1) stride = s_stride = bytes;
  if (sum == in && stride == s_stride) return true;
  int64_t s = (int64_t)(intptr_t)sum, x = (int64_t)(intptr_t)in;
  const int64_t end = s + (rows - 1) * s_stride + bytes;
  if (stride < 0) {
    x += (rows - 1) * stride;
    stride = -stride;
  }
  int64_t row = 0;                     // the first that ends behind the sums' start
  if (x + bytes <= s) row = stride == 0 ? rows : (s - x - bytes) / stride + 1;
  return row >= rows || x + row * stride >= end;
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
  const int per_warp = mx4::units_of(all, k);
  const int64_t units = cdiv64(k, 256 * per_warp);
  B2L_REQUIRE(all * units < (1ll << 31), "mxfp4_quantize: too many rows");
  const dim3 grid((unsigned)cdiv64(all * units, mx4::kWarps));
  B2L_DISPATCH_FLOAT(dtype, "mxfp4_quantize", {
    b2l_launch(per_warp == 1 ? mx4::quantize_kernel<T, 1> : mx4::quantize_kernel<T, 4>, grid, dim3(mx4::kWarps * 32), (size_t)0,
               (cudaStream_t)stream, (uint8_t*)codes, (uint8_t*)scales, (const T*)x, (uint32_t)all, (uint32_t)rows, (uint32_t)k,
               x_row_stride, mx4::k_tiles(k), (uint32_t)units);
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
  const int per_warp = mx4::units_of(all, k);
  const int64_t units = cdiv64(k, 256 * per_warp);
  B2L_REQUIRE(all * units < (1ll << 31), "mxfp4_dequantize: too many rows");
  const dim3 grid((unsigned)cdiv64(all * units, mx4::kWarps));
  B2L_DISPATCH_FLOAT(dtype, "mxfp4_dequantize", {
    b2l_launch(per_warp == 1 ? mx4::dequantize_kernel<T, 1> : mx4::dequantize_kernel<T, 4>, grid, dim3(mx4::kWarps * 32), (size_t)0,
               (cudaStream_t)stream, (T*)y, (const uint8_t*)codes, (const uint8_t*)scales, (uint32_t)all, (uint32_t)rows, (uint32_t)k,
               codes_row_stride, mx4::k_tiles(k), (uint32_t)units);
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
  if (residual) {
    B2L_REQUIRE(s_row_stride >= n || rows == 1, "skip_rmsnorm_mxfp4: the sums' rows overlap");
    B2L_REQUIRE(mx4::writable(sum, 2 * s_row_stride, x, 2 * x_row_stride, rows, 2 * n) &&
                    mx4::writable(sum, 2 * s_row_stride, residual, 2 * r_row_stride, rows, 2 * n),
                "skip_rmsnorm_mxfp4: the sums overlap other rows than their own of what is read");
  }
  if (dtype != B2L_F16 && dtype != B2L_BF16) B2L_UNSUPPORTED("skip_rmsnorm_mxfp4: dtype %d", dtype);
  B2L_REQUIRE(!residual || (const char*)weight + 2 * n <= (const char*)sum ||
                  (const char*)sum + 2 * ((rows == 1 ? 0 : (rows - 1) * s_row_stride) + n) <= (const char*)weight,
              "skip_rmsnorm_mxfp4: the sums overlap the weight");
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == B2L_F16)
    return mx4::launch_norm<__half>(codes, scales, sum, x, residual, weight, rows, n, x_row_stride, r_row_stride, s_row_stride, eps, st);
  return mx4::launch_norm<__nv_bfloat16>(codes, scales, sum, x, residual, weight, rows, n, x_row_stride, r_row_stride, s_row_stride, eps, st);
}
