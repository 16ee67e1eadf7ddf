// The 4-bit cache's writer (rotary positions on q and k, K and V rounded to codes and stored at their tokens' rows, one launch) and
// its reader.
//
// A group's minimum is one of its elements and stored as it is; scale = (maximum - minimum) / 15, rounded to the activations' type;
// the codes are chosen against the ROUNDED scale: code = (x - minimum) / scale, to nearest (ties to even), at most 15.  An element
// comes back within half a step, plus what the rounding of the scale leaves of the 15 steps.
// Bound by memory in prompts (each element is read and stored once) and by one trip to memory and back in a decode step.
#include "kv_int4.cuh"
#include <type_traits>

namespace {

struct WriteParams {
  const void *q, *k, *v, *cos, *sin;
  void *q_out, *k_out;
  uint8_t* cache;
  const void* index;
  int index_w;
  int64_t row_stride, max_tokens;
  int seq_len, n_qh, n_kh;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, cs_b, cs_s, qo_ts, qo_hs, ko_ts, ko_hs;
};

template <typename T> struct Ext;                // minimum and maximum of pairs; a NaN stays
template <> struct Ext<__half> {
  using T2 = __half2;
  static __device__ T2 lo(T2 a, T2 b) { return __hmin2_nan(a, b); }
  static __device__ T2 hi(T2 a, T2 b) { return __hmax2_nan(a, b); }
  static __device__ float2 f2(T2 a) { return __half22float2(a); }
};
template <> struct Ext<__nv_bfloat16> {
  using T2 = __nv_bfloat162;
  static __device__ T2 lo(T2 a, T2 b) { return __hmin2_nan(a, b); }
  static __device__ T2 hi(T2 a, T2 b) { return __hmax2_nan(a, b); }
  static __device__ float2 f2(T2 a) { return __bfloat1622float2(a); }
};
template <typename T2> __device__ __forceinline__ uint32_t bits(T2 v) { return *reinterpret_cast<uint32_t*>(&v); }
template <typename T2> __device__ __forceinline__ T2 as_pair(uint32_t v) { return *reinterpret_cast<T2*>(&v); }

template <typename T, bool VEC>
__device__ __forceinline__ void load8(uint32_t (&w)[4], const T* p) {
  if (VEC) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const uint32_t (&w)[4]) {
  if (VEC) {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    uint16_t* h = reinterpret_cast<uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) { h[2 * i] = (uint16_t)w[i]; h[2 * i + 1] = (uint16_t)(w[i] >> 16); }
  }
}

// (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin) in 32 bits, rounded once
template <typename T>
__device__ __forceinline__ void rotate(uint32_t (&a)[4], uint32_t (&b)[4], const uint32_t (&cv)[4], const uint32_t (&sv)[4]) {
  using T2 = typename Ext<T>::T2;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = Ext<T>::f2(as_pair<T2>(a[i])), y = Ext<T>::f2(as_pair<T2>(b[i]));
    const float2 c = Ext<T>::f2(as_pair<T2>(cv[i])), s = Ext<T>::f2(as_pair<T2>(sv[i]));
    a[i] = pack2<T>(x.x * c.x - y.x * s.x, x.y * c.y - y.y * s.y);
    b[i] = pack2<T>(y.x * c.x + x.x * s.x, y.y * c.y + x.y * s.y);
  }
}

// A group's stored (scale, minimum), and what turns an element into its code.  Differences and quotients are taken of values divided
// by 16, which is exact, so that no range of bf16 values overflows.
template <typename T>
struct Grid {
  uint32_t stored;
  float lo16, step16, inv;
  int way;                                        // 0 codes are zero, 1 by the reciprocal, 2 by division (steps near the ends of the range; one that was
                                                  // rounded to few bits may lead past 15, else 15.06 is the most)
  __device__ __forceinline__ void from(float lo, float hi) {
    lo16 = lo * 0.0625f;
    const float range16 = hi * 0.0625f - lo16;
    if (!(range16 < INFINITY)) {                  // an infinity or a NaN in the group: it reads as NaN
      const float nan = __int_as_float(0x7fc00000);
      stored = pack2<T>(nan, nan);
      way = 0;
      return;
    }
    stored = pack2<T>(__fdiv_rn(range16, 0.9375f), lo);
    step16 = kv4::scale_min<T>(stored).x * 0.0625f;
    way = step16 == 0.f ? 0 : step16 > (std::is_same<T, __half>::value ? 0x1p-18f : 1e-30f) && step16 < 1e30f ? 1 : 2;
    inv = __frcp_rn(step16);
  }
  // Quotient by the correctly rounded reciprocal and one correction with the remainder, which gives the correctly rounded quotient
  // (Markstein, IBM J. Res. Dev. 34, 1990): a difference of exactly half a step, which one value in some thousands of a 16-bit type
  // is, then goes to the even code as in exact arithmetic.
  __device__ __forceinline__ uint32_t code(float x) const {
    const float t = fmaf(x, 0.0625f, -lo16);
    float c;
    if (way == 1) {
      c = t * inv;
      c = fmaf(fmaf(-c, step16, t), inv, c);
    } else {
      c = way == 0 ? 0.f : fminf(__fdiv_rn(t, step16), 15.f);
    }
    const float near = c + 12582912.f;                           // 1.5 * 2^23: the sum's last bits are the nearest whole number
    uint32_t code = __float_as_uint(near);
    if (fabsf(c - (near - 12582912.f)) == 0.5f) {
      // Half a step of the difference that 32 bits hold.  What they do not (of an element some 2^13 times smaller than the minimum, or the
      // other way round) decides.
      const float x16 = x * 0.0625f, part = t + lo16, rest = (x16 - part) - (lo16 - (part - t));
      if (rest != 0.f) code = (uint32_t)(c + (rest > 0.f ? 0.5f : -0.5f));
    }
    return code & 15u;
  }
  __device__ __forceinline__ uint32_t codes(const uint32_t (&w)[4]) const {
    using T2 = typename Ext<T>::T2;
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = Ext<T>::f2(as_pair<T2>(w[i]));
      r |= code(x.x) << (8 * i) | code(x.y) << (8 * i + 4);
    }
    return r;
  }
};

// A thread holds eight elements of a head's lower half and the eight that rotate with them of its upper half; a head's threads are
// neighbours in a warp and find their groups' ends with one to four shuffles.  All of a token's heads -- q rotated, k rotated and
// stored, v stored -- are units of one grid: a decode step is one trip through L2, not one per head.  (8000 tokens of 28 + 4 + 4 heads of
// 128, bf16, 147 MB: blocks of 96 threads 29 us, of 288, a token's all heads, 33, with two tokens to a thread 42; deciding half steps exactly 2 more.)
template <typename T, int D, int GS, bool VEC>
__global__ void __launch_bounds__(128) kv4_write_kernel(const WriteParams p) {
  pdl_prologue();
  using X = Ext<T>;
  using T2 = typename X::T2;
  constexpr int HALF = D / 2, UNITS = HALF / 8;
  constexpr int NG = D / GS, LANES = (GS < HALF ? GS : HALF) / 8;   // threads that share a group of one half
  const int i = blockIdx.y * blockDim.x + threadIdx.x;
  const int h = i / UNITS, c = (i % UNITS) * 8;
  const bool is_q = h < p.n_qh, is_v = h >= p.n_qh + p.n_kh;
  const int hk = is_v ? h - p.n_qh - p.n_kh : h - p.n_qh;
  if (h >= p.n_qh + 2 * p.n_kh) return;             // a head's threads leave together; a warp's heads need not
  const T* src = is_q ? (const T*)p.q + (int64_t)h * p.q_hs : is_v ? (const T*)p.v + (int64_t)hk * p.v_hs : (const T*)p.k + (int64_t)hk * p.k_hs;
  const int64_t ts = is_q ? p.q_ts : is_v ? p.v_ts : p.k_ts;
  const bool turn = !is_v && p.cos != nullptr;
  const int64_t tok = blockIdx.x;
  uint32_t a[4], b[4];
  int64_t row = -1;
  load8<T, VEC>(a, src + tok * ts + c);
  load8<T, VEC>(b, src + tok * ts + c + HALF);
  if (!is_q) row = load_index(p.index, tok, p.index_w);
  if (turn) {
    uint32_t cv[4], sv[4];
    const int64_t at = p.seq_len == 1 ? tok : blockIdx.x / (unsigned)p.seq_len;
    const int64_t cs = at * p.cs_b + (tok - at * p.seq_len) * p.cs_s + c;
    load8<T, VEC>(cv, (const T*)p.cos + cs);
    load8<T, VEC>(sv, (const T*)p.sin + cs);
    rotate<T>(a, b, cv, sv);
    T* dst = is_q ? (T*)p.q_out + tok * p.qo_ts + (int64_t)h * p.qo_hs : (T*)p.k_out + tok * p.ko_ts + (int64_t)hk * p.ko_hs;
    if (is_q || p.k_out != nullptr) {
      store8<T, VEC>(dst + c, a);
      store8<T, VEC>(dst + c + HALF, b);
    }
  }
  if (is_q) return;
  // ends of this thread's group in either half (one group over both: of both)
  T2 lo_a = as_pair<T2>(a[0]), hi_a = lo_a, lo_b = as_pair<T2>(b[0]), hi_b = lo_b;
#pragma unroll
  for (int j = 1; j < 4; ++j) {
    lo_a = X::lo(lo_a, as_pair<T2>(a[j])); hi_a = X::hi(hi_a, as_pair<T2>(a[j]));
    lo_b = X::lo(lo_b, as_pair<T2>(b[j])); hi_b = X::hi(hi_b, as_pair<T2>(b[j]));
  }
  if (GS == D) { lo_a = lo_b = X::lo(lo_a, lo_b); hi_a = hi_b = X::hi(hi_a, hi_b); }
  // the head's threads: other heads of the warp may have left or be queries
  const unsigned mine = UNITS == 32 ? 0xffffffffu : ((1u << UNITS) - 1u) << ((threadIdx.x & 31) / UNITS * UNITS);
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) {
    lo_a = X::lo(lo_a, as_pair<T2>(__shfl_xor_sync(mine, bits(lo_a), o)));
    hi_a = X::hi(hi_a, as_pair<T2>(__shfl_xor_sync(mine, bits(hi_a), o)));
    lo_b = X::lo(lo_b, as_pair<T2>(__shfl_xor_sync(mine, bits(lo_b), o)));
    hi_b = X::hi(hi_b, as_pair<T2>(__shfl_xor_sync(mine, bits(hi_b), o)));
  }
  if (row < 0 || row >= p.max_tokens) return;   // a padded token has no row
  auto low = [](T2 v) { const float2 f = X::f2(v); return f.x != f.x || f.x < f.y ? f.x : f.y; };
  auto high = [](T2 v) { const float2 f = X::f2(v); return f.x != f.x || f.x > f.y ? f.x : f.y; };
  Grid<T> ga, gb;
  ga.from(low(lo_a), high(hi_a));
  if (GS == D) gb = ga;
  else gb.from(low(lo_b), high(hi_b));
  uint8_t* head = p.cache + row * p.row_stride + (int64_t)hk * kv4::head_bytes(D, GS);
  uint32_t* codes = reinterpret_cast<uint32_t*>(head + (is_v ? D / 2 : 0));
  codes[c / 8] = ga.codes(a);
  codes[(c + HALF) / 8] = gb.codes(b);
  if (c % GS == 0) {
    uint32_t* groups = reinterpret_cast<uint32_t*>(head + D) + (is_v ? NG : 0);
    groups[c / GS] = ga.stored;
    if (GS != D) groups[(c + HALF) / GS] = gb.stored;
  }
}

// Eight elements and R tokens a thread.
template <typename T, int D, int GS, int R>
__global__ void __launch_bounds__(256) kv4_read_kernel(T* out, const uint8_t* cache, const void* index, int index_w, int n_kh,
                                                       int64_t row_stride, int64_t max_tokens, int64_t tokens) {
  pdl_prologue();
  constexpr int NG = D / GS, UNITS = D / 8;
  const int i = blockIdx.y * blockDim.x + threadIdx.x, h = i / UNITS, c = i % UNITS;
  if (h >= 2 * n_kh) return;
  const bool is_v = h >= n_kh;
  int64_t row[R];
  uint32_t w[R], g[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t tok = (int64_t)blockIdx.x * R + r;
    row[r] = tok < tokens ? load_index(index, tok, index_w) : -1;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    w[r] = g[r] = 0u;
    if (row[r] < 0 || row[r] >= max_tokens) continue;   // zeros
    const uint8_t* head = cache + row[r] * row_stride + (int64_t)(is_v ? h - n_kh : h) * kv4::head_bytes(D, GS);
    w[r] = reinterpret_cast<const uint32_t*>(head + (is_v ? D / 2 : 0))[c];
    g[r] = reinterpret_cast<const uint32_t*>(head + D)[(is_v ? NG : 0) + c * 8 / GS];
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t tok = (int64_t)blockIdx.x * R + r;
    if (tok >= tokens) break;
    const float2 sm = kv4::scale_min<T>(g[r]);
    // 15 rounded steps may end above the type's largest number, which the group's maximum then was: no infinity (a NaN stays)
    constexpr float kMost = std::is_same<T, __half>::value ? 65504.f : 3.38953139e38f;
    auto one = [&](int at) {
      const float x = fmaf((float)(w[r] >> at & 15u), sm.x, sm.y);
      return x > kMost ? kMost : x;
    };
    auto two = [&](int at) { return pack2<T>(one(at), one(at + 4)); };
    reinterpret_cast<uint4*>(out)[(tok * 2 * n_kh + h) * UNITS + c] = make_uint4(two(0), two(8), two(16), two(24));
  }
}

// blocks of whole warps that share `units` threads evenly
struct Blocks { unsigned parts, threads; };
Blocks blocks_of(int64_t units, int most) {
  const int64_t parts = cdiv64(units, most);
  return {(unsigned)parts, (unsigned)(cdiv64(cdiv64(units, parts), 32) * 32)};
}

int check_cache(const char* what, const void* cache, int64_t row_stride, int64_t max_tokens, int n_kh, int head_dim, int group) {
  B2L_REQUIRE(kv4::shape_ok(head_dim, group), "%s: head_dim %d with groups of %d (head_dim 32, 64 or 128; groups of 32, 64 or 128, at most head_dim)",
              what, head_dim, group);
  B2L_REQUIRE(n_kh > 0 && max_tokens >= 0, "%s: bad shape", what);
  B2L_REQUIRE(row_stride >= kv4::row_bytes(n_kh, head_dim, group) && row_stride % 16 == 0 && (uintptr_t)cache % 16 == 0,
              "%s: cache rows must be 16-byte aligned and hold %lld bytes", what, (long long)kv4::row_bytes(n_kh, head_dim, group));
  return B2L_OK;
}

}  // namespace

extern "C" int64_t b2l_kv_int4_row_bytes(int num_kv_heads, int head_dim, int group) {
  return num_kv_heads > 0 && kv4::shape_ok(head_dim, group) ? kv4::row_bytes(num_kv_heads, head_dim, group) : 0;
}

extern "C" int b2l_kv_int4_write(void* q_out, void* k_out, const void* q, const void* k, const void* v, const void* cos, const void* sin,
                                 const void* select_index, int index_width, void* cache, int64_t cache_row_stride, int64_t max_tokens,
                                 int64_t tokens, int64_t seq_len, int n_qh, int n_kh, int head_dim, int group, int64_t q_tok_stride,
                                 int64_t q_head_stride, int64_t k_tok_stride, int64_t k_head_stride, int64_t v_tok_stride,
                                 int64_t v_head_stride, int64_t cs_batch_stride, int64_t cs_seq_stride, int64_t qo_tok_stride,
                                 int64_t qo_head_stride, int64_t ko_tok_stride, int64_t ko_head_stride, int dtype, void* stream) {
  B2L_REQUIRE(k && v && select_index && cache && (n_qh == 0 || (q && q_out)), "kv_int4_write: null pointer");
  B2L_REQUIRE(n_qh == 0 || (cos && sin), "kv_int4_write: query heads without positions");
  B2L_REQUIRE((cos == nullptr) == (sin == nullptr), "kv_int4_write: cos without sin");
  if (int rc = check_cache("kv_int4_write", cache, cache_row_stride, max_tokens, n_kh, head_dim, group)) return rc;
  B2L_REQUIRE(tokens >= 0 && n_qh >= 0 && seq_len > 0, "kv_int4_write: bad shape");
  B2L_REQUIRE(index_width == 4 || index_width == 8, "kv_int4_write: index width %d", index_width);
  B2L_REQUIRE(dtype == B2L_F16 || dtype == B2L_BF16, "kv_int4_write: dtype %d", dtype);
  B2L_REQUIRE(tokens < (1ll << 31) && seq_len < (1ll << 31), "kv_int4_write: too many tokens");
  if (tokens == 0) return B2L_OK;
  WriteParams p;
  p.q = q; p.k = k; p.v = v; p.cos = cos; p.sin = sin; p.q_out = q_out; p.k_out = k_out;
  p.cache = (uint8_t*)cache; p.index = select_index; p.index_w = index_width;
  p.row_stride = cache_row_stride; p.max_tokens = max_tokens;
  p.seq_len = (int)seq_len; p.n_qh = n_qh; p.n_kh = n_kh;
  p.q_ts = q_tok_stride; p.q_hs = q_head_stride; p.k_ts = k_tok_stride; p.k_hs = k_head_stride; p.v_ts = v_tok_stride;
  p.v_hs = v_head_stride; p.cs_b = cs_batch_stride; p.cs_s = cs_seq_stride; p.qo_ts = qo_tok_stride; p.qo_hs = qo_head_stride;
  p.ko_ts = ko_tok_stride; p.ko_hs = ko_head_stride;
  const int64_t strides[] = {q_tok_stride, q_head_stride, k_tok_stride, k_head_stride, v_tok_stride, v_head_stride, cs_batch_stride,
                             cs_seq_stride, qo_tok_stride, qo_head_stride, ko_tok_stride, ko_head_stride};
  bool vec = ((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)cos | (uintptr_t)sin | (uintptr_t)q_out | (uintptr_t)k_out) % 16 == 0;
  for (int64_t s : strides) vec = vec && s % 8 == 0;
  const Blocks bl = blocks_of(((int64_t)n_qh + 2 * (int64_t)n_kh) * (head_dim / 16), 128);
  B2L_REQUIRE(bl.parts <= 65535, "kv_int4_write: too many heads");
  const dim3 grid((unsigned)tokens, bl.parts);
  cudaStream_t st = (cudaStream_t)stream;
#define KV4_WRITE(TT)                                                                                   \
  KV4_DISPATCH_SHAPE(head_dim, group, {                                                                 \
    b2l_launch(vec ? kv4_write_kernel<TT, D, GS, true> : kv4_write_kernel<TT, D, GS, false>, grid, dim3(bl.threads), (size_t)0, st, p); \
  })
  if (dtype == B2L_F16) KV4_WRITE(__half);
  else KV4_WRITE(__nv_bfloat16);
#undef KV4_WRITE
  B2L_LAUNCH_CHECK();
  return B2L_OK;
}

extern "C" int b2l_kv_int4_read(void* out, const void* cache, int64_t cache_row_stride, int64_t max_tokens, const void* select_index,
                                int index_width, int64_t tokens, int n_kh, int head_dim, int group, int dtype, void* stream) {
  B2L_REQUIRE(out && cache && select_index, "kv_int4_read: null pointer");
  if (int rc = check_cache("kv_int4_read", cache, cache_row_stride, max_tokens, n_kh, head_dim, group)) return rc;
  B2L_REQUIRE(index_width == 4 || index_width == 8, "kv_int4_read: index width %d", index_width);
  B2L_REQUIRE(dtype == B2L_F16 || dtype == B2L_BF16, "kv_int4_read: dtype %d", dtype);
  B2L_REQUIRE(tokens >= 0 && tokens < (1ll << 31) && (uintptr_t)out % 16 == 0, "kv_int4_read: bad shape");
  if (tokens == 0) return B2L_OK;
  const Blocks bl = blocks_of(2 * (int64_t)n_kh * (head_dim / 8), 256);
  B2L_REQUIRE(bl.parts <= 65535, "kv_int4_read: too many heads");
  // Four tokens a thread, whose loads are on their way together, from eight blocks of one token to an SM on (one and four, us; 8 kv heads of 128:
  // 1000 tokens 2.3 and 3.0, 2000 3.7 and 4.0, 4000 5.9 and 5.3, 16000 23.8 and 16.4; 4 of 128: 1000 2.0 and 2.0, 4000 4.6 and 3.7; 2 of 64, blocks
  // of a warp, which start one after the other: 500 1.4 and 1.6, 1500 2.0 and 1.7, 8000 8.7 and 2.6).
  const bool four = tokens * bl.parts > 8ll * b2l_num_sms();
  const dim3 grid((unsigned)cdiv64(tokens, four ? 4 : 1), bl.parts);
  cudaStream_t st = (cudaStream_t)stream;
#define KV4_READ(TT)                                                                                                             \
  KV4_DISPATCH_SHAPE(head_dim, group, {                                                                                          \
    b2l_launch(four ? kv4_read_kernel<TT, D, GS, 4> : kv4_read_kernel<TT, D, GS, 1>, grid, dim3(bl.threads), (size_t)0, st, (TT*)out, \
               (const uint8_t*)cache, select_index, index_width, n_kh, cache_row_stride, max_tokens, tokens);                    \
  })
  if (dtype == B2L_F16) KV4_READ(__half);
  else KV4_READ(__nv_bfloat16);
#undef KV4_READ
  B2L_LAUNCH_CHECK();
  return B2L_OK;
}
