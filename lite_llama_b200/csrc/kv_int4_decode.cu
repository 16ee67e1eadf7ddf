// flash_decoding_int4: one query per sequence over a cache held in 4 bits (kv_int4.cuh).
//
//   out_h = sum_t softmax_t(scale q_h . k_t) v_t,   k_t = minimum + scale_t * code per group of elements (v_t too)
//
// Elements are not formed.  With codes c, q . k = sum over groups (s q . c + m sum(q)), so a key's scales meet the finished sums of
// its codes; and out = sum_t (p s) c + sum_t p m, so a value's scale is multiplied into the probability.  What is left of unpacking is
// a shift and a mask: four bits inside a half's fraction ARE a subnormal half, 2^-24 c in the lowest places, and a product of it is exact.
// The SUM of products is not: a tensor core lines products up by their operands' exponents, a subnormal's being 2^-14 however small it is,
// and drops what lies 24 bits or so below the largest.  Measured against the largest product of 16: 2^-15.9 with codes in the lowest places,
// 2^-20.4 four places higher, 2^-21.9 six.  So keys' codes go to bits 4 - 7 (seven integer instructions for a word of eight), values', which
// all add up with one sign, to the top of the fraction, bits 6 - 9 (eight).  (With the codes in the lowest places, five: 32 rows of 1000 - 2000
// tokens take 29.0 us instead of 30.2, and a query with one large element is off by 2^-14 of its score's parts.)
// The tokens are the 16 rows of an mma.sync tile and the group's query heads its 8 columns: the cache is the operand that fills the
// tile.  Queries are scaled by a power of two per head to the middle of the range of halves, which is exact down to 2^-32 of the
// head's largest element.  Probabilities are not rounded to 11 bits: what rounding leaves of p s is multiplied as well -- in the
// columns that up to four heads leave free, else in a second product -- since a code's products are larger than its value's.
//
// Work: tiles of 16 * TS or 32 * TS tokens of all rows, in equal shares over one wave of CTAs, whatever rows they belong to (the lengths are device
// data).  Whole token rows come by bulk copies into a ring (of the working warps: with a warp of its own for that, two CTAs to
// an SM leave a thread 96 registers, and spill); a warp takes 16 or 32 tokens of one kv head.  A row
// that lies in one share is written out; else its parts go to the workspace and a second kernel adds them up.
#include "kv_int4.cuh"
#include "attention_tmem.cuh"
#include <type_traits>

namespace {

constexpr int kMaxConsumers = 8, kMaxStages = 8, kUnit = 16, kCluster = 8, kFirst = 3;
// a row's start and end in tiles (150 rows of 200 - 400 tokens, 2 kv heads of 64: 13.5 us; 0 tiles 16.0, 2 tiles 15.0)
constexpr int kRowCost = 1;
// tokens of a share, at least a tile (one row of 1500 / 3900 tokens, 8 kv heads of 128: 11.5 / 12.4 us; of 64 tokens 13.3 / 14.2, 128: 15.5 / 16.9)
constexpr int kMinLog2 = 5, kMinTokens = 1 << kMinLog2;

struct Int4DecodeParams {
  const void* q; int64_t q_bs, q_hs; int q_vec;   // q_vec: heads on 16-byte boundaries
  void* out; int64_t o_bs, o_hs;
  const uint8_t* cache; int64_t row_stride, max_tokens;
  const int32_t* table; int64_t tab_rs, tab_cs, requests, width;
  const void* req_idx; int req_w;
  const void* seq_len; int len_w;
  int batch, Hq, Hkv, G, HB, nblk, qblocks, TS, TS_log2, stages, pitch;
  int64_t most;                                   // tokens of a row that the call's bound lets count
  float scale_log2;
  float* ws_o; float* ws_ml; int2* ws_info;       // parts [cta][2][HB * G]: rows, (largest score, sum); first and last CTA of a row
};

__device__ __forceinline__ uint32_t trans8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// as common.cuh's, but not volatile: products of the two units of a tile may change places
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float2 halves(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
// 2^e, e clamped to the range of normal numbers
__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e < -126 ? 1 : e > 127 ? 254 : e + 127) << 23); }

// the row of a tile's unit that stands at place i of eight: rows 0 - 3 and 4 - 7 as well as the even and the odd ones then lie in
// different banks (a row's pitch is 32 bytes past a multiple of 128)
__device__ __forceinline__ int place(int i) { return i ^ ((i >> 2) & 1); }

// units of 16 tokens that a warp takes together: two where their groups' scales leave the registers
constexpr int units_of(int d, int group) { return d / group > 2 ? 1 : 2; }

// One warp's work: up to 8 query heads of one kv head, U units of 16 tokens in turn.
// DUP: at most 4 heads; columns 4 - 7 are the same heads again and take what rounding leaves of p s.
template <typename T, int D, int GS, bool DUP>
struct Int4Consumer {
  static constexpr int NG = D / GS, NW = D / 32, MT = D / 16, U = units_of(D, GS);
  uint4 raw[NW];                                  // the query as it is in memory, between ask() and begin()
  uint32_t qb[NW][4];                             // a key word's query elements: nibbles (0, 4), (2, 6), (1, 5), (3, 7)
  float f[2], sq[2][NG];                          // per column: what a sum of codes is multiplied by; scaled sums of the query
  float O[MT][4], z[2][NG];                       // sums of p s c and of p m
  float m[2], base[2], l[2], m_lim[2];            // the maximum (base: 0 instead of -inf) that sums are relative to; above m_lim it is raised
  float v_scale[2][NG];                           // powers of two that p s is multiplied by before it is rounded
  static constexpr int kMostUp = 118;             // 2^kMostUp at most: times 2^8, a number
  int r, c;
  int k_at, g_at, v_at[2], step;                   // bytes from a unit's first row: key words, groups, value words of two tokens; eight rows

  using Pair = typename Vec2<T>::type;
  static __device__ __forceinline__ Pair as2(uint32_t w) { return *reinterpret_cast<Pair*>(&w); }
  static __device__ __forceinline__ Pair pair2(float x) {
    const uint32_t w = pack2<T>(x, x);
    return as2(w);
  }
  // a pair of elements as halves (bf16: after scaling, within their range)
  static __device__ __forceinline__ uint32_t to_half2(Pair x) {
    const uint32_t w = *reinterpret_cast<uint32_t*>(&x);
    if (std::is_same<T, __half>::value) return w;
    return pack2<__half>(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ int word_at(int k, int c) { return GS == 32 ? k * 4 + c : (k >> 1) * 8 + c * 2 + (k & 1); }
  static __device__ __forceinline__ constexpr int group_of(int k) { return GS == 32 ? k : GS == 64 ? k >> 1 : 0; }

  // the query's words of this lane's column, on their way while the ring is filled
  __device__ __forceinline__ void ask(const Int4DecodeParams& p, int b, int kvh, int head0, int heads) {
    const int col = DUP ? r & 3 : r;
    const T* q = reinterpret_cast<const T*>(p.q) + (int64_t)b * p.q_bs + (int64_t)(kvh * p.G + head0 + col) * p.q_hs;
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      raw[k] = make_uint4(0, 0, 0, 0);
      if (col < heads) {
        const T* w = q + word_at(k, c) * 8;
        if (p.q_vec) {
          raw[k] = *reinterpret_cast<const uint4*>(w);
        } else {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(w);
          raw[k] = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
        }
      }
    }
  }
  // Packed arithmetic, and the sums by the tensor cores from codes of 1: straight-line code runs from a cold instruction cache once a
  // segment, so its length is its time.
  __device__ __forceinline__ void begin(const Int4DecodeParams& p) {
    using T2 = typename Vec2<T>::type;
    T2 most = as2(raw[0].x & 0x7fff7fffu);
#pragma unroll
    for (int k = 0; k < NW; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) most = __hmax2_nan(most, as2((&raw[k].x)[i] & 0x7fff7fffu));
    const float2 ends = kv4::scale_min<T>(*reinterpret_cast<const uint32_t*>(&most));
    float big = ends.x > ends.y || ends.x != ends.x ? ends.x : ends.y;
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    // largest element to [2^8, 2^9), by 2^15 at most (a half multiplies); an infinity stays one
    int e = 8 - ((int)(__float_as_uint(big) >> 23) - 127);
    if (!(big < INFINITY) || big == 0.f) e = 0;
    constexpr int kMost = std::is_same<T, __half>::value ? 15 : 100;
    e = e < -kMost ? -kMost : e > kMost ? kMost : e;
    const T2 by = pair2(exp2i(e));
    float sums[NG][4];
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[g][i] = 0.f;
    const uint32_t one[4] = {0x00100010u, 0x00100010u, 0x00100010u, 0x00100010u};
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      qb[k][0] = to_half2(__hmul2(as2(__byte_perm(raw[k].x, raw[k].z, 0x5410)), by));
      qb[k][1] = to_half2(__hmul2(as2(__byte_perm(raw[k].y, raw[k].w, 0x5410)), by));
      qb[k][2] = to_half2(__hmul2(as2(__byte_perm(raw[k].x, raw[k].z, 0x7632)), by));
      qb[k][3] = to_half2(__hmul2(as2(__byte_perm(raw[k].y, raw[k].w, 0x7632)), by));
      mma(sums[group_of(k)], one, qb[k][0], qb[k][1]);
      mma(sums[group_of(k)], one, qb[k][2], qb[k][3]);
    }
    const float back = p.scale_log2 * exp2i(-e) * 1048576.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f[j] = __shfl_sync(0xffffffffu, back, (2 * c + j) * 4);
#pragma unroll
      for (int g = 0; g < NG; ++g) sq[j][g] = sums[g][j] * f[j];
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) O[t][i] = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      m[j] = m_lim[j] = -INFINITY;
      l[j] = base[j] = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        z[j][g] = 0.f;
        v_scale[j][g] = exp2i(kMostUp);
      }
    }
  }

  // a score above what the sums are scaled for: the maximum rises, and the sums so far are worth `fell` of what they were (O is left to rescale())
  __device__ __forceinline__ void raise(const float (&v)[U][2][2], float (&fell)[2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float mx = v[0][0][j];
#pragma unroll
      for (int x = 1; x < 2 * U; ++x) mx = fmaxf(mx, v[x >> 1][x & 1][j]);
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      if (mx > m[j]) {
        const float a = fast_exp2(m[j] - mx);     // m[j] = -inf at first: 0
        m[j] = base[j] = mx;
        l[j] *= a;
#pragma unroll
        for (int g = 0; g < NG; ++g) z[j][g] *= a;
        fell[j] = a;
      }
      m_lim[j] = m[j] + 8.f;
    }
  }

  // The power of two that a head's products with a group's scales are multiplied by before they are rounded to two halves, whose least
  // step is 2^-24: the largest p s so far -- of the sums as they are worth now, and of these tokens -- comes to 2^7 or above.  By the products,
  // per head and group, and not by the scales, which may lie any range apart: a wide token of little weight, or a wide group, must not take
  // the digits of the others.  A larger power than the last one is allowed by as much as the sums have fallen.  (One power for a warp, by
  // the largest scale: one row of 201 tokens 6.6 us instead of 6.85, the larger cases level; a value 2^-20 of a scale seen before was off by 1 %.)
  __device__ __forceinline__ void rescale(const float (&pr)[U][2][2], const uint32_t (&vg)[U][2][NG], const float (&fell)[2], bool fresh) {
    // powers of two by their exponents alone: what `fell` leaves room for (2^127 where nothing is left)
    float up[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) up[j] = __uint_as_float(0x7f000000u - (__float_as_uint(fell[j]) & 0x7f800000u));
    float by[2][NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float top[2] = {0.f, 0.f};                  // of what is a number
#pragma unroll
      for (int n = 0; n < U; ++n) {
        const float s0 = kv4::scale_min<T>(vg[n][0][g]).x, s1 = kv4::scale_min<T>(vg[n][1][g]).x;
#pragma unroll
        for (int j = 0; j < 2; ++j) top[j] = max3(top[j], pr[n][0][j] * s0, pr[n][1][j] * s1);
      }
      uint32_t e = __float_as_uint(top[0]) >> 23 | __float_as_uint(top[1]) >> 23 << 16;      // of both heads
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) e = __vmaxu2(e, __shfl_xor_sync(0xffffffffu, e, o));
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int want = 134 + 127 - (int)(j ? e >> 16 : e & 0xffffu);
        const float next = fminf(__int_as_float((want < 127 + kMostUp ? want : 127 + kMostUp) << 23), v_scale[j][g] * up[j]);
        by[j][g] = fell[j] * next * __uint_as_float(0x7f000000u - __float_as_uint(v_scale[j][g]));
        v_scale[j][g] = next;
      }
    }
    if (fresh) return;                            // O is zero
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        O[t][j] *= by[j][t * 16 / GS];
        O[t][2 + j] *= by[j][t * 16 / GS];
      }
  }

  __device__ __forceinline__ Int4Consumer(int lane, int pitch) {
    r = lane >> 2;
    c = lane & 3;
    step = 8 * pitch;
    k_at = place(r) * pitch + c * (GS == 32 ? 4 : 8);
    g_at = place(r) * pitch + D;
    v_at[0] = place(2 * c) * pitch + D / 2 + (GS == 32 ? r >> 1 : r) * 4;
    v_at[1] = place(2 * c + 1) * pitch + D / 2 + (GS == 32 ? r >> 1 : r) * 4;
  }

  // 16 U tokens at `at` (the head's bytes of the first), of which `valid` count; fresh: the first of a part
  __device__ __forceinline__ void tile(const uint8_t* at, int valid, bool fresh) {
    constexpr uint32_t kKey = 0x00f000f0u, kValue = 0x03c003c0u;   // 2^-20 code and 2^-18 code as halves
    // ---- scores: 16 tokens (rows) and 8 heads (columns) to a unit ----
    float acc[U][NG][4];
    uint32_t vg[U][2][NG];                        // the values' groups
    float v[U][2][2];
#pragma unroll
    for (int n = 0; n < U; ++n) {
      const uint8_t* u = at + 2 * n * step;
      uint32_t w0[NW], w1[NW];
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        if (GS == 32) {
          w0[k] = *reinterpret_cast<const uint32_t*>(u + k_at + k * 16);
          w1[k] = *reinterpret_cast<const uint32_t*>(u + k_at + step + k * 16);
        } else if ((k & 1) == 0) {
          const uint2 x = *reinterpret_cast<const uint2*>(u + k_at + k * 16), y = *reinterpret_cast<const uint2*>(u + k_at + step + k * 16);
          w0[k] = x.x; w0[k + 1] = x.y;
          w1[k] = y.x; w1[k + 1] = y.y;
        }
      }
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][g][i] = 0.f;
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        const uint32_t lo[4] = {w0[k] << 4 & kKey, w1[k] << 4 & kKey, w0[k] >> 4 & kKey, w1[k] >> 4 & kKey};
        const uint32_t hi[4] = {w0[k] & kKey, w1[k] & kKey, w0[k] >> 8 & kKey, w1[k] >> 8 & kKey};
        mma(acc[n][group_of(k)], lo, qb[k][0], qb[k][1]);
        mma(acc[n][group_of(k)], hi, qb[k][2], qb[k][3]);
      }
    }
#pragma unroll
    for (int n = 0; n < U; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t word[2 * NG];                    // groups of K, then of V
#pragma unroll
        for (int x = 0; x < NG; ++x) {
          const uint2 y = *reinterpret_cast<const uint2*>(at + g_at + (2 * n + i) * step + x * 8);
          word[2 * x] = y.x;
          word[2 * x + 1] = y.y;
        }
        float2 ks[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          ks[g] = kv4::scale_min<T>(word[g]);
          vg[n][i][g] = word[NG + g];
        }
        float tu[2], uu[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float t = ks[0].x * acc[n][0][2 * i + j], u = ks[0].y * sq[j][0];
#pragma unroll
          for (int g = 1; g < NG; ++g) {
            t = fmaf(ks[g].x, acc[n][g][2 * i + j], t);
            u = fmaf(ks[g].y, sq[j][g], u);
          }
          tu[j] = t;
          uu[j] = u;
        }
        f32x2_split(f32x2_fma(f32x2(tu[0], tu[1]), f32x2(f[0], f[1]), f32x2(uu[0], uu[1])), v[n][i][0], v[n][i][1]);
      }
    if (valid < 16 * U) {                         // a row's last tokens
#pragma unroll
      for (int n = 0; n < U; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (place(r) + 16 * n + 8 * i >= valid) {
            v[n][i][0] = v[n][i][1] = -INFINITY;
#pragma unroll
            for (int g = 0; g < NG; ++g) vg[n][i][g] = 0u;
          }
    }
    // the largest of a thread's 2 U values of either head
    auto largest = [](const float (&x)[U][2][2], int j) {
      const float y = fmaxf(x[0][0][j], x[0][1][j]);
      return U == 1 ? y : max3(y, x[U - 1][0][j], x[U - 1][1][j]);
    };
    float fell[2] = {1.f, 1.f};
    const bool risen = __any_sync(0xffffffffu, largest(v, 0) > m_lim[0] || largest(v, 1) > m_lim[1]);
    if (risen) raise(v, fell);
    // ---- probabilities; whether a product with a scale may be past the range of halves ----
    float pr[U][2][2];
#pragma unroll
    for (int n = 0; n < U; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f32x2_split(f32x2_add(f32x2(v[n][i][0], v[n][i][1]), f32x2(-base[0], -base[1])), pr[n][i][0], pr[n][i][1]);
#pragma unroll
        for (int j = 0; j < 2; ++j) pr[n][i][j] = fast_exp2(pr[n][i][j]);
        f32x2_split(f32x2_add(f32x2(l[0], l[1]), f32x2(pr[n][i][0], pr[n][i][1])), l[0], l[1]);
      }
    const uint64_t p_top = f32x2(largest(pr, 0), largest(pr, 1));
    float product = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      using T2 = typename Vec2<T>::type;
      T2 s = __hmax2(as2(vg[0][0][g]), as2(vg[0][1][g]));
      if (U == 2) s = __hmax2(s, __hmax2(as2(vg[U - 1][0][g]), as2(vg[U - 1][1][g])));
      float a, b;
      f32x2_split(f32x2_mul(p_top, f32x2(v_scale[0][g], v_scale[1][g])), a, b);
      product = fmaxf(product, fmaxf(a, b) * kv4::scale_min<T>(*reinterpret_cast<uint32_t*>(&s)).x);
    }
    if (__any_sync(0xffffffffu, risen || product > 32768.f)) rescale(pr, vg, fell, fresh);
#pragma unroll
    for (int n = 0; n < U; ++n) {
      // ---- probabilities, times the values' scales, as the second product's columns ----
      uint32_t pb[NG][2], rest[NG][2];
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 vs = kv4::scale_min<T>(vg[n][i][g]);
#pragma unroll
          for (int j = 0; j < 2; ++j) z[j][g] = fmaf(pr[n][i][j], vs.y, z[j][g]);
          float x, y, dx, dy;
          f32x2_split(f32x2_mul(f32x2(pr[n][i][0], pr[n][i][1]), f32x2(v_scale[0][g], v_scale[1][g])), x, y);
          x *= vs.x;
          y *= vs.x;
          const uint32_t near = pack2<__half>(x, y);
          const float2 back = halves(near);
          f32x2_split(f32x2_fma(f32x2(back.x, back.y), f32x2(-1.f, -1.f), f32x2(x, y)), dx, dy);
          const uint32_t left = pack2<__half>(dx, dy);
          if (DUP) {
            pb[g][i] = trans8x8(c < 2 ? near : left);
          } else {
            pb[g][i] = trans8x8(near);
            rest[g][i] = trans8x8(left);
          }
        }
      // ---- values: rows are elements, columns heads, the products run over tokens ----
      const uint8_t* u = at + 2 * n * step;
      auto add = [&](int tile, int g, const uint32_t (&a)[4]) {
        mma(O[tile], a, pb[g][0], pb[g][1]);
        if (!DUP) mma(O[tile], a, rest[g][0], rest[g][1]);
      };
      if (GS == 32) {
        const uint32_t pick = (r & 1) ? 0x7632u : 0x5410u;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          auto word = [&](int o) { return *reinterpret_cast<const uint32_t*>(u + o + g * 16); };
          const uint32_t x = __byte_perm(word(v_at[0]), word(v_at[1]), pick), y = __byte_perm(word(v_at[0] + step), word(v_at[1] + step), pick);
          const uint32_t a0[4] = {x << 6 & kValue, x << 2 & kValue, y << 6 & kValue, y << 2 & kValue};
          const uint32_t a1[4] = {x >> 2 & kValue, x >> 6 & kValue, y >> 2 & kValue, y >> 6 & kValue};
          add(g * 2, g, a0);
          add(g * 2 + 1, g, a1);
        }
      } else {
#pragma unroll
        for (int b = 0; b < D / 64; ++b) {
          const int g = b * 64 / GS;
          auto word = [&](int o) { return *reinterpret_cast<const uint32_t*>(u + o + b * 32); };
          const uint32_t e0 = word(v_at[0]), e1 = word(v_at[1]), e2 = word(v_at[0] + step), e3 = word(v_at[1] + step);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t x = __byte_perm(e0, e1, h ? 0x7632 : 0x5410), y = __byte_perm(e2, e3, h ? 0x7632 : 0x5410);
            const uint32_t a0[4] = {x << 6 & kValue, x << 2 & kValue, y << 6 & kValue, y << 2 & kValue};
            const uint32_t a1[4] = {x >> 2 & kValue, x >> 6 & kValue, y >> 2 & kValue, y >> 6 & kValue};
            add(b * 4 + h * 2, g, a0);
            add(b * 4 + h * 2 + 1, g, a1);
          }
        }
      }
    }
  }

  // the element that O[t][0] (and [1]) of this lane belongs to; O[t][2] (and [3]) to the next one
  __device__ __forceinline__ int element(int t) const {
    return GS == 32 ? (t >> 1) * 32 + r * 4 + (t & 1) * 2 : (t >> 2) * 64 + r * 8 + (t & 3) * 2;
  }
  // sums in true units, complete over the lanes
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], o);
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) z[j][g] += __shfl_xor_sync(0xffffffffu, z[j][g], o);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        float lo = O[t][j], hi = O[t][2 + j];
        if (DUP) {
          lo += __shfl_xor_sync(0xffffffffu, lo, 2);
          hi += __shfl_xor_sync(0xffffffffu, hi, 2);
        }
        const int g = GS == 32 ? t >> 1 : (t >> 2) * 64 / GS;
        const float by = exp2i(127 - (int)(__float_as_uint(v_scale[j][g]) >> 23));
        O[t][j] = fmaf(lo * 262144.f, by, z[j][g]);
        O[t][2 + j] = fmaf(hi * 262144.f, by, z[j][g]);
      }
    }
  }
};

struct Segment { int b, blk, first, last, tiles; };   // tiles [first, last) of a row of `tiles`

__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_smem(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float ld_peer(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// CLUSTER: a row and block of heads to a cluster of kCluster CTAs, whose parts meet in shared memory; else equal shares of all tiles.
template <typename T, int D, int GS, bool DUP, bool CLUSTER>
__global__ void __launch_bounds__(kMaxConsumers * 32, 2) kv4_decode_kernel(const Int4DecodeParams p) {
  pdl_prologue();   // everything below reads what earlier kernels of the step wrote
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int warp_sum[kMaxConsumers];
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem);
  uint64_t* empty_bar = full_bar + kMaxStages;
  uint8_t* ring = smem + 128;
  constexpr int kWarpTokens = kUnit * units_of(D, GS);
  const int tile_log2 = p.TS_log2 + (kWarpTokens == 32 ? 5 : 4), tile = 1 << tile_log2;
  const int warp_bytes = kWarpTokens * p.pitch, stage_bytes = warp_bytes << p.TS_log2;
  float* join = reinterpret_cast<float*>(ring + p.stages * stage_bytes);      // sums of the warps that share a head
  const int per_head = p.qblocks * 8 * (D + 2);
  int* prefix = reinterpret_cast<int*>(join + (p.TS - 1) * p.HB * per_head);  // tiles of the rows before, [batch + 1]
  int* lens = prefix + p.batch + 1;
  int* reqs = lens + p.batch;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nwarps = p.HB * p.qblocks * p.TS;
  const int heads_warps = p.HB * p.qblocks;
  auto length = [&](int r, int& req) {
    const int64_t n = load_index(p.seq_len, r, p.len_w), q = load_index(p.req_idx, r, p.req_w);
    req = (int)q;
    return q < 0 || q >= p.requests || n <= 0 ? 0 : n > p.most ? (int)p.most : (int)n;
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full_bar[s], nwarps);
      mbar_init(&empty_bar[s], nwarps);
    }
    mbar_fence_init();
  }

  auto cost = [&](int len) { return len > 0 ? ((len + tile - 1) >> tile_log2) + kRowCost : 0; };
  Segment seg;
  int all = 0, item = 0, item_end = 0, len0 = 0, req0 = 0;
  if (CLUSTER) {
    const int id = blockIdx.x / kCluster, rank = blockIdx.x - id * kCluster;
    seg.blk = id / p.batch;
    seg.b = id - seg.blk * p.batch;
    len0 = length(seg.b, req0);
    seg.tiles = (len0 + tile - 1) >> tile_log2;
    seg.first = seg.tiles * rank / kCluster;
    seg.last = seg.tiles * (rank + 1) / kCluster;
    item_end = seg.first < seg.last;
    __syncthreads();
  } else {
    // ---- tiles of the rows before each (a row counts kRowCost more: its start and end); a thread owns neighbouring rows ----
    const int per = p.batch <= 32 ? 1 : (p.batch + (int)blockDim.x - 1) / (int)blockDim.x, r_lo = threadIdx.x * per;
    const int r_hi = r_lo + per < p.batch ? r_lo + per : p.batch;
    int own = 0;
#pragma unroll 1
    for (int r = r_lo; r < r_hi; ++r) {
      lens[r] = length(r, reqs[r]);
      own += cost(lens[r]);
    }
    int upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    int at = upto - own;
    if (p.batch > 32) {                           // else the first warp has all rows
      if (lane == 31) warp_sum[warp] = upto;
      __syncthreads();
      at += __reduce_add_sync(0xffffffffu, lane < warp ? warp_sum[lane] : 0);
    }
#pragma unroll 1
    for (int r = r_lo; r < r_hi; ++r) {
      prefix[r] = at;
      at += cost(lens[r]);
    }
    if (r_hi == p.batch && r_lo < r_hi) prefix[p.batch] = at;
    __syncthreads();
    all = prefix[p.batch];
    // ---- this CTA's share of all tiles, heads' blocks one after the other ----
    const int total = all * p.nblk, least = tile_log2 < kMinLog2 ? kMinLog2 - tile_log2 : 0, worth = (total + (1 << least) - 1) >> least;
    const int shares = worth < (int)gridDim.x ? worth : (int)gridDim.x;
    if ((int)blockIdx.x >= shares) return;
    const int each = total / shares, more_by_one = total - each * shares;
    item = blockIdx.x * each + ((int)blockIdx.x < more_by_one ? blockIdx.x : more_by_one);
    item_end = item + each + ((int)blockIdx.x < more_by_one);
  }
  // the part of a row at `item`
  auto part_at = [&](int& item, Segment& s) -> bool {
    if (item >= item_end) return false;
    if (CLUSTER) {
      s = seg;
      item = item_end;
      return true;
    }
    s.blk = p.nblk == 1 ? 0 : item / all;
    const int x = item - s.blk * all;
    int lo = 0, n = p.batch;                      // the last row that begins at or before x, 32 at a look
#pragma unroll 1
    while (n > 1) {
      const int stride = (n + 31) >> 5, i = lane * stride;
      const int k = __popc(__ballot_sync(0xffffffffu, i < n && prefix[lo + i] <= x)) - 1;
      lo += k * stride;
      n = n - k * stride < stride ? n - k * stride : stride;
    }
    s.b = lo;
    s.tiles = prefix[lo + 1] - prefix[lo] - kRowCost;
    const int left = item_end - item, from = x - prefix[lo], to = left < prefix[lo + 1] - x ? from + left : s.tiles + kRowCost;
    s.first = from > kRowCost ? from - kRowCost : 0;
    s.last = to > kRowCost ? to - kRowCost : 0;   // may be empty: the part of a row's start that is only cost
    item += to - from;
    return true;
  };
  auto next = [&](int& item, Segment& s) -> bool {
    bool any;
    do any = part_at(item, s);
    while (any && s.first >= s.last);
    return any;
  };

  // ---- the ring's copies: each warp brings its part of a tile's token rows, whose table entries are read a tile ahead, one bulk copy to
  // a row.  (16 bytes a lane instead, measured when a code cost fewer instructions: 32 rows of 1000 - 2000 tokens, 8 kv heads of 128: 32 us, bulk
  // 29; one row of 201: 7.2 and 6.6; rows of 160 bytes, 150 of 200 - 400 tokens: 13.6 and 13.4.) ----
  const int hb = kv4::head_bytes(D, GS), mine = nwarps == 8 ? tile >> 3 : (tile + nwarps - 1) / nwarps;   // token rows of this warp, at most 32
  struct Place { Segment s; int item, t; bool more; };   // a tile of the share
  auto start_of = [&](Place& x) {
    x.item = item;
    x.more = next(x.item, x.s);
    x.t = x.s.first;
  };
  auto step_on = [&](Place& x) {
    if (++x.t == x.s.last) {
      x.more = next(x.item, x.s);
      x.t = x.s.first;
    }
  };
  auto rows_of = [&](const Place& x) {            // token rows of the tile
    const int left = (CLUSTER ? len0 : lens[x.s.b]) - x.t * tile;
    return left < tile ? left : tile;
  };
  auto entry = [&](const Place& x) -> int {       // this lane's
    const int i = warp * mine + lane;
    if (!x.more || lane >= mine || i >= rows_of(x)) return 0;
    return ld_upstream(p.table + (int64_t)(CLUSTER ? req0 : reqs[x.s.b]) * p.tab_rs + (int64_t)(x.t * tile + i) * p.tab_cs);
  };
  auto bring = [&](const Place& x, int row, int s) {
    const int from = x.s.blk * p.HB * hb, shift = from & 15, pieces = (shift + p.HB * hb + 15) >> 4;
    const int first = warp * mine, rows_here = rows_of(x) - first, mine_here = rows_here < mine ? rows_here : mine;
    const uint8_t* src = p.cache + (from - shift);
    uint8_t* dst = ring + s * stage_bytes + first * p.pitch;
    const int at = row < 0 || row >= p.max_tokens ? 0 : row;
    if (lane == 0) mbar_arrive_expect_tx(&full_bar[s], (uint32_t)((mine_here > 0 ? mine_here : 0) * pieces * 16));
    __syncwarp();
    if (lane < mine_here) bulk_g2s(dst + lane * p.pitch, src + (int64_t)at * p.row_stride, (uint32_t)pieces * 16u, &full_bar[s]);
  };

  // ===================== a warp: (kv head, block of query heads, unit of the tile) =====================
  const int ts = p.TS == 1 ? 0 : warp / heads_warps, wh = warp - ts * heads_warps;
  const int hl = p.qblocks == 1 ? wh : wh / p.qblocks, qblk = wh - hl * p.qblocks;
  const int head0 = qblk * 8, heads = p.G - head0 < 8 ? p.G - head0 : 8;
  Int4Consumer<T, D, GS, DUP> c(lane, p.pitch);
  // columns of this lane: heads 2c and 2c + 1 (DUP: the upper half of the columns repeats the lower)
  const bool counts = !DUP || c.c < 2;
  int s = 0, at_tile = 0;
  uint32_t phase = 0;
  // The first tiles are much of what a share reads: their entries are read together, and their rows asked for at once (the query before
  // them: behind them it waits for all of their bytes).
  Place ahead;
  start_of(ahead);
  bool got = next(item, seg);
  if (got) c.ask(p, seg.b, seg.blk * p.HB + hl, head0, heads);
  int row = 0;
  {
    Place look = ahead;
    int first_rows[kFirst];
#pragma unroll
    for (int f = 0; f < kFirst; ++f) {
      first_rows[f] = entry(look);
      if (look.more) step_on(look);
    }
    for (int f = 0; f < p.stages && ahead.more; ++f) {
      row = first_rows[0];
#pragma unroll
      for (int k = 1; k < kFirst; ++k) row = f == k ? first_rows[k] : row;
      if (f >= kFirst) row = entry(ahead);
      bring(ahead, row, f);
      step_on(ahead);
    }
    row = entry(ahead);
  }
  while (got) {
    const int len = CLUSTER ? len0 : lens[seg.b], kvh = seg.blk * p.HB + hl;
    const int off = ((seg.blk * p.HB * hb) & 15) + hl * hb + ts * warp_bytes;
    c.begin(p);
#pragma unroll 1
    for (int t = seg.first; t < seg.last; ++t, ++at_tile) {
      mbar_wait(&full_bar[s], phase);
      const int valid = len - t * tile - ts * kWarpTokens;
      if (valid > 0) c.tile(ring + s * stage_bytes + off, valid, t == seg.first);
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_bar[s]);
      if (at_tile > 0 && ahead.more) {            // into the stage of the tile before this one, which the others have left by now
        const int b = s == 0 ? p.stages - 1 : s - 1;
        mbar_wait(&empty_bar[b], s == 0 ? phase ^ 1u : phase);
        bring(ahead, row, b);
        step_on(ahead);
        row = entry(ahead);
      }
      if (++s == p.stages) { s = 0; phase ^= 1; }
    }
    const Segment done = seg;
    got = next(item, seg);
    if (got) c.ask(p, seg.b, seg.blk * p.HB + hl, head0, heads);
    c.finish();
    if (p.TS > 1) {
      auto bar = [&] { asm volatile("bar.sync 1, %0;" ::"r"(nwarps * 32) : "memory"); };
      bar();                                      // the sums before these have been read
      float* to_join = join + ((ts - 1) * p.HB * p.qblocks + wh) * 8 * (D + 2);
      if (ts > 0 && counts) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float* to = to_join + (2 * c.c + j) * (D + 2);
#pragma unroll
          for (int t = 0; t < D / 16; ++t) *reinterpret_cast<float2*>(to + c.element(t)) = make_float2(c.O[t][j], c.O[t][2 + j]);
          if (c.r == 0) *reinterpret_cast<float2*>(to + D) = make_float2(c.m[j], c.l[j]);
        }
      }
      bar();
      if (ts == 0 && counts) {
#pragma unroll 1
        for (int o = 1; o < p.TS; ++o) {
          const float* from = join + ((o - 1) * p.HB * p.qblocks + wh) * 8 * (D + 2);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float* x = from + (2 * c.c + j) * (D + 2);
            const float2 ml = *reinterpret_cast<const float2*>(x + D);
            const float mm = fmaxf(c.m[j], ml.x), base = mm == -INFINITY ? 0.f : mm;
            const float a = fast_exp2(c.m[j] - base), e = fast_exp2(ml.x - base);
            c.m[j] = mm;
            c.l[j] = c.l[j] * a + ml.y * e;
#pragma unroll
            for (int t = 0; t < D / 16; ++t) {
              const float2 y = *reinterpret_cast<const float2*>(x + c.element(t));
              c.O[t][j] = c.O[t][j] * a + y.x * e;
              c.O[t][2 + j] = c.O[t][2 + j] * a + y.y * e;
            }
          }
        }
      }
    }
    if (CLUSTER) break;
    const bool whole = done.first == 0 && done.last == done.tiles;
    if (ts == 0 && counts) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int head = head0 + 2 * c.c + j;
        if (2 * c.c + j >= heads) continue;
        if (whole) {
          const float inv = 1.f / c.l[j];
          T* to = reinterpret_cast<T*>(p.out) + (int64_t)done.b * p.o_bs + (int64_t)(kvh * p.G + head) * p.o_hs;
#pragma unroll
          for (int t = 0; t < D / 16; ++t) {
            to[c.element(t)] = from_f32<T>(c.O[t][j] * inv);
            to[c.element(t) + 1] = from_f32<T>(c.O[t][2 + j] * inv);
          }
        } else {
          const int64_t part = ((int64_t)blockIdx.x * 2 + (done.first == 0 ? 1 : 0)) * p.HB * p.G + hl * p.G + head;
#pragma unroll
          for (int t = 0; t < D / 16; ++t)
            *reinterpret_cast<float2*>(p.ws_o + part * D + c.element(t)) = make_float2(c.O[t][j], c.O[t][2 + j]);
          if (c.r == 0) *reinterpret_cast<float2*>(p.ws_ml + part * 2) = make_float2(c.m[j], c.l[j]);
        }
      }
      if (wh == 0 && lane == 0) {
        int* note = reinterpret_cast<int*>(p.ws_info + (int64_t)done.blk * p.batch + done.b);
        if (done.first == 0) note[0] = blockIdx.x;
        if (done.last == done.tiles) note[1] = blockIdx.x;
      }
    }
  }
  if (!CLUSTER) return;

  // ---- the cluster's parts, in the memory of the rings: [heads][D + 2] with the largest score and the sum; each CTA adds up its heads ----
  __syncthreads();                                // the ring has been read
  float* part = reinterpret_cast<float*>(ring);
  const int block_heads = p.HB * p.G, rank = blockIdx.x % kCluster;
  if (seg.first < seg.last) {
    if (ts == 0 && counts) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (2 * c.c + j >= heads) continue;
        float* to = part + (hl * p.G + head0 + 2 * c.c + j) * (D + 2);
#pragma unroll
        for (int t = 0; t < D / 16; ++t) *reinterpret_cast<float2*>(to + c.element(t)) = make_float2(c.O[t][j], c.O[t][2 + j]);
        if (c.r == 0) *reinterpret_cast<float2*>(to + D) = make_float2(c.m[j], c.l[j]);
      }
    }
  } else {
    for (int h = threadIdx.x; h < block_heads; h += blockDim.x) *reinterpret_cast<float2*>(part + h * (D + 2) + D) = make_float2(-INFINITY, 0.f);
  }
  __syncwarp();
  cluster_sync_all();
  constexpr int E = D / 32;
  for (int h = warp * kCluster + rank; h < block_heads; h += nwarps * kCluster) {
    float m[kCluster], l[kCluster], x[kCluster][E], M = -INFINITY;
#pragma unroll
    for (int k = 0; k < kCluster; ++k) {
      const uint32_t peer = peer_smem(smem_u32(part + h * (D + 2)), k);
      m[k] = ld_peer(peer + D * 4);
      l[k] = ld_peer(peer + D * 4 + 4);
#pragma unroll
      for (int e = 0; e < E; ++e) x[k][e] = ld_peer(peer + (e * 32 + lane) * 4);
      M = fmaxf(M, m[k]);
    }
    const float base = M == -INFINITY ? 0.f : M;
    float L = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll
    for (int k = 0; k < kCluster; ++k) {
      if (l[k] == 0.f && m[k] == -INFINITY) continue;   // a part without tokens: nothing was stored
      const float w = fast_exp2(m[k] - base);
      L = fmaf(l[k], w, L);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(x[k][e], w, o[e]);
    }
    T* to = reinterpret_cast<T*>(p.out) + (int64_t)seg.b * p.o_bs + (int64_t)(seg.blk * block_heads + h) * p.o_hs;
#pragma unroll
    for (int e = 0; e < E; ++e) to[e * 32 + lane] = from_f32<T>(len0 == 0 ? 0.f : o[e] / L);
  }
  __syncwarp();
  cluster_sync_all();                             // the peers have read this CTA's part
}

// The rows that several CTAs met in, and zeros for the empty ones.  Bound by latency: W warps take the parts of a row's head in turn,
// eight of each on their way together, and meet in shared memory (W = 1: four heads to a block, no meeting).
template <typename T, int D, int W>
__global__ void __launch_bounds__(W == 1 ? 128 : W * 32) kv4_decode_merge_kernel(const Int4DecodeParams p) {
  pdl_prologue();
  constexpr int E = D / 32, kAsk = 8;             // neighbouring elements of a lane
  __shared__ float sums[W][W == 1 ? 1 : D + 2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x, head = W == 1 ? blockIdx.y * 4 + warp : blockIdx.y;
  if (head >= p.Hq) return;
  const int kvh = head / p.G, blk = kvh / p.HB, local = (kvh - blk * p.HB) * p.G + head - kvh * p.G;
  const int2 who = __ldcg(p.ws_info + (int64_t)blk * p.batch + b);   // of an empty row: an earlier call's
  const int64_t len = load_index(p.seq_len, b, p.len_w), q = load_index(p.req_idx, b, p.req_w);
  T* out = reinterpret_cast<T*>(p.out) + (int64_t)b * p.o_bs + (int64_t)head * p.o_hs;
  if (len <= 0 || q < 0 || q >= p.requests || p.most <= 0) {
    for (int d = W == 1 ? lane : threadIdx.x; d < D; d += W * 32) out[d] = from_f32<T>(0.f);
    return;
  }
  const int n = who.y - who.x + 1;
  if (n < 2) return;                              // written by its only CTA
  const int first = W == 1 ? 0 : warp;
  auto part = [&](int i) { return ((int64_t)(who.x + i) * 2 + (i == 0 ? 1 : 0)) * p.HB * p.G + local; };
  float acc[E], M = -INFINITY, L = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 1
  for (int i0 = first; i0 < n; i0 += W * kAsk) {
    float x[kAsk][E];
    float2 ml[kAsk];
#pragma unroll
    for (int k = 0; k < kAsk; ++k) {
      const int i = i0 + W * k;
      ml[k] = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int e = 0; e < E; ++e) x[k][e] = 0.f;
      if (i < n) {
        ml[k] = __ldcg(reinterpret_cast<const float2*>(p.ws_ml) + part(i));
        const float* o = p.ws_o + part(i) * D + lane * E;
        if (E == 4) {
          const float4 y = __ldcg(reinterpret_cast<const float4*>(o));
          x[k][0] = y.x; x[k][1 % E] = y.y; x[k][2 % E] = y.z; x[k][3 % E] = y.w;
        } else if (E == 2) {
          const float2 y = __ldcg(reinterpret_cast<const float2*>(o));
          x[k][0] = y.x; x[k][1 % E] = y.y;
        } else {
          x[k][0] = __ldcg(o);
        }
      }
    }
    float mm = M;
#pragma unroll
    for (int k = 0; k < kAsk; ++k) mm = fmaxf(mm, ml[k].x);
    const float base = mm == -INFINITY ? 0.f : mm, a = fast_exp2(M - base);
    L *= a;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= a;
#pragma unroll
    for (int k = 0; k < kAsk; ++k) {
      const float w = fast_exp2(ml[k].x - base);
      L = fmaf(ml[k].y, w, L);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(x[k][e], w, acc[e]);
    }
    M = mm;
  }
  if constexpr (W == 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) out[lane * E + e] = from_f32<T>(acc[e] / L);
  } else {
#pragma unroll
  for (int e = 0; e < E; ++e) sums[warp][lane * E + e] = acc[e];
  if (lane == 0) { sums[warp][D] = M; sums[warp][D + 1] = L; }
  __syncthreads();
  if ((int)threadIdx.x < D) {
    float mm = -INFINITY, o = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) mm = fmaxf(mm, sums[w][D]);
    const float base = mm == -INFINITY ? 0.f : mm;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float a = fast_exp2(sums[w][D] - base);
      o = fmaf(sums[w][threadIdx.x], a, o);
      l = fmaf(sums[w][D + 1], a, l);
    }
    out[threadIdx.x] = from_f32<T>(o / l);
  }
  }
}

constexpr int kMaxBatch = 4096;                   // rows of one launch (their lengths lie in shared memory)
// Tokens of a row that a cluster takes.  One row of 201 / 650 / 1000 / 1400 tokens, 8 kv heads of 128: 6.9 / 10.3 / 12.3 / 16.0 us, in shares
// 9.4 / 11.7 / 11.0 / 11.4; 18 rows of 900: 16.1 and 18.4; 4 kv heads, 2 rows of 1000 / 1900: 9.2 / 13.1 and 11.8 / 10.9.
constexpr int kClusterMost = 1024;

struct Int4Plan { int HB, qblocks, TS, pitch, stages, smem, grid; bool cluster; };

// A function of sizes that the host knows, hence the same inside and outside a captured graph.
Int4Plan make_plan(int64_t batch, int G, int Hkv, int D, int group, int64_t max_len) {
  Int4Plan pl;
  pl.qblocks = (G + 7) / 8;
  pl.HB = 1;
  for (int h = 1; h * pl.qblocks <= kMaxConsumers; ++h)
    if (Hkv % h == 0) pl.HB = h;
  const int units = units_of(D, group);
  for (pl.TS = 1; 2 * pl.TS * pl.HB * pl.qblocks <= kMaxConsumers;) pl.TS *= 2;
  if (pl.TS > 8 / units) pl.TS = 8 / units;       // 128 tokens to a tile at most
  const int hb = kv4::head_bytes(D, group);
  const int bytes = ((pl.HB * hb + (pl.HB == Hkv ? 0 : 8)) + 15) / 16 * 16;
  pl.pitch = (bytes + 95) / 128 * 128 + 32;       // 32 bytes past a multiple of 128
  const int stage = pl.TS * units * kUnit * pl.pitch;
  const int rows = (int)(batch < kMaxBatch ? batch : kMaxBatch);
  const int fixed = 128 + (pl.TS - 1) * pl.HB * pl.qblocks * 8 * (D + 2) * 4 + (3 * rows + 1) * 4;
  // sixteen warps to an SM, each CTA with a ring of its part of the shared memory (1 KB of it is the system's)
  const int per_sm = 2 * kMaxConsumers / (pl.HB * pl.qblocks * pl.TS);
  const int cap = (b2l_max_smem_optin() + 1024) / per_sm - 1024 - 128;
  pl.stages = (cap - fixed) / stage;
  if (pl.stages > kMaxStages) pl.stages = kMaxStages;
  if (pl.stages < 2) pl.stages = 2;
  pl.smem = fixed + pl.stages * stage;
  const int tile = pl.TS * units * kUnit;
  const int64_t most = (int64_t)rows * cdiv64(max_len > 0 ? max_len : 1, tile > kMinTokens ? tile : kMinTokens) * (Hkv / pl.HB);
  const int64_t wave = (int64_t)per_sm * b2l_num_sms();
  pl.grid = (int)(most < wave ? most : wave);
  pl.cluster = batch * (Hkv / pl.HB) * kCluster <= wave && max_len <= kClusterMost && pl.HB * G * (D + 2) * 4 <= pl.stages * stage;
  if (pl.cluster) pl.grid = (int)(batch * (Hkv / pl.HB) * kCluster);
  return pl;
}

template <typename T, int D, int GS>
int launch_int4_decode(const Int4DecodeParams& p, const Int4Plan& pl, cudaStream_t st) {
  const dim3 grid((unsigned)pl.grid), block(pl.HB * pl.qblocks * pl.TS * 32);
  if (pl.cluster) {
    static int configured_cluster[2][64] = {{0}};
    auto kern = p.G <= 4 ? kv4_decode_kernel<T, D, GS, true, true> : kv4_decode_kernel<T, D, GS, false, true>;
    B2L_CUDA_CHECK(b2l_ensure_dynamic_smem(kern, pl.smem, configured_cluster[p.G <= 4]));
    b2l_hang_arm(st);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = pl.smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kCluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = b2l_pdl_enabled() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kern, p);
    B2L_LAUNCH_CHECK();
    return B2L_OK;
  }
  static int configured[2][64] = {{0}};
  auto kern = p.G <= 4 ? kv4_decode_kernel<T, D, GS, true, false> : kv4_decode_kernel<T, D, GS, false, false>;
  B2L_CUDA_CHECK(b2l_ensure_dynamic_smem(kern, pl.smem, configured[p.G <= 4]));
  b2l_launch(kern, grid, block, (size_t)pl.smem, st, p);
  B2L_LAUNCH_CHECK();
  // many parts to a row, or few: 16 warps to a head, or one (2 rows of 30000 tokens: 19.4 and 38.7 us; 32 rows of 1000 - 2000: 39.0 and 30.3)
  if ((int64_t)pl.grid > 24 * (int64_t)p.batch)
    b2l_launch(kv4_decode_merge_kernel<T, D, 16>, dim3((unsigned)p.batch, (unsigned)p.Hq), dim3(512), (size_t)0, st, p);
  else
    b2l_launch(kv4_decode_merge_kernel<T, D, 1>, dim3((unsigned)p.batch, (unsigned)((p.Hq + 3) / 4)), dim3(128), (size_t)0, st, p);
  B2L_LAUNCH_CHECK();
  return B2L_OK;
}

int64_t part_rows(const Int4Plan& pl, int G) { return 2ll * pl.grid * pl.HB * G; }

}  // namespace

extern "C" int64_t b2l_flash_decoding_int4_workspace_bytes(int64_t batch, int num_q_heads, int num_kv_heads, int head_dim, int group,
                                                           int64_t max_seq_len) {
  if (batch <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 || !kv4::shape_ok(head_dim, group)) return 0;
  const int G = num_q_heads / num_kv_heads;
  if (G > 8 * kMaxConsumers) return 0;
  const Int4Plan pl = make_plan(batch, G, num_kv_heads, head_dim, group, max_seq_len);
  const int64_t rows = batch < kMaxBatch ? batch : kMaxBatch;
  return part_rows(pl, G) * (head_dim + 2) * 4 + rows * (num_kv_heads / pl.HB) * 8 + 16;
}

extern "C" int b2l_flash_decoding_int4(void* out, const void* q, const void* cache, int64_t cache_row_stride, int64_t max_tokens,
                                       const void* b_req_tokens_table, int64_t table_req_stride, int64_t table_seq_stride,
                                       int64_t table_requests, int64_t table_width, const void* b_req_idx, int req_idx_width,
                                       const void* b_seq_len, int seq_len_width, int64_t batch, int num_q_heads, int num_kv_heads,
                                       int head_dim, int group, int64_t max_seq_len, float qk_scale, int64_t q_batch_stride,
                                       int64_t q_head_stride, int64_t o_batch_stride, int64_t o_head_stride, void* workspace,
                                       int64_t workspace_bytes, int dtype, void* stream) {
  B2L_REQUIRE(out && q && cache && b_req_tokens_table && b_req_idx && b_seq_len, "flash_decoding_int4: null pointer");
  B2L_REQUIRE(num_q_heads > 0 && num_kv_heads > 0 && num_q_heads % num_kv_heads == 0,
              "flash_decoding_int4: num_q_heads (%d) must be a multiple of num_kv_heads (%d)", num_q_heads, num_kv_heads);
  B2L_REQUIRE(num_q_heads / num_kv_heads <= 8 * kMaxConsumers, "flash_decoding_int4: more than %d query heads to a kv head", 8 * kMaxConsumers);
  B2L_REQUIRE(num_q_heads <= 65535, "flash_decoding_int4: too many heads");
  B2L_REQUIRE(kv4::shape_ok(head_dim, group), "flash_decoding_int4: head_dim %d with groups of %d (head_dim 32, 64 or 128; groups of 32, 64 or 128, at most head_dim)",
              head_dim, group);
  B2L_REQUIRE((req_idx_width == 4 || req_idx_width == 8) && (seq_len_width == 4 || seq_len_width == 8),
              "flash_decoding_int4: index widths must be 4 or 8");
  B2L_REQUIRE(cache_row_stride >= kv4::row_bytes(num_kv_heads, head_dim, group) && cache_row_stride % 16 == 0 && (uintptr_t)cache % 16 == 0,
              "flash_decoding_int4: cache rows must be 16-byte aligned and hold %lld bytes",
              (long long)kv4::row_bytes(num_kv_heads, head_dim, group));
  B2L_REQUIRE(dtype == B2L_F16 || dtype == B2L_BF16, "flash_decoding_int4: dtype %d", dtype);
  B2L_REQUIRE(batch >= 0 && max_tokens > 0 && table_requests >= 0 && table_width >= 0 && max_seq_len < (1ll << 31) - 256,
              "flash_decoding_int4: bad shape");
  if (batch == 0) return B2L_OK;
  const int G = num_q_heads / num_kv_heads, elem = 2;
  const Int4Plan pl = make_plan(batch, G, num_kv_heads, head_dim, group, max_seq_len);
  B2L_REQUIRE(pl.smem <= b2l_max_smem_optin(), "flash_decoding_int4: cache rows too long");
  B2L_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 &&
                  workspace_bytes >= b2l_flash_decoding_int4_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim, group, max_seq_len),
              "flash_decoding_int4: workspace too small");
  Int4DecodeParams p;
  p.q_bs = q_batch_stride; p.q_hs = q_head_stride; p.o_bs = o_batch_stride; p.o_hs = o_head_stride;
  p.cache = (const uint8_t*)cache; p.row_stride = cache_row_stride; p.max_tokens = max_tokens;
  p.table = (const int32_t*)b_req_tokens_table; p.tab_rs = table_req_stride; p.tab_cs = table_seq_stride;
  p.requests = table_requests; p.width = table_width;
  p.req_w = req_idx_width; p.len_w = seq_len_width;
  p.Hq = num_q_heads; p.Hkv = num_kv_heads; p.G = G; p.HB = pl.HB; p.qblocks = pl.qblocks; p.TS = pl.TS;
  p.stages = pl.stages; p.pitch = pl.pitch; p.nblk = num_kv_heads / pl.HB;
  for (p.TS_log2 = 0; 1 << p.TS_log2 < pl.TS;) ++p.TS_log2;     // a power of two
  p.most = max_seq_len < table_width ? max_seq_len : table_width;
  if (p.most < 0) p.most = 0;
  // the shares' sums, each row's kRowCost among them
  B2L_REQUIRE((batch < kMaxBatch ? batch : kMaxBatch) * (cdiv64(p.most, kUnit) + kRowCost) * num_kv_heads < (1ll << 31),
              "flash_decoding_int4: too many tokens");
  p.q_vec = (uintptr_t)q % 16 == 0 && q_batch_stride % 8 == 0 && q_head_stride % 8 == 0;
  p.scale_log2 = qk_scale * 1.4426950408889634f;
  p.ws_o = (float*)workspace;
  p.ws_ml = p.ws_o + part_rows(pl, G) * head_dim;
  p.ws_info = (int2*)(p.ws_ml + part_rows(pl, G) * 2);
  cudaStream_t st = (cudaStream_t)stream;
  for (int64_t b0 = 0; b0 < batch; b0 += kMaxBatch) {
    p.batch = (int)(batch - b0 < kMaxBatch ? batch - b0 : kMaxBatch);
    p.q = (const char*)q + b0 * q_batch_stride * elem;
    p.out = (char*)out + b0 * o_batch_stride * elem;
    p.req_idx = (const char*)b_req_idx + b0 * req_idx_width;
    p.seq_len = (const char*)b_seq_len + b0 * seq_len_width;
    int rc;
    if (dtype == B2L_F16) { KV4_DISPATCH_SHAPE(head_dim, group, { rc = launch_int4_decode<__half, D, GS>(p, pl, st); }); }
    else { KV4_DISPATCH_SHAPE(head_dim, group, { rc = launch_int4_decode<__nv_bfloat16, D, GS>(p, pl, st); }); }
    if (rc != B2L_OK) return rc;
  }
  return B2L_OK;
}
