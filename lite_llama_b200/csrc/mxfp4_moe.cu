// Routed experts in microscaled 4-bit floating point: tokens sorted by expert and back (the products: mxfp4_gemm.cu).
//
//   out[t] = sum_j weight[t, j] * down_e(silu(gate_e(x[t])) * up_e(x[t])),  e = ids[t, j]
//
// A slot (t, j) gets a row among its expert's; every expert's rows fill tiles of `tile` rows, and row r of tile i is row i tile + r of
// all buffers (with 64 rows to a tile row 128 i + r of their scales, so that a tile's scales start on a tile of their own).  Ids that name no expert get no
// row and add nothing.  A row's results do not depend on its place, so places are given out by atomics.
#include "mxfp4.cuh"
#include "pair.cuh"

namespace mx4 {

constexpr int kSortThreads = 1024;

// Ranks by counters in shared memory, tiles by a scan over experts.  Up to HELD slots a thread, whose ids are asked for together and stay in
// registers with their ranks; what is left goes through `place`.  CTAS > 1: a cluster parts the slots and adds up the counters, for
// the atomics of one CTA on a few addresses bound it (16000 slots over 128 experts: 9.1 us in one, with eight CTAs 5).
template <int HELD, int CTAS>
__global__ void __cluster_dims__(CTAS, 1, 1) __launch_bounds__(kSortThreads)
sort_kernel(int32_t* __restrict__ place, int32_t* __restrict__ table, const void* __restrict__ ids, int id_width, int slots, int tile,
            int experts) {
  extern __shared__ int counts[];      // of this CTA per expert, then the first row of its slots among all
  int* first = counts + experts;
  __shared__ int warp_sum[32], carry;
  pdl_prologue();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = CTAS == 1 ? 0 : (int)pair_rank();
  const int start = rank * kSortThreads + tid, step = CTAS * kSortThreads;
  for (int e = tid; e < experts; e += kSortThreads) counts[e] = 0;
  if (tid == 0) carry = 0;
  __syncthreads();
  auto expert_of = [&](int s) {
    const int64_t e = load_index(ids, s, id_width);
    return e >= 0 && e < experts ? (int)e : -1;
  };
  int held[HELD], at[HELD];
#pragma unroll
  for (int i = 0; i < HELD; ++i) held[i] = start + i * step < slots ? expert_of(start + i * step) : -1;
#pragma unroll
  for (int i = 0; i < HELD; ++i) at[i] = held[i] >= 0 ? atomicAdd(&counts[held[i]], 1) : -1;
  for (int s = start + HELD * step; s < slots; s += step) {
    const int e = expert_of(s);
    place[s] = e >= 0 ? atomicAdd(&counts[e], 1) : -1;
  }
  if (CTAS == 1) __syncthreads();
  else pair_sync();                    // all counters of the cluster
  for (int base = 0; base < experts; base += kSortThreads) {
    const int e = base + tid;
    int all = 0, before = 0;
    if (e < experts) {
      if (CTAS == 1) {
        all = counts[e];
      } else {
        uint32_t n[CTAS];
#pragma unroll
        for (int c = 0; c < CTAS; ++c) n[c] = ld_cluster_32(cluster_addr(counts + e, (uint32_t)c));
#pragma unroll
        for (int c = 0; c < CTAS; ++c) {
          if (c < rank) before += (int)n[c];
          all += (int)n[c];
        }
      }
    }
    const int tiles = (all + tile - 1) / tile;
    int sum = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      int w = warp_sum[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += up;
      }
      warp_sum[lane] = w;
    }
    __syncthreads();
    const int tile0 = carry + (warp ? warp_sum[warp - 1] : 0) + sum - tiles;
    if (e < experts) {
      first[e] = tile0 * tile + before;
      if (rank == 0) {
        for (int i = 0; i < tiles; ++i) {
          table[1 + 2 * (tile0 + i)] = e;
          table[2 + 2 * (tile0 + i)] = all - i * tile < tile ? all - i * tile : tile;
        }
      }
    }
    __syncthreads();
    if (tid == 0) carry += warp_sum[31];
    __syncthreads();
  }
  if (rank == 0 && tid == 0) table[0] = carry;
#pragma unroll
  for (int i = 0; i < HELD; ++i)
    if (start + i * step < slots) place[start + i * step] = held[i] >= 0 ? at[i] + first[held[i]] : -1;
  for (int s = start + HELD * step; s < slots; s += step) {
    const int e = expert_of(s);
    if (e >= 0) place[s] += first[e];
  }
  if (CTAS > 1) pair_sync();           // the peers have read this CTA's counters
}

// What sort_kernel gives for up to 32 slots, a lane each, by one warp: the lane's place.  An expert has one tile; `write`: place and table, too.
__device__ __forceinline__ int place_of_few(int32_t* place, int32_t* table, const void* ids, int id_width, int slots, int tile, int experts, bool write) {
  const int lane = threadIdx.x & 31;
  int64_t id = -1;
  if (lane < slots) id = load_index(ids, lane, id_width);
  const int e = id >= 0 && id < experts ? (int)id : -1;
  const uint32_t same = __match_any_sync(0xffffffffu, e), below = (1u << lane) - 1u;
  const uint32_t firsts = __ballot_sync(0xffffffffu, e >= 0 && (same & below) == 0u);
  int before = 0;                      // experts with a smaller number
#pragma unroll
  for (int o = 0; o < 32; ++o) {
    const int other = __shfl_sync(0xffffffffu, e, o);      // by the set bits, one after another: 1 us for 28 experts
    before += other < e ? (int)(firsts >> o & 1u) : 0;
  }
  const int to = e >= 0 ? before * tile + __popc(same & below) : -1;
  if (write) {
    if (lane < slots) place[lane] = to;
    if (firsts >> lane & 1u) {
      table[1 + 2 * before] = e;
      table[2 + 2 * before] = __popc(same);
    }
    if (lane == 0) table[0] = __popc(firsts);
  }
  return to;
}

// A token's row quantised once, as quantize_kernel does (mxfp4_quant.cu), and written to the rows of all its slots.
// Two units of 256 elements to a warp (U): the lanes of a block exchange codes, so that two of them have each unit's, 8 bytes a lane.
// FEW: every warp finds the places itself.
template <typename T, int U, bool FEW>
__global__ void __launch_bounds__(256)
scatter_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, const T* __restrict__ x, int32_t* __restrict__ place,
               int32_t* __restrict__ table, const void* __restrict__ ids, int id_width, int experts, uint32_t tokens, int top_k, uint32_t tile,
               uint32_t k, int64_t x_stride, int64_t ktiles, uint32_t units) {
  pdl_prologue();
  const int lane = threadIdx.x & 31;
  const uint32_t u = blockIdx.x * 8 + (threadIdx.x >> 5), row = u / units;
  if (row >= tokens) return;                           // whole warps
  const uint32_t first = (u - row * units) * (32 * U), chunks = k / 8;      // chunks of eight elements
  const T* src = x + row * x_stride + (int64_t)(first + lane) * 8;
  Raw8<T> v[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    zero_raw(v[i]);
    if (first + lane + 32 * i < chunks) load_raw(src + 256 * i, v[i]);
  }
  int mine;                            // the row's first 32 slots, a lane each; FEW: all slots
  if (FEW) mine = place_of_few(place, table, ids, id_width, (int)tokens * top_k, (int)tile, experts, u == 0);
  else mine = lane < top_k ? ld_upstream(place + (int64_t)row * top_k + lane) : -1;
  uint32_t code[U], byte[U];
#pragma unroll
  for (int i = 0; i < U; ++i) code[i] = quantise_raw(v[i], byte[i]);
  uint32_t block = (first + lane) >> 2;
  uint2 both = make_uint2(code[0], 0u);
  bool scaled = (lane & 3) == 0, in = first + lane < chunks;
  uint32_t at = (first + lane) * 4;
  if constexpr (U == 2) {
    // lane 4 b + j: bytes 8 (j & 1) of block b of unit j / 2, the codes of lanes 4 b + 2 (j & 1) and the next
    const int from = (lane & 28) | ((lane & 1) << 1);
    const uint32_t a0 = __shfl_sync(0xffffffffu, code[0], from), a1 = __shfl_sync(0xffffffffu, code[1], from);
    const uint32_t b0 = __shfl_sync(0xffffffffu, code[0], from + 1), b1 = __shfl_sync(0xffffffffu, code[1], from + 1);
    const bool second = (lane & 2) != 0;
    both = second ? make_uint2(a1, b1) : make_uint2(a0, b0);
    if (second) { byte[0] = byte[1]; block += 8; }
    scaled = (lane & 1) == 0;
    in = block < k / 32;
    at = block * 16 + (lane & 1) * 8;
  }
  const uint32_t half = tile == 64 ? ~63u : 0u;        // of tiles of 64 rows each has a tile of scales
  scaled = scaled && block < ((k / 32 + 3) & ~3u);
  uint8_t* out = codes + at;
  uint8_t* scale = scales + (block >> 2) * kTileBytes + (block & 3);
  for (int j = 0; j < top_k; ++j) {
    if (!FEW && j > 0 && (j & 31) == 0) mine = j + lane < top_k ? ld_upstream(place + (int64_t)row * top_k + j + lane) : -1;
    const int to = __shfl_sync(0xffffffffu, mine, FEW ? (int)row * top_k + j : j & 31);
    if (to < 0) continue;                              // whole warps
    if (in) {
      if (U == 2) *reinterpret_cast<uint2*>(out + (int64_t)to * (k / 2)) = both;
      else *reinterpret_cast<uint32_t*>(out + (int64_t)to * (k / 2)) = code[0];
    }
    if (scaled) scale[scale_word((int64_t)to + (to & half), 0, ktiles)] = (uint8_t)byte[0];
  }
}

// A token's expert rows (32 bits, in one piece or, SPLIT, in two planes of 16), weighted, added up in the order of its choices in 32 bits; eight
// outputs a thread.
template <typename T, typename W, bool SPLIT>
__global__ void __launch_bounds__(128)
combine_kernel(T* __restrict__ out, const void* __restrict__ y, const void* __restrict__ y_low, const int32_t* __restrict__ place,
               const W* __restrict__ weights, int64_t tokens, int top_k, int64_t n) {
  pdl_prologue();
  const uint32_t chunks = (uint32_t)(n / 8), i = blockIdx.x * 128 + threadIdx.x;
  if (i >= tokens * chunks) return;
  const uint32_t t = i / chunks, c = i - t * chunks;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int j0 = 0; j0 < top_k; j0 += 8) {              // eight rows requested together
    uint4 q[8], r[8];                  // upper and lower halves, or the first four and the others
    float w[8];
    int from[8];                       // all places first: one after another each would wait for the row before
#pragma unroll
    for (int j = 0; j < 8; ++j) from[j] = j0 + j < top_k ? ld_upstream(place + (int64_t)t * top_k + j0 + j) : -1;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      q[j] = r[j] = make_uint4(0u, 0u, 0u, 0u);
      w[j] = 0.f;
      if (from[j] >= 0) {
        const int64_t at = (int64_t)from[j] * n + c * 8;
        if (SPLIT) {
          q[j] = ldg_stream_128(reinterpret_cast<const uint16_t*>(y) + at);
          r[j] = ldg_stream_128(reinterpret_cast<const uint16_t*>(y_low) + at);
        } else {
          q[j] = ldg_stream_128(reinterpret_cast<const float*>(y) + at);
          r[j] = ldg_stream_128(reinterpret_cast<const float*>(y) + at + 4);
        }
        w[j] = to_f32(weights[(int64_t)t * top_k + j0 + j]);
      }
    }
    auto add = [&](int j) {
      const uint32_t *a = reinterpret_cast<const uint32_t*>(&q[j]), *b = reinterpret_cast<const uint32_t*>(&r[j]);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        if (SPLIT) {
          sum[2 * h] = fmaf(w[j], __uint_as_float(__byte_perm(b[h], a[h], 0x5410)), sum[2 * h]);
          sum[2 * h + 1] = fmaf(w[j], __uint_as_float(__byte_perm(b[h], a[h], 0x7632)), sum[2 * h + 1]);
        } else {
          sum[h] = fmaf(w[j], __uint_as_float(a[h]), sum[h]);
          sum[4 + h] = fmaf(w[j], __uint_as_float(b[h]), sum[4 + h]);
        }
      }
    };
    // by fours where issue is the bound, one by one where latency is
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (SPLIT || j0 + j < top_k) add(j);
    if (j0 + 4 < top_k) {
#pragma unroll
      for (int j = 4; j < 8; ++j)
        if (SPLIT || j0 + j < top_k) add(j);
    }
  }
  stg_128(out + (int64_t)t * n + c * 8, make_uint4(pack2<T>(sum[0], sum[1]), pack2<T>(sum[2], sum[3]), pack2<T>(sum[4], sum[5]), pack2<T>(sum[6], sum[7])));
}

template <typename T>
static int combine(void* out, const void* y, const void* y_low, const void* place, const void* weights, int wide, int64_t tokens, int top_k,
                   int64_t n, cudaStream_t st) {
  const dim3 grid((unsigned)cdiv64(tokens * (n / 8), 128));
#define COMBINE(W, SPLIT)                                                                                                              \
  b2l_launch(combine_kernel<T, W, SPLIT>, grid, dim3(128), (size_t)0, st, (T*)out, y, y_low, (const int32_t*)place, (const W*)weights, tokens, \
             top_k, n)
  if (y_low) {
    if (wide) COMBINE(float, true);
    else COMBINE(T, true);
  } else {
    if (wide) COMBINE(float, false);
    else COMBINE(T, false);
  }
#undef COMBINE
  B2L_LAUNCH_CHECK();
  return B2L_OK;
}

}  // namespace mx4

// Rows of an expert's tile.  64: the weights are the MMA's rows, for few rows an expert (or of few outputs, n of them in the first product); 128: the
// tokens are, in 256: on a pair of CTAs that share the weights (whole call, us, 64 / 128 / 256; 128 experts of 2048 x 768: 24 rows each 78 / 87,
// 48 94 / 94, 64 108 / 102 / 116, 256 318 / 209 / 212, 320 390 / 247 / 248, 1024 1191 / 702 / 708; 8 of 4096 x 1792: 320
// 84 / 71 / 66, 1024 228 / 152 / 143; 8 of 256 x 128, a quarter as many tiles as SMs: 512 17.2 / 21.1, half as many: 1024 23.8 / 22.7).
extern "C" int64_t b2l_mxfp4_moe_tile_rows(int64_t slots, int experts, int64_t n) {
  if (slots <= 800 || slots <= 48LL * experts || cdiv64(slots, 128) * cdiv64(n, 256) * 4 <= b2l_num_sms()) return 64;
  return slots < 320LL * experts ? 128 : 256;
}

extern "C" int64_t b2l_mxfp4_moe_max_tiles(int64_t slots, int tile_rows, int experts) {
  if (slots <= 0 || tile_rows <= 0 || experts <= 0) return 0;
  return slots / tile_rows + (slots < experts ? slots : experts);
}

extern "C" int b2l_mxfp4_moe_scatter(void* place, void* table, void* codes, void* scales, const void* x, const void* topk_ids, int id_width,
                                     int64_t tokens, int top_k, int tile_rows, int experts, int64_t k, int64_t x_row_stride, int dtype,
                                     void* stream) {
  B2L_REQUIRE(id_width == 4 || id_width == 8, "mxfp4_moe_scatter: topk_ids must be int32 or int64");
  B2L_REQUIRE(tokens >= 0 && top_k > 0 && top_k < (1 << 24) && tokens < (1ll << 24) && tokens * top_k < (1ll << 24) && experts > 0 && experts <= 4096,
              "mxfp4_moe_scatter: %lld tokens of %d slots over %d experts", (long long)tokens, top_k, experts);
  B2L_REQUIRE((tile_rows == 64 || tile_rows == 128 || tile_rows == 256) && k > 0 && k % 32 == 0 && k < (1ll << 30),
              "mxfp4_moe_scatter: tiles of %d rows, k=%lld (a multiple of 32)", tile_rows, (long long)k);
  if (tokens == 0) return B2L_OK;
  B2L_REQUIRE(place && table && topk_ids && codes && scales && x, "mxfp4_moe_scatter: null pointer");
  B2L_REQUIRE((uintptr_t)x % 16 == 0 && x_row_stride % 8 == 0 && (uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 4 == 0,
              "mxfp4_moe_scatter: rows must start on 16 bytes");
  B2L_REQUIRE(dtype == B2L_F16 || dtype == B2L_BF16, "mxfp4_moe_scatter: dtype %d", dtype);
  const int slots = (int)(tokens * top_k);
  // up to 32 slots in one launch (whole call, two -> one, us: 8 of 128 experts of 2048 x 768 16.4 -> 14.3, four tokens
  // 25.9 -> 24.0; 2 of 8 of 4096 x 1792 17.6 -> 15.4)
  const bool few = slots <= 32;
  // one unit a warp where there are few, or one to a row (one / two, us, 8 slots a token: 32 x 2048 2.1 / 2.2, 200 2.7 / 2.4, 2000 8.6 / 6.5, 8000
  // 29 / 22; two slots: 2000 x 4096 8.6 / 6.2, 4000 x 256 2.5 / 2.9)
  const int per_warp = few || k <= 256 || tokens * cdiv64(k, 256) < 8LL * b2l_num_sms() ? 1 : 2;
  const int64_t units = cdiv64(k, 256 * per_warp), grid = cdiv64(tokens * units, 8);
  B2L_REQUIRE(tokens * units < (1ll << 31), "mxfp4_moe_scatter: too many tokens");
  if (!few) {
    const bool many = slots > 4 * mx4::kSortThreads;
    auto kern = many ? mx4::sort_kernel<4, 8> : (slots <= mx4::kSortThreads ? mx4::sort_kernel<1, 1> : mx4::sort_kernel<4, 1>);
    b2l_launch(kern, dim3(many ? 8 : 1), dim3(mx4::kSortThreads), (size_t)experts * 8, (cudaStream_t)stream, (int32_t*)place, (int32_t*)table,
               topk_ids, id_width, slots, tile_rows, experts);
    B2L_LAUNCH_CHECK();
  }
#define SCATTER(T)                                                                                                                       \
  b2l_launch(few ? mx4::scatter_kernel<T, 1, true> : (per_warp == 1 ? mx4::scatter_kernel<T, 1, false> : mx4::scatter_kernel<T, 2, false>), \
             dim3((unsigned)grid), dim3(256), (size_t)0, (cudaStream_t)stream, (uint8_t*)codes, (uint8_t*)scales, (const T*)x, (int32_t*)place, \
             (int32_t*)table, topk_ids, id_width, experts, (uint32_t)tokens, top_k, (uint32_t)tile_rows, (uint32_t)k, x_row_stride,           \
             mx4::k_tiles(k), (uint32_t)units)
  if (dtype == B2L_F16) SCATTER(__half);
  else SCATTER(__nv_bfloat16);
#undef SCATTER
  B2L_LAUNCH_CHECK();
  return B2L_OK;
}

extern "C" int b2l_mxfp4_moe_combine(void* out, const void* y, const void* y_low, const void* place, const void* weights, int weights_f32, int64_t tokens,
                                     int top_k, int64_t n, int dtype, void* stream) {
  B2L_REQUIRE(tokens >= 0 && top_k > 0 && n > 0 && n % 8 == 0 && tokens * (n / 8) < (1ll << 31), "mxfp4_moe_combine: tokens=%lld n=%lld (a multiple of 8)",
              (long long)tokens, (long long)n);
  if (tokens == 0) return B2L_OK;
  B2L_REQUIRE(out && y && place && weights && ((uintptr_t)out | (uintptr_t)y | (uintptr_t)y_low) % 16 == 0, "mxfp4_moe_combine: null or misaligned pointer");
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == B2L_F16) return mx4::combine<__half>(out, y, y_low, place, weights, weights_f32, tokens, top_k, n, st);
  if (dtype == B2L_BF16) return mx4::combine<__nv_bfloat16>(out, y, y_low, place, weights, weights_f32, tokens, top_k, n, st);
  B2L_UNSUPPORTED("mxfp4_moe_combine: dtype %d", dtype);
}
