// Y = X W^T with both operands in microscaled 4-bit floating point, for up to 128 tokens (and for what the pair kernel leaves).
//
//   Y[t, n] = sum over blocks b of 2^(sx[t, b] + sw[n, b] - 254) * sum_i ex[t, 32 b + i] * ew[n, 32 b + i]
//
// The products of elements are exact, scales are powers of two, sums are in 32 bits on the tensor cores; rounded once.
//
// Bound: with few tokens the weights (17/32 bytes an element) are what streams.  128 weight rows are the rows of the MMA (they are
// most of the bytes), 32, 64 or 128 tokens its columns, so the tensor pipe is idle nearly always and the kernel is a ring of TMA copies: a CTA has
// four stages of 256 k (90 - 105 KiB) in flight and two CTAs share an SM.  A tile whose n leaves SMs idle is parted along k
// over a cluster of 2, 4 or 8 CTAs, whose sums are added up in shared memory in the order of the parts: nothing outlives the
// launch, so calls on several streams and captured graphs share nothing.  Up to 32 tokens every CTA sends its sums of a token to the CTA that
// owns it (st.async, counted by the owner's barrier), which is one way through the cluster; with more they lie where they are, between
// two barriers of the cluster, and each CTA fetches a share of the tile (one token, 4096 x 4096, us: 3.6 that way, 3.3 so).
#include "gemm_tc.cuh"
#include "mxfp4_mma.cuh"
#include "mxfp4_gemm.cuh"
#include "pair.cuh"

namespace mx4 {

constexpr int kThreads = 6 * 32;       // TMA producer, MMA issuer, four warps that read the accumulator

struct Params {
  void* y; int64_t ldy;                // [T, N] 16-bit, or the codes [T, N / 4] of silu(gate) * up
  uint8_t* y_scales; int64_t y_ktiles;
  const void* bias;                    // [N] in the output's type, or null
  const uint8_t* x_scales; const uint8_t* w_scales;
  const void* x16; int64_t ldx16;      // activations that the kernel quantises itself
  int64_t ktiles;                      // scale tiles along k
  int T, N, K, num_kb;
  int early;                           // weights may be requested before the previous kernel has ended
  int vec;                             // 8-byte stores of y
};

constexpr int kRawTokens = 8;          // activations that the kernel quantises itself: up to so many rows,
constexpr int kRawStages = 24;         // so many stages of 256 k of a CTA's part, and so many of both together

template <int BT, bool RAW> struct Ring {
  static constexpr int kStages = BT == 128 ? 3 : 4;
  static constexpr int kStage = 16384 + kSfBytes + (RAW ? 0 : BT * 128 + kSfBytes);   // W, its scales, X, its scales
  // RAW: X of all stages stays, eight rows of 128 bytes each and for every scale tile eight rows of 16; the MMA's columns from 8 on read
  // what follows, whatever it is, and are not looked at
  static constexpr int kRaw = kStages * kStage, kRawScales = kRaw + (kRawStages + 3) * 1024;
  static constexpr int kX = 16384 + kSfBytes;
  // Up to 32 tokens: [token of this CTA][part of k][128] sums
  static constexpr int kSums = RAW ? kRawScales + (2 * kRawStages + 3) * 128 : kStages * kStage;
  static constexpr int kSumBytes = BT == 32 ? (RAW ? kRawTokens : 32) * 512 : 0;
  static constexpr int kCols = BT + kStages * 16;                         // accumulator, then 16 columns of scales a stage
  static constexpr int kAlloc = kCols <= 128 ? 128 : 256;
  static constexpr int kSmem = 1024 + 1024 + kSums + kSumBytes;
};

struct __align__(8) Control {
  uint64_t full[8], empty[8], done, raw, sums;
  uint32_t tmem;
};

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}

// Four outputs of a token from their sums
template <typename T> __device__ __forceinline__ void store4(const Params& p, int64_t row, int n, float (&v)[4]) {
  T* out = reinterpret_cast<T*>(p.y) + row * p.ldy + n;
  const T* bias = reinterpret_cast<const T*>(p.bias);
  if (bias)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < p.N) v[j] += to_f32(bias[n + j]);
  if (p.vec && n < p.N) {              // N is a multiple of four
    *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < p.N) out[j] = from_f32<T>(v[j]);
  }
}
// Four activations of a token from the sums of their gate and up rows, e to e + 3 of the tile's 64; eight lanes hold a block (whole warps)
template <typename T>
__device__ __forceinline__ void store_unit4(const Params& p, bool in, int64_t row, int tile, int e, float (&g)[4], float (&u)[4], int lane) {
  const T* bias = p.bias ? reinterpret_cast<const T*>(p.bias) + (int64_t)tile * 128 + e : nullptr;
  uint32_t byte, code[1];
  quantise_unit<4, T>(g, u, bias, in, code, byte);
  if (!in) return;
  const int k = tile * 64 + e;
  *reinterpret_cast<uint16_t*>(reinterpret_cast<uint8_t*>(p.y) + row * p.ldy + k / 2) = (uint16_t)code[0];
  if ((lane & 7) == 0) {
    uint8_t* word = p.y_scales + scale_word(row, k >> 7, p.y_ktiles);
    word[(k >> 5) & 3] = (uint8_t)byte;
    // an odd number of tiles: the second half of the last word lies behind the end
    if (tile * 128 + 128 >= p.N && (tile & 1) == 0) word[((k >> 5) & 3) + 2] = 0;
  }
}

// This CTA's share of a tile: sums over the S parts of k in their order, all parts of an output asked for together (one after another
// they cost a trip to the other SM each: 128 tokens, 4096 x 4096, gated 13.1 us).  `sums`: [token][128] in every CTA of the cluster.
template <typename T, bool GATED, int S>
__device__ __forceinline__ void add_up(const Params& p, const uint8_t* sums, int tile, int m0, int tokens, uint32_t rank) {
  const int lane = threadIdx.x & 31;
  uint32_t base[S];
#pragma unroll
  for (int s = 0; s < S; ++s) base[s] = cluster_addr(sums, (uint32_t)s);
  if (!GATED) {
    // four outputs a thread
    for (int i = threadIdx.x + kThreads * rank; i < tokens * 32; i += kThreads * S) {
      const int t = i >> 5, n = tile * 128 + (i & 31) * 4;
      uint4 q[S];
#pragma unroll
      for (int s = 0; s < S; ++s) q[s] = ld_cluster_128(base[s] + i * 16);
      float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < S; ++s) {
        v[0] += __uint_as_float(q[s].x);
        v[1] += __uint_as_float(q[s].y);
        v[2] += __uint_as_float(q[s].z);
        v[3] += __uint_as_float(q[s].w);
      }
      store4<T>(p, m0 + t, n, v);
    }
  } else {
    // four activations a lane, eight lanes a block, two blocks a tile: 64 gate rows, then their up rows
    const int tasks = tokens * 16;
    for (int first = (int)(threadIdx.x & ~31u) + kThreads * (int)rank; first < tasks; first += kThreads * S) {
      const int i = first + lane, t = i >> 4, e = (i & 15) * 4;
      const bool in = i < tasks;
      float g[4] = {0.f, 0.f, 0.f, 0.f}, u[4] = {0.f, 0.f, 0.f, 0.f};
      if (in) {
        uint4 q[S], r[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
          q[s] = ld_cluster_128(base[s] + (t * 128 + e) * 4);
          r[s] = ld_cluster_128(base[s] + (t * 128 + 64 + e) * 4);
        }
#pragma unroll
        for (int s = 0; s < S; ++s) {
          g[0] += __uint_as_float(q[s].x); g[1] += __uint_as_float(q[s].y); g[2] += __uint_as_float(q[s].z); g[3] += __uint_as_float(q[s].w);
          u[0] += __uint_as_float(r[s].x); u[1] += __uint_as_float(r[s].y); u[2] += __uint_as_float(r[s].z); u[3] += __uint_as_float(r[s].w);
        }
      }
      store_unit4<T>(p, in, m0 + t, tile, e, g, u, lane);
    }
  }
}

// The tokens rank, rank + S, ... of a tile from their parts, [token][part][128] in this CTA: as add_up, by the 128 threads of four warps.
template <typename T, bool GATED, int S>
__device__ __forceinline__ void add_own(const Params& p, const float* sums, int tile, int rank, int tid) {
  const int lane = tid & 31, owned = p.T > rank ? (p.T - rank + S - 1) / S : 0;
  if (!GATED) {
    for (int i = tid; i < owned * 32; i += 128) {
      const int slot = i >> 5, n = tile * 128 + (i & 31) * 4;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const float4 q = *reinterpret_cast<const float4*>(sums + (slot * S + s) * 128 + (i & 31) * 4);
        v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
      }
      store4<T>(p, rank + slot * S, n, v);
    }
  } else {
    const int tasks = owned * 16;
    for (int first = tid & ~31; first < tasks; first += 128) {
      const int i = first + lane, slot = i >> 4, e = (i & 15) * 4;
      float g[4] = {0.f, 0.f, 0.f, 0.f}, u[4] = {0.f, 0.f, 0.f, 0.f};
      if (i < tasks) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const float* src = sums + (slot * S + s) * 128 + e;
          const float4 q = *reinterpret_cast<const float4*>(src), r = *reinterpret_cast<const float4*>(src + 64);
          g[0] += q.x; g[1] += q.y; g[2] += q.z; g[3] += q.w;
          u[0] += r.x; u[1] += r.y; u[2] += r.z; u[3] += r.w;
        }
      }
      store_unit4<T>(p, i < tasks, rank + slot * S, tile, e, g, u, lane);
    }
  }
}

__device__ __forceinline__ void send_f32(uint32_t to, float v, uint32_t bar) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(to), "r"(__float_as_uint(v)), "r"(bar) : "memory");
}

// A thread's output row over all tokens, each to the CTA that owns the token; then this CTA's tokens.
template <typename T, bool GATED, int S>
__device__ __forceinline__ void send_and_add(const Params& p, const uint32_t (&v)[32], float* sums, uint64_t* bar, int tile, int rank, int tid) {
  if (S == 1) {
#pragma unroll
    for (int t = 0; t < 32; ++t)
      if (t < p.T) sums[t * 128 + tid] = __uint_as_float(v[t]);
    asm volatile("bar.sync 1, 128;" ::: "memory");
  } else {
    uint32_t to[S], done[S];
#pragma unroll
    for (int c = 0; c < S; ++c) {
      to[c] = cluster_addr(sums, (uint32_t)c) + (rank * 128 + tid) * 4;
      done[c] = cluster_addr(bar, (uint32_t)c);
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");        // every CTA of the cluster runs and expects its sums
#pragma unroll
    for (int t = 0; t < 32; ++t)
      if (t < p.T) send_f32(to[t % S] + (t / S) * S * 512, __uint_as_float(v[t]), done[t % S]);
    if (rank < p.T) mbar_wait(bar, 0);
  }
  pdl_wait_prior();                    // y may still be read upstream
  add_own<T, GATED, S>(p, sums, tile, rank, tid);
}

// The rows of x in this CTA's part of k, quantised by the four warps that wait for the accumulator anyway: one launch less than with the quantiser
// by itself, and the same codes.  It pays while a warp has few units of 256 elements to do (quantiser and product -> this, us: one token, 6144 x
// 4096 5.1 -> 4.5, 4096 x 14336 8.2 -> 7.6; four tokens, 6144 x 4096, 16 units to a CTA, 5.3 -> 4.8; eight, 32 units, 5.4 -> 5.6; eight, 28672 x 4096,
// 128 units, 12.5 -> 17.9).
template <typename T, int BT>
__device__ __forceinline__ void quantise_rows(const Params& p, uint8_t* ring, int kb0, int stages, int warp, int lane) {
  using R = Ring<BT, true>;
  const T* x = reinterpret_cast<const T*>(p.x16);
  const int units = stages * p.T;
#pragma unroll 1
  for (int first = warp; first < units; first += 16) {           // four units of 256 k asked for together
    Raw8<T> v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int u = first + 4 * i, t = u / stages, k = (kb0 + u - t * stages) * kStageK + lane * 8;
      zero_raw(v[i]);
      if (u < units && k < p.K) load_raw(x + t * p.ldx16 + k, v[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int u = first + 4 * i, t = u / stages, s = u - t * stages;
      uint32_t byte;
      const uint32_t code = quantise_raw(v[i], byte);
      if (u >= units) break;                                     // whole warps
      *reinterpret_cast<uint32_t*>(ring + R::kRaw + s * 1024 + t * 128 + (((lane >> 2) ^ t) << 4) + (lane & 3) * 4) = code;
      if ((lane & 3) == 0) ring[R::kRawScales + (2 * s + (lane >> 4)) * 128 + t * 16 + ((lane >> 2) & 3)] = (uint8_t)byte;
    }
  }
}

template <typename T, int BT, bool GATED, bool RAW>
__global__ void __launch_bounds__(kThreads, 2)
stream_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const Params p) {
  using R = Ring<BT, RAW>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  Control* ctl = reinterpret_cast<Control*>(smem);
  uint8_t* ring = smem + 1024;
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;      // uniform (mxfp4_gemm_pair.cu)
  const uint32_t S = cluster_size(), rank = pair_rank();
  const int tile = blockIdx.x / S, m0 = blockIdx.y * BT;
  const int kb0 = (int)((int64_t)p.num_kb * rank / S), kb1 = (int)((int64_t)p.num_kb * (rank + 1) / S);
  if (warp == 0 && lane == 0) {
    if (!RAW) tma_prefetch_desc(&tmap_x);
    tma_prefetch_desc(&tmap_w);
    for (int s = 0; s < R::kStages; ++s) {
      mbar_init(&ctl->full[s], 1);
      mbar_init(&ctl->empty[s], 1);
    }
    mbar_init(&ctl->done, 1);
    mbar_init(&ctl->raw, 128);
    mbar_init(&ctl->sums, 1);
    mbar_fence_init();
    if (BT == 32 && S > 1 && (int)rank < p.T) mbar_arrive_expect_tx(&ctl->sums, (p.T - rank + S - 1) / S * S * 512);
  }
  __syncwarp();
  if (BT == 32 && S > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // waited for before the sums travel
  if (warp == 1) {
    tmem_alloc(&ctl->tmem, R::kAlloc);
    tmem_relinquish();
    pdl_launch_dependents();           // after the allocation: the next kernel's waits for this one's columns otherwise
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, ctl->tmem, 0);

  if (warp == 0) {
    // ===================== TMA producer =====================
    const uint8_t* ws = p.w_scales + (int64_t)tile * p.ktiles * kTileBytes;
    const uint8_t* xs = p.x_scales + (int64_t)(m0 >> 7) * p.ktiles * kTileBytes;
    auto sf_bytes = [&](int kb) { return (uint32_t)(2 * kb + 2 <= p.ktiles ? 2 : 1) * kTileBytes; };
    auto load_w = [&](int s, int kb) {
      uint8_t* st = ring + s * R::kStage;
      mbar_arrive_expect_tx(&ctl->full[s], RAW ? 16384 + sf_bytes(kb) : 16384 + BT * 128 + 2 * sf_bytes(kb));
      tma_load_2d_hint(st, &tmap_w, kb * 128, tile * 128, &ctl->full[s], kEvictFirst);
      bulk_g2s(st + 16384, ws + (int64_t)2 * kb * kTileBytes, sf_bytes(kb), &ctl->full[s]);
    };
    auto load_x = [&](int s, int kb) {
      if (RAW) return;
      uint8_t* st = ring + s * R::kStage + R::kX;
      tma_load_2d_hint(st, &tmap_x, kb * 128, m0, &ctl->full[s], kEvictLast);
      bulk_g2s(st + BT * 128, xs + (int64_t)2 * kb * kTileBytes, sf_bytes(kb), &ctl->full[s]);
    };
    const int pre = kb1 - kb0 < R::kStages ? kb1 - kb0 : R::kStages;
    if (!p.early) pdl_wait_prior();
    if (elect_one())
      for (int i = 0; i < pre; ++i) load_w(i, kb0 + i);
    __syncwarp();
    pdl_wait_prior();
    if (elect_one())
      for (int i = 0; i < pre; ++i) load_x(i, kb0 + i);
    __syncwarp();
    gemm::PipeState ps(R::kStages);
    for (int i = 0; i < pre; ++i) ps.advance();
    for (int kb = kb0 + pre; kb < kb1; ++kb) {
      mbar_wait(&ctl->empty[ps.stage], ps.phase ^ 1);
      if (elect_one()) {
        load_w(ps.stage, kb);
        load_x(ps.stage, kb);
      }
      __syncwarp();
      ps.advance();
    }
  } else if (warp == 1) {
    // ===================== MMA issuer =====================
    const uint64_t desc0 = umma_desc_sw128_kmajor(smem_u32(ring)), sf0 = scale_desc(smem_u32(ring));
    gemm::PipeState ps(R::kStages);
    if (RAW) mbar_wait(&ctl->raw, 0);
    for (int kb = kb0; kb < kb1; ++kb) {
      mbar_wait(&ctl->full[ps.stage], ps.phase);
      tc_fence_after();
      if (elect_one()) {
        const uint64_t base = (uint64_t)(ps.stage * R::kStage) >> 4;
        const uint64_t wd = desc0 + base, xd = RAW ? desc0 + ((R::kRaw + (kb - kb0) * 1024) >> 4) : wd + (R::kX >> 4);
        const uint64_t wsf = sf0 + base + (16384 >> 4);
        const uint64_t xsf = RAW ? sf0 + ((R::kRawScales + (kb - kb0) * 256) >> 4) : sf0 + base + ((R::kX + BT * 128) >> 4);
        const uint32_t sf = tmem + BT + ps.stage * 16;
        const int steps = (p.K - kb * kStageK + 63) >> 6;      // MMAs of 64 k that hold anything
        copy_scales<1>(sf, wsf);
        copy_scales<1>(sf + 8, xsf);
        if (steps > 2) {
          copy_scales<1>(sf + 4, wsf + (kTileBytes >> 4));
          copy_scales<1>(sf + 12, xsf + ((RAW ? 128 : kTileBytes) >> 4));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < steps)
            mma<1>(tmem, wd + 2 * j, xd + 2 * j, idesc(128, BT, j & 1), sf + (j >> 1) * 4, sf + 8 + (j >> 1) * 4,
                   (kb - kb0) | j ? 1u : 0u);
        tc_commit(kb + 1 == kb1 ? &ctl->done : &ctl->empty[ps.stage]);
      }
      __syncwarp();
      ps.advance();
    }
  } else {
    // ===================== this CTA's sums to shared memory, [token][128] =====================
    // done covers every MMA, and with it every copy into the ring: its memory is free
    const int quad = warp & 3;
    float* part = reinterpret_cast<float*>(ring) + quad * 32 + lane;
    if (RAW) {
      pdl_wait_prior();
      quantise_rows<T, BT>(p, ring, kb0, kb1 - kb0, quad, lane);
      fence_proxy_async_smem();
      mbar_arrive(&ctl->raw);
    }
    mbar_wait(&ctl->done, 0);
    tc_fence_after();
    if constexpr (BT == 32) {
      uint32_t v[32];
      tmem_ld_32x32b_x32(tmem + ((uint32_t)(quad * 32) << 16), v);
      tc_wait_ld();
      float* sums = reinterpret_cast<float*>(ring + R::kSums);
      const int tid = quad * 32 + lane;
      if (S == 1) send_and_add<T, GATED, 1>(p, v, sums, &ctl->sums, tile, (int)rank, tid);
      else if (S == 2) send_and_add<T, GATED, 2>(p, v, sums, &ctl->sums, tile, (int)rank, tid);
      else if (S == 4) send_and_add<T, GATED, 4>(p, v, sums, &ctl->sums, tile, (int)rank, tid);
      else send_and_add<T, GATED, 8>(p, v, sums, &ctl->sums, tile, (int)rank, tid);
    }
#pragma unroll 1
    for (int c = 0; BT != 32 && c < BT; c += 32) {
      if (m0 + c >= p.T) break;
      uint32_t v[32];
      tmem_ld_32x32b_x32(tmem + ((uint32_t)(quad * 32) << 16) + c, v);
      tc_wait_ld();
#pragma unroll
      for (int j = 0; j < 32; ++j) part[(c + j) * 128] = __uint_as_float(v[j]);
    }
  }
  tc_fence_before();
  if (BT == 32) {
    if (warp < 2 && S > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    __syncthreads();                   // the accumulator has been read
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(tmem, R::kAlloc);
    }
    return;
  }
  pair_sync();                         // all sums of the cluster are in place
  pdl_wait_prior();                    // y may still be read upstream
  const int tokens = p.T - m0 < BT ? p.T - m0 : BT;
  if (S == 1) add_up<T, GATED, 1>(p, ring, tile, m0, tokens, rank);
  else if (S == 2) add_up<T, GATED, 2>(p, ring, tile, m0, tokens, rank);
  else if (S == 4) add_up<T, GATED, 4>(p, ring, tile, m0, tokens, rank);
  else add_up<T, GATED, 8>(p, ring, tile, m0, tokens, rank);
  pair_sync_relaxed();                 // the peers have read this CTA's sums
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, R::kAlloc);
  }
}

// Parts of k: as many CTAs as keep every SM with two of them busy, two of two stages or more of four stages at least (one token,
// 4096 x 4096, us: eight parts of two stages 5.1, four of four 4.1; 6144 x 4096 four 5.0, two 5.6, eight 8.5 in two waves; 4096 x 14336 eight 7.6,
// four 8.2; 9728 x 896 two of two stages 3.7, one 3.9).
static int parts(int64_t tiles, int num_kb) {
  const int64_t room = 2 * b2l_num_sms();
  int s = 1;
  while (s < 8 && tiles * s * 2 <= room && num_kb >= (s == 1 ? 4 : 8 * s)) s *= 2;
  return s;
}

template <typename T, int BT, bool GATED, bool RAW>
static int launch(const CUtensorMap& tx, const CUtensorMap& tw, const Params& p, cudaStream_t st) {
  using R = Ring<BT, RAW>;
  auto kern = stream_kernel<T, BT, GATED, RAW>;
  static int configured[64] = {0};
  B2L_CUDA_CHECK(b2l_ensure_dynamic_smem(kern, R::kSmem, configured));
  const int64_t n_tiles = cdiv64(p.N, 128), m_tiles = cdiv64(p.T, BT);
  const int s = parts(n_tiles * m_tiles, p.num_kb);
  b2l_hang_arm(st);
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)(n_tiles * s), (unsigned)m_tiles);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = R::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)s;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = b2l_pdl_enabled() ? 2 : 1;
  B2L_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, tx, tw, p));
  B2L_LAUNCH_CHECK();
  return B2L_OK;
}

template <typename T>
static int stream_gemm(const void* x, int64_t x_stride, const void* w, int64_t w_stride, const Params& p, bool gated, cudaStream_t st) {
  const int bt = p.T <= 32 ? 32 : (p.T <= 64 ? 64 : 128);
  CUtensorMap tx, tw;
  int rc = b2l_make_tmap_2d(&tw, w, TMA_U8, (uint64_t)p.N, (uint64_t)p.K / 2, (uint64_t)w_stride, 128, 128, true);
  if (rc != B2L_OK) return rc;
  if (p.x16) return gated ? launch<T, 32, true, true>(tw, tw, p, st) : launch<T, 32, false, true>(tw, tw, p, st);
  rc = b2l_make_tmap_2d(&tx, x, TMA_U8, (uint64_t)p.T, (uint64_t)p.K / 2, (uint64_t)x_stride, (uint32_t)bt, 128, true);
  if (rc != B2L_OK) return rc;
#define STREAM(BT) (gated ? launch<T, BT, true, false>(tx, tw, p, st) : launch<T, BT, false, false>(tx, tw, p, st))
  return bt == 32 ? STREAM(32) : (bt == 64 ? STREAM(64) : STREAM(128));
#undef STREAM
}

// ---------------------------------------------------------------------------------------------------------------
// The same product for routed experts: tiles of up to 64 rows of one expert, {expert, rows} in a table on the device
// (mxfp4_moe.cu), row r of tile i in row 64 i + r of x and y and in row 128 i + r of their scales.
//
// Tiles of 128 rows or more are multiplied with the rows as the MMA's (mxfp4_gemm_pair.cu), where a thread holds a row's
// outputs: here its lane is an output, and bringing 128 columns out through shared memory took longer than the products (2000 tokens,
// 128 experts of 2048 x 768, both products 137 us, there 100).  Tiles of 32 rows were no faster at two rows an expert (58.7 against 56.1 us).
// Bound: the experts' weights, each read from memory once (further tiles of an expert find them in L2).  Persistent, one CTA to
// an SM with 180 KiB of copies in flight, the accumulator in two buffers: a tile's end overlaps the next one's products.
// ---------------------------------------------------------------------------------------------------------------
struct GroupedRing {
  static constexpr int BT = 64;        // rows of a tile
  static constexpr int kStage = 16384 + kSfBytes + BT * 128 + kSfBytes;
  static constexpr int kX = 16384 + kSfBytes;
  static constexpr int kStages = 7;
  static constexpr int kCols = 2 * BT + kStages * 16;
  static constexpr int kAlloc = 256;
  static constexpr int kOut = 32 * 128 * 4;
  static constexpr int kSmem = 1024 + 1024 + kStages * kStage + kOut;
};

struct GroupedParams {
  void* y; int64_t ldy;                // rows of 32-bit outputs (elements) or of codes (bytes)
  uint8_t* y_scales; int64_t y_ktiles;
  const uint8_t* x_scales; const uint8_t* w_scales;
  const int32_t* table;                // tiles, then {expert, rows} of each
  int64_t ktiles;
  int N, K, num_kb, n_tiles;
};

struct __align__(8) GroupedControl {
  uint64_t full[8], empty[8], acc_full[2], acc_empty[2];
  uint32_t tmem;
};

template <bool GATED>
__global__ void __launch_bounds__(kThreads, 1)
grouped_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const GroupedParams p) {
  using R = GroupedRing;
  constexpr int BT = R::BT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  GroupedControl* ctl = reinterpret_cast<GroupedControl*>(smem);
  uint8_t* ring = smem + 1024;
  float* out_stage = reinterpret_cast<float*>(ring + R::kStages * R::kStage);
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;      // uniform (mxfp4_gemm_pair.cu)
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmap_x);
    tma_prefetch_desc(&tmap_w);
    for (int s = 0; s < R::kStages; ++s) {
      mbar_init(&ctl->full[s], 1);
      mbar_init(&ctl->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&ctl->acc_full[b], 1);
      mbar_init(&ctl->acc_empty[b], 4);
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(&ctl->tmem, R::kAlloc);
    tmem_relinquish();
    pdl_launch_dependents();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, ctl->tmem, 0);
  pdl_wait_prior();                    // the table and the rows are upstream data
  const int items = ld_upstream(p.table) * p.n_tiles;

  if (warp == 0) {
    // ===================== TMA producer =====================
    gemm::PipeState ps(R::kStages);
    int next = (int)blockIdx.x < items ? ld_upstream(p.table + 1 + 2 * (blockIdx.x / p.n_tiles)) : 0;
    for (int it = blockIdx.x; it < items; it += gridDim.x) {
      const int tile = it / p.n_tiles, nt = it - tile * p.n_tiles;
      const int expert = next;
      if (it + (int)gridDim.x < items) next = ld_upstream(p.table + 1 + 2 * ((it + gridDim.x) / p.n_tiles));      // a tile ahead
      const int64_t w_tile = (int64_t)expert * p.n_tiles + nt;
      const uint8_t* ws = p.w_scales + w_tile * p.ktiles * kTileBytes;
      const uint8_t* xs = p.x_scales + (int64_t)tile * p.ktiles * kTileBytes;
      const int w_row = expert * p.N + nt * 128;
      for (int kb = 0; kb < p.num_kb; ++kb) {
        mbar_wait(&ctl->empty[ps.stage], ps.phase ^ 1);
        if (elect_one()) {
          uint8_t* st = ring + ps.stage * R::kStage;
          const uint32_t sf = (uint32_t)(2 * kb + 2 <= p.ktiles ? 2 : 1) * kTileBytes;
          uint64_t* full = &ctl->full[ps.stage];
          mbar_arrive_expect_tx(full, 16384 + BT * 128 + 2 * sf);
          tma_load_2d_hint(st, &tmap_w, kb * 128, w_row, full, kEvictNormal);
          bulk_g2s(st + 16384, ws + (int64_t)2 * kb * kTileBytes, sf, full);
          tma_load_2d_hint(st + R::kX, &tmap_x, kb * 128, tile * BT, full, kEvictLast);
          bulk_g2s(st + R::kX + BT * 128, xs + (int64_t)2 * kb * kTileBytes, sf, full);
        }
        __syncwarp();
        ps.advance();
      }
    }
  } else if (warp == 1) {
    // ===================== MMA issuer =====================
    const uint64_t desc0 = umma_desc_sw128_kmajor(smem_u32(ring)), sf0 = scale_desc(smem_u32(ring));
    gemm::PipeState ps(R::kStages);
    int turn = 0;
    for (int it = blockIdx.x; it < items; it += gridDim.x, ++turn) {
      const int buf = turn & 1;
      mbar_wait(&ctl->acc_empty[buf], ((turn >> 1) & 1) ^ 1);
      tc_fence_after();
      for (int kb = 0; kb < p.num_kb; ++kb) {
        mbar_wait(&ctl->full[ps.stage], ps.phase);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t base = (uint64_t)(ps.stage * R::kStage) >> 4;
          const uint64_t wd = desc0 + base, xd = wd + (R::kX >> 4);
          const uint64_t wsf = sf0 + base + (16384 >> 4), xsf = sf0 + base + ((R::kX + BT * 128) >> 4);
          const uint32_t sf = tmem + 2 * BT + ps.stage * 16;
          const int steps = (p.K - kb * kStageK + 63) >> 6;
          copy_scales<1>(sf, wsf);
          copy_scales<1>(sf + 8, xsf);
          if (steps > 2) {
            copy_scales<1>(sf + 4, wsf + (kTileBytes >> 4));
            copy_scales<1>(sf + 12, xsf + (kTileBytes >> 4));
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j < steps)
              mma<1>(tmem + buf * BT, wd + 2 * j, xd + 2 * j, idesc(128, BT, j & 1), sf + (j >> 1) * 4, sf + 8 + (j >> 1) * 4,
                     kb | j ? 1u : 0u);
          // nobody waits for the last stage of all, and no arrival may be on its way when the CTA leaves
          if (kb + 1 < p.num_kb || it + (int)gridDim.x < items) tc_commit(&ctl->empty[ps.stage]);
          if (kb + 1 == p.num_kb) tc_commit(&ctl->acc_full[buf]);
        }
        __syncwarp();
        ps.advance();
      }
    }
  } else {
    // ===================== four warps: 32 rows at a time through shared memory, [row][128] =====================
    const int quad = warp & 3, tid = quad * 32 + lane;
    float* mine = out_stage + quad * 32 + lane;
    int turn = 0;
    int next = (int)blockIdx.x < items ? ld_upstream(p.table + 2 + 2 * (blockIdx.x / p.n_tiles)) : 0;
    for (int it = blockIdx.x; it < items; it += gridDim.x, ++turn) {
      const int tile = it / p.n_tiles, nt = it - tile * p.n_tiles, buf = turn & 1;
      const int rows = next;
      if (it + (int)gridDim.x < items) next = ld_upstream(p.table + 2 + 2 * ((it + gridDim.x) / p.n_tiles));
      mbar_wait(&ctl->acc_full[buf], (turn >> 1) & 1);
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < BT; c += 32) {
        if (c < rows) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(tmem + ((uint32_t)(quad * 32) << 16) + buf * BT + c, v);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) mine[j * 128] = __uint_as_float(v[j]);
        }
        if (c + 32 == BT) {            // every row is on its way out: the accumulator is free
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctl->acc_empty[buf]);
        }
        if (c >= rows) continue;
        asm volatile("bar.sync 1, 128;" ::: "memory");
        const int here = rows - c < 32 ? rows - c : 32;
        if (!GATED) {
          for (int i = tid; i < here * 32; i += 128) {
            const int r = i >> 5, n = nt * 128 + (i & 31) * 4;
            if (n < p.N) stg_128(reinterpret_cast<float*>(p.y) + ((int64_t)tile * BT + c + r) * p.ldy + n, *reinterpret_cast<const uint4*>(out_stage + i * 4));
          }
        } else {
          for (int base = quad * 32; base < here * 8; base += 128) {
            const int i = base + lane, r = i >> 3, e = (i & 7) * 8;
            const bool in = i < here * 8;
            float g[8], u[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] = u[j] = 0.f;
            if (in) {
              const float* src = out_stage + r * 128 + e;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                g[j] = src[j];
                u[j] = src[64 + j];
              }
            }
            uint32_t byte, code[1];
            quantise_unit<8, __half>(g, u, nullptr, in, code, byte);
            if (in) {
              const int k = nt * 64 + e;
              *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(p.y) + ((int64_t)tile * BT + c + r) * p.ldy + k / 2) = code[0];
              if ((lane & 3) == 0) {
                uint8_t* word = p.y_scales + scale_word((int64_t)tile * 128 + c + r, k >> 7, p.y_ktiles);
                word[(k >> 5) & 3] = (uint8_t)byte;
                if (nt + 1 == p.n_tiles && (nt & 1) == 0) word[((k >> 5) & 3) + 2] = 0;
              }
            }
          }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, R::kAlloc);
  }
}

template <bool GATED>
static int launch_grouped(const CUtensorMap& tx, const CUtensorMap& tw, const GroupedParams& p, int64_t max_tiles, cudaStream_t st) {
  auto kern = grouped_kernel<GATED>;
  static int configured[64] = {0};
  B2L_CUDA_CHECK(b2l_ensure_dynamic_smem(kern, GroupedRing::kSmem, configured));
  const int64_t items = max_tiles * p.n_tiles;
  const int grid = (int)(items < b2l_num_sms() ? items : b2l_num_sms());
  b2l_launch(kern, dim3((unsigned)grid), dim3(kThreads), (size_t)GroupedRing::kSmem, st, tx, tw, p);
  B2L_LAUNCH_CHECK();
  return B2L_OK;
}

static int grouped_gemm(const void* x, const void* w, const GroupedParams& p, int64_t max_tiles, int experts, bool is_gated,
                        cudaStream_t st) {
  CUtensorMap tx, tw;
  int rc = b2l_make_tmap_2d(&tx, x, TMA_U8, (uint64_t)(max_tiles * GroupedRing::BT), (uint64_t)p.K / 2, (uint64_t)p.K / 2, (uint32_t)GroupedRing::BT, 128, true);
  if (rc != B2L_OK) return rc;
  rc = b2l_make_tmap_2d(&tw, w, TMA_U8, (uint64_t)experts * p.N, (uint64_t)p.K / 2, (uint64_t)p.K / 2, 128, 128, true);
  if (rc != B2L_OK) return rc;
  return is_gated ? launch_grouped<true>(tx, tw, p, max_tiles, st) : launch_grouped<false>(tx, tw, p, max_tiles, st);
}

}  // namespace mx4

// whether the product quantises 16-bit activations itself
extern "C" int64_t b2l_mxfp4_matmul_takes_16bit(int64_t t, int64_t n, int64_t k) {
  if (t < 1 || t > mx4::kRawTokens || n < 1 || k < 1) return 0;
  const int num_kb = (int)cdiv64(k, mx4::kStageK), s = mx4::parts(cdiv64(n, 128), num_kb);
  return (num_kb + s - 1) / s * t <= mx4::kRawStages;
}

extern "C" int b2l_mxfp4_matmul(void* y, void* y_scales, const void* x, const void* x_scales, const void* w, const void* w_scales,
                                const void* bias, int64_t t, int64_t n, int64_t k, int64_t x_row_stride, int64_t w_row_stride,
                                int64_t y_row_stride, int gated, int weights_ready, int dtype, void* stream) {
  B2L_REQUIRE(t >= 0 && n > 0 && k > 0 && k % 32 == 0 && t < (1ll << 30) && n < (1ll << 30) && k < (1ll << 30),
              "mxfp4_matmul: t=%lld n=%lld k=%lld (k a multiple of 32)", (long long)t, (long long)n, (long long)k);
  if (t == 0) return B2L_OK;
  const bool raw = x_scales == nullptr;
  B2L_REQUIRE(y && x && w && w_scales && (!gated || y_scales), "mxfp4_matmul: null pointer");
  B2L_REQUIRE(!raw || b2l_mxfp4_matmul_takes_16bit(t, n, k), "mxfp4_matmul: %lld rows of 16-bit activations want the quantiser first", (long long)t);
  B2L_REQUIRE(!gated || n % 128 == 0, "mxfp4_matmul: gate and up rows come in runs of 64 (n=%lld)", (long long)n);
  B2L_REQUIRE(((uintptr_t)x | (uintptr_t)x_scales | (uintptr_t)w | (uintptr_t)w_scales) % 16 == 0 &&
                  ((raw ? 2 * x_row_stride : x_row_stride) | w_row_stride) % 16 == 0 && (!gated || ((uintptr_t)y % 16 == 0 && y_row_stride % 16 == 0)),
              "mxfp4_matmul: rows of codes must start on 16 bytes");
  B2L_REQUIRE(dtype == B2L_F16 || dtype == B2L_BF16, "mxfp4_matmul: dtype %d", dtype);
  B2L_REQUIRE((cdiv64(t, 128) + cdiv64(n, 128)) * mx4::k_tiles(k) < (1ll << 29), "mxfp4_matmul: t=%lld n=%lld k=%lld", (long long)t, (long long)n, (long long)k);
  cudaStream_t st = (cudaStream_t)stream;
  mx4::PairCall g = {y, y_row_stride, y_scales, bias, x, x_scales, w, w_scales, t, n, k, x_row_stride, w_row_stride, gated != 0, weights_ready != 0};
  if (!raw && mx4::pair_wanted(g)) return mx4::pair_gemm(g, dtype, st);
  mx4::Params p;
  p.y = y; p.ldy = y_row_stride;
  p.y_scales = (uint8_t*)y_scales; p.y_ktiles = mx4::k_tiles(n / 2);
  p.bias = bias;
  p.x_scales = (const uint8_t*)x_scales; p.w_scales = (const uint8_t*)w_scales;
  p.x16 = raw ? x : nullptr; p.ldx16 = x_row_stride;
  p.ktiles = mx4::k_tiles(k);
  p.T = (int)t; p.N = (int)n; p.K = (int)k; p.num_kb = (int)cdiv64(k, mx4::kStageK);
  p.early = weights_ready;
  p.vec = n % 4 == 0 && y_row_stride % 4 == 0 && (uintptr_t)y % 8 == 0;
  if (dtype == B2L_F16) return mx4::stream_gemm<__half>(x, x_row_stride, w, w_row_stride, p, gated != 0, st);
  return mx4::stream_gemm<__nv_bfloat16>(x, x_row_stride, w, w_row_stride, p, gated != 0, st);
}

extern "C" int b2l_mxfp4_grouped_matmul(void* y, void* y_scales, const void* x, const void* x_scales, const void* w,
                                        const void* w_scales, const void* table, int64_t max_tiles, int tile_rows, int experts,
                                        int64_t n, int64_t k, int gated, void* stream) {
  B2L_REQUIRE(max_tiles >= 0 && experts > 0 && n > 0 && k > 0 && k % 32 == 0 && k < (1ll << 30) && n * experts < (1ll << 31) &&
                  max_tiles * cdiv64(n, 128) < (1ll << 31) && max_tiles * 256 < (1ll << 31) &&
                  (experts * cdiv64(n, 128) + 2 * max_tiles) * mx4::k_tiles(k) < (1ll << 29),
              "mxfp4_grouped_matmul: experts=%d n=%lld k=%lld (a multiple of 32) tiles=%lld", experts, (long long)n, (long long)k, (long long)max_tiles);
  B2L_REQUIRE(tile_rows == 64 || tile_rows == 128 || tile_rows == 256, "mxfp4_grouped_matmul: tiles of %d rows", tile_rows);
  if (max_tiles == 0) return B2L_OK;
  B2L_REQUIRE(y && x && x_scales && w && w_scales && table && (y_scales || (!gated && tile_rows == 64)), "mxfp4_grouped_matmul: null pointer");
  B2L_REQUIRE(!gated || n % 128 == 0, "mxfp4_grouped_matmul: gate and up rows come in runs of 64 (n=%lld)", (long long)n);
  B2L_REQUIRE(n % 32 == 0, "mxfp4_grouped_matmul: outputs come in units of 32 (n=%lld)", (long long)n);
  B2L_REQUIRE(((uintptr_t)x | (uintptr_t)x_scales | (uintptr_t)w | (uintptr_t)w_scales | (uintptr_t)y | (uintptr_t)y_scales) % 16 == 0,
              "mxfp4_grouped_matmul: rows must start on 16 bytes");
  cudaStream_t st = (cudaStream_t)stream;
  mx4::PairCall g = {y, gated ? n / 4 : n, y_scales, nullptr, x, x_scales, w, w_scales, max_tiles, n, k, k / 2, k / 2, gated != 0, false};
  if (tile_rows != 64) return mx4::rows_gemm(g, table, tile_rows, experts, st);
  mx4::GroupedParams p;
  p.y = y; p.ldy = gated ? n / 4 : n;
  p.y_scales = (uint8_t*)y_scales; p.y_ktiles = mx4::k_tiles(n / 2);
  p.x_scales = (const uint8_t*)x_scales; p.w_scales = (const uint8_t*)w_scales;
  p.table = (const int32_t*)table;
  p.ktiles = mx4::k_tiles(k);
  p.N = (int)n; p.K = (int)k; p.num_kb = (int)cdiv64(k, mx4::kStageK); p.n_tiles = (int)cdiv64(n, 128);
  return mx4::grouped_gemm(x, w, p, max_tiles, experts, gated != 0, st);
}
