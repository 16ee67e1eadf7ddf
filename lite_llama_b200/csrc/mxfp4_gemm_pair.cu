// Y = X W^T with both operands in microscaled 4-bit floating point, for prompt-sized batches, on CTA pairs.
//
// Bound: the tensor pipe (four times the rate of 16-bit operands), and right behind it what L2 can bring: a pair multiplies 256
// tokens x 256 outputs, 35 KiB per SM for 256 k.  As in gemm_pair.cu, with what the rate and the scales ask for:
//   * tokens are the MMA's rows, so a thread holds consecutive outputs of one token: 16-byte stores to shared memory and one TMA
//     store per 32 tokens x 64 outputs, or, for the gated unit, a token's 32 activations, which it quantises alone;
//   * 512 columns of tensor memory hold two accumulators of 256 only if the scales have none.  The accumulators overlap by 48 columns:
//     [0, 256) and [208, 464), scales behind them.  The shared columns are read out first and handed on at once, so a tile's products
//     start when a quarter of the tile before has been read, and the rest is written out under them;
//   * scales are TMA copies of whole tiles into every stage; both CTAs hold those of all 256 outputs.  Two sets of 24 columns take turns:
//     a set is written again when the MMAs of two stages ago have retired.
// ROUTED: the rows of routed experts, tiles of up to 128 rows of one expert by 256 of its weight rows, from a table on the device, on single
// CTAs (CTAS = 1); up to 256 rows on pairs, which fetch the weights once for both, where experts have so many.
#include "gemm_tc.cuh"
#include "mxfp4_mma.cuh"
#include "mxfp4_gemm.cuh"
#include "pair.cuh"

namespace mx4 {

constexpr int kPairThreads = 10 * 32;  // TMA producer, MMA issuer, eight warps that read the accumulator
constexpr int kPairRows = 128;         // tokens per CTA
constexpr int kPairBand = 16;          // token tiles per band: 16 x 256 rows x 4096 / 2 bytes = 8 MiB of L2

// Outputs in boxes by TMA, in rows that start anywhere, or of routed experts (in boxes)
enum Kind { kBoxes, kRagged, kRouted };

template <int BN, int CTAS, bool GATED, Kind KIND> struct PairRing {
  static constexpr int kStages = CTAS == 2 ? (GATED ? 6 : (KIND == kRouted ? 4 : 5)) : (GATED ? 4 : 3);
  static constexpr int kX = 16384, kW = BN / CTAS * 128;
  static constexpr int kXs = kX + kW, kWs = kXs + kSfBytes;
  static constexpr int kBytes = kWs + BN / 128 * kSfBytes;
  static constexpr int kOut = KIND == kRouted ? 8192 : 4096;               // boxes of a warp: 32 rows of 64 outputs, 16 bits of each
  static constexpr int kSmem = 1024 + 1024 + kStages * kBytes + (GATED ? 0 : 8 * kOut);
  static constexpr int kAcc1 = BN == 256 ? 208 : 128;                     // first column of the second accumulator
  static constexpr int kSf = BN == 256 ? 464 : 256;
  static constexpr int kSfSet = 8 + BN / 128 * 8;
};

struct PairParams {
  const void* bias;
  uint8_t* y; uint8_t* y_scales; int64_t ldy, y_ktiles;                   // gated: codes and scales
  const int32_t* table;                // experts: tiles, then {expert, rows} of each
  int T, N, K, num_kb, m_tiles, n_tiles, ktiles;
  int wide, tiles;                     // tiles of BN outputs; those and the halves behind them
  int early;                           // weights may be requested before the previous kernel has ended
};

struct __align__(8) PairControl {
  uint64_t full[6];                    // leader: both CTAs' operands and scales of a stage have landed
  uint64_t empty[6];                   // both: the MMAs of a stage have retired
  uint64_t acc_full[2];                // both: a tile's accumulator is complete
  uint64_t freed[2];                   // leader: all warps have read what the next tile's products overwrite
  uint32_t tmem;
};

// What differs between a pair and a single CTA
template <int CTAS> __device__ __forceinline__ void sync_all() {
  if (CTAS == 2) pair_sync_relaxed();
  else __syncthreads();
}
template <int CTAS> __device__ __forceinline__ void load_2d(void* dst, const void* map, int c0, int c1, uint64_t* bar) {
  if (CTAS == 2) tma_load_2d_pair(dst, map, c0, c1, leader_addr(bar), kEvictNormal);
  else tma_load_2d_hint(dst, map, c0, c1, bar, kEvictNormal);
}
template <int CTAS> __device__ __forceinline__ void commit(uint64_t* bar) {
  if (CTAS == 2) tc_commit_pair(bar);
  else tc_commit(bar);
}
// A tile of outputs: token tile (index of 128 rows for each CTA), first 128 outputs and how many of those, rows that hold anything, expert
struct Work { int m, n, width, rows, expert; };
template <int BN, int CTAS, bool ROUTED> __device__ __forceinline__ Work work_of(const PairParams& p, int t, int rank) {
  Work o;
  o.width = BN / 128;
  if (!ROUTED) {
    // the tiles that would make a last wave of less than half of the pairs come in halves
    const int behind = t - p.wide;
    const PairTile pt = pair_tile(behind < 0 ? t : p.wide + (behind >> 1), p.m_tiles, p.n_tiles, kPairBand);
    o.m = pt.m * 2 + rank;
    o.n = pt.n * (BN / 128);
    if (behind >= 0) {
      o.n += behind & 1;
      o.width = 1;
    }
    o.rows = p.T - o.m * kPairRows;
    o.expert = 0;
  } else {
    const int tile = t / p.n_tiles;
    o.m = tile * CTAS + rank;
    o.n = (t - tile * p.n_tiles) * (BN / 128);
    o.expert = ld_upstream(p.table + 1 + 2 * tile);
    o.rows = ld_upstream(p.table + 2 + 2 * tile) - rank * kPairRows;
  }
  return o;
}

template <typename T, int BN, bool GATED, int CTAS, Kind KIND>
__global__ void __launch_bounds__(kPairThreads, 1)
pair_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_xs,
            const __grid_constant__ CUtensorMap tmap_ws, const __grid_constant__ CUtensorMap tmap_y, const __grid_constant__ CUtensorMap tmap_low,
            const PairParams p) {
  using R = PairRing<BN, CTAS, GATED, KIND>;
  constexpr bool ROUTED = KIND == kRouted;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  PairControl* ctl = reinterpret_cast<PairControl*>(smem);
  uint8_t* ring = smem + 1024;
  uint8_t* out_stage = ring + R::kStages * R::kBytes;

  // one value for the warp, as far as the compiler can see: roles and addresses then live in uniform registers
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = CTAS == 2 ? pair_rank() : 0u;
  const int pairs = gridDim.x / CTAS, pair = blockIdx.x / CTAS;
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmap_x);
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_xs);
    tma_prefetch_desc(&tmap_ws);
    if (!GATED) tma_prefetch_desc(&tmap_y);
    if (!GATED && ROUTED) tma_prefetch_desc(&tmap_low);
    for (int s = 0; s < R::kStages; ++s) {
      mbar_init(&ctl->full[s], 1);
      mbar_init(&ctl->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&ctl->acc_full[b], 1);
      mbar_init(&ctl->freed[b], 8 * CTAS);
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    if (CTAS == 2) { tmem_alloc_pair(&ctl->tmem, 512); tmem_relinquish_pair(); }
    else { tmem_alloc(&ctl->tmem, 512); tmem_relinquish(); }
    pdl_launch_dependents();           // after the allocation (gemm_dense.cu)
  }
  tc_fence_before();
  __syncthreads();                     // the allocation's store to shared memory, which the relaxed barrier does not show
  if (CTAS == 2) pair_sync_relaxed();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, ctl->tmem, 0);
  if (ROUTED) pdl_wait_prior();        // the table is upstream data
  const int tiles = ROUTED ? ld_upstream(p.table) * p.n_tiles : p.tiles;

  if (warp == 0) {
    // ===================== TMA producer: this CTA's halves of both operands, its tokens' scales, all outputs' scales =====================
    auto expect = [&](int s) {
      if (rank == 0) mbar_arrive_expect_tx(&ctl->full[s], CTAS * R::kBytes);
    };
    auto load_w = [&](int s, int kb, const Work& wk) {
      uint8_t* st = ring + (size_t)s * R::kBytes;
      const int row = wk.expert * p.N + wk.n * 128 + (int)rank * (wk.width * (128 / CTAS));      // of half a tile the box holds twice as much
      const int ws = (wk.expert * ((p.N + 127) / 128) + wk.n) * p.ktiles * 4;                     // rows of 128 bytes
      load_2d<CTAS>(st + R::kX, &tmap_w, kb * 128, row, &ctl->full[s]);
#pragma unroll
      for (int h = 0; h < BN / 128; ++h) load_2d<CTAS>(st + R::kWs + h * kSfBytes, &tmap_ws, 0, ws + h * p.ktiles * 4 + kb * 8, &ctl->full[s]);
    };
    auto load_x = [&](int s, int kb, const Work& wk) {
      uint8_t* st = ring + (size_t)s * R::kBytes;
      load_2d<CTAS>(st, &tmap_x, kb * 128, wk.m * kPairRows, &ctl->full[s]);
      load_2d<CTAS>(st + R::kXs, &tmap_xs, 0, (wk.m * p.ktiles + kb * 2) * 4, &ctl->full[s]);
    };
    gemm::PipeState ps(R::kStages);
    int ahead = 0;                     // stages whose weights were requested before the previous kernel has ended
    if (!ROUTED && p.early && pair < tiles) {
      const Work wk = work_of<BN, CTAS, ROUTED>(p, pair, (int)rank);
      ahead = p.num_kb < R::kStages ? p.num_kb : R::kStages;
      if (elect_one())
        for (int s = 0; s < ahead; ++s) { expect(s); load_w(s, s, wk); }
      __syncwarp();
    }
    pdl_wait_prior();
    Work next = pair < tiles ? work_of<BN, CTAS, ROUTED>(p, pair, (int)rank) : Work{0, 0, 0, 0, 0};
    for (int t = pair; t < tiles; t += pairs) {
      const Work wk = next;
      if (t + pairs < tiles) next = work_of<BN, CTAS, ROUTED>(p, t + pairs, (int)rank);      // table entries are asked for a tile ahead
#pragma unroll 1
      for (int kb = 0; kb < p.num_kb; ++kb) {
        mbar_wait(&ctl->empty[ps.stage], ps.phase ^ 1);
        if (elect_one()) {
          if (ahead == 0) { expect(ps.stage); load_w(ps.stage, kb, wk); }
          load_x(ps.stage, kb, wk);
        }
        if (ahead > 0) --ahead;
        __syncwarp();
        ps.advance();
      }
    }
    // every stage handed back: no commit is still on its way to this CTA's barriers when it leaves
    for (int s = 0; s < R::kStages; ++s) {
      mbar_wait(&ctl->empty[ps.stage], ps.phase ^ 1);
      ps.advance();
    }
  } else if (warp == 1) {
    // ===================== MMA issuer (leader only) =====================
    // A step of 256 k is 512 cycles of the tensor pipe, and the issuer's own instructions take nearly as long: they bound the kernel
    // until warp index and column base were uniform to the compiler (1000 x 4096 x 14336 29.9 -> 24 us).  The loop unrolled over the
    // ring is slower (256 x 4096 x 4096 7.7 -> 8.8: instruction cache), a second elected region costs 120 ns a step.
    if (rank == 0) {
      const uint64_t desc0 = umma_desc_sw128_kmajor(smem_u32(ring)), sf0 = scale_desc(smem_u32(ring));
      gemm::PipeState ps(R::kStages), back(R::kStages);      // back: the stage two before
      int it = 0, i = 0;
      for (int t = pair; t < tiles; t += pairs, ++it) {
        const uint32_t acc = tmem + (it & 1) * R::kAcc1;
        const uint32_t id = BN == 256 && !ROUTED && t >= p.wide ? idesc(128 * CTAS, 128, 0) : idesc(128 * CTAS, BN, 0);
        if (BN == 256) {
          if (it >= 1) mbar_wait_spin(&ctl->freed[(it - 1) & 1], ((it - 1) >> 1) & 1);
        } else {
          if (it >= 2) mbar_wait_spin(&ctl->freed[it & 1], ((it - 2) >> 1) & 1);
        }
        tc_fence_after();
#pragma unroll 1
        for (int kb = 0; kb < p.num_kb; ++kb, ++i) {
          if (i >= 2) {
            mbar_wait_spin(&ctl->empty[back.stage], back.phase);
            back.advance();
          }
          mbar_wait_spin(&ctl->full[ps.stage], ps.phase);
          tc_fence_after();
          if (elect_one()) {
            const uint32_t base = (uint32_t)(ps.stage * R::kBytes) >> 4;
            const uint64_t xd = desc0 + base, wd = xd + (R::kX >> 4);
            const uint64_t xsf = sf0 + base + (R::kXs >> 4), wsf = xsf + (kSfBytes >> 4);
            const uint32_t sfa = tmem + R::kSf + (i & 1) * R::kSfSet, sfb = sfa + 8;
            const int steps = (p.K - kb * kStageK + 63) >> 6;
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (2 * j < steps) {
                copy_scales<CTAS>(sfa + 4 * j, xsf + j * (kTileBytes >> 4));
#pragma unroll
                for (int h = 0; h < BN / 128; ++h)
                  copy_scales<CTAS>(sfb + j * (BN / 32) + 4 * h, wsf + h * (kSfBytes >> 4) + j * (kTileBytes >> 4));
#pragma unroll
                for (int q = 2 * j; q < 2 * j + 2; ++q)
                  if (q < steps)
                    mma<CTAS>(acc, xd + 2 * q, wd + 2 * q, id | ((q & 1) ? kSecondHalf : 0u), sfa + j * 4, sfb + j * (BN / 32), kb | q ? 1u : 0u);
              }
            commit<CTAS>(&ctl->empty[ps.stage]);
            if (kb + 1 == p.num_kb) commit<CTAS>(&ctl->acc_full[it & 1]);
          }
          __syncwarp();
          ps.advance();
        }
      }
    }
  } else {
    // ===================== one thread per token, two warps to its columns =====================
    const int quad = warp & 3, half = (warp - 2) >> 2;
    // Only where a later tile's products wait for it: an arrival that nobody waits for could still be on its way to the leader when that
    // has left.
    bool awaited = false;
    auto hand_on = [&](int buf) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0 && awaited) {
        if (CTAS == 2) mbar_arrive_cluster(leader_addr(&ctl->freed[buf]));
        else mbar_arrive(&ctl->freed[buf]);
      }
    };
    pdl_wait_prior();                  // y may still be read upstream
    uint8_t* dst = out_stage + (quad + 4 * half) * R::kOut;
    int it = 0;
    Work next = pair < tiles ? work_of<BN, CTAS, ROUTED>(p, pair, (int)rank) : Work{0, 0, 0, 0, 0};
    for (int t = pair; t < tiles; t += pairs, ++it) {
      const Work wk = next;
      if (t + pairs < tiles) next = work_of<BN, CTAS, ROUTED>(p, t + pairs, (int)rank);
      const int buf = it & 1, m_warp = wk.m * kPairRows + quad * 32;
      awaited = t + (BN == 256 ? 1 : 2) * pairs < tiles;
      const bool any = quad * 32 < wk.rows;             // uniform over the warp
      const int end = (wk.n + wk.width) * 128 < p.N ? (wk.n + wk.width) * 128 : p.N;
      const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16) + buf * R::kAcc1;
      // the columns that both accumulators have: the first one's last, read by the second half's warps, the second one's first.  The other
      // half's warps are done with the tile before, which is what their arrival says.
      const bool shared = BN == 256 && half == 1 - buf;
      mbar_wait(&ctl->acc_full[buf], (it >> 1) & 1);
      tc_fence_after();
      if (BN == 256 && !shared) hand_on(buf);
      if (!GATED) {
#pragma unroll 1
        for (int j = 0; j < BN / 128; ++j) {
          const int c = half * (BN / 2) + (BN == 256 && buf == 0 ? 1 - j : j) * 64;
          uint32_t v[64];
          tmem_ld_32x32b_x32(acc + c, *reinterpret_cast<uint32_t(*)[32]>(v));
          tmem_ld_32x32b_x32(acc + c + 32, *reinterpret_cast<uint32_t(*)[32]>(v + 32));
          tc_wait_ld();
          if (BN == 256 ? shared && j == 0 : true) hand_on(buf);
          const int n0 = wk.n * 128 + c;
          if (n0 >= end || !any) continue;
          if (ROUTED) {
            // Sums stay in 32 bits, in two planes of 16 (boxes of 64 outputs, as 16-bit ones have): the upper halves, then the lower.  In 16
            // bits, as whole numbers with a scale for 64 of them, 2000 tokens over 128 experts took 113 us instead of 133 (16000 slots written
            // and read), but an output a thousand times its neighbours cost them all but six bits.  Two boxes and four stages on
            // pairs, or one box and five, us: 131072 slots of 2048 x 768 706 / 722, 8192 of 4096 x 1792 143 / 138.
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (lane == 0) bulk_wait_read<1>();       // the box's store before, which is the last but one, has read it
              __syncwarp();
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                uint32_t o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = __byte_perm(v[8 * q + 2 * e], v[8 * q + 2 * e + 1], h ? 0x5410 : 0x7632);
                *reinterpret_cast<uint4*>(dst + h * 4096 + lane * 128 + ((q ^ (lane & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
              }
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                tma_store_2d(h ? &tmap_low : &tmap_y, dst + h * 4096, n0, m_warp);
                bulk_commit();
              }
            }
            continue;
          }
          if (lane == 0) bulk_wait_read<0>();           // the store before has read the box
          __syncwarp();
          if (p.bias && KIND == kBoxes) {               // a branch of its own: without a bias nothing of it is issued
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const int n = n0 + 8 * q;                 // N is a multiple of 8
              const uint4 b4 = n < p.N ? ldg_128(reinterpret_cast<const T*>(p.bias) + n) : make_uint4(0u, 0u, 0u, 0u);
              const T* b = reinterpret_cast<const T*>(&b4);
#pragma unroll
              for (int e = 0; e < 8; ++e) v[8 * q + e] = __float_as_uint(__uint_as_float(v[8 * q + e]) + to_f32(b[e]));
            }
          }
          if (p.bias && KIND == kRagged) {
            const T* bias = reinterpret_cast<const T*>(p.bias) + n0;
            const float b0 = n0 + lane < p.N ? to_f32(bias[lane]) : 0.f, b1 = n0 + 32 + lane < p.N ? to_f32(bias[32 + lane]) : 0.f;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              v[e] = __float_as_uint(__uint_as_float(v[e]) + __shfl_sync(0xffffffffu, b0, e));
              v[32 + e] = __float_as_uint(__uint_as_float(v[32 + e]) + __shfl_sync(0xffffffffu, b1, e));
            }
          }
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float a = __uint_as_float(v[8 * q + 2 * e]), b = __uint_as_float(v[8 * q + 2 * e + 1]);
              o[e] = pack2<T>(a, b);
            }
            *reinterpret_cast<uint4*>(dst + lane * 128 + ((q ^ (lane & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
          }
          if (KIND != kRagged) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmap_y, dst, n0, m_warp);
              bulk_commit();
            }
          } else {                                      // two outputs a lane and row
            __syncwarp();
            const int rows = wk.rows - quad * 32, n = n0 + 2 * lane;
            T* y = reinterpret_cast<T*>(p.y) + (int64_t)m_warp * p.ldy + n;
            const uint8_t* src = dst + (lane & 3) * 4;
#pragma unroll 4
            for (int r = 0; r < 32 && r < rows; ++r, y += p.ldy) {
              const uint32_t two = *reinterpret_cast<const uint32_t*>(src + r * 128 + (((lane >> 2) ^ (r & 7)) << 4));
              const T* o = reinterpret_cast<const T*>(&two);
              if (n < end) y[0] = o[0];
              if (n + 1 < end) y[1] = o[1];
            }
            __syncwarp();
          }
        }
      } else {
        // A run of 64 gate and 64 up columns to each half (of the narrow tile's only run: a block of 32).  What lies on the shared columns is
        // read before anything else: the up columns of the first accumulator's second run, the gate columns of the second's first.
        constexpr int kBlocks = BN / 128;               // blocks of 32 activations to a warp
        const bool up_first = BN == 256 && buf == 0;
        const int c = BN == 256 ? half * 128 : half * 32;
        uint32_t held[32 * kBlocks];
#pragma unroll
        for (int h = 0; h < kBlocks; ++h)
          tmem_ld_32x32b_x32(acc + c + (up_first ? 64 : 0) + 32 * h, *reinterpret_cast<uint32_t(*)[32]>(held + 32 * h));
        tc_wait_ld();
        if (shared) hand_on(buf);
        const int n0 = wk.n * 128 + (BN == 256 ? c : 0), k = n0 / 2 + (BN == 256 ? 0 : half * 32), row = m_warp + lane;
        uint32_t bytes = 0;
        uint32_t codes[kBlocks][4];
#pragma unroll
        for (int h = 0; h < kBlocks; ++h) {
          uint32_t other[32];
          tmem_ld_32x32b_x32(acc + c + (up_first ? 0 : 64) + 32 * h, other);
          tc_wait_ld();
          if (BN != 256) hand_on(buf);
          const int n = n0 + (BN == 256 ? 32 * h : 32 * half);      // the block's gate rows
          float v[32], u[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            v[e] = __uint_as_float(up_first ? other[e] : held[32 * h + e]);
            u[e] = __uint_as_float(up_first ? held[32 * h + e] : other[e]);
          }
          const T* bias = p.bias && n < p.N ? reinterpret_cast<const T*>(p.bias) + n : nullptr;
          uint32_t byte;
          quantise_unit<32, T>(v, u, bias, quad * 32 + lane < wk.rows, codes[h], byte);
          bytes |= byte << (8 * h);
        }
        if (n0 < end && quad * 32 + lane < wk.rows) {   // N is a multiple of 128
          uint8_t* y = p.y + (int64_t)row * p.ldy + k / 2;
#pragma unroll
          for (int h = 0; h < kBlocks; ++h) stg_128(y + 16 * h, make_uint4(codes[h][0], codes[h][1], codes[h][2], codes[h][3]));
          uint8_t* word = p.y_scales + scale_word(row, k >> 7, p.y_ktiles) + ((k >> 5) & 3);
          const bool last = n0 + 128 == p.N && (k & 64) == 0;      // an odd number of runs: zeros behind the end
          if (BN == 256) {
            if (last) *reinterpret_cast<uint32_t*>(word) = bytes;
            else *reinterpret_cast<uint16_t*>(word) = (uint16_t)bytes;
          } else {
            word[0] = (uint8_t)bytes;
            if (last) word[2] = 0;
          }
        }
      }
    }
    if (!GATED && lane == 0) bulk_wait_read<0>();       // the boxes have been read; the stores end with the kernel
  }

  tc_fence_before();
  sync_all<CTAS>();                    // the peer's MMAs, commits and arrivals are over
  if (warp == 1) {
    if (CTAS == 2) tmem_dealloc_pair(tmem, 512);
    else tmem_dealloc(tmem, 512);
  }
}

// Maps and launch, for `rows` rows of x and y in tiles of 128 and `weight_rows` rows of w
template <typename T, int BN, bool GATED, int CTAS, Kind KIND>
static int launch_rows(const PairCall& g, PairParams& p, int64_t rows, int64_t experts, int64_t tiles, cudaStream_t st) {
  using R = PairRing<BN, CTAS, GATED, KIND>;
  const int sms = b2l_num_sms();
  p.bias = g.bias;
  p.y = (uint8_t*)g.y; p.y_scales = (uint8_t*)g.y_scales; p.ldy = g.ldy; p.y_ktiles = k_tiles(g.N / 2);
  p.N = (int)g.N; p.K = (int)g.K; p.num_kb = (int)cdiv64(g.K, kStageK); p.ktiles = (int)k_tiles(g.K);
  p.n_tiles = (int)cdiv64(g.N, BN);
  tiles *= p.n_tiles;
  // Halves for what is left of the last wave if that is at most half of one (us: 1000 x 28672 x 4096, 448 tiles
  // for 74 pairs, 54 -> 52; 300 x 28672 x 4096 32.5 -> 29.3)
  const int64_t pairs = sms / CTAS, rest = tiles % pairs;
  p.wide = (int)(KIND != kRouted && BN == 256 && tiles > pairs && 2 * rest <= pairs ? tiles - rest : tiles);
  p.tiles = (int)(p.wide + 2 * (tiles - p.wide));
  const int grid = CTAS * (int)(tiles < pairs ? tiles : pairs);
  CUtensorMap tx, tw, txs, tws, ty, tl;
  int rc = b2l_make_tmap_2d(&tx, g.x, TMA_U8, (uint64_t)rows, (uint64_t)g.K / 2, (uint64_t)g.ldx, kPairRows, 128, true);
  if (rc == B2L_OK) rc = b2l_make_tmap_2d(&tw, g.w, TMA_U8, (uint64_t)(experts * g.N), (uint64_t)g.K / 2, (uint64_t)g.ldw, BN / CTAS, 128, true);
  if (rc == B2L_OK) rc = b2l_make_tmap_2d(&txs, g.x_scales, TMA_U8, (uint64_t)(cdiv64(rows, 128) * p.ktiles * 4), 128, 128, 8, 128, false);
  if (rc == B2L_OK) rc = b2l_make_tmap_2d(&tws, g.w_scales, TMA_U8, (uint64_t)(experts * cdiv64(g.N, 128) * p.ktiles * 4), 128, 128, 8, 128, false);
  const bool boxes = !GATED && KIND != kRagged;
  if (rc == B2L_OK && boxes)
    rc = b2l_make_tmap_2d(&ty, g.y, std::is_same<T, __half>::value ? TMA_F16 : TMA_BF16, (uint64_t)rows, (uint64_t)g.N, (uint64_t)g.ldy * 2, 32, 64, true);
  const bool low = KIND == kRouted && !GATED;
  if (rc == B2L_OK && low) rc = b2l_make_tmap_2d(&tl, g.y_scales, TMA_F16, (uint64_t)rows, (uint64_t)g.N, (uint64_t)g.ldy * 2, 32, 64, true);
  if (rc != B2L_OK) return rc;
  if (!boxes) ty = tx;
  if (!low) tl = ty;
  auto kern = pair_kernel<T, BN, GATED, CTAS, KIND>;
  static int configured[64] = {0};
  B2L_CUDA_CHECK(b2l_ensure_dynamic_smem(kern, R::kSmem, configured));
  b2l_hang_arm(st);
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = R::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CTAS;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = b2l_pdl_enabled() ? 2 : 1;
  B2L_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, tx, tw, txs, tws, ty, tl, p));
  B2L_LAUNCH_CHECK();
  return B2L_OK;
}

template <typename T, int BN, bool GATED>
static int launch_pair(const PairCall& g, cudaStream_t st) {
  PairParams p;
  p.table = nullptr;
  p.T = (int)g.T;
  p.early = g.early ? 1 : 0;
  p.m_tiles = (int)cdiv64(g.T, 2 * kPairRows);
  if constexpr (!GATED) {
    // two bytes at a time: 2881 x 4563 x 7808 43 us, 63 with the streaming kernel; 2881 x 4560 x 7808 in boxes 39
    if (g.N % 8 != 0 || g.ldy % 8 != 0 || (uintptr_t)g.y % 16 != 0 || (uintptr_t)g.bias % 16 != 0)
      return launch_rows<T, BN, false, 2, kRagged>(g, p, g.T, 1, p.m_tiles, st);
  }
  return launch_rows<T, BN, GATED, 2, kBoxes>(g, p, g.T, 1, p.m_tiles, st);
}

// Up to 128 tokens half of a pair's rows are padding, and the streaming kernel is as fast or faster (65 - 128 tokens, us, streaming / pairs:
// 28672 x 4096 14.0 - 15.2 / 16.7, 4096 x 14336 13.1 / 17.6; 2048 x 2048 5.5 / 5.2).  With few tiles and a long k it parts k over more SMs, up to 256
// tokens: 256 x 4096 x 14336 14.3 / 17.7, 200 x 896 x 4864 6.6 / 7.8; but 256 x 4096 x 4096 9.4 / 8.1, 400 x 4096 x 14336 18.5 / 18.4.
bool pair_wanted(const PairCall& g) {
  return g.T > 128 && !(g.T <= 256 && cdiv64(g.N, 128) * 4 <= b2l_num_sms() && g.K > 16 * kStageK);
}

int pair_gemm(const PairCall& g, int dtype, cudaStream_t st) {
  const int64_t m_tiles = cdiv64(g.T, 2 * kPairRows), pairs = b2l_num_sms() / 2;
  // Waves x tile width is what the grid spends on the tensor pipe, and a narrow tile fetches its tokens twice as often (256 -> 128 outputs, us:
  // 600 x 2048 x 2048 6.2 -> 5.3, 777 x 4608 x 3584 9.2 -> 10.7, three waves for two 1000 x 6144 x 4096 14.2 -> 16.5; gated
  // 16.2 -> 17.2, 400 x 9728 x 896 9.6 -> 8.2).
  const int64_t w256 = cdiv64(m_tiles * cdiv64(g.N, 256), pairs) * 256, w128 = cdiv64(m_tiles * cdiv64(g.N, 128), pairs) * 128;
  const bool narrow = w128 * (g.gated ? 130 : 140) < w256 * 100;
#define PAIR(T) (narrow ? (g.gated ? launch_pair<T, 128, true>(g, st) : launch_pair<T, 128, false>(g, st)) \
                        : (g.gated ? launch_pair<T, 256, true>(g, st) : launch_pair<T, 256, false>(g, st)))
  if (dtype == B2L_F16) return PAIR(__half);
  return PAIR(__nv_bfloat16);
#undef PAIR
}

// Routed experts: g.T tiles of 128 or 256 rows at most, w of `experts` stacked matrices
int rows_gemm(const PairCall& g, const void* table, int tile_rows, int experts, cudaStream_t st) {
  PairParams p;
  p.table = (const int32_t*)table;
  p.T = p.m_tiles = p.early = 0;
  const int64_t rows = g.T * tile_rows;
  if (tile_rows == 128)
    return g.gated ? launch_rows<__half, 256, true, 1, kRouted>(g, p, rows, experts, g.T, st) : launch_rows<__half, 256, false, 1, kRouted>(g, p, rows, experts, g.T, st);
  return g.gated ? launch_rows<__half, 256, true, 2, kRouted>(g, p, rows, experts, g.T, st) : launch_rows<__half, 256, false, 2, kRouted>(g, p, rows, experts, g.T, st);
}

}  // namespace mx4
