// flash_attention_int4: portions of prompts over a cache held in 4 bits (kv_int4.cuh), on the 5th-generation tensor cores.
//
// Query j of a sequence's new tokens stands at position len - new + j and sees the cached tokens up to itself.
//
// A CTA works on 256 query rows of one kv head -- rows are (token, query head of the group), so that a key tile serves all heads of
// the group and a portion of few tokens still fills a tile -- as two tiles of 128 rows, over tiles of 128 keys:
//   warps 0, 1    tensor-core issuers: the scores S = Q K^T, and O += P V (A = P from tensor memory)
//   warps 2, 3    the head's bytes of the cache rows, through the request table, by asynchronous copies into a ring of units (64 keys of K
//                 or of V), a tile ahead
//   warps 4 - 11  codes to halves minimum + scale * code in the operands' swizzled layout.  A word of eight codes turns into one 16-byte
//                 chunk in the order 0 4 1 5 2 6 3 7: with the queries stored in the same order the scores are the same, and the
//                 outputs' order is undone at the end.
//   warps 12 - 19 softmax, a thread to a row of either tile: the row's scores from tensor memory once, P written back, the output rescaled
//                 where the running maximum rises by more than 2^8 (both by one factor, hence exact)
// Tensor memory: two buffers of 64 keys' scores for either tile, whose place the probabilities take | O0 | O1.  A softmax thread works on
// one half of a key tile (its registers suffice for that beside eight converting warps) while the products of the other run.  A step
// (a key tile of both row tiles) takes 4500 to 4900 cycles, bound by the conversion's and the softmax's instructions together; its four
// products would take 2050.
//
// READY: where five row blocks or more read a key tile on average and a CTA has ten steps or more, a kernel before this one converts
// each tile once into the workspace, as the tensor cores read it, and one warp fetches whole operands; the softmax warps then have
// registers for a whole row of 128 scores (S for both tiles in turn | P0 P1 | O0 | O1), which they free before the exponentials.  A
// step takes 2750 cycles, of which 2050 are the exponentials' issue alone.  The kernel before takes 8 - 12 us for 8000 keys of 8 heads.
// 512 tokens over 7500, 32 / 8 heads: 85 us (98 the other way).
// The operands are halves for both activation types: elements are rounded to 11 bits (as the 16-bit cache of an fp16 model rounds
// them), which for bf16 models are three bits more than reading the cache into their type would leave; elements of those beyond 65504
// count as 65504, and below 2^-14 they come in steps of 2^-24.  Queries of bf16 models are scaled by a power of two per row.  Probabilities are rounded to 11 bits, as in
// flash_attention_tc.cu; sums, maxima and outputs are held in 32.
// A value that is NaN enters as 0 and makes NaN of the rows that see it at the end, since 0 * NaN would reach the rows that do not.
//
// Work: key tiles of all row blocks of all sequences, in equal shares over one wave of CTAs (lengths are device data), down to one
// (5 tokens over 300, 8 kv heads: 11.7 us, two tiles at least 17.2; 64 over 500: 19.6 and 30.9).  A row block in several shares leaves parts in the workspace, which a second kernel adds up.
#include "kv_int4.cuh"
#include "attention_tmem.cuh"
#include <climits>
#include <type_traits>

namespace kv4p {

constexpr int kBM = 128, kBN = 128, kRows = 2 * kBM;
constexpr int kThreads = 640, kConvert = 256, kReadyThreads = 384, kKStages = 2, kVStages = 2, kSegs = 4;
constexpr int kUnits = 5, kUnitKeys = 64, kUnitPitch = 96;   // pitch: rows of four neighbours in different banks
constexpr int kMaxBatch = 128;                    // sequences of a launch (their sizes lie in shared memory)

struct Params {
  const void* q; int64_t q_ts, q_hs; int q_vec;
  void* out; int64_t o_ts, o_hs; int o_vec;
  const uint8_t* cache; int64_t row_stride, max_tokens;
  const int32_t* table; int64_t tab_rs, tab_cs, requests;
  const void *start, *fresh, *req, *len;
  int start_w, fresh_w, req_w, len_w;
  int batch, Hkv, G;
  uint64_t by_G;                                  // 2^64 / G, rounded up: n / G is the high half of n * by_G for n < 2^32 (G > 1)
  int64_t total, max_new, most;
  uint32_t items;                                 // row blocks (of all kv heads) that the workspace has notes for
  float scale_log2;
  float* ws_o; float2* ws_ml; int2* ws_info; int4* ws_item;
  uint8_t* ready; int4* ready_nan; int ready_tiles;   // operands made before: tiles [sequence][kv head][ready_tiles], K's image and V's
};

// a sequence: its m new tokens begin at row `start` of q, the first stands at position ctx, keys below `keys` are cached
struct Seq { int m, ctx, keys, start, req; };
__device__ __forceinline__ Seq sequence(const Params& p, int b) {
  const int64_t n = load_index(p.len, b, p.len_w), f = load_index(p.fresh, b, p.fresh_w), s = load_index(p.start, b, p.start_w);
  const int64_t r = load_index(p.req, b, p.req_w);
  int64_t m = f < 0 ? 0 : f, ctx = (n < 0 ? 0 : n) - m;
  if (m > p.max_new) m = p.max_new;
  if (s < 0 || s >= p.total) m = 0;
  else if (m > p.total - s) m = p.total - s;
  Seq q;
  q.m = (int)m;
  q.ctx = (int)(ctx < -(1ll << 30) ? -(1ll << 30) : ctx > (1ll << 30) ? (1ll << 30) : ctx);
  q.keys = r < 0 || r >= p.requests || n <= 0 ? 0 : (int)(n < p.most ? n : p.most);
  q.start = (int)s;
  q.req = (int)r;
  return q;
}
__device__ __forceinline__ int over_G(const Params& p, int n) { return p.G == 1 ? n : (int)__umul64hi((uint64_t)(uint32_t)n, p.by_G); }
__device__ __forceinline__ int row_blocks(const Params& p, const Seq& s) { return (s.m * p.G + kRows - 1) / kRows; }
// key tiles of tile t of row block rb: up to its last row's position (0: no rows; a tile that sees nothing takes one step for its zeros)
__device__ __forceinline__ int key_tiles(const Params& p, const Seq& s, int rb, int t) {
  const int first = rb * kRows + t * kBM, rows = s.m * p.G;
  if (first >= rows) return 0;
  const int last = (first + kBM < rows ? first + kBM : rows) - 1;
  int k = s.ctx + over_G(p, last) + 1;
  if (k > s.keys) k = s.keys;
  return k > 0 ? (k + kBN - 1) / kBN : 1;
}
// of both: the second sees no less, where it has rows
__device__ __forceinline__ int block_steps(const Params& p, const Seq& s, int rb) {
  const int b = key_tiles(p, s, rb, 1);
  return b > 0 ? b : key_tiles(p, s, rb, 0);
}

struct __align__(16) Ctl {
  uint64_t q_full[2], k_full[kKStages], k_empty[kKStages], v_full[kVStages], v_empty[kVStages];
  uint64_t raw_full[kUnits], raw_empty[kUnits];
  uint64_t s_free;                                // READY: one buffer for both tiles' scores
  uint64_t s_full[2][2], p_full[2][2], pv_done[2][2], seg_done[kSegs];   // of either half of a tile's scores: a phase is a key tile
  int nan_at[kSegs][4];                           // first key whose value group is NaN
  int8_t q_exp[2][kBM];                           // bf16: the power of two that a row of Q was divided by
  uint32_t tmem_base;
};
static_assert(sizeof(Ctl) <= 1024, "control block");

// steps [j0, j1) of a row block
struct Segment { int b, kvh, rb, j0, j1, steps, item; };

#define kv4_wait(bar, parity) mbar_wait_at<true>((bar), (parity), b2l_file_hash(__FILE__), __LINE__)

// an asynchronous copy of 4, 8 or 16 bytes to shared memory; zeros where `read` is false
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool read) {
  const int n = read ? BYTES : 0;
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(n), "n"(BYTES) : "memory");
}
// the barrier's arrival of this thread, once its copies so far are done
__device__ __forceinline__ void copy_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// codes of a word to halves minimum + scale * code, in the order 0 4 1 5 2 6 3 7
__device__ __forceinline__ uint4 to_halves(uint32_t w, __half2 s, __half2 m) {
  const uint32_t magic = 0x64006400u;             // 1024 + code
  const __half2 big = *reinterpret_cast<const __half2*>(&magic);
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = ((w >> (4 * i)) & 0x000f000fu) | magic;
    const __half2 v = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&x), big), s, m);
    r[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}
// the same for scales or minima that may lead past the halves' range or are too small for it, or NaN: rounded once
__device__ __forceinline__ uint4 to_halves_wide(uint32_t w, float s, float m) {
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x = fmaf((float)(w >> (4 * i) & 15u), s, m), y = fmaf((float)(w >> (4 * i + 16) & 15u), s, m);
    x = x > 65504.f ? 65504.f : x < -65504.f ? -65504.f : x;
    y = y > 65504.f ? 65504.f : y < -65504.f ? -65504.f : y;
    r[i] = pack2<__half>(x, y);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}
// A group's (scale, minimum) as halves; wide(): the top bit of either place is set where the fast conversion does not serve
template <typename T> struct Group;
template <> struct Group<__half> {
  static __device__ __forceinline__ uint32_t wide(uint32_t g) { return (g & 0x7fff7fffu) + 0x18001800u; }   // from 2048 on
  static __device__ __forceinline__ __half2 both(uint32_t g, int which) {
    const uint32_t x = __byte_perm(g, g, which ? 0x3232 : 0x1010);
    return *reinterpret_cast<const __half2*>(&x);
  }
};
template <> struct Group<__nv_bfloat16> {
  // from 2048 on, and, but for zero, below 2^-17, from where on a half holds all digits of a bf16 number
  static __device__ __forceinline__ uint32_t wide(uint32_t g) {
    const uint32_t x = g & 0x7fff7fffu;
    return (x + 0x3b003b00u) | ((x + 0x7fff7fffu) & ~(x + 0x49004900u));
  }
  static __device__ __forceinline__ __half2 both(uint32_t g, int which) {
    const float2 f = kv4::scale_min<__nv_bfloat16>(g);
    return __float2half2_rn(which ? f.y : f.x);
  }
};

// READY: operands that a kernel before this one has made come as whole tiles, and there are no converting warps.
template <typename T, int D, int GS, bool READY>
__global__ void __launch_bounds__(READY ? kReadyThreads : kThreads, 1) kv4_prompt_kernel(const Params p) {
  constexpr int kSoftmaxWarp = READY ? 4 : 12, kAll = READY ? kReadyThreads : kThreads;
  constexpr int DP = D < 64 ? 64 : D;             // a row of an operand is whole swizzle atoms of 64 halves
  constexpr int kTile = kBN * DP * 2, kHalf = kBN * 64 * 2, NG = D / GS;
  constexpr int kN = READY ? kBN : kBN / 2, kParts = kBN / kN;     // keys of a product; products of a key tile
  extern __shared__ __align__(1024) uint8_t smem[];
  Ctl* ctl = reinterpret_cast<Ctl*>(smem);
  uint8_t* q_s = smem + 1024;
  uint8_t* k_ring = q_s + 2 * kTile;
  uint8_t* v_ring = k_ring + kKStages * kTile;
  uint8_t* raw_ring = v_ring + kVStages * kTile;
  int* prefix = reinterpret_cast<int*>(raw_ring + (READY ? 0 : kUnits * kUnitKeys * kUnitPitch));   // steps of the sequences before, [batch + 1]
  int* items = prefix + kMaxBatch + 1;            // row blocks (of all kv heads) before
  Seq* seqs = reinterpret_cast<Seq*>(items + kMaxBatch);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.G;

  if (threadIdx.x == 0) {
    mbar_init(&ctl->s_free, 4);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&ctl->q_full[t], 4);
      for (int h = 0; h < 2; ++h) { mbar_init(&ctl->s_full[t][h], 1); mbar_init(&ctl->p_full[t][h], 4); mbar_init(&ctl->pv_done[t][h], 1); }
    }
    for (int s = 0; s < kKStages; ++s) { mbar_init(&ctl->k_full[s], READY ? 1 : kConvert / 32); mbar_init(&ctl->k_empty[s], 1); }
    for (int s = 0; s < kVStages; ++s) { mbar_init(&ctl->v_full[s], READY ? 1 : kConvert / 32); mbar_init(&ctl->v_empty[s], 1); }
    for (int s = 0; s < kUnits; ++s) { mbar_init(&ctl->raw_full[s], 64); mbar_init(&ctl->raw_empty[s], kConvert / 32); }
    for (int s = 0; s < kSegs; ++s) mbar_init(&ctl->seg_done[s], 8);
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(&ctl->tmem_base, 512);
    tmem_relinquish();
    pdl_launch_dependents();                      // only once this CTA owns its tensor memory
  }
  pdl_wait_prior();                               // lengths, table, cache, q are upstream data

  // ---- steps and row blocks per sequence (a warp each), then their sums ----
  for (int b = warp; b < p.batch; b += kAll / 32) {
    const Seq s = sequence(p, b);
    const int nb = row_blocks(p, s);
    int n = 0;
    for (int rb = lane; rb < nb; rb += 32) n += block_steps(p, s, rb);
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) {
      seqs[b] = s;
      prefix[b + 1] = n * p.Hkv;
      items[b] = nb * p.Hkv;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) {
    int steps = 0, blocks = 0;
    bool full = false;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
      const int b = b0 + lane;
      int s = b < p.batch ? prefix[b + 1] : 0;
      const int own = b < p.batch ? items[b] : 0;
      int k = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, s, o), y = __shfl_up_sync(0xffffffffu, k, o);
        if (lane >= o) { s += x; k += y; }
      }
      // Disjoint ranges of q fit into the workspace by its size.  Of others (stale starts), the sequences from the first on that does not fit
      // are left out.  (The sum up to it is below 2^32; what stands behind it in the scan is not used.)
      const unsigned past = __ballot_sync(0xffffffffu, full || (uint32_t)blocks + (uint32_t)k > p.items);
      bool out = false;
      if (past != 0u) {
        const int first = __ffs(past) - 1, from = first > 0 ? first - 1 : 0;
        const int s_kept = __shfl_sync(0xffffffffu, s, from), k_kept = __shfl_sync(0xffffffffu, k, from);
        full = true;
        out = lane >= first;
        if (out) {
          s = first > 0 ? s_kept : 0;
          k = first > 0 ? k_kept : 0;
        }
      }
      if (b < p.batch) {
        const int before = blocks + k - (out ? 0 : own);
        prefix[b + 1] = steps + s;
        items[b] = before;
        if (blockIdx.x == 0) p.ws_item[b] = make_int4(before, out ? 0 : seqs[b].m, seqs[b].start, 0);
      }
      steps += __shfl_sync(0xffffffffu, s, 31);
      blocks += __shfl_sync(0xffffffffu, k, 31);
    }
    if (lane == 0) prefix[0] = 0;
  }
  __syncthreads();
  const uint32_t tmem_base = ctl->tmem_base;

  const int total = prefix[p.batch], shares = total < (int)gridDim.x ? total : (int)gridDim.x;
  int step = 0, step_end = 0;
  if ((int)blockIdx.x < shares) {
    step = (int)((int64_t)blockIdx.x * total / shares);
    step_end = (int)((int64_t)(blockIdx.x + 1) * total / shares);
  }
  auto next = [&](Segment& g, Seq& s) -> bool {
    if (step >= step_end) return false;
    int lo = 0, n = p.batch;                      // the last sequence that begins at or before `step` and has steps
    while (n > 1) {
      const int half = n / 2;
      if (prefix[lo + half] <= step) { lo += half; n -= half; }
      else n = half;
    }
    s = seqs[lo];
    const int per_head = (prefix[lo + 1] - prefix[lo]) / p.Hkv, nb = row_blocks(p, s);
    int y = step - prefix[lo];
    g.b = lo;
    g.kvh = y / per_head;
    y -= g.kvh * per_head;
    g.steps = block_steps(p, s, 0);
    for (g.rb = 0; g.rb < nb - 1 && y >= g.steps;) {
      y -= g.steps;
      g.steps = block_steps(p, s, ++g.rb);
    }
    g.j0 = y;
    const int left = step_end - step;
    g.j1 = left < g.steps - y ? y + left : g.steps;
    g.item = items[lo] + g.kvh * nb + g.rb;
    step += g.j1 - g.j0;
    return true;
  };

  Segment seg;
  Seq seq;
  // registers per lane: 20 warps x 96 at launch >= 4 x 56 + 8 x 72 + 8 x 136
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp < 2) {
      // ===================== tensor-core issuers: warp 0 the scores, warp 1 P V =====================
      // Halves of a tile's scores alternate between its two buffers, and the probabilities take their place there: a buffer is written
      // again when P V of the half that was in it is done, half a tile after it was asked for.
      constexpr uint32_t idesc_s = umma_idesc(1u, 0u, 0u, 0u, 0u, kBM, kN);
      constexpr uint32_t idesc_o = umma_idesc(1u, 0u, 0u, 0u, 1u, kBM, DP);
      int ring = 0;
      uint32_t phase = 0, q_phase = 0, par = 0, used = 0;   // a bit to a tile: of its Q, of its key tiles; whether it had one
      while (next(seg, seq)) {
        const int nt0 = key_tiles(p, seq, seg.rb, 0), nt1 = key_tiles(p, seq, seg.rb, 1);
        for (int j = seg.j0; j < seg.j1; ++j) {
          kv4_wait(warp == 0 ? &ctl->k_full[ring] : &ctl->v_full[ring], phase);
#pragma unroll 1
          for (int x = 0; x < 2 * kParts; ++x) {
            const int t = x & 1, h = x >> 1;
            if (j >= (t ? nt1 : nt0)) continue;
            const bool last = h == kParts - 1 && (t == 1 || j >= nt1);    // the key tile's last reader
            if (warp == 0) {
              if (h == 0 && j == seg.j0) { kv4_wait(&ctl->q_full[t], q_phase >> t & 1u); q_phase ^= 1u << t; }
              if (READY) {
                if (used) { kv4_wait(&ctl->s_free, par); par ^= 1u; }      // the product before is in its threads' registers
                used = 1u;
              } else {
                if (used >> t & 1u) kv4_wait(&ctl->pv_done[t][h], (par >> t & 1u) ^ 1u);   // of the key tile before
                if (h == 1) { used |= 1u << t; par ^= 1u << t; }
              }
              tc_fence_after();
              if (elect_one()) {
                const uint64_t q_desc = umma_desc_sw128_kmajor(smem_u32(q_s + t * kTile));
                const uint64_t k_desc = umma_desc_sw128_kmajor(smem_u32(k_ring + ring * kTile + h * (kBN / 2) * 128));
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk) {
                  const uint64_t off = (uint64_t)(((kk >> 2) * kHalf + (kk & 3) * 32) >> 4);
                  umma_f16(tmem_base + (uint32_t)(READY ? 0 : t * 128 + h * 64), q_desc + off, k_desc + off, idesc_s, kk ? 1u : 0u);
                }
                if (last) tc_commit(&ctl->k_empty[ring]);
                tc_commit(&ctl->s_full[t][h]);
              }
            } else {
              kv4_wait(&ctl->p_full[t][h], par >> t & 1u);
              if (h == kParts - 1) par ^= 1u << t;
              tc_fence_after();
              if (elect_one()) {
                const uint32_t v_addr = smem_u32(v_ring + ring * kTile + h * (kBN / 2) * 128);
#pragma unroll
                for (int kk = 0; kk < kN / 16; ++kk) {
                  // 16 keys per step = two 8-row groups of 1024 B; elements 64 .. 127 are one LBO away
                  const uint64_t v_desc = umma_desc_sw128_mnmajor(v_addr + kk * 2048, kHalf, 1024);
                  umma_ts(tmem_base + 256u + (uint32_t)t * 128u, tmem_base + (uint32_t)(READY ? 128 + t * 64 : t * 128 + h * 64) + kk * 8, v_desc, idesc_o,
                          (j > seg.j0 || h || kk) ? 1u : 0u);
                }
                if (last) tc_commit(&ctl->v_empty[ring]);
                tc_commit(&ctl->pv_done[t][h]);
              }
            }
            __syncwarp();
          }
          if (++ring == (warp == 0 ? kKStages : kVStages)) { ring = 0; phase ^= 1u; }
        }
      }
    } else if (READY) {
      // ===================== operands' tiles =====================
      int ks = 0, vs = 0, nseg = 0;
      uint32_t kp = 1, vp = 1;
      for (; warp == 2 && next(seg, seq); ++nseg) {
        const int slot = nseg % kSegs;
        if (nseg >= kSegs) kv4_wait(&ctl->seg_done[slot], (uint32_t)(nseg / kSegs - 1) & 1u);
        if (lane < 4) ctl->nan_at[slot][lane] = INT_MAX;
        __syncwarp();
        int64_t at = ((int64_t)seg.b * p.Hkv + seg.kvh) * p.ready_tiles + seg.j0;
        for (int j = seg.j0; j < seg.j1; ++j, ++at) {
          const uint8_t* tile = p.ready + at * 2 * kTile;
          const int nan = lane < NG ? __ldcg(reinterpret_cast<const int*>(p.ready_nan + at) + lane) : INT_MAX;
          kv4_wait(&ctl->k_empty[ks], kp);
          if (elect_one()) {
            mbar_arrive_expect_tx(&ctl->k_full[ks], kTile);
            bulk_g2s(k_ring + ks * kTile, tile, kTile, &ctl->k_full[ks]);
          }
          __syncwarp();
          if (++ks == kKStages) { ks = 0; kp ^= 1u; }
          if (nan != INT_MAX) atomicMin(&ctl->nan_at[slot][lane], nan);
          __syncwarp();
          kv4_wait(&ctl->v_empty[vs], vp);
          if (elect_one()) {
            mbar_arrive_expect_tx(&ctl->v_full[vs], kTile);
            bulk_g2s(v_ring + vs * kTile, tile + kTile, kTile, &ctl->v_full[vs]);
          }
          __syncwarp();
          if (++vs == kVStages) { vs = 0; vp ^= 1u; }
        }
      }
    } else {
      // ===================== cache rows: codes and groups of 64 keys of one side, a unit =====================
      constexpr int kPiece = kv4::head_bytes(D, GS) % 16 == 0 ? 16 : 8, kLanes = D / 2 / kPiece, kGroupBytes = 4 * NG;
      const int wk = (warp - 2) * 32;             // this warp's keys of a unit
      int us = 0;
      uint32_t up = 1;
      while (next(seg, seq)) {
        const int32_t* entry = p.table + (int64_t)seq.req * p.tab_rs;
        const uint8_t* head = p.cache + (int64_t)seg.kvh * kv4::head_bytes(D, GS);
        auto row_of = [&](int j, int h) -> int {  // -1: past the sequence
          const int key = j * kBN + h * kUnitKeys + wk + lane;
          if (key >= seq.keys) return -1;
          const int row = ld_upstream(entry + (int64_t)key * p.tab_cs);
          return row >= 0 && row < p.max_tokens ? row : 0;
        };
        int ahead[2] = {row_of(seg.j0, 0), row_of(seg.j0, 1)};
        for (int j = seg.j0; j < seg.j1; ++j) {
          const int rows[2] = {ahead[0], ahead[1]};
          if (j + 1 < seg.j1) { ahead[0] = row_of(j + 1, 0); ahead[1] = row_of(j + 1, 1); }
#pragma unroll 1
          for (int u = 0; u < 4; ++u) {
            const int side = u >> 1, row = (u & 1) ? rows[1] : rows[0];
            kv4_wait(&ctl->raw_empty[us], up);
            uint8_t* unit = raw_ring + us * kUnitKeys * kUnitPitch + wk * kUnitPitch;
#pragma unroll
            for (int i = 0; i < kLanes; ++i) {    // 32 / kLanes keys at a time, kLanes neighbours to a key
              const int k = i * (32 / kLanes) + lane / kLanes, c = lane % kLanes * kPiece;
              const int r = __shfl_sync(0xffffffffu, row, k);
              copy_async<kPiece>(unit + k * kUnitPitch + c, head + (int64_t)(r < 0 ? 0 : r) * p.row_stride + side * (D / 2) + c, r >= 0);
            }
            copy_async<kGroupBytes>(unit + lane * kUnitPitch + D / 2, head + (int64_t)(row < 0 ? 0 : row) * p.row_stride + D + side * kGroupBytes,
                                    row >= 0);
            copy_async_arrive(&ctl->raw_full[us]);
            if (++us == kUnits) { us = 0; up ^= 1u; }
          }
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
  } else if (warp < kSoftmaxWarp) {
    // ===================== codes to operands =====================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    constexpr int NWD = D == 128 ? 2 : 1;         // words of a row and side that a thread takes (eight threads to a row)
    const int tid = threadIdx.x - 128, l = tid & 7, kq = tid >> 3;
    const bool on = l < D / 8;                    // D = 32: half of the threads store zeros
    const uint32_t spot = (uint32_t)(kq * 128 + ((l ^ (kq & 7)) << 4));
    int ks = 0, vs = 0, us = 0, nseg = 0;
    uint32_t kp = 1, vp = 1, up = 0;
    for (; next(seg, seq); ++nseg) {
      const int slot = nseg % kSegs;
      if (nseg >= kSegs) kv4_wait(&ctl->seg_done[slot], (uint32_t)(nseg / kSegs - 1) & 1u);
      if (tid < 4) ctl->nan_at[slot][tid] = INT_MAX;
      asm volatile("bar.sync 2, %0;" ::"n"(kConvert) : "memory");
#pragma unroll 1
      for (int j = seg.j0; j < seg.j1; ++j) {
#pragma unroll 1
        for (int u = 0; u < 4; ++u) {
          const int side = u >> 1, half = u & 1;
          if (half == 0) kv4_wait(side ? &ctl->v_empty[vs] : &ctl->k_empty[ks], side ? vp : kp);
          uint8_t* to = (side ? v_ring + vs * kTile : k_ring + ks * kTile) + half * kUnitKeys * 128 + spot;
          kv4_wait(&ctl->raw_full[us], up);
          const uint8_t* unit = raw_ring + us * kUnitKeys * kUnitPitch + kq * kUnitPitch;
          constexpr int kPass = kConvert / 8, NI = kUnitKeys / kPass;   // rows of all threads; rows of a thread and unit
          uint32_t w[NI][NWD], g[NI][NWD], wide = 0u;
#pragma unroll
          for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int k = 0; k < NWD; ++k) {
              const uint32_t* row = reinterpret_cast<const uint32_t*>(unit + i * kPass * kUnitPitch);
              w[i][k] = on ? row[k * 8 + l] : 0u;
              g[i][k] = on ? row[D / 8 + (k * 8 + l) * 8 / GS] : 0u;
              wide |= Group<T>::wide(g[i][k]);
            }
          if ((wide & 0x80008000u) == 0u) {
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
              for (int k = 0; k < NWD; ++k)
                *reinterpret_cast<uint4*>(to + k * kHalf + i * kPass * 128) = to_halves(w[i][k], Group<T>::both(g[i][k], 0), Group<T>::both(g[i][k], 1));
          } else {                                // outside the range of halves somewhere, or NaN
#pragma unroll 1
            for (int x = 0; x < NI * NWD; ++x) {
              const int i = x / NWD, k = x % NWD, group = (k * 8 + l) * 8 / GS;
              const uint32_t* row = reinterpret_cast<const uint32_t*>(unit + i * kPass * kUnitPitch);
              float2 f = on ? kv4::scale_min<T>(row[D / 8 + group]) : make_float2(0.f, 0.f);
              if (side == 1 && (f.x != f.x || f.y != f.y)) {
                f = make_float2(0.f, 0.f);
                atomicMin(&ctl->nan_at[slot][group], j * kBN + half * kUnitKeys + i * kPass + kq);
              }
              *reinterpret_cast<uint4*>(to + k * kHalf + i * kPass * 128) = to_halves_wide(on ? row[k * 8 + l] : 0u, f.x, f.y);
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctl->raw_empty[us]);
          if (++us == kUnits) { us = 0; up ^= 1u; }
          if (half == 1) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(side ? &ctl->v_full[vs] : &ctl->k_full[ks]);
            if (side) { if (++vs == kVStages) { vs = 0; vp ^= 1u; } }
            else if (++ks == kKStages) { ks = 0; kp ^= 1u; }
          }
        }
      }
    }
  } else {
    if (READY) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");   // 12 warps x 168 at launch >= 4 x 56 + 8 x 216
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
    // ===================== softmax: thread = query row = TMEM lane of tile t =====================
    const int t = (warp - kSoftmaxWarp) >> 2, quad = warp & 3;
    const int row = quad * 32 + lane;
    const uint32_t lane_base = tmem_base + ((uint32_t)(quad * 32) << 16);
    const uint32_t sb = lane_base + (READY ? 0u : (uint32_t)t * 128u), ob = lane_base + 256u + (uint32_t)t * 128u;
    constexpr float kLazy = 8.0f;                 // log2 units: rescale only when a tile exceeds m_used by 2^8
    uint32_t par = 0;                             // of the key tiles
    int nseg = 0;
    for (; next(seg, seq); ++nseg) {
      // A row tile without keys here has nothing to wait for: it must not arrive for a segment before all have left the slot's last one.
      if (nseg >= kSegs) kv4_wait(&ctl->seg_done[nseg % kSegs], (uint32_t)(nseg / kSegs - 1) & 1u);
      const int nt = key_tiles(p, seq, seg.rb, t), j_end = nt < seg.j1 ? nt : seg.j1;
      const int r = seg.rb * kRows + t * kBM + row;
      const int token = over_G(p, r), head = seg.kvh * G + r - token * G;
      const bool live = token < seq.m;
      const int64_t place = live ? seq.start + token : 0;
      const int64_t part = ((int64_t)blockIdx.x * 2 + (seg.j0 == 0 ? 1 : 0)) * kRows + t * kBM + row;
      const bool whole = seg.j0 == 0 && seg.j1 == seg.steps;
      float m_used = -INFINITY, l_run = 0.f;      // m_used: the maximum the accumulated P / O / l are scaled by
      if (j_end > seg.j0) {
        // The tile's rows of Q, in the operands' order: neighbouring threads take a row's 16-byte pieces, all asked for
        // before the first is converted (a row to a thread took 7 us, this 4).
        float scale = p.scale_log2;
        {
          constexpr int kLanes = D / 8, kPass = 128 / kLanes;      // pieces of a row; rows at a time
          const int tid = quad * 32 + lane, c = tid % kLanes;
          const int y0 = tid / kLanes, yr = seg.rb * kRows + t * kBM + y0;
          uint8_t* dst = q_s + t * kTile + (c >> 3) * kHalf + y0 * 128 + (((c & 7) ^ (y0 & 7)) << 4);
          {
            const int by = over_G(p, kPass), on = kPass - by * G;  // tokens and heads from a row to the next
            int yt = over_G(p, yr), yh = yr - yt * G;
            const T* src = reinterpret_cast<const T*>(p.q) + (int64_t)(seq.start + yt) * p.q_ts + (int64_t)(seg.kvh * G + yh) * p.q_hs + c * 8;
            const int64_t step = by * p.q_ts + on * p.q_hs, wrap = p.q_ts - G * p.q_hs;
#pragma unroll 2
            for (int i = 0; i < kBM / kPass; ++i) {
              const bool live_row = yt < seq.m;
              const T* from = live_row ? src : reinterpret_cast<const T*>(p.q);
              if (p.q_vec) {
                copy_async<16>(dst + i * kPass * 128, from, live_row);
              } else {
#pragma unroll 1
                for (int e = 0; e < 8; ++e)
                  reinterpret_cast<uint16_t*>(dst + i * kPass * 128)[e] = live_row ? reinterpret_cast<const uint16_t*>(from)[e] : (uint16_t)0;
              }
              yt += by;
              yh += on;
              src += step;
              if (yh >= G) { yh -= G; ++yt; src += wrap; }
            }
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
          constexpr int kTogether = 4;
#pragma unroll 1
          for (int i = 0; i < kBM / kPass; i += kTogether) {       // in place: a thread's own pieces
            uint4 x[kTogether];
#pragma unroll
            for (int k = 0; k < kTogether; ++k) x[k] = *reinterpret_cast<const uint4*>(dst + (i + k) * kPass * 128);
            if (std::is_same<T, __nv_bfloat16>::value) {
              float big[kTogether];
#pragma unroll
              for (int k = 0; k < kTogether; ++k) {
                const uint32_t* w = &x[k].x;
                big[k] = 0.f;
#pragma unroll
                for (int n = 0; n < 4; ++n) big[k] = max3(big[k], fabsf(__uint_as_float(w[n] << 16)), fabsf(__uint_as_float(w[n] & 0xffff0000u)));
              }
#pragma unroll
              for (int o = 1; o < kLanes; o <<= 1)
#pragma unroll
                for (int k = 0; k < kTogether; ++k) big[k] = fmaxf(big[k], __shfl_xor_sync(0xffffffffu, big[k], o));
#pragma unroll
              for (int k = 0; k < kTogether; ++k) {
                uint32_t* w = &x[k].x;
                int e = 8 - ((int)(__float_as_uint(big[k]) >> 23) - 127);
                if (!(big[k] < INFINITY) || big[k] == 0.f) e = 0;
                e = e < -100 ? -100 : e > 100 ? 100 : e;
                const float up = __int_as_float((e + 127) << 23);
#pragma unroll
                for (int n = 0; n < 4; ++n) w[n] = pack2<__half>(__uint_as_float(w[n] << 16) * up, __uint_as_float(w[n] & 0xffff0000u) * up);
                if (c == 0) ctl->q_exp[t][y0 + (i + k) * kPass] = (int8_t)e;
              }
            }
#pragma unroll
            for (int k = 0; k < kTogether; ++k)
              *reinterpret_cast<uint4*>(dst + (i + k) * kPass * 128) = make_uint4(
                  __byte_perm(x[k].x, x[k].z, 0x5410), __byte_perm(x[k].x, x[k].z, 0x7632), __byte_perm(x[k].y, x[k].w, 0x5410), __byte_perm(x[k].y, x[k].w, 0x7632));
          }
          if (D < DP) {                                            // the atom's other half
            for (int i = tid; i < kBM * 4; i += 128)
              *reinterpret_cast<uint4*>(q_s + t * kTile + (i >> 2) * 128 + ((((i & 3) + 4) ^ ((i >> 2) & 7)) << 4)) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          asm volatile("bar.sync %0, 128;" ::"r"(3 + t) : "memory");
          if (std::is_same<T, __nv_bfloat16>::value) scale *= __int_as_float((127 - (int)ctl->q_exp[t][row]) << 23);
          if (lane == 0) mbar_arrive(&ctl->q_full[t]);
        }
        const int pos = seq.ctx + token, see = live ? (pos < seq.keys - 1 ? pos : seq.keys - 1) : -1;   // last key that counts
        const int see_all = __reduce_min_sync(0xffffffffu, live ? see : INT_MAX);

        // Loops stay rolled and the mask is a pass of its own: with copies for masked tiles and for either half the roles' code did not
        // fit into the instruction cache (6000 cycles a step, most of them waiting for instructions).
#pragma unroll 1
        for (int j = seg.j0; j < j_end; ++j) {
          const bool masked = (j + 1) * kBN - 1 > see_all;
#pragma unroll 1
          for (int h = 0; h < kParts; ++h) {
            kv4_wait(&ctl->s_full[t][h], par);
            tc_fence_after();
            const uint32_t buf = sb + (uint32_t)h * 64u;
            uint32_t sv[kN];
#pragma unroll
            for (int c = 0; c < kN; c += 32) tmem_ld_32x32b_x32(buf + c, *reinterpret_cast<uint32_t(*)[32]>(sv + c));
            tc_wait_ld();
            if (READY) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&ctl->s_free);
            }
            if (masked) {
              const int limit = see - j * kBN - h * kN;            // key column i is visible iff i <= limit
#pragma unroll
              for (int i = 0; i < kN; ++i) sv[i] = i <= limit ? sv[i] : 0xff800000u;
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < kN; i += 8)
#pragma unroll
              for (int c = 0; c < 4; ++c) mx[c] = max3(mx[c], __uint_as_float(sv[i + 2 * c]), __uint_as_float(sv[i + 2 * c + 1]));
            const float m_half = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * scale;
            const bool grow = m_half > m_used + kLazy;             // at first m_used = -inf: true
            const float m_new = grow ? m_half : m_used;
            const float base = m_new == -INFINITY ? 0.f : m_new;   // nothing visible yet: avoid inf - inf
            if (READY && j > seg.j0) { kv4_wait(&ctl->pv_done[t][0], par ^ 1u); tc_fence_after(); }   // P's place is free, O rests
            if (__any_sync(0xffffffffu, grow)) {
              const float alpha = grow ? fast_exp2(m_used - base) : 1.0f;
              l_run *= alpha;
              if (j > seg.j0 || h) {
                if (!READY) { kv4_wait(&ctl->pv_done[t][h ^ 1], h ? par : par ^ 1u); tc_fence_after(); }   // of the half before, the last one asked for
#pragma unroll 1
                for (int c = 0; c < DP; c += 32) {
                  uint32_t v[32];
                  tmem_ld_32x32b_x32(ob + c, v);
                  tc_wait_ld();
#pragma unroll
                  for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
                  tmem_st_32x32b_x32(ob + c, v);
                }
              }
            }
            m_used = m_new;
            const uint64_t scale2 = f32x2(scale, scale), base2 = f32x2(-base, -base);
            uint64_t lsum2 = 0ull;
#pragma unroll
            for (int c = 0; c < kN; c += 32) {
              uint32_t pk[16];
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                float p0, p1;
                f32x2_split(f32x2_fma(f32x2(__uint_as_float(sv[c + i]), __uint_as_float(sv[c + i + 1])), scale2, base2), p0, p1);
                p0 = fast_exp2(p0);
                p1 = fast_exp2(p1);
                lsum2 = f32x2_add(lsum2, f32x2(p0, p1));
                pk[i >> 1] = pack2<__half>(p0, p1);
              }
              tmem_st_32x32b_x16((READY ? lane_base + 128u + (uint32_t)t * 64u : buf) + (c >> 1), pk);
            }
            float l0, l1;
            f32x2_split(lsum2, l0, l1);
            l_run += l0 + l1;
            tc_wait_st_();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctl->p_full[t][h]);
          }
          par ^= 1u;
        }
        kv4_wait(&ctl->pv_done[t][kParts - 1], par ^ 1u);      // the last half's, and with it all before
        tc_fence_after();
        // columns are in the operands' order: of eight, 0 4 1 5 2 6 3 7
        const float inv = whole ? (l_run == 0.f ? 0.f : 1.0f / l_run) : 1.f;
        T* orow = reinterpret_cast<T*>(p.out) + place * p.o_ts + (int64_t)(live ? head : 0) * p.o_hs;
        float* prow = p.ws_o + part * D;
        constexpr int kFrom[8] = {0, 2, 4, 6, 1, 3, 5, 7};
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(ob + c, v);          // warp-collective: outside the row predicate
          tc_wait_ld();
          const bool nan = see >= ctl->nan_at[nseg % kSegs][c / GS];
          if (live) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              float x[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) x[k] = nan ? __int_as_float(0x7fc00000) : __uint_as_float(v[i + kFrom[k]]) * inv;
              if (whole) {
                const uint4 w = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
                if (p.o_vec) {
                  *reinterpret_cast<uint4*>(orow + c + i) = w;
                } else {
#pragma unroll
                  for (int k = 0; k < 8; ++k) orow[c + i + k] = from_f32<T>(x[k]);
                }
              } else {
                *reinterpret_cast<float4*>(prow + c + i) = make_float4(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<float4*>(prow + c + i + 4) = make_float4(x[4], x[5], x[6], x[7]);
              }
            }
          }
        }
      }
      if (!whole) {
        p.ws_ml[part] = make_float2(m_used, l_run);
        if (t == 0 && row == 0) {
          int* note = reinterpret_cast<int*>(p.ws_info + seg.item);
          if (seg.j0 == 0) note[0] = blockIdx.x;
          if (seg.j1 == seg.steps) note[1] = blockIdx.x;
        }
      } else if (t == 0 && row == 0) {
        p.ws_info[seg.item] = make_int2(blockIdx.x, blockIdx.x);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->seg_done[nseg % kSegs]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, 512);
}

// Operands of one tile of 128 keys of a kv head, as the tensor cores read them.  Where many row blocks read a tile, its codes are
// converted once here instead of beside the products of each.
template <typename T, int D, int GS>
__global__ void __launch_bounds__(256, 6) kv4_prompt_ready_kernel(const Params p) {
  pdl_prologue();
  constexpr int DP = D < 64 ? 64 : D, kTile = kBN * DP * 2, kHalf = kBN * 64 * 2, NG = D / GS, NWD = D == 128 ? 2 : 1, NI = kBN / 32;
  __shared__ int nan_at[4];
  const int tile = blockIdx.x >> 1, side = blockIdx.x & 1, kvh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, l = tid & 7, kq = tid >> 3;
  const Seq s = sequence(p, b);
  if (s.m == 0 || tile * kBN >= s.keys) {
    // a sequence that sees nothing takes one step for its zeros: of zero operands
    if (s.m == 0 || tile > 0) return;
  }
  if (tid < 4) nan_at[tid] = INT_MAX;
  __syncthreads();
  uint32_t w[NI][NWD], g[NI][NWD];
  int row[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int key = tile * kBN + i * 32 + kq;
    row[i] = -1;
    if (key < s.keys && l < D / 8) {
      const int r = ld_upstream(p.table + (int64_t)s.req * p.tab_rs + (int64_t)key * p.tab_cs);
      row[i] = r >= 0 && r < p.max_tokens ? r : 0;
    }
  }
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int k = 0; k < NWD; ++k) {
      w[i][k] = g[i][k] = 0u;
      if (row[i] >= 0) {
        const uint32_t* head = reinterpret_cast<const uint32_t*>(p.cache + (int64_t)row[i] * p.row_stride + (int64_t)kvh * kv4::head_bytes(D, GS));
        w[i][k] = __ldcg(head + side * (D / 8) + k * 8 + l);
        g[i][k] = __ldcg(head + D / 4 + side * NG + (k * 8 + l) * 8 / GS);
      }
    }
  const int64_t at = ((int64_t)b * p.Hkv + kvh) * p.ready_tiles + tile;
  uint8_t* to = p.ready + (at * 2 + side) * kTile + kq * 128 + ((l ^ (kq & 7)) << 4);
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int k = 0; k < NWD; ++k) {
      const uint32_t x = g[i][k];
      uint4 v;
      if ((Group<T>::wide(x) & 0x80008000u) == 0u) {
        v = to_halves(w[i][k], Group<T>::both(x, 0), Group<T>::both(x, 1));
      } else {
        float2 f = kv4::scale_min<T>(x);
        if (side == 1 && (f.x != f.x || f.y != f.y)) {
          f = make_float2(0.f, 0.f);
          atomicMin(&nan_at[(k * 8 + l) * 8 / GS], tile * kBN + i * 32 + kq);
        }
        v = to_halves_wide(w[i][k], f.x, f.y);
      }
      *reinterpret_cast<uint4*>(to + k * kHalf + i * 32 * 128) = v;
    }
  if (side == 0) return;
  __syncthreads();
  if (tid < 4) reinterpret_cast<int*>(p.ready_nan + at)[tid] = nan_at[tid];
}

// Row blocks that several CTAs met in.  Bound by latency, or by the parts' bytes: a warp asks for the parts of its R rows together, before
// their weights are known, and lanes share the largest scores and sums.
template <typename T, int D, int R>
__global__ void __launch_bounds__(256) kv4_prompt_merge_kernel(const Params p) {
  pdl_prologue();
  constexpr int E = D / 32, kTogether = 16 / R, kLook = 32 / R;      // parts of a row asked for together; lanes that look at one row's
  const int b = blockIdx.z, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r0 = blockIdx.x * 8 * R;
  const int4 s = __ldcg(p.ws_item + b);           // row blocks before, m, start: left in the workspace by the first CTA
  const int rows = s.y * p.G;
  if (r0 >= rows) return;
  const int rb = r0 / kRows, nb = (rows + kRows - 1) / kRows;
  const int2 who = __ldcg(p.ws_info + s.x + kvh * nb + rb);
  const int n = who.y - who.x + 1;
  if (n < 2) return;                              // written by its only CTA
  const int in_block = r0 - rb * kRows + warp * R, here = rows - (r0 + warp * R);
  auto part_of = [&](int i) { return ((int64_t)(who.x + i) * 2 + (i == 0 ? 1 : 0)) * kRows + in_block; };
  float x[kTogether][R][E], acc[R][E];
  auto ask = [&](int from) {
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      if (from + i >= n) continue;
      const float* row = p.ws_o + part_of(from + i) * D + lane * E;
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (E == 4) *reinterpret_cast<float4*>(x[i][k]) = __ldcg(reinterpret_cast<const float4*>(row + k * D));
        else if (E == 2) *reinterpret_cast<float2*>(x[i][k]) = __ldcg(reinterpret_cast<const float2*>(row + k * D));
        else x[i][k][0] = __ldcg(row + k * D);
      }
    }
  };
  auto look = [&](int from) -> float2 {           // lane (row, part): its largest score and its sum
    const int i = from + lane % kLook;
    return i < n ? __ldcg(p.ws_ml + part_of(i) + lane / kLook) : make_float2(-INFINITY, 0.f);
  };
  ask(0);
  const float2 first = look(0);
  float M = first.x;
#pragma unroll 1
  for (int from = kLook; from < n; from += kLook) M = fmaxf(M, look(from).x);
#pragma unroll
  for (int o = 1; o < kLook; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  const float base = M == -INFINITY ? 0.f : M;
  float L = 0.f, w = 0.f;
#pragma unroll
  for (int k = 0; k < R; ++k)
#pragma unroll
    for (int e = 0; e < E; ++e) acc[k][e] = 0.f;
#pragma unroll 1
  for (int from = 0; from < n; from += kTogether) {
    if (from % kLook == 0) {
      const float2 ml = from == 0 ? first : look(from);
      // A sum of zero: of keys that the row does not see, nothing was stored.  A weight that is zero counts: the part may hold a NaN.
      w = ml.y == 0.f ? -1.f : fast_exp2(ml.x - base);
      if (!(w < 0.f)) L = fmaf(ml.y, w, L);
    }
#pragma unroll
    for (int i = 0; i < kTogether; ++i)
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const float wi = __shfl_sync(0xffffffffu, w, k * kLook + from % kLook + i);
        if (!(wi < 0.f)) {
#pragma unroll
          for (int e = 0; e < E; ++e) acc[k][e] = fmaf(x[i][k][e], wi, acc[k][e]);
        }
      }
    ask(from + kTogether);
  }
#pragma unroll
  for (int o = 1; o < kLook; o <<= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const float sum = __shfl_sync(0xffffffffu, L, k * kLook), inv = sum == 0.f ? 0.f : 1.0f / sum;
    if (k >= here) continue;
    const int r = r0 + warp * R + k, token = over_G(p, r), head = kvh * p.G + r - token * p.G;
    T* out = reinterpret_cast<T*>(p.out) + (int64_t)(s.z + token) * p.o_ts + (int64_t)head * p.o_hs + lane * E;
    if (p.o_vec && E == 4) {
      *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(acc[k][0] * inv, acc[k][1 % E] * inv), pack2<T>(acc[k][2 % E] * inv, acc[k][3 % E] * inv));
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) out[e] = from_f32<T>(acc[k][e] * inv);
    }
  }
}

struct Plan { int grid, smem, ready_tiles; int64_t items, rows, steps, ready_bytes; };   // ready_tiles 0: operands are made beside the products

// Row blocks of a portion, on average, from which on operands are made ready.  1 x 320 / 384 / 512 tokens (5 to 8 blocks) over 7500: 72.0 /
// 76.1 / 89.6 us ready, 72.7 / 80.2 / 98.5 converted beside the products; 256 (4 blocks): 66.5 and 64.6; 6 x 290 / 400 at most over 1200:
// 73.2 / 82.3 and 76.2 / 90.0; 6 x 200: 58.5 and 54.2.
constexpr int kReadyBlocks = 5;
// And steps of a CTA, by the bounds.  One portion of 1000 tokens over none / 1000 (7 / 15 steps): 52.6 / 61.0 us ready, 49.9 / 64.2 the other
// way; 500 over 1000 / 2000 / 4000 (6 / 10 / 17): 45.5 / 51.9 / 64.7 and 44.7 / 51.4 / 68.1; 2000 over 6000: 215 and 279.
constexpr int kReadySteps = 10;
// Their room in the workspace at most: 65536 keys of 8 heads.  It grows with batch * max_seq_len, of which ragged steps use a part.
constexpr int64_t kReadyMost = 256ll << 20;
// Parts of a row block from which on a warp merges one row at a time, sixteen parts together, instead of four rows, four parts together:
// 64 tokens over 7500 (9 parts, 8 kv heads) 34.7 us and 39.4, 128 tokens (6 parts) 48.8 and 48.1, 256 tokens 67.5 and 61.7.
constexpr int kManyParts = 8;

Plan make_plan(int64_t batch, int64_t total, int G, int Hkv, int D, int64_t max_len) {
  Plan pl;
  const int DP = D < 64 ? 64 : D;
  const int64_t rows = batch < kMaxBatch ? batch : kMaxBatch, tiles = cdiv64(max_len > 0 ? max_len : 1, kBN);
  const int lists = (2 * kMaxBatch + 1) * 4 + kMaxBatch * (int)sizeof(Seq);
  pl.items = (cdiv64(total * G, kRows) + rows) * Hkv;   // of disjoint ranges of q at most; the kernel takes no more
  pl.steps = pl.items * tiles;
  pl.grid = (int)(pl.steps < b2l_num_sms() ? pl.steps : b2l_num_sms());
  if (pl.grid < 1) pl.grid = 1;
  pl.rows = 2ll * pl.grid * kRows;
  // A tile is read by every row block that sees it: converted once for all of them where they are several, with room for the tiles
  // of the bounds.
  const int64_t tile = 2ll * kBN * DP * 2;
  const bool ready = total * G > (kReadyBlocks - 1) * kRows * batch && rows * Hkv * tiles <= kReadyMost / tile &&
                     pl.steps >= (int64_t)kReadySteps * b2l_num_sms();
  pl.ready_tiles = ready ? (int)tiles : 0;
  pl.ready_bytes = ready ? rows * Hkv * tiles * (tile + 16) : 0;
  pl.smem = 1024 + (2 + kKStages + kVStages) * kBN * DP * 2 + (ready ? 0 : kUnits * kUnitKeys * kUnitPitch) + lists;
  return pl;
}
// partial rows, notes, sequences, each from a multiple of 16 bytes on; the ready operands first
int64_t workspace_for(const Plan& pl, int D) { return pl.ready_bytes + pl.rows * (D + 2) * 4 + (pl.items + 1) / 2 * 16 + (int64_t)kMaxBatch * 16; }

template <typename T, int D, int GS>
int launch(const Params& p, const Plan& pl, cudaStream_t st) {
  static int configured[2][64] = {{0}};
  const bool ready = pl.ready_tiles > 0;
  auto kern = ready ? kv4_prompt_kernel<T, D, GS, true> : kv4_prompt_kernel<T, D, GS, false>;
  B2L_CUDA_CHECK(b2l_ensure_dynamic_smem(kern, pl.smem, configured[ready]));
  if (ready) {
    b2l_launch(kv4_prompt_ready_kernel<T, D, GS>, dim3(2u * (unsigned)pl.ready_tiles, (unsigned)p.Hkv, (unsigned)p.batch), dim3(256), (size_t)0, st, p);
    B2L_LAUNCH_CHECK();
  }
  b2l_launch(kern, dim3((unsigned)pl.grid), dim3(ready ? kReadyThreads : kThreads), (size_t)pl.smem, st, p);
  B2L_LAUNCH_CHECK();
  // many parts to a row block, or few: a row to a warp, or four
  if (pl.grid > kManyParts * pl.items)
    b2l_launch(kv4_prompt_merge_kernel<T, D, 1>, dim3((unsigned)cdiv64(p.max_new * p.G, 8), (unsigned)p.Hkv, (unsigned)p.batch), dim3(256), (size_t)0, st, p);
  else
    b2l_launch(kv4_prompt_merge_kernel<T, D, 4>, dim3((unsigned)cdiv64(p.max_new * p.G, 32), (unsigned)p.Hkv, (unsigned)p.batch), dim3(256), (size_t)0, st, p);
  B2L_LAUNCH_CHECK();
  return B2L_OK;
}

}  // namespace kv4p

extern "C" int64_t b2l_flash_attention_int4_workspace_bytes(int64_t batch, int64_t total_tokens, int num_q_heads, int num_kv_heads,
                                                            int head_dim, int group, int64_t max_seq_len) {
  if (batch <= 0 || total_tokens <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 || !kv4::shape_ok(head_dim, group))
    return 0;
  return kv4p::workspace_for(kv4p::make_plan(batch, total_tokens, num_q_heads / num_kv_heads, num_kv_heads, head_dim, max_seq_len), head_dim);
}

extern "C" int b2l_flash_attention_int4(void* out, const void* q, const void* cache, int64_t cache_row_stride, int64_t max_tokens,
                                        const void* b_start_loc, int start_width, const void* b_new_len, int new_width,
                                        const void* b_req_tokens_table, int64_t table_req_stride, int64_t table_seq_stride,
                                        int64_t table_requests, int64_t table_width, const void* b_req_idx, int req_width,
                                        const void* b_seq_len, int len_width, int64_t batch, int64_t total_tokens, int64_t max_new_len,
                                        int num_q_heads, int num_kv_heads, int head_dim, int group, int64_t max_seq_len, float qk_scale,
                                        int64_t q_tok_stride, int64_t q_head_stride, int64_t o_tok_stride, int64_t o_head_stride,
                                        void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
  using namespace kv4p;
  const char* what = "flash_attention_int4";
  B2L_REQUIRE(out && q && cache && b_start_loc && b_new_len && b_req_tokens_table && b_req_idx && b_seq_len, "%s: null pointer", what);
  B2L_REQUIRE(num_q_heads > 0 && num_kv_heads > 0 && num_q_heads % num_kv_heads == 0 && num_kv_heads <= 65535,
              "%s: num_q_heads (%d) must be a multiple of num_kv_heads (%d)", what, num_q_heads, num_kv_heads);
  B2L_REQUIRE(kv4::shape_ok(head_dim, group), "%s: head_dim %d with groups of %d (head_dim 32, 64 or 128; groups of 32, 64 or 128, at most head_dim)",
              what, head_dim, group);
  for (int w : {start_width, new_width, req_width, len_width}) B2L_REQUIRE(w == 4 || w == 8, "%s: index widths must be 4 or 8", what);
  B2L_REQUIRE(cache_row_stride >= kv4::row_bytes(num_kv_heads, head_dim, group) && cache_row_stride % 16 == 0 && (uintptr_t)cache % 16 == 0,
              "%s: cache rows must be 16-byte aligned and hold %lld bytes", what, (long long)kv4::row_bytes(num_kv_heads, head_dim, group));
  B2L_REQUIRE(dtype == B2L_F16 || dtype == B2L_BF16, "%s: dtype %d", what, dtype);
  B2L_REQUIRE(qk_scale > 0.f && qk_scale < INFINITY, "%s: qk_scale must be positive", what);
  B2L_REQUIRE(batch >= 0 && total_tokens >= 0 && max_tokens > 0 && max_tokens < (1ll << 31) && table_requests >= 0 && table_width >= 0 &&
                  max_new_len >= 0 && max_new_len < (1ll << 30) && max_seq_len < (1ll << 30), "%s: bad shape", what);
  if (batch == 0 || total_tokens == 0 || max_new_len == 0) return B2L_OK;
  const int G = num_q_heads / num_kv_heads;
  const int64_t most = max_seq_len < table_width ? max_seq_len : table_width;
  const Plan pl = make_plan(batch, total_tokens, G, num_kv_heads, head_dim, max_seq_len);
  B2L_REQUIRE(pl.steps < (1ll << 31) && total_tokens * G < (1ll << 31), "%s: too many tokens", what);
  B2L_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 &&
                  workspace_bytes >= workspace_for(pl, head_dim),
              "%s: workspace too small", what);
  Params p;
  p.q = q; p.q_ts = q_tok_stride; p.q_hs = q_head_stride;
  p.q_vec = (uintptr_t)q % 16 == 0 && q_tok_stride % 8 == 0 && q_head_stride % 8 == 0;
  p.out = out; p.o_ts = o_tok_stride; p.o_hs = o_head_stride;
  p.o_vec = (uintptr_t)out % 16 == 0 && o_tok_stride % 8 == 0 && o_head_stride % 8 == 0;
  p.cache = (const uint8_t*)cache; p.row_stride = cache_row_stride; p.max_tokens = max_tokens;
  p.table = (const int32_t*)b_req_tokens_table; p.tab_rs = table_req_stride; p.tab_cs = table_seq_stride; p.requests = table_requests;
  p.start_w = start_width; p.fresh_w = new_width; p.req_w = req_width; p.len_w = len_width;
  p.Hkv = num_kv_heads; p.G = G; p.by_G = G > 1 ? ~0ull / G + 1 : 0;
  p.total = total_tokens; p.max_new = max_new_len < total_tokens ? max_new_len : total_tokens;
  p.most = most < 0 ? 0 : most;
  p.items = (uint32_t)pl.items;
  p.scale_log2 = qk_scale * 1.4426950408889634f;
  char* ws = (char*)workspace;
  p.ready = (uint8_t*)ws;
  p.ready_tiles = pl.ready_tiles;
  p.ready_nan = (int4*)(ws + pl.ready_bytes / (2ll * kBN * (head_dim < 64 ? 64 : head_dim) * 2 + 16) * (2ll * kBN * (head_dim < 64 ? 64 : head_dim) * 2));
  p.ws_o = (float*)(ws + pl.ready_bytes);
  p.ws_ml = (float2*)(p.ws_o + pl.rows * head_dim);
  p.ws_info = (int2*)(p.ws_ml + pl.rows);
  p.ws_item = (int4*)((char*)p.ws_info + (pl.items + 1) / 2 * 16);
  cudaStream_t st = (cudaStream_t)stream;
  for (int64_t b0 = 0; b0 < batch; b0 += kMaxBatch) {
    p.batch = (int)(batch - b0 < kMaxBatch ? batch - b0 : kMaxBatch);
    p.start = (const char*)b_start_loc + b0 * start_width;
    p.fresh = (const char*)b_new_len + b0 * new_width;
    p.req = (const char*)b_req_idx + b0 * req_width;
    p.len = (const char*)b_seq_len + b0 * len_width;
    int rc;
    if (dtype == B2L_F16) { KV4_DISPATCH_SHAPE(head_dim, group, { rc = launch<__half, D, GS>(p, pl, st); }); }
    else { KV4_DISPATCH_SHAPE(head_dim, group, { rc = launch<__nv_bfloat16, D, GS>(p, pl, st); }); }
    if (rc != B2L_OK) return rc;
  }
  return B2L_OK;
}
