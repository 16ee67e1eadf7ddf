// Slot maps of a ragged step, from the requests' lengths: where each request's new tokens begin in the flat batch, and for every new
// token its position in its sequence and its row of the pool -- the table's entry, or the next row of a list, which is then
// entered into the table.  One launch, nothing read by the host.
//
// start(b) = sum of new(b') over b' < b.  Token t belongs to the last b with start(b) <= t and new(b) > 0.  Every block adds up the
// lengths by itself, 1024 at a time, instead of a scan with a second launch: latency is the bound (a step's lengths are a few KB in L2).
#include "common.cuh"
#include <cstdint>

namespace {

constexpr int kThreads = 256, kPer = 4, kChunk = kThreads * kPer;   // lengths added up at a time; tokens of a block

struct MapParams {
  const void *req, *ctx, *fresh, *pool;
  int req_w, ctx_w, fresh_w, pool_w;
  int32_t *table, *rows, *start, *length;
  int64_t* position;
  int64_t tab_rs, tab_cs, requests, width;
  int64_t batch, total;
};

// a length as it counts: 64-bit ones too fit into 32 bits, so that no sum of them leaves 64
__device__ __forceinline__ int64_t length_of(const void* lens, int64_t b, int width) {
  const int64_t n = load_index(lens, b, width);
  return n < 0 ? 0 : n > INT32_MAX ? INT32_MAX : n;
}
__device__ __forceinline__ int32_t int32_at_most(int64_t n) { return n > INT32_MAX ? INT32_MAX : (int32_t)n; }

__global__ void __launch_bounds__(kThreads) slot_maps_kernel(const MapParams p) {
  pdl_prologue();
  __shared__ int64_t ends[kChunk];                 // of the requests in hand, in the flat batch
  __shared__ int64_t warp_sum[kThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool heads = blockIdx.x == 0;              // this block also writes what belongs to the requests
  const int64_t lo = (int64_t)blockIdx.x * kChunk, hi = lo + kChunk < p.total ? lo + kChunk : p.total;
  int64_t base = 0;
  for (int64_t b0 = 0; b0 < p.batch && (heads || base < hi); b0 += kChunk) {
    const int64_t b = b0 + threadIdx.x * kPer;
    int64_t n[kPer], own = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      n[i] = b + i < p.batch ? length_of(p.fresh, b + i, p.fresh_w) : 0;
      own += n[i];
    }
    int64_t upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    __syncthreads();                               // the chunk before is done with
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    int64_t at = base + upto - own;
    for (int w = 0; w < warp; ++w) at += warp_sum[w];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (heads && b + i < p.batch) {
        p.start[b + i] = int32_at_most(at);
        p.length[b + i] = int32_at_most(length_of(p.ctx, b + i, p.ctx_w) + n[i]);
      }
      at += n[i];
      ends[threadIdx.x * kPer + i] = at;
    }
    __syncthreads();
    const int64_t chunk_end = ends[kChunk - 1];
#pragma unroll 1
    for (int64_t t = lo + threadIdx.x; t < hi; t += kThreads) {
      if (t < base || t >= chunk_end) continue;
      int first = 0, count = kChunk;               // the first request that ends behind t
      while (count > 0) {
        const int half = count / 2;
        if (ends[first + half] <= t) { first += half + 1; count -= half + 1; }
        else count = half;
      }
      const int64_t begin = first > 0 ? ends[first - 1] : base;
      const int64_t r = load_index(p.req, b0 + first, p.req_w), pos = length_of(p.ctx, b0 + first, p.ctx_w) + t - begin;
      int32_t row = -1;
      if (r >= 0 && r < p.requests && pos < p.width) {
        int32_t* entry = p.table + r * p.tab_rs + pos * p.tab_cs;
        if (p.pool != nullptr) *entry = row = (int32_t)load_index(p.pool, t, p.pool_w);
        else row = *entry;
      }
      p.rows[t] = row;
      p.position[t] = pos;
    }
    base = chunk_end;
  }
  // padding behind the last request
  for (int64_t t = (lo > base ? lo : base) + threadIdx.x; t < hi; t += kThreads) {
    p.rows[t] = -1;
    p.position[t] = 0;
  }
}

}  // namespace

extern "C" int b2l_slot_maps(void* rows, void* position, void* start, void* length, const void* req_idx, int req_width,
                             const void* ctx_len, int ctx_width, const void* new_len, int new_width, const void* pool_rows,
                             int pool_width, void* table, int64_t table_req_stride, int64_t table_seq_stride, int64_t requests,
                             int64_t width, int64_t batch, int64_t total_tokens, void* stream) {
  B2L_REQUIRE(table && (total_tokens <= 0 || (rows && position)) && (batch <= 0 || (start && length && req_idx && ctx_len && new_len)),
              "slot_maps: null pointer");
  for (int w : {req_width, ctx_width, new_width, pool_rows ? pool_width : 4})
    B2L_REQUIRE(w == 4 || w == 8, "slot_maps: index widths must be 4 or 8");
  B2L_REQUIRE(batch >= 0 && total_tokens >= 0 && requests >= 0 && width >= 0 && total_tokens < (1ll << 31), "slot_maps: bad shape");
  if (batch == 0 && total_tokens == 0) return B2L_OK;
  MapParams p;
  p.req = req_idx; p.ctx = ctx_len; p.fresh = new_len; p.pool = pool_rows;
  p.req_w = req_width; p.ctx_w = ctx_width; p.fresh_w = new_width; p.pool_w = pool_width;
  p.table = (int32_t*)table; p.rows = (int32_t*)rows; p.start = (int32_t*)start; p.length = (int32_t*)length;
  p.position = (int64_t*)position;
  p.tab_rs = table_req_stride; p.tab_cs = table_seq_stride; p.requests = requests; p.width = width;
  p.batch = batch; p.total = total_tokens;
  const int64_t blocks = cdiv64(total_tokens, kChunk);
  b2l_launch(slot_maps_kernel, dim3((unsigned)(blocks > 0 ? blocks : 1)), dim3(kThreads), (size_t)0, (cudaStream_t)stream, p);
  B2L_LAUNCH_CHECK();
  return B2L_OK;
}
