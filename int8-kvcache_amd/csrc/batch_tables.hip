// Block tables, slot mapping, positions and lengths of a ragged batch, from request lengths.
//
// Everything follows from two exclusive prefix sums over the requests: of their new tokens and of
// the blocks they take from the free list.  A token finds its request by binary search among the
// token starts; the token at a block's first position writes that block's table entry, and reads
// no entry that another token writes (a new block's id comes from the free list itself), so
// nothing has to wait for anything.
//
// Bound: latency (a decode step of 32 requests moves 1.3 KB), or the 20 bytes written per token of
// a large prefill.  Up to kMostScanned requests every workgroup scans all lengths itself, one or
// two requests per thread, instead of a scan kernel running first: one launch.  Measured: 4.3 us
// for 32 requests of one token, 4.9 for 1021, 8.3 for 61 requests of 16384 (20 MB, 2.4 TB/s: the
// launch and the scan are about half of that).

#include <hip/hip_runtime.h>

#include <cstdint>

#include "serving_ops.h"
#include "wave_scan.h"

namespace int8kv_serving {
namespace {

constexpr int kFewThreads = 256;    // workgroups for at most as many requests ...
constexpr int kManyThreads = 1024;  // ... and for up to twice as many as these
constexpr int kMostScanned = 2 * kManyThreads;
constexpr int kTokensPerThread = 4;
constexpr int64_t kLongest = 0x7fffffff;

struct TableArgs {
  const void* computed;
  const void* fresh;
  int64_t requests;
  int32_t* tables;
  int64_t width;
  int64_t table_stride;
  uint32_t block_size;
  int32_t block_shift;  // log2 of it, or -1
  const int32_t* free_blocks;
  int64_t num_free;
  const int64_t* free_start;
  int64_t tokens;
  int32_t* query_starts;
  int32_t* seq_lens;
  int64_t* positions;
  int64_t* slots;
  int32_t* token_requests;
  int64_t* free_end;
  int64_t* ws_taken;  // [requests] blocks taken before each request (two launches)
  int64_t* ws_free;   // [1] free_start as it was before the call (two launches)
};

template <bool L64>
__device__ __forceinline__ uint32_t length_at(const void* p, int64_t i) {
  const int64_t v = L64 ? reinterpret_cast<const int64_t*>(p)[i]
                        : (int64_t) reinterpret_cast<const int32_t*>(p)[i];
  return (uint32_t)(v < 0 ? 0 : (v > kLongest ? kLongest : v));
}

__device__ __forceinline__ uint32_t block_of(const TableArgs& a, uint32_t position) {
  return a.block_shift >= 0 ? position >> a.block_shift : position / a.block_size;
}

// Blocks of the first `length` (below 2^32) tokens, as far as the table holds them.
__device__ __forceinline__ uint32_t blocks_for(const TableArgs& a, uint32_t length) {
  const uint32_t whole = block_of(a, length);
  const uint32_t blocks = whole + (length - whole * a.block_size != 0 ? 1 : 0);
  return blocks < (uint32_t)a.width ? blocks : (uint32_t)a.width;
}

// Blocks that a request with c tokens takes for n more (c + n below 2^32).
__device__ __forceinline__ uint32_t blocks_taken(const TableArgs& a, uint32_t c, uint32_t n) {
  return blocks_for(a, c + n) - blocks_for(a, c);
}

// The sequence length of a request with c tokens computed and n new ones.
__device__ __forceinline__ int32_t sequence_length(uint32_t c, uint32_t n) {
  const uint32_t length = c + n;
  return (int32_t)(length < (uint32_t)kLongest ? length : (uint32_t)kLongest);
}

// The outputs of token t of request r (its first token at `first`, `c` tokens computed before,
// `before` blocks taken by the requests before it).
__device__ __forceinline__ void write_token(const TableArgs& a, int64_t t, int64_t r, int64_t first,
                                            uint32_t c, int64_t before, int64_t free_start) {
  const uint32_t p = c + (uint32_t)(t - first);  // < 2^32: both are below 2^31
  const uint32_t block = block_of(a, p);
  const uint32_t within = p - block * a.block_size;
  int64_t slot = -1;
  if (block < (uint32_t)a.width) {
    const uint32_t have = blocks_for(a, c);
    int32_t id;
    if (block < have) {
      id = a.tables[r * a.table_stride + block];
    } else {
      const int64_t i = free_start + before + (block - have);
      id = i >= 0 && i < a.num_free ? a.free_blocks[i] : -1;
      if (within == 0) a.tables[r * a.table_stride + block] = id;
    }
    if (id >= 0) slot = (int64_t)id * a.block_size + within;
  }
  a.positions[t] = p;
  a.slots[t] = slot;
  a.token_requests[t] = (int32_t)r;
}

__device__ __forceinline__ void write_padding(const TableArgs& a, int64_t t) {
  a.positions[t] = 0;
  a.slots[t] = -1;
  a.token_requests[t] = -1;
}

// Last request whose first token is at or before t (starts[requests] is the number of tokens
// held, and t < that).
template <typename P>
__device__ __forceinline__ int32_t find_request(P starts, int32_t requests, int32_t t) {
  int32_t lo = 0, hi = requests;
  while (hi - lo > 1) {
    const int32_t mid = (int32_t)(((uint32_t)lo + (uint32_t)hi) >> 1);
    if (starts[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

// One launch: every workgroup scans all requests (REQUESTS consecutive ones per thread), then
// writes its tokens; the first one writes the requests' outputs too.
template <int THREADS, int REQUESTS, bool L64>
__global__ __launch_bounds__(THREADS) void tables_kernel(TableArgs a) {
  constexpr int kMost = THREADS * REQUESTS;
  constexpr int kWaves = THREADS / 64;
  __shared__ int32_t s_start[kMost + 1];
  __shared__ uint32_t s_computed[kMost];
  __shared__ int64_t s_taken[kMost];
  __shared__ uint64_t s_wave[kWaves];
  const int64_t free_start = a.free_start ? *a.free_start : 0;
  const int32_t requests = (int32_t)a.requests;
  const int32_t r0 = REQUESTS * (int32_t)threadIdx.x;
  uint32_t c[REQUESTS], n[REQUESTS];
  uint64_t sum = 0, total;
#pragma unroll
  for (int j = 0; j < REQUESTS; ++j) {
    c[j] = r0 + j < requests ? length_at<L64>(a.computed, r0 + j) : 0;
    n[j] = r0 + j < requests ? length_at<L64>(a.fresh, r0 + j) : 0;
    sum += n[j];
  }
  uint64_t at = workgroup_scan<kWaves, uint64_t>(sum, s_wave, total);
  uint64_t taken = 0;
#pragma unroll
  for (int j = 0; j < REQUESTS; ++j) {
    const uint64_t end = at + n[j];
    const uint32_t b = at < (uint64_t)a.tokens ? (uint32_t)at : (uint32_t)a.tokens;
    const uint32_t e = end < (uint64_t)a.tokens ? (uint32_t)end : (uint32_t)a.tokens;
    at = end;
    n[j] = e - b;  // the tokens that fit
    taken += blocks_taken(a, c[j], n[j]);
    if (r0 + j <= requests) s_start[r0 + j] = (int32_t)b;
    if (r0 + j < requests) s_computed[r0 + j] = c[j];
  }
  if (requests == kMost && threadIdx.x == THREADS - 1)
    s_start[kMost] = (int32_t)(total < (uint64_t)a.tokens ? total : (uint64_t)a.tokens);
  uint64_t all_taken;
  uint64_t before = workgroup_scan<kWaves, uint64_t>(taken, s_wave, all_taken);
#pragma unroll
  for (int j = 0; j < REQUESTS; ++j) {
    if (r0 + j < requests) s_taken[r0 + j] = (int64_t)before;
    before += blocks_taken(a, c[j], n[j]);
  }
  __syncthreads();
  const int32_t held = s_start[requests];
  const int64_t t0 = (int64_t)blockIdx.x * (THREADS * kTokensPerThread) + threadIdx.x;
#pragma unroll
  for (int j = 0; j < kTokensPerThread; ++j) {
    const int64_t t = t0 + j * THREADS;
    if (t >= a.tokens) break;
    if (t >= held) {
      write_padding(a, t);
      continue;
    }
    const int32_t r = find_request(s_start, requests, (int32_t)t);
    write_token(a, t, r, s_start[r], s_computed[r], s_taken[r], free_start);
  }
  if (blockIdx.x == 0) {
#pragma unroll
    for (int j = 0; j < REQUESTS; ++j) {
      const int32_t r = r0 + j;
      if (r < requests) {
        a.query_starts[r] = s_start[r];
        a.seq_lens[r] = sequence_length(c[j], n[j]);
      }
    }
    // (In place of free_start only where this is the only workgroup: every thread read it before
    // the scan's barriers.)
    if (threadIdx.x == 0) {
      a.query_starts[requests] = held;
      *a.free_end = free_start + (int64_t)all_taken;
    }
  }
}

// More requests than a workgroup scans on the side: the scan once, each thread a contiguous span
// of requests, then the tokens.
template <bool L64>
__global__ __launch_bounds__(kManyThreads) void scan_kernel(TableArgs a) {
  constexpr int kWaves = kManyThreads / 64;
  __shared__ uint64_t s_wave[kWaves];
  const int64_t free_start = a.free_start ? *a.free_start : 0;
  const int64_t per = (a.requests + kManyThreads - 1) / kManyThreads;
  const int64_t r0 = threadIdx.x * per;
  const int64_t r1 = r0 + per < a.requests ? r0 + per : a.requests;
  uint64_t sum = 0, total;
  for (int64_t r = r0; r < r1; ++r) sum += length_at<L64>(a.fresh, r);
  uint64_t at = workgroup_scan<kWaves, uint64_t>(sum, s_wave, total);
  const uint64_t first = at;
  const auto fitting = [&](int64_t r, uint32_t& start) {
    const uint64_t end = at + length_at<L64>(a.fresh, r);
    start = at < (uint64_t)a.tokens ? (uint32_t)at : (uint32_t)a.tokens;
    at = end;
    return (end < (uint64_t)a.tokens ? (uint32_t)end : (uint32_t)a.tokens) - start;
  };
  uint64_t taken = 0;
  for (int64_t r = r0; r < r1; ++r) {
    uint32_t start;
    const uint32_t c = length_at<L64>(a.computed, r);
    const uint32_t n = fitting(r, start);
    a.query_starts[r] = (int32_t)start;
    a.seq_lens[r] = sequence_length(c, n);
    taken += blocks_taken(a, c, n);
  }
  uint64_t all_taken;
  uint64_t before = workgroup_scan<kWaves, uint64_t>(taken, s_wave, all_taken);
  at = first;
  for (int64_t r = r0; r < r1; ++r) {
    uint32_t start;
    a.ws_taken[r] = (int64_t)before;
    const uint32_t n = fitting(r, start);
    before += blocks_taken(a, length_at<L64>(a.computed, r), n);
  }
  if (threadIdx.x == 0) {
    a.query_starts[a.requests] = (int32_t)(total < (uint64_t)a.tokens ? total : (uint64_t)a.tokens);
    *a.ws_free = free_start;
    *a.free_end = free_start + (int64_t)all_taken;
  }
}

template <bool L64>
__global__ __launch_bounds__(kFewThreads) void tokens_kernel(TableArgs a) {
  const int32_t held = a.query_starts[a.requests];
  const int64_t free_start = *a.ws_free;
  const int64_t t0 = (int64_t)blockIdx.x * (kFewThreads * kTokensPerThread) + threadIdx.x;
#pragma unroll
  for (int j = 0; j < kTokensPerThread; ++j) {
    const int64_t t = t0 + j * kFewThreads;
    if (t >= a.tokens) break;
    if (t >= held) {
      write_padding(a, t);
      continue;
    }
    const int32_t r = find_request(a.query_starts, (int32_t)a.requests, (int32_t)t);
    write_token(a, t, r, a.query_starts[r], length_at<L64>(a.computed, r), a.ws_taken[r], free_start);
  }
}

uint32_t grid_for(int64_t tokens, int threads) {
  const int64_t per_wg = threads * kTokensPerThread;
  return (uint32_t)((tokens + per_wg - 1) / per_wg);
}

template <int THREADS, int REQUESTS, bool L64>
void launch_one(const TableArgs& a, hipStream_t s) {
  const uint32_t grid = grid_for(a.tokens, THREADS);
  hipLaunchKernelGGL((tables_kernel<THREADS, REQUESTS, L64>), dim3(grid > 0 ? grid : 1),
                     dim3(THREADS), 0, s, a);
}

template <bool L64>
void launch(const TableArgs& a, bool in_place, hipStream_t s) {
  // free_end in place of free_start: one workgroup alone may read and write it in one launch.
  if (a.requests <= kFewThreads && !(in_place && grid_for(a.tokens, kFewThreads) > 1))
    return launch_one<kFewThreads, 1, L64>(a, s);
  if (a.requests <= kManyThreads && !(in_place && grid_for(a.tokens, kManyThreads) > 1))
    return launch_one<kManyThreads, 1, L64>(a, s);
  if (a.requests <= kMostScanned && !(in_place && grid_for(a.tokens, kManyThreads) > 1))
    return launch_one<kManyThreads, 2, L64>(a, s);
  hipLaunchKernelGGL(scan_kernel<L64>, dim3(1), dim3(kManyThreads), 0, s, a);
  const uint32_t grid = grid_for(a.tokens, kFewThreads);
  if (grid > 0) hipLaunchKernelGGL(tokens_kernel<L64>, dim3(grid), dim3(kFewThreads), 0, s, a);
}

}  // namespace
}  // namespace int8kv_serving

using namespace int8kv_serving;

extern "C" size_t int8kv_batch_tables_workspace_bytes(int64_t requests) {
  if (requests < 0 || requests > 0x7ffffffe) return 0;
  return 16 + 8 * (size_t)requests;
}

extern "C" int int8kv_batch_tables(const void* computed_lens, const void* new_lens, int lens_dtype,
                                   int64_t requests, int32_t* block_tables, int64_t table_width,
                                   int64_t table_row_stride, int32_t block_size,
                                   const int32_t* free_blocks, int64_t num_free,
                                   const int64_t* free_start, int64_t num_tokens,
                                   int32_t* query_starts, int32_t* seq_lens, int64_t* positions,
                                   int64_t* slot_mapping, int32_t* token_requests,
                                   int64_t* free_end, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  if (!query_starts || !free_end) return INT8KV_E_NULL;
  if (requests > 0 && (!computed_lens || !new_lens || !seq_lens)) return INT8KV_E_NULL;
  if (requests > 0 && table_width > 0 && !block_tables) return INT8KV_E_NULL;
  if (num_free > 0 && !free_blocks) return INT8KV_E_NULL;
  if (num_tokens > 0 && (!positions || !slot_mapping || !token_requests)) return INT8KV_E_NULL;
  if (lens_dtype != INT8KV_I32 && lens_dtype != INT8KV_I64) return INT8KV_E_DTYPE;
  if (requests < 0 || requests > 0x7ffffffe || table_width < 0 || table_width > 0x7fffffff ||
      block_size < 1 || block_size > 65536 || num_free < 0 || num_tokens < 0 ||
      num_tokens > 0x7fffffff)
    return INT8KV_E_SHAPE;
  if (requests > 1 && table_row_stride < table_width) return INT8KV_E_STRIDE;
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 ||
      workspace_bytes < int8kv_batch_tables_workspace_bytes(requests))
    return INT8KV_E_WORKSPACE;
  TableArgs a;
  a.computed = computed_lens;
  a.fresh = new_lens;
  a.requests = requests;
  a.tables = block_tables;
  a.width = table_width;
  a.table_stride = table_row_stride;
  a.block_size = (uint32_t)block_size;
  a.block_shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz((unsigned)block_size) : -1;
  a.free_blocks = free_blocks;
  a.num_free = num_free;
  a.free_start = free_start;
  a.tokens = num_tokens;
  a.query_starts = query_starts;
  a.seq_lens = seq_lens;
  a.positions = positions;
  a.slots = slot_mapping;
  a.token_requests = token_requests;
  a.free_end = free_end;
  a.ws_free = static_cast<int64_t*>(workspace);
  a.ws_taken = a.ws_free + 2;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (lens_dtype == INT8KV_I64)
    launch<true>(a, free_start == free_end, s);
  else
    launch<false>(a, free_start == free_end, s);
  return (int)hipGetLastError();
}
