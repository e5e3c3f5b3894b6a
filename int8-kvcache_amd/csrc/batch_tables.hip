// Block tables, slot mapping, positions and lengths of a ragged batch, from request lengths.
//
// Everything follows from two exclusive prefix sums over the requests: of their new tokens and of
// the blocks they take from the free list.  A token finds its request by binary search among the
// token starts; the token at a block's first position writes that block's table entry, and reads
// no entry that another token writes (a new block's id comes from the free list itself), so
// nothing has to wait for anything.
//
// Bound: latency.  A decode step of 32 requests moves 1.3 KB, and even a prefill of a million
// tokens writes 20 bytes per token.  Up to kOneLaunch requests every workgroup scans all lengths
// itself (in LDS) instead of a scan kernel running first: one launch.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "serving_ops.h"

namespace int8kv_serving {
namespace {

constexpr int kThreads = 256;
constexpr int kOneLaunch = 2048;  // requests whose prefix sums a workgroup keeps in LDS (40 KB)
constexpr int kTokensPerThread = 4;
constexpr int kScanThreads = 1024;
constexpr int64_t kLongest = 0x7fffffff;

struct TableArgs {
  const void* computed;
  const void* fresh;
  int64_t requests;
  int32_t* tables;
  int64_t width;
  int64_t table_stride;
  uint32_t block_size;
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
__device__ __forceinline__ int64_t length_at(const void* p, int64_t i) {
  const int64_t v = L64 ? reinterpret_cast<const int64_t*>(p)[i]
                        : (int64_t) reinterpret_cast<const int32_t*>(p)[i];
  return v < 0 ? 0 : (v > kLongest ? kLongest : v);
}

// Exclusive prefix sum of one value per thread over a workgroup of THREADS; returns the total too.
template <int THREADS>
__device__ __forceinline__ int64_t workgroup_scan(int64_t v, int64_t& total, int64_t* s_wave) {
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  int64_t inc = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t up = __shfl_up(inc, d, 64);
    if (lane >= d) inc += up;
  }
  __syncthreads();  // s_wave may still be read from the scan before
  if (lane == 63) s_wave[wave] = inc;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < wave) before += s_wave[w];
    total += s_wave[w];
  }
  return before + inc - v;
}

__device__ __forceinline__ int64_t blocks_for(int64_t len, uint32_t bs, int64_t width) {
  const uint32_t n = (uint32_t)len;  // both parts of a length are below 2^31
  const int64_t b = n / bs + (n % bs != 0 ? 1 : 0);
  return b < width ? b : width;
}

// Blocks that a request with c tokens takes for n more.
__device__ __forceinline__ int64_t blocks_taken(int64_t c, int64_t n, uint32_t bs, int64_t width) {
  return blocks_for(c + n, bs, width) - blocks_for(c, bs, width);
}

// One workgroup: the prefix sums of all requests, each thread a contiguous span of them.
// start(r, tokens before r) and taken(r, blocks before r) receive them; start(requests, ...) too.
template <int THREADS, bool L64, typename Start, typename Taken>
__device__ __forceinline__ void scan_requests(const TableArgs& a, int64_t* s_wave, Start start,
                                              Taken taken, int64_t& all_taken) {
  const int64_t per = (a.requests + THREADS - 1) / THREADS;
  const int64_t r0 = threadIdx.x * per;
  const int64_t r1 = r0 + per < a.requests ? r0 + per : a.requests;
  int64_t sum = 0;
  for (int64_t r = r0; r < r1; ++r) sum += length_at<L64>(a.fresh, r);
  int64_t total;
  int64_t at = workgroup_scan<THREADS>(sum, total, s_wave);
  int64_t blocks = 0;
  for (int64_t r = r0; r < r1; ++r) {
    const int64_t n = length_at<L64>(a.fresh, r);
    const int64_t b = at < a.tokens ? at : a.tokens;
    const int64_t e = at + n < a.tokens ? at + n : a.tokens;
    start(r, b, e);
    blocks += blocks_taken(length_at<L64>(a.computed, r), e - b, a.block_size, a.width);
    at += n;
  }
  int64_t before = workgroup_scan<THREADS>(blocks, all_taken, s_wave);
  at = 0;
  for (int64_t r = r0; r < r1; ++r) {
    const int64_t t = taken(r, before);
    before += t;
  }
}

// The outputs of token t of request r (its first token at `first`, `c` tokens computed before,
// `before` blocks taken by the requests before it).
__device__ __forceinline__ void write_token(const TableArgs& a, int64_t t, int64_t r, int64_t first,
                                            int64_t c, int64_t before, int64_t free_start) {
  const uint32_t p = (uint32_t)(c + (t - first));  // < 2^32: both are below 2^31
  const uint32_t block = p / a.block_size;
  const uint32_t within = p - block * a.block_size;
  int64_t slot = -1;
  if (block < a.width) {
    const int64_t have = blocks_for(c, a.block_size, a.width);
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
__device__ __forceinline__ int64_t find_request(P starts, int64_t requests, int64_t t) {
  int64_t lo = 0, hi = requests;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if ((int64_t)starts[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

// The sequence length of a request with c tokens computed and n new ones.
__device__ __forceinline__ int32_t sequence_length(int64_t c, int64_t n) {
  return (int32_t)(c + n < kLongest ? c + n : kLongest);
}

template <bool L64>
__global__ __launch_bounds__(kThreads) void tables_kernel(TableArgs a) {
  __shared__ int32_t s_start[kOneLaunch + 1];
  __shared__ int32_t s_computed[kOneLaunch];
  __shared__ int64_t s_taken[kOneLaunch];
  __shared__ int64_t s_wave[kThreads / 64];
  const int64_t free_start = a.free_start ? *a.free_start : 0;
  int64_t all_taken;
  if (a.requests == 0 && threadIdx.x == 0) s_start[0] = 0;
  scan_requests<kThreads, L64>(
      a, s_wave,
      [&](int64_t r, int64_t b, int64_t e) {
        s_start[r] = (int32_t)b;
        s_start[r + 1] = (int32_t)e;  // the next request's own start: the same value
        s_computed[r] = (int32_t)length_at<L64>(a.computed, r);
      },
      [&](int64_t r, int64_t before) {
        s_taken[r] = before;
        return blocks_taken(s_computed[r], s_start[r + 1] - s_start[r], a.block_size, a.width);
      },
      all_taken);
  __syncthreads();
  const int64_t held = s_start[a.requests];
  const int64_t t0 = (int64_t)blockIdx.x * (kThreads * kTokensPerThread) + threadIdx.x;
#pragma unroll
  for (int j = 0; j < kTokensPerThread; ++j) {
    const int64_t t = t0 + j * kThreads;
    if (t >= a.tokens) break;
    if (t >= held) {
      write_padding(a, t);
      continue;
    }
    const int64_t r = find_request(s_start, a.requests, t);
    write_token(a, t, r, s_start[r], s_computed[r], s_taken[r], free_start);
  }
  if (blockIdx.x == 0) {
    for (int64_t r = threadIdx.x; r <= a.requests; r += kThreads) {
      a.query_starts[r] = s_start[r];
      if (r < a.requests)
        a.seq_lens[r] = sequence_length(s_computed[r], s_start[r + 1] - s_start[r]);
    }
    // (In place of free_start only where this is the only workgroup: every thread read it before
    // the scan's barriers.)
    if (threadIdx.x == 0) *a.free_end = free_start + all_taken;
  }
}

// More requests than a workgroup scans on the side: the scan once, then the tokens.
template <bool L64>
__global__ __launch_bounds__(kScanThreads) void scan_kernel(TableArgs a) {
  __shared__ int64_t s_wave[kScanThreads / 64];
  const int64_t free_start = a.free_start ? *a.free_start : 0;
  int64_t all_taken;
  scan_requests<kScanThreads, L64>(
      a, s_wave,
      [&](int64_t r, int64_t b, int64_t e) {
        a.query_starts[r] = (int32_t)b;
        if (r == a.requests - 1) a.query_starts[a.requests] = (int32_t)e;
        a.seq_lens[r] = sequence_length(length_at<L64>(a.computed, r), e - b);
      },
      [&](int64_t r, int64_t before) {
        a.ws_taken[r] = before;
        // (The starts written above, by this thread: they hold the tokens kept.)
        const int64_t c = length_at<L64>(a.computed, r);
        const int64_t b = a.query_starts[r];
        const int64_t n = length_at<L64>(a.fresh, r);
        return blocks_taken(c, b + n < a.tokens ? n : a.tokens - b, a.block_size, a.width);
      },
      all_taken);
  if (a.requests == 0 && threadIdx.x == 0) a.query_starts[0] = 0;
  if (threadIdx.x == 0) {
    *a.ws_free = free_start;
    *a.free_end = free_start + all_taken;
  }
}

template <bool L64>
__global__ __launch_bounds__(kThreads) void tokens_kernel(TableArgs a) {
  const int64_t held = a.query_starts[a.requests];
  const int64_t free_start = *a.ws_free;
  const int64_t t0 = (int64_t)blockIdx.x * (kThreads * kTokensPerThread) + threadIdx.x;
#pragma unroll
  for (int j = 0; j < kTokensPerThread; ++j) {
    const int64_t t = t0 + j * kThreads;
    if (t >= a.tokens) break;
    if (t >= held) {
      write_padding(a, t);
      continue;
    }
    const int64_t r = find_request(a.query_starts, a.requests, t);
    write_token(a, t, r, a.query_starts[r], length_at<L64>(a.computed, r), a.ws_taken[r], free_start);
  }
}

template <bool L64>
void launch(const TableArgs& a, bool one_launch, hipStream_t s) {
  const int64_t per_wg = kThreads * kTokensPerThread;
  const uint32_t grid = (uint32_t)((a.tokens + per_wg - 1) / per_wg);
  if (one_launch) {
    hipLaunchKernelGGL(tables_kernel<L64>, dim3(grid > 0 ? grid : 1), dim3(kThreads), 0, s, a);
    return;
  }
  hipLaunchKernelGGL(scan_kernel<L64>, dim3(1), dim3(kScanThreads), 0, s, a);
  if (grid > 0) hipLaunchKernelGGL(tokens_kernel<L64>, dim3(grid), dim3(kThreads), 0, s, a);
}

}  // namespace
}  // namespace int8kv_serving

using namespace int8kv_serving;

extern "C" size_t int8kv_batch_tables_workspace_bytes(int64_t requests) {
  if (requests < 0 || requests > 0x7fffffff) return 0;
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
  // free_end in place of free_start: one workgroup alone may read and write it in one launch.
  const bool in_place = free_start == free_end && num_tokens > kThreads * kTokensPerThread;
  const bool one_launch = requests <= kOneLaunch && !in_place;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (lens_dtype == INT8KV_I64)
    launch<true>(a, one_launch, s);
  else
    launch<false>(a, one_launch, s);
  return (int)hipGetLastError();
}
