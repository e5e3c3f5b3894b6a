// Low-rank adapters of many requests beside a shared projection:
//   out[t] = bf16(base[t] + scale[a] (x[t] A[a]^T) B[a]^T),  a = adapter of token t.
//
// A plan groups the tokens by adapter into tiles of one adapter each (16 tokens, or 64 in larger
// batches); the products then run tile by tile on matrix instructions, in two launches: x A^T into
// fp32 partial sums (split along k), then those times B^T, the scale and the base.
//
// Precision: the first product's sums stay fp32.  They enter the second one as two bf16 parts,
// the upper bits and the rest (together 17 bits, of a rank-wide vector), so that both products run
// on bf16 matrix instructions and the result differs from an fp32 one by less than its own
// rounding to bf16 does.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "serving_ops.h"

namespace int8kv_serving {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int64_t kMaxTokens = 1 << 24;
constexpr int kMaxAdapters = 4096;
constexpr int kMaxRank = 128;
constexpr int64_t kMaxWidth = 1 << 20;
constexpr int kPlanThreads = 1024;
constexpr int kTileRows = 16;

__device__ __forceinline__ float bf16_value(uint32_t h) { return __uint_as_float(h << 16); }
__device__ __forceinline__ uint32_t bf16_bits(float f) {
  return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f));
}

// ------------------------------------------------------------------------------------ plan
// int32 words: [0] tiles, [1] tokens with an adapter, [2..3] unused; the token of every position
// (grouped by adapter, those without one last); adapter, first position and rows of every tile
// (adapter -1: tokens without one).
struct Plan {
  int32_t* head;
  int32_t* order;
  int32_t* tile_adapter;
  int32_t* tile_start;
  int32_t* tile_rows;
};

int64_t max_tiles(int64_t tokens, int32_t adapters, int rows) {
  const int64_t groups = (int64_t)adapters + 1 < tokens ? (int64_t)adapters + 1 : tokens;
  return tokens / rows + groups;  // each group rounds up by less than one tile
}

Plan plan_at(const void* p, int64_t tokens, int32_t adapters) {
  int32_t* w = static_cast<int32_t*>(const_cast<void*>(p));
  const int64_t tiles = max_tiles(tokens, adapters, kTileRows);
  Plan q;
  q.head = w;
  q.order = w + 4;
  q.tile_adapter = q.order + tokens;
  q.tile_start = q.tile_adapter + tiles;
  q.tile_rows = q.tile_start + tiles;
  return q;
}

template <bool L64>
__device__ __forceinline__ int32_t adapter_of(const void* ids, int64_t t, int32_t adapters) {
  const int64_t a = L64 ? static_cast<const int64_t*>(ids)[t]
                        : (int64_t) static_cast<const int32_t*>(ids)[t];
  return a >= 0 && a < adapters ? (int32_t)a : adapters;  // `adapters`: none
}

// Exclusive prefix sum over the workgroup.
__device__ __forceinline__ int32_t plan_scan(int32_t v, int32_t* s_wave, int32_t& total) {
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  int32_t inc = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int32_t up = __shfl_up(inc, d, 64);
    if (lane >= d) inc += up;
  }
  __syncthreads();
  if (lane == 63) s_wave[wave] = inc;
  __syncthreads();
  int32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) before += s_wave[w];
    total += s_wave[w];
  }
  return before + inc - v;
}

// Lanes of the wave with this lane's group: adds their number to *counter (one lane's atomic) and
// returns this lane's place.  Neighbouring tokens mostly share their adapter.
__device__ __forceinline__ int32_t take_place(int32_t group, bool valid, int32_t* counters) {
  uint64_t todo = __ballot(valid);
  int32_t place = 0;
  const int lane = threadIdx.x & 63;
  while (todo) {
    const int leader = __ffsll((unsigned long long)todo) - 1;
    const int32_t g = __shfl(group, leader, 64);
    const uint64_t same = __ballot(valid && group == g);
    int32_t at = 0;
    if (lane == leader) at = atomicAdd(&counters[g], (int32_t)__popcll(same));
    at = __shfl(at, leader, 64);
    if (valid && group == g)
      place = at + (int32_t)__popcll(same & (((uint64_t)1 << lane) - 1));
    todo &= ~same;
  }
  return place;
}

// One workgroup: counts, offsets and places.  The order of tokens within a group may differ from
// call to call; no result depends on it (a token's row is computed alike at every place).
template <bool L64>
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(const void* ids, int32_t tokens,
                                                            int32_t adapters, int tile, Plan plan) {
  __shared__ int32_t s_count[kMaxAdapters + 1];
  __shared__ int32_t s_wave[kPlanThreads / 64];
  for (int32_t g = threadIdx.x; g <= adapters; g += kPlanThreads) s_count[g] = 0;
  __syncthreads();
  for (int32_t t0 = 0; t0 < tokens; t0 += kPlanThreads) {
    const int32_t t = t0 + (int32_t)threadIdx.x;
    const bool valid = t < tokens;
    take_place(valid ? adapter_of<L64>(ids, t, adapters) : 0, valid, s_count);
  }
  __syncthreads();
  // Offsets of the groups and of their tiles; each thread a contiguous span of groups.
  const int32_t per = (adapters + 1 + kPlanThreads - 1) / kPlanThreads;
  const int32_t g0 = (int32_t)threadIdx.x * per;
  const int32_t g1 = g0 + per < adapters + 1 ? g0 + per : adapters + 1;
  int32_t rows = 0, tiles = 0;
  for (int32_t g = g0; g < g1; ++g) {
    rows += s_count[g];
    tiles += (s_count[g] + tile - 1) / tile;
  }
  int32_t all_rows, all_tiles;
  int32_t row = plan_scan(rows, s_wave, all_rows);
  int32_t at = plan_scan(tiles, s_wave, all_tiles);
  for (int32_t g = g0; g < g1; ++g) {
    const int32_t n = s_count[g];
    for (int32_t i = 0; i < n; i += tile) {
      plan.tile_adapter[at] = g < adapters ? g : -1;
      plan.tile_start[at] = row + i;
      plan.tile_rows[at] = n - i < tile ? n - i : tile;
      ++at;
    }
    s_count[g] = row;  // now the group's next place
    if (g == adapters) plan.head[1] = row;
    row += n;
  }
  if (threadIdx.x == 0) plan.head[0] = all_tiles;
  __syncthreads();
  for (int32_t t0 = 0; t0 < tokens; t0 += kPlanThreads) {
    const int32_t t = t0 + (int32_t)threadIdx.x;
    const bool valid = t < tokens;
    const int32_t p = take_place(valid ? adapter_of<L64>(ids, t, adapters) : 0, valid, s_count);
    if (valid) plan.order[p] = t;
  }
}

// -------------------------------------------------------------------------------- products
struct LoraArgs {
  const uint16_t* base;
  int64_t base_stride;
  const uint16_t* x;
  int64_t x_stride;
  const uint16_t* a;
  int64_t a_adapter, a_row;
  const uint16_t* b;
  int64_t b_adapter, b_row;
  const float* scales;
  uint16_t* out;
  int64_t out_stride;
  float* part;  // [splits][tokens (in plan order)][rank]
  Plan plan;
  int32_t tokens, k, n, rank;
  int32_t splits;   // parts of k
  int32_t chunk;    // k of a part (a multiple of 32)
  int32_t chunks;   // column chunks of the second product
};

__device__ __forceinline__ bf16x8 load8(const uint16_t* p) {
  return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(p));
}
__device__ __forceinline__ bf16x8 zero8() {
  return __builtin_bit_cast(bf16x8, u32x4{0u, 0u, 0u, 0u});
}

// x A^T of one tile and one part of k.  Four waves take the part's 32-wide steps in turn; RT:
// 16-row tiles of A.  Operands straight from memory: lane (i, g) holds 8 consecutive k of row i.
constexpr int kShrinkWaves = 4;
template <int RT>
__global__ __launch_bounds__(kShrinkWaves * 64) void shrink_kernel(LoraArgs a) {
  __shared__ f32x4 s_acc[kShrinkWaves][RT][64];
  const int32_t tile = blockIdx.x / a.splits;
  const int32_t split = blockIdx.x - tile * a.splits;
  if (tile >= a.plan.head[0]) return;
  const int32_t adapter = a.plan.tile_adapter[tile];
  if (adapter < 0) return;
  const int32_t start = a.plan.tile_start[tile];
  const int32_t rows = a.plan.tile_rows[tile];
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int i = lane & 15;
  const int g = lane >> 4;
  const int32_t token = a.plan.order[start + (i < rows ? i : rows - 1)];
  const uint16_t* xp = a.x + token * a.x_stride + 8 * g;
  const uint16_t* ap[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int32_t r = 16 * rt + i;
    ap[rt] = a.a + adapter * a.a_adapter + (int64_t)(r < a.rank ? r : a.rank - 1) * a.a_row + 8 * g;
  }
  f32x4 acc[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) acc[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int32_t k0 = split * a.chunk;
  const int32_t k1 = k0 + a.chunk < a.k ? k0 + a.chunk : a.k;
  for (int32_t k = k0 + 32 * wave; k < k1; k += 32 * kShrinkWaves) {
    const bool in = k + 8 * g < k1;  // k is a multiple of 8
    const bf16x8 xv = in ? load8(xp + k) : zero8();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const bf16x8 av = in ? load8(ap[rt] + k) : zero8();
      acc[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, xv, acc[rt], 0, 0, 0);
    }
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) s_acc[wave][rt][lane] = acc[rt];
  __syncthreads();
  // Lane (i, g) of tile rt: ranks 16 rt + 4 g .. + 3 of token i.
  for (int rt = wave; rt < RT; rt += kShrinkWaves) {
    f32x4 y = s_acc[0][rt][lane];
#pragma unroll
    for (int w = 1; w < kShrinkWaves; ++w) y += s_acc[w][rt][lane];
    const int32_t r = 16 * rt + 4 * g;
    if (i < rows && r < a.rank)
      *reinterpret_cast<f32x4*>(a.part + ((int64_t)split * a.tokens + start + i) * a.rank + r) = y;
  }
}

// The second product of one tile and one chunk of columns.  The rank-wide vectors are staged in
// LDS as two bf16 parts, upper (truncated: no overflow) and rest; along the product's inner axis
// first all upper parts, then all rests, against the same row of B.
constexpr int kExpandWaves = 4;
constexpr int kWaveColumns = 64;
constexpr int kExpandColumns = kExpandWaves * kWaveColumns;
template <int RT>
__global__ __launch_bounds__(kExpandWaves * 64) void expand_kernel(LoraArgs a) {
  constexpr int kPad = 8;
  __shared__ __align__(16) uint16_t s_h[kTileRows][2 * 16 * RT + kPad];
  const int32_t tile = blockIdx.x / a.chunks;
  const int32_t chunk = blockIdx.x - tile * a.chunks;
  if (tile >= a.plan.head[0]) return;
  const int32_t adapter = a.plan.tile_adapter[tile];
  const int32_t start = a.plan.tile_start[tile];
  const int32_t rows = a.plan.tile_rows[tile];
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int i = lane & 15;
  const int g = lane >> 4;
  if (adapter < 0) {
    if (a.out == a.base && a.out_stride == a.base_stride) return;
    const int32_t c0 = chunk * kExpandColumns;
    const int32_t c1 = c0 + kExpandColumns < a.n ? c0 + kExpandColumns : a.n;
    const int32_t pieces = (c1 - c0) / 8;
    for (int32_t p = threadIdx.x; p < rows * pieces; p += kExpandWaves * 64) {
      const int32_t r = p / pieces;
      const int64_t t = a.plan.order[start + r];
      const int32_t c = c0 + 8 * (p - r * pieces);
      *reinterpret_cast<u32x4*>(a.out + t * a.out_stride + c) =
          *reinterpret_cast<const u32x4*>(a.base + t * a.base_stride + c);
    }
    return;
  }
  const int32_t quads = a.rank / 4;
  for (int32_t p = threadIdx.x; p < rows * quads; p += kExpandWaves * 64) {
    const int32_t r = p / quads;
    const int32_t c = 4 * (p - r * quads);
    f32x4 h = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int32_t s = 0; s < a.splits; ++s)
      h += *reinterpret_cast<const f32x4*>(a.part + ((int64_t)s * a.tokens + start + r) * a.rank + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t hi = __float_as_uint(h[j]) >> 16;
      const float rest = h[j] - bf16_value(hi);
      s_h[r][c + j] = (uint16_t)hi;
      s_h[r][a.rank + c + j] = fabsf(h[j]) < INFINITY ? (uint16_t)bf16_bits(rest) : 0;
    }
  }
  __syncthreads();
  // Columns of this wave: lane g's 16 consecutive ones, 4 per matrix tile j (row 4 g + r of tile
  // j's operand is column 16 g + 4 j + r), so a token's 64 columns are one 128-byte line.
  const int32_t col0 = chunk * kExpandColumns + wave * kWaveColumns;
  if (col0 >= a.n) return;
  const uint16_t* bp[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int32_t c = col0 + 16 * (i >> 2) + 4 * j + (i & 3);
    bp[j] = a.b + adapter * a.b_adapter + (int64_t)(c < a.n ? c : a.n - 1) * a.b_row;
  }
  f32x4 acc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int32_t granules = a.rank / 8;  // 8-wide pieces of one part
  const int row = i < rows ? i : rows - 1;
  for (int32_t s = 0; s < 2 * granules; s += 4) {
    const int32_t p = s + g;
    const bool in = p < 2 * granules;
    const int32_t at = p < granules ? p : p - granules;
    const bf16x8 hv = in ? load8(&s_h[row][8 * p]) : zero8();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bf16x8 bv = in ? load8(bp[j] + 8 * at) : zero8();
      acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bv, hv, acc[j], 0, 0, 0);
    }
  }
  if (i >= rows) return;
  const int64_t t = a.plan.order[start + i];
  const float scale = a.scales ? a.scales[adapter] : 1.0f;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int32_t c = col0 + 16 * g + 8 * half;
    if (c >= a.n) break;
    const u32x4 v = *reinterpret_cast<const u32x4*>(a.base + t * a.base_stride + c);
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4 d = acc[2 * half + (j >> 1)];
      const float lo = d[2 * (j & 1)] * scale + bf16_value(v[j] & 0xffffu);
      const float hi = d[2 * (j & 1) + 1] * scale + bf16_value(v[j] >> 16);
      o[j] = bf16_bits(lo) | (bf16_bits(hi) << 16);
    }
    *reinterpret_cast<u32x4*>(a.out + t * a.out_stride + c) = o;
  }
}

bool rows16(const void* p, int64_t stride) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride % 8 == 0;
}

int splits_for(int64_t tiles, int64_t k) {
  const int64_t steps = (k + 127) / 128;
  int64_t s = (512 + tiles - 1) / (tiles > 0 ? tiles : 1);
  s = s < 1 ? 1 : (s > 8 ? 8 : s);
  return (int)(s < steps ? s : steps);
}

bool lora_sizes_ok(int64_t tokens, int32_t adapters, int64_t k, int32_t rank) {
  return tokens >= 0 && tokens <= kMaxTokens && adapters >= 1 && adapters <= kMaxAdapters &&
         k >= 8 && k % 8 == 0 && k <= kMaxWidth && rank >= 8 && rank % 8 == 0 && rank <= kMaxRank;
}

template <int RT>
void launch_lora(const LoraArgs& a, int64_t tiles, hipStream_t s) {
  hipLaunchKernelGGL(shrink_kernel<RT>, dim3((unsigned)(tiles * a.splits)),
                     dim3(kShrinkWaves * 64), 0, s, a);
  hipLaunchKernelGGL(expand_kernel<RT>, dim3((unsigned)(tiles * a.chunks)),
                     dim3(kExpandWaves * 64), 0, s, a);
}

}  // namespace
}  // namespace int8kv_serving

using namespace int8kv_serving;

extern "C" size_t int8kv_lora_plan_bytes(int64_t tokens, int32_t num_adapters) {
  if (tokens < 0 || tokens > kMaxTokens || num_adapters < 1 || num_adapters > kMaxAdapters) return 0;
  return 4 * (size_t)(4 + tokens + 3 * max_tiles(tokens, num_adapters, kTileRows));
}

extern "C" int int8kv_lora_plan(const void* adapter_ids, int ids_dtype, int64_t tokens,
                                int32_t num_adapters, void* plan, size_t plan_bytes, void* stream) {
  if (!plan || (tokens != 0 && !adapter_ids)) return INT8KV_E_NULL;
  if (ids_dtype != INT8KV_I32 && ids_dtype != INT8KV_I64) return INT8KV_E_DTYPE;
  const size_t need = int8kv_lora_plan_bytes(tokens, num_adapters);
  if (need == 0) return INT8KV_E_SHAPE;
  if (plan_bytes < need || reinterpret_cast<uintptr_t>(plan) % 16) return INT8KV_E_WORKSPACE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Plan p = plan_at(plan, tokens, num_adapters);
  auto kernel = ids_dtype == INT8KV_I64 ? plan_kernel<true> : plan_kernel<false>;
  hipLaunchKernelGGL(kernel, dim3(1), dim3(kPlanThreads), 0, s, adapter_ids, (int32_t)tokens,
                     num_adapters, kTileRows, p);
  return (int)hipGetLastError();
}

extern "C" size_t int8kv_lora_workspace_bytes(int64_t tokens, int32_t num_adapters, int64_t k,
                                              int32_t rank) {
  if (!lora_sizes_ok(tokens, num_adapters, k, rank)) return 0;
  const int64_t tiles = max_tiles(tokens, num_adapters, kTileRows);
  return (size_t)(tokens > 0 ? tokens : 1) * rank * 4 * splits_for(tiles, k);
}

extern "C" int int8kv_lora_add(const void* base, int64_t base_row_stride, const void* x,
                               int64_t tokens, int64_t k, int64_t x_row_stride, const void* lora_a,
                               const int64_t lora_a_strides[2], const void* lora_b,
                               const int64_t lora_b_strides[2], int32_t num_adapters, int32_t rank,
                               int64_t n, const float* scales, const void* plan, size_t plan_bytes,
                               void* out, int64_t out_row_stride, void* workspace,
                               size_t workspace_bytes, void* stream) {
  if (!lora_a || !lora_a_strides || !lora_b || !lora_b_strides || !plan) return INT8KV_E_NULL;
  if (tokens != 0 && (!base || !x || !out)) return INT8KV_E_NULL;
  if (!lora_sizes_ok(tokens, num_adapters, k, rank) || n < 8 || n % 8 || n > kMaxWidth)
    return INT8KV_E_SHAPE;
  // (The stride of a single row or adapter is never used.)
  if (tokens <= 1) base_row_stride = out_row_stride = n, x_row_stride = k;
  const int64_t a_adapter = num_adapters > 1 ? lora_a_strides[0] : 0;
  const int64_t b_adapter = num_adapters > 1 ? lora_b_strides[0] : 0;
  if (!rows16(base, base_row_stride) || !rows16(x, x_row_stride) || !rows16(out, out_row_stride) ||
      !rows16(lora_a, a_adapter) || lora_a_strides[1] % 8 || !rows16(lora_b, b_adapter) ||
      lora_b_strides[1] % 8 || x_row_stride < k || base_row_stride < n || out_row_stride < n ||
      lora_a_strides[1] < k || lora_b_strides[1] < rank)
    return INT8KV_E_STRIDE;
  if (plan_bytes < int8kv_lora_plan_bytes(tokens, num_adapters) ||
      reinterpret_cast<uintptr_t>(plan) % 16)
    return INT8KV_E_WORKSPACE;
  if (tokens == 0) return INT8KV_OK;
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 ||
      workspace_bytes < int8kv_lora_workspace_bytes(tokens, num_adapters, k, rank))
    return INT8KV_E_WORKSPACE;
  LoraArgs a;
  a.base = static_cast<const uint16_t*>(base);
  a.base_stride = base_row_stride;
  a.x = static_cast<const uint16_t*>(x);
  a.x_stride = x_row_stride;
  a.a = static_cast<const uint16_t*>(lora_a);
  a.a_adapter = a_adapter;
  a.a_row = lora_a_strides[1];
  a.b = static_cast<const uint16_t*>(lora_b);
  a.b_adapter = b_adapter;
  a.b_row = lora_b_strides[1];
  a.scales = scales;
  a.out = static_cast<uint16_t*>(out);
  a.out_stride = out_row_stride;
  a.part = static_cast<float*>(workspace);
  a.plan = plan_at(plan, tokens, num_adapters);
  a.tokens = (int32_t)tokens;
  a.k = (int32_t)k;
  a.n = (int32_t)n;
  a.rank = rank;
  const int64_t tiles = max_tiles(tokens, num_adapters, kTileRows);
  a.splits = splits_for(tiles, k);
  a.chunk = (int32_t)(((k + a.splits - 1) / a.splits + 31) / 32 * 32);
  a.chunks = (int32_t)((n + kExpandColumns - 1) / kExpandColumns);
  if (tiles * a.chunks > 0x7fffffff) return INT8KV_E_SHAPE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int tiles_of_rank = (rank + 15) / 16;
  if (tiles_of_rank <= 1)
    launch_lora<1>(a, tiles, s);
  else if (tiles_of_rank <= 2)
    launch_lora<2>(a, tiles, s);
  else if (tiles_of_rank <= 4)
    launch_lora<4>(a, tiles, s);
  else
    launch_lora<8>(a, tiles, s);
  return (int)hipGetLastError();
}
