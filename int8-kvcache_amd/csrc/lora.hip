// Low-rank adapters of many requests beside a shared projection:
//   out[t] = bf16(base[t] + scale[a] (x[t] A[a]^T) B[a]^T),  a = adapter of token t.
//
// A plan groups the tokens by adapter into tiles of one adapter each (16 tokens, or 64 in larger
// batches); the products then run tile by tile on matrix instructions, in two launches: x A^T into
// fp32 partial sums (split along k), then those times B^T, the scale and the base; or in one, where
// A is small.
//
// Precision: the first product's sums stay fp32.  They enter the second one as two bf16 parts,
// the upper bits and the rest (together 17 bits, of a rank-wide vector), so that both products run
// on bf16 matrix instructions and the result differs from an fp32 one by less than its own
// rounding to bf16 does.
//
// Bound: for few tokens by the adapters' bytes and two launches (one token, 3584 x 4608, rank 16:
// 7.4 us, where a launch that exits at once takes 2 to 3; 1100 tokens on 16 adapters, 18944 x 3584,
// rank 32: 25 us, whose bytes alone take 14 at a copy's rate); for many by reading the base and
// writing the result (6007 tokens, 3584 x 37888: 222 us, of them 210 in the second product at
// 4.4 TB/s).

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
constexpr int kPlanTokens = 16;  // tokens per thread whose places stay in registers

__device__ __forceinline__ float bf16_value(uint32_t h) { return __uint_as_float(h << 16); }
__device__ __forceinline__ uint32_t bf16_bits(float f) {
  return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f));
}

// ------------------------------------------------------------------------------------ plan
// {adapter, rows} of every tile (adapter -1: tokens without one; rows 0: an unused tile), then the
// tokens of every tile, `tile` each (what lies behind its rows is not set).
struct Plan {
  int2* head;
  int32_t* token;
  int32_t tiles;  // at most
};

// Tokens per tile: 16 (one matrix tile), or 64 where the adapters have 32 tokens or more each: an
// adapter's weights are then read for 64 tokens at a time where that counts (6007 tokens on 5
// adapters, rank 64, 3584 x 37888: 595 us with tiles of 16, most of it the traffic of B, 454 with 64
// and nothing else changed); below that the tiles would be mostly empty.
int tile_rows(int64_t tokens, int32_t adapters) {
  return tokens >= 32 * (int64_t)adapters && tokens >= 64 ? 64 : 16;
}

int64_t max_tiles(int64_t tokens, int32_t adapters, int rows) {
  const int64_t groups = (int64_t)adapters + 1 < tokens ? (int64_t)adapters + 1 : tokens;
  return tokens / rows + groups;  // each group rounds up by less than one tile
}

Plan plan_at(const void* p, int64_t tokens, int32_t adapters) {
  Plan q;
  q.tiles = (int32_t)max_tiles(tokens, adapters, tile_rows(tokens, adapters));
  q.head = static_cast<int2*>(const_cast<void*>(p));
  q.token = reinterpret_cast<int32_t*>(q.head + (q.tiles + 1) / 2 * 2);
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

// The next place of group g (the active lanes' own).  Neighbours in a prefill share their adapter:
// then one lane counts for all of them.
__device__ __forceinline__ int32_t next_place(int32_t* s_count, int32_t g) {
  const uint64_t active = __ballot(true);
  const int32_t first = __builtin_amdgcn_readfirstlane(g);
  if (__ballot(g == first) != active) return atomicAdd(&s_count[g], 1);
  const int32_t before = (int32_t)__popcll(active & ((1ull << (threadIdx.x & 63)) - 1));
  int32_t at = 0;
  if (before == 0) at = atomicAdd(&s_count[first], (int32_t)__popcll(active));
  return __builtin_amdgcn_readfirstlane(at) + before;
}

// One workgroup: a token's place in its group from a counter in LDS, then the groups' first tiles.
// The order of tokens within a group may differ from call to call; no result depends on it (a
// token's row is computed alike at every place).  HELD: all places stay in registers; otherwise
// they are counted a second time.
template <bool L64, bool HELD>
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(const void* ids, int32_t tokens,
                                                            int32_t adapters, int tile, Plan plan) {
  __shared__ int32_t s_count[kMaxAdapters + 1];
  __shared__ int32_t s_tile[kMaxAdapters + 1];
  __shared__ int32_t s_wave[kPlanThreads / 64];
  int32_t group[HELD ? kPlanTokens : 1], place[HELD ? kPlanTokens : 1];
  if constexpr (HELD) {
#pragma unroll
    for (int j = 0; j < kPlanTokens; ++j) {
      const int32_t t = j * kPlanThreads + (int32_t)threadIdx.x;
      group[j] = t < tokens ? adapter_of<L64>(ids, t, adapters) : -1;
    }
  }
  for (int32_t g = threadIdx.x; g <= adapters; g += kPlanThreads) s_count[g] = 0;
  __syncthreads();
  if constexpr (HELD) {
#pragma unroll
    for (int j = 0; j < kPlanTokens; ++j)
      if (group[j] >= 0) place[j] = next_place(s_count, group[j]);
  } else {
    for (int32_t t = threadIdx.x; t < tokens; t += kPlanThreads)
      next_place(s_count, adapter_of<L64>(ids, t, adapters));
  }
  __syncthreads();
  // The groups' first tiles; each thread a contiguous span of groups.
  const int32_t per = (adapters + 1 + kPlanThreads - 1) / kPlanThreads;
  const int32_t g0 = (int32_t)threadIdx.x * per;
  const int32_t g1 = g0 + per < adapters + 1 ? g0 + per : adapters + 1;
  int32_t tiles = 0;
  for (int32_t g = g0; g < g1; ++g) tiles += (s_count[g] + tile - 1) / tile;
  int32_t all_tiles;
  int32_t at = plan_scan(tiles, s_wave, all_tiles);
  for (int32_t g = g0; g < g1; ++g) {
    const int32_t n = s_count[g];
    s_tile[g] = at;
    for (int32_t i = 0; i < n; i += tile)
      plan.head[at++] = int2{g < adapters ? g : -1, n - i < tile ? n - i : tile};
    s_count[g] = 0;
  }
  for (int32_t i = all_tiles + (int32_t)threadIdx.x; i < plan.tiles; i += kPlanThreads)
    plan.head[i] = int2{-1, 0};
  __syncthreads();
  if constexpr (HELD) {
#pragma unroll
    for (int j = 0; j < kPlanTokens; ++j)
      if (group[j] >= 0)
        plan.token[s_tile[group[j]] * tile + place[j]] = j * kPlanThreads + (int32_t)threadIdx.x;
  } else {
    for (int32_t t = threadIdx.x; t < tokens; t += kPlanThreads) {
      const int32_t g = adapter_of<L64>(ids, t, adapters);
      plan.token[s_tile[g] * tile + next_place(s_count, g)] = t;
    }
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
  float* part;  // [splits][tiles x rows of a tile][rank]
  uint16_t* staged;  // [tiles x rows of a tile][2][rank]: their sums in two parts, or null
  Plan plan;
  int32_t tiles;       // of the products: the plan's, or its quarters (tile_shift 2)
  int32_t tile_shift;
  int32_t k, n, rank;
  int32_t splits;  // parts of k
  int32_t chunk;   // k of a part (a multiple of 32)
  int32_t halves;  // parts of the rank, 64 each (first product)
  int32_t chunks;  // column chunks (second product), taken in `groups` of `run`
  int32_t groups, run;
};

__device__ __forceinline__ bf16x8 load8(const uint16_t* p) {
  return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(p));
}
// 16 bytes of base or out; STREAM: past the caches.
template <bool STREAM>
__device__ __forceinline__ u32x4 load16(const uint16_t* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
  return *reinterpret_cast<const u32x4*>(p);
}
template <bool STREAM>
__device__ __forceinline__ void store16(uint16_t* p, u32x4 v) {
  if constexpr (STREAM)
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(p));
  else
    *reinterpret_cast<u32x4*>(p) = v;
}
// {adapter, rows} of a tile of 16 x TT tokens.
template <int TT>
__device__ __forceinline__ int2 head_of(const LoraArgs& a, int32_t tile) {
  int2 head = a.plan.head[TT == 1 ? tile >> a.tile_shift : tile];
  if constexpr (TT == 1) {
    const int32_t rows = head.y - 16 * (tile & ((1 << a.tile_shift) - 1));
    head.y = rows < 0 ? 0 : (rows < 16 ? rows : 16);
  }
  return head;
}
__device__ __forceinline__ bf16x8 zero8() {
  return __builtin_bit_cast(bf16x8, u32x4{0u, 0u, 0u, 0u});
}

// x A^T of one tile (TT x 16 tokens), one part of k and at most 64 ranks (RT x 16).  The waves
// take the part's 32-wide steps in turn, each with its next step's operands in flight, and add up
// through LDS.  Operands straight from memory: lane (i, g) holds 8 consecutive k of row i.
template <int TT>
constexpr int kShrinkWaves = TT == 1 ? 4 : 8;
template <int TT, int RT>
__global__ __launch_bounds__(kShrinkWaves<TT> * 64) void shrink_kernel(LoraArgs a) {
  constexpr int kRows = 16 * TT;
  constexpr int kWaves = kShrinkWaves<TT>;
  __shared__ f32x4 s_acc[kWaves / 2][TT * RT][64];
  const int32_t per_tile = a.splits * a.halves;
  const int32_t tile = blockIdx.x / per_tile;
  const int32_t rest = blockIdx.x - tile * per_tile;
  const int32_t split = rest / a.halves;
  const int32_t r0 = 64 * (rest - split * a.halves);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15;
  const int g = lane >> 4;
  const int2 head = head_of<TT>(a, tile);
  int32_t token[TT];
#pragma unroll
  for (int tt = 0; tt < TT; ++tt) token[tt] = a.plan.token[tile * kRows + 16 * tt + i];
  const int32_t adapter = __builtin_amdgcn_readfirstlane(head.x);
  const int32_t rows = __builtin_amdgcn_readfirstlane(head.y);
  if (adapter < 0 || rows == 0) return;
  const int32_t first = __builtin_amdgcn_readlane(token[0], 0);
  const uint16_t* xp[TT];
#pragma unroll
  for (int tt = 0; tt < TT; ++tt)
    xp[tt] = a.x + (int64_t)(16 * tt + i < rows ? token[tt] : first) * a.x_stride + 8 * g;
  const uint16_t* ap[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int32_t r = r0 + 16 * rt + i;
    ap[rt] = a.a + adapter * a.a_adapter + (int64_t)(r < a.rank ? r : a.rank - 1) * a.a_row + 8 * g;
  }
  f32x4 acc[TT][RT];
#pragma unroll
  for (int tt = 0; tt < TT; ++tt)
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) acc[tt][rt] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int32_t k0 = split * a.chunk;
  const int32_t k1 = k0 + a.chunk < a.k ? k0 + a.chunk : a.k;
  // Steps in flight: as many as leave the tile's operands room in the registers.
  constexpr int kFlight = TT * RT == 1 ? 4 : (TT * RT <= 4 ? 2 : 1);
  constexpr int kStep = 32 * kWaves;
  bf16x8 xv[kFlight][TT], av[kFlight][RT];
  const auto request = [&](int f, int32_t k) {
    const bool in = k + 8 * g < k1;  // k is a multiple of 8
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) xv[f][tt] = in ? load8(xp[tt] + k) : zero8();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) av[f][rt] = in ? load8(ap[rt] + k) : zero8();
  };
  int32_t k = k0 + 32 * wave;
#pragma unroll
  for (int f = 0; f < kFlight; ++f) request(f, k + f * kStep);
  for (; k < k1; k += kFlight * kStep) {
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      bf16x8 x[TT], w[RT];
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) x[tt] = xv[f][tt];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) w[rt] = av[f][rt];
      request(f, k + (kFlight + f) * kStep);
#pragma unroll
      for (int tt = 0; tt < TT; ++tt)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          acc[tt][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[rt], x[tt], acc[tt][rt], 0, 0, 0);
    }
  }
  // The upper half of the waves hands its sums to the lower half, until wave 0 has all.
#pragma unroll
  for (int half = kWaves / 2; half >= 1; half >>= 1) {
    if (wave >= half && wave < 2 * half)
#pragma unroll
      for (int tt = 0; tt < TT; ++tt)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s_acc[wave - half][tt * RT + rt][lane] = acc[tt][rt];
    __syncthreads();
    if (wave < half)
#pragma unroll
      for (int tt = 0; tt < TT; ++tt)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[tt][rt] += s_acc[wave][tt * RT + rt][lane];
    __syncthreads();
  }
  // Lane (i, g) of tile (tt, rt): ranks 16 rt + 4 g .. + 3 of token 16 tt + i.
  if (wave == 0)
#pragma unroll
    for (int tt = 0; tt < TT; ++tt)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int32_t r = r0 + 16 * rt + 4 * g;
        const int64_t row = ((int64_t)split * a.tiles + tile) * kRows + 16 * tt + i;
        if (16 * tt + i < rows && r < a.rank)
          *reinterpret_cast<f32x4*>(a.part + row * a.rank + r) = acc[tt][rt];
      }
}

// Rank r's value of a token as two bf16 parts: upper (truncated: no overflow) and rest.
__device__ __forceinline__ void stage_value(uint16_t* row, int32_t r, int32_t rank, float h) {
  const uint32_t hi = __float_as_uint(h) >> 16;
  row[r] = (uint16_t)hi;
  row[rank + r] = fabsf(h) < INFINITY ? (uint16_t)bf16_bits(h - bf16_value(hi)) : 0;
}

// Eight columns: bf16(base + scale * products).
__device__ __forceinline__ u32x4 add_scaled(const float* product, float scale, u32x4 base) {
  const f32x4 d[2] = {*reinterpret_cast<const f32x4*>(product),
                      *reinterpret_cast<const f32x4*>(product + 4)};
  u32x4 o;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float lo = d[j >> 1][2 * (j & 1)] * scale + bf16_value(base[j] & 0xffffu);
    const float hi = d[j >> 1][2 * (j & 1) + 1] * scale + bf16_value(base[j] >> 16);
    o[j] = bf16_bits(lo) | (bf16_bits(hi) << 16);
  }
  return o;
}

// The parts' sums, once, where many workgroups of the second product would each add them up; left
// as the two bf16 parts (what lies behind a tile's rows or was not written: any bits, which reach
// no row of a result).  Bound by latency: 2 to 4 us.
constexpr int kSumThreads = 256;
__global__ __launch_bounds__(kSumThreads) void sum_kernel(LoraArgs a, int32_t rows) {
  constexpr int kTogether = 8;
  const int32_t quads = a.rank / 4;
  const int64_t q = (int64_t)blockIdx.x * kSumThreads + threadIdx.x;
  const int64_t all = (int64_t)a.tiles * rows * quads;
  if (q >= all) return;
  const f32x4* part = reinterpret_cast<const f32x4*>(a.part);
  f32x4 h = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int32_t s0 = 0; s0 < a.splits; s0 += kTogether) {
    f32x4 y[kTogether];
#pragma unroll
    for (int u = 0; u < kTogether; ++u) y[u] = part[(s0 + u < a.splits ? s0 + u : 0) * all + q];
#pragma unroll
    for (int u = 0; u < kTogether; ++u)
      if (s0 + u < a.splits) h += y[u];
  }
  const int64_t row = q / quads;
  const int32_t c = 4 * (int32_t)(q - row * quads);
#pragma unroll
  for (int j = 0; j < 4; ++j) stage_value(a.staged + row * 2 * a.rank, c + j, a.rank, h[j]);
}

// The second product of one tile and one chunk of columns.  The rank-wide vectors are staged in
// LDS as two bf16 parts, upper (truncated: no overflow) and rest; along the product's inner axis
// first all upper parts, then all rests, against the same row of B.  NS: 32-wide steps of that
// axis; PAIRED: the rank is a multiple of 32, and the second half of the steps meets the first
// half's operands of B.  B's operands stay in registers for all tokens of the tile.
// Tiles of 64 tokens: a workgroup takes a run of column chunks, so that the vectors are read for
// more than 256 columns, and the workgroups of one die (every eighth) take the same columns of all
// tiles in turn, so that B is read into one L2 cache only.
// Loads are requested as early as their addresses are known: the partial sums (which depend on the
// tile's number alone), then B and the first base rows.  Base and out are read and written in
// whole 128-byte lines, eight lanes each; the products get there through LDS (in operand order,
// where neighbouring lanes hold different rows, 6007 x 37888 took 437 us instead of 365).
constexpr int kExpandWaves = 4;
constexpr int kWaveColumns = 64;
constexpr int kExpandColumns = kExpandWaves * kWaveColumns;
constexpr int kXcds = 8;
constexpr int64_t kInfinityCacheBytes = 256 << 20;  // base and out beyond it stream past the caches
template <int TT, int NS, bool PAIRED, bool STREAM>
__global__ __launch_bounds__(kExpandWaves * 64) void expand_kernel(LoraArgs a) {
  constexpr int kRows = 16 * TT;
  constexpr int kPad = 8;
  constexpr int kHeld = PAIRED ? NS / 2 : NS;
  __shared__ __align__(16) uint16_t s_h[kRows][32 * NS + kPad];
  __shared__ __align__(16) float s_out[kExpandWaves][16][kWaveColumns + 4];
  __shared__ __align__(16) float s_way[TT == 1 ? 4 * kExpandWaves * 64 : 4];
  int32_t tile, group;
  if constexpr (TT == 1) {
    tile = blockIdx.x / a.groups;
    group = blockIdx.x - tile * a.groups;
  } else {
    const int32_t at = blockIdx.x / kXcds;
    const int32_t round = at / a.tiles;
    tile = at - round * a.tiles;
    group = round * kXcds + blockIdx.x % kXcds;
    if (group >= a.groups) return;
  }
  const int32_t chunk0 = group * a.run;
  const int32_t chunk1 = chunk0 + a.run < a.chunks ? chunk0 + a.run : a.chunks;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15;
  const int g = lane >> 4;
  const int2 head = head_of<TT>(a, tile);
  // As an operand lane (i, g) holds token i; in base and out lane l holds columns 8 (l % 8) .. + 7
  // of rows l / 8 and 8 + l / 8.
  const int line = lane >> 3;
  int32_t token[TT][2];
#pragma unroll
  for (int tt = 0; tt < TT; ++tt)
#pragma unroll
    for (int h = 0; h < 2; ++h) token[tt][h] = a.plan.token[tile * kRows + 16 * tt + 8 * h + line];
  // The tile's vectors, four values per thread and round (those behind its rows are not set; they
  // meet no other row).
  const int32_t quads = a.rank / 4;
  const int64_t split_stride = (int64_t)a.tiles * kRows * a.rank;
  const float* part = a.part + (int64_t)tile * kRows * a.rank;
  constexpr int kTogether = 8;  // partial sums requested together
  f32x4 y[kTogether];
  // Tiles of 16 have fewer values than threads: then thread (p, way) adds every ways-th sum of p.
  const int32_t ways = TT == 1 && kRows * quads <= kExpandWaves * 32 ? kExpandWaves * 64 / (kRows * quads) : 1;
  const int32_t way = ways > 1 ? (int32_t)threadIdx.x / (kRows * quads) : 0;
  const int32_t p0 = (int32_t)threadIdx.x - way * kRows * quads;
  const auto request_parts = [&](int32_t p, int32_t s0) {
#pragma unroll
    for (int u = 0; u < kTogether; ++u) {
      const int32_t s = s0 + u * ways;
      y[u] = *reinterpret_cast<const f32x4*>(part + (s < a.splits ? s : 0) * split_stride +
                                             4 * (p < kRows * quads ? p : 0));
    }
  };
  // Summed already: 16-byte pieces of the two parts.
  const int32_t row_pieces = a.rank / 4;
  const uint16_t* sums = a.staged + (int64_t)tile * kRows * 2 * a.rank;
  const bool summed = TT > 1 && a.staged;
  if (summed) {
#pragma unroll
    for (int u = 0; u < kTogether; ++u) {
      const int32_t p = (int32_t)threadIdx.x + u * kExpandWaves * 64;
      y[u] = *reinterpret_cast<const f32x4*>(sums + 8 * (p < kRows * row_pieces ? p : 0));
    }
  } else {
    request_parts(p0, way);
  }
  const int32_t adapter = __builtin_amdgcn_readfirstlane(head.x);
  const int32_t rows = __builtin_amdgcn_readfirstlane(head.y);
  if (rows == 0) return;
  const int32_t first = __builtin_amdgcn_readlane(token[0][0], 0);
  const int32_t granules = a.rank / 8;  // 8-wide pieces of one part
  int32_t col0 = chunk0 * kExpandColumns + wave * kWaveColumns;
  int32_t col = col0 + 8 * (lane & 7);  // this lane's in base and out
  bool in = col < a.n;
  u32x4 base[TT][2];  // of all the tile's tokens: requested a chunk ahead
  const auto request_base = [&](int tt) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t t = 16 * tt + 8 * h + line < rows ? token[tt][h] : first;
      base[tt][h] = in ? load16<STREAM>(a.base + t * a.base_stride + col) : u32x4{0u, 0u, 0u, 0u};
    }
  };
  if (adapter < 0) {
    if (a.out == a.base && a.out_stride == a.base_stride) return;
    for (int32_t chunk = chunk0; chunk < chunk1; ++chunk) {
      in = col < a.n;
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) request_base(tt);
#pragma unroll
      for (int tt = 0; tt < TT; ++tt)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (in && 16 * tt + 8 * h + line < rows)
            store16<STREAM>(a.out + (int64_t)token[tt][h] * a.out_stride + col, base[tt][h]);
      col += kExpandColumns;
    }
    return;
  }
#pragma unroll
  for (int tt = 0; tt < TT; ++tt) request_base(tt);
  // Row 4 g + r of matrix tile j's operand is column 16 j + 4 g + r.
  bf16x8 bv[kHeld][4];
  const auto request_b = [&]() {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int32_t c = col0 + 16 * j + i;
      const uint16_t* bp = a.b + adapter * a.b_adapter + (int64_t)(c < a.n ? c : a.n - 1) * a.b_row;
#pragma unroll
      for (int s = 0; s < kHeld; ++s) {
        const int32_t p = 4 * s + g;
        bv[s][j] = p < 2 * granules ? load8(bp + 8 * (p < granules ? p : p - granules)) : zero8();
      }
    }
  };
  request_b();
  const float scale = a.scales ? a.scales[adapter] : 1.0f;
  const auto stage = [&](int32_t p, f32x4 h) {
    const int32_t r = p / quads;
    const int32_t c = 4 * (p - r * quads);
#pragma unroll
    for (int j = 0; j < 4; ++j) stage_value(&s_h[r][0], c + j, a.rank, h[j]);
  };
  if (summed) {
    static_assert(TT == 1 || kRows * kMaxRank / 4 <= kTogether * kExpandWaves * 64, "one round");
#pragma unroll
    for (int u = 0; u < kTogether; ++u) {
      const int32_t p = (int32_t)threadIdx.x + u * kExpandWaves * 64;
      const int32_t r = p / row_pieces;
      if (p < kRows * row_pieces) *reinterpret_cast<f32x4*>(&s_h[r][8 * (p - r * row_pieces)]) = y[u];
    }
  }
  for (int32_t p = summed ? kRows * quads : p0; p < kRows * quads; p += kExpandWaves * 64) {
    f32x4 h = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int32_t s0 = way; s0 < a.splits; s0 += kTogether * ways) {
      if (p != p0 || s0 != way) request_parts(p, s0);
#pragma unroll
      for (int u = 0; u < kTogether; ++u)
        if (s0 + u * ways < a.splits) h += y[u];
    }
    if (ways == 1)
      stage(p, h);
    else if (way < ways)
      *reinterpret_cast<f32x4*>(&s_way[4 * threadIdx.x]) = h;
  }
  if (ways > 1) {
    __syncthreads();
    if ((int32_t)threadIdx.x < kRows * quads) {
      f32x4 h = *reinterpret_cast<const f32x4*>(&s_way[4 * threadIdx.x]);
      for (int32_t w = 1; w < ways; ++w)
        h += *reinterpret_cast<const f32x4*>(&s_way[4 * (threadIdx.x + w * kRows * quads)]);
      stage(threadIdx.x, h);
    }
  }
  __syncthreads();
  for (int32_t chunk = chunk0; chunk < chunk1; ++chunk) {
    if (chunk > chunk0) request_b();
    const int32_t here = col;
    const bool in_here = in;
    if (chunk + 1 < chunk1) {
      col0 += kExpandColumns;
      col += kExpandColumns;
      in = col < a.n;
    }
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
      if (16 * tt >= rows) break;  // (uniform)
      const u32x4 v[2] = {base[tt][0], base[tt][1]};
      if (chunk + 1 < chunk1) request_base(tt);
      f32x4 acc[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const int32_t p = 4 * s + g;
        const bf16x8 hv = p < 2 * granules ? load8(&s_h[16 * tt + i][8 * p]) : zero8();
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bv[s % kHeld][j], hv, acc[j], 0, 0, 0);
      }
      // (The wave's own buffer, and a wave's LDS accesses run in order: no barrier.)
#pragma unroll
      for (int j = 0; j < 4; ++j) *reinterpret_cast<f32x4*>(&s_out[wave][i][16 * j + 4 * g]) = acc[j];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4 o = add_scaled(&s_out[wave][8 * h + line][8 * (lane & 7)], scale, v[h]);
        if (in_here && 16 * tt + 8 * h + line < rows)
          store16<STREAM>(a.out + (int64_t)token[tt][h] * a.out_stride + here, o);
      }
    }
  }
}

// Both products of one tile of 16 tokens and 512 columns, for adapters whose A is small: every
// workgroup forms the tile's x A^T itself (its waves take the 32-wide steps of k in turn and add up
// through LDS), which saves the first product's launch and the partial sums' way through memory.
// B and the base rows are requested before the first product.  Bound by one launch's chain of loads
// (plan, then x, A, B and base) and by the rate at which a compute unit loads A.  One token, 1024 x
// 4096, rank 8: 4.2 us.
constexpr int kBothWaves = 8;
constexpr int kBothColumns = kBothWaves * kWaveColumns;
template <int RT, int NS, bool PAIRED>
__global__ __launch_bounds__(kBothWaves * 64) void both_kernel(LoraArgs a) {
  constexpr int kHeld = PAIRED ? NS / 2 : NS;
  constexpr int kFlight = RT == 1 ? 8 : 6;
  constexpr int kStep = 32 * kBothWaves;
  __shared__ __align__(16) uint16_t s_h[16][32 * NS + 8];
  __shared__ union {
    f32x4 acc[kBothWaves][RT * 64];
    float out[kBothWaves][16][kWaveColumns + 4];
  } s;
  const int32_t tile = blockIdx.x / a.groups;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15;
  const int g = lane >> 4;
  const int line = lane >> 3;
  const int2 head = head_of<1>(a, tile);
  const int32_t mine = a.plan.token[tile * 16 + i];
  int32_t token[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) token[h] = a.plan.token[tile * 16 + 8 * h + line];
  const int32_t adapter = __builtin_amdgcn_readfirstlane(head.x);
  const int32_t rows = __builtin_amdgcn_readfirstlane(head.y);
  if (rows == 0) return;
  const int32_t first = __builtin_amdgcn_readlane(mine, 0);
  const int32_t col0 = (int32_t)(blockIdx.x - tile * a.groups) * kBothColumns + wave * kWaveColumns;
  const int32_t col = col0 + 8 * (lane & 7);
  const bool in = col < a.n;
  u32x4 base[2];
  const auto request_base = [&]() {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t t = 8 * h + line < rows ? token[h] : first;
      base[h] = load16<false>(a.base + t * a.base_stride + (in ? col : 0));
    }
  };
  const auto store = [&](int h, u32x4 v) {
    if (in && 8 * h + line < rows)
      store16<false>(a.out + (int64_t)token[h] * a.out_stride + col, v);
  };
  if (adapter < 0) {
    if (a.out == a.base && a.out_stride == a.base_stride) return;
    request_base();
#pragma unroll
    for (int h = 0; h < 2; ++h) store(h, base[h]);
    return;
  }
  const uint16_t* xp = a.x + (int64_t)(i < rows ? mine : first) * a.x_stride + 8 * g;
  const uint16_t* ap[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int32_t r = 16 * rt + i;
    ap[rt] = a.a + adapter * a.a_adapter + (int64_t)(r < a.rank ? r : a.rank - 1) * a.a_row + 8 * g;
  }
  f32x4 acc[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) acc[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
  bf16x8 xv[kFlight], av[kFlight][RT];
  const auto request = [&](int f, int32_t k) {
    const bool inside = k + 8 * g < a.k;  // k is a multiple of 8
    xv[f] = inside ? load8(xp + k) : zero8();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) av[f][rt] = inside ? load8(ap[rt] + k) : zero8();
  };
  int32_t k = 32 * wave;
#pragma unroll
  for (int f = 0; f < kFlight; ++f) request(f, k + f * kStep);
  const int32_t granules = a.rank / 8;
  bf16x8 bv[kHeld][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int32_t c = col0 + 16 * j + i;
    const uint16_t* bp = a.b + adapter * a.b_adapter + (int64_t)(c < a.n ? c : a.n - 1) * a.b_row;
#pragma unroll
    for (int t = 0; t < kHeld; ++t) {
      const int32_t p = 4 * t + g;
      bv[t][j] = p < 2 * granules ? load8(bp + 8 * (p < granules ? p : p - granules)) : zero8();
    }
  }
  request_base();
  const float scale = a.scales ? a.scales[adapter] : 1.0f;
  for (; k < a.k; k += kFlight * kStep) {
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      const bf16x8 x = xv[f];
      bf16x8 w[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) w[rt] = av[f][rt];
      request(f, k + (kFlight + f) * kStep);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
        acc[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[rt], x, acc[rt], 0, 0, 0);
    }
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) s.acc[wave][rt * 64 + lane] = acc[rt];
  __syncthreads();
  // Value v of the tile: of rank 16 rt + 4 g + c and token i, v = 4 (64 rt + 16 g + i) + c.
  for (int32_t v = threadIdx.x; v < RT * 256; v += kBothWaves * 64) {
    float h = 0.0f;
#pragma unroll
    for (int w = 0; w < kBothWaves; ++w) h += reinterpret_cast<const float*>(s.acc[w])[v];
    const int32_t r = 16 * (v >> 8) + 4 * ((v >> 6) & 3) + (v & 3);
    if (r < a.rank) stage_value(&s_h[(v >> 2) & 15][0], r, a.rank, h);
  }
  __syncthreads();
  f32x4 sum[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) sum[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int t = 0; t < NS; ++t) {
    const int32_t p = 4 * t + g;
    const bf16x8 hv = p < 2 * granules ? load8(&s_h[i][8 * p]) : zero8();
#pragma unroll
    for (int j = 0; j < 4; ++j)
      sum[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bv[t % kHeld][j], hv, sum[j], 0, 0, 0);
  }
  // (The wave's own buffer.)
#pragma unroll
  for (int j = 0; j < 4; ++j) *reinterpret_cast<f32x4*>(&s.out[wave][i][16 * j + 4 * g]) = sum[j];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    store(h, add_scaled(&s.out[wave][8 * h + line][8 * (lane & 7)], scale, base[h]));
}

bool rows16(const void* p, int64_t stride) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride % 8 == 0;
}

// Whether the first pn and qn columns of two matrices' rows share memory (rows of different strides:
// whether the matrices' extents do).
bool rows_overlap(const void* p, int64_t ps, int64_t pn, const void* q, int64_t qs, int64_t qn,
                  int64_t rows) {
  const int64_t at = (int64_t)(reinterpret_cast<intptr_t>(q) - reinterpret_cast<intptr_t>(p)) / 2;
  if (at >= (rows - 1) * ps + pn || at + (rows - 1) * qs + qn <= 0) return false;
  if (rows == 1 || ps != qs) return true;
  const int64_t column = (at % ps + ps) % ps;
  return column < pn || column + qn > ps;
}

// Parts of k.  Tiles of 16 tokens: about four workgroups of four waves per compute unit (32 tokens
// on 24 adapters, the four projections of a layer: 35 us with 12-16 parts, 37 with 8, 56 with 2).
// Tiles of 64: eight waves, as many workgroups as run at a time, nearly two per unit up to rank 32
// and one above, where the registers leave room for no more (1100 tokens, 18944 x 3584, rank 32, 34
// tiles: 24.3 us with 12 parts, 27.7 with 7, 27.9 with 16; 1057 tokens, 18944 x 37888, rank 64, 20 tiles:
// 55 with 12, 62 with 16, 64 with 6).  A part has at least two steps per wave.
int splits_for(int64_t tiles, int64_t k, int rows, int32_t rank) {
  const int64_t shortest = 2 * 32 * (rows == 16 ? kShrinkWaves<1> : kShrinkWaves<4>);
  const int64_t most = k / shortest < 32 ? k / shortest : 32;
  int64_t s;
  if (rows == 16) {
    s = (1024 + tiles - 1) / (tiles > 0 ? tiles : 1);
    s = s < 16 ? s : 16;
  } else {
    s = (rank <= 32 ? 416 : 256) / (tiles * ((rank + 63) / 64));
  }
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : s);
}

// A plan's tiles of 64 tokens as four of 16, which have more workgroups with shorter chains but
// read A and B four times as often: up to 96 MB of that (16000 tokens, 512 x 512, rank 8, 17 MB: 12.4
// us, 26.2 in tiles of 64; 512, 3584 x 4608, rank 16, 13 MB: 9.7 and 12.1; 4942, 512 x 4376, rank
// 24, 74 MB: 30.4 and 35.2; 2000, 3584 x 4608, rank 32, 75 MB: 23.9 and 23.4; 160, 3584 x 37888,
// rank 64, 106 MB: 22.5 and 22.7; 1100, 18944 x 3584, rank 32, 196 MB: 36.9 and 33.3; 3000, 4096 x
// 4096, rank 64, 231 MB: 41.1 and 31.8).
bool taken_as_quarters(int64_t tiles, int64_t k, int32_t rank, int64_t n) {
  return 4 * tiles * rank * (k + n) * 2 <= 96 << 20;
}

// Both products in one launch?  A launch costs about 2.5 us and one compute unit loads A at about
// 30 bytes a ns, so where an adapter's A has at most 64 KB, and all workgroups' together 64 KB per
// compute unit (one token: 1024 x 4096, rank 8: 6.6 us in two launches, 4.2 in one; 2048 x 4608,
// rank 16: 6.5 and 5.6; 3584 x 4608, 112 KB: 6.5 and 7.2; 100 tokens on 40 adapters, 1024 x 4096,
// rank 16: 7.9 and 6.5; 250, 2048 x 4608: 8.4 and 10.6).
bool both_at_once(int64_t tiles, int rows, int64_t k, int32_t rank, int64_t n) {
  constexpr int64_t kMost = 64 << 10, kUnits = 256;
  const int64_t bytes = 2 * rank * k;
  return rows == 16 && rank <= 32 && bytes <= kMost &&
         tiles * ((n + kBothColumns - 1) / kBothColumns) * bytes <= kMost * kUnits;
}

bool lora_sizes_ok(int64_t tokens, int32_t adapters, int64_t k, int32_t rank) {
  return tokens >= 0 && tokens <= kMaxTokens && adapters >= 1 && adapters <= kMaxAdapters &&
         k >= 8 && k % 8 == 0 && k <= kMaxWidth && rank >= 8 && rank % 8 == 0 && rank <= kMaxRank;
}

template <int TT>
void launch_shrink(const LoraArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.tiles * a.splits * a.halves)), block(kShrinkWaves<TT> * 64);
  if (a.rank <= 16)
    hipLaunchKernelGGL((shrink_kernel<TT, 1>), grid, block, 0, s, a);
  else if (a.rank <= 32)
    hipLaunchKernelGGL((shrink_kernel<TT, 2>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((shrink_kernel<TT, 4>), grid, block, 0, s, a);
}

void launch_both(const LoraArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.tiles * a.groups)), block(kBothWaves * 64);
  const bool paired = a.rank % 32 == 0;
  switch ((2 * a.rank + 31) / 32) {
#define INT8KV_BOTH(RT, NS, PAIRED) \
  hipLaunchKernelGGL((both_kernel<RT, NS, PAIRED>), grid, block, 0, s, a)
    case 1: INT8KV_BOTH(1, 1, false); break;
    case 2:
      if (paired)
        INT8KV_BOTH(2, 2, true);
      else
        INT8KV_BOTH(2, 2, false);
      break;
#undef INT8KV_BOTH
    default: break;
  }
}

template <int TT, bool STREAM>
void launch_expand(const LoraArgs& a, hipStream_t s) {
  const int64_t groups = TT == 1 ? a.groups : (a.groups + kXcds - 1) / kXcds * kXcds;
  const dim3 grid((unsigned)(a.tiles * groups)), block(kExpandWaves * 64);
  const bool paired = a.rank % 32 == 0;
  switch ((2 * a.rank + 31) / 32) {
#define INT8KV_EXPAND(NS, PAIRED) \
  hipLaunchKernelGGL((expand_kernel<TT, NS, PAIRED, STREAM>), grid, block, 0, s, a)
    case 1: INT8KV_EXPAND(1, false); break;
    case 2:
      if (paired)
        INT8KV_EXPAND(2, true);
      else
        INT8KV_EXPAND(2, false);
      break;
    case 3: INT8KV_EXPAND(3, false); break;
    case 4:
      if (paired)
        INT8KV_EXPAND(4, true);
      else
        INT8KV_EXPAND(4, false);
      break;
    case 5: INT8KV_EXPAND(5, false); break;
    case 6:
      if (paired)
        INT8KV_EXPAND(6, true);
      else
        INT8KV_EXPAND(6, false);
      break;
    case 7: INT8KV_EXPAND(7, false); break;
    case 8:
      if (paired)
        INT8KV_EXPAND(8, true);
      else
        INT8KV_EXPAND(8, false);
      break;
#undef INT8KV_EXPAND
    default: break;
  }
}

}  // namespace
}  // namespace int8kv_serving

using namespace int8kv_serving;

extern "C" size_t int8kv_lora_plan_bytes(int64_t tokens, int32_t num_adapters) {
  if (tokens < 0 || tokens > kMaxTokens || num_adapters < 1 || num_adapters > kMaxAdapters) return 0;
  const int rows = tile_rows(tokens, num_adapters);
  const int64_t tiles = max_tiles(tokens, num_adapters, rows);
  return 16 + 8 * (size_t)((tiles + 1) / 2 * 2) + 4 * (size_t)(tiles * rows);
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
  const bool held = tokens <= kPlanTokens * kPlanThreads;
  auto kernel = ids_dtype == INT8KV_I64 ? (held ? plan_kernel<true, true> : plan_kernel<true, false>)
                                        : (held ? plan_kernel<false, true> : plan_kernel<false, false>);
  hipLaunchKernelGGL(kernel, dim3(1), dim3(kPlanThreads), 0, s, adapter_ids, (int32_t)tokens,
                     num_adapters, tile_rows(tokens, num_adapters), p);
  return (int)hipGetLastError();
}

extern "C" size_t int8kv_lora_workspace_bytes(int64_t tokens, int32_t num_adapters, int64_t k,
                                              int32_t rank) {
  if (!lora_sizes_ok(tokens, num_adapters, k, rank)) return 0;
  const int rows = tile_rows(tokens, num_adapters);
  const int64_t tiles = max_tiles(tokens, num_adapters, rows);
  int64_t parts = splits_for(tiles, k, rows, rank);
  if (rows == 64) {  // with their sums, or taken as quarters
    const int64_t quarters = splits_for(4 * tiles, k, 16, rank);
    parts = parts + 1 > quarters ? parts + 1 : quarters;
  }
  return 16 + (size_t)(tiles * rows * rank * 4 * parts);
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
  const bool in_place = out == base && out_row_stride == base_row_stride;
  if ((!in_place && rows_overlap(out, out_row_stride, n, base, base_row_stride, n, tokens)) ||
      rows_overlap(out, out_row_stride, n, x, x_row_stride, k, tokens))
    return INT8KV_E_STRIDE;
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
  a.k = (int32_t)k;
  a.n = (int32_t)n;
  a.rank = rank;
  int64_t tiles = a.plan.tiles;
  int rows = tile_rows(tokens, num_adapters);
  a.chunks = (int32_t)((n + kExpandColumns - 1) / kExpandColumns);
  a.tile_shift = 0;
  if (rows == 64 && taken_as_quarters(tiles, k, rank, n)) {
    rows = 16;
    a.tile_shift = 2;
    tiles *= 4;
  }
  a.tiles = (int32_t)tiles;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (both_at_once(tiles, rows, k, rank, n)) {
    a.groups = (int32_t)((n + kBothColumns - 1) / kBothColumns);
    launch_both(a, s);
    return (int)hipGetLastError();
  }
  a.splits = splits_for(tiles, k, rows, rank);
  a.chunk = (int32_t)(((k + a.splits - 1) / a.splits + 31) / 32 * 32);
  a.halves = (rank + 63) / 64;
  // Runs of chunks: while there are about fourteen workgroups per compute unit (99 tiles of 148
  // chunks: runs of 4 240 us, 2 255, 8 265, 1 300).
  int64_t run = rows == 16 ? 1 : tiles * a.chunks / 3584;
  a.run = (int32_t)(run < 1 ? 1 : (run < 8 ? run : 8));
  a.groups = (a.chunks + a.run - 1) / a.run;
  if (tiles * (a.groups + kXcds) > 0x7fffffff) return INT8KV_E_SHAPE;
  a.staged = nullptr;
  if (rows == 64) {
    launch_shrink<4>(a, s);
    // The parts' sums in a launch of their own, where a workgroup of the second product would need
    // more than four rounds of loads for them (148 tokens, 18944 x 3584, rank 64, 32 parts: 31.6 us
    // without, 19.4 with; 3294, 3936 x 4608, rank 128, 2 parts: 61.6 and 50.9; 500, 4096 x 4096,
    // rank 32, 8 parts, two rounds: 13.7 and 15.0), or all of them would read more than 32 MB of
    // parts (4907, 2048 x 3584, rank 32: 34.5 and 31.8; 6007, 3584 x 37888, rank 64: 232 and 226).
    const int64_t rounds = rank / 16 * ((a.splits + 7) / 8);
    if (rounds > 4 || tiles * a.groups * a.splits * rows * rank * 4 > 32 << 20) {
      a.staged = reinterpret_cast<uint16_t*>(a.part + (int64_t)a.splits * tiles * rows * rank);
      const int64_t quads = tiles * rows * rank / 4;
      hipLaunchKernelGGL(sum_kernel, dim3((unsigned)((quads + kSumThreads - 1) / kSumThreads)),
                         dim3(kSumThreads), 0, s, a, rows);
    }
    if (4 * tokens * n > kInfinityCacheBytes)
      launch_expand<4, true>(a, s);
    else
      launch_expand<4, false>(a, s);
  } else {
    launch_shrink<1>(a, s);
    launch_expand<1, false>(a, s);
  }
  return (int)hipGetLastError();
}
