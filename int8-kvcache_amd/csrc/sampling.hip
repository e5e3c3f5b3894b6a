// Sampling: one token per row of logits, with temperature, top-k, top-p and min-p, from a given
// uniform number per row.
//
// A token's weight is w = exp((v - M) / T), M the row's maximum.  The tokens in order of falling
// logit (equal ones by index) make top-k, top-p and min-p each a prefix of one order, so what is
// kept is described by a cut: every token above a key tau, and the first `ties` tokens (by index)
// at tau.  The token is then the inverse of the cumulative kept weight in index order.
//
// Which token comes out depends on sums over the whole vocabulary, next to borders that a
// rounding could move, so weights are exact to about 2^-41 (2^-44 at 152064 tokens): 2^y by a
// polynomial in 64 bits, rounded to a fixed-point integer.
// Integer sums do not depend on their order: chunking and atomics cannot change a result.
//
// Launches: chunk_kernel reads the logits once (maxima, and masses where the row needs its whole
// one); bins_kernel and gather_kernel, where some row may have a nucleus cut over a long row, find
// its bin and the tokens in it; row_kernel finishes a row.  What bounds them: the first pass by
// memory where no mass is needed (37 MB of 61 x 152064 fp32: 9.0 us, 4.1 TB/s) and by 64-bit
// arithmetic where it is (156 MB of 256 x 152064 fp32: 43.5 us, 3.6 TB/s; a copy of that size reads
// and writes 5 TB/s); the others by the latency of their steps, each a load, a barrier or a scan of
// one workgroup that waits for the one before (about 1 us each).

#include <hip/hip_runtime.h>

#include <cstdint>

#include "int8kv_common.h"
#include "serving_ops.h"
#include "wave_scan.h"

namespace int8kv_serving {
namespace {

using int8kv::kBF16;
using int8kv::kF16;
using int8kv::kF32;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 1024;  // of the workgroup that finishes a row
constexpr int kWaves = kThreads / 64;
constexpr int kChunkThreads = 256;     // of a workgroup of the first pass ...
constexpr int kChunkElements = 4096;   // ... and the elements it reads: 16 per thread
constexpr int kPieceElements = 256;    // elements whose maximum the first pass keeps
constexpr int kMaxTiles = kThreads;    // one per thread in the tile scan
constexpr int kList = 4096;            // tokens a row's exact order is made of
constexpr int64_t kMaxVocab = 1 << 21;  // 513 chunks at most
constexpr int64_t kMaxRows = 1 << 16;
constexpr int64_t kGroupRows = 1024;  // rows that share a workspace (60 KB each) and its launches

struct SampleArgs {
  const void* logits;
  int64_t rows;
  int64_t row_stride;  // elements
  int32_t vocab;
  int32_t frac;  // fraction bits of a weight
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t* out;
  int32_t chunks;   // of the first pass, per row, taken in `runs` of `run_chunks`
  int32_t runs, run_chunks;
  int32_t pieces;   // kChunkElements / kPieceElements of each chunk
  int32_t parts;    // workgroups per row of the histogram pass (0: it does not run)
  float* chunk_max;      // [rows][chunks]
  uint64_t* chunk_mass;  // [rows][chunks] (rows without a filter), in units of the chunk's own maximum
  float* piece_max;      // [rows][pieces]
  uint64_t* bin_mass;    // [rows][kBins]
  uint64_t* tile_mass;   // [rows][kMaxTiles]
  uint64_t* list;        // [rows][kList] places
  int32_t* list_count;   // [rows] tokens of the list
};

// ------------------------------------------------------------------------------ row access
// A row as slots: slot 0 the elements before the first 16-byte boundary, slots 1 .. whole 16-byte
// vectors, the last slot what is left.  Elements a slot lacks read as -inf (weight 0).
template <int DT>
struct Row {
  static constexpr int kE = DT == kF32 ? 4 : 8;     // elements of a vector
  static constexpr int kSize = DT == kF32 ? 4 : 2;  // bytes of one
  const char* p;
  const u32x4* body;  // the whole vectors (any readable memory if there are none)
  int32_t vocab, head, vectors;

  __device__ __forceinline__ Row(const SampleArgs& a, int64_t r) {
    p = static_cast<const char*>(a.logits) + r * a.row_stride * kSize;
    vocab = a.vocab;
    const int32_t off = (int32_t)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / kSize;
    head = off < vocab ? off : vocab;
    vectors = (vocab - head) / kE;
    body = vectors > 0 ? reinterpret_cast<const u32x4*>(p + (int64_t)head * kSize)
                       : reinterpret_cast<const u32x4*>(a.chunk_mass);
  }
  __device__ __forceinline__ int32_t slots() const { return vectors + 2; }
  // Index of a slot's first element.
  __device__ __forceinline__ int32_t first(int32_t s) const {
    return s == 0 ? 0 : head + (s - 1) * kE;
  }
  static __device__ __forceinline__ float value_in(const void* values, int32_t i) {
    if constexpr (DT == kF32)
      return static_cast<const float*>(values)[i];
    else if constexpr (DT == kBF16)
      return __uint_as_float((uint32_t) static_cast<const uint16_t*>(values)[i] << 16);
    else
      return (float)static_cast<const _Float16*>(values)[i];
  }
  __device__ __forceinline__ float element(int32_t i) const { return value_in(p, i); }
  // A slot's vector, requested without a branch (an edge slot requests a neighbour's).
  __device__ __forceinline__ u32x4 request(int32_t s) const {
    const int32_t i = s - 1 < vectors - 1 ? s - 1 : vectors - 1;
    return body[i > 0 ? i : 0];
  }
  // The slot's values from what request() gave, NaN as it is.  INNER: no edge slot.
  template <bool INNER>
  __device__ __forceinline__ void values(int32_t s, u32x4 raw, float (&v)[kE]) const {
    if constexpr (DT == kF32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(raw[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) int8kv::unpack2<DT>(raw[j], v[2 * j], v[2 * j + 1]);
    }
    if (!INNER && !(s >= 1 && s <= vectors)) {
      const int32_t i0 = first(s);
      const int32_t n = s == 0 ? head : (s == vectors + 1 ? vocab - i0 : 0);
#pragma unroll
      for (int j = 0; j < kE; ++j) v[j] = j < n ? element(i0 + j) : -INFINITY;
    }
  }
  // The slot's values, NaN as -inf.
  __device__ __forceinline__ void load(int32_t s, float (&v)[kE]) const {
    values<false>(s, request(s), v);
#pragma unroll
    for (int j = 0; j < kE; ++j) v[j] = fmaxf(v[j], -INFINITY);  // (fmaxf: the number, if one is NaN)
  }
};

// Keys order as the values do; -0 and +0 are one value.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// ---------------------------------------------------------------------------------- weights
// w(v) = 2^((v - M) log2(e) / T) in units of 2^-frac.  With y = n + f, |f| <= 1/2, 2^f by a
// polynomial (interpolation at Chebyshev nodes, relative error 2e-12, exactly 1 at f = 0).
__device__ __forceinline__ double exp2_part(double f) {
  double p = 0x1.63b2d796ba66ap-20;
  p = fma(p, f, 0x1.00c0e4e15180ap-16);
  p = fma(p, f, 0x1.4308c7183da5dp-13);
  p = fma(p, f, 0x1.5d877598350fdp-10);
  p = fma(p, f, 0x1.3b2ab70ad2564p-7);
  p = fma(p, f, 0x1.c6b08da70cce3p-5);
  p = fma(p, f, 0x1.ebfbdff82a734p-3);
  p = fma(p, f, 0x1.62e42fef9cc69p-1);
  return fma(p, f, 1.0);
}
// 2^(frac + n), n >= -102.
__device__ __forceinline__ double exp2_scale(int32_t n, int32_t frac) {
  return __hiloint2double((n + (1023 + frac)) << 20, 0);
}
constexpr double kRound = 0x1.8p52;  // y + kRound - kRound: y rounded to an integer, left in the low bits

// Rounded to integers by adding 2^52: the integer is left in the low bits.
//
// 19 operations of 64 bits, each 8 cycles of a wave where 32-bit ones take 4.
struct Weights {
  double c;    // log2(e) / T
  double top;  // M
  float topf;
  int32_t frac;

  __device__ __forceinline__ uint64_t operator()(float v) const {
    if (topf == INFINITY) return v == topf ? (uint64_t)1 << frac : 0;
    const double y = fmax(((double)v - top) * c, -100.0);  // (NaN, of -inf and T = inf: -100, weight 0)
    const double t = y + kRound;
    const double p = exp2_part(y - (t - kRound));
    const double r = fma(p, exp2_scale(__double2loint(t), frac), 0x1p52);
    return (uint64_t)__double_as_longlong(r) - 0x4330000000000000ull;
  }
};

// The same up to the last bits of y for ordinary temperatures and logits, added to a sum that
// starts at 2^52 (at most 16 weights: below 2^53, so that each is rounded to an integer): 15
// 64-bit operations per weight instead of 19, and no test.  A row's chunk masses and the choice
// within the chunk both use it.
struct FastWeights {
  double c, k;  // y = v c - k
  float low;    // y is about -99.5 here: weight 0
  int32_t frac;

  // `rate`: log2(e) / t.
  __device__ __forceinline__ FastWeights(double rate, float t, float top, int32_t fraction) {
    c = rate;
    k = (double)top * c;
    low = top - 69.0f * t;  // (about 100 ln 2)
    frac = fraction;
  }
  // The maximum's weight is exactly 2^frac, and `low` lies below the maximum.
  static __device__ __forceinline__ bool fits(float t, float top) {
    return t > 0x1p-10f && t < 0x1p10f && fabsf(top) < 64.0f * t;
  }
  __device__ __forceinline__ double add(float v, double sum) const {
    const double y = fma((double)fmaxf(v, low), c, -k);
    const double t = y + kRound;
    const double p = exp2_part(y - (t - kRound));
    return fma(p, exp2_scale(__double2loint(t), frac), sum);
  }
  __device__ __forceinline__ uint64_t operator()(float v) const { return value(add(v, 0x1p52)); }
  static __device__ __forceinline__ uint64_t value(double sum) {
    return (uint64_t)__double_as_longlong(sum) - 0x4330000000000000ull;
  }
};

// ------------------------------------------------------------------------- workgroup sums
// Barrier for data exchanged through LDS: loads in flight stay in flight.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_max(float v) {
  const uint32_t b = __float_as_uint(v);
  return fmaxf(v, __uint_as_float(dpp<CTRL, ROWS>(b, b)));
}
// The largest (or smallest) of the lanes' values, in lane 63.
template <bool LARGEST>
__device__ __forceinline__ uint32_t wave_extreme(uint32_t v) {
  const auto pick = [](uint32_t a, uint32_t b) { return (a > b) == LARGEST ? a : b; };
  v = pick(v, dpp<0x111, 0xf>(v, v));
  v = pick(v, dpp<0x112, 0xf>(v, v));
  v = pick(v, dpp<0x114, 0xf>(v, v));
  v = pick(v, dpp<0x118, 0xf>(v, v));
  v = pick(v, dpp<0x142, 0xa>(v, v));
  return pick(v, dpp<0x143, 0xc>(v, v));
}
// Running maximum: lane 15 of each 16, then lanes 31 and 63 hold their 32 lanes', then lane 63 all.
__device__ __forceinline__ float max_to_31(float m) {
  m = dpp_max<0x111, 0xf>(m);
  m = dpp_max<0x112, 0xf>(m);
  m = dpp_max<0x114, 0xf>(m);
  m = dpp_max<0x118, 0xf>(m);
  return dpp_max<0x142, 0xa>(m);
}
__device__ __forceinline__ float max_to_63(float m) { return dpp_max<0x143, 0xc>(m); }
__device__ __forceinline__ float wave_max(float m) {
  return __uint_as_float(last_lane(__float_as_uint(max_to_63(max_to_31(m)))));
}
// --------------------------------------------------------------------------- row parameters
struct Params {
  double u;
  float t;      // temperature
  int32_t k;    // 0: off
  double p;     // >= 1: off
  double m;     // 0: off
  bool greedy;  // the first maximum, whatever u is
};

__device__ __forceinline__ Params row_params(const SampleArgs& a, int64_t r) {
  Params q;
  const double u = a.u[r];
  q.u = u > 0.0 ? (u < 1.0 ? u : 0x1.fffffffffffffp-1) : 0.0;
  q.t = a.temperature ? a.temperature[r] : 1.0f;
  const int32_t k = a.top_k ? a.top_k[r] : 0;
  q.k = k > 0 && k < a.vocab ? k : 0;
  const float p = a.top_p ? a.top_p[r] : 1.0f;
  q.p = p < 1.0f ? (double)p : 2.0;
  const float m = a.min_p ? a.min_p[r] : 0.0f;
  q.m = m > 0.0f ? (double)m : 0.0;
  // One token kept, the first of the order: nothing to draw.
  q.greedy = !(q.t > 0.0f) || q.k == 1 || q.p <= 0.0 || q.m > 1.0;
  return q;
}

// Smallest integer weight that min-p keeps: w >= m 2^frac.
__device__ __forceinline__ uint64_t least_weight(double m, int32_t frac) {
  return m > 0.0 ? (uint64_t)ceil(m * __longlong_as_double((int64_t)(1023 + frac) << 52)) : 0;
}

// floor(u z) for 0 <= u < 1, exactly: u = mant 2^-sh with a 53-bit mant.
__device__ __forceinline__ uint64_t scaled(double u, uint64_t z) {
  if (!(u > 0.0)) return 0;
  const uint64_t bits = (uint64_t)__double_as_longlong(u);
  const int e = (int)(bits >> 52);
  if (e == 0) return 0;  // below 2^-1022
  const uint64_t mant = (bits & 0xfffffffffffffull) | 0x10000000000000ull;
  const int sh = 1075 - e;  // >= 53
  const uint64_t hi = __umul64hi(mant, z), lo = mant * z;
  if (sh < 64) return (hi << (64 - sh)) | (lo >> sh);
  return sh < 128 ? hi >> (sh - 64) : 0;
}

// ------------------------------------------------------------------------------- histogram
// Bins of d = M - v, 128 to an octave from 2^-10 to 256, one below and one above: fine where a
// cut can lie whatever the temperature, and monotone in v (the subtraction rounds monotonically).
constexpr int kBinShift = 16;  // 7 mantissa bits
constexpr int kBinBase = (127 - 10) << 7;
constexpr int kBins = 18 * 128 + 2;
constexpr int kThreadBins = (kBins + kThreads - 1) / kThreads;
__device__ __forceinline__ int32_t bin_of(float v, float top) {
  const float d = v == top ? 0.0f : top - v;
  const int32_t b = (int32_t)(__float_as_uint(d) >> kBinShift) - kBinBase + 1;
  return b < 0 ? 0 : (b < kBins ? b : kBins - 1);
}

// Rows with a nucleus cut alone: their histogram pass and gathering run over many workgroups.  (A
// row of at most kList tokens lists them all.)
__device__ __forceinline__ bool needs_bins(const SampleArgs& a, const Params& q) {
  return a.parts > 0 && !q.greedy && q.k == 0 && q.p < 1.0;
}

// Rows with a long top-k: where those passes run, their list is gathered there too, since one
// workgroup reads a long row's tiles slowly.  (61 x 152064 fp32 beside rows with a nucleus cut:
// top-k 256 takes 23.0 us in row_kernel, 257 takes 11.4 there and 16.4 in gather_kernel, where the
// other rows' parts hide it; 1000 took 37.5 and takes 13.4 and 23.3.)
constexpr int kLongList = 256;
__device__ __forceinline__ bool needs_list(const SampleArgs& a, const Params& q) {
  return a.parts > 0 && !q.greedy && q.k > kLongList && q.k <= kList;
}

// Tokens waiting for their weights, so that those are computed by whole waves: places in a round's
// vectors, which lie beside them.
constexpr int kQueue = 8192;
constexpr int kTogether = 4;  // vectors per thread and round
struct Queue {
  u32x4 raw[kTogether * kThreads];
  uint16_t place[kQueue];
  int32_t length[2];  // of even and of odd rounds
};

// ------------------------------------------------------------------------------ first pass
// A run of chunks of one row, each held in registers while the next one is loaded: the maxima of
// their pieces and their own, and, for rows whose whole mass is needed, the sum of their weights in
// units of their own maximum (so that the data is read once).  Clears the row's bins where they
// will be used.  Workgroups of four waves: four share a compute unit (106 registers a lane),
// so that one reads while another computes.
template <int DT>
__global__ __launch_bounds__(kChunkThreads) void chunk_kernel(SampleArgs a) {
  constexpr int kE = Row<DT>::kE;
  constexpr int kSteps = kChunkElements / kChunkThreads / kE;
  constexpr int kPieceSlots = kPieceElements / kE;  // 32 or 64: half a wave's slots, or a wave's
  __shared__ float s_max[2][kChunkThreads / 64];
  __shared__ uint64_t s_sum[2][kChunkThreads / 64];
  const int64_t r = blockIdx.x / a.runs;
  const int32_t run = (int32_t)(blockIdx.x - r * a.runs);
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const Row<DT> row(a, r);
  const int32_t c0 = run * a.run_chunks;
  const int32_t c1 = c0 + a.run_chunks < a.chunks ? c0 + a.run_chunks : a.chunks;
  int32_t slot0 = c0 * (kSteps * kChunkThreads) + (int32_t)threadIdx.x;
  u32x4 raw[kSteps];
#pragma unroll
  for (int j = 0; j < kSteps; ++j) raw[j] = row.request(slot0 + j * kChunkThreads);
  const Params q = row_params(a, r);
  if (needs_bins(a, q)) {
    for (int32_t b = run * kChunkThreads + (int32_t)threadIdx.x; b < kBins; b += a.runs * kChunkThreads) {
      a.bin_mass[r * kBins + b] = 0;
    }
  }
  if (run == 0 && threadIdx.x == 0) a.list_count[r] = 0;
  // Rows whose whole mass is needed: without a filter, and with a nucleus cut alone.
  const bool summed = !q.greedy && q.k == 0 && (q.p < 1.0 ? a.parts > 0 : !(q.m > 0.0));
  const double rate = 0x1.71547652b82fep+0 / (double)q.t;
  for (int32_t c = c0; c < c1; ++c) {
    const int buf = c & 1;
    float v[kSteps][kE];
    if (c > 0 && (c + 1) * (kSteps * kChunkThreads) <= row.vectors) {
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
        row.template values<true>(slot0 + j * kChunkThreads, raw[j], v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
        row.template values<false>(slot0 + j * kChunkThreads, raw[j], v[j]);
    }
#pragma unroll
    for (int j = 0; j < kSteps; ++j)  // (behind the last chunk: the last vector again)
      raw[j] = row.request(c + 1 < c1 ? slot0 + (kSteps + j) * kChunkThreads : 0);
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      float m = v[j][0];
#pragma unroll
      for (int e = 1; e < kE; ++e) m = fmaxf(m, v[j][e]);
      m = max_to_31(m);
      if (kPieceSlots == 64) m = max_to_63(m);
      if (lane % kPieceSlots == kPieceSlots - 1)
        a.piece_max[r * a.pieces + (slot0 + j * kChunkThreads) / kPieceSlots] = m;
      top = fmaxf(top, m);
    }
    if (kPieceSlots == 32) top = max_to_63(top);
    if (lane == 63) s_max[buf][wave] = top;
    lds_barrier();
    top = s_max[buf][0];
#pragma unroll
    for (int w = 1; w < kChunkThreads / 64; ++w) top = fmaxf(top, s_max[buf][w]);
    if (threadIdx.x == 0) a.chunk_max[r * a.chunks + c] = top;
    if (summed) {
      uint64_t sum = 0;
      if (FastWeights::fits(q.t, top)) {
        const FastWeights w(rate, q.t, top, a.frac);
        double part = 0x1p52;
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
#pragma unroll
          for (int e = 0; e < kE; ++e) part = w.add(v[j][e], part);
        sum = FastWeights::value(part);
      } else if (top > -INFINITY) {
        const Weights w{rate, (double)top, top, a.frac};
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
#pragma unroll
          for (int e = 0; e < kE; ++e) sum += w(v[j][e]);
      }
      sum = wave_sum(sum);
      if (lane == 0) s_sum[buf][wave] = sum;
      lds_barrier();
      if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < kChunkThreads / 64; ++w) sum += s_sum[buf][w];
        a.chunk_mass[r * a.chunks + c] = sum;
      }
    }
    slot0 += kSteps * kChunkThreads;
  }
}

// One chunk per thread: its maximum, and its mass in units of that (where it was summed).
struct Chunk {
  float top;
  uint64_t mass;
};
__device__ __forceinline__ Chunk own_chunk(const SampleArgs& a, int64_t r) {
  const int64_t i = r * a.chunks + ((int32_t)threadIdx.x < a.chunks ? (int32_t)threadIdx.x : 0);
  Chunk c{a.chunk_max[i], a.chunk_mass[i]};
  if ((int32_t)threadIdx.x >= a.chunks) c = Chunk{-INFINITY, 0};
  return c;
}

// The row's maximum from its chunks' (s_max: kWaves).
__device__ __forceinline__ float row_max(const Chunk& chunk, float* s_max) {
  float m = wave_max(chunk.top);
  if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) m = fmaxf(m, s_max[w]);
  return m;
}

// The row's mass from its chunks', each scaled from its own maximum to the row's: returns the mass
// before this thread's chunk, `mass` its own and `factor` its scale.
__device__ __forceinline__ uint64_t scan_chunks(const Chunk& chunk, const Params& q, float top,
                                                uint64_t* s_wave, uint64_t& mass, double& factor,
                                                uint64_t& total) {
  mass = chunk.mass;
  factor = 1.0;
  if (mass > 0 && chunk.top < top) {
    factor = exp2(fmax(((double)chunk.top - (double)top) * (0x1.71547652b82fep+0 / (double)q.t), -200.0));
    mass = (uint64_t)rint((double)mass * factor);
  }
  return workgroup_scan<kWaves, uint64_t>(mass, s_wave, total);
}

// Tiles of a row: 1, 2, 4 ... pieces, at most kMaxTiles of them, each a power of two of slots.
template <int DT>
struct Tiles {
  int32_t count, shift, slots;  // slots = 1 << shift
  int32_t pieces_shift;

  __device__ __forceinline__ explicit Tiles(const SampleArgs& a) {
    pieces_shift = 0;
    while ((a.pieces >> pieces_shift) > kMaxTiles) ++pieces_shift;
    count = (a.pieces + (1 << pieces_shift) - 1) >> pieces_shift;
    shift = (Row<DT>::kE == 8 ? 5 : 6) + pieces_shift;
    slots = 1 << shift;
  }
  // The tile of a token.
  __device__ __forceinline__ int32_t of(const Row<DT>& row, int32_t index) const {
    constexpr int kShift = Row<DT>::kE == 8 ? 3 : 2;
    return (index < row.head ? 0 : 1 + ((index - row.head) >> kShift)) >> shift;
  }
  __device__ __forceinline__ float max_of(const SampleArgs& a, int64_t r, int32_t tile) const {
    float m = -INFINITY;
    for (int32_t i = tile << pieces_shift; i < (tile + 1) << pieces_shift && i < a.pieces; ++i)
      m = fmaxf(m, a.piece_max[r * a.pieces + i]);
    return m;
  }
};

// Adds this thread's tile to the list of those to visit, one addition per wave.
__device__ __forceinline__ void push_visit(bool wanted, int32_t tile, int32_t* visit, int32_t* visits) {
  const uint64_t m = __ballot(wanted);
  if (m == 0) return;
  const int lane = threadIdx.x & 63;
  int32_t at = 0;
  if (lane == 0) at = atomicAdd(visits, (int32_t)__popcll(m));
  at = __builtin_amdgcn_readfirstlane(at) + (int32_t)__popcll(m & ((1ull << lane) - 1));
  if (wanted) visit[at] = tile;
}

// Reads the tiles visit[0 .. visits), four slots per thread at a time and the next four in flight,
// and calls token(value, index) for every token that is at least `from` (not -inf), by whole waves:
// what a round finds is queued first, as places in its vectors (values and indices, found by a test
// per bit: 200 x 50257, the histogram pass 23 us and the gathering 18 instead of 20 and 16).  A wave
// that wants at least half of its values calls whole(values, mask, slot) for its slots instead
// (274 x 32000 bf16, nearly flat: the histogram pass 34 us, with the queue alone 61; with a quarter
// instead of half, 200 x 50257 took 25 us instead of 23).  One
// workgroup; queue.length is 0 before and after.  Rounds count in two lengths by turns: a wave that
// leaves a round where nothing was found may count in the next before others have read this one's.
template <int DT, typename Token, typename Whole>
__device__ __forceinline__ void read_tiles(const Row<DT>& row, const Tiles<DT>& tiles,
                                           const int32_t* visit, int32_t visits, float from,
                                           Queue& queue, Token token, Whole whole) {
  constexpr int kE = Row<DT>::kE;
  constexpr uint32_t kDense = 64 * kTogether * kE / 2;
  static_assert(kTogether * kThreads * kE <= 1 << 16, "a place has 16 bits");
  const int lane = threadIdx.x & 63;
  const int32_t items = visits << tiles.shift;
  const float least = fmaxf(from, -3.4028235e38f);
  const auto slot_of = [&](int32_t i) {
    return i < items ? (visit[i >> tiles.shift] << tiles.shift) + (i & (tiles.slots - 1)) : -1;
  };
  u32x4 raw[kTogether];
#pragma unroll
  for (int u = 0; u < kTogether; ++u) raw[u] = row.request(slot_of(u * kThreads + (int32_t)threadIdx.x));
  int32_t round = 0;
  for (int32_t i0 = 0; i0 < items; i0 += kTogether * kThreads) {
    int32_t* length = &queue.length[round++ & 1];
    uint32_t hits = 0;  // one bit per value
#pragma unroll
    for (int u = 0; u < kTogether; ++u) {
      const int32_t slot = slot_of(i0 + u * kThreads + (int32_t)threadIdx.x);
      if (slot >= 0) {
        float v[kE];
        row.template values<false>(slot, raw[u], v);
#pragma unroll
        for (int j = 0; j < kE; ++j) hits |= v[j] >= least ? 1u << (u * kE + j) : 0u;
      }
    }
    uint32_t incl = wave_scan<uint32_t>((uint32_t)__popc(hits));
    uint32_t all = last_lane(incl);
    if (all > kDense) {  // (uniform)
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
        const int32_t slot = slot_of(i0 + u * kThreads + (int32_t)threadIdx.x);
        if (slot < 0) continue;
        float v[kE];
        row.template values<false>(slot, raw[u], v);
        whole(v, (hits >> (u * kE)) & ((1u << kE) - 1), slot);
      }
      hits = 0;
      all = 0;
    } else if (all > 0) {
#pragma unroll
      for (int u = 0; u < kTogether; ++u) queue.raw[u * kThreads + threadIdx.x] = raw[u];
    }
#pragma unroll
    for (int u = 0; u < kTogether; ++u)
      raw[u] = row.request(slot_of(i0 + (kTogether + u) * kThreads + (int32_t)threadIdx.x));
    // (Barriers that leave the requests in flight.)
    for (int32_t found = kQueue + 1; found > kQueue;) {
      if (all > 0) {
        int32_t at = 0;
        if (lane == 63) at = atomicAdd(length, (int32_t)all);
        at = (int32_t)last_lane((uint32_t)at) + (int32_t)(incl - (uint32_t)__popc(hits));
        while (hits && at < kQueue) {
          const int32_t b = __ffs((int)hits) - 1;
          queue.place[at++] =
              (uint16_t)((b / kE * kThreads + (int32_t)threadIdx.x) * kE + b % kE);
          hits &= hits - 1;
        }
      }
      lds_barrier();
      found = *length;
      if (found == 0) break;
      const int32_t queued = found < kQueue ? found : kQueue;
      for (int32_t i = threadIdx.x; i < queued; i += kThreads) {
        const int32_t place = queue.place[i];
        const int32_t slot = slot_of(i0 + place / kE);
        const int32_t index = row.first(slot) + place % kE;
        const bool inner = slot >= 1 && slot <= row.vectors;
        token(inner ? Row<DT>::value_in(queue.raw, place) : row.element(index), index);
      }
      if (found > kQueue) {  // what is left goes into the next turn
        incl = wave_scan<uint32_t>((uint32_t)__popc(hits));
        all = last_lane(incl);
      }
      lds_barrier();
      if (threadIdx.x == 0) *length = 0;
      lds_barrier();
    }
  }
}

// The same for tokens far apart (a few per tile): slots that hold one are queued whole and looked
// through afterwards, so that reading costs a maximum and a comparison per slot.
constexpr int kSlotQueue = 1024;
struct SlotQueue {
  u32x4 raw[kSlotQueue];
  int32_t slot[kSlotQueue];
  int32_t length;
};
template <int DT, typename Token>
__device__ __forceinline__ void read_tiles_sparse(const Row<DT>& row, const Tiles<DT>& tiles,
                                                  const int32_t* visit, int32_t visits, float from,
                                                  SlotQueue& queue, Token token) {
  constexpr int kE = Row<DT>::kE;
  const int32_t items = visits << tiles.shift;
  const float least = fmaxf(from, -3.4028235e38f);
  const auto slot_of = [&](int32_t i) {
    return i < items ? (visit[i >> tiles.shift] << tiles.shift) + (i & (tiles.slots - 1)) : -1;
  };
  const auto look = [&](int32_t slot, u32x4 raw) {
    float v[kE];
    row.template values<false>(slot, raw, v);
#pragma unroll
    for (int j = 0; j < kE; ++j)
      if (v[j] >= least) token(v[j], row.first(slot) + j);
  };
  u32x4 raw[kTogether];
  int32_t slot[kTogether];
  const auto request = [&](int32_t i0) {
#pragma unroll
    for (int u = 0; u < kTogether; ++u) {
      slot[u] = slot_of(i0 + u * kThreads + (int32_t)threadIdx.x);
      raw[u] = row.request(slot[u]);
    }
  };
  request(0);
  for (int32_t i0 = 0; i0 < items; i0 += kTogether * kThreads) {
    u32x4 now[kTogether];
    int32_t at[kTogether];
#pragma unroll
    for (int u = 0; u < kTogether; ++u) {
      now[u] = raw[u];
      at[u] = slot[u];
    }
    if (i0 + kTogether * kThreads < items) request(i0 + kTogether * kThreads);
#pragma unroll
    for (int u = 0; u < kTogether; ++u) {
      if (i0 + u * kThreads >= items) break;  // (uniform)
      if (at[u] < 0) continue;
      float v[kE];
      row.template values<false>(at[u], now[u], v);
      float m = v[0];
#pragma unroll
      for (int j = 1; j < kE; ++j) m = fmaxf(m, v[j]);
      if (m >= least) {
        const int32_t place = atomicAdd(&queue.length, 1);
        if (place < kSlotQueue) {
          queue.raw[place] = now[u];
          queue.slot[place] = at[u];
        } else {
          look(at[u], now[u]);
        }
      }
    }
  }
  __syncthreads();
  // One value per thread.
  const int32_t n = queue.length < kSlotQueue ? queue.length : kSlotQueue;
  for (int32_t i = threadIdx.x; i < n * kE; i += kThreads) {
    const int32_t slot = queue.slot[i / kE];
    const int32_t index = row.first(slot) + i % kE;
    const bool whole = slot >= 1 && slot <= row.vectors;
    float v = Row<DT>::value_in(queue.raw, i);
    if (!whole) v = index < (slot == 0 ? row.head : row.vocab) ? row.element(index) : -INFINITY;
    if (v >= least) token(v, index);
  }
  __syncthreads();
}

// ------------------------------------------------------------------------ histogram pass
// One part of one row with a nucleus cut alone: the weights of its tokens per bin, added to the
// row's (integers: in any order).  Tokens with w < (1 - p) Z / vocab cannot be kept (they and all
// behind them weigh less than (1 - p) Z together) and are left out.  Two copies of the histogram
// lie interleaved, a lane's copy by its number: most tokens fall into about a hundred bins, and
// lanes that meet on one address go one after the other (four copies: no faster).
struct PartShared {
  Queue queue;
  uint64_t mass[2 * kBins];
  int32_t visit[kMaxTiles];
  uint64_t wave64[kWaves];
  float wave_max[kWaves];
  int32_t visits;
};

// The least logit that a token of a nucleus can have, with a margin for the roundings.
__device__ __forceinline__ float nucleus_from(const SampleArgs& a, const Params& q, float top,
                                              uint64_t total) {
  if (top == INFINITY) return top;
  // In 32 bits: a bound, and every thread of the workgroup computes it (in 64 bits 1.3 us of the
  // histogram pass).  The argument is off by 2^-22 of it at most, and so is its logarithm, which
  // is off by 2^-22 of itself besides.
  const float z = (float)((double)total * __longlong_as_double((int64_t)(1023 - a.frac) << 52));
  const float x = (float)(1.0 - q.p) * z / (float)a.vocab;
  const float d = (-logf(x) * (1.0f + 0x1p-18f) + 0x1p-18f) * q.t;
  return d > 0.0f ? (float)((double)top - (double)d) - (fabsf(top) + d) * 0x1p-20f : top;
}

template <int DT>
__global__ __launch_bounds__(kThreads) void bins_kernel(SampleArgs a) {
  __shared__ PartShared s;
  const int64_t r = blockIdx.x / a.parts;
  const int32_t part = (int32_t)(blockIdx.x - r * a.parts);
  const int t = threadIdx.x;
  const Params q = row_params(a, r);
  if (!needs_bins(a, q)) return;
  const Tiles<DT> tiles(a);
  const int32_t per = (tiles.count + a.parts - 1) / a.parts;
  const int32_t tile = part * per + t;
  const float tile_max = t < per && tile < tiles.count ? tiles.max_of(a, r, tile) : -INFINITY;
  const Chunk chunk = own_chunk(a, r);
  for (int32_t b = t; b < 2 * kBins; b += kThreads) s.mass[b] = 0;
  if (t == 0) s.visits = s.queue.length[0] = s.queue.length[1] = 0;
  const float top = row_max(chunk, s.wave_max);
  if (top == -INFINITY) return;
  uint64_t mass, total;
  double factor;
  scan_chunks(chunk, q, top, s.wave64, mass, factor, total);
  const float from = nucleus_from(a, q, top, total);
  push_visit(tile_max >= from && tile_max > -INFINITY, tile, s.visit, &s.visits);
  __syncthreads();
  const Row<DT> row(a, r);
  const Weights w{0x1.71547652b82fep+0 / (double)q.t, (double)top, top, a.frac};
  const auto count = [&](float v, int32_t) {
    atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[2 * bin_of(v, top) + (t & 1)]),
              (unsigned long long)w(v));
  };
  read_tiles(row, tiles, s.visit, s.visits, from, s.queue, count,
             [&](const float (&v)[Row<DT>::kE], uint32_t wanted, int32_t) {
#pragma unroll
    for (int j = 0; j < Row<DT>::kE; ++j)
      if (wanted & (1u << j)) count(v[j], 0);
  });
  __syncthreads();
  for (int32_t b = t; b < kBins; b += kThreads) {
    const uint64_t m = s.mass[2 * b] + s.mass[2 * b + 1];
    if (m)
      atomicAdd(reinterpret_cast<unsigned long long*>(&a.bin_mass[r * kBins + b]), (unsigned long long)m);
  }
}

// -------------------------------------------------------------------------- the general cut
// For rows whose cut falls among more tokens than the list holds (thousands of equal logits, or
// logits far closer together than the bins): digit by digit over the keys, reading the row again
// for each.
constexpr int kDigits = 2048;
struct General {
  uint64_t mass[kDigits];
  uint32_t count[kDigits];
  uint64_t wave64[kWaves];
  uint32_t wave32[kWaves];
  uint64_t found64[2];
  uint32_t found32[4];
};

// Every token with a key above tau is kept, and the first `ties` tokens at it.
struct Cut {
  uint32_t tau;
  uint32_t ties;
};

// The key at which a prefix of the order ends, digit by digit from the top (11, 11 and 10 bits; a
// 16-bit type's keys differ in the first 22 only).  BY_MASS: the first `want` units of weight,
// else the first `want` tokens; tokens at -inf are not counted.  Returns the key with the tokens and the mass
// above it and the tokens at it, or false where the row has less than `want`.
template <int DT, bool BY_MASS>
__device__ bool select_key(const Row<DT>& row, const Weights& w, uint64_t want, bool need_mass,
                           General& s, uint32_t& key, uint32_t& count_above, uint64_t& mass_above,
                           uint32_t& at_key) {
  constexpr int kLevels = DT == kF32 ? 3 : 2;
  uint32_t prefix = 0, mask = 0;
  count_above = 0;
  mass_above = 0;
  for (int level = 0; level < kLevels; ++level) {
    const int shift = level == 0 ? 21 : (level == 1 ? 10 : 0);
    const uint32_t digit = level == 2 ? 1023u : 2047u;
    __syncthreads();
    for (int b = threadIdx.x; b < kDigits; b += kThreads) {
      s.mass[b] = 0;
      s.count[b] = 0;
    }
    if (threadIdx.x == 0) s.found32[0] = 0xffffffffu;
    __syncthreads();
    for (int32_t q = threadIdx.x; q < row.slots(); q += kThreads) {
      float v[Row<DT>::kE];
      row.load(q, v);
#pragma unroll
      for (int j = 0; j < Row<DT>::kE; ++j) {
        const uint32_t k = key_of(v[j]);
        if (v[j] > -INFINITY && (k & mask) == prefix) {
          const uint32_t b = (k >> shift) & digit;
          atomicAdd(&s.count[b], 1u);
          if (BY_MASS || need_mass)
            atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[b]), (unsigned long long)w(v[j]));
        }
      }
    }
    __syncthreads();
    // Thread i holds bins 2047 - 2 i and 2046 - 2 i: the bins from the largest key down.
    const int b0 = kDigits - 1 - 2 * (int)threadIdx.x;
    const uint32_t c0 = s.count[b0], c1 = s.count[b0 - 1];
    const uint64_t m0 = s.mass[b0], m1 = s.mass[b0 - 1];
    uint32_t ctot;
    uint64_t mtot;
    const uint32_t cb = workgroup_scan<kWaves, uint32_t>(c0 + c1, s.wave32, ctot);
    const uint64_t mb = workgroup_scan<kWaves, uint64_t>(m0 + m1, s.wave64, mtot);
    const uint64_t left = want - (BY_MASS ? mass_above : (uint64_t)count_above);
    const uint64_t x0 = BY_MASS ? mb : (uint64_t)cb;
    const uint64_t x1 = x0 + (BY_MASS ? m0 : (uint64_t)c0);
    const uint64_t x2 = x1 + (BY_MASS ? m1 : (uint64_t)c1);
    if (x0 < left && left <= x2) {  // one thread
      const bool second = x1 < left;
      s.found32[0] = (uint32_t)(second ? b0 - 1 : b0);
      s.found32[1] = second ? cb + c0 : cb;
      s.found32[2] = second ? c1 : c0;
      s.found64[0] = second ? mb + m0 : mb;
    }
    __syncthreads();
    const uint32_t bin = s.found32[0];
    if (bin == 0xffffffffu) return false;
    prefix |= bin << shift;
    mask |= digit << shift;
    count_above += s.found32[1];
    mass_above += s.found64[0];
    at_key = s.found32[2];
  }
  // The low bits of a 16-bit type's key: zero, or one for negative values (their bits complemented).
  key = DT == kF32 ? prefix : (prefix & 0x80000000u ? prefix : prefix | 0x3ffu);
  return true;
}

// The cut of top-k and top-p.
template <int DT>
__device__ Cut find_cut(const Row<DT>& row, const Weights& w, const Params& q, General& s) {
  Cut cut{0u, 0u};
  uint32_t key, above, at_key;
  uint64_t mass;
  uint64_t kept = 0;  // S(n_k)
  bool have = false;
  if (q.k > 0) {
    if (select_key<DT, false>(row, w, (uint64_t)q.k, q.p < 1.0, s, key, above, mass, at_key)) {
      cut.tau = key;
      cut.ties = (uint32_t)q.k - above;
      kept = mass + cut.ties * w(value_of(key));
      have = true;
    }
  }
  if (q.p < 1.0) {
    if (!have) {
      uint64_t sum = 0;
      for (int32_t i = threadIdx.x; i < row.slots(); i += kThreads) {
        float v[Row<DT>::kE];
        row.load(i, v);
#pragma unroll
        for (int j = 0; j < Row<DT>::kE; ++j) sum += w(v[j]);
      }
      workgroup_scan<kWaves, uint64_t>(sum, s.wave64, kept);
    }
    // Tokens whose preceding mass is below p S(n_k): up to the one that reaches it.
    uint64_t want = (uint64_t)ceil(q.p * (double)kept);
    want = want < 1 ? 1 : (want > kept ? kept : want);
    if (select_key<DT, true>(row, w, want, true, s, key, above, mass, at_key)) {
      const uint64_t each = w(value_of(key));
      uint64_t n = each > 0 ? (want - mass + each - 1) / each : at_key;
      cut.tau = key;
      cut.ties = (uint32_t)(n < at_key ? n : at_key);
    }
  }
  return cut;
}


// ------------------------------------------------------------------------------ one row
// A token's place in the order: its key, equal keys by index, larger is earlier.
__device__ __forceinline__ uint64_t place_of(uint32_t key, int32_t index) {
  return ((uint64_t)key << 32) | (uint32_t)~(uint32_t)index;
}
__device__ __forceinline__ uint32_t place_key(uint64_t place) { return (uint32_t)(place >> 32); }
__device__ __forceinline__ int32_t place_index(uint64_t place) { return (int32_t)~(uint32_t)place; }

struct RowShared {
  union {
    General general;
    struct {
      uint64_t place[kList];
      uint64_t bin_mass[kBins];
      uint32_t bin_count[kBins];
    } list;
  };
  SlotQueue queue;
  uint64_t tile_mass[kMaxTiles];
  uint32_t tile_ties[kMaxTiles];
  int32_t visit[kMaxTiles];
  uint64_t wave64[kWaves];
  uint32_t wave32[kWaves];
  float wave_max[kWaves];
  uint64_t value64[4];
  int32_t value32[8];
  int32_t visits, length;
};

// The order of at most kRanked places: four threads per place count the larger ones.  INDEXED: the
// places' numbers by index too, left behind (index_ranks) in the order of the places.
constexpr int kRanked = kThreads / 4;
__device__ __forceinline__ int32_t* index_ranks(uint64_t* s) {
  return reinterpret_cast<int32_t*>(s + 2 * kRanked) + 2 * kRanked;
}
template <bool INDEXED>
__device__ __forceinline__ uint64_t rank_places(int32_t n, uint64_t* s) {
  uint64_t* sorted = s + kRanked;
  int32_t* rank = reinterpret_cast<int32_t*>(s + 2 * kRanked);
  int32_t* by_index = rank + kRanked;
  const int t = threadIdx.x;
  const int e = t % kRanked;
  if (t < 2 * kRanked) rank[t] = 0;
  __syncthreads();
  const int32_t per = (n + 3) / 4;
  const int32_t j0 = t / kRanked * per;
  const int32_t j1 = j0 + per < n ? j0 + per : n;
  if (e < n) {
    const uint64_t mine = s[e];
    int32_t above = 0, before = 0;
#pragma unroll 8
    for (int32_t j = j0; j < j1; ++j) {
      const uint64_t other = s[j];
      above += other > mine ? 1 : 0;
      if (INDEXED) before += (uint32_t)other > (uint32_t)mine ? 1 : 0;
    }
    if (above) atomicAdd(&rank[e], above);
    if (INDEXED && before) atomicAdd(&by_index[e], before);
  }
  __syncthreads();
  if (t < n) {  // (n <= kRanked; places differ)
    sorted[rank[t]] = s[t];
    if (INDEXED) index_ranks(s)[rank[t]] = by_index[t];
  }
  __syncthreads();
  return t < n ? sorted[t] : 0;
}

// What comes before the list of a row: the mass of the tokens before it, and, with top-p alone, the
// whole row's (else the list holds all tokens that count).
struct ListCut {
  uint64_t before;
  uint64_t all_mass;
};

// Sorts the list's n places (at most kRanked) and finds the last kept one.
__device__ __forceinline__ uint64_t cut_short_list(const Weights& w, const Params& q,
                                                   const ListCut& cut, int32_t n, RowShared& s) {
  const int t = threadIdx.x;
  const uint64_t x = rank_places<true>(n, s.list.place);
  const uint64_t weight = t < n ? w(value_of(place_key(x))) : 0;
  __syncthreads();
  uint64_t total;
  const uint64_t before = workgroup_scan<kWaves, uint64_t>(weight, s.wave64, total);
  // S(n_k): of the first k, or everything.
  int32_t last = q.k > 0 && q.k < n ? q.k - 1 : n - 1;
  if (t == 0) {
    s.value32[0] = -1;
    s.value64[2] = 0;
  }
  __syncthreads();
  if (q.p < 1.0) {
    if (t == last) s.value64[0] = before + weight;
    __syncthreads();
    const uint64_t kept = q.k > 0 || cut.all_mass == 0 ? s.value64[0] : cut.all_mass;
    // Tokens whose preceding mass is below p S(n_k).
    uint64_t want = (uint64_t)ceil(q.p * (double)kept);
    want = want < 1 ? 1 : want;
    const uint64_t at = cut.before + before;
    // (One of them: the token that reaches `want`, or the list's last.)
    if (at < want && (at + weight >= want || t == n - 1) && t < n) s.value32[0] = t;
    __syncthreads();
    last = s.value32[0] < last ? s.value32[0] : last;
  }
  __syncthreads();
  if (t == last) s.value64[2] = x;
  if (t < kRanked) s.list.place[t] = x;  // (the sorted list stays in place for the caller)
  __syncthreads();
  return s.value64[2];
}

// The members of one sub-bin of the list, in order: thread i gets the i-th of `count` (more than
// kRanked: they are not ordered).  They are put behind the list's n places.
template <typename SubBin>
__device__ __forceinline__ uint64_t members(int32_t n, int32_t bin, SubBin sub_bin, RowShared& s,
                                            int32_t& count) {
  uint64_t* found = reinterpret_cast<uint64_t*>(&s.queue);
  if (threadIdx.x == 0) s.length = 0;
  __syncthreads();
  for (int32_t i = threadIdx.x; i < n; i += kThreads)
    if (sub_bin(s.list.place[i]) == bin) {
      const int32_t at = atomicAdd(&s.length, 1);
      if (at < kRanked) found[at] = s.list.place[i];
    }
  __syncthreads();
  count = s.length;
  return count <= kRanked ? rank_places<false>(count, found) : 0;
}

// The place, among those of the list within [low, high], at which their number (BY_MASS: their mass)
// reaches `want`; `upto` is their mass up to it.  2048 sub-bins of equal ranges of places between
// the outermost ones, again within the one that is reached, until that can be put in order: equal
// logits differ in their indices, so two turns are the rule.
constexpr int kSub = 2 * kThreads;
static_assert(kSub <= kBins, "the row's bins are reused");
template <bool BY_MASS>
__device__ __forceinline__ uint64_t narrow(const Weights& w, bool weighed, int32_t n, uint64_t low,
                                           uint64_t high, uint64_t want, RowShared& s,
                                           uint64_t& upto) {
  const int t = threadIdx.x;
  uint64_t mass_before = 0;
  for (;;) {
    const auto within = [&](uint64_t place) { return place >= low && place <= high; };
    uint64_t first = 0, last = ~0ull;
    for (int32_t i = t; i < n; i += kThreads) {
      const uint64_t p = s.list.place[i];
      if (within(p)) {
        first = p > first ? p : first;
        last = p < last ? p : last;
      }
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint64_t f = __shfl_xor((unsigned long long)first, d, 64);
      const uint64_t l = __shfl_xor((unsigned long long)last, d, 64);
      first = f > first ? f : first;
      last = l < last ? l : last;
    }
    __syncthreads();
    if (t == 0) {
      s.value64[2] = 0;
      s.value64[3] = ~0ull;
    }
    for (int32_t b = t; b < kSub; b += kThreads) {
      s.list.bin_mass[b] = 0;
      s.list.bin_count[b] = 0;
    }
    __syncthreads();
    if ((t & 63) == 0) {
      atomicMax(reinterpret_cast<unsigned long long*>(&s.value64[2]), (unsigned long long)first);
      atomicMin(reinterpret_cast<unsigned long long*>(&s.value64[3]), (unsigned long long)last);
    }
    __syncthreads();
    high = s.value64[2];
    low = s.value64[3];
    const uint64_t range = high - low;
    const int shift = range < (uint64_t)kSub ? 0 : 64 - 11 - __clzll((long long)range);
    const auto sub_bin = [&](uint64_t place) {
      return within(place) ? (int32_t)((high - place) >> shift) : -1;
    };
    for (int32_t i = t; i < n; i += kThreads) {
      const uint64_t p = s.list.place[i];
      const int32_t b = sub_bin(p);
      if (b < 0) continue;
      atomicAdd(&s.list.bin_count[b], 1u);
      if (weighed)
        atomicAdd(reinterpret_cast<unsigned long long*>(&s.list.bin_mass[b]),
                  (unsigned long long)w(value_of(place_key(p))));
    }
    __syncthreads();
    const uint32_t c0 = s.list.bin_count[2 * t], c1 = s.list.bin_count[2 * t + 1];
    const uint64_t m0 = s.list.bin_mass[2 * t], m1 = s.list.bin_mass[2 * t + 1];
    uint32_t count_all;
    uint64_t mass_all;
    const uint32_t cb = workgroup_scan<kWaves, uint32_t>(c0 + c1, s.wave32, count_all);
    const uint64_t mb = workgroup_scan<kWaves, uint64_t>(m0 + m1, s.wave64, mass_all);
    const uint64_t x0 = BY_MASS ? mb : (uint64_t)cb;
    const uint64_t x1 = x0 + (BY_MASS ? m0 : (uint64_t)c0);
    const uint64_t x2 = x1 + (BY_MASS ? m1 : (uint64_t)c1);
    if (x0 < want && want <= x2) {  // one thread
      const bool second = x1 < want;
      s.value32[6] = second ? 2 * t + 1 : 2 * t;
      s.value64[0] = second ? mb + m0 : mb;
      s.value64[1] = want - (second ? x1 : x0);
    }
    __syncthreads();
    const int32_t bin = s.value32[6];
    mass_before += s.value64[0];
    want = s.value64[1];
    int32_t count;
    const uint64_t place = members(n, bin, sub_bin, s, count);
    if (count > kRanked) {
      low = high - ((uint64_t)bin << shift) - ((1ull << shift) - 1);  // (may wrap below 0: clamped)
      if (low > high) low = 0;
      high -= (uint64_t)bin << shift;
      __syncthreads();
      continue;
    }
    const uint64_t mass = weighed && t < count ? w(value_of(place_key(place))) : 0;
    uint64_t sum;
    const uint64_t at = workgroup_scan<kWaves, uint64_t>(mass, s.wave64, sum);
    if (BY_MASS ? at < want && want <= at + mass : t + 1 == (int32_t)want) {  // one thread
      s.value64[0] = place;
      s.value64[1] = mass_before + at + mass;
    }
    __syncthreads();
    upto = s.value64[1];
    const uint64_t found = s.value64[0];
    __syncthreads();
    return found;
  }
}

// The last kept place of a longer list: its tokens' counts and masses in sub-bins of equal key
// ranges, then the exact order within the two sub-bins where the cuts fall.
__device__ __forceinline__ uint64_t cut_by_bins(const Weights& w, const Params& q,
                                                const ListCut& cut, int32_t n, RowShared& s) {
  uint64_t last;
  const int t = threadIdx.x;
  uint32_t high = 0, low = 0xffffffffu;
  for (int32_t i = t; i < n; i += kThreads) {
    const uint32_t k = place_key(s.list.place[i]);
    high = k > high ? k : high;
    low = k < low ? k : low;
  }
  if (t == 0) {
    s.wave32[0] = 0;
    s.wave32[1] = 0xffffffffu;
  }
  for (int32_t b = t; b < kSub; b += kThreads) {
    s.list.bin_mass[b] = 0;
    s.list.bin_count[b] = 0;
  }
  __syncthreads();
  high = wave_extreme<true>(high);
  low = wave_extreme<false>(low);
  if ((t & 63) == 63) {
    atomicMax(&s.wave32[0], high);
    atomicMin(&s.wave32[1], low);
  }
  __syncthreads();
  high = s.wave32[0];
  const uint32_t range = high - s.wave32[1];
  const int shift = range < (uint32_t)kSub ? 0 : 32 - 11 - __clz((int)range);  // range >> shift < kSub
  const auto sub_bin = [&](uint64_t place) { return (int32_t)((high - place_key(place)) >> shift); };
  // The places that a sub-bin can hold.
  const auto highest = [&](int32_t bin) {
    return ((uint64_t)(high - ((uint32_t)bin << shift)) << 32) | 0xffffffffu;
  };
  const auto lowest = [&](int32_t bin) {
    const uint32_t key = high - ((uint32_t)bin << shift), width = (1u << shift) - 1;
    return (uint64_t)(key > width ? key - width : 0) << 32;
  };
  for (int32_t i = t; i < n; i += kThreads) {
    const uint64_t p = s.list.place[i];
    const int32_t b = sub_bin(p);
    atomicAdd(&s.list.bin_count[b], 1u);
    if (q.p < 1.0)
      atomicAdd(reinterpret_cast<unsigned long long*>(&s.list.bin_mass[b]),
                (unsigned long long)w(value_of(place_key(p))));
  }
  __syncthreads();
  const uint32_t c0 = s.list.bin_count[2 * t], c1 = s.list.bin_count[2 * t + 1];
  const uint64_t m0 = s.list.bin_mass[2 * t], m1 = s.list.bin_mass[2 * t + 1];
  uint32_t count_all;
  uint64_t mass_all = 0, mb = 0;
  const uint32_t cb = workgroup_scan<kWaves, uint32_t>(c0 + c1, s.wave32, count_all);
  if (q.p < 1.0) mb = workgroup_scan<kWaves, uint64_t>(m0 + m1, s.wave64, mass_all);
  const bool top_k = q.k > 0 && q.k <= n;  // (n: the row may have more tokens than its list)
  uint64_t kept = mass_all;
  last = 0;  // (everything)
  int32_t count;
  if (top_k) {
    const uint32_t k = (uint32_t)q.k;
    if (cb < k && k <= cb + c0 + c1) {  // one thread
      const bool second = cb + c0 < k;
      s.value32[6] = second ? 2 * t + 1 : 2 * t;
      s.value32[7] = (int32_t)(k - (second ? cb + c0 : cb));
      s.value64[0] = second ? mb + m0 : mb;
    }
    __syncthreads();
    const int32_t left = s.value32[7];
    kept = s.value64[0];
    const int32_t bin = s.value32[6];
    const uint64_t place = members(n, bin, sub_bin, s, count);
    if (count > kRanked) {
      uint64_t upto;
      last = narrow<false>(w, q.p < 1.0, n, lowest(bin), highest(bin), (uint64_t)left, s, upto);
      kept += upto;
    } else {
      if (t == left - 1) s.value64[1] = place;
      uint64_t sum = 0;
      if (q.p < 1.0)
        workgroup_scan<kWaves, uint64_t>(t < left ? w(value_of(place_key(place))) : 0, s.wave64, sum);
      else
        __syncthreads();
      kept += sum;
      last = s.value64[1];
      __syncthreads();
    }
  } else if (q.k == 0 && cut.all_mass > 0) {
    kept = cut.all_mass;
  }
  if (q.p < 1.0) {
    uint64_t want = (uint64_t)ceil(q.p * (double)kept);
    want = want < 1 ? 1 : want;
    want = want > cut.before ? want - cut.before : 1;
    want = want < mass_all ? want : mass_all;
    if (mb < want && want <= mb + m0 + m1) {  // one thread
      const bool second = mb + m0 < want;
      s.value32[6] = second ? 2 * t + 1 : 2 * t;
      s.value64[0] = second ? mb + m0 : mb;
    }
    __syncthreads();
    const uint64_t before_bin = s.value64[0];
    const int32_t bin = s.value32[6];
    const uint64_t place = members(n, bin, sub_bin, s, count);
    if (count > kRanked) {
      uint64_t upto;
      return narrow<true>(w, true, n, lowest(bin), highest(bin), want - before_bin, s, upto);
    }
    const uint64_t mass = t < count ? w(value_of(place_key(place))) : 0;
    uint64_t sum;
    const uint64_t at = before_bin + workgroup_scan<kWaves, uint64_t>(mass, s.wave64, sum);
    if (at < want && want <= at + mass) s.value64[1] = place;  // one thread
    __syncthreads();
    last = s.value64[1];
    __syncthreads();
  }
  return last;
}

__device__ __forceinline__ uint64_t cut_list(const Weights& w, const Params& q, const ListCut& cut,
                                             int32_t n, RowShared& s) {
  return n <= kRanked ? cut_short_list(w, q, cut, n, s) : cut_by_bins(w, q, cut, n, s);
}

// The first token, in index order, at which the kept weight exceeds `target`, within the slots
// [s0, s1) (one wave).
template <int DT, typename WeightOf>
__device__ __forceinline__ int32_t pick_in_slots(const Row<DT>& row, int32_t s0, int32_t s1,
                                                 uint64_t target, WeightOf weight_of) {
  constexpr int kE = Row<DT>::kE;
  const int lane = threadIdx.x & 63;
  for (int32_t q0 = s0; q0 < s1; q0 += 64) {
    const int32_t q = q0 + lane;
    uint64_t x[kE];
    uint64_t mass = 0;
    float v[kE];
    row.load(q < s1 ? q : s1 - 1, v);
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      x[j] = q < s1 ? weight_of(v[j], row.first(q) + j) : 0;
      mass += x[j];
    }
    const uint64_t incl = wave_scan<uint64_t>(mass);
    const uint64_t before = incl - mass;
    const bool here = before <= target && target < incl;
    const uint64_t any = __ballot(here);
    if (any) {
      int32_t pick = 0;
      uint64_t sum = before;
      bool done = false;
#pragma unroll
      for (int j = 0; j < kE; ++j) {
        sum += x[j];
        if (!done && sum > target) {
          pick = row.first(q) + j;
          done = true;
        }
      }
      return __shfl(pick, __ffsll((unsigned long long)any) - 1, 64);
    }
    target -= __shfl((unsigned long long)incl, 63, 64);
  }
  return 0;  // (not reached: target lies below the sum of [s0, s1))
}

// Rows without a filter: the chunk that holds the target from the chunks' masses, then the token.
template <int DT>
__device__ __forceinline__ void finish_plain(const SampleArgs& a, const Row<DT>& row, int64_t r,
                                             const Params& q, const Chunk& chunk, float top,
                                             RowShared& s) {
  constexpr int kE = Row<DT>::kE;
  constexpr int kChunkSlots = kChunkElements / kE;  // at most kThreads
  const int t = threadIdx.x;
  const double c = 0x1.71547652b82fep+0 / (double)q.t;
  if (t == 0) {
    s.value64[0] = 0;
    s.value32[0] = 0;
  }
  uint64_t mass, total;
  double factor;
  const uint64_t before = scan_chunks(chunk, q, top, s.wave64, mass, factor, total);
  const uint64_t target = scaled(q.u, total);
  if (before <= target && target < before + mass) {  // one thread
    uint64_t left = target - before;
    if (chunk.top < top) left = (uint64_t)((double)left / factor);
    s.value64[0] = left < chunk.mass ? left : chunk.mass - 1;
    s.value32[0] = t;
    s.wave_max[0] = chunk.top;
  }
  __syncthreads();
  // The chunk's slots, one per thread.
  const float cm = s.wave_max[0];
  uint64_t left = s.value64[0];
  const int32_t slot = s.value32[0] * kChunkSlots + t;
  float v[kE];
  uint64_t x[kE];
  uint64_t sum = 0;
  row.load(t < kChunkSlots ? slot : row.slots(), v);  // (past the row: -inf)
  if (FastWeights::fits(q.t, cm)) {
    const FastWeights w(c, q.t, cm, a.frac);
#pragma unroll
    for (int j = 0; j < kE; ++j) x[j] = w(v[j]);
  } else {
    const Weights w{c, (double)cm, cm, a.frac};
#pragma unroll
    for (int j = 0; j < kE; ++j) x[j] = w(v[j]);
  }
#pragma unroll
  for (int j = 0; j < kE; ++j) sum += x[j];
  uint64_t all;
  uint64_t at = workgroup_scan<kWaves, uint64_t>(sum, s.wave64, all);
  if (left >= all) left = all - 1;  // (a sum of several weights may round otherwise than each)
  if (at <= left && left < at + sum) {  // one thread
    int32_t pick = 0;
    bool done = false;
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      at += x[j];
      if (!done && at > left) {
        pick = row.first(slot) + j;
        done = true;
      }
    }
    a.out[r] = pick;
  }
}

// The kept weights of the tiles are in s.tile_mass: picks the tile, then the token in it.
template <int DT, typename WeightOf>
__device__ __forceinline__ void finish_tiles(const SampleArgs& a, const Row<DT>& row, int64_t r,
                                             const Params& q, int32_t tiles, int32_t tile_slots,
                                             RowShared& s, WeightOf weight_of) {
  const int t = threadIdx.x;
  const uint64_t mass = t < tiles ? s.tile_mass[t] : 0;
  if (t == 0) {
    s.value64[0] = 0;
    s.value32[0] = 0;
  }
  uint64_t total;
  const uint64_t before = workgroup_scan<kWaves, uint64_t>(mass, s.wave64, total);
  const uint64_t target = scaled(q.u, total);
  if (before <= target && target < before + mass) {  // one thread
    s.value64[0] = target - before;
    s.value32[0] = t;
  }
  __syncthreads();
  if (t < 64) {
    const int32_t s0 = s.value32[0] * tile_slots;
    const int32_t s1 = s0 + tile_slots < row.slots() ? s0 + tile_slots : row.slots();
    const int32_t pick = pick_in_slots(row, s0, s1, s.value64[0], weight_of);
    if (t == 0) a.out[r] = pick;
  }
}

// Rows whose list is short and holds every kept token: the list in index order.
__device__ __forceinline__ void finish_list(const SampleArgs& a, int64_t r, const Params& q,
                                            const Weights& w, uint64_t least, int32_t n,
                                            uint64_t last_place, RowShared& s) {
  const int t = threadIdx.x;
  uint64_t* place_at = reinterpret_cast<uint64_t*>(&s.queue);
  uint64_t* mass_at = place_at + kRanked;
  if (t < n) {
    const uint64_t mine = s.list.place[t];
    const uint64_t x = mine >= last_place ? w(value_of(place_key(mine))) : 0;
    const int32_t at = index_ranks(s.list.place)[t];
    place_at[at] = mine;
    mass_at[at] = x >= least ? x : 0;
  }
  __syncthreads();
  const uint64_t place = t < n ? place_at[t] : 0;
  const uint64_t mass = t < n ? mass_at[t] : 0;
  uint64_t total;
  const uint64_t before = workgroup_scan<kWaves, uint64_t>(mass, s.wave64, total);
  const uint64_t target = scaled(q.u, total);
  if (before <= target && target < before + mass) a.out[r] = place_index(place);  // one thread
}

// The general path: cut by digits, then the kept weight of every tile, ties counted by index.
// (Not inlined, and given a copy of the arguments: the row kernel keeps its registers.)
template <int DT>
__device__ __attribute__((noinline)) void finish_general(const SampleArgs& a, int64_t r, float top,
                                                         RowShared& s) {
  const Row<DT> row(a, r);
  const Params q = row_params(a, r);
  const Weights w{0x1.71547652b82fep+0 / (double)q.t, (double)top, top, a.frac};
  const uint64_t least = least_weight(q.m, a.frac);
  const int32_t tiles = Tiles<DT>(a).count, tile_slots = Tiles<DT>(a).slots;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  __syncthreads();
  const Cut cut = find_cut(row, w, q, s.general);
  uint64_t tie_weight = cut.ties > 0 ? w(value_of(cut.tau)) : 0;
  if (tie_weight < least) tie_weight = 0;
  for (int32_t t = wave; t < tiles; t += kWaves) {
    uint64_t mass = 0;
    uint32_t ties = 0;
    for (int32_t i = lane; i < tile_slots; i += 64) {
      const int32_t slot = t * tile_slots + i;
      if (slot < row.slots()) {
        float v[Row<DT>::kE];
        row.load(slot, v);
#pragma unroll
        for (int j = 0; j < Row<DT>::kE; ++j) {
          const uint32_t k = key_of(v[j]);
          const uint64_t x = w(v[j]);
          mass += k > cut.tau && x >= least ? x : 0;
          ties += k == cut.tau ? 1u : 0u;
        }
      }
    }
    mass = wave_sum(mass);
    const uint64_t n = wave_sum((uint64_t)ties);
    if (lane == 0) {
      s.tile_mass[t] = mass;
      s.tile_ties[t] = (uint32_t)n;
    }
  }
  __syncthreads();
  // The index of the last kept tie, in the tile where their count is reached.
  const int t = threadIdx.x;
  const uint32_t n = t < tiles ? s.tile_ties[t] : 0;
  uint32_t all_ties;
  const uint32_t before = workgroup_scan<kWaves, uint32_t>(n, s.wave32, all_ties);
  const uint32_t left = cut.ties > before ? cut.ties - before : 0;
  if (t == 0) s.value32[2] = -1;
  __syncthreads();
  if (t < tiles) {
    s.tile_mass[t] += (n < left ? n : left) * tie_weight;
    if (left > 0 && left <= n) {  // one thread
      s.value32[2] = t;
      s.value32[3] = (int32_t)left;
    }
  }
  __syncthreads();
  if (wave == 0 && s.value32[2] >= 0) {
    const int32_t s0 = s.value32[2] * tile_slots;
    const int32_t s1 = s0 + tile_slots < row.slots() ? s0 + tile_slots : row.slots();
    const int32_t at = pick_in_slots(row, s0, s1, (uint64_t)(s.value32[3] - 1), [&](float v, int32_t) {
      return (uint64_t)(key_of(v) == cut.tau ? 1 : 0);
    });
    if (lane == 0) s.value64[1] = place_of(cut.tau, at);
  }
  __syncthreads();
  const uint64_t last = s.value32[2] >= 0 ? s.value64[1] : 0;  // (no cut: every token)
  __syncthreads();
  finish_tiles(a, row, r, q, tiles, tile_slots, s, [&](float v, int32_t i) {
    const uint64_t x = w(v);
    return place_of(key_of(v), i) >= last && x >= least ? x : (uint64_t)0;
  });
}

// The bin in which the cumulative sum of `bins` reaches `want`, and what comes before that bin;
// kBins if the whole does not reach it.
template <typename T, typename Shared>
__device__ __forceinline__ int32_t find_bin(const T* bins, T want, T* s_wave, Shared& s, T& before,
                                            T& total) {
  const int32_t b0 = (int32_t)threadIdx.x * kThreadBins;
  T x[kThreadBins];
  T sum = 0;
#pragma unroll
  for (int j = 0; j < kThreadBins; ++j) {
    x[j] = b0 + j < kBins ? bins[b0 + j] : 0;
    sum += x[j];
  }
  if (threadIdx.x == 0) s.value32[6] = kBins;
  T at = workgroup_scan<kWaves, T>(sum, s_wave, total);
  if (at < want && want <= at + sum) {  // one thread
    int32_t bin = b0;
#pragma unroll
    for (int j = 0; j < kThreadBins; ++j)
      if (at < want && want <= at + x[j]) {
        bin = b0 + j;
        s.value64[0] = at;
        at = want;  // (found)
      } else {
        at += x[j];
      }
    s.value32[6] = bin;
  }
  __syncthreads();
  before = (T)s.value64[0];
  const int32_t bin = s.value32[6];
  __syncthreads();
  return bin;
}

// The bin down to which a list for top-k is gathered, from the tiles' maxima (in `counts`, zero
// before): all bins where every live token fits the list, else for a top-k of at most half the
// tiles that of the k-th largest maximum (at least k tokens, hardly more than twice as many), and
// for a larger one a guess as if the tiles were random samples of the row.  -1: more than three
// tokens per tile, where such a guess is often wrong.
template <int DT, typename Shared>
__device__ __forceinline__ int32_t list_bin(const Tiles<DT>& tiles, int32_t top_k, float tile_max,
                                            float top, uint32_t* counts, Shared& s,
                                            uint32_t* s_wave) {
  if (tile_max > -INFINITY) atomicAdd(&counts[bin_of(tile_max, top)], 1u);
  const uint32_t live = (uint32_t)__syncthreads_count(tile_max > -INFINITY);
  const uint32_t k = (uint32_t)top_k;
  if ((live << tiles.pieces_shift) <= kList / kPieceElements) return kBins - 1;
  if (k > 3 * live) return -1;
  uint32_t rank = k, before, all;
  if (k > live / 2) {
    const float share = 1.0f - expf(-1.3f * (float)k / (float)live - 0.3f);
    rank = (uint32_t)ceilf((float)live * share);
    rank = rank < live ? rank : live;
  }
  return find_bin<uint32_t>(counts, rank, s_wave, s, before, all);
}

// The bin in which a nucleus cut alone falls (`total`: the row's mass).
template <typename Shared>
__device__ __forceinline__ int32_t nucleus_bin(const Params& q, uint64_t total,
                                               const uint64_t* bin_mass, Shared& s,
                                               uint64_t& before, uint64_t& binned) {
  const uint64_t want = (uint64_t)ceil(q.p * (double)total);
  int32_t bin = find_bin<uint64_t>(bin_mass, want < 1 ? 1 : want, s.wave64, s, before, binned);
  // (Roundings: the tokens left out weigh less than (1 - p) Z, but p Z may be all but Z.)
  if (bin == kBins) bin = find_bin<uint64_t>(bin_mass, binned, s.wave64, s, before, binned);
  return bin;
}

// The smallest value of a bin, or a little less (d is rounded, and so is the value from it: both
// errors are relative to d or to top, whichever is larger).
__device__ __forceinline__ float bin_from(int32_t bin, float top) {
  if (bin >= kBins - 1) return -INFINITY;
  if (top == INFINITY) return top;
  const float d = __uint_as_float((uint32_t)(bin + kBinBase) << kBinShift);  // the next bin's least d
  return (float)((double)top - (double)d) - (fabsf(top) + d) * 0x1p-20f;
}

constexpr int kTileCopies = 4;
struct GatherShared {
  union {
    uint64_t bin_mass[kBins];
    Queue queue;  // (once the bin is found)
  };
  uint64_t place[kList];
  uint64_t tile_mass[kTileCopies * kMaxTiles];
  int32_t visit[kMaxTiles];
  uint64_t wave64[kWaves];
  uint32_t wave32[kWaves];
  float wave_max[kWaves];
  uint64_t value64[1];
  int32_t value32[7];
  int32_t visits, length;
};

// One part of the tiles of a row with a nucleus cut alone, its histogram finished: the tokens of
// the bin where the cut falls, and the mass of those before it per tile (four copies, a lane's by
// its number: neighbours share a tile).  For rows with a long top-k, the tokens of all bins down to
// the list's.
template <int DT>
__global__ __launch_bounds__(kThreads) void gather_kernel(SampleArgs a) {
  __shared__ GatherShared s;
  const int64_t r = blockIdx.x / a.parts;
  const int32_t part = (int32_t)(blockIdx.x - r * a.parts);
  const int t = threadIdx.x;
  const Params q = row_params(a, r);
  const bool listed = needs_list(a, q);
  if (!needs_bins(a, q) && !listed) return;
  const Tiles<DT> tiles(a);
  const int32_t per = (tiles.count + a.parts - 1) / a.parts;
  const int32_t tile0 = part * per;
  const int32_t tile1 = tile0 + per < tiles.count ? tile0 + per : tiles.count;
  if (tile0 >= tile1) return;
  for (int32_t b = t; b < kBins; b += kThreads) s.bin_mass[b] = listed ? 0 : a.bin_mass[r * kBins + b];
  const float any_max = listed && t < tiles.count ? tiles.max_of(a, r, t) : -INFINITY;
  const float tile_max = t < tile1 - tile0 ? tiles.max_of(a, r, tile0 + t) : -INFINITY;
  const Chunk chunk = own_chunk(a, r);
  if (t == 0) s.visits = s.length = 0;
#pragma unroll
  for (int c = 0; c < kTileCopies; ++c) s.tile_mass[c * kMaxTiles + t] = 0;
  const float top = row_max(chunk, s.wave_max);  // (with a barrier)
  if (top == -INFINITY) return;
  const Row<DT> row(a, r);
  const Weights w{0x1.71547652b82fep+0 / (double)q.t, (double)top, top, a.frac};
  const uint64_t least = least_weight(q.m, a.frac);
  // The list's bins: [least_bin, bin].
  int32_t bin, least_bin = 0;
  if (listed) {
    bin = list_bin(tiles, q.k, any_max, top, reinterpret_cast<uint32_t*>(s.bin_mass), s, s.wave32);
    if (bin < 0) return;  // (an empty list)
    __syncthreads();
  } else {
    uint64_t mass, total, before, binned;
    double factor;
    scan_chunks(chunk, q, top, s.wave64, mass, factor, total);
    bin = least_bin = nucleus_bin(q, total, s.bin_mass, s, before, binned);
  }
  const float from = bin_from(bin, top);
  if (t < 2) s.queue.length[t] = 0;
  push_visit(tile_max >= from && tile_max > -INFINITY, tile0 + t, s.visit, &s.visits);
  __syncthreads();
  // The mass that a token adds to its tile, or its place in the list.
  const auto take = [&](float v, int32_t index) {
    const int32_t b = bin_of(v, top);
    if (b < least_bin) {
      const uint64_t x = w(v);
      return x >= least ? x : (uint64_t)0;
    }
    if (b <= bin) {
      const int32_t at = atomicAdd(&s.length, 1);
      if (at < kList) s.place[at] = place_of(key_of(v), index);
    }
    return (uint64_t)0;
  };
  const auto add = [&](int32_t tile, uint64_t x) {
    if (x > 0)
      atomicAdd(reinterpret_cast<unsigned long long*>(
                    &s.tile_mass[kTileCopies * (tile - tile0) + (t & (kTileCopies - 1))]),
                (unsigned long long)x);
  };
  read_tiles(row, tiles, s.visit, s.visits, from, s.queue,
             [&](float v, int32_t index) { add(tiles.of(row, index), take(v, index)); },
             [&](const float (&v)[Row<DT>::kE], uint32_t wanted, int32_t slot) {
    uint64_t sum = 0;
#pragma unroll
    for (int j = 0; j < Row<DT>::kE; ++j)
      if (wanted & (1u << j)) sum += take(v[j], row.first(slot) + j);
    add(slot >> tiles.shift, sum);
  });
  __syncthreads();
  if (t < tile1 - tile0) {
    uint64_t m = 0;
#pragma unroll
    for (int c = 0; c < kTileCopies; ++c) m += s.tile_mass[kTileCopies * t + c];
    a.tile_mass[r * kMaxTiles + tile0 + t] = m;
  }
  const int32_t n = s.length;
  if (t == 0) s.value32[6] = n > 0 ? atomicAdd(&a.list_count[r], n) : 0;
  __syncthreads();
  const int32_t at = s.value32[6];
  for (int32_t i = t; i < n && i < kList && at + i < kList; i += kThreads)
    a.list[r * kList + at + i] = s.place[i];
}

// One row.  Rows without a filter need the chunks' masses only.  Otherwise the cut lies in a list
// of tokens that are put in exact order: the one that gather_kernel left, else all tokens down to
// the bin that list_bin gives.  Where that bin was too high or too low, the row's tokens are counted
// per bin, which gives it exactly (32 x 50257 fp32, top-k 1000: 28.6 us; by the digits 88).  Tiles
// whose maximum shows that they hold no token of the list or before it are not read.
//
// Bound by its steps' latency: 32 x 152064 bf16 with all filters 13 us, of those 1.7 for the maximum,
// 1.7 for the bin, 3.2 for reading 50 tiles, 2.6 for the order and cut and 1.5 for the choice; a row
// without a filter 6.
template <int DT>
__global__ __launch_bounds__(kThreads) void row_kernel(SampleArgs a) {
  __shared__ RowShared s;
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x;
  const Row<DT> row(a, r);
  const Params q = row_params(a, r);
  const Tiles<DT> tiles(a);
  const bool filter = q.k > 0 || q.p < 1.0;
  const bool counted = needs_bins(a, q);  // histogram and list are there
  const bool listed = needs_list(a, q);   // a list is
  const float tile_max = t < tiles.count ? tiles.max_of(a, r, t) : -INFINITY;
  const Chunk chunk = own_chunk(a, r);
  s.tile_mass[t] = counted && t < tiles.count ? a.tile_mass[r * kMaxTiles + t] : 0;
  if (filter)
    for (int32_t b = t; b < kBins; b += kThreads) {
      if (counted)
        s.list.bin_mass[b] = a.bin_mass[r * kBins + b];
      else
        s.list.bin_count[b] = 0;
    }
  if (t == 0) {
    s.length = counted || listed ? a.list_count[r] : 0;
    s.visits = s.queue.length = 0;
    s.value32[4] = kMaxTiles;  // first tile with the maximum
  }
  const float top = row_max(chunk, s.wave_max);
  __syncthreads();
  if (top == -INFINITY) {
    if (t == 0) a.out[r] = 0;
    return;
  }
  if (q.greedy) {
    if (tile_max == top) atomicMin(&s.value32[4], t);
    __syncthreads();
    if (t < 64) {
      const int32_t s0 = s.value32[4] << tiles.shift;
      const int32_t s1 = s0 + tiles.slots < row.slots() ? s0 + tiles.slots : row.slots();
      const int32_t pick = pick_in_slots(row, s0, s1, 0, [&](float v, int32_t) {
        return (uint64_t)(v == top ? 1 : 0);
      });
      if (t == 0) a.out[r] = pick;
    }
    return;
  }
  if (!filter && !(q.m > 0.0)) {
    finish_plain(a, row, r, q, chunk, top, s);
    return;
  }
  const Weights w{0x1.71547652b82fep+0 / (double)q.t, (double)top, top, a.frac};
  const uint64_t least = least_weight(q.m, a.frac);
  ListCut cut{0, 0};
  bool confirmed = true;
  if (counted) {
    uint64_t mass, total, binned;
    double factor;
    scan_chunks(chunk, q, top, s.wave64, mass, factor, total);
    nucleus_bin(q, total, s.list.bin_mass, s, cut.before, binned);
    cut.all_mass = total < binned ? binned : total;
    const int32_t n = s.length < kList ? s.length : kList;
    for (int32_t i = t; i < n; i += kThreads) s.list.place[i] = a.list[r * kList + i];
  } else {
    int32_t last = kBins - 1;
    bool counting = false;
    bool done = false;
    if (listed) {
      const int32_t n = s.length;
      done = n >= q.k && n <= kList;
      counting = !done;
      for (int32_t i = t; i < n && done; i += kThreads) s.list.place[i] = a.list[r * kList + i];
      __syncthreads();
      if (t == 0 && !done) s.length = 0;
    } else if (filter) {
      confirmed = q.k <= kList;  // (no list could hold it)
      if (confirmed) last = list_bin(tiles, q.k > 0 ? q.k : kList, tile_max, top, s.list.bin_count, s, s.wave32);
      counting = last < 0;
      last = counting ? kBins - 1 : last;
    } else {
      // min-p alone: w >= m is M - v <= -T ln m (and a little more, for the roundings).
      const float d = (-logf((float)q.m) * (1.0f + 0x1p-18f) + 0x1p-18f) * q.t;
      last = bin_of((float)((double)top - (double)d) - (fabsf(top) + d) * 0x1p-20f, top);
    }
    // A guess that was too high or too low is followed by a count of the row's tokens per bin, and
    // that by the list down to the bin of the k-th.
    for (int turn = counting ? 1 : 0; confirmed && !done; ++turn) {
      if (counting) {
        __syncthreads();
        for (int32_t b = t; b < kBins; b += kThreads) s.list.bin_count[b] = 0;
      }
      const float from = bin_from(last, top);
      push_visit(tile_max >= from && tile_max > -INFINITY, t, s.visit, &s.visits);
      __syncthreads();
      // (min-p alone lists nothing: its tokens' weights go to their tiles.)
      read_tiles_sparse(row, tiles, s.visit, s.visits, from, s.queue, [&](float v, int32_t index) {
        if (filter) {
          const int32_t b = bin_of(v, top);
          if (b > last) return;
          if (counting) {
            atomicAdd(&s.list.bin_count[b], 1u);
            return;
          }
          const int32_t at = atomicAdd(&s.length, 1);
          if (at < kList) s.list.place[at] = place_of(key_of(v), index);
        } else {
          const uint64_t x = w(v);
          if (x >= least && x > 0)
            atomicAdd(reinterpret_cast<unsigned long long*>(&s.tile_mass[tiles.of(row, index)]),
                      (unsigned long long)x);
        }
      });
      if (!filter) break;
      if (counting) {
        uint32_t before, all;
        const int32_t bin = find_bin<uint32_t>(s.list.bin_count, (uint32_t)q.k, s.wave32, s, before, all);
        last = bin < last ? bin : last;  // (kBins: fewer than k tokens in all)
        counting = false;
      } else {
        // The list holds the first k tokens, or every live one.
        const int32_t n = s.length;
        const bool enough = last == kBins - 1 || n >= q.k;
        if (n <= kList && enough) break;
        confirmed = turn == 0 && q.k > 0;
        counting = true;
        if (!enough) last = kBins - 1;
      }
      __syncthreads();
      if (t == 0) s.length = s.visits = s.queue.length = 0;
      __syncthreads();
    }
  }
  __syncthreads();
  uint64_t last_place = 0;
  if (filter) {
    const int32_t n = s.length;
    if (n > kList || !confirmed) {
      const SampleArgs copy = a;
      finish_general<DT>(copy, r, top, s);
      return;
    }
    last_place = cut_list(w, q, cut, n, s);
    if (!counted && n <= kRanked) {
      finish_list(a, r, q, w, least, n, last_place, s);
      return;
    }
    for (int32_t i = t; i < n; i += kThreads) {
      const uint64_t p = s.list.place[i];
      const uint64_t x = w(value_of(place_key(p)));
      if (p >= last_place && x >= least)
        atomicAdd(reinterpret_cast<unsigned long long*>(
                      &s.tile_mass[tiles.of(row, place_index(p))]),
                  (unsigned long long)x);
    }
    __syncthreads();
  }
  finish_tiles(a, row, r, q, tiles.count, tiles.slots, s, [&](float v, int32_t i) {
    const uint64_t x = w(v);
    return v > -INFINITY && place_of(key_of(v), i) >= last_place && x >= least ? x : (uint64_t)0;
  });
}

int frac_bits(int64_t vocab) {
  int b = 0;
  while (((int64_t)1 << b) < vocab) ++b;
  return 62 - b < 47 ? 62 - b : 47;  // (16 weights stay below 2^52)
}

}  // namespace
}  // namespace int8kv_serving

using namespace int8kv_serving;

namespace {

// Chunks of a row of any alignment (a slot more at either end than its vectors).
int64_t chunks_of(int64_t vocab, bool f32) {
  const int64_t e = f32 ? 4 : 8;
  return (vocab / e + 2 + kChunkElements / e - 1) / (kChunkElements / e);
}

int64_t align16(int64_t n) { return (n + 15) / 16 * 16; }

// Workspace: masses and lists (64 bits), then counts and maxima.
int64_t workspace_of(int64_t rows, int64_t chunks, SampleArgs* a, char* base) {
  const int64_t pieces = chunks * (kChunkElements / kPieceElements);
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at = align16(at + bytes);
    return here;
  };
  const int64_t chunk_mass = take(rows * chunks * 8), bin_mass = take(rows * kBins * 8),
                tile_mass = take(rows * kMaxTiles * 8), list = take(rows * kList * 8),
                list_count = take(rows * 4), chunk_max = take(rows * chunks * 4),
                piece_max = take(rows * pieces * 4);
  if (a) {
    a->chunks = (int32_t)chunks;
    a->pieces = (int32_t)pieces;
    a->chunk_mass = reinterpret_cast<uint64_t*>(base + chunk_mass);
    a->bin_mass = reinterpret_cast<uint64_t*>(base + bin_mass);
    a->tile_mass = reinterpret_cast<uint64_t*>(base + tile_mass);
    a->list = reinterpret_cast<uint64_t*>(base + list);
    a->list_count = reinterpret_cast<int32_t*>(base + list_count);
    a->chunk_max = reinterpret_cast<float*>(base + chunk_max);
    a->piece_max = reinterpret_cast<float*>(base + piece_max);
  }
  return at;
}

template <int DT>
void launch_sample(const SampleArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(chunk_kernel<DT>, dim3((unsigned)(a.rows * a.runs)), dim3(kChunkThreads), 0, s,
                     a);
  if (a.parts > 0) {
    const dim3 grid((unsigned)(a.rows * a.parts));
    hipLaunchKernelGGL(bins_kernel<DT>, grid, dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL(gather_kernel<DT>, grid, dim3(kThreads), 0, s, a);
  }
  hipLaunchKernelGGL(row_kernel<DT>, dim3((unsigned)a.rows), dim3(kThreads), 0, s, a);
}

// How the passes of a.rows rows are cut.
void plan_launches(SampleArgs& a) {
  // Runs of chunks long enough for the loads of one to hide behind the weights of another, while
  // there are enough of them to fill the compute units.
  const int64_t per_unit = a.rows * a.chunks / 2048;
  a.run_chunks = (int32_t)(per_unit < 1 ? 1 : (per_unit < 8 ? per_unit : 8));
  a.runs = (a.chunks + a.run_chunks - 1) / a.run_chunks;
  // The histogram pass and the gathering behind it run where some row may have a nucleus cut alone
  // and more tokens than its list holds.  A compute unit takes one of their workgroups.  Without a
  // top-k in the call every row may be such a one: one turn of the units (120 rows of 50257: 13 and
  // 11 us with 2 parts, 16 and 18 with 4, 18 and 15 with 1).  With one, rows of other settings leave
  // at once: up to two turns (61 rows of mixed settings, 152064: 11 and 13 us with 8 parts, 16 and 16
  // with 4, 9 and 16 with 12).
  a.parts = 0;
  if (a.top_p && a.pieces > kList / kPieceElements) {
    const int64_t most = (a.vocab + 4 * kThreads - 1) / (4 * kThreads);
    const int64_t turns = a.top_k && a.rows <= 128 ? 512 : 256;
    const int64_t want = turns / a.rows < 1 ? 1 : turns / a.rows;
    a.parts = (int32_t)(want < most ? want : most);
  }
}

}  // namespace

extern "C" size_t int8kv_sample_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows < 0 || rows > kMaxRows || vocab < 1 || vocab > kMaxVocab) return 0;
  const int64_t chunks = chunks_of(vocab, true);  // at least those of the 16-bit types
  const int64_t group = rows < kGroupRows ? rows : kGroupRows;
  return (size_t)workspace_of(group > 0 ? group : 1, chunks, nullptr, nullptr);
}

extern "C" int int8kv_sample_rows(const void* logits, int logits_dtype, int64_t rows, int64_t vocab,
                                  int64_t row_stride, const float* uniforms,
                                  const float* temperature, const int32_t* top_k,
                                  const float* top_p, const float* min_p, int64_t* out,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  if (rows != 0 && (!logits || !uniforms || !out)) return INT8KV_E_NULL;
  if (logits_dtype != INT8KV_F32 && logits_dtype != INT8KV_F16 && logits_dtype != INT8KV_BF16)
    return INT8KV_E_DTYPE;
  if (rows < 0 || rows > kMaxRows || vocab < 1 || vocab > kMaxVocab) return INT8KV_E_SHAPE;
  const uintptr_t size = logits_dtype == INT8KV_F32 ? 4 : 2;
  if (row_stride < vocab || reinterpret_cast<uintptr_t>(logits) % size) return INT8KV_E_STRIDE;
  if (rows == 0) return INT8KV_OK;
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 ||
      workspace_bytes < int8kv_sample_workspace_bytes(rows, vocab))
    return INT8KV_E_WORKSPACE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  for (int64_t r0 = 0; r0 < rows; r0 += kGroupRows) {
    const int64_t n = rows - r0 < kGroupRows ? rows - r0 : kGroupRows;
    SampleArgs a;
    a.logits = static_cast<const char*>(logits) + r0 * row_stride * (int64_t)size;
    a.rows = n;
    a.row_stride = row_stride;
    a.vocab = (int32_t)vocab;
    a.frac = frac_bits(vocab);
    a.u = uniforms + r0;
    a.temperature = temperature ? temperature + r0 : nullptr;
    a.top_k = top_k ? top_k + r0 : nullptr;
    a.top_p = top_p ? top_p + r0 : nullptr;
    a.min_p = min_p ? min_p + r0 : nullptr;
    a.out = out + r0;
    workspace_of(n, chunks_of(vocab, logits_dtype == INT8KV_F32), &a, static_cast<char*>(workspace));
    plan_launches(a);
    if (logits_dtype == INT8KV_F32)
      launch_sample<kF32>(a, s);
    else if (logits_dtype == INT8KV_BF16)
      launch_sample<kBF16>(a, s);
    else
      launch_sample<kF16>(a, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return INT8KV_OK;
}
