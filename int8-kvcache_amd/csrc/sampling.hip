// Sampling: one token per row of logits, with temperature, top-k, top-p and min-p, from a given
// uniform number per row.
//
// A token's weight is w = exp((v - M) / T), M the row's maximum.  The tokens in order of falling
// logit (equal ones by index) make top-k, top-p and min-p each a prefix of one order, so what is
// kept is described by a cut: every token above a key tau, and the first `ties` tokens (by index)
// at tau.  The token is then the inverse of the cumulative kept weight in index order.
//
// Which token comes out depends on sums over the whole vocabulary, next to borders that a
// rounding could move, so weights are exact to about 2^-44: 2^y by a polynomial in 64 bits (the
// vector rate of 64-bit multiply-adds is that of 32-bit ones), rounded to a fixed-point integer.
// Integer sums do not depend on their order: chunking and atomics cannot change a result.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "int8kv_common.h"
#include "serving_ops.h"

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
  int32_t chunks;   // of the first pass, per row
  int32_t pieces;   // kChunkElements / kPieceElements of each chunk
  int32_t parts;    // workgroups per row of the histogram pass (0: it does not run)
  float* chunk_max;      // [rows][chunks]
  uint64_t* chunk_mass;  // [rows][chunks] (rows without a filter), in units of the chunk's own maximum
  float* piece_max;      // [rows][pieces]
  uint64_t* bin_mass;    // [rows][kBins]
  uint32_t* bin_count;   // [rows][kBins]
};

// ------------------------------------------------------------------------------ row access
// A row as slots: slot 0 the elements before the first 16-byte boundary, slots 1 .. whole 16-byte
// vectors, the last slot what is left.  Elements a slot lacks read as -inf (weight 0).
template <int DT>
struct Row {
  static constexpr int kE = DT == kF32 ? 4 : 8;  // elements of a vector
  const char* p;
  int32_t vocab, head, vectors;

  __device__ __forceinline__ Row(const SampleArgs& a, int64_t r) {
    constexpr int size = DT == kF32 ? 4 : 2;
    p = static_cast<const char*>(a.logits) + r * a.row_stride * size;
    vocab = a.vocab;
    const int32_t off = (int32_t)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / size;
    head = off < vocab ? off : vocab;
    vectors = (vocab - head) / kE;
  }
  __device__ __forceinline__ int32_t slots() const { return vectors + 2; }
  // Index of a slot's first element.
  __device__ __forceinline__ int32_t first(int32_t s) const {
    return s == 0 ? 0 : head + (s - 1) * kE;
  }
  __device__ __forceinline__ float element(int32_t i) const {
    if constexpr (DT == kF32)
      return reinterpret_cast<const float*>(p)[i];
    else if constexpr (DT == kBF16)
      return __uint_as_float((uint32_t) reinterpret_cast<const uint16_t*>(p)[i] << 16);
    else
      return (float)reinterpret_cast<const _Float16*>(p)[i];
  }
  // The slot's values, NaN as -inf.
  __device__ __forceinline__ void load(int32_t s, float (&v)[kE]) const {
    if (s >= 1 && s <= vectors) {
      const char* q = p + (int64_t)head * (DT == kF32 ? 4 : 2) + 16 * (int64_t)(s - 1);
      if constexpr (DT == kF32) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(q);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = x[j];
      } else {
        int8kv::load8_f32<DT>(q, v);
      }
    } else {
      const int32_t i0 = first(s);
      const int32_t n = s == 0 ? head : (s == vectors + 1 ? vocab - i0 : 0);
#pragma unroll
      for (int j = 0; j < kE; ++j) v[j] = j < n ? element(i0 + j) : -INFINITY;
    }
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
// w(v) = 2^((v - M) log2(e) / T) in units of 2^-frac, rounded to even.  With y = n + f, |f| <= 1/2,
// 2^f by a polynomial (interpolation at Chebyshev nodes, relative error 4e-14, exactly 1 at f = 0)
// and the rounding by adding 2^52: the integer is left in the low bits.
struct Weights {
  double c;    // log2(e) / T
  double top;  // M
  float topf;
  int32_t frac;

  __device__ __forceinline__ uint64_t operator()(float v) const {
    constexpr double kMagic = 0x1.8p52;
    double y = ((double)v - top) * c;
    y = v == topf ? 0.0 : fmax(y, -100.0);  // (NaN, from infinities: -100, weight 0)
    const double t = y + kMagic;
    const double f = y - (t - kMagic);
    const int32_t n = (int32_t)__double_as_longlong(t);
    double p = 0x1.b63880fccd758p-24;
    p = fma(p, f, 0x1.63d13634289c7p-20);
    p = fma(p, f, 0x1.ffcb951552801p-17);
    p = fma(p, f, 0x1.4308ac85ac77dp-13);
    p = fma(p, f, 0x1.5d87fe86fea1cp-10);
    p = fma(p, f, 0x1.3b2ab7181b747p-7);
    p = fma(p, f, 0x1.c6b08d7047e51p-5);
    p = fma(p, f, 0x1.ebfbdff823cedp-3);
    p = fma(p, f, 0x1.62e42fefa39efp-1);
    p = fma(p, f, 1.0);
    const double scale = __longlong_as_double((int64_t)(1023 + frac + n) << 52);
    const double r = fma(p, scale, 0x1p52);
    return (uint64_t)__double_as_longlong(r) - 0x4330000000000000ull;
  }
};

// ------------------------------------------------------------------------- workgroup sums
__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor((unsigned long long)v, d, 64);
  return v;
}
// Inclusive prefix sum over the wave.
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T up = __shfl_up(v, d, 64);
    if (lane >= d) v += up;
  }
  return v;
}
// Exclusive prefix sum over the workgroup; s_wave: kWaves values.
template <typename T>
__device__ __forceinline__ T workgroup_scan(T v, T* s_wave, T& total) {
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const T inc = wave_scan(v);
  __syncthreads();
  if (lane == 63) s_wave[wave] = inc;
  __syncthreads();
  T before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) before += s_wave[w];
    total += s_wave[w];
  }
  return before + inc - v;
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
// Bins of d = M - v, 64 to an octave from 2^-10 to 256, one below and one above: fine where a
// cut can lie whatever the temperature, and monotone in v (the subtraction rounds monotonically).
constexpr int kBinShift = 17;                        // 6 mantissa bits
constexpr int kBinBase = (127 - 10) << 6;
constexpr int kOctaveBins = 18 * 64;
constexpr int kBins = kOctaveBins + 2;
__device__ __forceinline__ int32_t bin_of(float v, float top) {
  const float d = v == top ? 0.0f : top - v;
  const int32_t b = (int32_t)(__float_as_uint(d) >> kBinShift) - kBinBase + 1;
  return b < 0 ? 0 : (b < kBins ? b : kBins - 1);
}

// Rows whose top-k cut is found from the piece maxima alone: at least half of the pieces lie
// below the k-th largest maximum.
__device__ __forceinline__ bool by_pieces(const SampleArgs& a, const Params& q) {
  return q.k > 0 && q.k <= a.pieces / 2;
}
__device__ __forceinline__ bool needs_bins(const SampleArgs& a, const Params& q) {
  return !q.greedy && (q.k > 0 || q.p < 1.0) && !by_pieces(a, q);
}

template <int DT>
__device__ __forceinline__ void add_to_bins(const Row<DT>& row, const Weights& w, const Params& q,
                                            int32_t s0, int32_t s1, uint64_t* mass,
                                            uint32_t* count) {
  for (int32_t i = s0 + (int32_t)threadIdx.x; i < s1; i += kThreads) {
    float v[Row<DT>::kE];
    row.load(i, v);
#pragma unroll
    for (int j = 0; j < Row<DT>::kE; ++j)
      if (v[j] > -INFINITY) {
        const int32_t b = bin_of(v[j], w.topf);
        if (q.k > 0) atomicAdd(&count[b], 1u);
        if (q.p < 1.0)
          atomicAdd(reinterpret_cast<unsigned long long*>(&mass[b]), (unsigned long long)w(v[j]));
      }
  }
}

__device__ __forceinline__ float wave_max(float m) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
  return m;
}

// ------------------------------------------------------------------------------ first pass
// One chunk of one row, held in registers: the maxima of its pieces and its own, and, for rows
// without a filter, the sum of its weights in units of its own maximum (so that the data is read
// once).  Clears the row's bins where they will be used.
template <int DT>
__global__ __launch_bounds__(kChunkThreads) void chunk_kernel(SampleArgs a) {
  constexpr int kE = Row<DT>::kE;
  constexpr int kSteps = kChunkElements / kChunkThreads / kE;
  constexpr int kPieceSlots = kPieceElements / kE;  // 32 or 64: half a wave's slots, or a wave's
  __shared__ float s_max[kChunkThreads / 64];
  __shared__ uint64_t s_sum[kChunkThreads / 64];
  const int64_t r = blockIdx.x / a.chunks;
  const int32_t c = (int32_t)(blockIdx.x - r * a.chunks);
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const Row<DT> row(a, r);
  const int32_t slot0 = c * (kSteps * kChunkThreads) + (int32_t)threadIdx.x;
  float v[kSteps][kE];
#pragma unroll
  for (int j = 0; j < kSteps; ++j) row.load(slot0 + j * kChunkThreads, v[j]);
  const Params q = row_params(a, r);
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    float m = v[j][0];
#pragma unroll
    for (int e = 1; e < kE; ++e) m = fmaxf(m, v[j][e]);
#pragma unroll
    for (int d = kPieceSlots / 2; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    if (lane % kPieceSlots == 0)
      a.piece_max[r * a.pieces + (slot0 + j * kChunkThreads) / kPieceSlots] = m;
    top = fmaxf(top, m);
  }
  top = wave_max(top);
  if (lane == 0) s_max[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kChunkThreads / 64; ++w) top = fmaxf(top, s_max[w]);
  if (threadIdx.x == 0) a.chunk_max[r * a.chunks + c] = top;
  if (a.parts > 0 && needs_bins(a, q)) {
    for (int32_t b = c * kChunkThreads + (int32_t)threadIdx.x; b < kBins; b += a.chunks * kChunkThreads) {
      a.bin_mass[r * kBins + b] = 0;
      a.bin_count[r * kBins + b] = 0;
    }
  }
  if (q.greedy || q.k > 0 || q.p < 1.0 || q.m > 0.0) return;
  uint64_t sum = 0;
  if (top > -INFINITY) {
    const Weights w{0x1.71547652b82fep+0 / (double)q.t, (double)top, top, a.frac};
#pragma unroll
    for (int j = 0; j < kSteps; ++j)
#pragma unroll
      for (int e = 0; e < kE; ++e) sum += w(v[j][e]);
  }
  sum = wave_sum(sum);
  if (lane == 0) s_sum[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < kChunkThreads / 64; ++w) sum += s_sum[w];
    a.chunk_mass[r * a.chunks + c] = sum;
  }
}

// The row's maximum from its chunks' (one value per thread; s_max: kWaves).
__device__ __forceinline__ float row_max(const SampleArgs& a, int64_t r, float* s_max) {
  float m = (int32_t)threadIdx.x < a.chunks ? a.chunk_max[r * a.chunks + threadIdx.x] : -INFINITY;
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) m = fmaxf(m, s_max[w]);
  return m;
}

// ------------------------------------------------------------------------ histogram pass
// One part of one row: its tokens and weights per bin, added to the row's (integers: in any order).
template <int DT>
__global__ __launch_bounds__(kThreads) void bins_kernel(SampleArgs a) {
  __shared__ uint64_t s_mass[kBins];
  __shared__ uint32_t s_count[kBins];
  __shared__ float s_max[kWaves];
  const int64_t r = blockIdx.x / a.parts;
  const int32_t part = (int32_t)(blockIdx.x - r * a.parts);
  const Params q = row_params(a, r);
  if (!needs_bins(a, q)) return;
  const float top = row_max(a, r, s_max);
  if (top == -INFINITY) return;
  for (int32_t b = threadIdx.x; b < kBins; b += kThreads) {
    s_mass[b] = 0;
    s_count[b] = 0;
  }
  __syncthreads();
  const Row<DT> row(a, r);
  const Weights w{0x1.71547652b82fep+0 / (double)q.t, (double)top, top, a.frac};
  const int32_t per = (row.slots() + a.parts - 1) / a.parts;
  const int32_t s1 = (part + 1) * per < row.slots() ? (part + 1) * per : row.slots();
  add_to_bins(row, w, q, part * per, s1, s_mass, s_count);
  __syncthreads();
  for (int32_t b = threadIdx.x; b < kBins; b += kThreads) {
    if (s_mass[b])
      atomicAdd(reinterpret_cast<unsigned long long*>(&a.bin_mass[r * kBins + b]),
                (unsigned long long)s_mass[b]);
    if (s_count[b]) atomicAdd(&a.bin_count[r * kBins + b], s_count[b]);
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
    const uint32_t cb = workgroup_scan<uint32_t>(c0 + c1, s.wave32, ctot);
    const uint64_t mb = workgroup_scan<uint64_t>(m0 + m1, s.wave64, mtot);
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
      workgroup_scan<uint64_t>(sum, s.wave64, kept);
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
  uint64_t tile_mass[kMaxTiles];
  float tile_max[kMaxTiles];
  uint32_t tile_ties[kMaxTiles];
  uint64_t wave64[kWaves];
  uint32_t wave32[kWaves];
  float wave_max[kWaves];
  uint64_t value64[4];
  int32_t value32[8];
};

// Sorts N = kThreads * P places, largest first: value e of thread t is number t P + e.  Partners
// within a thread by registers, within a wave by lane exchange, else through LDS.
template <int P>
__device__ __forceinline__ void sort_places(uint64_t (&x)[P], uint64_t* s) {
  constexpr int kN = kThreads * P;
  const int t = threadIdx.x;
  for (int size = 2; size <= kN; size <<= 1) {
    for (int step = size >> 1; step >= 1; step >>= 1) {
      if (step >= 64 * P) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < P; ++e) s[t * P + e] = x[e];
        __syncthreads();
      }
      if (step >= P) {
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const int i = t * P + e;
          const uint64_t y = step >= 64 * P
                                 ? s[i ^ step]
                                 : (uint64_t)__shfl_xor((unsigned long long)x[e], step / P, 64);
          const bool larger = ((i & size) == 0) == ((i & step) == 0);
          x[e] = (y > x[e]) == larger ? y : x[e];
        }
      } else if constexpr (P > 1) {
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const int i = t * P + e;
          const int o = e ^ step;
          if (o > e) {  // (step is 1 or 2: resolved when unrolled over both)
            const bool down = (i & size) == 0;
            uint64_t lo = x[0], hi = x[0];
#pragma unroll
            for (int z = 0; z < P; ++z) {
              lo = z == e ? x[z] : lo;
              hi = z == o ? x[z] : hi;
            }
            const bool swap = (hi > lo) == down && hi != lo;
#pragma unroll
            for (int z = 0; z < P; ++z) x[z] = swap ? (z == e ? hi : (z == o ? lo : x[z])) : x[z];
          }
        }
      }
    }
  }
}

// What the exact order of the list means for the row (cut_list): everything before the list
// (base tokens and mass per group) and where its two groups lie.
struct ListCut {
  bool top_k, top_p;
  uint32_t k_left;     // tokens that top-k still keeps of its group
  int32_t k_group;     // list position where top-k's group begins
  uint64_t k_mass;     // mass before top-k's group
  uint64_t p_mass;     // mass before the list's first token
  uint64_t all_mass;   // the whole row's (top-p without top-k) ...
  bool whole;          // ... or the list's, if it holds every live token
};

// Sorts the list's n places and finds the last kept one.
template <int P>
__device__ uint64_t cut_list(const Weights& w, const Params& q, const ListCut& cut, int32_t n,
                             RowShared& s) {
  uint64_t x[P];
  const int t = threadIdx.x;
#pragma unroll
  for (int e = 0; e < P; ++e) x[e] = t * P + e < n ? s.list.place[t * P + e] : 0;
  sort_places<P>(x, s.list.place);
  uint64_t weight[P];
  uint64_t sum = 0;
#pragma unroll
  for (int e = 0; e < P; ++e) {
    weight[e] = t * P + e < n ? w(value_of(place_key(x[e]))) : 0;
    sum += weight[e];
  }
  __syncthreads();
  uint64_t total;
  const uint64_t before = workgroup_scan<uint64_t>(sum, s.wave64, total);
  // S(n_k): the mass before top-k's group and of the tokens it keeps of it.  Position of the last.
  const int32_t k_last = cut.top_k ? cut.k_group + (int32_t)cut.k_left - 1 : n - 1;
  if (t == 0) {
    s.value64[0] = 0;
    s.value64[1] = 0;
    s.value32[0] = -1;
  }
  __syncthreads();
  uint64_t at = before;
#pragma unroll
  for (int e = 0; e < P; ++e) {
    const int32_t i = t * P + e;
    if (i == cut.k_group) s.value64[0] = at;
    at += weight[e];
    if (i == k_last) s.value64[1] = at;
  }
  __syncthreads();
  int32_t last = k_last;
  if (cut.top_p) {
    const uint64_t kept = cut.top_k   ? cut.k_mass + (s.value64[1] - s.value64[0])
                          : cut.whole ? total
                                      : cut.all_mass;
    // Tokens whose preceding mass is below p S(n_k).
    uint64_t want = (uint64_t)ceil(q.p * (double)kept);
    want = want < 1 ? 1 : want;
    at = cut.p_mass + before;
    int32_t mine = -1;
#pragma unroll
    for (int e = 0; e < P; ++e) {
      if (t * P + e < n && at < want) mine = t * P + e;
      at += weight[e];
    }
    if (mine >= 0) atomicMax(&s.value32[0], mine);
    __syncthreads();
    last = s.value32[0] < last ? s.value32[0] : last;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < P; ++e)
    if (t * P + e == last) s.value64[2] = x[e];
  // (The sorted list stays in place for the caller.)
#pragma unroll
  for (int e = 0; e < P; ++e) s.list.place[t * P + e] = x[e];
  __syncthreads();
  return s.value64[2];
}

__device__ __forceinline__ uint64_t cut_list_any(const Weights& w, const Params& q,
                                                 const ListCut& cut, int32_t n, RowShared& s) {
  if (n <= kThreads) return cut_list<1>(w, q, cut, n, s);
  if (n <= 2 * kThreads) return cut_list<2>(w, q, cut, n, s);
  return cut_list<4>(w, q, cut, n, s);
}

// Adds this lane's tokens to the list (those with `in`); more than kList of them only count.
__device__ __forceinline__ void append(bool in, uint64_t place, RowShared& s) {
  const uint64_t mask = __ballot(in);
  if (mask == 0) return;
  const int lane = threadIdx.x & 63;
  const int leader = __ffsll((unsigned long long)mask) - 1;
  int32_t at = 0;
  if (lane == leader) at = atomicAdd(&s.value32[1], (int32_t)__popcll(mask));
  at = __shfl(at, leader, 64) + (int32_t)__popcll(mask & (((uint64_t)1 << lane) - 1));
  if (in && at < kList) s.list.place[at] = place;
}

// The k-th largest of the tiles' maxima (k <= tiles).
__device__ float kth_tile_max(const SampleArgs& a, int32_t k, int32_t tiles, RowShared& s) {
  uint64_t x[1];
  x[0] = (int32_t)threadIdx.x < tiles ? place_of(key_of(s.tile_max[threadIdx.x]), threadIdx.x) : 0;
  sort_places<1>(x, s.list.place);
  if ((int32_t)threadIdx.x == k - 1) s.value64[3] = x[0];
  __syncthreads();
  const float v = value_of(place_key(s.value64[3]));
  __syncthreads();
  return v;
}

template <int DT>
__device__ __forceinline__ int32_t tile_of(const Row<DT>& row, int32_t index, int32_t tile_slots) {
  return (index < row.head ? 0 : 1 + (index - row.head) / Row<DT>::kE) / tile_slots;
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
    const uint64_t incl = wave_scan<unsigned long long>(mass);
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
__device__ void finish_plain(const SampleArgs& a, const Row<DT>& row, int64_t r, const Params& q,
                             float top, RowShared& s) {
  constexpr int kChunkSlots = kChunkElements / Row<DT>::kE;
  const int t = threadIdx.x;
  const double c = 0x1.71547652b82fep+0 / (double)q.t;
  uint64_t mass = 0, own = 0;
  double factor = 1.0;
  float m = -INFINITY;
  if (t < a.chunks) {
    m = a.chunk_max[r * a.chunks + t];
    own = a.chunk_mass[r * a.chunks + t];
    mass = own;
    if (m < top) {
      factor = exp2(fmax(((double)m - (double)top) * c, -200.0));
      mass = (uint64_t)rint((double)own * factor);
    }
  }
  if (t == 0) {
    s.value64[0] = 0;
    s.value32[0] = 0;
  }
  uint64_t total;
  const uint64_t before = workgroup_scan<uint64_t>(mass, s.wave64, total);
  const uint64_t target = scaled(q.u, total);
  if (before <= target && target < before + mass) {  // one thread
    uint64_t left = target - before;
    if (m < top) left = (uint64_t)((double)left / factor);
    s.value64[0] = left < own ? left : own - 1;
    s.value32[0] = t;
    s.wave_max[0] = m;
  }
  __syncthreads();
  if (t < 64) {
    const float cm = s.wave_max[0];
    const Weights w{c, (double)cm, cm, a.frac};
    const int32_t s0 = s.value32[0] * kChunkSlots;
    const int32_t s1 = s0 + kChunkSlots < row.slots() ? s0 + kChunkSlots : row.slots();
    const int32_t pick =
        pick_in_slots(row, s0, s1, s.value64[0], [&](float v, int32_t) { return w(v); });
    if (t == 0) a.out[r] = pick;
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
  const uint64_t before = workgroup_scan<uint64_t>(mass, s.wave64, total);
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

// The general path: cut by digits, then the kept weight of every tile, ties counted by index.
template <int DT>
__device__ void finish_general(const SampleArgs& a, const Row<DT>& row, int64_t r, const Weights& w,
                               const Params& q, uint64_t least, int32_t tiles, int32_t tile_slots,
                               RowShared& s) {
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
  const uint32_t before = workgroup_scan<uint32_t>(n, s.wave32, all_ties);
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

// One row.  Rows without a filter need the chunks' masses only.  Otherwise the cut lies in a list
// of tokens that are put in exact order: with a top-k of at most half the pieces, all tokens at or
// above the k-th largest piece maximum (at least k of them, hardly more than twice k); else the
// tokens of the bins that the cuts fall into.  Tiles whose maximum shows that they hold no kept
// token are not read.
template <int DT>
__global__ __launch_bounds__(kThreads) void row_kernel(SampleArgs a) {
  constexpr int kE = Row<DT>::kE;
  __shared__ RowShared s;
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x;
  const int lane = t & 63;
  const int wave = t >> 6;
  const Row<DT> row(a, r);
  const Params q = row_params(a, r);
  const float top = row_max(a, r, s.wave_max);
  __syncthreads();
  if (top == -INFINITY) {
    if (t == 0) a.out[r] = 0;
    return;
  }
  const bool filter = q.k > 0 || q.p < 1.0;
  if (!q.greedy && !filter && !(q.m > 0.0)) {
    finish_plain(a, row, r, q, top, s);
    return;
  }
  // Tiles: one or more pieces, at most kMaxTiles.
  const int32_t per_tile = (a.pieces + kMaxTiles - 1) / kMaxTiles;
  const int32_t tiles = (a.pieces + per_tile - 1) / per_tile;
  const int32_t tile_slots = per_tile * (kPieceElements / kE);
  if (t < tiles) {
    float m = -INFINITY;
    for (int32_t i = t * per_tile; i < (t + 1) * per_tile && i < a.pieces; ++i)
      m = fmaxf(m, a.piece_max[r * a.pieces + i]);
    s.tile_max[t] = m;
    s.tile_mass[t] = 0;
  }
  if (t == 0) {
    s.value32[1] = 0;           // list length
    s.value32[4] = kMaxTiles;   // first tile with the maximum
    s.value32[5] = 0;           // list members before top-k's bin
  }
  __syncthreads();
  if (q.greedy) {
    if (t < tiles && s.tile_max[t] == top) atomicMin(&s.value32[4], t);
    __syncthreads();
    if (wave == 0) {
      const int32_t s0 = s.value32[4] * tile_slots;
      const int32_t s1 = s0 + tile_slots < row.slots() ? s0 + tile_slots : row.slots();
      const int32_t pick = pick_in_slots(row, s0, s1, 0, [&](float v, int32_t) {
        return (uint64_t)(v == top ? 1 : 0);
      });
      if (lane == 0) a.out[r] = pick;
    }
    return;
  }
  const Weights w{0x1.71547652b82fep+0 / (double)q.t, (double)top, top, a.frac};
  const uint64_t least = least_weight(q.m, a.frac);
  ListCut cut{q.k > 0, q.p < 1.0, (uint32_t)q.k, 0, 0, 0, 0, false};
  int32_t first_bin = kBins, last_bin = -1, k_bin = -1;  // bins of the list: [first, last] and k_bin
  float list_from = INFINITY;                            // or all tokens from this value on
  if (filter && by_pieces(a, q) && per_tile == 1) {
    list_from = kth_tile_max(a, q.k, tiles, s);
  } else if (filter) {
    uint64_t* mass = s.list.bin_mass;
    uint32_t* count = s.list.bin_count;
    for (int32_t b = t; b < kBins; b += kThreads) {
      mass[b] = a.parts > 0 && needs_bins(a, q) ? a.bin_mass[r * kBins + b] : 0;
      count[b] = a.parts > 0 && needs_bins(a, q) ? a.bin_count[r * kBins + b] : 0;
    }
    __syncthreads();
    if (!(a.parts > 0 && needs_bins(a, q))) add_to_bins(row, w, q, 0, row.slots(), mass, count);
    __syncthreads();
    // Thread t holds bins 2 t and 2 t + 1: the largest logits first.
    const int32_t b0 = 2 * t;
    const bool in0 = b0 < kBins, in1 = b0 + 1 < kBins;
    const uint64_t m0 = in0 ? mass[b0] : 0, m1 = in1 ? mass[b0 + 1] : 0;
    const uint32_t c0 = in0 ? count[b0] : 0, c1 = in1 ? count[b0 + 1] : 0;
    uint64_t all_mass;
    uint32_t all_count;
    const uint64_t mb = workgroup_scan<uint64_t>(m0 + m1, s.wave64, all_mass);
    const uint32_t cb = workgroup_scan<uint32_t>(c0 + c1, s.wave32, all_count);
    cut.all_mass = all_mass;
    cut.top_k = q.k > 0 && (uint32_t)q.k < all_count;  // (else it keeps every live token)
    uint64_t low = all_mass, high = all_mass;           // bounds of S(n_k)
    if (cut.top_k) {
      const uint32_t k = (uint32_t)q.k;
      if (cb < k && k <= cb + c0 + c1) {  // one thread
        const bool second = cb + c0 < k;
        s.value32[6] = second ? b0 + 1 : b0;
        s.value32[7] = (int32_t)(k - (second ? cb + c0 : cb));
        s.value64[0] = second ? mb + m0 : mb;
        s.value64[1] = second ? m1 : m0;
      }
      __syncthreads();
      k_bin = s.value32[6];
      cut.k_left = (uint32_t)s.value32[7];
      cut.k_mass = low = s.value64[0];
      high = low + s.value64[1];
      first_bin = last_bin = k_bin;
      __syncthreads();
    }
    if (cut.top_p) {
      uint64_t want0 = (uint64_t)ceil(q.p * (double)low), want1 = (uint64_t)ceil(q.p * (double)high);
      want0 = want0 < 1 ? 1 : want0;
      want1 = want1 < 1 ? 1 : want1;
      const uint64_t x1 = mb + m0, x2 = x1 + m1;
      if (mb < want0 && want0 <= x2) {  // one thread
        const bool second = x1 < want0;
        s.value32[6] = second ? b0 + 1 : b0;
        s.value64[0] = second ? x1 : mb;
      }
      if (mb < want1 && want1 <= x2) s.value32[7] = x1 < want1 ? b0 + 1 : b0;
      __syncthreads();
      first_bin = s.value32[6];
      last_bin = s.value32[7];
      cut.p_mass = s.value64[0];
      __syncthreads();
    }
    if (!cut.top_k && !cut.top_p) first_bin = kBins;  // top-k keeps every live token
  }
  // Gather the list; the weights of the tokens before it go to their tiles.
  const int32_t reach = last_bin > k_bin ? last_bin : k_bin;
  const bool by_value = list_from < INFINITY;
  for (int32_t tile = wave; tile < tiles; tile += kWaves) {
    const float m = s.tile_max[tile];
    if (m == -INFINITY) continue;
    if (by_value ? m < list_from : (first_bin < kBins && bin_of(m, top) > reach)) continue;
    uint64_t mass = 0;
    for (int32_t i = lane; i < tile_slots; i += 64) {
      const int32_t slot = tile * tile_slots + i;
      float v[kE];
      if (slot < row.slots()) {
        row.load(slot, v);
      } else {
#pragma unroll
        for (int j = 0; j < kE; ++j) v[j] = -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < kE; ++j) {
        bool in;
        if (by_value) {
          in = v[j] >= list_from && v[j] > -INFINITY;
        } else {
          const int32_t b = bin_of(v[j], top);
          const bool live = v[j] > -INFINITY;
          in = live && ((b >= first_bin && b <= last_bin) || b == k_bin);
          if (live && b < first_bin) {
            const uint64_t x = w(v[j]);
            mass += x >= least ? x : 0;
          }
          const uint64_t before = __ballot(in && b < k_bin);
          if (before && lane == 0) atomicAdd(&s.value32[5], (int32_t)__popcll(before));
        }
        append(in, place_of(key_of(v[j]), row.first(slot) + j), s);
      }
    }
    if (!by_value) {
      mass = wave_sum(mass);
      if (lane == 0) s.tile_mass[tile] = mass;
    }
  }
  __syncthreads();
  const int32_t n = s.value32[1];
  uint64_t last = 0;
  if (by_value || first_bin < kBins) {
    if (n > kList) {
      finish_general(a, row, r, w, q, least, tiles, tile_slots, s);
      return;
    }
    cut.k_group = s.value32[5];
    if (by_value && n < q.k) {  // fewer live tokens than top-k keeps, and all of them listed
      cut.top_k = false;
      cut.whole = true;
    }
    last = cut_list_any(w, q, cut, n, s);
    for (int32_t i = t; i < n; i += kThreads) {
      const uint64_t p = s.list.place[i];
      const uint64_t x = w(value_of(place_key(p)));
      if (p >= last && x >= least)
        atomicAdd(reinterpret_cast<unsigned long long*>(
                      &s.tile_mass[tile_of(row, place_index(p), tile_slots)]),
                  (unsigned long long)x);
    }
    __syncthreads();
  }
  finish_tiles(a, row, r, q, tiles, tile_slots, s, [&](float v, int32_t i) {
    const uint64_t x = w(v);
    return v > -INFINITY && place_of(key_of(v), i) >= last && x >= least ? x : (uint64_t)0;
  });
}

int frac_bits(int64_t vocab) {
  int b = 0;
  while (((int64_t)1 << b) < vocab) ++b;
  return 62 - b < 48 ? 62 - b : 48;
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

// Workspace: masses of chunks and bins (64 bits), then chunk and piece maxima and bin counts.
int64_t workspace_of(int64_t rows, int64_t chunks, SampleArgs* a, char* base) {
  const int64_t pieces = chunks * (kChunkElements / kPieceElements);
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at = align16(at + bytes);
    return here;
  };
  const int64_t chunk_mass = take(rows * chunks * 8), bin_mass = take(rows * kBins * 8),
                chunk_max = take(rows * chunks * 4), piece_max = take(rows * pieces * 4),
                bin_count = take(rows * kBins * 4);
  if (a) {
    a->chunks = (int32_t)chunks;
    a->pieces = (int32_t)pieces;
    a->chunk_mass = reinterpret_cast<uint64_t*>(base + chunk_mass);
    a->bin_mass = reinterpret_cast<uint64_t*>(base + bin_mass);
    a->chunk_max = reinterpret_cast<float*>(base + chunk_max);
    a->piece_max = reinterpret_cast<float*>(base + piece_max);
    a->bin_count = reinterpret_cast<uint32_t*>(base + bin_count);
  }
  return at;
}

template <int DT>
void launch_sample(const SampleArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(chunk_kernel<DT>, dim3((unsigned)(a.rows * a.chunks)), dim3(kChunkThreads), 0,
                     s, a);
  if (a.parts > 0)
    hipLaunchKernelGGL(bins_kernel<DT>, dim3((unsigned)(a.rows * a.parts)), dim3(kThreads), 0, s, a);
  hipLaunchKernelGGL(row_kernel<DT>, dim3((unsigned)a.rows), dim3(kThreads), 0, s, a);
}

}  // namespace

extern "C" size_t int8kv_sample_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows < 0 || rows > kMaxRows || vocab < 1 || vocab > kMaxVocab) return 0;
  const int64_t chunks = chunks_of(vocab, true);  // at least those of the 16-bit types
  return (size_t)workspace_of(rows > 0 ? rows : 1, chunks, nullptr, nullptr);
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
  SampleArgs a;
  a.logits = logits;
  a.rows = rows;
  a.row_stride = row_stride;
  a.vocab = (int32_t)vocab;
  a.frac = frac_bits(vocab);
  a.u = uniforms;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.out = out;
  hipStream_t s = static_cast<hipStream_t>(stream);
  workspace_of(rows, chunks_of(vocab, logits_dtype == INT8KV_F32), &a, static_cast<char*>(workspace));
  // The histogram pass runs where some row may need it (a nucleus cut, whose mass is the whole
  // row's; a large top-k alone is counted by its own row): about two workgroups per compute unit.
  a.parts = 0;
  if (top_p) {
    const int64_t most = (vocab + 4 * kThreads - 1) / (4 * kThreads);
    const int64_t want = 512 / rows < 1 ? 1 : 512 / rows;
    a.parts = (int32_t)(want < most ? want : most);
  }
  if (logits_dtype == INT8KV_F32)
    launch_sample<kF32>(a, s);
  else if (logits_dtype == INT8KV_BF16)
    launch_sample<kBF16>(a, s);
  else
    launch_sample<kF16>(a, s);
  return (int)hipGetLastError();
}
