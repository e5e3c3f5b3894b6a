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

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr int kMaxTiles = kThreads;  // one per thread in the tile scan
constexpr int64_t kMaxVocab = 1 << 22;

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
struct Cut {
  uint32_t tau;   // keys above are kept ...
  uint32_t ties;  // ... and the first `ties` tokens with key tau
};

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

// ------------------------------------------------------------------------------ one workgroup
struct Shared {
  uint64_t mass[kBins];
  uint32_t count[kBins];
  uint64_t wave64[kWaves];
  uint32_t wave32[kWaves];
  float wave_max[kWaves];
  int32_t wave_at[kWaves];
  uint64_t found64[2];
  uint32_t found32[4];
};

// The row's maximum and its first index (-inf and 0 for a row without finite values).
template <int DT>
__device__ __forceinline__ void row_max(const Row<DT>& row, Shared& s, float& top, int32_t& at) {
  float m = -INFINITY;
  int32_t mi = 0x7fffffff;
  for (int32_t q = threadIdx.x; q < row.slots(); q += kThreads) {
    float v[Row<DT>::kE];
    row.load(q, v);
#pragma unroll
    for (int j = 0; j < Row<DT>::kE; ++j)
      if (v[j] > m) {
        m = v[j];
        mi = row.first(q) + j;
      }
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    const float om = __shfl_xor(m, d, 64);
    const int32_t oi = __shfl_xor(mi, d, 64);
    if (om > m || (om == m && oi < mi)) {
      m = om;
      mi = oi;
    }
  }
  if ((threadIdx.x & 63) == 0) {
    s.wave_max[threadIdx.x >> 6] = m;
    s.wave_at[threadIdx.x >> 6] = mi;
  }
  __syncthreads();
  top = s.wave_max[0];
  at = s.wave_at[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w)
    if (s.wave_max[w] > top || (s.wave_max[w] == top && s.wave_at[w] < at)) {
      top = s.wave_max[w];
      at = s.wave_at[w];
    }
  if (top == -INFINITY) at = 0;
}

// The key at which a prefix of the order ends, digit by digit from the top (11, 11 and 10 bits; a
// 16-bit type's keys differ in the first 22 only).  BY_MASS: the first `want` units of weight,
// else the first `want` tokens; tokens at -inf are not counted.  Returns the key with the tokens and the mass
// above it and the tokens at it, or false where the row has less than `want`.
template <int DT, bool BY_MASS>
__device__ bool select_key(const Row<DT>& row, const Weights& w, uint64_t want, bool need_mass,
                           Shared& s, uint32_t& key, uint32_t& count_above, uint64_t& mass_above,
                           uint32_t& at_key) {
  constexpr int kLevels = DT == kF32 ? 3 : 2;
  uint32_t prefix = 0, mask = 0;
  count_above = 0;
  mass_above = 0;
  for (int level = 0; level < kLevels; ++level) {
    const int shift = level == 0 ? 21 : (level == 1 ? 10 : 0);
    const uint32_t digit = level == 2 ? 1023u : 2047u;
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
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
    const int b0 = kBins - 1 - 2 * (int)threadIdx.x;
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
__device__ Cut find_cut(const Row<DT>& row, const Weights& w, const Params& q, Shared& s) {
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

// Kept weight of a slot's elements above the cut, and the number of its ties.
template <int N>
__device__ __forceinline__ uint64_t slot_mass(const float (&v)[N], const Weights& w, uint32_t tau,
                                              uint64_t least, uint32_t& ties) {
  uint64_t sum = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint32_t k = key_of(v[j]);
    const uint64_t x = w(v[j]);
    sum += k > tau && x >= least ? x : 0;
    ties += k == tau ? 1u : 0u;
  }
  return sum;
}

// The index of the first kept token whose cumulative weight exceeds `target`, within the slots
// [s0, s1) (one wave; `ties` tied tokens and `target` units of weight remain before them).
template <int DT>
__device__ int32_t pick_in_slots(const Row<DT>& row, const Weights& w, Cut cut, uint64_t least,
                                 uint64_t tie_weight, int32_t s0, int32_t s1, uint32_t ties,
                                 uint64_t target) {
  constexpr int kE = Row<DT>::kE;
  const int lane = threadIdx.x & 63;
  for (int32_t q0 = s0; q0 < s1; q0 += 64) {
    float v[kE];
    uint32_t n = 0;
    uint64_t mass = 0;
    const int32_t q = q0 + lane;
    if (q < s1) {
      row.load(q, v);
      mass = slot_mass(v, w, cut.tau, least, n);
    }
    const uint32_t tie_incl = wave_scan<uint32_t>(n);
    const uint32_t tie_before = tie_incl - n;
    const uint32_t left = ties > tie_before ? ties - tie_before : 0;  // tied tokens this lane may keep
    const uint32_t mine = n < left ? n : left;
    mass += mine * tie_weight;
    const uint64_t incl = wave_scan<unsigned long long>(mass);
    const uint64_t before = incl - mass;
    const bool here = before <= target && target < incl;
    const uint64_t any = __ballot(here);
    if (any) {
      int32_t pick = 0;
      if (here) {
        uint64_t sum = before;
        uint32_t tl = left;
        bool done = false;
#pragma unroll
        for (int j = 0; j < kE; ++j) {
          const uint32_t k = key_of(v[j]);
          uint64_t x = w(v[j]);
          if (k == cut.tau) {
            x = tl > 0 ? tie_weight : 0;
            tl -= tl > 0 ? 1 : 0;
          } else if (k < cut.tau || x < least) {
            x = 0;
          }
          sum += x;
          if (!done && sum > target) {
            pick = row.first(q) + j;
            done = true;
          }
        }
      }
      return __shfl(pick, __ffsll((unsigned long long)any) - 1, 64);
    }
    const uint32_t all_ties = __shfl(tie_incl, 63, 64);
    ties = ties > all_ties ? ties - all_ties : 0;
    target -= __shfl((unsigned long long)incl, 63, 64);
  }
  return 0;  // (not reached: target lies below the sum of [s0, s1))
}

template <int DT>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  __shared__ Shared s;
  __shared__ uint64_t s_tile_mass[kMaxTiles];
  __shared__ uint32_t s_tile_ties[kMaxTiles];
  const int64_t r = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const Row<DT> row(a, r);
  const Params q = row_params(a, r);
  float top;
  int32_t first;
  row_max(row, s, top, first);
  if (q.greedy || top == -INFINITY) {
    if (threadIdx.x == 0) a.out[r] = first;
    return;
  }
  const Weights w{0x1.71547652b82fep+0 / (double)q.t, (double)top, top, a.frac};
  const uint64_t least = least_weight(q.m, a.frac);
  Cut cut{0u, 0u};
  if (q.k > 0 || q.p < 1.0) cut = find_cut(row, w, q, s);
  uint64_t tie_weight = cut.ties > 0 ? w(value_of(cut.tau)) : 0;
  if (tie_weight < least) tie_weight = 0;
  // Kept weight per tile of slots, in index order.
  const int32_t per_tile = 64 * ((row.slots() + 64 * kMaxTiles - 1) / (64 * kMaxTiles));
  const int32_t tiles = (row.slots() + per_tile - 1) / per_tile;
  for (int32_t t = wave; t < tiles; t += kWaves) {
    uint64_t mass = 0;
    uint32_t ties = 0;
    for (int32_t i = 0; i < per_tile; i += 64) {
      const int32_t slot = t * per_tile + i + lane;
      if (slot < row.slots()) {
        float v[Row<DT>::kE];
        row.load(slot, v);
        mass += slot_mass(v, w, cut.tau, least, ties);
      }
    }
    mass = wave_sum(mass);
    const uint64_t n = wave_sum((uint64_t)ties);
    if (lane == 0) {
      s_tile_mass[t] = mass;
      s_tile_ties[t] = (uint32_t)n;
    }
  }
  __syncthreads();
  const int32_t t = threadIdx.x;
  uint64_t mass = t < tiles ? s_tile_mass[t] : 0;
  const uint32_t n = t < tiles ? s_tile_ties[t] : 0;
  uint32_t all_ties;
  const uint32_t tie_before = workgroup_scan<uint32_t>(n, s.wave32, all_ties);
  const uint32_t left = cut.ties > tie_before ? cut.ties - tie_before : 0;
  mass += (n < left ? n : left) * tie_weight;
  uint64_t total;
  const uint64_t before = workgroup_scan<uint64_t>(mass, s.wave64, total);
  const uint64_t target = scaled(q.u, total);
  if (before <= target && target < before + mass) {  // one thread
    s.found32[0] = (uint32_t)t;
    s.found32[1] = left;
    s.found64[0] = target - before;
  }
  __syncthreads();
  if (wave == 0) {
    const int32_t s0 = (int32_t)s.found32[0] * per_tile;
    const int32_t s1 = s0 + per_tile < row.slots() ? s0 + per_tile : row.slots();
    const int32_t pick = pick_in_slots(row, w, cut, least, tie_weight, s0, s1, s.found32[1], s.found64[0]);
    if (lane == 0) a.out[r] = pick;
  }
}

int frac_bits(int64_t vocab) {
  int b = 0;
  while (((int64_t)1 << b) < vocab) ++b;
  return 62 - b < 48 ? 62 - b : 48;
}

}  // namespace
}  // namespace int8kv_serving

using namespace int8kv_serving;

extern "C" size_t int8kv_sample_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows < 0 || rows > 0x7fffffff || vocab < 1 || vocab > kMaxVocab) return 0;
  return 16;
}

extern "C" int int8kv_sample_rows(const void* logits, int logits_dtype, int64_t rows, int64_t vocab,
                                  int64_t row_stride, const float* uniforms,
                                  const float* temperature, const int32_t* top_k,
                                  const float* top_p, const float* min_p, int64_t* out,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  if (rows != 0 && (!logits || !uniforms || !out)) return INT8KV_E_NULL;
  if (logits_dtype != INT8KV_F32 && logits_dtype != INT8KV_F16 && logits_dtype != INT8KV_BF16)
    return INT8KV_E_DTYPE;
  if (rows < 0 || rows > 0x7fffffff || vocab < 1 || vocab > kMaxVocab) return INT8KV_E_SHAPE;
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
  const dim3 grid((unsigned)rows), block(kThreads);
  if (logits_dtype == INT8KV_F32)
    hipLaunchKernelGGL(sample_kernel<kF32>, grid, block, 0, s, a);
  else if (logits_dtype == INT8KV_BF16)
    hipLaunchKernelGGL(sample_kernel<kBF16>, grid, block, 0, s, a);
  else
    hipLaunchKernelGGL(sample_kernel<kF16>, grid, block, 0, s, a);
  return (int)hipGetLastError();
}
