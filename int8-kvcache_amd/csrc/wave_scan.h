// Prefix sums over a wave by lane moves (DPP), and over a workgroup, for gfx950 (wave64).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace int8kv_serving {

// A lane's value moved along the wave without LDS (DPP): CTRL row_shr 1, 2, 4, 8 within 16 lanes,
// row_bcast 15 and 31 across them.  Lanes without a source keep `old`.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t old, uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)old, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_add(uint32_t v) {
  return v + dpp<CTRL, ROWS>(0u, v);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_add(uint64_t v) {
  const uint32_t lo = dpp<CTRL, ROWS>(0u, (uint32_t)v);
  const uint32_t hi = dpp<CTRL, ROWS>(0u, (uint32_t)(v >> 32));
  return v + (((uint64_t)hi << 32) | lo);
}
// Inclusive prefix sum over the wave.
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
  v = dpp_add<0x111, 0xf>(v);
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);
  return dpp_add<0x143, 0xc>(v);
}
__device__ __forceinline__ uint32_t last_lane(uint32_t v, int lane = 63) {
  return (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ uint64_t last_lane(uint64_t v, int lane = 63) {
  return ((uint64_t)last_lane((uint32_t)(v >> 32), lane) << 32) | last_lane((uint32_t)v, lane);
}
__device__ __forceinline__ uint64_t wave_sum(uint64_t v) { return last_lane(wave_scan(v)); }
// Exclusive prefix sum over a workgroup of WAVES (1, 2, 4, 8 or 16) waves; s_wave: WAVES values.
template <int WAVES, typename T>
__device__ __forceinline__ T workgroup_scan(T v, T* s_wave, T& total) {
  static_assert(WAVES <= 16 && (WAVES & (WAVES - 1)) == 0, "the waves' sums are scanned by 16 lanes");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T inc = wave_scan(v);
  __syncthreads();
  if (lane == 63) s_wave[wave] = inc;
  __syncthreads();
  T w = s_wave[lane & (WAVES - 1)];
  w = dpp_add<0x111, 0xf>(w);
  w = dpp_add<0x112, 0xf>(w);
  w = dpp_add<0x114, 0xf>(w);
  w = dpp_add<0x118, 0xf>(w);
  total = last_lane(w, WAVES - 1);
  const T before = wave > 0 ? last_lane(w, wave - 1) : 0;
  return before + inc - v;
}

}  // namespace int8kv_serving
