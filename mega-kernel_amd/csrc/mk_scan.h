// Sums and maxima over the lanes of a wave and the waves of a workgroup on MI355X (gfx950), of 32- and 64-bit
// numbers, by DPP: no LDS traffic but a workgroup's one number per wave.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mk {

// v of another lane by DPP, 0 where there is none
template <int CTRL, int ROWS, typename V>
__device__ __forceinline__ V from_lane(V v) {
  if constexpr (sizeof(V) == 4) {
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
  } else {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(V, (uint64_t)hi << 32 | lo);
  }
}
template <typename V>
__device__ __forceinline__ V at_lane(V v, int lane) {
  if constexpr (sizeof(V) == 4) {
    return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
  } else {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(V, (uint64_t)hi << 32 | lo);
  }
}
// op over lanes 0 .. this one of each 16, and of the wave; 0 is op's neutral number
template <typename V, typename F>
__device__ __forceinline__ V scan_row16(V v, F op) {
  v = op(v, from_lane<0x111, 0xf>(v));  // row_shr 1, 2, 4, 8
  v = op(v, from_lane<0x112, 0xf>(v));
  v = op(v, from_lane<0x114, 0xf>(v));
  return op(v, from_lane<0x118, 0xf>(v));
}
template <typename V, typename F>
__device__ __forceinline__ V scan_wave(V v, F op) {
  v = scan_row16(v, op);
  v = op(v, from_lane<0x142, 0xa>(v));  // row_bcast 15, 31
  return op(v, from_lane<0x143, 0xc>(v));
}
template <typename V>
__device__ __forceinline__ V plus(V a, V b) { return a + b; }
template <typename V>
__device__ __forceinline__ V sum_over_wave(V v) { return at_lane(scan_wave(v, plus<V>), 63); }
template <typename V>
__device__ __forceinline__ V max_over_wave(V v) {  // of numbers that are not negative
  return at_lane(scan_wave(v, [](V a, V b) { return a > b ? a : b; }), 63);
}

// Sums over the threads up to this one, over all WAVES waves of the workgroup and over the waves before this one, each in
// an order of its own. `lds` holds WAVES numbers. For numbers that round: the sum before a thread is the one up to the
// thread before it. (Taken as a difference, a small sum before a large number would be rounded to the large one's digits.)
template <int WAVES, typename V>
__device__ __forceinline__ V block_upto(V v, V* lds, V& total, V& waves) {
  static_assert(WAVES <= 16 && (WAVES & (WAVES - 1)) == 0);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const V x = scan_wave(v, plus<V>);
  __syncthreads();
  if (lane == 63) lds[w] = x;
  __syncthreads();
  const V y = scan_row16(lds[lane & (WAVES - 1)], plus<V>);  // every wave: the waves' sums, up to each
  total = at_lane(y, WAVES - 1);
  const V before = at_lane(y, w > 0 ? w - 1 : 0);
  waves = w ? before : (V)0;
  return waves + x;
}
template <int WAVES, typename V>
__device__ __forceinline__ V block_upto(V v, V* lds, V& total) {
  V waves;
  return block_upto<WAVES>(v, lds, total, waves);
}
// Sums over the threads before this one and over all, of whole numbers.
template <int WAVES, typename V>
__device__ __forceinline__ V block_before(V v, V* lds, V& total) {
  static_assert(V(0.5) == V(0), "a sum that rounds has no exact difference");
  return block_upto<WAVES>(v, lds, total) - v;
}

}  // namespace mk
