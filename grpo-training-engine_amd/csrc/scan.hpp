// Prefixes and reductions of unsigned integers over the lanes of a wave and the threads of a
// block, by DPP moves and one LDS slot per wave (gfx950).
#pragma once

#include "common.hpp"

namespace grpo {

// v of the lane that DPP control CTRL names, 0 where it names none.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp0(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
template <int CTRL>
__device__ __forceinline__ uint64_t dpp0(uint64_t v) {
  return dpp0<CTRL>((uint32_t)v) | ((uint64_t)dpp0<CTRL>((uint32_t)(v >> 32)) << 32);
}
// Inclusive prefix over each row of 16 lanes, and over the wave: shifts by 1, 2, 4, 8
// within the rows, then lane 15 of rows 0 and 2 to the rows after them, then lane 31 to
// the upper half.
template <typename T, typename F>
__device__ __forceinline__ T row_prefix(T v, F&& op) {
  v = op(v, dpp0<0x111>(v));
  v = op(v, dpp0<0x112>(v));
  v = op(v, dpp0<0x114>(v));
  return op(v, dpp0<0x118>(v));
}
template <typename T, typename F>
__device__ __forceinline__ T wave_prefix(T v, F&& op) {
  v = row_prefix(v, op);
  const T below = dpp0<0x142>(v);
  v = op(v, (threadIdx.x & 16) ? below : 0);
  const T half = dpp0<0x143>(v);
  return op(v, (threadIdx.x & 32) ? half : 0);
}
struct Add {
  template <typename T>
  __device__ __forceinline__ T operator()(T a, T b) const { return a + b; }
};
struct Max {
  __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return max(a, b); }
};
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) {
  return (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ uint64_t lane_value(uint64_t v, int lane) {
  return lane_value((uint32_t)v, lane) | ((uint64_t)lane_value((uint32_t)(v >> 32), lane) << 32);
}

// Block-wide sum / max over NW <= 16 waves through one LDS slot per wave.  Every
// thread gets the result; the trailing barrier lets the slots be reused.
template <int NW, typename T, typename F>
__device__ __forceinline__ T block_reduce(T v, T* slots, F&& op) {
  const int lane = threadIdx.x & 63;
  v = wave_prefix(v, op);
  if (lane == 63) slots[threadIdx.x >> 6] = v;
  __syncthreads();
  const T s = lane < NW ? slots[lane] : 0;
  __syncthreads();
  return lane_value(row_prefix(s, op), 15);
}
template <int NW, typename T>
__device__ __forceinline__ T block_sum(T v, T* slots) {
  return block_reduce<NW>(v, slots, Add());
}
template <int NW>
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* slots) {
  return block_reduce<NW>(v, slots, Max());
}

// Exclusive prefix over a block of 1024 threads (thread order) of a (u64, u32) pair: one row
// of lanes scans the sixteen waves' sums.
__device__ __forceinline__ void block_excl_scan(uint64_t& a, uint32_t& b, uint64_t* sa,
                                                uint32_t* sb) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint64_t ia = wave_prefix(a, Add());
  const uint32_t ib = wave_prefix(b, Add());
  if (lane == 63) {
    sa[wave] = ia;
    sb[wave] = ib;
  }
  __syncthreads();
  const uint64_t va = row_prefix(sa[lane & 15], Add());
  const uint32_t vb = row_prefix(sb[lane & 15], Add());
  __syncthreads();
  a = ia - a + (wave ? lane_value(va, wave - 1) : 0);
  b = ib - b + (wave ? lane_value(vb, wave - 1) : 0);
}

}  // namespace grpo
