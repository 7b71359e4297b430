// Sums, maxima and running sums over the lanes of a wave, by moves that take no trip through LDS.
#pragma once
#include "common.h"

namespace amoe {

typedef unsigned long long u64;

// Over the N lanes of a group (16 or 64), the same in all of them.
template <int N, class Join>
__device__ __forceinline__ float lanes_all(float v, Join join) {
  static_assert(N == 16 || N == 64, "a row or the whole wave");
  v = join(v, as_f32(row_rotate<8>(as_u32(v))));
  v = join(v, as_f32(row_rotate<4>(as_u32(v))));
  v = join(v, as_f32(row_rotate<2>(as_u32(v))));
  v = join(v, as_f32(row_rotate<1>(as_u32(v))));
  if constexpr (N == 64) {
    uint32_t a = as_u32(v), b = a;
    swap_odd_rows(a, b);
    v = join(as_f32(a), as_f32(b));
    a = b = as_u32(v);
    swap_half_waves(a, b);
    v = join(as_f32(a), as_f32(b));
  }
  return v;
}
template <int N = 64>
__device__ __forceinline__ float lanes_sum(float v) {
  return lanes_all<N>(v, [](float a, float b) __attribute__((always_inline)) { return a + b; });
}
__device__ __forceinline__ float wave_largest(float v) {
  return lanes_all<64>(v, [](float a, float b) __attribute__((always_inline)) { return fmaxf(a, b); });
}

__device__ __forceinline__ u64 join_words(uint32_t hi, uint32_t lo) { return ((u64)hi << 32) | lo; }
__device__ __forceinline__ u64 wave_total(u64 v) {
  v += join_words(row_rotate<8>((uint32_t)(v >> 32)), row_rotate<8>((uint32_t)v));
  v += join_words(row_rotate<4>((uint32_t)(v >> 32)), row_rotate<4>((uint32_t)v));
  v += join_words(row_rotate<2>((uint32_t)(v >> 32)), row_rotate<2>((uint32_t)v));
  v += join_words(row_rotate<1>((uint32_t)(v >> 32)), row_rotate<1>((uint32_t)v));
  uint32_t ah = (uint32_t)(v >> 32), al = (uint32_t)v, bh = ah, bl = al;
  swap_odd_rows(ah, bh);
  swap_odd_rows(al, bl);
  v = join_words(ah, al) + join_words(bh, bl);
  ah = bh = (uint32_t)(v >> 32);
  al = bl = (uint32_t)v;
  swap_half_waves(ah, bh);
  swap_half_waves(al, bl);
  return join_words(ah, al) + join_words(bh, bl);
}
// sums up to and with the lane's
__device__ __forceinline__ int wave_scan(int n) {
  uint32_t v = (uint32_t)n;
  v += row_from_below<1>(v);
  v += row_from_below<2>(v);
  v += row_from_below<4>(v);
  v += row_from_below<8>(v);
  v += odd_rows_from_below(v);
  v += upper_half_from_below(v);
  return (int)v;
}
__device__ __forceinline__ u64 wave_scan(u64 v) {
  v += join_words(row_from_below<1>((uint32_t)(v >> 32)), row_from_below<1>((uint32_t)v));
  v += join_words(row_from_below<2>((uint32_t)(v >> 32)), row_from_below<2>((uint32_t)v));
  v += join_words(row_from_below<4>((uint32_t)(v >> 32)), row_from_below<4>((uint32_t)v));
  v += join_words(row_from_below<8>((uint32_t)(v >> 32)), row_from_below<8>((uint32_t)v));
  v += join_words(odd_rows_from_below((uint32_t)(v >> 32)), odd_rows_from_below((uint32_t)v));
  v += join_words(upper_half_from_below((uint32_t)(v >> 32)), upper_half_from_below((uint32_t)v));
  return v;
}
// what lane `src` holds (the same for the whole wave)
__device__ __forceinline__ u64 wave_read(u64 v, int src) { return join_words(wave_read((uint32_t)(v >> 32), src), wave_read((uint32_t)v, src)); }

}  // namespace amoe
