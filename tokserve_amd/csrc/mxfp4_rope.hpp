// Eight values of a row at a time, rotated (rope_common.hpp) on their way to MXFP4.
#pragma once

#include "mxfp4_common.hpp"
#include "rope_common.hpp"

namespace tks {

template <typename T, bool VEC>
__device__ __forceinline__ MxEight<T> load8(const T *p) {
  if constexpr (VEC) return mx_load8<T>(p);
  return mx_load8_any<T>(p);
}

template <typename T>
__device__ __forceinline__ void floats8(const MxEight<T> &x, float *f) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) unpack<T>(x.v[i], f + i * Vec<T>::N);
}

// Values d .. d+7 of the row at x, rotated at the table rows c and s, rounded to T: the pair
// of each value is half a row away (half is a multiple of 16).
template <typename T, bool VEC>
__device__ __forceinline__ MxEight<T> rotated8(const T *x, const T *c, const T *s, int d,
                                               int half) {
  const bool first = d < half;
  const int at = first ? d : d - half;
  float lo[8], hi[8], cf[8], sf[8], o1[8], o2[8];
  floats8<T>(load8<T, VEC>(x + at), lo);
  floats8<T>(load8<T, VEC>(x + at + half), hi);
  floats8<T>(load8<T, VEC>(c + at), cf);
  floats8<T>(load8<T, VEC>(s + at), sf);
  rotate_math<T, 8>(lo, hi, cf, sf, o1, o2);
#pragma unroll
  for (int j = 0; j < 8; ++j) o1[j] = fp32_value(first ? o1[j] : o2[j]);
  MxEight<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.v[i] = pack<T>(o1 + i * Vec<T>::N);
  return r;
}

// Threads to a row of DH values, eight each: a divisor of 64, so that a row lies in one wave
// (Dh 96: a quad of each sixteen idles).
__host__ __device__ __forceinline__ int row_threads(int head_dim) {
  return head_dim == 96 ? 16 : head_dim / 8;
}

}  // namespace tks
