// MXFP4 (OCP microscaled 4-bit floating point): 32 consecutive values x of a row share one
// power-of-two scale and are held as e2m1 codes.
//
//   E     = clamp(e - 2, 2, 252), e the biased fp32 exponent of max |x| (0 for 0 and fp32
//           subnormals); 255 where a value is NaN or infinite
//   scale = 2^(E - 127) (e8m0), NaN for E = 255
//   code  = x / scale rounded to nearest, ties to the even code, at most 6 in magnitude: of
//           0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign bit; 0 throughout a block with E = 255
//
// Two codes to a byte, the even element in the low nibble. max |x| / scale lies in [4, 8), so
// the largest code of a block is 4 or 6. A decoded value, code * scale, has two significant
// bits and at least 2^-126 in magnitude if it is not 0: exact in fp32 and bf16.
//
// The gfx950 converters v_cvt_scalef32_pk_* do x / scale, its rounding and its saturation
// in one instruction per pair, and the decoding likewise.
#pragma once

#include "common.hpp"

namespace tks {

constexpr int kMxBlock = 32;
constexpr uint32_t kMxNan = 255;

typedef uint32_t mx_u32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t mx_u16x2 __attribute__((ext_vector_type(2)));

// Scale byte of a block from the biased fp32 exponent of its largest magnitude.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t exponent) {
  return exponent == 255 ? kMxNan : max(exponent, 4u) - 2;
}

// The scale as the converters take it: they read a float's exponent field as e8m0, 0 being
// 2^-127 and 255 a NaN for every code.
__device__ __forceinline__ float mx_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight consecutive values of a row in registers, as stored.
template <typename T>
struct MxEight {
  uint4 v[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ MxEight<T> mx_load8(const T *p) {
  MxEight<T> x;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) x.v[i] = ld16(p + i * Vec<T>::N);
  return x;
}
// The same without the 16-byte alignment.
template <typename T>
__device__ __forceinline__ MxEight<T> mx_load8_any(const T *p) {
  T t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = p[i];
  MxEight<T> x;
  __builtin_memcpy(&x, t, sizeof(x));
  return x;
}

// Largest magnitude of the eight as the bits of a T (its sign bit clear): such bits order as
// the magnitudes do, infinities and NaN last.
template <typename T>
__device__ __forceinline__ uint32_t mx_largest(const MxEight<T> &x) {
  if constexpr (sizeof(T) == 4) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t w[4] = {x.v[i].x, x.v[i].y, x.v[i].z, x.v[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) m = max(m, w[j] & 0x7fffffffu);
    }
    return m;
  } else {
    const uint32_t w[4] = {x.v[0].x, x.v[0].y, x.v[0].z, x.v[0].w};
    mx_u16x2 m = {0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t a = w[j] & 0x7fff7fffu;
      mx_u16x2 h;
      __builtin_memcpy(&h, &a, 4);
      m = __builtin_elementwise_max(m, h);
    }
    return max(static_cast<uint32_t>(m[0]), static_cast<uint32_t>(m[1]));
  }
}

// Biased fp32 exponent of a magnitude given as a T's bits.
template <typename T>
__device__ __forceinline__ uint32_t mx_exponent(uint32_t bits) {
  if constexpr (sizeof(T) == 4) return bits >> 23;
  if constexpr (__is_same(T, bf16_t)) return bits >> 7;
  if (bits >= 0x7c00u) return 255;
  const uint16_t h = static_cast<uint16_t>(bits);
  _Float16 f;
  __builtin_memcpy(&f, &h, 2);
  return __float_as_uint(static_cast<float>(f)) >> 23;
}

// The codes of the eight, element 0 in the low nibble.
template <typename T>
__device__ __forceinline__ uint32_t mx_codes(const MxEight<T> &x, uint32_t scale_byte) {
  uint32_t c = 0;
#if __HIP_DEVICE_COMPILE__
  const float s = mx_scale(scale_byte);
  if constexpr (sizeof(T) == 4) {
    float f[8];
    __builtin_memcpy(f, &x, 32);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[0], f[1], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[2], f[3], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[4], f[5], s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[6], f[7], s, 3);
  } else if constexpr (__is_same(T, bf16_t)) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    pair p[4];
    __builtin_memcpy(p, &x, 16);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, p[0], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, p[1], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, p[2], s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, p[3], s, 3);
  } else {
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
    pair p[4];
    __builtin_memcpy(p, &x, 16);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, p[0], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, p[1], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, p[2], s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, p[3], s, 3);
  }
#else
  (void)x;
#endif
  return scale_byte == kMxNan ? 0 : c;
}

// Quantizes a block held by four neighbouring lanes of a DPP quad, eight values each (every
// lane of the quad active): this lane's codes, and the block's scale byte in every lane.
template <typename T>
__device__ __forceinline__ uint32_t mx_quantize(const MxEight<T> &x, uint32_t *scale_byte) {
  uint32_t m = mx_largest<T>(x);
  m = max(m, static_cast<uint32_t>(
                 __builtin_amdgcn_mov_dpp(static_cast<int>(m), kDppQuadSwap1, 0xF, 0xF, true)));
  m = max(m, static_cast<uint32_t>(
                 __builtin_amdgcn_mov_dpp(static_cast<int>(m), kDppQuadSwap2, 0xF, 0xF, true)));
  *scale_byte = mx_scale_byte(mx_exponent<T>(m));
  return mx_codes<T>(x, *scale_byte);
}

// Quantizes a block that the lane holds alone: its 16 bytes of codes and its scale byte.
template <typename T>
__device__ __forceinline__ uint4 mx_quantize_block(const MxEight<T> (&x)[4],
                                                   uint32_t *scale_byte) {
  uint32_t m = mx_largest<T>(x[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) m = max(m, mx_largest<T>(x[i]));
  *scale_byte = mx_scale_byte(mx_exponent<T>(m));
  return make_uint4(mx_codes<T>(x[0], *scale_byte), mx_codes<T>(x[1], *scale_byte),
                    mx_codes<T>(x[2], *scale_byte), mx_codes<T>(x[3], *scale_byte));
}

// Codes 2 SEL and 2 SEL + 1 of a word times the scale, as floats.
template <int SEL>
__device__ __forceinline__ void mx_pair(uint32_t codes, float scale, float *out) {
#if __HIP_DEVICE_COMPILE__
  const auto f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, SEL);
  out[0] = f[0];
  out[1] = f[1];
#else
  (void)codes; (void)scale; (void)out;
#endif
}
__device__ __forceinline__ void mx_values8(uint32_t codes, float scale, float *out) {
  mx_pair<0>(codes, scale, out);
  mx_pair<1>(codes, scale, out + 2);
  mx_pair<2>(codes, scale, out + 4);
  mx_pair<3>(codes, scale, out + 6);
}

// Eight floats rounded to T and stored (16-byte aligned with VEC).
template <typename T, bool VEC>
__device__ __forceinline__ void mx_store8(T *p, const float *f) {
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < 8; i += Vec<T>::N) st16(p + i, pack<T>(f + i));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = from_float<T>(f[i]);
  }
}

}  // namespace tks
