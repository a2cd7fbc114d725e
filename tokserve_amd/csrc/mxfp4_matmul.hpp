// What the MXFP4 products share: the block-scaled matrix instruction, the arguments, and the
// order of scale bytes that the tiled kernel reads.
#pragma once

#include "mxfp4_common.hpp"

namespace tks {

typedef int mx_op __attribute__((ext_vector_type(8)));
typedef float mx_f4 __attribute__((ext_vector_type(4)));

// B . A^T of a 16-row tile each over 128 of K: D[4 g + r][i] with B's rows as the instruction's
// first operand, so a lane holds four consecutive columns n of the output row m = i. The scale
// bytes are byte SEL of sb and sa.
template <int SEL>
__device__ __forceinline__ mx_f4 mx_mfma(uint4 b, uint4 a, mx_f4 c, uint32_t sb, uint32_t sa) {
#if __HIP_DEVICE_COMPILE__
  // (e2m1, format 4, takes the first four registers of an operand.)
  const mx_op x = {static_cast<int>(b.x), static_cast<int>(b.y), static_cast<int>(b.z),
                   static_cast<int>(b.w), 0, 0, 0, 0};
  const mx_op y = {static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z),
                   static_cast<int>(a.w), 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, SEL, sb, SEL, sa);
#else
  (void)b; (void)a; (void)sb; (void)sa;
  return c;
#endif
}

struct MatmulArgs {
  const uint8_t *a, *as;  // (M, K) codes and scale bytes, contiguous
  const uint8_t *b, *bs;  // (N, K)
  int64_t m, n, k;
  void *out;
  int64_t o_rs;
};

// Scale bytes as the tiled kernel reads them: per 512 of K ("window") and row 16 bytes, the
// dword of lane group g holding the blocks 4 t + g of the window's four steps t in byte t; 0
// for blocks past K. All rows of a window are together, so that the 16 rows of a tile are one
// run of 256 bytes.
constexpr int kWindow = 512;
inline __host__ __device__ int64_t windows(int64_t k) { return (k + kWindow - 1) / kWindow; }
__device__ __forceinline__ int64_t window_scale_at(int64_t block, int64_t row, int64_t rows) {
  const int64_t w = block >> 4;
  const int j = static_cast<int>(block & 15);
  return (w * rows + row) * 16 + 4 * (j & 3) + (j >> 2);
}
// (The last tile reads whole tiles of rows: 256 more, whose values matter to no result.)
inline int64_t window_scale_bytes(int64_t rows, int64_t k) {
  return (rows * windows(k) + 256) * 16;
}

// The tiled product over A's and B's codes and window-ordered scales (16-byte aligned).
int32_t launch_matmul_tiles(const MatmulArgs &p, int32_t dtype, hipStream_t s);
// A's and B's scale bytes (rows, k / 32) into window order.
int32_t launch_window_scales(const uint8_t *a_scales, int64_t m, uint8_t *a_out,
                             const uint8_t *b_scales, int64_t n, uint8_t *b_out, int64_t k,
                             hipStream_t s);
// Rows of `dtype` to codes and window-ordered scales, and B's scales (n, k / 32) into window
// order, in one launch.
int32_t launch_quantize_windows(const void *x, int64_t x_rs, int64_t m, int64_t k, uint8_t *codes,
                                uint8_t *scales, const uint8_t *b_scales, int64_t n,
                                uint8_t *b_out, int32_t dtype, hipStream_t s);

}  // namespace tks
