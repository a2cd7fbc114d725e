// Rows to MXFP4 and back (mxfp4_common.hpp). A lane takes eight consecutive values, so a
// block is the work of four neighbouring lanes and a wave's loads and stores are contiguous.
// Bound by HBM: one pass, 16-byte loads, kItems of them in flight per thread. bf16, 11,264 x
// 2,048: 11 us there and 10 back, 5.1 TB/s in a row (a large copy's rate).
#include "mxfp4_common.hpp"

#include <algorithm>

namespace tks {
namespace {

constexpr int kThreads = 256;
constexpr int kItems = 4;  // eights per thread

// The eight-value groups of `rows` rows of `eights` groups each: group i of this thread.
__device__ __forceinline__ int64_t group_index(int i) {
  return (static_cast<int64_t>(blockIdx.x) * kItems + i) * kThreads + threadIdx.x;
}

// Element offset of group `at` in rows of stride `rs`.
__device__ __forceinline__ int64_t group_offset(int64_t at, int64_t eights, int64_t rs) {
  const int64_t r = at / eights;
  return r * rs + (at - r * eights) * 8;
}

// total: groups in all. FLAT: the rows are contiguous, group i at element 8 i.
template <typename T, bool VEC, bool FLAT>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const T *__restrict__ x, int64_t rs,
                                                            int64_t total, int64_t eights,
                                                            uint32_t *__restrict__ codes,
                                                            uint8_t *__restrict__ scales) {
  MxEight<T> v[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int64_t at = group_index(i);
    if (at >= total) continue;  // whole blocks: total is a multiple of 4
    const T *p = x + (FLAT ? at * 8 : group_offset(at, eights, rs));
    v[i] = VEC ? mx_load8<T>(p) : mx_load8_any<T>(p);
  }
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int64_t at = group_index(i);
    if (at >= total) continue;
    uint32_t s;
    codes[at] = mx_quantize<T>(v[i], &s);
    if ((threadIdx.x & 3) == 0) scales[at >> 2] = static_cast<uint8_t>(s);
  }
}

template <typename T, bool VEC, bool FLAT>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(const uint32_t *__restrict__ codes,
                                                              const uint8_t *__restrict__ scales,
                                                              int64_t total, int64_t eights,
                                                              T *__restrict__ out, int64_t rs) {
  uint32_t c[kItems];
  uint8_t s[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int64_t at = group_index(i);
    if (at >= total) continue;
    c[i] = codes[at];
    s[i] = scales[at >> 2];
  }
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int64_t at = group_index(i);
    if (at >= total) continue;
    float f[8];
    mx_values8(c[i], mx_scale(s[i]), f);
    mx_store8<T, VEC>(out + (FLAT ? at * 8 : group_offset(at, eights, rs)), f);
  }
}

bool rows_ok(int64_t rows, int64_t cols, const void *codes) {
  return rows >= 0 && cols > 0 && cols % kMxBlock == 0 &&
         (reinterpret_cast<uintptr_t>(codes) & 3) == 0;
}

// Workgroups of a launch over `total` groups, 0 if they are too many for one.
int64_t grid_of(int64_t total) {
  const int64_t n = ceil_div(total, kThreads * kItems);
  return n <= 0x7fffffff ? n : 0;
}

template <typename T>
void launch_quantize(const void *x, int64_t rs, int64_t rows, int64_t cols, void *codes,
                     void *scales, unsigned grid, hipStream_t s) {
  const bool flat = rs == cols || rows == 1;
  const bool vec = aligned16(x) && (flat || rs * sizeof(T) % 16 == 0);
  const int64_t total = rows * cols / 8;
  const T *in = static_cast<const T *>(x);
  uint32_t *c = static_cast<uint32_t *>(codes);
  uint8_t *e = static_cast<uint8_t *>(scales);
  if (vec && flat)
    quantize_kernel<T, true, true><<<grid, kThreads, 0, s>>>(in, rs, total, cols / 8, c, e);
  else if (vec)
    quantize_kernel<T, true, false><<<grid, kThreads, 0, s>>>(in, rs, total, cols / 8, c, e);
  else
    quantize_kernel<T, false, false><<<grid, kThreads, 0, s>>>(in, rs, total, cols / 8, c, e);
}

template <typename T>
void launch_dequantize(const void *codes, const void *scales, int64_t rows, int64_t cols,
                       void *out, int64_t rs, unsigned grid, hipStream_t s) {
  const bool flat = rs == cols || rows == 1;
  const bool vec = aligned16(out) && (flat || rs * sizeof(T) % 16 == 0);
  const int64_t total = rows * cols / 8;
  T *o = static_cast<T *>(out);
  const uint32_t *c = static_cast<const uint32_t *>(codes);
  const uint8_t *e = static_cast<const uint8_t *>(scales);
  if (vec && flat)
    dequantize_kernel<T, true, true><<<grid, kThreads, 0, s>>>(c, e, total, cols / 8, o, rs);
  else if (vec)
    dequantize_kernel<T, true, false><<<grid, kThreads, 0, s>>>(c, e, total, cols / 8, o, rs);
  else
    dequantize_kernel<T, false, false><<<grid, kThreads, 0, s>>>(c, e, total, cols / 8, o, rs);
}

}  // namespace
}  // namespace tks

using namespace tks;

extern "C" int32_t tks_mxfp4_quantize(const void *input, int64_t input_row_stride,
                                      int64_t num_rows, int64_t num_cols, void *codes,
                                      void *scales, int32_t dtype, tks_stream_t stream) {
  if (!valid_dtype(dtype)) return TKS_ERR_TYPE;
  if (!rows_ok(num_rows, num_cols, codes)) return TKS_ERR_VALUE;
  if (num_rows == 0) return TKS_OK;
  if (!input || !codes || !scales) return TKS_ERR_VALUE;
  if (num_rows > INT64_MAX / 4 / num_cols) return TKS_ERR_VALUE;
  const int64_t grid = grid_of(num_rows * num_cols / 8);
  if (grid == 0) return TKS_ERR_VALUE;
  const unsigned g = static_cast<unsigned>(grid);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TKS_FLOAT32:
      launch_quantize<float>(input, input_row_stride, num_rows, num_cols, codes, scales, g, s);
      break;
    case TKS_FLOAT16:
      launch_quantize<_Float16>(input, input_row_stride, num_rows, num_cols, codes, scales, g, s);
      break;
    default:
      launch_quantize<bf16_t>(input, input_row_stride, num_rows, num_cols, codes, scales, g, s);
      break;
  }
  return check_launch();
}

extern "C" int32_t tks_mxfp4_dequantize(const void *codes, const void *scales, int64_t num_rows,
                                        int64_t num_cols, void *out, int64_t out_row_stride,
                                        int32_t dtype, tks_stream_t stream) {
  if (!valid_dtype(dtype)) return TKS_ERR_TYPE;
  if (!rows_ok(num_rows, num_cols, codes)) return TKS_ERR_VALUE;
  if (num_rows == 0) return TKS_OK;
  if (!codes || !scales || !out) return TKS_ERR_VALUE;
  if (num_rows > INT64_MAX / 4 / num_cols) return TKS_ERR_VALUE;
  const int64_t grid = grid_of(num_rows * num_cols / 8);
  if (grid == 0) return TKS_ERR_VALUE;
  const unsigned g = static_cast<unsigned>(grid);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TKS_FLOAT32:
      launch_dequantize<float>(codes, scales, num_rows, num_cols, out, out_row_stride, g, s);
      break;
    case TKS_FLOAT16:
      launch_dequantize<_Float16>(codes, scales, num_rows, num_cols, out, out_row_stride, g, s);
      break;
    default:
      launch_dequantize<bf16_t>(codes, scales, num_rows, num_cols, out, out_row_stride, g, s);
      break;
  }
  return check_launch();
}
