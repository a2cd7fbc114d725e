// Products of MXFP4 matrices, out[m, n] = sum_k A[m, k] B[n, k], on the block-scaled matrix
// instructions: a lane of v_mfma_scale_f32_16x16x128_f8f6f4 holds 32 consecutive e2m1 codes
// of one row and their scale byte, i.e. one MXFP4 block, so codes and scales go from memory
// to the operands as they are stored. Lane 16 g + i holds row i and the g-th of four blocks;
// which four blocks of K those are is free as long as A and B agree. Products of two codes
// are exact in the accumulator; sums are fp32.
#include "mxfp4_matmul.hpp"

#include <algorithm>

namespace tks {
namespace {

// ------------------------------------------------------------------------
// Few rows: the weights stream from HBM straight to the operands.
// ------------------------------------------------------------------------

// One workgroup per 16 columns of the output and 16 MT rows of it, its waves taking chunks of
// 512 of K in turn (a lane then reads 64 consecutive bytes of its row, four blocks); their
// sums meet in LDS, in wave order.
constexpr int kChunk = 512;
constexpr int kWaves = 4;

struct Chunk {
  uint4 v[4];
  uint32_t s;
};

// Lane group g's four blocks of chunk `c` of a row: blocks past the row are zeros with scale 1.
__device__ __forceinline__ Chunk load_chunk(const uint8_t *codes, const uint8_t *scales,
                                            int64_t row, int64_t blocks, int64_t c, int g) {
  Chunk r;
  const int64_t first = c * (kChunk / kMxBlock) + 4 * g;
  const uint8_t *p = codes + (row * blocks + first) * 16;
  const uint8_t *s = scales + row * blocks + first;
  if (first + 4 <= blocks) {
#pragma unroll
    for (int j = 0; j < 4; ++j) r.v[j] = ld16(p + 16 * j);
    __builtin_memcpy(&r.s, s, 4);
  } else {
    r.s = 0x7f7f7f7fu;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r.v[j] = make_uint4(0, 0, 0, 0);
      if (first + j < blocks) {
        r.v[j] = ld16(p + 16 * j);
        r.s = (r.s & ~(0xffu << (8 * j))) | static_cast<uint32_t>(s[j]) << (8 * j);
      }
    }
  }
  return r;
}

template <typename T, int MT>
__global__ __launch_bounds__(64 * kWaves) void matmul_few_kernel(MatmulArgs p) {
  __shared__ mx_f4 part[kWaves][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, i = lane & 15;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * (16 * MT);
  const int64_t blocks = p.k / kMxBlock;
  const int64_t chunks = (p.k + kChunk - 1) / kChunk;
  const int64_t n = min(n0 + i, p.n - 1);  // rows past the last are not stored
  mx_f4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = mx_f4{0.f, 0.f, 0.f, 0.f};
  for (int64_t c = wave; c < chunks; c += kWaves) {
    const Chunk b = load_chunk(p.b, p.bs, n, blocks, c, g);
    Chunk a[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
      a[t] = load_chunk(p.a, p.as, min(m0 + 16 * t + i, p.m - 1), blocks, c, g);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      acc[t] = mx_mfma<0>(b.v[0], a[t].v[0], acc[t], b.s, a[t].s);
      acc[t] = mx_mfma<1>(b.v[1], a[t].v[1], acc[t], b.s, a[t].s);
      acc[t] = mx_mfma<2>(b.v[2], a[t].v[2], acc[t], b.s, a[t].s);
      acc[t] = mx_mfma<3>(b.v[3], a[t].v[3], acc[t], b.s, a[t].s);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) part[wave][t][lane] = acc[t];
  __syncthreads();
  for (int e = threadIdx.x; e < MT * 64; e += 64 * kWaves) {
    const int t = e >> 6, from = e & 63;
    mx_f4 sum = part[0][t][from];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) sum += part[w][t][from];
    const int64_t m = m0 + 16 * t + (from & 15);
    const int64_t col = n0 + 4 * (from >> 4);
    if (m >= p.m) continue;
    T *o = static_cast<T *>(p.out) + m * p.o_rs + col;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (col + r < p.n) o[r] = from_float<T>(sum[r]);
  }
}

template <typename T>
int32_t launch_few(const MatmulArgs &p, hipStream_t s) {
  const int mt = static_cast<int>(std::min<int64_t>(4, ceil_div(p.m, 16)));
  const int64_t gx = ceil_div(p.n, 16), gy = ceil_div(p.m, 16 * mt);
  if (gx > 0x7fffffff || gy > 65535) return TKS_ERR_VALUE;
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
  switch (mt) {
    case 1: matmul_few_kernel<T, 1><<<grid, 64 * kWaves, 0, s>>>(p); break;
    case 2: matmul_few_kernel<T, 2><<<grid, 64 * kWaves, 0, s>>>(p); break;
    case 3: matmul_few_kernel<T, 3><<<grid, 64 * kWaves, 0, s>>>(p); break;
    default: matmul_few_kernel<T, 4><<<grid, 64 * kWaves, 0, s>>>(p); break;
  }
  return check_launch();
}

// The rows from which the tiled kernel is used, and the K its 32-bit offsets reach.
constexpr int64_t kTileRows = 65;
constexpr int64_t kTileDepth = int64_t{1} << 24;
bool tiled(int64_t m, int64_t k) { return m >= kTileRows && k <= kTileDepth; }

int32_t launch_few_of(const MatmulArgs &p, int32_t dtype, hipStream_t s) {
  switch (dtype) {
    case TKS_FLOAT32: return launch_few<float>(p, s);
    case TKS_FLOAT16: return launch_few<_Float16>(p, s);
    default: return launch_few<bf16_t>(p, s);
  }
}

int64_t padded(int64_t bytes) { return ceil_div(bytes, 256) * 256; }

constexpr int64_t kMaxDim = int64_t{1} << 40;

bool shape_ok(int64_t m, int64_t n, int64_t k) {
  return m >= 0 && n >= 0 && k > 0 && k % kMxBlock == 0 && m <= kMaxDim / k && n <= kMaxDim / k;
}

bool workspace_ok(const void *workspace, int64_t bytes, int64_t needed) {
  return needed == 0 || (workspace != nullptr && aligned16(workspace) && bytes >= needed);
}

}  // namespace
}  // namespace tks

using namespace tks;

// Both scales in window order, for the tiled kernel.
extern "C" int64_t tks_mxfp4_matmul_workspace_bytes(int64_t num_rows, int64_t num_cols,
                                                    int64_t depth) {
  if (!shape_ok(num_rows, num_cols, depth)) return -1;
  if (!tiled(num_rows, depth) || num_cols == 0) return 0;
  return padded(window_scale_bytes(num_rows, depth)) + window_scale_bytes(num_cols, depth);
}

extern "C" int32_t tks_mxfp4_matmul(const void *a_codes, const void *a_scales,
                                    const void *b_codes, const void *b_scales, int64_t num_rows,
                                    int64_t num_cols, int64_t depth, void *out,
                                    int64_t out_row_stride, void *workspace,
                                    int64_t workspace_bytes, int32_t dtype, tks_stream_t stream) {
  if (!valid_dtype(dtype)) return TKS_ERR_TYPE;
  if (!shape_ok(num_rows, num_cols, depth)) return TKS_ERR_VALUE;
  if (num_rows == 0 || num_cols == 0) return TKS_OK;
  if (!a_codes || !a_scales || !b_codes || !b_scales || !out || !aligned16(a_codes) ||
      !aligned16(b_codes))
    return TKS_ERR_VALUE;
  if (!workspace_ok(workspace, workspace_bytes,
                    tks_mxfp4_matmul_workspace_bytes(num_rows, num_cols, depth)))
    return TKS_ERR_WORKSPACE;
  MatmulArgs p{static_cast<const uint8_t *>(a_codes), static_cast<const uint8_t *>(a_scales),
               static_cast<const uint8_t *>(b_codes), static_cast<const uint8_t *>(b_scales),
               num_rows, num_cols, depth, out, out_row_stride};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!tiled(num_rows, depth)) return launch_few_of(p, dtype, s);
  uint8_t *as = static_cast<uint8_t *>(workspace);
  uint8_t *bs = as + padded(window_scale_bytes(num_rows, depth));
  int32_t st = launch_window_scales(p.as, num_rows, depth, as, s);
  if (st == TKS_OK) st = launch_window_scales(p.bs, num_cols, depth, bs, s);
  if (st != TKS_OK) return st;
  p.as = as;
  p.bs = bs;
  return launch_matmul_tiles(p, dtype, s);
}

// The rows' codes and their scales (in window order for the tiled kernel, which takes the
// weight's so too).
extern "C" int64_t tks_mxfp4_linear_workspace_bytes(int64_t num_rows, int64_t num_cols,
                                                    int64_t depth) {
  if (!shape_ok(num_rows, num_cols, depth)) return -1;
  if (num_rows == 0 || num_cols == 0) return 0;
  const int64_t codes = padded(num_rows * depth / 2);
  if (!tiled(num_rows, depth)) return codes + num_rows * (depth / kMxBlock);
  return codes + padded(window_scale_bytes(num_rows, depth)) + window_scale_bytes(num_cols, depth);
}

extern "C" int32_t tks_mxfp4_linear(const void *input, int64_t input_row_stride,
                                    const void *weight_codes, const void *weight_scales,
                                    int64_t num_rows, int64_t num_cols, int64_t depth, void *out,
                                    int64_t out_row_stride, void *workspace,
                                    int64_t workspace_bytes, int32_t dtype, tks_stream_t stream) {
  if (!valid_dtype(dtype)) return TKS_ERR_TYPE;
  if (!shape_ok(num_rows, num_cols, depth)) return TKS_ERR_VALUE;
  if (num_rows == 0 || num_cols == 0) return TKS_OK;
  if (!input || !weight_codes || !weight_scales || !out || !aligned16(weight_codes))
    return TKS_ERR_VALUE;
  if (!workspace_ok(workspace, workspace_bytes,
                    tks_mxfp4_linear_workspace_bytes(num_rows, num_cols, depth)))
    return TKS_ERR_WORKSPACE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint8_t *codes = static_cast<uint8_t *>(workspace);
  uint8_t *as = codes + padded(num_rows * depth / 2);
  MatmulArgs p{codes, as, static_cast<const uint8_t *>(weight_codes),
               static_cast<const uint8_t *>(weight_scales), num_rows, num_cols, depth, out,
               out_row_stride};
  if (!tiled(num_rows, depth)) {
    const int32_t st = tks_mxfp4_quantize(input, input_row_stride, num_rows, depth, codes, as,
                                          dtype, stream);
    return st != TKS_OK ? st : launch_few_of(p, dtype, s);
  }
  uint8_t *bs = as + padded(window_scale_bytes(num_rows, depth));
  const int32_t st = launch_quantize_windows(input, input_row_stride, num_rows, depth, codes, as,
                                             p.bs, num_cols, bs, dtype, s);
  if (st != TKS_OK) return st;
  p.bs = bs;
  return launch_matmul_tiles(p, dtype, s);
}
