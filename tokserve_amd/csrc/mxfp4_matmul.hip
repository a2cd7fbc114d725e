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
// 512 of K in turn, four blocks of its row a lane; their
// sums meet in LDS, in wave order. (With a chunk's loads issued a chunk ahead: no faster but for
// one row of a long K, 11008 -> 4096 13.0 -> 9.6 us, and 16 rows 4096 -> 8192 8.3 -> 9.4.) With ROWS the activations come as they are and each lane
// quantizes the four blocks it needs: all the workgroups do that work again, a fraction of a
// microsecond of it, and a launch is saved.
constexpr int kChunk = 512;
constexpr int kWaves = 4;

struct Chunk {
  uint4 v[4];
  uint32_t s;
};

// Lane group g's four blocks of chunk `c` of a row, 4 j + g for j = 0 .. 3 (the lanes of a row
// then read 64 consecutive bytes at a time); blocks past the row are zeros with scale 1.
__device__ __forceinline__ Chunk load_chunk(const uint8_t *codes, const uint8_t *scales,
                                            int64_t row, int64_t blocks, int64_t c, int g) {
  Chunk r;
  const int64_t first = c * (kChunk / kMxBlock);
  const uint8_t *p = codes + (row * blocks + first + g) * 16;
  const uint8_t *s = scales + row * blocks + first;
  if (first + 16 <= blocks) {
    uint32_t w[4];
    __builtin_memcpy(w, s, 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) r.v[j] = ld16(p + 64 * j);
    // Byte g of each of the four words.
    const uint32_t pick = 0x0c0c0400u + 0x0101u * g;
    r.s = __builtin_amdgcn_perm(w[1], w[0], pick) |
          __builtin_amdgcn_perm(w[3], w[2], pick) << 16;
  } else {
    r.s = 0x7f7f7f7fu;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r.v[j] = make_uint4(0, 0, 0, 0);
      if (first + 4 * j + g < blocks) {
        r.v[j] = ld16(p + 64 * j);
        r.s = (r.s & ~(0xffu << (8 * j))) | static_cast<uint32_t>(s[4 * j + g]) << (8 * j);
      }
    }
  }
  return r;
}

// The same of a row of values.
template <typename T>
__device__ __forceinline__ Chunk quantize_chunk(const T *row, int64_t blocks, int64_t c, int g) {
  Chunk r;
  r.s = 0;
  const int64_t first = c * (kChunk / kMxBlock) + g;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t s = 127;
    r.v[j] = make_uint4(0, 0, 0, 0);
    if (first + 4 * j < blocks) {
      MxEight<T> x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = mx_load8<T>(row + (first + 4 * j) * kMxBlock + 8 * e);
      r.v[j] = mx_quantize_block<T>(x, &s);
    }
    r.s |= s << (8 * j);
  }
  return r;
}

struct FewArgs {
  MatmulArgs p;
  const void *x;  // ROWS: (M, K) values
  int64_t x_rs;
  bool vec;  // output rows can be stored four values at a time
};

template <typename T, int MT, int NT, bool ROWS>
__global__ __launch_bounds__(64 * kWaves) void matmul_few_kernel(FewArgs f) {
  const MatmulArgs &p = f.p;
  __shared__ mx_f4 part[kWaves][MT][NT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, i = lane & 15;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * NT);
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * (16 * MT);
  const int64_t blocks = p.k / kMxBlock;
  const int64_t chunks = (p.k + kChunk - 1) / kChunk;
  mx_f4 acc[MT][NT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) acc[t][u] = mx_f4{0.f, 0.f, 0.f, 0.f};
  for (int64_t c = wave; c < chunks; c += kWaves) {
    // (Rows past the last are read as the last and not stored.)
    Chunk b[NT], a[MT];
#pragma unroll
    for (int u = 0; u < NT; ++u)
      b[u] = load_chunk(p.b, p.bs, min(n0 + 16 * u + i, p.n - 1), blocks, c, g);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int64_t m = min(m0 + 16 * t + i, p.m - 1);
      if constexpr (ROWS)
        a[t] = quantize_chunk<T>(static_cast<const T *>(f.x) + m * f.x_rs, blocks, c, g);
      else
        a[t] = load_chunk(p.a, p.as, m, blocks, c, g);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        acc[t][u] = mx_mfma<0>(b[u].v[0], a[t].v[0], acc[t][u], b[u].s, a[t].s);
        acc[t][u] = mx_mfma<1>(b[u].v[1], a[t].v[1], acc[t][u], b[u].s, a[t].s);
        acc[t][u] = mx_mfma<2>(b[u].v[2], a[t].v[2], acc[t][u], b[u].s, a[t].s);
        acc[t][u] = mx_mfma<3>(b[u].v[3], a[t].v[3], acc[t][u], b[u].s, a[t].s);
      }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) part[wave][t][u][lane] = acc[t][u];
  __syncthreads();
  for (int e = threadIdx.x; e < MT * NT * 64; e += 64 * kWaves) {
    const int t = e / (64 * NT), u = e / 64 % NT, from = e & 63;
    mx_f4 sum = part[0][t][u][from];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) sum += part[w][t][u][from];
    const int64_t m = m0 + 16 * t + (from & 15);
    const int64_t col = n0 + 16 * u + 4 * (from >> 4);
    if (m >= p.m) continue;
    T *o = static_cast<T *>(p.out) + m * p.o_rs + col;
    T v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = from_float<T>(sum[r]);
    if (f.vec && col + 4 <= p.n) {
      __builtin_memcpy(__builtin_assume_aligned(o, 4 * sizeof(T)), v, sizeof(v));
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (col + r < p.n) o[r] = v[r];
    }
  }
}

template <typename T, int MT, int NT, bool ROWS>
int32_t launch_few_kernel(const FewArgs &f, hipStream_t s) {
  const int64_t gx = ceil_div(f.p.n, 16 * NT), gy = ceil_div(f.p.m, 16 * MT);
  if (gx > 0x7fffffff || gy > 65535) return TKS_ERR_VALUE;
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
  matmul_few_kernel<T, MT, NT, ROWS><<<grid, 64 * kWaves, 0, s>>>(f);
  return check_launch();
}

// Where there are columns enough for every CU, two tiles of them share what is read of A. us
// with one and with two, of 48 rows: 2048 -> 2560 4.4 and 5.3, 2048 -> 11264 9.4 and 8.5, 4096 ->
// 8192 12.0 and 9.3 (16 rows of it 7.2 and 6.3). Eight waves instead of four: level.
constexpr int64_t kWideCols = 8192;
template <typename T, int MT, bool ROWS>
int32_t launch_few_mt(const FewArgs &f, hipStream_t s) {
  if constexpr (!ROWS)
    if (f.p.n >= kWideCols) return launch_few_kernel<T, MT, 2, ROWS>(f, s);
  return launch_few_kernel<T, MT, 1, ROWS>(f, s);
}

template <typename T, bool ROWS>
int32_t launch_few(const FewArgs &f, hipStream_t s) {
  if constexpr (ROWS) {
    return launch_few_mt<T, 1, ROWS>(f, s);
  } else {
    switch (std::min<int64_t>(4, ceil_div(f.p.m, 16))) {
      case 1: return launch_few_mt<T, 1, ROWS>(f, s);
      case 2: return launch_few_mt<T, 2, ROWS>(f, s);
      case 3: return launch_few_mt<T, 3, ROWS>(f, s);
      default: return launch_few_mt<T, 4, ROWS>(f, s);
    }
  }
}

// The rows from which the tiled kernel is used, fewer where its 64 columns of a workgroup still
// are work for most CUs and K is short (48 rows: 2048 -> 11264 6.7 us, 8.5 below; 2048 -> 2560
// 4.7 and 4.4; 4096 -> 8192 10.1 and 9.3; 5632 -> 2048 12.7 and 8.0), and the K its 32-bit
// offsets reach.
constexpr int64_t kTileRows = 65, kTileRowsWide = 33, kTileDepthWide = 2048;
constexpr int64_t kTileDepth = int64_t{1} << 24;
bool tiled(int64_t m, int64_t n, int64_t k) {
  if (k > kTileDepth) return false;
  return m >= kTileRows || (m >= kTileRowsWide && n >= kWideCols && k <= kTileDepthWide);
}

// Whether a projection's product quantizes the rows itself: every 16 columns do so again. us so
// and in two launches, from a graph (eager a launch more costs the host 3 us): bf16 16 rows
// 2048 -> 2560 4.6 and 5.9, 2048 -> 11264 10.2 and 8.9; 4 rows -> 11264 7.1 and 7.9; one row ->
// 11264 6.7 and 6.5; fp32 4 rows -> 2560 4.3 and 5.5, 4096 -> 8192 11.4 and 8.9.
constexpr int64_t kRowsInPlace = 16;
constexpr int64_t kOutputsInPlace = 1 << 16;
bool in_place(const void *x, int64_t x_rs, int64_t m, int64_t n, int32_t dtype) {
  const int elem = elem_bytes(dtype);
  return m <= kRowsInPlace && m * n <= (elem == 2 ? kOutputsInPlace : kOutputsInPlace / 4) &&
         aligned16(x) && x_rs * elem % 16 == 0;
}

// (x: the rows' values, or null where p holds their codes.)
template <typename T>
int32_t launch_few_of(const FewArgs &f, hipStream_t s) {
  return f.x ? launch_few<T, true>(f, s) : launch_few<T, false>(f, s);
}
int32_t launch_few_dtype(const MatmulArgs &p, const void *x, int64_t x_rs, int32_t dtype,
                         hipStream_t s) {
  const int four = 4 * elem_bytes(dtype);
  const FewArgs f{p, x, x_rs,
                  reinterpret_cast<uintptr_t>(p.out) % four == 0 && p.o_rs % 4 == 0};
  switch (dtype) {
    case TKS_FLOAT32: return launch_few_of<float>(f, s);
    case TKS_FLOAT16: return launch_few_of<_Float16>(f, s);
    default: return launch_few_of<bf16_t>(f, s);
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

// Both scales in window order, for the tiled kernel. (Putting A's in order is a launch that a
// projection does not have: the tiles pay from kTileRows rows on only.)
extern "C" int64_t tks_mxfp4_matmul_workspace_bytes(int64_t num_rows, int64_t num_cols,
                                                    int64_t depth) {
  if (!shape_ok(num_rows, num_cols, depth)) return -1;
  if (num_cols == 0 || !tiled(num_rows, 0, depth)) return 0;
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
  if (!tiled(num_rows, 0, depth)) return launch_few_dtype(p, nullptr, 0, dtype, s);
  uint8_t *as = static_cast<uint8_t *>(workspace);
  uint8_t *bs = as + padded(window_scale_bytes(num_rows, depth));
  const int32_t st =
      launch_window_scales(p.as, num_rows, as, p.bs, num_cols, bs, depth, s);
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
  if (!tiled(num_rows, num_cols, depth)) return codes + num_rows * (depth / kMxBlock);
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
  if (!tiled(num_rows, num_cols, depth)) {
    if (in_place(input, input_row_stride, num_rows, num_cols, dtype))
      return launch_few_dtype(p, input, input_row_stride, dtype, s);
    const int32_t st = tks_mxfp4_quantize(input, input_row_stride, num_rows, depth, codes, as,
                                          dtype, stream);
    return st != TKS_OK ? st : launch_few_dtype(p, nullptr, 0, dtype, s);
  }
  uint8_t *bs = as + padded(window_scale_bytes(num_rows, depth));
  const int32_t st = launch_quantize_windows(input, input_row_stride, num_rows, depth, codes, as,
                                             p.bs, num_cols, bs, dtype, s);
  if (st != TKS_OK) return st;
  p.bs = bs;
  return launch_matmul_tiles(p, dtype, s);
}
