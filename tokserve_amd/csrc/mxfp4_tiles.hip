// The tiled MXFP4 product, for more rows than the weights' stream alone would pay for.
//
// A workgroup of 2 x 2 waves computes 32 MI x 32 NI of the output, a wave 16 MI x 16 NI: K in
// steps of 128, one v_mfma_scale 16x16x128 per pair of 16-row tiles. A's codes go through LDS
// (both waves of a row of waves read them), B's from L2 straight to the operands: either path
// alone, LDS or the vector cache, would be the bound. Nothing is waited for in the step that
// asks for it. In step s
//   - A's codes of step s + 1 go from LDS to the operands of the next step,
//   - those of step s + 2, in registers since step s - 1, go to LDS, and those of s + 3 are asked
//     for in their place,
//   - B's operands of step s + 1 are asked for,
// while the matrix unit works on step s; a barrier ends it. The LDS ring has four slots and
// the steps are unrolled by four: a scale dword holds a row's bytes of four steps (one window,
// mxfp4_matmul.hpp), which the instruction picks its byte from.
//
// Past K the codes read are those of the last block, and both scales 2^-127, whose product
// with any two codes is below the smallest fp32: adding it changes nothing.
#include "mxfp4_matmul.hpp"

#include <algorithm>

namespace tks {
namespace {

constexpr int kThreads = 256;

// Workgroup -> tile: the workgroups of an XCD (every eighth) take neighbouring tiles, in
// columns of `kBand` tile rows, so that the tiles its L2 holds are read by many of them.
constexpr int kXcds = 8;
constexpr int kBand = 8;
__device__ __forceinline__ void tile_of(int64_t id, int64_t tiles_m, int64_t tiles_n, int64_t *tm,
                                        int64_t *tn) {
  const int64_t total = tiles_m * tiles_n;
  const int64_t per = total / kXcds, rest = total % kXcds;
  const int64_t x = id % kXcds;
  const int64_t t = x * per + min(x, rest) + id / kXcds;
  const int64_t band = t / (kBand * tiles_n);
  const int64_t rows = min(static_cast<int64_t>(kBand), tiles_m - band * kBand);
  const int64_t in = t - band * kBand * tiles_n;
  *tm = band * kBand + in % rows;
  *tn = in / rows;
}

template <typename T, int MI, int NI, bool VEC>
__global__ __launch_bounds__(kThreads) void matmul_tiles_kernel(MatmulArgs p, int64_t tiles_m,
                                                                int64_t tiles_n) {
  constexpr int BM = 32 * MI, BN = 32 * NI;
  constexpr int kSlots = 4;
  constexpr int kStage = BM * 64 / 16 / kThreads;  // 16-byte pieces of an A step per thread
  static_assert(kStage * 16 * kThreads == BM * 64, "whole pieces");
  __shared__ __align__(16) uint8_t ring[kSlots][BM * 64];

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, i = lane & 15;
  const int wm = wave >> 1, wn = wave & 1;
  int64_t tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, &tm, &tn);
  const int64_t m0 = tm * BM, n0 = tn * BN;
  const int last_m = static_cast<int>(min<int64_t>(p.m - m0, BM)) - 1;
  const int last_n = static_cast<int>(min<int64_t>(p.n - n0, BN)) - 1;
  const int row_bytes = static_cast<int>(p.k / 2);
  const int blocks = static_cast<int>(p.k / kMxBlock);
  const int wins = static_cast<int>(windows(p.k));
  const uint8_t *a = p.a + m0 * row_bytes;
  const uint8_t *b = p.b + n0 * row_bytes;

  // A's piece q of this thread: row t / 4 + 64 q, block t % 4 of the step. In LDS a row's four
  // blocks are permuted by its bits 2 and 3, so that the 16 rows of an operand read touch all
  // banks once.
  uint32_t a_off[kStage];
  int a_lds[kStage];
  const int piece = threadIdx.x & 3;
#pragma unroll
  for (int q = 0; q < kStage; ++q) {
    const int row = (threadIdx.x >> 2) + 64 * q;
    a_off[q] = static_cast<uint32_t>(min(row, last_m)) * row_bytes;
    a_lds[q] = row * 64 + 16 * (piece ^ ((row >> 2) & 3));
  }
  const int read_at = (16 * MI * wm + i) * 64 + 16 * (g ^ ((i >> 2) & 3));
  uint32_t b_off[NI];
#pragma unroll
  for (int t = 0; t < NI; ++t)
    b_off[t] = static_cast<uint32_t>(min(16 * (NI * wn + t) + i, last_n)) * row_bytes;
  // (Scales are padded to whole tiles of rows: those past the last are read and not used.)
  const uint8_t *as = p.as + (m0 + 16 * MI * wm) * 16;
  const uint8_t *bs = p.bs + (n0 + 16 * NI * wn) * 16;
  const uint32_t s_off = 16 * i + 4 * g;

  uint4 stage[kStage], af[2][MI], bf[2][NI];
  uint32_t sa[MI], sb[NI], sa_next[MI], sb_next[NI];
  mx_f4 acc[MI][NI];
#pragma unroll
  for (int x = 0; x < MI; ++x)
#pragma unroll
    for (int y = 0; y < NI; ++y) acc[x][y] = mx_f4{0.f, 0.f, 0.f, 0.f};

  auto fetch_a = [&](int step) {
    const uint32_t at = 16u * static_cast<uint32_t>(min(4 * step + piece, blocks - 1));
#pragma unroll
    for (int q = 0; q < kStage; ++q) stage[q] = ld16(a + (a_off[q] + at));
  };
  auto put_a = [&](int slot) {
#pragma unroll
    for (int q = 0; q < kStage; ++q) st16(&ring[slot][a_lds[q]], stage[q]);
  };
  auto get_a = [&](int slot, uint4 *f) {
#pragma unroll
    for (int t = 0; t < MI; ++t) f[t] = ld16(&ring[slot][read_at + 1024 * t]);
  };
  auto fetch_b = [&](int step, uint4 *f) {
    const uint32_t at = 16u * static_cast<uint32_t>(min(4 * step + g, blocks - 1));
#pragma unroll
    for (int t = 0; t < NI; ++t) f[t] = ld16(b + (b_off[t] + at));
  };
  auto fetch_scales = [&](uint32_t *xa, uint32_t *xb) {
#pragma unroll
    for (int t = 0; t < MI; ++t) xa[t] = *reinterpret_cast<const uint32_t *>(as + (s_off + 256 * t));
#pragma unroll
    for (int t = 0; t < NI; ++t) xb[t] = *reinterpret_cast<const uint32_t *>(bs + (s_off + 256 * t));
  };

  fetch_scales(sa, sb);
  fetch_a(0);
  put_a(0);
  fetch_a(1);
  fetch_b(0, bf[0]);
  put_a(1);
  fetch_a(2);
  __syncthreads();
  get_a(0, af[0]);

#define TKS_STEP(T4)                                                                           \
  {                                                                                            \
    constexpr int cur = T4 & 1, nxt = cur ^ 1;                                                 \
    get_a((T4 + 1) & 3, af[nxt]);                                                              \
    fetch_b(step + T4 + 1, bf[nxt]);                                                           \
    put_a((T4 + 2) & 3);                                                                       \
    fetch_a(step + T4 + 3);                                                                    \
    _Pragma("unroll") for (int x = 0; x < MI; ++x) {                                           \
      _Pragma("unroll") for (int y = 0; y < NI; ++y)                                           \
          acc[x][y] = mx_mfma<T4>(bf[cur][y], af[cur][x], acc[x][y], sb[y], sa[x]);            \
    }                                                                                          \
    __syncthreads();                                                                           \
  }
  for (int win = 0; win < wins; ++win) {
    if (win + 1 < wins) {
      as += p.m * 16;
      bs += p.n * 16;
    }
    fetch_scales(sa_next, sb_next);
    const int step = 4 * win;
    TKS_STEP(0)
    TKS_STEP(1)
    TKS_STEP(2)
    TKS_STEP(3)
#pragma unroll
    for (int t = 0; t < MI; ++t) sa[t] = sa_next[t];
#pragma unroll
    for (int t = 0; t < NI; ++t) sb[t] = sb_next[t];
  }
#undef TKS_STEP

  T *out = static_cast<T *>(p.out) + m0 * p.o_rs + n0;
#pragma unroll
  for (int x = 0; x < MI; ++x) {
    const int row = 16 * (MI * wm + x) + i;
    if (row > last_m) continue;
    T *o = out + row * p.o_rs;
#pragma unroll
    for (int y = 0; y < NI; ++y) {
      const int col = 16 * (NI * wn + y) + 4 * g;
      if constexpr (VEC) {
        if (col > last_n) continue;
        T v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = from_float<T>(acc[x][y][r]);
        __builtin_memcpy(__builtin_assume_aligned(o + col, 4 * sizeof(T)), v, sizeof(v));
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (col + r <= last_n) o[col + r] = from_float<T>(acc[x][y][r]);
      }
    }
  }
}

// ------------------------------------------------------------------------
// Window-ordered scales
// ------------------------------------------------------------------------

// Row r's window w: 16 bytes, zeros past K.
__device__ __forceinline__ void window_scales(const uint8_t *scales, int64_t rows, int64_t blocks,
                                              int64_t item, uint8_t *out) {
  const int64_t w = item / rows, r = item - w * rows;
  const uint8_t *s = scales + r * blocks + 16 * w;
  const int left = static_cast<int>(min<int64_t>(blocks - 16 * w, 16));
  uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (j < left) v[j & 3] |= static_cast<uint32_t>(s[j]) << (8 * (j >> 2));
  st16(out + item * 16, make_uint4(v[0], v[1], v[2], v[3]));
}

__global__ __launch_bounds__(kThreads) void window_scales_kernel(const uint8_t *scales,
                                                                 int64_t rows, int64_t blocks,
                                                                 int64_t total, uint8_t *out) {
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (item < total) window_scales(scales, rows, blocks, item, out);
}

// The first `quant` workgroups quantize (a thread eight values, kItems times), the others put
// B's scales in order.
constexpr int kItems = 4;
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void quantize_windows_kernel(
    const T *__restrict__ x, int64_t rs, int64_t m, int64_t eights, uint32_t *__restrict__ codes,
    uint8_t *__restrict__ scales, int64_t quant, const uint8_t *__restrict__ b_scales, int64_t n,
    uint8_t *__restrict__ b_out) {
  const int64_t blocks = eights / 4;
  if (blockIdx.x >= quant) {
    const int64_t item = (blockIdx.x - quant) * kThreads + threadIdx.x;
    if (item < n * windows(blocks * kMxBlock)) window_scales(b_scales, n, blocks, item, b_out);
    return;
  }
  const int64_t total = m * eights;
  MxEight<T> v[kItems];
  int64_t row[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int64_t at = (static_cast<int64_t>(blockIdx.x) * kItems + i) * kThreads + threadIdx.x;
    row[i] = at / eights;
    if (at >= total) continue;
    const T *src = x + row[i] * rs + (at - row[i] * eights) * 8;
    v[i] = VEC ? mx_load8<T>(src) : mx_load8_any<T>(src);
  }
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int64_t at = (static_cast<int64_t>(blockIdx.x) * kItems + i) * kThreads + threadIdx.x;
    if (at >= total) continue;
    uint32_t s;
    codes[at] = mx_quantize<T>(v[i], &s);
    const int64_t block = (at - row[i] * eights) >> 2;
    const int sub = threadIdx.x & 3;
    if (sub == 0) scales[window_scale_at(block, row[i], m)] = static_cast<uint8_t>(s);
    if (block == blocks - 1)  // zeros up to the window's end, a quarter of them each
      for (int64_t z = blocks + sub; z < ((blocks + 15) & ~int64_t{15}); z += 4)
        scales[window_scale_at(z, row[i], m)] = 0;
  }
}

template <typename T, int MI, int NI>
void launch_tiles(const MatmulArgs &p, hipStream_t s) {
  const int64_t tm = ceil_div(p.m, 32 * MI), tn = ceil_div(p.n, 32 * NI);
  const unsigned grid = static_cast<unsigned>(tm * tn);
  const bool vec = p.n % 4 == 0 && p.o_rs % 4 == 0 &&
                   reinterpret_cast<uintptr_t>(p.out) % (4 * sizeof(T)) == 0;
  if (vec)
    matmul_tiles_kernel<T, MI, NI, true><<<grid, kThreads, 0, s>>>(p, tm, tn);
  else
    matmul_tiles_kernel<T, MI, NI, false><<<grid, kThreads, 0, s>>>(p, tm, tn);
}

template <typename T>
int32_t launch(const MatmulArgs &p, hipStream_t s) {
  if (ceil_div(p.m, 64) > 0x7fffffff / ceil_div(p.n, 64)) return TKS_ERR_VALUE;
  const int64_t tiles = ceil_div(p.m, 256) * ceil_div(p.n, 256);
  const int64_t half = ceil_div(p.m, 128) * ceil_div(p.n, 128);
  if (tiles >= 200)
    launch_tiles<T, 8, 8>(p, s);
  else if (half >= 200)
    launch_tiles<T, 4, 4>(p, s);
  else
    launch_tiles<T, 2, 2>(p, s);
  return check_launch();
}

}  // namespace

int32_t launch_matmul_tiles(const MatmulArgs &p, int32_t dtype, hipStream_t s) {
  switch (dtype) {
    case TKS_FLOAT32: return launch<float>(p, s);
    case TKS_FLOAT16: return launch<_Float16>(p, s);
    default: return launch<bf16_t>(p, s);
  }
}

int32_t launch_window_scales(const uint8_t *scales, int64_t rows, int64_t k, uint8_t *out,
                             hipStream_t s) {
  const int64_t total = rows * windows(k);
  if (ceil_div(total, kThreads) > 0x7fffffff) return TKS_ERR_VALUE;
  window_scales_kernel<<<static_cast<unsigned>(ceil_div(total, kThreads)), kThreads, 0, s>>>(
      scales, rows, k / kMxBlock, total, out);
  return check_launch();
}

int32_t launch_quantize_windows(const void *x, int64_t x_rs, int64_t m, int64_t k, uint8_t *codes,
                                uint8_t *scales, const uint8_t *b_scales, int64_t n,
                                uint8_t *b_out, int32_t dtype, hipStream_t s) {
  const int64_t quant = ceil_div(m * (k / 8), kThreads * kItems);
  const int64_t grid = quant + ceil_div(n * windows(k), kThreads);
  if (grid > 0x7fffffff) return TKS_ERR_VALUE;
  const bool vec = aligned16(x) && x_rs * elem_bytes(dtype) % 16 == 0;
  const unsigned g = static_cast<unsigned>(grid);
  uint32_t *c = reinterpret_cast<uint32_t *>(codes);
#define TKS_QUANT(TYPE)                                                                        \
  if (vec)                                                                                     \
    quantize_windows_kernel<TYPE, true><<<g, kThreads, 0, s>>>(                                \
        static_cast<const TYPE *>(x), x_rs, m, k / 8, c, scales, quant, b_scales, n, b_out);   \
  else                                                                                         \
    quantize_windows_kernel<TYPE, false><<<g, kThreads, 0, s>>>(                               \
        static_cast<const TYPE *>(x), x_rs, m, k / 8, c, scales, quant, b_scales, n, b_out)
  switch (dtype) {
    case TKS_FLOAT32: TKS_QUANT(float); break;
    case TKS_FLOAT16: TKS_QUANT(_Float16); break;
    default: TKS_QUANT(bf16_t); break;
  }
#undef TKS_QUANT
  return check_launch();
}

}  // namespace tks
