// The tiled MXFP4 product, for more rows than the weights' stream alone would pay for.
//
// A workgroup of 2 x 2 waves computes 32 MI x 32 NI of the output, a wave 16 MI x 16 NI: one
// v_mfma_scale 16x16x128 per pair of 16-row tiles and 128 of K. Codes and scales go from L2 to
// LDS without passing through registers, in units of 256 of K (128 bytes of a row: requests of
// whole cache lines; in units of 128 the same loads reach half the rate, 31 against 60 bytes
// per clock and CU), two units and the scales of two windows (mxfp4_matmul.hpp) at a time.
//
// A unit is two phases. While the matrix unit works on one, the operands of the next are read
// from LDS: all of B's into a second set of registers, each of A's into the registers of the
// one that was just used. So a unit's last LDS read is in its first phase, and in its second
// its LDS is filled again, two units ahead, a few loads after each row of products. A barrier
// per unit makes the next unit's codes visible and this one's LDS free.
//
// What bounds it: at 8192 x 8192 x 4096, 164 - 183 us (3.0 - 3.4 PFLOP/s), 155 without the
// stores; of the matrix unit's nominal rate that is a third, of the rate that it keeps up in
// this loop without loads (power: the clock falls) six tenths. Tiles of 256 x 256, one wave
// per SIMD, take 186 us, since nothing covers a tile's first loads and its stores; two
// workgroups of 128 x 128 per CU cover each other's.
//
// With few tiles a workgroup is four such groups of waves (below).
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

// 16 bytes per lane from base + off to LDS address `to` (wave-uniform) + 16 * lane. As asm, so
// that the compiler, which cannot tell the ring's slots apart, does not make every LDS read
// wait for it: unit_barrier waits, and nothing else in the loop counts as such a load.
__device__ __forceinline__ void load_lds_async(const uint8_t *base, uint32_t off, uint32_t to) {
#if __HIP_DEVICE_COMPILE__
  // (A wait state between the write of m0 and its use.)
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off),
               "s"(base), "s"(to)
               : "memory", "m0");
#else
  (void)base; (void)off; (void)to;
#endif
}

// The wave's loads into LDS are there, its LDS reads done, and so those of the others.
__device__ __forceinline__ void unit_barrier() {
#if __HIP_DEVICE_COMPILE__
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#endif
}

// mx_mfma<SEL> with the sum in place, in accumulation registers (left to itself the compiler
// moves them about: 2048 x 11264 x 2048 36.8 -> 54.7 us).
// The compiler does not see what the instruction needs around it: the wait states after a
// VALU write of an operand are here, those before a VALU read of a sum are settle_sums.
template <int SEL>
__device__ __forceinline__ void mfma_in_place(uint4 b4, uint4 a4, mx_f4 &c, uint32_t sb,
                                              uint32_t sa) {
#if __HIP_DEVICE_COMPILE__
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  const u4 b = {b4.x, b4.y, b4.z, b4.w}, a = {a4.x, a4.y, a4.z, a4.w};
#define TKS_MFMA(sel)                                                                          \
  asm volatile("s_nop 1\n\tv_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 " sel                \
      " cbsz:4 blgp:4"                                                                         \
      : "+a"(c)                                                                                \
      : "v"(b), "v"(a), "v"(sb), "v"(sa))
  if constexpr (SEL == 0) TKS_MFMA("op_sel_hi:[0,0,0]");
  if constexpr (SEL == 1) TKS_MFMA("op_sel:[1,1,0] op_sel_hi:[0,0,0]");
  if constexpr (SEL == 2) TKS_MFMA("op_sel_hi:[1,1,0]");
  if constexpr (SEL == 3) TKS_MFMA("op_sel:[1,1,0] op_sel_hi:[1,1,0]");
#undef TKS_MFMA
#else
  (void)b4; (void)a4; (void)sb; (void)sa; (void)c;
#endif
}
// (In the loop's last round, not after it: what the compiler moves between the loop's registers
// and those of its exit comes right behind the loop.)
__device__ __forceinline__ void settle_sums() {
#if __HIP_DEVICE_COMPILE__
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#endif
}

// Four floats as 16-bit T, packed.
template <typename T>
__device__ __forceinline__ uint2 four16(mx_f4 f) {
  T t[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) t[r] = from_float<T>(f[r]);
  uint2 v;
  __builtin_memcpy(&v, t, 8);
  return v;
}
// Of lane groups g, g + 1 (g even): the first gets both groups' v, the second both groups' w.
__device__ __forceinline__ uint4 swap_halves(uint2 v, uint2 w) {
#if __HIP_DEVICE_COMPILE__
  const auto x = __builtin_amdgcn_permlane16_swap(v.x, w.x, false, false);
  const auto y = __builtin_amdgcn_permlane16_swap(v.y, w.y, false, false);
  return make_uint4(x[0], y[0], x[1], y[1]);
#else
  return make_uint4(v.x, v.y, w.x, w.y);
#endif
}

__device__ __forceinline__ uint32_t lds_base(const void *p) {
  return __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void *)p)));
}

// GROUPS: sets of 2 x 2 waves that take the windows of K in turn, each with LDS of its own;
// their sums meet in LDS, in the groups' order.
template <typename T, int MI, int NI, int GROUPS, bool VEC>
__global__ __launch_bounds__(kThreads *GROUPS, 1) void matmul_tiles_kernel(MatmulArgs p,
                                                                           int64_t tiles_m,
                                                                           int64_t tiles_n) {
  constexpr int BM = 32 * MI, BN = 32 * NI, kRows = BM + BN;
  constexpr int kUnitBytes = kRows * 128;
  constexpr int kLoads = kRows / 32;                // a wave's loads of a unit, 8 rows each
  constexpr int kPart = (kLoads + MI - 1) / MI;     // of them after each row of products
  static_assert(kRows % 64 == 0 && GROUPS >= 1, "");
  static_assert(GROUPS == 1 || MI * NI * 4096 <= 2 * kUnitBytes, "");  // the sums meet there
  __shared__ __align__(1024) uint8_t rings[GROUPS][2][kUnitBytes];
  __shared__ __align__(1024) uint8_t scale_rings[GROUPS][2][kRows * 16];

  const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) & 3;
  const int uw = __builtin_amdgcn_readfirstlane(wave);
  const int group = GROUPS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  uint8_t(*ring)[kUnitBytes] = rings[group];
  uint8_t(*scale_ring)[kRows * 16] = scale_rings[group];
  const int g = lane >> 4, i = lane & 15;
  const int wm = wave >> 1, wn = wave & 1;
  const int row_bytes = static_cast<int>(p.k / 2);
  const int blocks = static_cast<int>(p.k / kMxBlock);
  const int wins = static_cast<int>(windows(p.k));

  // In LDS the eight blocks of a row (of a unit) are permuted by its bits 1 to 3, so that the 16
  // rows of an operand read fall on different banks. Load q of a wave is rows 8 (4 q + wave) and
  // up: lane's row is lane / 8 of them, and its block the one whose place lane % 8 is.
  const int load_block = (lane & 7) ^ ((lane >> 4) & 3) ^ ((wave & 1) << 2);
  const int perm = (i >> 1) & 7;
  const int place[2] = {16 * (g ^ perm), 16 * ((4 + g) ^ perm)};  // of a phase's block
  const int read_a = (16 * MI * wm + i) * 128, read_b = (BM + 16 * NI * wn + i) * 128;
  const int read_sa = (16 * MI * wm + i) * 16 + 4 * g;
  const int read_sb = (BM + 16 * NI * wn + i) * 16 + 4 * g;
  const uint32_t ring_at = lds_base(&ring[0][0]), scale_at = lds_base(&scale_ring[0][0]);

  int64_t tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, &tm, &tn);
  const int64_t m0 = tm * BM, n0 = tn * BN;
  const int last_m = static_cast<int>(min<int64_t>(p.m - m0, BM)) - 1;
  const int last_n = static_cast<int>(min<int64_t>(p.n - n0, BN)) - 1;
  const uint8_t *a = p.a + m0 * row_bytes, *b = p.b + n0 * row_bytes;
  const uint8_t *as = p.as + m0 * 16, *bs = p.bs + n0 * 16;
  uint32_t off[kLoads];
#pragma unroll
  for (int q = 0; q < kLoads; ++q) {
    const int row = 8 * (4 * q + wave) + (lane >> 3);
    off[q] = static_cast<uint32_t>(32 * q < BM ? min(row, last_m) : min(row - BM, last_n)) *
             row_bytes;
  }
  // (Windows and units are counted within the group.)
  auto window_of = [&](int win) { return GROUPS * win + group; };
  auto fetch = [&](int unit, int slot, int from, int to) {
    if (GROUPS > 1) unit = 2 * window_of(unit >> 1) + (unit & 1);
    const uint32_t at = 16u * static_cast<uint32_t>(min(8 * unit + load_block, blocks - 1));
#pragma unroll
    for (int q = 0; q < kLoads; ++q)
      if (q >= from && q < to)
        load_lds_async(32 * q < BM ? a : b, off[q] + at,
                       ring_at + slot * kUnitBytes + (4 * q + uw) * 1024);
  };
  auto fetch_scales = [&](int win) {
    const int64_t w = GROUPS > 1 ? min(window_of(win), wins - 1) : win;
    const uint8_t *wa = as + w * (p.m * 16), *wb = bs + w * (p.n * 16);
    const int row = 64 * uw;  // (BM is a multiple of 64)
    if (row < kRows)
      load_lds_async(row < BM ? wa : wb, static_cast<uint32_t>(16 * ((row < BM ? row : row - BM) + lane)),
                     scale_at + (win & 1) * (kRows * 16) + row * 16);
  };

  uint4 af[MI], bf[2][NI];
  uint32_t sa[MI], sb[NI];
  mx_f4 acc[MI][NI];
  auto get_scales = [&](int win) {
    const uint8_t *s = scale_ring[win & 1];
#pragma unroll
    for (int t = 0; t < MI; ++t)
      sa[t] = *reinterpret_cast<const uint32_t *>(s + read_sa + 256 * t);
#pragma unroll
    for (int t = 0; t < NI; ++t)
      sb[t] = *reinterpret_cast<const uint32_t *>(s + read_sb + 256 * t);
    if (GROUPS > 1 && window_of(win) >= wins) {  // past K
#pragma unroll
      for (int t = 0; t < MI; ++t) sa[t] = 0;
#pragma unroll
      for (int t = 0; t < NI; ++t) sb[t] = 0;
    }
  };

  fetch_scales(0);
  fetch(0, 0, 0, kLoads);
  fetch(1, 1, 0, kLoads);
  const int rounds = (wins + GROUPS - 1) / GROUPS, units = 2 * rounds;
#pragma unroll
  for (int x = 0; x < MI; ++x)
#pragma unroll
    for (int y = 0; y < NI; ++y) acc[x][y] = mx_f4{0.f, 0.f, 0.f, 0.f};
  unit_barrier();
  get_scales(0);
#pragma unroll
  for (int t = 0; t < NI; ++t) bf[0][t] = ld16(&ring[0][read_b + place[0] + 2048 * t]);
#pragma unroll
  for (int t = 0; t < MI; ++t) af[t] = ld16(&ring[0][read_a + place[0] + 2048 * t]);

  // Phase T4 of a window: products of the operands at hand; those of the next phase, NEXT of
  // the unit in SLOT, are read, and with FETCH unit `unit` goes to the other slot.
#define TKS_PHASE(T4, SLOT, NEXT, FETCH)                                                       \
  {                                                                                            \
    constexpr int cur = T4 & 1;                                                                \
    const uint8_t *from = &ring[SLOT][place[NEXT]];                                            \
    _Pragma("unroll") for (int t = 0; t < NI; ++t) bf[cur ^ 1][t] =                            \
        ld16(from + read_b + 2048 * t);                                                        \
    _Pragma("unroll") for (int x = 0; x < MI; ++x) {                                           \
      _Pragma("unroll") for (int y = 0; y < NI; ++y)                                           \
          mfma_in_place<T4>(bf[cur][y], af[x], acc[x][y], sb[y], sa[x]);                       \
      af[x] = ld16(from + read_a + 2048 * x);                                                  \
      if (FETCH && unit < units) fetch(unit, SLOT ^ 1, kPart * x, kPart * x + kPart);          \
      __builtin_amdgcn_sched_barrier(0);                                                       \
    }                                                                                          \
  }
  for (int win = 0; win < rounds; ++win) {
    int unit = 2 * win + 2;
    TKS_PHASE(0, 0, 1, false)
    unit_barrier();
    if (win + 1 < rounds) fetch_scales(win + 1);
    TKS_PHASE(1, 1, 0, true)
    ++unit;
    TKS_PHASE(2, 1, 1, false)
    unit_barrier();
    TKS_PHASE(3, 0, 0, true)
    if (win + 1 < rounds)
      get_scales(win + 1);
    else
      settle_sums();
  }
#undef TKS_PHASE

  T *out = static_cast<T *>(p.out) + m0 * p.o_rs + n0;
  auto store = [&](int x, const mx_f4 *sums) {
    const int row = 16 * (MI * wm + x) + i;
    T *o = out + row * p.o_rs;
#pragma unroll
    for (int y = 0; y < NI; ++y) {
      const int col = 16 * (NI * wn + y) + 4 * g;
      if constexpr (VEC && sizeof(T) == 2) {
        // Four columns are 8 bytes: lanes of neighbouring groups exchange halves of two column
        // tiles, so that each stores 16 (2048 x 11264: 42.9 -> 39.3 us).
        if (y & 1) continue;
        const uint2 v = four16<T>(sums[y]), w = four16<T>(sums[y + 1]);
        const uint4 both = swap_halves(v, w);
        const int at = 16 * (NI * wn + y + (g & 1)) + 8 * (g >> 1);
        if (row <= last_m && at <= last_n) st16(o + at, both);
      } else if constexpr (VEC) {
        const mx_f4 v = sums[y];
        if (row <= last_m && col <= last_n)
          st16(o + col, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]),
                                   __float_as_uint(v[2]), __float_as_uint(v[3])));
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (row <= last_m && col + r <= last_n) o[col + r] = from_float<T>(sums[y][r]);
      }
    }
  };
  if constexpr (GROUPS == 1) {
#pragma unroll
    for (int x = 0; x < MI; ++x) store(x, acc[x]);
  } else {
    // (Every LDS read of the loop that matters is done, every load into LDS has come.) Group
    // x adds up the x-th row of tiles of each wave of the four.
    auto sums_of = [&](int from, int x, int y) {
      return reinterpret_cast<mx_f4 *>(&rings[from][0][0]) + ((x * NI + y) * 4 + wave) * 64 + lane;
    };
    __syncthreads();
#pragma unroll
    for (int x = 0; x < MI; ++x)
#pragma unroll
      for (int y = 0; y < NI; ++y) *sums_of(group, x, y) = acc[x][y];
    __syncthreads();
    for (int x = group; x < MI; x += GROUPS) {
      mx_f4 sums[NI];
#pragma unroll
      for (int y = 0; y < NI; ++y) {
        sums[y] = *sums_of(0, x, y);
#pragma unroll
        for (int from = 1; from < GROUPS; ++from) sums[y] += *sums_of(from, x, y);
      }
      store(x, sums);
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

__global__ __launch_bounds__(kThreads) void window_scales_kernel(
    const uint8_t *a_scales, int64_t m, uint8_t *a_out, const uint8_t *b_scales, int64_t n,
    uint8_t *b_out, int64_t blocks) {
  const int64_t w = windows(blocks * kMxBlock);
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (item < m * w)
    window_scales(a_scales, m, blocks, item, a_out);
  else if (item < (m + n) * w)
    window_scales(b_scales, n, blocks, item - m * w, b_out);
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

template <typename T, int MI, int NI, int GROUPS = 1>
int32_t launch_tiles(const MatmulArgs &p, hipStream_t s) {
  const int64_t tm = ceil_div(p.m, 32 * MI), tn = ceil_div(p.n, 32 * NI);
  if (tm > 0x7fffffff / tn) return TKS_ERR_VALUE;
  const unsigned grid = static_cast<unsigned>(tm * tn);
  // (Whole 16-byte pieces of a row: eight 16-bit columns, four fp32.)
  const bool vec = p.n * sizeof(T) % 16 == 0 && p.o_rs * sizeof(T) % 16 == 0 && aligned16(p.out);
  if (vec)
    matmul_tiles_kernel<T, MI, NI, GROUPS, true><<<grid, kThreads * GROUPS, 0, s>>>(p, tm, tn);
  else
    matmul_tiles_kernel<T, MI, NI, GROUPS, false><<<grid, kThreads * GROUPS, 0, s>>>(p, tm, tn);
  return check_launch();
}

// The largest tiles that still give each CU enough of them. us at 128 x 128, 64 x 128 and
// 64 x 64 (bf16):
//   2048 x 11264 x 2048 (1,408 tiles of 128 x 128)  36.8, 49.3, 53.0
//   1024 x 11264 x 2048 (704)                       23.3, 28.6, 28.3
//   2048 x 2048 x 5632  (256)                       21.9, 20.4, 23.0
//   300 x 11264 x 2048  (264; 440 of 64 x 128)      12.4, 10.0, 10.4
//   777 x 2048 x 5632   (112; 208)                  16.1, 13.1, 12.6
//   512 x 2048 x 2048   (64; 128)                   8.3, 6.6, 5.7
// With no more tiles of 64 x 64 than CUs a workgroup waits for its loads most of the time, and
// four groups of waves have four times as many on the way. us of a projection, its rows'
// quantisation included, with one group and with four:
//   128 x 2048 x 5632 (64 tiles) 16.4, 13.2     128 x 8192 x 4096 (256) 14.9, 12.8
//   256 x 4096 x 11008 (256)     32.3, 24.9     128 x 2048 x 2048 (64)  9.7, 9.0
//   777 x 2048 x 5632 (416)      20.6, 24.2     512 x 2560 x 2048 (320) 11.0, 13.7
constexpr int64_t kFewTiles = 256;
template <typename T>
int32_t launch(const MatmulArgs &p, hipStream_t s) {
  if (ceil_div(p.m, 128) * ceil_div(p.n, 128) >= 512) return launch_tiles<T, 4, 4>(p, s);
  if (ceil_div(p.m, 64) * ceil_div(p.n, 128) >= 256) return launch_tiles<T, 2, 4>(p, s);
  if (ceil_div(p.m, 64) * ceil_div(p.n, 64) <= kFewTiles && windows(p.k) >= 4)
    return launch_tiles<T, 2, 2, 4>(p, s);
  return launch_tiles<T, 2, 2>(p, s);
}

}  // namespace

int32_t launch_matmul_tiles(const MatmulArgs &p, int32_t dtype, hipStream_t s) {
  switch (dtype) {
    case TKS_FLOAT32: return launch<float>(p, s);
    case TKS_FLOAT16: return launch<_Float16>(p, s);
    default: return launch<bf16_t>(p, s);
  }
}

int32_t launch_window_scales(const uint8_t *a_scales, int64_t m, uint8_t *a_out,
                             const uint8_t *b_scales, int64_t n, uint8_t *b_out, int64_t k,
                             hipStream_t s) {
  const int64_t grid = ceil_div((m + n) * windows(k), kThreads);
  if (grid > 0x7fffffff) return TKS_ERR_VALUE;
  window_scales_kernel<<<static_cast<unsigned>(grid), kThreads, 0, s>>>(
      a_scales, m, a_out, b_scales, n, b_out, k / kMxBlock);
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
