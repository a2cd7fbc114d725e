// Decode attention over MXFP4 K/V pools: one query token per sequence, fp32/fp16/bf16.
//
// One workgroup of kWaves waves per (sequence, KV head[, split]); a wave takes tiles of 32
// keys, dealt round to the waves. Everything goes through 16x16x32 bf16 MFMAs, whose operands
// hold eight values of the contracted axis per lane (lane = 16 g + i):
//
//   S^T (16 keys x 16 heads) = K . Q^T   A: lane i a key, eight dims; B: lane i a head
//   O^T (16 dims x 16 heads) += V^T . P^T  A: lane i a dim, eight keys; B: lane i a head
//
// A decoded e2m1 value has two significant bits and its scale is a power of two, so K and V
// are exact in bf16 whatever the query's type, and a query or a probability of more bits is
// the sum of two (fp16) or three (fp32) bf16 parts, one MFMA each: products exact, sums fp32.
//
// The contracted axis may be cut among the lanes in any order that both operands share:
//  * Q.K: lane group g takes the dims [g Dh / 4, (g + 1) Dh / 4), so a lane's share of a K row
//    is one load of Dh / 8 bytes with one scale byte (Dh 128: a block; Dh 64: half of one).
//  * P.V: the score tile leaves lane (g, head) with rows 4 g + r of each 16-key half t; key
//    slot 8 g + 4 t + r of the second product is that score, so probabilities never cross
//    lanes. Row 4 g + r is key 4 r + g of the half (K rows are loaded in that order), which
//    makes the V loads of one r four adjacent rows. A lane loads Dh / 16 dims of its eight
//    keys, converts them in pairs of dims, and v_perm pairs the keys up instead.
// So K and V go from HBM to registers to the matrix cores, and LDS holds the merge alone.
//
// The softmax is online, in the log2 domain, with a lazy reference: a wave rescales its sums
// when some score passes the reference by more than 8 (2^8 is harmless in bf16 and fp32).
//
// What bounds it is reading the pools, and the waits for them: a tile's loads are issued a tile
// ahead, from an address that the wave holds in scalar registers (its pages are looked up 32
// tiles at a time) and 32-bit lane offsets. bf16, 256 sequences of 128-8,192 keys (about 2,000
// on average), Dh 128, 8 KV heads of 4 query heads each: 110 us, 5.2 TB/s; with each lane's
// address in 64 bits and every tile waited for as soon as asked for: 212 us. fp16, 128
// sequences of 0-1,152 keys, Dh 64, 4 KV heads of 8 query heads each: 11 us (18), most of it
// the launch and the longest sequence's chain of tiles.
#include "attention_common.hpp"
#include "mxfp4_kv.hpp"

#include <type_traits>

namespace tks {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr float kSlack = 8.f;
constexpr int kLookUp = 32;  // tiles whose pages a wave looks up at once

typedef Mfma<bf16_t> Bf;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

template <typename T>
struct Parts;
template <>
struct Parts<bf16_t> { static constexpr int N = 1; };
template <>
struct Parts<_Float16> { static constexpr int N = 2; };
template <>
struct Parts<float> { static constexpr int N = 3; };

// Eight floats as the sum of N bf16 parts: exact for the bits that a T has.
template <int N>
__device__ __forceinline__ void split_parts(float *x, Bf::v8 *parts) {
#pragma unroll
  for (int p = 0; p < N; ++p)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __bf16 h = static_cast<__bf16>(x[i]);
      parts[p][i] = h;
      if (p + 1 < N) x[i] -= static_cast<float>(h);
    }
}

// Byte pair SEL (two codes) of a word times the scale, as packed bf16.
template <int SEL>
__device__ __forceinline__ uint32_t pair_bits(uint32_t codes, float scale) {
#if __HIP_DEVICE_COMPILE__
  const bf16x2 v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, SEL);
  uint32_t b;
  __builtin_memcpy(&b, &v, 4);
  return b;
#else
  (void)codes; (void)scale;
  return 0;
#endif
}
__device__ __forceinline__ uint32_t pair_bits(uint32_t codes, float scale, int sel) {
  return sel == 0   ? pair_bits<0>(codes, scale)
         : sel == 1 ? pair_bits<1>(codes, scale)
         : sel == 2 ? pair_bits<2>(codes, scale)
                    : pair_bits<3>(codes, scale);
}

__device__ __forceinline__ Bf::v8 eight_of(const uint32_t *w) {
  Bf::v8 r;
  __builtin_memcpy(&r, w, 16);
  return r;
}

// A tile's codes and scale bytes as loaded. NB = Dh / 32.
template <int NB>
struct Tile {
  static constexpr int KS = NB == 3 ? 3 : 1;  // scale bytes of a lane's share of a K row
  static constexpr int VB = NB == 3 ? 3 : 1;  // loads of a lane's share of a V row
  uint32_t k[2][NB];
  uint8_t ks[2][KS];
  uint32_t v[2][4][VB];
  uint8_t vs[2][4][VB];
};

// Byte offsets of lane (g, i)'s shares in a K and a V row.
template <int NB>
__device__ __forceinline__ uint32_t k_share(int g) { return 4 * NB * g; }
template <int NB>
__device__ __forceinline__ uint32_t v_share(int i) {
  return NB == 4 ? 4 * i : NB == 2 ? 2 * i : i;
}
// The share of K and V rows at p, their scale bytes at s (rows from `row` on).
template <int NB>
__device__ __forceinline__ void load_k(const uint8_t *p, const uint8_t *s, uint32_t row, int g,
                                       uint32_t *k, uint8_t *ks) {
  __builtin_memcpy(k, __builtin_assume_aligned(p + (row * (16 * NB) + k_share<NB>(g)),
                                               NB == 4 ? 16 : NB == 2 ? 8 : 4),
                   4 * NB);
  if constexpr (NB == 3) {
#pragma unroll
    for (int j = 0; j < 3; ++j) ks[j] = s[row * NB + ((3 * g + j) >> 2)];
  } else {
    ks[0] = s[row * NB + g * NB / 4];
  }
}
template <int NB>
__device__ __forceinline__ void load_v(const uint8_t *p, const uint8_t *s, uint32_t row, int c,
                                       uint32_t *v, uint8_t *vs) {
  const uint32_t at = row * (16 * NB) + v_share<NB>(c);
  if constexpr (NB == 4) {
    v[0] = *reinterpret_cast<const uint32_t *>(p + at);
    vs[0] = s[row * NB + (c >> 2)];
  } else if constexpr (NB == 2) {
    v[0] = *reinterpret_cast<const uint16_t *>(p + at);
    vs[0] = s[row * NB + (c >> 3)];
  } else if constexpr (NB == 1) {
    v[0] = p[at];
    vs[0] = s[row];
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      v[j] = p[at + 16 * j];
      vs[j] = s[row * NB + j];
    }
  }
}
// Output dim of A row i of P.V product jj.
template <int NB>
__device__ __forceinline__ int dim_of(int i, int jj) {
  return NB == 3 ? 32 * (jj >> 1) + 2 * i + (jj & 1) : 2 * NB * i + jj;
}

// PAGED16: blocks of a multiple of 16 tokens; a half tile then lies in one block.
template <typename T, int NB, bool PAGED16>
__global__ __launch_bounds__(kThreads, 2) void decode_mx_kernel(MxDecodeArgs a) {
  constexpr int DH = 32 * NB;
  constexpr int P = Parts<T>::N;
  constexpr int J = 2 * NB;  // P.V products: 16 dims each
  __shared__ float m_s[kWaves][16], l_s[kWaves][16];
  __shared__ __align__(16) float acc_s[kWaves][16][DH];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, i = lane & 15;
  const int kvh = blockIdx.x, split = blockIdx.z;
  const int b = a.seq_order ? a.seq_order[blockIdx.y] : static_cast<int>(blockIdx.y);
  const int G = a.group;
  const int len = min(max(a.seq_lens[b], 0), a.key_cap);
  const int begin = split * a.split_keys;
  T *out = static_cast<T *>(a.out) + b * a.o_ss + static_cast<int64_t>(kvh) * G * a.o_hs;
  if (begin >= len) {
    if (split == 0)
      for (int e = threadIdx.x; e < G * DH; e += kThreads)
        out[(e / DH) * a.o_hs + e % DH] = from_float<T>(0.f);
    return;
  }
  const int end = min(len, begin + a.split_keys);
  const int tiles = (end - begin + 31) / 32;
  const int32_t *bt = a.bt + static_cast<int64_t>(b) * a.bt_stride;
  const int BS = a.kc.block_size;

  // The query as the B operand of Q.K: head i (zeros past the group), dims of group g.
  Bf::v8 q[P][NB];
  const T *q_row = static_cast<const T *>(a.q) + b * a.q_ss +
                   (static_cast<int64_t>(kvh) * G + min(i, G - 1)) * a.q_hs + 8 * NB * g;
  MxEight<T> raw[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j)
    raw[j] = a.q_vec ? mx_load8<T>(q_row + 8 * j) : mx_load8_any<T>(q_row + 8 * j);
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    float x[8];
#pragma unroll
    for (int e = 0; e < static_cast<int>(sizeof(T) / 2); ++e)
      unpack<T>(raw[j].v[e], x + e * Vec<T>::N);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = i < G ? x[e] : 0.f;
    Bf::v8 parts[P];
    split_parts<P>(x, parts);
#pragma unroll
    for (int p = 0; p < P; ++p) q[p][j] = parts[p];
  }

  // Pool row of a key (clamped to the last one: its loads are masked).
  auto row_of = [&](int key) -> int64_t {
    key = min(key, end - 1);
    const int page = key / BS;
    return a.kc.row(block_of(bt, page, a.kc.num_blocks), kvh, key - page * BS);
  };
  // With PAGED16 a half tile is a page of 16 rows, id = pool row / 16 (of this layer): lane 2 n + h
  // holds that of half h of the wave's tile `from` + n, so that a table entry is read long before
  // its keys are.
  int pages = 0;
  auto look_up = [&](int from) {
    const int key = begin + 32 * (wave + kWaves * (from + (lane >> 1))) + 16 * (lane & 1);
    if (key < end) {
      const int page = key / BS;
      const int64_t block = block_of(bt, page, a.kc.num_blocks);
      pages = static_cast<int>((block * a.kc.num_kv_heads + kvh) * (BS >> 4)) +
              ((key - page * BS) >> 4);
    }
  };
  const int64_t layer_row = a.kc.layer_base * BS;
  const int k_row = 4 * (i & 3) + (i >> 2);  // key of A row i of a half tile
  auto load = [&](int n, Tile<NB> &t) {
    const int base = begin + 32 * (wave + kWaves * n);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (PAGED16) {
        // (A page's address in scalar registers, the lane's part of it 32 bits.)
        const int64_t row =
            layer_row + 16 * static_cast<int64_t>(__builtin_amdgcn_readlane(
                                 pages, 2 * (n & (kLookUp - 1)) + h));
        const uint8_t *kp = a.kc.codes + row * (16 * NB), *ks = a.kc.scales + row * NB;
        const uint8_t *vp = a.vc.codes + row * (16 * NB), *vs = a.vc.scales + row * NB;
        load_k<NB>(kp, ks, k_row, g, t.k[h], t.ks[h]);
#pragma unroll
        for (int r = 0; r < 4; ++r) load_v<NB>(vp, vs, 4 * r + g, i, t.v[h][r], t.vs[h][r]);
      } else {
        const int64_t k_at = row_of(base + 16 * h + k_row);
        load_k<NB>(a.kc.codes + k_at * (16 * NB), a.kc.scales + k_at * NB, 0, g, t.k[h], t.ks[h]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int64_t at = row_of(base + 16 * h + 4 * r + g);
          load_v<NB>(a.vc.codes + at * (16 * NB), a.vc.scales + at * NB, 0, i, t.v[h][r],
                     t.vs[h][r]);
        }
      }
    }
  };

  float ref = -INFINITY, l = 0.f;
  Bf::f4 acc[J];
#pragma unroll
  for (int jj = 0; jj < J; ++jj) acc[jj] = Bf::f4{0.f, 0.f, 0.f, 0.f};

  // whole_tile: all 32 keys of the tile are the sequence's.
  auto process = [&](const Tile<NB> &t, int base, auto whole_tile) {
    constexpr bool whole = decltype(whole_tile)::value;
    float s[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      Bf::f4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const float scale = mx_scale(t.ks[h][NB == 3 ? j : 0]);
        const uint32_t w[4] = {pair_bits<0>(t.k[h][j], scale), pair_bits<1>(t.k[h][j], scale),
                               pair_bits<2>(t.k[h][j], scale), pair_bits<3>(t.k[h][j], scale)};
#pragma unroll
        for (int p = 0; p < P; ++p) d = Bf::run(eight_of(w), q[p][j], d);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[4 * h + r] = d[r] * a.scale_log2;
        if (!whole && base + 16 * h + 4 * r + g >= end) s[4 * h + r] = -INFINITY;
      }
    }
    float top = s[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) top = nan_max(top, s[e]);
    if (__builtin_amdgcn_ballot_w64(top > ref + kSlack) != 0) {
      const float next = nan_max(ref, xgroup_max(top));
      const float alpha = next == ref ? 1.f : fast_exp2(ref - next);
      ref = next;
      l *= alpha;
#pragma unroll
      for (int jj = 0; jj < J; ++jj) acc[jj] *= alpha;
    }
    const float from = ref == -INFINITY ? 0.f : ref;
    float pr[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      pr[e] = fast_exp2(s[e] - from);
      l += pr[e];
    }
    Bf::v8 pp[P];
    split_parts<P>(pr, pp);
#pragma unroll
    for (int p = 0; p < NB; ++p) {  // dims 2p and 2p + 1 of the lane
      uint32_t w[8], lo[4], hi[4];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t code = t.v[e >> 2][e & 3][NB == 3 ? p : 0];
        uint32_t sb = t.vs[e >> 2][e & 3][NB == 3 ? p : 0];
        uint32_t c = code;
        if (!whole && base + 16 * (e >> 2) + 4 * (e & 3) + g >= end) c = 0, sb = 127;
        w[e] = pair_bits(c, mx_scale(sb), NB == 3 ? 0 : p);
      }
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        lo[m] = __builtin_amdgcn_perm(w[2 * m + 1], w[2 * m], 0x05040100u);
        hi[m] = __builtin_amdgcn_perm(w[2 * m + 1], w[2 * m], 0x07060302u);
      }
#pragma unroll
      for (int k = 0; k < P; ++k) {
        acc[2 * p] = Bf::run(eight_of(lo), pp[k], acc[2 * p]);
        acc[2 * p + 1] = Bf::run(eight_of(hi), pp[k], acc[2 * p + 1]);
      }
    }
  };

  // The next tile's loads are in flight while one is worked on. Only the split's last tile may
  // be a part of one; its wave works on it after the others of its own.
  const int mine = (tiles - wave + kWaves - 1) / kWaves;
  const int whole = (end - begin) / 32 > wave ? ((end - begin) / 32 - wave + kWaves - 1) / kWaves : 0;
  if (mine > 0) {
    Tile<NB> even, odd;
    int looked_up = 0;
    // (Past the last tile the last one again: were the loads in a branch, a tile's would all
    // have to be waited for before the next one is worked on.)
    auto fetch = [&](int n, Tile<NB> &t) {
      n = min(n, mine - 1);
      if constexpr (PAGED16)
        if (n >= looked_up + kLookUp) look_up(looked_up += kLookUp);
      load(n, t);
    };
    auto base_of = [&](int n) { return begin + 32 * (wave + kWaves * n); };
    if constexpr (PAGED16) look_up(0);
    load(0, even);
    int n = 0;
    for (; n + 1 < whole; n += 2) {
      fetch(n + 1, odd);
      process(even, base_of(n), std::true_type{});
      fetch(n + 2, even);
      process(odd, base_of(n + 1), std::true_type{});
    }
    if (n < whole) {
      fetch(n + 1, odd);
      process(even, base_of(n), std::true_type{});
      even = odd;
      ++n;
    }
    if (n < mine) process(even, base_of(n), std::false_type{});
  }
  l = xgroup_sum(l);

  if (g == 0) {
    m_s[wave][i] = ref;
    l_s[wave][i] = l;
  }
  if (i < G) {
#pragma unroll
    for (int jj = 0; jj < J; ++jj)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc_s[wave][i][dim_of<NB>(4 * g + r, jj)] = acc[jj][r];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < G * DH; e += kThreads) {
    const int h = e / DH, d = e - h * DH;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, m_s[w][h]);
    float L = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = m_s[w][h] == M ? 1.f : exp2f(m_s[w][h] - M);
      L += f * l_s[w][h];
      o += f * acc_s[w][h][d];
    }
    const int qh = kvh * G + h;
    if (a.max_splits == 1) {
      out[h * a.o_hs + d] = from_float<T>(o / L);
    } else {
      const int64_t w = (static_cast<int64_t>(b) * a.num_q_heads + qh) * a.max_splits + split;
      if (d == 0) {
        a.ws_m[w] = M;
        a.ws_l[w] = L;
      }
      a.ws_acc[w * DH + d] = o;
    }
  }
}

template <typename T, int NB>
int32_t launch(const MxDecodeArgs &a, int32_t num_seqs, hipStream_t s) {
  const dim3 grid(a.kc.num_kv_heads, num_seqs, a.max_splits);
  if (a.kc.block_size % 16 == 0)
    decode_mx_kernel<T, NB, true><<<grid, kThreads, 0, s>>>(a);
  else
    decode_mx_kernel<T, NB, false><<<grid, kThreads, 0, s>>>(a);
  return check_launch();
}

template <typename T>
int32_t launch_dh(const MxDecodeArgs &a, int32_t num_seqs, hipStream_t s) {
  switch (a.kc.head_dim / 32) {
    case 1: return launch<T, 1>(a, num_seqs, s);
    case 2: return launch<T, 2>(a, num_seqs, s);
    case 3: return launch<T, 3>(a, num_seqs, s);
    default: return launch<T, 4>(a, num_seqs, s);
  }
}

}  // namespace

int32_t launch_decode_mxfp4(const MxDecodeArgs &a, int32_t dtype, int32_t num_seqs,
                            hipStream_t s) {
  switch (dtype) {
    case TKS_FLOAT32: return launch_dh<float>(a, num_seqs, s);
    case TKS_FLOAT16: return launch_dh<_Float16>(a, num_seqs, s);
    default: return launch_dh<bf16_t>(a, num_seqs, s);
  }
}

}  // namespace tks
