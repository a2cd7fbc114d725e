// Attention of a wave's queries over MXFP4 K/V pools, 32 keys at a time, which the decode and
// the prefill share. Everything goes through 16x16x32 bf16 MFMAs, whose operands hold eight
// values of the contracted axis per lane (lane = 16 g + i):
//
//   S^T (16 keys x 16 rows) = K . Q^T     A: lane i a key, eight dims; B: lane i a row of queries
//   O^T (16 dims x 16 rows) += V^T . P^T  A: lane i a dim, eight keys; B: lane i a row
//
// A decoded e2m1 value has two significant bits and its scale is a power of two, so K and V
// are exact in bf16 whatever the query's type, and a query or a probability of more bits is
// the sum of two (fp16) or three (fp32) bf16 parts, one MFMA each: products exact, sums fp32.
//
// The contracted axis may be cut among the lanes in any order that both operands share:
//  * Q.K: lane group g takes the dims [g Dh / 4, (g + 1) Dh / 4), so a lane's share of a K row
//    is one load of Dh / 8 bytes with one scale byte (Dh 128: a block; Dh 64: half of one).
//  * P.V: the score tile leaves lane (g, row) with keys 4 g + r of each 16-key half t; key
//    slot 8 g + 4 t + r of the second product is that score, so probabilities never cross
//    lanes. Row 4 g + r is key 4 r + g of the half (K rows are loaded in that order), which
//    makes the V loads of one r four adjacent rows. A lane loads Dh / 16 dims of its eight
//    keys, converts them in pairs of dims, and v_perm pairs the keys up instead.
// So K and V go from HBM or L2 to registers to the matrix cores.
//
// The softmax is online, in the log2 domain, with a lazy reference: a wave rescales its sums
// when some score passes the reference by more than 8 (2^8 is harmless in bf16 and fp32).
#pragma once

#include "attention_common.hpp"
#include "mxfp4_kv.hpp"
#include "mxfp4_rope.hpp"

#include <type_traits>

namespace tks {
namespace {

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
// A row that is a sequence's last key, as it goes to the pools, in LDS.
template <int NB>
struct NewRow {
  __align__(16) uint8_t k[16 * NB], v[16 * NB];
  uint8_t ks[NB], vs[NB];
};
// It in place of key `in` of a loaded tile (lane (g, i), which holds key k_row of K).
template <int NB>
__device__ __forceinline__ void patch(Tile<NB> &t, const NewRow<NB> &row, int in, int g, int i,
                                      int k_row) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (in >> 4 != h) continue;
    if (k_row == (in & 15)) load_k<NB>(row.k, row.ks, 0, g, t.k[h], t.ks[h]);
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (4 * r + g == (in & 15)) load_v<NB>(row.v, row.vs, 0, i, t.v[h][r], t.vs[h][r]);
  }
}
// Output dim of A row i of P.V product jj.
template <int NB>
__device__ __forceinline__ int dim_of(int i, int jj) {
  return NB == 3 ? 32 * (jj >> 1) + 2 * i + (jj & 1) : 2 * NB * i + jj;
}

// 16 rows. PAGED16: blocks of a multiple of 16 tokens; a half tile of keys then lies in one
// block. CAUSAL: the rows see different numbers of keys.
template <typename T, int NB, bool PAGED16, bool CAUSAL>
struct MxAttention {
  static constexpr int P = Parts<T>::N;
  static constexpr int J = 2 * NB;  // P.V products: 16 dims each
  Bf::v8 q[P][NB];
  float ref, l;  // (l: the lane's share of the sum)
  Bf::f4 acc[J];
  int limit;    // CAUSAL: keys that the lane's row sees
  float scale;  // of raw scores, > 0 (or NaN)

  // The lane's row, whose values from 8 NB g on are at `row` (zeros if not live), and the
  // scores' scale in log2 units. A negative one negates the queries, a zero one makes their
  // finite values zeros, so that row maxima are those of the raw scores.
  __device__ __forceinline__ void start(const T *row, bool live, bool vec, float scale_log2) {
    MxEight<T> raw[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j)
      raw[j] = vec ? mx_load8<T>(row + 8 * j) : mx_load8_any<T>(row + 8 * j);
    start(raw, live, scale_log2);
  }
  // The same of a row that starts at `row` (16-byte aligned as the others), rotated at the table
  // rows c and s.
  __device__ __forceinline__ void start_rotated(const T *row, const T *c, const T *s, int g,
                                                bool live, float scale_log2) {
    MxEight<T> raw[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      raw[j] = rotated8<T, true>(row, c, s, 8 * (NB * g + j), 16 * NB);
      __builtin_amdgcn_sched_barrier(0);  // (one at a time: registers)
    }
    start(raw, live, scale_log2);
  }
  __device__ __forceinline__ void start(const MxEight<T> (&raw)[NB], bool live,
                                        float scale_log2) {
    const float sign = scale_log2 < 0.f ? -1.f : scale_log2 == 0.f ? 0.f : 1.f;
    scale = scale_log2 == 0.f ? 1.f : fabsf(scale_log2);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      float x[8];
#pragma unroll
      for (int e = 0; e < static_cast<int>(sizeof(T) / 2); ++e)
        unpack<T>(raw[j].v[e], x + e * Vec<T>::N);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = live ? x[e] * sign : 0.f;
      Bf::v8 parts[P];
      split_parts<P>(x, parts);
#pragma unroll
      for (int p = 0; p < P; ++p) q[p][j] = parts[p];
    }
    ref = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int jj = 0; jj < J; ++jj) acc[jj] = Bf::f4{0.f, 0.f, 0.f, 0.f};
  }

  // 32 raw scores (a lane's eight of its row) to probabilities; hidden(e): the row does not
  // see the e-th.
  template <typename Hidden>
  __device__ __forceinline__ void softmax(const Bf::f4 *d, Bf::v8 *pp, Hidden hidden) {
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = hidden(e) ? -INFINITY : d[e >> 2][e & 3];
    float top = s[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) top = nan_max(top, s[e]);
    top *= scale;
    if (__builtin_amdgcn_ballot_w64(top > ref + kSlack) != 0) {
      const float next = nan_max(ref, xgroup_max(top));
      const float alpha = next == ref ? 1.f : fast_exp2(ref - next);
      ref = next;
      l *= alpha;
#pragma unroll
      for (int jj = 0; jj < J; ++jj) acc[jj] *= alpha;
    }
    const float from = ref == -INFINITY ? 0.f : -ref;
    float pr[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      pr[e] = fast_exp2(__builtin_fmaf(s[e], scale, from));
      l += pr[e];
    }
    split_parts<P>(pr, pp);
  }

  // Dims 2p and 2p + 1 of the lane (at the tile's e-th key: lo and hi halves of w[e]).
  __device__ __forceinline__ void add_values(int p, const uint32_t *w, const Bf::v8 *pp) {
    uint32_t lo[4], hi[4];
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

  // 0 times a NaN that a row does not see would be NaN. So in a tile that not every row sees
  // whole, NaN values are zeros, and here the sums acc[jj] of the rows that do see one become
  // NaN, by a sum over keys of "is NaN" (operand bits: 1 or 0) times "is seen".
  template <typename Hidden>
  __device__ __forceinline__ void strike(int jj, const uint32_t *nan, Hidden hidden) {
    Bf::v8 sees;
#pragma unroll
    for (int e = 0; e < 8; ++e) sees[e] = static_cast<__bf16>(hidden(e) ? 0.f : 1.f);
    const Bf::f4 hits = Bf::run(eight_of(nan), sees, Bf::f4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (hits[r] > 0.f) acc[jj][r] = __builtin_nanf("");
  }

  // The 32 keys from `base` on. whole_tile: every row sees them all; else keys from `end` on
  // are nobody's.
  template <typename Whole>
  __device__ __forceinline__ void process(const Tile<NB> &t, int base, int end, int g, Whole) {
    constexpr bool whole = Whole::value;
    auto key_of = [&](int e) { return base + 16 * (e >> 2) + 4 * (e & 3) + g; };
    auto hidden = [&](int e) { return !whole && key_of(e) >= (CAUSAL ? limit : end); };
    Bf::f4 d[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      d[h] = Bf::f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const float by = mx_scale(t.ks[h][NB == 3 ? j : 0]);
        const uint32_t w[4] = {pair_bits<0>(t.k[h][j], by), pair_bits<1>(t.k[h][j], by),
                               pair_bits<2>(t.k[h][j], by), pair_bits<3>(t.k[h][j], by)};
#pragma unroll
        for (int p = 0; p < P; ++p) d[h] = Bf::run(eight_of(w), q[p][j], d[h]);
      }
    }
    Bf::v8 pp[P];
    softmax(d, pp, hidden);
#pragma unroll
    for (int p = 0; p < NB; ++p) {
      uint32_t w[8], nan[4] = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t c = t.v[e >> 2][e & 3][NB == 3 ? p : 0];
        uint32_t sb = t.vs[e >> 2][e & 3][NB == 3 ? p : 0];
        if constexpr (!whole) {
          if (key_of(e) >= end) c = 0, sb = 127;
          if (CAUSAL && sb == 255) {
            nan[e >> 1] |= e & 1 ? 0x3f800000u : 0x3f80u;
            c = 0, sb = 127;
          }
        }
        w[e] = pair_bits(c, mx_scale(sb), NB == 3 ? 0 : p);
      }
      add_values(p, w, pp);
      if constexpr (CAUSAL && !whole)
        if (__builtin_amdgcn_ballot_w64((nan[0] | nan[1] | nan[2] | nan[3]) != 0) != 0) {
          strike(2 * p, nan, hidden);  // (a block's dims are all NaN)
          strike(2 * p + 1, nan, hidden);
        }
    }
  }

  // Keys [begin, end) of the sequence whose blocks bt lists, begin a multiple of 16: of their
  // tiles of 32 the wave takes number `first` and every `stride`-th after it. Every row sees
  // those before `whole_end`. With `last` (not null), key end - 1, at or behind `whole_end`, is
  // that row.
  __device__ __forceinline__ void run(const MxPool &kc, const MxPool &vc, const int32_t *bt,
                                      int kvh, int begin, int end, int whole_end, int first,
                                      int stride, int lane, const NewRow<NB> *last = nullptr) {
    const int g = lane >> 4, i = lane & 15;
    const int BS = kc.block_size;
    // Without PAGED16: rows (of this layer) of the keys of two of the wave's tiles, 2 pair and
    // 2 pair + 1, a lane each; those of the next two are looked up meanwhile. (Past the end the
    // last key's, masked.)
    int rows = 0, next_rows = 0, pair = 0;
    auto rows_of = [&](int of) {
      const int tile = 2 * of + (lane >> 5);
      const int key = min(begin + 32 * (first + stride * tile) + (lane & 31), end - 1);
      const int page = key / BS;
      return static_cast<int>((block_of(bt, page, kc.num_blocks) * kc.num_kv_heads + kvh) * BS) +
             key - page * BS;
    };
    // With PAGED16 a half tile is a page of 16 rows, id = pool row / 16 (of this layer): lane
    // 2 n + h holds that of half h of the wave's tile `from` + n, so that a table entry is read
    // long before its keys are. (Past the end: some page of the layer's, masked.)
    int pages = 0;
    auto look_up = [&](int from) {
      const int key = begin + 32 * (first + stride * (from + (lane >> 1))) + 16 * (lane & 1);
      if (key < end) {
        const int page = key / BS;
        const int64_t block = block_of(bt, page, kc.num_blocks);
        pages = static_cast<int>((block * kc.num_kv_heads + kvh) * (BS >> 4)) +
                ((key - page * BS) >> 4);
      }
    };
    const int64_t layer_row = kc.layer_base * BS;
    const int k_row = 4 * (i & 3) + (i >> 2);  // key of A row i of a half tile
    auto base_of = [&](int n) { return begin + 32 * (first + stride * n); };
    auto load = [&](int n, Tile<NB> &t) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (PAGED16) {
          // (A page's address in scalar registers, the lane's part of it 32 bits.)
          const int64_t row =
              layer_row + 16 * static_cast<int64_t>(__builtin_amdgcn_readlane(
                                   pages, 2 * (n & (kLookUp - 1)) + h));
          const uint8_t *kp = kc.codes + row * (16 * NB), *ks = kc.scales + row * NB;
          const uint8_t *vp = vc.codes + row * (16 * NB), *vs = vc.scales + row * NB;
          load_k<NB>(kp, ks, k_row, g, t.k[h], t.ks[h]);
#pragma unroll
          for (int r = 0; r < 4; ++r) load_v<NB>(vp, vs, 4 * r + g, i, t.v[h][r], t.vs[h][r]);
        } else {
          auto row_of = [&](int key) {  // of the tile
            return layer_row + __builtin_amdgcn_ds_bpermute(4 * (32 * (n & 1) + key), rows);
          };
          const int64_t k_at = row_of(16 * h + k_row);
          load_k<NB>(kc.codes + k_at * (16 * NB), kc.scales + k_at * NB, 0, g, t.k[h], t.ks[h]);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int64_t at = row_of(16 * h + 4 * r + g);
            load_v<NB>(vc.codes + at * (16 * NB), vc.scales + at * NB, 0, i, t.v[h][r],
                       t.vs[h][r]);
          }
        }
      }
    };

    // The next tile's loads are in flight while one is worked on.
    auto of_wave = [&](int tiles) { return tiles > first ? (tiles - first + stride - 1) / stride : 0; };
    const int mine = of_wave((end - begin + 31) / 32);
    const int whole = of_wave(max(whole_end - begin, 0) / 32);
    if (mine == 0) return;
    Tile<NB> even, odd;
    int looked_up = 0;
    // (Past the last tile the last one again: were the loads in a branch, a tile's would all
    // have to be waited for before the next one is worked on.)
    auto fetch = [&](int n, Tile<NB> &t) {
      n = min(n, mine - 1);
      if constexpr (PAGED16) {
        if (n >= looked_up + kLookUp) look_up(looked_up += kLookUp);
      } else if (n >> 1 > pair) {
        rows = next_rows;
        next_rows = rows_of(++pair + 1);
      }
      load(n, t);
    };
    if constexpr (PAGED16) {
      look_up(0);
    } else {
      rows = rows_of(0);
      next_rows = rows_of(1);
    }
    load(0, even);
    int n = 0;
    for (; n + 1 < whole; n += 2) {
      fetch(n + 1, odd);
      process(even, base_of(n), end, g, std::true_type{});
      fetch(n + 2, even);
      process(odd, base_of(n + 1), end, g, std::true_type{});
    }
    if (n < whole) {
      fetch(n + 1, odd);
      process(even, base_of(n), end, g, std::true_type{});
      even = odd;
      ++n;
    }
    for (; n < mine; ++n) {
      if constexpr (CAUSAL) fetch(n + 1, odd);
      if (!CAUSAL && last != nullptr && end - base_of(n) <= 32)
        patch<NB>(even, *last, end - 1 - base_of(n), g, i, k_row);
      process(even, base_of(n), end, g, std::false_type{});
      if constexpr (CAUSAL) even = odd;
    }
  }
};

}  // namespace
}  // namespace tks
