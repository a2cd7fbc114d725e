// Chunked-prefill attention over MXFP4 K/V pools, fp32/fp16/bf16, straight from the pools.
//
// The rows of a (sequence, KV head) are its (query token, head of the group) pairs, row =
// token * G + head, each seeing the keys up to its token's own position; a wave computes 16 of
// them (mxfp4_attention.hpp). Two forms:
//
//  * shared: the four waves of a workgroup take different rows and walk the same keys. A tile
//    of 32 keys is decoded once, to bf16 in LDS ([key][dim], double-buffered, one barrier a
//    tile), while the next one's codes are on their way to registers; V's operand comes out of
//    it transposed (ds_read_b64_tr_b16). What bounds it is a tile's chain (scores, softmax,
//    values, barrier), which three waves per SIMD do not cover: bf16, 16 x 512 tokens, Dh 128,
//    324 us, the matrix pipe busy a quarter of it. Tiles of 64 keys are level.
//  * apart: the four waves take the same rows, the tiles of keys dealt round, each decoding
//    its own in registers; their sums meet in LDS. Where there are few rows the longest chain
//    of tiles sets the time, and this quarters it.
//
// us of each (apart, shared), kv heads 8 of Dh 128 under 32 heads, 4,096 earlier keys: bf16 4 x
// 128 tokens 44, 109; 16 x 64 85, 115; 16 x 128 163, 147; 512 earlier keys: 4 x 128 22, 26; 16 x
// 64 35, 27; fp32 5 x 1-333 tokens, Dh 64, to 1,024 earlier: 23, 32 (over decoded fp32 pages, as
// before these: 61); fp32 16 x 512, Dh 128, to 2,048 earlier: 642, 573 (1,590); bf16 4 x 200-400,
// Dh 96, to 1,024 earlier: 76, 45 (3,910: nothing but a plain kernel takes such pages).
#include "mxfp4_attention.hpp"

#include <algorithm>

namespace tks {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kXcds = 8;

// What a workgroup works on: rows [row0, row0 + count) of a sequence and KV head. All the tiles
// of a (sequence, KV head) are on one XCD, whose L2 then holds its pages; the last tiles,
// which see the most keys, come first.
struct Work {
  int kvh, b, q0, base_pos;  // (position of query token 0, below 0 where keys are missing)
  int64_t rows, row0;        // rows: of the sequence; none left: row0 >= rows
  const int32_t *bt;
};
__device__ __forceinline__ Work work_of(const MxPrefillArgs &a, int count) {
  Work w{};
  const int slot = blockIdx.x / kXcds;
  const int pair = (slot / a.tiles) * kXcds + blockIdx.x % kXcds;
  if (pair >= a.num_seqs * a.kc.num_kv_heads) return w;
  const int tile = a.tiles - 1 - slot % a.tiles, rank = pair / a.kc.num_kv_heads;
  w.kvh = pair % a.kc.num_kv_heads;
  w.b = a.seq_order ? min(max(a.seq_order[rank], 0), a.num_seqs - 1) : rank;
  w.q0 = min(max(a.cu_q[w.b], 0), a.num_tokens);
  const int q_len = min(a.cu_q[w.b + 1], a.num_tokens) - w.q0;
  w.rows = static_cast<int64_t>(q_len) * a.group;
  w.row0 = static_cast<int64_t>(tile) * count;
  w.base_pos = min(max(a.seq_lens[w.b], 0), a.key_cap) - q_len;
  w.bt = a.bt + static_cast<int64_t>(w.b) * a.bt_stride;
  return w;
}
// Keys that row `row` sees (0 or less: none).
__device__ __forceinline__ int seen_by(const Work &w, int64_t row, int G) {
  return w.base_pos + static_cast<int>(row) / G + 1;
}

// The lane's row (row0 + i) to the wave's operands.
template <typename T, int NB, bool PAGED16>
struct Rows {
  MxAttention<T, NB, PAGED16, true> at;
  int64_t out;  // offset of the row's output
  bool live;
  __device__ __forceinline__ void start(const MxPrefillArgs &a, const Work &w, int64_t row0, int g,
                                        int i) {
    live = row0 + i < w.rows;
    const int row = static_cast<int>(live ? row0 + i : w.rows - 1), t = row / a.group;
    const int64_t head = w.kvh * a.group + row - t * a.group;
    at.limit = live ? w.base_pos + t + 1 : 0;
    out = (w.q0 + t) * a.o_ts + head * a.o_hs;
    at.start(static_cast<const T *>(a.q) + (w.q0 + t) * a.q_ts + head * a.q_hs + 8 * NB * g, live,
             a.q_vec, a.scale_log2);
  }
};

template <typename T, int NB, bool PAGED16>
__global__ __launch_bounds__(kThreads, 2) void prefill_mx_apart_kernel(MxPrefillArgs a) {
  constexpr int DH = 32 * NB;
  constexpr int J = 2 * NB;
  __shared__ float m_s[kWaves][16], l_s[kWaves][16];
  __shared__ __align__(16) float acc_s[kWaves][16][DH];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, i = lane & 15;
  const int G = a.group;
  const Work w = work_of(a, 16);
  if (w.row0 >= w.rows) return;

  Rows<T, NB, PAGED16> r;
  r.start(a, w, w.row0, g, i);
  auto &at = r.at;
  at.run(a.kc, a.vc, w.bt, w.kvh, 0, max(seen_by(w, min(w.row0 + 16, w.rows) - 1, G), 0),
         max(seen_by(w, w.row0, G), 0), wave, kWaves, lane);
  const float sum = xgroup_sum(at.l);
  if (g == 0) {
    m_s[wave][i] = at.ref;
    l_s[wave][i] = sum;
  }
#pragma unroll
  for (int jj = 0; jj < J; ++jj)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc_s[wave][i][dim_of<NB>(4 * g + e, jj)] = at.acc[jj][e];
  __syncthreads();
  for (int e = threadIdx.x; e < 16 * DH; e += kThreads) {
    const int x = e / DH, d = e - x * DH;
    if (w.row0 + x >= w.rows) continue;
    const int row = static_cast<int>(w.row0) + x, t = row / G;
    float M = -INFINITY;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) M = fmaxf(M, m_s[v][x]);
    float L = 0.f, o = 0.f;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      const float f = m_s[v][x] == M ? 1.f : exp2f(m_s[v][x] - M);
      L += f * l_s[v][x];
      o += f * acc_s[v][x][d];
    }
    const int64_t head = w.kvh * G + row - t * G;
    static_cast<T *>(a.out)[(w.q0 + t) * a.o_ts + head * a.o_hs + d] =
        from_float<T>(w.base_pos + t >= 0 ? o / L : 0.f);  // (a row of no keys: zeros)
  }
}

// A tile of K and V in LDS as bf16, [key][dim], the 16-byte chunks of a row permuted by its
// number so that neither operand's read has bank conflicts.
template <int NB>
struct KeyTile {
  static constexpr int CPR = NB == 1 ? 4 : NB == 2 ? 8 : 16;  // chunks of a row (96 dims: 12 used)
  static constexpr int kBytes = 32 * CPR * 16;
  static __device__ __forceinline__ int k_at(int row, int chunk) {
    const int by = NB >= 3 ? row : NB == 2 ? row >> 1 : row >> 2;
    return 16 * (row * CPR + (chunk ^ (by & (CPR - 1))));
  }
  static __device__ __forceinline__ int v_at(int row, int chunk) {
    const int by = NB >= 3 ? 2 * (row & 7) : NB == 2 ? row & 7 : row >> 1;
    return 16 * (row * CPR + (chunk ^ (by & (CPR - 1))));
  }
};

__device__ __forceinline__ void lds_barrier() {
#if __HIP_DEVICE_COMPILE__
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#endif
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
// Within 16 lanes, element e of lane j: element j % 4 of what lane 4 e + j / 4 addressed.
__device__ __forceinline__ uint2 read_transposed(const uint8_t *p) {
#if __HIP_DEVICE_COMPILE__
  const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4 *)p);
  uint2 r;
  __builtin_memcpy(&r, &v, 8);
  return r;
#else
  (void)p;
  return make_uint2(0, 0);
#endif
}

template <typename T, int NB, bool PAGED16>
__global__ __launch_bounds__(kThreads, 2) void prefill_mx_shared_kernel(MxPrefillArgs a) {
  constexpr int J = 2 * NB;
  constexpr int kRows = 16 * kWaves;
  constexpr int kUnits = 128 * NB;  // 16 values each, of a tile's K and V
  constexpr int U = (kUnits + kThreads - 1) / kThreads;
  using Keys = KeyTile<NB>;
  __shared__ __align__(16) uint8_t ring[2][2][Keys::kBytes];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, i = lane & 15;
  const int G = a.group;
  const Work w = work_of(a, kRows);
  if (w.row0 >= w.rows) return;
  // Keys that some and that every row of the workgroup sees.
  const int end = max(seen_by(w, min(w.row0 + kRows, w.rows) - 1, G), 0);
  const int whole_end = max(seen_by(w, w.row0, G), 0);

  Rows<T, NB, PAGED16> r;
  r.start(a, w, w.row0 + 16 * wave, g, i);
  auto &at = r.at;

  // A thread's units of a tile: 16 values of a row each. K's come first, then V's (a wave's are
  // all of one).
  struct Unit {
    uint2 codes;
    uint32_t scale;
  };
  Unit unit[U];
  const int BS = a.kc.block_size;
  const int64_t layer_row = a.kc.layer_base * BS;
  int pages = 0;
  auto look_up = [&](int from) {  // as MxAttention::run's
    const int key = 32 * (from + (lane >> 1)) + 16 * (lane & 1);
    if (key < end) {
      const int page = key / BS;
      const int64_t block = block_of(w.bt, page, a.kc.num_blocks);
      pages = static_cast<int>((block * a.kc.num_kv_heads + w.kvh) * (BS >> 4)) +
              ((key - page * BS) >> 4);
    }
  };
  auto page_row = [&](int step, int h) {
    return layer_row + 16 * static_cast<int64_t>(__builtin_amdgcn_readlane(
                                pages, 2 * (step & (kLookUp - 1)) + h));
  };
  auto each_unit = [&](auto f) {
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int u = static_cast<int>(threadIdx.x) + kThreads * k;
      if (kUnits % kThreads != 0 && u >= kUnits) continue;
      const bool of_v = 64 * wave + kThreads * k >= 64 * NB;
      const int v = of_v ? u - 64 * NB : u, row = v / (2 * NB);
      f(unit[k], of_v, row, v - row * (2 * NB));
    }
  };
  auto load = [&](int step) {
    each_unit([&](Unit &x, bool of_v, int row, int part) {
      const MxPool &pool = of_v ? a.vc : a.kc;
      if constexpr (PAGED16 && NB % 2 == 0) {
        // (A wave's rows are all of one page: its address in scalar registers.)
        const int64_t from = page_row(step, __builtin_amdgcn_readfirstlane(row >> 4));
        const uint32_t in = row & 15;
        x.codes = *reinterpret_cast<const uint2 *>(pool.codes + from * (16 * NB) +
                                                   (in * (16 * NB) + 8 * part));
        x.scale = (pool.scales + from * NB)[in * NB + (part >> 1)];
      } else {
        int64_t from;
        if constexpr (PAGED16) {
          const int64_t first = page_row(step, 0), second = page_row(step, 1);
          from = (row < 16 ? first : second) + (row & 15);
        } else {
          const int key = min(32 * step + row, end - 1), pg = key / BS;
          from = a.kc.row(block_of(w.bt, pg, a.kc.num_blocks), w.kvh, key - pg * BS);
        }
        x.codes = *reinterpret_cast<const uint2 *>(pool.codes + from * (16 * NB) + 8 * part);
        x.scale = pool.scales[from * NB + (part >> 1)];
      }
    });
  };
  auto write = [&](int step, auto stage) {
    each_unit([&](Unit &x, bool of_v, int row, int part) {
      if (32 * step + 32 > end && 32 * step + row >= end) {
        // (Keys that no row sees are zeros: what the pool has there may be NaN.)
        x.codes = make_uint2(0, 0);
        x.scale = 127;
      }
      // Half of the lanes write their second chunk first, so that eight lanes' are of eight
      // different bank groups.
      const bool second = NB == 2 ? !of_v && (row & 1) : NB == 4 && part >= 4;
      const uint32_t c0 = second ? x.codes.y : x.codes.x, c1 = second ? x.codes.x : x.codes.y;
      const int chunk = 2 * part + second;
      const float scale = mx_scale(x.scale);
      uint8_t *to = ring[decltype(stage)::value][of_v];
      st16(to + (of_v ? Keys::v_at(row, chunk) : Keys::k_at(row, chunk)),
           make_uint4(pair_bits<0>(c0, scale), pair_bits<1>(c0, scale), pair_bits<2>(c0, scale),
                      pair_bits<3>(c0, scale)));
      st16(to + (of_v ? Keys::v_at(row, chunk ^ 1) : Keys::k_at(row, chunk ^ 1)),
           make_uint4(pair_bits<0>(c1, scale), pair_bits<1>(c1, scale), pair_bits<2>(c1, scale),
                      pair_bits<3>(c1, scale)));
    });
  };

  // Lane (g, i): scores of keys 16 h + 4 g + r, so V's operand is rows 4 g + r of both halves.
  auto compute = [&](int step, auto stage, auto whole_tile) {
    constexpr bool whole = decltype(whole_tile)::value;
    const uint8_t *ks = ring[decltype(stage)::value][0], *vs = ring[decltype(stage)::value][1];
    auto hidden = [&](int e) {
      return !whole && 32 * step + 16 * (e >> 2) + 4 * g + (e & 3) >= at.limit;
    };
    Bf::f4 d[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      d[h] = Bf::f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const uint4 w = ld16(ks + Keys::k_at(16 * h + i, g * NB + j));
        Bf::v8 k;
        __builtin_memcpy(&k, &w, 16);
#pragma unroll
        for (int p = 0; p < Parts<T>::N; ++p) d[h] = Bf::run(k, at.q[p][j], d[h]);
      }
    }
    Bf::v8 pp[Parts<T>::N];
    at.softmax(d, pp, hidden);
#pragma unroll
    for (int jj = 0; jj < J; ++jj) {
      uint32_t w[4], nan[4] = {0, 0, 0, 0};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint2 half = read_transposed(
            vs + Keys::v_at(16 * h + 4 * g + (i >> 2), 2 * jj + ((i >> 1) & 1)) + 8 * (i & 1));
        w[2 * h] = half.x;
        w[2 * h + 1] = half.y;
      }
      if constexpr (!whole) {
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const bool lo = (w[m] & 0x7fffu) > 0x7f80u, hi = (w[m] & 0x7fffffffu) >= 0x7f810000u;
          nan[m] = (lo ? 0x3f80u : 0) | (hi ? 0x3f800000u : 0);
          w[m] = (lo ? 0 : w[m] & 0xffffu) | (hi ? 0 : w[m] & 0xffff0000u);
        }
      }
#pragma unroll
      for (int k = 0; k < Parts<T>::N; ++k) at.acc[jj] = Bf::run(eight_of(w), pp[k], at.acc[jj]);
      if constexpr (!whole)
        if (__builtin_amdgcn_ballot_w64((nan[0] | nan[1] | nan[2] | nan[3]) != 0) != 0)
          at.strike(jj, nan, hidden);
    }
  };

  // A tile's values are on their way to registers while the one before is worked on, and go to
  // the LDS of the one before that.
  const int steps = (end + 31) / 32;
  int looked_up = 0;
  if constexpr (PAGED16) look_up(0);
  if (steps > 0) {
    load(0);
    write(0, std::integral_constant<int, 0>());
    load(min(1, steps - 1));
  }
  lds_barrier();
  auto turn = [&](int step, auto stage, auto whole_tile) {
    compute(step, stage, whole_tile);
    if (step + 1 < steps) {
      write(step + 1, std::integral_constant<int, 1 - decltype(stage)::value>());
      const int next = min(step + 2, steps - 1);
      if constexpr (PAGED16)
        if (next >= looked_up + kLookUp) look_up(looked_up += kLookUp);
      load(next);
    }
    lds_barrier();
  };
  typedef std::integral_constant<int, 0> Even;
  typedef std::integral_constant<int, 1> Odd;
  // (Two loops, not a choice in one: it would have the sums copied from path to path.)
  const int whole = whole_end / 64 * 2;  // tiles that every row sees, in pairs
  int step = 0;
  for (; step < whole; step += 2) {
    turn(step, Even(), std::true_type{});
    turn(step + 1, Odd(), std::true_type{});
  }
  for (; step < steps; step += 2) {
    turn(step, Even(), std::false_type{});
    if (step + 1 < steps) turn(step + 1, Odd(), std::false_type{});
  }
  if (!r.live) return;
  const float sum = xgroup_sum(at.l);
  const float by = at.limit > 0 ? 1.f / sum : 0.f;  // (a row of no keys: zeros)
  T *o = static_cast<T *>(a.out) + r.out + 4 * g;
#pragma unroll
  for (int jj = 0; jj < J; ++jj) {
    T v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = from_float<T>(at.acc[jj][e] * by);
    if (a.o_vec) {
      __builtin_memcpy(__builtin_assume_aligned(o + 16 * jj, 4 * sizeof(T)), v, sizeof(v));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) o[16 * jj + e] = v[e];
    }
  }
}

// Fewer rows than make this many workgroups of the shared form (most of two a CU): apart.
constexpr int64_t kSharedFrom = 449;

template <typename T, int NB>
int32_t launch(MxPrefillArgs a, int32_t max_query_len, hipStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.num_tokens) * a.group * a.kc.num_kv_heads;
  const bool shared = ceil_div(rows, 16 * kWaves) >= kSharedFrom;
  const int64_t tiles =
      ceil_div(static_cast<int64_t>(max_query_len) * a.group, shared ? 16 * kWaves : 16);
  const int64_t pairs = static_cast<int64_t>(a.num_seqs) * a.kc.num_kv_heads;
  const int64_t per_xcd = ceil_div(pairs, kXcds);
  if (tiles == 0) return TKS_OK;
  if (per_xcd > 0x7fffffff / kXcds || tiles > 0x7fffffff / (per_xcd * kXcds)) return TKS_ERR_VALUE;
  a.tiles = static_cast<int32_t>(tiles);
  const unsigned grid = static_cast<unsigned>(per_xcd * kXcds * tiles);
  const bool paged16 = a.kc.block_size % 16 == 0;
  if (shared && paged16)
    prefill_mx_shared_kernel<T, NB, true><<<grid, kThreads, 0, s>>>(a);
  else if (shared)
    prefill_mx_shared_kernel<T, NB, false><<<grid, kThreads, 0, s>>>(a);
  else if (paged16)
    prefill_mx_apart_kernel<T, NB, true><<<grid, kThreads, 0, s>>>(a);
  else
    prefill_mx_apart_kernel<T, NB, false><<<grid, kThreads, 0, s>>>(a);
  return check_launch();
}

template <typename T>
int32_t launch_dh(const MxPrefillArgs &a, int32_t max_query_len, hipStream_t s) {
  switch (a.kc.head_dim / 32) {
    case 1: return launch<T, 1>(a, max_query_len, s);
    case 2: return launch<T, 2>(a, max_query_len, s);
    case 3: return launch<T, 3>(a, max_query_len, s);
    default: return launch<T, 4>(a, max_query_len, s);
  }
}

}  // namespace

int32_t launch_prefill_mxfp4(const MxPrefillArgs &a, int32_t max_query_len, int32_t dtype,
                             hipStream_t s) {
  switch (dtype) {
    case TKS_FLOAT32: return launch_dh<float>(a, max_query_len, s);
    case TKS_FLOAT16: return launch_dh<_Float16>(a, max_query_len, s);
    default: return launch_dh<bf16_t>(a, max_query_len, s);
  }
}

}  // namespace tks
