// Decode attention over MXFP4 K/V pools: one query token per sequence, fp32/fp16/bf16.
//
// One workgroup of kWaves waves per (sequence, KV head[, split]); a wave takes tiles of 32
// keys (mxfp4_attention.hpp: a row is a head of the group), dealt round to the waves. LDS
// holds the merge alone.
//
// What bounds it is reading the pools, and the waits for them: a tile's loads are issued a tile
// ahead, from an address that the wave holds in scalar registers (its pages are looked up 32
// tiles at a time) and 32-bit lane offsets. bf16, 256 sequences of 128-8,192 keys (about 2,000
// on average), Dh 128, 8 KV heads of 4 query heads each: 110 us, 5.2 TB/s; with each lane's
// address in 64 bits and every tile waited for as soon as asked for: 212 us. fp16, 128
// sequences of 0-1,152 keys, Dh 64, 4 KV heads of 8 query heads each: 11 us (18), most of it
// the launch and the longest sequence's chain of tiles. In blocks of 5 tokens the rows of two
// tiles are looked up at once, a lane each: the former case 133 us (each lane looking up its own:
// 251), 38 sequences of 128-927 keys 10 us (19; 8.5 in blocks of 16).
#include "mxfp4_attention.hpp"

namespace tks {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;

// The sequence's new K and V rows of a KV head, rotated and quantized, to `row` and their slot's
// place in the pools: by the first threads, eight values each. False: they have no slot.
template <typename T, int NB>
__device__ __forceinline__ bool append_row(const MxDecodeArgs &a, int b, int kvh, const T *crow,
                                           const T *srow, NewRow<NB> &row) {
  constexpr int DH = 32 * NB;
  const int E = row_threads(DH);
  const MxDecodeRope &p = a.step;
  const int64_t slot = p.slots[b];
  if (slot < 0 || slot >= a.kc.num_blocks * a.kc.block_size) return false;
  const int n = threadIdx.x, d = (n % E) * 8;
  if (n < 2 * E && d < DH) {
    const bool is_k = n < E;
    const T *src = is_k ? static_cast<const T *>(p.k) + b * p.k_ss + kvh * p.k_hs
                        : static_cast<const T *>(p.v) + b * p.v_ss + kvh * p.v_hs;
    MxEight<T> x;
    if (is_k)
      x = rotated8<T, true>(src, crow, srow, d, DH / 2);
    else
      x = mx_load8<T>(src + d);
    uint32_t s;
    const uint32_t codes = mx_quantize<T>(x, &s);
    const int64_t block = slot / a.kc.block_size;
    const MxPool &pool = is_k ? a.kc : a.vc;
    const int64_t at = pool.row(block, kvh, static_cast<int>(slot - block * a.kc.block_size));
    *reinterpret_cast<uint32_t *>(pool.codes + at * (DH / 2) + d / 2) = codes;
    *reinterpret_cast<uint32_t *>((is_k ? row.k : row.v) + d / 2) = codes;
    if ((d & 31) == 0) {
      pool.scales[at * NB + d / 32] = static_cast<uint8_t>(s);
      (is_k ? row.ks : row.vs)[d / 32] = static_cast<uint8_t>(s);
    }
  }
  return true;
}

// ROPE: a decode step (MxDecodeRope). The workgroup that holds the sequence's last key appends it
// (of a sequence of no keys: the first), and attends to it from LDS, since what another workgroup
// of the CU has in its L1 may be older. bf16, 4 KV heads of Dh 64, 512 keys, in a decode graph: 1.0
// us less than with the append in a launch of its own for one sequence, 1.1 for 128.
template <typename T, int NB, bool PAGED16, bool ROPE>
__global__ __launch_bounds__(kThreads, 2) void decode_mx_kernel(MxDecodeArgs a) {
  constexpr int DH = 32 * NB;
  constexpr int J = 2 * NB;  // P.V products: 16 dims each
  __shared__ float m_s[kWaves][16], l_s[kWaves][16];
  __shared__ __align__(16) float acc_s[kWaves][16][DH];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, i = lane & 15;
  const int kvh = blockIdx.x, split = blockIdx.z;
  const int rank = blockIdx.y;
  const int b = a.seq_order ? min(max(a.seq_order[rank], 0), static_cast<int>(gridDim.y) - 1) : rank;
  const int G = a.group;
  const int len = min(max(a.seq_lens[b], 0), a.key_cap);
  const int begin = split * a.split_keys;
  const T *crow = nullptr, *srow = nullptr;
  bool appended = false;
  __shared__ NewRow<NB> new_row;
  if constexpr (ROPE) {
    const int64_t pos = min(max(a.step.positions[b], int64_t{0}), a.step.table_len - 1);
    crow = static_cast<const T *>(a.step.cos_t) + pos * (DH / 2);
    srow = static_cast<const T *>(a.step.sin_t) + pos * (DH / 2);
    if (len > 0 ? begin < len && len - begin <= a.split_keys : split == 0) {
      // (Under a bound that cuts the sequence short the new row is not among the keys.)
      appended = append_row<T, NB>(a, b, kvh, crow, srow, new_row) && a.seq_lens[b] <= a.key_cap;
      __syncthreads();
    }
  }
  T *out = static_cast<T *>(a.out) + b * a.o_ss + static_cast<int64_t>(kvh) * G * a.o_hs;
  if (begin >= len) {
    if (split == 0)
      for (int e = threadIdx.x; e < G * DH; e += kThreads)
        out[(e / DH) * a.o_hs + e % DH] = from_float<T>(0.f);
    return;
  }
  const int end = min(len, begin + a.split_keys);
  const int head = min(i, G - 1);  // (rows past the group: zeros)
  MxAttention<T, NB, PAGED16, false> at;
  const T *q = static_cast<const T *>(a.q) + b * a.q_ss +
               (static_cast<int64_t>(kvh) * G + head) * a.q_hs;
  if constexpr (ROPE)
    at.start_rotated(q, crow, srow, g, i < G, a.scale_log2);
  else
    at.start(q + 8 * NB * g, i < G, a.q_vec, a.scale_log2);
  at.run(a.kc, a.vc, a.bt + static_cast<int64_t>(b) * a.bt_stride, kvh, begin, end,
         appended ? end - 1 : end, wave, kWaves, lane, appended ? &new_row : nullptr);
  const float l = xgroup_sum(at.l);

  if (g == 0) {
    m_s[wave][i] = at.ref;
    l_s[wave][i] = l;
  }
  if (i < G) {
#pragma unroll
    for (int jj = 0; jj < J; ++jj)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc_s[wave][i][dim_of<NB>(4 * g + r, jj)] = at.acc[jj][r];
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
  const bool paged16 = a.kc.block_size % 16 == 0;
  if (a.rope && paged16)
    decode_mx_kernel<T, NB, true, true><<<grid, kThreads, 0, s>>>(a);
  else if (a.rope)
    decode_mx_kernel<T, NB, false, true><<<grid, kThreads, 0, s>>>(a);
  else if (paged16)
    decode_mx_kernel<T, NB, true, false><<<grid, kThreads, 0, s>>>(a);
  else
    decode_mx_kernel<T, NB, false, false><<<grid, kThreads, 0, s>>>(a);
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
