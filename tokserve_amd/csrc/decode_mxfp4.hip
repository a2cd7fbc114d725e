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

template <typename T, int NB, bool PAGED16>
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
  at.start(static_cast<const T *>(a.q) + b * a.q_ss +
               (static_cast<int64_t>(kvh) * G + head) * a.q_hs + 8 * NB * g,
           i < G, a.q_vec, a.scale_log2);
  at.run(a.kc, a.vc, a.bt + static_cast<int64_t>(b) * a.bt_stride, kvh, begin, end, end, wave,
         kWaves, lane);
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
