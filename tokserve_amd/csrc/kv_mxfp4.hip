// MXFP4 K/V pools (mxfp4_common.hpp): the quantizing appends (plain, and with the step's RoPE
// fused in), the decoding block-table gather, and the decoding of the pages that a prefill
// reads. The pools hold codes, [L, NB, Hkv, BS, Dh / 2] bytes, beside scale bytes
// [L, NB, Hkv, BS, Dh / 32].
//
// A thread takes eight consecutive values of a row everywhere, so a block of 32 is the work
// of four neighbouring lanes. All of it is bound by the bytes of the 16-bit or fp32 side: bf16,
// 16 sequences, 8 KV heads of 128, appending 1-512 tokens each 9 us, gathering up to 2,560 keys
// each 21 us (4.2 TB/s of the two), decoding such pages 33 us (3.8 TB/s); a few tokens are a
// launch's 2.5 us.
#include "attention_common.hpp"
#include "mxfp4_kv.hpp"
#include "mxfp4_rope.hpp"

#include <algorithm>
#include <type_traits>

namespace tks {
namespace {

constexpr int kThreads = 256;

struct MxAppendArgs {
  const void *k, *v;  // new rows per token and KV head, in the model dtype
  int64_t k_ts, k_hs, v_ts, v_hs;
  MxPool kc, vc;
  int64_t num_tokens;
  const int64_t *slots;
  // With the RoPE fused in: query rows rotated into qo, key rows rotated before they are
  // quantized (and written to ko when it is given).
  const void *q;
  void *qo, *ko;
  int64_t q_ts, q_hs, qo_ts, qo_hs, ko_ts, ko_hs;
  int32_t num_q_heads;
  const int64_t *positions;
  const void *cos_t, *sin_t;
  int64_t table_len;
};

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T *p, const MxEight<T> &x) {
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) st16(p + i * Vec<T>::N, x.v[i]);
  } else {
    T t[8];
    __builtin_memcpy(t, &x, sizeof(x));
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = t[i];
  }
}

// A token's eights: those of its K rows, of its V rows and, with the RoPE, of its query rows
// (in that order, so quads of lanes that quantize share a block). One thread each, the tokens
// one after another. The rotation may be in place: a row's values are all read, by the one
// instruction of its wave, before any is written.
template <typename T, bool ROPE, bool VEC>
__global__ __launch_bounds__(kThreads) void append_mx_kernel(MxAppendArgs a) {
  const int DH = a.kc.head_dim, E = row_threads(DH);
  const int kv = a.kc.num_kv_heads * E;
  const int per_token = 2 * kv + (ROPE ? a.num_q_heads * E : 0);
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t t = item / per_token;
  if (t >= a.num_tokens) return;
  int rem = static_cast<int>(item - t * per_token);
  const T *crow = nullptr, *srow = nullptr;
  if constexpr (ROPE) {
    int64_t pos = a.positions[t];
    pos = pos < 0 ? 0 : (pos >= a.table_len ? a.table_len - 1 : pos);
    crow = static_cast<const T *>(a.cos_t) + pos * (DH / 2);
    srow = static_cast<const T *>(a.sin_t) + pos * (DH / 2);
    if (rem >= 2 * kv) {
      rem -= 2 * kv;
      const int h = rem / E, d = (rem - h * E) * 8;
      const T *src = static_cast<const T *>(a.q) + t * a.q_ts + h * a.q_hs;
      T *dst = static_cast<T *>(a.qo) + t * a.qo_ts + h * a.qo_hs;
      if (d >= DH) return;
      const MxEight<T> x = rotated8<T, VEC>(src, crow, srow, d, DH / 2);
      __builtin_amdgcn_wave_barrier();
      store8<T, VEC>(dst + d, x);
      return;
    }
  }
  const bool is_k = rem < kv;
  if (!is_k) rem -= kv;
  const int h = rem / E, d = (rem - h * E) * 8;
  if (d >= DH) return;
  const T *src = is_k ? static_cast<const T *>(a.k) + t * a.k_ts + h * a.k_hs
                      : static_cast<const T *>(a.v) + t * a.v_ts + h * a.v_hs;
  MxEight<T> x;
  if (ROPE && is_k) {
    x = rotated8<T, VEC>(src, crow, srow, d, DH / 2);
    __builtin_amdgcn_wave_barrier();
    if (a.ko != nullptr)
      store8<T, VEC>(static_cast<T *>(a.ko) + t * a.ko_ts + h * a.ko_hs + d, x);
  } else {
    x = load8<T, VEC>(src + d);
  }
  const int64_t slot = a.slots[t];
  const MxPool &pool = is_k ? a.kc : a.vc;
  if (slot < 0 || slot >= pool.num_blocks * pool.block_size) return;  // (all four lanes alike)
  uint32_t s;
  const uint32_t codes = mx_quantize<T>(x, &s);
  const int64_t block = slot / pool.block_size;
  const int64_t row = pool.row(block, h, static_cast<int>(slot - block * pool.block_size));
  *reinterpret_cast<uint32_t *>(pool.codes + row * (DH / 2) + d / 2) = codes;
  if ((d & 31) == 0) pool.scales[row * (DH / 32) + d / 32] = static_cast<uint8_t>(s);
}

// One thread per eight values of a gathered K row and the V row's same eight.
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void gather_mx_kernel(
    MxPool kc, MxPool vc, const int32_t *__restrict__ bt, int32_t bt_stride,
    const int32_t *__restrict__ seq_lens, const int32_t *__restrict__ cu, int32_t max_seq_len,
    T *__restrict__ k_out, T *__restrict__ v_out, int64_t o_ts, int64_t o_hs) {
  const int b = blockIdx.y;
  const int DH = kc.head_dim, E = DH / 8;
  const int per_token = kc.num_kv_heads * E;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t p = item / per_token;
  if (p >= max_seq_len || p >= seq_lens[b]) return;
  const int rem = static_cast<int>(item - p * per_token);
  const int h = rem / E, d = (rem - h * E) * 8;
  const int64_t page = p / kc.block_size;
  const int64_t block = bt[static_cast<int64_t>(b) * bt_stride + page];
  if (block < 0 || block >= kc.num_blocks) return;
  const int64_t row = kc.row(block, h, static_cast<int>(p - page * kc.block_size));
  const int64_t dst = (cu[b] + p) * o_ts + h * o_hs + d;
  float f[8];
  kc.values8(row, d, f);
  mx_store8<T, VEC>(k_out + dst, f);
  vc.values8(row, d, f);
  mx_store8<T, VEC>(v_out + dst, f);
}

// The pages that a batch reads, decoded into a dense pool of T: page (b, p) at block b * W + p
// (W pages to a sequence, at most the table's width), with the identity table and the V rows'
// marks beside it. A workgroup decodes a page, eight values a thread at a time.
template <typename T, int NB>
__global__ __launch_bounds__(kThreads) void decode_mx_pages_kernel(
    MxPool kc, MxPool vc, const int32_t *__restrict__ bt, int32_t bt_stride,
    const int32_t *__restrict__ seq_lens, int32_t width, T *__restrict__ k_out,
    T *__restrict__ v_out, int32_t *__restrict__ table_out, uint8_t *__restrict__ marks) {
  constexpr int kEights = 4 * NB;  // of a row
  const int at = blockIdx.x, b = at / width, p = at - b * width;
  if (threadIdx.x == 0) table_out[at] = at;
  if (p * static_cast<int64_t>(kc.block_size) >= seq_lens[b]) return;
  const int64_t block = block_of(bt + static_cast<int64_t>(b) * bt_stride, p, kc.num_blocks);
  const int64_t from = (kc.layer_base + block * kc.num_kv_heads) * kc.block_size;
  const int rows = kc.num_kv_heads * kc.block_size;
  const int64_t to = static_cast<int64_t>(at) * rows;
  const uint32_t *k_codes = reinterpret_cast<const uint32_t *>(kc.codes + from * (16 * NB));
  const uint32_t *v_codes = reinterpret_cast<const uint32_t *>(vc.codes + from * (16 * NB));
  const uint8_t *k_scales = kc.scales + from * NB, *v_scales = vc.scales + from * NB;
  T *k_to = k_out + to * (32 * NB), *v_to = v_out + to * (32 * NB);
#pragma unroll 4
  for (int e = threadIdx.x; e < rows * kEights; e += kThreads) {
    float f[8];
    mx_values8(k_codes[e], mx_scale(k_scales[e >> 2]), f);
    mx_store8<T, true>(k_to + 8 * e, f);
    uint32_t row_scales = 0;  // of all the V row's blocks
    const int r = e / kEights;
    __builtin_memcpy(&row_scales, v_scales + r * NB, NB);
    // (A NaN block would reach rows that do not see it, as 0 * NaN: mx_marks_kernel has them.)
    const uint32_t scale = (row_scales >> (8 * (e / 4 % NB))) & 255;
    const bool nan = scale == 255;
    mx_values8(nan ? 0 : v_codes[e], mx_scale(nan ? 127 : scale), f);
    mx_store8<T, true>(v_to + 8 * e, f);
    if (e % kEights == 0) {
      uint32_t mark = 0;
#pragma unroll
      for (int j = 0; j < NB; ++j)
        mark |= static_cast<uint32_t>(((row_scales >> (8 * j)) & 255) == 255) << j;
      marks[to + r] = static_cast<uint8_t>(mark);
    }
  }
}

// One workgroup per (sequence, KV head): the first key of each 32 dims that is NaN, and NaN to
// those dims of the rows from its position on. A launch that mostly finds nothing: 5 us for 16
// sequences of up to 2,560 keys.
template <typename T>
__global__ __launch_bounds__(kThreads) void mx_marks_kernel(MxPrefillArgs a,
                                                            const uint8_t *__restrict__ marks,
                                                            int32_t width) {
  __shared__ int first[4];
  const int b = blockIdx.y, kvh = blockIdx.x, BS = a.kc.block_size, G = a.group;
  const int len = min(max(a.seq_lens[b], 0), a.key_cap);
  if (threadIdx.x < 4) first[threadIdx.x] = INT32_MAX;
  __syncthreads();
  for (int key = 16 * static_cast<int>(threadIdx.x); key < len; key += 16 * kThreads) {
    const int page = key / BS;
    const int64_t at =
        ((static_cast<int64_t>(b) * width + page) * a.kc.num_kv_heads + kvh) * BS + key - page * BS;
    const uint4 v = *reinterpret_cast<const uint4 *>(marks + at);
    // (Of a last page's rows past `len` too, which no row sees.)
    if ((v.x | v.y | v.z | v.w) == 0) continue;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    for (int e = 0; e < 16 && key + e < len; ++e)
      for (int j = 0; j < 4; ++j)
        if ((w[e >> 2] >> (8 * (e & 3) + j)) & 1) atomicMin(&first[j], key + e);
  }
  __syncthreads();
  const int q0 = min(max(a.cu_q[b], 0), a.num_tokens);
  const int q_len = min(a.cu_q[b + 1], a.num_tokens) - q0;
  for (int j = 0; j < a.kc.head_dim / kMxBlock; ++j) {
    if (first[j] == INT32_MAX) continue;
    const int from = max(first[j] - (len - q_len), 0);  // the first token that sees it
    const int64_t items = static_cast<int64_t>(q_len - from) * G * kMxBlock;
    for (int64_t e = threadIdx.x; e < items; e += kThreads) {
      const int64_t row = e / kMxBlock, t = q0 + from + row / G;
      static_cast<T *>(a.out)[t * a.o_ts + (static_cast<int64_t>(kvh) * G + row % G) * a.o_hs +
                              j * kMxBlock + e % kMxBlock] = from_float<T>(__builtin_nanf(""));
    }
  }
}

template <typename T>
bool rows_vec(const void *p, int64_t ts, int64_t hs) {
  return aligned16(p) && ts * sizeof(T) % 16 == 0 && hs * sizeof(T) % 16 == 0;
}

template <typename T>
int32_t launch_append(const MxAppendArgs &a, bool rope, hipStream_t s) {
  const int64_t per_token =
      (2 * static_cast<int64_t>(a.kc.num_kv_heads) + (rope ? a.num_q_heads : 0)) *
      row_threads(a.kc.head_dim);
  if (per_token > 0x7fffffff) return TKS_ERR_VALUE;
  const int64_t grid = ceil_div(a.num_tokens * per_token, kThreads);
  if (grid > 0x7fffffff) return TKS_ERR_VALUE;
  bool vec = rows_vec<T>(a.k, a.k_ts, a.k_hs) && rows_vec<T>(a.v, a.v_ts, a.v_hs);
  if (rope)
    vec = vec && rows_vec<T>(a.q, a.q_ts, a.q_hs) && rows_vec<T>(a.qo, a.qo_ts, a.qo_hs) &&
          (a.ko == nullptr || rows_vec<T>(a.ko, a.ko_ts, a.ko_hs)) && aligned16(a.cos_t) &&
          aligned16(a.sin_t);
  const unsigned g = static_cast<unsigned>(grid);
  if (rope && vec)
    append_mx_kernel<T, true, true><<<g, kThreads, 0, s>>>(a);
  else if (rope)
    append_mx_kernel<T, true, false><<<g, kThreads, 0, s>>>(a);
  else if (vec)
    append_mx_kernel<T, false, true><<<g, kThreads, 0, s>>>(a);
  else
    append_mx_kernel<T, false, false><<<g, kThreads, 0, s>>>(a);
  return check_launch();
}

int32_t append_impl(MxAppendArgs a, bool rope, void *key_cache, void *value_cache,
                    void *k_scales, void *v_scales, int32_t num_layers, int64_t num_blocks,
                    int32_t num_kv_heads, int32_t block_size, int32_t head_dim,
                    int32_t layer_index, int32_t dtype, tks_stream_t stream) {
  if (!valid_dtype(dtype)) return TKS_ERR_TYPE;
  if (!mx_pool_ok(num_layers, num_blocks, num_kv_heads, block_size, head_dim) ||
      a.num_tokens < 0 || (rope && (a.num_q_heads < 0 || a.table_len <= 0)))
    return TKS_ERR_VALUE;
  if (layer_index < 0 || layer_index >= num_layers) return TKS_ERR_INDEX;
  if (a.num_tokens == 0) return TKS_OK;
  if (a.num_tokens > 0x7fffffff || !mx_pools_given(key_cache, value_cache, k_scales, v_scales) ||
      !a.k || !a.v || !a.slots)
    return TKS_ERR_VALUE;
  if (rope && ((a.num_q_heads > 0 && (!a.q || !a.qo)) || !a.positions || !a.cos_t || !a.sin_t))
    return TKS_ERR_VALUE;
  a.kc = mx_pool(key_cache, k_scales, num_blocks, num_kv_heads, block_size, head_dim, layer_index);
  a.vc =
      mx_pool(value_cache, v_scales, num_blocks, num_kv_heads, block_size, head_dim, layer_index);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TKS_FLOAT32: return launch_append<float>(a, rope, s);
    case TKS_FLOAT16: return launch_append<_Float16>(a, rope, s);
    default: return launch_append<bf16_t>(a, rope, s);
  }
}

}  // namespace

MxScratch mx_carve_pages(void *ws, int32_t num_seqs, int32_t width, int32_t num_kv_heads,
                         int32_t block_size, int32_t head_dim, int32_t dtype) {
  const int64_t pages = static_cast<int64_t>(num_seqs) * width;
  const int64_t pool =
      ceil_div(pages * num_kv_heads * block_size * head_dim * elem_bytes(dtype), 256) * 256;
  const int64_t table = ceil_div(pages * 4, 256) * 256;
  const int64_t marks = ceil_div(pages * num_kv_heads * block_size, 256) * 256;
  char *base = static_cast<char *>(ws);
  MxScratch r;
  r.k = base;
  r.v = base ? base + pool : nullptr;
  r.table = base ? reinterpret_cast<int32_t *>(base + 2 * pool) : nullptr;
  r.marks = base ? reinterpret_cast<uint8_t *>(base + 2 * pool + table) : nullptr;
  r.bytes = 2 * pool + table + marks;
  return r;
}

int32_t launch_decode_mx_pages(const MxPool &kc, const MxPool &vc, const int32_t *bt,
                               int32_t bt_stride, const int32_t *seq_lens, int32_t num_seqs,
                               int32_t width, const MxScratch &to, int32_t dtype, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>(num_seqs) * static_cast<unsigned>(width);
  auto run = [&](auto zero, auto nb) {
    typedef decltype(zero) T;
    decode_mx_pages_kernel<T, decltype(nb)::value><<<grid, kThreads, 0, s>>>(
        kc, vc, bt, bt_stride, seq_lens, width, static_cast<T *>(to.k), static_cast<T *>(to.v),
        to.table, to.marks);
  };
  auto run_dh = [&](auto zero) {
    if (kc.head_dim == 64)
      run(zero, std::integral_constant<int, 2>());
    else
      run(zero, std::integral_constant<int, 4>());
  };
  if (dtype == TKS_FLOAT16)
    run_dh(_Float16());
  else
    run_dh(bf16_t());
  return check_launch();
}

int32_t launch_mx_marks(const MxPrefillArgs &a, const MxScratch &from, int32_t width,
                        int32_t dtype, hipStream_t s) {
  const dim3 grid(a.kc.num_kv_heads, a.num_seqs);
  if (dtype == TKS_FLOAT16)
    mx_marks_kernel<_Float16><<<grid, kThreads, 0, s>>>(a, from.marks, width);
  else
    mx_marks_kernel<bf16_t><<<grid, kThreads, 0, s>>>(a, from.marks, width);
  return check_launch();
}

}  // namespace tks

using namespace tks;

extern "C" int32_t tks_kv_append_mxfp4(const void *key, int64_t key_token_stride,
                                       int64_t key_head_stride, const void *value,
                                       int64_t value_token_stride, int64_t value_head_stride,
                                       int64_t num_tokens, void *key_cache, void *value_cache,
                                       void *k_scales, void *v_scales, int32_t num_layers,
                                       int64_t num_blocks, int32_t num_kv_heads,
                                       int32_t block_size, int32_t head_dim, int32_t layer_index,
                                       const int64_t *slot_mapping, int32_t dtype,
                                       tks_stream_t stream) {
  MxAppendArgs a{};
  a.k = key;
  a.k_ts = key_token_stride;
  a.k_hs = key_head_stride;
  a.v = value;
  a.v_ts = value_token_stride;
  a.v_hs = value_head_stride;
  a.num_tokens = num_tokens;
  a.slots = slot_mapping;
  return append_impl(a, false, key_cache, value_cache, k_scales, v_scales, num_layers, num_blocks,
                     num_kv_heads, block_size, head_dim, layer_index, dtype, stream);
}

extern "C" int32_t tks_rope_kv_append_mxfp4(
    const void *query, void *query_out, int64_t q_ts, int64_t q_hs, int64_t qo_ts, int64_t qo_hs,
    int32_t num_q_heads, const void *key, void *key_out, int64_t k_ts, int64_t k_hs, int64_t ko_ts,
    int64_t ko_hs, const void *value, int64_t v_ts, int64_t v_hs, int32_t num_kv_heads,
    int64_t num_tokens, int32_t head_dim, const int64_t *positions, const void *cos_cache,
    const void *sin_cache, int64_t cache_len, void *key_cache, void *value_cache, void *k_scales,
    void *v_scales, int32_t num_layers, int64_t num_blocks, int32_t block_size,
    int32_t layer_index, const int64_t *slot_mapping, int32_t dtype, tks_stream_t stream) {
  MxAppendArgs a{};
  a.k = key;
  a.k_ts = k_ts;
  a.k_hs = k_hs;
  a.v = value;
  a.v_ts = v_ts;
  a.v_hs = v_hs;
  a.num_tokens = num_tokens;
  a.slots = slot_mapping;
  a.q = query;
  a.qo = query_out;
  a.q_ts = q_ts;
  a.q_hs = q_hs;
  a.qo_ts = qo_ts;
  a.qo_hs = qo_hs;
  a.num_q_heads = num_q_heads;
  a.ko = key_out;
  a.ko_ts = ko_ts;
  a.ko_hs = ko_hs;
  a.positions = positions;
  a.cos_t = cos_cache;
  a.sin_t = sin_cache;
  a.table_len = cache_len;
  return append_impl(a, true, key_cache, value_cache, k_scales, v_scales, num_layers, num_blocks,
                     num_kv_heads, block_size, head_dim, layer_index, dtype, stream);
}

extern "C" int32_t tks_paged_gather_mxfp4(
    const void *key_cache, const void *value_cache, const void *k_scales, const void *v_scales,
    int32_t num_layers, int64_t num_blocks, int32_t num_kv_heads, int32_t block_size,
    int32_t head_dim, int32_t layer_index, const int32_t *block_tables, int32_t block_table_stride,
    const int32_t *seq_lens, const int32_t *cu_seqlens, int32_t num_seqs, int32_t max_seq_len,
    void *key_out, void *value_out, int64_t out_token_stride, int64_t out_head_stride,
    int32_t dtype, tks_stream_t stream) {
  if (!valid_dtype(dtype)) return TKS_ERR_TYPE;
  if (!mx_pool_ok(num_layers, num_blocks, num_kv_heads, block_size, head_dim) || num_seqs < 0 ||
      max_seq_len < 0 || block_table_stride < 0)
    return TKS_ERR_VALUE;
  if (layer_index < 0 || layer_index >= num_layers) return TKS_ERR_INDEX;
  if (num_seqs == 0 || max_seq_len == 0) return TKS_OK;
  if (num_seqs > 65535 || ceil_div(max_seq_len, block_size) > block_table_stride)
    return TKS_ERR_VALUE;
  if (!mx_pools_given(key_cache, value_cache, k_scales, v_scales) || !block_tables || !seq_lens ||
      !cu_seqlens || !key_out || !value_out)
    return TKS_ERR_VALUE;
  const int64_t items = static_cast<int64_t>(max_seq_len) * num_kv_heads * (head_dim / 8);
  if (ceil_div(items, kThreads) > 0x7fffffff) return TKS_ERR_VALUE;
  const MxPool kc = mx_pool(const_cast<void *>(key_cache), const_cast<void *>(k_scales),
                            num_blocks, num_kv_heads, block_size, head_dim, layer_index);
  const MxPool vc = mx_pool(const_cast<void *>(value_cache), const_cast<void *>(v_scales),
                            num_blocks, num_kv_heads, block_size, head_dim, layer_index);
  const dim3 grid(static_cast<unsigned>(ceil_div(items, kThreads)), num_seqs);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define TKS_MX_GATHER(TYPE, VEC)                                                               \
  gather_mx_kernel<TYPE, VEC><<<grid, kThreads, 0, s>>>(                                       \
      kc, vc, block_tables, block_table_stride, seq_lens, cu_seqlens, max_seq_len,             \
      static_cast<TYPE *>(key_out), static_cast<TYPE *>(value_out), out_token_stride,          \
      out_head_stride)
#define TKS_MX_GATHER_OF(TYPE)                                                                 \
  if (rows_vec<TYPE>(key_out, out_token_stride, out_head_stride) && aligned16(value_out))      \
    TKS_MX_GATHER(TYPE, true);                                                                 \
  else                                                                                         \
    TKS_MX_GATHER(TYPE, false)
  switch (dtype) {
    case TKS_FLOAT32: TKS_MX_GATHER_OF(float); break;
    case TKS_FLOAT16: TKS_MX_GATHER_OF(_Float16); break;
    default: TKS_MX_GATHER_OF(bf16_t); break;
  }
#undef TKS_MX_GATHER_OF
#undef TKS_MX_GATHER
  return check_launch();
}
