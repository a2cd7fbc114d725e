// MXFP4 K/V pools as the kernels address them, and the scratch pool that a prefill of many rows
// decodes the pages it reads into.
#pragma once

#include "mxfp4_common.hpp"

namespace tks {

// One layer's K or V pool: codes, Dh / 2 bytes to a row, and Dh / 32 scale bytes to a row.
struct MxPool {
  uint8_t *codes, *scales;
  int64_t layer_base;  // layer * NB * Hkv
  int64_t num_blocks;
  int32_t block_size, num_kv_heads, head_dim;

  // Row (of the whole pool) of offset `r` in a block.
  __host__ __device__ __forceinline__ int64_t row(int64_t block, int h, int r) const {
    return (layer_base + block * num_kv_heads + h) * block_size + r;
  }
  // Values d .. d+7 of a row (d a multiple of 8).
  __device__ __forceinline__ void values8(int64_t row, int d, float *f) const {
    const uint32_t c = *reinterpret_cast<const uint32_t *>(codes + row * (head_dim / 2) + d / 2);
    mx_values8(c, mx_scale(scales[row * (head_dim / 32) + d / 32]), f);
  }
};

constexpr int kMxMaxDh = 128;

inline bool mx_pool_ok(int32_t num_layers, int64_t num_blocks, int32_t num_kv_heads,
                       int32_t block_size, int32_t head_dim) {
  return num_layers > 0 && num_blocks > 0 && num_kv_heads > 0 && block_size > 0 &&
         head_dim > 0 && head_dim <= kMxMaxDh && head_dim % kMxBlock == 0;
}
// Attention over blocks that are no multiple of 16 numbers a layer's rows in 32 bits.
inline bool mx_rows_ok(int64_t num_blocks, int32_t num_kv_heads, int32_t block_size) {
  return block_size % 16 == 0 ||
         num_blocks <= INT32_MAX / (static_cast<int64_t>(num_kv_heads) * block_size);
}

// Codes are read and written four bytes at a time at least, sixteen in the decode.
inline bool mx_pools_given(const void *kc, const void *vc, const void *ks, const void *vs) {
  return kc && vc && ks && vs && aligned16(kc) && aligned16(vc);
}

inline MxPool mx_pool(void *codes, void *scales, int64_t num_blocks, int32_t num_kv_heads,
                      int32_t block_size, int32_t head_dim, int32_t layer_index) {
  return MxPool{static_cast<uint8_t *>(codes),
                static_cast<uint8_t *>(scales),
                static_cast<int64_t>(layer_index) * num_blocks * num_kv_heads,
                num_blocks,
                block_size,
                num_kv_heads,
                head_dim};
}

// Pages decoded for a prefill (16-bit types, Dh 64 or 128, blocks of a multiple of 16 tokens): pools of the
// query's dtype, num_seqs * width blocks, the identity block table, and a byte per V row (in
// the pools' order), bit j: its j-th block is NaN, zeros in the pool.
struct MxScratch {
  void *k, *v;
  int32_t *table;
  uint8_t *marks;
  int64_t bytes;
};
MxScratch mx_carve_pages(void *ws, int32_t num_seqs, int32_t width, int32_t num_kv_heads,
                         int32_t block_size, int32_t head_dim, int32_t dtype);
int32_t launch_decode_mx_pages(const MxPool &kc, const MxPool &vc, const int32_t *bt,
                               int32_t bt_stride, const int32_t *seq_lens, int32_t num_seqs,
                               int32_t width, const MxScratch &to, int32_t dtype, hipStream_t s);
struct MxPrefillArgs;
// NaN to the outputs of the rows that see a marked block.
int32_t launch_mx_marks(const MxPrefillArgs &a, const MxScratch &from, int32_t width,
                        int32_t dtype, hipStream_t s);

// A decode step's new rows, one per sequence: its query rows are rotated at their positions,
// the rotated K row and the V row quantized to their slots, the sequence's last key. All are
// read 16 bytes at a time.
struct MxDecodeRope {
  const void *k, *v;
  int64_t k_ss, k_hs, v_ss, v_hs;
  const int64_t *positions, *slots;
  const void *cos_t, *sin_t;
  int64_t table_len;
};

// Decode attention over MXFP4 pools (decode_mxfp4.hip).
struct MxDecodeArgs {
  bool rope;
  MxDecodeRope step;
  const void *q;
  int64_t q_ss, q_hs;
  bool q_vec;  // query rows can be read 16 bytes at a time
  MxPool kc, vc;
  const int32_t *bt;
  int32_t bt_stride;
  const int32_t *seq_lens, *seq_order;
  int32_t num_q_heads, group;
  float scale_log2;
  int32_t split_keys;  // keys of a split: a multiple of the block size
  int32_t max_splits;
  int32_t key_cap;  // keys any sequence may have
  void *out;
  int64_t o_ss, o_hs;
  float *ws_m, *ws_l, *ws_acc;
};
int32_t launch_decode_mxfp4(const MxDecodeArgs &a, int32_t dtype, int32_t num_seqs,
                            hipStream_t s);

// Chunked prefill over them (prefill_mxfp4.hip).
struct MxPrefillArgs {
  const void *q;
  int64_t q_ts, q_hs;
  bool q_vec, o_vec;  // rows can be read and written 16 bytes at a time
  MxPool kc, vc;
  const int32_t *bt;
  int32_t bt_stride;
  const int32_t *seq_lens, *cu_q, *seq_order;
  int32_t num_seqs, num_tokens, group;
  float scale_log2;
  int32_t key_cap;  // keys any sequence may have
  int32_t tiles;    // of a sequence and KV head
  void *out;
  int64_t o_ts, o_hs;
};
int32_t launch_prefill_mxfp4(const MxPrefillArgs &a, int32_t max_query_len, int32_t dtype,
                             hipStream_t s);

}  // namespace tks
