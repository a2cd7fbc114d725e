// Device kernels of the operators an iteration calls, registered with the dispatcher
// from here: the addresses, strides and stream go to the C entry points without passing
// through Python (torch_ops.py declares the schemas and fake kernels, and keeps the other
// operators' device kernels). Small calls last as long as the host takes for them: the
// fused decode of 8 sequences 20.6 us through the ctypes binding and 12.5 us from here, the
// greedy choice of 16 rows 10.6 and 6.8 us, a 1.1B model's iteration (about 200 calls)
// 5,060 and 4,000 us.
//
// The entry points are looked up in libtokserve_hip.so on the first call, so loading this
// library does not touch HIP. It is loaded and registered by torch_ops.py, which first
// compares the versions it was built against (of torch, and of the C ABI that it calls
// through) with those it is loaded into. Errors are raised by tokserve_amd.kernels._lib, which maps a
// status to its exception.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Exceptions.h>
#include <torch/library.h>
#include <torch/headeronly/version.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <dlfcn.h>

#include <atomic>
#include <initializer_list>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>

#include "tokserve_hip.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

#define TKS_ENTRY_POINTS(X)              \
  X(tks_paged_attention_decode_workspace_bytes) \
  X(tks_paged_attention_decode)          \
  X(tks_paged_attention_decode_fp8)      \
  X(tks_paged_attention_decode_fp8_rows) \
  X(tks_paged_attention_prefill)         \
  X(tks_paged_attention_prefill_fp8_workspace_bytes) \
  X(tks_paged_attention_prefill_fp8)     \
  X(tks_paged_attention_prefill_fp8_rows) \
  X(tks_rope_append_paged_decode)        \
  X(tks_rope_append_paged_decode_fp8)    \
  X(tks_rope_append_paged_decode_fp8_rows) \
  X(tks_rope_kv_append)                  \
  X(tks_rope_kv_append_fp8)              \
  X(tks_rope_kv_append_fp8_rows)         \
  X(tks_kv_append)                       \
  X(tks_kv_append_fp8)                   \
  X(tks_kv_append_fp8_rows)              \
  X(tks_kv_append_mxfp4)                 \
  X(tks_paged_gather)                    \
  X(tks_paged_gather_fp8)                \
  X(tks_paged_gather_fp8_rows)           \
  X(tks_paged_gather_mxfp4)              \
  X(tks_rms_norm)                        \
  X(tks_argmax)                          \
  X(tks_silu_mul)                        \
  X(tks_mxfp4_quantize)                  \
  X(tks_mxfp4_dequantize)                \
  X(tks_mxfp4_matmul_workspace_bytes)    \
  X(tks_mxfp4_matmul)                    \
  X(tks_mxfp4_linear_workspace_bytes)    \
  X(tks_mxfp4_linear)                    \
  X(tks_paged_attention_decode_mxfp4)    \
  X(tks_paged_attention_prefill_mxfp4_workspace_bytes) \
  X(tks_paged_attention_prefill_mxfp4)   \
  X(tks_rope_append_paged_decode_mxfp4)  \
  X(tks_rope_kv_append_mxfp4)

struct Library {
#define TKS_FIELD(name) decltype(&::name) name = nullptr;
  TKS_ENTRY_POINTS(TKS_FIELD)
#undef TKS_FIELD
};

// f() with the GIL held, its exception passed on as a kernel in Python would raise it.
template <typename F>
auto with_python(F f) {
  pybind11::gil_scoped_acquire gil;
  try {
    return f();
  } catch (pybind11::error_already_set &raised) {
    raised.restore();
    python_error error;
    error.persist();
    throw error;
  }
}

// The library _lib.load() loads (and checks).
Library look_up() {
  const std::string path = with_python([] {
    pybind11::module_ lib = pybind11::module_::import("tokserve_amd.kernels._lib");
    lib.attr("load")();
    return std::string(pybind11::str(lib.attr("library_path")()));
  });
  void *handle = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  if (handle == nullptr) throw std::runtime_error(dlerror());
  Library l;
#define TKS_LOOK_UP(name)                                            \
  l.name = reinterpret_cast<decltype(l.name)>(dlsym(handle, #name)); \
  if (l.name == nullptr) throw std::runtime_error(std::string("missing ") + #name);
  TKS_ENTRY_POINTS(TKS_LOOK_UP)
#undef TKS_LOOK_UP
  return l;
}

const Library &library() {
  static std::atomic<const Library *> ready{nullptr};
  if (const Library *l = ready.load(std::memory_order_acquire)) return *l;
  // Without the GIL, which look_up() takes under the lock of the static below.
  std::optional<pybind11::gil_scoped_release> released;
  if (PyGILState_Check()) released.emplace();
  static const Library loaded = look_up();
  ready.store(&loaded, std::memory_order_release);
  return loaded;
}

void check(int32_t status, const char *operation) {
  if (status == TKS_OK) return;
  with_python([&] {
    return pybind11::module_::import("tokserve_amd.kernels._lib").attr("check")(status, operation)
        .is_none();  // (raises)
  });
}

int32_t code(const Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return TKS_FLOAT32;
    case at::kHalf: return TKS_FLOAT16;
    case at::kBFloat16: return TKS_BFLOAT16;
    default: break;
  }
  return with_python([&] {
    return pybind11::module_::import("tokserve_amd.kernels._lib")
        .attr("dtype_code")(pybind11::handle(
            reinterpret_cast<PyObject *>(torch::getTHPDtype(t.scalar_type()))))
        .cast<int32_t>();  // (raises)
  });
}

tks_stream_t stream_of(const Tensor &t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

const void *ptr(const OptTensor &t) { return t ? t->const_data_ptr() : nullptr; }
void *mut(const OptTensor &t) { return t ? t->mutable_data_ptr() : nullptr; }
template <typename T>
T *as(const Tensor &t) { return static_cast<T *>(t.mutable_data_ptr()); }
template <typename T>
T *as(const OptTensor &t) { return static_cast<T *>(mut(t)); }
int32_t i32(int64_t x) { return static_cast<int32_t>(x); }
bool fp8(const Tensor &pool) { return pool.scalar_type() == at::kFloat8_e4m3fn; }
// MXFP4 pools hold two codes to an element.
bool mxfp4(const Tensor &pool) { return pool.scalar_type() == at::kFloat4_e2m1fn_x2; }
int32_t head_dim(const Tensor &pool) { return i32(pool.size(4) * (mxfp4(pool) ? 2 : 1)); }

// Scratch memory of one call, undefined for 0 bytes: from the caching allocator on the
// launch's stream, so no other call, stream or thread shares it.
Tensor scratch(int64_t bytes, const Tensor &query, const char *use) {
  TORCH_CHECK_VALUE(bytes >= 0, "invalid ", use, " workspace query");
  return bytes == 0 ? Tensor() : at::empty({bytes}, query.options().dtype(at::kByte));
}

// Split partials of a decode: the caller's workspace, or scratch.
// The MXFP4 matrix operators, and the cache's and the attention over MXFP4 pools, check their
// arguments here (Python does the same for traced calls): there the checks of a small product
// took 5 us of its 12.6, those of an append and a gather 11 of 21, of a decode 7 of 12.
bool is_float(const Tensor &t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf ||
         t.scalar_type() == at::kBFloat16;
}

void one_device(const char *op, const Tensor &first, std::initializer_list<const Tensor *> others) {
  TORCH_CHECK_VALUE(first.is_cuda(), op, " requires HIP device tensors");
  for (const Tensor *t : others) {
    if (t == nullptr) continue;
    TORCH_CHECK_VALUE(t->is_cuda(), op, " requires HIP device tensors");
    TORCH_CHECK_VALUE(t->device() == first.device(), op, ": tensors must use the same device");
  }
}

const Tensor *maybe(const OptTensor &t) { return t ? &*t : nullptr; }

void check_mxfp4_pools(const char *op, const Tensor &kc, const Tensor &vc,
                       const OptTensor &k_scales, const OptTensor &v_scales) {
  TORCH_CHECK_VALUE(kc.dim() == 5 && kc.sizes() == vc.sizes(),
                    "KV pools must both have shape (L, NB, Hkv, BS, Dh)");
  TORCH_CHECK_VALUE(kc.scalar_type() == vc.scalar_type(), "KV pools must use the same dtype");
  TORCH_CHECK_VALUE(kc.is_contiguous() && vc.is_contiguous(), "KV pools must be contiguous");
  const int64_t half = kc.size(4);
  TORCH_CHECK_VALUE(half % 16 == 0 && half >= 16 && half <= 64,
                    "MXFP4 KV pools need a head_dim of 32, 64, 96 or 128");
  TORCH_CHECK_VALUE(k_scales || v_scales, op, ": MXFP4 KV pools need k_scales and v_scales");
  TORCH_CHECK_VALUE(k_scales && v_scales, op, ": k_scales and v_scales go together");
  for (const Tensor *t : {&*k_scales, &*v_scales}) {
    const char *name = t == &*k_scales ? "k_scales" : "v_scales";
    TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat8_e8m0fnu, name,
                     " of MXFP4 pools must be float8_e8m0fnu");
    TORCH_CHECK_VALUE(t->dim() == 5 && t->sizes().slice(0, 4) == kc.sizes().slice(0, 4) &&
                          t->size(4) == half / 16 && t->is_contiguous(),
                      name, " must be a contiguous (L, NB, Hkv, BS, Dh / 32) tensor");
  }
}

Tensor int_tensor(const Tensor &t, at::ScalarType type, const char *name) {
  TORCH_CHECK_TYPE(t.scalar_type() == type, name, " must be torch.",
                   type == at::kLong ? "int64" : "int32");
  return t.contiguous();
}

// The arguments that decode and prefill share; query, tables, lengths and order as the kernels
// take them.
struct AttentionArgs {
  Tensor query, tables, lens;
  OptTensor order;
};
AttentionArgs check_mxfp4_attention(const char *op, const Tensor &query, const Tensor &kc,
                                    const Tensor &vc, const Tensor &tables, const Tensor &lens,
                                    const OptTensor &order, const Tensor &out,
                                    const OptTensor &k_scales, const OptTensor &v_scales,
                                    const Tensor *more, const char *rows) {
  one_device(op, query, {&kc, &vc, &tables, &lens, maybe(order), &out, maybe(k_scales),
                         maybe(v_scales), more});
  check_mxfp4_pools(op, kc, vc, k_scales, v_scales);
  TORCH_CHECK_VALUE(query.dim() == 3 && query.size(2) == 2 * kc.size(4), "query must have shape (",
                    rows, ", Hq, Dh) with the pool's Dh");
  TORCH_CHECK_TYPE(is_float(query), op, ": query must be float32, float16 or bfloat16");
  TORCH_CHECK_VALUE(kc.size(2) > 0 && query.size(1) % kc.size(2) == 0,
                    "query head count must be divisible by KV head count");
  TORCH_CHECK_VALUE(out.sizes() == query.sizes() && out.scalar_type() == query.scalar_type() &&
                        (out.numel() == 0 || out.stride(2) == 1),
                    "out must match query and be contiguous in head_dim");
  AttentionArgs r{query.stride(2) == 1 ? query : query.contiguous(),
                  int_tensor(tables, at::kInt, "block_tables"),
                  int_tensor(lens, at::kInt, "seq_lens"), order};
  TORCH_CHECK_VALUE(tables.dim() == 2 && lens.dim() == 1 && lens.size(0) == tables.size(0),
                    "block_tables (B, max_blocks) and seq_lens (B,) must match query");
  if (order) {
    r.order = int_tensor(*order, at::kInt, "seq_order");
    TORCH_CHECK_VALUE(order->dim() == 1 && order->size(0) == lens.size(0),
                      "seq_order must have shape (B,)");
  }
  return r;
}

Tensor decode_workspace(const OptTensor &given, const Tensor &query, const Tensor &pool,
                        int64_t max_seq_len, int64_t pages_per_split) {
  if (given) return *given;
  return scratch(library().tks_paged_attention_decode_workspace_bytes(
                     i32(query.size(0)), i32(query.size(1)), i32(pool.size(2)), head_dim(pool),
                     i32(pool.size(3)), i32(max_seq_len), i32(pages_per_split)),
                 query, "decode");
}

void paged_attention_decode(const Tensor &q, const Tensor &key_cache,
                            const Tensor &value_cache, const Tensor &tables,
                            const Tensor &lens, const OptTensor &order, int64_t layer_index, int64_t max_seq_len, double scale,
                            int64_t pages_per_split, double k_scale, double v_scale,
                            const Tensor &out, const OptTensor &workspace,
                            const OptTensor &k_scales, const OptTensor &v_scales) {
  AttentionArgs args{q, tables, lens, order};
  if (mxfp4(key_cache)) {
    const char *op = "paged_attention_decode";
    args = check_mxfp4_attention(op, q, key_cache, value_cache, tables, lens, order, out, k_scales,
                                 v_scales, maybe(workspace), "B");
    TORCH_CHECK_VALUE(lens.size(0) == q.size(0),
                      "block_tables (B, max_blocks) and seq_lens (B,) must match query");
    TORCH_CHECK_VALUE(!workspace || (workspace->scalar_type() == at::kByte &&
                                     workspace->is_contiguous()),
                      "workspace must be a contiguous uint8 tensor");
  }
  const Tensor &query = args.query, &block_tables = args.tables, &seq_lens = args.lens;
  const OptTensor &seq_order = args.order;
  const c10::DeviceGuard guard(query.device());
  const Library &l = library();
  const Tensor ws = decode_workspace(workspace, query, key_cache, max_seq_len, pages_per_split);
  void *ws_ptr = ws.defined() ? ws.mutable_data_ptr() : nullptr;
  const int64_t ws_bytes = ws.defined() ? ws.numel() : 0;
  const Tensor &kc = key_cache;
  auto call = [&](auto entry, auto scales, auto... factors) {
    return std::apply(
        [&](auto... rows) {
          return entry(query.const_data_ptr(), query.stride(0), query.stride(1),
                       kc.const_data_ptr(), value_cache.const_data_ptr(), rows...,
                       i32(kc.size(0)), kc.size(1), i32(kc.size(2)), i32(kc.size(3)),
                       head_dim(kc), i32(layer_index), as<int32_t>(block_tables),
                       i32(block_tables.size(1)), as<int32_t>(seq_lens), as<int32_t>(seq_order),
                       i32(query.size(0)), i32(query.size(1)), i32(max_seq_len),
                       static_cast<float>(scale), i32(pages_per_split), out.mutable_data_ptr(),
                       out.stride(0), out.stride(1), ws_ptr, ws_bytes, factors..., code(query),
                       stream_of(query));
        },
        scales);
  };
  const auto none = std::tuple<>();
  check(mxfp4(kc) ? call(l.tks_paged_attention_decode_mxfp4,
                         std::make_tuple(ptr(k_scales), ptr(v_scales)))
        : k_scales ? call(l.tks_paged_attention_decode_fp8_rows,
                        std::make_tuple(as<const float>(k_scales), as<const float>(v_scales)))
        : fp8(kc) ? call(l.tks_paged_attention_decode_fp8, none, static_cast<float>(k_scale),
                         static_cast<float>(v_scale))
                  : call(l.tks_paged_attention_decode, none),
        "paged_attention_decode");
}

// The decoded pages of fp8 pools.
Tensor fp8_pages(const Tensor &query, const Tensor &pool, int64_t num_seqs, int64_t table_width,
                 int64_t max_seq_len) {
  return scratch(library().tks_paged_attention_prefill_fp8_workspace_bytes(
                     i32(num_seqs), i32(query.size(1)), i32(pool.size(2)), head_dim(pool),
                     i32(pool.size(3)), i32(table_width), i32(max_seq_len), code(query)),
                 query, "fp8 prefill");
}

void paged_attention_prefill(const Tensor &q, const Tensor &key_cache,
                             const Tensor &value_cache, const Tensor &tables,
                             const Tensor &lens, const Tensor &cu, const OptTensor &order,
                             int64_t layer_index,
                             int64_t max_query_len, int64_t max_seq_len, double scale,
                             double k_scale, double v_scale, const Tensor &out,
                             const OptTensor &k_scales, const OptTensor &v_scales) {
  AttentionArgs args{q, tables, lens, order};
  Tensor cu_seqlens_q = cu;
  if (mxfp4(key_cache)) {
    args = check_mxfp4_attention("paged_attention_prefill", q, key_cache, value_cache, tables,
                                 lens, order, out, k_scales, v_scales, &cu, "N");
    cu_seqlens_q = int_tensor(cu, at::kInt, "cu_seqlens_q");
    TORCH_CHECK_VALUE(cu.dim() == 1 && cu.size(0) == lens.size(0) + 1,
                      "block_tables (B, max_blocks), seq_lens (B,), cu_seqlens_q (B+1,)");
  }
  const Tensor &query = args.query, &block_tables = args.tables, &seq_lens = args.lens;
  const OptTensor &seq_order = args.order;
  const c10::DeviceGuard guard(query.device());
  const Library &l = library();
  const Tensor &kc = key_cache;
  auto call = [&](auto entry, auto scales, auto... tail) {
    return std::apply(
        [&](auto... rows) {
          return entry(query.const_data_ptr(), query.stride(0), query.stride(1),
                       kc.const_data_ptr(), value_cache.const_data_ptr(), rows...,
                       i32(kc.size(0)), kc.size(1), i32(kc.size(2)), i32(kc.size(3)),
                       head_dim(kc), i32(layer_index), as<int32_t>(block_tables),
                       i32(block_tables.size(1)), as<int32_t>(seq_lens),
                       as<int32_t>(cu_seqlens_q), as<int32_t>(seq_order), i32(seq_lens.size(0)),
                       query.size(0), i32(query.size(1)), i32(max_query_len), i32(max_seq_len),
                       static_cast<float>(scale), out.mutable_data_ptr(), out.stride(0),
                       out.stride(1), tail..., code(query), stream_of(query));
        },
        scales);
  };
  const auto none = std::tuple<>();
  int32_t status;
  if (mxfp4(kc)) {
    const Tensor ws = scratch(l.tks_paged_attention_prefill_mxfp4_workspace_bytes(
                                  i32(seq_lens.size(0)), query.size(0), i32(query.size(1)),
                                  i32(kc.size(2)), head_dim(kc), i32(kc.size(3)),
                                  i32(max_seq_len), code(query)),
                              query, "MXFP4 prefill");
    status = call(l.tks_paged_attention_prefill_mxfp4,
                  std::make_tuple(ptr(k_scales), ptr(v_scales)),
                  ws.defined() ? ws.mutable_data_ptr() : nullptr, ws.defined() ? ws.numel() : 0);
  } else if (fp8(kc)) {
    const Tensor ws =
        fp8_pages(query, kc, seq_lens.size(0), block_tables.size(1), max_seq_len);
    void *ws_ptr = ws.defined() ? ws.mutable_data_ptr() : nullptr;
    const int64_t ws_bytes = ws.defined() ? ws.numel() : 0;
    status = k_scales ? call(l.tks_paged_attention_prefill_fp8_rows,
                             std::make_tuple(as<const float>(k_scales), as<const float>(v_scales)),
                             ws_ptr, ws_bytes)
                      : call(l.tks_paged_attention_prefill_fp8, none, ws_ptr, ws_bytes,
                             static_cast<float>(k_scale), static_cast<float>(v_scale));
  } else {
    status = call(l.tks_paged_attention_prefill, none);
  }
  check(status, "paged_attention_prefill");
}

void rope_append_paged_decode(
    const Tensor &query, const Tensor &key, const Tensor &value, const Tensor &positions,
    const Tensor &cos, const Tensor &sin, const Tensor &slot_mapping, const Tensor &key_cache,
    const Tensor &value_cache, const Tensor &block_tables, const Tensor &seq_lens,
    const OptTensor &seq_order, int64_t layer_index, int64_t max_seq_len, double scale,
    int64_t pages_per_split, const Tensor &out, const OptTensor &workspace, double k_scale,
    double v_scale, const OptTensor &k_scales, const OptTensor &v_scales) {
  const c10::DeviceGuard guard(query.device());
  const Library &l = library();
  const Tensor ws = decode_workspace(workspace, query, key_cache, max_seq_len, pages_per_split);
  void *ws_ptr = ws.defined() ? ws.mutable_data_ptr() : nullptr;
  const int64_t ws_bytes = ws.defined() ? ws.numel() : 0;
  const Tensor &kc = key_cache;
  auto call = [&](auto entry, auto scales, auto... factors) {
    return std::apply(
        [&](auto... rows) {
          return entry(query.const_data_ptr(), query.stride(0), query.stride(1),
                       key.const_data_ptr(), key.stride(0), key.stride(1),
                       value.const_data_ptr(), value.stride(0), value.stride(1),
                       as<int64_t>(positions), cos.const_data_ptr(), sin.const_data_ptr(),
                       cos.size(0), as<int64_t>(slot_mapping), kc.mutable_data_ptr(),
                       value_cache.mutable_data_ptr(), rows..., i32(kc.size(0)), kc.size(1),
                       i32(kc.size(2)), i32(kc.size(3)), head_dim(kc), i32(layer_index),
                       as<int32_t>(block_tables), i32(block_tables.size(1)),
                       as<int32_t>(seq_lens), as<int32_t>(seq_order), i32(query.size(0)),
                       i32(query.size(1)), i32(max_seq_len), static_cast<float>(scale),
                       i32(pages_per_split), out.mutable_data_ptr(), out.stride(0),
                       out.stride(1), ws_ptr, ws_bytes, factors..., code(query),
                       stream_of(query));
        },
        scales);
  };
  const auto none = std::tuple<>();
  check(mxfp4(kc) ? call(l.tks_rope_append_paged_decode_mxfp4,
                         std::make_tuple(mut(k_scales), mut(v_scales)))
        : k_scales ? call(l.tks_rope_append_paged_decode_fp8_rows,
                        std::make_tuple(as<float>(k_scales), as<float>(v_scales)))
        : fp8(kc) ? call(l.tks_rope_append_paged_decode_fp8, none, static_cast<float>(k_scale),
                         static_cast<float>(v_scale))
                  : call(l.tks_rope_append_paged_decode, none),
        "rope_append_paged_decode");
}

void rope_kv_append(const Tensor &query, const Tensor &key, const Tensor &value,
                    const Tensor &positions, const Tensor &cos, const Tensor &sin,
                    const Tensor &key_cache, const Tensor &value_cache,
                    const Tensor &slot_mapping, int64_t layer_index, const Tensor &query_out,
                    const OptTensor &key_out, double k_scale, double v_scale,
                    const OptTensor &k_scales, const OptTensor &v_scales) {
  const c10::DeviceGuard guard(query.device());
  const Library &l = library();
  const Tensor &kc = key_cache;
  auto call = [&](auto entry, auto scales, auto... factors) {
    return std::apply(
        [&](auto... rows) {
          return entry(query.const_data_ptr(), query_out.mutable_data_ptr(), query.stride(0),
                       query.stride(1), query_out.stride(0), query_out.stride(1),
                       i32(query.size(1)), key.const_data_ptr(), mut(key_out), key.stride(0),
                       key.stride(1), key_out ? key_out->stride(0) : 0,
                       key_out ? key_out->stride(1) : 0, value.const_data_ptr(),
                       value.stride(0), value.stride(1), i32(kc.size(2)), query.size(0),
                       head_dim(kc), as<int64_t>(positions), cos.const_data_ptr(),
                       sin.const_data_ptr(), cos.size(0), kc.mutable_data_ptr(),
                       value_cache.mutable_data_ptr(), rows..., i32(kc.size(0)), kc.size(1),
                       i32(kc.size(3)), i32(layer_index), as<int64_t>(slot_mapping), factors...,
                       code(query), stream_of(query));
        },
        scales);
  };
  const auto none = std::tuple<>();
  check(mxfp4(kc) ? call(l.tks_rope_kv_append_mxfp4,
                         std::make_tuple(mut(k_scales), mut(v_scales)))
        : k_scales ? call(l.tks_rope_kv_append_fp8_rows,
                        std::make_tuple(as<float>(k_scales), as<float>(v_scales)))
        : fp8(kc) ? call(l.tks_rope_kv_append_fp8, none, static_cast<float>(k_scale),
                         static_cast<float>(v_scale))
                  : call(l.tks_rope_kv_append, none),
        "rope_kv_append");
}

void rope_kv_append_(const Tensor &query, const Tensor &key, const Tensor &value,
                     const Tensor &positions, const Tensor &cos, const Tensor &sin,
                     const Tensor &key_cache, const Tensor &value_cache,
                     const Tensor &slot_mapping, int64_t layer_index, const OptTensor &key_out,
                     double k_scale, double v_scale, const OptTensor &k_scales,
                     const OptTensor &v_scales) {
  rope_kv_append(query, key, value, positions, cos, sin, key_cache, value_cache, slot_mapping,
                 layer_index, query, key_out, k_scale, v_scale, k_scales, v_scales);
}

void kv_append(const Tensor &key_rows, const Tensor &value_rows, const Tensor &key_cache,
               const Tensor &value_cache, const Tensor &slot_mapping, int64_t layer_index,
               double k_scale, double v_scale, const OptTensor &k_scales,
               const OptTensor &v_scales) {
  const Tensor &kc = key_cache;
  Tensor key = key_rows, value = value_rows, slots = slot_mapping;
  if (mxfp4(kc)) {
    const char *op = "kv_append";
    one_device(op, key, {&value, &kc, &value_cache, &slots, maybe(k_scales), maybe(v_scales)});
    check_mxfp4_pools(op, kc, value_cache, k_scales, v_scales);
    TORCH_CHECK_VALUE(key.dim() == 3 && key.sizes() == value.sizes(),
                      "key and value must have shape (N, Hkv, Dh)");
    TORCH_CHECK_VALUE(key.size(1) == kc.size(2) && key.size(2) == 2 * kc.size(4),
                      "key rows must match the pool's (Hkv, Dh)");
    TORCH_CHECK_VALUE(is_float(key) && value.scalar_type() == key.scalar_type(),
                      "keys and values must match the storage dtype");
    TORCH_CHECK_VALUE(slots.dim() == 1 && slots.size(0) == key.size(0),
                      "slot_mapping must have shape (N,)");
    slots = int_tensor(slots, at::kLong, "slot_mapping");
    if (key.stride(2) != 1) key = key.contiguous();
    if (value.stride(2) != 1) value = value.contiguous();
  }
  const c10::DeviceGuard guard(key.device());
  const Library &l = library();
  auto call = [&](auto entry, auto scales, auto... factors) {
    return std::apply(
        [&](auto... rows) {
          return entry(key.const_data_ptr(), key.stride(0), key.stride(1),
                       value.const_data_ptr(), value.stride(0), value.stride(1), key.size(0),
                       kc.mutable_data_ptr(), value_cache.mutable_data_ptr(), rows...,
                       i32(kc.size(0)), kc.size(1), i32(kc.size(2)), i32(kc.size(3)),
                       head_dim(kc), i32(layer_index), as<int64_t>(slots), factors...,
                       code(key), stream_of(key));
        },
        scales);
  };
  const auto none = std::tuple<>();
  check(mxfp4(kc) ? call(l.tks_kv_append_mxfp4, std::make_tuple(mut(k_scales), mut(v_scales)))
        : k_scales ? call(l.tks_kv_append_fp8_rows,
                          std::make_tuple(as<float>(k_scales), as<float>(v_scales)))
        : fp8(kc) ? call(l.tks_kv_append_fp8, none, static_cast<float>(k_scale),
                         static_cast<float>(v_scale))
                  : call(l.tks_kv_append, none),
        "kv_append");
}

void paged_gather(const Tensor &key_cache, const Tensor &value_cache, const Tensor &tables,
                  const Tensor &lens, const Tensor &cu, int64_t layer_index,
                  int64_t max_seq_len, const Tensor &key_out, const Tensor &value_out,
                  double k_scale, double v_scale, const OptTensor &k_scales,
                  const OptTensor &v_scales) {
  const Tensor &kc = key_cache;
  Tensor block_tables = tables, seq_lens = lens, cu_seqlens = cu;
  if (mxfp4(kc)) {
    const char *op = "paged_gather";
    one_device(op, kc, {&value_cache, &tables, &lens, &cu, &key_out, &value_out, maybe(k_scales),
                        maybe(v_scales)});
    check_mxfp4_pools(op, kc, value_cache, k_scales, v_scales);
    TORCH_CHECK_VALUE(tables.dim() == 2, "block_tables must have shape (B, max_blocks)");
    block_tables = int_tensor(tables, at::kInt, "block_tables");
    seq_lens = int_tensor(lens, at::kInt, "seq_lens");
    cu_seqlens = int_tensor(cu, at::kInt, "cu_seqlens");
    TORCH_CHECK_VALUE(lens.numel() >= tables.size(0) && cu.numel() >= tables.size(0),
                      "seq_lens and cu_seqlens must have an entry per row of block_tables");
    TORCH_CHECK_VALUE(key_out.dim() == 3 && key_out.size(1) == kc.size(2) &&
                          key_out.size(2) == 2 * kc.size(4),
                      "outputs must have shape (S, Hkv, Dh)");
    TORCH_CHECK_VALUE(value_out.sizes() == key_out.sizes() &&
                          value_out.strides() == key_out.strides(),
                      "key_out and value_out must share shape and strides");
    TORCH_CHECK_VALUE(key_out.stride(2) == 1, "outputs must be contiguous in head_dim");
    TORCH_CHECK_VALUE(is_float(key_out) && value_out.scalar_type() == key_out.scalar_type(),
                      "outputs must match the storage dtype");
  }
  const c10::DeviceGuard guard(key_cache.device());
  const Library &l = library();
  auto call = [&](auto entry, auto scales, auto... factors) {
    return std::apply(
        [&](auto... rows) {
          return entry(kc.const_data_ptr(), value_cache.const_data_ptr(), rows...,
                       i32(kc.size(0)), kc.size(1), i32(kc.size(2)), i32(kc.size(3)),
                       head_dim(kc), i32(layer_index), as<int32_t>(block_tables),
                       i32(block_tables.size(1)), as<int32_t>(seq_lens), as<int32_t>(cu_seqlens),
                       i32(block_tables.size(0)), i32(max_seq_len), key_out.mutable_data_ptr(),
                       value_out.mutable_data_ptr(), key_out.stride(0), key_out.stride(1),
                       factors..., code(key_out), stream_of(key_out));
        },
        scales);
  };
  const auto none = std::tuple<>();
  check(mxfp4(kc) ? call(l.tks_paged_gather_mxfp4, std::make_tuple(ptr(k_scales), ptr(v_scales)))
        : k_scales ? call(l.tks_paged_gather_fp8_rows,
                          std::make_tuple(as<const float>(k_scales), as<const float>(v_scales)))
        : fp8(kc) ? call(l.tks_paged_gather_fp8, none, static_cast<float>(k_scale),
                         static_cast<float>(v_scale))
                  : call(l.tks_paged_gather, none),
        "paged_gather");
}

void rms_norm(const Tensor &input, const Tensor &weight, double epsilon,
              const OptTensor &residual, const Tensor &out, const OptTensor &residual_out) {
  check(library().tks_rms_norm(
            input.const_data_ptr(), input.stride(0), ptr(residual),
            residual ? residual->stride(0) : 0, mut(residual_out),
            residual_out ? residual_out->stride(0) : 0, weight.const_data_ptr(),
            out.mutable_data_ptr(), out.stride(0), input.size(0), i32(input.size(1)),
            static_cast<float>(epsilon), code(input), code(weight), code(out), stream_of(input)),
        "rms_norm");
}

void greedy_argmax(const Tensor &logits, const Tensor &out) {
  check(library().tks_argmax(logits.const_data_ptr(), logits.stride(0), logits.size(0),
                             logits.size(1), as<int64_t>(out), code(logits), stream_of(logits)),
        "greedy_argmax");
}

void silu_mul(const Tensor &gate_up, const Tensor &out) {
  check(library().tks_silu_mul(gate_up.const_data_ptr(), gate_up.stride(0), gate_up.size(0),
                               gate_up.size(1) / 2, out.mutable_data_ptr(), out.stride(0),
                               code(gate_up), stream_of(gate_up)),
        "silu_mul");
}

bool same_lead(const Tensor &a, const Tensor &b) {
  return a.dim() == b.dim() && a.sizes().slice(0, a.dim() - 1) == b.sizes().slice(0, b.dim() - 1);
}

int64_t float_depth(const char *op, const Tensor &t, const char *name) {
  TORCH_CHECK_TYPE(is_float(t), op, ": ", name, " must be float32, float16 or bfloat16");
  const int64_t depth = t.dim() ? t.size(-1) : 0;
  TORCH_CHECK_VALUE(depth >= 1 && depth % 32 == 0, op, ": the last dimension of ", name,
                    " must be a positive multiple of 32");
  return depth;
}

int64_t mxfp4_depth(const char *op, const Tensor &codes, const Tensor &scales, const char *name) {
  TORCH_CHECK_TYPE(codes.scalar_type() == at::kFloat4_e2m1fn_x2 &&
                       scales.scalar_type() == at::kFloat8_e8m0fnu,
                   op, ": ", name, " codes must be float4_e2m1fn_x2 and scales float8_e8m0fnu");
  const int64_t half = codes.dim() ? codes.size(-1) : 0;
  TORCH_CHECK_VALUE(half >= 1 && half % 16 == 0, op, ": ", name,
                    " must hold a positive multiple of 32 values a row");
  TORCH_CHECK_VALUE(same_lead(codes, scales) && scales.size(-1) == half / 16, op, ": ", name,
                    " scales must have one entry per 32 values");
  TORCH_CHECK_VALUE(codes.is_contiguous() && scales.is_contiguous(), op, ": ", name,
                    " codes and scales must be contiguous");
  return 2 * half;
}

int64_t weight_depth(const char *op, const Tensor &codes, const Tensor &scales, const char *name) {
  TORCH_CHECK_VALUE(codes.dim() == 2 && codes.size(0) >= 1, op, ": ", name,
                    " must have shape (N, K) and at least one row");
  return mxfp4_depth(op, codes, scales, name);
}

void check_rows_out(const char *op, const Tensor &out, const Tensor &rows, int64_t width) {
  TORCH_CHECK_VALUE(same_lead(out, rows) && out.size(-1) == width &&
                        (out.numel() == 0 || out.stride(-1) == 1),
                    op, ": out must have shape (..., ", width, ") after the rows', its last "
                    "dimension contiguous");
  TORCH_CHECK_VALUE(out.dim() == 2 || out.is_contiguous(), op,
                    ": an out of other than two dimensions must be contiguous");
}

void check_space(const char *op, const OptTensor &workspace) {
  TORCH_CHECK_VALUE(!workspace || (workspace->scalar_type() == at::kByte &&
                                   workspace->is_contiguous()),
                    op, ": workspace must be a contiguous uint8 tensor");
}

// Rows and row stride of a matrix whose last dimension is `width` long and contiguous (of
// other than two dimensions: contiguous).
int64_t rows_of(const Tensor &t, int64_t width) {
  return t.dim() == 2 ? t.size(0) : t.numel() / width;
}
int64_t row_stride(const Tensor &t, int64_t width) { return t.dim() == 2 ? t.stride(0) : width; }
// The input as such a matrix, copied where it is not one.
Tensor as_rows(const Tensor &t) {
  return t.dim() == 2 ? (t.stride(1) == 1 ? t : t.contiguous()) : t.contiguous();
}

void mxfp4_quantize(const Tensor &input, const Tensor &codes, const Tensor &scales) {
  const char *op = "mxfp4_quantize";
  one_device(op, input, {&codes, &scales});
  const int64_t depth = float_depth(op, input, "inputs");
  TORCH_CHECK_VALUE(mxfp4_depth(op, codes, scales, "output") == depth && same_lead(codes, input),
                    op, ": codes must have shape (..., K / 2)");
  const c10::DeviceGuard guard(input.device());
  const Tensor x = as_rows(input);
  check(library().tks_mxfp4_quantize(x.const_data_ptr(), row_stride(x, depth), rows_of(x, depth),
                                     depth, codes.mutable_data_ptr(), scales.mutable_data_ptr(),
                                     code(x), stream_of(x)),
        op);
}

void mxfp4_dequantize(const Tensor &codes, const Tensor &scales, const Tensor &out) {
  const char *op = "mxfp4_dequantize";
  one_device(op, codes, {&scales, &out});
  TORCH_CHECK_TYPE(is_float(out), op, ": out must be float32, float16 or bfloat16");
  const int64_t depth = mxfp4_depth(op, codes, scales, "input");
  check_rows_out(op, out, codes, depth);
  const c10::DeviceGuard guard(codes.device());
  check(library().tks_mxfp4_dequantize(codes.const_data_ptr(), scales.const_data_ptr(),
                                       rows_of(out, depth), depth, out.mutable_data_ptr(),
                                       row_stride(out, depth), code(out), stream_of(out)),
        op);
}

void mxfp4_matmul(const Tensor &a_codes, const Tensor &a_scales, const Tensor &b_codes,
                  const Tensor &b_scales, const Tensor &out, const OptTensor &workspace) {
  const char *op = "mxfp4_matmul";
  one_device(op, a_codes, {&a_scales, &b_codes, &b_scales, &out, maybe(workspace)});
  TORCH_CHECK_TYPE(is_float(out), op, ": out must be float32, float16 or bfloat16");
  const int64_t depth = mxfp4_depth(op, a_codes, a_scales, "A");
  TORCH_CHECK_VALUE(weight_depth(op, b_codes, b_scales, "B") == depth, op, ": B must have A's K");
  const int64_t width = b_codes.size(0);
  check_rows_out(op, out, a_codes, width);
  check_space(op, workspace);
  const c10::DeviceGuard guard(a_codes.device());
  const Library &l = library();
  const int64_t rows = rows_of(out, width);
  const Tensor ws = workspace ? *workspace
                              : scratch(l.tks_mxfp4_matmul_workspace_bytes(rows, width, depth),
                                        out, op);
  check(l.tks_mxfp4_matmul(a_codes.const_data_ptr(), a_scales.const_data_ptr(),
                           b_codes.const_data_ptr(), b_scales.const_data_ptr(), rows, width, depth,
                           out.mutable_data_ptr(), row_stride(out, width),
                           ws.defined() ? ws.mutable_data_ptr() : nullptr,
                           ws.defined() ? ws.numel() : 0, code(out), stream_of(out)),
        op);
}

void mxfp4_linear(const Tensor &input, const Tensor &weight_codes, const Tensor &weight_scales,
                  const Tensor &out, const OptTensor &workspace) {
  const char *op = "mxfp4_linear";
  one_device(op, input, {&weight_codes, &weight_scales, &out, maybe(workspace)});
  const int64_t depth = float_depth(op, input, "inputs");
  TORCH_CHECK_VALUE(out.scalar_type() == input.scalar_type(), op,
                    ": out must have the inputs' dtype");
  TORCH_CHECK_VALUE(weight_depth(op, weight_codes, weight_scales, "the weight") == depth, op,
                    ": the weight must have the inputs' K");
  const int64_t width = weight_codes.size(0);
  check_rows_out(op, out, input, width);
  check_space(op, workspace);
  const c10::DeviceGuard guard(input.device());
  const Library &l = library();
  const Tensor x = as_rows(input);
  const int64_t rows = rows_of(x, depth);
  const Tensor ws = workspace ? *workspace
                              : scratch(l.tks_mxfp4_linear_workspace_bytes(rows, width, depth), x,
                                        op);
  check(l.tks_mxfp4_linear(x.const_data_ptr(), row_stride(x, depth), weight_codes.const_data_ptr(),
                           weight_scales.const_data_ptr(), rows, width, depth,
                           out.mutable_data_ptr(), row_stride(out, width),
                           ws.defined() ? ws.mutable_data_ptr() : nullptr,
                           ws.defined() ? ws.numel() : 0, code(x), stream_of(x)),
        op);
}

}  // namespace

extern "C" const char *tks_torch_built_for(void) { return TORCH_VERSION; }

extern "C" int32_t tks_torch_abi_version(void) { return TKS_ABI_VERSION; }

// Registers the device kernels, once; null, or why not.
extern "C" const char *tks_torch_register(void) {
  static std::string error;
  try {
    static const torch::Library kernels = [] {
      torch::Library m(torch::Library::IMPL, "tokserve_amd", c10::DispatchKey::CUDA, __FILE__,
                       __LINE__);
      m.impl("paged_attention_decode", paged_attention_decode);
      m.impl("paged_attention_prefill", paged_attention_prefill);
      m.impl("rope_append_paged_decode", rope_append_paged_decode);
      m.impl("rope_kv_append", rope_kv_append);
      m.impl("rope_kv_append_", rope_kv_append_);
      m.impl("kv_append", kv_append);
      m.impl("paged_gather", paged_gather);
      m.impl("rms_norm", rms_norm);
      m.impl("greedy_argmax", greedy_argmax);
      m.impl("silu_mul", silu_mul);
      m.impl("mxfp4_quantize", mxfp4_quantize);
      m.impl("mxfp4_dequantize", mxfp4_dequantize);
      m.impl("mxfp4_matmul", mxfp4_matmul);
      m.impl("mxfp4_linear", mxfp4_linear);
      return m;
    }();
  } catch (const std::exception &raised) {
    error = raised.what();
    return error.c_str();
  }
  return nullptr;
}
