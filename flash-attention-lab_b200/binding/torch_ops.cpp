// PyTorch binding of the C ABI for eager calls (flash_lab/ops.py calls it when it is built).
//
// The same work as the ctypes path of flash_lab/ops.py (_prefill / _decode): allocate o, lse and
// the decode workspace with ATen on the inputs' device, fill flb_attn_params /
// flb_decode_params, call flb_prefill_fwd / flb_decode_fwd on the device's current stream and
// turn a nonzero status into RuntimeError with the library's message. Calling through here
// instead of ctypes keeps an eager call's host cost near the reference's C++ extension
// (csrc/bindings.cpp there), which registers its ops the same way. No kernel code is here: the
// library behind include/flash_lab_b200.h does the work.
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <initializer_list>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>
#include <unordered_map>
#include <utility>

#include "flash_lab_b200.h"

namespace {

int dtype_code(at::ScalarType t, bool allow_fp32) {
  switch (t) {
    case at::kBFloat16: return FLB_BF16;
    case at::kHalf: return FLB_FP16;
    case at::kFloat:
      if (allow_fp32) return FLB_FP32;
      [[fallthrough]];
    default: return -1;
  }
}

// The message flash_lab/ops.py raises for a failed call: "<what>: <status>: <detail>".
[[noreturn]] void raise_status(const char* what, int status) {
  std::string msg = std::string(what) + ": " + flb_status_string(status);
  const char* detail = flb_last_error();
  if (detail != nullptr && detail[0] != '\0') msg += std::string(": ") + detail;
  throw std::runtime_error(msg);
}

flb_stream_t current_stream(const at::Tensor& t) {
  return reinterpret_cast<flb_stream_t>(at::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

std::tuple<at::Tensor, at::Tensor> prefill(const at::Tensor& q, const at::Tensor& k,
                                           const at::Tensor& v, bool causal, double scale,
                                           int64_t status) {
  const int code = dtype_code(q.scalar_type(), false);
  if (code < 0 || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
    throw std::runtime_error("prefill takes bf16 or fp16 tensors of one dtype, got " +
                             std::string(c10::toString(q.scalar_type())));
  if (q.stride(-1) != 1 || k.stride(-1) != 1 || v.stride(-1) != 1)
    throw std::runtime_error("q, k, v must be contiguous in head_dim");
  const c10::cuda::CUDAGuard guard(q.device());
  const int64_t batch = q.size(0), seqlen_q = q.size(1), heads = q.size(2), head_dim = q.size(3);
  at::Tensor o = at::empty({batch, seqlen_q, heads, head_dim}, q.options());
  at::Tensor lse = at::empty({batch, heads, seqlen_q}, q.options().dtype(at::kFloat));
  flb_attn_params p{};
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.o = o.data_ptr();
  p.lse = lse.data_ptr<float>();
  p.q_batch_stride = q.stride(0);
  p.q_seq_stride = q.stride(1);
  p.q_head_stride = q.stride(2);
  p.k_batch_stride = k.stride(0);
  p.k_seq_stride = k.stride(1);
  p.k_head_stride = k.stride(2);
  p.v_batch_stride = v.stride(0);
  p.v_seq_stride = v.stride(1);
  p.v_head_stride = v.stride(2);
  p.o_batch_stride = o.stride(0);
  p.o_seq_stride = o.stride(1);
  p.o_head_stride = o.stride(2);
  p.batch = static_cast<int32_t>(batch);
  p.seqlen_q = static_cast<int32_t>(seqlen_q);
  p.seqlen_k = static_cast<int32_t>(k.size(1));
  p.heads = static_cast<int32_t>(heads);
  p.heads_kv = static_cast<int32_t>(k.size(2));
  p.head_dim = static_cast<int32_t>(head_dim);
  p.causal = causal ? 1 : 0;
  p.dtype = code;
  p.softmax_scale = static_cast<float>(scale);
  p.status = reinterpret_cast<int32_t*>(status);
  if (int st = flb_prefill_fwd(&p, current_stream(q))) raise_status("flb_prefill_fwd", st);
  return {o, lse};
}

std::tuple<at::Tensor, at::Tensor> decode(const at::Tensor& q, const at::Tensor& k_cache,
                                          const at::Tensor& v_cache, const at::Tensor& seq_lens,
                                          const std::optional<at::Tensor>& block_tables,
                                          double scale, int64_t num_splits, bool allow_splits,
                                          int64_t status, int64_t sm_count) {
  const int code = dtype_code(q.scalar_type(), true);
  if (code < 0)
    throw std::runtime_error("decode takes bf16, fp16 or fp32, got " +
                             std::string(c10::toString(q.scalar_type())));
  // q is [B, H, D], or [B, 1, H, D] (one query token per sequence), and o takes its shape.
  const bool q4 = q.dim() == 4 && q.size(1) == 1;
  if ((q.dim() != 3 && !q4) || k_cache.dim() != 4)
    throw std::runtime_error("q must be [B, H, D], caches [B, S_max, H_kv, D]");
  if (seq_lens.scalar_type() != at::kInt || !seq_lens.is_contiguous())
    throw std::runtime_error("seq_lens must be contiguous int32");
  const c10::cuda::CUDAGuard guard(q.device());
  const int hd = q4 ? 2 : 1;   // q's head dimension
  const int64_t batch = q.size(0), heads = q.size(hd), head_dim = q.size(hd + 1);
  const int64_t heads_kv = k_cache.size(2);
  flb_decode_params p{};
  int64_t max_seqlen = k_cache.size(1);
  if (block_tables.has_value()) {
    const at::Tensor& bt = *block_tables;
    if (bt.scalar_type() != at::kInt || bt.dim() != 2 || bt.stride(1) != 1)
      throw std::runtime_error("block_tables must be [B, max_blocks] int32 with unit column stride");
    max_seqlen = bt.size(1) * k_cache.size(1);
    p.block_tables = bt.data_ptr<int32_t>();
    p.block_table_stride = bt.stride(0);
    p.page_size = static_cast<int32_t>(k_cache.size(1));
    p.num_blocks = static_cast<int32_t>(k_cache.size(0));
  }
  // num_splits 0 lets the library choose (the count of flb_decode_num_splits, and one CTA per
  // SM for a length-balanced launch); the resolved count sizes the workspace.
  int32_t splits = 1, abi_splits = 1;
  if (allow_splits) {
    if (num_splits > 0) {
      splits = abi_splits = static_cast<int32_t>(num_splits);
    } else {
      abi_splits = 0;
      splits = flb_decode_num_splits(static_cast<int32_t>(batch), static_cast<int32_t>(heads),
                                     static_cast<int32_t>(heads_kv),
                                     static_cast<int32_t>(head_dim),
                                     static_cast<int32_t>(max_seqlen),
                                     static_cast<int32_t>(sm_count));
    }
  }
  const size_t ws_bytes = flb_decode_workspace_bytes(
      static_cast<int32_t>(batch), static_cast<int32_t>(heads), static_cast<int32_t>(head_dim),
      splits);
  at::Tensor workspace;
  if (ws_bytes > 0)
    workspace = at::empty({static_cast<int64_t>(ws_bytes)}, q.options().dtype(at::kByte));
  at::Tensor o = q4 ? at::empty({batch, 1, heads, head_dim}, q.options())
                    : at::empty({batch, heads, head_dim}, q.options());
  at::Tensor lse = at::empty({batch, heads}, q.options().dtype(at::kFloat));
  p.q = q.data_ptr();
  p.k_cache = k_cache.data_ptr();
  p.v_cache = v_cache.data_ptr();
  p.o = o.data_ptr();
  p.lse = lse.data_ptr<float>();
  p.seq_lens = seq_lens.data_ptr<int32_t>();
  p.q_batch_stride = q.stride(0);
  p.q_head_stride = q.stride(hd);
  p.k_batch_stride = k_cache.stride(0);
  p.k_seq_stride = k_cache.stride(1);
  p.k_head_stride = k_cache.stride(2);
  p.v_batch_stride = v_cache.stride(0);
  p.v_seq_stride = v_cache.stride(1);
  p.v_head_stride = v_cache.stride(2);
  p.o_batch_stride = o.stride(0);
  p.o_head_stride = o.stride(hd);
  p.batch = static_cast<int32_t>(batch);
  p.heads = static_cast<int32_t>(heads);
  p.heads_kv = static_cast<int32_t>(heads_kv);
  p.head_dim = static_cast<int32_t>(head_dim);
  p.max_seqlen = static_cast<int32_t>(max_seqlen);
  p.num_splits = abi_splits;
  p.dtype = code;
  p.softmax_scale = static_cast<float>(scale);
  p.workspace = ws_bytes > 0 ? workspace.data_ptr() : nullptr;
  p.workspace_bytes = ws_bytes;
  p.status = reinterpret_cast<int32_t*>(status);
  if (int st = flb_decode_fwd(&p, current_stream(q))) raise_status("flb_decode_fwd", st);
  return {o, lse};
}

// The KV-cache ops (flash_lab/kvcache.py, which checks shapes and dtypes before calling these).
using OptTensor = std::optional<at::Tensor>;

int cache_dtype_code(at::ScalarType t) {
  return t == at::kChar ? static_cast<int>(FLB_INT8) : dtype_code(t, true);
}

int32_t size32(int64_t n) {
  if (n < 0 || n > INT32_MAX) throw std::runtime_error("a size does not fit in 32 bits");
  return static_cast<int32_t>(n);
}

const int32_t* i32_ptr(const OptTensor& t) {
  return t.has_value() ? t->data_ptr<int32_t>() : nullptr;
}

flb_kv_cache cache_struct(const at::Tensor& k_cache, const at::Tensor& v_cache,
                          const at::Tensor& seq_lens, const OptTensor& block_tables,
                          const OptTensor& k_scale, const OptTensor& v_scale) {
  if (k_cache.dim() != 4 || v_cache.dim() != 4 || v_cache.sizes() != k_cache.sizes() ||
      v_cache.scalar_type() != k_cache.scalar_type() || k_cache.stride(3) != 1 ||
      v_cache.stride(3) != 1)
    throw std::runtime_error("caches must be two alike 4-D tensors, contiguous in head_dim");
  flb_kv_cache c{};
  c.k_cache = k_cache.data_ptr();
  c.v_cache = v_cache.data_ptr();
  c.k_batch_stride = k_cache.stride(0);
  c.k_seq_stride = k_cache.stride(1);
  c.k_head_stride = k_cache.stride(2);
  c.v_batch_stride = v_cache.stride(0);
  c.v_seq_stride = v_cache.stride(1);
  c.v_head_stride = v_cache.stride(2);
  for (const OptTensor* s : {&k_scale, &v_scale}) {
    if (s->has_value() && ((*s)->dim() != 3 || (*s)->sizes() != k_cache.sizes().slice(0, 3)))
      throw std::runtime_error("scales must be [outer, rows, H_kv] like the cache");
  }
  if (k_scale.has_value()) {
    c.k_scale = k_scale->data_ptr<float>();
    c.ks_batch_stride = k_scale->stride(0);
    c.ks_seq_stride = k_scale->stride(1);
    c.ks_head_stride = k_scale->stride(2);
  }
  if (v_scale.has_value()) {
    c.v_scale = v_scale->data_ptr<float>();
    c.vs_batch_stride = v_scale->stride(0);
    c.vs_seq_stride = v_scale->stride(1);
    c.vs_head_stride = v_scale->stride(2);
  }
  c.batch = size32(seq_lens.numel());
  c.heads_kv = size32(k_cache.size(2));
  c.head_dim = size32(k_cache.size(3));
  c.max_seqlen = size32(k_cache.size(1));
  c.dtype = cache_dtype_code(k_cache.scalar_type());
  if (block_tables.has_value()) {
    if (block_tables->dim() != 2 || block_tables->size(0) != c.batch ||
        block_tables->stride(1) != 1)
      throw std::runtime_error("block_tables must be [B, max_blocks] int32 with unit column stride");
    c.block_tables = block_tables->data_ptr<int32_t>();
    c.block_table_stride = block_tables->stride(0);
    c.page_size = size32(k_cache.size(1));
    c.num_blocks = size32(k_cache.size(0));
    c.max_seqlen = size32(block_tables->size(1) * k_cache.size(1));
  } else if (k_cache.size(0) != c.batch) {
    throw std::runtime_error("the cache and seq_lens differ in batch size");
  }
  return c;
}

flb_kv_rows rows_struct(const at::Tensor& k, const at::Tensor& v, const flb_kv_cache& c,
                        const OptTensor& cu_seqlens, const at::Tensor& seq_lens,
                        int64_t rows_per_seq) {
  if (k.dim() != 3 || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type() ||
      k.size(1) != c.heads_kv || k.size(2) != c.head_dim || k.stride(2) != 1 || v.stride(2) != 1)
    throw std::runtime_error("k and v must be [rows, H_kv, D], contiguous in head_dim");
  if (cu_seqlens.has_value() && cu_seqlens->numel() != int64_t{c.batch} + 1)
    throw std::runtime_error("cu_seqlens must be [B + 1]");
  flb_kv_rows r{};
  r.k = k.data_ptr();
  r.v = v.data_ptr();
  r.k_row_stride = k.stride(0);
  r.k_head_stride = k.stride(1);
  r.v_row_stride = v.stride(0);
  r.v_head_stride = v.stride(1);
  r.cu_seqlens = i32_ptr(cu_seqlens);
  r.seq_lens = seq_lens.data_ptr<int32_t>();
  r.rows = size32(k.size(0));
  r.rows_per_seq = size32(rows_per_seq);
  r.dtype = dtype_code(k.scalar_type(), true);
  return r;
}

void kv_append(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache,
               const at::Tensor& v_cache, const at::Tensor& seq_lens, const OptTensor& cu_seqlens,
               const OptTensor& block_tables, const OptTensor& k_scale, const OptTensor& v_scale,
               int64_t rows_per_seq) {
  const c10::cuda::CUDAGuard guard(k.device());
  const flb_kv_cache c = cache_struct(k_cache, v_cache, seq_lens, block_tables, k_scale, v_scale);
  const flb_kv_rows r = rows_struct(k, v, c, cu_seqlens, seq_lens, rows_per_seq);
  if (int st = flb_kv_append(&c, &r, current_stream(k))) raise_status("flb_kv_append", st);
  // As for any in-place write, so that autograd notices where it had saved one of these. Tensors of
  // inference mode have no version.
  auto written = [](const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  };
  written(k_cache);
  written(v_cache);
  if (k_scale.has_value()) written(*k_scale);
  if (v_scale.has_value()) written(*v_scale);
}

std::tuple<at::Tensor, at::Tensor> kv_gather(const at::Tensor& k_cache, const at::Tensor& v_cache,
                                             const at::Tensor& seq_lens,
                                             const at::Tensor& cu_seqlens,
                                             const OptTensor& block_tables,
                                             const OptTensor& k_scale, const OptTensor& v_scale,
                                             int64_t total, at::ScalarType dtype) {
  const c10::cuda::CUDAGuard guard(k_cache.device());
  const flb_kv_cache c = cache_struct(k_cache, v_cache, seq_lens, block_tables, k_scale, v_scale);
  const auto options = k_cache.options().dtype(dtype);
  at::Tensor k = at::empty({total, k_cache.size(2), k_cache.size(3)}, options);
  at::Tensor v = at::empty({total, k_cache.size(2), k_cache.size(3)}, options);
  const flb_kv_rows r = rows_struct(k, v, c, cu_seqlens, seq_lens, 0);
  if (int st = flb_kv_gather(&c, &r, current_stream(k_cache))) raise_status("flb_kv_gather", st);
  return {k, v};
}

std::tuple<at::Tensor, at::Tensor> extend(const at::Tensor& q_in, const at::Tensor& k_cache,
                                          const at::Tensor& v_cache, const at::Tensor& seq_lens,
                                          const OptTensor& cu_seqlens,
                                          const OptTensor& block_tables, const OptTensor& k_scale,
                                          const OptTensor& v_scale, int64_t rows_per_seq,
                                          bool causal, double scale, int64_t status,
                                          int64_t sm_count) {
  if (q_in.dim() != 3 || q_in.stride(2) != 1)
    throw std::runtime_error("q must be [rows, H, D], contiguous in head_dim");
  const c10::cuda::CUDAGuard guard(q_in.device());
  // Queries expanded over rows or heads are copied.
  const bool expanded = (q_in.size(0) > 1 && q_in.stride(0) == 0) ||
                        (q_in.size(1) > 1 && q_in.stride(1) == 0);
  const at::Tensor q = expanded ? q_in.contiguous() : q_in;
  const flb_kv_cache c = cache_struct(k_cache, v_cache, seq_lens, block_tables, k_scale, v_scale);
  if (q.size(2) != c.head_dim) throw std::runtime_error("q and the cache differ in head_dim");
  if (cu_seqlens.has_value() && cu_seqlens->numel() != int64_t{c.batch} + 1)
    throw std::runtime_error("cu_seqlens must be [B + 1]");
  flb_extend_params p{};
  p.rows = size32(q.size(0));
  p.heads = size32(q.size(1));
  at::Tensor o = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
  at::Tensor lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
  const size_t ws_bytes = flb_extend_workspace_bytes(p.rows, p.heads, c.heads_kv, c.head_dim,
                                                     static_cast<int32_t>(sm_count));
  at::Tensor workspace = at::empty({static_cast<int64_t>(ws_bytes)}, q.options().dtype(at::kByte));
  p.q = q.data_ptr();
  p.o = o.data_ptr();
  p.lse = lse.data_ptr<float>();
  p.q_row_stride = q.stride(0);
  p.q_head_stride = q.stride(1);
  p.o_row_stride = o.stride(0);
  p.o_head_stride = o.stride(1);
  p.cu_seqlens = i32_ptr(cu_seqlens);
  p.seq_lens = seq_lens.data_ptr<int32_t>();
  p.rows_per_seq = size32(rows_per_seq);
  p.causal = causal ? 1 : 0;
  p.dtype = dtype_code(q.scalar_type(), false);
  p.softmax_scale = static_cast<float>(scale);
  p.workspace = workspace.data_ptr();
  p.workspace_bytes = ws_bytes;
  p.status = reinterpret_cast<int32_t*>(status);
  if (int st = flb_extend_fwd(&c, &p, current_stream(q))) raise_status("flb_extend_fwd", st);
  return {o, lse};
}

// Eager calls whose metadata (shapes, strides, dtypes, devices and the arguments that the checks
// read) passed flash_lab/kvcache.py's checks before go straight to the ops above: *_known() records a
// call that passed, *_fast() runs a recorded one and returns None for any other. The checks depend
// on nothing else, so every error still comes from Python, in its order.
struct Known {
  int64_t status = 0, sm_count = 0;
};

class KnownCalls {
 public:
  const Known* find(const std::string& key) const {
    const auto it = calls_.find(key);
    return it == calls_.end() ? nullptr : &it->second;
  }
  void add(std::string key, Known value) {
    if (calls_.size() >= 4096) calls_.clear();   // many distinct shapes: start over, not grow
    calls_[std::move(key)] = value;
  }

 private:
  std::unordered_map<std::string, Known> calls_;   // under the GIL
};

KnownCalls g_known;

template <typename V>
void put(std::string& key, V value) {
  key.append(reinterpret_cast<const char*>(&value), sizeof(value));
}

// Appends the metadata of plain tensors (or None); false for anything else.
bool put_tensors(std::string& key, std::initializer_list<py::handle> tensors) {
  for (const py::handle& h : tensors) {
    if (h.is_none()) {
      key.push_back('n');
      continue;
    }
    if (!THPVariable_CheckExact(h.ptr())) return false;
    const at::Tensor& t = THPVariable_Unpack(h.ptr());
    key.push_back('t');
    put(key, static_cast<int16_t>(t.scalar_type()));
    put(key, static_cast<int16_t>(t.device().type()));
    put(key, static_cast<int16_t>(t.device().index()));
    put(key, static_cast<int16_t>(t.dim()));
    for (int64_t n : t.sizes()) put(key, n);
    for (int64_t n : t.strides()) put(key, n);
  }
  return true;
}

OptTensor optional_tensor(py::handle h) {
  return h.is_none() ? OptTensor{} : OptTensor{THPVariable_Unpack(h.ptr())};
}

// Rows as the ops take them, [rows, H, D], and rows per sequence (0: from cu_seqlens).
at::Tensor flat_rows(const at::Tensor& x, bool ragged, int64_t* per_seq) {
  *per_seq = ragged ? 0 : x.dim() == 4 ? x.size(1) : 1;
  return x.dim() == 4 ? x.flatten(0, 1) : x;
}

bool append_key(std::string& key, py::handle k, py::handle v, py::handle kc, py::handle vc,
                py::handle lens, py::handle cu, py::handle tables, py::handle ks, py::handle vs) {
  key.push_back('a');
  return put_tensors(key, {k, v, kc, vc, lens, cu, tables, ks, vs});
}

void append_known(py::handle k, py::handle v, py::handle kc, py::handle vc, py::handle lens,
                  py::handle cu, py::handle tables, py::handle ks, py::handle vs) {
  std::string key;
  if (append_key(key, k, v, kc, vc, lens, cu, tables, ks, vs)) g_known.add(std::move(key), {});
}

py::object append_fast(py::handle k, py::handle v, py::handle kc, py::handle vc, py::handle lens,
                       py::handle cu, py::handle tables, py::handle ks, py::handle vs) {
  std::string key;
  if (!append_key(key, k, v, kc, vc, lens, cu, tables, ks, vs) || g_known.find(key) == nullptr)
    return py::none();
  int64_t per_seq = 0;
  const at::Tensor k3 = flat_rows(THPVariable_Unpack(k.ptr()), !cu.is_none(), &per_seq);
  const at::Tensor v3 = flat_rows(THPVariable_Unpack(v.ptr()), !cu.is_none(), &per_seq);
  kv_append(k3, v3, THPVariable_Unpack(kc.ptr()), THPVariable_Unpack(vc.ptr()),
            THPVariable_Unpack(lens.ptr()), optional_tensor(cu), optional_tensor(tables),
            optional_tensor(ks), optional_tensor(vs), per_seq);
  return py::bool_(true);
}

bool gather_key(std::string& key, py::handle kc, py::handle vc, py::handle lens, py::handle cu,
                int64_t total, py::handle tables, py::handle ks, py::handle vs, int dtype) {
  key.push_back('g');
  put(key, total);
  put(key, dtype);
  return put_tensors(key, {kc, vc, lens, cu, tables, ks, vs});
}

int dtype_of(py::handle dtype) {   // -1: not given
  return dtype.is_none() ? -1 : static_cast<int>(py::cast<at::ScalarType>(dtype));
}

void gather_known(py::handle kc, py::handle vc, py::handle lens, py::handle cu, int64_t total,
                  py::handle tables, py::handle ks, py::handle vs, py::handle dtype) {
  std::string key;
  if (gather_key(key, kc, vc, lens, cu, total, tables, ks, vs, dtype_of(dtype)))
    g_known.add(std::move(key), {});
}

py::object gather_fast(py::handle kc, py::handle vc, py::handle lens, py::handle cu, int64_t total,
                       py::handle tables, py::handle ks, py::handle vs, py::handle dtype) {
  std::string key;
  const int code = dtype_of(dtype);
  if (!gather_key(key, kc, vc, lens, cu, total, tables, ks, vs, code) ||
      g_known.find(key) == nullptr)
    return py::none();
  const at::Tensor& k_cache = THPVariable_Unpack(kc.ptr());
  const at::ScalarType own = k_cache.scalar_type();
  const at::ScalarType out = code >= 0           ? static_cast<at::ScalarType>(code)
                             : own == at::kChar ? at::kBFloat16
                                                : own;
  return py::cast(kv_gather(k_cache, THPVariable_Unpack(vc.ptr()), THPVariable_Unpack(lens.ptr()),
                            THPVariable_Unpack(cu.ptr()), optional_tensor(tables),
                            optional_tensor(ks), optional_tensor(vs), total, out));
}

// `entry` tells the callers of extend apart, whose checks differ.
bool extend_key(std::string& key, int entry, py::handle q, py::handle kc, py::handle vc,
                py::handle lens, py::handle cu, py::handle tables, py::handle ks, py::handle vs,
                bool causal, double scale) {
  key.push_back('e');
  put(key, entry);
  put(key, causal);
  put(key, scale);
  return put_tensors(key, {q, kc, vc, lens, cu, tables, ks, vs});
}

void extend_known(int entry, py::handle q, py::handle kc, py::handle vc, py::handle lens,
                  py::handle cu, py::handle tables, py::handle ks, py::handle vs, bool causal,
                  double scale, int64_t status, int64_t sm_count) {
  std::string key;
  if (extend_key(key, entry, q, kc, vc, lens, cu, tables, ks, vs, causal, scale))
    g_known.add(std::move(key), {status, sm_count});
}

// o and lse in the shapes of q.
py::object extend_fast(int entry, py::handle q, py::handle kc, py::handle vc, py::handle lens,
                       py::handle cu, py::handle tables, py::handle ks, py::handle vs,
                       bool causal, double scale) {
  std::string key;
  if (!extend_key(key, entry, q, kc, vc, lens, cu, tables, ks, vs, causal, scale))
    return py::none();
  const Known* known = g_known.find(key);
  if (known == nullptr) return py::none();
  const at::Tensor& rows = THPVariable_Unpack(q.ptr());
  int64_t per_seq = 0;
  const at::Tensor flat = flat_rows(rows, !cu.is_none(), &per_seq);
  auto [o, lse] = extend(flat, THPVariable_Unpack(kc.ptr()), THPVariable_Unpack(vc.ptr()),
                         THPVariable_Unpack(lens.ptr()), optional_tensor(cu),
                         optional_tensor(tables), optional_tensor(ks), optional_tensor(vs), per_seq,
                         causal, scale, known->status, known->sm_count);
  if (rows.dim() == 4) {
    o = o.view(rows.sizes());
    lse = lse.view(rows.sizes().slice(0, 3));
  }
  return py::make_tuple(o, lse);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "flash_lab's eager ops: ATen allocation + the sm_100a library's C ABI";
  m.def("prefill", &prefill, "o, lse of one prefill call (flb_prefill_fwd)");
  m.def("decode", &decode, "o, lse of one decode call (flb_decode_fwd)");
  m.def("kv_append", &kv_append, "writes rows into a KV cache (flb_kv_append)");
  m.def("kv_gather", &kv_gather, "k, v read back from a KV cache (flb_kv_gather)");
  m.def("extend", &extend, "o, lse of new tokens over a KV cache (flb_extend_fwd)");
  m.def("append_known", &append_known);
  m.def("append_fast", &append_fast, "kv_append of a call that passed the checks before, or None");
  m.def("gather_known", &gather_known);
  m.def("gather_fast", &gather_fast, "kv_gather of a call that passed the checks before, or None");
  m.def("extend_known", &extend_known);
  m.def("extend_fast", &extend_fast, "extend of a call that passed the checks before, or None");
  m.def("abi_version", &flb_version);
}
