// Host side of the decode-side operators: argument checks, outputs and workspaces, and the call of the C ABI
// (include/cq_b200.h) on the tensors' device and its current stream.
//
// These operators take a few microseconds on the GPU, less than their checks and a ctypes call with thirty arguments
// take in Python (11 us for the W4A16 linear, 15 us for the attention; here 5.8 and 5.7 us), so a decode step would wait for
// its host.  The Python functions of ops.py and kvcache.py document them and pass their arguments on.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <variant>

#include "../../include/cq_b200.h"

namespace py = pybind11;
using at::Tensor;
using Opt = std::optional<Tensor>;

namespace {

std::string text(const std::string& s) { return s; }
std::string text(int64_t v) { return std::to_string(v); }
std::string text(at::ScalarType t) { return c10::toString(t); }
std::string text(at::IntArrayRef v) {
  std::string s = "[";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + "]";
}
template <typename... Ts>
[[noreturn]] void refuse(const Ts&... parts) {
  std::string s;
  ((s += text(parts)), ...);
  throw py::value_error(s);
}

void check_status(const char* name, int status) {
  if (status != CQ_OK) py::module_::import("comfy_quant_bench_b200._lib").attr("check")(name, status);   // raises
}

// every tensor on one CUDA device: its index
void on_device(const Tensor& t, int& index) {
  if (!t.is_cuda()) refuse("comfy_quant_bench_b200 ops run on CUDA tensors only (no CPU fallback)");
  const int i = t.get_device();
  if (index < 0) index = i;
  else if (index != i) refuse("tensors on different devices: cuda:", index, " and cuda:", i);
}
void on_device(const Opt& t, int& index) {
  if (t) on_device(*t, index);
}
template <typename... Ts>
int device_of(const Ts&... ts) {
  int index = -1;
  (on_device(ts, index), ...);
  return index;
}

void* stream_of(int index) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream(); }
template <typename T = void>
T* ptr(const Opt& t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}
bool aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
bool half_type(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return CQ_DT_BF16;
    case at::kHalf: return CQ_DT_F16;
    case at::kFloat8_e4m3fn: return CQ_DT_FP8_E4M3;
    default: return -1;
  }
}

Tensor bytes_like(const Tensor& t, int64_t n) { return at::empty({n}, t.options().dtype(at::kByte)); }

// -------------------------------------------------------------------------------------------------------------
// W4A16 linear
// -------------------------------------------------------------------------------------------------------------

Tensor w4a16_linear(const Tensor& x, const Tensor& qweight, const Tensor& scale, const Tensor& zeros, Opt bias, int64_t group,
                    const Opt& out_arg) {
  const at::ScalarType dt = x.scalar_type();
  if (!half_type(dt)) refuse("x must be bf16 or f16, got ", dt);
  if (qweight.dim() != 2 || (qweight.scalar_type() != at::kChar && qweight.scalar_type() != at::kByte))
    refuse("qweight must be int8 or uint8 [N, K/2]");
  if (x.dim() < 1) refuse("x must have a last dimension of K");
  const int64_t k = x.size(-1), n = qweight.size(0);
  if (k != 2 * qweight.size(1)) refuse("Input K=", k, " does not match qweight K=", 2 * qweight.size(1));
  if ((group != 32 && group != 64 && group != 128) || k % group != 0)
    refuse("group_size must be 32, 64 or 128 and divide K=", k, ", got ", group);
  for (const Tensor* t : {&scale, &zeros})
    if (t->scalar_type() != at::kBFloat16 || t->dim() != 2 || t->size(0) != k / group || t->size(1) != n)
      refuse("scale and zeros must be bf16 [", k / group, ", ", n, "]");
  if (!qweight.is_contiguous() || !scale.is_contiguous() || !zeros.is_contiguous())
    refuse("qweight, scale and zeros must be contiguous");
  if (bias && bias->numel() != n) refuse("bias must have ", n, " elements");
  const int index = device_of(x, qweight, scale, zeros, bias, out_arg);
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));

  Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, k});
  if (!aligned16(x2) || (k > 1 && x2.stride(1) != 1) || (x2.size(0) > 1 && (x2.stride(0) % 8 != 0 || x2.stride(0) < k)))
    x2 = x2.clone(at::MemoryFormat::Contiguous);
  const int64_t m = x2.size(0), ldx = m > 1 ? x2.stride(0) : k;
  if (bias && (bias->scalar_type() != dt || bias->dim() != 1 || !bias->is_contiguous()))
    bias = bias->reshape({n}).to(dt).contiguous();
  auto shape = x.sizes().vec();
  shape.back() = n;
  Tensor out;
  if (out_arg) {
    out = *out_arg;
    if (out.scalar_type() != dt || out.sizes() != at::IntArrayRef(shape) || !out.is_contiguous())
      refuse("out must be contiguous ", dt, " of shape ", at::IntArrayRef(shape));
  } else {
    out = at::empty(shape, x.options());
  }
  const int64_t bytes = cq_w4a16_workspace_bytes(m, k, static_cast<int>(group));
  Opt ws;
  if (bytes > 0) ws = bytes_like(x, bytes);
  check_status("cq_w4a16_linear",
               cq_w4a16_linear(x2.data_ptr(), ldx, dtype_code(dt), m, k, n, qweight.data_ptr(), scale.data_ptr(),
                               zeros.data_ptr(), static_cast<int>(group), ptr(bias), out.data_ptr(), ptr(ws), bytes,
                               stream_of(index)));
  return out;
}

// -------------------------------------------------------------------------------------------------------------
// root-mean-square norm with the residual's addition
// -------------------------------------------------------------------------------------------------------------

// x as rows [M, C] whose last dimension is contiguous, 16-byte aligned where the width allows; a copy where it has to be
Tensor norm_rows(const Tensor& x, int64_t c) {
  Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, c});
  const int64_t ld = x2.size(0) > 1 ? x2.stride(0) : c;
  if ((c > 1 && x2.stride(1) != 1) || ld < c || (c % 8 == 0 && (!aligned16(x2) || ld % 8 != 0)))
    x2 = x2.clone(at::MemoryFormat::Contiguous);
  return x2;
}

py::tuple add_rmsnorm(const Tensor& x, Tensor weight, const Opt& residual, double eps, const std::optional<std::string>& quant,
                      int64_t group, const Opt& out_residual) {
  const at::ScalarType dt = x.scalar_type();
  if (!half_type(dt)) refuse("x must be bf16 or f16, got ", dt);
  if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > 32768) refuse("x must have a last dimension of 1 to 32768");
  const int64_t c = x.size(-1);
  if (weight.numel() != c) refuse("weight must have ", c, " elements");
  if (residual && (residual->scalar_type() != dt || residual->sizes() != x.sizes()))
    refuse("residual must be ", dt, " of shape ", x.sizes());
  int kind = CQ_NORM_SAME;
  if (quant) {
    if (*quant == "int8") kind = CQ_NORM_INT8;
    else if (*quant == "fp8") kind = CQ_NORM_FP8;
    else refuse("quant must be None, 'int8' or 'fp8', got '", *quant, "'");
  }
  if (group != 0 && (kind == CQ_NORM_SAME || (group != 32 && group != 64 && group != 128) || c % group != 0))
    refuse("group_size must be 0, or 32, 64 or 128 and divide ", c, " with an 8-bit output, got ", group);
  if (out_residual) {
    if (!residual) refuse("out_residual goes with a residual");
    if (out_residual->scalar_type() != dt || out_residual->sizes() != x.sizes() || !out_residual->is_contiguous())
      refuse("out_residual must be contiguous ", dt, " of shape ", x.sizes());
    if (c % 8 == 0 && !aligned16(*out_residual)) refuse("out_residual must be 16-byte aligned");
  }
  const int index = device_of(x, weight, residual, out_residual);
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));
  const Tensor x2 = norm_rows(x, c);
  const int64_t m = x2.size(0);
  Opt r2, h;
  if (residual) {
    r2 = norm_rows(*residual, c);
    h = out_residual ? *out_residual : at::empty(x.sizes(), x.options());
  }
  if (weight.scalar_type() != dt || weight.dim() != 1 || !weight.is_contiguous() || !aligned16(weight))
    weight = weight.reshape({c}).to(dt).clone(at::MemoryFormat::Contiguous);
  const at::ScalarType ot = kind == CQ_NORM_INT8 ? at::kChar : kind == CQ_NORM_FP8 ? at::kFloat8_e4m3fn : dt;
  const Tensor out = at::empty(x.sizes(), x.options().dtype(ot));
  Opt scale;
  if (quant) scale = group ? at::empty({c / group, m}, x.options().dtype(at::kFloat)) : at::empty({m}, x.options().dtype(at::kFloat));
  auto ld = [&](const Opt& t) { return t && t->dim() == 2 && m > 1 ? t->stride(0) : c; };
  check_status("cq_add_rmsnorm",
               cq_add_rmsnorm(x2.data_ptr(), ld(x2), ptr(r2), ld(r2), weight.data_ptr(), dtype_code(dt), m, c,
                              static_cast<float>(eps), kind, group, ptr(h), c, out.data_ptr(), ptr<float>(scale),
                              stream_of(index)));
  const Tensor kept = residual ? *h : x;
  if (quant) return py::make_tuple(out, *scale, kept);
  return py::make_tuple(out, kept);
}

// -------------------------------------------------------------------------------------------------------------
// sampling
// -------------------------------------------------------------------------------------------------------------

using Each = std::variant<Tensor, double>;     // one number, or one for each row

// an [n] array of a row parameter, or none and its number
Opt row_param(const Each& p, int64_t n, at::ScalarType type, const char* name, double least, double most, double& one) {
  if (const Tensor* t = std::get_if<Tensor>(&p)) {
    if (t->scalar_type() != type || t->dim() != 1 || t->size(0) != n) refuse(name, " must be a number or ", type, " [", n, "]");
    return *t;
  }
  one = std::get<double>(p);
  if (!(one >= least && one <= most)) refuse(name, " is out of range: ", std::to_string(one));
  if (type == at::kInt && one != std::floor(one)) refuse(name, " must be a whole number, got ", std::to_string(one));
  return std::nullopt;
}

py::object sample_tokens(const Tensor& logits_arg, const Tensor& uniform_arg, const Each& temperature, const Each& top_k,
                         const Each& top_p, const Each& min_p, bool return_logprob) {
  const at::ScalarType dt = logits_arg.scalar_type();
  if (logits_arg.dim() != 2 || (!half_type(dt) && dt != at::kFloat)) refuse("logits must be bf16, f16 or f32 [rows, vocab]");
  const int64_t rows = logits_arg.size(0), vocab = logits_arg.size(1);
  if (vocab < 1 || vocab > 327680) refuse("vocab must be 1 to 327680, got ", vocab);
  if (uniform_arg.scalar_type() != at::kFloat || uniform_arg.dim() != 1 || uniform_arg.size(0) != rows)
    refuse("uniform must be f32 [", rows, "]");
  double t = 0, k = 0, p = 0, m = 0;
  Opt ts = row_param(temperature, rows, at::kFloat, "temperature", 0, 1e30, t);
  Opt ks = row_param(top_k, rows, at::kInt, "top_k", 0, 2147483647.0, k);
  Opt ps = row_param(top_p, rows, at::kFloat, "top_p", 0, 1, p);
  Opt ms = row_param(min_p, rows, at::kFloat, "min_p", 0, 1, m);
  const int index = device_of(logits_arg, uniform_arg, ts, ks, ps, ms);
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));
  Tensor logits = logits_arg;
  if ((vocab > 1 && logits.stride(1) != 1) || (rows > 1 && logits.stride(0) < vocab)) logits = logits.clone(at::MemoryFormat::Contiguous);
  const Tensor uniform = uniform_arg.contiguous();
  for (Opt* o : {&ts, &ks, &ps, &ms})
    if (*o) *o = (*o)->contiguous();
  const Tensor tokens = at::empty({rows}, logits.options().dtype(at::kLong));
  Opt logprob;
  if (return_logprob) logprob = at::empty({rows}, logits.options().dtype(at::kFloat));
  check_status("cq_sample",
               cq_sample(logits.data_ptr(), rows > 1 ? logits.stride(0) : vocab, dt == at::kFloat ? CQ_DT_F32 : dtype_code(dt),
                         rows, vocab, uniform.data_ptr<float>(), ptr<const float>(ts), static_cast<float>(t),
                         ptr<const int32_t>(ks), static_cast<int64_t>(k), ptr<const float>(ps), static_cast<float>(p),
                         ptr<const float>(ms), static_cast<float>(m), tokens.data_ptr<int64_t>(), ptr<float>(logprob),
                         stream_of(index)));
  if (return_logprob) return py::make_tuple(tokens, *logprob);
  return py::cast(tokens);
}

// -------------------------------------------------------------------------------------------------------------
// paged cache
// -------------------------------------------------------------------------------------------------------------

void i32(const Tensor& t, int64_t dim, const char* name) {
  if (t.scalar_type() != at::kInt || t.dim() != dim || (!t.is_contiguous() && t.numel() > 0 && t.stride(-1) != 1))
    refuse(name, " must be int32 with ", dim, " dimension(s), its last one contiguous");
}

void cache_pair(const Tensor& k, const Tensor& v, int64_t dim) {
  if (k.dim() != dim || k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type() || dtype_code(k.scalar_type()) < 0)
    refuse("key and value cache must be bf16, f16 or float8_e4m3fn tensors of one shape and type: ", dim,
           " dimensions ending in [num_pages, kv_heads, page_size, head_dim]");
  if (k.strides() != v.strides() || k.stride(-1) != 1)
    refuse("key and value cache must have the same strides, the last one 1");
}

const float* head_scale(const Opt& s, int64_t heads, at::ScalarType cache, const char* name) {
  if (!s) return nullptr;
  if (cache != at::kFloat8_e4m3fn) refuse(name, " goes with a float8_e4m3fn cache");
  if (s->scalar_type() != at::kFloat || s->dim() != 1 || s->size(0) != heads || !s->is_contiguous())
    refuse(name, " must be contiguous f32 [", heads, "]");
  return s->data_ptr<float>();
}

// Rows that share memory (one row expanded to several, an overlapping view): the kernels take tables whose rows lie at
// least their width apart.
bool rows_overlap(const Tensor& table) { return table.size(0) > 1 && table.stride(0) < table.size(1); }
// a table that is only read: such a view is taken as its copy
Tensor read_table(const Tensor& table) { return rows_overlap(table) ? table.contiguous() : table; }
// one that is written has to have rows of its own
void written_table(const Tensor& table, const char* name) {
  if (rows_overlap(table)) refuse(name, " is written, but its rows share memory: strides ", table.strides(), " for shape ", table.sizes());
}
int64_t row_stride(const Tensor& table) { return table.size(0) > 1 ? table.stride(0) : table.size(1); }

using Prefix = std::variant<Tensor, int64_t>;   // tokens that all rows share

py::object attention(const Tensor& q_arg, const Tensor& k_cache, const Tensor& v_cache, const Tensor& table_arg,
                     const Tensor& lens, const Prefix* shared, int64_t weight_parts, const Opt& rows, std::optional<double> scale,
                     int64_t window, int64_t sinks, const Opt& k_scale, const Opt& v_scale, const Opt& out_arg, bool return_lse) {
  const at::ScalarType dt = q_arg.scalar_type(), ct = k_cache.scalar_type();
  if (q_arg.dim() != 3 || !half_type(dt)) refuse("q must be bf16 or f16 [B, q_heads, D]");
  const int64_t b = q_arg.size(0), hq = q_arg.size(1), d = q_arg.size(2);
  cache_pair(k_cache, v_cache, 4);
  const int64_t pages = k_cache.size(0), hk = k_cache.size(1), page = k_cache.size(2);
  if (k_cache.size(3) != d || (d != 64 && d != 128 && d != 256))
    refuse("head_dim must be 64, 128 or 256 in q and the caches, got ", d, " and ", k_cache.size(3));
  if (hk < 1 || hq < 1 || hq % hk != 0) refuse("q_heads (", hq, ") must be a multiple of kv_heads (", hk, ")");
  if (ct != dt && ct != at::kFloat8_e4m3fn) refuse("the caches must hold ", dt, " or float8_e4m3fn, got ", ct);
  if (window < 0 || sinks < 0) refuse("window and sinks must not be negative");
  i32(table_arg, 2, "block_table");
  i32(lens, 1, "seq_lens");
  const int64_t table_rows = table_arg.size(0), width = table_arg.size(1);
  if (lens.size(0) != table_rows) refuse("seq_lens must have one entry per table row (", table_rows, ")");
  if (rows) {
    i32(*rows, 1, "rows");
    if (rows->size(0) != b) refuse("rows must have ", b, " entries");
  } else if (b > table_rows) {
    refuse(b, " queries for ", table_rows, " table rows");
  }
  Opt prefix;
  int64_t prefix_len = 0;
  if (shared) {
    if (const Tensor* t = std::get_if<Tensor>(shared)) {
      if (t->scalar_type() != at::kInt || t->numel() != 1) refuse("prefix must be an int or an int32 tensor of one element");
      prefix = *t;
    } else {
      prefix_len = std::get<int64_t>(*shared);
      if (prefix_len < 0 || prefix_len > 2147483647) refuse("prefix must not be negative, got ", prefix_len);
    }
  }
  const int index = device_of(q_arg, k_cache, v_cache, table_arg, lens, rows, k_scale, v_scale, out_arg, prefix);
  const float* ks = head_scale(k_scale, hk, ct, "k_scale");
  const float* vs = head_scale(v_scale, hk, ct, "v_scale");
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));

  const Tensor table = read_table(table_arg);
  Tensor q = q_arg;
  if (!aligned16(q) || q.stride(2) != 1 || q.stride(0) % 8 != 0 || q.stride(1) % 8 != 0)
    q = q.clone(at::MemoryFormat::Contiguous);
  Tensor out;
  if (out_arg) {
    out = *out_arg;
    if (out.scalar_type() != dt || out.sizes() != q.sizes() || !out.is_contiguous())
      refuse("out must be contiguous ", dt, " [", b, ", ", hq, ", ", d, "]");
  } else {
    out = at::empty({b, hq, d}, q.options());
  }
  Opt lse, ws;
  if (return_lse) lse = at::empty({b, hq}, q.options().dtype(at::kFloat));
  const float factor = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(d)));
  if (shared) {
    const int64_t bytes = cq_prefix_attention_workspace_bytes(b, hq, hk, d, width * page);
    if (bytes > 0) ws = bytes_like(q, bytes);
    check_status("cq_prefix_attention",
                 cq_prefix_attention_parts(q.data_ptr(), q.stride(0), q.stride(1), dtype_code(dt), b, hq, hk, d, k_cache.data_ptr(),
                                           v_cache.data_ptr(), dtype_code(ct), pages, page, k_cache.stride(0),
                                           k_cache.stride(1), k_cache.stride(2), static_cast<const int32_t*>(table.data_ptr()),
                                           table_rows, width, row_stride(table), ptr<const int32_t>(rows),
                                           static_cast<const int32_t*>(lens.data_ptr()), ptr<const int32_t>(prefix),
                                           prefix_len, static_cast<int>(weight_parts), factor, ks, vs, out.data_ptr(),
                                           ptr<float>(lse), ptr(ws), bytes, stream_of(index)));
    if (return_lse) return py::make_tuple(out, *lse);
    return py::cast(out);
  }
  const int64_t bytes = cq_paged_attention_workspace_bytes(b, hq, hk, d, width * page, window, sinks);
  if (bytes > 0) ws = bytes_like(q, bytes);
  check_status("cq_paged_attention",
               cq_paged_attention(q.data_ptr(), q.stride(0), q.stride(1), dtype_code(dt), b, hq, hk, d, k_cache.data_ptr(),
                                  v_cache.data_ptr(), dtype_code(ct), pages, page, k_cache.stride(0), k_cache.stride(1),
                                  k_cache.stride(2), static_cast<const int32_t*>(table.data_ptr()), table_rows, width,
                                  row_stride(table), ptr<const int32_t>(rows), static_cast<const int32_t*>(lens.data_ptr()),
                                  factor, window, sinks, ks, vs, out.data_ptr(), ptr<float>(lse), ptr(ws), bytes, stream_of(index)));
  if (return_lse) return py::make_tuple(out, *lse);
  return py::cast(out);
}

py::object paged_attention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& table, const Tensor& lens,
                           const Opt& rows, std::optional<double> scale, int64_t window, int64_t sinks, const Opt& k_scale,
                           const Opt& v_scale, const Opt& out, bool return_lse) {
  return attention(q, k_cache, v_cache, table, lens, nullptr, 0, rows, scale, window, sinks, k_scale, v_scale, out, return_lse);
}
py::object prefix_attention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& table,
                            const Tensor& lens, const Prefix& prefix, const Opt& rows, std::optional<double> scale,
                            const Opt& k_scale, const Opt& v_scale, const Opt& out, bool return_lse,
                            std::optional<int64_t> weight_parts) {
  if (weight_parts && *weight_parts != 1 && *weight_parts != 2) refuse("weight_parts must be None, 1 or 2, got ", *weight_parts);
  return attention(q, k_cache, v_cache, table, lens, &prefix, weight_parts.value_or(0), rows, scale, 0, 0, k_scale, v_scale, out, return_lse);
}

// x, or a contiguous copy where its rows are not 16-byte aligned
Tensor aligned_rows(const Tensor& x) {
  bool ok = aligned16(x) && x.stride(-1) == 1;
  for (int64_t i = 0; i + 1 < x.dim(); ++i) ok = ok && x.stride(i) % 8 == 0;
  return ok ? x : x.clone(at::MemoryFormat::Contiguous);
}

void append_kv(const Tensor& k_arg, const Tensor& v_arg, const Tensor& k_cache, const Tensor& v_cache, const Tensor& table_arg,
               const Tensor& rows, const Tensor& positions, const Opt& k_scale, const Opt& v_scale) {
  const at::ScalarType dt = k_arg.scalar_type(), ct = k_cache.scalar_type();
  const int64_t dim = k_arg.dim();
  if ((dim != 3 && dim != 4) || k_arg.sizes() != v_arg.sizes() || dt != v_arg.scalar_type() || !half_type(dt))
    refuse("k and v must be bf16 or f16 of one shape, [T, kv_heads, D] or [layers, T, kv_heads, D]");
  cache_pair(k_cache, v_cache, dim + 1);
  const int64_t layers = dim == 4 ? k_arg.size(0) : 1, t = k_arg.size(-3), hk = k_arg.size(-2), d = k_arg.size(-1);
  if ((dim == 4 && k_cache.size(0) != layers) || k_cache.size(-3) != hk || k_cache.size(-1) != d)
    refuse("caches ", k_cache.sizes(), " do not fit k ", k_arg.sizes());
  if (ct != dt && ct != at::kFloat8_e4m3fn) refuse("the caches must hold ", dt, " or float8_e4m3fn, got ", ct);
  i32(table_arg, 2, "block_table");
  i32(rows, 1, "rows");
  i32(positions, 1, "positions");
  if (rows.size(0) != t || positions.size(0) != t) refuse("rows and positions must have one entry per token (", t, ")");
  const int index = device_of(k_arg, v_arg, k_cache, v_cache, table_arg, rows, positions, k_scale, v_scale);
  const float* ks = head_scale(k_scale, hk, ct, "k_scale");
  const float* vs = head_scale(v_scale, hk, ct, "v_scale");
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));
  const Tensor table = read_table(table_arg);
  const Tensor k = aligned_rows(k_arg), v = aligned_rows(v_arg);
  check_status("cq_kv_append",
               cq_kv_append(k.data_ptr(), dim == 4 ? k.stride(0) : 0, k.stride(-3), k.stride(-2), v.data_ptr(),
                            dim == 4 ? v.stride(0) : 0, v.stride(-3), v.stride(-2), dtype_code(dt), layers, t, hk, d,
                            k_cache.data_ptr(), v_cache.data_ptr(), dtype_code(ct), k_cache.size(-4), k_cache.size(-2),
                            dim == 4 ? k_cache.stride(0) : 0, k_cache.stride(-4), k_cache.stride(-3), k_cache.stride(-2),
                            static_cast<const int32_t*>(table.data_ptr()), table.size(0), table.size(1), row_stride(table),
                            static_cast<const int32_t*>(rows.data_ptr()), static_cast<const int32_t*>(positions.data_ptr()),
                            ks, vs, stream_of(index)));
}

void head_norm(const Opt& w, int64_t d, const char* name) {
  if (w && w->numel() != d) refuse(name, " must have ", d, " elements");
}
// a norm weight as the kernel reads it: of the type, contiguous and aligned
Opt norm_weight(const Opt& w, at::ScalarType dt) {
  if (!w || (w->scalar_type() == dt && w->dim() == 1 && w->is_contiguous() && aligned16(*w))) return w;
  return w->reshape({w->numel()}).to(dt).clone(at::MemoryFormat::Contiguous);
}

py::object append_rotated(const Tensor& q_arg, const Tensor& k_arg, const Tensor& v_arg, const Tensor& k_cache,
                          const Tensor& v_cache, const Tensor& table_arg, const Tensor& rows, const Tensor& positions,
                          const Tensor& rope_arg, bool interleaved, const Opt& q_norm_arg, const Opt& k_norm_arg, double eps,
                          const Opt& k_scale, const Opt& v_scale, bool return_k) {
  const at::ScalarType dt = q_arg.scalar_type(), ct = k_cache.scalar_type();
  if (q_arg.dim() != 3 || !half_type(dt)) refuse("q must be bf16 or f16 [T, q_heads, D]");
  if (k_arg.dim() != 3 || k_arg.sizes() != v_arg.sizes() || k_arg.scalar_type() != dt || v_arg.scalar_type() != dt)
    refuse("k and v must be ", dt, " of one shape, [T, kv_heads, D]");
  cache_pair(k_cache, v_cache, 4);
  const int64_t t = q_arg.size(0), hq = q_arg.size(1), d = q_arg.size(2), hk = k_arg.size(1);
  if (k_arg.size(0) != t || k_arg.size(2) != d) refuse("k ", k_arg.sizes(), " does not fit q ", q_arg.sizes());
  if (k_cache.size(1) != hk || k_cache.size(3) != d) refuse("caches ", k_cache.sizes(), " do not fit k ", k_arg.sizes());
  if (hq < 1 || hk < 1 || d < 16 || d > 256 || d % 8 != 0) refuse("head_dim must be a multiple of 8 from 16 to 256, got ", d);
  if (ct != dt && ct != at::kFloat8_e4m3fn) refuse("the caches must hold ", dt, " or float8_e4m3fn, got ", ct);
  i32(table_arg, 2, "block_table");
  i32(rows, 1, "rows");
  i32(positions, 1, "positions");
  if (rows.size(0) != t || positions.size(0) != t) refuse("rows and positions must have one entry per token (", t, ")");
  if (rope_arg.scalar_type() != at::kFloat || rope_arg.dim() != 3 || rope_arg.size(2) != 2 || rope_arg.size(0) < 1 ||
      !rope_arg.is_contiguous())
    refuse("rope must be contiguous f32 [positions, rot_dim / 2, 2]");
  const int64_t rot = 2 * rope_arg.size(1);
  if (rot < 16 || rot % 16 != 0 || rot > d) refuse("rope must turn a multiple of 16 columns, at most D=", d, ", got ", rot);
  head_norm(q_norm_arg, d, "q_norm");
  head_norm(k_norm_arg, d, "k_norm");
  const int index = device_of(q_arg, k_arg, v_arg, k_cache, v_cache, table_arg, rows, positions, rope_arg, q_norm_arg,
                              k_norm_arg, k_scale, v_scale);
  const float* ks = head_scale(k_scale, hk, ct, "k_scale");
  const float* vs = head_scale(v_scale, hk, ct, "v_scale");
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));
  const Tensor table = read_table(table_arg);
  const Tensor rope = aligned16(rope_arg) ? rope_arg : rope_arg.clone();
  const Tensor q = aligned_rows(q_arg), k = aligned_rows(k_arg), v = aligned_rows(v_arg);
  const Opt q_norm = norm_weight(q_norm_arg, dt), k_norm = norm_weight(k_norm_arg, dt);
  const Tensor q_out = at::empty({t, hq, d}, q.options());
  Opt k_out;
  if (return_k) k_out = at::empty({t, hk, d}, q.options());
  check_status("cq_kv_append_rotated",
               cq_kv_append_rotated(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
                                    v.stride(0), v.stride(1), dtype_code(dt), t, hq, hk, d, rope.data_ptr<float>(), rope.size(0),
                                    rot, interleaved, ptr(q_norm), ptr(k_norm), static_cast<float>(eps), q_out.data_ptr(),
                                    ptr(k_out), k_cache.data_ptr(), v_cache.data_ptr(), dtype_code(ct), k_cache.size(0),
                                    k_cache.size(2), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
                                    static_cast<const int32_t*>(table.data_ptr()), table.size(0), table.size(1),
                                    row_stride(table), static_cast<const int32_t*>(rows.data_ptr()),
                                    static_cast<const int32_t*>(positions.data_ptr()), ks, vs, stream_of(index)));
  if (return_k) return py::make_tuple(q_out, *k_out);
  return py::cast(q_out);
}

// caches [layers, num_pages, kv_heads, page_size, D] whose pages are one block each
struct PageLayout {
  int64_t layers = 0, layer_bytes = 0, page_bytes = 0;
};
PageLayout page_layout(const Tensor& k, const Tensor& v, int64_t pages) {
  cache_pair(k, v, 5);
  if (k.size(1) != pages) refuse("the caches have ", k.size(1), " pages, ref_counts ", pages);
  const int64_t per = k.size(2) * k.size(3) * k.size(4);
  if (!k.is_contiguous() && (k.stride(1) != per || k.stride(2) != k.size(3) * k.size(4) || k.stride(3) != k.size(4)))
    refuse("a layer of the caches must be contiguous, so that a page is one block");
  const int64_t size = static_cast<int64_t>(k.element_size());
  return {k.size(0), k.stride(0) * size, per * size};
}

py::object pages_update(const Tensor& table, const Tensor& lens, const Tensor& refs, int64_t page_size, const Opt& free_rows,
                        const Opt& src, const Opt& dst, const Opt& reserve, const Opt& counts, int64_t count,
                        const Opt& k_cache, const Opt& v_cache) {
  i32(table, 2, "block_table");
  written_table(table, "block_table");
  i32(lens, 1, "seq_lens");
  i32(refs, 1, "ref_counts");
  if (lens.size(0) != table.size(0)) refuse("seq_lens must have one entry per table row (", table.size(0), ")");
  if (!free_rows && !src && !dst && !reserve) refuse("rows must be an int32 tensor");
  if (src.has_value() != dst.has_value()) refuse("src and dst must both be int32 tensors");
  if (counts && !reserve) refuse("rows must be an int32 tensor, one entry per count");
  if (reserve && (!k_cache || !v_cache)) refuse("the caches are needed to reserve");
  if (free_rows) i32(*free_rows, 1, "rows");
  if (src) i32(*src, 1, "src");
  if (dst) i32(*dst, 1, "dst");
  if (src && src->size(0) != dst->size(0)) refuse("src and dst must have the same number of rows");
  if (reserve) i32(*reserve, 1, "rows");
  if (counts) {
    i32(*counts, 1, "count");
    if (counts->size(0) != reserve->size(0)) refuse("count must have one entry per row");
  }
  if (count < 0) refuse("count must not be negative");
  const int index = device_of(table, lens, refs, free_rows, src, dst, reserve, counts, k_cache, v_cache);
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));
  const int64_t pages = refs.size(0), n = reserve ? reserve->size(0) : 0;
  PageLayout layout;
  Opt start, copies, ws;
  int64_t bytes = 0;
  if (reserve) {
    layout = page_layout(*k_cache, *v_cache, pages);
    start = at::empty({n}, lens.options());
    copies = at::empty({n, 2}, lens.options());
    bytes = cq_pages_workspace_bytes(pages, n);
    if (bytes > 0) ws = bytes_like(lens, bytes);
  }
  check_status("cq_pages_update",
               cq_pages_update(static_cast<int32_t*>(table.data_ptr()), table.size(0), table.size(1), row_stride(table),
                               static_cast<int32_t*>(lens.data_ptr()), static_cast<int32_t*>(refs.data_ptr()), pages, page_size,
                               ptr<const int32_t>(free_rows), free_rows ? free_rows->size(0) : 0, ptr<const int32_t>(src),
                               ptr<const int32_t>(dst), dst ? dst->size(0) : 0, ptr<const int32_t>(reserve), n,
                               ptr<const int32_t>(counts), count, ptr<int32_t>(start), ptr<int32_t>(copies), ptr(k_cache),
                               ptr(v_cache), layout.layers, layout.layer_bytes, layout.page_bytes, ptr(ws), bytes,
                               stream_of(index)));
  if (!reserve) return py::none();
  return py::make_tuple(*start, *copies);
}

py::tuple compact_pages(const Tensor& table_arg, const Tensor& refs, const Tensor& k_cache, const Tensor& v_cache,
                        const Opt& out_table_arg, const Opt& out_refs_arg) {
  i32(table_arg, 2, "block_table");
  i32(refs, 1, "ref_counts");
  if (out_table_arg) {
    i32(*out_table_arg, 2, "out_table");
    written_table(*out_table_arg, "out_table");
    if (out_table_arg->sizes() != table_arg.sizes()) refuse("out_table must have the shape of block_table");
  }
  if (out_refs_arg) {
    i32(*out_refs_arg, 1, "out_refs");
    if (out_refs_arg->size(0) != refs.size(0)) refuse("out_refs must have the shape of ref_counts");
  }
  const int index = device_of(table_arg, refs, k_cache, v_cache, out_table_arg, out_refs_arg);
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));
  const int64_t pages = refs.size(0);
  const PageLayout layout = page_layout(k_cache, v_cache, pages);
  const Tensor table = read_table(table_arg);
  const Tensor out_table = out_table_arg ? *out_table_arg : at::empty(table.sizes(), refs.options());
  const Tensor out_refs = out_refs_arg ? *out_refs_arg : at::empty({pages}, refs.options());
  const Tensor moves = at::empty({pages / 2, 2}, refs.options());
  const Tensor ws = at::empty({pages}, refs.options());
  check_status("cq_pages_compact",
               cq_pages_compact(static_cast<const int32_t*>(table.data_ptr()), table.size(0), table.size(1), row_stride(table),
                                static_cast<int32_t*>(out_table.data_ptr()), row_stride(out_table),
                                static_cast<const int32_t*>(refs.data_ptr()), static_cast<int32_t*>(out_refs.data_ptr()), pages,
                                static_cast<int32_t*>(moves.data_ptr()), k_cache.data_ptr(), v_cache.data_ptr(), layout.layers,
                                layout.layer_bytes, layout.page_bytes, ws.data_ptr(), 4 * pages, stream_of(index)));
  return py::make_tuple(out_table, out_refs, moves);
}

}  // namespace

PYBIND11_MODULE(_decode, m) {
  m.def("w4a16_linear", &w4a16_linear);
  m.def("add_rmsnorm", &add_rmsnorm);
  m.def("sample_tokens", &sample_tokens);
  m.def("paged_attention", &paged_attention);
  m.def("prefix_attention", &prefix_attention);
  m.def("append_kv", &append_kv);
  m.def("append_rotated", &append_rotated);
  m.def("pages_update", &pages_update);
  m.def("compact_pages", &compact_pages);
}
