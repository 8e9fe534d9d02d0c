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

#include "../../include/cq_b200.h"

namespace py = pybind11;
using at::Tensor;
using Opt = std::optional<Tensor>;

namespace {

std::string text(const char* s) { return s; }
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

py::object paged_attention(const Tensor& q_arg, const Tensor& k_cache, const Tensor& v_cache, const Tensor& table_arg,
                           const Tensor& lens, const Opt& rows, std::optional<double> scale, int64_t window, int64_t sinks,
                           const Opt& k_scale, const Opt& v_scale, const Opt& out_arg, bool return_lse) {
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
  const int index = device_of(q_arg, k_cache, v_cache, table_arg, lens, rows, k_scale, v_scale, out_arg);
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
  const int64_t bytes = cq_paged_attention_workspace_bytes(b, hq, hk, d, width * page, window, sinks);
  if (bytes > 0) ws = bytes_like(q, bytes);
  check_status("cq_paged_attention",
               cq_paged_attention(q.data_ptr(), q.stride(0), q.stride(1), dtype_code(dt), b, hq, hk, d, k_cache.data_ptr(),
                                  v_cache.data_ptr(), dtype_code(ct), pages, page, k_cache.stride(0), k_cache.stride(1),
                                  k_cache.stride(2), static_cast<const int32_t*>(table.data_ptr()), table_rows, width,
                                  row_stride(table), ptr<const int32_t>(rows), static_cast<const int32_t*>(lens.data_ptr()),
                                  static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(d))), window, sinks,
                                  ks, vs, out.data_ptr(), ptr<float>(lse), ptr(ws), bytes, stream_of(index)));
  if (return_lse) return py::make_tuple(out, *lse);
  return py::cast(out);
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
  m.def("paged_attention", &paged_attention);
  m.def("append_kv", &append_kv);
  m.def("pages_update", &pages_update);
  m.def("compact_pages", &compact_pages);
}
