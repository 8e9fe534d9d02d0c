// extern "C" entry points of the decode-side operators (declared in include/cq_b200.h): the W4A16 linear and the
// paged key-value cache.  Argument checks on the host, then kernel launches on the caller's stream.
#include <cstdint>

#include "kernels.cuh"

namespace {

constexpr int64_t kMaxTokens = 1 << 20;          // of a W4A16 linear
constexpr int64_t kMaxSharedBits = 200 * 1024;   // bytes of the page and row bitmaps in one CTA's shared memory

bool valid16(int dtype) { return dtype == CQ_DT_BF16 || dtype == CQ_DT_F16; }
bool valid_page_size(int64_t s) { return s >= 8 && s <= 1024 && (s & (s - 1)) == 0; }
bool valid_head_dim(int64_t d) { return d == 64 || d == 128 || d == 256; }
bool fits_int(int64_t v) { return v >= 0 && v <= 0x7FFFFFFF; }

// sizes of a paged cache's bookkeeping
int check_tables(int64_t table_rows, int64_t table_width, int64_t table_stride, int64_t num_pages, int64_t page_size) {
  if (!fits_int(table_rows) || table_rows > (1 << 24) || !fits_int(table_width) || table_width > (1 << 20) ||
      table_stride < table_width || num_pages < 1 || !fits_int(num_pages) || !valid_page_size(page_size) ||
      table_width * page_size > 0x7FFFFFFF - 1024)      // room for a tile's key index past the row's end
    return CQ_ERR_SHAPE;
  return CQ_OK;
}

}  // namespace

extern "C" {

int64_t cq_w4a16_workspace_bytes(int64_t M, int64_t K, int group) {
  if (M < 0 || M > kMaxTokens || (group != 32 && group != 64 && group != 128) || K < group || K % group != 0 || K > kMaxK)
    return -1;
  return cq::w4a16_workspace(static_cast<int>(M), static_cast<int>(K), group);
}

int cq_w4a16_linear(const void* x, int64_t ldx, int dtype, int64_t M, int64_t K, int64_t N, const void* qweight,
                    const void* scale, const void* zeros, int group, const void* bias, void* out, void* workspace,
                    int64_t workspace_bytes, void* stream) {
  if (!valid16(dtype) || (group != 32 && group != 64 && group != 128)) return CQ_ERR_ARG;
  if (M < 0 || M > kMaxTokens || N < 0 || N > kMaxRows || K < group || K % group != 0 || K > kMaxK || ldx < K)
    return CQ_ERR_SHAPE;
  const int64_t need = cq_w4a16_workspace_bytes(M, K, group);
  if (workspace_bytes < need) return CQ_ERR_SHAPE;
  if (M == 0 || N == 0) return CQ_OK;
  if (x == nullptr || qweight == nullptr || scale == nullptr || zeros == nullptr || out == nullptr ||
      (workspace == nullptr && need > 0))
    return CQ_ERR_ARG;
  if (!aligned(x, 16) || ldx % 8 != 0 || !aligned(qweight, 16) || !aligned(scale, 2) || !aligned(zeros, 2) ||
      !aligned(bias, 2) || !aligned(out, 2) || !aligned(workspace, 256))
    return CQ_ERR_ALIGN;
  if (int dv = check_device()) return dv;
  const cq::W4A16Args a{x, static_cast<const uint8_t*>(qweight), static_cast<const __nv_bfloat16*>(scale),
                        static_cast<const __nv_bfloat16*>(zeros), bias, out, ldx, static_cast<int>(M),
                        static_cast<int>(N), static_cast<int>(K), group, dtype == CQ_DT_F16 ? 1 : 0};
  return cuda_status(cq::launch_w4a16(a, workspace, static_cast<cudaStream_t>(stream)));
}

int64_t cq_paged_attention_workspace_bytes(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                           int64_t span, int64_t window, int64_t sinks) {
  if (!fits_int(batch) || q_heads < 1 || kv_heads < 1 || q_heads > 4096 || q_heads % kv_heads != 0 ||
      !valid_head_dim(head_dim) || !fits_int(span) || window < 0 || sinks < 0)
    return -1;
  return cq::paged_attention_workspace(batch, static_cast<int>(q_heads), static_cast<int>(kv_heads),
                                       static_cast<int>(head_dim), span, window, sinks);
}

int cq_paged_attention(const void* q, int64_t q_batch_stride, int64_t q_head_stride, int dtype, int64_t batch,
                       int64_t q_heads, int64_t kv_heads, int64_t head_dim, const void* k_cache, const void* v_cache,
                       int cache_dtype, int64_t num_pages, int64_t page_size, int64_t page_stride,
                       int64_t head_stride, int64_t token_stride, const int32_t* block_table, int64_t table_rows,
                       int64_t table_width, int64_t table_stride, const int32_t* rows, const int32_t* seq_lens,
                       float scale, int64_t window, int64_t sinks, const float* k_scale, const float* v_scale,
                       void* out, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!valid16(dtype) || (cache_dtype != dtype && cache_dtype != CQ_DT_FP8_E4M3)) return CQ_ERR_ARG;
  if (window < 0 || sinks < 0) return CQ_ERR_ARG;
  if (int rc = check_tables(table_rows, table_width, table_stride, num_pages, page_size)) return rc;
  if (!fits_int(batch) || batch > 65535 || q_heads < 1 || kv_heads < 1 || q_heads > 4096 || q_heads % kv_heads != 0 ||
      !valid_head_dim(head_dim))
    return CQ_ERR_SHAPE;
  const int64_t need = cq_paged_attention_workspace_bytes(batch, q_heads, kv_heads, head_dim, table_width * page_size,
                                                          window, sinks);
  if (workspace_bytes < need) return CQ_ERR_SHAPE;
  if (batch == 0) return CQ_OK;
  if (q == nullptr || k_cache == nullptr || v_cache == nullptr || seq_lens == nullptr || out == nullptr ||
      (block_table == nullptr && table_width > 0) || (workspace == nullptr && need > 0))
    return CQ_ERR_ARG;
  const int vec = cache_dtype == CQ_DT_FP8_E4M3 ? 16 : 8;      // elements of a 16-byte access
  if (!aligned(q, 16) || q_batch_stride % 8 != 0 || q_head_stride % 8 != 0 || !aligned(k_cache, 16) ||
      !aligned(v_cache, 16) || page_stride % vec != 0 || head_stride % vec != 0 || token_stride % vec != 0 ||
      !aligned(block_table, 4) || !aligned(rows, 4) || !aligned(seq_lens, 4) || !aligned(k_scale, 4) ||
      !aligned(v_scale, 4) || !aligned(out, 16) || !aligned(lse, 4) || !aligned(workspace, 16))
    return CQ_ERR_ALIGN;
  if (int dv = check_device()) return dv;
  const int64_t top = 0x7FFFFFFF;
  const cq::PagedAttnArgs a{q, q_batch_stride, q_head_stride, k_cache, v_cache, page_stride, head_stride,
                            token_stride, block_table, table_stride, rows, seq_lens, k_scale, v_scale, out, lse,
                            workspace, static_cast<int>(batch), static_cast<int>(q_heads),
                            static_cast<int>(kv_heads), static_cast<int>(head_dim), static_cast<int>(num_pages),
                            static_cast<int>(page_size), static_cast<int>(table_rows), static_cast<int>(table_width),
                            dtype, cache_dtype, static_cast<int>(window < top ? window : top),
                            static_cast<int>(sinks < top ? sinks : top), scale};
  return cuda_status(cq::launch_paged_attention(a, static_cast<cudaStream_t>(stream)));
}

int64_t cq_pages_workspace_bytes(int64_t num_pages, int64_t reserved_rows) {
  if (!fits_int(num_pages) || !fits_int(reserved_rows)) return -1;
  return 4 * (2 * reserved_rows + num_pages);
}

int cq_pages_update(int32_t* block_table, int64_t table_rows, int64_t table_width, int64_t table_stride,
                    int32_t* seq_lens, int32_t* ref_counts, int64_t num_pages, int64_t page_size,
                    const int32_t* free_rows, int64_t n_free, const int32_t* src_rows, const int32_t* dst_rows,
                    int64_t n_fork, const int32_t* reserve_rows, int64_t n_reserve, const int32_t* counts,
                    int64_t count, int32_t* start, int32_t* copies, void* k_cache, void* v_cache, int64_t layers,
                    int64_t layer_bytes, int64_t page_bytes, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_tables(table_rows, table_width, table_stride, num_pages, page_size)) return rc;
  if (!fits_int(n_free) || !fits_int(n_fork) || !fits_int(n_reserve) || !fits_int(count) || layers < 0 ||
      layers > 65535 || n_free > table_rows || n_fork > table_rows || n_reserve > table_rows)
    return CQ_ERR_SHAPE;
  if (layers > 0 && (page_bytes < 16 || page_bytes % 16 != 0 || layer_bytes % 16 != 0)) return CQ_ERR_SHAPE;
  if (n_reserve > 0 && workspace_bytes < cq_pages_workspace_bytes(num_pages, n_reserve)) return CQ_ERR_SHAPE;
  if (cq::pages_branch_shared(static_cast<int>(table_rows), static_cast<int>(num_pages)) > kMaxSharedBits)
    return CQ_ERR_CAPACITY;
  if (n_free == 0 && n_fork == 0 && n_reserve == 0) return CQ_OK;
  if (block_table == nullptr || seq_lens == nullptr || ref_counts == nullptr || (n_free > 0 && free_rows == nullptr) ||
      (n_fork > 0 && (src_rows == nullptr || dst_rows == nullptr)) ||
      (n_reserve > 0 && (reserve_rows == nullptr || start == nullptr || copies == nullptr || workspace == nullptr)) ||
      (layers > 0 && (k_cache == nullptr || v_cache == nullptr)))
    return CQ_ERR_ARG;
  if (!aligned(block_table, 4) || !aligned(seq_lens, 4) || !aligned(ref_counts, 4) || !aligned(free_rows, 4) ||
      !aligned(src_rows, 4) || !aligned(dst_rows, 4) || !aligned(reserve_rows, 4) || !aligned(counts, 4) ||
      !aligned(start, 4) || !aligned(copies, 8) || !aligned(workspace, 4) || !aligned(k_cache, 16) ||
      !aligned(v_cache, 16))
    return CQ_ERR_ALIGN;
  if (int dv = check_device()) return dv;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cq::PagesArgs a{block_table, table_stride, seq_lens, ref_counts, free_rows, src_rows, dst_rows, reserve_rows,
                        counts, start, copies, static_cast<int*>(workspace), static_cast<int>(table_rows),
                        static_cast<int>(table_width), static_cast<int>(num_pages), static_cast<int>(page_size),
                        static_cast<int>(n_free), static_cast<int>(n_fork), static_cast<int>(n_reserve),
                        static_cast<int>(count)};
  if (cudaError_t e = cq::launch_pages_branch(a, st)) return cuda_status(e);
  if (n_reserve == 0 || layers == 0) return CQ_OK;
  const cq::PagesCopyArgs c{copies, k_cache, v_cache, layer_bytes, page_bytes, static_cast<int>(n_reserve),
                            static_cast<int>(layers), static_cast<int>(num_pages)};
  return cuda_status(cq::launch_pages_copy(c, st));
}

int cq_pages_compact(const int32_t* block_table, int64_t table_rows, int64_t table_width, int64_t table_stride,
                     int32_t* table_out, int64_t out_stride, const int32_t* ref_counts, int32_t* refs_out,
                     int64_t num_pages, int32_t* moves, void* k_cache, void* v_cache, int64_t layers,
                     int64_t layer_bytes, int64_t page_bytes, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_tables(table_rows, table_width, table_stride, num_pages, 16)) return rc;
  if (out_stride < table_width || layers < 0 || layers > 65535) return CQ_ERR_SHAPE;
  if (layers > 0 && (page_bytes < 16 || page_bytes % 16 != 0 || layer_bytes % 16 != 0)) return CQ_ERR_SHAPE;
  if (workspace_bytes < 4 * num_pages) return CQ_ERR_SHAPE;
  if (num_pages / 8 > kMaxSharedBits) return CQ_ERR_CAPACITY;
  if (ref_counts == nullptr || refs_out == nullptr || workspace == nullptr || (num_pages > 1 && moves == nullptr) ||
      (table_rows * table_width > 0 && (block_table == nullptr || table_out == nullptr)) ||
      (layers > 0 && (k_cache == nullptr || v_cache == nullptr)))
    return CQ_ERR_ARG;
  if (!aligned(block_table, 4) || !aligned(table_out, 4) || !aligned(ref_counts, 4) || !aligned(refs_out, 4) ||
      !aligned(moves, 8) || !aligned(workspace, 4) || !aligned(k_cache, 16) || !aligned(v_cache, 16))
    return CQ_ERR_ALIGN;
  if (int dv = check_device()) return dv;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cq::CompactArgs a{block_table, table_out, table_stride, out_stride, ref_counts, refs_out, moves,
                          static_cast<int*>(workspace), static_cast<int>(table_rows), static_cast<int>(table_width),
                          static_cast<int>(num_pages)};
  if (cudaError_t e = cq::launch_pages_compact(a, st)) return cuda_status(e);
  if (layers == 0) return CQ_OK;
  const cq::PagesCopyArgs c{moves, k_cache, v_cache, layer_bytes, page_bytes, static_cast<int>(num_pages / 2),
                            static_cast<int>(layers), static_cast<int>(num_pages)};
  return cuda_status(cq::launch_pages_copy(c, st));
}

int cq_kv_append(const void* k_new, int64_t k_layer_stride, int64_t k_token_stride, int64_t k_head_stride,
                 const void* v_new, int64_t v_layer_stride, int64_t v_token_stride, int64_t v_head_stride, int dtype,
                 int64_t layers, int64_t tokens, int64_t kv_heads, int64_t head_dim, void* k_cache, void* v_cache,
                 int cache_dtype, int64_t num_pages, int64_t page_size, int64_t layer_stride, int64_t page_stride,
                 int64_t head_stride, int64_t token_stride, const int32_t* block_table, int64_t table_rows,
                 int64_t table_width, int64_t table_stride, const int32_t* rows, const int32_t* positions,
                 const float* k_scale, const float* v_scale, void* stream) {
  if (!valid16(dtype) || (cache_dtype != dtype && cache_dtype != CQ_DT_FP8_E4M3)) return CQ_ERR_ARG;
  if (int rc = check_tables(table_rows, table_width, table_stride, num_pages, page_size)) return rc;
  if (!fits_int(tokens) || layers < 0 || layers > 65535 || kv_heads < 1 || kv_heads > 4096 || head_dim < 8 ||
      head_dim % 8 != 0 || head_dim > 1024)
    return CQ_ERR_SHAPE;
  if (tokens == 0 || layers == 0) return CQ_OK;
  if (k_new == nullptr || v_new == nullptr || k_cache == nullptr || v_cache == nullptr || rows == nullptr ||
      positions == nullptr || (block_table == nullptr && table_width > 0))
    return CQ_ERR_ARG;
  if (!aligned(k_new, 16) || !aligned(v_new, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16) ||
      k_layer_stride % 8 != 0 || k_token_stride % 8 != 0 || k_head_stride % 8 != 0 || v_layer_stride % 8 != 0 ||
      v_token_stride % 8 != 0 || v_head_stride % 8 != 0 || layer_stride % 8 != 0 || page_stride % 8 != 0 ||
      head_stride % 8 != 0 || token_stride % 8 != 0 || !aligned(block_table, 4) || !aligned(rows, 4) ||
      !aligned(positions, 4) || !aligned(k_scale, 4) || !aligned(v_scale, 4))
    return CQ_ERR_ALIGN;
  if (int dv = check_device()) return dv;
  const cq::AppendArgs a{k_new, v_new, k_layer_stride, k_token_stride, k_head_stride, v_layer_stride, v_token_stride,
                         v_head_stride, k_cache, v_cache, layer_stride, page_stride, head_stride, token_stride,
                         block_table, table_stride, rows, positions, k_scale, v_scale, static_cast<int>(layers),
                         static_cast<int>(tokens), static_cast<int>(kv_heads), static_cast<int>(head_dim),
                         static_cast<int>(num_pages), static_cast<int>(page_size), static_cast<int>(table_rows),
                         static_cast<int>(table_width), dtype, cache_dtype};
  return cuda_status(cq::launch_kv_append(a, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
