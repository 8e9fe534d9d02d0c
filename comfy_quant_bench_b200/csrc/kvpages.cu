// Bookkeeping and data movement of a paged key-value cache.
//
// State, all on the device so that no step waits for the host: block tables int32 [rows, width] (-1: no page), tokens
// per row int32 [rows], and the number of table rows that hold each page, int32 [pages] (0: free).  Pages are always
// taken lowest index first and rows served in the order given, so every result is a function of the state alone.
//
// pages_branch_kernel: free a list of rows, fork rows (destination rows take the source rows' pages and one more
// reference to each), then make room for new tokens: a row whose last page is partly filled and held by another row
// too gets its own copy of it (copy on write), and pages are taken for what does not fit.  One CTA: each phase is
// short and needs the one before it.  All lists of rows are checked before any phase begins, so a wrong list changes
// nothing; whether the free pages suffice is known when the rows are freed and forked, and then only the reservation is
// refused.
#include "decode_common.cuh"

namespace cq {

namespace pages {
constexpr int kThreads = 1024;
constexpr int kMaxShared = 200 * 1024;   // bytes of the row and page bitmaps
constexpr int kPlainShared = 47 * 1024;  // what a launch may ask for as it is: 48 KB less the kernels' static arrays
constexpr int kSiteFree = 101, kSiteFork = 102, kSiteReserve = 103;   // device status sites
}  // namespace pages

// inclusive block sum of one int per thread; *total receives the sum over the block
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();                       // the previous scan's warp_sums are read
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  int s = warp_sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  *total = __shfl_sync(0xffffffffu, s, 31);
  const int before = __shfl_sync(0xffffffffu, s, (warp + 31) & 31);
  return v + (warp > 0 ? before : 0);
}

// marks `rows` in the bitmap `seen`; whether each is in range and listed once (the same answer to all threads)
__device__ bool mark_rows(const int* rows, int n, int table_rows, uint32_t* seen) {
  for (int i = threadIdx.x; i < (table_rows + 31) / 32; i += blockDim.x) seen[i] = 0;
  __syncthreads();
  int bad = 0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int r = rows[i];
    if (r < 0 || r >= table_rows || (atomicOr(&seen[r >> 5], 1u << (r & 31)) >> (r & 31) & 1u)) bad = 1;
  }
  return !__syncthreads_or(bad);
}
__device__ __forceinline__ bool marked(const uint32_t* seen, int r) { return seen[r >> 5] >> (r & 31) & 1u; }

__device__ __forceinline__ int held_pages(int len, int page_size, int width) {
  if (len <= 0) return 0;
  const int n = (len - 1) / page_size + 1;
  return n < width ? n : width;
}

// bitmap of the free pages (bit set: no row holds it), one word per 32 pages
__device__ void free_bitmap(const int* refs, int num_pages, uint32_t* bits) {
  const int lane = threadIdx.x & 31;
  const int padded = (num_pages + 31) & ~31;
  for (int p = threadIdx.x; p < padded; p += blockDim.x) {
    const bool f = p < num_pages && __ldcg(refs + p) <= 0;
    const uint32_t w = __ballot_sync(0xffffffffu, f);
    if (lane == 0) bits[p >> 5] = w;
  }
  __syncthreads();
}

// Lanes that work on one table row: each row is a chain of dependent loads, so with short rows many of them at a time.
// 128 rows of 56 pages, the whole branching kernel: 23 us with a warp per row, 15 us with eight lanes.
__device__ __forceinline__ int lanes_of_row(int width) { return width >= 512 ? 32 : 8; }

__global__ void __launch_bounds__(pages::kThreads) pages_branch_kernel(const PagesArgs a) {
  extern __shared__ uint32_t dyn[];
  __shared__ int warp_sums[32];
  __shared__ int over;
  uint32_t* seen = dyn;                                  // [table_rows] bits
  uint32_t* bits = dyn + (a.table_rows + 31) / 32;       // [num_pages] bits
  const int tid = threadIdx.x;
  const int per = lanes_of_row(a.table_width), sub = tid & (per - 1), group = tid / per, groups = blockDim.x / per;
  const uint32_t mates = per == 32 ? 0xffffffffu : 0xffu << (tid & 24);   // the lanes of this thread's row
  grid_dep_launch();                                     // the copies may be set up while this runs
  if (tid == 0) over = 0;

  // the lists: each names rows of the table once, a fork's source is no destination, and a destination is empty or freed
  // here; `site` has the same value in all threads
  int site = 0;
  if (a.n_free > 0 && !mark_rows(a.free_rows, a.n_free, a.table_rows, seen)) site = pages::kSiteFree;
  if (site == 0 && a.n_fork > 0) {
    const bool same = a.dst == a.free_rows && a.n_fork == a.n_free;      // `seen` has the destinations already
    int bad = 0;
    for (int i = tid; i < a.n_fork; i += blockDim.x) {
      const int s = a.src[i], d = a.dst[i];
      if (d < 0 || d >= a.table_rows || !((a.n_free > 0 && marked(seen, d)) || a.lens[d] == 0)) bad = 1;
      if (s < 0 || s >= a.table_rows || (same && marked(seen, s))) bad = 1;
    }
    if (__syncthreads_or(bad) || (!same && !mark_rows(a.dst, a.n_fork, a.table_rows, seen))) site = pages::kSiteFork;
    else if (!same) {
      for (int i = tid; i < a.n_fork; i += blockDim.x)
        if (marked(seen, a.src[i])) bad = 1;
      if (__syncthreads_or(bad)) site = pages::kSiteFork;
    }
  }
  if (site == 0 && a.n_res > 0 && (a.res_rows != a.dst || a.n_res != a.n_fork) &&
      !mark_rows(a.res_rows, a.n_res, a.table_rows, seen))
    site = pages::kSiteReserve;

  if (site == 0 && a.n_free > 0) {
    for (int i = group; i < a.n_free; i += groups) {
      const int r = a.free_rows[i];
      int* row = a.table + r * a.table_stride;
      const int held = held_pages(a.lens[r], a.page_size, a.table_width);
      __syncwarp(mates);                                  // every lane has read the row's length
#pragma unroll 4
      for (int j = sub; j < held; j += per) {
        const int p = row[j];
        if (p >= 0 && p < a.num_pages) atomicSub(&a.refs[p], 1);
        row[j] = -1;
      }
      if (sub == 0) a.lens[r] = 0;
    }
    __syncthreads();
  }
  if (site == 0 && a.n_fork > 0) {
    for (int i = group; i < a.n_fork; i += groups) {
      const int s = a.src[i], d = a.dst[i];
      const int len = a.lens[s], held = held_pages(len, a.page_size, a.table_width);
#pragma unroll 4
      for (int j = sub; j < held; j += per) {
        const int p = a.table[s * a.table_stride + j];
        a.table[d * a.table_stride + j] = p;
        if (p >= 0 && p < a.num_pages) atomicAdd(&a.refs[p], 1);
      }
      if (sub == 0) a.lens[d] = len;
    }
    __syncthreads();
  }
  if (a.n_res == 0) {
    if (site != 0 && tid == 0) record_status(CQ_ERR_ARG, site);
    return;
  }
  int code = CQ_OK;
  if (site != 0) code = CQ_ERR_ARG;
  else site = pages::kSiteReserve;
  int total = 0;
  if (code == CQ_OK) {
    // pages that each row needs, and where its share of the free pages begins
    for (int i0 = 0; i0 < a.n_res; i0 += blockDim.x) {
      const int i = i0 + tid;
      int need = 0;
      if (i < a.n_res) {
        const int r = a.res_rows[i];
        const int len = max(__ldcg(a.lens + r), 0), cnt = a.counts != nullptr ? a.counts[i] : a.count;
        const int64_t top = static_cast<int64_t>(len) + cnt;
        if (cnt < 0 || top > static_cast<int64_t>(a.table_width) * a.page_size) over = 1;
        else if (cnt > 0) {
          need = static_cast<int>((top + a.page_size - 1) / a.page_size) - (len + a.page_size - 1) / a.page_size;
          if (len % a.page_size != 0) {
            const int p = __ldcg(a.table + r * a.table_stride + len / a.page_size);
            if (p < 0 || p >= a.num_pages) over = 1;
            else if (__ldcg(a.refs + p) > 1) need = (need + 1) | (1 << 30);       // bit 30: copy on write
          }
        }
      }
      int sum;
      const int own = need & ~(1 << 30), incl = block_scan(own, warp_sums, &sum);
      if (i < a.n_res) { a.ws[2 * i] = need; a.ws[2 * i + 1] = total + incl - own; }
      total = min(total + sum, a.num_pages + 1);            // at most 1024 x width per step: no overflow
    }
    // the free pages in order; entry k of the list is the k-th lowest
    free_bitmap(a.refs, a.num_pages, bits);
    const int words = (a.num_pages + 31) / 32, each = (words + blockDim.x - 1) / blockDim.x;
    int mine = 0, frees;
    for (int w = tid * each; w < min(words, (tid + 1) * each); ++w) mine += __popc(bits[w]);
    int rank = block_scan(mine, warp_sums, &frees) - mine;
    if (over || frees < total) code = CQ_ERR_CAPACITY;
    else {
      int* list = a.ws + 2 * a.n_res;
      for (int w = tid * each; w < min(words, (tid + 1) * each) && rank < total; ++w)
        for (uint32_t m = bits[w]; m != 0 && rank < total; m &= m - 1) list[rank++] = 32 * w + __ffs(m) - 1;
    }
    __syncthreads();
  }
  if (code != CQ_OK) {
    for (int i = tid; i < a.n_res; i += blockDim.x) {
      a.start[i] = -1;
      a.copies[2 * i] = -1;
      a.copies[2 * i + 1] = -1;
    }
    if (tid == 0) record_status(code, site);
    return;
  }
  const int* list = a.ws + 2 * a.n_res;
  for (int i = group; i < a.n_res; i += groups) {
    const int r = a.res_rows[i], need = a.ws[2 * i], first = a.ws[2 * i + 1], len = max(__ldcg(a.lens + r), 0);
    const bool cow = need >> 30 & 1;
    const int own = need & ~(1 << 30), at = (len + a.page_size - 1) / a.page_size - (cow ? 1 : 0);
    int* row = a.table + r * a.table_stride;
    const int old = cow ? __ldcg(row + at) : -1;
    __syncwarp(mates);                                // every lane has read the row's length
    for (int j = sub; j < own; j += per) {
      const int p = list[first + j];
      row[at + j] = p;
      a.refs[p] = 1;
    }
    if (sub == 0) {
      a.start[i] = len;
      a.copies[2 * i] = old;
      a.copies[2 * i + 1] = cow ? list[first] : -1;
      a.lens[r] = len + (a.counts != nullptr ? a.counts[i] : a.count);
      if (cow) atomicSub(&a.refs[old], 1);
    }
  }
}

int64_t pages_branch_shared(int table_rows, int num_pages) {
  return 4 * ((static_cast<int64_t>(table_rows) + 31) / 32 + (static_cast<int64_t>(num_pages) + 31) / 32);
}

cudaError_t launch_pages_branch(const PagesArgs& a, cudaStream_t st) {
  const int64_t smem = pages_branch_shared(a.table_rows, a.num_pages);
  if (smem > pages::kPlainShared) {
    static unsigned long long devices = 0;
    const cudaError_t e = allow_shared(pages_branch_kernel, pages::kMaxShared, devices);
    if (e != cudaSuccess) return e;
  }
  pages_branch_kernel<<<1, pages::kThreads, smem, st>>>(a);
  return cudaGetLastError();
}

// pages_copy_kernel: page moves[i][0] -> page moves[i][1] in every layer of the key and the value cache; a negative
// entry moves nothing.  No destination is a source, so the order does not matter.  A CTA per page, layer and cache: bound by
// HBM (moving 0.69 GB takes 224 us, 6.2 TB/s counting both ways, and few pages the launch).
__global__ void __launch_bounds__(256) pages_copy_kernel(const PagesCopyArgs a) {
  grid_dep_launch();
  grid_dep_wait();                                        // the list is written
  const int2 mv = reinterpret_cast<const int2*>(a.moves)[blockIdx.x];
  if (mv.x < 0 || mv.x >= a.num_pages || mv.y < 0 || mv.y >= a.num_pages) return;
  const int64_t layer = blockIdx.y * a.layer_bytes;
  char* base = static_cast<char*>(blockIdx.z == 0 ? a.k : a.v) + layer;
  const uint4* from = reinterpret_cast<const uint4*>(base + mv.x * a.page_bytes);
  uint4* to = reinterpret_cast<uint4*>(base + mv.y * a.page_bytes);
  for (int64_t i = threadIdx.x; i < a.page_bytes / 16; i += 256) to[i] = __ldcs(from + i);
}

cudaError_t launch_pages_copy(const PagesCopyArgs& a, cudaStream_t st) {
  if (a.n == 0) return cudaSuccess;
  return launch_early(pages_copy_kernel, dim3(a.n, a.layers, 2), 256, 0, st, a);
}

// pages_compact_kernel: with L live pages (held by some row), the live pages at L and above move, in order, to the
// free pages below L, in order.  map[p]: the new index of page p.  refs_out may be refs.
__global__ void __launch_bounds__(pages::kThreads) pages_compact_kernel(const CompactArgs a, const int remap) {
  extern __shared__ uint32_t bits[];
  __shared__ int warp_sums[32];
  const int tid = threadIdx.x;
  grid_dep_launch();
  free_bitmap(a.refs, a.num_pages, bits);
  const int words = (a.num_pages + 31) / 32, each = (words + blockDim.x - 1) / blockDim.x;
  const int w0 = min(words, tid * each), w1 = min(words, (tid + 1) * each);
  auto live_word = [&](int w) {
    const int left = a.num_pages - 32 * w;
    return ~bits[w] & (left >= 32 ? 0xffffffffu : (1u << left) - 1u);
  };
  int mine = 0, live, holes_total, movers_total;
  for (int w = w0; w < w1; ++w) mine += __popc(live_word(w));
  block_scan(mine, warp_sums, &live);
  auto below = [&](int w) { return 32 * w >= live ? 0u : live - 32 * w >= 32 ? 0xffffffffu : (1u << (live - 32 * w)) - 1u; };
  int nh = 0, nm = 0;
  for (int w = w0; w < w1; ++w) {
    nh += __popc(bits[w] & below(w));
    nm += __popc(live_word(w) & ~below(w));
  }
  int h = block_scan(nh, warp_sums, &holes_total) - nh;
  int m = block_scan(nm, warp_sums, &movers_total) - nm;
  for (int w = w0; w < w1; ++w) {
    for (uint32_t x = bits[w] & below(w); x != 0; x &= x - 1) a.moves[2 * h++ + 1] = 32 * w + __ffs(x) - 1;
    for (uint32_t x = live_word(w) & ~below(w); x != 0; x &= x - 1) a.moves[2 * m++] = 32 * w + __ffs(x) - 1;
  }
  for (int k = movers_total + tid; k < a.num_pages / 2; k += blockDim.x) {
    a.moves[2 * k] = -1;
    a.moves[2 * k + 1] = -1;
  }
  for (int p = tid; p < a.num_pages; p += blockDim.x) {
    a.map[p] = p;
    if (p < live && !(bits[p >> 5] >> (p & 31) & 1u)) a.refs_out[p] = a.refs[p];
  }
  __syncthreads();
  for (int k = tid; k < movers_total; k += blockDim.x) {
    const int from = a.moves[2 * k], to = a.moves[2 * k + 1];
    a.map[from] = to;
    a.refs_out[to] = a.refs[from];
  }
  __syncthreads();
  for (int p = live + tid; p < a.num_pages; p += blockDim.x) a.refs_out[p] = 0;
  if (remap) {
    for (int i = tid; i < a.table_rows * a.table_width; i += blockDim.x) {
      const int r = i / a.table_width, j = i - r * a.table_width;
      const int p = a.table[r * a.table_stride + j];
      a.table_out[r * a.out_stride + j] = p >= 0 && p < a.num_pages ? a.map[p] : p;
    }
  }
}

// table entries to the pages' new indexes; table_out may be table
__global__ void __launch_bounds__(256) pages_remap_kernel(const CompactArgs a) {
  const int64_t n = static_cast<int64_t>(a.table_rows) * a.table_width;
  grid_dep_launch();
  grid_dep_wait();                                        // the map is written
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int64_t r = i / a.table_width, j = i - r * a.table_width;
    const int p = a.table[r * a.table_stride + j];
    a.table_out[r * a.out_stride + j] = p >= 0 && p < a.num_pages ? a.map[p] : p;
  }
}

cudaError_t launch_pages_compact(const CompactArgs& a, cudaStream_t st) {
  const int smem = (a.num_pages + 31) / 32 * 4;
  if (smem > pages::kPlainShared) {
    static unsigned long long devices = 0;
    const cudaError_t e = allow_shared(pages_compact_kernel, pages::kMaxShared, devices);
    if (e != cudaSuccess) return e;
  }
  // a table of a few thousand entries is remapped by the planning CTA itself: one launch (3 us) less
  const int64_t n = static_cast<int64_t>(a.table_rows) * a.table_width;
  const bool small = n <= 8 * pages::kThreads;
  pages_compact_kernel<<<1, pages::kThreads, smem, st>>>(a, small ? 1 : 0);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || small) return e;
  const int64_t ctas = (n + 255) / 256;
  return launch_early(pages_remap_kernel, dim3(static_cast<unsigned>(ctas < 1184 ? ctas : 1184)), 256, 0, st, a);
}

// kv_append_kernel: new keys and values [layers, T, Hkv, D] into their rows' pages.  A token whose row, position or
// page is out of range is skipped (a refused reservation gives positions of -1).  An 8-bit cache holds x / scale,
// rounded to the nearest even and kept inside the format's finite range (NaN stays NaN).
// A thread moves eight elements (16 bytes in, 16 or 8 out): bound by launch and latency (128 tokens in 32 layers, 8 heads
// of 128: 11.5 us; element by element it took 28).
__global__ void __launch_bounds__(256) kv_append_kernel(const AppendArgs a) {
  grid_dep_launch();
  const int64_t t = blockIdx.x, layer = blockIdx.y;
  const int per = a.Hkv * a.D / 8;                        // eights of a token's keys, and of its values
  grid_dep_wait();                                        // positions, tables and copied pages are written
  const int row = a.rows[t];
  const int pos = a.positions[t];
  if (row < 0 || row >= a.table_rows || pos < 0 || pos / a.page_size >= a.table_width) return;
  const int page = a.table[row * a.table_stride + pos / a.page_size];
  if (page < 0 || page >= a.num_pages) return;
  const int64_t base = layer * a.layer_stride + page * a.page_stride + (pos % a.page_size) * a.tok_stride;
  for (int i = threadIdx.x; i < 2 * per; i += blockDim.x) {
    const bool value = i >= per;
    const int e = 8 * (value ? i - per : i), h = e / a.D, d = e - h * a.D;
    const int64_t from = layer * (value ? a.vn_sl : a.kn_sl) + t * (value ? a.vn_st : a.kn_st) + h * (value ? a.vn_sh : a.kn_sh) + d;
    const int64_t at = base + h * a.head_stride + d;
    const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(value ? a.v_new : a.k_new) + from);
    void* cache = value ? a.v : a.k;
    if (a.cache_dtype != CQ_DT_FP8_E4M3) {
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(cache) + at) = raw;
      continue;
    }
    const float* scales = value ? a.v_scale : a.k_scale;
    const float scale = scales != nullptr ? scales[h] : 1.0f;
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t out[2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = a.dtype == CQ_DT_F16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[j]))
                                            : make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
      const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(f.x, scale), __fdiv_rn(f.y, scale)), __NV_SATFINITE, __NV_E4M3);
      out[j >> 1] = j & 1 ? out[j >> 1] | two << 16 : two;
    }
    *reinterpret_cast<uint2*>(static_cast<__nv_fp8_storage_t*>(cache) + at) = make_uint2(out[0], out[1]);
  }
}

cudaError_t launch_kv_append(const AppendArgs& a, cudaStream_t st) {
  if (a.T == 0 || a.layers == 0) return cudaSuccess;
  const int threads = (2 * a.Hkv * a.D / 8 + 31) / 32 * 32;
  return launch_early(kv_append_kernel, dim3(a.T, a.layers), threads < 256 ? threads : 256, 0, st, a);
}

}  // namespace cq
