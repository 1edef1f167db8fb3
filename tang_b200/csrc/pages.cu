// Pages of a KV cache that several sequences hold at once (include/tangq.h, tq_pages_*): forked samples of one prompt share its pages,
// and only a page that a sequence is about to write, and that another one holds too, is copied.  No reference counterpart; the slots of
// crates/tang-infer/src/kv_cache.rs:12-160 hold one sequence each.
//
// All bookkeeping is on the device, in one CTA per call, so that a generation loop can be recorded in a graph: the host never learns
// which page went where.  A call is all or nothing: every thread checks one sequence of the list, and unless all are fine nothing is
// written and the status word says why.  Pages are handed out lowest number first, in the order of the list, so that the same calls give
// the same tables.  What is copied is listed by that CTA and moved by a second kernel over all SMs.
// What bounds it: the copied bytes, where there are many (64 half pages in 32 arrays, 134 MB each way, 54 us with the calls before), else launches and one
// CTA's chain of loads: tq_pages_free 2.9 us for 64 sequences, tq_pages_fork 5.9 (0.6 and 1.5 of these for the look at all table
// entries before any is changed), tq_pages_extend without a copy 6.2 (two kernels).
#include <new>

#include "common.cuh"
#include "pages.h"

namespace tq {

constexpr int kBookThreads = kPageCalls;
constexpr int kScanPages = 8;          // pages that a thread looks at per turn
constexpr int kCopyThreads = 256;
constexpr int kCopyChunk = kCopyThreads * 4 * 16;   // bytes that a CTA moves per turn

struct PagesParams {
  int *refs, *tables, *lens;
  int n_pages, page_rows, n_seqs, table_ld;
  int *n_copies, *from, *to, *rows, *list, *marks, *refused;
  int* err;
};

__device__ __forceinline__ int pages_of(int positions, int page_rows) { return (positions + page_rows - 1) / page_rows; }

// Sum of v over the lower threads of the CTA and, in *total, over all of them.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* warp_sums, T* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  T incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  __syncthreads();                     // (the sums of the call before have been read)
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  T base = 0, all = 0;
#pragma unroll 8
  for (int w = 0; w < kBookThreads / 32; ++w) {
    base += w < warp ? warp_sums[w] : 0;
    all += warp_sums[w];
  }
  *total = all;
  return base + incl - v;
}

// Appends to list[0 .. most) the lowest pages p >= from with (refs[p] == 0) == free, in order; how many pages of the pool qualify at least
// (it stops looking once `most` are found).
__device__ __forceinline__ int find_pages(const int* refs, int from, int end, bool free, int most, int* list, int* warp_sums) {
  int found = 0;
  for (int base = from; base < end && found < most; base += kBookThreads * kScanPages) {
    const int first = base + (int)threadIdx.x * kScanPages;
    unsigned hit = 0;
#pragma unroll
    for (int i = 0; i < kScanPages; ++i)
      if (first + i < end && (refs[first + i] == 0) == free) hit |= 1u << i;
    int total;
    int at = found + block_scan(__popc(hit), warp_sums, &total);
#pragma unroll
    for (int i = 0; i < kScanPages; ++i)
      if (hit >> i & 1u) {
        if (at < most) list[at] = first + i;
        ++at;
      }
    found += total;
  }
  return found;
}

// Whether tables name a page that does not exist (this library did not write them): of sequences seqs[i] the first pages_of(lens[i]) entries, a warp per
// sequence, and for the whole CTA.
__device__ __forceinline__ bool names_no_page(const PagesParams& p, const int* seqs, const int* lens, int n) {
  bool none = false;
  for (int i = threadIdx.x >> 5; i < n; i += kBookThreads / 32) {
    const int pages = pages_of(lens[i], p.page_rows);
    for (int j = threadIdx.x & 31; j < pages; j += 32) {
      const int page = p.tables[(size_t)seqs[i] * p.table_ld + j];
      none = none || page < 0 || page >= p.n_pages;
    }
  }
  return __syncthreads_or(none);
}

// One sequence per thread: valid, and in the list once.  (The mark is taken back by the threads that set it.)
__device__ __forceinline__ bool mark_once(const PagesParams& p, int s) {
  return s >= 0 && s < p.n_seqs && atomicExch(&p.marks[s], 1) == 0;
}

__device__ __forceinline__ bool sound(const PagesParams& p, int len) { return len >= 0 && len <= 0x7fffffff - p.page_rows && pages_of(len, p.page_rows) <= p.table_ld; }

__global__ void __launch_bounds__(kBookThreads) pages_extend_kernel(const PagesParams p, const int* seqs, const int* counts, int n) {
  __shared__ long long warp_needs[kBookThreads / 32];
  __shared__ int warp_sums[kBookThreads / 32], first_s[kBookThreads + 1], last_s[kBookThreads], seq_s[kBookThreads], at_s[kBookThreads];
  pdl_wait();
  pdl_launch_dependents();
  const int t = threadIdx.x, P = p.page_rows;
  int s = -1, c = 0, len = 0, last = -1, need = 0;
  bool bad = false, marked = false, cow = false;
  if (t == 0) *p.n_copies = 0;
  if (t < n) {
    s = seqs[t];
    c = counts ? counts[t] : 1;
    marked = mark_once(p, s);
    bad = !marked || c < 0;
    if (!bad) {
      len = p.lens[s];
      bad = !sound(p, len);
      if (!bad && c > 0 && len % P != 0) {
        last = p.tables[(size_t)s * p.table_ld + len / P];
        bad = last < 0 || last >= p.n_pages;
      }
    }
  }
  last_s[t] = bad ? -1 : last;
  bad = __syncthreads_or(bad);
  bool full = false;
  if (!bad && t < n) {
    if (last >= 0) {
      // earlier sequences of the list that hold the same page take a copy each: the last holder keeps it
      int before = 0;
      const int holders = p.refs[last];
      if (holders > 1)
        for (int u = 0; u < t; ++u) before += last_s[u] == last;
      cow = holders - before > 1;
    }
    full = c > 0x7fffffff - P - len || pages_of(len + c, P) > p.table_ld;
    if (!full) need = (cow ? 1 : 0) + pages_of(len + c, P) - pages_of(len, P);
  }
  if (marked) p.marks[s] = 0;
  full = __syncthreads_or(full);
  long long needs = 0;                 // (1024 sequences of 2^24 pages each are more than 32 bits)
  int n_copies = 0;
  const int first = (int)block_scan<long long>(need, warp_needs, &needs), copy_at = block_scan(cow ? 1 : 0, warp_sums, &n_copies);
  full = full || needs > p.n_pages;
  const int total = (int)needs;
  if (!bad && !full && total > 0) full = find_pages(p.refs, 0, p.n_pages, true, total, p.list, warp_sums) < total;
  if (bad || full) {
    if (t == 0) atomicCAS(p.err, 0, bad ? (int)DERR_PAGE_LIST : (int)DERR_PAGES);
    if (s >= 0 && s < p.n_seqs) p.refused[s] = 1;      // (the step that stands behind this call in a graph runs all the same)
    return;
  }
  first_s[t] = first;
  seq_s[t] = s;
  at_s[t] = pages_of(len, P) - (cow ? 1 : 0);
  __syncthreads();                     // (and the list is written)
  if (cow) {
    p.from[copy_at] = last;
    p.to[copy_at] = p.list[first];
    p.rows[copy_at] = len % P;
    atomicSub(&p.refs[last], 1);
  }
  if (t < n) {
    p.lens[s] = len + c;
    if (c > 0) p.refused[s] = 0;
  }
  if (t == 0) *p.n_copies = n_copies;
  for (int i = t; i < total; i += kBookThreads) {
    int lo = 0, hi = n;                // the last sequence whose first page is at most i
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first_s[mid] <= i) lo = mid;
      else hi = mid;
    }
    const int page = p.list[i];
    p.refs[page] = 1;
    p.tables[(size_t)seq_s[lo] * p.table_ld + at_s[lo] + (i - first_s[lo])] = page;
  }
}

__global__ void __launch_bounds__(kBookThreads) pages_fork_kernel(const PagesParams p, const int* src, const int* dst, const int* keep, int n) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ int src_s[kBookThreads], dst_s[kBookThreads], len_s[kBookThreads];
  const int t = threadIdx.x;
  int s = -1, d = -1, len = 0;
  bool bad = false, marked = false;
  if (t < n) {
    s = src[t];
    d = dst[t];
    marked = mark_once(p, d);
    bad = !marked || s < 0 || s >= p.n_seqs;
    if (!bad) {
      len = p.lens[s];
      bad = p.lens[d] != 0 || !sound(p, len);
      if (keep) {
        bad = bad || keep[t] < 0;
        len = min(len, keep[t]);
      }
    }
  }
  __syncthreads();
  if (t < n && !bad) bad = __ldcg(&p.marks[s]) != 0;     // a source that is a destination too
  src_s[t] = s;
  dst_s[t] = d;
  len_s[t] = len;
  bad = __syncthreads_or(bad);
  if (marked) p.marks[d] = 0;
  if (!bad) bad = names_no_page(p, src_s, len_s, n);
  for (int i = t >> 5; i < n && !bad; i += kBookThreads / 32) {      // a warp per pair
    const int pages = pages_of(len_s[i], p.page_rows);
    for (int j = t & 31; j < pages; j += 32) {
      const int page = p.tables[(size_t)src_s[i] * p.table_ld + j];
      atomicAdd(&p.refs[page], 1);
      p.tables[(size_t)dst_s[i] * p.table_ld + j] = page;
    }
  }
  if (bad) {
    if (t == 0) atomicCAS(p.err, 0, (int)DERR_PAGE_LIST);
  } else if (t < n) {
    p.lens[d] = len;
  }
}

__global__ void __launch_bounds__(kBookThreads) pages_free_kernel(const PagesParams p, const int* seqs, int n) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ int seq_s[kBookThreads], len_s[kBookThreads];
  const int t = threadIdx.x;
  int s = -1, len = 0;
  bool bad = false, marked = false;
  if (t < n) {
    s = seqs[t];
    marked = mark_once(p, s);
    bad = !marked;
    if (!bad) {
      len = p.lens[s];
      bad = !sound(p, len);
    }
  }
  seq_s[t] = s;
  len_s[t] = len;
  bad = __syncthreads_or(bad);
  if (marked) p.marks[s] = 0;
  if (!bad) bad = names_no_page(p, seq_s, len_s, n);
  for (int i = t >> 5; i < n && !bad; i += kBookThreads / 32) {
    const int pages = pages_of(len_s[i], p.page_rows);
    for (int j = t & 31; j < pages; j += 32) {
      int* at = &p.tables[(size_t)seq_s[i] * p.table_ld + j];
      const int page = *at;
      *at = -1;
      atomicSub(&p.refs[page], 1);
    }
  }
  if (bad) {
    if (t == 0) atomicCAS(p.err, 0, (int)DERR_PAGE_LIST);
  } else if (t < n) {
    p.lens[s] = 0;
  }
}

// With u pages in use, those numbered u and above move to the free ones below u, both in order.  `list` becomes where a page is found now.
__global__ void __launch_bounds__(kBookThreads) pages_compact_kernel(const PagesParams p, int* used_out) {
  __shared__ int warp_sums[kBookThreads / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int t = threadIdx.x;
  int mine = 0, used;
  for (int i = t; i < p.n_pages; i += kBookThreads) mine += p.refs[i] != 0;
  block_scan(mine, warp_sums, &used);
  const int moves = find_pages(p.refs, 0, used, true, p.n_pages, p.to, warp_sums);
  find_pages(p.refs, used, p.n_pages, false, moves, p.from, warp_sums);
  for (int i = t; i < p.n_pages; i += kBookThreads) p.list[i] = i;
  __syncthreads();
  for (int i = t; i < moves; i += kBookThreads) {
    const int to = p.to[i], from = p.from[i];
    p.list[from] = to;
    p.refs[to] = p.refs[from];
    p.refs[from] = 0;
  }
  if (t == 0) {
    *p.n_copies = moves;
    if (used_out) *used_out = used;
  }
}

struct CopyParams {
  void* const* arrays;
  int n_arrays;
  size_t row_bytes, page_bytes;
  const int *n_copies, *from, *to, *rows;              // rows null: whole pages
  const int *remap, *lens;                             // remap null: the tables stay
  int* tables;
  int n_seqs, table_ld, n_pages, page_rows;
};

// A CTA takes (copy, array, part of the page) in turn; a thread has four 16-byte loads in flight.
__global__ void __launch_bounds__(kCopyThreads) pages_copy_kernel(const CopyParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int n = *p.n_copies, t = threadIdx.x;
  if (n == 0) return;
  const size_t parts = (p.page_bytes + kCopyChunk - 1) / kCopyChunk, items = (size_t)n * p.n_arrays * parts;
  for (size_t i = blockIdx.x; i < items; i += gridDim.x) {
    const size_t pair = i / parts, part = i - pair * parts;
    const int c = (int)(pair / p.n_arrays), a = (int)(pair - (size_t)c * p.n_arrays);
    const size_t bytes = p.rows ? (size_t)p.rows[c] * p.row_bytes : p.page_bytes;
    char* base = static_cast<char*>(p.arrays[a]);
    const char* src = base + (size_t)p.from[c] * p.page_bytes;
    char* dst = base + (size_t)p.to[c] * p.page_bytes;
    uint4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const size_t at = part * kCopyChunk + (size_t)(k * kCopyThreads + t) * 16;
      if (at < bytes) v[k] = *reinterpret_cast<const uint4*>(src + at);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const size_t at = part * kCopyChunk + (size_t)(k * kCopyThreads + t) * 16;
      if (at < bytes) *reinterpret_cast<uint4*>(dst + at) = v[k];
    }
  }
  if (p.remap) {
    const size_t entries = (size_t)p.n_seqs * p.table_ld;
    for (size_t i = (size_t)blockIdx.x * kCopyThreads + t; i < entries; i += (size_t)gridDim.x * kCopyThreads) {
      const int s = (int)(i / p.table_ld), j = (int)(i - (size_t)s * p.table_ld);
      const int page = p.tables[i];
      if (j < pages_of(p.lens[s], p.page_rows) && page >= 0 && page < p.n_pages) p.tables[i] = p.remap[page];
    }
  }
}

static PagesParams params_of(const tq_pages* p) {
  PagesParams k;
  const size_t m = pages_max_copies(p);
  k.refs = p->refs;
  k.tables = p->tables;
  k.lens = p->lens;
  k.n_pages = p->n_pages;
  k.page_rows = p->page_rows;
  k.n_seqs = p->n_seqs;
  k.table_ld = p->table_ld;
  k.n_copies = p->ws;
  k.from = pages_copies(p);
  k.to = k.from + m;
  k.rows = k.to + m;
  k.list = pages_list(p);
  k.marks = pages_marks(p);
  k.refused = pages_refused(p);
  k.err = p->ctx->dev_err;
  return k;
}

static int launch_copies(tq_pages* p, const PagesParams& k, bool whole) {
  tq_ctx* ctx = p->ctx;
  CopyParams c;
  c.arrays = p->arrays;
  c.n_arrays = p->n_arrays;
  c.row_bytes = p->row_bytes;
  c.page_bytes = p->row_bytes * p->page_rows;
  c.n_copies = k.n_copies;
  c.from = k.from;
  c.to = k.to;
  c.rows = whole ? nullptr : k.rows;
  c.remap = whole ? k.list : nullptr;
  c.lens = k.lens;
  c.tables = k.tables;
  c.n_seqs = k.n_seqs;
  c.table_ld = k.table_ld;
  c.n_pages = k.n_pages;
  c.page_rows = k.page_rows;
  TQ_CUDA(ctx, launch_k(ctx, pages_copy_kernel, dim3((unsigned)ctx->sm_count * 8), dim3(kCopyThreads), 0, c));
  return TQ_OK;
}

static void release(tq_pages* p) {
  if (p->owns) {
    cudaFree(p->refs);
    cudaFree(p->tables);
    cudaFree(p->lens);
  }
  if (p->arrays) cudaFree(p->arrays);
  if (p->ws) cudaFree(p->ws);
  delete p;
}

}  // namespace tq

using namespace tq;

extern "C" {

int tq_pages_create(tq_ctx* ctx, size_t n_pages, size_t page_rows, size_t n_seqs, size_t table_ld, int* refs_dev, int* tables_dev, int* lens_dev,
                    tq_pages** out) {
  if (int st = bind(ctx)) return st;
  TQ_REQUIRE(ctx, out != nullptr, "tq_pages_create: null argument");
  *out = nullptr;
  TQ_REQUIRE(ctx, !ctx->capturing, "tq_pages_create: not during graph capture");
  TQ_REQUIRE(ctx, n_pages > 0 && n_pages <= (1u << 24) && n_seqs > 0 && n_seqs <= (1u << 20) && table_ld > 0 && table_ld <= (1u << 24),
             "tq_pages_create: 1 to 2^24 pages and table entries, 1 to 2^20 sequences");
  TQ_REQUIRE(ctx, page_rows >= 16 && page_rows <= 1024 && (page_rows & (page_rows - 1)) == 0,
             "tq_pages_create: a page has 16, 32, 64 .. 1024 positions");
  TQ_REQUIRE(ctx, (refs_dev != nullptr) == (tables_dev != nullptr) && (refs_dev != nullptr) == (lens_dev != nullptr),
             "tq_pages_create: the three arrays are all the caller's or all the library's");
  tq_pages* p = new (std::nothrow) tq_pages();
  if (!p) return fail(ctx, TQ_ENOMEM, "out of host memory");
  p->ctx = ctx;
  p->n_pages = (int)n_pages;
  p->page_rows = (int)page_rows;
  p->n_seqs = (int)n_seqs;
  p->table_ld = (int)table_ld;
  cudaError_t e = cudaMalloc(&p->ws, pages_ws_ints(p) * sizeof(int));
  if (e == cudaSuccess) e = cudaMemsetAsync(p->ws, 0, pages_ws_ints(p) * sizeof(int), ctx->stream);
  if (refs_dev) {
    p->refs = refs_dev;
    p->tables = tables_dev;
    p->lens = lens_dev;
  } else {
    p->owns = true;
    if (e == cudaSuccess) e = cudaMalloc(&p->refs, n_pages * sizeof(int));
    if (e == cudaSuccess) e = cudaMalloc(&p->tables, n_seqs * table_ld * sizeof(int));
    if (e == cudaSuccess) e = cudaMalloc(&p->lens, n_seqs * sizeof(int));
    if (e == cudaSuccess) e = cudaMemsetAsync(p->refs, 0, n_pages * sizeof(int), ctx->stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(p->tables, 0xFF, n_seqs * table_ld * sizeof(int), ctx->stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(p->lens, 0, n_seqs * sizeof(int), ctx->stream);
  }
  if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->stream);
  if (e != cudaSuccess) {
    release(p);
    cudaGetLastError();
    return fail(ctx, e == cudaErrorMemoryAllocation ? TQ_ENOMEM : TQ_ECUDA, "tq_pages_create: %s", cudaGetErrorString(e));
  }
  p->id = ++ctx->pool_ids;
  p->next = ctx->pools;
  ctx->pools = p;
  *out = p;
  return TQ_OK;
}

int tq_pages_destroy(tq_pages* p) {
  if (!p) return TQ_OK;
  if (tq_ctx* ctx = p->ctx) {          // (null: the context went first, and its stream was waited for)
    bind(ctx);
    cudaStreamSynchronize(ctx->stream);
    for (tq_pages** at = &ctx->pools; *at; at = &(*at)->next)
      if (*at == p) {
        *at = p->next;
        break;
      }
  }
  release(p);
  return TQ_OK;
}

int tq_pages_arrays(tq_pages* p, void* const* bases_host, size_t n_arrays, size_t row_bytes) {
  if (!p) return TQ_EINVAL;
  tq_ctx* ctx = p->ctx;
  if (int st = bind(ctx)) return st;
  TQ_REQUIRE(ctx, !ctx->capturing, "tq_pages_arrays: not during graph capture");
  TQ_REQUIRE(ctx, bases_host && n_arrays > 0 && n_arrays <= (1u << 16), "tq_pages_arrays: 1 to 65536 arrays");
  TQ_REQUIRE(ctx, row_bytes > 0 && row_bytes % 16 == 0 && row_bytes <= (1u << 24), "tq_pages_arrays: rows are a multiple of 16 bytes");
  for (size_t i = 0; i < n_arrays; ++i)
    TQ_REQUIRE(ctx, bases_host[i] && ((uintptr_t)bases_host[i] & 15) == 0, "tq_pages_arrays: array %zu is not 16-byte aligned", i);
  void** fresh = nullptr;
  TQ_CUDA(ctx, cudaMalloc(&fresh, n_arrays * sizeof(void*)));
  cudaError_t e = cudaMemcpyAsync(fresh, bases_host, n_arrays * sizeof(void*), cudaMemcpyHostToDevice, ctx->stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->stream);
  if (e != cudaSuccess) {
    cudaFree(fresh);
    return fail(ctx, TQ_ECUDA, "tq_pages_arrays: %s", cudaGetErrorString(e));
  }
  if (p->arrays) {
    cudaFree(p->arrays);
    p->id = ++ctx->pool_ids;
  }
  p->arrays = fresh;
  p->n_arrays = (int)n_arrays;
  p->row_bytes = row_bytes;
  return TQ_OK;
}

int tq_pages_data(const tq_pages* p, int** refs_dev, int** tables_dev, int** lens_dev) {
  if (!p) return TQ_EINVAL;
  if (refs_dev) *refs_dev = p->refs;
  if (tables_dev) *tables_dev = p->tables;
  if (lens_dev) *lens_dev = p->lens;
  return TQ_OK;
}

int tq_pages_extend(tq_pages* p, const int* seqs_dev, const int* counts_dev, size_t n) {
  if (!p) return TQ_EINVAL;
  tq_ctx* ctx = p->ctx;
  if (int st = bind(ctx)) return st;
  if (n == 0) return TQ_OK;
  TQ_REQUIRE(ctx, seqs_dev != nullptr, "tq_pages_extend: null list");
  TQ_REQUIRE(ctx, n <= (size_t)kPageCalls, "tq_pages_extend: at most %d sequences in a call", kPageCalls);
  TQ_REQUIRE(ctx, p->arrays != nullptr, "tq_pages_extend: a shared page cannot be copied before tq_pages_arrays names the caches");
  const PagesParams k = params_of(p);
  if (int st = pages_use(ctx, p)) return st;
  TQ_CUDA(ctx, launch_k(ctx, pages_extend_kernel, dim3(1), dim3(kBookThreads), 0, k, seqs_dev, counts_dev, (int)n));
  return launch_copies(p, k, false);
}

int tq_pages_fork(tq_pages* p, const int* src_dev, const int* dst_dev, const int* keep_dev, size_t n) {
  if (!p) return TQ_EINVAL;
  tq_ctx* ctx = p->ctx;
  if (int st = bind(ctx)) return st;
  if (n == 0) return TQ_OK;
  TQ_REQUIRE(ctx, src_dev && dst_dev, "tq_pages_fork: null list");
  TQ_REQUIRE(ctx, n <= (size_t)kPageCalls, "tq_pages_fork: at most %d sequences in a call", kPageCalls);
  if (int st = pages_use(ctx, p)) return st;
  TQ_CUDA(ctx, launch_k(ctx, pages_fork_kernel, dim3(1), dim3(kBookThreads), 0, params_of(p), src_dev, dst_dev, keep_dev, (int)n));
  return TQ_OK;
}

int tq_pages_free(tq_pages* p, const int* seqs_dev, size_t n) {
  if (!p) return TQ_EINVAL;
  tq_ctx* ctx = p->ctx;
  if (int st = bind(ctx)) return st;
  if (n == 0) return TQ_OK;
  TQ_REQUIRE(ctx, seqs_dev != nullptr, "tq_pages_free: null list");
  TQ_REQUIRE(ctx, n <= (size_t)kPageCalls, "tq_pages_free: at most %d sequences in a call", kPageCalls);
  if (int st = pages_use(ctx, p)) return st;
  TQ_CUDA(ctx, launch_k(ctx, pages_free_kernel, dim3(1), dim3(kBookThreads), 0, params_of(p), seqs_dev, (int)n));
  return TQ_OK;
}

int tq_pages_compact(tq_pages* p, int* used_out_dev) {
  if (!p) return TQ_EINVAL;
  tq_ctx* ctx = p->ctx;
  if (int st = bind(ctx)) return st;
  TQ_REQUIRE(ctx, p->arrays != nullptr, "tq_pages_compact: pages cannot be moved before tq_pages_arrays names the caches");
  const PagesParams k = params_of(p);
  if (int st = pages_use(ctx, p)) return st;
  TQ_CUDA(ctx, launch_k(ctx, pages_compact_kernel, dim3(1), dim3(kBookThreads), 0, k, used_out_dev));
  return launch_copies(p, k, true);
}

}  // extern "C"
