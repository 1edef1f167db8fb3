// Decode attention over a cache of pages (include/tangq.h: tq_gqa_decode_paged): the attention of tq_gqa_decode (attention.cu) for one new
// token per sequence, where position j of a sequence is row j % page_rows of page table[j / page_rows], and the positions that a group
// of sequences shares are the first member's.
#include <cuda_bf16.h>

#include <cfloat>

#include "attn_mma.cuh"
#include "pages.h"

namespace tq {

constexpr int kPaDim = 128;

struct PagedParams {
  const __nv_bfloat16 *q, *k, *v;      // q [batch][n_heads][128]; pages [n_pages][page_rows][n_kv][128]
  const int *tables, *lens, *seqs;     // seqs null: sequence b of the batch is sequence b of the pool
  const int *group_starts, *shared;    // null: nothing is shared
  int batch, n_groups, max_shared, max_len;
  int n_pages, page_shift, n_seqs, table_ld;
  int n_heads, n_kv, group;            // group: query heads of a KV head
  float scale_log2;
  void* out;
  int out_f32;
  int* err;
};

// What a sequence of the batch attends: its length, its table, and the table of the positions below `shared`.
struct PagedSeq {
  int len, shared;
  const int *table, *first;
};
__device__ __forceinline__ int paged_row_of(const PagedParams& p, int b) {
  const int s = p.seqs ? p.seqs[b] : b;
  return s >= 0 && s < p.n_seqs ? s : -1;
}
__device__ __forceinline__ PagedSeq paged_seq(const PagedParams& p, int b) {
  PagedSeq a{0, 0, p.tables, p.tables};
  const int s = paged_row_of(p, b);
  if (s < 0) {
    atomicCAS(p.err, 0, (int)DERR_PAGE_LIST);
    return a;
  }
  a.len = min(max(p.lens[s], 0), p.max_len);
  a.table = a.first = p.tables + (size_t)s * p.table_ld;
  if (p.group_starts) {
    int lo = 0, hi = p.n_groups;       // the last group that starts at b or before
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.group_starts[mid] <= b) lo = mid;
      else hi = mid;
    }
    const int f = paged_row_of(p, min(max(p.group_starts[lo], 0), b));
    a.shared = f < 0 ? 0 : min(max(p.shared[lo], 0), p.max_shared);
    if (f >= 0) a.first = p.tables + (size_t)f * p.table_ld;
  }
  return a;
}

// A warp per query head and sequence, a position after the other: lane i has four of the 128 values.
__global__ void __launch_bounds__(128) paged_decode_kernel(const PagedParams p) {
  __shared__ float m_s[4], l_s[4], o_s[4][kPaDim];
  pdl_wait();
  pdl_launch_dependents();
  const int head = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kvh = head / p.group;
  const PagedSeq a = paged_seq(p, b);
  const size_t row = (size_t)p.n_kv * kPaDim, at = ((size_t)b * p.n_heads + head) * kPaDim;
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -FLT_MAX, l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = __bfloat162float(p.q[at + 4 * lane + i]);
  for (int j = warp; j < a.len; j += 4) {
    const int page = (j < a.shared ? a.first : a.table)[j >> p.page_shift];
    if (page < 0 || page >= p.n_pages) {
      atomicCAS(p.err, 0, (int)DERR_POSITION);
      continue;
    }
    const size_t r = ((((size_t)page << p.page_shift) + (j & ((1 << p.page_shift) - 1))) * row) + (size_t)kvh * kPaDim + 4 * lane;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) s = fmaf(q[i], __bfloat162float(p.k[r + i]), s);
    s = warp_sum(s) * p.scale_log2;
    const float mn = fmaxf(m, s), f = exp2f(m - mn), w = exp2f(s - mn);
    m = mn;
    l = l * f + w;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] * f + w * __bfloat162float(p.v[r + i]);
  }
  if (lane == 0) {
    m_s[warp] = m;
    l_s[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) o_s[warp][4 * lane + i] = o[i];
  __syncthreads();
  const int d = threadIdx.x;
  float M = -FLT_MAX, L = 0.f, O = 0.f;
  for (int w = 0; w < 4; ++w) M = fmaxf(M, m_s[w]);
  for (int w = 0; w < 4; ++w) {
    const float f = exp2f(m_s[w] - M);
    L += l_s[w] * f;
    O += o_s[w][d] * f;
  }
  const float y = L > 0.f ? O / L : 0.f;
  if (p.out_f32) static_cast<float*>(p.out)[at + d] = y;
  else static_cast<__nv_bfloat16*>(p.out)[at + d] = __float2bfloat16_rn(y);
}

}  // namespace tq

using namespace tq;

extern "C" int tq_gqa_decode_paged(tq_ctx* ctx, const void* q_dev, const void* k_pages_dev, const void* v_pages_dev, const tq_pages* pages,
                                   const int* seqs_dev, size_t batch, const int* group_starts_dev, const int* shared_dev, size_t n_groups,
                                   size_t max_shared, size_t n_heads, size_t n_kv_heads, size_t head_dim, size_t max_len, void* out_dev,
                                   int out_dtype) {
  if (int st = bind(ctx)) return st;
  if (batch == 0) return TQ_OK;
  TQ_REQUIRE(ctx, q_dev && k_pages_dev && v_pages_dev && pages && out_dev, "tq_gqa_decode_paged: null pointer");
  TQ_REQUIRE(ctx, pages->ctx->device == ctx->device, "tq_gqa_decode_paged: the pool belongs to another device");
  TQ_REQUIRE(ctx, head_dim == (size_t)kPaDim, "tq_gqa_decode_paged: head_dim must be %d", kPaDim);
  TQ_REQUIRE(ctx, n_kv_heads > 0 && n_heads % n_kv_heads == 0 && n_heads / n_kv_heads >= 1 && n_heads / n_kv_heads <= 8 && n_heads <= 65535,
             "tq_gqa_decode_paged: n_heads/n_kv_heads must be 1..8");
  TQ_REQUIRE(ctx, out_dtype == TQ_BF16 || out_dtype == TQ_F32, "tq_gqa_decode_paged: out must be bf16 or f32");
  TQ_REQUIRE(ctx, batch <= 65535 && (seqs_dev || batch <= (size_t)pages->n_seqs), "tq_gqa_decode_paged: more sequences than the pool has");
  const size_t most = (size_t)pages->table_ld * pages->page_rows;
  TQ_REQUIRE(ctx, max_len > 0 && max_len <= 0x7fffffff - 1024, "tq_gqa_decode_paged: max_len must bound the sequence lengths");
  TQ_REQUIRE(ctx, (group_starts_dev != nullptr) == (shared_dev != nullptr) && (group_starts_dev == nullptr || (n_groups > 0 && n_groups <= batch)),
             "tq_gqa_decode_paged: groups have starts and shared lengths, at most one per sequence");
  TQ_REQUIRE(ctx, (((uintptr_t)q_dev | (uintptr_t)k_pages_dev | (uintptr_t)v_pages_dev | (uintptr_t)out_dev) & 15) == 0,
             "tq_gqa_decode_paged: arrays must be 16-byte aligned");
  PagedParams p;
  p.q = static_cast<const __nv_bfloat16*>(q_dev);
  p.k = static_cast<const __nv_bfloat16*>(k_pages_dev);
  p.v = static_cast<const __nv_bfloat16*>(v_pages_dev);
  p.tables = pages->tables;
  p.lens = pages->lens;
  p.seqs = seqs_dev;
  p.group_starts = group_starts_dev;
  p.shared = shared_dev;
  p.batch = (int)batch;
  p.n_groups = (int)n_groups;
  p.max_len = (int)(max_len < most ? max_len : most);
  p.max_shared = (int)(max_shared < (size_t)p.max_len ? max_shared : (size_t)p.max_len);
  p.n_pages = pages->n_pages;
  p.page_shift = 31 - __builtin_clz((unsigned)pages->page_rows);
  p.n_seqs = pages->n_seqs;
  p.table_ld = pages->table_ld;
  p.n_heads = (int)n_heads;
  p.n_kv = (int)n_kv_heads;
  p.group = (int)(n_heads / n_kv_heads);
  p.scale_log2 = 1.44269504088896340736f / sqrtf((float)head_dim);
  p.out = out_dev;
  p.out_f32 = out_dtype == TQ_F32;
  p.err = ctx->dev_err;
  TQ_CUDA(ctx, launch_k(ctx, paged_decode_kernel, dim3((unsigned)n_heads, (unsigned)batch), dim3(128), 0, p));
  return TQ_OK;
}
