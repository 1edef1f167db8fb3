// Causal attention of several sequences' new positions, packed, over their pages (include/tangq.h: tq_gqa_prefill_paged).
#include <cfloat>

#include "attn_mma.cuh"
#include "page_rows.cuh"

namespace tq {

struct PackedPrefillParams {
  PackedSeqs s;
  const __nv_bfloat16* q;
  const uint8_t *k, *v;
  size_t row_bytes;
  int n_heads, n_kv, max_len;
  float scale_log2;
  __nv_bfloat16* out;
  int* err;
};

// Values 4 lane .. of a head of a cache row.
template <bool Q4>
__device__ __forceinline__ void row_values(const uint8_t* row, int n_kv, int head, int lane, float (&x)[4]) {
  if constexpr (Q4) {
    const uint32_t w = *reinterpret_cast<const uint16_t*>(row + head * kQ4HeadBytes + 2 * lane);
    const float s = bf16_bits_to_float(*reinterpret_cast<const uint16_t*>(row + n_kv * kQ4HeadBytes + 2 * (head * kQ4HeadScales + lane / 8)));
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)((int)(w >> (4 * i) & 15u) - 8) * s;
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(row + 2 * (head * kRowDim + 4 * lane));
    x[0] = __uint_as_float(w.x << 16);
    x[1] = __uint_as_float(w.x & 0xFFFF0000u);
    x[2] = __uint_as_float(w.y << 16);
    x[3] = __uint_as_float(w.y & 0xFFFF0000u);
  }
}

// A warp takes a row's head, key by key.
template <bool Q4>
__global__ void __launch_bounds__(128) paged_prefill_rows_kernel(const PackedPrefillParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, m = blockIdx.x, h = 4 * blockIdx.y + (threadIdx.x >> 5);
  if (h >= p.n_heads) return;
  const PackedRow row = packed_row(p.s, m, lane);
  if (row.bad && lane == 0 && h == 0) atomicCAS(p.err, 0, (int)DERR_PAGE_LIST);
  if (row.seq < 0) return;
  const size_t at = ((size_t)m * p.n_heads + h) * kRowDim + 4 * lane;
  const int kv = h / (p.n_heads / p.n_kv), end = min(row.pos + 1, p.max_len);
  float q[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, top = -FLT_MAX, l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = __bfloat162float(p.q[at + i]);
  for (int j = 0; j < end; ++j) {
    int place = page_row_of(p.s, row.seq, j);
    if (place < 0) {
      if (lane == 0) atomicCAS(p.err, 0, (int)DERR_POSITION);
      return;
    }
    float k[4], v[4], s = 0.f;
    row_values<Q4>(p.k + (size_t)place * p.row_bytes, p.n_kv, kv, lane, k);
    row_values<Q4>(p.v + (size_t)place * p.row_bytes, p.n_kv, kv, lane, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) s = fmaf(q[i], k[i], s);
    s = warp_sum(s) * p.scale_log2;
    const float mn = fmaxf(top, s), f = ex2_ftz(top - mn), w = ex2_ftz(s - mn);
    top = mn;
    l = l * f + w;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = fmaf(w, v[i], acc[i] * f);
  }
  const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) p.out[at + i] = __float2bfloat16_rn(acc[i] * inv);
}

}  // namespace tq

using namespace tq;

extern "C" int tq_gqa_prefill_paged(tq_ctx* ctx, const void* q_dev, const void* k_pages_dev, const void* v_pages_dev, int page_rows_as, const tq_pages* pages,
                                    const int* seqs_dev, const int* seq_rows_dev, size_t batch, size_t rows, size_t n_heads, size_t n_kv_heads,
                                    size_t head_dim, size_t max_len, void* out_dev) {
  if (int st = bind(ctx)) return st;
  if (batch == 0 || rows == 0) return TQ_OK;
  if (int st = check_packed(ctx, "tq_gqa_prefill_paged", pages, seqs_dev, seq_rows_dev, batch, rows, n_kv_heads, head_dim, page_rows_as)) return st;
  TQ_REQUIRE(ctx, q_dev && k_pages_dev && v_pages_dev && out_dev, "tq_gqa_prefill_paged: null pointer");
  TQ_REQUIRE(ctx, n_heads % n_kv_heads == 0 && n_heads / n_kv_heads >= 1 && n_heads / n_kv_heads <= 8, "tq_gqa_prefill_paged: n_heads/n_kv_heads must be 1..8");
  TQ_REQUIRE(ctx, max_len > 0 && max_len <= (1u << 30), "tq_gqa_prefill_paged: max_len must bound the sequence lengths");
  TQ_REQUIRE(ctx, (((uintptr_t)q_dev | (uintptr_t)k_pages_dev | (uintptr_t)v_pages_dev | (uintptr_t)out_dev) & 15) == 0,
             "tq_gqa_prefill_paged: arrays must be 16-byte aligned");
  const bool q4 = page_rows_as == TQ_PAGES_Q4;
  PackedPrefillParams p;
  p.s = packed_seqs(pages, seqs_dev, seq_rows_dev, batch, rows);
  p.q = static_cast<const __nv_bfloat16*>(q_dev);
  p.k = static_cast<const uint8_t*>(k_pages_dev);
  p.v = static_cast<const uint8_t*>(v_pages_dev);
  p.row_bytes = q4 ? q4_row_bytes(n_kv_heads) : n_kv_heads * kRowDim * 2;
  p.n_heads = (int)n_heads;
  p.n_kv = (int)n_kv_heads;
  p.max_len = (int)max_len;
  p.scale_log2 = 1.44269504088896340736f / sqrtf((float)head_dim);
  p.out = static_cast<__nv_bfloat16*>(out_dev);
  p.err = ctx->dev_err;
  if (int st = pages_use(ctx, pages)) return st;
  TQ_CUDA(ctx, launch_k(ctx, q4 ? paged_prefill_rows_kernel<true> : paged_prefill_rows_kernel<false>, dim3((unsigned)rows, (unsigned)((n_heads + 3) / 4)),
                        dim3(128), 0, p));
  return TQ_OK;
}
