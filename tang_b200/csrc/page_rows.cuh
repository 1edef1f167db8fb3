// Packed rows of several sequences over a pool of pages, and cache rows of 4 bits, as the kernels of page_rows.cu, paged_prefill.cu and
// paged_q4.cu see them.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "pages.h"

namespace tq {

constexpr int kRowDim = 128;           // values of a head
constexpr int kQ4Block = 32;           // values that share a scale
constexpr int kQ4HeadBytes = kRowDim / 2, kQ4HeadScales = kRowDim / kQ4Block;
__host__ __device__ inline size_t q4_row_bytes(size_t n_kv) { return (n_kv * (kQ4HeadBytes + 2 * kQ4HeadScales) + 15) / 16 * 16; }

// Two f32 numbers in one operation.  (A product that goes into a sum may come out as one fused operation.)
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// A pool's state and a list of sequences whose last positions are packed rows (include/tangq.h: tq_kv_append_paged).
struct PackedSeqs {
  const int *tables, *lens, *refs, *refused;           // of the pool
  const int *seqs, *seq_rows;                          // null: sequence i of the list is i of the pool; row i is sequence i's
  int batch, rows, n_seqs, table_ld, n_pages, page_shift;
};

inline PackedSeqs packed_seqs(const tq_pages* pages, const int* seqs, const int* seq_rows, size_t batch, size_t rows) {
  return PackedSeqs{pages->tables, pages->lens, pages->refs, pages_refused(pages), seqs, seq_rows, (int)batch, (int)rows, pages->n_seqs, pages->table_ld,
                    pages->n_pages, 31 - __builtin_clz((unsigned)pages->page_rows)};
}

// Sequence i of the list as a sequence of the pool, -1 where there is none.
__device__ __forceinline__ int packed_seq(const PackedSeqs& p, int i) {
  const int s = p.seqs ? p.seqs[i] : i;
  return s >= 0 && s < p.n_seqs ? s : -1;
}

// Where a packed row stands.
struct PackedRow {
  int seq, pos;                        // of the pool (-1: nowhere), position
  int i;                               // of the list
  bool bad;                            // there is something to report
};
// Row m's, by a whole warp.  Rows behind the last sequence are nowhere, and that is nothing to report.
__device__ __forceinline__ PackedRow packed_row(const PackedSeqs& p, int m, int lane) {
  PackedRow r{-1, 0, m, false};
  int first = m, count = 1;
  if (p.seq_rows) {
    int below = 0;                     // starts at or before the row
#pragma unroll 4
    for (int j = lane; j <= p.batch; j += 32) below += p.seq_rows[j] <= m;
    below = __reduce_add_sync(0xffffffffu, below);
    if (below > p.batch) return r;
    r.bad = below == 0;
    if (r.bad) return r;
    r.i = below - 1;
    first = p.seq_rows[r.i];
    const int end = p.seq_rows[below];
    count = end - first;
    r.bad = first < 0 || m < first || m >= end || end > p.rows;        // (starts that do not ascend)
    if (r.bad) return r;
  }
  const int s = packed_seq(p, r.i), len = s < 0 ? 0 : p.lens[s];
  r.bad = s < 0 || len < count || len > (long long)p.table_ld << p.page_shift;
  if (r.bad) return r;
  r.seq = s;
  r.pos = len - count + (m - first);
  return r;
}

// Cache row of a position, the cache seen as one; -1 where the table names a page that does not exist.
__device__ __forceinline__ int page_row_of(const PackedSeqs& p, int seq, int pos, int* page_out = nullptr) {
  const int page = p.tables[(size_t)seq * p.table_ld + (pos >> p.page_shift)];
  if (page < 0 || page >= p.n_pages) return -1;
  if (page_out) *page_out = page;
  return (page << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
}

// What calls over packed rows ask of their arguments.
inline int check_packed(tq_ctx* ctx, const char* call, const tq_pages* pages, const int* seqs, const int* seq_rows, size_t batch, size_t rows, size_t n_kv,
                        size_t head_dim, int page_rows_as) {
  TQ_REQUIRE(ctx, pages, "%s: null pointer", call);
  TQ_REQUIRE(ctx, pages->ctx == ctx, "%s: the pool belongs to another context", call);
  TQ_REQUIRE(ctx, head_dim == (size_t)kRowDim, "%s: head_dim must be %d", call, kRowDim);
  TQ_REQUIRE(ctx, page_rows_as == TQ_PAGES_BF16 || page_rows_as == TQ_PAGES_Q4, "%s: pages hold rows of bf16 or of 4 bits", call);
  TQ_REQUIRE(ctx, batch <= (size_t)kPageCalls && (seqs || batch <= (size_t)pages->n_seqs), "%s: at most %d sequences, and no more than the pool has", call,
             kPageCalls);
  TQ_REQUIRE(ctx, seq_rows || rows == batch, "%s: without starts every sequence has one row", call);
  TQ_REQUIRE(ctx, rows < (1u << 30), "%s: too many rows", call);
  TQ_REQUIRE(ctx, n_kv >= 1 && n_kv <= 1024 && (size_t)pages->n_pages * pages->page_rows < (1ull << 31), "%s: too many positions or heads", call);
  return TQ_OK;
}

}  // namespace tq
