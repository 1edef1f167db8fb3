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
};
// Starts need not be what they should be: they are the device's.  Rows seq_rows[i] .. seq_rows[i+1]-1 are sequence i's if no start before seq_rows[i] is larger (the first
// one is 0) and they end neither before they begin nor behind the last row; such rows are never two sequences'.  Every kernel goes by that, whatever else the list
// holds, so that a row which is appended is attended, and one which is not is left alone by all of them.
//
// Row m's, by a whole warp, which reports what is wrong with it, or with the list.  Rows behind the last sequence are nowhere, and that is nothing to report.
__device__ __forceinline__ PackedRow packed_row(const PackedSeqs& p, int m, int lane, int* err) {
  const PackedRow nowhere{-1, 0};
  auto report = [&] {
    if (lane == 0) atomicCAS(err, 0, (int)DERR_PAGE_LIST);
  };
  int i = m, first = m, count = 1;
  if (p.seq_rows) {
    unsigned seen = 0;                 // starts at or before the row; from bit 16 on, those that are not what they should be
#pragma unroll 4
    for (int j = lane; j <= p.batch; j += 32) {
      const int start = p.seq_rows[j], next = j < p.batch ? p.seq_rows[j + 1] : p.rows;
      seen += (start <= m) + (start > next || (j == 0 && start != 0) ? 1u << 16 : 0u);
    }
    seen = __reduce_add_sync(0xffffffffu, seen);
    if (seen >> 16) {
      report();
      int largest = 0;                 // of the starts before the first one behind the row
      for (seen = 0; (int)seen <= p.batch && p.seq_rows[seen] <= m; ++seen) largest = max(largest, p.seq_rows[seen]);
      if (seen == 0 || (int)seen > p.batch) return nowhere;
      if (p.seq_rows[seen - 1] != largest || (seen == 1 && largest != 0) || p.seq_rows[seen] > p.rows) return nowhere;
    }
    if ((int)seen > p.batch) return nowhere;
    i = (int)seen - 1;
    first = p.seq_rows[i];
    count = p.seq_rows[i + 1] - first;
  }
  const int s = packed_seq(p, i), len = s < 0 ? 0 : p.lens[s];
  if (s < 0 || len < count || len > (long long)p.table_ld << p.page_shift) {
    report();
    return nowhere;
  }
  return PackedRow{s, len - count + (m - first)};
}

// Cache row of a position, the cache seen as one; -1 where the table names a page that does not exist.
__device__ __forceinline__ int page_row_of(const PackedSeqs& p, int seq, int pos, int* page_out = nullptr) {
  const int page = p.tables[(size_t)seq * p.table_ld + (pos >> p.page_shift)];
  if (page < 0 || page >= p.n_pages) return -1;
  if (page_out) *page_out = page;
  return (page << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
}

// Two arrays that share no byte.
inline bool apart(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
  return (uintptr_t)a + a_bytes <= (uintptr_t)b || (uintptr_t)b + b_bytes <= (uintptr_t)a;
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
