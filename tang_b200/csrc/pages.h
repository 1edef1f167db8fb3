// A pool of cache pages (pages.cu) as the kernels that read it see it (paged_attention.cu).
#pragma once

#include "internal.h"

struct tq_pages {
  tq_ctx* ctx = nullptr;
  int *refs = nullptr, *tables = nullptr, *lens = nullptr;   // [n_pages], [n_seqs][table_ld], [n_seqs]
  int n_pages = 0, page_rows = 0, n_seqs = 0, table_ld = 0;
  void** arrays = nullptr;      // device: the caches' base pointers
  int n_arrays = 0;
  size_t row_bytes = 0;
  int* ws = nullptr;            // [0] copies to make; then their from, to and rows, a list of pages, a mark per sequence (zero between calls), refusals
  bool owns = false;
};

namespace tq {

constexpr int kPageCalls = 1024;   // sequences of one call: a thread each
inline size_t pages_max_copies(const tq_pages* p) { return p->n_pages > kPageCalls ? (size_t)p->n_pages : (size_t)kPageCalls; }
inline int* pages_copies(const tq_pages* p) { return p->ws + 4; }
inline int* pages_list(const tq_pages* p) { return pages_copies(p) + 3 * pages_max_copies(p); }
inline int* pages_marks(const tq_pages* p) { return pages_list(p) + p->n_pages; }
// Per sequence: not zero from a refused tq_pages_extend on until one that gives it new positions.  Its last position is then an old one, which a step must
// not write.
inline int* pages_refused(const tq_pages* p) { return pages_marks(p) + p->n_seqs; }
inline size_t pages_ws_ints(const tq_pages* p) { return 4 + 3 * pages_max_copies(p) + p->n_pages + 2 * (size_t)p->n_seqs; }

}  // namespace tq
