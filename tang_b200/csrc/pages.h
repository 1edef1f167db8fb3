// A pool of cache pages (pages.cu) as the kernels that read it see it (paged_attention.cu).
#pragma once

#include <cstdlib>

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
  tq_pages* next = nullptr;     // of the context's
  unsigned long long id = 0;    // another one when the arrays are: recorded graphs hold the old list
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

// Before a kernel that reads or writes the pool is launched: an open capture takes its number down.
inline int pages_use(tq_ctx* ctx, const tq_pages* p) {
  if (!ctx->capturing) return TQ_OK;
  for (size_t i = 0; i < ctx->n_recorded_pools; ++i)
    if (ctx->recorded_pools[i] == p->id) return TQ_OK;
  if (ctx->n_recorded_pools == ctx->recorded_pools_room) {
    const size_t room = 2 * ctx->recorded_pools_room + 4;
    void* fresh = realloc(ctx->recorded_pools, room * sizeof(unsigned long long));
    if (!fresh) return fail(ctx, TQ_ENOMEM, "out of host memory");
    ctx->recorded_pools = static_cast<unsigned long long*>(fresh);
    ctx->recorded_pools_room = room;
  }
  ctx->recorded_pools[ctx->n_recorded_pools++] = p->id;
  return TQ_OK;
}
inline bool pages_live(const tq_ctx* ctx, unsigned long long id) {
  for (const tq_pages* p = ctx->pools; p; p = p->next)
    if (p->id == id) return true;
  return false;
}

}  // namespace tq
