// Decode attention over a cache of pages (include/tangq.h: tq_gqa_decode_paged): the attention of tq_gqa_decode (attention.cu) for one new
// token per sequence, where position j of a sequence is row j % page_rows of page table[j / page_rows], and the positions that a group
// of sequences shares are the first member's.
#include <cuda_bf16.h>

#include <cfloat>
#include <type_traits>

#include "attn_mma.cuh"
#include "attn_umma.cuh"
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

__device__ __forceinline__ int paged_row_of(const PagedParams& p, int b) {
  const int s = p.seqs ? p.seqs[b] : b;
  return s >= 0 && s < p.n_seqs ? s : -1;
}
// ---------------------------------------------------------------------------------------------
// Units, tiles, items, pieces.  A unit is what meets the same keys: the rows (member, query head of one KV head) of up to 128 / group members of a group
// over the group's shared positions, in whole tiles of 128, or one sequence's query heads over the rest.  The tiles of all units of a KV head stand in one
// list, shared ones first, and are cut into items of equal length; CTAs, one an SM, take two items each and then the next one that nobody has, whatever
// the lengths of the sequences and the speeds of the SMs.  (Items of all KV heads that stand at the same place of their lists follow one another: a cache
// row holds all heads, and its 256 bytes a head are fetched at the same time.)  A piece is what an item has of a unit.  Its odd and its even tiles belong
// to different softmax groups, which keep sums and products of their own and leave a partial result each.
// ---------------------------------------------------------------------------------------------
constexpr int kPuThreads = 384;
constexpr int kPuTile = 4 * kPfBox / 2;               // bytes of 128 rows of keys or values
constexpr int kPuRing = 5;
constexpr int kPuWeights = 2 * 32 * 128;              // a parity's weights where keys are the lanes: 32 rows of 128 keys, in two halves
constexpr int kPuMeet = 2 * 2 * 4 * 32 * 4;           // [parity][maxima, sums][warp][row]
constexpr float kPuLargest = 7.9228162514264338e28f;  // 2^96: a weight above it is too far from its reference
constexpr int kPuHeader = 384;                        // barriers, items
constexpr int kPuReaders = 11;                        // warps that are told the items
constexpr int kPuBatch = 1024;                        // sequences of a call
constexpr size_t kPuFixed = 2 * (size_t)kPfBox + kPuRing * (size_t)kPuTile + 2 * (size_t)kPuWeights + kPuMeet + kPuHeader;

// In shared memory, behind the buffers.
struct PuPlan {
  int *own, *last, *pre, *eff;                        // [batch + 1] own tiles of the sequences before; [batch] shared tiles << 8 | keys of the last tile - 1;
                                                      // [groups + 1] units' shared tiles of the groups before; [groups] tiles that a group shares
  int batch, groups, group, per_tile, pre_tiles, total;
  int n_kv, pre_len, own_len, pre_items, items;       // tiles of an item, items of a KV head
};
struct PuUnit {
  bool pre;
  int b0, rows, tiles, tile, shared_tiles, last;      // b0: (first) sequence of the batch; tile: the asked one; last: keys of the last tile
  int slot;                                           // first row of its partial results, without what KV head and item add
};

__device__ __forceinline__ int pu_group_start(const PagedParams& p, int g) { return min(max(p.group_starts[g], 0), p.batch); }
__device__ __forceinline__ int pu_group_end(const PagedParams& p, int g, int start) { return g + 1 < p.n_groups ? max(pu_group_start(p, g + 1), start) : p.batch; }
__device__ __forceinline__ int pu_last_not_above(const int* a, int n, int v) {      // the last i < n with a[i] <= v (a ascends from 0)
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}
__device__ __forceinline__ PuUnit pu_locate(const PagedParams& p, const PuPlan& l, int f) {
  PuUnit u;
  u.pre = f < l.pre_tiles;
  if (u.pre) {
    const int g = pu_last_not_above(l.pre, l.groups, f), start = pu_group_start(p, g), members = pu_group_end(p, g, start) - start;
    u.tiles = l.eff[g];
    const int rest = f - l.pre[g], rt = rest / u.tiles;
    u.tile = rest - rt * u.tiles;
    u.b0 = start + rt * l.per_tile;
    u.rows = min(l.per_tile, members - rt * l.per_tile) * l.group;
    u.shared_tiles = 0;
    u.last = kPfTile;
    u.slot = u.b0 * l.group;
  } else {
    const int h = f - l.pre_tiles, b = pu_last_not_above(l.own, l.batch, h);
    u.tiles = l.own[b + 1] - l.own[b];
    u.tile = h - l.own[b];
    u.b0 = b;
    u.rows = l.group;
    u.shared_tiles = l.last[b] >> 8;
    u.last = (l.last[b] & 255) + 1;
    u.slot = b * l.group;
  }
  return u;
}

// From a tile of the list to the next one, f, which exists.
__device__ __forceinline__ void pu_step(const PagedParams& p, const PuPlan& l, PuUnit& u, int f) {
  if (++u.tile < u.tiles) return;
  if (u.pre) {
    u = pu_locate(p, l, f);
    return;
  }
  int b = u.b0 + 1;
  while (l.own[b + 1] == l.own[b]) ++b;
  u.tiles = l.own[b + 1] - l.own[b];
  u.tile = 0;
  u.b0 = b;
  u.shared_tiles = l.last[b] >> 8;
  u.last = (l.last[b] & 255) + 1;
  u.slot = b * l.group;
}
// Rows that are laid out for a unit whose keys are the tensor memory's lanes (0: its rows are), each as two terms but for the 32 of bf16 results.
template <int TERMS>
__device__ __forceinline__ int pu_wide(const PuUnit& u) { return u.rows <= 8 ? 8 : u.rows <= 16 ? 16 : u.rows <= 32 && TERMS == 1 ? 32 : 0; }
__device__ __forceinline__ int pu_keys(const PuUnit& u) { return u.tile == u.tiles - 1 ? u.last : kPfTile; }

// A role's place in the CTA's items.
struct PuCursor {
  PuUnit u;
  int f, end, kv, item;                               // tile of the list, the item's end; item: its number among the KV head's shared or own ones
  int piece;                                          // first tile of the piece
};
__device__ __forceinline__ void pu_begin(const PagedParams& p, const PuPlan& l, PuCursor& c, int item) {
  const int k = item / l.n_kv;
  c.kv = item - k * l.n_kv;
  const bool pre = k < l.pre_items;
  c.item = pre ? k : k - l.pre_items;
  c.f = pre ? c.item * l.pre_len : l.pre_tiles + c.item * l.own_len;
  c.end = pre ? min(c.f + l.pre_len, l.pre_tiles) : min(c.f + l.own_len, l.total);
  c.piece = c.f;
  c.u = pu_locate(p, l, c.f);
}
// Within an item: to the next tile, which exists.
__device__ __forceinline__ void pu_next(const PagedParams& p, const PuPlan& l, PuCursor& c) {
  ++c.f;
  pu_step(p, l, c.u, c.f);
  if (c.u.tile == 0) c.piece = c.f;
}
__device__ __forceinline__ int pu_piece_end(const PuCursor& c) { return min(c.end, c.f + c.u.tiles - c.u.tile); }
// Places in the ring, in the order in which they are needed: keys 0, keys 1, values 0, keys 2, values 1 ..
__device__ __forceinline__ int pu_keys_at(int t) { return t == 0 ? 0 : 2 * t - 1; }
__device__ __forceinline__ int pu_values_at(int t) { return 2 * t + 2; }

// What the kernel that joins the pieces has to know: where a sequence's tiles stand in a KV head's list, and how the list is cut.
struct PuSeqPlan {
  int own_f, own_tiles, pre_f, pre_tiles;             // (the place among the own, the shared tiles)
};

struct PuParams {
  PagedParams a;
  int per_tile, per_quarter;                          // members of a row tile; of a row tile that fits 32 rows
  int max_pre, max_own;                               // items of a KV head at most
  float *own_o, *own_ml, *pre_o, *pre_ml;             // partial results: [row][2][128], [row][2][2]
  PuSeqPlan* plan;
  int* plan_cut;                                      // [2] tiles of a shared, an own item
  int* counter;                                       // items handed out beyond the first two of every CTA; zero between calls
};

__device__ __forceinline__ void pu_scan(int* a, int n, int lane) {      // a[0 .. n-1] become the sums before them, a[n] the sum; one warp
  int sum = 0;
  for (int base = 0; base < n; base += 32) {
    const int v = base + lane < n ? a[base + lane] : 0;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int w = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += w;
    }
    if (base + lane < n) a[base + lane] = sum + incl - v;
    sum += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) a[n] = sum;
}

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float (&v)[8]) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}

template <int TERMS>
__global__ void __launch_bounds__(kPuThreads, 1)
paged_decode_kernel(const __grid_constant__ CUtensorMap q_own, const __grid_constant__ CUtensorMap q_quarter, const __grid_constant__ CUtensorMap q_whole,
                    const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const __grid_constant__ PuParams pp) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];   // (the swizzled buffers come first)
  const PagedParams& p = pp.a;
  uint8_t *q_s = smem_raw, *kv_s = q_s + 2 * kPfBox;
  uint8_t* w_s = kv_s + kPuRing * kPuTile;            // [parity]
  float* meet_s = reinterpret_cast<float*>(w_s + 2 * kPuWeights);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(meet_s + kPuMeet / 4);  // [4]
  uint64_t* q_empty = q_full + 4;                     // [4]
  uint64_t* kv_full = q_empty + 4;                    // [ring]
  uint64_t* kv_empty = kv_full + kPuRing;
  uint64_t* v_raw = kv_empty + kPuRing;               // [ring] values of a last tile, before the rows behind the last key are zeroed
  uint64_t* s_full = v_raw + kPuRing;                       // [parity]
  uint64_t* p_full = s_full + 2;
  uint64_t* o_done = p_full + 2;
  uint64_t* o_free = o_done + 2;
  uint64_t* item_full = o_free + 2;                   // [4]
  uint64_t* item_empty = item_full + 4;
  uint64_t* met = item_empty + 4;                     // [parity] the four warps of a softmax group
  int* item_s = reinterpret_cast<int*>(met + 2);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(item_s + 4);
  PuPlan l;
  l.own = reinterpret_cast<int*>(q_full) + kPuHeader / 4;
  l.last = l.own + p.batch + 1;
  l.pre = l.last + p.batch;
  l.eff = l.pre + p.n_groups + 1;
  l.batch = p.batch;
  l.groups = p.n_groups;
  l.group = p.group;
  l.per_tile = pp.per_tile;
  l.n_kv = p.n_kv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < 4; ++i) {
        mbar_init(&q_full[i], 1);
        mbar_init(&q_empty[i], 1);
        mbar_init(&item_full[i], 1);
        mbar_init(&item_empty[i], kPuReaders);
      }
      for (int i = 0; i < kPuRing; ++i) {
        mbar_init(&kv_full[i], 1);
        mbar_init(&kv_empty[i], 1);
        mbar_init(&v_raw[i], 1);
      }
      for (int x = 0; x < 2; ++x) {
        mbar_init(&s_full[x], 1);
        mbar_init(&p_full[x], 4);
        mbar_init(&o_done[x], 1);
        mbar_init(&o_free[x], 4);
        mbar_init(&met[x], 4);
      }
      mbar_init_fence();
    }
  } else if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
  } else if (warp == 3 && lane == 0) {
    prefetch_map(&q_own);
    prefetch_map(&k_map);
    prefetch_map(&v_map);
  }
  tc_fence_before();
  pdl_wait();
  pdl_launch_dependents();
  auto give_up = [&](int code) { atomicCAS(p.err, 0, code); };
  if (threadIdx.x == 0 && (smem_u32(smem_raw) & 1023)) give_up(DERR_TMEM);

  // ---- the plan: every CTA makes it for itself
  for (int b = threadIdx.x; b < p.batch; b += kPuThreads) {
    const int s = paged_row_of(p, b);
    if (s < 0 && blockIdx.x == 0) give_up(DERR_PAGE_LIST);
    l.own[b] = s < 0 ? 0 : min(max(p.lens[s], 0), p.max_len);
    l.last[b] = 0;
  }
  __syncthreads();
  for (int g = warp; g < p.n_groups; g += kPuThreads / 32) {
    // no more than the shortest member has, in whole tiles
    const int start = pu_group_start(p, g), end = pu_group_end(p, g, start);
    int least = min(max(p.shared[g], 0), p.max_shared);
    for (int b = start + lane; b < end; b += 32) least = min(least, l.own[b]);
    for (int o = 16; o > 0; o >>= 1) least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
    const int tiles = end - start > 1 ? least / kPfTile : 0;
    for (int b = start + lane; b < end; b += 32) l.last[b] = tiles << 8;
    if (lane == 0) {
      l.eff[g] = tiles;
      l.pre[g] = tiles * ((end - start + pp.per_tile - 1) / pp.per_tile);
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b < p.batch; b += kPuThreads) {
    const int len = l.own[b], shared = l.last[b] >> 8, tiles = (len + kPfTile - 1) / kPfTile;
    l.own[b] = tiles - shared;
    l.last[b] |= tiles > shared ? len - 1 - (tiles - 1) * kPfTile : 0;
  }
  __syncthreads();
  if (warp == 0) pu_scan(l.own, p.batch, lane);
  if (warp == 1) pu_scan(l.pre, p.n_groups, lane);
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  l.pre_tiles = l.pre[p.n_groups];
  l.total = l.pre_tiles + l.own[p.batch];
  const int own_tiles = l.own[p.batch];
  l.pre_len = max(1, (l.pre_tiles + pp.max_pre - 1) / pp.max_pre);
  // (as many turns of the CTAs as leave items of about four tiles, up to eight: shorter ones cost more than they balance)
  const int turns = max(1, min(pp.max_own / pp.max_pre, own_tiles / (4 * pp.max_pre)));
  l.own_len = max(1, (own_tiles + pp.max_pre * turns - 1) / (pp.max_pre * turns));
  l.pre_items = (l.pre_tiles + l.pre_len - 1) / l.pre_len;
  l.items = (l.pre_items + (own_tiles + l.own_len - 1) / l.own_len) * p.n_kv;
  if (blockIdx.x == 0) {               // for the kernel that joins the pieces
    for (int b = threadIdx.x; b < p.batch; b += kPuThreads) {
      int pre_f = 0;
      const int shared = l.last[b] >> 8;
      if (shared) {
        int lo = 0, hi = p.n_groups;   // the group with b: the last that starts there or before
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (pu_group_start(p, mid) <= b) lo = mid;
          else hi = mid;
        }
        pre_f = l.pre[lo] + (b - pu_group_start(p, lo)) / pp.per_tile * l.eff[lo];
      }
      pp.plan[b] = PuSeqPlan{l.own[b], l.own[b + 1] - l.own[b], pre_f, shared};
    }
    if (threadIdx.x == 0) {
      pp.plan_cut[0] = l.pre_len;
      pp.plan_cut[1] = l.own_len;
    }
  }
  // One arrival for the warp.  The lanes meet before it and behind it: none may wait for what the arrival lets happen before it is made.
  auto arrive = [&](uint64_t* bar) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
    __syncwarp();
  };
  // ---- items: warp 0 hands them on to the others (-1: there are no more)
  int it = 0;
  auto take = [&](bool& ok) {
    const int slot = it & 3;
    ok = __all_sync(0xffffffffu, ok && mbar_wait_spin(&item_full[slot], (uint32_t)((it >> 2) & 1)));
    const int item = __shfl_sync(0xffffffffu, ok ? item_s[slot] : -1, 0);
    arrive(&item_empty[slot]);
    ++it;
    return item;
  };

  if (warp == 0 || warp == 2) {
    // ---- copies: the keys of every tile (warp 0); the queries of every unit and the values of every tile (warp 2).  A lane per box: a page's rows, half
    // their columns.  The page of the next tile is asked for before the wait of this one.
    const bool values = warp == 2;
    const int box_rows = min(1 << p.page_shift, kPfTile), boxes = kPfTile / box_rows, j = lane >> 1, c = lane & 1;
    uint32_t q_used = 0;               // phases of the query slots
    int own_pieces = 0;
    bool ok = true;
    const int* table = nullptr;
    auto page_of = [&](const PuCursor& w, bool fresh) {
      if (fresh) {
        const int s = paged_row_of(p, w.u.pre ? pu_group_start(p, pu_last_not_above(l.pre, l.groups, w.f)) : w.u.b0);
        table = p.tables + (size_t)max(s, 0) * p.table_ld;
      }
      return j < boxes && j * box_rows < pu_keys(w.u) ? table[((w.u.shared_tiles + w.u.tile) * kPfTile + j * box_rows) >> p.page_shift] : 0;
    };
    // the items that come: the next one, and the one behind it, which is on its way
    const int n_ctas = (int)gridDim.x;
    int coming = (int)blockIdx.x, behind = (int)blockIdx.x + n_ctas;
    auto next_item = [&]() {
      if (values) return take(ok);
      const int item = coming < l.items ? coming : -1, slot = it & 3;
      coming = __shfl_sync(0xffffffffu, behind, 0);
      if (coming < l.items && lane == 0) behind = 2 * n_ctas + atomicAdd(pp.counter, 1);
      ok = __all_sync(0xffffffffu, ok && mbar_wait_spin(&item_empty[slot], (uint32_t)((it >> 2) & 1) ^ 1u));
      if (lane == 0) {
        item_s[slot] = item;
        mbar_arrive(&item_full[slot]);
      }
      __syncwarp();
      ++it;
      return ok ? item : -1;
    };
    PuCursor cur, next;
    int page = 0, page_next = 0, item = next_item();
    bool more = item >= 0, fresh_next = true;
    if (more) {
      pu_begin(p, l, next, item);
      page_next = page_of(next, true);
    }
    for (int t = 0; more && ok; ++t) {
      cur = next;
      page = page_next;
      const bool fresh = fresh_next;
      if (next.f + 1 < next.end) {
        pu_next(p, l, next);
      } else {
        item = next_item();
        more = item >= 0;
        if (more) pu_begin(p, l, next, item);
      }
      if (more) {
        fresh_next = next.piece == next.f;
        page_next = page_of(next, fresh_next);
      }
      const PuUnit& u = cur.u;
      if (values && fresh) {
        const int slot = u.pre ? 0 : own_pieces++ & 3;
        for (int k = 0; k < 4; ++k)
          if (ok && (u.pre || k == slot)) {
            ok = mbar_wait_spin(&q_empty[k], ((q_used >> k) & 1u) ^ 1u);
            q_used ^= 1u << k;
          }
        if (!ok) break;
        const bool whole = pu_wide<TERMS>(u) == 0;
        const uint32_t rows = (uint32_t)((whole ? pp.per_tile : u.pre ? pp.per_quarter : 1) * p.group);
        if (lane == 0) mbar_arrive_expect_tx(&q_full[slot], 2u * rows * 128u);
        __syncwarp();
        if (lane < 2) tma_load_3d(q_s + c * kPfBox + 16 * slot * 128, whole ? &q_whole : u.pre ? &q_quarter : &q_own, 64 * c, cur.kv * p.group, u.b0, &q_full[slot]);
        __syncwarp();
      }
      const int keys = pu_keys(u), used = (keys + box_rows - 1) / box_rows, r = values ? pu_values_at(t) : pu_keys_at(t), slot = r % kPuRing;
      if (j < used && (page < 0 || page >= p.n_pages)) {
        give_up(DERR_POSITION);
        page = 0;
      }
      const int row = (page << p.page_shift) + (((u.shared_tiles + u.tile) * kPfTile) & ((1 << p.page_shift) - 1) & ~(box_rows - 1));
      ok = ok && mbar_wait_spin(&kv_empty[slot], (uint32_t)((r / kPuRing) & 1) ^ 1u);
      if (!ok) break;
      uint64_t* bar = values && (keys & 15) ? &v_raw[slot] : &kv_full[slot];
      if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(used * box_rows) * 256u);
      __syncwarp();
      if (j < used) tma_load_2d(kv_s + slot * kPuTile + c * kPfBox + j * box_rows * 128, values ? &v_map : &k_map, cur.kv * kPaDim + 64 * c, row, bar);
      __syncwarp();
    }
    if (!ok) give_up(DERR_EMPTY_WAIT);
  } else if (warp == 3) {
    // ---- value rows between the last key and the next multiple of 16: whatever the cache holds there must not meet a weight of zero
    uint32_t used = 0;                 // phases of v_raw
    bool ok = true;
    int t = 0;                         // tiles before the piece
    for (int item = take(ok); item >= 0 && ok; item = take(ok)) {
      PuCursor c;
      pu_begin(p, l, c, item);
      while (ok) {
        const int end = pu_piece_end(c);
        t += end - c.f;
        const PuUnit& u = c.u;
        if (u.tile + end - c.f == u.tiles && (u.last & 15)) {
          const int slot = pu_values_at(t - 1) % kPuRing;
          ok = mbar_wait_spin(&v_raw[slot], (used >> slot) & 1u);
          used ^= 1u << slot;
          if (!ok) break;
          uint8_t* at = kv_s + slot * kPuTile;
          const int rows = 16 - (u.last & 15);
          for (int k = lane; k < 2 * rows * 8; k += 32) {             // (a row's 128 bytes of either box, whatever their order)
            const int box = (k >> 3) & 1, row = u.last + (k >> 4);
            *reinterpret_cast<uint4*>(at + box * kPfBox + row * 128 + 16 * (k & 7)) = make_uint4(0u, 0u, 0u, 0u);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          arrive(&kv_full[slot]);
        }
        if (end == c.end) break;
        c.u.tile += end - 1 - c.f;
        c.f = end - 1;
        pu_next(p, l, c);
      }
    }
    if (!ok) give_up(DERR_EMPTY_WAIT);
    __syncwarp();
  } else if (warp == 1) {
    // ---- products: the scores of a tile, then the weighted values of the tile before
    const bool leader = elect_one();
    const uint32_t idesc_o = umma_idesc_bf16(kPaDim) | (1u << 16);     // (bit 16: B is N-major; bit 15: A is M-major)
    const uint64_t qd = umma_desc_sw128(q_s), kd = umma_desc_sw128(kv_s), vd = pf_desc_mn(kv_s), wd = umma_desc_sw128(w_s);
    uint32_t q_seen = 0;
    int made[2] = {0, 0}, freed[2] = {0, 0};          // tiles of a parity so far, results read
    bool ok = true;
    struct Tile {
      int steps, wide;                                // 16-key steps, layout
      bool first;                                     // of its parity in the piece
    };
    auto values = [&](int t, const Tile& w) {
      const int x = t & 1, r = pu_values_at(t), slot = r % kPuRing;
      const uint32_t s_t = tmem + (uint32_t)(x * 256), o_t = s_t + 128u;
      bool good = mbar_wait_spin(&kv_full[slot], (uint32_t)((r / kPuRing) & 1)) && mbar_wait_spin(&p_full[x], (uint32_t)(made[x] & 1));
      ++made[x];
      if (good && w.first) {
        good = freed[x] == 0 || mbar_wait_spin(&o_free[x], (uint32_t)((freed[x] - 1) & 1));
        ++freed[x];
      }
      if (!good) return false;
      tc_fence_after();
      if (leader) {
        const uint64_t at = vd + (uint64_t)(slot * (kPuTile >> 4));
        if (w.wide) {
          const uint32_t idesc = umma_idesc_bf16(w.wide == 8 ? 16 : 32) | (1u << 15);
          for (int k = 0; k < w.steps; ++k)
            umma_f16(o_t, at + (uint64_t)(k * (2048 >> 4)), wd + (uint64_t)(x * (kPuWeights >> 4) + (k >> 2) * (kPuWeights >> 5) + 2 * (k & 3)), idesc, !w.first || k != 0);
        } else {
          for (int k = 0; k < w.steps; ++k) umma_f16_ts(o_t, s_t + 8u * k, at + (uint64_t)(k * (2048 >> 4)), idesc_o, !w.first || k != 0);
          if (TERMS == 2)
            for (int k = 0; k < w.steps; ++k) umma_f16_ts(o_t, s_t + 64u + 8u * k, at + (uint64_t)(k * (2048 >> 4)), idesc_o, 1u);
        }
        umma_commit(&o_done[x]);
        umma_commit(&kv_empty[slot]);
      }
      __syncwarp();
      return true;
    };
    PuCursor c;
    Tile before{};
    bool fresh[2] = {true, true};
    int own_pieces = 0, q_slot = 0, t = 0, item = take(ok);
    if (item >= 0) pu_begin(p, l, c, item);
    while (item >= 0 && ok) {
      const int x = t & 1, r = pu_keys_at(t), slot = r % kPuRing;
      const PuUnit& u = c.u;
      if (c.f == c.piece) {
        fresh[0] = fresh[1] = true;
        q_slot = u.pre ? 0 : own_pieces++ & 3;
        ok = mbar_wait_spin(&q_full[q_slot], (q_seen >> q_slot) & 1u);
        q_seen ^= 1u << q_slot;
      }
      // (the scores' columns hold the weights of the parity's tile before until its products are done)
      ok = ok && mbar_wait_spin(&kv_full[slot], (uint32_t)((r / kPuRing) & 1)) && (made[x] == 0 || mbar_wait_spin(&o_done[x], (uint32_t)((made[x] - 1) & 1)));
      if (!ok) break;
      tc_fence_after();
      const int keys = pu_keys(u);
      const Tile now{(keys + 15) >> 4, pu_wide<TERMS>(u), fresh[x]};
      fresh[x] = false;
      if (leader) {
        const uint32_t s_t = tmem + (uint32_t)(x * 256);
        const uint32_t idesc = umma_idesc_bf16(now.wide ? (now.wide == 32 ? 32 : 16) : kPfTile);
        const uint64_t kt = kd + (uint64_t)(slot * (kPuTile >> 4)), qt = qd + (uint64_t)(q_slot * (16 * 128 >> 4));
        const uint64_t da = now.wide ? kt : qt, db = now.wide ? qt : kt;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint64_t off = (uint64_t)((k >> 2) * (kPfBox >> 4) + 2 * (k & 3));
          umma_f16(s_t, da + off, db + off, idesc, k != 0);
        }
        umma_commit(&s_full[x]);
        umma_commit(&kv_empty[slot]);
        if (c.f + 1 == pu_piece_end(c))
          for (int k = 0; k < 4; ++k)
            if (u.pre || k == q_slot) umma_commit(&q_empty[k]);
      }
      __syncwarp();
      if (t > 0) ok = values(t - 1, before);
      before = now;
      ++t;
      if (c.f + 1 < c.end) {
        pu_next(p, l, c);
      } else {
        item = take(ok);
        if (item >= 0) pu_begin(p, l, c, item);
      }
    }
    if (ok && t > 0) ok = values(t - 1, before);
    if (!ok) give_up(DERR_FULL_WAIT);
  } else if (warp >= 4) {
    // ---- softmax of the tiles of a parity.  More than 32 rows: S = Q K^T, a thread per row, the weights over the scores' columns.  Up to 32: the keys are
    // the tensor memory's lanes, S^T = K Q^T and O^T = V^T P, with as many columns as there are rows (a product of 128 x 128 x 16 takes 84 cycles for four
    // rows too, one of 128 x 16 x 16 a fraction): a thread per key, whose weights go to shared memory, each as two bf16 terms in rows of their own.
    // The reference that scores are taken from is their maximum in the unit's first tile: a bf16 weight may be as large as an f32 one, so that
    // nothing is rescaled; a weight above 2^96 leaves a sum that is no number, and the joining kernel goes through the row's keys one by one.
    const int x = (warp - 4) >> 2, q4 = warp & 3;
    const uint32_t s_t = tmem + ((uint32_t)(32 * q4) << 16) + (uint32_t)(x * 256), o_t = s_t + 128u;
    float *max_s = meet_s + x * 256, *sum_s = max_s + 128;             // [warp][32 rows]
    int meetings = 0;
    bool ok = true, first = true;
    auto meet = [&]() {                // (a barrier of the group whose wait ends, as every other's)
      arrive(&met[x]);
      ok = __all_sync(0xffffffffu, ok && mbar_wait_spin(&met[x], (uint32_t)(meetings++ & 1)));
    };
    float ref[16], sums[32], largest = 0.f;            // (32 rows: the references stay in max_s)
    int done = 0;                      // tiles of this parity
    PuCursor cur;
    const PuUnit& u = cur.u;
    int place = 0;                     // the group's first tile of the piece is the piece's first or second: its partial result's place
    // a tile whose lanes are keys
    auto keyed = [&](auto rows_c) {
      constexpr int NR = decltype(rows_c)::value;
      constexpr bool kTwo = NR < 32;
      float v[NR];
      __syncwarp();
      if constexpr (NR == 8) tmem_ld8(s_t, v);
      else if constexpr (NR == 16) tmem_ld16(s_t, v);
      else pf_ld32(s_t, v);
      const int key = 32 * q4 + lane;
      const bool seen = key < pu_keys(u);
      if (first) {
        float mine = -FLT_MAX;
#pragma unroll
        for (int r = 0; r < NR; ++r)
          if (r < u.rows) {
            const float mx = warp_max(seen ? v[r] : -FLT_MAX);
            if (lane == r) mine = mx;
          }
        max_s[32 * q4 + lane] = mine;
        meet();
        if constexpr (NR == 32) {
          const float mx = fmaxf(fmaxf(max_s[lane], max_s[32 + lane]), fmaxf(max_s[64 + lane], max_s[96 + lane]));
          meet();                                      // (everyone has read: a warp's own 32 become the references)
          max_s[32 * q4 + lane] = mx;
          __syncwarp();
        } else {
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            ref[r] = fmaxf(fmaxf(max_s[r], max_s[32 + r]), fmaxf(max_s[64 + r], max_s[96 + r]));
            ref[r] = ref[r] == -FLT_MAX ? ref[r] : ref[r] * p.scale_log2;
          }
        }
#pragma unroll
        for (int r = 0; r < NR; ++r) sums[r] = 0.f;
      }
      uint8_t* at = w_s + x * kPuWeights + (key >> 6) * (kPuWeights / 2) + 2 * (key & 7);
      const int chunk = (key & 63) >> 3;
#pragma unroll
      for (int r = 0; r < NR; ++r)
        if (r < u.rows) {
          float from;
          if constexpr (NR == 32) from = max_s[32 * q4 + r] == -FLT_MAX ? -FLT_MAX : max_s[32 * q4 + r] * p.scale_log2;
          else from = ref[r];
          const float w = seen ? ex2(fmaf(v[r], p.scale_log2, -from)) : 0.f;
          sums[r] += w;
          largest = fmaxf(largest, w);
          const __nv_bfloat16 hi = __float2bfloat16_rn(w);
          *reinterpret_cast<__nv_bfloat16*>(at + r * 128 + ((chunk ^ (r & 7)) << 4)) = hi;
          if constexpr (kTwo) *reinterpret_cast<__nv_bfloat16*>(at + (NR + r) * 128 + ((chunk ^ (r & 7)) << 4)) = __float2bfloat16_rn(w - __bfloat162float(hi));
        }
      tc_fence_before();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    };
    auto keyed_out = [&](auto rows_c, float* to_o, float* to_ml) {
      constexpr int NR = decltype(rows_c)::value;
      constexpr bool kTwo = NR < 32;
      float o[32];
      __syncwarp();
      if constexpr (NR == 8) {
        float w[16];
        tmem_ld16(o_t, w);
#pragma unroll
        for (int r = 0; r < 8; ++r) o[r] = w[r] + w[8 + r];
      } else {
        pf_ld32(o_t, o);
        if constexpr (kTwo)
#pragma unroll
          for (int r = 0; r < NR; ++r) o[r] += o[NR + r];
      }
      tc_fence_before();
      arrive(&o_free[x]);                              // (the next unit's products may begin)
      float mine = 0.f;
#pragma unroll
      for (int r = 0; r < NR; ++r)
        if (r < u.rows) {
          to_o[(size_t)r * 2 * kPaDim + 32 * q4 + lane] = o[r];
          const float sum = warp_sum(largest > kPuLargest ? NAN : sums[r]);
          if (lane == r) mine = sum;
        }
      sum_s[32 * q4 + lane] = mine;
      meet();
      if (q4 == 0 && lane < u.rows) {
        const float mx = fmaxf(fmaxf(max_s[lane], max_s[32 + lane]), fmaxf(max_s[64 + lane], max_s[96 + lane]));
        *reinterpret_cast<float2*>(to_ml + lane * 4) =
            make_float2(mx == -FLT_MAX ? mx : mx * p.scale_log2, (sum_s[lane] + sum_s[32 + lane]) + (sum_s[64 + lane] + sum_s[96 + lane]));
      }
      meet();                                          // (the next unit's maxima go where these were)
    };
    using R8 = std::integral_constant<int, 8>;
    using R16 = std::integral_constant<int, 16>;
    using R32 = std::integral_constant<int, 32>;
    int item = take(ok);
    if (item >= 0) pu_begin(p, l, cur, item);
    bool begun = false;                // the group has had a tile of the piece
    for (int t = 0; item >= 0 && ok; ++t) {
      if (t > 0) {
        if (cur.f + 1 < cur.end) {
          pu_next(p, l, cur);
        } else {
          item = take(ok);
          if (item < 0) break;
          pu_begin(p, l, cur, item);
        }
      }
      if (cur.f == cur.piece) begun = false;
      if ((t & 1) != x) continue;
      first = !begun;
      if (first) {
        begun = true;
        place = (cur.f - cur.piece) & 1;
        largest = 0.f;
      }
      const int wide = pu_wide<TERMS>(u), r = 32 * q4 + lane;
      const bool live = r < u.rows;
      ok = __all_sync(0xffffffffu, mbar_wait_spin(&s_full[x], (uint32_t)(done & 1)));
      if (!ok) break;
      tc_fence_after();
      if (wide == 8) {
        keyed(R8());
      } else if (wide == 16) {
        keyed(R16());
      } else if (TERMS == 1 && wide == 32) {
        keyed(R32());
      } else {
        __syncwarp();
        if (first) {
          float mx = -FLT_MAX;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float v[32];
            pf_ld32(s_t + 32u * c, v);
#pragma unroll
            for (int j = 0; j < 32; ++j) mx = fmaxf(mx, v[j]);
          }
          ref[0] = mx == -FLT_MAX ? mx : mx * p.scale_log2;
          sums[0] = 0.f;
        }
        __syncwarp();
        uint32_t low[TERMS == 2 ? 64 : 1];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v[32];
          pf_ld32(s_t + 32u * c, v);
          uint32_t w[16];
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float w0 = ex2(fmaf(v[2 * j], p.scale_log2, -ref[0])), w1 = ex2(fmaf(v[2 * j + 1], p.scale_log2, -ref[0]));
            sum[j & 3] += w0 + w1;
            if constexpr (TERMS == 2) split_bf16(w0, w1, w[j], low[16 * c + j]);
            else w[j] = pack_bf16(w0, w1);
          }
          sums[0] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          tmem_st16(s_t + 16u * c, w);                 // over scores that this thread has read
        }
        largest = sums[0];
        if constexpr (TERMS == 2)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t w[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = low[16 * c + j];
            tmem_st16(s_t + 64u + 16u * c, w);
          }
        tmem_st_wait();
        tc_fence_before();
      }
      arrive(&p_full[x]);
      ++done;
      if (cur.f + 2 < pu_piece_end(cur)) continue;

      // ---- the piece's result
      ok = __all_sync(0xffffffffu, mbar_wait_spin(&o_done[x], (uint32_t)((done - 1) & 1)));
      if (!ok) break;
      tc_fence_after();
      const int apart = u.pre ? 128 : 8;
      const size_t row0 = (size_t)cur.kv * (p.batch * p.group + apart * (u.pre ? pp.max_pre : pp.max_own)) + u.slot + apart * cur.item;
      float *to_o = (u.pre ? pp.pre_o : pp.own_o) + (row0 * 2 + place) * kPaDim, *to_ml = (u.pre ? pp.pre_ml : pp.own_ml) + (row0 * 2 + place) * 2;
      if (wide == 8) {
        keyed_out(R8(), to_o, to_ml);
      } else if (wide == 16) {
        keyed_out(R16(), to_o, to_ml);
      } else if (TERMS == 1 && wide == 32) {
        keyed_out(R32(), to_o, to_ml);
      } else {
#pragma unroll 1
        for (int c = 0; c < kPaDim; c += 32) {
          float o[32];
          __syncwarp();
          pf_ld32(o_t + (uint32_t)c, o);
          float4* o_row = reinterpret_cast<float4*>(to_o + (size_t)r * 2 * kPaDim + c);
          if (live)
#pragma unroll
            for (int j = 0; j < 8; ++j) o_row[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
        }
        tc_fence_before();
        arrive(&o_free[x]);
        if (live)
          *reinterpret_cast<float2*>(to_ml + r * 4) = make_float2(ref[0], largest > kPuLargest ? NAN : sums[0]);
      }
    }
    if (!ok) give_up(DERR_TMEM);
  }
  tc_fence_before();
  __syncthreads();
  __syncwarp();                        // (the release is one instruction of the whole warp)
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// Joins the pieces of a query head: a warp per head, four columns a lane.
__global__ void __launch_bounds__(128) paged_join_kernel(const PuParams pp) {
  pdl_wait();
  pdl_launch_dependents();
  const PagedParams& p = pp.a;
  const int b = blockIdx.x, lane = threadIdx.x & 31;
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *pp.counter = 0;
  const PuSeqPlan q = pp.plan[b];
  const int cut[2] = {pp.plan_cut[1], pp.plan_cut[0]};
  const int head = (int)(blockIdx.y * 4 + (threadIdx.x >> 5));
  if (head < p.n_heads) {
    const int kv = head / p.group, h = head - kv * p.group;
    // tiles of the own and of the shared part, first item and number of (item, place)s
    const int f[2] = {q.own_f, q.pre_f}, e[2] = {q.own_f + q.own_tiles, q.pre_f + q.pre_tiles}, apart[2] = {8, 128}, most[2] = {pp.max_own, pp.max_pre};
    int c[2] = {0, 0}, places[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (e[k] > f[k]) {
        c[k] = f[k] / cut[k];
        places[k] = 2 * ((e[k] - 1) / cut[k] - c[k] + 1);
      }
    const int all = places[0] + places[1];
    float top = -FLT_MAX, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int base = 0; base < all; base += 32) {
      // a lane per place: its row of the partial results (the second one of a piece of one tile is none), maximum and sum
      const int i = base + lane;
      const float *row = nullptr, *ml = nullptr;
      if (i < all) {
        const int k = i >= places[0], j = k ? i - places[0] : i, item = c[k] + (j >> 1), x = j & 1;
        const int lo = max(f[k], item * cut[k]), hi = min(e[k], (item + 1) * cut[k]);
        if (hi - lo > x) {
          const size_t r = ((size_t)kv * (p.batch * p.group + apart[k] * most[k]) + b * p.group + h + (size_t)apart[k] * item) * 2 + x;
          row = (k ? pp.pre_o : pp.own_o) + r * kPaDim;
          ml = (k ? pp.pre_ml : pp.own_ml) + r * 2;
        }
      }
      float2 mine = make_float2(-FLT_MAX, 0.f);
      if (ml) mine = *reinterpret_cast<const float2*>(ml);
      const float to = fmaxf(top, warp_max(mine.x)), f0 = ex2(top - to), w = ex2(mine.x - to);
      top = to;
      l = l * f0 + warp_sum(mine.y * w);
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] *= f0;
      const int count = min(32, all - base);
#pragma unroll 8
      for (int k = 0; k < count; ++k) {
        const float* from = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, (unsigned long long)row, k));
        const float wk = __shfl_sync(0xffffffffu, w, k);
        if (from) {
          const float4 v = *reinterpret_cast<const float4*>(from + 4 * lane);
          o[0] = fmaf(v.x, wk, o[0]);
          o[1] = fmaf(v.y, wk, o[1]);
          o[2] = fmaf(v.z, wk, o[2]);
          o[3] = fmaf(v.w, wk, o[3]);
        }
      }
    }
    const size_t at = ((size_t)b * p.n_heads + head) * kPaDim + 4 * lane;
    if (__any_sync(0xffffffffu, l != l || o[0] != o[0] || o[1] != o[1] || o[2] != o[2] || o[3] != o[3])) {
      // A score far above those of its unit's first tile, or an infinite value beside a weight that is zero as a second term: once more, key by key.
      const int s = paged_row_of(p, b), len = s < 0 ? 0 : min(max(p.lens[s], 0), p.max_len);
      float m = -FLT_MAX, x[4];
      l = o[0] = o[1] = o[2] = o[3] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __bfloat162float(p.q[at + i]);
      for (int j = 0; j < len; ++j) {
        const int page = min(max(p.tables[(size_t)s * p.table_ld + (j >> p.page_shift)], 0), p.n_pages - 1);
        const size_t r = (((size_t)page << p.page_shift) + (j & ((1 << p.page_shift) - 1))) * p.n_kv * kPaDim + (size_t)kv * kPaDim;
        attend_row(p.k + r, 0, p.v + r, 0, 0, 1, x, p.scale_log2, lane, m, l, o);
      }
    }
    const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;              // (a NaN stays one)
    if (p.out_f32) {
      *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    } else {
      uint2 w;
      w.x = pack_bf16(o[0] * inv, o[1] * inv);
      w.y = pack_bf16(o[2] * inv, o[3] * inv);
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at) = w;
    }
  }
}

// Rows of `row` bf16 [rows], boxes of 64 columns x `box_rows` rows in the 128-byte swizzle.
static bool encode_pages(CUtensorMap* map, const void* base, size_t row, size_t rows, unsigned box_rows) {
  return encode_bf16_k64(map, base, rows, row, row, box_rows);
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
  TQ_REQUIRE(ctx, batch <= (size_t)kPuBatch && (seqs_dev || batch <= (size_t)pages->n_seqs), "tq_gqa_decode_paged: at most %d sequences, and no more than the pool has", kPuBatch);
  const size_t most = (size_t)pages->table_ld * pages->page_rows;
  TQ_REQUIRE(ctx, max_len > 0 && max_len <= (1u << 30), "tq_gqa_decode_paged: max_len must bound the sequence lengths");
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
  p.n_groups = group_starts_dev ? (int)n_groups : 0;
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
  PuParams pp;
  pp.per_tile = 128 / p.group;
  pp.per_quarter = 32 / p.group;
  const size_t tiles = batch * (((size_t)p.max_len + kPfTile - 1) / kPfTile) * n_kv_heads;
  TQ_REQUIRE(ctx, tiles < (1ull << 30) && (size_t)p.n_pages * pages->page_rows < (1ull << 31), "tq_gqa_decode_paged: too many positions");
  const size_t n_ctas = tiles < (size_t)ctx->sm_count ? tiles : (size_t)ctx->sm_count;
  // A CTA takes one item of shared tiles (whose partial results are many rows) and eight of the others, if there are as many tiles.
  const size_t per_kv = ((size_t)ctx->sm_count + n_kv_heads - 1) / n_kv_heads;
  pp.max_pre = (int)per_kv;
  pp.max_own = (int)(8 * per_kv);
  // partial results, the sequences' plans
  const size_t own_rows = (batch * n_heads + 8 * n_kv_heads * pp.max_own) * 2, pre_rows = p.n_groups ? (batch * n_heads + 128 * n_kv_heads * pp.max_pre) * 2 : 0;
  const size_t floats = (own_rows + pre_rows) * (kPaDim + 2);
  if (int st = ensure_scratch(ctx, floats * sizeof(float) + (batch + 1) * sizeof(PuSeqPlan))) return st;
  pp.own_o = static_cast<float*>(ctx->scratch);
  pp.pre_o = pp.own_o + own_rows * kPaDim;
  pp.own_ml = pp.pre_o + pre_rows * kPaDim;
  pp.pre_ml = pp.own_ml + own_rows * 2;
  pp.plan = reinterpret_cast<PuSeqPlan*>(pp.pre_ml + pre_rows * 2);
  pp.plan_cut = reinterpret_cast<int*>(pp.plan + batch);
  pp.counter = ctx->dev_err + kTileCounters;          // (the last of the counters)
  pp.a = p;
  CUtensorMap qo, qq, qw, km, vm;
  const size_t row = n_kv_heads * kPaDim, rows = (size_t)p.n_pages * pages->page_rows;
  const unsigned g = (unsigned)p.group, box = pages->page_rows < kPfTile ? (unsigned)pages->page_rows : (unsigned)kPfTile;
  auto q_map = [&](CUtensorMap* m, int members) { return encode_bf16_boxes(m, q_dev, kPaDim, n_heads, batch, kPaDim * 2, n_heads * kPaDim * 2, g, (unsigned)members); };
  if (!q_map(&qo, 1) || !q_map(&qq, pp.per_quarter) || !q_map(&qw, pp.per_tile) || !encode_pages(&km, k_pages_dev, row, rows, box) ||
      !encode_pages(&vm, v_pages_dev, row, rows, box))
    return fail(ctx, TQ_ECUDA, "cuTensorMapEncodeTiled failed");
  const size_t smem = kPuFixed + (2 * batch + 1 + 2 * (size_t)p.n_groups + 1) * sizeof(int);
  auto kern = p.out_f32 ? paged_decode_kernel<2> : paged_decode_kernel<1>;
  TQ_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kPuFixed + (4 * kPuBatch + 2) * sizeof(int))));
  TQ_CUDA(ctx, launch_k(ctx, kern, dim3((unsigned)n_ctas), dim3(kPuThreads), smem, qo, qq, qw, km, vm, pp));
  TQ_CUDA(ctx, launch_k(ctx, paged_join_kernel, dim3((unsigned)batch, (unsigned)((n_heads + 3) / 4)), dim3(128), 0, pp));
  return TQ_OK;
}
