// Decode attention over a cache of pages (include/tangq.h: tq_gqa_decode_paged): the attention of tq_gqa_decode (attention.cu) for one new
// token per sequence, where position j of a sequence is row j % page_rows of page table[j / page_rows], and the positions that a group
// of sequences shares are the first member's.
#include <cuda_bf16.h>

#include <cfloat>

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
// Units, tiles, pieces.  A unit is what meets the same keys: the rows (member, query head of one KV head) of up to 128 / group members of a group over
// the group's shared positions, in whole tiles of 128, or one sequence's query heads over the rest.  All tiles of all units stand in one list, shared ones
// first, and CTA c of N takes tiles T c / N .. T (c + 1) / N - 1: the same number each, whatever the lengths.  Odd and even tiles of the list belong
// to different softmax groups, which keep maximum, sum and products of their own: a piece (unit, CTA, parity) leaves one partial result.
// ---------------------------------------------------------------------------------------------
constexpr int kPuThreads = 384;
constexpr int kPuTile = 4 * kPfBox / 2;               // bytes of 128 rows of keys or values
constexpr int kPuRing = 5;
constexpr int kPuStageLd = 17;                        // words between rows of a group's staging
constexpr int kPuStage = 128 * kPuStageLd * 4;
constexpr int kPuHeader = 512;
constexpr int kPuBatch = 1024;                        // sequences of a call
constexpr size_t kPuFixed = kPuHeader + 1024 + 2 * (size_t)kPfBox + kPuRing * (size_t)kPuTile + 2 * (size_t)kPuStage;

// In shared memory, behind the buffers.
struct PuPlan {
  int *own, *last, *pre, *eff;                        // [batch + 1] own tiles of the sequences before; [batch] shared tiles << 8 | keys of the last tile - 1;
                                                      // [groups + 1] shared tiles of the groups before; [groups] tiles that a group shares
  int batch, groups, n_kv, group, per_tile, pre_tiles, total;
};
struct PuUnit {
  bool pre;
  int b0, kv, rows, tiles, tile, shared_tiles, last;  // b0: (first) sequence of the batch; tile: the asked one; last: keys of the last tile
  int slot;                                           // first row of its partial results at CTA 0
  int q_slot;
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
    const int row_tiles = (members + l.per_tile - 1) / l.per_tile;
    u.tiles = l.eff[g];
    const int rest = f - l.pre[g], unit = rest / u.tiles, rt = unit % row_tiles;
    u.tile = rest - unit * u.tiles;
    u.kv = unit / row_tiles;
    u.b0 = start + rt * l.per_tile;
    u.rows = min(l.per_tile, members - rt * l.per_tile) * l.group;
    u.shared_tiles = 0;
    u.last = kPfTile;
    u.slot = (start * l.n_kv + u.kv * members + rt * l.per_tile) * l.group;
    u.q_slot = 0;
  } else {
    const int h = f - l.pre_tiles, b = pu_last_not_above(l.own, l.batch, h / l.n_kv);
    u.tiles = l.own[b + 1] - l.own[b];
    const int rest = h - l.own[b] * l.n_kv;
    u.kv = rest / u.tiles;
    u.tile = rest - u.kv * u.tiles;
    u.b0 = b;
    u.rows = l.group;
    u.shared_tiles = l.last[b] >> 8;
    u.last = (l.last[b] & 255) + 1;
    u.slot = (b * l.n_kv + u.kv) * l.group;
    u.q_slot = (b * l.n_kv + u.kv) & 3;
  }
  return u;
}

// What the kernel that joins the pieces has to know of a sequence, and the total behind them all.
struct PuSeqPlan {
  int own_f, own_tiles;                               // first tile of (sequence, KV head 0) in the list, tiles per KV head
  int pre_f, pre_kv, pre_tiles;                       // first tile of its row tile's unit for KV head 0, tiles between KV heads, tiles of the unit
  int pre_row, pre_row_kv;                            // its first row among the partial results, rows between KV heads
  int pad;
};

struct PuParams {
  PagedParams a;
  int per_tile, per_quarter;                          // members of a row tile; of a row tile that fits 32 rows
  float *own_o, *own_ml, *pre_o, *pre_ml;             // partial results: [row][parity][128], [row][parity][2]
  PuSeqPlan* plan;
  int* plan_total;
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

template <int TERMS>
__global__ void __launch_bounds__(kPuThreads, 1)
paged_decode_kernel(const __grid_constant__ CUtensorMap q_own, const __grid_constant__ CUtensorMap q_quarter, const __grid_constant__ CUtensorMap q_whole,
                    const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const __grid_constant__ PuParams pp) {
  extern __shared__ uint8_t smem_raw[];
  const PagedParams& p = pp.a;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem_raw);            // [4]
  uint64_t* q_empty = q_full + 4;                     // [4]
  uint64_t* kv_full = q_empty + 4;                    // [ring]
  uint64_t* kv_empty = kv_full + kPuRing;
  uint64_t* v_raw = kv_empty + kPuRing;               // [ring] values of a last tile, before the rows behind the last key are zeroed
  uint64_t* s_full = v_raw + kPuRing;                       // [parity]
  uint64_t* p_full = s_full + 2;
  uint64_t* o_done = p_full + 2;
  uint64_t* o_free = o_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_free + 2);
  uint8_t* q_s = smem_raw + kPuHeader + ((1024 - ((smem_u32(smem_raw) + kPuHeader) & 1023)) & 1023);
  uint8_t* kv_s = q_s + 2 * kPfBox;
  float* stage_s = reinterpret_cast<float*>(kv_s + kPuRing * kPuTile);
  PuPlan l;
  l.own = reinterpret_cast<int*>(stage_s) + 2 * kPuStage / 4;
  l.last = l.own + p.batch + 1;
  l.pre = l.last + p.batch;
  l.eff = l.pre + p.n_groups + 1;
  l.batch = p.batch;
  l.groups = p.n_groups;
  l.n_kv = p.n_kv;
  l.group = p.group;
  l.per_tile = pp.per_tile;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < 4; ++i) {
        mbar_init(&q_full[i], 1);
        mbar_init(&q_empty[i], 1);
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
      }
      mbar_init_fence();
    }
  } else if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
  } else if (warp == 2 && lane == 0) {
    prefetch_map(&q_own);
    prefetch_map(&k_map);
    prefetch_map(&v_map);
  }
  tc_fence_before();
  pdl_wait();
  pdl_launch_dependents();
  auto give_up = [&](int code) { atomicCAS(p.err, 0, code); };

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
      l.pre[g] = tiles * ((end - start + pp.per_tile - 1) / pp.per_tile) * p.n_kv;
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
  l.total = l.pre_tiles + l.own[p.batch] * p.n_kv;
  const int f0 = (int)((long long)l.total * blockIdx.x / gridDim.x), f1 = (int)((long long)l.total * (blockIdx.x + 1) / gridDim.x), n = f1 - f0;
  if (blockIdx.x == 0) {               // for the kernel that joins the pieces
    for (int b = threadIdx.x; b < p.batch; b += kPuThreads) {
      PuSeqPlan q;
      q.own_tiles = l.own[b + 1] - l.own[b];
      q.own_f = l.pre_tiles + l.own[b] * p.n_kv;
      q.pre_tiles = l.last[b] >> 8;
      q.pre_f = q.pre_kv = q.pre_row = q.pre_row_kv = q.pad = 0;
      pp.plan[b] = q;
    }
    __syncthreads();
    for (int g = warp; g < p.n_groups; g += kPuThreads / 32) {
      const int start = pu_group_start(p, g), end = pu_group_end(p, g, start), members = end - start, row_tiles = (members + pp.per_tile - 1) / pp.per_tile;
      for (int b = start + lane; b < end; b += 32) {
        const int rt = (b - start) / pp.per_tile;
        PuSeqPlan* q = &pp.plan[b];
        q->pre_f = l.pre[g] + rt * l.eff[g];
        q->pre_kv = row_tiles * l.eff[g];
        q->pre_row = (start * p.n_kv + b - start) * p.group;
        q->pre_row_kv = members * p.group;
      }
    }
    if (threadIdx.x == 0) *pp.plan_total = l.total;
  }

  if (warp == 0) {
    // ---- copies: queries of every unit, keys and values of every tile; a lane per box
    uint32_t q_used = 0;               // phases of the query slots
    PuUnit u;
    int page_next = 0;
    const int* table = p.tables;
    const int box_rows = min(1 << p.page_shift, kPfTile), boxes = kPfTile / box_rows;
    bool ok = true;
    // the page of box `lane / 2` of a tile (the boxes' halves are the lanes' parity)
    auto page_of = [&](const PuUnit& w, const int* t, int tile, int keys) {
      const int j = lane >> 1, at = tile * kPfTile + j * box_rows;
      if (j >= boxes || j * box_rows >= keys) return -1;
      int page = t[at >> p.page_shift];
      if (page < 0 || page >= p.n_pages) {
        give_up(DERR_POSITION);
        page = 0;
      }
      return page;
    };
    for (int i = 0; i < n && ok; ++i) {
      if (i == 0 || ++u.tile == u.tiles) {
        u = pu_locate(p, l, f0 + i);
        const int first = u.pre ? pu_group_start(p, pu_last_not_above(l.pre, l.groups, f0 + i)) : u.b0, s = paged_row_of(p, first);
        table = p.tables + (size_t)max(s, 0) * p.table_ld;
        page_next = page_of(u, table, u.shared_tiles + u.tile, u.tile == u.tiles - 1 ? u.last : kPfTile);
        if (u.pre) {
          for (int j = 0; j < 4 && ok; ++j) ok = mbar_wait_spin(&q_empty[j], ((q_used >> j) & 1u) ^ 1u);
          q_used ^= 15u;
          if (!ok) break;
          if (lane == 0) {
            if (u.rows <= 32) {
              mbar_arrive_expect_tx(&q_full[0], 8u * (uint32_t)(pp.per_quarter * p.group) * 128u);
              for (int j = 0; j < 8; ++j) tma_load_3d(q_s + (j & 1) * kPfBox + (j >> 1) * 32 * 128, &q_quarter, 64 * (j & 1), u.kv * p.group, u.b0, &q_full[0]);
            } else {
              mbar_arrive_expect_tx(&q_full[0], 2u * (uint32_t)(pp.per_tile * p.group) * 128u);
              for (int j = 0; j < 2; ++j) tma_load_3d(q_s + j * kPfBox, &q_whole, 64 * j, u.kv * p.group, u.b0, &q_full[0]);
            }
          }
        } else {
          ok = mbar_wait_spin(&q_empty[u.q_slot], ((q_used >> u.q_slot) & 1u) ^ 1u);
          q_used ^= 1u << u.q_slot;
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_full[u.q_slot], 8u * (uint32_t)p.group * 128u);
            for (int j = 0; j < 8; ++j)
              tma_load_3d(q_s + (j & 1) * kPfBox + ((j >> 1) * 32 + 8 * u.q_slot) * 128, &q_own, 64 * (j & 1), u.kv * p.group, u.b0, &q_full[u.q_slot]);
          }
        }
        __syncwarp();
      }
      const bool is_last = u.tile == u.tiles - 1;
      const int keys = is_last ? u.last : kPfTile, page = page_next, tile = u.shared_tiles + u.tile;
      if (!is_last) page_next = page_of(u, table, tile + 1, u.tile + 1 == u.tiles - 1 ? u.last : kPfTile);
      const int used = (keys + box_rows - 1) / box_rows, j = lane >> 1, c = lane & 1;
      const int row = (page << p.page_shift) + ((tile * kPfTile) & ((1 << p.page_shift) - 1) & ~(box_rows - 1));
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int r = 2 * i + kv, slot = r % kPuRing;
        ok = ok && mbar_wait_spin(&kv_empty[slot], (uint32_t)((r / kPuRing) & 1) ^ 1u);
        if (!ok) break;
        uint64_t* bar = kv && (keys & 15) ? &v_raw[slot] : &kv_full[slot];
        if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(used * box_rows) * 256u);
        __syncwarp();
        if (j < used) tma_load_2d(kv_s + slot * kPuTile + c * kPfBox + j * box_rows * 128, kv ? &v_map : &k_map, u.kv * kPaDim + 64 * c, row, bar);
        __syncwarp();
      }
    }
    if (!ok) give_up(DERR_EMPTY_WAIT);
  } else if (warp == 3) {
    // ---- value rows between the last key and the next multiple of 16: whatever the cache holds there must not meet a weight of zero
    PuUnit u;
    uint32_t used = 0;                 // phases of v_raw
    bool ok = true;
    for (int i = 0; i < n && ok;) {
      u = pu_locate(p, l, f0 + i);
      const int end = i + u.tiles - u.tile;           // behind the unit's last tile
      if (end <= n && (u.last & 15)) {
        const int r = 2 * (end - 1) + 1, slot = r % kPuRing;
        ok = mbar_wait_spin(&v_raw[slot], (used >> slot) & 1u);
        used ^= 1u << slot;
        if (!ok) break;
        uint8_t* at = kv_s + slot * kPuTile;
        const int rows = 16 - (u.last & 15);
        for (int k = lane; k < 2 * rows * 8; k += 32) {               // (a row's 128 bytes of either box, whatever their order)
          const int box = (k >> 3) & 1, row = u.last + (k >> 4);
          *reinterpret_cast<uint4*>(at + box * kPfBox + row * 128 + 16 * (k & 7)) = make_uint4(0u, 0u, 0u, 0u);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&kv_full[slot]);
      }
      i = end;
    }
    if (!ok) give_up(DERR_EMPTY_WAIT);
    __syncwarp();
  } else if (warp == 1) {
    // ---- products: the scores of a tile, then the weighted values of the tile before
    const bool leader = elect_one();
    const uint32_t idesc_o = umma_idesc_bf16(kPaDim) | (1u << 16);     // (bit 16: B is N-major)
    const uint64_t qd = umma_desc_sw128(q_s), kd = umma_desc_sw128(kv_s), vd = pf_desc_mn(kv_s);
    uint32_t q_seen = 0;
    int made[2] = {0, 0}, freed[2] = {0, 0};          // tiles of a parity so far, results read
    bool ok = true;
    PuUnit u, before;
    bool fresh[2] = {true, true}, before_fresh = false;                // the parity's next tile is its first of the unit
    auto values = [&](int i, const PuUnit& w, bool first) {
      const int x = (f0 + i) & 1, r = 2 * i + 1, slot = r % kPuRing;
      const uint32_t s_t = tmem + (uint32_t)(x * 256), o_t = s_t + 128u;
      bool good = mbar_wait_spin(&kv_full[slot], (uint32_t)((r / kPuRing) & 1)) && mbar_wait_spin(&p_full[x], (uint32_t)(made[x] & 1));
      ++made[x];
      if (good && first) {
        good = freed[x] == 0 || mbar_wait_spin(&o_free[x], (uint32_t)((freed[x] - 1) & 1));
        ++freed[x];
      }
      if (!good) return false;
      tc_fence_after();
      if (leader) {
        const int steps = w.tile == w.tiles - 1 ? (w.last + 15) >> 4 : 8;
        const uint64_t at = vd + (uint64_t)(slot * (kPuTile >> 4));
        for (int k = 0; k < steps; ++k) umma_f16_ts(o_t, s_t + 8u * k, at + (uint64_t)(k * (2048 >> 4)), idesc_o, !first || k != 0);
        if (TERMS == 2 || w.rows <= 32)
          for (int k = 0; k < steps; ++k) umma_f16_ts(o_t, s_t + 64u + 8u * k, at + (uint64_t)(k * (2048 >> 4)), idesc_o, 1u);
        umma_commit(&o_done[x]);
        umma_commit(&kv_empty[slot]);
      }
      __syncwarp();
      return true;
    };
    for (int i = 0; i < n && ok; ++i) {
      const int x = (f0 + i) & 1, r = 2 * i, slot = r % kPuRing;
      if (i == 0 || ++u.tile == u.tiles) {
        u = pu_locate(p, l, f0 + i);
        fresh[0] = fresh[1] = true;
        ok = mbar_wait_spin(&q_full[u.q_slot], (q_seen >> u.q_slot) & 1u);
        q_seen ^= 1u << u.q_slot;
      }
      // (the scores' columns hold the weights of the parity's tile before until its products are done)
      ok = ok && mbar_wait_spin(&kv_full[slot], (uint32_t)((r / kPuRing) & 1)) && (made[x] == 0 || mbar_wait_spin(&o_done[x], (uint32_t)((made[x] - 1) & 1)));
      if (!ok) break;
      tc_fence_after();
      if (leader) {
        const uint32_t s_t = tmem + (uint32_t)(x * 256);
        const uint32_t idesc_s = umma_idesc_bf16(u.tile == u.tiles - 1 ? (u.last + 15) & ~15 : kPfTile);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t off = (uint32_t)((k >> 2) * (kPfBox >> 4) + 2 * (k & 3));
          umma_f16(s_t, qd + off, kd + (uint32_t)(slot * (kPuTile >> 4)) + off, idesc_s, k != 0);
        }
        umma_commit(&s_full[x]);
        umma_commit(&kv_empty[slot]);
        if (i == n - 1 || u.tile == u.tiles - 1)
          for (int j = 0; j < 4; ++j)
            if (u.pre || j == u.q_slot) umma_commit(&q_empty[j]);
      }
      __syncwarp();
      const bool first = fresh[x];
      fresh[x] = false;
      if (i > 0) ok = values(i - 1, before, before_fresh);
      before = u;
      before_fresh = first;
    }
    if (ok && n > 0) ok = values(n - 1, before, before_fresh);
    if (!ok) give_up(DERR_FULL_WAIT);
  } else if (warp >= 4) {
    // ---- softmax of the tiles of a parity.  More than 32 rows: a thread per row.  Up to 32: the queries stand in all four quarters of the tensor
    // memory's lanes, and a warp takes 32 of the tile's keys for them (weights of zero for the others), so that a thread has 32 scores instead of 128.
    const int x = (warp - 4) >> 2, q4 = warp & 3;
    const uint32_t s_t = tmem + ((uint32_t)(32 * q4) << 16) + (uint32_t)(x * 256), o_t = s_t + 128u;
    float* stage = stage_s + x * (kPuStage / 4);
    float m = -FLT_MAX, l_sum = 0.f;
    bool ok = true, first = true;
    int done = 0;                      // tiles of this parity
    PuUnit u;
    int unit_end = 0;                  // the tile behind the unit's last, or the CTA's
    for (int i = (f0 & 1) == x ? 0 : 1; i < n && ok; i += 2) {
      if (i >= unit_end) {
        u = pu_locate(p, l, f0 + i);
        unit_end = min(n, i + u.tiles - u.tile);
        first = true;
        m = -FLT_MAX;
        l_sum = 0.f;
      } else {
        u.tile += 2;
      }
      const bool quarter = u.rows <= 32;
      const int r = quarter ? lane - (u.pre ? 0 : 8 * u.q_slot) : 32 * q4 + lane;
      const bool live = r >= 0 && r < u.rows;
      ok = __all_sync(0xffffffffu, mbar_wait_spin(&s_full[x], (uint32_t)(done & 1)));
      if (!ok) break;
      tc_fence_after();
      auto rescale = [&](float mx) {                   // (the products so far are done: these scores were asked for after them)
        const bool grown = live && mx > m;
        if (first) {
          m = mx;
        } else if (__any_sync(0xffffffffu, grown)) {
          const float to = grown ? mx : m, f = ex2(m - to);
#pragma unroll 1
          for (int c = 0; c < kPaDim; c += 32) {
            float o[32];
            pf_ld32(o_t + (uint32_t)c, o);
            uint32_t w0[16], w1[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              w0[j] = __float_as_uint(o[j] * f);
              w1[j] = __float_as_uint(o[16 + j] * f);
            }
            tmem_st16(o_t + (uint32_t)c, w0);
            tmem_st16(o_t + (uint32_t)c + 16u, w1);
          }
          l_sum *= f;
          m = to;
        }
      };
      if (quarter) {
        const int keys = min(max((u.tile == u.tiles - 1 ? u.last : kPfTile) - 32 * q4, 0), 32);
        float v[32];
        pf_ld32(s_t + 32u * q4, v);
        float mx = -FLT_MAX;
#pragma unroll
        for (int j = 0; j < 32; ++j) mx = fmaxf(mx, j < keys ? v[j] : -FLT_MAX);
        rescale(mx == -FLT_MAX ? mx : mx * p.scale_log2);
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float w0 = 2 * j < keys ? ex2(fmaf(v[2 * j], p.scale_log2, -m)) : 0.f, w1 = 2 * j + 1 < keys ? ex2(fmaf(v[2 * j + 1], p.scale_log2, -m)) : 0.f;
          sum[j & 3] += w0 + w1;
          split_bf16(w0, w1, hi[j], lo[j]);
        }
        l_sum += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        uint32_t zero[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) zero[j] = 0u;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (q == q4) {
            tmem_st16(s_t + 16u * q, hi);
            tmem_st16(s_t + 64u + 16u * q, lo);
          } else {
            tmem_st16(s_t + 16u * q, zero);
            tmem_st16(s_t + 64u + 16u * q, zero);
          }
        }
      } else {
        float mx = -FLT_MAX;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v[32];
          pf_ld32(s_t + 32u * c, v);
#pragma unroll
          for (int j = 0; j < 32; ++j) mx = fmaxf(mx, v[j]);
        }
        rescale(mx == -FLT_MAX ? mx : mx * p.scale_log2);
        uint32_t low[TERMS == 2 ? 64 : 1];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v[32];
          pf_ld32(s_t + 32u * c, v);
          uint32_t w[16];
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float w0 = ex2(fmaf(v[2 * j], p.scale_log2, -m)), w1 = ex2(fmaf(v[2 * j + 1], p.scale_log2, -m));
            sum[j & 3] += w0 + w1;
            if constexpr (TERMS == 2) split_bf16(w0, w1, w[j], low[16 * c + j]);
            else w[j] = pack_bf16(w0, w1);
          }
          l_sum += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          tmem_st16(s_t + 16u * c, w);                 // over scores that this thread has read
        }
        if constexpr (TERMS == 2)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t w[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = low[16 * c + j];
            tmem_st16(s_t + 64u + 16u * c, w);
          }
      }
      first = false;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[x]);
      ++done;
      if (i + 2 < unit_end) continue;

      // ---- the piece's result
      ok = __all_sync(0xffffffffu, mbar_wait_spin(&o_done[x], (uint32_t)((done - 1) & 1)));
      if (!ok) break;
      tc_fence_after();
      const size_t row0 = (size_t)u.slot + (size_t)(u.pre ? 128 : 8) * blockIdx.x;
      float *to_o = u.pre ? pp.pre_o : pp.own_o, *to_ml = u.pre ? pp.pre_ml : pp.own_ml;
      if (!quarter) {
        float* o_row = to_o + ((row0 + r) * 2 + x) * kPaDim;
#pragma unroll 1
        for (int c = 0; c < kPaDim; c += 32) {
          float o[32];
          pf_ld32(o_t + (uint32_t)c, o);
          if (live)
#pragma unroll
            for (int j = 0; j < 8; ++j) reinterpret_cast<float4*>(o_row + c)[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
        }
        if (live) *reinterpret_cast<float2*>(to_ml + ((row0 + r) * 2 + x) * 2) = make_float2(m, l_sum);
      } else {
        // the four warps' parts of a row meet here: their maxima and sums, then 16 or 64 columns at a time
        auto meet = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1 + x) : "memory"); };
        if (live) {
          stage[(4 * r + q4) * 2] = m;
          stage[(4 * r + q4) * 2 + 1] = l_sum;
        }
        meet();
        float top = -FLT_MAX, all = 0.f;
        if (live) {
#pragma unroll
          for (int w = 0; w < 4; ++w) top = fmaxf(top, stage[(4 * r + w) * 2]);
#pragma unroll
          for (int w = 0; w < 4; ++w) all += stage[(4 * r + w) * 2 + 1] * ex2(stage[(4 * r + w) * 2] - top);
          if (q4 == 0) *reinterpret_cast<float2*>(to_ml + ((row0 + r) * 2 + x) * 2) = make_float2(top, all);
        }
        const float f = ex2(m - top);
        const int t = (int)(threadIdx.x & 127);
        meet();
        if (u.rows <= 8) {
          constexpr int kLd = 65;                      // [warp][8 rows][64 columns]
#pragma unroll 1
          for (int c = 0; c < kPaDim; c += 64) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float o[32];
              pf_ld32(o_t + (uint32_t)(c + 32 * h), o);
              if (live)
#pragma unroll
                for (int j = 0; j < 32; ++j) stage[(q4 * 8 + r) * kLd + 32 * h + j] = o[j] * f;
            }
            meet();
            for (int k = t; k < u.rows * 64; k += 128) {
              const int row = k >> 6, col = k & 63;
              float sum = 0.f;
#pragma unroll
              for (int w = 0; w < 4; ++w) sum += stage[(w * 8 + row) * kLd + col];
              to_o[((row0 + row) * 2 + x) * kPaDim + c + col] = sum;
            }
            meet();
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < kPaDim; c += 16) {
            float o[16];
            tmem_ld16(o_t + (uint32_t)c, o);
            if (live)
#pragma unroll
              for (int j = 0; j < 16; ++j) stage[(q4 * 32 + r) * kPuStageLd + j] = o[j] * f;
            meet();
            for (int k = t; k < u.rows * 16; k += 128) {
              const int row = k >> 4, col = k & 15;
              float sum = 0.f;
#pragma unroll
              for (int w = 0; w < 4; ++w) sum += stage[(w * 32 + row) * kPuStageLd + col];
              to_o[((row0 + row) * 2 + x) * kPaDim + c + col] = sum;
            }
            meet();
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_free[x]);
    }
    if (!ok) give_up(DERR_TMEM);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// Joins the pieces of a query head: a warp per head, four columns a lane.
__global__ void __launch_bounds__(128) paged_join_kernel(const PuParams pp, int n_ctas) {
  pdl_wait();
  pdl_launch_dependents();
  const PagedParams& p = pp.a;
  const int b = blockIdx.x, lane = threadIdx.x & 31;
  const PuSeqPlan q = pp.plan[b];
  const int total = *pp.plan_total;
  for (int head = (int)(blockIdx.y * 4 + (threadIdx.x >> 5)); head < p.n_heads; head += gridDim.y * 4) {
    const int kv = head / p.group, h = head - kv * p.group;
    // tiles of the list, first CTA and number of (CTA, parity) places of the own and of the shared part
    int f[2], e[2], c[2], places[2];
    f[0] = q.own_f + kv * q.own_tiles;
    e[0] = f[0] + q.own_tiles;
    f[1] = q.pre_f + kv * q.pre_kv;
    e[1] = f[1] + q.pre_tiles;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      c[k] = places[k] = 0;
      if (e[k] > f[k]) {
        c[k] = (int)(((long long)(f[k] + 1) * n_ctas - 1) / total);
        places[k] = 2 * ((int)(((long long)e[k] * n_ctas - 1) / total) - c[k] + 1);
      }
    }
    const size_t own_row = (size_t)(b * p.n_kv + kv) * p.group + h, pre_row = (size_t)q.pre_row + (size_t)kv * q.pre_row_kv + h;
    const int all = places[0] + places[1];
    // place i: its row of the partial results, or none
    auto row_of = [&](int i, bool& pre) -> long long {
      pre = i >= places[0];
      const int k = pre, j = pre ? i - places[0] : i, cta = c[k] + (j >> 1), x = j & 1;
      const int lo = max(f[k], (int)((long long)total * cta / n_ctas)), hi = min(e[k], (int)((long long)total * (cta + 1) / n_ctas));
      if (hi - lo < 1 || (hi - lo == 1 && (lo & 1) != x)) return -1;
      return (long long)(((pre ? pre_row : own_row) + (size_t)(pre ? 128 : 8) * cta) * 2 + x);
    };
    float top = -FLT_MAX;
    for (int i = lane; i < all; i += 32) {
      bool pre;
      const long long r = row_of(i, pre);
      if (r >= 0) top = fmaxf(top, (pre ? pp.pre_ml : pp.own_ml)[2 * r]);
    }
    top = warp_max(top);
    float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < all; ++i) {
      bool pre;
      const long long r = row_of(i, pre);
      if (r < 0) continue;
      const float2 ml = *reinterpret_cast<const float2*>((pre ? pp.pre_ml : pp.own_ml) + 2 * r);
      const float4 v = *reinterpret_cast<const float4*>((pre ? pp.pre_o : pp.own_o) + r * kPaDim + 4 * lane);
      const float w = ex2(ml.x - top);
      l += ml.y * w;
      o[0] = fmaf(v.x, w, o[0]);
      o[1] = fmaf(v.y, w, o[1]);
      o[2] = fmaf(v.z, w, o[2]);
      o[3] = fmaf(v.w, w, o[3]);
    }
    const size_t at = ((size_t)b * p.n_heads + head) * kPaDim + 4 * lane;
    if (__any_sync(0xffffffffu, o[0] != o[0] || o[1] != o[1] || o[2] != o[2] || o[3] != o[3])) {
      // An infinite value times a weight of zero, in the quarters that do not have its key, is no number, though the sum may be infinite: once more,
      // key by key.
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
  PuParams pp;
  pp.per_tile = 128 / p.group;
  pp.per_quarter = 32 / p.group;
  const size_t tiles = batch * (((size_t)p.max_len + kPfTile - 1) / kPfTile) * n_kv_heads;
  TQ_REQUIRE(ctx, tiles < (1ull << 30) && (size_t)p.n_pages * pages->page_rows < (1ull << 31), "tq_gqa_decode_paged: too many positions");
  const size_t n_ctas = tiles < (size_t)ctx->sm_count ? tiles : (size_t)ctx->sm_count;
  // partial results, the sequences' plans
  const size_t own_rows = (batch * n_heads + 8 * n_ctas) * 2, pre_rows = p.n_groups ? (batch * n_heads + 128 * n_ctas) * 2 : 0;
  const size_t floats = (own_rows + pre_rows) * (kPaDim + 2);
  if (int st = ensure_scratch(ctx, floats * sizeof(float) + (batch + 1) * sizeof(PuSeqPlan))) return st;
  pp.own_o = static_cast<float*>(ctx->scratch);
  pp.pre_o = pp.own_o + own_rows * kPaDim;
  pp.own_ml = pp.pre_o + pre_rows * kPaDim;
  pp.pre_ml = pp.own_ml + own_rows * 2;
  pp.plan = reinterpret_cast<PuSeqPlan*>(pp.pre_ml + pre_rows * 2);
  pp.plan_total = reinterpret_cast<int*>(pp.plan + batch);
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
  TQ_CUDA(ctx, launch_k(ctx, paged_join_kernel, dim3((unsigned)batch, (unsigned)((n_heads + 3) / 4)), dim3(128), 0, pp, (int)n_ctas));
  return TQ_OK;
}
