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
// Units, tiles, runs, pieces.  A unit is what meets the same keys: the rows (member, query head of one KV head) of up to 128 / group members of a group
// over the group's shared positions, in whole tiles of 128, or one sequence's query heads over the rest.  The tiles of all units of a KV head stand in
// two lists, one of shared and one of own tiles, and every CTA, one an SM, takes a share of either: as many tiles of the one and of the other as everybody
// else.  CTAs that stand at the same place of the KV heads' lists are neighbours: a cache row holds all heads, and its 256 bytes a head are fetched at the
// same time.  A run is what a share has of a unit; a long one is cut into pieces (kPuWindow).  A piece's odd and even tiles belong to different softmax
// groups, which take scores from the run's one reference, so that the products of both go to the same columns (two sets of columns, for pieces that follow
// one another).  A run leaves a partial result, to which each of its pieces adds; a second kernel joins those of a row, in the order of the list.
// (64 sequences of 2048 positions and 8 KV heads take 97 us.  One list of all heads' tiles, cut for 148 CTAs rather than 144, took 98 us.  Shorter shares,
// handed out as CTAs get to them because SMs differ in speed by a fifth, took 102: they make more partial results than they balance.)
//
// What bounds it: the bytes of the cache, once, where sequences are long (537 MB in 97 us, 5.5 TB/s; the steady state is 2800 cycles for a tile of 64 KB,
// which is an SM's share of the memory's rate); beside them a start of 5 us (lengths, plan, first pages, first tile: six loads in a row) and 4 us until the
// second kernel is through, which are most of a small call (one sequence of 700 positions 8.5 us, 8 samples of a prompt of 2040 16.0, of which 5.5 come with
// the first shared tile: queries, the first instructions of that path and 128 rows to read out).  A shared tile of 128 rows is a product for the scores and
// two for the weights' terms, of two softmax groups in turn, and 64 KB from L2 (64 samples with 512 positions of their own: 35.5 us behind a prompt of
// 2048, 38.7 of 4096, 45.0 of 8192).
// ---------------------------------------------------------------------------------------------
constexpr int kPuThreads = 416;
constexpr int kPuTile = 4 * kPfBox / 2;               // bytes of 128 rows of keys or values
constexpr int kPuRing = 5;
constexpr int kPuWeights = 2 * 32 * 128;              // a parity's weights where keys are the lanes: three terms of eight rows (32 columns) of 128 keys, in two halves
constexpr int kPuOnes = 1024;                         // eight rows of 64 ones
constexpr int kPuMeet = (2 + 2) * 128 * 4;            // maxima [parity][warp][row], references [run's parity][row, or warp and row]
constexpr float kPuLargest = 7.9228162514264338e28f;  // 2^96: a weight above it is too far from its reference
constexpr int kPuHeader = 640;                        // barriers, pieces
constexpr int kPuReaders = 12;                        // warps that are told the pieces
constexpr int kPuPieces = 4;                          // pieces that are told ahead
// Tiles of a piece, own and shared ones, for f32 and for bf16 results: the tensor core truncates what it adds up, about 4e-9 of a sum for a position (64
// sequences of 16384 positions in one piece each, with values of one sign, were off by 7e-5).  f32 results of 64 sequences of up to 2048 positions: error
// from 64 bits 1.9e-6 in pieces of 16 tiles, 1.2e-6 in pieces of 8 (the attention over slots 1.4e-6, f32 arithmetic 0.9e-6), 56.6 and 57.8 us; 64 samples of a
// prompt of 8192, whose shared tiles add both terms of a weight to the same sums, 3.6e-6 in pieces of 8 tiles, 2.8e-6 in pieces of 4, 36.9 and 42.5 us.
// Powers of two; only a run's first piece has another number, 1 more at most and 2 at least: so the last tiles of a run's pieces have the same parity, and
// a thread that adds to a partial result adds to what it wrote itself.
constexpr int kPuWindow[2][2] = {{8, 4}, {128, 128}};
__device__ __forceinline__ int pu_piece(int left, int window) { return left <= window + 1 ? left : ((left - 2) & (window - 1)) + 2; }
// f32 results: groups of up to so many rows are attended by eight rows at a time, keys as the lanes, with three terms of a weight; more rows than that read the
// same tiles too often.  16 rows: 16 groups of four samples 39.5 -> 40.6 us and 1.9e-6 -> 0.9e-6 of error from 64 bits, four groups behind prompts of 8192
// 31.1 -> 34.5 and 2.7e-6 -> 0.8e-6; 32 rows: 8 groups behind prompts of 2040 41.8 -> 61.1 for 2.6e-6 -> 0.8e-6; 64 rows: 40.6 -> 97.8.
constexpr int kPuFewRows = 16;
constexpr int kPuBatch = 1024;                        // sequences of a call
constexpr size_t kPuFixed = 2 * (size_t)kPfBox + kPuRing * (size_t)kPuTile + 2 * (size_t)kPuWeights + kPuOnes + kPuMeet + kPuHeader;

// In shared memory, behind the buffers.
struct PuPlan {
  int *own, *last, *pre;                              // [batch + 1] own tiles of the sequences before; [batch] shared tiles << 8 | keys of the last tile - 1;
                                                      // [groups + 1] units' shared tiles of the groups before
  int batch, groups, group, per_tile, per_eight, few;
  __device__ __forceinline__ int unit(int members) const { return members <= few ? per_eight : per_tile; }      // members of a unit of such a group
  int share[2];                                       // own, shared tiles of a CTA
};
// What the kernel that joins the pieces has to know: where a sequence's tiles stand in a KV head's list.
struct PuSeqPlan {
  int own_f, own_tiles, pre_f, pre_tiles;
};
struct PuUnit {
  int b0, head, rows, tiles, tile, shared_tiles, last;  // b0: (first) sequence of the batch; head: whose pages; tile: the asked one; last: keys of the last
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
// Tile f of a KV head's shared (pre) or own tiles.
__device__ __forceinline__ PuUnit pu_locate(const PagedParams& p, const PuPlan& l, bool pre, int f) {
  PuUnit u;
  if (pre) {
    const int g = pu_last_not_above(l.pre, l.groups, f), start = pu_group_start(p, g), members = pu_group_end(p, g, start) - start;
    u.tiles = l.last[start] >> 8;
    const int rest = f - l.pre[g], rt = rest < u.tiles ? 0 : rest / u.tiles;
    u.tile = rest - rt * u.tiles;
    u.b0 = start + rt * l.unit(members);
    u.head = start;                    // the group's first member
    u.rows = min(l.unit(members), members - rt * l.unit(members)) * l.group;
    u.shared_tiles = 0;
    u.last = kPfTile;
  } else {
    const int b = pu_last_not_above(l.own, l.batch, f);
    u.tiles = l.own[b + 1] - l.own[b];
    u.tile = f - l.own[b];
    u.b0 = u.head = b;
    u.rows = l.group;
    u.shared_tiles = l.last[b] >> 8;
    u.last = (l.last[b] & 255) + 1;
  }
  return u;
}
// A piece as the roles are told of it, in shared memory.
struct __align__(16) PuPiece {
  int n, tile, last, rows;                            // tiles (0: there are no more pieces), the first one's place in the sequence, keys of the last one, rows
  int kv, b0, seq, out;                               // KV head, (first) sequence of the batch, its row of the tables; first row of its run's partial results
  int what, pad[3];                                   // bits: see below
  __device__ __forceinline__ bool pre() const { return what & 1; }                 // of shared tiles
  __device__ __forceinline__ bool keyed() const { return what & 2; }               // the keys are the lanes
  __device__ __forceinline__ bool later() const { return what & 4; }               // not its run's first piece
  __device__ __forceinline__ bool more() const { return what & 8; }                // not its run's last piece
  __device__ __forceinline__ int run() const { return (what >> 4) & 1; }           // the run's parity
  __device__ __forceinline__ uint32_t phase() const { return (uint32_t)what >> 5; }       // and that of the runs before with the same
};
// Places in the ring, in the order in which they are needed: keys 0, keys 1, values 0, keys 2, values 1 ..
__device__ __forceinline__ int pu_keys_at(int t) { return t == 0 ? 0 : 2 * t - 1; }
__device__ __forceinline__ int pu_values_at(int t) { return 2 * t + 2; }

struct PuParams {
  PagedParams a;
  int per_tile, per_eight, few, n_shares;             // members of a row tile; of eight rows; of a group that is attended by eight rows; CTAs of a KV head
  int window[2];                                      // own, shared tiles of a piece
  float *own_o, *own_ml, *pre_o, *pre_ml;             // partial results: [row][128], [row][2] references and sums (of the groups)
  PuSeqPlan* plan;                                    // [batch]
  int* share;                                         // [2]
};

template <typename F>
__device__ __forceinline__ void pu_scan(int* a, int n, int lane, F value) {      // a[i] becomes the sum of the values before i, a[n] the whole; one warp
  int sum = 0;
  for (int base = 0; base < n; base += 32) {
    const int v = base + lane < n ? value(base + lane) : 0;
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

__device__ __forceinline__ float redux_max(float v) {                  // of the warp's values; NaN is none of them
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ void st_global8(float* to, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
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

// LONG: there may be runs of several pieces.  (The form without has less code to fetch: one sequence of 700 positions 9.4 us, with it 9.8.)
template <bool LONG>
__global__ void __launch_bounds__(kPuThreads, 1)
paged_decode_kernel(const __grid_constant__ CUtensorMap q_eight, const __grid_constant__ CUtensorMap q_whole,
                    const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const __grid_constant__ PuParams pp) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];   // (the swizzled buffers come first)
  const PagedParams& p = pp.a;
  uint8_t *q_s = smem_raw, *kv_s = q_s + 2 * kPfBox;
  uint8_t* w_s = kv_s + kPuRing * kPuTile;            // [parity]
  uint8_t* ones_s = w_s + 2 * kPuWeights;
  float* meet_s = reinterpret_cast<float*>(ones_s + kPuOnes);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(meet_s + kPuMeet / 4);  // [4]
  uint64_t* q_empty = q_full + 4;                     // [4]
  uint64_t* kv_full = q_empty + 4;                    // [ring]
  uint64_t* kv_empty = kv_full + kPuRing;
  uint64_t* v_raw = kv_empty + kPuRing;               // [ring] values of a last tile, before the rows behind the last key are zeroed
  uint64_t* s_full = v_raw + kPuRing;                       // [parity]
  uint64_t* p_full = s_full + 2;
  uint64_t* o_done = p_full + 2;
  uint64_t* o_free = o_done + 2;
  uint64_t* piece_full = o_free + 2;                  // [kPuPieces]
  uint64_t* piece_empty = piece_full + kPuPieces;
  uint64_t* met = piece_empty + kPuPieces;            // [parity] the four warps of a softmax group
  uint64_t* ref_full = met + 2;                       // [run's parity]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ref_full + 2);
  volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);
  PuPiece* piece_s = reinterpret_cast<PuPiece*>(q_full) + (kPuHeader / sizeof(PuPiece) - kPuPieces);
  PuPlan l;
  l.own = reinterpret_cast<int*>(q_full) + kPuHeader / 4;
  l.last = l.own + p.batch + 1;
  l.pre = l.last + p.batch;
  l.batch = p.batch;
  l.group = p.group;
  l.per_tile = pp.per_tile;
  l.per_eight = pp.per_eight;
  l.few = pp.few;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < 4; ++i) {
        mbar_init(&q_full[i], 1);
        mbar_init(&q_empty[i], 1);
      }
      for (int i = 0; i < kPuPieces; ++i) {
        mbar_init(&piece_full[i], 1);
        mbar_init(&piece_empty[i], kPuReaders);
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
        mbar_init(&ref_full[x], 4);
      }
      *failed = 0;
      mbar_init_fence();
    }
  } else if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
  } else if (warp == 3) {
    if (lane == 0) {
      prefetch_map(&q_eight);
      prefetch_map(&k_map);
      prefetch_map(&v_map);
    }
    for (int i = lane; i < kPuOnes / 16; i += 32) reinterpret_cast<uint4*>(ones_s)[i] = make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  tc_fence_before();
  pdl_wait();
  pdl_launch_dependents();
  auto give_up = [&](int code) { atomicCAS(p.err, 0, code); };
  auto abandon = [&](int code) {
    give_up(code);
    *failed = 1;
  };
  if (threadIdx.x == 0 && (smem_u32(smem_raw) & 1023)) give_up(DERR_TMEM);

  // ---- the plan: every CTA makes it for itself
  // (what is read of the groups is on its way before the sequences' lengths, which two loads in a row bring)
  bool bad = false;                    // starts that do not ascend from 0: nothing is shared, and the status word says why
  for (int g = threadIdx.x; g < p.n_groups; g += kPuThreads) {
    const int start = p.group_starts[g], next = g + 1 < p.n_groups ? p.group_starts[g + 1] : p.batch;
    l.pre[g] = min(max(p.shared[g], 0), p.max_shared);
    bad = bad || start < 0 || start > next || next > p.batch || (g == 0 && start != 0);
  }
  for (int b = threadIdx.x; b < p.batch; b += kPuThreads) {
    const int s = paged_row_of(p, b);
    if (s < 0 && blockIdx.x == 0) give_up(DERR_PAGE_LIST);
    l.own[b] = s < 0 ? 0 : min(max(p.lens[s], 0), p.max_len);
    l.last[b] = 0;
  }
  bad = __syncthreads_or(bad);
  if (bad && threadIdx.x == 0 && blockIdx.x == 0) give_up(DERR_PAGE_LIST);
  l.groups = bad ? 0 : p.n_groups;
  for (int g = warp; g < l.groups; g += kPuThreads / 32) {
    // no more than the shortest member has, in whole tiles
    const int start = pu_group_start(p, g), end = pu_group_end(p, g, start), members = end - start;
    int least = l.pre[g];
    for (int b = start + lane; b < end; b += 32) least = min(least, l.own[b]);
    least = __reduce_min_sync(0xffffffffu, least);
    const int tiles = members > 1 ? least / kPfTile : 0;
    for (int b = start + lane; b < end; b += 32) l.last[b] = tiles << 8;
    if (lane == 0) l.pre[g] = members <= l.unit(members) ? tiles : tiles * ((members + l.unit(members) - 1) / l.unit(members));
  }
  if (l.groups) __syncthreads();
  if (warp == 0)
    pu_scan(l.own, p.batch, lane, [&](int b) {
      const int len = l.own[b], shared = l.last[b] >> 8, tiles = (len + kPfTile - 1) / kPfTile;
      l.last[b] |= tiles > shared ? len - 1 - (tiles - 1) * kPfTile : 0;
      return tiles - shared;
    });
  if (warp == 1) pu_scan(l.pre, l.groups, lane, [&](int g) { return l.pre[g]; });
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int pre_tiles = l.pre[l.groups], own_tiles = l.own[p.batch];
#pragma unroll
  for (int k = 0; k < 2; ++k) l.share[k] = max(1, ((k ? pre_tiles : own_tiles) + pp.n_shares - 1) / pp.n_shares);
  // One arrival for the warp.  The lanes meet before it and behind it: none may wait for what the arrival lets happen before it is made.
  auto arrive = [&](uint64_t* bar) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
    __syncwarp();
  };
  // ---- pieces, as warp 12 tells them
  int told = 0;
  auto take = [&](bool& ok, PuPiece& w) {
    const int slot = told % kPuPieces;
    ok = __all_sync(0xffffffffu, ok && mbar_wait_spin(&piece_full[slot], (uint32_t)((told / kPuPieces) & 1)));
    if (ok) w = piece_s[slot];
    else w.n = 0;
    arrive(&piece_empty[slot]);
    ++told;
  };

  if (warp == 12) {
    // ---- what to do: the CTA's two shares, in pieces
    bool ok = true;
    auto tell = [&](const PuPiece& w) {
      const int slot = told % kPuPieces;
      ok = __all_sync(0xffffffffu, ok && mbar_wait_spin(&piece_empty[slot], (uint32_t)((told / kPuPieces) & 1) ^ 1u));
      if (lane == 0) {
        piece_s[slot] = w;
        mbar_arrive(&piece_full[slot]);
      }
      __syncwarp();
      ++told;
    };
    const int cta = (int)blockIdx.x / p.n_kv;            // of the KV head
    PuPiece w{};
    w.kv = (int)blockIdx.x - cta * p.n_kv;
    // Own tiles first where there are several shared ones: the first burst of copies is the own tiles', which only one CTA reads, and shared ones find the
    // other heads' rows in L2 by the time they are needed (64 samples by fours 59.2 us, the other way 60.4; one prefix 44.9 and 46.6; but 8 samples with a
    // shared tile a CTA 16.6 and 16.0).
    const bool own_first = l.share[1] > 1;
    int run = 0;
#pragma unroll 1
    for (int turn = 0; turn < 2 && ok; ++turn) {
      const int k = (turn == 0) != own_first;            // 1: shared tiles
      const int share = k ? l.share[1] : l.share[0], from = share * cta, most = min(from + share, k ? pre_tiles : own_tiles), apart = k ? 128 : 8;
      for (int f = from; f < most && ok;) {
        const PuUnit u = pu_locate(p, l, k, f);
        int left = min(most - f, u.tiles - u.tile);
        f += left;
        const int last = u.tile + left == u.tiles ? u.last : kPfTile;
        w.tile = u.shared_tiles + u.tile;
        w.rows = u.rows;
        w.b0 = u.b0;
        w.seq = max(paged_row_of(p, u.head), 0);
        w.out = w.kv * (p.batch * p.group + apart * pp.n_shares) + u.b0 * p.group + apart * cta;
        w.what = k | (u.rows <= 8) << 1 | (run & 3) << 4;
        for (++run; left > 0 && ok; w.what |= 4, w.tile += w.n) {
          w.n = LONG ? pu_piece(left, pp.window[k]) : left;
          left -= w.n;
          w.what = left > 0 ? w.what | 8 : w.what & ~8;
          w.last = left > 0 ? kPfTile : last;
          tell(w);
        }
      }
    }
    w.n = 0;
    if (ok) tell(w);
    if (!ok) abandon(DERR_EMPTY_WAIT);
  } else if (warp == 0 || warp == 2) {
    // ---- copies: the keys of every tile (warp 0); the queries of every piece and the values of every tile (warp 2).  A lane per box: a page's rows, half
    // their columns.  The warp holds the pages of the next 32 boxes' rows (four tiles or more), and has asked for those behind them.
    const bool values = warp == 2;
    const int box_rows = min(1 << p.page_shift, kPfTile), boxes = kPfTile / box_rows, j = lane >> 1, c = lane & 1;
    uint32_t q_used = 0;               // phases of the query slots
    int own_pieces = 0;
    bool ok = true;
    const int tiles_ahead = 32 / boxes;
    auto pages_from = [&](const PuPiece& w, int i0) {
      const int i = i0 + lane / boxes, row = lane % boxes * box_rows;
      return i < w.n && row < (i == w.n - 1 ? w.last : kPfTile) ? p.tables[(size_t)w.seq * p.table_ld + (((w.tile + i) * kPfTile + row) >> p.page_shift)] : 0;
    };
    PuPiece w, next;
    take(ok, next);
    int pages = 0, ahead = next.n ? pages_from(next, 0) : 0;
    for (int t = 0; next.n && ok;) {
      w = next;
      if (values) {
        const int slot = w.pre() ? 0 : own_pieces++ & 3;
        for (int k = 0; k < 4; ++k)
          if (ok && (w.pre() || k == slot)) {
            ok = __all_sync(0xffffffffu, mbar_wait_spin(&q_empty[k], ((q_used >> k) & 1u) ^ 1u));
            q_used ^= 1u << k;
          }
        if (!ok) break;
        const bool whole = !w.keyed();
        const uint32_t rows = (uint32_t)((whole ? pp.per_tile : pp.per_eight) * p.group);
        if (lane == 0) mbar_arrive_expect_tx(&q_full[slot], 2u * rows * 128u);
        __syncwarp();
        if (lane < 2) tma_load_3d(q_s + c * kPfBox + 16 * slot * 128, whole ? &q_whole : &q_eight, 64 * c, w.kv * p.group, w.b0, &q_full[slot]);
        __syncwarp();
      }
      for (int i = 0; i < w.n && ok; ++i, ++t) {
        const int k = i % tiles_ahead;
        if (k == 0) pages = ahead;
        int page = __shfl_sync(0xffffffffu, pages, k * boxes + min(j, boxes - 1));
        const int keys = i == w.n - 1 ? w.last : kPfTile, used = (keys + box_rows - 1) / box_rows, r = values ? pu_values_at(t) : pu_keys_at(t), slot = r % kPuRing;
        if (j < used && (page < 0 || page >= p.n_pages)) {
          give_up(DERR_POSITION);
          page = 0;
        }
        const int row = (page << p.page_shift) + (((w.tile + i) * kPfTile) & ((1 << p.page_shift) - 1) & ~(box_rows - 1));
        ok = __all_sync(0xffffffffu, ok && mbar_wait_spin(&kv_empty[slot], (uint32_t)((r / kPuRing) & 1) ^ 1u));
        if (!ok) break;
        uint64_t* bar = values && (keys & 15) ? &v_raw[slot] : &kv_full[slot];
        if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(used * box_rows) * 256u);
        __syncwarp();
        if (j < used) tma_load_2d(kv_s + slot * kPuTile + c * kPfBox + j * box_rows * 128, values ? &v_map : &k_map, w.kv * kPaDim + 64 * c, row, bar);
        __syncwarp();
        if (k == 0) {
          if (i + tiles_ahead < w.n) {
            ahead = pages_from(w, i + tiles_ahead);
          } else {
            take(ok, next);
            ahead = next.n ? pages_from(next, 0) : 0;
          }
        }
      }
    }
    if (!ok) abandon(DERR_EMPTY_WAIT);
  } else if (warp == 3) {
    // ---- value rows between the last key and the next multiple of 16: whatever the cache holds there must not meet a weight of zero
    if (blockIdx.x == 0) {             // (before that: what the kernel that joins the pieces has to know)
      for (int b = lane; b < p.batch; b += 32) {
        const int shared = l.last[b] >> 8;
        int pre_f = 0;
        if (shared) {
          int lo = 0, hi = l.groups;   // the group with b: the last that starts there or before
          while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (pu_group_start(p, mid) <= b) lo = mid;
            else hi = mid;
          }
          const int start = pu_group_start(p, lo);
          pre_f = l.pre[lo] + (b - start) / l.unit(pu_group_end(p, lo, start) - start) * shared;
        }
        pp.plan[b] = PuSeqPlan{l.own[b], l.own[b + 1] - l.own[b], pre_f, shared};
      }
      if (lane < 2) pp.share[lane] = lane ? l.share[1] : l.share[0];
      __syncwarp();
    }
    uint32_t used = 0;                 // phases of v_raw
    bool ok = true;
    int t = 0;                         // tiles up to the piece's end
    PuPiece w;
    for (take(ok, w); w.n && ok; take(ok, w)) {
      t += w.n;
      if (!(w.last & 15)) continue;
      const int slot = pu_values_at(t - 1) % kPuRing;
      ok = __all_sync(0xffffffffu, mbar_wait_spin(&v_raw[slot], (used >> slot) & 1u));
      used ^= 1u << slot;
      if (!ok) break;
      uint8_t* at = kv_s + slot * kPuTile;
      const int rows = 16 - (w.last & 15);
      for (int k = lane; k < 2 * rows * 8; k += 32) {             // (a row's 128 bytes of either box, whatever their order)
        const int box = (k >> 3) & 1, row = w.last + (k >> 4);
        *reinterpret_cast<uint4*>(at + box * kPfBox + row * 128 + 16 * (k & 7)) = make_uint4(0u, 0u, 0u, 0u);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      arrive(&kv_full[slot]);
    }
    if (!ok) abandon(DERR_EMPTY_WAIT);
    __syncwarp();
  } else if (warp == 1) {
    // ---- products: the scores of a tile, then the weighted values of the tile before
    const bool leader = elect_one();
    const uint32_t idesc_o = umma_idesc_bf16(kPaDim) | (1u << 16);     // (bit 16: B is N-major; bit 15: A is M-major)
    const uint64_t qd = umma_desc_sw128(q_s), kd = umma_desc_sw128(kv_s), vd = pf_desc_mn(kv_s), wd = umma_desc_sw128(w_s);
    const uint64_t od = umma_desc_sw128(ones_s) & ~((uint64_t)0x3FFF << 32);      // (all groups of eight rows are the same one)
    uint32_t q_seen = 0;
    int made[2] = {0, 0}, freed[2] = {0, 0};          // tiles of a parity so far, pieces of a parity
    bool ok = true;
    struct Tile {
      int steps;                                      // of 16 keys
      bool keyed, first;                                     // of the piece
      int piece;                                      // its parity
    };
    auto values = [&](int t, const Tile& w) {
      const int x = t & 1, r = pu_values_at(t), slot = r % kPuRing;
      const uint32_t s_t = tmem + (uint32_t)(x * 128), o_t = tmem + 256u + (uint32_t)(w.piece * 128);
      bool good = __all_sync(0xffffffffu, mbar_wait_spin(&kv_full[slot], (uint32_t)((r / kPuRing) & 1)) && mbar_wait_spin(&p_full[x], (uint32_t)(made[x] & 1)));
      ++made[x];
      if (good && w.first) {
        good = __all_sync(0xffffffffu, freed[w.piece] == 0 || mbar_wait_spin(&o_free[w.piece], (uint32_t)((freed[w.piece] - 1) & 1)));
        ++freed[w.piece];
      }
      if (!good) return false;
      tc_fence_after();
      if (leader) {
        const uint64_t at = vd + (uint64_t)(slot * (kPuTile >> 4));
        if (w.keyed) {
          const uint32_t idesc = umma_idesc_bf16(32);
          for (int k = 0; k < w.steps; ++k) {
            const uint64_t wk = wd + (uint64_t)(x * (kPuWeights >> 4) + (k >> 2) * (kPuWeights >> 5) + 2 * (k & 3));
            umma_f16(o_t, at + (uint64_t)(k * (2048 >> 4)), wk, idesc | (1u << 15), !w.first || k != 0);
            umma_f16(o_t + 64u, od, wk, idesc, !w.first || k != 0);    // the weights' sums, in every lane
          }
        } else {
          for (int k = 0; k < w.steps; ++k) umma_f16_ts(o_t, s_t + 8u * k, at + (uint64_t)(k * (2048 >> 4)), idesc_o, !w.first || k != 0);
          for (int k = 0; k < w.steps; ++k) umma_f16_ts(o_t, s_t + 64u + 8u * k, at + (uint64_t)(k * (2048 >> 4)), idesc_o, 1u);
        }
        umma_commit(&o_done[x]);
        umma_commit(&kv_empty[slot]);
      }
      __syncwarp();
      return true;
    };
    Tile before{};
    PuPiece w;
    int own_pieces = 0, t = 0, piece = 0;
    for (take(ok, w); w.n && ok; piece ^= 1, take(ok, w)) {
      const int q_slot = w.pre() ? 0 : own_pieces++ & 3;
      ok = __all_sync(0xffffffffu, mbar_wait_spin(&q_full[q_slot], (q_seen >> q_slot) & 1u));
      q_seen ^= 1u << q_slot;
      for (int i = 0; i < w.n && ok; ++i, ++t) {
        const int x = t & 1, r = pu_keys_at(t), slot = r % kPuRing;
        // (the scores' columns hold the weights of the parity's tile before until its products are done)
        ok = __all_sync(0xffffffffu, ok && mbar_wait_spin(&kv_full[slot], (uint32_t)((r / kPuRing) & 1)) &&
                                         (made[x] == 0 || mbar_wait_spin(&o_done[x], (uint32_t)((made[x] - 1) & 1))));
        if (!ok) break;
        tc_fence_after();
        const int keys = i == w.n - 1 ? w.last : kPfTile;
        const Tile now{(keys + 15) >> 4, w.keyed(), i == 0, piece};
        if (leader) {
          const uint32_t s_t = tmem + (uint32_t)(x * 128);
          const uint32_t idesc = umma_idesc_bf16(now.keyed ? 16 : kPfTile);
          const uint64_t kt = kd + (uint64_t)(slot * (kPuTile >> 4)), qt = qd + (uint64_t)(q_slot * (16 * 128 >> 4));
          const uint64_t da = now.keyed ? kt : qt, db = now.keyed ? qt : kt;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint64_t off = (uint64_t)((k >> 2) * (kPfBox >> 4) + 2 * (k & 3));
            umma_f16(s_t, da + off, db + off, idesc, k != 0);
          }
          umma_commit(&s_full[x]);
          umma_commit(&kv_empty[slot]);
          if (i == w.n - 1)
            for (int k = 0; k < 4; ++k)
              if (w.pre() || k == q_slot) umma_commit(&q_empty[k]);
        }
        __syncwarp();
        if (t > 0) ok = values(t - 1, before);
        before = now;
      }
    }
    if (ok && t > 0) ok = values(t - 1, before);
    if (!ok) abandon(DERR_FULL_WAIT);
  } else if (warp >= 4) {
    // ---- softmax of the tiles of a parity.  More than eight rows: S = Q K^T, a thread per row, the weights over the scores' columns.  Up to eight: the keys
    // are the tensor memory's lanes, S^T = K Q^T with 16 columns and O^T = V^T P with 32 (a product of 128 x 128 x 16 takes 84 cycles for four rows too,
    // one of 128 x 16 x 16 a fraction): a thread per key, whose weights go to shared memory, and the weights' sums come from a product with ones.  (Both ways for 9
    // to 32 rows, with two terms of a weight: 16 groups of four samples 41.8 us with keys as lanes and 42.4 with rows, 64 samples by fours 71.6 and 70.4.)
    // A weight is bf16 terms, each the rounding of what those before leave.  Two, within 2^-16 of it as in the attention over slots, where rows are the lanes
    // (one, within 2^-8, would be as far off as the rounding of a bf16 result).  Three, an f32 number's bits, where keys are: their columns are there and cost
    // nothing (8 sequences of up to 700 positions, f32 results: error from 64 bits 1.9e-6 with two, 0.5e-6 with three, 14.2 us both), while a third product of
    // 128 rows does (64 samples of a prompt of 8192 42.5 -> 50.7 us for 2.8e-6 -> 2.1e-6).
    // The reference that scores are taken from is their maximum in the run's first tile, which the group with that tile tells the other one: a bf16 weight
    // may be as large as an f32 one, so that nothing is rescaled; a weight above 2^96 becomes no number, and the joining kernel goes through the row's keys
    // one by one.
    const int x = (warp - 4) >> 2, q4 = warp & 3, t128 = 32 * q4 + lane;
    const uint32_t s_t = tmem + ((uint32_t)(32 * q4) << 16) + (uint32_t)(x * 128);
    uint32_t o_t = 0;                  // of the piece
    float *max_s = meet_s + x * 128, *ref_s = nullptr;                 // [warp][8 rows]; the run's references
    int meetings = 0;
    bool ok = true, first = true, leads = true;      // the group's first tile of the run; it is the piece's first
    int slot = 0;                      // the piece's parity
    auto meet = [&]() {                // (a barrier of the group whose wait ends, as every other's)
      arrive(&met[x]);
      ok = __all_sync(0xffffffffu, ok && mbar_wait_spin(&met[x], (uint32_t)(meetings++ & 1)));
    };
    float ref = 0.f, sum_all = 0.f;    // of the thread's row, and its weights' sum in the run
    int done = 0;                      // tiles of this parity
    PuPiece u{};
    // a tile whose lanes are keys
    auto keyed = [&](bool seen) {
      float v[8];
      __syncwarp();
      tmem_ld8(s_t, v);
      if (first && leads) {
        float mine = -FLT_MAX;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const float mx = redux_max(seen ? v[r] : -FLT_MAX);
          if (lane == r) mine = mx;
        }
        if (lane < 8) max_s[8 * q4 + lane] = mine;
        meet();
        const int r = lane & 7;
        const float mx = fmaxf(fmaxf(max_s[r], max_s[8 + r]), fmaxf(max_s[16 + r], max_s[24 + r]));
        if (lane < 8) ref_s[8 * q4 + lane] = mx == -FLT_MAX ? mx : mx * p.scale_log2;      // (a copy for every warp)
        arrive(&ref_full[u.run()]);
      }
      const float4 f0 = *reinterpret_cast<const float4*>(&ref_s[8 * q4]), f1 = *reinterpret_cast<const float4*>(&ref_s[8 * q4 + 4]);
      if (first) ref = ref_s[8 * q4 + (lane & 7)];
      const float from[8] = {f0.x, f0.y, f0.z, f0.w, f1.x, f1.y, f1.z, f1.w};
      // (rows behind the last one have columns and places too, which nobody reads: without branches the eight go side by side)
      uint8_t* at = w_s + x * kPuWeights + (t128 >> 6) * (kPuWeights / 2) + 2 * (t128 & 7);
      const int chunk = (t128 & 63) >> 3;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const float e = ex2(fmaf(v[r], p.scale_log2, -from[r])), w = !seen ? 0.f : e > kPuLargest ? NAN : e;
        const __nv_bfloat16 hi = __float2bfloat16_rn(w);
        uint8_t* to = at + r * 128 + ((chunk ^ r) << 4);
        const float rest = w - __bfloat162float(hi);
        const __nv_bfloat16 second = __float2bfloat16_rn(rest);
        *reinterpret_cast<__nv_bfloat16*>(to) = hi;
        *reinterpret_cast<__nv_bfloat16*>(to + 1024) = second;
        *reinterpret_cast<__nv_bfloat16*>(to + 2048) = __float2bfloat16_rn(rest - __bfloat162float(second));
      }
      tc_fence_before();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    };
    auto keyed_out = [&](float* to_o, float* to_ml) {
      float o[8], low[2][8], sum[8], sum_low[2][8], was[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) was[r] = LONG && u.later() && r < u.rows ? to_o[r * kPaDim + t128] : 0.f;
      __syncwarp();
      tmem_ld8(o_t, o);
      tmem_ld8(o_t + 8u, low[0]);
      tmem_ld8(o_t + 16u, low[1]);
      tmem_ld8(o_t + 64u, sum);
      tmem_ld8(o_t + 72u, sum_low[0]);
      tmem_ld8(o_t + 80u, sum_low[1]);
      tc_fence_before();
      arrive(&o_free[slot]);                           // (the products of the piece after the next may begin)
      float l = 0.f;                                   // of the lane's row
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        if (r < u.rows) to_o[r * kPaDim + t128] = was[r] + (o[r] + (low[0][r] + low[1][r]));
        if (lane == r) l = sum[r] + (sum_low[0][r] + sum_low[1][r]);
      }
      sum_all = LONG && u.later() ? sum_all + l : l;
      if (!(LONG && u.more()) && q4 == 0 && lane < u.rows) *reinterpret_cast<float4*>(to_ml + lane * 4) = make_float4(ref, sum_all, ref, 0.f);
    };
    int t0 = 0, piece = 0;             // tiles and pieces before the piece
    for (take(ok, u); u.n && ok; t0 += u.n, ++piece, take(ok, u)) {
      const int place = (x - t0) & 1;  // the group's first tile is the piece's first or second
      leads = place == 0;
      slot = piece & 1;
      o_t = tmem + ((uint32_t)(32 * q4) << 16) + 256u + (uint32_t)(slot * 128);
      ref_s = meet_s + 256 + u.run() * 128;
      float *to_o = (u.pre() ? pp.pre_o : pp.own_o) + (size_t)u.out * kPaDim, *to_ml = (u.pre() ? pp.pre_ml : pp.own_ml) + (size_t)u.out * 4;
      for (int i = place; i < u.n && ok; i += 2) {
        first = i == place && !(LONG && u.later());
        const int r = 32 * q4 + lane;
        const bool live = r < u.rows;
        ok = __all_sync(0xffffffffu, mbar_wait_spin(&s_full[x], (uint32_t)(done & 1)) &&
                                         (!first || leads || mbar_wait_spin(&ref_full[u.run()], u.phase())));
        if (!ok) break;
        tc_fence_after();
        if (u.keyed()) {
          keyed(t128 < (i == u.n - 1 ? u.last : kPfTile));
        } else {
          __syncwarp();
          if (first && leads) {
            float mx = -FLT_MAX;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              float v[32];
              pf_ld32(s_t + 32u * c, v);
#pragma unroll
              for (int j = 0; j < 32; ++j) mx = fmaxf(mx, v[j]);
            }
            ref_s[r] = mx == -FLT_MAX ? mx : mx * p.scale_log2;
            arrive(&ref_full[u.run()]);
          }
          if (first) {
            ref = ref_s[r];
            sum_all = 0.f;
          }
          __syncwarp();
          // Weights take the first half of the scores' columns.  Second terms take the other half: quarters in the order 0, 2, 1, 3, so that only three
          // sixteens wait in registers for columns that are read.
          uint32_t keep[3][16];                       // second terms of quarter 0; weights and second terms of quarter 2
#pragma unroll
          for (int step = 0; step < 4; ++step) {
            const int c = step == 1 ? 2 : step == 2 ? 1 : step;
            float v[32];
            pf_ld32(s_t + 32u * c, v);
            uint32_t w[16], low[16];
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float w0 = ex2(fmaf(v[2 * j], p.scale_log2, -ref)), w1 = ex2(fmaf(v[2 * j + 1], p.scale_log2, -ref));
              sum[j & 3] += w0 + w1;
              split_bf16(w0, w1, w[j], low[j]);
            }
            sum_all += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            if (step == 0) {                               // (over scores that this thread has read)
              tmem_st16(s_t, w);
#pragma unroll
              for (int j = 0; j < 16; ++j) keep[0][j] = low[j];
            } else if (step == 1) {
              tmem_st16(s_t + 64u, keep[0]);
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                keep[1][j] = w[j];
                keep[2][j] = low[j];
              }
            } else {
              tmem_st16(s_t + 16u * c, w);
              tmem_st16(s_t + 64u + 16u * c, low);
              if (step == 2) tmem_st16(s_t + 32u, keep[1]);
              else tmem_st16(s_t + 96u, keep[2]);
            }
          }
          tmem_st_wait();
          tc_fence_before();
        }
        arrive(&p_full[x]);
        ++done;
        // (a sum each of the two groups; a run of one tile has one)
        if (!u.keyed() && live && i + 2 >= u.n && !(LONG && u.more())) {
          const float2 ml = make_float2(ref, sum_all > kPuLargest ? NAN : sum_all);
          if (u.n > 1) *reinterpret_cast<float2*>(to_ml + r * 4 + 2 * place) = ml;
          else *reinterpret_cast<float4*>(to_ml + r * 4) = make_float4(ml.x, ml.y, ml.x, 0.f);
        }
        if (i + 1 < u.n) continue;

        // ---- the piece's result, by the group that has its last tile (the same for all pieces of a run)
        ok = __all_sync(0xffffffffu, mbar_wait_spin(&o_done[x], (uint32_t)((done - 1) & 1)));
        if (!ok) break;
        tc_fence_after();
        if (u.keyed()) {
          keyed_out(to_o, to_ml);
        } else {
#pragma unroll 1
          for (int c = 0; c < kPaDim; c += 32) {
            float o[32];
            __syncwarp();
            pf_ld32(o_t + (uint32_t)c, o);
            if (live) {
              float* o_row = to_o + (size_t)r * kPaDim + c;          // (whole sectors: 32 bytes a store)
              if (LONG && u.later())
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                  const float4 was = *reinterpret_cast<const float4*>(o_row + j);
                  o[j] += was.x;
                  o[j + 1] += was.y;
                  o[j + 2] += was.z;
                  o[j + 3] += was.w;
                }
#pragma unroll
              for (int j = 0; j < 32; j += 8) st_global8(o_row + j, &o[j]);
            }
          }
          tc_fence_before();
          arrive(&o_free[slot]);
        }
      }
    }
    if (!ok) abandon(DERR_TMEM);
  }
  tc_fence_before();
  __syncthreads();
  if (*failed && threadIdx.x == 0) {
    // copies and products that are still in flight target this CTA's memories: give them time to land before leaving
    for (int i = 0; i < 10000; ++i) __nanosleep(1000);
  }
  __syncthreads();
  __syncwarp();                        // (the release is one instruction of the whole warp)
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// Joins the partial results of a query head, in their order: a CTA, every fourth result a warp, four columns a lane.  It is launched while the kernel
// above runs and fits beside it (that one is held to 128 registers a thread), so that nothing but loads stands between the last piece and the result.
__global__ void __launch_bounds__(128) paged_join_kernel(const PuParams pp) {
  __shared__ float4 part[4][32];
  __shared__ float2 part_ml[4];
  __shared__ bool again;
  pdl_wait();
  pdl_launch_dependents();
  const PagedParams& p = pp.a;
  const int head = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const PuSeqPlan q = pp.plan[b];
  const int own_share = pp.share[0], pre_share = pp.share[1];
  const int kv = head / p.group, h = head - kv * p.group;
  // CTAs (of the KV head) with the row's own and shared tiles
  const int own_c = q.own_f / own_share, pre_c = q.pre_f / pre_share;
  const int own = q.own_tiles ? (q.own_f + q.own_tiles - 1) / own_share - own_c + 1 : 0, pre = q.pre_tiles ? (q.pre_f + q.pre_tiles - 1) / pre_share - pre_c + 1 : 0;
  float top = -FLT_MAX, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int base = 0; base < own + pre; base += 32) {
    // a lane per partial result: its row, reference and sums
    const int i = base + lane;
    const float* row = nullptr;
    float4 mine = make_float4(-FLT_MAX, 0.f, 0.f, 0.f);
    if (i < own + pre) {
      const bool k = i >= own;
      const int cta = k ? pre_c + i - own : own_c + i, apart = k ? 128 : 8;
      const size_t r = (size_t)kv * (p.batch * p.group + apart * pp.n_shares) + b * p.group + h + (size_t)apart * cta;
      row = (k ? pp.pre_o : pp.own_o) + r * kPaDim;
      mine = *reinterpret_cast<const float4*>((k ? pp.pre_ml : pp.own_ml) + r * 4);
    }
    float4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float* from = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, (unsigned long long)row, 4 * k + warp));
      v[k] = from ? *reinterpret_cast<const float4*>(from + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const float to = fmaxf(top, redux_max(mine.x)), f0 = ex2(top - to), w = ex2(mine.x - to);
    top = to;
    l = l * f0 + warp_sum((mine.y + mine.w) * w);
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] *= f0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float wk = __shfl_sync(0xffffffffu, w, 4 * k + warp);
      o[0] = fmaf(v[k].x, wk, o[0]);
      o[1] = fmaf(v[k].y, wk, o[1]);
      o[2] = fmaf(v[k].z, wk, o[2]);
      o[3] = fmaf(v[k].w, wk, o[3]);
    }
  }
  if (warp) part[warp][lane] = make_float4(o[0], o[1], o[2], o[3]);
  __syncthreads();
  const size_t at = ((size_t)b * p.n_heads + head) * kPaDim + 4 * lane;
  if (warp == 0) {
#pragma unroll
    for (int k = 1; k < 4; ++k) {
      const float4 v = part[k][lane];
      o[0] += v.x;
      o[1] += v.y;
      o[2] += v.z;
      o[3] += v.w;
    }
    const float largest = fmaxf(fmaxf(fabsf(o[0]), fabsf(o[1])), fmaxf(fabsf(o[2]), fabsf(o[3])));
    const bool bad = __any_sync(0xffffffffu, !(l + largest <= FLT_MAX) || o[0] != o[0] || o[1] != o[1] || o[2] != o[2] || o[3] != o[3]);
    if (lane == 0) again = bad;
  }
  __syncthreads();
  if (again) {
    // A score far above those of its run's first tile, whose weight, or weight times value, is no f32 number any more, or an infinite value beside a weight
    // that is zero as a second term: once more, four keys a warp at a time, the shared tiles' from the group's first sequence.  (One sequence of 100000
    // positions 14 ms, 105 by one warp and key by key; 0.1 where no row is attended again.)
    const int s = paged_row_of(p, b), len = s < 0 ? 0 : min(max(p.lens[s], 0), p.max_len);
    int head_s = s;                    // whose pages
    if (q.pre_tiles) {
      int g = p.n_groups - 1;          // the last group that starts there or before
      while (g > 0 && pu_group_start(p, g) > b) --g;
      head_s = max(paged_row_of(p, pu_group_start(p, g)), 0);
    }
    float m = -FLT_MAX, x[4];
    l = o[0] = o[1] = o[2] = o[3] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __bfloat162float(p.q[at + i]);
    auto four = [](const __nv_bfloat16* from, float (&to)[4]) {
      const uint2 w = *reinterpret_cast<const uint2*>(from);
      to[0] = __uint_as_float(w.x << 16);
      to[1] = __uint_as_float(w.x & 0xFFFF0000u);
      to[2] = __uint_as_float(w.y << 16);
      to[3] = __uint_as_float(w.y & 0xFFFF0000u);
    };
    for (int j0 = 4 * warp; j0 < len; j0 += 16) {      // (of one page: a page has 16 rows or more)
      const int from = j0 < q.pre_tiles * kPfTile ? head_s : s;
      const int page = min(max(p.tables[(size_t)from * p.table_ld + (j0 >> p.page_shift)], 0), p.n_pages - 1);
      const size_t row = ((size_t)page << p.page_shift) + (j0 & ((1 << p.page_shift) - 1));
      float sc[4], v[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const size_t r = ((row + i) * p.n_kv + kv) * kPaDim + 4 * lane;
        float k[4];
        four(p.k + r, k);
        four(p.v + r, v[i]);
        sc[i] = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) sc[i] = fmaf(x[c], k[c], sc[i]);
      }
      float mn = m;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sc[i] = warp_sum(sc[i]) * p.scale_log2;
        if (j0 + i < len) mn = fmaxf(mn, sc[i]);
      }
      const float f = ex2(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] *= f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (j0 + i < len) {
          const float w = ex2(sc[i] - mn);
          l += w;
#pragma unroll
          for (int c = 0; c < 4; ++c) o[c] += w * v[i][c];
        }
    }
    part[warp][lane] = make_float4(o[0], o[1], o[2], o[3]);
    if (lane == 0) part_ml[warp] = make_float2(m, l);
    __syncthreads();
    m = fmaxf(fmaxf(part_ml[0].x, part_ml[1].x), fmaxf(part_ml[2].x, part_ml[3].x));
    l = o[0] = o[1] = o[2] = o[3] = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 v = part[k][lane];
      const float f = ex2(part_ml[k].x - m);
      l += part_ml[k].y * f;
      o[0] += v.x * f;
      o[1] += v.y * f;
      o[2] += v.z * f;
      o[3] += v.w * f;
    }
  }
  if (warp) return;
  const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;                // (a NaN stays one)
  if (p.out_f32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
  } else {
    uint2 w;
    w.x = pack_bf16(o[0] * inv, o[1] * inv);
    w.y = pack_bf16(o[2] * inv, o[3] * inv);
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at) = w;
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
  TQ_REQUIRE(ctx, pages->ctx == ctx, "tq_gqa_decode_paged: the pool belongs to another context");
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
  if (p.max_shared > 1 << 29) p.max_shared = 1 << 29; // (what the plan's 23 bits of tiles hold; the rest is attended by each member)
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
  pp.per_eight = 8 / p.group;
  pp.few = p.out_f32 ? kPuFewRows / p.group : 0;
  const size_t tiles = batch * (((size_t)p.max_len + kPfTile - 1) / kPfTile) * n_kv_heads;
  TQ_REQUIRE(ctx, tiles < (1ull << 30) && (size_t)p.n_pages * pages->page_rows < (1ull << 31), "tq_gqa_decode_paged: too many positions");
  const size_t most_ctas = tiles < (size_t)ctx->sm_count ? tiles : (size_t)ctx->sm_count;
  pp.n_shares = (int)(most_ctas > n_kv_heads ? most_ctas / n_kv_heads : 1);
  const size_t n_ctas = pp.n_shares * n_kv_heads;
  // partial results (rows of either kind: the list's, and what a CTA adds), the sequences' plans
  // (tiles of a run: no more than a sequence has)
  const size_t longest[2] = {((size_t)p.max_len + kPfTile - 1) / kPfTile, p.n_groups ? (size_t)p.max_shared / kPfTile : 0};
  bool pieces = false;
  for (int k = 0; k < 2; ++k) {
    pp.window[k] = kPuWindow[!p.out_f32][k];
    pieces = pieces || longest[k] > (size_t)pp.window[k] + 1;
  }
  auto kern = pieces ? paged_decode_kernel<true> : paged_decode_kernel<false>;
  const size_t own_rows = batch * n_heads + 8 * n_ctas, pre_rows = p.n_groups ? batch * n_heads + 128 * n_ctas : 0, floats = (own_rows + pre_rows) * (kPaDim + 4);
  if (int st = ensure_scratch(ctx, floats * sizeof(float) + (batch + 1) * sizeof(PuSeqPlan))) return st;
  pp.own_o = static_cast<float*>(ctx->scratch);
  pp.pre_o = pp.own_o + own_rows * kPaDim;
  pp.own_ml = pp.pre_o + pre_rows * kPaDim;
  pp.pre_ml = pp.own_ml + own_rows * 4;
  pp.plan = reinterpret_cast<PuSeqPlan*>(pp.pre_ml + pre_rows * 4);
  pp.share = reinterpret_cast<int*>(pp.plan + batch);
  pp.a = p;
  CUtensorMap qe, qw, km, vm;
  const size_t row = n_kv_heads * kPaDim, rows = (size_t)p.n_pages * pages->page_rows;
  const unsigned g = (unsigned)p.group, box = pages->page_rows < kPfTile ? (unsigned)pages->page_rows : (unsigned)kPfTile;
  auto q_map = [&](CUtensorMap* m, int members) { return encode_bf16_boxes(m, q_dev, kPaDim, n_heads, batch, kPaDim * 2, n_heads * kPaDim * 2, g, (unsigned)members); };
  if (!q_map(&qe, pp.per_eight) || !q_map(&qw, pp.per_tile) || !encode_pages(&km, k_pages_dev, row, rows, box) ||
      !encode_pages(&vm, v_pages_dev, row, rows, box))
    return fail(ctx, TQ_ECUDA, "cuTensorMapEncodeTiled failed");
  const size_t smem = kPuFixed + (2 * batch + 1 + (size_t)p.n_groups + 1) * sizeof(int);
  if (int st = pages_use(ctx, pages)) return st;
  TQ_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kPuFixed + (3 * kPuBatch + 2) * sizeof(int))));
  TQ_CUDA(ctx, launch_k(ctx, kern, dim3((unsigned)n_ctas), dim3(kPuThreads), smem, qe, qw, km, vm, pp));
  TQ_CUDA(ctx, launch_k(ctx, paged_join_kernel, dim3((unsigned)n_heads, (unsigned)batch), dim3(128), 0, pp));
  return TQ_OK;
}
