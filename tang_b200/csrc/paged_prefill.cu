// Causal attention of several sequences' new positions, packed, over their pages (include/tangq.h: tq_gqa_prefill_paged).
//
// A CTA takes a tile of 128 rows (128 / group positions x the group's heads of one KV head) of a sequence and walks its keys in blocks of 64:
//   warp 0        queries, then blocks of keys: tensor copies page by page, or, for pages of 4 bits, codes that it turns into the same bf16 rows
//   warp 1        issues the products: a block's S = Q K^T (both from shared memory), then O += P V of the block before (P from tensor memory, V N-major)
//   warp 2        blocks of values, likewise; rows behind the last key are zeros (whatever a page holds there must not meet a weight of zero)
//                 (values of keys that not all rows of the tile see, 127 keys at most, are looked at: those that are no number are zeros too, and are added to
//                 the results of the rows that see them.  Rows that met such a value attended again over all of their keys, by a warp while the others
//                 waited, took a time that grew with the sequence and could outlast the waits' limit)
//   warp 3        finds out what the CTA does: its own tile, then those that it takes over from CTAs of the grid that have not begun (the hardware
//                 hands them out one by one), looked up while the tile before is worked on
//   warps 4..7    softmax, a thread a row, and the results
// Tensor memory: two blocks' S / P and O, 256 columns, so that two CTAs share an SM: one's products run while the other's weights are computed.  The roles go
// from tile to tile on their own: copies and scores of the next one run while the results of this one are stored (a tile a CTA: look-up, first copies and results
// took 10000 of 21000 cycles for 8 blocks).  A weight is one bf16 number, and the sum that results are
// divided by is that of the numbers as they entered: a row of a few keys, where the roundings do not average out, is then nearer (the largest weight need not
// be 1 for that, so that the reference may lag: a row's sums are rescaled only when its maximum grew by more than 2^8; sums with a running reference are those of
// Milakov and Gimelshein, Online normalizer calculation for softmax, 2018).  It begins 2^8 above the maximum, so that weights are 2^-8 to 1: sums hold what those of
// weights of at most 1 hold, and values of 2^-110 count.  What the lag costs is that the largest weight is rounded like the others: errors against 64 bits of 1.70e-3
// to 2.19e-3, with a reference that follows every maximum 1.70e-3 to 1.89e-3, but one prompt of 4096 then takes 183 instead of 146 us; the results' own rounding is
// 1.57e-3 to 1.66e-3.
// Few rows: a tile's keys are cut into parts, a CTA each, and a second kernel joins the results.
//
// What bounds it: products of 128 x 64 x 16 take 48 cycles, the bytes of their operands (32 would do for the multiplications), of 128 x 128 x 16 from tensor memory
// 64: 640 a block, 1280 for two CTAs' blocks, beside 1000 of a scheduler's special function unit and 900 of its issue slots.  One prompt of 4096 positions, 32 heads,
// 8 KV heads, 118 to 122 us (1140 TFLOP/s; 141 to 147 at the power limit, where a quarter of the weights as polynomials, to spare the special function unit, made 141
// into 149), 13 prompts of up to 1237 80 us (94 to 97 at the power limit), 57 blocks and 8 tiles a CTA, where what lies between tiles is a quarter of the time.  Over 4
// bits the same takes 1.35 to 1.45 times as long: one warp each unpacks keys and values, on the schedulers of two of the softmax warps.  A few rows are a chain of blocks of
// 0.8 to 1 us (64 behind 2000 keys 16.4 us, one block 8.2).  Scores of 128 keys at a time, which cost the tensor core less, wait for the products of the tile before:
// 167 us.
#include <cfloat>
#include <type_traits>

#include "attn_mma.cuh"
#include "attn_umma.cuh"
#include "page_rows.cuh"

namespace tq {

constexpr int kPpThreads = 256;
constexpr int kPpBlock = 64;                          // keys whose scores are computed, and become weights, at a time
constexpr int kPpSlots = 2;                           // of keys, and of values: a block each
constexpr int kPpBox = kPpBlock * 128;                // bytes of a block's 64 columns
constexpr int kPpTile = 2 * kPpBox;
constexpr int kPpItems = 2;                            // tiles that the roles are told ahead
constexpr int kPpAhead = 2;                            // the next tile is asked for when so many blocks of keys are still to be copied
constexpr int kPpStored = 4;                          // a tile's values are all there at most two tiles before its results are stored
constexpr int kPpReaders = 7;                         // warps that are told
constexpr int kPpStage = 32 * 64;                     // bytes of results that a warp stores at a time
constexpr size_t kPpSmem = 1024 + 1024 + 2 * (size_t)kPfBox + 2 * kPpSlots * (size_t)kPpTile + 4 * (size_t)kPpStage;
constexpr float kPpLag = 8.f;                         // how far a row's maximum may grow before its reference does (log2)
constexpr int kPpMaxParts = 32;                       // a lane of the join each (2 rows behind 65536 keys 44.7 us, 64 with 16 parts, 109 with 8; 16 behind 32768 41.5, 41.1, 61.5)

struct PackedPrefillParams {
  PackedSeqs s;
  const __nv_bfloat16* q;
  const uint8_t *k, *v;
  size_t row_bytes;
  int n_heads, n_kv, group, max_len;
  int per_tile, parts;                 // positions of a row tile; parts of a tile's keys
  float scale_log2;
  __nv_bfloat16* out;
  float *part_o, *part_ml;             // [part][rows][n_heads][128], [..][2] (reference and sum) where there are several
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

// Values that are no number, of keys lo .. hi - 1 of a block in shared memory, become zeros, by a warp; says whether there were any.
__device__ __forceinline__ bool pp_zero_values(uint8_t* tile, int lo, int hi, int lane) {
  // (a lane: 16 bytes of every other key, whatever their order in its half of the columns)
  uint8_t* mine = tile + ((lane >> 3) & 1) * kPpBox + (lo + (lane >> 4)) * 128 + 16 * (lane & 7);
  const int n = (hi - lo + 1 - (lane >> 4)) >> 1;
  uint32_t z[2] = {0u, 0u};            // products with zero: NaN if there is one, or an infinity
#pragma unroll 4
  for (int k = 0; k < n; ++k) {
    const uint4 x = *reinterpret_cast<const uint4*>(mine + 256 * k);
    z[0] = bf16x2_fma(x.x, 0u, z[0]);
    z[1] = bf16x2_fma(x.y, 0u, z[1]);
    z[0] = bf16x2_fma(x.z, 0u, z[0]);
    z[1] = bf16x2_fma(x.w, 0u, z[1]);
  }
  const uint32_t nan = ((z[0] & 0x7FFF7FFFu) + 0x007F007Fu) | ((z[1] & 0x7FFF7FFFu) + 0x007F007Fu);
  if (!__any_sync(0xffffffffu, (nan & 0x80008000u) != 0)) return false;
#pragma unroll 1
  for (int k = 0; k < n; ++k) {
    uint32_t* w = reinterpret_cast<uint32_t*>(mine + 256 * k);
    for (int i = 0; i < 4; ++i) {
      if ((w[i] & 0x7F80u) == 0x7F80u) w[i] &= 0xFFFF0000u;
      if ((w[i] & 0x7F800000u) == 0x7F800000u) w[i] &= 0xFFFFu;
    }
  }
  return true;
}

// What a CTA does.
struct PpItem {
  int seq, kv, part;                   // of the pool (-1: there is no more), KV head, part of the keys
  int row0, rows;                      // first packed row, rows
  int pos0;                            // position of the first row
  int block0, blocks;                  // blocks of keys: the part's first, how many
  int k_end;                           // keys that the last row sees, or the bound
};
// Tile x of all sequences, the longest of each sequence first, by one warp.
__device__ __forceinline__ PpItem pp_item(const PackedPrefillParams& p, int x, int kv, int part, int lane) {
  PpItem it{-1, kv, part, 0, 0, 0, 0, 0, 0};
  int i = -1, first = 0, count = 0, tile = 0, s = -1, len = 0;
  if (!p.s.seq_rows) {
    if (x < p.s.batch) {
      i = x, first = x, count = 1;
      s = packed_seq(p.s, i);
      len = s < 0 ? 0 : p.s.lens[s];
    }
  } else {
    int before = 0, largest = 0;       // tiles of the sequences before; the largest start so far, once some are not as they should be
    bool bad = false;
    for (int base = 0; base < p.s.batch; base += 32) {
      const int j = base + lane;
      int f = -0x7fffffff - 1, c = 0, js = -1, jl = 0;
      bool odd = false;
      if (j < p.s.batch) {
        const int b = p.s.seq_rows[j + 1];
        f = p.s.seq_rows[j];
        js = packed_seq(p.s, j);       // (on their way beside the starts)
        jl = js < 0 ? 0 : p.s.lens[js];
        odd = f < 0 || b < f || b > p.s.rows || (j == 0 && f != 0);
        c = odd ? 0 : b - f;
      }
      const bool was = bad;
      bad = bad || __any_sync(0xffffffffu, odd);
      if (bad) {                       // (packed_row has the rule)
        int most = f;
        if (lane == 0 && base > 0) most = max(most, was ? largest : p.s.seq_rows[base - 1]);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int w = __shfl_up_sync(0xffffffffu, most, o);
          if (lane >= o) most = max(most, w);
        }
        if (most != f) c = 0;
        largest = __shfl_sync(0xffffffffu, most, 31);
      }
      const int tiles = (c + p.per_tile - 1) / p.per_tile;
      int incl = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int w = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += w;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, x >= before + incl - tiles && x < before + incl);
      if (hit && i < 0) {
        const int src = __ffs(hit) - 1;
        i = base + src;
        first = __shfl_sync(0xffffffffu, f, src);
        count = __shfl_sync(0xffffffffu, c, src);
        s = __shfl_sync(0xffffffffu, js, src);
        len = __shfl_sync(0xffffffffu, jl, src);
        tile = __shfl_sync(0xffffffffu, before + incl, src) - 1 - x;   // (the last tile first)
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
      if (i >= 0 && x > 0) break;      // (the first tile's CTAs look at all starts)
    }
    if (bad && lane == 0) atomicCAS(p.err, 0, (int)DERR_PAGE_LIST);
  }
  if (i < 0) return it;
  if (s < 0 || len < count || len > (long long)p.s.table_ld << p.s.page_shift) {
    if (lane == 0) atomicCAS(p.err, 0, (int)DERR_PAGE_LIST);
    return it;
  }
  it.seq = s;
  it.row0 = first + tile * p.per_tile;
  it.rows = min(p.per_tile, count - tile * p.per_tile);
  it.pos0 = len - count + tile * p.per_tile;
  it.k_end = min(it.pos0 + it.rows, p.max_len);
  const int all = (it.k_end + kPpBlock - 1) / kPpBlock, per = max((all + p.parts - 1) / p.parts, 4);
  it.block0 = min(part * per, all);
  it.blocks = min(per, all - it.block0);
  return it;
}

// Adds a pair of bf16 to f32 sums.
__device__ __forceinline__ void add_bf16x2(float& a, float& b, uint32_t w) {
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tadd.f32.bf16 %0, lo, %0;\n\tadd.f32.bf16 %1, hi, %1;\n\t}" : "+f"(a), "+f"(b) : "r"(w));
}
// 32 columns of the warp's lanes; nothing may touch v before pp_landed.
__device__ __forceinline__ void pp_ask(uint32_t taddr, float (&v)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
               "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
                 "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
                 "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]),
                 "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void pp_landed(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]),
                 "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]),
                 "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]),
                 "+f"(v[31])::"memory");
}

// Pages of 4 bits: a loader's blocks.  A lane takes keys lane and lane + 32 of a block: their codes are asked for a block ahead, their pages two.
struct PpCodes {
  uint4 w[4];
  uint2 s;
};
__device__ __forceinline__ void pp_convert(uint8_t* tile, int key, const PpCodes& x) {
#pragma unroll
  for (int b = 0; b < 4; ++b) {        // a scale's 32 values
    const uint32_t half = b < 2 ? x.s.x : x.s.y, sc = prmt(half, half, b & 1 ? 0x3232 : 0x1010), off = bf16x2_mul(sc, 0xC1C0C1C0u);      // -24 s
    const uint32_t w[4] = {x.w[b].x, x.w[b].y, x.w[b].z, x.w[b].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t a[4];
      dequant_q4_word_24(w[i], a);
#pragma unroll
      for (int j = 0; j < 4; ++j) a[j] = bf16x2_fma(a[j], sc, off);
      const int c = 4 * (b & 1) + i;   // 16-byte chunk of the row's half
      *reinterpret_cast<uint4*>(tile + (b >> 1) * kPpBox + key * 128 + ((c ^ (key & 7)) << 4)) =
          make_uint4(prmt(a[0], a[1], 0x5410), prmt(a[2], a[3], 0x5410), prmt(a[0], a[1], 0x7632), prmt(a[2], a[3], 0x7632));
    }
  }
}

// Shared-memory descriptor of a block of values: keys are k, their 64-column halves a box apart (MN-major, 128-byte swizzle).
__device__ __forceinline__ uint64_t pp_desc_values(const void* smem_ptr) {
  return (uint64_t)((smem_u32(smem_ptr) >> 4) & 0x3FFF) | (uint64_t)(kPpBox >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// Asks for a CTA of this grid that has not begun: its place is then the asking CTA's to do, and it never begins.  The answer lands in 16 bytes of shared memory.
__device__ __forceinline__ void ask_for_cta(uint32_t answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool answered_cta(uint32_t answer, int& x, int& y, int& z) {
  uint32_t ok, a = 0, b = 0, c = 0;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t"
      "ld.shared.b128 r, [%4];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, %2, %3, _}, r;\n\t}"
      : "=r"(ok), "+r"(a), "+r"(b), "+r"(c)
      : "r"(answer)
      : "memory");
  x = (int)a, y = (int)b, z = (int)c;
  return ok != 0;
}

// Values that were made zeros, to the results of the tile's rows that see them, by a warp: a weight is positive, so that an infinity stays one.
template <bool Q4>
__device__ __forceinline__ void pp_give_back(const PackedPrefillParams& p, int seq, int kv, int part, int row0, int rows, int pos0, int first, int end) {
  const int lane = threadIdx.x & 31;
  int key = max(pos0 + 1, first);
  float seen[4] = {0.f, 0.f, 0.f, 0.f};                // of the lane's four columns, the keys up to a position
#pragma unroll 1
  for (int r = 0; r < rows; ++r) {
#pragma unroll 1
    for (const int behind = min(min(pos0 + r, p.max_len - 1) + 1, end); key < behind; ++key) {
      float v[4];
      row_values<Q4>(p.v + (size_t)max(page_row_of(p.s, seq, key), 0) * p.row_bytes, p.n_kv, kv, lane, v);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!(fabsf(v[i]) <= FLT_MAX)) seen[i] += v[i];
    }
    if (!__any_sync(0xffffffffu, seen[0] != 0.f || seen[1] != 0.f || seen[2] != 0.f || seen[3] != 0.f)) continue;
#pragma unroll 1
    for (int h = 0; h < p.group; ++h) {
      const size_t at = ((size_t)(row0 + r) * p.n_heads + kv * p.group + h) * kRowDim + 4 * lane;
      if (p.parts > 1) {
        float4* to = reinterpret_cast<float4*>(p.part_o + (size_t)part * p.s.rows * p.n_heads * kRowDim + at);
        const float4 x = *to;
        *to = make_float4(x.x + seen[0], x.y + seen[1], x.z + seen[2], x.w + seen[3]);
      } else {
        uint2* to = reinterpret_cast<uint2*>(p.out + at);
        const uint2 x = *to;
        *to = make_uint2(pack_bf16(__uint_as_float(x.x << 16) + seen[0], __uint_as_float(x.x & 0xFFFF0000u) + seen[1]),
                         pack_bf16(__uint_as_float(x.y << 16) + seen[2], __uint_as_float(x.y & 0xFFFF0000u) + seen[3]));
      }
    }
  }
}

template <bool Q4>
__global__ void __launch_bounds__(kPpThreads, 2)
paged_prefill_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                     const __grid_constant__ PackedPrefillParams p) {
  extern __shared__ uint8_t smem_raw[];
  // (phases run on from tile to tile: block R of all that the CTA does uses slots and columns R & 1)
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem_raw);
  uint64_t* q_empty = q_full + 1;
  uint64_t* k_full = q_empty + 1;                     // [slots]
  uint64_t* k_empty = k_full + kPpSlots;
  uint64_t* v_full = k_empty + kPpSlots;
  uint64_t* v_empty = v_full + kPpSlots;
  uint64_t* v_raw = v_empty + kPpSlots;               // a last block's values, before the rows behind the last key are zeroed
  uint64_t* s_full = v_raw + 1;                       // [parity of the block]
  uint64_t* p_full = s_full + 2;                      // likewise
  uint64_t* o_done = p_full + 2;                      // likewise: whoever waits for a block's products has seen those of the block two before
  uint64_t* o_free = o_done + 2;                      // a tile's sums have been read
  uint64_t* item_full = o_free + 1;                   // [items]
  uint64_t* item_empty = item_full + kPpItems;
  uint64_t* answer_bar = item_empty + kPpItems;
  uint64_t* nearly = answer_bar + 1;                  // a tile's last keys but a few have been asked for
  uint64_t* stored = nearly + 1;                      // [kPpStored] a tile's results have been stored
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(stored + kPpStored);
  volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);
  PpItem* item_s = reinterpret_cast<PpItem*>(smem_raw + 512);
  const uint32_t answer = smem_u32(smem_raw) + 768;
  uint8_t* q_s = smem_raw + 1024 + ((1024 - ((smem_u32(smem_raw) + 1024) & 1023)) & 1023);
  uint8_t *k_s = q_s + 2 * kPfBox, *v_s = k_s + kPpSlots * kPpTile, *stage_s = v_s + kPpSlots * kPpTile;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    if (lane == 0) {
      mbar_init(q_full, 1);
      mbar_init(q_empty, 1);
      mbar_init(o_free, 4);
      mbar_init(answer_bar, 1);
      mbar_init(nearly, 1);
      for (int i = 0; i < kPpStored; ++i) mbar_init(&stored[i], 4);
      for (int i = 0; i < kPpItems; ++i) {
        mbar_init(&item_full[i], 1);
        mbar_init(&item_empty[i], kPpReaders);
      }
      for (int s = 0; s < kPpSlots; ++s) {
        mbar_init(&k_full[s], 1);
        mbar_init(&k_empty[s], 1);
        mbar_init(&v_full[s], 1);
        mbar_init(&v_empty[s], 1);
      }
      mbar_init(v_raw, 1);
      for (int x = 0; x < 2; ++x) {
        mbar_init(&s_full[x], 1);
        mbar_init(&p_full[x], 4);
        mbar_init(&o_done[x], 1);
      }
      *failed = 0;
      mbar_init_fence();
    }
  } else if (warp == 1) {
    tmem_alloc(tmem_slot, 256);
  } else if (warp == 3 && lane == 0) {
    prefetch_map(&q_map);
    if (!Q4) {
      prefetch_map(&k_map);
      prefetch_map(&v_map);
    }
  }
  tc_fence_before();
  pdl_wait();
  pdl_launch_dependents();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto give_up = [&](int code) {
    atomicCAS(p.err, 0, code);
    *failed = 1;
  };
  // One arrival for the warp, whose lanes meet before it and behind it.
  auto arrive = [&](uint64_t* bar) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
    __syncwarp();
  };
  int told = 0;                        // tiles that the warp has been told
  auto take = [&](bool& ok, PpItem& it) {
    const int slot = told % kPpItems;
    ok = __all_sync(0xffffffffu, ok && mbar_wait_spin(&item_full[slot], (uint32_t)(told / kPpItems & 1)));
    if (ok) it = item_s[slot];
    else it.seq = -1;
    arrive(&item_empty[slot]);
    ++told;
    return it.seq >= 0;
  };

  // (registers: 256 threads of 128 at the start, then 128 of 88 or 104 and 128 of 168 or 152, the same in all)
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Q4 ? 104 : 88));
    if (warp == 3) {
      // ---- what to do
      bool ok = true;
      int x = blockIdx.x, y = blockIdx.y, z = blockIdx.z;
      for (int asked = 0;; ++asked) {
        const PpItem it = pp_item(p, y, x, z, lane);
        if (it.seq >= 0 && (it.blocks > 0 || p.parts > 1)) {
          const int slot = told % kPpItems;
          ok = __all_sync(0xffffffffu, mbar_wait_spin(&item_empty[slot], (uint32_t)(told / kPpItems & 1) ^ 1u));
          if (lane == 0) item_s[slot] = it;
          arrive(&item_full[slot]);
          // (not earlier: CTAs that are just being started elsewhere would be taken, and a long tile's CTA would hold the next one)
          ok = __all_sync(0xffffffffu, ok && mbar_wait_spin(nearly, (uint32_t)(told & 1)));
          ++told;
        }
        if (ok && lane == 0) {
          mbar_arrive_expect_tx(answer_bar, 16);
          ask_for_cta(answer, answer_bar);
        }
        __syncwarp();
        ok = __all_sync(0xffffffffu, ok && mbar_wait_spin(answer_bar, (uint32_t)(asked & 1)));
        if (!ok || !answered_cta(answer, x, y, z)) break;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // (the answer has been read before the next one is written)
        __syncwarp();
      }
      const int slot = told % kPpItems;                // the end
      ok = __all_sync(0xffffffffu, ok && mbar_wait_spin(&item_empty[slot], (uint32_t)(told / kPpItems & 1) ^ 1u));
      if (lane == 0) item_s[slot].seq = -1;
      arrive(&item_full[slot]);
      if (!ok && lane == 0) give_up(DERR_EMPTY_WAIT);
    }
    if (warp == 0 || warp == 2) {
      // ---- blocks of keys (and queries), blocks of values
      const bool values = warp == 2;
      uint64_t *full = values ? v_full : k_full, *empty = values ? v_empty : k_empty;
      uint8_t* to = values ? v_s : k_s;
      const int box_rows = min(1 << p.s.page_shift, kPpBlock), boxes = kPpBlock / box_rows;
      bool ok = true;
      int run = 0, tiles = 0, cuts = 0;                // blocks, tiles with keys, and blocks of values that the warp has waited for so far
      PpItem it;
      while (take(ok, it)) {
        const int n = it.blocks, call = max(n - kPpAhead, 0);
        if (n == 0) {
          if (!values) arrive(nearly);
          continue;
        }
        // Values of keys that some rows of the tile do not see meet weights of zero, and zero times a value that is no number is NaN.  They are zeros for all rows,
        // then; those that do see them get them back when the results are there.
        bool bad = false;
        const int* table = p.s.tables + (size_t)it.seq * p.s.table_ld;
        if (!values) {
          ok = __all_sync(0xffffffffu, mbar_wait_spin(q_empty, (uint32_t)(tiles & 1) ^ 1u));
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(q_full, 2u * p.per_tile * p.group * 128u);
          __syncwarp();
          if (lane < 2) tma_load_3d(q_s + lane * kPfBox, &q_map, 64 * lane, it.kv * p.group, it.row0, q_full);
          __syncwarp();
          ++tiles;
        }
        if constexpr (Q4) {
          const uint8_t* from = (values ? p.v : p.k) + it.kv * kQ4HeadBytes;
          const int steps = 2 * n, key0 = it.block0 * kPpBlock + lane, scales = p.n_kv * kQ4HeadBytes - it.kv * kQ4HeadBytes + it.kv * 2 * kQ4HeadScales;
          auto page_at = [&](int m) {  // of key `lane` of step m
            const int key = key0 + 32 * m;
            return m < steps && key < it.k_end ? table[key >> p.s.page_shift] : 0;
          };
          auto codes_at = [&](int m, int page) {
            PpCodes x;
            const int key = key0 + 32 * m;
            if (m < steps && key < it.k_end) {
              if (page < 0 || page >= p.s.n_pages) {
                atomicCAS(p.err, 0, (int)DERR_POSITION);
                page = 0;
              }
              const uint8_t* row = from + ((size_t)(page << p.s.page_shift) + (key & ((1 << p.s.page_shift) - 1))) * p.row_bytes;
#pragma unroll
              for (int i = 0; i < 4; ++i) x.w[i] = *reinterpret_cast<const uint4*>(row + 16 * i);
              x.s = *reinterpret_cast<const uint2*>(row + scales);
            } else {                   // rows of zeros
#pragma unroll
              for (int i = 0; i < 4; ++i) x.w[i] = make_uint4(0u, 0u, 0u, 0u);
              x.s = make_uint2(0u, 0u);
            }
            return x;
          };
          auto turn = [&](uint8_t* tile, int row, int m, PpCodes& x) {
            if (values && key0 + 32 * m > it.pos0) {   // (behind the last key: scales of zero)
              auto no_number_at = [](uint32_t w, uint32_t e) { return (w & e) == e; };
              const bool no_number[4] = {no_number_at(x.s.x, 0x7F80u), no_number_at(x.s.x, 0x7F800000u), no_number_at(x.s.y, 0x7F80u), no_number_at(x.s.y, 0x7F800000u)};
              if (no_number[0] || no_number[1] || no_number[2] || no_number[3]) {
                bad = true;
                x.s = make_uint2((no_number[0] ? 0u : x.s.x & 0xFFFFu) | (no_number[1] ? 0u : x.s.x & 0xFFFF0000u),
                                 (no_number[2] ? 0u : x.s.y & 0xFFFFu) | (no_number[3] ? 0u : x.s.y & 0xFFFF0000u));
              }
            }
            pp_convert(tile, row, x);
          };
          PpCodes even = codes_at(0, page_at(0)), odd = codes_at(1, page_at(1));
          int even_page = page_at(2), odd_page = page_at(3);
          for (int i = 0; i < n && ok; ++i, ++run) {
            const int slot = run % kPpSlots;
            ok = __all_sync(0xffffffffu, mbar_wait_spin(&empty[slot], (uint32_t)(run / kPpSlots & 1) ^ 1u));
            if (!ok) break;
            turn(to + slot * kPpTile, lane, 2 * i, even);
            even = codes_at(2 * i + 2, even_page);
            even_page = page_at(2 * i + 4);
            turn(to + slot * kPpTile, 32 + lane, 2 * i + 1, odd);
            odd = codes_at(2 * i + 3, odd_page);
            odd_page = page_at(2 * i + 5);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            arrive(&full[slot]);
            if (!values && i == call) arrive(nearly);
          }
        } else {
          // a lane per box: a page's rows, half their columns
          const int j = lane >> 1, c = lane & 1;
          auto page_at = [&](int i) {
            const int key = (it.block0 + i) * kPpBlock + j * box_rows;
            return i < n && j < boxes && key < it.k_end ? table[key >> p.s.page_shift] : 0;
          };
          int next = page_at(0);
          for (int i = 0; i < n && ok; ++i, ++run) {
            int page = next;
            next = page_at(i + 1);
            const int slot = run % kPpSlots, key = (it.block0 + i) * kPpBlock, keys = min(kPpBlock, it.k_end - key), used = (keys + box_rows - 1) / box_rows;
            if (page < 0 || page >= p.s.n_pages) {
              atomicCAS(p.err, 0, (int)DERR_POSITION);
              page = 0;
            }
            const int row = (page << p.s.page_shift) + (key & ((1 << p.s.page_shift) - 1) & ~(box_rows - 1));
            ok = __all_sync(0xffffffffu, mbar_wait_spin(&empty[slot], (uint32_t)(run / kPpSlots & 1) ^ 1u));
            if (!ok) break;
            const int unseen = max(it.pos0 + 1 - key, 0);              // keys from there on are not seen by the first row
            const bool cut = values && (keys < kPpBlock || unseen < keys);
            uint64_t* bar = cut ? v_raw : &full[slot];
            if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(used * box_rows) * 256u);
            __syncwarp();
            if (j < used) tma_load_2d(to + slot * kPpTile + c * kPpBox + j * box_rows * 128, values ? &v_map : &k_map, it.kv * kRowDim + 64 * c, row, bar);
            __syncwarp();
            if (!values && i == call) arrive(nearly);
            if (cut) {                 // (the tile's last block, or those that its rows end in)
              ok = __all_sync(0xffffffffu, mbar_wait_spin(v_raw, (uint32_t)(cuts++ & 1)));
              if (!ok) break;
              uint8_t* at = to + slot * kPpTile;
              if (unseen < keys) bad = pp_zero_values(at, unseen, keys, lane) || bad;
              for (int k = lane; k < 2 * (kPpBlock - keys) * 8; k += 32)     // (a row's 128 bytes of either box, whatever their order)
                *reinterpret_cast<uint4*>(at + ((k >> 3) & 1) * kPpBox + (keys + (k >> 4)) * 128 + 16 * (k & 7)) = make_uint4(0u, 0u, 0u, 0u);
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              arrive(&full[slot]);
            }
          }
        }
        if (values) {
          if (__any_sync(0xffffffffu, ok && bad)) {
            ok = __all_sync(0xffffffffu, mbar_wait_spin(&stored[tiles % kPpStored], (uint32_t)(tiles / kPpStored & 1)));
            if (!ok) break;
            pp_give_back<Q4>(p, it.seq, it.kv, it.part, it.row0, it.rows, it.pos0, it.block0 * kPpBlock, min((it.block0 + n) * kPpBlock, it.k_end));
          }
          ++tiles;
        }
      }
      if (!ok && lane == 0) give_up(DERR_EMPTY_WAIT);
    } else if (warp == 1) {
      // ---- products: a block's scores, then the weighted values of the block before
      const bool leader = elect_one();
      const uint32_t idesc_s = umma_idesc_bf16(kPpBlock), idesc_o = umma_idesc_bf16(kRowDim) | (1u << 16);     // (bit 16: B is N-major)
      const uint64_t qd = umma_desc_sw128(q_s), kd = umma_desc_sw128(k_s), vd = pp_desc_values(v_s);
      const uint32_t o_t = tmem + 128u;
      bool ok = true;
      int run = 0, tiles = 0;          // blocks and tiles with keys before this one
      PpItem it;
      while (take(ok, it)) {
        const int n = it.blocks;
        if (n == 0) continue;
        ok = __all_sync(0xffffffffu, mbar_wait_spin(q_full, (uint32_t)(tiles & 1)));
        for (int j = 0; j <= n && ok; ++j) {
          if (j < n) {
            const int r = run + j, slot = r % kPpSlots;
            // (the scores' columns hold the weights of the block two before until its products are done)
            ok = __all_sync(0xffffffffu, mbar_wait_spin(&k_full[slot], (uint32_t)(r / kPpSlots & 1)) &&
                                             (r < 2 || mbar_wait_spin(&o_done[r & 1], (uint32_t)((r - 2) >> 1 & 1))));
            if (!ok) break;
            tc_fence_after();
            if (leader) {
              const uint64_t kt = kd + (uint64_t)(slot * (kPpTile >> 4));
#pragma unroll
              for (int k = 0; k < 8; ++k)
                umma_f16(tmem + (uint32_t)((r & 1) * kPpBlock), qd + (uint64_t)((k >> 2) * (kPfBox >> 4) + 2 * (k & 3)),
                         kt + (uint64_t)((k >> 2) * (kPpBox >> 4) + 2 * (k & 3)), idesc_s, k != 0);
              umma_commit(&s_full[r & 1]);
              umma_commit(&k_empty[slot]);
              if (j + 1 == n) umma_commit(q_empty);
            }
            __syncwarp();
          }
          if (j > 0) {
            const int r = run + j - 1, slot = r % kPpSlots;
            ok = __all_sync(0xffffffffu, mbar_wait_spin(&v_full[slot], (uint32_t)(r / kPpSlots & 1)) && mbar_wait_spin(&p_full[r & 1], (uint32_t)(r >> 1 & 1)) &&
                                             (j > 1 || tiles == 0 || mbar_wait_spin(o_free, (uint32_t)((tiles - 1) & 1))));
            if (!ok) break;
            tc_fence_after();
            if (leader) {
              const uint64_t vt = vd + (uint64_t)(slot * (kPpTile >> 4));
#pragma unroll
              for (int k = 0; k < kPpBlock / 16; ++k)
                umma_f16_ts(o_t, tmem + (uint32_t)((r & 1) * kPpBlock) + 8u * k, vt + (uint64_t)(k * (2048 >> 4)), idesc_o, ((j - 1) | k) != 0);
              umma_commit(&o_done[r & 1]);
              umma_commit(&v_empty[slot]);
            }
            __syncwarp();
          }
        }
        run += n;
        ++tiles;
      }
      if (!ok && lane == 0) give_up(DERR_FULL_WAIT);
    }
  } else {
    // ---- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Q4 ? 152 : 168));
    const int q4 = warp & 3, r = 32 * q4 + lane, r_pos = r / p.group, r_head = r - r_pos * p.group;
    const uint32_t s_t = tmem + ((uint32_t)(32 * q4) << 16), o_t = s_t + 128u;
    const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2);
    const bool parts = p.parts > 1;
    uint8_t* mine_s = stage_s + q4 * kPpStage;
    bool ok = true;
    int run = 0, tiles = 0;            // blocks and tiles with keys before this one
    PpItem it;
    while (take(ok, it)) {
      const int n = it.blocks, head = it.kv * p.group + r_head;
      const bool live = r_pos < min(p.per_tile, it.rows);
      const int limit = live ? min(it.pos0 + r_pos, p.max_len - 1) : -1;                           // the last key of this row
      float m = -FLT_MAX, l = 0.f;
#pragma unroll 1
      for (int j = 0; j < n && ok; ++j) {
        const uint32_t b_t = s_t + (uint32_t)(((run + j) & 1) * kPpBlock);
        ok = __all_sync(0xffffffffu, mbar_wait_spin(&s_full[(run + j) & 1], (uint32_t)((run + j) >> 1 & 1)));
        if (!ok) break;
        tc_fence_after();
        __syncwarp();
        float v[2][32];
        pp_ask(b_t, v[0]);
        pp_ask(b_t + 32u, v[1]);
        pp_landed(v[0]);
        pp_landed(v[1]);
        const int last = limit - (it.block0 + j) * kPpBlock;      // keys 0 .. last of the block count
        if (!__all_sync(0xffffffffu, last >= kPpBlock - 1)) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int k = 0; k < 32; ++k) v[c][k] = 32 * c + k <= last ? v[c][k] : -INFINITY;
        }
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          mx[c] = fmaxf(v[c >> 1][16 * (c & 1)], v[c >> 1][16 * (c & 1) + 1]);
#pragma unroll
          for (int k = 2; k < 16; k += 2) mx[c] = fmaxf(mx[c], fmaxf(v[c >> 1][16 * (c & 1) + k], v[c >> 1][16 * (c & 1) + k + 1]));
        }
        const float top = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2, -FLT_MAX);
        // (m: 2^8 above the maximum that it follows, so that no weight is above 1 before the maximum has grown so far)
        if (j == 0) {
          m = top + kPpLag;
        } else if (__any_sync(0xffffffffu, top > m)) {
          ok = __all_sync(0xffffffffu, mbar_wait_spin(&o_done[(run + j - 1) & 1], (uint32_t)((run + j - 1) >> 1 & 1)));
          if (!ok) break;
          tc_fence_after();
          __syncwarp();
          const float m_new = top > m ? top + kPpLag : m, f = ex2(m - m_new);
#pragma unroll 1
          for (int c = 0; c < kRowDim; c += 16) {
            float o[16];
            uint32_t w[16];
            tmem_ld16(o_t + (uint32_t)c, o);
#pragma unroll
            for (int k = 0; k < 16; ++k) w[k] = __float_as_uint(o[k] * f);
            tmem_st16(o_t + (uint32_t)c, w);
          }
          l *= f;
          m = m_new;
        }
        const uint64_t less = pack2(-m, -m);
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t w[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float a, b;
            const uint64_t t = fma2(pack2(v[c][2 * k], v[c][2 * k + 1]), scale2, less);
            unpack2(t, a, b);
            a = ex2(a);
            b = ex2(b);
            w[k] = pack_bf16(a, b);
            add_bf16x2(sum[2 * (k & 1)], sum[2 * (k & 1) + 1], w[k]);
          }
          tmem_st16(b_t + 16u * c, w);                  // over scores that this thread has read
        }
        tmem_st_wait();
        tc_fence_before();
        arrive(&p_full[(run + j) & 1]);
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      }
      if (ok && n) ok = __all_sync(0xffffffffu, mbar_wait_spin(&o_done[(run + n - 1) & 1], (uint32_t)((run + n - 1) >> 1 & 1)));
      if (!ok) break;
      run += n;
      tc_fence_after();
      __syncwarp();
      const size_t at = ((size_t)(live ? it.row0 + r_pos : 0) * p.n_heads + head) * kRowDim;
      const size_t part_at = (size_t)it.part * p.s.rows * p.n_heads * kRowDim;
      if (parts && live) *reinterpret_cast<float2*>(p.part_ml + (part_at + at) / (kRowDim / 2)) = make_float2(m, l);
      if (n) {
        const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
        // Rows go over shared memory 64 bytes at a time, so that four lanes store what stands together (a lane with a row of its own would store to 32 places at once).
        // Code of its own for parts (f32) and results (bf16): left to the compiler, which of them it writes changes with what stands around it, 4 % of many short prompts.
        const unsigned to_store = __ballot_sync(0xffffffffu, live);
        auto store = [&](auto of_parts) {
          constexpr bool PARTS = decltype(of_parts)::value;
          uint8_t* base = PARTS ? reinterpret_cast<uint8_t*>(p.part_o + part_at) : reinterpret_cast<uint8_t*>(p.out);
          const unsigned long long row_bytes_at = (unsigned long long)at * (PARTS ? 4 : 2);
          unsigned long long to[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) to[k] = __shfl_sync(0xffffffffu, row_bytes_at, 8 * k + (lane >> 2)) + 16 * (lane & 3);
#pragma unroll 1
          for (int c = 0; c < kRowDim; c += 32) {
            float o[32];
            __syncwarp();
            pp_ask(o_t + (uint32_t)c, o);
            pp_landed(o);
            if (c == kRowDim - 32) {     // (the next tile's products may begin)
              tc_fence_before();
              arrive(o_free);
            }
#pragma unroll
            for (int half = 0; half < (PARTS ? 2 : 1); ++half) {
              uint8_t* row = mine_s + lane * 64;
              const int turn = (lane >> 1) & 3;          // (eight lanes' 16 bytes meet all banks)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                uint4 y;
                if constexpr (PARTS) {
                  const float* x = &o[16 * half + 4 * k];
                  y = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
                } else {
                  const float* x = &o[8 * k];
                  y = make_uint4(pack_bf16(x[0] * inv, x[1] * inv), pack_bf16(x[2] * inv, x[3] * inv), pack_bf16(x[4] * inv, x[5] * inv), pack_bf16(x[6] * inv, x[7] * inv));
                }
                *reinterpret_cast<uint4*>(row + ((k ^ turn) << 4)) = y;
              }
              __syncwarp();
              uint4 y[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int from = 8 * k + (lane >> 2);
                y[k] = *reinterpret_cast<const uint4*>(mine_s + from * 64 + (((lane & 3) ^ ((from >> 1) & 3)) << 4));
              }
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (to_store >> (8 * k + (lane >> 2)) & 1u) *reinterpret_cast<uint4*>(base + to[k] + (PARTS ? 4 * (c + 16 * half) : 2 * c)) = y[k];
              __syncwarp();
            }
          }
        };
        if (parts) store(std::true_type{});
        else store(std::false_type{});
        arrive(&stored[tiles++ % kPpStored]);
      }
    }
    if (!ok && lane == 0) give_up(DERR_TMEM);
  }
  tc_fence_before();
  __syncthreads();
  if (*failed && threadIdx.x == 0) {
    // copies and products that are still in flight target this CTA's memories: give them time to land before leaving
    for (int i = 0; i < 10000; ++i) __nanosleep(1000);
  }
  __syncthreads();
  __syncwarp();                        // (the release is one instruction of the whole warp)
  if (warp == 1) tmem_dealloc(tmem, 256);
}

// Joins the parts of a row's head, in their order: a warp, four columns a lane.
__global__ void __launch_bounds__(128) paged_prefill_join_kernel(const PackedPrefillParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const size_t i = (size_t)blockIdx.x * 4 + (threadIdx.x >> 5), heads = (size_t)p.s.rows * p.n_heads;      // the row's head
  if (i >= heads) return;
  // rows that nobody attended for are left as they are
  const int m = (int)(i / p.n_heads);
  if (packed_row(p.s, m, lane, p.err).seq < 0) return;
  const float2 ml = lane < p.parts ? *reinterpret_cast<const float2*>(p.part_ml + (lane * heads + i) * 2) : make_float2(-FLT_MAX, 0.f);
  const float top = warp_max(ml.x), w = ex2(ml.x - top), l = warp_sum(ml.y * w);
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int base = 0; base < p.parts; base += 8) {      // (eight on their way at a time)
    float4 v[8];
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      f[k] = __shfl_sync(0xffffffffu, w, base + k);
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      // (a part without keys of this row has left nothing)
      if (__shfl_sync(0xffffffffu, ml.y, base + k) != 0.f) v[k] = *reinterpret_cast<const float4*>(p.part_o + ((size_t)(base + k) * heads + i) * kRowDim + 4 * lane);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      o[0] = fmaf(v[k].x, f[k], o[0]);
      o[1] = fmaf(v[k].y, f[k], o[1]);
      o[2] = fmaf(v[k].z, f[k], o[2]);
      o[3] = fmaf(v[k].w, f[k], o[3]);
    }
  }
  const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
  *reinterpret_cast<uint2*>(p.out + i * kRowDim + 4 * lane) = make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
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
  TQ_REQUIRE(ctx, apart(q_dev, rows * n_heads * kRowDim * 2, out_dev, rows * n_heads * kRowDim * 2),
             "tq_gqa_prefill_paged: results need a buffer of their own (they are stored while other rows' queries are read)");
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
  p.group = (int)(n_heads / n_kv_heads);
  p.per_tile = kPfTile / p.group;
  // Tiles there may be; parts of their keys, of four blocks or more, where these leave SMs idle (each takes two CTAs).
  const size_t tiles = seq_rows_dev ? rows / p.per_tile + (batch < rows ? batch : rows) : rows;
  const size_t most = (size_t)pages->table_ld * pages->page_rows, longest = max_len < most ? max_len : most, ctas = tiles * n_kv_heads;
  TQ_REQUIRE(ctx, tiles <= 65535, "tq_gqa_prefill_paged: too many rows");
  size_t parts = 1;
  if (ctas < 2 * (size_t)ctx->sm_count) {
    parts = 2 * (size_t)ctx->sm_count / ctas;          // (one more would begin when the others are through)
    const size_t few = longest / (4 * kPpBlock);
    parts = parts > few ? few : parts;
    parts = parts < 1 ? 1 : parts > (size_t)kPpMaxParts ? (size_t)kPpMaxParts : parts;
  }
  p.parts = (int)parts;
  p.part_o = p.part_ml = nullptr;
  if (parts > 1) {
    const size_t heads = parts * rows * n_heads;
    if (int st = ensure_scratch(ctx, heads * (kRowDim + 2) * sizeof(float))) return st;
    p.part_o = static_cast<float*>(ctx->scratch);
    p.part_ml = p.part_o + heads * kRowDim;
  }
  CUtensorMap qm, km = {}, vm = {};
  const size_t row = n_kv_heads * kRowDim, cache_rows = (size_t)pages->n_pages * pages->page_rows;
  const unsigned box = pages->page_rows < kPpBlock ? (unsigned)pages->page_rows : (unsigned)kPpBlock;
  if (!encode_bf16_boxes(&qm, q_dev, kRowDim, n_heads, rows, kRowDim * 2, n_heads * kRowDim * 2, (unsigned)p.group, (unsigned)p.per_tile) ||
      (!q4 && (!encode_bf16_k64(&km, k_pages_dev, cache_rows, row, row, box) || !encode_bf16_k64(&vm, v_pages_dev, cache_rows, row, row, box))))
    return fail(ctx, TQ_ECUDA, "cuTensorMapEncodeTiled failed");
  if (int st = pages_use(ctx, pages)) return st;
  auto kern = q4 ? paged_prefill_kernel<true> : paged_prefill_kernel<false>;
  TQ_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPpSmem));
  TQ_CUDA(ctx, launch_k(ctx, kern, dim3((unsigned)n_kv_heads, (unsigned)tiles, (unsigned)parts), dim3(kPpThreads), kPpSmem, qm, km, vm, p));
  if (parts > 1) TQ_CUDA(ctx, launch_k(ctx, paged_prefill_join_kernel, dim3((unsigned)((rows * n_heads + 3) / 4)), dim3(128), 0, p));
  return TQ_OK;
}
