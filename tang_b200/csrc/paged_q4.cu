// Decode attention over pages of 4 bits (include/tangq.h: tq_gqa_decode_paged_q4): the attention of tq_gqa_decode_paged (paged_attention.cu)
// for one new token per sequence, where a cache row is 64 bytes of codes and four scales a head (page_rows.cu).
//
// A warp works alone: no barrier, no wait but for its own copies.  It holds the query heads of one KV head as the columns of mma.sync's B operand and walks
// chunks of 32 keys, which it copies to its own ring in shared memory a chunk ahead: S^T = K Q^T (keys are rows), softmax weights from a reference that
// begins 2^8 above the largest score and moves when one is above it (so that no weight is above 1), O^T = V^T P^T.  Codes become bf16 in registers, exactly:
// 24 + c is four bits in the mantissa of 16, and fma(24 + c, s, -24 s) = c s, where s has 5 significant bits and c 3.  Which row, column or step a value
// takes is free, as long as both operands agree:
// a lane's 16 bytes of a key are its part of all eight steps of the scores, a lane's 8 bytes of four keys its part of all 128 rows of O.
// Weights are two bf16 terms, within 2^-16.  Up to four query heads, columns 4 to 7 repeat columns 0 to 3 and take the second terms, so that these cost nothing.
//
// What bounds it: a warp's way through a chunk, scores, vote, exponentials, transposes and values one after the other: 3.4 us for 32 keys and values of a head, 790
// instructions, of which 400 unpack (a word of eight codes four shifts, four masks, four fused operations), 100 ask for the next chunk and 32 are products.  Four warps a
// scheduler issue 0.58 a cycle of them, and ask for 47 % of the memory's rate.  64 sequences of up to 4096 positions, 8 KV heads, 156 MB,
// 51.3 us (3.0 TB/s, 47 % of the memory's rate; the same without any copies 47); one sequence of 700 8.4 us; three of up to 65537 30.9.  Tensor copies instead of
// cp.async 53.3 us (boxes of 64 and of 16 bytes); one sum of the scores of a half chunk instead of two 53.2; 12 warps an SM with three chunks each 53.9.
#include <cfloat>

#include "attn_mma.cuh"
#include "page_rows.cuh"

namespace tq {

constexpr int kQdWarps = 4, kQdCtas = 4, kQdChunk = 32, kQdStages = 2;        // warps of a CTA, CTAs of an SM
constexpr int kQdKeyBytes = 64, kQdValueBytes = 80;    // of a row in shared memory (80: four rows' 8-byte reads meet all banks)
constexpr int kQdStageBytes = kQdChunk * (kQdKeyBytes + kQdValueBytes + 16);
constexpr float kQdLag = 8.f;          // how far a maximum may grow before its reference does (log2)

struct Q4DecodeParams {
  PackedSeqs s;
  const __nv_bfloat16* q;
  const uint8_t *k, *v;
  size_t row_bytes;
  int n_heads, n_kv, group, max_len, n_shares;         // n_shares: warps of a KV head
  float scale_log2;
  float *o, *ml;                       // partial results [kv][batch + n_shares][group][128], [..][2]
  int2* plan;                          // [batch] a sequence's first share, how many have a part of it
  __nv_bfloat16* out;
  int* err;
};

__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(valid ? 8u : 0u) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {           // of an 8 x 8 matrix of 16 bits, a row in four lanes
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ int q4d_len(const Q4DecodeParams& p, int b) {
  const int s = packed_seq(p.s, b);
  return s < 0 ? 0 : min(max(p.s.lens[s], 0), p.max_len);
}

// SPLIT: up to four query heads of a KV head.
template <bool SPLIT>
__global__ void __launch_bounds__(32 * kQdWarps, kQdCtas) q4_decode_kernel(const Q4DecodeParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  int* before = reinterpret_cast<int*>(smem + kQdWarps * kQdStages * kQdStageBytes);       // [batch + 1] chunks of the sequences before
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl_wait();
  pdl_launch_dependents();
  for (int b = threadIdx.x; b < p.s.batch; b += 32 * kQdWarps) {
    if (blockIdx.x == 0 && packed_seq(p.s, b) < 0) atomicCAS(p.err, 0, (int)DERR_PAGE_LIST);
    before[b] = (q4d_len(p, b) + kQdChunk - 1) / kQdChunk;
  }
  __syncthreads();
  if (warp == 0) {
    int sum = 0;
    for (int base = 0; base < p.s.batch; base += 32) {
      const int v = base + lane < p.s.batch ? before[base + lane] : 0;
      int incl = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int w = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += w;
      }
      if (base + lane < p.s.batch) before[base + lane] = sum + incl - v;
      sum += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) before[p.s.batch] = sum;
  }
  __syncthreads();
  const int total = before[p.s.batch], share = max(1, (total + p.n_shares - 1) / p.n_shares);
  const int w = blockIdx.x * kQdWarps + warp, c = w / p.n_kv, kv = w - c * p.n_kv;         // neighbours: the KV heads of the same rows
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b < p.s.batch; b += 32 * kQdWarps) {
      const int f = before[b], n = before[b + 1] - f;
      p.plan[b] = make_int2(f / share, n ? (f + n - 1) / share - f / share + 1 : 0);
    }
  if (c >= p.n_shares) return;
  const int from = c * share, to = min(from + share, total);
  if (from >= to) return;

  uint8_t* ring = smem + warp * kQdStages * kQdStageBytes;
  const uint32_t ring_a = smem_u32(ring);
  // ---- copies: the page of key `lane` of the chunk that is asked for next is loaded a turn ahead
  int ask = from, ask_b = 0;           // the chunk that is asked for next, its sequence
  {
    int lo = 0, hi = p.s.batch;        // the last sequence that begins at or before it (those without chunks stand before it)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] <= from) lo = mid;
      else hi = mid;
    }
    ask_b = lo;
  }
  int b = ask_b, ask_pos = 0, ask_len = q4d_len(p, b), page = 0;
  const int* table = p.s.tables + (size_t)max(packed_seq(p.s, b), 0) * p.s.table_ld;
  auto look_up = [&] {
    ask_pos = (ask - before[ask_b]) * kQdChunk + lane;
    if (ask < to && ask_pos < ask_len) page = table[ask_pos >> p.s.page_shift];
  };
  look_up();
  auto request = [&](int stage) {
    const uint32_t at = ring_a + stage * kQdStageBytes;
    if (ask < to) {
      int mine = -1;                   // cache row, none behind the end
      if (ask_pos < ask_len) {
        if (page >= 0 && page < p.s.n_pages) mine = (page << p.s.page_shift) + (ask_pos & ((1 << p.s.page_shift) - 1));
        else atomicCAS(p.err, 0, (int)DERR_POSITION);
      }
      ++ask;
      if (ask < to && before[ask_b + 1] <= ask) {
        do ++ask_b;
        while (before[ask_b + 1] <= ask);
        ask_len = q4d_len(p, ask_b);
        table = p.s.tables + (size_t)max(packed_seq(p.s, ask_b), 0) * p.s.table_ld;
      }
      look_up();
#pragma unroll
      for (int i = 0; i < kQdChunk / 8; ++i) {
        const int key = 8 * i + (lane >> 2), row = __shfl_sync(0xffffffffu, mine, key);
        const size_t src = (size_t)max(row, 0) * p.row_bytes + kv * kQ4HeadBytes + 16 * t;
        cp_async16(at + key * kQdKeyBytes + 16 * t, p.k + src, row >= 0);
        cp_async16(at + kQdChunk * kQdKeyBytes + key * kQdValueBytes + 16 * t, p.v + src, row >= 0);
      }
      const size_t src = (size_t)max(mine, 0) * p.row_bytes + p.n_kv * kQ4HeadBytes + kv * 2 * kQ4HeadScales;
      const uint32_t sc = at + kQdChunk * (kQdKeyBytes + kQdValueBytes) + 8 * lane;
      cp_async8(sc, p.k + src, mine >= 0);
      cp_async8(sc + 8 * kQdChunk, p.v + src, mine >= 0);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kQdStages - 1; ++i) request(i);

  uint32_t q[8][2];                    // steps' columns: the head of column g, this lane's 32 values
  float o[8][4], ref[2] = {0.f, 0.f}, sum[2] = {0.f, 0.f};             // heads 2t, 2t + 1
  int stage = 0;
  bool first = true;
  int len = 0;
#pragma unroll 1
  for (int f = from; f < to; ++f) {
    if (first) {
      while (b + 1 < p.s.batch && before[b + 1] <= f) ++b;
      len = q4d_len(p, b);
      const int h = SPLIT ? (g & 3) : g;
      const uint4* src = reinterpret_cast<const uint4*>(p.q + ((size_t)b * p.n_heads + kv * p.group + min(h, p.group - 1)) * kRowDim + 32 * t);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 x = h < p.group ? src[i] : make_uint4(0u, 0u, 0u, 0u);
        q[2 * i][0] = prmt(x.x, x.z, 0x5410);
        q[2 * i][1] = prmt(x.x, x.z, 0x7632);
        q[2 * i + 1][0] = prmt(x.y, x.w, 0x5410);
        q[2 * i + 1][1] = prmt(x.y, x.w, 0x7632);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
      sum[0] = sum[1] = 0.f;
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(kQdStages - 2) : "memory");
    __syncwarp();                      // (everybody's copies of this chunk, and everybody is done with the one before)
    request(stage == 0 ? kQdStages - 1 : stage - 1);
    const uint8_t* at = ring + stage * kQdStageBytes;
    if (++stage == kQdStages) stage = 0;

    // ---- scores: rows are keys, columns are heads
    float s[2][4];
    const uint16_t* ks = reinterpret_cast<const uint16_t*>(at + kQdChunk * (kQdKeyBytes + kQdValueBytes));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[h][0] = s[h][1] = s[h][2] = s[h][3] = 0.f;
      float more[4] = {0.f, 0.f, 0.f, 0.f};            // (two sums: half as many products wait for one another)
      uint32_t words[2][4], sc[2], off[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key = 16 * h + 8 * i + g;
        const uint4 x = *reinterpret_cast<const uint4*>(at + key * kQdKeyBytes + 16 * t);
        words[i][0] = x.x;
        words[i][1] = x.y;
        words[i][2] = x.z;
        words[i][3] = x.w;
        sc[i] = ks[key * kQ4HeadScales + t] * 0x10001u;
        off[i] = bf16x2_mul(sc[i], 0xC1C0C1C0u);       // -24 s
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a[2][4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          dequant_q4_word_24(words[r][i], a[r]);
#pragma unroll
          for (int j = 0; j < 4; ++j) a[r][j] = bf16x2_fma(a[r][j], sc[r], off[r]);
        }
        mma_bf16_16816(s[h], a[0][0], a[1][0], a[0][1], a[1][1], q[2 * i][0], q[2 * i][1]);
        mma_bf16_16816(more, a[0][2], a[1][2], a[0][3], a[1][3], q[2 * i + 1][0], q[2 * i + 1][1]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) s[h][j] += more[j];
    }
    const int left = len - (f - before[b]) * kQdChunk;                 // keys of the chunk
    if (left < kQdChunk) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[h][j] = 16 * h + 8 * (j >> 1) + g < left ? s[h][j] : -INFINITY;
    }
    float top[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) top[j] = fmaxf(fmaxf(s[0][j], s[0][2 + j]), fmaxf(s[1][j], s[1][2 + j])) * p.scale_log2;
    if (__any_sync(0xffffffffu, first || top[0] > ref[0] || top[1] > ref[1])) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], x));
        // (2^8 above the maximum that it follows: no weight is above 1 before the maximum has grown so far)
        const float to_ref = fmaxf(first ? -FLT_MAX : ref[j], top[j] + kQdLag), by = first ? 0.f : ex2_ftz(ref[j] - to_ref);
        ref[j] = to_ref;
        if (!first) {
          sum[j] *= by;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            o[i][j] *= by;
            o[i][2 + j] *= by;
          }
        }
      }
    }
    first = false;

    // ---- weights, as columns of the second product
    uint32_t hi[2][2], lo[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float w0 = ex2_ftz(fmaf(s[h][2 * i], p.scale_log2, -ref[0])), w1 = ex2_ftz(fmaf(s[h][2 * i + 1], p.scale_log2, -ref[1]));
        sum[0] += w0;
        sum[1] += w1;
        uint32_t a, b2;
        split_bf16(w0, w1, a, b2);
        if (SPLIT) {
          hi[h][i] = transpose8(t < 2 ? a : b2);
        } else {
          hi[h][i] = transpose8(a);
          lo[h][i] = transpose8(b2);
        }
      }

    // ---- values: rows are the 128 columns of V, 16 g + n in products n / 2, its row g or g + 8
    const uint8_t* vs = at + kQdChunk * kQdKeyBytes;
    const uint16_t* vsc = ks + kQdChunk * kQ4HeadScales + (g >> 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint2 x[4];
      uint32_t sc[2], off[2];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const uint2*>(vs + (16 * h + 8 * (i >> 1) + 2 * t + (i & 1)) * kQdValueBytes + 8 * g);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint16_t* at2 = vsc + (16 * h + 8 * i + 2 * t) * kQ4HeadScales;
        sc[i] = (uint32_t)at2[0] | (uint32_t)at2[kQ4HeadScales] << 16;
        off[i] = bf16x2_mul(sc[i], 0xC1C0C1C0u);
      }
#pragma unroll
      for (int part = 0; part < 4; ++part) {           // four of the lane's 16 columns
        uint32_t a[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t u = part < 2 ? x[2 * i].x : x[2 * i].y, v = part < 2 ? x[2 * i + 1].x : x[2 * i + 1].y;
          dequant_q4_word_24(prmt(u, v, part & 1 ? 0x7632 : 0x5410), a[i]);
#pragma unroll
          for (int j = 0; j < 4; ++j) a[i][j] = bf16x2_fma(a[i][j], sc[i], off[i]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mma_bf16_16816(o[2 * part + j], a[0][2 * j], a[0][2 * j + 1], a[1][2 * j], a[1][2 * j + 1], hi[h][0], hi[h][1]);
          if (!SPLIT) mma_bf16_16816(o[2 * part + j], a[0][2 * j], a[0][2 * j + 1], a[1][2 * j], a[1][2 * j + 1], lo[h][0], lo[h][1]);
        }
      }
    }

    // ---- the sequence's end, or the share's
    if (f + 1 == to || before[b + 1] == f + 1) {
      const size_t row = ((size_t)kv * (p.s.batch + p.n_shares) + b + c) * p.group;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], x);
        if (SPLIT)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            o[i][j] += __shfl_xor_sync(0xffffffffu, o[i][j], 2);
            o[i][2 + j] += __shfl_xor_sync(0xffffffffu, o[i][2 + j], 2);
          }
        const int h = 2 * t + j;
        if (h < p.group) {
          float* to_o = p.o + (row + h) * kRowDim + 16 * g;
#pragma unroll
          for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(to_o)[i] = make_float4(o[2 * i][j], o[2 * i][2 + j], o[2 * i + 1][j], o[2 * i + 1][2 + j]);
          if (g == 0) *reinterpret_cast<float2*>(p.ml + (row + h) * 2) = make_float2(ref[j], sum[j]);
        }
      }
      first = true;
    }
  }
}

// Joins the partial results of a query head, in the order of the chunks: WARPS warps, every WARPS-th result each, four columns a lane; eight of a warp's are on
// their way at a time (one after the other: 230 of a sequence of 65537 positions took 25 us).
template <int WARPS>
__global__ void __launch_bounds__(WARPS > 1 ? 32 * WARPS : 128) q4_join_kernel(const Q4DecodeParams p) {
  __shared__ float4 part[WARPS][32];
  __shared__ float2 part_ml[WARPS];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int i = WARPS > 1 ? blockIdx.x : 4 * blockIdx.x + warp, first = WARPS > 1 ? warp : 0;
  if (i >= p.s.batch * p.n_heads) return;
  const int b = i / p.n_heads, head = i - b * p.n_heads, kv = head / p.group;
  const int2 plan = p.plan[b];
  const size_t row0 = ((size_t)kv * (p.s.batch + p.n_shares) + b + plan.x) * p.group + head - kv * p.group;
  float top = -FLT_MAX, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int base = first; base < plan.y; base += 8 * WARPS) {
    float2 ml[8];
    float4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int piece = base + k * WARPS;
      const size_t row = row0 + (size_t)piece * p.group;
      ml[k] = make_float2(-FLT_MAX, 0.f);
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (piece < plan.y) {
        ml[k] = *reinterpret_cast<const float2*>(p.ml + row * 2);
        v[k] = *reinterpret_cast<const float4*>(p.o + row * kRowDim + 4 * lane);
      }
    }
    float to = top;
#pragma unroll
    for (int k = 0; k < 8; ++k) to = fmaxf(to, ml[k].x);
    const float f0 = ex2_ftz(top - to);
    top = to;
    l *= f0;
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] *= f0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float f = ex2_ftz(ml[k].x - to);
      l = fmaf(ml[k].y, f, l);
      o[0] = fmaf(v[k].x, f, o[0]);
      o[1] = fmaf(v[k].y, f, o[1]);
      o[2] = fmaf(v[k].z, f, o[2]);
      o[3] = fmaf(v[k].w, f, o[3]);
    }
  }
  if (WARPS > 1) {
    part[warp][lane] = make_float4(o[0], o[1], o[2], o[3]);
    if (lane == 0) part_ml[warp] = make_float2(top, l);
    __syncthreads();
    if (warp) return;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) top = fmaxf(top, part_ml[k].x);
    l = o[0] = o[1] = o[2] = o[3] = 0.f;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) {
      const float4 v = part[k][lane];
      const float f = ex2_ftz(part_ml[k].x - top);
      l = fmaf(part_ml[k].y, f, l);
      o[0] = fmaf(v.x, f, o[0]);
      o[1] = fmaf(v.y, f, o[1]);
      o[2] = fmaf(v.z, f, o[2]);
      o[3] = fmaf(v.w, f, o[3]);
    }
  }
  const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;                // (a NaN stays one)
  *reinterpret_cast<uint2*>(p.out + ((size_t)b * p.n_heads + head) * kRowDim + 4 * lane) =
      make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
}

}  // namespace tq

using namespace tq;

extern "C" int tq_gqa_decode_paged_q4(tq_ctx* ctx, const void* q_dev, const void* k_pages_dev, const void* v_pages_dev, const tq_pages* pages,
                                      const int* seqs_dev, size_t batch, size_t n_heads, size_t n_kv_heads, size_t head_dim, size_t max_len, void* out_dev) {
  if (int st = bind(ctx)) return st;
  if (batch == 0) return TQ_OK;
  if (int st = check_packed(ctx, "tq_gqa_decode_paged_q4", pages, seqs_dev, nullptr, batch, batch, n_kv_heads, head_dim, TQ_PAGES_Q4)) return st;
  TQ_REQUIRE(ctx, q_dev && k_pages_dev && v_pages_dev && out_dev, "tq_gqa_decode_paged_q4: null pointer");
  TQ_REQUIRE(ctx, n_heads % n_kv_heads == 0 && n_heads / n_kv_heads >= 1 && n_heads / n_kv_heads <= 8, "tq_gqa_decode_paged_q4: n_heads/n_kv_heads must be 1..8");
  TQ_REQUIRE(ctx, max_len > 0 && max_len <= (1u << 30), "tq_gqa_decode_paged_q4: max_len must bound the sequence lengths");
  TQ_REQUIRE(ctx, (((uintptr_t)q_dev | (uintptr_t)k_pages_dev | (uintptr_t)v_pages_dev | (uintptr_t)out_dev) & 15) == 0,
             "tq_gqa_decode_paged_q4: arrays must be 16-byte aligned");
  const size_t most = (size_t)pages->table_ld * pages->page_rows;
  Q4DecodeParams p;
  p.s = packed_seqs(pages, seqs_dev, nullptr, batch, batch);
  p.q = static_cast<const __nv_bfloat16*>(q_dev);
  p.k = static_cast<const uint8_t*>(k_pages_dev);
  p.v = static_cast<const uint8_t*>(v_pages_dev);
  p.row_bytes = q4_row_bytes(n_kv_heads);
  p.n_heads = (int)n_heads;
  p.n_kv = (int)n_kv_heads;
  p.group = (int)(n_heads / n_kv_heads);
  p.max_len = (int)(max_len < most ? max_len : most);
  p.scale_log2 = 1.44269504088896340736f / sqrtf((float)head_dim);
  p.out = static_cast<__nv_bfloat16*>(out_dev);
  p.err = ctx->dev_err;
  const size_t chunks = batch * (((size_t)p.max_len + kQdChunk - 1) / kQdChunk);
  TQ_REQUIRE(ctx, chunks < (1ull << 30), "tq_gqa_decode_paged_q4: too many positions");
  // All SMs' warps, or as many as there may be chunks.
  const size_t most_warps = (size_t)ctx->sm_count * kQdCtas * kQdWarps, shares = most_warps > n_kv_heads ? most_warps / n_kv_heads : 1;
  p.n_shares = (int)(shares < chunks ? shares : chunks);
  const size_t n_ctas = (p.n_shares * n_kv_heads + kQdWarps - 1) / kQdWarps, rows = (batch + p.n_shares) * n_heads;
  if (int st = ensure_scratch(ctx, rows * (kRowDim + 2) * sizeof(float) + batch * sizeof(int2))) return st;
  p.o = static_cast<float*>(ctx->scratch);
  p.ml = p.o + rows * kRowDim;
  p.plan = reinterpret_cast<int2*>(p.ml + rows * 2);
  if (int st = pages_use(ctx, pages)) return st;
  const size_t smem = kQdWarps * kQdStages * kQdStageBytes + (batch + 1) * sizeof(int), most_smem = kQdWarps * kQdStages * kQdStageBytes + (kPageCalls + 1) * sizeof(int);
  auto kern = p.group <= 4 ? q4_decode_kernel<true> : q4_decode_kernel<false>;
  TQ_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most_smem));
  TQ_CUDA(ctx, launch_k(ctx, kern, dim3((unsigned)n_ctas), dim3(32 * kQdWarps), smem, p));
  // A warp a query head where a sequence has few parts on the average (in CTAs of four heads), sixteen where it has many.  (From 16 on: 64 sequences of up to 4096
  // positions take 51.3 us, from 4 on 73.8; one of 700 8.6 and 8 of 8000 23.6, from 64 on 12.4 and 32.9.)
  const unsigned heads = (unsigned)(batch * n_heads);
  if ((size_t)p.n_shares > 16 * batch) TQ_CUDA(ctx, launch_k(ctx, q4_join_kernel<16>, dim3(heads), dim3(512), 0, p));
  else TQ_CUDA(ctx, launch_k(ctx, q4_join_kernel<1>, dim3((heads + 3) / 4), dim3(128), 0, p));
  return TQ_OK;
}
