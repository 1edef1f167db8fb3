// Rows of a cache of pages (include/tangq.h: tq_kv_append_paged, tq_kv_read_paged): the new tokens of several sequences go to their pages, with the
// rotation of queries and keys on the way (crates/tang-train/examples/smollm.rs:84-95 does it for one token and a cache of one sequence), and are read back.
// A cache row is bf16 or of 4 bits: s = the block's largest magnitude / 7, rounded up to 5 significant bits, an integer c = x / s rounded to nearest
// even, within -7 .. 7, and the value c s, which is a bf16 number (3 + 5 bits): what reads 4 bits multiplies the same numbers as what reads bf16.
#include "page_rows.cuh"

namespace tq {

constexpr int kAppendThreads = 128;

struct AppendParams {
  PackedSeqs s;
  const void* x;
  size_t ldx;
  const float *cos_t, *sin_t;
  int n_positions, n_heads, n_kv;
  __nv_bfloat16* q_out;
  uint8_t *k, *v;                      // cache rows of row_bytes
  size_t row_bytes;
  int* err;
};

// The scale of 32 values whose largest magnitude is amax.  Blocks below 2^-100 are zeros, those of 2^120 and above NaN: 24 s, which the readers
// form, is then a normal number.  A product with a number just below 1 / 7, rounded up to 5 bits, is the scale or, where amax / 7 is on the border, the number
// below it; seven times 5 bits are exact, and tell.
__device__ __forceinline__ float q4_scale(float amax) {
  if (!(amax < 1.329227995784916e36f)) return __uint_as_float(0x7FC00000u);
  if (amax < 7.888609052210118e-31f) return 0.f;
  const float s = __uint_as_float((__float_as_uint(amax * 0.14285707f) + 0x7FFFFu) & 0xFFF80000u);
  return 7.f * s < amax ? __uint_as_float(__float_as_uint(s) + 0x80000u) : s;
}

__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// The codes of eight values of a scale s, the first in the lowest four bits: 8 + x / s rounded to nearest even.  The quotient comes from the reciprocal with one
// correction by its remainder, which fused operations have exactly (Markstein, Computation of elementary functions on the IBM RISC System/6000 processor, 1990): 2^-46
// of it off before its last rounding.  s has 5 bits, a tie (k + 1/2) s nine at most, so that the f32 numbers beside a tie are 2^-24 (1 + 2^-9) of it away and their
// quotients do not round to one.  (The compiler's division instead: 5800 rows of 1024 keys and values from bf16 41.8 us.)  Adding 1.5 * 2^23 + 8 leaves the code in the
// number's low bits, and what else is in them is the same for all.
__device__ __forceinline__ uint32_t q4_codes(const float (&x)[8], float s) {
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  inv = __fmaf_rn(__fmaf_rn(-s, inv, 1.f), inv, inv);
  const uint64_t inv2 = pack2(inv, inv), less = pack2(-s, -s), up = pack2(12582920.f, 12582920.f);
  uint32_t word = 0, rest = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = j / 2 * 4 + j % 2;   // (and i + 2: the rotation's pairs)
    const uint64_t v = pack2(x[i], x[i + 2]), q = mul2(v, inv2);
    float a, b;
    unpack2(add2(fma2(fma2(q, less, v), inv2, q), up), a, b);
    word += (__float_as_uint(a) << (4 * i)) + (__float_as_uint(b) << (4 * i + 8));
    rest += (0x4B400000u << (4 * i)) + (0x4B400000u << (4 * i + 8));
  }
  return word - rest;
}

// A CTA takes ROWS rows and 128 eighths of a head: 32 bytes (f32) in, 16 or 4 out for a thread and row.  Rows' places are looked up by a warp each
// (starts, sequence, length, page, holders: five loads one after the other) while the values are on their way.  What bounds it: the bytes (5000 rows of 32 + 16
// heads f32 to bf16 pages, 200 MB, 35.0 us, 5.7 TB/s), beside the look-ups (CTAs of 256 threads 37.1, of 512 44.1; eight rows each 47.2); to 4 bits
// instructions and loads on their way, 73 % of the issue slots (5973 rows from bf16 31.7 us; 30 instead of 28 in an earlier form with single products and quotients, 32
// with two groups of columns a thread, for half as many look-ups; one warp's lanes for all rows' look-ups no difference).  With its reading back 38.8: in the earlier
// form four rows 37.0, two 39.2, three 37.7, four in shared memory by cp.async 39.0.  A single row 4.2 us.
template <typename X, int ROWS, bool Q4>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const AppendParams p) {
  __shared__ int place_s[ROWS], pos_s[ROWS];           // cache row (-1: none), position
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, m0 = blockIdx.x * ROWS;
  const int at = 8 * (blockIdx.y * kAppendThreads + threadIdx.x), width = (p.n_heads + 2 * p.n_kv) * kRowDim;   // value of the row
  uint4 raw[ROWS][sizeof(X) / 2];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
    if (at < width && m0 + r < p.s.rows) {
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const X*>(p.x) + (size_t)(m0 + r) * p.ldx + at);
#pragma unroll
      for (int i = 0; i < (int)sizeof(X) / 2; ++i) raw[r][i] = src[i];
    }
  if (warp < ROWS) {
    int place = -1, pos = 0;
    if (m0 + warp < p.s.rows) {
      const PackedRow row = packed_row(p.s, m0 + warp, lane, p.err);
      int why = 0, page = 0, same = 0;
      if (row.seq >= 0) {
        const int refused = p.s.refused[row.seq];      // (on its way beside the page)
        pos = row.pos;
        place = page_row_of(p.s, row.seq, pos, &page);
        if (place < 0 || pos >= p.n_positions) {
          why = DERR_POSITION;
        } else {
          // a position that is not the sequence's to write: the pool refused to make room, the page has other holders, or the sequence stands in the
          // list twice
          if (p.s.seqs)
#pragma unroll 4
            for (int j = lane; j < p.s.batch; j += 32) same += p.s.seqs[j] == row.seq;
          same = p.s.seqs ? (int)__reduce_add_sync(0xffffffffu, same) : 1;
          if (same != 1 || refused != 0 || p.s.refs[page] != 1) why = DERR_PAGE_LIST;
        }
      }
      if (why) {
        place = -1;
        if (lane == 0 && blockIdx.y == 0) atomicCAS(p.err, 0, why);
      }
    }
    if (lane == 0) {
      place_s[warp] = place;
      pos_s[warp] = pos;
    }
  }
  __syncthreads();
  const int head = at / kRowDim, d = at % kRowDim;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int place = place_s[r], pos = pos_s[r];
    if (place < 0) continue;           // (the whole CTA)
    float x[8];
    if (at < width) {
      if constexpr (sizeof(X) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(reinterpret_cast<const uint32_t*>(&raw[r][0])[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w = reinterpret_cast<const uint32_t*>(&raw[r][0])[i];
          x[2 * i] = __uint_as_float(w << 16);
          x[2 * i + 1] = __uint_as_float(w & 0xFFFF0000u);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
    }
    if (head < p.n_heads + p.n_kv) {
      const float4 c4 = *reinterpret_cast<const float4*>(p.cos_t + (size_t)pos * (kRowDim / 2) + d / 2);
      const float4 s4 = *reinterpret_cast<const float4*>(p.sin_t + (size_t)pos * (kRowDim / 2) + d / 2);
      const uint64_t cs[2] = {pack2(c4.x, c4.y), pack2(c4.z, c4.w)}, sn[2] = {pack2(s4.x, s4.y), pack2(s4.z, s4.w)};
      // Each product is rounded: which 4-bit integer a value becomes does not depend on how a compiler joins them.  It does join packed products with
      // packed sums, .rn or not (results a bit off), and leaves the single sums alone, which the bit-for-bit tests hold it to.
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const uint64_t x0 = pack2(x[i], x[i + 2]), x1 = pack2(x[i + 1], x[i + 3]), c = cs[i / 4], s = sn[i / 4];
        float a0, a1, b0, b1;
        unpack2(mul2(x0, c), a0, a1);
        unpack2(mul2(x1, s), b0, b1);
        x[i] = __fsub_rn(a0, b0), x[i + 2] = __fsub_rn(a1, b1);
        unpack2(mul2(x0, s), a0, a1);
        unpack2(mul2(x1, c), b0, b1);
        x[i + 1] = __fadd_rn(a0, b0), x[i + 3] = __fadd_rn(a1, b1);
      }
    }
    const bool key = head < p.n_heads + p.n_kv;
    const int kv_head = head - p.n_heads - (key ? 0 : p.n_kv);
    uint8_t* row = (key ? p.k : p.v) + (size_t)place * p.row_bytes;
    if constexpr (Q4) {
      if (__any_sync(0xffffffffu, head >= p.n_heads && at < width)) {  // (a warp of queries alone has nothing to do here)
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = max_or_nan(amax, fabsf(x[i]));
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) amax = max_or_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (head >= p.n_heads && at < width) {
          const float s = q4_scale(amax);
          *reinterpret_cast<uint32_t*>(row + kv_head * kQ4HeadBytes + d / 2) = s > 0.f ? q4_codes(x, s) : 0x88888888u;
          if (d % kQ4Block == 0) {
            uint16_t* to = reinterpret_cast<uint16_t*>(row + p.n_kv * kQ4HeadBytes) + kv_head * kQ4HeadScales;
            to[d / kQ4Block] = (uint16_t)(__float_as_uint(s) >> 16);
            if (kv_head == p.n_kv - 1 && (p.n_kv & 1) && d == 0) *reinterpret_cast<uint2*>(to + kQ4HeadScales) = make_uint2(0u, 0u);      // (the row's end)
          }
        }
      }
      if (head >= p.n_heads) continue;
    }
    if (at >= width) continue;
    __nv_bfloat16* dst = head < p.n_heads ? p.q_out + (size_t)(m0 + r) * p.n_heads * kRowDim + at : reinterpret_cast<__nv_bfloat16*>(row) + kv_head * kRowDim + d;
    uint4 o;
    __nv_bfloat162* pk = reinterpret_cast<__nv_bfloat162*>(&o);
#pragma unroll
    for (int i = 0; i < 4; ++i) pk[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(dst) = o;
  }
}

struct ReadParams {
  PackedSeqs s;
  const uint8_t *k, *v;
  size_t row_bytes;
  int n_kv;
  __nv_bfloat16 *k_out, *v_out;
  int* err;
};

// A CTA takes ROWS rows: eight values a thread and turn, keys and then values.  5973 rows of 8 heads from 4 bits, 31 MB, 8.3 us (a single row 4.2): start, look-up, loads and
// stores once each, too short for the memory's rate (4.8).
template <bool Q4, int ROWS>
__global__ void __launch_bounds__(kAppendThreads) kv_read_kernel(const ReadParams p) {
  __shared__ int place_s[ROWS];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, m0 = blockIdx.x * ROWS;
  if (warp < ROWS) {
    int place = -1;
    if (m0 + warp < p.s.rows) {
      const PackedRow row = packed_row(p.s, m0 + warp, lane, p.err);
      if (row.seq >= 0) place = page_row_of(p.s, row.seq, row.pos);
      if (row.seq >= 0 && place < 0 && lane == 0) atomicCAS(p.err, 0, (int)DERR_POSITION);
    }
    if (lane == 0) place_s[warp] = place;
  }
  __syncthreads();
  const int parts = p.n_kv * (kRowDim / 8);
  for (int i = threadIdx.x; i < 2 * parts; i += kAppendThreads) {
    const bool key = i < parts;
    const int part = key ? i : i - parts;
    const uint8_t* base = key ? p.k : p.v;
    __nv_bfloat16* to = (key ? p.k_out : p.v_out) + ((size_t)m0 * parts + part) * 8;
    if constexpr (Q4) {
      uint32_t w[ROWS];
      uint16_t s[ROWS];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const uint8_t* row = base + (size_t)max(place_s[r], 0) * p.row_bytes;
        w[r] = *reinterpret_cast<const uint32_t*>(row + 4 * part);
        s[r] = *reinterpret_cast<const uint16_t*>(row + p.n_kv * kQ4HeadBytes + 2 * (part / 4));
      }
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const uint32_t sc = s[r] * 0x10001u, off = bf16x2_mul(sc, 0xC1C0C1C0u);          // -24 s
        uint32_t a[4];
        dequant_q4_word_24(w[r], a);
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = bf16x2_fma(a[j], sc, off);
        if (place_s[r] >= 0)
          *reinterpret_cast<uint4*>(to + (size_t)r * parts * 8) =
              make_uint4(prmt(a[0], a[1], 0x5410), prmt(a[2], a[3], 0x5410), prmt(a[0], a[1], 0x7632), prmt(a[2], a[3], 0x7632));
      }
    } else {
      uint4 x[ROWS];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) x[r] = *reinterpret_cast<const uint4*>(base + (size_t)max(place_s[r], 0) * p.row_bytes + 16 * part);
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
        if (place_s[r] >= 0) *reinterpret_cast<uint4*>(to + (size_t)r * parts * 8) = x[r];
    }
  }
}

}  // namespace tq

using namespace tq;

extern "C" {

size_t tq_q4_row_bytes(size_t n_kv_heads) { return q4_row_bytes(n_kv_heads); }

int tq_kv_append_paged(tq_ctx* ctx, const void* x_dev, int x_dtype, size_t ldx, const float* cos_dev, const float* sin_dev, size_t n_positions,
                       const tq_pages* pages, const int* seqs_dev, const int* seq_rows_dev, size_t batch, size_t rows, size_t n_heads, size_t n_kv_heads,
                       size_t head_dim, void* q_out_dev, void* k_pages_dev, void* v_pages_dev, int page_rows_as) {
  if (int st = bind(ctx)) return st;
  if (batch == 0 || rows == 0) return TQ_OK;
  if (int st = check_packed(ctx, "tq_kv_append_paged", pages, seqs_dev, seq_rows_dev, batch, rows, n_kv_heads, head_dim, page_rows_as)) return st;
  TQ_REQUIRE(ctx, x_dev && cos_dev && sin_dev && q_out_dev && k_pages_dev && v_pages_dev, "tq_kv_append_paged: null pointer");
  TQ_REQUIRE(ctx, x_dtype == TQ_F32 || x_dtype == TQ_BF16, "tq_kv_append_paged: rows are f32 or bf16");
  TQ_REQUIRE(ctx, n_heads >= 1 && n_heads <= 65535, "tq_kv_append_paged: too many heads");
  const size_t width = (n_heads + 2 * n_kv_heads) * kRowDim;
  if (ldx == 0) ldx = width;
  TQ_REQUIRE(ctx, ldx >= width && ldx * dtype_size(x_dtype) % 16 == 0, "tq_kv_append_paged: rows stand a multiple of 16 bytes apart and do not overlap");
  TQ_REQUIRE(ctx, (((uintptr_t)x_dev | (uintptr_t)cos_dev | (uintptr_t)sin_dev | (uintptr_t)q_out_dev | (uintptr_t)k_pages_dev | (uintptr_t)v_pages_dev) & 15) == 0,
             "tq_kv_append_paged: arrays must be 16-byte aligned");
  TQ_REQUIRE(ctx, apart(x_dev, ((rows - 1) * ldx + width) * dtype_size(x_dtype), q_out_dev, rows * n_heads * kRowDim * 2),
             "tq_kv_append_paged: queries need a buffer of their own (they are stored while other rows are read)");
  TQ_REQUIRE(ctx, n_positions >= 1, "tq_kv_append_paged: tables of the rotation without positions");
  AppendParams p;
  p.s = packed_seqs(pages, seqs_dev, seq_rows_dev, batch, rows);
  p.x = x_dev;
  p.ldx = ldx;
  p.cos_t = cos_dev;
  p.sin_t = sin_dev;
  p.n_positions = (int)(n_positions < 0x7fffffff ? n_positions : 0x7fffffff);
  p.n_heads = (int)n_heads;
  p.n_kv = (int)n_kv_heads;
  p.q_out = static_cast<__nv_bfloat16*>(q_out_dev);
  p.k = static_cast<uint8_t*>(k_pages_dev);
  p.v = static_cast<uint8_t*>(v_pages_dev);
  const bool q4 = page_rows_as == TQ_PAGES_Q4;
  p.row_bytes = q4 ? q4_row_bytes(n_kv_heads) : n_kv_heads * kRowDim * 2;
  p.err = ctx->dev_err;
  if (int st = pages_use(ctx, pages)) return st;
  const unsigned parts = (unsigned)((width / 8 + kAppendThreads - 1) / kAppendThreads);
  // Four rows a CTA once that leaves a CTA for every SM.
  const size_t many = 4;
  const bool several = rows * parts >= many * (size_t)ctx->sm_count;
  const dim3 grid((unsigned)(several ? (rows + many - 1) / many : rows), parts), block(kAppendThreads);
  auto go = [&](auto kern) { return launch_k(ctx, kern, grid, block, 0, p); };
  if (x_dtype == TQ_F32) {
    TQ_CUDA(ctx, q4 ? (several ? go(kv_append_kernel<float, 4, true>) : go(kv_append_kernel<float, 1, true>))
                    : (several ? go(kv_append_kernel<float, 4, false>) : go(kv_append_kernel<float, 1, false>)));
  } else {
    using bf = __nv_bfloat16;
    TQ_CUDA(ctx, q4 ? (several ? go(kv_append_kernel<bf, 4, true>) : go(kv_append_kernel<bf, 1, true>))
                    : (several ? go(kv_append_kernel<bf, 4, false>) : go(kv_append_kernel<bf, 1, false>)));
  }
  return TQ_OK;
}

int tq_kv_read_paged(tq_ctx* ctx, const void* k_pages_dev, const void* v_pages_dev, int page_rows_as, const tq_pages* pages, const int* seqs_dev,
                     const int* seq_rows_dev, size_t batch, size_t rows, size_t n_kv_heads, size_t head_dim, void* k_out_dev, void* v_out_dev) {
  if (int st = bind(ctx)) return st;
  if (batch == 0 || rows == 0) return TQ_OK;
  if (int st = check_packed(ctx, "tq_kv_read_paged", pages, seqs_dev, seq_rows_dev, batch, rows, n_kv_heads, head_dim, page_rows_as)) return st;
  TQ_REQUIRE(ctx, k_pages_dev && v_pages_dev && k_out_dev && v_out_dev, "tq_kv_read_paged: null pointer");
  TQ_REQUIRE(ctx, (((uintptr_t)k_pages_dev | (uintptr_t)v_pages_dev | (uintptr_t)k_out_dev | (uintptr_t)v_out_dev) & 15) == 0,
             "tq_kv_read_paged: arrays must be 16-byte aligned");
  ReadParams p;
  p.s = packed_seqs(pages, seqs_dev, seq_rows_dev, batch, rows);
  p.k = static_cast<const uint8_t*>(k_pages_dev);
  p.v = static_cast<const uint8_t*>(v_pages_dev);
  const bool q4 = page_rows_as == TQ_PAGES_Q4;
  p.row_bytes = q4 ? q4_row_bytes(n_kv_heads) : n_kv_heads * kRowDim * 2;
  p.n_kv = (int)n_kv_heads;
  p.k_out = static_cast<__nv_bfloat16*>(k_out_dev);
  p.v_out = static_cast<__nv_bfloat16*>(v_out_dev);
  p.err = ctx->dev_err;
  if (int st = pages_use(ctx, pages)) return st;
  const bool four = rows >= 4 * (size_t)ctx->sm_count;
  auto kern = q4 ? (four ? kv_read_kernel<true, 4> : kv_read_kernel<true, 1>) : (four ? kv_read_kernel<false, 4> : kv_read_kernel<false, 1>);
  TQ_CUDA(ctx, launch_k(ctx, kern, dim3((unsigned)(four ? (rows + 3) / 4 : rows)), dim3(kAppendThreads), 0, p));
  return TQ_OK;
}

}  // extern "C"
