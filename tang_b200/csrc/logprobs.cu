// Log probabilities of given tokens, entropy and the most likely tokens of rows of logits (include/tangq.h: tq_token_logprobs).  The
// reference has none; the softmax is that of Sampler::sample without its filters (crates/tang-infer/src/sampling.rs:119-142).
//
// With m the largest logit, c how many logits equal it and s the sum of exp(x - m) over the others,
//     log sum exp x = m + log c + log1p(s / c),      H = log c + log1p(s / c) + sum (m - x) exp(x - m) / (c + s),
// so that a model that is sure of a token (log probability and entropy near zero) loses nothing to the addition of the leading one.
#include <cuda_bf16.h>

#include <cfloat>

#include "common.cuh"
#include "internal.h"

namespace tq {

constexpr int kLpThreads = 512;
constexpr int kLpMaxTop = 64;

struct LogprobParams {
  const void* x;                       // [slices][rows][ld] f32 or bf16
  int bf16;
  size_t ld;
  int slices, rows, cols, n_tokens, top;
  const int* tokens;                   // [rows][n_tokens] or null
  float *logprob, *entropy;            // [rows][n_tokens], [rows]
  int* top_ids;                        // [rows][top]
  float* top_logprob;
};

__device__ __forceinline__ float lp_at(const LogprobParams& p, int row, int i) {
  const int sl = i / p.cols;
  const size_t at = ((size_t)sl * p.rows + row) * p.ld + (i - sl * p.cols);
  return p.bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.x)[at]) : static_cast<const float*>(p.x)[at];
}

// (larger value, else lower index); a value that is not a number loses to everything
struct LpBest {
  float v;
  int i;
};
__device__ __forceinline__ bool lp_before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

__global__ void __launch_bounds__(kLpThreads) token_logprobs_kernel(const LogprobParams p) {
  __shared__ float red[3][kLpThreads / 32];
  __shared__ float best_v[kLpThreads / 32];
  __shared__ int best_i[kLpThreads / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.x, t = threadIdx.x, warp = t >> 5, lane = t & 31, V = p.slices * p.cols;
  constexpr int W = kLpThreads / 32;
  float m = -INFINITY;
  bool nan = false;
  for (int i = t; i < V; i += kLpThreads) {
    const float v = lp_at(p, row, i);
    nan = nan || v != v;
    m = fmaxf(m, v);
  }
  m = warp_max(m);
  if (lane == 0) red[0][warp] = m;
  nan = __syncthreads_or(nan);
  for (int w = 0; w < W; ++w) m = fmaxf(m, red[0][w]);
  __syncthreads();
  float s = 0.f, u = 0.f, c = 0.f;
  for (int i = t; i < V; i += kLpThreads) {
    const float v = lp_at(p, row, i), d = v - m;
    if (v == m) {
      c += 1.f;
    } else if (d > -INFINITY) {
      const float e = expf(d);
      s += e;
      u -= d * e;
    }
  }
  s = warp_sum(s);
  u = warp_sum(u);
  c = warp_sum(c);
  if (lane == 0) {
    red[0][warp] = s;
    red[1][warp] = u;
    red[2][warp] = c;
  }
  __syncthreads();
  s = u = c = 0.f;
  for (int w = 0; w < W; ++w) {
    s += red[0][w];
    u += red[1][w];
    c += red[2][w];
  }
  float log_s = logf(c) + log1pf(s / c), h = log_s + u / (c + s);
  if (m == -INFINITY) log_s = h = 0.f;                 // no logit at all: nothing has a probability
  if (nan || m == INFINITY) log_s = h = NAN;
  auto logprob = [&](float v) { return v == -INFINITY && log_s == log_s ? -INFINITY : (v - m) - log_s; };
  if (t == 0 && p.entropy) p.entropy[row] = h;
  for (int j = t; j < p.n_tokens; j += kLpThreads) {
    const int tok = p.tokens[(size_t)row * p.n_tokens + j];
    p.logprob[(size_t)row * p.n_tokens + j] = tok < 0 ? 0.f : tok >= V ? NAN : logprob(lp_at(p, row, tok));
  }
  float last_v = INFINITY;
  int last_i = -1;
  for (int k = 0; k < p.top; ++k) {
    float bv = -INFINITY;
    int bi = 0x7fffffff;
    for (int i = t; i < V; i += kLpThreads) {
      const float v = lp_at(p, row, i);
      if (v == v && lp_before(last_v, last_i, v, i) && (bi == 0x7fffffff || lp_before(v, i, bv, bi))) {
        bv = v;
        bi = i;
      }
    }
    auto meet = [&](float v, int i) {
      if (i != 0x7fffffff && (bi == 0x7fffffff || lp_before(v, i, bv, bi))) {
        bv = v;
        bi = i;
      }
    };
    for (int o = 16; o > 0; o >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
      const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
      meet(ov, oi);
    }
    __syncthreads();
    if (lane == 0) {
      best_v[warp] = bv;
      best_i[warp] = bi;
    }
    __syncthreads();
    for (int w = 0; w < W; ++w) meet(best_v[w], best_i[w]);
    if (t == 0) {
      p.top_ids[(size_t)row * p.top + k] = bi == 0x7fffffff ? -1 : bi;
      p.top_logprob[(size_t)row * p.top + k] = bi == 0x7fffffff ? NAN : logprob(bv);
    }
    last_v = bv;
    last_i = bi;
  }
}

}  // namespace tq

using namespace tq;

extern "C" int tq_token_logprobs(tq_ctx* ctx, const void* logits_dev, int dtype, size_t ld, size_t slices, size_t rows, size_t cols, const int* tokens_dev,
                                 size_t n_tokens, size_t top, float* logprob_out_dev, float* entropy_out_dev, int* top_ids_out_dev,
                                 float* top_logprob_out_dev) {
  if (int st = bind(ctx)) return st;
  if (rows == 0) return TQ_OK;
  TQ_REQUIRE(ctx, logits_dev != nullptr && slices > 0 && cols > 0, "tq_token_logprobs: null pointer or empty vocabulary");
  TQ_REQUIRE(ctx, dtype == TQ_F32 || dtype == TQ_BF16, "tq_token_logprobs: logits must be f32 or bf16");
  TQ_REQUIRE(ctx, slices < (1u << 16) && cols < (1ull << 31) && slices * cols < (1ull << 31) && rows < (1ull << 31), "tq_token_logprobs: vocabulary or rows too large");
  if (ld == 0) ld = cols;
  TQ_REQUIRE(ctx, ld >= cols, "tq_token_logprobs: rows overlap");
  TQ_REQUIRE(ctx, ((uintptr_t)logits_dev & (dtype == TQ_F32 ? 3 : 1)) == 0, "tq_token_logprobs: logits are not aligned to their type");
  TQ_REQUIRE(ctx, n_tokens == 0 || (tokens_dev && logprob_out_dev && n_tokens < (1u << 20)), "tq_token_logprobs: given tokens need their ids and a place for the results");
  TQ_REQUIRE(ctx, top <= (size_t)kLpMaxTop && top <= slices * cols, "tq_token_logprobs: at most %d of the most likely tokens, and no more than there are", kLpMaxTop);
  TQ_REQUIRE(ctx, top == 0 || (top_ids_out_dev && top_logprob_out_dev), "tq_token_logprobs: the most likely tokens need places for ids and log probabilities");
  LogprobParams p;
  p.x = logits_dev;
  p.bf16 = dtype == TQ_BF16;
  p.ld = ld;
  p.slices = (int)slices;
  p.rows = (int)rows;
  p.cols = (int)cols;
  p.n_tokens = (int)n_tokens;
  p.top = (int)top;
  p.tokens = tokens_dev;
  p.logprob = logprob_out_dev;
  p.entropy = entropy_out_dev;
  p.top_ids = top_ids_out_dev;
  p.top_logprob = top_logprob_out_dev;
  TQ_CUDA(ctx, launch_k(ctx, token_logprobs_kernel, dim3((unsigned)rows), dim3(kLpThreads), 0, p));
  return TQ_OK;
}
