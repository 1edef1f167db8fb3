// Log probabilities of given tokens, entropy and the most likely tokens of rows of logits (include/tangq.h: tq_token_logprobs).  The
// reference has none; the softmax is that of Sampler::sample without its filters (crates/tang-infer/src/sampling.rs:119-142).
//
// With m the largest logit, c how many logits equal it and s the sum of exp(x - m) over the others,
//     log sum exp x = m + log c + log1p(s / c),      H = log c + log1p(s / c) + sum (m - x) exp(x - m) / (c + s),
// so that a model that is sure of a token (log probability and entropy near zero) loses nothing to the addition of the leading one.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <cfloat>

#include "common.cuh"
#include "internal.h"

namespace tq {

namespace cg = cooperative_groups;

constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpMaxTop = 64;
constexpr int kLpLoads = 4;            // 16-byte loads of a thread in flight, twice
constexpr int kLpGroups = kLpThreads / 4;
constexpr int kLpList = 512;           // candidates that a CTA sorts
constexpr int kLpMaxCluster = 8;
constexpr float kLpLog2e = 1.4426950408889634f;

struct LogprobParams {
  const void* x;                       // [slices][rows][ld]
  size_t ld;
  int slices, rows, cols, n_tokens, top;
  const int* tokens;                   // [rows][n_tokens] or null
  float *logprob, *entropy;            // [rows][n_tokens], [rows]
  int* top_ids;                        // [rows][top]
  float* top_logprob;
};

__device__ __forceinline__ float lp_float(float v) { return v; }
__device__ __forceinline__ float lp_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ const T* lp_slice(const LogprobParams& p, int row, int sl) {
  return static_cast<const T*>(p.x) + ((size_t)sl * p.rows + row) * p.ld;
}
template <typename T>
__device__ __forceinline__ float lp_at(const LogprobParams& p, int row, int i) {
  const int sl = i / p.cols;
  return lp_float(lp_slice<T>(p, row, sl)[i - sl * p.cols]);
}
__device__ __forceinline__ uint4 lp_load(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void lp_unpack(const uint4& v, float (&x)[4], float) {
  x[0] = __uint_as_float(v.x);
  x[1] = __uint_as_float(v.y);
  x[2] = __uint_as_float(v.z);
  x[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void lp_unpack(const uint4& v, float (&x)[8], __nv_bfloat16) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ float lp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// (larger value, else lower index)
__device__ __forceinline__ bool lp_before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

// Part of a row: its largest logit m, how many equal it, the sum of exp(x - m) over the others, and sum (m - x) exp(x - m).
struct LpState {
  float m = -INFINITY, c = 0.f, s = 0.f, u = 0.f;

  __device__ __forceinline__ void rise(float to) {      // to >= m
    if (to > m) {
      const float f = m == -INFINITY ? 0.f : lp_ex2((m - to) * kLpLog2e);
      u = f == 0.f && u == u ? 0.f : f * (u + (to - m) * (c + s));
      s = m == -INFINITY ? s * 0.f : f * (s + c);       // (a NaN stays one)
      c = 0.f;
      m = to;
    }
  }
  template <bool ENT, int N>
  __device__ __forceinline__ void add(const float (&x)[N]) {
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = x[i] - base, e = lp_ex2(d * kLpLog2e);
      if (x[i] == m) c += 1.f;
      else s += e;
      if (ENT) u = fmaf(fmaxf(d, -1e4f), -e, u);        // (e is 0 there, and -infinity times that is not)
    }
  }
};

// The elements first .. end-1 of a segment that this thread takes: up to one before the first 16-byte boundary, every 512th 16 bytes, up to one
// behind the last.
template <typename T>
struct LpSegment {
  static constexpr int N = 16 / (int)sizeof(T);
  const T* base;
  int head, vecs, tail0, n;            // elements before the vectors, vectors, first element behind them, all
  __device__ __forceinline__ LpSegment(const T* b, int count) : base(b), n(count) {
    head = min(n, (int)((16 - ((uintptr_t)b & 15)) & 15) / (int)sizeof(T));
    vecs = (n - head) / N;
    tail0 = head + vecs * N;
  }
};

template <typename T, bool ENT>
__global__ void __launch_bounds__(kLpThreads, 2) token_logprobs_kernel(const LogprobParams p) {
  constexpr int N = LpSegment<T>::N;
  __shared__ float red[4][kLpWarps];
  __shared__ float4 part;              // this CTA's state
  __shared__ __align__(16) float group_max[kLpGroups];
  __shared__ float thr_s;
  __shared__ int n_above, n_equal;
  __shared__ float list_v[kLpList];    // above the threshold
  __shared__ int list_i[kLpList], equal_i[kLpList];
  __shared__ float top_v[kLpMaxTop];   // this CTA's largest, in order
  __shared__ int top_i[kLpMaxTop];
  __shared__ float all_v[kLpMaxCluster * kLpMaxTop];
  __shared__ int all_i[kLpMaxCluster * kLpMaxTop];
  pdl_wait();
  pdl_launch_dependents();
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = (int)(blockIdx.x / C), t = threadIdx.x, warp = t >> 5, lane = t & 31, V = p.slices * p.cols, top = p.top;
  const int lo = (int)((long long)V * rank / C) & ~63, hi = rank == C - 1 ? V : (int)((long long)V * (rank + 1) / C) & ~63;
  int token = -1;
  float token_x = 0.f;
  if (rank == 0 && t < p.n_tokens) {   // (on their way while the row is read)
    token = p.tokens[(size_t)row * p.n_tokens + t];
    if (token >= 0 && token < V) token_x = lp_at<T>(p, row, token);
  }

  // ---- one pass: maximum and sums of this thread's elements
  LpState a;
  for (int at = lo; at < hi;) {
    const int sl = at / p.cols, in = at - sl * p.cols, n = min(hi - at, p.cols - in);
    const LpSegment<T> g(lp_slice<T>(p, row, sl) + in, n);
    const uint4 none = sizeof(T) == 4 ? make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u) : make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u);
    uint4 v[kLpLoads];
    auto fetch = [&](int first) {
#pragma unroll
      for (int k = 0; k < kLpLoads; ++k) {
        const int i = first + k * kLpThreads + t;
        v[k] = i < g.vecs ? lp_load(g.base + g.head + i * N) : none;
      }
    };
    fetch(0);
    if (t < g.head || g.tail0 + t < n) {               // (both at most 7 elements)
      float x[2] = {-INFINITY, -INFINITY};
      if (t < g.head) x[0] = lp_float(g.base[t]);
      if (g.tail0 + t < n) x[1] = lp_float(g.base[g.tail0 + t]);
      a.rise(fmaxf(a.m, fmaxf(x[0], x[1])));
      a.template add<ENT>(x);
    }
    for (int first = 0; first < g.vecs; first += kLpLoads * kLpThreads) {
      uint4 w[kLpLoads];
#pragma unroll
      for (int k = 0; k < kLpLoads; ++k) w[k] = v[k];
      if (first + kLpLoads * kLpThreads < g.vecs) fetch(first + kLpLoads * kLpThreads);
#pragma unroll
      for (int k = 0; k < kLpLoads; ++k) {
        float x[N];
        lp_unpack(w[k], x, T());
        float mx = x[0];
#pragma unroll
        for (int i = 1; i < N; ++i) mx = fmaxf(mx, x[i]);
        a.rise(fmaxf(a.m, mx));
        a.template add<ENT>(x);
      }
    }
    at += n;
  }
  const float mine = a.m;

  // ---- the CTA's state: lanes, then warps
  auto meet_warp = [&](LpState& st) {
    const float m = warp_max(st.m);
    st.rise(m);
    st.c = warp_sum(st.c);
    st.s = warp_sum(st.s);
    if (ENT) st.u = warp_sum(st.u);
  };
  meet_warp(a);
  if (lane == 0) {
    red[0][warp] = a.m;
    red[1][warp] = a.c;
    red[2][warp] = a.s;
    red[3][warp] = a.u;
  }
  if (top) {
    const float g2 = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, 1)), g4 = fmaxf(g2, __shfl_xor_sync(0xffffffffu, g2, 2));
    if ((t & 3) == 0) group_max[t >> 2] = g4;
    if (t == 0) n_above = n_equal = 0;
    if (t < kLpMaxTop) top_i[t] = 0x7fffffff;
  }
  __syncthreads();
  if (warp == 0) {
    LpState b;
    if (lane < kLpWarps) {
      b.m = red[0][lane];
      b.c = red[1][lane];
      b.s = red[2][lane];
      b.u = red[3][lane];
    }
    meet_warp(b);
    if (lane == 0) part = make_float4(b.m, b.c, b.s, b.u);
  }

  // ---- the CTA's `top` largest.  The top-th largest of the 128 groups' maxima is a lower bound of the top-th largest element: few elements are above
  // it, and only the threads whose own maximum reaches it have any.
  if (top) {
    if (t >= kLpThreads - kLpGroups) {
      const int me = t - (kLpThreads - kLpGroups);
      const float v = group_max[me];
      int before = 0;
#pragma unroll 8
      for (int j = 0; j < kLpGroups / 4; ++j) {
        const float4 w = reinterpret_cast<const float4*>(group_max)[j];
        before += lp_before(w.x, 4 * j, v, me) + lp_before(w.y, 4 * j + 1, v, me) + lp_before(w.z, 4 * j + 2, v, me) + lp_before(w.w, 4 * j + 3, v, me);
      }
      if (before == top - 1) thr_s = v;
    }
    __syncthreads();
    const float thr = thr_s;
    if (mine >= thr) {
      auto offer = [&](float x, int i) {
        if (x > thr) {
          const int k = atomicAdd(&n_above, 1);
          if (k < kLpList) {
            list_v[k] = x;
            list_i[k] = i;
          }
        } else if (x == thr) {
          const int k = atomicAdd(&n_equal, 1);
          if (k < kLpList) equal_i[k] = i;
        }
      };
      for (int at = lo; at < hi;) {
        const int sl = at / p.cols, in = at - sl * p.cols, n = min(hi - at, p.cols - in);
        const LpSegment<T> g(lp_slice<T>(p, row, sl) + in, n);
        if (t < g.head) offer(lp_float(g.base[t]), at + t);
        if (g.tail0 + t < n) offer(lp_float(g.base[g.tail0 + t]), at + g.tail0 + t);
#pragma unroll 4
        for (int i = t; i < g.vecs; i += kLpThreads) {
          float x[N];
          lp_unpack(lp_load(g.base + g.head + i * N), x, T());
          float mx = x[0];
#pragma unroll
          for (int j = 1; j < N; ++j) mx = fmaxf(mx, x[j]);
          if (mx >= thr)
#pragma unroll
            for (int j = 0; j < N; ++j) offer(x[j], at + g.head + i * N + j);
        }
        at += n;
      }
    }
    __syncthreads();
    const int above = n_above, equal = n_equal;
    if (above <= kLpList) {
      for (int i = t; i < above; i += kLpThreads) {
        const float v = list_v[i];
        const int id = list_i[i];
        int before = 0;
        for (int j = 0; j < above; ++j) before += lp_before(list_v[j], list_i[j], v, id);
        if (before < top) {
          top_v[before] = v;
          top_i[before] = id;
        }
      }
      const int want = top - above;
      if (want > 0 && equal <= kLpList) {
        for (int i = t; i < equal; i += kLpThreads) {
          const int id = equal_i[i];
          int before = 0;
          for (int j = 0; j < equal; ++j) before += equal_i[j] < id;
          if (before < want) {
            top_v[above + before] = thr;
            top_i[above + before] = id;
          }
        }
      } else if (want > 0) {
        // many equal ones: the first of them in the order of the row
        int found = 0;
        for (int base = lo; base < hi && found < want; base += kLpThreads) {
          const bool hit = base + t < hi && lp_at<T>(p, row, base + t) == thr;
          const unsigned ballot = __ballot_sync(0xffffffffu, hit);
          __syncthreads();
          if (lane == 0) list_i[warp] = __popc(ballot);
          __syncthreads();
          int at = found + __popc(ballot & ((1u << lane) - 1u));
          for (int w = 0; w < kLpWarps; ++w) {
            at += w < warp ? list_i[w] : 0;
            found += list_i[w];
          }
          if (hit && at < want) {
            top_v[above + at] = thr;
            top_i[above + at] = base + t;
          }
        }
      }
    } else {
      // more above the bound than the list holds (they sit in few threads' elements): the next in order, one after the other
      float last_v = INFINITY;
      int last_i = -1;
      for (int k = 0; k < top; ++k) {
        float bv = -INFINITY;
        int bi = 0x7fffffff;
        auto meet = [&](float v, int i) {
          if (i != 0x7fffffff && (bi == 0x7fffffff || lp_before(v, i, bv, bi))) {
            bv = v;
            bi = i;
          }
        };
        for (int i = lo + t; i < hi; i += kLpThreads) {
          const float v = lp_at<T>(p, row, i);
          if (v == v && lp_before(last_v, last_i, v, i)) meet(v, i);
        }
        for (int o = 16; o > 0; o >>= 1) {
          const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
          const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
          meet(ov, oi);
        }
        __syncthreads();
        if (lane == 0) {
          list_v[warp] = bv;
          list_i[warp] = bi;
        }
        __syncthreads();
        for (int w = 0; w < kLpWarps; ++w) meet(list_v[w], list_i[w]);
        if (t == 0) {
          top_v[k] = bv;
          top_i[k] = bi;
        }
        last_v = bv;
        last_i = bi;
      }
    }
  }

  // ---- the row: the first CTA of the cluster reads the others' states and lists
  if (C > 1) cluster.sync();
  else __syncthreads();
  if (rank == 0) {
    LpState r;
    {
      float4 q[kLpMaxCluster];
#pragma unroll
      for (int k = 0; k < kLpMaxCluster; ++k)
        if (k < C) q[k] = C > 1 ? *cluster.map_shared_rank(&part, k) : part;
#pragma unroll
      for (int k = 0; k < kLpMaxCluster; ++k)
        if (k < C) r.m = fmaxf(r.m, q[k].x);
      const float m = r.m;
#pragma unroll
      for (int k = 0; k < kLpMaxCluster; ++k) {
        if (k >= C) break;
        LpState b;
        b.m = q[k].x;
        b.c = q[k].y;
        b.s = q[k].z;
        b.u = q[k].w;
        b.rise(m);
        r.c += b.c;
        r.s += b.s;
        r.u += b.u;
      }
    }
    float log_s = logf(r.c) + log1pf(r.s / r.c), h = log_s + r.u / (r.c + r.s);
    if (r.m == -INFINITY) log_s = h = r.s;             // no logit at all (0: nothing has a probability), or a NaN
    if (r.m == INFINITY) log_s = h = NAN;
    auto logprob = [&](float v) { return v == -INFINITY && log_s == log_s ? -INFINITY : (v - r.m) - log_s; };
    if (ENT && t == 0 && p.entropy) p.entropy[row] = h;
    if (t < p.n_tokens) p.logprob[(size_t)row * p.n_tokens + t] = token < 0 ? 0.f : token >= V ? NAN : logprob(token_x);
    for (int j = t + kLpThreads; j < p.n_tokens; j += kLpThreads) {
      const int tok = p.tokens[(size_t)row * p.n_tokens + j];
      p.logprob[(size_t)row * p.n_tokens + j] = tok < 0 ? 0.f : tok >= V ? NAN : logprob(lp_at<T>(p, row, tok));
    }
    if (top) {
      if (C == 1) {
        if (t < top) {
          const int id = top_i[t];
          p.top_ids[(size_t)row * top + t] = id == 0x7fffffff ? -1 : id;
          p.top_logprob[(size_t)row * top + t] = id == 0x7fffffff ? NAN : logprob(top_v[t]);
        }
      } else {
        const int all = C * top;
        for (int i = t; i < all; i += kLpThreads) {
          const int k = i / top, j = i - k * top;
          all_i[i] = *cluster.map_shared_rank(&top_i[j], k);
          all_v[i] = *cluster.map_shared_rank(&top_v[j], k);
        }
        __syncthreads();
        int have = 0;
        for (int i = t; i < all; i += kLpThreads) {
          const int id = all_i[i];
          if (id == 0x7fffffff) continue;
          const float v = all_v[i];
          int before = 0;
          for (int j = 0; j < all; ++j) before += all_i[j] != 0x7fffffff && lp_before(all_v[j], all_i[j], v, id);
          if (before < top) {
            p.top_ids[(size_t)row * top + before] = id;
            p.top_logprob[(size_t)row * top + before] = logprob(v);
          }
          ++have;
        }
        if (t < top) {                                 // (fewer numbers than places)
          have = 0;
          for (int j = 0; j < all; ++j) have += all_i[j] != 0x7fffffff;
          if (t >= have) {
            p.top_ids[(size_t)row * top + t] = -1;
            p.top_logprob[(size_t)row * top + t] = NAN;
          }
        }
      }
    }
  }
  if (C > 1) cluster.sync();           // (nobody leaves while its memory is read)
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
  // CTAs of a row (a cluster): as many as keep the GPU's CTA slots (two an SM) filled, none with less than 2048 logits.
  const size_t V = slices * cols;
  int C = 1;
  while (C < kLpMaxCluster && rows * C < 4 * (size_t)ctx->sm_count && V / (2 * C) >= 2048) C *= 2;
  const bool ent = entropy_out_dev != nullptr;
  auto kern = dtype == TQ_BF16 ? (ent ? token_logprobs_kernel<__nv_bfloat16, true> : token_logprobs_kernel<__nv_bfloat16, false>)
                               : (ent ? token_logprobs_kernel<float, true> : token_logprobs_kernel<float, false>);
  TQ_REQUIRE(ctx, rows < (size_t)(0x7fffffff / kLpMaxCluster), "tq_token_logprobs: too many rows");
  TQ_CUDA(ctx, launch_k_cluster(ctx, kern, dim3((unsigned)(rows * C)), dim3(kLpThreads), 0, dim3((unsigned)C), p));
  return TQ_OK;
}
