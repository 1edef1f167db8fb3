// Log probabilities of given tokens, entropy and the most likely tokens of rows of logits (include/tangq.h: tq_token_logprobs).  The
// reference has none; the softmax is that of Sampler::sample without its filters (crates/tang-infer/src/sampling.rs:119-142).
//
// With m the largest logit, c how many logits equal it and s the sum of exp(x - m) over the others,
//     log sum exp x = m + log c + log1p(s / c),      H = log c + log1p(s / c) + sum (m - x) exp(x - m) / (c + s),
// so that a model that is sure of a token (log probability and entropy near zero) loses nothing to the addition of the leading one.
//
// What bounds it: the logits' bytes where rows are many (1024 x 128256 f32 79 us, 6.6 TB/s; as many bytes of bf16 85 us, 6.2 TB/s, where
// every logit costs an exponential, a share of a maximum and half an addition and multiplication; from a graph over six inputs: calls from Python over one
// input take 93 to 98); the latency of the launch, the
// cluster's meeting and, with alternatives, of sorting 128 maxima where they are few (one row of 32000 4.0 us, 6.6 with five alternatives).
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <cfloat>

#include "common.cuh"
#include "internal.h"

namespace tq {

namespace cg = cooperative_groups;

constexpr int kLpThreads = 256, kLpPerSm = 4;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpMaxTop = 64;
constexpr int kLpLoads = 4;            // 16-byte loads of a thread in flight, twice
constexpr int kLpGroups = 128;         // of neighbouring threads; four warps sort their maxima
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
__device__ __forceinline__ void lp_set(uint32_t& w, float v) { w = __float_as_uint(v); }
__device__ __forceinline__ void lp_set(uint32_t& w, __nv_bfloat16 v) { w = (w & 0xFFFF0000u) | __bfloat16_as_ushort(v); }
__device__ __forceinline__ float lp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two f32 operations of one instruction.
__device__ __forceinline__ unsigned long long lp_pair(float x, float y) {
  unsigned long long r;
  asm("mov.b64 %0, {%1,%2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 lp_split(unsigned long long v) {
  float2 r;
  asm("mov.b64 {%0,%1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ unsigned long long lp_fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long lp_add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The cluster's barrier, in the forms that ask nothing of where a warp's lanes are: they come from branches.
__device__ __forceinline__ void lp_cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void lp_cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// The largest of 16 bytes of logits (NaN is none of them); bf16 by pairs.
__device__ __forceinline__ float lp_largest(const uint4& v, float) {
  return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
}
__device__ __forceinline__ __nv_bfloat162 lp_largest2(const uint4& v) {
  return __hmax2(__hmax2(reinterpret_cast<const __nv_bfloat162&>(v.x), reinterpret_cast<const __nv_bfloat162&>(v.y)),
                 __hmax2(reinterpret_cast<const __nv_bfloat162&>(v.z), reinterpret_cast<const __nv_bfloat162&>(v.w)));
}
__device__ __forceinline__ float lp_largest(const uint4& v, __nv_bfloat16) {
  const __nv_bfloat162 m = lp_largest2(v);
  return fmaxf(__low2float(m), __high2float(m));
}
template <int K>
__device__ __forceinline__ float lp_largest(const uint4 (&v)[K], float) {
  float m = lp_largest(v[0], 0.f);
#pragma unroll
  for (int k = 1; k < K; ++k) m = fmaxf(m, lp_largest(v[k], 0.f));
  return m;
}
template <int K>
__device__ __forceinline__ float lp_largest(const uint4 (&v)[K], __nv_bfloat16) {
  __nv_bfloat162 m = lp_largest2(v[0]);
#pragma unroll
  for (int k = 1; k < K; ++k) m = __hmax2(m, lp_largest2(v[k]));
  return fmaxf(__low2float(m), __high2float(m));
}

// Larger for a larger logit and, among equals (the zeros too), for a lower index; 0 is nobody's.
__device__ __forceinline__ unsigned long long lp_key(float v, int i) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return (unsigned long long)(b >> 31 ? ~b : b | 0x80000000u) << 32 | (0xFFFFFFFFu - (uint32_t)i);
}
__device__ __forceinline__ float lp_key_value(unsigned long long k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float(o >> 31 ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ int lp_key_index(unsigned long long k) { return (int)(0xFFFFFFFFu - (uint32_t)k); }

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
};

// What a thread has read.  Exponents are fma(x, log2 e, -base), one instruction instead of the two of (x - b) log2 e, with base = b log2 e rounded and
// b the largest logit of the warp's first batch: it only moves where a batch goes kLpSlack beyond it, so that the loop needs no maximum but the
// thread's own.  What the rounding of base adds to every exponent alike, `off`, is taken out at the end (it would be too large from |b| = 2^20 on:
// there, and before anything but -infinity was seen, the two instructions are used).
// The 16 bytes with the thread's largest logit are held back: the row's largest must not be added before it is known (the sum of the others would be
// lost against it where a model is sure).  Where another vector has the same one, that is among s, which is no loss there.  Without alternatives it is
// enough to do so where a batch goes beyond what the warp has seen (2048 rows of 128256 bf16 91 -> 86 us, with entropies 98 -> 94); f32 with entropies has
// each thread look after its own all the same (256 rows 23.2 us, the other way 24.0).
constexpr float kLpSlack = 20.f;
template <typename T, bool ENT, bool TOP>
struct LpRunning {
  static constexpr int N = 16 / (int)sizeof(T);
  static constexpr bool EACH = TOP || (ENT && sizeof(T) == 4);
  static constexpr uint32_t kNone = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;        // -infinity
  float b = -INFINITY, base = 0.f, off = 0.f;
  unsigned long long s = 0, u = 0;                      // two sums each, of even and of odd places; u: of exponent * exponential
  float warps = -INFINITY;                              // the largest that the warp has read
  float mine = -INFINITY, second = -INFINITY;           // the largest of `held` and of all other vectors
  uint4 held = make_uint4(kNone, kNone, kNone, kNone);
  int where = -1;                                       // the row's place of its first logit (-1: not 16 bytes of the row)

  static __device__ __forceinline__ uint4 none() { return make_uint4(kNone, kNone, kNone, kNone); }
  __device__ __forceinline__ bool far() const { return !(fabsf(b) <= 1048576.f); }
  __device__ __forceinline__ void take(float a0, float a1) {
    const unsigned long long e = lp_pair(lp_ex2(a0), lp_ex2(a1));
    s = lp_add2(s, e);
    if (ENT) u = lp_fma2(lp_pair(fmaxf(a0, -1e4f), fmaxf(a1, -1e4f)), e, u);             // (e is 0 there, and -infinity times that is not)
  }
  // K vectors, the first of them at place `at` of the row and the others `step` apart (-1: nowhere)
  template <int K>
  __device__ __forceinline__ void add(uint4 (&v)[K], int at, int step) {
    float top = -INFINITY;
    auto hold = [&](int k, float mx) {
      if (mx > mine) {                                  // (selects, no branch)
        const uint4 w = held;
        held = v[k];
        v[k] = w;
        mine = mx;
        if (TOP) where = at < 0 ? -1 : at + k * step;
      }
    };
    if constexpr (EACH) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const float mx = lp_largest(v[k], T());
        top = fmaxf(top, mx);
        if (TOP) second = fmaxf(second, fminf(mx, mine));
        hold(k, mx);
      }
    } else {
      top = lp_largest(v, T());
    }
    // (the warp's largest rises a few times in a row: 3.4 of 16 batches)
    if (__any_sync(0xffffffffu, top > (EACH ? b + kLpSlack : warps))) {
      if constexpr (!EACH)
#pragma unroll
        for (int k = 0; k < K; ++k) hold(k, lp_largest(v[k], T()));
      warps = fmaxf(warps, warp_max(top));
      if (warps > b + kLpSlack) {
        const float was = b, off_was = off;
        b = warps;
        base = far() ? 0.f : b * kLpLog2e;
        off = far() ? 0.f : fmaf(b, kLpLog2e, -base);
        if (was != -INFINITY) {
          const float by = fmaxf((was - b) * kLpLog2e - off_was + off, -1e4f), f = lp_ex2(by);
          const unsigned long long f2 = lp_pair(f, f);
          if (ENT) u = lp_fma2(lp_fma2(lp_pair(by, by), s, u), f2, 0ull);
          s = lp_fma2(s, f2, 0ull);
        }
      }
    }
    if (!far()) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float x[N];
        lp_unpack(v[k], x, T());
#pragma unroll
        for (int i = 0; i < N; i += 2) {
          const float2 a = lp_split(lp_fma2(lp_pair(x[i], x[i + 1]), lp_pair(kLpLog2e, kLpLog2e), lp_pair(-base, -base)));
          take(a.x, a.y);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float x[N];
        lp_unpack(v[k], x, T());
#pragma unroll
        for (int i = 0; i < N; i += 2)
          take(x[i] == -INFINITY ? -INFINITY : (x[i] - b) * kLpLog2e, x[i + 1] == -INFINITY ? -INFINITY : (x[i + 1] - b) * kLpLog2e);
      }
    }
  }
  // All of it relative to m, the largest logit of the CTA.
  __device__ __forceinline__ LpState state(float m) const {
    LpState r;
    r.m = m;
    const float by = b == -INFINITY ? 0.f : fmaxf((b - m) * kLpLog2e - off, -1e4f), f = lp_ex2(by);
    const float2 s2 = lp_split(s), u2 = lp_split(u);
    const float sum = s2.x + s2.y;
    r.s = sum * f;
    if (ENT) r.u = -fmaf(by, sum, u2.x + u2.y) * f * 0.693147180559945309f;
    float x[N];
    lp_unpack(held, x, T());
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = x[i] - m, e = lp_ex2(d * kLpLog2e);
      if (x[i] == m) {
        r.c += 1.f;
      } else if (x[i] != -INFINITY) {
        r.s += e;
        if (ENT) r.u = fmaf(fmaxf(d, -1e4f), -e, r.u);
      }
    }
    return r;
  }
};

// The elements first .. end-1 of a segment that this thread takes: up to one before the first 16-byte boundary, every 256th 16 bytes, up to one
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

template <typename T, bool ENT, bool TOP>
__global__ void __launch_bounds__(kLpThreads, kLpPerSm) token_logprobs_kernel(const LogprobParams p) {
  constexpr int N = LpSegment<T>::N;
  __shared__ float red[4][kLpWarps];
  __shared__ float4 parts[kLpMaxCluster];              // the CTAs' states, and
  __shared__ __align__(16) float group_max[kLpGroups];
  __shared__ float thr_s;
  __shared__ int n_above, n_equal;
  __shared__ __align__(16) unsigned long long list[kLpList];           // above the threshold
  __shared__ unsigned long long equal_list[kLpList];
  __shared__ int scan[kLpThreads];     // threads that have any of them
  __shared__ int n_scan;
  __shared__ __align__(16) unsigned long long all_k[kLpMaxCluster * kLpMaxTop + 2];        // their largest, each in order, in the first CTA
  __shared__ unsigned long long top_k[kLpMaxTop];                      // this CTA's largest, in order
  pdl_wait();
  pdl_launch_dependents();
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = (int)(blockIdx.x / C), t = threadIdx.x, warp = t >> 5, lane = t & 31, V = p.slices * p.cols, top = TOP ? p.top : 0;
  const int lo = (int)((long long)V * rank / C) & ~63, hi = rank == C - 1 ? V : (int)((long long)V * (rank + 1) / C) & ~63;
  if (C > 1) lp_cluster_arrive();      // (this CTA runs: the others may write to its memory)
  int token = -1;
  float token_x = 0.f;
  if (rank == 0 && t < p.n_tokens) {   // (on their way while the row is read)
    token = p.tokens[(size_t)row * p.n_tokens + t];
    if (token >= 0 && token < V) token_x = lp_at<T>(p, row, token);
  }

  // ---- one pass: maximum and sums of this thread's elements
  LpRunning<T, ENT, TOP> sums;
  for (int at = lo; at < hi;) {
    const int sl = at / p.cols, in = at - sl * p.cols, n = min(hi - at, p.cols - in);
    const LpSegment<T> g(lp_slice<T>(p, row, sl) + in, n);
    uint4 v[kLpLoads];
    auto fetch = [&](int first) {
#pragma unroll
      for (int k = 0; k < kLpLoads; ++k) {
        const int i = first + k * kLpThreads + t;
        v[k] = i < g.vecs ? lp_load(g.base + g.head + i * N) : sums.none();
      }
    };
    fetch(0);
    if (g.head > 0 || g.tail0 < n) {                   // (at most 7 elements each)
      uint4 x[1] = {sums.none()};
      if (t < g.head) lp_set(x[0].x, g.base[t]);
      if (g.tail0 + t < n) lp_set(x[0].y, g.base[g.tail0 + t]);
      sums.add(x, -1, 0);
    }
    for (int first = 0; first < g.vecs; first += kLpLoads * kLpThreads) {
      uint4 w[kLpLoads];
#pragma unroll
      for (int k = 0; k < kLpLoads; ++k) w[k] = v[k];
      if (first + kLpLoads * kLpThreads < g.vecs) fetch(first + kLpLoads * kLpThreads);
      sums.add(w, at + g.head + (first + t) * N, kLpThreads * N);
    }
    at += n;
  }

  // ---- the CTA's state
  const float mine = sums.mine;
  {
    const float m = warp_max(mine);
    if (lane == 0) red[0][warp] = m;
  }
  if constexpr (TOP) {
    float g = mine;
#pragma unroll
    for (int o = 1; o < kLpThreads / kLpGroups; o *= 2) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (t % (kLpThreads / kLpGroups) == 0) group_max[t / (kLpThreads / kLpGroups)] = g;
    if (t == 0) n_above = n_equal = n_scan = 0;
    if (t < kLpMaxTop) top_k[t] = 0ull;
  }
  __syncthreads();
  {
    float m = red[0][0];
#pragma unroll
    for (int w = 1; w < kLpWarps; ++w) m = fmaxf(m, red[0][w]);
    LpState a = sums.state(m);
    a.c = warp_sum(a.c);
    a.s = warp_sum(a.s);
    if (ENT) a.u = warp_sum(a.u);
    if (lane == 0) {
      red[1][warp] = a.c;
      red[2][warp] = a.s;
      red[3][warp] = a.u;
    }
  }

  // ---- the CTA's `top` largest.  The top-th largest of the 128 groups' maxima is a lower bound of the top-th largest element: few elements are above
  // it, and only the threads whose own maximum reaches it have any.
  if constexpr (TOP) {
    if (t >= kLpThreads - kLpGroups) {
      // every warp sorts 32 maxima, largest first; a maximum's rank is its place there and how many of the other three lists are before it
      const int me = t - (kLpThreads - kLpGroups), w = me >> 5;
      float v = group_max[me];
#pragma unroll
      for (int k = 2; k <= 32; k *= 2)
#pragma unroll
        for (int j = k / 2; j > 0; j /= 2) {
          const float o = __shfl_xor_sync(0xffffffffu, v, j);
          v = ((lane & k) == 0) == ((lane & j) == 0) ? fmaxf(v, o) : fminf(v, o);
        }
      group_max[me] = v;
      asm volatile("bar.sync 1, %0;" ::"n"(kLpGroups) : "memory");
      int before = lane;
#pragma unroll
      for (int q = 1; q < 4; ++q) {
        const int other = (w + q) & 3;
        const bool first = other < w;                  // (among equals, the lower list's)
        int n = 0;
#pragma unroll
        for (int half = 16; half > 0; half /= 2) {
          const float o = group_max[32 * other + n + half - 1];
          if (first ? o >= v : o > v) n += half;
        }
        if (n == 31 && (first ? group_max[32 * other + 31] >= v : group_max[32 * other + 31] > v)) n = 32;
        before += n;
      }
      if (before == top - 1) thr_s = v;
    }
    __syncthreads();
    const float thr = thr_s;
    auto offer = [&](float x, int i) {
      if (x > thr) {
        const int k = atomicAdd(&n_above, 1);
        if (k < kLpList) list[k] = lp_key(x, i);
      } else if (x == thr) {
        const int k = thr == -INFINITY ? kLpList : atomicAdd(&n_equal, 1);
        if (k < kLpList) equal_list[k] = lp_key(x, i);
      }
    };
    if (t == 0 && thr == -INFINITY) n_equal = kLpList + 1;            // (any number of them: see below)
    if (mine == -INFINITY) {
    } else if (sums.second >= thr || (mine >= thr && sums.where < 0)) {
      scan[atomicAdd(&n_scan, 1)] = t;
    } else if (mine >= thr) {
      float x[N];
      lp_unpack(sums.held, x, T());
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (x[j] >= thr) offer(x[j], sums.where + j);
    }
    __syncthreads();
    // (few) threads with more than one such vector: eight lanes read all of one's again, eight 16-byte loads each at a time
    for (int q = t >> 3; q < n_scan; q += kLpThreads / 8) {
      const int owner = scan[q], o8 = t & 7;
      for (int at = lo; at < hi;) {
        const int sl = at / p.cols, in = at - sl * p.cols, n = min(hi - at, p.cols - in);
        const LpSegment<T> g(lp_slice<T>(p, row, sl) + in, n);
        if (o8 == 0 && owner < g.head) offer(lp_float(g.base[owner]), at + owner);
        if (o8 == 0 && g.tail0 + owner < n) offer(lp_float(g.base[g.tail0 + owner]), at + g.tail0 + owner);
        for (int first = owner + o8 * kLpThreads; first < g.vecs; first += 64 * kLpThreads) {
          uint4 v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (first + 8 * k * kLpThreads < g.vecs) v[k] = lp_load(g.base + g.head + (first + 8 * k * kLpThreads) * N);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (first + 8 * k * kLpThreads >= g.vecs) break;
            float x[N];
            lp_unpack(v[k], x, T());
            float mx = x[0];
#pragma unroll
            for (int j = 1; j < N; ++j) mx = fmaxf(mx, x[j]);
            if (mx >= thr)
#pragma unroll
              for (int j = 0; j < N; ++j) offer(x[j], at + g.head + (first + 8 * k * kLpThreads) * N + j);
          }
        }
        at += n;
      }
    }
    __syncthreads();
    const int above = n_above, equal = n_equal;
    if (above <= kLpList) {
      for (int i = t; i < above; i += kLpThreads) {
        const unsigned long long me = list[i];
        int before = 0;
#pragma unroll 4
        for (int j = 0; j < above; ++j) before += list[j] > me;
        if (before < top) top_k[before] = me;
      }
      const int want = top - above;
      if (want > 0 && equal <= kLpList) {
        for (int i = t; i < equal; i += kLpThreads) {
          const unsigned long long me = equal_list[i];
          int before = 0;
#pragma unroll 4
          for (int j = 0; j < equal; ++j) before += equal_list[j] > me;
          if (before < want) top_k[above + before] = me;
        }
      } else if (want > 0) {
        // many equal ones: the first of them in the order of the row
        int found = 0;
        for (int base = lo; base < hi && found < want; base += kLpThreads) {
          const bool hit = base + t < hi && lp_at<T>(p, row, base + t) == thr;
          const unsigned ballot = __ballot_sync(0xffffffffu, hit);
          __syncthreads();
          if (lane == 0) scan[warp] = __popc(ballot);
          __syncthreads();
          int at = found + __popc(ballot & ((1u << lane) - 1u));
          for (int w = 0; w < kLpWarps; ++w) {
            at += w < warp ? scan[w] : 0;
            found += scan[w];
          }
          if (hit && at < want) top_k[above + at] = lp_key(thr, base + t);
        }
      }
    } else {
      // more above the bound than the list holds (they sit in few threads' elements): the next in order, one after the other
      unsigned long long last = ~0ull;
      for (int k = 0; k < top; ++k) {
        unsigned long long best = 0ull;
        for (int i = lo + t; i < hi; i += kLpThreads) {
          const float v = lp_at<T>(p, row, i);
          const unsigned long long key = lp_key(v, i);
          if (v == v && key < last && key > best) best = key;
        }
        for (int o = 16; o > 0; o >>= 1) {
          const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
          best = other > best ? other : best;
        }
        __syncthreads();
        if (lane == 0) list[warp] = best;
        __syncthreads();
        for (int w = 0; w < kLpWarps; ++w) best = list[w] > best ? list[w] : best;
        if (t == 0) top_k[k] = best;
        last = best;
      }
    }
  }

  // ---- the row: every CTA of the cluster writes its state and its list to the first one's memory
  if (C > 1) lp_cluster_wait();
  __syncthreads();
  if (t == 0) {
    LpState r;
#pragma unroll
    for (int w = 0; w < kLpWarps; ++w) {
      r.m = fmaxf(r.m, red[0][w]);
      r.c += red[1][w];
      r.s += red[2][w];
      if (ENT) r.u += red[3][w];
    }
    *(C > 1 ? cluster.map_shared_rank(&parts[rank], 0) : parts) = make_float4(r.m, r.c, r.s, r.u);
  }
  if (TOP && C > 1 && t < top) *cluster.map_shared_rank(&all_k[rank * top + t], 0) = top_k[t];
  if (C > 1) {
    lp_cluster_arrive();
    lp_cluster_wait();
  } else {
    __syncthreads();
  }
  if (rank == 0) {
    LpState r;
    {
      float m = -INFINITY;
#pragma unroll
      for (int k = 0; k < kLpMaxCluster; ++k)
        if (k < C) m = fmaxf(m, parts[k].x);
      r.m = m;
#pragma unroll
      for (int k = 0; k < kLpMaxCluster; ++k) {
        if (k >= C) break;
        const float4 q = parts[k];
        LpState b;
        b.m = q.x;
        b.c = q.y;
        b.s = q.z;
        b.u = q.w;
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
    if constexpr (TOP) {
      // place k of the row, a key or nobody's
      auto put = [&](int k, unsigned long long key) {
        p.top_ids[(size_t)row * top + k] = key ? lp_key_index(key) : -1;
        p.top_logprob[(size_t)row * top + k] = key ? logprob(lp_key_value(key)) : NAN;
      };
      if (C == 1) {
        if (t < top) put(t, top_k[t]);
      } else {
        // (a key's place is how many are before it; searching the lists, which are in order, is more code and was 1 us slower)
        const int all = C * top;
        if (t == 0 && (all & 1)) all_k[all] = 0ull;    // (read as the second of two)
        int have = 0;
        for (int i = t; i - t < all; i += kLpThreads) {
          const unsigned long long me = i < all ? all_k[i] : 0ull;
          have += __syncthreads_count(me != 0ull);
          if (!me) continue;
          int before = 0;
#pragma unroll 8
          for (int j = 0; j < all; j += 2) {
            const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(&all_k[j]);
            before += (two.x > me) + (two.y > me);
          }
          if (before < top) put(before, me);
        }
        if (t >= have && t < top) put(t, 0ull);        // (fewer numbers than places)
      }
    }
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
  // (32-bit places: a thread's next one may lie up to a turn of 1024 vectors behind the row's end)
  TQ_REQUIRE(ctx, slices < (1u << 16) && cols < (1ull << 31) && slices * cols <= (1ull << 31) - (1u << 16) && rows < (1ull << 31),
             "tq_token_logprobs: vocabulary or rows too large");
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
  // CTAs of a row (a cluster): as many as fit the GPU at once (four an SM), none with less than 2048 logits.  More, smaller ones cost more than they
  // balance, fewer leave SMs idle; us for one, two, four, eight: 64 rows of 128256 f32 23.7, 14.6, 10.3, 9.8, 256 rows 27.5, 22.3, 26.1, 33.0,
  // one row of 32000 6.5, 5.2, 4.6, 4.3.  Forms without alternatives or entropies leave their bookkeeping out of the loop: 2048 rows of 128256 bf16
  // 86 us, 95 with entropies, 108 with 20 alternatives, 122 with both.
  const size_t V = slices * cols, slots = (size_t)ctx->sm_count * kLpPerSm;
  size_t C = slots / rows < V / 2048 ? slots / rows : V / 2048;
  C = C < 1 ? 1 : C > (size_t)kLpMaxCluster ? (size_t)kLpMaxCluster : C;
  const bool ent = entropy_out_dev != nullptr;
  using bf = __nv_bfloat16;
  void (*kern)(LogprobParams);
  if (top) kern = dtype == TQ_BF16 ? (ent ? token_logprobs_kernel<bf, true, true> : token_logprobs_kernel<bf, false, true>)
                                   : (ent ? token_logprobs_kernel<float, true, true> : token_logprobs_kernel<float, false, true>);
  else kern = dtype == TQ_BF16 ? (ent ? token_logprobs_kernel<bf, true, false> : token_logprobs_kernel<bf, false, false>)
                               : (ent ? token_logprobs_kernel<float, true, false> : token_logprobs_kernel<float, false, false>);
  TQ_REQUIRE(ctx, rows < (size_t)(0x7fffffff / kLpMaxCluster), "tq_token_logprobs: too many rows");
  TQ_CUDA(ctx, launch_k_cluster(ctx, kern, dim3((unsigned)(rows * C)), dim3(kLpThreads), 0, dim3((unsigned)C), p));
  return TQ_OK;
}
