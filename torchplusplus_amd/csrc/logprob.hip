// Log probabilities of given tokens, entropy and the largest logits of rows of logits x:
//   m = max_j x_j, Z = sum_j e^(x_j - m)
//   logprob(t) = x_t - m - ln Z,   H = ln Z + (1 / Z) sum_j e^(x_j - m) (m - x_j)
// and the same of the `top` largest logits, the lowest index first among equal ones.
// Both terms of H are sums of terms not below 0: nothing cancels. Terms of x_j = -inf are
// 0. A row with a NaN or +inf, or of -inf alone, has no distribution: its results are NaN
// (and its top tokens -1; of -inf alone the lowest). A token outside [0, V) is padding, its
// log probability 0.
//
// One pass over the row: a thread keeps its running maximum with the two sums, and the
// place where it met that maximum first. The rows are 2 or 4 V bytes and everything else is
// small, so HBM bounds the pass.
//
// The largest: of 64 groups of threads the `top`-th largest maximum bounds the `top`-th
// largest logit from below, so only threads whose maximum reaches it have any of them: those
// threads' elements are read again (from the caches), the ones that reach the bound kept in
// LDS and ranked by counting. Order is by (value, index) as one 64-bit key, so equal logits,
// and rows of one value alone, are bounded like any other.
#include "tpp_common.hpp"

namespace tpp {

constexpr int kLpThreads = 256, kLpRun = 8, kLpStep = kLpThreads * kLpRun; // elements an iteration
constexpr int kLpMaxTop = 32, kLpRoom = 1024;

typedef unsigned long long u64;

struct LpArgs {
  const void *x;
  const int64_t *tok;
  float *lp, *ent, *top_lp;
  int64_t *top_id;
  int64_t x_s, V;
  int top;
};

// Larger floats as larger words (-0 as 0); the place breaks ties, lower first.
__device__ __forceinline__ unsigned lp_order(float x) {
  const unsigned u = __float_as_uint(x + 0.f);
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float lp_value(unsigned o) {
  return __uint_as_float(o ^ (~(unsigned)((int)o >> 31) | 0x80000000u));
}
__device__ __forceinline__ u64 lp_key(float x, unsigned place) { return ((u64)lp_order(x) << 32) | (0xffffffffu - place); }

// Eight elements from any address of their type's alignment; -inf past the row's end.
template <typename P> struct LpVec {
  typedef P type __attribute__((ext_vector_type(kLpRun), aligned(sizeof(P))));
};
template <typename P> __device__ __forceinline__ void lp_load(const P *row, int64_t at, int64_t n, float (&x)[kLpRun]) {
  typedef typename LpVec<P>::type V;
  if (at + kLpRun <= n) {
    const V v = *reinterpret_cast<const V *>(row + at);
#pragma unroll
    for (int e = 0; e < kLpRun; ++e) x[e] = to_f32(v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < kLpRun; ++e) x[e] = at + e < n ? to_f32(row[at + e]) : -INFINITY;
  }
}

struct LpSums { // of elements met so far: maximum, sum of e^(x - m), sum of e^(x - m) (x - m)
  float m, s, t;
  // terms relative to the larger maximum mn
  __device__ __forceinline__ void shift(float mn) {
    // (no terms yet: s = t = 0; far apart: 0 times -inf is none)
    const float d = m == -INFINITY ? 0.f : fmaxf(m - mn, -1e30f);
    const float a = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
    t = a * fmaf(s, d, t), s *= a, m = mn;
  }
  __device__ __forceinline__ void add(LpSums o) {
    const float mn = fmaxf(m, o.m);
    if (mn == -INFINITY) {
      s += o.s; // a NaN stays one
      return;
    }
    shift(mn), o.shift(mn);
    s += o.s, t += o.t;
  }
};

__device__ __forceinline__ LpSums lp_wave(LpSums a) {
#pragma unroll
  for (int sh = 1; sh < kWave; sh <<= 1) {
    LpSums o;
    o.m = __shfl_xor(a.m, sh, kWave), o.s = __shfl_xor(a.s, sh, kWave), o.t = __shfl_xor(a.t, sh, kWave);
    a.add(o);
  }
  return a;
}

template <typename P> __global__ __launch_bounds__(kLpThreads) void logprob_kernel(LpArgs p) {
  __shared__ LpSums s_sum[4];
  __shared__ u64 s_max[kLpThreads], s_cand[kLpRoom], s_bound, s_best[4];
  __shared__ int s_active[kLpThreads], s_n[2];
  const int tid = threadIdx.x, lane = lane_id(), w = wave_id();
  const int64_t r = blockIdx.x, n = p.V;
  const P *row = (const P *)p.x + r * p.x_s;
  const int iters = (int)((n + kLpStep - 1) / kLpStep);

  LpSums a = {-INFINITY, 0.f, 0.f};
  int first = 0; // iteration in which this thread met its maximum
  for (int i = 0; i < iters; ++i) {
    float x[kLpRun];
    lp_load(row, (int64_t)i * kLpStep + tid * kLpRun, n, x);
    float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    if (mx > a.m) a.shift(mx), first = i;
    const float mu = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
    for (int e = 0; e < kLpRun; ++e) {
      const float d = x[e] - mu, f = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
      a.s += f;
      a.t = fmaf(f, fmaxf(d, -1e30f), a.t); // (0 times -inf is none)
    }
  }
  const LpSums ws = lp_wave(a);
  if (lane == 0) s_sum[w] = ws;
  const u64 mine = lp_key(a.m, (unsigned)(first * kLpThreads + tid)); // place: the run of eight
  s_max[tid] = mine;
  if (tid < 2) s_n[tid] = 0;
  __syncthreads();
  LpSums all = s_sum[0];
#pragma unroll
  for (int i = 1; i < 4; ++i) all.add(s_sum[i]);
  const bool nan = all.s != all.s; // a NaN, or +inf less +inf
  const float log_z = all.m == -INFINITY ? NAN : logf(all.s);
  if (tid == 0) {
    const int64_t t = p.tok[r];
    p.lp[r] = t < 0 || t >= n ? 0.f : to_f32(row[t]) - all.m - log_z;
    p.ent[r] = log_z - all.t / all.s;
  }
  if (p.top == 0) return;
  if (nan) { // (the whole block)
    if (tid < p.top) p.top_lp[r * p.top + tid] = NAN, p.top_id[r * p.top + tid] = -1;
    return;
  }

  // the bound: the top-th largest of 64 groups' maxima (four threads a group)
  if (w == 0) {
    u64 g = s_max[lane];
#pragma unroll
    for (int i = 1; i < 4; ++i) g = max(g, s_max[i * kWave + lane]);
    int rank = 0;
    for (int l = 0; l < kWave; ++l) rank += __shfl(g, l, kWave) > g;
    if (rank == p.top - 1) s_bound = g;
  }
  __syncthreads();
  const u64 bound = s_bound;
  if (mine >= bound) s_active[atomicAdd(&s_n[0], 1)] = tid;
  __syncthreads();
  const int active = s_n[0];
  // an element as a key with its run's place: reaches the bound or not
  auto each = [&](auto f) {
    for (int k = w; k < active; k += 4)
      for (int i = lane; i < iters; i += kWave) {
        const unsigned run = (unsigned)(i * kLpThreads + s_active[k]);
        if ((int64_t)run * kLpRun >= n) continue;
        float x[kLpRun];
        lp_load(row, (int64_t)run * kLpRun, n, x);
#pragma unroll
        for (int e = 0; e < kLpRun; ++e)
          if ((int64_t)run * kLpRun + e < n && lp_key(x[e], run) >= bound) f(lp_key(x[e], run * kLpRun + e));
      }
  };
  each([&](u64 key) {
    const int at = atomicAdd(&s_n[1], 1);
    if (at < kLpRoom) s_cand[at] = key;
  });
  __syncthreads();
  const int found = s_n[1];
  auto put = [&](int rank, u64 key) {
    p.top_lp[r * p.top + rank] = lp_value((unsigned)(key >> 32)) - all.m - log_z;
    p.top_id[r * p.top + rank] = (int64_t)(0xffffffffu - (unsigned)key);
  };
  if (found <= kLpRoom) {
    for (int c = tid; c < found; c += kLpThreads) {
      const u64 key = s_cand[c];
      int rank = 0;
      for (int k = 0; k < found; ++k) rank += s_cand[k] > key;
      if (rank < p.top) put(rank, key);
    }
    return;
  }
  // more than the list holds (most of a few threads' elements among the largest): one
  // after the other
  u64 last = ~0ull;
  for (int k = 0; k < p.top; ++k) {
    u64 best = 0;
    each([&](u64 key) {
      if (key < last) best = max(best, key);
    });
#pragma unroll
    for (int sh = 1; sh < kWave; sh <<= 1) best = max(best, (u64)__shfl_xor(best, sh, kWave));
    __syncthreads();
    if (lane == 0) s_best[w] = best;
    __syncthreads();
    last = max(max(s_best[0], s_best[1]), max(s_best[2], s_best[3]));
    if (tid == 0) put(k, last);
  }
}

} // namespace tpp

using namespace tpp;

extern "C" size_t tpp_token_logprobs_workspace_size(int64_t N, int64_t V, int64_t top, int dtype) { return 0; }

extern "C" int tpp_token_logprobs(const void *logits, int64_t row_stride, const int64_t *tokens, float *logprobs,
                                  float *entropy, float *top_logprobs, int64_t *top_tokens, int64_t N, int64_t V,
                                  int64_t top, int dtype, void *workspace, size_t ws_bytes, void *stream) {
  const char *name = "tpp_token_logprobs";
  if (dtype != TPP_F16 && dtype != TPP_BF16 && dtype != TPP_F32)
    return set_error(TPP_E_UNSUPPORTED, "%s: unsupported dtype %d", name, dtype);
  if (N < 0 || V < 1 || row_stride < 0) return set_error(TPP_E_INVALID, "%s: invalid shapes", name);
  if (top < 0 || top > kLpMaxTop || top > V)
    return set_error(TPP_E_UNSUPPORTED, "%s: %lld alternatives, 0 to %d (and at most the vocabulary) are handled", name,
                     (long long)top, kLpMaxTop);
  if (V > 0x7fff0000LL || N > 0xffffff) return set_error(TPP_E_UNSUPPORTED, "%s: too large", name);
  if (N == 0) return TPP_OK;
  if (!logits || !tokens || !logprobs || !entropy || (top > 0 && (!top_logprobs || !top_tokens)))
    return set_error(TPP_E_INVALID, "%s: null pointer", name);
  LpArgs a = {};
  a.x = logits, a.tok = tokens, a.lp = logprobs, a.ent = entropy, a.top_lp = top_logprobs, a.top_id = top_tokens;
  a.x_s = row_stride, a.V = V, a.top = (int)top;
  hipStream_t st = as_stream(stream);
  auto go = [&](auto zero) {
    typedef decltype(zero) P;
    logprob_kernel<P><<<dim3((unsigned)N), dim3(kLpThreads), 0, st>>>(a);
    return check_launch(name);
  };
  return dtype == TPP_F32 ? go(0.f) : dtype == TPP_F16 ? go(f16(0)) : go(bf16(0));
}
