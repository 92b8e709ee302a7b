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
// small, so HBM bounds the pass: 1024 bf16 rows of 151936, 311 MB, 58 us (5.4 TB/s). Rows
// that do not fill the card are cut into chunks, a block each, whose sums and largest logits
// the row's last block to finish joins: it is found by an arrival word, and the chunks'
// results go past the caches, since the blocks may run on any XCD. Captured calls, and those
// of more rows than there are words, join in a second launch. A chain of trips to memory
// bounds such calls: 8 bf16 rows of 151936 with five alternatives 8.3 us, 77 fp32 rows of 50257
// with 20 alternatives 11.7. Of the first's 7.2 in the kernel the loads are 1.2, the sums of a
// block 0.4 twice, the selections 1.7 and 1.0, and the exchange 1.5 (the rest waits for the
// ragged chunk).
//
// The largest: of 64 groups of threads the `top`-th largest maximum bounds the `top`-th
// largest logit from below, so only threads whose maximum reaches it have any of them. Those
// threads' elements that reach the bound go to a list in LDS and are ranked by counting.
// Every wave finds the bound by itself, bit by bit from ballots; the upper 16 bits of the
// value do. Where more elements reach it than there is room for (many equal ones, or the
// largest in fewer groups than `top`), the bound is the `top`-th largest maximum of all threads
// to the last bit of (value, place): no two are equal, so `top` threads reach it and no more.
// Up to kLpHeld iterations a thread's elements are loaded at once and stay in registers, and
// the runs of eight that reach the bound go to LDS, kLpHeld of each such thread at most; longer
// ones are read again from the caches.
#include "tpp_common.hpp"

namespace tpp {

constexpr int kLpThreads = 256, kLpRun = 8, kLpStep = kLpThreads * kLpRun; // elements an iteration
constexpr int kLpMaxTop = 32, kLpRoom = 1024;
constexpr int kLpHeld = 8, kLpRuns = kLpMaxTop * kLpHeld; // (runs of kLpMaxTop threads)

typedef unsigned long long u64;

struct LpArgs {
  const void *x;
  const int64_t *tok;
  float *lp, *ent, *top_lp;
  int64_t *top_id;
  int64_t x_s, V;
  int top;
  u64 *sums, *keys; // of chunks: maximum and the two sums, two words; their largest logits
  unsigned *arrived; // a word a row, or null
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

// A block's exchange.
struct LpShared {
  float sum[4][3];
  u64 max[kLpThreads], cand[kLpRoom + 32], best[4];
  int active[kLpThreads], n[2];       // threads, or runs, that reach the bound; entries of active and cand
  float run[kLpRuns][kLpRun];         // values of those runs
};
static_assert(kLpRuns <= kLpThreads, "a run's place is in active");

// The sums of a block's threads. Each thread's largest key is in s.max then, for lp_select.
__device__ __forceinline__ LpSums lp_block(const LpSums &a, u64 mine, LpShared &s) {
  float mx = row16_max(a.m);
  mx = fmaxf(fmaxf(readlane_f32(mx, 0), readlane_f32(mx, 16)), fmaxf(readlane_f32(mx, 32), readlane_f32(mx, 48)));
  LpSums ws = a;
  ws.shift(mx);
  ws.s = wave_sum(ws.s), ws.t = wave_sum(ws.t);
  if (lane_id() == 0) s.sum[wave_id()][0] = ws.m, s.sum[wave_id()][1] = ws.s, s.sum[wave_id()][2] = ws.t;
  s.max[threadIdx.x] = mine;
  if (threadIdx.x < 2) s.n[threadIdx.x] = 0;
  __syncthreads();
  LpSums all = {fmaxf(fmaxf(s.sum[0][0], s.sum[1][0]), fmaxf(s.sum[2][0], s.sum[3][0])), 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    LpSums x = {s.sum[i][0], s.sum[i][1], s.sum[i][2]};
    x.shift(all.m);
    all.s += x.s, all.t += x.t;
  }
  return all;
}

// The `top` largest of a block's elements, put(rank, key) once for each rank (all of them
// where there are fewer), behind lp_block. `mine`, given there: a bound of this thread's keys
// that one of them reaches. begin(bound), then scan(bound, f) any number of times: f(key) for
// every key that reaches the bound.
template <typename BEGIN, typename SCAN, typename PUT>
__device__ __forceinline__ void lp_select(LpShared &s, int top, BEGIN begin, SCAN scan, PUT put) {
  const int tid = threadIdx.x, lane = lane_id(), w = wave_id();
  // the top-th largest of 64 groups (four threads a group)
  u64 g = s.max[lane];
#pragma unroll
  for (int i = 1; i < 4; ++i) g = max(g, s.max[i * kWave + lane]);
  const unsigned hi = (unsigned)(g >> 32);
  unsigned b = 0;
#pragma unroll
  for (int bit = 31; bit >= 16; --bit)
    if (__popcll(__ballot(hi >= (b | 1u << bit))) >= top) b |= 1u << bit;
  u64 bound = (u64)b << 32;
  auto list = [&] {
    begin(bound);
    scan(bound, [&](u64 key) {
      const int at = atomicAdd(&s.n[1], 1);
      if (at < kLpRoom) s.cand[at] = key;
    });
    __syncthreads();
  };
  list();
  int found = s.n[1];
  if (found > kLpRoom || s.n[0] > kLpRuns) { // the top-th largest of the threads
    u64 each[kLpThreads / kWave];
#pragma unroll
    for (int i = 0; i < kLpThreads / kWave; ++i) each[i] = s.max[i * kWave + lane];
    bound = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const u64 higher = bound | 1ull << bit;
      int n = 0;
#pragma unroll
      for (int i = 0; i < kLpThreads / kWave; ++i) n += __popcll(__ballot(each[i] >= higher));
      if (n >= top) bound = higher;
    }
    __syncthreads();
    if (tid < 2) s.n[tid] = 0;
    __syncthreads();
    list();
    found = s.n[1];
  }
  if (found <= kLpRoom) {
    // four threads a candidate, a quarter of the list each (every wave pads the list with zeros)
    if (lane < 32) s.cand[found + lane] = 0;
    for (int c = tid / 4; c < (found + 63) / 64 * 64; c += kLpThreads / 4) {
      const u64 key = s.cand[min(c, found)];
      int rank = 0;
      for (int k = tid % 4; k < found; k += 32)
#pragma unroll
        for (int j = 0; j < 8; ++j) rank += s.cand[k + 4 * j] > key;
      rank = (int)group_sum<4>((float)rank);
      if (tid % 4 == 0 && c < found && rank < top) put(rank, key);
    }
    return;
  }
  // more than the list holds (most of a few threads' elements among the largest): one
  // after the other
  u64 last = ~0ull;
  for (int k = 0; k < top; ++k) {
    u64 best = 0;
    scan(bound, [&](u64 key) {
      if (key < last) best = max(best, key);
    });
#pragma unroll
    for (int sh = 1; sh < kWave; sh <<= 1) best = max(best, (u64)__shfl_xor(best, sh, kWave));
    __syncthreads();
    if (lane == 0) s.best[w] = best;
    __syncthreads();
    last = max(max(s.best[0], s.best[1]), max(s.best[2], s.best[3]));
    if (tid == 0) put(k, last);
  }
}

// What the row's results are made of, by the block that has all of it.
struct LpRow {
  float m, log_z;
  bool nan; // a NaN, or +inf less +inf
};
// The row's token's logit, asked for behind the first loads of the row: it takes two trips.
struct LpToken {
  float x;
  bool real;
};
template <typename P> __device__ __forceinline__ LpToken lp_token(const LpArgs &p, int64_t r, int64_t t) {
  return {to_f32(((const P *)p.x)[r * p.x_s + min(max(t, (int64_t)0), p.V - 1)]), t >= 0 && t < p.V};
}
__device__ __forceinline__ LpRow lp_finish(const LpArgs &p, int64_t r, const LpSums &all, const LpToken &k) {
  const LpRow o = {all.m, all.m == -INFINITY ? NAN : logf(all.s), all.s != all.s};
  if (threadIdx.x == 0) {
    p.lp[r] = k.real ? k.x - all.m - o.log_z : 0.f;
    p.ent[r] = o.log_z - all.t / all.s;
  }
  if (o.nan && (int)threadIdx.x < p.top) p.top_lp[r * p.top + threadIdx.x] = NAN, p.top_id[r * p.top + threadIdx.x] = -1;
  return o;
}
__device__ __forceinline__ void lp_put(const LpArgs &p, int64_t r, const LpRow &o, int rank, u64 key) {
  p.top_lp[r * p.top + rank] = lp_value((unsigned)(key >> 32)) - o.m - o.log_z;
  p.top_id[r * p.top + rank] = (int64_t)(0xffffffffu - (unsigned)key);
}

// To and from another block of the launch.
__device__ __forceinline__ void lp_store(u64 *p, u64 x) {
  __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ u64 lp_fetch(const u64 *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The chunks of a row, by one block.
__device__ __forceinline__ void lp_join(const LpArgs &p, int64_t r, int chunks, const LpToken &k, LpShared &s) {
  constexpr int kKeep = 4; // keys a thread keeps (past them, memory is asked again)
  const int tid = threadIdx.x;
  const u64 *sums = p.sums + r * chunks * 2, *in = p.keys + r * chunks * p.top;
  const int n = chunks * p.top;
  LpSums a = {-INFINITY, 0.f, 0.f};
  u64 key[kKeep], mine = 0;
#pragma unroll
  for (int j = 0; j < kKeep; ++j) key[j] = j * kLpThreads + tid < n ? lp_fetch(in + j * kLpThreads + tid) : 0;
  for (int c = tid; c < chunks; c += kLpThreads) {
    const u32x2 x = __builtin_bit_cast(u32x2, lp_fetch(sums + c * 2)), y = __builtin_bit_cast(u32x2, lp_fetch(sums + c * 2 + 1));
    a.add(LpSums{__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(y[0])});
  }
#pragma unroll
  for (int j = 0; j < kKeep; ++j) mine = max(mine, key[j]);
  for (int c = kKeep * kLpThreads + tid; c < n; c += kLpThreads) mine = max(mine, lp_fetch(in + c));
  const LpRow o = lp_finish(p, r, lp_block(a, mine, s), k);
  if (p.top && !o.nan)
    lp_select(s, p.top, [](u64) {},
              [&](u64 bound, auto f) {
#pragma unroll
                for (int j = 0; j < kKeep; ++j)
                  if (j * kLpThreads + tid < n && key[j] >= bound) f(key[j]);
                for (int c = kKeep * kLpThreads + tid; c < n; c += kLpThreads) {
                  const u64 x = lp_fetch(in + c);
                  if (x >= bound) f(x);
                }
              },
              [&](int rank, u64 key) { lp_put(p, r, o, rank, key); });
}

// A row (WHOLE), or chunk blockIdx.y of one: `steps` iterations of the block. HELD: at most
// kLpHeld of them, in registers throughout.
template <typename P, bool WHOLE, bool HELD> __global__ __launch_bounds__(kLpThreads) void logprob_kernel(LpArgs p, int steps) {
  constexpr int U = HELD ? kLpHeld : 4; // iterations whose loads are in flight
  typedef typename LpVec<P>::type V;
  __shared__ LpShared s;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x, base = WHOLE ? 0 : (int64_t)blockIdx.y * steps * kLpStep;
  const P *row = (const P *)p.x + r * p.x_s;
  const int64_t n = WHOLE ? p.V : min(p.V, base + (int64_t)steps * kLpStep);
  const int iters = (int)((n - base + kLpStep - 1) / kLpStep), full = (int)((n - base) / kLpStep);

  const int64_t tok = p.tok[r];
  const P *mine_at = row + base + tid * kLpRun;
  auto at = [&](int i) { return base + (int64_t)i * kLpStep + tid * kLpRun; }; // this thread's elements of iteration i
  V v[U];
  if constexpr (HELD) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u < full) v[u] = __builtin_nontemporal_load((const V *)(mine_at + u * kLpStep));
    if (full < iters) {
      V end;
#pragma unroll
      for (int e = 0; e < kLpRun; ++e) end[e] = row[min(at(full) + e, n - 1)];
#pragma unroll
      for (int e = 0; e < kLpRun; ++e) end[e] = at(full) + e < n ? end[e] : P(-INFINITY);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u == full) v[u] = end;
    }
  } else if (full >= U) {
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = __builtin_nontemporal_load((const V *)(mine_at + u * kLpStep));
  }
  const LpToken token = lp_token<P>(p, r, tok);

  LpSums a = {-INFINITY, 0.f, 0.f};
  int first = 0;    // iteration in which this thread met its maximum
  float most[U];    // HELD: of every iteration
  auto largest = [](const float (&x)[kLpRun]) {
    return fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
  };
  auto add = [&](const float (&x)[kLpRun]) {
    const float mu = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
    for (int e = 0; e < kLpRun; ++e) {
      const float d = x[e] - mu, f = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
      a.s += f;
      a.t = fmaf(f, fmaxf(d, -1e30f), a.t); // (0 times -inf is none)
    }
  };
  auto values = [](const V &v, float (&x)[kLpRun]) {
#pragma unroll
    for (int e = 0; e < kLpRun; ++e) x[e] = to_f32(v[e]);
  };
  float x[kLpRun];
  if constexpr (HELD) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u >= iters) continue;
      values(v[u], x);
      most[u] = largest(x);
      if (most[u] > a.m) a.m = most[u], first = u;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u >= iters) continue;
      values(v[u], x);
      add(x);
    }
  } else {
    auto step = [&](int i) {
      const float mx = largest(x);
      if (mx > a.m) a.shift(mx), first = i;
      add(x);
    };
    int i = 0;
    if (full >= U)
      for (; i + U <= full; i += U)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          values(v[u], x);
          // (past the last whole round: an iteration that is there, not used)
          const int next = i + u + U < full / U * U ? i + u + U : i + u;
          v[u] = __builtin_nontemporal_load((const V *)(mine_at + (int64_t)next * kLpStep));
          step(i + u);
        }
    for (; i < iters; ++i) {
      lp_load(row, at(i), n, x);
      step(i);
    }
  }

  const unsigned run0 = (unsigned)(base / kLpRun); // a place is a run of eight, counted over the row
  const u64 mine = lp_key(a.m, run0 + (unsigned)(first * kLpThreads + tid));
  const LpSums all = lp_block(a, mine, s);
  auto begin = [&](u64 bound) {
    if constexpr (HELD) {
      auto hit = [&](int u) { return u < iters && lp_key(most[u], run0 + (unsigned)(u * kLpThreads + tid)) >= bound; };
      int hits = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) hits += hit(u);
      const int upto = wave_scan(hits), all = __builtin_amdgcn_readlane(upto, kWave - 1);
      int k = 0;
      if (lane_id() == 0 && all) k = atomicAdd(&s.n[0], all);
      k = __builtin_amdgcn_readfirstlane(k) + upto - hits;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!hit(u)) continue;
        if (k < kLpRuns) {
          s.active[k] = (int)(run0 + (unsigned)(u * kLpThreads + tid));
          values(v[u], x);
#pragma unroll
          for (int e = 0; e < kLpRun; e += 4) *reinterpret_cast<f32x4 *>(&s.run[k][e]) = f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
        }
        ++k;
      }
    } else {
      if (mine >= bound) s.active[atomicAdd(&s.n[0], 1)] = tid;
    }
    __syncthreads();
  };
  auto reach = [&](float x, unsigned run, int e, u64 bound, auto f) {
    if (lp_key(x, run) >= bound && (int64_t)run * kLpRun + e < n) f(lp_key(x, run * kLpRun + e));
  };
  auto scan = [&](u64 bound, auto f) {
    if constexpr (HELD) {
      const int work = min(s.n[0], kLpRuns) * kLpRun;
      for (int i = tid; i < work; i += kLpThreads) reach(s.run[i / kLpRun][i % kLpRun], s.active[i / kLpRun], i % kLpRun, bound, f);
    } else {
      // their iterations over the block (a wave a thread would wait for memory once for each)
      const unsigned work = (unsigned)(s.n[0] * iters);
      for (unsigned i = tid; i < work; i += kLpThreads) {
        const unsigned k = i / (unsigned)iters, run = run0 + (i - k * (unsigned)iters) * kLpThreads + s.active[k];
        if ((int64_t)run * kLpRun >= n) continue;
        lp_load(row, (int64_t)run * kLpRun, n, x);
#pragma unroll
        for (int e = 0; e < kLpRun; ++e) reach(x[e], run, e, bound, f);
      }
    }
  };
  if constexpr (WHOLE) {
    const LpRow o = lp_finish(p, r, all, token);
    if (p.top && !o.nan) lp_select(s, p.top, begin, scan, [&](int rank, u64 key) { lp_put(p, r, o, rank, key); });
  } else {
    const int chunks = gridDim.y;
    const int64_t slot = r * chunks + blockIdx.y;
    if (tid == 0) {
      lp_store(p.sums + slot * 2, __builtin_bit_cast(u64, u32x2{__float_as_uint(all.m), __float_as_uint(all.s)}));
      lp_store(p.sums + slot * 2 + 1, (u64)__float_as_uint(all.t));
    }
    if (p.top && all.s == all.s) { // (else the row is NaN, no key is used)
      u64 *out = p.keys + slot * p.top;
      if (n - base < p.top && tid >= n - base && tid < p.top) lp_store(out + tid, 0); // fewer elements: below every key
      lp_select(s, p.top, begin, scan, [&](int rank, u64 key) { lp_store(out + rank, key); });
    }
    if (!p.arrived) return;
    __shared__ int s_last;
    asm volatile("" ::: "memory");
    vm_wait<0>(); // this wave's results are in memory
    __syncthreads();
    if (tid == 0) {
      const unsigned old = __hip_atomic_fetch_add(p.arrived + r, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s_last = (int)old == chunks - 1;
      if (s_last) __hip_atomic_store(p.arrived + r, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (s_last) lp_join(p, r, chunks, token, s);
  }
}

template <typename P> __global__ __launch_bounds__(kLpThreads) void logprob_join_kernel(LpArgs p, int chunks) {
  __shared__ LpShared s;
  lp_join(p, blockIdx.x, chunks, lp_token<P>(p, blockIdx.x, p.tok[blockIdx.x]), s);
}

// Chunks of a row (1: none), of `steps` iterations. As many as fill the CUs k times over, by
// estimated time in us, from measurements of 1 to 1024 rows: 4; an iteration 0.1 and 0.14 for
// each of the CU's blocks (16-bit logits, twice that for fp32); 1 a block for what it selects; 3
// for the join; 2.5 where elements are not held. Measured, bf16 rows of 151936, k = 1 and 2: 8
// with five alternatives 7.2 and 7.6 (in the kernel), 4 with 20 7.7 and 10.2. A few blocks more
// than CUs are the worst: 130 rows with 32 alternatives, 260 chunks 27.6, 1040 20.9, 300 rows
// with five, whole 30.7, halves 26.5.
struct LpPlan {
  int chunks, steps;
};
static LpPlan lp_plan(int64_t N, int64_t V, int dtype) {
  const int cus = device_cu_count() > 0 ? device_cu_count() : 256;
  const int64_t iters = (V + kLpStep - 1) / kLpStep;
  LpPlan best = {1, (int)iters};
  double least = 0;
  for (int k = 1; k <= 6; ++k) {
    int64_t c = k * cus / N;
    if (c < 1) c = 1;
    if (c > iters) c = iters;
    const int64_t steps = (iters + c - 1) / c;
    c = (iters + steps - 1) / steps;
    const double blocks = (double)((N * c + cus - 1) / cus);
    const double us = 4 + steps * (0.1 + (dtype == TPP_F32 ? 0.28 : 0.14) * blocks) + blocks + (c > 1 ? 3 : 0) + (steps > kLpHeld ? 2.5 : 0);
    if (k == 1 || us < least) least = us, best = {(int)c, (int)steps};
  }
  return best;
}

} // namespace tpp

using namespace tpp;

extern "C" size_t tpp_token_logprobs_workspace_size(int64_t N, int64_t V, int64_t top, int dtype) {
  if (N <= 0 || V <= 0 || top < 0) return 0;
  const LpPlan pl = lp_plan(N, V, dtype);
  return pl.chunks > 1 ? (size_t)N * pl.chunks * (2 + (size_t)top) * sizeof(u64) : 0;
}

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
  const LpPlan pl = lp_plan(N, V, dtype);
  if (pl.chunks > 1) {
    if (!workspace || !aligned16(workspace) || ws_bytes < tpp_token_logprobs_workspace_size(N, V, top, dtype))
      return set_error(TPP_E_WORKSPACE, "%s: workspace missing, unaligned or too small", name);
    a.sums = (u64 *)workspace, a.keys = a.sums + N * pl.chunks * 2;
  }
  hipStream_t st = as_stream(stream);
  if (pl.chunks > 1) a.arrived = arrival_words(st, N);
  auto go = [&](auto zero) {
    typedef decltype(zero) P;
    const dim3 grid((unsigned)N, (unsigned)pl.chunks);
    const bool held = pl.steps <= kLpHeld;
    if (pl.chunks == 1) {
      if (held) logprob_kernel<P, true, true><<<grid, dim3(kLpThreads), 0, st>>>(a, pl.steps);
      else logprob_kernel<P, true, false><<<grid, dim3(kLpThreads), 0, st>>>(a, pl.steps);
    } else {
      if (held) logprob_kernel<P, false, true><<<grid, dim3(kLpThreads), 0, st>>>(a, pl.steps);
      else logprob_kernel<P, false, false><<<grid, dim3(kLpThreads), 0, st>>>(a, pl.steps);
      if (!a.arrived) logprob_join_kernel<P><<<dim3((unsigned)N), dim3(kLpThreads), 0, st>>>(a, pl.chunks);
    }
    return check_launch(name);
  };
  return dtype == TPP_F32 ? go(0.f) : dtype == TPP_F16 ? go(f16(0)) : go(bf16(0));
}
