// Verification of drafted tokens against the target's probabilities, from
// given uniform numbers.
//
// Rows of probabilities: target_probs[b, 0] follows the context, row t + 1
// follows drafted token t. A mass that is not finite or not above zero counts
// as zero. Three forms:
//  * chain with the draft's probabilities q (rejection sampling): token i
//    stays while u_i q_i(x_i) < p_i(x_i). The next token comes from
//    max(p_n - q_n, 0) at the first token n that does not stay, from p_T
//    behind the last, and from p_n at a token that is none (padding).
//  * chain and tree of tokens chosen without a draw: at a node the target's
//    own draw is made in two parts, over the node's children by inverse CDF
//    (child c stays if below(c) <= u_depth < below(c) + p(x_c), below(c) the
//    mass of its earlier siblings, a token met before having none), and, where
//    no child stays, over the vocabulary without the children.
// The next token is the first index at which the running sum of those weights
// passes u_T times their sum (the last positive one where rounding leaves
// none). Where the weights have no mass the row itself is used, and where that
// has none the token is -1.
//
// All sums are fp64: a border of the inverse CDF is met by an fp32 sum over
// 150000 tokens at one draw in a few hundred, so the token would depend on the
// order of the sum.
//
// Two launches. The first cuts the row that the walk ends at into chunks of 4096
// masses and sums each; the second finds the chunk and the index. Every wave of the
// first repeats the walk (one gather of a mass per drafted token, all at once, then
// a walk in registers): cheaper than a launch of its own, or a barrier. Every wave
// of the second scans the chunks' sums. What bounds it: the latency of two launches,
// of three dependent trips to memory in the first (tokens, their masses, the row) and
// two in the second (the chunks' sums, the chunk), and there of three scans of fp64
// sums over a wave, one after the other; the rows are B V 4 bytes (with q twice that).
// 8 chains of 5 over 150000 tokens 10.5 us, 16 trees of 31 11.7; in one launch, the last
// block of a sequence to finish picking, 11.9 for the chains.
#include "tpp_common.hpp"

namespace tpp {

constexpr int kVerChunk = 4096;
constexpr int kVerMaxT = 64;

struct VerState { // one per sequence, written by the first launch for the second
  int row;        // row of target_probs the next token is drawn from
  int rejected;   // weights are max(p - q, 0)
  unsigned long long children;
};

struct VerArgs {
  const int64_t *tok;   // [B, T]
  const int32_t *parents; // [B, T] or null: a chain
  const void *p, *q;
  int64_t p_sb, p_st, q_sb, q_st;
  const float *u; // [B, T + 1]
  int T, chunks;
  int64_t V;
  int32_t *accepted, *path; // [B], [B, T]
  int64_t *next;            // [B]
  double *part;             // [B, chunks, 2]
  VerState *state;          // [B]
};

__device__ __forceinline__ double mass(float x) { // NaN fails both
  return x > 0.f && x < INFINITY ? (double)x : 0.0;
}
__device__ __forceinline__ double readlane_f64(double v, int lane) {
  const u32x2 w = __builtin_bit_cast(u32x2, v);
  const u32x2 r = {(unsigned)__builtin_amdgcn_readlane((int)w[0], lane),
                   (unsigned)__builtin_amdgcn_readlane((int)w[1], lane)};
  return __builtin_bit_cast(double, r);
}

// The walk, by one whole wave (lane i = drafted token i).
template <typename P>
__device__ __forceinline__ VerState ver_walk(const VerArgs &a, int64_t b, bool write, int &tok) {
  const int lane = lane_id(), T = a.T;
  const bool in = lane < T;
  const int64_t t64 = in ? a.tok[b * T + lane] : -1;
  int par = in ? (a.parents ? a.parents[b * T + lane] : lane - 1) : -3;
  if (par < -1 || par >= lane) par = -3; // padding: no node's child
  const bool valid = in && par != -3 && t64 >= 0 && t64 < a.V;
  tok = valid ? (int)t64 : -1;
  const float u = in ? a.u[b * (T + 1) + lane] : 0.f;
  double pm = 0.0, qm = 0.0;
  if (valid) {
    pm = mass(to_f32(((const P *)a.p)[b * a.p_sb + (int64_t)(par + 1) * a.p_st + tok]));
    if (a.q) qm = mass(to_f32(((const P *)a.q)[b * a.q_sb + (int64_t)lane * a.q_st + tok]));
  }
  VerState st;
  int n = 0;
  if (a.q) { // a chain
    const bool stays = valid && (double)u * qm < pm;
    const unsigned long long gone = ~__ballot(stays);
    n = gone ? min(__builtin_ctzll(gone), T) : T;
    st.row = n;
    st.rejected = n < T && ((__ballot(valid) >> n) & 1);
    st.children = 0;
    if (write && in) a.path[b * T + lane] = lane < n ? lane : -1;
  } else {
    // down from the context: the node's children in order, `below` the mass of
    // those passed; a token that an earlier sibling has counts as none
    int cur = -1, mine = -1;
    while (n < T) {
      const unsigned long long kids = __ballot(valid && par == cur);
      const double ud = (double)readlane_f32(u, n);
      double below = 0.0;
      int hit = -1;
      for (unsigned long long c = kids; c && hit < 0; c &= c - 1) {
        const int j = __builtin_ctzll(c);
        if (__ballot(tok == __builtin_amdgcn_readlane(tok, j)) & kids & ((1ull << j) - 1)) continue;
        const double up = below + readlane_f64(pm, j);
        if (below <= ud && ud < up) hit = j;
        below = up;
      }
      if (hit < 0) break;
      if (lane == n) mine = hit;
      cur = hit;
      ++n;
    }
    st.row = cur + 1;
    st.rejected = 0;
    st.children = __ballot(valid && par == cur);
    if (write && in) a.path[b * T + lane] = lane < n ? mine : -1;
  }
  if (write && lane == 0) {
    a.accepted[b] = n;
    a.state[b] = st;
  }
  return st;
}

constexpr int kVerEach = kVerChunk / 256; // masses of a thread

// A thread's masses of a chunk of n: i-th at place(i). Unconditional loads from
// clamped places, all before the first use; VEC: 16 bytes at a time.
template <bool RUNS> __device__ __forceinline__ int ver_place(int i, int per) {
  // RUNS: a thread's masses are neighbours; else 256 threads' runs of `per` are
  return RUNS ? threadIdx.x * kVerEach + i : (i / per * 256 + threadIdx.x) * per + i % per;
}
template <typename P, bool RUNS, bool VEC>
__device__ __forceinline__ void ver_load(const P *row, int n, float (&x)[kVerEach]) {
  constexpr int PER = VEC ? 16 / sizeof(P) : 1;
  typedef P V __attribute__((ext_vector_type(PER)));
#pragma unroll
  for (int i = 0; i < kVerEach; i += PER) {
    const int at = ver_place<RUNS>(i, PER);
    if constexpr (PER == 1) {
      x[i] = to_f32(row[min(at, n - 1)]);
    } else { // n is a multiple of PER
      const V v = *reinterpret_cast<const V *>(row + min(at, n - PER));
#pragma unroll
      for (int e = 0; e < PER; ++e) x[i + e] = to_f32(v[e]);
    }
    if (at >= n)
#pragma unroll
      for (int e = 0; e < PER; ++e) x[i + e] = 0.f;
  }
}
// Weights of the draw w and masses of the row f of a thread's part of a chunk.
template <typename P, bool RUNS, bool VEC>
__device__ __forceinline__ void ver_weights(const VerArgs &a, int64_t b, const VerState &st, int tok, int64_t base,
                                            double (&w)[kVerEach], double (&f)[kVerEach]) {
  const int n = (int)min((int64_t)kVerChunk, a.V - base);
  float x[kVerEach], y[kVerEach];
  ver_load<P, RUNS, VEC>((const P *)a.p + b * a.p_sb + (int64_t)st.row * a.p_st + base, n, x);
  if (st.rejected) ver_load<P, RUNS, VEC>((const P *)a.q + b * a.q_sb + (int64_t)st.row * a.q_st + base, n, y);
#pragma unroll
  for (int i = 0; i < kVerEach; ++i) {
    f[i] = mass(x[i]);
    w[i] = st.rejected ? fmax(f[i] - mass(y[i]), 0.0) : f[i];
  }
  for (unsigned long long c = st.children; c; c &= c - 1) {
    const int64_t at = (int64_t)__builtin_amdgcn_readlane(tok, __builtin_ctzll(c)) - base;
    if (at < 0 || at >= kVerChunk) continue;
#pragma unroll
    for (int i = 0; i < kVerEach; ++i)
      if (ver_place<RUNS>(i, VEC ? 16 / sizeof(P) : 1) == at) w[i] = 0.0;
  }
}
__device__ __forceinline__ double tree_sum(const double (&v)[kVerEach]) {
  double t[kVerEach / 2];
#pragma unroll
  for (int i = 0; i < kVerEach / 2; ++i) t[i] = v[2 * i] + v[2 * i + 1];
#pragma unroll
  for (int m = kVerEach / 4; m > 0; m /= 2)
#pragma unroll
    for (int i = 0; i < m; ++i) t[i] = t[2 * i] + t[2 * i + 1];
  return t[0];
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int sh = 1; sh < kWave; sh <<= 1) v += __shfl_xor(v, sh, kWave);
  return v;
}

template <typename P, bool VEC> __global__ __launch_bounds__(256) void ver_sum_kernel(VerArgs a) {
  __shared__ double red[4][2];
  const int64_t b = blockIdx.y;
  int tok;
  const VerState st = ver_walk<P>(a, b, blockIdx.x == 0 && threadIdx.x < kWave, tok);
  double w[kVerEach], f[kVerEach];
  ver_weights<P, false, VEC>(a, b, st, tok, (int64_t)blockIdx.x * kVerChunk, w, f);
  const double ws = wave_sum_f64(tree_sum(w)), fs = wave_sum_f64(tree_sum(f));
  if (lane_id() == 0) red[wave_id()][0] = ws, red[wave_id()][1] = fs;
  __syncthreads();
  if (threadIdx.x < 2)
    a.part[(b * a.chunks + blockIdx.x) * 2 + threadIdx.x] =
        (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
}

// inclusive sum over the wave's lanes
__device__ __forceinline__ double wave_scan_f64(double v) {
  const int lane = lane_id();
#pragma unroll
  for (int sh = 1; sh < kWave; sh <<= 1) {
    const double o = __shfl_up(v, sh, kWave);
    if (lane >= sh) v += o;
  }
  return v;
}

template <typename P, bool VEC> __global__ __launch_bounds__(256) void ver_pick_kernel(VerArgs a) {
  __shared__ double s_wave[4];
  __shared__ int s_found[4], s_last[4];
  const int64_t b = blockIdx.x;
  const int lane = lane_id();
  const VerState st = a.state[b];
  const int tok = lane < a.T ? (int)a.tok[b * a.T + lane] : -1;
  const double u = fmax((double)a.u[b * (a.T + 1) + a.T], 0.0);
  const double *part = a.part + b * a.chunks * 2;
  // 64 chunks at a time: the running sums of the draw's weights (which 0), or,
  // where those have none, of the whole row (1), to the end, then to the chunk
  int chunk = -1, which = 0;
  double before = 0.0, thr = 0.0;
  for (; which < 2 && chunk < 0; ++which) {
    double total = 0.0;
    for (int c = 0; c < a.chunks; c += kWave)
      total += __shfl(wave_scan_f64(c + lane < a.chunks ? part[(c + lane) * 2 + which] : 0.0), kWave - 1, kWave);
    if (!(total > 0.0)) continue;
    thr = u * total;
    double carry = 0.0;
    for (int c = 0; c < a.chunks; c += kWave) {
      const double own = c + lane < a.chunks ? part[(c + lane) * 2 + which] : 0.0;
      const double v = wave_scan_f64(own);
      const unsigned long long hit = __ballot(carry + v > thr && own > 0.0), pos = __ballot(own > 0.0);
      if (hit || pos) { // else, so far, the last chunk with mass
        const int l = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(pos);
        chunk = c + l, before = carry + (__shfl(v, l, kWave) - __shfl(own, l, kWave));
      }
      if (hit) break;
      carry += __shfl(v, kWave - 1, kWave);
    }
    if (chunk >= 0) break;
  }
  if (chunk < 0) { // (every wave)
    if (threadIdx.x == 0) a.next[b] = -1;
    return;
  }
  chunk = __builtin_amdgcn_readfirstlane(chunk);
  const int64_t base = (int64_t)chunk * kVerChunk;
  double w[kVerEach], f[kVerEach];
  ver_weights<P, true, VEC>(a, b, st, tok, base, w, f);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kVerEach; ++i) {
    w[i] = which ? f[i] : w[i];
    sum += w[i];
  }
  const double incl = wave_scan_f64(sum);
  if (lane == kWave - 1) s_wave[wave_id()] = incl;
  __syncthreads();
  double run = before;
  for (int i = 0; i < wave_id(); ++i) run += s_wave[i];
  run += incl - sum;
  int found = 0x7fffffff, last = -1;
#pragma unroll
  for (int i = 0; i < kVerEach; ++i) {
    run += w[i];
    if (w[i] > 0.0) {
      last = threadIdx.x * kVerEach + i;
      if (run > thr) found = min(found, last);
    }
  }
  // the first that passes, or the last with mass, of the wave, then of the block
  const unsigned long long hit = __ballot(found != 0x7fffffff), pos = __ballot(last >= 0);
  const int wf = hit ? __shfl(found, __builtin_ctzll(hit), kWave) : 0x7fffffff;
  const int wl = pos ? __shfl(last, 63 - __builtin_clzll(pos), kWave) : -1;
  if (lane == 0) s_found[wave_id()] = wf, s_last[wave_id()] = wl;
  __syncthreads();
  if (threadIdx.x == 0) {
    const int ff = min(min(s_found[0], s_found[1]), min(s_found[2], s_found[3]));
    const int ll = max(max(s_last[0], s_last[1]), max(s_last[2], s_last[3]));
    a.next[b] = base + (ff != 0x7fffffff ? ff : ll);
  }
}

static int64_t ver_chunks(int64_t V) { return (V + kVerChunk - 1) / kVerChunk; }

} // namespace tpp

using namespace tpp;

extern "C" size_t tpp_verify_draft_workspace_size(int64_t B, int64_t V) {
  if (B <= 0 || V <= 0) return 0;
  return (size_t)B * (size_t)ver_chunks(V) * 2 * sizeof(double) + (size_t)B * sizeof(VerState);
}

extern "C" int tpp_verify_draft(const int64_t *draft_tokens, const int32_t *parents,
                                const void *target_probs, const int64_t *target_strides,
                                const void *draft_probs, const int64_t *draft_strides,
                                const float *uniforms, int32_t *accepted, int32_t *path,
                                int64_t *next_token, int64_t B, int64_t T, int64_t V, int dtype,
                                void *workspace, size_t ws_bytes, void *stream) {
  const char *name = "tpp_verify_draft";
  if (!draft_tokens || !target_probs || !target_strides || !uniforms || !accepted || !path || !next_token ||
      (draft_probs && !draft_strides))
    return set_error(TPP_E_INVALID, "%s: null pointer", name);
  if (draft_probs && parents)
    return set_error(TPP_E_UNSUPPORTED, "%s: draft_probs go with a chain, not with a tree", name);
  if (dtype != TPP_F16 && dtype != TPP_BF16 && dtype != TPP_F32)
    return set_error(TPP_E_UNSUPPORTED, "%s: unsupported dtype %d", name, dtype);
  if (T < 1 || T > kVerMaxT)
    return set_error(TPP_E_UNSUPPORTED, "%s: %lld drafted tokens, 1 to %d are handled", name, (long long)T, kVerMaxT);
  if (B < 0 || V < 1 || V > 0x7fffffffLL) return set_error(TPP_E_INVALID, "%s: invalid shapes", name);
  if (B > 65535) return set_error(TPP_E_UNSUPPORTED, "%s: too many sequences", name);
  if (B == 0) return TPP_OK;
  if (!workspace || ((uintptr_t)workspace & 7) || ws_bytes < tpp_verify_draft_workspace_size(B, V))
    return set_error(TPP_E_WORKSPACE, "%s: workspace missing, unaligned or too small", name);
  VerArgs a = {};
  a.tok = draft_tokens, a.parents = parents, a.p = target_probs, a.q = draft_probs;
  a.p_sb = target_strides[0], a.p_st = target_strides[1];
  if (draft_probs) a.q_sb = draft_strides[0], a.q_st = draft_strides[1];
  a.u = uniforms, a.T = (int)T, a.V = V, a.chunks = (int)ver_chunks(V);
  a.accepted = accepted, a.path = path, a.next = next_token;
  a.part = (double *)workspace;
  a.state = (VerState *)(a.part + (size_t)B * a.chunks * 2);
  hipStream_t st = as_stream(stream);
  // 16 bytes at a time where every row begins at such an address and ends whole
  const int es = dtype == TPP_F32 ? 4 : 2;
  uint64_t low = (uint64_t)(uintptr_t)target_probs | (uint64_t)(a.p_sb * es) | (uint64_t)(a.p_st * es) | (uint64_t)(V * es);
  if (draft_probs) low |= (uint64_t)(uintptr_t)draft_probs | (uint64_t)(a.q_sb * es) | (uint64_t)(a.q_st * es);
  const bool vec = !(low & 15);
  auto go = [&](auto zero) {
    typedef decltype(zero) P;
    const dim3 grid((unsigned)a.chunks, (unsigned)B);
    if (vec) {
      ver_sum_kernel<P, true><<<grid, dim3(256), 0, st>>>(a);
      ver_pick_kernel<P, true><<<dim3((unsigned)B), dim3(256), 0, st>>>(a);
    } else {
      ver_sum_kernel<P, false><<<grid, dim3(256), 0, st>>>(a);
      ver_pick_kernel<P, false><<<dim3((unsigned)B), dim3(256), 0, st>>>(a);
    }
  };
  if (dtype == TPP_F32) go(0.f);
  else if (dtype == TPP_F16) go(f16(0));
  else go(bf16(0));
  return check_launch(name);
}
