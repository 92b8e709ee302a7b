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
// Two launches. The first cuts the row that the walk ends at into chunks of
// 4096 masses and sums each (every block repeats the walk: a gather of one
// mass per drafted token, all at once, then a walk in registers; cheaper than
// a launch of its own). The second finds the chunk and the index. What bounds
// it: the latency of both launches and the dependent gathers; the rows are
// B V 4 bytes (with q twice that).
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
__device__ VerState ver_walk(const VerArgs &a, int64_t b, bool write) {
  const int lane = lane_id(), T = a.T;
  const bool in = lane < T;
  const int64_t t64 = in ? a.tok[b * T + lane] : -1;
  int par = in ? (a.parents ? a.parents[b * T + lane] : lane - 1) : -3;
  if (par < -1 || par >= lane) par = -3; // padding: no node's child
  const bool valid = in && par != -3 && t64 >= 0 && t64 < a.V;
  const int tok = valid ? (int)t64 : -1;
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
    // mass of earlier siblings; a token that one of them has counts as none
    double below = 0.0;
    bool dup = !valid;
    for (int j = 0; j < T; ++j) {
      const int pj = __builtin_amdgcn_readlane(par, j), tj = __builtin_amdgcn_readlane(tok, j);
      const double mj = readlane_f64(dup ? 0.0 : pm, j);
      if (j < lane && pj == par) {
        below += mj;
        dup |= tj == tok;
      }
    }
    int cur = -1, mine = -1;
    while (n < T) {
      const double ud = (double)readlane_f32(u, n);
      const unsigned long long hit = __ballot(!dup && par == cur && below <= ud && ud < below + pm);
      if (!hit) break;
      cur = __builtin_ctzll(hit);
      if (lane == n) mine = cur;
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

// Bits of a chunk's masses that are children of the node (one per token).
__device__ __forceinline__ void mark_children(const VerArgs &a, int64_t b, const VerState &st,
                                              int64_t base, unsigned *ex) {
  for (int i = threadIdx.x; i < kVerChunk / 32; i += blockDim.x) ex[i] = 0;
  __syncthreads();
  if (threadIdx.x < a.T && ((st.children >> threadIdx.x) & 1)) {
    const int64_t t = a.tok[b * a.T + threadIdx.x] - base;
    if (t >= 0 && t < kVerChunk) atomicOr(&ex[t / 32], 1u << (t % 32));
  }
  __syncthreads();
}

// weights of index base + i (i in the chunk): of the draw, and of the row
template <typename P>
__device__ __forceinline__ void weights(const P *p, const P *q, int i, const unsigned *ex, double &w,
                                        double &full) {
  full = mass(to_f32(p[i]));
  w = q ? fmax(full - mass(to_f32(q[i])), 0.0) : ((ex[i / 32] >> (i % 32)) & 1) ? 0.0 : full;
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int sh = 1; sh < kWave; sh <<= 1) v += __shfl_xor(v, sh, kWave);
  return v;
}

template <typename P> __global__ __launch_bounds__(256) void ver_sum_kernel(VerArgs a) {
  __shared__ unsigned ex[kVerChunk / 32];
  __shared__ double red[4][2];
  __shared__ VerState s_st;
  const int64_t b = blockIdx.y;
  if (wave_id() == 0) {
    const VerState st = ver_walk<P>(a, b, blockIdx.x == 0);
    if (threadIdx.x == 0) s_st = st;
  }
  __syncthreads();
  const VerState st = s_st;
  const int64_t base = (int64_t)blockIdx.x * kVerChunk;
  const int n = (int)min((int64_t)kVerChunk, a.V - base);
  mark_children(a, b, st, base, ex);
  const P *p = (const P *)a.p + b * a.p_sb + (int64_t)st.row * a.p_st + base;
  const P *q = st.rejected ? (const P *)a.q + b * a.q_sb + (int64_t)st.row * a.q_st + base : nullptr;
  double w = 0.0, f = 0.0;
#pragma unroll 8
  for (int i = threadIdx.x; i < n; i += 256) {
    double wi, fi;
    weights(p, q, i, ex, wi, fi);
    w += wi, f += fi;
  }
  w = wave_sum_f64(w), f = wave_sum_f64(f);
  if (lane_id() == 0) red[wave_id()][0] = w, red[wave_id()][1] = f;
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

template <typename P> __global__ __launch_bounds__(1024) void ver_pick_kernel(VerArgs a) {
  __shared__ unsigned ex[kVerChunk / 32];
  __shared__ double s_wave[16], s_before, s_thr;
  __shared__ int s_chunk, s_which, s_found, s_last;
  const int64_t b = blockIdx.x;
  const VerState st = a.state[b];
  const double *part = a.part + b * a.chunks * 2;
  if (wave_id() == 0) {
    const int lane = lane_id();
    double total = 0.0;
    int which = 0;
    for (; which < 2; ++which) { // the draw's weights, else the whole row
      total = 0.0;
      for (int c = 0; c < a.chunks; c += kWave) {
        const double v = wave_scan_f64(c + lane < a.chunks ? part[(c + lane) * 2 + which] : 0.0);
        total += __shfl(v, kWave - 1, kWave);
      }
      if (total > 0.0) break;
    }
    const float u = a.u[b * (a.T + 1) + a.T];
    const double thr = fmax((double)u, 0.0) * total;
    int chunk = -1;
    double before = 0.0;
    if (which < 2) {
      double carry = 0.0;
      int lastpos = -1; // the last chunk with mass
      double lastbefore = 0.0;
      for (int c = 0; c < a.chunks && chunk < 0; c += kWave) {
        const double own = c + lane < a.chunks ? part[(c + lane) * 2 + which] : 0.0;
        const double v = wave_scan_f64(own);
        const unsigned long long hit = __ballot(carry + v > thr && own > 0.0), pos = __ballot(own > 0.0);
        const int l = hit ? __builtin_ctzll(hit) : pos ? 63 - __builtin_clzll(pos) : 0;
        const double bf = carry + __shfl(v, l, kWave) - __shfl(own, l, kWave);
        if (hit) chunk = c + l, before = bf;
        else if (pos) lastpos = c + l, lastbefore = bf;
        carry += __shfl(v, kWave - 1, kWave);
      }
      if (chunk < 0) chunk = lastpos, before = lastbefore;
    }
    if (lane == 0) s_chunk = chunk, s_which = which, s_before = before, s_thr = thr, s_found = 0x7fffffff, s_last = -1;
  }
  __syncthreads();
  const int chunk = s_chunk, which = s_which;
  if (chunk < 0) {
    if (threadIdx.x == 0) a.next[b] = -1;
    return;
  }
  const int64_t base = (int64_t)chunk * kVerChunk;
  const int n = (int)min((int64_t)kVerChunk, a.V - base);
  mark_children(a, b, st, base, ex);
  const P *p = (const P *)a.p + b * a.p_sb + (int64_t)st.row * a.p_st + base;
  const P *q = st.rejected ? (const P *)a.q + b * a.q_sb + (int64_t)st.row * a.q_st + base : nullptr;
  double w[4], sum = 0.0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = threadIdx.x * 4 + j;
    double x = 0.0, f = 0.0;
    if (i < n) weights(p, q, i, ex, x, f);
    w[j] = which ? f : x;
    sum += w[j];
  }
  const double incl = wave_scan_f64(sum);
  if (lane_id() == kWave - 1) s_wave[wave_id()] = incl;
  __syncthreads();
  double run = s_before;
  for (int i = 0; i < wave_id(); ++i) run += s_wave[i];
  run += incl - sum;
  int found = 0x7fffffff, last = -1;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    run += w[j];
    if (w[j] > 0.0) {
      last = threadIdx.x * 4 + j;
      if (run > s_thr) found = min(found, last);
    }
  }
  if (found != 0x7fffffff) atomicMin(&s_found, found);
  if (last >= 0) atomicMax(&s_last, last);
  __syncthreads();
  if (threadIdx.x == 0) a.next[b] = base + (s_found != 0x7fffffff ? s_found : s_last);
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
  auto go = [&](auto zero) {
    typedef decltype(zero) P;
    ver_sum_kernel<P><<<dim3((unsigned)a.chunks, (unsigned)B), dim3(256), 0, st>>>(a);
    ver_pick_kernel<P><<<dim3((unsigned)B), dim3(1024), 0, st>>>(a);
  };
  if (dtype == TPP_F32) go(0.f);
  else if (dtype == TPP_F16) go(f16(0));
  else go(bf16(0));
  return check_launch(name);
}
