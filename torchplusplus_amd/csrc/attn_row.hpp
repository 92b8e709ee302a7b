// One query row over given keys by one wave, for any head size up to 256 and any
// alignment: the kernels of last resort of packed_attention.hip and
// paged_attention.hip, and the rows that their matrix-core kernels sum again.
#pragma once
#include "tpp_common.hpp"

namespace tpp {

// What a wave has of a row: the running maximum of scale q.k in the exp2 domain, the
// sum of weights and the weighted sums of V, element 64 c + lane in acc[c].
struct AttnRow {
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  bool seen = false; // a row that sees nothing is 0, one whose scores are all -inf NaN
  __device__ __forceinline__ float out(int c) const { return seen ? acc[c] / l : 0.f; }
};

// A weight is times 2^-20, so that sums over 2^20 values of V near the end of bfloat16
// stay finite where their mean is.
constexpr float kRowUp = -20.f;

// Keys lo .. hi - 1; at(j, k, v): the rows of key j, false where it is not seen. Four
// keys at a time, all their loads ahead of the first reduction.
template <typename T, typename AT>
__device__ __forceinline__ void attn_row(AttnRow &r, const T *q, int D, int lo, int hi, float scale_log2, AT at) {
  constexpr int U = 4;
  const int lane = lane_id();
  float qv[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) qv[c] = c * 64 + lane < D ? to_f32(q[c * 64 + lane]) : 0.f;
  for (int j0 = lo; j0 < hi; j0 += U) {
    float s[U], v[U][4];
    bool see[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const T *kr = nullptr, *vr = nullptr;
      see[u] = j0 + u < hi && at(j0 + u, kr, vr); // wave-uniform
      s[u] = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bool on = see[u] && c * 64 + lane < D;
        s[u] += on ? qv[c] * to_f32(kr[c * 64 + lane]) : 0.f;
        v[u][c] = on ? to_f32(vr[c * 64 + lane]) : 0.f;
      }
    }
    float mn = r.m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s[u] = see[u] ? wave_sum(s[u]) * scale_log2 : -INFINITY;
      mn = fmaxf(mn, s[u]);
      r.seen = r.seen || see[u];
    }
    const float mc = mn == -INFINITY ? 0.f : mn, a = __builtin_amdgcn_exp2f(r.m - mc);
    r.l *= a;
#pragma unroll
    for (int c = 0; c < 4; ++c) r.acc[c] *= a;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!see[u]) continue; // (its weight of 0 times an infinity would be a NaN)
      const float e = __builtin_amdgcn_exp2f(s[u] - mc + kRowUp);
      r.l += e;
#pragma unroll
      for (int c = 0; c < 4; ++c) r.acc[c] = fmaf(e, v[u][c], r.acc[c]);
    }
    r.m = mn;
  }
}

} // namespace tpp
