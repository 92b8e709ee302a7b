// Attention of drafted tokens over a KV cache of 16-bit values or 8-bit codes.
//
//   o[b, t, h] = softmax_j(scale q[b, t, h] . K[b, j, h / G]) V[b, j, h / G]
// over the keys j < len_b of the sequence's context and those keys len_b + i
// that hold drafted token i where i is t or one of its ancestors (G = Hq / Hkv
// query heads share a KV head). `parents` gives each drafted token's parent:
// an earlier token, or -1 for the context's last; any other value marks
// padding, which sees nothing, as do its children. One token per sequence is
// decode over the cache. A row that sees nothing is 0.
// A code's value is code * 2^(exponent byte - 127), see kv_quant.hip; a row
// with exponent 255 is NaN.
#include "tpp_common.hpp"

namespace tpp {

constexpr int kTreeMaxT = 64;

struct TreeArgs {
  const void *q, *k, *v;
  void *o;
  const uint8_t *ke, *ve; // exponent bytes of coded caches
  const int32_t *seqlens, *parents;
  int64_t q_s[3], o_s[3];           // {batch, token, head}
  int64_t k_s[3], v_s[3], e_s[2];   // {batch, head, position}; {batch, head}
  int B, T, Hq, Hkv, G, Lmax;
  float scale_log2;
};

// Bit i of the result: this lane's token (lane index < T) sees drafted token
// i. Ancestors by doubling: after step s a lane holds those up to 2^s levels up.
__device__ __forceinline__ unsigned long long tree_bits(const TreeArgs &p, int b, int L) {
  const int lane = lane_id();
  int up = lane < p.T ? (p.parents ? p.parents[(int64_t)b * p.T + lane] : lane - 1) : -2;
  int none = up < -1 || up >= lane;
  if (none) up = -1;
  unsigned lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
#pragma unroll
  for (int s = 0; s < 6; ++s) {
    const int at = max(up, 0);
    const unsigned l = __shfl((int)lo, at, kWave), h = __shfl((int)hi, at, kWave);
    const int nn = __shfl(none, at, kWave), u2 = __shfl(up, at, kWave);
    if (up >= 0) {
      lo |= l, hi |= h, none |= nn;
      up = u2;
    }
  }
  // a token whose own row would lie past the cache's end sees nothing either
  return none || lane >= p.Lmax - L ? 0ull : ((unsigned long long)hi << 32) | lo;
}

// An element of a cache row as fp32 (KIND 0: of type T, else a tpp_code).
template <typename T, int KIND>
__device__ __forceinline__ float cache_value(const void *row, int d, float sc) {
  if constexpr (KIND == 0) return to_f32(((const T *)row)[d]);
  else if constexpr (KIND == TPP_CODE_E4M3)
    return __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t *)row)[d], 0) * sc;
  else return (float)((const int8_t *)row)[d] * sc;
}
__device__ __forceinline__ float exp_scale(const uint8_t *e, int64_t i) {
  return __uint_as_float(e[i] == 255 ? 0x7fc00000u : (unsigned)e[i] << 23);
}

// Any head size up to 256, any alignment: one wave per (sequence, token,
// head), keys one at a time with a wave reduction.
template <typename T, int KIND>
__global__ __launch_bounds__(64) void tree_generic_kernel(TreeArgs p, int D) {
  const int lane = lane_id(), t = blockIdx.x % p.T, h = blockIdx.x / p.T, b = blockIdx.y;
  const int hk = h / p.G;
  const int L = min(max(p.seqlens[b], 0), p.Lmax);
  const unsigned long long bits = tree_bits(p, b, L);
  const unsigned lo = __builtin_amdgcn_readlane((int)(unsigned)bits, t);
  const unsigned hi = __builtin_amdgcn_readlane((int)(unsigned)(bits >> 32), t);
  const unsigned long long see = ((unsigned long long)hi << 32) | lo;
  const T *qp = (const T *)p.q + b * p.q_s[0] + t * p.q_s[1] + h * p.q_s[2];
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < 4; ++c) q[c] = c * 64 + lane < D ? to_f32(qp[c * 64 + lane]) : 0.f;
  constexpr int EB = KIND == 0 ? 2 : 1;
  const char *kp = (const char *)p.k + (b * p.k_s[0] + hk * p.k_s[1]) * EB;
  const char *vp = (const char *)p.v + (b * p.v_s[0] + hk * p.v_s[1]) * EB;
  const int64_t eb = b * p.e_s[0] + hk * p.e_s[1];
  float m = -INFINITY, l = 0.f;
  const int end = see ? L + 64 - __builtin_clzll(see) : 0;
  for (int j = 0; j < end; ++j) {
    if (j >= L && !((see >> (j - L)) & 1)) continue;
    const char *kr = kp + (int64_t)j * p.k_s[2] * EB, *vr = vp + (int64_t)j * p.v_s[2] * EB;
    const float ks = KIND ? exp_scale(p.ke, eb + j) : 1.f, vs = KIND ? exp_scale(p.ve, eb + j) : 1.f;
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c * 64 + lane < D) s += q[c] * cache_value<T, KIND>(kr, c * 64 + lane, ks);
    s = wave_sum(s) * p.scale_log2;
    const float mn = fmaxf(m, s), mc = mn == -INFINITY ? 0.f : mn;
    const float a = __builtin_amdgcn_exp2f(m - mc), e = __builtin_amdgcn_exp2f(s - mc);
    l = l * a + e;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c * 64 + lane < D) o[c] = o[c] * a + e * cache_value<T, KIND>(vr, c * 64 + lane, vs);
    m = mn;
  }
  T *op = (T *)p.o + b * p.o_s[0] + t * p.o_s[1] + h * p.o_s[2];
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (c * 64 + lane < D) op[c * 64 + lane] = from_f32<T>(end ? o[c] / l : 0.f);
}

} // namespace tpp

using namespace tpp;

extern "C" size_t tpp_tree_attn_workspace_size(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int) {
  return 0;
}

extern "C" int tpp_tree_attn(const void *q, const void *k, const void *v, void *o, const void *k_exps,
                             const void *v_exps, const int64_t *q_strides, const int64_t *k_strides,
                             const int64_t *v_strides, const int64_t *exp_strides,
                             const int64_t *o_strides, const int32_t *seqlens,
                             const int32_t *parents, int64_t B, int64_t T, int64_t Hq, int64_t Hkv,
                             int64_t D, int64_t Lmax, float softmax_scale, int code, int dtype,
                             void *workspace, size_t ws_bytes, void *stream) {
  const char *name = "tpp_tree_attn";
  if (!q || !k || !v || !o || !seqlens || !q_strides || !k_strides || !v_strides || !o_strides)
    return set_error(TPP_E_INVALID, "%s: null pointer", name);
  if (!half_type(dtype)) return set_error(TPP_E_UNSUPPORTED, "%s: unsupported dtype %d", name, dtype);
  if (code != 0 && code != TPP_CODE_E4M3 && code != TPP_CODE_INT8)
    return set_error(TPP_E_UNSUPPORTED, "%s: unsupported code type %d", name, code);
  if (code && (!k_exps || !v_exps || !exp_strides))
    return set_error(TPP_E_INVALID, "%s: a coded cache needs its exponents", name);
  if (T < 1 || T > kTreeMaxT)
    return set_error(TPP_E_UNSUPPORTED, "%s: %lld drafted tokens, 1 to %d are handled", name, (long long)T, kTreeMaxT);
  if (B < 0 || Hkv < 1 || Hq < 1 || Hq % Hkv || Lmax < 1 || Lmax > 0x7fffffffLL - 256 || D < 1)
    return set_error(TPP_E_INVALID, "%s: invalid shapes", name);
  if (D > 256 || B > 65535 || Hq > 65535)
    return set_error(TPP_E_UNSUPPORTED, "%s: head_dim above 256, or too many sequences or heads", name);
  if (B == 0) return TPP_OK;
  TreeArgs a = {};
  a.q = q, a.k = k, a.v = v, a.o = o, a.ke = (const uint8_t *)k_exps, a.ve = (const uint8_t *)v_exps;
  a.seqlens = seqlens, a.parents = parents;
  for (int i = 0; i < 3; ++i)
    a.q_s[i] = q_strides[i], a.o_s[i] = o_strides[i], a.k_s[i] = k_strides[i], a.v_s[i] = v_strides[i];
  if (code) a.e_s[0] = exp_strides[0], a.e_s[1] = exp_strides[1];
  a.B = (int)B, a.T = (int)T, a.Hq = (int)Hq, a.Hkv = (int)Hkv, a.G = (int)(Hq / Hkv), a.Lmax = (int)Lmax;
  const float sc = softmax_scale > 0.f ? softmax_scale : 1.f / sqrtf((float)D);
  a.scale_log2 = sc * 1.4426950408889634f;
  hipStream_t st = as_stream(stream);
  (void)workspace, (void)ws_bytes;
  const dim3 grid((unsigned)(Hq * T), (unsigned)B);
  return TPP_DISPATCH_HALF(dtype, [&] {
    if (code == 0) tree_generic_kernel<T, 0><<<grid, dim3(64), 0, st>>>(a, (int)D);
    else if (code == TPP_CODE_E4M3) tree_generic_kernel<T, TPP_CODE_E4M3><<<grid, dim3(64), 0, st>>>(a, (int)D);
    else tree_generic_kernel<T, TPP_CODE_INT8><<<grid, dim3(64), 0, st>>>(a, (int)D);
    return check_launch(name);
  });
}
