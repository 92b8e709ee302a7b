// Attention of sequences of different lengths packed one behind the other: query
// token i of sequence b (rows cu_q[b] .. cu_q[b + 1] - 1) sees keys of rows cu_k[b] ..
// cu_k[b + 1] - 1 of its own sequence,
//   o[i, h] = softmax_j(scale q[i, h] . k[j, h / G]) v[j, h / G],
// causal and window bounds aligned bottom-right in each sequence (query i at key i + Lk -
// Lq). A row that sees nothing is 0, one whose scores are all -inf NaN.
#include "attn_row.hpp"

namespace tpp {

struct PackedArgs {
  const void *q, *k, *v;
  void *o;
  int64_t q_ss, q_sh, k_ss, k_sh, v_ss, v_sh, o_ss, o_sh;
  const int32_t *cu_q, *cu_k; // [B + 1]
  int B, Nq, Nk, Hq, Hkv;
  float scale_log2;
  int left, right; // window, -1 = unbounded; causal => right = 0
  int fill;        // rows of no sequence become 0 (else they stay as they were)
};

// Rows of sequence b; what is given is cut to the tensors, so that no read or write
// leaves them. Sequences B and B + 1 are the rows behind the last and ahead of the first.
struct PackedSeq {
  int q0, Sq, k0, Sk;
};
__device__ __forceinline__ PackedSeq packed_seq(const PackedArgs &p, int b) {
  PackedSeq s = {0, 0, 0, 0};
  const int qa = b > p.B ? 0 : min(max(p.cu_q[b], 0), p.Nq);
  const int qe = b < p.B ? p.cu_q[b + 1] : b == p.B ? p.Nq : p.cu_q[0];
  s.q0 = qa, s.Sq = max(min(qe, p.Nq) - qa, 0);
  if (b < p.B) {
    s.k0 = min(max(p.cu_k[b], 0), p.Nk);
    s.Sk = max(min(p.cu_k[b + 1], p.Nk) - s.k0, 0);
  }
  return s;
}

// Any head size up to 256, any alignment: one wave per (token, head).
template <typename T> __global__ __launch_bounds__(64) void packed_generic_kernel(PackedArgs p, int D) {
  const int lane = lane_id(), i = blockIdx.x, h = blockIdx.y, hk = h / (p.Hq / p.Hkv);
  // the sequence: the first whose end is past the token (64 ends at a time)
  int b = -1;
  for (int c = 0; c < p.B && b < 0; c += kWave) {
    const bool past = c + lane < p.B && i < p.cu_q[c + lane + 1];
    const unsigned long long hit = __ballot(past);
    if (hit) b = c + __builtin_ctzll(hit);
  }
  AttnRow r;
  const PackedSeq s = b < 0 ? PackedSeq{0, 0, 0, 0} : packed_seq(p, b);
  const bool none = b < 0 || i < s.q0 || i >= s.q0 + s.Sq;
  if (none && !p.fill) return;
  if (!none) {
    const int at = i - s.q0 + s.Sk - s.Sq; // the query's key
    const int lo = p.left >= 0 && (int64_t)at - p.left > 0 ? at - p.left : 0;
    const int hi = p.right >= 0 && (int64_t)at + p.right + 1 < s.Sk ? max(at + p.right + 1, 0) : s.Sk;
    attn_row<T>(r, (const T *)p.q + i * p.q_ss + h * p.q_sh, D, lo, hi, p.scale_log2,
                [&](int j, const T *&k, const T *&v) {
                  k = (const T *)p.k + (int64_t)(s.k0 + j) * p.k_ss + hk * p.k_sh;
                  v = (const T *)p.v + (int64_t)(s.k0 + j) * p.v_ss + hk * p.v_sh;
                  return true;
                });
  }
  T *op = (T *)p.o + i * p.o_ss + h * p.o_sh;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (c * 64 + lane < D) op[c * 64 + lane] = from_f32<T>(r.out(c));
}

} // namespace tpp

using namespace tpp;

extern "C" size_t tpp_attn_packed_workspace_size(int64_t B, int64_t Nq, int64_t Nk, int64_t Hq, int64_t Hkv, int64_t D) {
  return 0;
}

extern "C" int tpp_attn_packed(const void *q, const void *k, const void *v, void *o, const int64_t *q_strides,
                               const int64_t *k_strides, const int64_t *v_strides, const int64_t *o_strides,
                               const int32_t *cu_q, const int32_t *cu_k, int64_t B, int64_t Nq, int64_t Nk,
                               int64_t Hq, int64_t Hkv, int64_t D, float softmax_scale, int causal, int window_left,
                               int window_right, int fill, int dtype, void *workspace, size_t ws_bytes,
                               void *stream) {
  const char *name = "tpp_attn_packed";
  if (!q_strides || !k_strides || !v_strides || !o_strides)
    return set_error(TPP_E_INVALID, "%s: null stride array", name);
  if (!half_type(dtype)) return set_error(TPP_E_UNSUPPORTED, "%s: unsupported dtype %d", name, dtype);
  if (B < 0 || Nq < 0 || Nk < 0 || Hkv < 1 || Hq < 1 || Hq % Hkv || D < 1)
    return set_error(TPP_E_INVALID, "%s: invalid shapes", name);
  if (!cu_k && Nk != Nq) return set_error(TPP_E_INVALID, "%s: keys of their own need cu_k", name);
  if (D > 256 || Hq > 65535 || B > (1 << 20) || Nq >= (1 << 26) || Nk > (1 << 30))
    return set_error(TPP_E_UNSUPPORTED, "%s: head_dim above 256, or too many heads, sequences or tokens", name);
  if (Nq == 0 || (B == 0 && !fill)) return TPP_OK;
  if (!q || !o || (Nk > 0 && (!k || !v)) || !cu_q) return set_error(TPP_E_INVALID, "%s: null pointer", name);
  PackedArgs a = {};
  a.q = q, a.k = k, a.v = v, a.o = o;
  a.q_ss = q_strides[0], a.q_sh = q_strides[1], a.k_ss = k_strides[0], a.k_sh = k_strides[1];
  a.v_ss = v_strides[0], a.v_sh = v_strides[1], a.o_ss = o_strides[0], a.o_sh = o_strides[1];
  a.cu_q = cu_q, a.cu_k = cu_k ? cu_k : cu_q;
  a.B = (int)B, a.Nq = (int)Nq, a.Nk = (int)Nk, a.Hq = (int)Hq, a.Hkv = (int)Hkv;
  const float sc = softmax_scale > 0.f ? softmax_scale : 1.f / sqrtf((float)D);
  a.scale_log2 = sc * 1.4426950408889634f;
  a.left = window_left < 0 ? -1 : window_left;
  a.right = causal ? 0 : window_right < 0 ? -1 : window_right;
  a.fill = fill;
  hipStream_t st = as_stream(stream);
  return TPP_DISPATCH_HALF(dtype, [&] {
    packed_generic_kernel<T><<<dim3((unsigned)Nq, (unsigned)Hq), dim3(64), 0, st>>>(a, (int)D);
    return check_launch(name);
  });
}
