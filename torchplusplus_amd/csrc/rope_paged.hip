// The step between a packed batch's fused projection and its attention, in one pass: per
// head RMSNorm of q and k (y = x / sqrt(mean(x^2) + eps) * w; none without weights),
// rotate-half RoPE at each token's own position, keys and values into their rows of a
// paged cache:
//   q_out, k_out = y cos(p) + (-y_hi, y_lo) sin(p),  page rows = k_out, v
// cos and sin are rows of tables [ctx, D]. One rounding, at the end. A token at a position
// outside [0, ctx) is padding: its q and k become 0 and no page row is written, nor is one
// for a slot outside [0, pages * page_size).
//
// Bound by HBM: q, k and v are read once, q, k and the two page rows written once. D / 16
// lanes share a row, each with 8 elements of either half, so a rotation's pair is in one
// lane and the norm is a DPP sum over the row's lanes. 16000 tokens of 16 + 8 + 8 heads of
// 128, 295 MB: 48.5 us in the trace, 6.1 TB/s; 32 tokens: 3.1, a launch and one round trip.
#include "tpp_common.hpp"

namespace tpp {

struct RopePagedArgs {
  const void *qkv;
  void *q, *k, *kp, *vp; // k: null if the rotated keys are wanted in their pages alone
  const void *qw, *kw, *cos, *sin;
  const int32_t *pos;
  const int64_t *slots;
  int64_t qkv_s, kp_s[3], vp_s[3]; // token; {page, head, row}
  int64_t slots_end;               // pages * page_size
  int N, Hq, Hk, ctx, lpage;
  float eps;
};

template <typename T, typename CS, int LPR>
__global__ __launch_bounds__(256) void rope_paged_kernel(RopePagedArgs p) {
  constexpr int D = LPR * 16;
  typedef typename VecT<T>::v8 V8;
  const int H = p.Hq + 2 * p.Hk;
  const int64_t row = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int i0 = (threadIdx.x % LPR) * 8;
  const bool valid = row < (int64_t)p.N * H;
  const int tok = valid ? (int)(row / H) : 0, head = valid ? (int)(row - (int64_t)tok * H) : 0;
  const bool is_q = head < p.Hq, is_k = !is_q && head < p.Hq + p.Hk;
  const T *src = (const T *)p.qkv + tok * p.qkv_s + (int64_t)head * D;
  const int pos = p.pos[tok];
  const bool real = pos >= 0 && pos < p.ctx;
  const int64_t slot = is_q ? 0 : p.slots[tok], cr = (int64_t)(real ? pos : 0) * D;
  const V8 r1 = ld_nt(reinterpret_cast<const V8 *>(src + i0));
  const V8 r2 = ld_nt(reinterpret_cast<const V8 *>(src + D / 2 + i0));
  const T *nw = (const T *)(is_q ? p.qw : p.kw);
  float x1[8], x2[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x1[j] = to_f32(r1[j]), x2[j] = to_f32(r2[j]);
  if (is_q || is_k) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += x1[j] * x1[j] + x2[j] * x2[j];
    ss = group_sum<LPR>(ss); // (the lanes of a row are all here)
    float c1[8], c2[8], s1[8], s2[8];
    load_cs8((const CS *)p.cos + cr + i0, c1);
    load_cs8((const CS *)p.cos + cr + D / 2 + i0, c2);
    load_cs8((const CS *)p.sin + cr + i0, s1);
    load_cs8((const CS *)p.sin + cr + D / 2 + i0, s2);
    if (nw) {
      const float inv = rsqrtf(ss / (float)D + p.eps);
      float w1[8], w2[8];
      load8(nw + i0, w1);
      load8(nw + D / 2 + i0, w2);
#pragma unroll
      for (int j = 0; j < 8; ++j) x1[j] = x1[j] * inv * w1[j], x2[j] = x2[j] * inv * w2[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = x1[j], b = x2[j];
      x1[j] = real ? a * c1[j] - b * s1[j] : 0.f;
      x2[j] = real ? b * c2[j] + a * s2[j] : 0.f;
    }
  }
  if (!valid) return;
  if (is_q || (is_k && p.k)) {
    T *dst = is_q ? (T *)p.q + ((int64_t)tok * p.Hq + head) * D : (T *)p.k + ((int64_t)tok * p.Hk + head - p.Hq) * D;
    store8(dst + i0, x1);
    store8(dst + D / 2 + i0, x2);
  }
  if (is_q || !real || slot < 0 || slot >= p.slots_end) return;
  const int hk = is_k ? head - p.Hq : head - p.Hq - p.Hk;
  const int64_t *st = is_k ? p.kp_s : p.vp_s;
  T *dst = (T *)(is_k ? p.kp : p.vp) + (slot >> p.lpage) * st[0] + hk * st[1] + (slot & ((1 << p.lpage) - 1)) * st[2];
  store8(dst + i0, x1);
  store8(dst + D / 2 + i0, x2);
}

} // namespace tpp

using namespace tpp;

extern "C" int tpp_qkv_rope_paged(const void *qkv, int64_t qkv_stride, void *q_out, void *k_out, void *k_pages,
                                  void *v_pages, const int64_t *k_strides, const int64_t *v_strides,
                                  const void *q_norm_w, const void *k_norm_w, const void *cos, const void *sin,
                                  int64_t ctx, const int32_t *positions, const int64_t *slots, int64_t N,
                                  int64_t Hq, int64_t Hkv, int64_t D, int64_t pages, int64_t page_size, float eps,
                                  int dtype, int cs_dtype, void *stream) {
  const char *name = "tpp_qkv_rope_paged";
  if (!k_strides || !v_strides) return set_error(TPP_E_INVALID, "%s: null stride array", name);
  if (!half_type(dtype)) return set_error(TPP_E_UNSUPPORTED, "%s: unsupported dtype %d", name, dtype);
  if (cs_dtype != TPP_F16 && cs_dtype != TPP_BF16 && cs_dtype != TPP_F32)
    return set_error(TPP_E_UNSUPPORTED, "%s: cos/sin dtype must be f16, bf16 or f32", name);
  if (D != 64 && D != 128 && D != 256)
    return set_error(TPP_E_UNSUPPORTED, "%s: head_dim %lld not in {64,128,256}", name, (long long)D);
  if (N < 0 || Hq < 1 || Hkv < 1 || Hq > 65535 || Hkv > 65535 || ctx < 1 || ctx > 0x7fffffffLL || pages < 0 ||
      pages > 0x7fffffffLL || qkv_stride < (Hq + 2 * Hkv) * D)
    return set_error(TPP_E_INVALID, "%s: invalid shapes", name);
  int lpage = 4;
  while (lpage < 10 && (1 << lpage) != page_size) ++lpage;
  if ((1 << lpage) != page_size)
    return set_error(TPP_E_UNSUPPORTED, "%s: pages of %lld rows; powers of two from 16 to 1024 are handled", name,
                     (long long)page_size);
  const int64_t rpb = 256 / (D / 16), rows = N * (Hq + 2 * Hkv);
  if (N > 0x7fffffffLL || (rows + rpb - 1) / rpb > 0xffffff) // (a grid has fewer than 2^32 threads)
    return set_error(TPP_E_UNSUPPORTED, "%s: too many tokens", name);
  if (N == 0) return TPP_OK;
  if (!qkv || !q_out || !cos || !sin || !positions || !slots || (pages > 0 && (!k_pages || !v_pages)))
    return set_error(TPP_E_INVALID, "%s: null pointer", name);
  uint64_t low = 0;
  for (const void *x : {qkv, (const void *)q_out, (const void *)k_out, (const void *)k_pages, (const void *)v_pages,
                        q_norm_w, k_norm_w, cos, sin})
    low |= (uint64_t)(uintptr_t)x;
  for (int i = 0; i < 3; ++i) low |= (uint64_t)(k_strides[i] * 2) | (uint64_t)(v_strides[i] * 2);
  if ((low | (uint64_t)(qkv_stride * 2)) & 15)
    return set_error(TPP_E_INVALID, "%s: 16-byte aligned pointers and strides required", name);
  RopePagedArgs a = {};
  a.qkv = qkv, a.q = q_out, a.k = k_out, a.kp = k_pages, a.vp = v_pages;
  a.qw = q_norm_w, a.kw = k_norm_w, a.cos = cos, a.sin = sin, a.pos = positions, a.slots = slots;
  a.qkv_s = qkv_stride;
  for (int i = 0; i < 3; ++i) a.kp_s[i] = k_strides[i], a.vp_s[i] = v_strides[i];
  a.slots_end = pages << lpage;
  a.N = (int)N, a.Hq = (int)Hq, a.Hk = (int)Hkv, a.ctx = (int)ctx, a.lpage = lpage, a.eps = eps;
  hipStream_t st = as_stream(stream);
  return TPP_DISPATCH_HALF(dtype, [&] {
    auto go = [&](auto *tab, auto lpr) {
      typedef std::remove_pointer_t<decltype(tab)> CS;
      rope_paged_kernel<T, CS, decltype(lpr)::value><<<dim3((unsigned)((rows + rpb - 1) / rpb)), dim3(256), 0, st>>>(a);
    };
    auto dims = [&](auto *tab) {
      if (D == 64) go(tab, std::integral_constant<int, 4>{});
      else if (D == 128) go(tab, std::integral_constant<int, 8>{});
      else go(tab, std::integral_constant<int, 16>{});
    };
    if (cs_dtype == TPP_F32) dims((float *)nullptr);
    else if (cs_dtype == TPP_F16) dims((f16 *)nullptr);
    else dims((bf16 *)nullptr);
    return check_launch(name);
  });
}
