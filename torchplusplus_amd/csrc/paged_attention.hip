// Attention of one new token a sequence over a cache held in pages:
//   o[b, h] = softmax_j(scale q[b, h] . K[j, h / G]) V[j, h / G],  j < seqlens[b],
// key j in row j % page_size of page block_tables[b, j / page_size] (and, in a window,
// j >= seqlens[b] - 1 - left). The positions of an entry that is no page (outside [0,
// pages)) are not seen. A row that sees nothing is 0, one whose scores are all -inf NaN.
#include "attn_row.hpp"

namespace tpp {

struct PagedArgs {
  const void *q, *k, *v;
  void *o;
  int64_t q_s[2], o_s[2];   // {sequence, head}
  int64_t k_s[3], v_s[3];   // {page, head, row}
  const int32_t *table, *seqlens;
  int64_t t_sb;
  int B, Hq, Hkv, G, pages, lpage, Lmax; // pages of 2^lpage rows; Lmax: the table's positions
  float scale_log2;
  int left;
};

// Any head size up to 256, any alignment: one wave per (sequence, head).
template <typename T> __global__ __launch_bounds__(64) void paged_generic_kernel(PagedArgs p, int D) {
  const int lane = lane_id(), h = blockIdx.x, b = blockIdx.y, hk = h / p.G;
  const int L = min(max(p.seqlens[b], 0), p.Lmax);
  const int lo = p.left >= 0 ? max(L - 1 - p.left, 0) : 0;
  const int32_t *table = p.table + b * p.t_sb;
  AttnRow r;
  attn_row<T>(r, (const T *)p.q + b * p.q_s[0] + h * p.q_s[1], D, lo, L, p.scale_log2,
              [&](int j, const T *&k, const T *&v) {
                const int pg = __builtin_amdgcn_readfirstlane(table[j >> p.lpage]);
                if (pg < 0 || pg >= p.pages) return false;
                const int64_t row = j & ((1 << p.lpage) - 1);
                k = (const T *)p.k + pg * p.k_s[0] + hk * p.k_s[1] + row * p.k_s[2];
                v = (const T *)p.v + pg * p.v_s[0] + hk * p.v_s[1] + row * p.v_s[2];
                return true;
              });
  T *op = (T *)p.o + b * p.o_s[0] + h * p.o_s[1];
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (c * 64 + lane < D) op[c * 64 + lane] = from_f32<T>(r.out(c));
}

} // namespace tpp

using namespace tpp;

extern "C" size_t tpp_attn_paged_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t Lmax) { return 0; }

extern "C" int tpp_attn_paged(const void *q, const void *k_pages, const void *v_pages, void *o,
                              const int64_t *q_strides, const int64_t *k_strides, const int64_t *v_strides,
                              const int64_t *o_strides, const int32_t *block_tables, int64_t table_stride,
                              int64_t table_pages, const int32_t *seqlens, int64_t B, int64_t Hq, int64_t Hkv,
                              int64_t D, int64_t pages, int64_t page_size, float softmax_scale, int window_left,
                              int dtype, void *workspace, size_t ws_bytes, void *stream) {
  const char *name = "tpp_attn_paged";
  if (!q_strides || !k_strides || !v_strides || !o_strides)
    return set_error(TPP_E_INVALID, "%s: null stride array", name);
  if (!half_type(dtype)) return set_error(TPP_E_UNSUPPORTED, "%s: unsupported dtype %d", name, dtype);
  if (B < 0 || Hkv < 1 || Hq < 1 || Hq % Hkv || D < 1 || pages < 0 || table_pages < 0 || table_stride < 0)
    return set_error(TPP_E_INVALID, "%s: invalid shapes", name);
  int lpage = 4;
  while (lpage < 10 && (1 << lpage) != page_size) ++lpage;
  if ((1 << lpage) != page_size)
    return set_error(TPP_E_UNSUPPORTED, "%s: pages of %lld rows; powers of two from 16 to 1024 are handled", name,
                     (long long)page_size);
  if (D > 256 || B > 65535 || Hq > 65535 || pages > 0x7fffffffLL || table_pages > (0x7fffffffLL >> lpage) - 1)
    return set_error(TPP_E_UNSUPPORTED, "%s: head_dim above 256, or too many sequences, heads or pages", name);
  if (B == 0) return TPP_OK;
  if (!q || !o || !seqlens || (pages > 0 && (!k_pages || !v_pages)) || (table_pages > 0 && !block_tables))
    return set_error(TPP_E_INVALID, "%s: null pointer", name);
  PagedArgs a = {};
  a.q = q, a.k = k_pages, a.v = v_pages, a.o = o;
  for (int i = 0; i < 2; ++i) a.q_s[i] = q_strides[i], a.o_s[i] = o_strides[i];
  for (int i = 0; i < 3; ++i) a.k_s[i] = k_strides[i], a.v_s[i] = v_strides[i];
  a.table = block_tables, a.t_sb = table_stride, a.seqlens = seqlens;
  a.B = (int)B, a.Hq = (int)Hq, a.Hkv = (int)Hkv, a.G = (int)(Hq / Hkv);
  a.pages = (int)pages, a.lpage = lpage, a.Lmax = (int)(table_pages << lpage);
  const float sc = softmax_scale > 0.f ? softmax_scale : 1.f / sqrtf((float)D);
  a.scale_log2 = sc * 1.4426950408889634f;
  a.left = window_left < 0 ? -1 : window_left;
  hipStream_t st = as_stream(stream);
  return TPP_DISPATCH_HALF(dtype, [&] {
    paged_generic_kernel<T><<<dim3((unsigned)Hq, (unsigned)B), dim3(64), 0, st>>>(a, (int)D);
    return check_launch(name);
  });
}
