// Rotary embedding at given positions: q and k rows of [B, S, H, D] (free
// batch / token / head strides) rotated at positions[b, s], pair by pair:
//   half layout:        pair j = elements (j, j + R/2)
//   interleaved layout: pair j = elements (2j, 2j + 1)
//   a' = a cos(t) - b sin(t), b' = b cos(t) + a sin(t), t = pos * inv_freq[j],
// cos and sin times `factor`, for the first R elements of a head; the rest of
// a head, and tokens at negative positions (padding), are copied. Drafted
// tokens of a tree sit at positions that are no run, which tables indexed by
// the token (rope.hip) do not serve.
//
// The angle is formed here and not read from a table: a table of a 10^6-token
// context is 1 GB in fp32, and the rows a batch needs are scattered over it.
// pos * inv_freq needs more than fp32 (at position 10^6 its rounding is 0.06
// rad), so the turns pos * inv_freq / (2 pi) are formed in fp64, reduced to
// [-1/2, 1/2] there, and only then rounded to fp32: v_sin_f32 / v_cos_f32 take
// turns and were within 1.3e-7 of sin and cos over that range.
//
// Bound by HBM: each element is read once and written once. A thread owns PW
// pairs of one token (16-byte accesses at PW = 8) in one head, or in four where there
// is work enough: their loads are in flight while the angles are worked out (4 x 4096
// tokens, 16 + 8 heads of 128, half of each turned: 45.0 -> 41.6 us, 4.84 TB/s, 95% of
// a copy's rate). Non-temporal stores were 19% slower.
#include "tpp_common.hpp"

namespace tpp {

struct RopeAtArgs {
  const void *q, *k;
  void *qo, *ko;
  int64_t qs[3], ks[3], qos[3], kos[3]; // {batch, token, head} strides
  const void *pos;
  int64_t pos_sb;
  const double *inv_freq;
  float factor;
  int S, Hq, Hk, D, R, pos64;
  unsigned upt, hgroups, units; // units = B * S * hgroups * upt
};

template <typename T, int PW, bool IL, int U>
__global__ __launch_bounds__(256) void rope_at_kernel(RopeAtArgs p) {
  typedef uint16_t W __attribute__((ext_vector_type(PW))); // PW elements
  const unsigned id = blockIdx.x * 256u + threadIdx.x; // (units < 2^32)
  if (id >= p.units) return;
  // unit (fastest), head group, token
  const unsigned r = id / p.upt, tok = r / p.hgroups;
  const int u = (int)(id - r * p.upt), hg = (int)(r - tok * p.hgroups);
  const int64_t b = tok / (unsigned)p.S, s = tok - (unsigned)b * (unsigned)p.S;
  const int64_t at = b * p.pos_sb + s;
  const int64_t pos = p.pos64 ? ((const int64_t *)p.pos)[at] : ((const int32_t *)p.pos)[at];
  // the unit's two runs of PW elements: of pairs, or past R copied
  const bool turn = u * 2 * PW < p.R && pos >= 0;
  const int lo = IL || u * 2 * PW >= p.R ? u * 2 * PW : u * PW;
  const int hi = IL || u * 2 * PW >= p.R ? lo + PW : lo + p.R / 2;
  if (!turn && p.q == p.qo && p.k == p.ko) return; // in place: nothing to copy
  const int H = p.Hq + p.Hk, h0 = hg * U, h1 = min(h0 + U, H);
  // U heads' loads before anything is worked out
  T *dst[U];
  W x[U], y[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int hc = min(h0 + i, h1 - 1); // (past the last: the last again, not stored)
    const bool isq = hc < p.Hq;
    const int hh = isq ? hc : hc - p.Hq;
    const int64_t *is = isq ? p.qs : p.ks, *os = isq ? p.qos : p.kos;
    const T *src = (const T *)(isq ? p.q : p.k) + b * is[0] + s * is[1] + hh * is[2];
    dst[i] = (T *)(isq ? p.qo : p.ko) + b * os[0] + s * os[1] + hh * os[2];
    x[i] = ld_nt(reinterpret_cast<const W *>(src + lo)), y[i] = ld_nt(reinterpret_cast<const W *>(src + hi));
  }
  float c[PW], sn[PW];
  if (turn) {
#pragma unroll
    for (int j = 0; j < PW; ++j) {
      const double t = (double)pos * (p.inv_freq[u * PW + j] * 0.15915494309189535); // 1 / (2 pi)
      const float f = (float)(t - __builtin_rint(t));
      c[j] = __builtin_amdgcn_cosf(f) * p.factor;
      sn[j] = __builtin_amdgcn_sinf(f) * p.factor;
    }
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if (i && h0 + i >= h1) break;
    if (turn) {
      float v[2 * PW];
#pragma unroll
      for (int j = 0; j < PW; ++j) {
        v[j] = to_f32(__builtin_bit_cast(T, (uint16_t)x[i][j]));
        v[PW + j] = to_f32(__builtin_bit_cast(T, (uint16_t)y[i][j]));
      }
#pragma unroll
      for (int j = 0; j < PW; ++j) {
        const int ia = IL ? 2 * j : j, ib = IL ? 2 * j + 1 : PW + j;
        const float a = v[ia], bb = v[ib];
        v[ia] = a * c[j] - bb * sn[j];
        v[ib] = bb * c[j] + a * sn[j];
      }
#pragma unroll
      for (int j = 0; j < PW; ++j) {
        x[i][j] = __builtin_bit_cast(uint16_t, from_f32<T>(v[j]));
        y[i][j] = __builtin_bit_cast(uint16_t, from_f32<T>(v[PW + j]));
      }
    }
    *reinterpret_cast<W *>(dst[i] + lo) = x[i];
    *reinterpret_cast<W *>(dst[i] + hi) = y[i];
  }
}

} // namespace tpp

using namespace tpp;

extern "C" int tpp_rope_at(const void *q, const void *k, void *q_out, void *k_out,
                           const int64_t *q_strides, const int64_t *k_strides,
                           const int64_t *qo_strides, const int64_t *ko_strides,
                           const void *positions, int64_t pos_stride, int pos_is_64,
                           const double *inv_freq, float factor, int64_t B, int64_t S, int64_t Hq,
                           int64_t Hk, int64_t D, int64_t R, int interleaved, int dtype,
                           void *stream) {
  const char *name = "tpp_rope_at";
  if (!q || !q_out || (Hk > 0 && (!k || !k_out)) || !positions || !inv_freq || !q_strides ||
      !qo_strides || (Hk > 0 && (!k_strides || !ko_strides)))
    return set_error(TPP_E_INVALID, "%s: null pointer", name);
  if (!half_type(dtype)) return set_error(TPP_E_UNSUPPORTED, "%s: unsupported dtype %d", name, dtype);
  if (B < 0 || S < 0 || Hq < 1 || Hk < 0 || D < 2 || D % 2 || R < 2 || R % 2 || R > D || pos_stride < 0)
    return set_error(TPP_E_INVALID, "%s: invalid shapes (even head_dim, even rotary <= head_dim)", name);
  if (S > 0x7fffffffLL || Hq + Hk > 65536 || D > 65536)
    return set_error(TPP_E_UNSUPPORTED, "%s: too many tokens, heads or elements", name);
  if (B == 0 || S == 0) return TPP_OK;
  RopeAtArgs a = {};
  a.q = q, a.k = Hk ? k : q, a.qo = q_out, a.ko = Hk ? k_out : q_out;
  // pairs per thread: the widest whose accesses are whole and aligned
  uint64_t low = (uint64_t)(uintptr_t)q | (uint64_t)(uintptr_t)q_out;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = q_strides[i], a.qos[i] = qo_strides[i];
    low |= (uint64_t)(a.qs[i] * 2) | (uint64_t)(a.qos[i] * 2);
    if (Hk) {
      a.ks[i] = k_strides[i], a.kos[i] = ko_strides[i];
      low |= (uint64_t)(a.ks[i] * 2) | (uint64_t)(a.kos[i] * 2);
    }
  }
  if (Hk) low |= (uint64_t)(uintptr_t)k | (uint64_t)(uintptr_t)k_out;
  int pw = 8;
  while (pw > 1 && ((low & (2 * pw - 1)) || (R / 2) % pw || (D - R) % (2 * pw))) pw /= 2;
  a.pos = positions, a.pos_sb = pos_stride, a.pos64 = pos_is_64 ? 1 : 0;
  a.inv_freq = inv_freq, a.factor = factor;
  a.S = (int)S, a.Hq = (int)Hq, a.Hk = (int)Hk, a.D = (int)D, a.R = (int)R;
  a.upt = (unsigned)(D / (2 * pw));
  const int64_t H = Hq + Hk;
  // threads of four heads where they still fill the card (2048 a CU), else of one
  const bool four = B * S * ((H + 3) / 4) * a.upt >= 2048 * 256;
  a.hgroups = (unsigned)(four ? (H + 3) / 4 : H);
  if (B > (int64_t)(0xffffff00u / ((uint64_t)S * a.hgroups * a.upt)))
    return set_error(TPP_E_UNSUPPORTED, "%s: too many rows", name);
  a.units = (unsigned)(B * S * a.hgroups * a.upt);
  const unsigned blocks = (a.units + 255) / 256;
  hipStream_t st = as_stream(stream);
  return TPP_DISPATCH_HALF(dtype, [&] {
    auto go = [&](auto w) {
      constexpr int PW = decltype(w)::value;
      const dim3 grid(blocks), block(256);
      if (four) {
        if (interleaved) rope_at_kernel<T, PW, true, 4><<<grid, block, 0, st>>>(a);
        else rope_at_kernel<T, PW, false, 4><<<grid, block, 0, st>>>(a);
      } else if (interleaved) {
        rope_at_kernel<T, PW, true, 1><<<grid, block, 0, st>>>(a);
      } else {
        rope_at_kernel<T, PW, false, 1><<<grid, block, 0, st>>>(a);
      }
    };
    if (pw == 8) go(std::integral_constant<int, 8>{});
    else if (pw == 4) go(std::integral_constant<int, 4>{});
    else if (pw == 2) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 1>{});
    return check_launch(name);
  });
}
