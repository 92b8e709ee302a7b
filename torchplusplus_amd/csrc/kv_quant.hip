// A KV cache of 8-bit codes: writing it and reading it back.
//
// A row (one head of one token, D elements) is D codes and one exponent byte
// E: x ~ code * 2^(E - 127). E is the least power of two for which every code
// is in range (max|x| <= M 2^(E - 127), M = 448 in e4m3 and 127 in int8), kept
// in 1 .. 254 so that 2^(E - 127) is a normal float; code = x / 2^(E - 127)
// rounded half to even. With powers of two the division is exact, so a code
// is the one correct rounding of its element (relative error at most 2^-4 in
// e4m3, absolute at most 2^(E - 128) in int8) and decoding is exact in
// bfloat16. A bfloat16 past the largest value below 2^128 that a row of codes holds
// (240 * 2^120 in e4m3, 127 * 2^121 in int8) is stored as that: the nearest code, 256 or
// 64 times more, would read back as infinity. A scale of max / M exactly would use int8's range better by up to
// one bit (half a bit on average), at four bytes a row and two more roundings.
// A row with an infinity or a NaN gets E = 255 and codes 0 and reads back as
// NaN throughout.
//
// Bound by HBM: append reads 2 bytes and writes 1 an element, read the other
// way round. 8 x 2048 tokens, 8 heads of 128, into e4m3: 24.5 us (4.1 TB/s, 26.1 with
// one row a thread); 8 x 2304 positions back: 19.5 us (5.8 TB/s, part of the codes from
// the caches, where a call before left them).
#include "tpp_common.hpp"

namespace tpp {

struct KvAppendArgs {
  const void *x[2];         // k, v [B, S, H, D]
  int64_t xs[2][3];         // {batch, token, head}
  void *codes[2];           // [B, H, Lmax, D]
  uint8_t *exps[2];         // [B, H, Lmax]
  int64_t cs[2], es[2];     // {batch, head}
  const int32_t *positions; // [B] or null: `start`
  const int32_t *counts;    // [B] or null: S
  int64_t start, rows, S;   // rows = B * S * H
  int H, Lmax;
};

template <int LPR> __device__ __forceinline__ unsigned group_umax(unsigned v) {
  auto dpp = [](unsigned x, auto c) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, decltype(c)::value, 0xf, 0xf, false);
  };
  v = max(v, dpp(v, std::integral_constant<int, kDppQuadXor1>{}));
  v = max(v, dpp(v, std::integral_constant<int, kDppQuadXor2>{}));
  v = max(v, dpp(v, std::integral_constant<int, kDppRowHalfMirror>{}));
  if constexpr (LPR >= 16) v = max(v, dpp(v, std::integral_constant<int, kDppRowMirror>{}));
  if constexpr (LPR >= 32) v = max(v, (unsigned)__shfl_xor((int)v, 16, kWave));
  return v;
}

// The largest value below 2^128 that a row of codes holds.
template <int CODE> constexpr float kCodedMax = CODE == TPP_CODE_E4M3 ? 0x1.ep127f : 0x1.fcp127f;

// The exponent byte for a row whose largest magnitude has the float bits `u`.
template <int CODE> __device__ __forceinline__ int row_exponent(unsigned u) {
  if (u >= 0x7f800000u) return 255; // an infinity or a NaN
  u = min(u, __builtin_bit_cast(unsigned, kCodedMax<CODE>));
  // M = 1.75 * 2^8 or 1.984375 * 2^6: one more where the mantissa is past M's
  const int e = CODE == TPP_CODE_E4M3 ? (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u)
                                      : (int)(u >> 23) - 6 + ((u & 0x7fffffu) > 0x7e0000u);
  return max(e, 1);
}

// D / 8 lanes a row, 8 elements (16 bytes in, 8 out) a lane, U rows a thread: their
// loads before the first use. Rows run over a head's tokens, so that a block writes
// one run of codes.
template <typename T, int CODE, int D, int U>
__global__ __launch_bounds__(256) void kv_append_kernel(KvAppendArgs p) {
  typedef typename VecT<T>::v8 V8;
  constexpr int LPR = D / 8, RPP = 256 / LPR; // rows of a pass
  const int c = threadIdx.x % LPR, w = blockIdx.y;
  const int64_t row0 = (int64_t)blockIdx.x * (RPP * U) + threadIdx.x / LPR;
  V8 t[U];
  bool put[U];
  int64_t pos[U], bb[U];
  int hh[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const unsigned row = (unsigned)(row0 + i * RPP < p.rows ? row0 + i * RPP : p.rows - 1); // (rows < 2^32)
    const unsigned bh = row / (unsigned)p.S;
    const int64_t s = row - bh * (unsigned)p.S, b = bh / (unsigned)p.H;
    const int h = (int)(bh - (unsigned)b * (unsigned)p.H);
    t[i] = ld_nt(reinterpret_cast<const V8 *>((const T *)p.x[w] + b * p.xs[w][0] + s * p.xs[w][1] + h * p.xs[w][2] + c * 8));
    pos[i] = (p.positions ? (int64_t)p.positions[b] : p.start) + s;
    put[i] = row0 + i * RPP < p.rows && pos[i] >= 0 && pos[i] < p.Lmax && !(p.counts && s >= p.counts[b]);
    bb[i] = b, hh[i] = h;
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    float x[8];
    unsigned u = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = to_f32(t[i][j]);
      u = max(u, __float_as_uint(x[j]) & 0x7fffffffu);
    }
    u = group_umax<LPR>(u);
    const int e = row_exponent<CODE>(u);
    if (__is_same(T, bf16) && u > __builtin_bit_cast(unsigned, kCodedMax<CODE>)) // (hardly ever)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __builtin_amdgcn_fmed3f(x[j], -kCodedMax<CODE>, kCodedMax<CODE>);
    // times 2^(127 - e): exact, or below half the least code
    const float inv = e == 255 ? 0.f : __uint_as_float((unsigned)(254 - e) << 23);
    u32x2 out = {0u, 0u};
    if (e != 255) {
      if constexpr (CODE == TPP_CODE_E4M3) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          int v = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j] * inv, x[4 * j + 1] * inv, 0, false);
          out[j] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j + 2] * inv, x[4 * j + 3] * inv, v, true);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          out[j / 4] |= ((unsigned)(int)__builtin_rintf(x[j] * inv) & 0xffu) << (8 * (j % 4));
      }
    }
    if (!put[i]) continue; // (whole rows of lanes)
    uint8_t *dst = (uint8_t *)p.codes[w] + bb[i] * p.cs[0] + hh[i] * p.cs[1] + pos[i] * D + c * 8;
    *reinterpret_cast<u32x2 *>(dst) = out;
    if (c == 0) p.exps[w][bb[i] * p.es[0] + hh[i] * p.es[1] + pos[i]] = (uint8_t)e;
  }
}

struct KvReadArgs {
  const void *codes[2];
  const uint8_t *exps[2];
  int64_t cs[2], es[2];
  void *out[2]; // [B, H, len, D] contiguous
  int64_t chunks; // B * H * len * D / 8
  int64_t len;
  int H;
};

template <typename T, int CODE, int D, int U>
__global__ __launch_bounds__(256) void kv_read_kernel(KvReadArgs p) {
  constexpr int LPR = D / 8;
  const int w = blockIdx.y;
  const int64_t id0 = (int64_t)blockIdx.x * (256 * U) + threadIdx.x;
  u32x2 t[U];
  int e[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int64_t id = id0 + i * 256 < p.chunks ? id0 + i * 256 : p.chunks - 1;
    const unsigned row = (unsigned)(id / LPR), bh = row / (unsigned)p.len, b0 = bh / (unsigned)p.H; // (rows < 2^32)
    const int64_t pos = row - bh * (unsigned)p.len, b = b0, h = bh - b0 * (unsigned)p.H;
    t[i] = ld_nt(reinterpret_cast<const u32x2 *>((const uint8_t *)p.codes[w] + b * p.cs[0] + h * p.cs[1] + pos * D +
                                                 (id % LPR) * 8));
    e[i] = p.exps[w][b * p.es[0] + h * p.es[1] + pos];
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    // 2^(e - 127); e = 255 is a NaN (bits of a NaN: exponent field 255, mantissa not 0)
    const float sc = __uint_as_float(e[i] == 255 ? 0x7fc00000u : (unsigned)e[i] << 23);
    float v[8];
    if constexpr (CODE == TPP_CODE_E4M3) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)t[i][j], false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)t[i][j], true);
        v[4 * j] = lo[0], v[4 * j + 1] = lo[1], v[4 * j + 2] = hi[0], v[4 * j + 3] = hi[1];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (float)(int8_t)(t[i][j / 4] >> (8 * (j % 4)));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] *= sc;
      // a code rounded up from the largest fp16 may stand for 65536
      if constexpr (__is_same(T, f16)) v[j] = v[j] != v[j] ? v[j] : fminf(fmaxf(v[j], -65504.f), 65504.f);
    }
    if (id0 + i * 256 < p.chunks) store8((T *)p.out[w] + (id0 + i * 256) * 8, v);
  }
}

static int check_codes(const char *name, const void *kc, const void *vc, const void *ke,
                       const void *ve, int64_t B, int64_t H, int64_t D, int64_t Lmax, int code,
                       int dtype) {
  if (!kc || !vc || !ke || !ve) return set_error(TPP_E_INVALID, "%s: null pointer", name);
  if (!half_type(dtype)) return set_error(TPP_E_UNSUPPORTED, "%s: unsupported dtype %d", name, dtype);
  if (code != TPP_CODE_E4M3 && code != TPP_CODE_INT8)
    return set_error(TPP_E_UNSUPPORTED, "%s: unsupported code type %d", name, code);
  if (D != 64 && D != 128 && D != 256)
    return set_error(TPP_E_UNSUPPORTED, "%s: head_dim %lld is not 64, 128 or 256", name, (long long)D);
  if (B < 0 || H < 1 || Lmax < 0 || Lmax > 0x7fffffffLL || H > 0x7fffffffLL)
    return set_error(TPP_E_INVALID, "%s: invalid shapes", name);
  if (((uintptr_t)kc | (uintptr_t)vc) & 7)
    return set_error(TPP_E_INVALID, "%s: codes must be 8-byte aligned", name);
  return TPP_OK;
}

} // namespace tpp

using namespace tpp;

extern "C" int tpp_kv_quant_append(const void *k, const void *v, const int64_t *k_strides,
                                   const int64_t *v_strides, void *k_codes, void *v_codes,
                                   void *k_exps, void *v_exps, const int64_t *code_strides,
                                   const int64_t *exp_strides, const int32_t *positions,
                                   int64_t start, const int32_t *counts, int64_t B, int64_t S,
                                   int64_t H, int64_t D, int64_t Lmax, int code, int dtype,
                                   void *stream) {
  const char *name = "tpp_kv_quant_append";
  if (int rc = check_codes(name, k_codes, v_codes, k_exps, v_exps, B, H, D, Lmax, code, dtype)) return rc;
  if (!k || !v || !k_strides || !v_strides || !code_strides || !exp_strides)
    return set_error(TPP_E_INVALID, "%s: null pointer", name);
  if (S < 0) return set_error(TPP_E_INVALID, "%s: invalid shapes", name);
  if (B == 0 || S == 0) return TPP_OK;
  KvAppendArgs a = {};
  uint64_t low = (uint64_t)(uintptr_t)k | (uint64_t)(uintptr_t)v;
  for (int i = 0; i < 3; ++i) {
    a.xs[0][i] = k_strides[i], a.xs[1][i] = v_strides[i];
    low |= (uint64_t)(k_strides[i] * 2) | (uint64_t)(v_strides[i] * 2);
  }
  if (low & 15) return set_error(TPP_E_INVALID, "%s: k and v rows must be 16-byte aligned", name);
  if ((code_strides[0] | code_strides[1]) & 7)
    return set_error(TPP_E_INVALID, "%s: code rows must be 8-byte aligned", name);
  a.x[0] = k, a.x[1] = v;
  a.codes[0] = k_codes, a.codes[1] = v_codes, a.exps[0] = (uint8_t *)k_exps, a.exps[1] = (uint8_t *)v_exps;
  for (int i = 0; i < 2; ++i) a.cs[i] = code_strides[i], a.es[i] = exp_strides[i];
  a.positions = positions, a.counts = counts, a.start = start, a.S = S, a.H = (int)H, a.Lmax = (int)Lmax;
  a.rows = B * S * H;
  // four rows a thread where that still fills the card (2048 threads a CU)
  const bool four = a.rows * (D / 8) * 2 >= 4LL * 2048 * 256;
  const int64_t per = 256 / (D / 8) * (four ? 4 : 1), blocks = (a.rows + per - 1) / per;
  if (S > 0x7fffffffLL || blocks > 0x7fffffffLL || a.rows > 0xffffffffLL) return set_error(TPP_E_UNSUPPORTED, "%s: too many rows", name);
  hipStream_t st = as_stream(stream);
  return TPP_DISPATCH_HALF(dtype, [&] {
    auto go = [&](auto cd, auto dd) {
      const dim3 grid((unsigned)blocks, 2);
      if (four) kv_append_kernel<T, decltype(cd)::value, decltype(dd)::value, 4><<<grid, dim3(256), 0, st>>>(a);
      else kv_append_kernel<T, decltype(cd)::value, decltype(dd)::value, 1><<<grid, dim3(256), 0, st>>>(a);
    };
    auto by_d = [&](auto cd) {
      if (D == 64) go(cd, std::integral_constant<int, 64>{});
      else if (D == 128) go(cd, std::integral_constant<int, 128>{});
      else go(cd, std::integral_constant<int, 256>{});
    };
    if (code == TPP_CODE_E4M3) by_d(std::integral_constant<int, TPP_CODE_E4M3>{});
    else by_d(std::integral_constant<int, TPP_CODE_INT8>{});
    return check_launch(name);
  });
}

extern "C" int tpp_kv_quant_read(const void *k_codes, const void *v_codes, const void *k_exps,
                                 const void *v_exps, const int64_t *code_strides,
                                 const int64_t *exp_strides, void *k_out, void *v_out, int64_t B,
                                 int64_t H, int64_t len, int64_t D, int64_t Lmax, int code, int dtype,
                                 void *stream) {
  const char *name = "tpp_kv_quant_read";
  if (int rc = check_codes(name, k_codes, v_codes, k_exps, v_exps, B, H, D, Lmax, code, dtype)) return rc;
  if (!k_out || !v_out || !code_strides || !exp_strides)
    return set_error(TPP_E_INVALID, "%s: null pointer", name);
  if (len < 0 || len > Lmax) return set_error(TPP_E_INVALID, "%s: length %lld of %lld", name, (long long)len, (long long)Lmax);
  if (!aligned16(k_out) || !aligned16(v_out) || ((code_strides[0] | code_strides[1]) & 7))
    return set_error(TPP_E_INVALID, "%s: outputs must be 16-byte, code rows 8-byte aligned", name);
  if (B == 0 || len == 0) return TPP_OK;
  KvReadArgs a = {};
  a.codes[0] = k_codes, a.codes[1] = v_codes, a.exps[0] = (const uint8_t *)k_exps, a.exps[1] = (const uint8_t *)v_exps;
  for (int i = 0; i < 2; ++i) a.cs[i] = code_strides[i], a.es[i] = exp_strides[i];
  a.out[0] = k_out, a.out[1] = v_out, a.len = len, a.H = (int)H;
  a.chunks = B * H * len * (D / 8);
  // four chunks of 8 a thread where that still fills the card
  const bool four = a.chunks * 2 >= 4LL * 2048 * 256;
  const int64_t per = four ? 1024 : 256, blocks = (a.chunks + per - 1) / per;
  if (blocks > 0x7fffffffLL || a.chunks / (D / 8) > 0xffffffffLL) return set_error(TPP_E_UNSUPPORTED, "%s: too many rows", name);
  hipStream_t st = as_stream(stream);
  return TPP_DISPATCH_HALF(dtype, [&] {
    auto go = [&](auto cd, auto dd) {
      const dim3 grid((unsigned)blocks, 2);
      if (four) kv_read_kernel<T, decltype(cd)::value, decltype(dd)::value, 4><<<grid, dim3(256), 0, st>>>(a);
      else kv_read_kernel<T, decltype(cd)::value, decltype(dd)::value, 1><<<grid, dim3(256), 0, st>>>(a);
    };
    auto by_d = [&](auto cd) {
      if (D == 64) go(cd, std::integral_constant<int, 64>{});
      else if (D == 128) go(cd, std::integral_constant<int, 128>{});
      else go(cd, std::integral_constant<int, 256>{});
    };
    if (code == TPP_CODE_E4M3) by_d(std::integral_constant<int, TPP_CODE_E4M3>{});
    else by_d(std::integral_constant<int, TPP_CODE_INT8>{});
    return check_launch(name);
  });
}
