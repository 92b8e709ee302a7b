// Attention of drafted tokens over a KV cache of 16-bit values or 8-bit codes.
//
//   o[b, t, h] = softmax_j(scale q[b, t, h] . K[b, j, h / G]) V[b, j, h / G]
// over the keys j < len_b of the sequence's context and those keys len_b + i
// that hold drafted token i where i is t or one of its ancestors (G = Hq / Hkv
// query heads share a KV head). `parents` gives each drafted token's parent:
// an earlier token, or -1 for the context's last; any other value marks
// padding, which sees nothing, as do its children. One token per sequence is
// decode over the cache. A row that sees nothing is 0; one that sees scores of -inf
// alone is NaN, as its softmax is.
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
__device__ __forceinline__ int tree_parent(const TreeArgs &p, int b) {
  const int lane = lane_id();
  return lane >= p.T ? -2 : p.parents ? p.parents[(int64_t)b * p.T + lane] : lane - 1;
}
__device__ __forceinline__ unsigned long long tree_bits(const TreeArgs &p, int up, int L) {
  const int lane = lane_id();
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
// head), keys one at a time with a wave reduction, so bound by latency, 1 us a key (one
// token over 4096 int8 keys of 256, 16 / 4 heads: 4.3 ms; 16-bit 8.3).
template <typename T, int KIND>
__global__ __launch_bounds__(64) void tree_generic_kernel(TreeArgs p, int D) {
  const int lane = lane_id(), t = blockIdx.x % p.T, h = blockIdx.x / p.T, b = blockIdx.y;
  const int hk = h / p.G;
  const int L = min(max(p.seqlens[b], 0), p.Lmax);
  const unsigned long long bits = tree_bits(p, tree_parent(p, b), L);
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

// ---------------------------------------------------------------------------
// Head sizes 64 and 128, 16-byte rows: on the matrix cores.
//
// The T G query rows of a KV head (row = token * G + head of the group) are the
// columns of S^T = K Q^T and of O^T = V^T P^T (16x16x32), NC groups of 16 a
// block; the four lanes with equal lane % 16 share a query row, so the softmax
// needs two exchanges. A block is 4 waves over one split of the sequence's keys;
// each wave streams its own tiles of KT keys (8 KB of K) by LDS-DMA into a
// private slot: no barrier in the loop, the next K tile is requested once this
// one's fragments are in registers, the next V tile after this one's. Waves are
// merged through LDS, splits by the pair's last block (tree_merge_here) or by
// tree_merge_kernel, a second launch. Bound by HBM up to 32 rows (32 sequences of 4096
// e4m3 keys, 16 / 8 heads of 128, one token: 48.8 us, 5.5 TB/s; of bfloat16 84.2 us, 6.4
// TB/s), by the products and the softmax past that (tree_rows_kernel).
//
// Key order: S^T gives lane quarter u the keys 16 st + 4 u + i (i = 0 .. 3) of
// tile st. The product with V takes them as its K index 8 u + j of step c: j < 4
// from st = 2 c, the others from st = 2 c + 1, so P never leaves its registers,
// and the transposing LDS reads of V fetch rows in that order.
//
// Codes stay codes up to the registers: a tile of codes has half the bytes and
// twice the keys. K fragments become T (exact: e4m3 and int8 values fit both
// types), V fragments bfloat16; the exponents are applied to the scores and to
// the probabilities. P keeps its fp32 bits: it is the sum of three values of V's
// type, whose products are summed in fp32. In bfloat16 those are 8 bits each, all of
// P down to 2^-100 of the largest (2^-118 is the least that counts). In fp16 they are
// 11 bits each at 2^15, 2^26 and 2^37 times P (1 at most), each folded into the next
// at its scale: 22 bits of a weight down to 2^-40 of the largest, 11 to 2^-51, and what
// is cut is below 2^-61, so that V up to 65504 over 2^20 keys loses less than half of
// fp16's least step. (Two parts at one scale lost every weight below 2^-39, and in
// bfloat16 the last 8 bits.) Over codes, whose powers of two P is multiplied by, all
// of its bits count where the product is above 2^-102.
// ---------------------------------------------------------------------------
// Keys of a tile: 8 KB of K, 32 or 64. The kernel of up to 32 rows takes 32 of coded
// caches too: of 16 rows three blocks a CU instead of two (32 sequences of 2098 e4m3
// keys, 16 / 8 heads, 28.9 -> 26.7 us; one of 700 int8 keys 8.8 -> 7.6 us), of 32 rows
// the three parts of P for half the keys, which stay in registers (8 trees of 16 over
// 1500-2288 e4m3 keys, 37.5 -> 20.0 us).
constexpr int tree_keys(int kind, int d) { return d * (kind ? 1 : 2) == 256 ? 32 : 64; }
template <int KIND, int D, int KEYS = tree_keys(KIND, D)> struct TreeTile {
  static constexpr int ROWB = D * (KIND ? 1 : 2); // bytes of a row
  static constexpr int KT = KEYS;                 // keys of a tile
  static constexpr int UPR = ROWB / 16, TILEB = KT * ROWB;
  // 16-byte unit u of row r is stored at u ^ ksw(r) in a K tile: 16 lanes that
  // read one unit of 16 rows hit all 64 banks
  static __device__ __forceinline__ int ksw(int r) { return (r / (16 / UPR)) & (UPR - 1); }
  // and at u ^ vsw(r) in a V tile: so do 32 lanes of a transposing read (8 rows
  // of two units, or rows r .. r + 7 and r + 16 .. r + 23 of one)
  static __device__ __forceinline__ int vsw(int r) {
    if constexpr (KIND == 0) return D == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3);
    else return D == 128 ? ((r >> 1) & 3) | ((r >> 2) & 4) : ((r >> 2) & 1) | ((r >> 3) & 2);
  }
};

template <typename T>
__device__ __forceinline__ f32x4 mfma16x16(typename VecT<T>::v8 a, typename VecT<T>::v8 b, f32x4 c) {
  if constexpr (__is_same(T, bf16)) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// eight codes as values of type T
template <typename T, int KIND>
__device__ __forceinline__ typename VecT<T>::v8 codes8(unsigned a, unsigned b) {
  typedef typename VecT<T>::v8 V8;
  if constexpr (KIND == TPP_CODE_E4M3) {
    auto two = [](unsigned c, auto hi) {
      if constexpr (__is_same(T, bf16))
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.f, decltype(hi)::value));
      else
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.f, decltype(hi)::value));
    };
    u32x4 r;
    r[0] = two(a, std::false_type{}), r[1] = two(a, std::true_type{});
    r[2] = two(b, std::false_type{}), r[3] = two(b, std::true_type{});
    return __builtin_bit_cast(V8, r);
  } else {
    V8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = from_f32<T>((float)(int8_t)((j < 4 ? a : b) >> (8 * (j % 4))));
    return v;
  }
}
// 2^(e - 127) for byte I of w (255: infinity, which codes of 0 make a NaN)
template <int I> __device__ __forceinline__ float exp_of(unsigned w) {
  return __uint_as_float(((w >> (8 * I)) & 0xffu) << 23);
}

// Eight probabilities, a's then b's, as the sum of three values of type PT each, all
// cut and not rounded: a part is what the ones ahead leave, in fp16 times 2^11 more than
// the one ahead of it (kPartUp), so that it does not fall among the subnormals.
constexpr float kPartUp = 2048.f;
template <typename PT>
__device__ __forceinline__ void three_parts(const f32x4 &a, const f32x4 &b, typename VecT<PT>::v8 (&r)[3]) {
  u32x4 w[3];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float x = j < 2 ? a[2 * j] : b[2 * j - 4], y = j < 2 ? a[2 * j + 1] : b[2 * j - 3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      if constexpr (__is_same(PT, bf16)) { // a bfloat16 is the upper half of a float
        w[i][j] = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
        if (i < 2) {
          x -= __uint_as_float(__float_as_uint(x) & 0xffff0000u);
          y -= __uint_as_float(__float_as_uint(y) & 0xffff0000u);
        }
      } else {
        const auto t = __builtin_amdgcn_cvt_pkrtz(x, y);
        w[i][j] = __builtin_bit_cast(unsigned, t);
        if (i < 2) x = (x - (float)t[0]) * kPartUp, y = (y - (float)t[1]) * kPartUp;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) r[i] = __builtin_bit_cast(typename VecT<PT>::v8, w[i]);
}

// the largest over lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float quarter_max(float v) {
  const unsigned u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const unsigned w = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
  const auto c = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  return fmaxf(__uint_as_float(c[0]), __uint_as_float(c[1]));
}

// One wave's part: NC groups of 16 query rows and what they have summed up.
template <typename T, int KIND, int D, int NC, int KEYS = tree_keys(KIND, D)> struct TreeWave {
  typedef typename VecT<T>::v8 V8;
  typedef std::conditional_t<KIND == 0, T, bf16> PT; // type of P and V operands
  typedef typename VecT<PT>::v8 P8;
  typedef TreeTile<KIND, D, KEYS> TT;
  static constexpr int KT = TT::KT, ROWB = TT::ROWB, UPR = TT::UPR, EB = KIND ? 1 : 2, EX = KIND ? 1 : 0;
  static constexpr int NST = KT / 16, NX = ROWB / 64, NCS = KT / 32, NT = D / 16;
  static constexpr bool kApart = !__is_same(PT, bf16);  // parts of P have scales of their own
  // The reference maximum moves when a tile's passes it by 2^8, for that rescales every
  // sum (2 trees of 33 over 26000 keys 89.1 -> 86.9 us). P is times 2^-8, so 1 at most
  // all the same: above 1 it took finite values from 2^120 on to infinity. Not in fp16,
  // whose parts have no such room: there P is times 2^15.
  static constexpr float kLazy = kApart ? 0.f : 8.f;
  static constexpr float kUp = kApart ? 15.f : -kLazy;

  V8 qf[NC][D / 32];
  unsigned long long see[NC];
  f32x4 o[NC][NT];
  float m[NC], l[NC];
  unsigned ko[NX], vo[NT], ea;
  int t[NC];

  // query rows row[i] (clamped by the caller), asked for
  __device__ __forceinline__ void ask(const TreeArgs &p, int b, int hk, unsigned g_inv, const int (&row)[NC]) {
    const int u4 = lane_id() >> 4;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      t[i] = div_inv((unsigned)row[i], g_inv);
      const T *qp = row_of((const T *)p.q, p.q_s, p, b, hk, row[i], t[i]);
#pragma unroll
      for (int k = 0; k < D / 32; ++k) // codes: a 16-byte read holds both steps of 64 elements
        qf[i][k] = *reinterpret_cast<const V8 *>(qp + (KIND ? (k / 2) * 64 + u4 * 16 + (k & 1) * 8 : k * 32 + u4 * 8));
    }
  }
  template <typename E>
  static __device__ __forceinline__ E *row_of(E *base, const int64_t (&st)[3], const TreeArgs &p, int b, int hk,
                                              int row, int tok) {
    return base + (int64_t)b * st[0] + (int64_t)tok * st[1] + (int64_t)(hk * p.G + row - tok * p.G) * st[2];
  }
  // The rows have come, the first tiles are in flight: no wait for the rows
  // inside the loop. LDS addresses of a tile's K and V and of its exponents.
  __device__ __forceinline__ void begin(unsigned long long bits, unsigned kbase, unsigned vbase, unsigned ebase) {
    const int lane = lane_id(), u4 = lane >> 4, l16 = lane & 15;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      see[i] = ((unsigned long long)(unsigned)__shfl((int)(bits >> 32), t[i], kWave) << 32) |
               (unsigned)__shfl((int)bits, t[i], kWave);
      m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) asm volatile("" ::"v"(qf[i][k]));
#pragma unroll
      for (int tt = 0; tt < NT; ++tt) o[i][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    ea = ebase + u4 * 16;
#pragma unroll
    for (int x = 0; x < NX; ++x) ko[x] = kbase + (unsigned)((l16 * UPR + ((4 * x + u4) ^ TT::ksw(l16))) * 16);
#pragma unroll
    for (int tt = 0; tt < NT; ++tt) {
      if constexpr (KIND == 0) { // lane a + 4 r at row 4 u + r, element 16 tt + 4 a
        const int kl = 4 * u4 + ((lane >> 2) & 3), a = lane & 3;
        vo[tt] = vbase + kl * ROWB + (((2 * tt) ^ TT::vsw(kl)) << 4) + 8 * a;
      } else { // lane a + 2 r at row 4 u + r (r < 4) or 16 + 4 u + r - 4, byte 16 tt + 8 a
        const int rr = (lane >> 1) & 7, kl = 16 * (rr >> 2) + 4 * u4 + (rr & 3);
        vo[tt] = vbase + kl * ROWB + ((tt ^ TT::vsw(kl)) << 4) + 8 * (lane & 1);
      }
    }
  }

  // One tile, keys kb .. kb + KT - 1, `off` bytes on in the ring (its exponents
  // eoff). after_k / after_v: its K / V fragments are in registers; wait_v: until
  // its V has landed.
  template <typename AK, typename WV, typename AV>
  __device__ __forceinline__ void step(const TreeArgs &p, int kb, int L, unsigned off, unsigned eoff, AK after_k,
                                       WV wait_v, AV after_v) {
    const int u4 = lane_id() >> 4;
    const bool edge = kb + KT > L;
    const float c2 = p.scale_log2;
    f32x4 s[NC][NST];
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int st = 0; st < NST; ++st) s[i][st] = f32x4{0.f, 0.f, 0.f, 0.f};
    u32x4 kr[NX][NST], ex[2];
    static_for<NX>([&](auto xx) {
      constexpr int x = decltype(xx)::value;
      static_for<NST>([&](auto tt) {
        constexpr int st = decltype(tt)::value;
        kr[x][st] = lds_read_b128<st * 16 * ROWB, u32x4>(ko[x] + off);
      });
    });
    if constexpr (KIND != 0) ex[0] = lds_read_b128<0, u32x4>(ea + eoff), ex[1] = lds_read_b128<64, u32x4>(ea + eoff);
    // The products of one wave go ahead of the other's softmax on the SIMD: the matrix
    // cores stay busy under it (2 trees of 33 over 26000 e4m3 keys, 32 / 4 heads: 80.1
    // -> 76.2 us; the other way round 80.7).
    __builtin_amdgcn_s_setprio(1);
    static_for<NX>([&](auto xx) {
      constexpr int x = decltype(xx)::value;
      lds_wait_tied<(NX - 1 - x) * NST + 2 * EX>(kr[x]);
      if constexpr (x == NX - 1) { // every K fragment is in registers
        if constexpr (KIND != 0) lds_wait_tied<0>(ex);
        asm volatile("" ::: "memory");
        after_k();
      }
      __builtin_amdgcn_sched_barrier(0);
      // (products into one accumulator are kept apart: back to back each would
      // wait for the one ahead)
      if constexpr (KIND == 0) {
#pragma unroll
        for (int st = 0; st < NST; ++st)
#pragma unroll
          for (int i = 0; i < NC; ++i)
            s[i][st] = mfma16x16<T>(__builtin_bit_cast(V8, kr[x][st]), qf[i][x], s[i][st]);
      } else {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int st = 0; st < NST; ++st) {
            const V8 f = codes8<T, KIND>(kr[x][st][2 * u], kr[x][st][2 * u + 1]);
#pragma unroll
            for (int i = 0; i < NC; ++i) s[i][st] = mfma16x16<T>(f, qf[i][2 * x + u], s[i][st]);
          }
      }
      __builtin_amdgcn_sched_barrier(0);
    });

    __builtin_amdgcn_s_setprio(0);
    P8 pt[NC][NCS][3];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      if constexpr (KIND != 0)
        static_for<4 * NST>([&](auto rr) {
          constexpr int r = decltype(rr)::value;
          s[i][r / 4][r % 4] *= exp_of<r % 4>(ex[0][r / 4]);
        });
      unsigned keep[NCS]; // bit 16 (st % 2) + e: score e of tile st
      if (edge) {
        const unsigned ninf = __float_as_uint(-INFINITY);
#pragma unroll
        for (int c = 0; c < NCS; ++c) {
          const int rel = kb + 32 * c - L;
          const unsigned k32 = rel >= 64 ? 0u
                               : rel >= 0 ? (unsigned)(see[i] >> rel)
                               : rel > -32 ? ((unsigned)see[i] << -rel) | ((1u << -rel) - 1u)
                                           : ~0u;
          keep[c] = k32 >> (4 * u4);
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const unsigned bm = (unsigned)__builtin_amdgcn_sbfe((int)keep[c], (r >> 2) * 16 + (r & 3), 1);
            float &x = reinterpret_cast<float *>(&s[i][2 * c + (r >> 2)])[r & 3];
            x = __uint_as_float((__float_as_uint(x) & bm) | (ninf & ~bm));
          }
        }
      }
      float mt = -INFINITY;
#pragma unroll
      for (int st = 0; st < NST; ++st)
        mt = fmaxf(mt, fmaxf(fmaxf(s[i][st][0], s[i][st][1]), fmaxf(s[i][st][2], s[i][st][3])));
      mt = quarter_max(mt);
      const bool move = (mt - m[i]) * c2 > kLazy;
      const float m_new = move ? mt : m[i];
      const float mc = m_new == -INFINITY ? 0.f : m_new * c2;
      const float alpha = move ? __builtin_amdgcn_exp2f(m[i] * c2 - mc) : 1.f;
      float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < NST; ++st)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = __builtin_amdgcn_exp2f(fmaf(s[i][st][r], c2, kUp - mc));
          s[i][st][r] = e;
          ps[r] += e;
        }
      l[i] = l[i] * alpha + ((ps[0] + ps[1]) + (ps[2] + ps[3]));
      m[i] = m_new;
      if (__any(move)) {
#pragma unroll
        for (int tt = 0; tt < NT; ++tt)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[i][tt][r] *= alpha;
      }
      if constexpr (KIND != 0) {
        static_for<4 * NST>([&](auto rr) {
          constexpr int r = decltype(rr)::value;
          s[i][r / 4][r % 4] *= exp_of<r % 4>(ex[1][r / 4]);
        });
        if (edge) { // a masked row of NaN: 0 times infinity above
#pragma unroll
          for (int c = 0; c < NCS; ++c)
#pragma unroll
            for (int r = 0; r < 8; ++r) {
              float &x = reinterpret_cast<float *>(&s[i][2 * c + (r >> 2)])[r & 3];
              x = __uint_as_float(__float_as_uint(x) &
                                  (unsigned)__builtin_amdgcn_sbfe((int)keep[c], (r >> 2) * 16 + (r & 3), 1));
            }
        }
      }
#pragma unroll
      for (int c = 0; c < NCS; ++c) three_parts<PT>(s[i][2 * c], s[i][2 * c + 1], pt[i][c]);
    }

    wait_v();
    __builtin_amdgcn_s_setprio(1);
    // DT d tiles of a step at a time
    constexpr int DT = KIND == 0 && NC == 2 ? 2 : 4, R = KIND ? DT : 2 * DT, NG = NCS * NT / DT;
    // fp16 parts have scales of their own: t to the scale of the part ahead, plus y
    auto fold = [](auto &t, auto y) {
#pragma unroll
      for (int j = 0; j < (NC == 1 ? 4 : 2); ++j)
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const f32x4 a = y(j, i);
#pragma unroll
          for (int e = 0; e < 4; ++e) t[j][i][e] = fmaf(t[j][i][e], 1.f / kPartUp, a[e]);
        }
    };
    typedef std::conditional_t<KIND == 0, s16x4, u32x2> VR;
    VR vr[2][R];
    auto vfrag = [&](auto gg) {
      constexpr int g = decltype(gg)::value, c = g / (NT / DT), t0 = DT * (g % (NT / DT));
#pragma unroll
      for (int j = 0; j < DT; ++j) {
        if constexpr (KIND == 0) {
          vr[g % 2][2 * j] = lds_read_tr16<c * 32 * ROWB>(vo[t0 + j] + off);
          vr[g % 2][2 * j + 1] = lds_read_tr16<c * 32 * ROWB + 16 * ROWB>(vo[t0 + j] + off);
        } else {
          vr[g % 2][j] = lds_read_tr8<c * 32 * ROWB>(vo[t0 + j] + off);
        }
      }
    };
    vfrag(std::integral_constant<int, 0>{});
    static_for<NG>([&](auto gg) {
      constexpr int g = decltype(gg)::value, c = g / (NT / DT), t0 = DT * (g % (NT / DT));
      if constexpr (g + 1 < NG) vfrag(std::integral_constant<int, g + 1>{});
      lds_wait_tied<(g + 1 < NG ? R : 0)>(vr[g % 2]);
      if constexpr (g + 1 == NG) {
        asm volatile("" ::: "memory");
        after_v();
      }
      __builtin_amdgcn_sched_barrier(0);
      // the parts of P, the least first
      constexpr int JG = NC == 1 ? 4 : 2;
#pragma unroll
      for (int j0 = 0; j0 < DT; j0 += JG) {
        P8 f[JG];
        f32x4 t[JG][NC];
#pragma unroll
        for (int j = 0; j < JG; ++j) {
          if constexpr (KIND == 0) {
            typedef short s16x8 __attribute__((ext_vector_type(8)));
            const s16x8 r12 = __builtin_shufflevector(vr[g % 2][2 * (j0 + j)], vr[g % 2][2 * (j0 + j) + 1], 0, 1, 2, 3, 4, 5, 6, 7);
            f[j] = __builtin_bit_cast(P8, r12);
          } else {
            f[j] = codes8<PT, KIND>(vr[g % 2][j0 + j][0], vr[g % 2][j0 + j][1]);
          }
#pragma unroll
          for (int i = 0; i < NC; ++i)
            t[j][i] = mfma16x16<PT>(f[j], pt[i][c][2], kApart ? f32x4{0.f, 0.f, 0.f, 0.f} : o[i][t0 + j0 + j]);
        }
        if constexpr (kApart) fold(t, [](int, int) { return f32x4{0.f, 0.f, 0.f, 0.f}; });
#pragma unroll
        for (int j = 0; j < JG; ++j)
#pragma unroll
          for (int i = 0; i < NC; ++i) t[j][i] = mfma16x16<PT>(f[j], pt[i][c][1], t[j][i]);
        if constexpr (kApart) fold(t, [&](int j, int i) { return o[i][t0 + j0 + j]; });
#pragma unroll
        for (int j = 0; j < JG; ++j)
#pragma unroll
          for (int i = 0; i < NC; ++i) o[i][t0 + j0 + j] = mfma16x16<PT>(f[j], pt[i][c][0], t[j][i]);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    __builtin_amdgcn_s_setprio(0);
  }

  // l over the four lanes of a row. A row that sees nothing gets a weight of 1 on
  // nothing: 0 after the merges, where a row of scores of -inf, with no weight, is 0 / 0.
  // True where a sum is not finite.
  __device__ __forceinline__ bool end(const TreeArgs &p) {
    f32x4 zero = {0.f, 0.f, 0.f, 0.f}; // or NaN (64 comparisons took 0.8 us here)
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      l[i] += __shfl_xor(l[i], 16, kWave);
      l[i] += __shfl_xor(l[i], 32, kWave);
      if (!see[i]) l[i] = 1.f, m[i] = 0.f;
#pragma unroll
      for (int tt = 0; tt < NT; ++tt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!see[i]) o[i][tt][e] = 0.f;
          zero[e] = fmaf(o[i][tt][e], 0.f, zero[e]);
        }
    }
    const float z = (zero[0] + zero[1]) + (zero[2] + zero[3]);
    return z != z;
  }
  __device__ __forceinline__ float top(const TreeArgs &p, int i) const {
    return m[i] == -INFINITY ? -INFINITY : m[i] * p.scale_log2;
  }

  // A row behind the context that is not finite, times a weight of 0, is a NaN in
  // the products of those that do not see it; so is an infinity among 16-bit values
  // times a part of P that is 0. A wave that had such a tile and has a sum that is not
  // finite sums again, key by key over what each row sees: its n tiles from key
  // `first`, `stride` apart, up to k_end (a row with a NaN among its scores is NaN
  // without). put(i, q, d, x): the sum of element d of row q of group i.
  template <typename PUT>
  __device__ __forceinline__ void again(const TreeArgs &p, int b, int hk, const char *ks, const char *vs, int64_t eb,
                                        int first, int stride, int n, int k_end, int L, unsigned g_inv,
                                        const int (&row0)[NC], int rows, PUT put) const {
    const int lane = lane_id();
#pragma unroll
    for (int i = 0; i < NC; ++i)
      for (int q = 0; q < 16 && row0[i] + q < rows; ++q) {
        const unsigned long long sq = ((unsigned long long)(unsigned)__shfl((int)(see[i] >> 32), q, kWave) << 32) |
                                      (unsigned)__shfl((int)see[i], q, kWave);
        const float mq = __shfl(m[i], q, kWave), mc = mq == -INFINITY ? 0.f : mq * p.scale_log2;
        const float lq = __shfl(l[i], q, kWave);
        const T *qp = row_of((const T *)p.q, p.q_s, p, b, hk, row0[i] + q, div_inv((unsigned)(row0[i] + q), g_inv));
        float acc[D / 64];
#pragma unroll
        for (int c = 0; c < D / 64; ++c) acc[c] = lq == lq ? 0.f : lq;
        for (int it = 0; it < n && sq && lq == lq; ++it)
          for (int j = first + it * stride; j < min(first + it * stride + KT, k_end); ++j) {
            if (j >= L && !((sq >> (j - L)) & 1)) continue;
            const char *kr = ks + (int64_t)j * p.k_s[2] * EB, *vr = vs + (int64_t)j * p.v_s[2] * EB;
            const float fk = KIND ? exp_scale(p.ke, eb + j) : 1.f, fv = KIND ? exp_scale(p.ve, eb + j) : 1.f;
            float sd = 0.f;
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
              sd += to_f32(qp[c * 64 + lane]) * cache_value<T, KIND>(kr, c * 64 + lane, fk);
            const float e = __builtin_amdgcn_exp2f(fmaf(wave_sum(sd), p.scale_log2, kUp - mc));
#pragma unroll
            for (int c = 0; c < D / 64; ++c) acc[c] += e * cache_value<T, KIND>(vr, c * 64 + lane, fv);
          }
#pragma unroll
        for (int c = 0; c < D / 64; ++c) put(i, q, c * 64 + lane, acc[c]);
      }
  }
};

// The caller's block: its pair, and the keys of its split in whole batches of
// `stride` keys (none: c0 >= end).
struct TreeBlock {
  int pair, b, hk, qt, split, L, end, live;
  int64_t c0, c1;
};
template <int STRIDE>
__device__ __forceinline__ void tree_split(const TreeArgs &p, int nsplit, unsigned nsplit_inv, TreeBlock &k) {
  k.L = min(max(p.seqlens[k.b], 0), p.Lmax), k.end = min(k.L + p.T, p.Lmax);
  const int nbatch = (int)((unsigned)(k.end + STRIDE - 1) / (unsigned)STRIDE);
  const int per = div_inv((unsigned)(nbatch + nsplit - 1), nsplit_inv);
  k.live = (int)((unsigned)(nbatch + per - 1) / (unsigned)per);
  k.c0 = (int64_t)k.split * per * STRIDE;
  k.c1 = k.c0 + (int64_t)per * STRIDE < k.end ? k.c0 + (int64_t)per * STRIDE : k.end;
}
__device__ __forceinline__ TreeBlock tree_block(const TreeArgs &p, unsigned hkv_inv, int by_xcd) {
  TreeBlock k; // blocks of a pair on one XCD where pairs divide by them
  k.pair = by_xcd ? blockIdx.z * 8 + (blockIdx.x & 7) : blockIdx.z;
  k.qt = by_xcd ? blockIdx.x >> 3 : blockIdx.x, k.split = blockIdx.y;
  k.b = div_inv(k.pair, hkv_inv), k.hk = k.pair - k.b * p.Hkv;
  return k;
}

// A wave's LDS-DMA of tile units j0 .. j0 + N - 1 (1 KB each) of K or V. Byte
// offsets of this lane's units from the tile's first row: a tile whose keys all
// exist is one uniform address and these. Else keys past the last read its row
// (masked).
template <int KIND, int D, int N, int POL, int KEYS = tree_keys(KIND, D)> struct TreeDma {
  typedef TreeTile<KIND, D, KEYS> TT;
  static constexpr int EB = KIND ? 1 : 2, KPI = 64 / TT::UPR;
  unsigned off[N];
  int j0;
  bool kt;
  __device__ __forceinline__ int unit(int j) const {
    const int key = (j0 + j) * KPI + lane_id() / TT::UPR;
    return (lane_id() % TT::UPR) ^ (kt ? TT::ksw(key) : TT::vsw(key));
  }
  __device__ __forceinline__ void begin(bool k, int first_unit, int64_t stride) {
    kt = k, j0 = first_unit;
#pragma unroll
    for (int j = 0; j < N; ++j)
      off[j] = (unsigned)(((j0 + j) * KPI + lane_id() / TT::UPR) * (int)stride * EB + (unit(j) << 4));
  }
  __device__ __forceinline__ void issue(const char *rows, int64_t stride, int base, int end, char *dst) const {
    const char *src = rows + (int64_t)base * stride * EB;
    if (base + TT::KT <= end) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        __builtin_amdgcn_global_load_lds((const void *)(src + off[j]),
                                         (__attribute__((address_space(3))) void *)(dst + (j0 + j) * 1024), 16, 0, POL);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int key = (j0 + j) * KPI + lane_id() / TT::UPR;
        __builtin_amdgcn_global_load_lds(
            (const void *)(src + (int64_t)min(key, end - 1 - base) * stride * EB + (unit(j) << 4)),
            (__attribute__((address_space(3))) void *)(dst + (j0 + j) * 1024), 16, 0, POL);
      }
    }
  }
};
// The exponents of a tile as the lanes read them: quarter u's four dwords (keys
// 16 st + 4 u .. + 3 in dword st) of K at 16 u, of V 64 bytes on (lanes 32 - 63
// repeat 0 - 31).
__device__ __forceinline__ void issue_exps(const TreeArgs &p, int64_t eb, int base, unsigned *dst) {
  const int lane = lane_id(), at = 16 * (lane & 3) + 4 * ((lane >> 2) & 3);
  __builtin_amdgcn_global_load_lds((const void *)((lane & 16 ? p.ve : p.ke) + eb + min(base + at, p.Lmax - 4)),
                                   (__attribute__((address_space(3))) void *)dst, 4, 0, 0);
}
template <typename P> __device__ __forceinline__ unsigned lds_addr(P *x) {
  return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) char *)x;
}

// Four floats to and from memory past the caches, for another block of the launch
// that may run on another XCD.
__device__ __forceinline__ void store_through(float *p, const f32x4 &x) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32x2 w = {__float_as_uint(x[2 * i]), __float_as_uint(x[2 * i + 1])};
    __hip_atomic_store((unsigned long long *)p + i, __builtin_bit_cast(unsigned long long, w), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
  }
}
__device__ __forceinline__ f32x4 load_through(const float *p) {
  f32x4 x;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32x2 w = __builtin_bit_cast(
        u32x2, __hip_atomic_load((const unsigned long long *)p + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    x[2 * i] = __uint_as_float(w[0]), x[2 * i + 1] = __uint_as_float(w[1]);
  }
  return x;
}

// Merging a row's splits, in one order wherever it is done: four parts, part g the
// splits g, g + 4, .. (four at a time), then the parts.
constexpr int kMergeParts = 4, kMergeAhead = 4;
template <int NP> struct TreeMerge { // parts g0, g0 + step, .. of a row, chunk c of four values
  float m[NP], l[NP];
  f32x4 o[NP];
  float ma[NP][kMergeAhead], la[NP][kMergeAhead];
  f32x4 oa[NP][kMergeAhead];
  // the splits s0 .. s0 + 15, those past `last` read it (and are not used); HERE:
  // maxima and weights past the L1
  template <int D, bool HERE>
  __device__ __forceinline__ void load(const float *ws_o, const float *ws_ml, int64_t slot, int c, int s0, int g0,
                                       int step, int last) {
#pragma unroll
    for (int n = 0; n < NP; ++n)
#pragma unroll
      for (int j = 0; j < kMergeAhead; ++j) {
        const int64_t at = slot + min(s0 + j * kMergeParts + g0 + n * step, last);
        if constexpr (HERE) {
          ma[n][j] = __hip_atomic_load(&ws_ml[at * 2], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          la[n][j] = __hip_atomic_load(&ws_ml[at * 2 + 1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        } else {
          ma[n][j] = ws_ml[at * 2], la[n][j] = ws_ml[at * 2 + 1];
        }
        if constexpr (HERE) oa[n][j] = load_through(ws_o + at * D + c * 4);
        else oa[n][j] = *reinterpret_cast<const f32x4 *>(ws_o + at * D + c * 4);
      }
  }
  __device__ __forceinline__ void begin() {
#pragma unroll
    for (int n = 0; n < NP; ++n) m[n] = -INFINITY, l[n] = 0.f, o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ void add(int s0, int g0, int step, int live) {
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      float mn = m[n];
#pragma unroll
      for (int j = 0; j < kMergeAhead; ++j)
        if (s0 + j * kMergeParts + g0 + n * step < live) mn = fmaxf(mn, ma[n][j]);
      const float mu = mn == -INFINITY ? 0.f : mn, a = __builtin_amdgcn_exp2f(m[n] - mu);
      l[n] *= a;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] *= a;
#pragma unroll
      for (int j = 0; j < kMergeAhead; ++j) {
        if (s0 + j * kMergeParts + g0 + n * step >= live) break; // (such a slot may hold anything)
        const float cf = __builtin_amdgcn_exp2f(ma[n][j] - mu);
        l[n] += la[n][j] * cf;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] += oa[n][j][e] * cf;
      }
      m[n] = mn;
    }
  }
};
// The parts of a row, from LDS (pitch f32x4 values of o, two of m and l): chunk c of
// the output.
template <typename T>
__device__ __forceinline__ typename VecT<T>::v4 tree_merge_parts(const f32x4 *o, int pitch, const float *ml) {
  float mx = -INFINITY, ls = 0.f;
#pragma unroll
  for (int g = 0; g < kMergeParts; ++g) mx = fmaxf(mx, ml[g * 2]);
  const float mu = mx == -INFINITY ? 0.f : mx;
  f32x4 os = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int g = 0; g < kMergeParts; ++g) {
    const float cf = __builtin_amdgcn_exp2f(ml[g * 2] - mu);
    ls += ml[g * 2 + 1] * cf;
    const f32x4 x = o[g * pitch];
#pragma unroll
    for (int e = 0; e < 4; ++e) os[e] += x[e] * cf;
  }
  typename VecT<T>::v4 ov;
  const float inv = 1.f / ls;
#pragma unroll
  for (int e = 0; e < 4; ++e) ov[e] = from_f32<T>(os[e] * inv);
  return ov;
}

// LDS bytes of the merge by a block: four parts of 256 / (D / 4) rows, with their
// maxima and weights.
template <int D> constexpr int tree_merge_lds = kMergeParts * (256 * 16 + 256 / (D / 4) * 8);

// The splits of up to 16 rows, by the pair's last block to finish: one launch instead
// of two, 7.8 -> 5.5 us where the sequences are so short that they need no merge. The
// block counts itself in on an arrival word; what it has summed went past the caches
// before, and comes so, since the blocks may run on any XCD. Captured calls take the
// second launch, as do more rows: 32 of 8 sequences took 32.0 us so for 21.4.
template <typename T, int D>
__device__ __forceinline__ void tree_merge_here(const TreeArgs &p, const TreeBlock &k, int rows, int nsplit,
                                                const float *__restrict__ ws_o, const float *__restrict__ ws_ml,
                                                unsigned g_inv, unsigned *__restrict__ arrived, char *lds) {
  constexpr int C4 = D / 4, NG = 256 / C4;
  __shared__ int s_last;
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0F70); // vmcnt(0): this wave's sums are in the L2
  __syncthreads();
  if (threadIdx.x == 0) {
    const unsigned old = __hip_atomic_fetch_add(arrived + k.pair, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = (int)old == k.live - 1;
    if (s_last) __hip_atomic_store(arrived + k.pair, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!s_last) return;
  // NG groups of lanes over the rows, up to four (one a part) a row
  const int grp = threadIdx.x / C4, c = threadIdx.x % C4;
  f32x4 *const s_o = reinterpret_cast<f32x4 *>(lds);                           // [row][part][chunk]
  float *const s_ml = reinterpret_cast<float *>(lds + NG * kMergeParts * C4 * 16); // [row][part][2]
  auto run = [&](auto npc) {
    constexpr int NP = decltype(npc)::value, STEP = kMergeParts / NP, RPB = NG / STEP;
    for (int base = 0; base < rows; base += RPB) {
      const int q = grp / STEP, g0 = grp % STEP, r = min(base + q, rows - 1);
      const int64_t slot = ((int64_t)k.pair * rows + r) * nsplit;
      TreeMerge<NP> mg;
      mg.begin();
      for (int s0 = 0; s0 < k.live; s0 += kMergeParts * kMergeAhead) {
        mg.template load<D, true>(ws_o, ws_ml, slot, c, s0, g0, STEP, k.live - 1);
        mg.add(s0, g0, STEP, k.live);
      }
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        const int at = q * kMergeParts + g0 + n * STEP;
        s_o[at * C4 + c] = mg.o[n];
        if (c == 0) s_ml[at * 2] = mg.m[n], s_ml[at * 2 + 1] = mg.l[n];
      }
      __syncthreads();
      if (g0 == 0 && base + q < rows) {
        const int t = div_inv((unsigned)r, g_inv), g = r - t * p.G;
        T *op = (T *)p.o + (int64_t)k.b * p.o_s[0] + (int64_t)t * p.o_s[1] + (int64_t)(k.hk * p.G + g) * p.o_s[2];
        *reinterpret_cast<typename VecT<T>::v4 *>(op + c * 4) =
            tree_merge_parts<T>(s_o + q * kMergeParts * C4 + c, C4, s_ml + q * kMergeParts * 2);
      }
      __syncthreads();
    }
  };
  if (rows * kMergeParts <= NG) run(std::integral_constant<int, 1>{});
  else if (rows * 2 <= NG) run(std::integral_constant<int, 2>{});
  else run(std::integral_constant<int, 4>{});
}

// Up to 32 rows a block: the four waves share the rows and split the keys.
template <typename T, int KIND, int D, int NC>
__global__ __launch_bounds__(256, KIND && NC == 1 ? 3 : 2) void tree_tile_kernel(TreeArgs p, float *__restrict__ ws_o,
                                                           float *__restrict__ ws_ml, int nsplit,
                                                           unsigned nsplit_inv, unsigned hkv_inv,
                                                           unsigned g_inv, int by_xcd,
                                                           unsigned *__restrict__ arrived) {
  constexpr int KEYS = KIND ? 32 : tree_keys(KIND, D);
  typedef TreeTile<KIND, D, KEYS> TT;
  typedef TreeWave<T, KIND, D, NC, KEYS> W;
  constexpr int KT = TT::KT, NW = 4, STRIDE = NW * KT, NDMA = TT::TILEB / 1024, C4 = D / 4, ROWS = 16 * NC;
  // a wave's tiles, later its rows
  constexpr int SLOT = 2 * TT::TILEB > ROWS * D * 4 ? 2 * TT::TILEB : ROWS * D * 4;
  constexpr int kRing = NW * SLOT, kMerge = NC == 1 ? tree_merge_lds<D> : 0;
  __shared__ __attribute__((aligned(16))) char smem[kRing > kMerge ? kRing : kMerge];
  __shared__ __attribute__((aligned(16))) unsigned s_e[NW][64];
  __shared__ float s_m[NW][ROWS], s_l[NW][ROWS];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int u4 = lane >> 4, l16 = lane & 15;
  TreeBlock k = tree_block(p, hkv_inv, by_xcd);
  // what no length has a part in is asked for first: loads return in order, so a
  // load behind the first tiles would wait for them
  const int up = tree_parent(p, k.b);
  const int rows = p.T * p.G;
  W wv;
  int row0[NC], row[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) row0[i] = k.qt * ROWS + i * 16, row[i] = min(row0[i] + l16, rows - 1);
  wv.ask(p, k.b, k.hk, g_inv, row);
  tree_split<STRIDE>(p, nsplit, nsplit_inv, k);
  if (k.c0 >= k.end) return;
  const int first = (int)k.c0 + w * KT, k_end = (int)k.c1;
  const int n = first < k_end ? (k_end - first + STRIDE - 1) / STRIDE : 0; // this wave's tiles

  const char *ks = (const char *)p.k + ((int64_t)k.b * p.k_s[0] + (int64_t)k.hk * p.k_s[1]) * W::EB;
  const char *vs = (const char *)p.v + ((int64_t)k.b * p.v_s[0] + (int64_t)k.hk * p.v_s[1]) * W::EB;
  const int64_t eb = (int64_t)k.b * p.e_s[0] + (int64_t)k.hk * p.e_s[1];
  char *const ring = smem + w * SLOT;
  TreeDma<KIND, D, NDMA, kCpolNT, KEYS> dk, dv;
  dk.begin(true, 0, p.k_s[2]);
  dv.begin(false, 0, p.v_s[2]);
  auto issue_k = [&](int base) {
    dk.issue(ks, p.k_s[2], base, k.end, ring);
    if constexpr (KIND != 0) issue_exps(p, eb, base, s_e[w]);
  };
  auto issue_v = [&](int base) { dv.issue(vs, p.v_s[2], base, k.end, ring + TT::TILEB); };
  if (n > 0) {
    issue_k(first);
    issue_v(first);
  }
  wv.begin(tree_bits(p, up, k.L), lds_addr(ring), lds_addr(ring) + TT::TILEB, lds_addr(s_e[w]));
  for (int it = 0; it < n; ++it) {
    const int kb = first + it * STRIDE;
    const bool more = it + 1 < n;
    vm_wait<NDMA>(); // this tile's K (and exponents) landed, its V may be in flight
    wv.step(p, kb, k.L, 0, 0,
            [&] { if (more) issue_k(kb + STRIDE); },
            [&] { // the next K may be in flight
              if (more) vm_wait<NDMA + W::EX>();
              else vm_wait<0>();
            },
            [&] { if (more) issue_v(kb + STRIDE); });
  }

  // The wave's rows, then the block's: chunk c (4 values) of row r at c ^ r
  f32x4 *const part = reinterpret_cast<f32x4 *>(ring);
  const bool odd = wv.end(p);
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int r = i * 16 + l16;
#pragma unroll
    for (int tt = 0; tt < W::NT; ++tt) part[r * C4 + ((tt * 4 + u4) ^ (r & (C4 - 1)))] = wv.o[i][tt];
    if (u4 == 0) s_m[w][r] = wv.top(p, i), s_l[w][r] = wv.l[i];
  }
  if (n > 0 && (KIND == 0 || first + (n - 1) * STRIDE + KT > k.L) && __any(odd))
    wv.again(p, k.b, k.hk, ks, vs, eb, first, STRIDE, n, k_end, k.L, g_inv, row0, rows, [&](int i, int q, int d, float x) {
      const int r = i * 16 + q;
      reinterpret_cast<float *>(part + r * C4 + ((d / 4) ^ (r & (C4 - 1))))[d % 4] = x;
    });
  __syncthreads();
  for (int idx = tid; idx < ROWS * C4; idx += 64 * NW) {
    const int q = idx / C4, c = idx % C4, r = row0[0] + q;
    if (r >= rows) break;
    float mx = -INFINITY;
#pragma unroll
    for (int ww = 0; ww < NW; ++ww) mx = fmaxf(mx, s_m[ww][q]);
    const float mu = mx == -INFINITY ? 0.f : mx;
    float ls = 0.f;
    f32x4 os = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ww = 0; ww < NW; ++ww) {
      const float cf = __builtin_amdgcn_exp2f(s_m[ww][q] - mu);
      ls += s_l[ww][q] * cf;
      const f32x4 pr = reinterpret_cast<const f32x4 *>(smem + ww * SLOT)[q * C4 + (c ^ (q & (C4 - 1)))];
#pragma unroll
      for (int e = 0; e < 4; ++e) os[e] += pr[e] * cf;
    }
    if (k.live == 1) {
      T *op = W::row_of((T *)p.o, p.o_s, p, k.b, k.hk, r, div_inv((unsigned)r, g_inv));
      typename VecT<T>::v4 ov;
      const float inv = 1.f / ls;
#pragma unroll
      for (int e = 0; e < 4; ++e) ov[e] = from_f32<T>(os[e] * inv);
      *reinterpret_cast<typename VecT<T>::v4 *>(op + c * 4) = ov;
    } else {
      const int64_t slot = ((int64_t)k.pair * rows + r) * nsplit + k.split;
      if (NC == 1 && arrived) {
        store_through(ws_o + slot * D + c * 4, os);
        if (c == 0) {
          __hip_atomic_store(&ws_ml[slot * 2], mx, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          __hip_atomic_store(&ws_ml[slot * 2 + 1], ls, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
      } else {
        *reinterpret_cast<f32x4 *>(ws_o + slot * D + c * 4) = os;
        if (c == 0) ws_ml[slot * 2] = mx, ws_ml[slot * 2 + 1] = ls;
      }
    }
  }
  if constexpr (NC == 1)
    if (arrived && k.live > 1) tree_merge_here<T, D>(p, k, rows, nsplit, ws_o, ws_ml, g_inv, arrived, smem);
}

// More rows: the four waves share the tiles of the split's keys, each with rows
// of its own (up to two groups of 16), in a ring of four tiles: one barrier a
// tile, after which the slot of the tile before last is asked for anew. With
// waves that stream their own tiles, 264 rows over 32700 e4m3 keys moved 9 times
// the cache through the L1s and took 122 us where the DMA alone took 44. Bound by the
// sum of matrix and VALU work, of which two waves a SIMD hide half: 70-104 us for 2 x 264
// rows over 20000-32700 e4m3 keys and 4 KV heads.
template <typename T, int KIND, int D>
__global__ __launch_bounds__(256, 2) void tree_rows_kernel(TreeArgs p, float *__restrict__ ws_o,
                                                           float *__restrict__ ws_ml, int nsplit,
                                                           unsigned nsplit_inv, unsigned hkv_inv,
                                                           unsigned g_inv, int by_xcd, int groups) {
  typedef TreeTile<KIND, D> TT;
  constexpr int KT = TT::KT, NW = 4, ST = 4, N = TT::TILEB / 1024 / NW, EX = KIND ? 1 : 0, PER = 2 * N + EX;
  __shared__ __attribute__((aligned(16))) char smem[ST * 2 * TT::TILEB];
  __shared__ __attribute__((aligned(16))) unsigned s_e[ST][64];

  const int lane = lane_id(), w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  TreeBlock k = tree_block(p, hkv_inv, by_xcd);
  const int up = tree_parent(p, k.b);
  const int rows = p.T * p.G;

  // rows 16 (qt groups + w + 4 i) .. of this wave, i < nc
  auto run = [&](auto ncc) {
    constexpr int NC = decltype(ncc)::value;
    typedef TreeWave<T, KIND, D, NC> W;
    W wv;
    int row0[NC], row[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i)
      row0[i] = (k.qt * groups + w + 4 * i) * 16, row[i] = min(row0[i] + (lane & 15), rows - 1);
    wv.ask(p, k.b, k.hk, g_inv, row);
    tree_split<KT>(p, nsplit, nsplit_inv, k);
    if (k.c0 >= k.end) return; // the whole block
    const int first = (int)k.c0, k_end = (int)k.c1, n = (k_end - first + KT - 1) / KT;
    const char *ks = (const char *)p.k + ((int64_t)k.b * p.k_s[0] + (int64_t)k.hk * p.k_s[1]) * W::EB;
    const char *vs = (const char *)p.v + ((int64_t)k.b * p.v_s[0] + (int64_t)k.hk * p.v_s[1]) * W::EB;
    const int64_t eb = (int64_t)k.b * p.e_s[0] + (int64_t)k.hk * p.e_s[1];
    TreeDma<KIND, D, N, 0> dk, dv;
    dk.begin(true, w * N, p.k_s[2]);
    dv.begin(false, w * N, p.v_s[2]);
    auto issue = [&](int it) { // (every wave brings the exponents: the same bytes)
      char *const slot = smem + (it & (ST - 1)) * (2 * TT::TILEB);
      dk.issue(ks, p.k_s[2], first + it * KT, k.end, slot);
      if constexpr (KIND != 0) issue_exps(p, eb, first + it * KT, s_e[it & (ST - 1)]);
      dv.issue(vs, p.v_s[2], first + it * KT, k.end, slot + TT::TILEB);
    };
    for (int it = 0; it < ST - 1; ++it)
      if (it < n) issue(it);
    wv.begin(tree_bits(p, up, k.L), lds_addr(smem), lds_addr(smem) + TT::TILEB, lds_addr(s_e[0]));
    for (int it = 0; it < n; ++it) {
      if (it + 2 < n) vm_wait<2 * PER>(); // this wave's part of tile `it` landed
      else if (it + 1 < n) vm_wait<PER>();
      else vm_wait<0>();
      lds_barrier(); // everybody's part, and everybody is done with tile it - 1
      if (it + 3 < n) issue(it + 3);
      wv.step(p, first + it * KT, k.L, (it & (ST - 1)) * (2 * TT::TILEB), (it & (ST - 1)) * 256, [] {}, [] {}, [] {});
    }
    const bool odd = wv.end(p);
    auto put = [&](int i, int q, int d, auto x, float l) { // x: one value or four
      constexpr int M = sizeof(x) / 4;
      const int r = row0[i] + q;
      if (k.live == 1) {
        T *op = W::row_of((T *)p.o, p.o_s, p, k.b, k.hk, r, div_inv((unsigned)r, g_inv)) + d;
        const float inv = 1.f / l;
        if constexpr (M == 4) {
          typename VecT<T>::v4 ov;
#pragma unroll
          for (int e = 0; e < 4; ++e) ov[e] = from_f32<T>(x[e] * inv);
          *reinterpret_cast<typename VecT<T>::v4 *>(op) = ov;
        } else {
          *op = from_f32<T>(x * inv);
        }
      } else {
        *reinterpret_cast<decltype(x) *>(ws_o + (((int64_t)k.pair * rows + r) * nsplit + k.split) * D + d) = x;
      }
    };
    const bool redo = (KIND == 0 || first + n * KT > k.L) && __any(odd);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int q = lane & 15, u4 = lane >> 4;
      if (row0[i] + q >= rows) continue;
      if (!redo)
#pragma unroll
        for (int tt = 0; tt < W::NT; ++tt) put(i, q, tt * 16 + u4 * 4, wv.o[i][tt], wv.l[i]);
      if (u4 == 0 && k.live > 1) {
        const int64_t slot = ((int64_t)k.pair * rows + row0[i] + q) * nsplit + k.split;
        ws_ml[slot * 2] = wv.top(p, i), ws_ml[slot * 2 + 1] = wv.l[i];
      }
    }
    if (redo)
      wv.again(p, k.b, k.hk, ks, vs, eb, first, KT, n, k_end, k.L, g_inv, row0, rows,
               [&](int i, int q, int d, float x) { put(i, q, d, x, __shfl(wv.l[i], q, kWave)); });
  };
  // a block's last groups may leave waves with one, or none: those bring their
  // part of the tiles all the same (as one group, of rows past the last)
  const int have = min(groups, (rows + 15) / 16 - k.qt * groups);
  if (w + 4 < have) run(std::integral_constant<int, 2>{});
  else run(std::integral_constant<int, 1>{});
}

// The splits of every row, which are runs of batches of 2^lstride keys: a part a
// group of D / 4 lanes, the first splits' loads before the sequence's length has come
// (slots that no split wrote are read and not used): a chain of length, maxima and
// sums would be three trips to memory, twice the launch's time.
template <typename T, int D>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs p, const float *__restrict__ ws_o,
                                                         const float *__restrict__ ws_ml, int nsplit,
                                                         unsigned nsplit_inv, unsigned g_inv, int lstride) {
  constexpr int C4 = D / 4, RPB = 256 / (C4 * kMergeParts);
  __shared__ f32x4 s_o[RPB * kMergeParts * C4];
  __shared__ float s_ml[RPB * kMergeParts * 2];
  const int grp = threadIdx.x / C4, q = grp / kMergeParts, g0 = grp % kMergeParts, c = threadIdx.x % C4;
  const int rows = p.T * p.G, r = min((int)blockIdx.x * RPB + q, rows - 1);
  const int hk = blockIdx.y, b = blockIdx.z;
  const int64_t slot = (((int64_t)b * p.Hkv + hk) * rows + r) * nsplit;
  const int len = p.seqlens[b];
  TreeMerge<1> mg;
  mg.begin();
  mg.template load<D, false>(ws_o, ws_ml, slot, c, 0, g0, 1, nsplit - 1);
  const int L = min(max(len, 0), p.Lmax), end = min(L + p.T, p.Lmax);
  const int nbatch = (int)(((unsigned)end + (1u << lstride) - 1) >> lstride);
  const int per = div_inv((unsigned)(nbatch + nsplit - 1), nsplit_inv);
  const int live = (int)((unsigned)(nbatch + per - 1) / (unsigned)per);
  if (live == 1) return; // written by the tile kernel
  for (int s0 = 0; s0 < live; s0 += kMergeParts * kMergeAhead) {
    if (s0) mg.template load<D, false>(ws_o, ws_ml, slot, c, s0, g0, 1, nsplit - 1);
    mg.add(s0, g0, 1, live);
  }
  s_o[grp * C4 + c] = mg.o[0];
  if (c == 0) s_ml[grp * 2] = mg.m[0], s_ml[grp * 2 + 1] = mg.l[0];
  __syncthreads();
  if (g0 || (int)blockIdx.x * RPB + q >= rows) return;
  const int t = div_inv((unsigned)r, g_inv), g = r - t * p.G;
  T *op = (T *)p.o + (int64_t)b * p.o_s[0] + (int64_t)t * p.o_s[1] + (int64_t)(hk * p.G + g) * p.o_s[2];
  *reinterpret_cast<typename VecT<T>::v4 *>(op + c * 4) =
      tree_merge_parts<T>(s_o + q * kMergeParts * C4 + c, C4, s_ml + q * kMergeParts * 2);
}

// How a call is cut: groups of 16 query rows a block (nc: of a wave that shares
// them with the other three; 0: the waves' own), blocks a pair, splits of the keys
// in batches of 2^lstride.
struct TreePlan {
  int nc, groups, qtiles, nsplit, lstride;
};
static TreePlan tree_plan(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t Lmax, int code) {
  TreePlan pl = {0, 0, 0, 0, 0};
  if (D != 64 && D != 128) return pl;
  const int64_t groups = (T * (Hq / Hkv) + 15) / 16;
  pl.nc = groups > 2 ? 0 : (int)groups;
  pl.qtiles = groups > 2 ? (int)((groups + 7) / 8) : 1;
  pl.groups = (int)((groups + pl.qtiles - 1) / pl.qtiles);
  const int lkt = D * (code ? 1 : 2) == 256 || (code && pl.nc) ? 5 : 6;
  pl.lstride = pl.nc ? lkt + 2 : lkt;
  const int64_t most = (Lmax + (4 << lkt) - 1) >> (lkt + 2), blocks = B * Hkv * pl.qtiles;
  const int cus = device_cu_count() > 0 ? device_cu_count() : 256;
  // Two blocks a CU, as many as are resident at once: with 3, 4 and 8 a CU 8 trees of 16
  // over 1500-2288 keys took 25.5, 31.1 and 32.6 us for 21.4, 32 tokens over 2098 keys
  // 31.4, 32.2 and 39.3 for 28.9, and mixed lengths gained nothing.
  int64_t ns = 2 * (int64_t)cus / blocks;
  if (ns > most) ns = most;
  pl.nsplit = (int)(ns > 256 ? 256 : ns < 1 ? 1 : ns);
  return pl;
}

} // namespace tpp

using namespace tpp;

extern "C" size_t tpp_tree_attn_workspace_size(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                               int64_t Lmax, int code) {
  if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || Lmax <= 0) return 0;
  const TreePlan pl = tree_plan(B, T, Hq, Hkv, D, Lmax, code);
  return pl.nsplit > 1 ? (size_t)(B * T * Hq) * pl.nsplit * (D + 2) * sizeof(float) : 0;
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
  // the matrix-core kernel: whole 16-byte rows, exponents by fours
  uint64_t low = (uint64_t)(uintptr_t)q | (uint64_t)(uintptr_t)k | (uint64_t)(uintptr_t)v, low_o = (uint64_t)(uintptr_t)o;
  for (int i = 0; i < 3; ++i) {
    low |= (uint64_t)(a.q_s[i] * 2) | (uint64_t)(a.k_s[i] * (code ? 1 : 2)) | (uint64_t)(a.v_s[i] * (code ? 1 : 2));
    low_o |= (uint64_t)(a.o_s[i] * 2);
  }
  bool tiles = (D == 64 || D == 128) && !(low & 15) && !(low_o & 7) && B * Hkv <= 65535;
  // (div_inv of a row by G is exact below this)
  tiles = tiles && (uint64_t)(T * a.G) * (uint64_t)a.G < 1ull << 32;
  // (a tile's rows by 32-bit byte offsets)
  for (int64_t r : {a.k_s[2], a.v_s[2]}) tiles = tiles && r >= 0 && r < (1 << 23);
  if (code)
    tiles = tiles && Lmax % 4 == 0 &&
            !(((uint64_t)(uintptr_t)k_exps | (uint64_t)(uintptr_t)v_exps | (uint64_t)a.e_s[0] | (uint64_t)a.e_s[1]) & 3);
  if (!tiles) {
    const dim3 grid((unsigned)(Hq * T), (unsigned)B);
    return TPP_DISPATCH_HALF(dtype, [&] {
      if (code == 0) tree_generic_kernel<T, 0><<<grid, dim3(64), 0, st>>>(a, (int)D);
      else if (code == TPP_CODE_E4M3) tree_generic_kernel<T, TPP_CODE_E4M3><<<grid, dim3(64), 0, st>>>(a, (int)D);
      else tree_generic_kernel<T, TPP_CODE_INT8><<<grid, dim3(64), 0, st>>>(a, (int)D);
      return check_launch(name);
    });
  }
  const TreePlan pl = tree_plan(B, T, Hq, Hkv, D, Lmax, code);
  const int64_t rows = T * a.G, pairs = B * Hkv;
  float *ws_o = (float *)workspace, *ws_ml = nullptr;
  if (pl.nsplit > 1) {
    if (!workspace || ((uintptr_t)workspace & 127) || ws_bytes < tpp_tree_attn_workspace_size(B, T, Hq, Hkv, D, Lmax, code))
      return set_error(TPP_E_WORKSPACE, "%s: workspace missing, unaligned or too small", name);
    ws_ml = ws_o + (size_t)(pairs * rows) * pl.nsplit * D;
  }
  const bool by_xcd = pairs % 8 == 0;
  // the merge by a pair's last block
  unsigned *arrived = pl.nsplit > 1 && pl.nc == 1 ? arrival_words(st, pairs) : nullptr;
  const dim3 grid(by_xcd ? 8 * pl.qtiles : pl.qtiles, pl.nsplit, (unsigned)(by_xcd ? pairs / 8 : pairs));
  const unsigned ninv = inv_of(pl.nsplit), hinv = inv_of((int)Hkv), ginv = inv_of(a.G);
  return TPP_DISPATCH_HALF(dtype, [&] {
    auto by_d = [&](auto kd, auto dd) {
      constexpr int KIND = decltype(kd)::value, DD = decltype(dd)::value;
      if (pl.nc == 0)
        tree_rows_kernel<T, KIND, DD><<<grid, dim3(256), 0, st>>>(a, ws_o, ws_ml, pl.nsplit, ninv, hinv, ginv, by_xcd, pl.groups);
      else if (pl.nc == 1)
        tree_tile_kernel<T, KIND, DD, 1><<<grid, dim3(256), 0, st>>>(a, ws_o, ws_ml, pl.nsplit, ninv, hinv, ginv, by_xcd, arrived);
      else
        tree_tile_kernel<T, KIND, DD, 2><<<grid, dim3(256), 0, st>>>(a, ws_o, ws_ml, pl.nsplit, ninv, hinv, ginv, by_xcd, nullptr);
      if (pl.nsplit > 1 && !arrived)
        tree_merge_kernel<T, DD><<<dim3((unsigned)((rows + 256 / DD - 1) / (256 / DD)), (unsigned)Hkv, (unsigned)B), dim3(256), 0, st>>>(
            a, ws_o, ws_ml, pl.nsplit, ninv, ginv, pl.lstride);
    };
    auto by_kind = [&](auto kd) {
      if (D == 64) by_d(kd, std::integral_constant<int, 64>{});
      else by_d(kd, std::integral_constant<int, 128>{});
    };
    if (code == 0) by_kind(std::integral_constant<int, 0>{});
    else if (code == TPP_CODE_E4M3) by_kind(std::integral_constant<int, TPP_CODE_E4M3>{});
    else by_kind(std::integral_constant<int, TPP_CODE_INT8>{});
    return check_launch(name);
  });
}
