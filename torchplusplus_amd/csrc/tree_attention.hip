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

// ---------------------------------------------------------------------------
// Head sizes 64 and 128, 16-byte rows: on the matrix cores.
//
// The T G query rows of a KV head (row = token * G + head of the group) are the
// columns of S^T = K Q^T and of O^T = V^T P^T (32x32x16; a lane owns one query
// row, so the softmax needs one exchange, with lane ^ 32). A block is 4 waves
// over NQ tiles of 32 rows and one split of the sequence's keys; each wave
// streams its own tiles of KT keys (8 KB of K) by LDS-DMA into a private slot:
// no barrier in the loop, the next K tile is requested once this one's
// fragments are in registers, the next V tile after this one's. Waves are
// merged through LDS, splits by tree_merge_kernel (a second launch: the splits'
// arrival counters would have to be shared by calls, which two replayed graphs
// may not do).
//
// Codes stay codes up to the registers: a tile of codes has half the bytes and
// twice the keys. K fragments become T (exact: e4m3 and int8 values fit both
// types), V fragments bfloat16; the exponents are applied to the scores and to
// the probabilities, 2 x 16 a lane and 32 keys, where scaling the operands would
// take 4 D / 64 times as many. P of a coded cache is rounded to bfloat16 (its
// range holds p 2^e, fp16's does not), else to T, in fp16 times 2^15 so that
// weights down to 2^-39 of the largest are kept; each weight is off by 2^-9 (fp16:
// 2^-12) at most, the sum of weights is kept in fp32 from the unrounded ones.
// ---------------------------------------------------------------------------
template <int KIND, int D> struct TreeTile {
  static constexpr int ROWB = D * (KIND ? 1 : 2);  // bytes of a row
  static constexpr int KT = ROWB == 256 ? 32 : 64; // keys of a tile
  static constexpr int UPR = ROWB / 16, TILEB = KT * ROWB;
  // 16-byte unit u of row r is stored at u ^ ksw(r) in a K tile (so that 8
  // lanes reading one unit of 8 rows hit distinct banks), at u ^ vsw(r) in a V
  // tile (distinct banks for the transposing reads)
  static __device__ __forceinline__ int ksw(int r) {
    return UPR == 4 ? (r ^ (r >> 2)) & 3 : r & (UPR - 1);
  }
  static __device__ __forceinline__ int vsw(int r) {
    if constexpr (KIND == 0) return vswz<D>(r);
    else return D == 128 ? 2 * ((r >> 1) & 3) : 2 * ((r >> 2) & 1);
  }
};

// eight codes as values of type T
template <typename T, int KIND>
__device__ __forceinline__ typename VecT<T>::v8 codes8(unsigned a, unsigned b) {
  typedef typename VecT<T>::v8 V8;
  u32x4 r;
  if constexpr (KIND == TPP_CODE_E4M3) {
    auto two = [](unsigned c, auto hi) {
      if constexpr (__is_same(T, bf16))
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.f, decltype(hi)::value));
      else
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.f, decltype(hi)::value));
    };
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
  return __uint_as_float((I == 3 ? w >> 1 : w << (23 - 8 * I)) & 0x7f800000u);
}

template <typename T, int KIND, int D, int NQ>
__global__ __launch_bounds__(256, NQ == 1 ? 2 : 1) void tree_tile_kernel(TreeArgs p, float *__restrict__ ws_o,
                                                        float *__restrict__ ws_ml, int nsplit,
                                                        unsigned nsplit_inv, unsigned hkv_inv,
                                                        unsigned g_inv, int by_xcd) {
  typedef typename VecT<T>::v8 V8;
  typedef std::conditional_t<KIND == 0, T, bf16> PT; // type of P and V operands
  typedef typename VecT<PT>::v8 P8;
  typedef TreeTile<KIND, D> TT;
  constexpr int KT = TT::KT, NB = KT / 32, NW = 4, STRIDE = NW * KT, ROWB = TT::ROWB, UPR = TT::UPR;
  constexpr int KPI = 64 / UPR, NDMA = KT / KPI, EX = KIND ? 1 : 0, NT = D / 32, C4 = D / 4;
  static_assert(2 * TT::TILEB >= 32 * D * 4 && (KIND == 0 || NB == 2), "a wave's rows fit its tiles");
  __shared__ __attribute__((aligned(16))) char smem[NW * 2 * TT::TILEB];
  __shared__ __attribute__((aligned(16))) unsigned s_e[NW][64];
  __shared__ float s_m[NW][32], s_l[NW][32];
  constexpr float kUp = KIND == 0 && !__is_same(T, bf16) ? 15.f : 0.f;

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, ql = lane & 31;
  const int pair = by_xcd ? blockIdx.z * 8 + (blockIdx.x & 7) : blockIdx.z;
  const int qt = by_xcd ? blockIdx.x >> 3 : blockIdx.x, split = blockIdx.y;
  const int b = div_inv(pair, hkv_inv), hk = pair - b * p.Hkv;
  const int L = min(max(p.seqlens[b], 0), p.Lmax), end = min(L + p.T, p.Lmax);
  const int nbatch = (int)((unsigned)(end + STRIDE - 1) / (unsigned)STRIDE);
  const int per = div_inv((unsigned)(nbatch + nsplit - 1), nsplit_inv);
  const int64_t c0 = (int64_t)split * per * STRIDE;
  if (c0 >= end) return;
  const int k_end = (int)(c0 + (int64_t)per * STRIDE < end ? c0 + (int64_t)per * STRIDE : end);
  const int first = (int)c0 + w * KT;
  const int n = first < k_end ? (k_end - first + STRIDE - 1) / STRIDE : 0; // this wave's tiles

  constexpr int EB = KIND ? 1 : 2;
  const char *ks = (const char *)p.k + ((int64_t)b * p.k_s[0] + (int64_t)hk * p.k_s[1]) * EB;
  const char *vs = (const char *)p.v + ((int64_t)b * p.v_s[0] + (int64_t)hk * p.v_s[1]) * EB;
  const int64_t eb = (int64_t)b * p.e_s[0] + (int64_t)hk * p.e_s[1];
  const int dkey = lane / UPR, dslot = lane % UPR;
  char *const ring = smem + w * (2 * TT::TILEB);
  // exponents of a tile as the lanes of half h read them: 8 dwords of K (scores
  // 32 st + 8 g + 4 h .. + 3 in dword 4 st + g), 8 of V 64 bytes on
  const uint8_t *es = nullptr;
  int edw = 0;
  if constexpr (KIND != 0) {
    es = (lane & 16 ? p.ve : p.ke) + eb;
    edw = 4 * (((lane >> 2) & 1) * 8 + (lane & 3) * 2 + ((lane >> 3) & 1));
  }
  auto issue = [&](bool kt, int base) {
    const char *src = kt ? ks : vs;
    const int64_t ss = (kt ? p.k_s[2] : p.v_s[2]) * EB;
#pragma unroll
    for (int j = 0; j < NDMA; ++j) {
      const int key = j * KPI + dkey;
      const int ch = dslot ^ (kt ? TT::ksw(key) : TT::vsw(key));
      __builtin_amdgcn_global_load_lds((const void *)(src + (int64_t)min(base + key, end - 1) * ss + ch * 16),
                                       (__attribute__((address_space(3))) void *)(ring + (kt ? 0 : TT::TILEB) + j * 1024),
                                       16, 0, kCpolNT);
    }
    if constexpr (KIND != 0)
      if (kt) // (lanes 32 - 63 repeat 0 - 31)
        __builtin_amdgcn_global_load_lds((const void *)(es + min(base + edw, p.Lmax - 4)),
                                         (__attribute__((address_space(3))) void *)s_e[w], 4, 0, 0);
  };
  if (n > 0) {
    issue(true, first);
    issue(false, first);
  }

  // this lane's query row of each tile: its fragments, and what it sees
  const unsigned long long bits = tree_bits(p, b, L);
  const int rows = p.T * p.G;
  V8 qf[NQ][D / 16];
  unsigned long long see[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const int r = min((qt * NQ + i) * 32 + ql, rows - 1);
    const int t = div_inv((unsigned)r, g_inv), g = r - t * p.G;
    see[i] = ((unsigned long long)(unsigned)__shfl((int)(bits >> 32), t, kWave) << 32) |
             (unsigned)__shfl((int)bits, t, kWave);
    const T *qp = (const T *)p.q + (int64_t)b * p.q_s[0] + (int64_t)t * p.q_s[1] + (int64_t)(hk * p.G + g) * p.q_s[2];
#pragma unroll
    for (int k = 0; k < D / 16; ++k) // codes: a 16-byte read holds both steps of 32 elements
      qf[i][k] = *reinterpret_cast<const V8 *>(qp + (KIND ? (k / 2) * 32 + h * 16 + (k & 1) * 8 : k * 16 + h * 8));
  }
  // waited for here (with the first tiles): no wait for them inside the loop
#pragma unroll
  for (int i = 0; i < NQ; ++i)
#pragma unroll
    for (int k = 0; k < D / 16; ++k) asm volatile("" ::"v"(qf[i][k]));

  f32x16 o[NQ][NT];
  float m_run[NQ], l_run[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    m_run[i] = -INFINITY, l_run[i] = 0.f;
#pragma unroll
    for (int tt = 0; tt < NT; ++tt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[i][tt][r] = 0.f;
  }
  const float c2 = p.scale_log2;
  const unsigned base0 = (unsigned)(uintptr_t)(const __attribute__((address_space(3))) char *)ring;
  const unsigned ebase = (unsigned)(uintptr_t)(const __attribute__((address_space(3))) unsigned *)s_e[w] + h * 32;
  const int grp = lane >> 4;
  unsigned vo[NT];
#pragma unroll
  for (int tt = 0; tt < NT; ++tt) {
    if constexpr (KIND == 0) {
      const int a4 = lane & 3, kl = 4 * (grp >> 1) + ((lane >> 2) & 3), d0 = tt * 32 + 16 * (grp & 1) + 4 * a4;
      vo[tt] = base0 + TT::TILEB + kl * ROWB + (((d0 >> 3) ^ TT::vsw(kl)) << 4) + ((d0 & 7) << 1);
    } else {
      const int rr = (lane >> 1) & 7, kl = 8 * (rr >> 2) + 4 * (grp >> 1) + (rr & 3);
      vo[tt] = base0 + TT::TILEB + kl * ROWB + (((2 * tt + (grp & 1)) ^ TT::vsw(kl)) << 4) + 8 * (lane & 1);
    }
  }

  for (int it = 0; it < n; ++it) {
    const int kb = first + it * STRIDE;
    const bool more = it + 1 < n, edge = kb + KT > L;
    vm_wait<NDMA>(); // this tile's K (and exponents) landed, its V may be in flight
    f32x16 s[NQ][NB];
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
      for (int st = 0; st < NB; ++st)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[i][st][r] = 0.f;
    u32x4 ex[4];
    if constexpr (KIND == 0) {
      constexpr int KS = D / 16, NS = KS * NB / 2;
      V8 kr[3][2];
      auto kfrag = [&](auto ii) {
        constexpr int x = decltype(ii)::value;
        static_for<2>([&](auto jj) {
          constexpr int j = decltype(jj)::value, k = NB == 2 ? x : 2 * x + j;
          const unsigned a = base0 + (unsigned)((ql * UPR + ((k * 2 + h) ^ TT::ksw(ql))) * 16);
          kr[x % 3][j] = lds_read_b128<(NB == 2 ? j : 0) * 32 * ROWB, V8>(a);
        });
      };
      kfrag(std::integral_constant<int, 0>{});
      kfrag(std::integral_constant<int, 1>{});
      static_for<NS>([&](auto ii) {
        constexpr int x = decltype(ii)::value;
        if constexpr (x + 2 < NS) kfrag(std::integral_constant<int, x + 2>{});
        lds_wait_tied<(x + 2 < NS ? 2 : NS - 1 - x) * 2>(kr[x % 3]);
        if constexpr (x == NS - 1) { // every K fragment is in registers
          asm volatile("" ::: "memory");
          if (more) issue(true, kb + STRIDE);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < NQ; ++i)
            s[i][j % NB] = mfma32x32<T>(kr[x % 3][j], qf[i][NB == 2 ? x : 2 * x + j], s[i][j % NB]);
        __builtin_amdgcn_sched_barrier(0);
      });
    } else {
      constexpr int NP = D / 32; // 16-byte reads: two steps of a half's 8 elements
      u32x4 kr[NP][2];
      static_for<NP>([&](auto ii) {
        constexpr int x = decltype(ii)::value;
        const unsigned a = base0 + (unsigned)((ql * UPR + ((2 * x + h) ^ TT::ksw(ql))) * 16);
        kr[x][0] = lds_read_b128<0, u32x4>(a);
        kr[x][1] = lds_read_b128<32 * ROWB, u32x4>(a);
      });
      ex[0] = lds_read_b128<0, u32x4>(ebase), ex[1] = lds_read_b128<16, u32x4>(ebase);
      ex[2] = lds_read_b128<64, u32x4>(ebase), ex[3] = lds_read_b128<80, u32x4>(ebase);
      static_for<NP>([&](auto ii) {
        constexpr int x = decltype(ii)::value;
        lds_wait_tied<2 * (NP - 1 - x) + 4>(kr[x]);
        if constexpr (x == NP - 1) {
          lds_wait_tied<0>(ex);
          asm volatile("" ::: "memory");
          if (more) issue(true, kb + STRIDE);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            const V8 f = codes8<T, KIND>(kr[x][st][2 * u], kr[x][st][2 * u + 1]);
#pragma unroll
            for (int i = 0; i < NQ; ++i) s[i][st] = mfma32x32<T>(f, qf[i][2 * x + u], s[i][st]);
          }
        __builtin_amdgcn_sched_barrier(0);
      });
    }

    P8 pb[NQ][2 * NB];
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      if constexpr (KIND != 0)
#pragma unroll
        for (int st = 0; st < NB; ++st)
          static_for<16>([&](auto rr) {
            constexpr int r = decltype(rr)::value;
            s[i][st][r] *= exp_of<r % 4>(ex[st][r / 4]);
          });
      unsigned keep[NB]; // bit 8 g + e: score register 4 g + e
      if (edge) {
        const unsigned ninf = __float_as_uint(-INFINITY);
#pragma unroll
        for (int st = 0; st < NB; ++st) {
          const int rel = kb + 32 * st - L;
          const unsigned k32 = rel >= 64 ? 0u
                               : rel >= 0 ? (unsigned)(see[i] >> rel)
                               : rel > -32 ? ((unsigned)see[i] << -rel) | ((1u << -rel) - 1u)
                                           : ~0u;
          keep[st] = k32 >> (4 * h);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const unsigned bm = (unsigned)__builtin_amdgcn_sbfe((int)keep[st], (r >> 2) * 8 + (r & 3), 1);
            s[i][st][r] = __uint_as_float((__float_as_uint(s[i][st][r]) & bm) | (ninf & ~bm));
          }
        }
      }
      float mx[4] = {s[i][0][0], s[i][0][1], s[i][0][2], s[i][0][3]};
#pragma unroll
      for (int st = 0; st < NB; ++st)
#pragma unroll
        for (int r = st == 0 ? 4 : 0; r < 16; ++r) mx[r & 3] = fmaxf(mx[r & 3], s[i][st][r]);
      float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
      mt = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
      const bool move = mt > m_run[i];
      const float m_new = move ? mt : m_run[i];
      const float mc = m_new == -INFINITY ? 0.f : m_new * c2;
      const float alpha = move ? __builtin_amdgcn_exp2f(m_run[i] * c2 - mc) : 1.f;
      float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < NB; ++st)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float e = __builtin_amdgcn_exp2f(fmaf(s[i][st][r], c2, kUp - mc));
          s[i][st][r] = e;
          ps[r & 3] += e;
        }
      l_run[i] = l_run[i] * alpha + ((ps[0] + ps[1]) + (ps[2] + ps[3]));
      m_run[i] = m_new;
      if (__any(move)) {
#pragma unroll
        for (int tt = 0; tt < NT; ++tt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[i][tt][r] *= alpha;
      }
      if constexpr (KIND != 0) {
#pragma unroll
        for (int st = 0; st < NB; ++st)
          static_for<16>([&](auto rr) {
            constexpr int r = decltype(rr)::value;
            s[i][st][r] *= exp_of<r % 4>(ex[2 + st][r / 4]);
          });
        if (edge) { // a masked row of NaN: 0 times infinity above
#pragma unroll
          for (int st = 0; st < NB; ++st)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              s[i][st][r] = __uint_as_float(__float_as_uint(s[i][st][r]) &
                                            (unsigned)__builtin_amdgcn_sbfe((int)keep[st], (r >> 2) * 8 + (r & 3), 1));
        }
      }
#pragma unroll
      for (int c = 0; c < 2 * NB; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) pb[i][c][j] = from_f32<PT>(s[i][c >> 1][(c & 1) * 8 + j]);
    }

    // this tile's V landed (the next K may be in flight)
    if (more) vm_wait<NDMA + EX>();
    else vm_wait<0>();
    constexpr int R = KIND ? NT : 2 * NT;
    typedef std::conditional_t<KIND == 0, s16x4, u32x2> VR;
    VR vr[2][R];
    auto vfrag = [&](auto cc) {
      constexpr int c = decltype(cc)::value;
#pragma unroll
      for (int tt = 0; tt < NT; ++tt) {
        if constexpr (KIND == 0) {
          vr[c % 2][2 * tt] = lds_read_tr16<c * 16 * ROWB>(vo[tt]);
          vr[c % 2][2 * tt + 1] = lds_read_tr16<c * 16 * ROWB + 8 * ROWB>(vo[tt]);
        } else {
          vr[c % 2][tt] = lds_read_tr8<c * 16 * ROWB>(vo[tt]);
        }
      }
    };
    vfrag(std::integral_constant<int, 0>{});
    static_for<2 * NB>([&](auto cc) {
      constexpr int c = decltype(cc)::value;
      if constexpr (c + 1 < 2 * NB) vfrag(std::integral_constant<int, c + 1>{});
      lds_wait_tied<(c + 1 < 2 * NB ? R : 0)>(vr[c % 2]);
      if constexpr (c + 1 == 2 * NB) {
        asm volatile("" ::: "memory");
        if (more) issue(false, kb + STRIDE);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int tt = 0; tt < NT; ++tt) {
        P8 f;
        if constexpr (KIND == 0) {
          typedef short s16x8 __attribute__((ext_vector_type(8)));
          const s16x8 r12 = __builtin_shufflevector(vr[c % 2][2 * tt], vr[c % 2][2 * tt + 1], 0, 1, 2, 3, 4, 5, 6, 7);
          f = __builtin_bit_cast(P8, r12);
        } else {
          f = codes8<PT, KIND>(vr[c % 2][tt][0], vr[c % 2][tt][1]);
        }
#pragma unroll
        for (int i = 0; i < NQ; ++i) o[i][tt] = mfma32x32<PT>(f, pb[i][c], o[i][tt]);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  }

  // The wave's rows, then the block's: row ql's chunk c of 4 values at c ^ ql
  f32x4 *const part = reinterpret_cast<f32x4 *>(ring);
  const int live = (int)((unsigned)(nbatch + per - 1) / (unsigned)per);
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const int r0 = (qt * NQ + i) * 32;
    if (r0 >= rows) break; // all waves
    if (i) __syncthreads();
    bool odd = false;
    float l = l_run[i] + __shfl_xor(l_run[i], 32, kWave), m = m_run[i];
    if (!see[i]) l = 0.f, m = -INFINITY;
#pragma unroll
    for (int tt = 0; tt < NT; ++tt)
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = see[i] ? o[i][tt][rg * 4 + e] : 0.f;
          odd |= !(fabsf(v[e]) < INFINITY);
        }
        part[ql * C4 + ((tt * 8 + rg * 2 + h) ^ (ql & (C4 - 1)))] = v;
      }
    if (h == 0) s_m[w][ql] = m == -INFINITY ? m : m * c2, s_l[w][ql] = l;
    // A row behind the context that is not finite, times a weight of 0, is a
    // NaN in the products of those that do not see it: a wave with such a tile
    // and a sum that is not finite sums again, over what each row sees.
    if (n > 0 && first + (n - 1) * STRIDE + KT > L && __any(odd)) {
      for (int q = 0; q < 32 && r0 + q < rows; ++q) {
        const unsigned long long sq = ((unsigned long long)(unsigned)__shfl((int)(see[i] >> 32), q, kWave) << 32) |
                                      (unsigned)__shfl((int)see[i], q, kWave);
        if (!sq) continue;
        const int t = div_inv((unsigned)(r0 + q), g_inv), g = r0 + q - t * p.G;
        const T *qp = (const T *)p.q + (int64_t)b * p.q_s[0] + (int64_t)t * p.q_s[1] + (int64_t)(hk * p.G + g) * p.q_s[2];
        const float mq = __shfl(m_run[i], q, kWave), mc = mq == -INFINITY ? 0.f : mq * c2;
        float acc[D / 64];
#pragma unroll
        for (int c = 0; c < D / 64; ++c) acc[c] = 0.f;
        for (int it = 0; it < n; ++it)
          for (int j = first + it * STRIDE; j < min(first + it * STRIDE + KT, k_end); ++j) {
            if (j >= L && !((sq >> (j - L)) & 1)) continue;
            const char *kr = ks + (int64_t)j * p.k_s[2] * EB, *vr = vs + (int64_t)j * p.v_s[2] * EB;
            const float fk = KIND ? exp_scale(p.ke, eb + j) : 1.f, fv = KIND ? exp_scale(p.ve, eb + j) : 1.f;
            float sd = 0.f;
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
              sd += to_f32(qp[c * 64 + lane]) * cache_value<T, KIND>(kr, c * 64 + lane, fk);
            const float e = __builtin_amdgcn_exp2f(fmaf(wave_sum(sd), c2, kUp - mc));
#pragma unroll
            for (int c = 0; c < D / 64; ++c) acc[c] += e * cache_value<T, KIND>(vr, c * 64 + lane, fv);
          }
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const int d = c * 64 + lane;
          reinterpret_cast<float *>(part + q * C4 + ((d / 4) ^ (q & (C4 - 1))))[d % 4] = acc[c];
        }
      }
    }
    __syncthreads();
    for (int idx = tid; idx < 32 * C4; idx += 64 * NW) {
      const int row = idx / C4, c = idx % C4, r = r0 + row;
      if (r >= rows) break;
      float mx = -INFINITY;
#pragma unroll
      for (int ww = 0; ww < NW; ++ww) mx = fmaxf(mx, s_m[ww][row]);
      const float mu = mx == -INFINITY ? 0.f : mx;
      float ls = 0.f;
      f32x4 os = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ww = 0; ww < NW; ++ww) {
        const float cf = __builtin_amdgcn_exp2f(s_m[ww][row] - mu);
        ls += s_l[ww][row] * cf;
        const f32x4 pr = reinterpret_cast<const f32x4 *>(smem + ww * (2 * TT::TILEB))[row * C4 + (c ^ (row & (C4 - 1)))];
#pragma unroll
        for (int e = 0; e < 4; ++e) os[e] += pr[e] * cf;
      }
      if (live == 1) {
        const int t = div_inv((unsigned)r, g_inv), g = r - t * p.G;
        T *op = (T *)p.o + (int64_t)b * p.o_s[0] + (int64_t)t * p.o_s[1] + (int64_t)(hk * p.G + g) * p.o_s[2];
        typename VecT<T>::v4 ov;
        const float inv = ls != 0.f ? 1.f / ls : 0.f; // (NaN stays NaN)
#pragma unroll
        for (int e = 0; e < 4; ++e) ov[e] = from_f32<T>(os[e] * inv);
        *reinterpret_cast<typename VecT<T>::v4 *>(op + c * 4) = ov;
      } else {
        const int64_t slot = ((int64_t)pair * rows + r) * nsplit + split;
        *reinterpret_cast<f32x4 *>(ws_o + slot * D + c * 4) = os;
        if (c == 0) ws_ml[slot * 2] = mx, ws_ml[slot * 2 + 1] = ls;
      }
    }
  }
}

// The splits of every row: D / 4 lanes a row.
template <typename T, int D, int STRIDE>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs p, const float *__restrict__ ws_o,
                                                         const float *__restrict__ ws_ml, int nsplit,
                                                         unsigned nsplit_inv, unsigned g_inv) {
  constexpr int C4 = D / 4, RPB = 256 / C4;
  const int rows = p.T * p.G, r = blockIdx.x * RPB + threadIdx.x / C4, c = threadIdx.x % C4;
  const int hk = blockIdx.y, b = blockIdx.z;
  if (r >= rows) return;
  const int L = min(max(p.seqlens[b], 0), p.Lmax), end = min(L + p.T, p.Lmax);
  const int nbatch = (int)((unsigned)(end + STRIDE - 1) / (unsigned)STRIDE);
  const int per = div_inv((unsigned)(nbatch + nsplit - 1), nsplit_inv);
  const int live = (int)((unsigned)(nbatch + per - 1) / (unsigned)per);
  if (live == 1) return; // written by the tile kernel
  const int64_t slot = (((int64_t)b * p.Hkv + hk) * rows + r) * nsplit;
  float mx = -INFINITY;
#pragma unroll 8
  for (int s = 0; s < live; ++s) mx = fmaxf(mx, ws_ml[(slot + s) * 2]);
  const float mu = mx == -INFINITY ? 0.f : mx;
  float ls = 0.f;
  f32x4 os = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int s = 0; s < live; ++s) {
    const float cf = __builtin_amdgcn_exp2f(ws_ml[(slot + s) * 2] - mu);
    ls += ws_ml[(slot + s) * 2 + 1] * cf;
    const f32x4 pr = *reinterpret_cast<const f32x4 *>(ws_o + (slot + s) * D + c * 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) os[e] += pr[e] * cf;
  }
  const int t = div_inv((unsigned)r, g_inv), g = r - t * p.G;
  T *op = (T *)p.o + (int64_t)b * p.o_s[0] + (int64_t)t * p.o_s[1] + (int64_t)(hk * p.G + g) * p.o_s[2];
  typename VecT<T>::v4 ov;
  const float inv = ls != 0.f ? 1.f / ls : 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) ov[e] = from_f32<T>(os[e] * inv);
  *reinterpret_cast<typename VecT<T>::v4 *>(op + c * 4) = ov;
}

// How a call is cut: query tiles a block, blocks a pair, splits of the keys.
struct TreePlan {
  int nq, qtiles, nsplit;
};
static TreePlan tree_plan(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t Lmax, int code) {
  TreePlan pl = {0, 0, 0};
  if (D != 64 && D != 128) return pl;
  const int64_t rows = T * (Hq / Hkv);
  pl.nq = rows > 32 ? 2 : 1;
  pl.qtiles = (int)((rows + 32 * pl.nq - 1) / (32 * pl.nq));
  const int kt = D * (code ? 1 : 2) == 256 ? 32 : 64;
  const int64_t most = (Lmax + 4 * kt - 1) / (4 * kt), blocks = B * Hkv * pl.qtiles;
  const int cus = device_cu_count() > 0 ? device_cu_count() : 256;
  int64_t ns = (2 * (int64_t)cus + blocks - 1) / blocks;
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
    if (!workspace || !aligned16(workspace) || ws_bytes < tpp_tree_attn_workspace_size(B, T, Hq, Hkv, D, Lmax, code))
      return set_error(TPP_E_WORKSPACE, "%s: workspace missing, unaligned or too small", name);
    ws_ml = ws_o + (size_t)(pairs * rows) * pl.nsplit * D;
  }
  const bool by_xcd = pairs % 8 == 0;
  const dim3 grid(by_xcd ? 8 * pl.qtiles : pl.qtiles, pl.nsplit, (unsigned)(by_xcd ? pairs / 8 : pairs));
  const unsigned ninv = inv_of(pl.nsplit), hinv = inv_of((int)Hkv), ginv = inv_of(a.G);
  return TPP_DISPATCH_HALF(dtype, [&] {
    auto go = [&](auto kd, auto dd, auto nn) {
      constexpr int KIND = decltype(kd)::value, DD = decltype(dd)::value, NQ = decltype(nn)::value;
      tree_tile_kernel<T, KIND, DD, NQ><<<grid, dim3(256), 0, st>>>(a, ws_o, ws_ml, pl.nsplit, ninv, hinv, ginv, by_xcd);
      if (pl.nsplit > 1)
        tree_merge_kernel<T, DD, 4 * TreeTile<KIND, DD>::KT>
              <<<dim3((unsigned)((rows + 1024 / DD - 1) / (1024 / DD)), (unsigned)Hkv, (unsigned)B), dim3(256), 0, st>>>(
                  a, ws_o, ws_ml, pl.nsplit, ninv, ginv);
    };
    auto by_q = [&](auto kd, auto dd) {
      if (pl.nq == 1) go(kd, dd, std::integral_constant<int, 1>{});
      else go(kd, dd, std::integral_constant<int, 2>{});
    };
    auto by_d = [&](auto kd) {
      if (D == 64) by_q(kd, std::integral_constant<int, 64>{});
      else by_q(kd, std::integral_constant<int, 128>{});
    };
    if (code == 0) by_d(std::integral_constant<int, 0>{});
    else if (code == TPP_CODE_E4M3) by_d(std::integral_constant<int, TPP_CODE_E4M3>{});
    else by_d(std::integral_constant<int, TPP_CODE_INT8>{});
    return check_launch(name);
  });
}
