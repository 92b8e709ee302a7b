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
#include "tree_wave.hpp"

namespace tpp {

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
  auto at = [&](int j, const char *&kr, const char *&vr) {
    kr = ks + (int64_t)j * p.k_s[2] * W::EB, vr = vs + (int64_t)j * p.v_s[2] * W::EB;
    return true;
  };
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int r = i * 16 + l16;
#pragma unroll
    for (int tt = 0; tt < W::NT; ++tt) part[r * C4 + ((tt * 4 + u4) ^ (r & (C4 - 1)))] = wv.o[i][tt];
    if (u4 == 0) s_m[w][r] = wv.top(p, i), s_l[w][r] = wv.l[i];
  }
  if (n > 0 && (KIND == 0 || first + (n - 1) * STRIDE + KT > k.L) && __any(odd))
    wv.again(p, k.b, k.hk, at, eb, first, STRIDE, n, k_end, k.L, g_inv, row0, rows, [&](int i, int q, int d, float x) {
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
    if (arrived && k.live > 1) tree_merge_here<T, D>(p, k, rows, (int64_t)k.pair * rows * nsplit, nsplit, ws_o, ws_ml, g_inv, arrived, smem);
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
    auto at = [&](int j, const char *&kr, const char *&vr) {
      kr = ks + (int64_t)j * p.k_s[2] * W::EB, vr = vs + (int64_t)j * p.v_s[2] * W::EB;
      return true;
    };
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
      wv.again(p, k.b, k.hk, at, eb, first, KT, n, k_end, k.L, g_inv, row0, rows,
               [&](int i, int q, int d, float x) { put(i, q, d, x, __shfl(wv.l[i], q, kWave)); });
  };
  // a block's last groups may leave waves with one, or none: those bring their
  // part of the tiles all the same (as one group, of rows past the last)
  const int have = min(groups, (rows + 15) / 16 - k.qt * groups);
  if (w + 4 < have) run(std::integral_constant<int, 2>{});
  else run(std::integral_constant<int, 1>{});
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
