// Attention of sequences of different lengths packed one behind the other: query
// token i of sequence b (rows cu_q[b] .. cu_q[b + 1] - 1) sees keys of rows cu_k[b] ..
// cu_k[b + 1] - 1 of its own sequence,
//   o[i, h] = softmax_j(scale q[i, h] . k[j, h / G]) v[j, h / G],
// causal and window bounds aligned bottom-right in each sequence (query i at key i + Lk -
// Lq). A row that sees nothing is 0, one whose scores are all -inf NaN.
//
// Head sizes 64 and 128 with 16-byte rows run on the matrix cores, on the kernels of
// attention_prefill.hpp with each query tile's sequence in place of the batch index. Grids are
// sized by what is known on the host, the number of tokens and of sequences: N tokens in B
// sequences have at most N / tile + B query tiles.
//  * short or few sequences: packed_wave_kernel, tiles of 32 queries of one head (of a few
//    queries behind cached keys: of as many heads as fill the tile), each wave on its own. A
//    block finds its sequence by a scan of the lengths, so it is one launch.
//  * else attn_prefill_kernel, 128 queries of two heads (or 64 of four, 256 of one) a tile: a
//    block each, or, where they are many, one block a CU that loops over its share of them.
//    That static dealing wants the tiles from the heaviest to the lightest: packed_plan_kernel
//    sorts them first.
#include "attention_prefill.hpp"

namespace tpp {

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

// A query row of a lane: its sequence, its index there and whether it is to be written.
struct PackedRow {
  PackedSeq seq;
  int i;
  bool real;
};
// Self-attention: tile `t` is rows 32 t .. 32 t + 31 of the batch, whatever sequences they are
// of, so that short ones share a tile. packed_find searches in 64 parts for the first sequence
// that ends past the tile's first row, or up to 63 ahead of it; packed_row_self takes it from
// there, given the begins and ends of the 64 sequences from `lo`, a lane each.
__device__ __forceinline__ int packed_find(const PackedArgs &p, int t) {
  int lo = 0, hi = p.B; // the sequence is in [lo, hi), or there is none
  while (hi - lo > kWave) {
    const int step = (hi - lo + kWave - 1) / kWave, at = min(lo + (lane_id() + 1) * step, hi) - 1;
    const unsigned long long past = __ballot(p.cu_q[at + 1] > t * 32);
    const int l = past ? __builtin_ctzll(past) : kWave - 1;
    const int next = lo + l * step;
    hi = min(next + step, hi), lo = min(next, hi);
  }
  return lo;
}
__device__ __forceinline__ PackedRow packed_row_self(const PackedArgs &p, int t, int lo, int begin, int end) {
  const int first = t * 32, r = min(first + (lane_id() & 31), p.Nq - 1);
  const bool in = first + (lane_id() & 31) < p.Nq;
  PackedRow o = {{r, 0, 0, 0}, 0, in && p.fill != 0}; // of no sequence
  bool found = false;
  auto take = [&](int lo, int begin, int end) { // whether sequences behind these may have rows in the tile
    if (lo + lane_id() >= p.B) begin = end = 0x7fffffff;
    // (mostly one or two do)
    for (unsigned long long hit = __ballot(end > first && begin < first + 32); hit; hit &= hit - 1) {
      const int l = __builtin_ctzll(hit);
      // (packed_seq's rows, without another trip to memory)
      const int q0 = max(__builtin_amdgcn_readlane(begin, l), 0), q1 = min(__builtin_amdgcn_readlane(end, l), p.Nq);
      if (!found && r >= q0 && r < q1) found = true, o = {{q0, q1 - q0, q0, q1 - q0}, r - q0, in};
    }
    return __builtin_amdgcn_readlane(end, kWave - 1) < first + 32;
  };
  // (the first apart: values loaded in a loop are waited for, with every DMA, where it begins)
  if (take(lo, begin, end))
    for (int at = lo + kWave; at < p.B; at += kWave)
      if (!take(at, p.cu_q[min(at + lane_id(), p.B)], p.cu_q[min(at + lane_id() + 1, p.B)])) break;
  return o;
}

// ---------------------------------------------------------------------------
// Short or few sequences: a wave has 32 queries of one head and streams its own KT-key tiles of
// K and V by LDS-DMA into a slot of its own, the next K tile asked for once this one's
// fragments are in registers, the next V tile after this one's. No wave waits for another.
// SH = 1: the four waves of a block are four heads of the same queries. SH = 4: they share one
// head's keys, every fourth tile each, and are merged through LDS. (Eight waves a row were
// slower everywhere: the rate at which a CU's LDS-DMA brings tiles, ~80 bytes a ns, bounds
// both where sequences are not short. Short ones are the launch and a chain of trips to memory,
// 6.8 us for one of 230 tokens, 11.8 for 64 of 3 to 200.) The keys that rows see rise with the
// rows, so the first and last row that see any give the wave's range; keys of a tile that a row
// does not see, other sequences' among them, are masked.
// ---------------------------------------------------------------------------
template <typename T, int D, int SH, bool SELF>
__global__ __launch_bounds__(256, 2) void packed_wave_kernel(PackedArgs p, int nh, int lg) {
  constexpr bool SPLIT = SH > 1;
  typedef typename VecT<T>::v8 V8;
  typedef typename VecT<T>::v4 V4;
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  constexpr int KT = kSplitTile<D>, NB = KT / 32, CPR = D / 8, NT = D / 32, TU = KT * CPR, KPI = 64 / CPR;
  constexpr int NW = 4, NDMA = KT / KPI, KS = D / 16, LDO = D + 4, RBY = D * 2, ORPI = 64 / CPR;
  constexpr float kUp = kWeightUp<T, true>;
  constexpr int kRing = NW * 2 * TU * 16, kMerge = SPLIT ? NW * 32 * LDO * 4 : 0;
  __shared__ __attribute__((aligned(16))) char smem[kRing > kMerge ? kRing : kMerge];
  __shared__ float s_m[NW][32], s_l[NW][32];
  __shared__ unsigned s_bad;
  __shared__ int s_cu[NW][2][kWave];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, ql = lane & 31;
  const int e = blockIdx.x / nh, hb = blockIdx.x - e * nh;
  // rows: 32 >> lg queries of 1 << lg heads that share their keys, a query's heads side by side
  const int hq = (SPLIT ? hb : hb * 4 + w) << lg, heads = (1 << lg) - 1;
  if (hq >= p.Hq) return;
  const int hk = hq / (p.Hq / p.Hkv);
  const char *kp = (const char *)((const T *)p.k + (int64_t)hk * p.k_sh);
  const char *vp = (const char *)((const T *)p.v + (int64_t)hk * p.v_sh);
  char *const ring = smem + w * (2 * TU * 16);
  const int dkey = lane / CPR, dslot = lane % CPR;
  int row_lo = 0, row_hi = p.Nk - 1;
  // the tile at row kb; keys ahead of row_lo or behind row_hi read those rows (masked)
  auto issue = [&](const char *head, int64_t ss, int kb, char *dst, auto swizzle) {
    const int rb = min(max(kb, row_lo), row_hi);
    const char *tb = head + (int64_t)rb * ss * 2;
#pragma unroll
    for (int j = 0; j < NDMA; ++j) {
      const int key = j * KPI + dkey, rel = min(max(kb + key, row_lo), row_hi) - rb;
      __builtin_amdgcn_global_load_lds((const void *)(tb + (unsigned)(rel * (int)ss * 2 + ((dslot ^ swizzle(key)) << 4))),
                                       (__attribute__((address_space(3))) void *)(dst + j * 1024), 16, 0, 0);
    }
  };
  auto issue_k = [&](int kb) { issue(kp, p.k_ss, kb, ring, [](int r) { return r & (CPR - 1); }); };
  auto issue_v = [&](int kb) { issue(vp, p.v_ss, kb, ring + TU * 16, [](int r) { return vswz<D>(r); }); };
  V8 qf[KS];
  auto ask_q = [&](int qrow) {
    const T *qp = (const T *)p.q + (int64_t)qrow * p.q_ss + (int64_t)(hq + (ql & heads)) * p.q_sh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const V8 *>(qp + ks * 16 + h * 8);
  };

  // Tiles go from the keys' end down: a causal tile of self-attention ends with its queries, so
  // they and the first keys can be asked for ahead of the sequences' lengths. With shared keys,
  // where there are few waves, that saves a trip to memory (one sequence of 230: 7.3 -> 6.8 us);
  // without, the loads of all waves at once are what the first tile waits for, and keys that are
  // of no use add to them (64 of 3 to 200: 11.8 -> 12.8).
  PackedRow row;
  const bool early = SELF && SPLIT && p.right == 0;
  const int kearly = min(e * 32 + 32, p.Nq), kw = SPLIT ? w * KT : 0; // (this wave's first tile ends at kend - kw)
  const bool asked = early && kearly - kw > 0;
  if constexpr (SELF) {
    // The lengths come by LDS-DMA, ahead of the query rows: loads return in the order they were
    // asked for, but for a value in a register the compiler waits for every DMA.
    const int lo = packed_find(p, e);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      __builtin_amdgcn_global_load_lds((const void *)(p.cu_q + min(lo + lane + i, p.B)),
                                       (__attribute__((address_space(3))) void *)s_cu[w][i], 4, 0, 0);
    asm volatile("" ::: "memory");
    ask_q(min(e * 32 + ql, p.Nq - 1));
    if (asked) {
      issue_k(kearly - kw - KT);
      issue_v(kearly - kw - KT);
      vm_wait<KS + 2 * NDMA>();
    } else {
      vm_wait<KS>();
    }
    float begin = lds_read_b32<0>(lds_offset(s_cu[w][0]) + 4 * lane), end = lds_read_b32<0>(lds_offset(s_cu[w][1]) + 4 * lane);
    asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(begin), "+v"(end)::"memory");
    row = packed_row_self(p, e, lo, __float_as_int(begin), __float_as_int(end));
  } else {
    PackedSeq seq = {0, 0, 0, 0};
    const int qt = packed_tile(p, e, 32 >> lg, seq);
    if (qt < 0) return; // (every wave)
    const int i = (qt * 32 + ql) >> lg;
    row = {seq, min(i, seq.Sq - 1), i < seq.Sq};
    ask_q(row.seq.q0 + row.i);
  }
  const int qrow = row.seq.q0 + row.i;
  const KeyRange kr = packed_keys(p, row.i, row.seq.Sq, row.seq.Sk);
  const int klo = row.seq.k0 + kr.lo, khi = row.seq.k0 + kr.hi; // rows of k and v that the row sees
  const bool sees = row.real && kr.lo < kr.hi;
  const unsigned seeing = (unsigned)__ballot(sees);
  const int ra = seeing ? __builtin_ctz(seeing) : 0, rb = seeing ? 31 - __builtin_clz(seeing) : 0;
  const int kmin = __builtin_amdgcn_readlane(klo, ra), kmax = seeing ? __builtin_amdgcn_readlane(khi, rb) : kmin;
  // keys [all_lo, all_hi) are seen by every row that sees any
  const int all_lo = __builtin_amdgcn_readlane(klo, rb), all_hi = __builtin_amdgcn_readlane(khi, ra);
  const int kend = early ? kearly : kmax, k0 = kend - kw - KT; // (kmax <= kearly)
  const bool any = kmin < kmax && k0 + KT > kmin;
  row_lo = kmin, row_hi = max(kmax - 1, kmin);
  if (any && !asked) {
    issue_k(k0);
    issue_v(k0);
  }
  f32x16 o[NT];
#pragma unroll
  for (int tt = 0; tt < NT; ++tt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[tt][i] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;
  const float c2 = p.scale_log2;
  const unsigned kbase = lds_offset(ring);
  unsigned ko[KS], vo[NT];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) ko[ks] = kbase + (unsigned)((ql * CPR + ((ks * 2 + h) ^ (ql & (CPR - 1)))) * 16);
  // V operand addresses within a tile (attn_prefill_kernel explains the layout)
  const int grp = lane >> 4, a4 = lane & 3, c4 = (lane >> 2) & 3, kl = 4 * (grp >> 1) + c4;
#pragma unroll
  for (int tt = 0; tt < NT; ++tt) {
    const int d0 = tt * 32 + 16 * (grp & 1) + 4 * a4;
    vo[tt] = kbase + TU * 16 + kl * D * 2 + (((d0 >> 3) ^ vswz<D>(kl)) << 4) + ((d0 & 7) << 1);
  }
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks])); // here, not in the loop

  for (int kb = k0; any && kb + KT > kmin; kb -= SH * KT) {
    const bool more = kb - SH * KT + KT > kmin;
    vm_wait<NDMA>(); // this tile's K landed, its V may be in flight
    // S^T = K Q^T: eight fragments, read i is K step i (two blocks of 32 keys: step i / 2)
    V8 kr[4][2];
    static_for<8>([&](auto ii) {
      constexpr int i = decltype(ii)::value;
      kr[i / 2][i % 2] = lds_read_b128<(NB == 2 ? i % 2 : 0) * 32 * D * 2, V8>(ko[NB == 2 ? i / 2 : i]);
    });
    f32x16 s[NB];
#pragma unroll
    for (int st = 0; st < NB; ++st)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[st][i] = 0.f;
    static_for<4>([&](auto ii) {
      constexpr int i = decltype(ii)::value;
      lds_wait_tied<(3 - i) * 2>(kr[i]);
      if constexpr (i == 3) { // every K fragment is in registers
        asm volatile("" ::: "memory");
        if (more) issue_k(kb - SH * KT);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 2; ++j) s[j % NB] = mfma32x32<T>(kr[i][j], qf[NB == 2 ? i : 2 * i + j], s[j % NB]);
      __builtin_amdgcn_sched_barrier(0);
    });
    // online softmax, as attn_prefill_kernel
    if (kb < all_lo || kb + KT > all_hi) {
      const int jb = kb + h * 4;
      const int ca = max(klo - jb, 0), cb = min(khi - 1 - jb, KT - 1);
      const unsigned ninf = __float_as_uint(-INFINITY);
#pragma unroll
      for (int st = 0; st < NB; ++st) {
        const int l0 = max(ca - 32 * st, 0), h0 = min(cb - 32 * st, 31);
        const unsigned keep = l0 <= h0 ? ((2u << h0) - 1u) & ~((1u << l0) - 1u) : 0u;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const unsigned bm = (unsigned)__builtin_amdgcn_sbfe((int)keep, (i >> 2) * 8 + (i & 3), 1);
          s[st][i] = __uint_as_float((__float_as_uint(s[st][i]) & bm) | (ninf & ~bm));
        }
      }
    }
    float mx[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
#pragma unroll
    for (int st = 0; st < NB; ++st)
#pragma unroll
      for (int i = st == 0 ? 4 : 0; i < 16; ++i) mx[i & 3] = fmaxf(mx[i & 3], s[st][i]);
    float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
    mt = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
    const bool move = (mt - m_run) * c2 > 8.f;
    const float m_new = move ? mt : m_run;
    const float mc = m_new == -INFINITY ? 0.f : m_new * c2;
    const float alpha = move ? __builtin_amdgcn_exp2f(m_run * c2 - mc) : 1.f;
    float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int st = 0; st < NB; ++st)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[st][i], c2, kUp - mc));
        s[st][i] = x;
        ps[i & 3] += x;
      }
    l_run = l_run * alpha + ((ps[0] + ps[1]) + (ps[2] + ps[3]));
    m_run = m_new;
    if (__any(move)) {
#pragma unroll
      for (int tt = 0; tt < NT; ++tt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[tt][i] *= alpha;
    }
    // The one rounding of the weights, to the type of V, as attn_prefill_kernel's (l has them
    // unrounded): what a second product with the rest of them would keep is half the matrix work
    // again. Off the 64-bit form by 0.0019-0.0023 (bf16) and 0.00022-0.00027 (fp16) relative,
    // outputs rounded alone by 0.0016-0.0017 and 0.00019-0.00021.
    V8 pb[2 * NB];
#pragma unroll
    for (int c = 0; c < 2 * NB; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) pb[c][j] = from_f32<T>(s[c >> 1][(c & 1) * 8 + j]);
    // O^T += V^T P^T
    if (more) vm_wait<NDMA>(); // the next K may be in flight
    else vm_wait<0>();
    constexpr int R = 2 * NT, NC = 2 * NB;
    s16x4 vr[NC][R];
    static_for<NC>([&](auto cc) {
      constexpr int c = decltype(cc)::value;
#pragma unroll
      for (int tt = 0; tt < NT; ++tt) {
        vr[c][2 * tt] = lds_read_tr16<c * 32 * D>(vo[tt]);
        vr[c][2 * tt + 1] = lds_read_tr16<c * 32 * D + 16 * D>(vo[tt]);
      }
    });
    static_for<NC>([&](auto cc) {
      constexpr int c = decltype(cc)::value;
      lds_wait_tied<(NC - 1 - c) * R>(vr[c]);
      if constexpr (c == NC - 1) { // every V fragment is in registers
        asm volatile("" ::: "memory");
        if (more) issue_v(kb - SH * KT);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int tt = 0; tt < NT; ++tt) {
        const s16x8 r12 = __builtin_shufflevector(vr[c][2 * tt], vr[c][2 * tt + 1], 0, 1, 2, 3, 4, 5, 6, 7);
        o[tt] = mfma32x32<T>(__builtin_bit_cast(V8, r12), pb[c], o[tt]);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  }

  if (!any) vm_wait<0>(); // (asked for and not used: the slots are written to below)
  const float l = l_run + __shfl_xor(l_run, 32, kWave);
  // rows of k and v that the block's tiles had
  const int had_lo = max(kend - (kend - kmin + KT - 1) / KT * KT, 0), had_hi = min(kend, p.Nk);
  // values that are not finite and not seen (packed_row_again): the rows in `bad`, by `waves`
  auto again = [&](unsigned bad, int w0, int waves) {
    if (!packed_odd_values<T, D>(p, hk, had_lo, all_lo) && !packed_odd_values<T, D>(p, hk, all_hi, had_hi)) return;
    for (int n = 0; bad; bad &= bad - 1, ++n) {
      if (n % waves != w0) continue;
      const int l = __builtin_ctz(bad);
      packed_row_again<T, D>(p, __builtin_amdgcn_readlane(qrow, l), __builtin_amdgcn_readlane(klo, l),
                             __builtin_amdgcn_readlane(khi, l), hq + (l & heads), hk);
    }
  };
  if constexpr (!SPLIT) {
    // the rows through LDS, so that a store instruction writes whole rows
    const float inv = 1.f / l; // (rows whose scores are all -inf are NaN)
    float z = 0.f;
#pragma unroll
    for (int tt = 0; tt < NT; ++tt)
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {
        V4 pk;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          z = fmaf(o[tt][rg * 4 + i], 0.f, z);
          pk[i] = from_f32<T>(sees ? o[tt][rg * 4 + i] * inv : 0.f);
        }
        *reinterpret_cast<V4 *>(ring + ql * RBY + ((tt * 4 + rg) ^ (ql % CPR)) * 16 + h * 8) = pk;
      }
    T *const op = (T *)p.o + (int64_t)hq * p.o_sh;
    const unsigned reals = (unsigned)__ballot(row.real);
#pragma unroll
    for (int r = 0; r < 32 / ORPI; ++r) {
      const int n = r * ORPI + lane / CPR, c = lane % CPR;
      const V8 x = *reinterpret_cast<const V8 *>(ring + n * RBY + ((c ^ (n % CPR)) * 16));
      const int at = __shfl(qrow, n, kWave);
      if (reals >> n & 1) *reinterpret_cast<V8 *>(op + (int64_t)at * p.o_ss + (int64_t)(n & heads) * p.o_sh + c * 8) = x;
    }
    unsigned long long bad = __ballot(z != z && l == l && sees);
    if (bad) {
      vm_wait<0>(); // the rows above are written before
      again((unsigned)(bad | (bad >> 32)), 0, 1);
    }
  } else {
    if (tid == 0) s_bad = 0;
    __syncthreads(); // every wave is done with its slot
    float *const mo = reinterpret_cast<float *>(smem) + (w * 32 + ql) * LDO;
#pragma unroll
    for (int tt = 0; tt < NT; ++tt)
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {
        f32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = o[tt][rg * 4 + i];
        *reinterpret_cast<f32x4 *>(mo + tt * 32 + rg * 8 + h * 4) = x;
      }
    if (h == 0) s_m[w][ql] = m_run, s_l[w][ql] = l;
    __syncthreads();
    const unsigned reals = (unsigned)__ballot(row.real);
    for (int idx = tid; idx < 32 * CPR; idx += 64 * NW) { // (whole waves)
      const int n = idx / CPR, c = idx % CPR, at = __shfl(qrow, n, kWave);
      if (!(reals >> n & 1)) continue;
      float mx = -INFINITY;
#pragma unroll
      for (int g = 0; g < NW; ++g) mx = fmaxf(mx, s_m[g][n]);
      const float ms = mx == -INFINITY ? 0.f : mx;
      float ls = 0.f, v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
#pragma unroll
      for (int g = 0; g < NW; ++g) {
        const float a = __builtin_amdgcn_exp2f((s_m[g][n] - ms) * c2);
        ls += a * s_l[g][n];
        const float *x = reinterpret_cast<const float *>(smem) + (g * 32 + n) * LDO + c * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += a * x[i];
      }
      const bool sees = seeing >> n & 1;
      const float inv = 1.f / ls;
      float z = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) z = fmaf(v[i], 0.f, z), v[i] = sees ? v[i] * inv : 0.f;
      if (z != z && ls == ls && sees) atomicOr(&s_bad, 1u << n);
      store8((T *)p.o + (int64_t)at * p.o_ss + (int64_t)(hq + (n & heads)) * p.o_sh + c * 8, v);
    }
    __syncthreads(); // every row above is written, and what is odd known
    if (s_bad) again(s_bad, w, NW);
  }
}

// The query tiles of every sequence, those with the most key tiles first: a counting sort by
// one block. A wave loads 64 sequences at once and takes its share of them; a lane a tile.
constexpr int kPlanBins = 1024;
__device__ __forceinline__ int plan_bin(int tiles) { // falling, one by one up to 512, then by 64s
  return kPlanBins - 1 - (tiles < 512 ? tiles : 512 + min((tiles - 512) >> 6, 511));
}
__global__ __launch_bounds__(1024) void packed_plan_kernel(PackedArgs p, int QL, int32_t *__restrict__ plan, int room) {
  __shared__ int s_at[kPlanBins], s_sum[16];
  const int tid = threadIdx.x, lane = lane_id(), w = wave_id(), count = packed_count(p);
  s_at[tid] = 0;
  __syncthreads();
  auto each = [&](auto f) { // (sequence, tile, its bin)
    for (int c = 0; c < count; c += kWave) {
      PackedSeq mine = {0, 0, 0, 0};
      if (c + lane < count) mine = packed_seq(p, c + lane);
      for (int l = w; l < min(count - c, kWave); l += 16) {
        PackedSeq s;
        s.q0 = __builtin_amdgcn_readlane(mine.q0, l), s.Sq = __builtin_amdgcn_readlane(mine.Sq, l);
        s.k0 = __builtin_amdgcn_readlane(mine.k0, l), s.Sk = __builtin_amdgcn_readlane(mine.Sk, l);
        for (int t = lane; t * QL < s.Sq; t += kWave) {
          const KeyBand kb = key_band(t * QL, min(t * QL + QL, s.Sq) - 1, s.Sq, s.Sk, p.left, p.right, kKvTile);
          f(s, t, plan_bin(kb.t_end - kb.t_begin));
        }
      }
    }
  };
  each([&](const PackedSeq &, int, int bin) { atomicAdd(&s_at[bin], 1); });
  __syncthreads();
  const int n = s_at[tid];
  int sum = wave_scan(n);
  if (lane == kWave - 1) s_sum[w] = sum;
  __syncthreads();
  for (int i = 0; i < w; ++i) sum += s_sum[i];
  s_at[tid] = sum - n;
  if (tid == 1023) plan[0] = min(sum, room);
  __syncthreads();
  each([&](const PackedSeq &s, int t, int bin) {
    const int at = atomicAdd(&s_at[bin], 1); // (the order inside a bin changes no result)
    if (at < 0 || at >= room) return;         // (lengths that do not ascend)
    int32_t *it = plan + kPlanHead + at * kPlanItem;
    it[0] = s.q0, it[1] = t * QL, it[2] = s.Sq, it[3] = s.k0, it[4] = s.Sk;
  });
}

// How a call is cut: the kernel (share: packed_wave_kernel's waves a row, 0: attn_prefill_kernel),
// query heads (packed_wave_kernel: their logarithm too) and queries of a tile, the most tiles
// there can be.
struct PackedPlan {
  bool tiles;
  int share, lg, hpb, QL;
  int64_t most;
  bool plan;
};
// Estimated times in us, of sequences of the batch's mean lengths (no other is known here),
// from measurements of 1 to 256 sequences of 17 to 8000 tokens (bf16, 16 / 8 heads of 128, the
// middle line for heads of 64):
//  * packed_wave_kernel: 2.5, 4.5 for each 2048 waves, and the longest row's tiles, 0.8 each,
//    or all waves' tiles at 1.1 ns (16 KB each from the L2s); with its keys shared by four
//    waves 4, 4.2 for each 512 blocks, and the row's share of tiles or 0.93 ns.
//  * attn_prefill_kernel: 7 with its plan, and 4.5 and 2.0 (1.2) a tile of 64 keys for all tiles
//    over the CUs, or the longest tile alone, 4.5 and 1.6 (1.2).
// Measured, e.g.: one sequence of 230 6.8 (17.8 on the other kernel), of 1000 17 (38), 64 of 3 to
// 200 12 (32; fp16, 16 / 16 heads of 64), 16 of 200 17 (21); and back, 16 of 1000 139 (107), eight
// of 501 to 4001 278 (188: 770 TFLOP/s, 5 us of it the plan's launch).
// What the mean does not show: long and short sequences in one batch take the kernel that suits
// their mean (eight of 2000 171 us, with 200 of 8, 7 on their own, 233), and one part of a prompt
// of 512 behind 4000 keys beside 31 single tokens there, 59 and 44 on their own, 230: the tokens'
// heads do not share tiles. Keys are not split over blocks: 33 behind 8000 keys 53-60 us, 32
// behind 30000 209, 6.5 and 24 at the copy's rate.
static PackedPlan packed_plan(int64_t B, int64_t Nq, int64_t Nk, int64_t Hq, int64_t Hkv, int64_t D, int left, int right,
                              bool self) {
  PackedPlan pl = {};
  if (D != 64 && D != 128) return pl;
  pl.tiles = true;
  const double cus = device_cu_count() > 0 ? device_cu_count() : 256, kt = D == 128 ? 32 : 64;
  auto most = [&](int64_t QL) { return self && QL == 32 ? (Nq + 31) / 32 : Nq / QL + (B + 2 < Nq ? B + 2 : Nq); };
  const double n = B > 0 ? B : 1, lq = Nq / n, lk = Nk / n;
  // keys that the last query sees, and that one does on the average
  double longest = lk, mean = right >= 0 && lq <= lk ? lk - lq / 2 : lk;
  if (left >= 0 && right >= 0 && left + right + 33.0 < longest) longest = left + right + 33.0;
  if (mean > longest) mean = longest;
  // few queries a sequence: the heads of a group fill the tile, which reads their keys once (17
  // sequences of one query behind 2410 keys, 16 / 2 heads, 61 -> 23 us; 11 of 4 behind 3865, 32 / 4
  // heads of 64, 57 -> 22; 32 of 16 behind 2000, 16 / 8 heads, 80 -> 50)
  int lg = 0;
  while (!self && lg < 5 && (Hq / Hkv) % (2 << lg) == 0 && lq * (2 << lg) <= 32) ++lg;
  const double items = (double)most(32 >> lg) * (Hq >> lg), work = items * (mean / kt + 0.5), chain = longest / kt + 1;
  auto larger = [](double a, double b) { return a > b ? a : b; };
  const double alone = 2.5 + 4.5 * larger(1, items / (8 * cus)) + larger(0.8 * chain, 1.1e-3 * work);
  double best = alone;
  pl.share = 1;
  const double shared = 4 + 4.2 * larger(1, items / (2 * cus)) + larger(0.8 * chain / 4 + 1, 0.93e-3 * work);
  if (shared < best) best = shared, pl.share = 4;
  const int64_t G = Hq / Hkv;
  const int hpb = G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1, QL = kPrefillWaves / hpb * 32;
  const double each = D == 128 ? 2.0 : 1.2, last = D == 128 ? 1.6 : 1.2;
  const double whole = 7 + larger((double)most(QL) * (Hq / hpb) / cus * (4.5 + each * (mean / 64 + 1)), 4.5 + last * (longest / 64 + 1));
  // (a grid has fewer than 2^32 threads)
  if (whole < best || most(32 >> lg) * (pl.share == 1 ? ((Hq >> lg) + 3) / 4 : Hq >> lg) > 0xffffff) pl.share = 0;
  pl.lg = lg, pl.hpb = pl.share ? 1 << lg : hpb, pl.QL = pl.share ? 32 >> lg : QL;
  pl.most = most(pl.QL);
  // up to two tiles a CU a block each, from the last to the first, and no list of them (its
  // launch: six turns behind 2500 tokens 46.9 -> 43.0 us; four prompts of 2000, 2.06 tiles a
  // CU, 90.7 with the list, 118 without)
  pl.plan = !pl.share && pl.most * (Hq / hpb) > 2 * cus;
  return pl;
}

} // namespace tpp

using namespace tpp;

// A window that reaches past every key is none (and query + window stays below 2^31).
static int packed_window(int x, int64_t Nq, int64_t Nk) { return x < 0 || x >= Nq + Nk ? -1 : x; }

extern "C" size_t tpp_attn_packed_workspace_size(int64_t B, int64_t Nq, int64_t Nk, int64_t Hq, int64_t Hkv, int64_t D,
                                                 int causal, int window_left, int window_right, int self) {
  if (B < 0 || Nq <= 0 || Nk < 0 || Hkv <= 0 || Hq <= 0) return 0;
  const PackedPlan pl = packed_plan(B, Nq, Nk, Hq, Hkv, D, packed_window(window_left, Nq, Nk),
                                    causal ? 0 : packed_window(window_right, Nq, Nk), self != 0);
  return pl.plan ? (size_t)(kPlanHead + pl.most * kPlanItem) * sizeof(int32_t) : 0;
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
  if (D > 256 || Hq > 65535 || B > (1 << 20) || Nq >= (1 << 26) || Nk > (1 << 29))
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
  a.scale_log2 = sc * kLog2e;
  a.left = packed_window(window_left, Nq, Nk), a.right = causal ? 0 : packed_window(window_right, Nq, Nk);
  a.fill = fill;
  hipStream_t st = as_stream(stream);
  // the matrix-core kernels: whole 16-byte rows, a tile's rows by 32-bit byte offsets
  uint64_t low = (uint64_t)(uintptr_t)q | (uint64_t)(uintptr_t)k | (uint64_t)(uintptr_t)v | (uint64_t)(uintptr_t)o;
  for (const int64_t x : {a.q_ss, a.q_sh, a.k_ss, a.k_sh, a.v_ss, a.v_sh, a.o_ss, a.o_sh}) low |= (uint64_t)(x * 2);
  const PackedPlan pl = packed_plan(B, Nq, Nk, Hq, Hkv, D, a.left, a.right, !cu_k);
  const bool fits = !(low & 15) && a.k_ss >= 0 && a.v_ss >= 0 && kKvTile * a.k_ss * 2 < (1LL << 31) &&
                    kKvTile * a.v_ss * 2 < (1LL << 31) && pl.most * Hq < (1LL << 31);
  if (!pl.tiles || !fits)
    return TPP_DISPATCH_HALF(dtype, [&] {
      packed_generic_kernel<T><<<dim3((unsigned)Nq, (unsigned)Hq), dim3(64), 0, st>>>(a, (int)D);
      return check_launch(name);
    });
  // packed_wave_kernel without shared keys: blocks of four heads
  const int nh = pl.share == 1 ? ((int)Hq / pl.hpb + 3) / 4 : (int)Hq / pl.hpb;
  const int64_t items = pl.most * nh;
  if (pl.plan) {
    if (!workspace || !aligned16(workspace) ||
        ws_bytes < tpp_attn_packed_workspace_size(B, Nq, Nk, Hq, Hkv, D, causal, window_left, window_right, !cu_k))
      return set_error(TPP_E_WORKSPACE, "%s: workspace missing, unaligned or too small", name);
    a.plan = (const int32_t *)workspace;
    packed_plan_kernel<<<dim3(1), dim3(1024), 0, st>>>(a, pl.QL, (int32_t *)workspace, (int)pl.most);
  }
  return TPP_DISPATCH_HALF(dtype, [&] {
    auto go = [&](auto dd) {
      constexpr int DD = decltype(dd)::value;
      const dim3 grid((unsigned)items);
      if (pl.share == 1 && !cu_k) packed_wave_kernel<T, DD, 1, true><<<grid, dim3(256), 0, st>>>(a, nh, pl.lg);
      else if (pl.share == 1) packed_wave_kernel<T, DD, 1, false><<<grid, dim3(256), 0, st>>>(a, nh, pl.lg);
      else if (pl.share && !cu_k) packed_wave_kernel<T, DD, 4, true><<<grid, dim3(256), 0, st>>>(a, nh, pl.lg);
      else if (pl.share) packed_wave_kernel<T, DD, 4, false><<<grid, dim3(256), 0, st>>>(a, nh, pl.lg);
      else {
        const int cus = device_cu_count() > 0 ? device_cu_count() : 256;
        attn_prefill_kernel<T, DD, kPrefillQG, kPrefillWaves>
            <<<dim3((unsigned)(!pl.plan || items < cus ? items : cus)), dim3(64 * kPrefillWaves), 0, st>>>(a, pl.hpb);
      }
    };
    if (D == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 64>{});
    return check_launch(name);
  });
}
