// Prefill attention on the matrix cores: the kernels of attention.hip, for a batch of one
// length, of which packed_attention.hip takes attn_prefill_kernel for sequences of different
// lengths packed one behind the other. attention.hip's head explains the layouts.
#pragma once
#include "attn_row.hpp"

namespace tpp {

struct AttnArgs {
  static constexpr bool kPacked = false;
  const void *q, *k, *v;
  void *o;
  int64_t q_sb, q_ss, q_sh;
  int64_t k_sb, k_ss, k_sh;
  int64_t v_sb, v_ss, v_sh;
  int64_t o_sb, o_ss, o_sh;
  int B, Sq, Sk, Hq, Hkv;
  float scale_log2; // softmax scale * log2(e)
  int left, right;  // window, -1 = unbounded; causal => right = 0
};

// A packed batch: sequence b has rows cu_q[b] .. cu_q[b + 1] - 1 of q and o, and cu_k[b] ..
// cu_k[b + 1] - 1 of k and v; no batch strides, and Sq and Sk are each sequence's own.
struct PackedArgs : AttnArgs {
  static constexpr bool kPacked = true;
  const int32_t *cu_q, *cu_k; // [B + 1]
  const int32_t *plan;        // attn_prefill_kernel's query tiles (packed_plan_kernel); null: a block a tile
  int Nq, Nk;
  int fill; // rows of no sequence become 0 (else they stay as they were)
};

// Rows of sequence b. What is given is cut to the tensors, so that no read or write leaves
// them. Sequences B and B + 1 are the rows behind the last and ahead of the first: they have
// no keys.
struct PackedSeq {
  int q0, Sq, k0, Sk;
};
__device__ __forceinline__ PackedSeq packed_seq(const PackedArgs &p, int b) {
  PackedSeq s = {0, 0, 0, 0};
  const int qa = b > p.B ? 0 : min(max(p.cu_q[b], 0), p.Nq);
  const int qe = b < p.B ? p.cu_q[b + 1] : b == p.B ? p.Nq : p.cu_q[0];
  s.q0 = qa, s.Sq = min(max(qe, qa), p.Nq) - qa;
  if (b < p.B) {
    s.k0 = min(max(p.cu_k[b], 0), p.Nk);
    s.Sk = min(max(p.cu_k[b + 1], s.k0), p.Nk) - s.k0;
  }
  return s;
}
// Sequences with rows to write.
__device__ __forceinline__ int packed_count(const PackedArgs &p) { return p.fill ? p.B + 2 : p.B; }

// The sequence and the tile in it of query tile `t`, counted over the batch in tiles of QL
// queries; -1 past the last. By every wave, 256 sequences' lengths in flight at once.
__device__ __forceinline__ int packed_tile(const PackedArgs &p, int t, int QL, PackedSeq &out) {
  constexpr int U = 4;
  const int lane = lane_id(), count = packed_count(p);
  for (int c0 = 0, before = 0; c0 < count; c0 += U * kWave) {
    PackedSeq s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s[u] = {0, 0, 0, 0};
      if (c0 + u * kWave + lane < count) s[u] = packed_seq(p, c0 + u * kWave + lane);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int n = (s[u].Sq + QL - 1) / QL;
      const int sum = wave_scan(n); // tiles up to this lane's sequence
      const unsigned long long hit = __ballot(before + sum > t);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        out.q0 = __builtin_amdgcn_readlane(s[u].q0, l), out.Sq = __builtin_amdgcn_readlane(s[u].Sq, l);
        out.k0 = __builtin_amdgcn_readlane(s[u].k0, l), out.Sk = __builtin_amdgcn_readlane(s[u].Sk, l);
        const int own = __builtin_amdgcn_readlane(n, l), at = t - before - (__builtin_amdgcn_readlane(sum, l) - own);
        return at >= 0 && at < own ? at : -1; // (lengths that do not ascend may add up to anything)
      }
      before += __builtin_amdgcn_readlane(sum, kWave - 1);
      if (c0 + (u + 1) * kWave >= count) return -1;
    }
  }
  return -1;
}

// Keys lo .. hi - 1 that query i of a sequence sees (none: lo >= hi).
struct KeyRange {
  int lo, hi;
};
__device__ __forceinline__ KeyRange packed_keys(const PackedArgs &p, int i, int Sq, int Sk) {
  const int at = i + Sk - Sq;
  return {p.left >= 0 ? max(at - p.left, 0) : 0, p.right >= 0 ? min(at + p.right + 1, Sk) : Sk};
}

// exp2 of the weights' reference: P is stored times 2^this. Above bfloat16's weights of 1 at
// most, times 2^8 before the reference moves, sums of finite values near the type's end would
// be infinite; fp16's weights want the room above them, not to lose those below 2^-24.
template <typename T, bool PACKED> constexpr float kWeightUp = !PACKED ? 0.f : __is_same(T, bf16) ? -20.f : 7.f;

// Row qrow of q and o again, by one wave from its definition over rows klo .. khi - 1 of k and
// v: an infinity or NaN among the values that a row does not see, times its weight of 0, is a
// NaN in the sums of a tile.
template <typename T, int D>
__device__ __forceinline__ void packed_row_again(const PackedArgs &p, int qrow, int klo, int khi, int hq, int hk) {
  AttnRow r;
  attn_row<T>(r, (const T *)p.q + (int64_t)qrow * p.q_ss + hq * p.q_sh, D, klo, khi, p.scale_log2,
              [&](int j, const T *&k, const T *&v) {
                k = (const T *)p.k + (int64_t)j * p.k_ss + hk * p.k_sh;
                v = (const T *)p.v + (int64_t)j * p.v_ss + hk * p.v_sh;
                return true;
              });
  T *op = (T *)p.o + (int64_t)qrow * p.o_ss + hq * p.o_sh;
#pragma unroll
  for (int c = 0; c < D / 64; ++c) op[c * 64 + lane_id()] = from_f32<T>(r.out(c));
}
// Whether a value that is not finite stands in rows [a, b) of v (one wave).
template <typename T, int D>
__device__ __forceinline__ bool packed_odd_values(const PackedArgs &p, int hk, int a, int b) {
  bool odd = false;
  for (int j = a; j < b; ++j)
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const float x = to_f32(((const T *)p.v)[(int64_t)j * p.v_ss + hk * p.v_sh + c * 64 + lane_id()]);
      odd = odd || !(fabsf(x) < INFINITY);
    }
  return __any(odd);
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kKvTile = 64;
// 32-query groups per prefill wave (each K / V^T fragment read from LDS feeds
// every group's products). Two groups need more than the 512 VGPRs of a wave
// at D = 128 and spill, so one group is used.
constexpr int kPrefillQG = 1;
// waves per prefill block: 8 = two per SIMD, so one wave's softmax (VALU)
// overlaps the other's MFMAs
constexpr int kPrefillWaves = 8;

template <typename T>
__device__ __forceinline__ f32x16 mfma32x32(typename VecT<T>::v8 a, typename VecT<T>::v8 b,
                                            f32x16 c) {
  if constexpr (__is_same(T, bf16))
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// V tiles are stored row-major like K ([key][16-byte unit]) and read as
// MFMA operands with ds_read_b64_tr_b16, whose 16-lane groups return lane
// 4a+b the b-th 16-bit element of the words lanes a, a+4, a+8, a+12 point at:
// pointing lane a'+4c' at V[k0 + c'][d0 + 4a'] gives lane l of the group
// V[k0 + 0..3][d0 + l]. Unit u of key row r is stored at u ^ vswz(r): the
// 32 lanes one read cycle serves (4 keys x 32 columns) then hit distinct
// banks (D = 128: 256-byte rows, XOR 4*(r%4); D = 64: 128-byte rows, two
// per bank row, XOR 4*((r/2)%2)).
template <int D> __device__ __forceinline__ int vswz(int r) {
  if constexpr (D == 128) return 4 * (r & 3);
  else return 4 * ((r >> 1) & 1);
}

// Tiles [t_begin, t_end) of `kt` keys that queries q0 .. q_last see (causal
// and window bounds are aligned bottom-right: query i sits at key i + Sk - Sq).
struct KeyBand {
  int t_begin, t_end;
};
__host__ __device__ inline KeyBand key_band(int q0, int q_last, int Sq, int Sk, int left, int right,
                                            int kt) {
  const int off = Sk - Sq;
  int hi = Sk, lo = 0;
  if (right >= 0) {
    const int64_t lim = (int64_t)q_last + off + right + 1;
    hi = lim < hi ? (int)lim : hi;
  }
  if (left >= 0) {
    const int64_t lim = (int64_t)q0 + off - left;
    lo = lim > 0 ? (int)lim : 0;
  }
  const int tb = lo / kt;
  return {tb, hi > lo ? (hi + kt - 1) / kt : tb};
}

// Key-split prefill: the tiles of a query tile's band that chunk `split`
// takes (the last one to the band's end, whatever the plan expected), and the
// chunks of the band that have a tile. The kernel and the merge both go by
// these two.
__host__ __device__ inline KeyBand key_chunk(const KeyBand &kb, int split, int ct, int nsmax) {
  const int t0 = kb.t_begin + split * ct;
  return {t0, split == nsmax - 1 || kb.t_end < t0 + ct ? kb.t_end : t0 + ct};
}
__host__ __device__ inline int key_chunks(const KeyBand &kb, int ct, int nsmax) {
  const int n = (kb.t_end - kb.t_begin + ct - 1) / ct;
  return n < nsmax ? n : nsmax; // the workspace has nsmax slots per row
}

// K / V ring slots of the prefill kernel: tile t in slot (t - t_begin) % 3
constexpr int kPrefillSlots = 3;
template <typename T, int D> struct PrefillSmem {
  typedef typename VecT<T>::v8 V8;
  V8 k[kPrefillSlots][kKvTile * D / 8];  // [key][chunk ^ (key % (D/8))]
  V8 v[kPrefillSlots][kKvTile * D / 8];  // [key][chunk ^ vswz(key)]
};

// Packed batches: `plan` holds the number of query tiles, then for each the sequence's first
// row of q, the tile's first query, the sequence's Sq, its first row of k and its Sk.
constexpr int kPlanHead = 8, kPlanItem = 8;

template <typename T, int D, int QG, int NW, typename A>
__global__ __launch_bounds__(64 * NW) void attn_prefill_kernel(A p, int hpb) {
  constexpr bool PACKED = A::kPacked;
  typedef typename VecT<T>::v8 V8;
  constexpr int CPR = D / 8; // 16-byte chunks per row
  constexpr int NT = D / 32; // 32-row MFMA tiles along D
  __shared__ PrefillSmem<T, D> sm;

  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int h = lane >> 5, ql = lane & 31;
  const int G = p.Hq / p.Hkv;
  const int wph = NW / hpb;  // waves per head
  const int qt_len = wph * 32 * QG;
  int Sq = p.Sq, Sk = p.Sk; // packed: of the item's sequence (setup)
  int nqt = (Sq + qt_len - 1) / qt_len;
  const int nhg = p.Hq / hpb;
  int npair = p.B * nhg;
  PackedSeq own = {0, 0, 0, 0}; // packed, no plan: the block's one tile
  int own_q0 = 0;
  if constexpr (PACKED) {
    npair = nhg; // one list of query tiles for every head
    if (p.plan) {
      nqt = __builtin_amdgcn_readfirstlane(p.plan[0]);
    } else {
      own_q0 = packed_tile(p, (gridDim.x - 1 - blockIdx.x) / nhg, qt_len, own) * qt_len; // (late tiles first)
      if (own_q0 < 0) return;
      nqt = gridDim.x / nhg;
    }
  }
  const int nitems = npair * nqt;
  int off = Sk - Sq;

  // Work items (query tile qt, batch x head-group pair) in a fixed order,
  // heavy (late) query tiles first; the block loops over its share of them.
  // When the pairs split evenly over the 8 XCDs (workgroups are dealt to
  // them round-robin, XCD = blockIdx % 8), an XCD runs only its own pairs,
  // so the K / V tiles its blocks share stay in its L2, and each of its S
  // blocks takes the XCD's items in boustrophedon order (rounds alternate
  // direction), which evens out the heavy and light tiles per block.
  const bool xcd_split = npair % 8 == 0 && gridDim.x % 8 == 0 && !(PACKED && gridDim.x == (unsigned)nitems);
  auto next_item = [&](int &k, int &qt, int &rest) -> bool {
    if (xcd_split) {
      const int S = gridDim.x / 8, slot = blockIdx.x / 8, per = npair / 8, ni = nitems / 8;
      for (;; ++k) {
        if (k * S >= ni) return false;
        const int j = (k & 1) ? (k + 1) * S - 1 - slot : k * S + slot;
        if (j >= ni) continue;
        rest = (blockIdx.x % 8) * per + j % per;
        qt = PACKED ? j / per : nqt - 1 - j / per;
        return true;
      }
    }
    const int it = blockIdx.x + k * gridDim.x;
    if (it >= nitems) return false;
    qt = PACKED ? it / npair : nqt - 1 - it / npair;
    rest = it % npair;
    return true;
  };
  // the item's state (set by setup)
  int b, hq, hk, q0, q_last, qw, t_begin, t_end;
  const T *qp, *kp, *vp;
  int seq_q = 0, seq_k = 0; // packed: the sequence's first rows
  auto setup = [&](int qt, int rest) {
    b = rest / nhg;
    const int hg = rest % nhg;
    hq = hg * hpb + w / wph;
    hk = (hg * hpb) / G;
    q0 = qt * qt_len;
    if constexpr (PACKED) {
      if (p.plan) {
        const int32_t *it = p.plan + kPlanHead + qt * kPlanItem;
        int x[5];
#pragma unroll
        for (int i = 0; i < 5; ++i) x[i] = __builtin_amdgcn_readfirstlane(it[i]);
        seq_q = x[0], q0 = x[1], Sq = x[2], seq_k = x[3], Sk = x[4];
      } else {
        seq_q = own.q0, q0 = own_q0, Sq = own.Sq, seq_k = own.k0, Sk = own.Sk;
      }
      off = Sk - Sq;
   }
    q_last = (q0 + qt_len < Sq ? q0 + qt_len : Sq) - 1;
    qw = q0 + (w % wph) * 32 * QG; // first query of this wave
    // key band of the whole item
    int hi = Sk, lo = 0;
    if (p.right >= 0) {
      const int lim = q_last + off + p.right + 1;
      hi = lim < hi ? lim : hi;
    }
    if (p.left >= 0) {
      const int lim = q0 + off - p.left;
      lo = lim > 0 ? lim : 0;
    }
    t_begin = lo / kKvTile;
    t_end = hi > lo ? (hi + kKvTile - 1) / kKvTile : t_begin;
    qp = (const T *)p.q + (int64_t)b * p.q_sb + (int64_t)hq * p.q_sh;
    kp = (const T *)p.k + (int64_t)b * p.k_sb + (int64_t)hk * p.k_sh;
    vp = (const T *)p.v + (int64_t)b * p.v_sb + (int64_t)hk * p.v_sh;
    if constexpr (PACKED) {
      qp += (int64_t)seq_q * p.q_ss;
      kp += (int64_t)seq_k * p.k_ss;
      vp += (int64_t)seq_k * p.v_ss;
    }
  };

  V8 zero;
#pragma unroll
  for (int i = 0; i < 8; ++i) zero[i] = (T)0.0f;

  // QG groups of 32 queries per wave share every K / V fragment read from LDS
  V8 qf[QG][D / 16];
  auto load_q = [&] {
#pragma unroll
    for (int g = 0; g < QG; ++g) {
      const int qi = qw + g * 32 + ql;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
        qf[g][ks] = qi < Sq
                        ? *reinterpret_cast<const V8 *>(qp + (int64_t)qi * p.q_ss + ks * 16 + h * 8)
                        : zero;
    }
  };
  int kitem = 0, qt0, rest0;
  if (!next_item(kitem, qt0, rest0)) return;
  setup(qt0, rest0);
  load_q();

  // The block's waves form two groups of NW/2 (waves w and w + NW/2 share a
  // SIMD). The leading group runs half an iteration ahead of the trailing
  // one, so on every SIMD one wave's MFMA phase (PV of tile t-1, then QK^T of
  // tile t) overlaps the other wave's softmax phase (VALU). Each iteration
  // has two workgroup barriers, one per phase change; the trailing group
  // passes one barrier before its first iteration, the leading group one
  // after its last.
  const bool lead = __builtin_amdgcn_readfirstlane(w) < NW / 2; // wave-uniform
  constexpr int NWL = NW / 2;

  // K and V tiles go HBM/L2 -> LDS by LDS-DMA (no staging registers): the
  // leading group fetches the K tiles, the trailing group the V tiles.
  // Instruction i of a group's wave wu fills 64 slots = 64/CPR keys; lane l
  // fetches the chunk that lands in its slot. The address is a wave-uniform
  // tile base plus a per-lane 32-bit byte offset fixed for the whole kernel
  // (the launch checks 64 rows fit in 2^31 bytes). Keys past Sk are clamped
  // to Sk-1 on the last tile (finite data; those scores are masked, so their
  // P is 0).
  constexpr int KPI = 64 / CPR;                 // keys per DMA instruction
  constexpr int KDMA = kKvTile / KPI / NWL;     // DMA instructions per wave per tile
  constexpr int NDMA = KDMA;                    // ... per wave per iteration
  const int wu = __builtin_amdgcn_readfirstlane(w) % NWL; // wave index within its group
  const int dkey = lane / CPR, dslot = lane % CPR;
  const int64_t dss = lead ? p.k_ss : p.v_ss; // row stride of this wave's tiles
  // Offsets of full tiles, and of the last tile when Sk is not a multiple of
  // the tile: its keys past Sk read key Sk-1 (the clamp computed here once,
  // not per tile)
  const int kb_last = ((Sk - 1) / kKvTile) * kKvTile;
  unsigned doff[KDMA], doffl[KDMA];
#pragma unroll
  for (int i = 0; i < KDMA; ++i) {
    const int key = (i * NWL + wu) * KPI + dkey;
    const int kk = min(key, Sk - 1 - kb_last);
    const int ch = lead ? dslot ^ (key & (CPR - 1)) : dslot ^ vswz<D>(key); // K / V swizzle
    doff[i] = (unsigned)((key * dss + ch * 8) * (int64_t)sizeof(T));
    doffl[i] = (unsigned)((kk * dss + ch * 8) * (int64_t)sizeof(T));
  }
  // DMA instruction i (< KDMA) of this wave's share of tile t (K tile for the
  // leading group, V tile for the trailing group) into ring slot `slot`
  auto dma = [&](int i, int t, int slot) {
    const int kb = t * kKvTile;
    const char *tb = (const char *)((lead ? kp : vp) + (int64_t)kb * dss);
    V8 *dst = lead ? sm.k[slot] : sm.v[slot];
    const int key0 = (i * NWL + wu) * KPI;
    unsigned o;
    if constexpr (PACKED) // the last tile is the item's own: rows past it less
      o = doff[i] - (unsigned)(max(key0 + dkey - (Sk - 1 - kb), 0) * (int)(dss * (int64_t)sizeof(T)));
    else
      o = kb + kKvTile > Sk ? doffl[i] : doff[i];
    __builtin_amdgcn_global_load_lds((const void *)(tb + o),
                                     (__attribute__((address_space(3))) void *)&dst[key0 * CPR],
                                     16, 0, 0);
  };

  f32x16 o[QG][NT];                // reset at the start of every item
  float m_run[QG], l_run[QG];

  f32x16 s[QG][2];
  V8 pb[QG][4];

  // S^T = K Q^T for the K tile in slot buf. The K fragments of step ks + 2
  // are requested before the MFMAs of step ks (scheduling barriers keep the
  // compiler from pulling the reads back next to their use), so LDS latency
  // hides behind the matrix work. The reads are inline asm with explicit
  // waits, like the V reads (from plain LDS loads the compiler waited for
  // all outstanding reads every third step).
  auto qk = [&](int buf) {
    const unsigned kbase = (unsigned)(uintptr_t)(const __attribute__((address_space(3))) char *)&sm.k[buf][0];
    // step ks, key row st * 32 + ql: the st = 1 row is 32 rows (32 * D * 2
    // bytes) after the st = 0 row, with the same swizzle
    auto kfrag = [&](int ks, V8 (&dst)[2]) {
      const unsigned a = kbase + (unsigned)((ql * CPR + ((ks * 2 + h) ^ (ql & (CPR - 1)))) * 16);
      dst[0] = lds_read_b128<0, V8>(a);
      dst[1] = lds_read_b128<32 * D * 2, V8>(a);
    };
    constexpr int KS = D / 16;
    V8 kr[3][2];
#pragma unroll
    for (int g = 0; g < QG; ++g)
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[g][st][r] = 0.f;
    kfrag(0, kr[0]);
    kfrag(1, kr[1]);
    static_for<KS>([&](auto kk) {
      constexpr int ks = decltype(kk)::value;
      if constexpr (ks + 2 < KS) kfrag(ks + 2, kr[(ks + 2) % 3]);
      // the reads of steps ks + 1, ks + 2 stay in flight
      lds_wait_tied<(ks + 2 < KS ? 2 : KS - 1 - ks) * 2>(kr[ks % 3]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int g = 0; g < QG; ++g) s[g][st] = mfma32x32<T>(kr[ks % 3][st], qf[g][ks], s[g][st]);
      __builtin_amdgcn_sched_barrier(0);
    });
  };

  // Online softmax on raw scores of tile t: the running max m is kept
  // unscaled and exp2(scale*log2e*(s - m)) is one FMA + v_exp_f32 per score
  // (scale > 0 preserves the max). Masking only on band edges.
  // issue(j) is called at evenly spaced points of the exponentials with
  // j = 0 .. NDMA-1 (the waves put their DMA instructions there: a burst of
  // them would stall issue on the vector-memory queue)
  auto softmax = [&](int t, auto &&issue) {
    const int kb = t * kKvTile;
    const bool edge = (p.right >= 0 && kb + kKvTile - 1 > q0 + off + p.right) ||
                      (p.left >= 0 && kb < q_last + off - p.left) || (kb + kKvTile > Sk);
    const float c2 = p.scale_log2;
    constexpr float kUp = kWeightUp<T, PACKED>;
#pragma unroll
    for (int g = 0; g < QG; ++g) {
      const int qi = qw + g * 32 + ql;
      float mt = -INFINITY;
      if (edge) {
        // score register (st, r) holds key kb + 4h + c, c = 32st + 8(r/4) + r%4;
        // it is kept iff lo <= key <= hi, i.e. c in [lo - jb, hi - jb] with
        // jb = kb + 4h. Per lane one 32-bit mask per st holds the kept c's;
        // each score then costs a bit extract (0 or -1) and a bit select,
        // with no VCC round trip
        const int qpos = qi + off;
        int hi = Sk - 1;
        if (p.right >= 0) hi = min(hi, qpos + p.right);
        const int lo = p.left >= 0 ? max(qpos - p.left, 0) : 0;
        const int jb = kb + h * 4;
        const int ca = max(lo - jb, 0), cb = min(hi - jb, 63); // kept c: [ca, cb] (empty if ca > cb)
        const unsigned ninf = __float_as_uint(-INFINITY);
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          const int l0 = max(ca - 32 * st, 0), h0 = min(cb - 32 * st, 31);
          const unsigned keep = l0 <= h0 ? ((2u << h0) - 1u) & ~((1u << l0) - 1u) : 0u;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const unsigned bm = (unsigned)__builtin_amdgcn_sbfe((int)keep, (r >> 2) * 8 + (r & 3), 1);
            s[g][st][r] = __uint_as_float((__float_as_uint(s[g][st][r]) & bm) | (ninf & ~bm));
          }
        }
      }
      // max and sum as trees (a 32-long dependent chain of VALU ops costs
      // its full latency per step); the max as chains of three for v_max3
      auto max3 = [](float a, float b, float c) { return fmaxf(fmaxf(a, b), c); };
      float m1[11];
#pragma unroll
      for (int i = 0; i < 10; ++i) {
        const int a = 3 * i, b = 3 * i + 1, c = 3 * i + 2;
        m1[i] = max3(s[g][a >> 4][a & 15], s[g][b >> 4][b & 15], s[g][c >> 4][c & 15]);
      }
      m1[10] = fmaxf(s[g][1][14], s[g][1][15]);
      const float m2a = max3(m1[0], m1[1], m1[2]), m2b = max3(m1[3], m1[4], m1[5]);
      const float m2c = max3(m1[6], m1[7], m1[8]), m2d = fmaxf(m1[9], m1[10]);
      mt = fmaxf(max3(m2a, m2b, m2c), m2d);
      {
        // the other half of the wave holds the other 4-key groups
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mt), __float_as_uint(mt),
                                                         false, false);
        mt = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
      }
      // lazy rescale: the reference max m_run only moves when the tile max
      // exceeds it by more than 8 in the exp2 domain (or on the first finite
      // tile), so P <= 2^8 and O, l keep fp32 headroom; O / l is unchanged by
      // the choice of m_run, and the O rescale then runs on few tiles
      const bool move = (mt - m_run[g]) * c2 > 8.f; // false for NaN (both -inf)
      const float m_new = move ? mt : m_run[g];
      const float mc = m_new == -INFINITY ? 0.f : m_new * c2;
      const float alpha = move ? __builtin_amdgcn_exp2f(m_run[g] * c2 - mc) : 1.f;
      float ps[8];
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          constexpr int kStride = 32 / NDMA;
          if (g == 0 && (st * 16 + r) % kStride == 0) issue((st * 16 + r) / kStride);
          const float e = __builtin_amdgcn_exp2f(fmaf(s[g][st][r], c2, PACKED ? kUp - mc : -mc));
          s[g][st][r] = e;
          // the first term of each partial sum starts it (0 + e == e)
          ps[r & 7] = (st == 0 && r < 8) ? e : ps[r & 7] + e;
        }
#pragma unroll
      for (int n = 4; n >= 1; n >>= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) ps[i] += ps[i + n];
      l_run[g] = l_run[g] * alpha + ps[0];
      m_run[g] = m_new;
      if (__any(move)) {
#pragma unroll
        for (int tt = 0; tt < NT; ++tt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[g][tt][r] *= alpha;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) pb[g][c][j] = from_f32<T>(s[g][c >> 1][(c & 1) * 8 + j]);
    }
  };

  // O^T += V^T P^T for the V tile in slot buf: the A operand of 16-key step c
  // for lane half h holds keys 16c + 4h + 0..3 (first read) and
  // 16c + 8 + 4h + 0..3 (second), the key order of the score registers (P
  // stays the B operand unchanged). The V fragments of step c + 2 are
  // requested before the MFMAs of step c.
  //
  // Key rows 16c + kl and 16c + kl + 8 (kl = 4(grp/2) + c4 < 16) have the
  // swizzle of kl, so a lane's address for step c is its step-0 address plus
  // the constant 32cD bytes (+16D for the second read): one base register per
  // 32-column slab, the step in the instruction's offset.
  auto pv = [&](int buf) {
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    constexpr int R = 2 * NT; // LDS reads per 16-key step
    const int grp = lane >> 4, a4 = lane & 3, c4 = (lane >> 2) & 3;
    const int kl = 4 * (grp >> 1) + c4;
    const unsigned vbase = (unsigned)(uintptr_t)(const __attribute__((address_space(3))) char *)&sm.v[buf][0];
    unsigned vb[NT];
#pragma unroll
    for (int tt = 0; tt < NT; ++tt) {
      const int d0 = tt * 32 + 16 * (grp & 1) + 4 * a4; // this lane's 4 columns
      vb[tt] = vbase + kl * D * 2 + (((d0 >> 3) ^ vswz<D>(kl)) << 4) + ((d0 & 7) << 1);
    }
    s16x4 vr[3][R];
    auto vfrag = [&](auto cc) {
      constexpr int c = decltype(cc)::value;
#pragma unroll
      for (int tt = 0; tt < NT; ++tt) {
        vr[c % 3][2 * tt] = lds_read_tr16<c * 32 * D>(vb[tt]);
        vr[c % 3][2 * tt + 1] = lds_read_tr16<c * 32 * D + 16 * D>(vb[tt]);
      }
    };
    auto step = [&](auto cc) {
      constexpr int c = decltype(cc)::value;
      if constexpr (c + 2 < 4) vfrag(std::integral_constant<int, c + 2>{});
      // reads of the later steps already issued stay in flight (LDS reads
      // complete in order)
      constexpr int later = (c + 2 < 4 ? 2 : 3 - c) * R;
      lds_wait_tied<later>(vr[c % 3]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int tt = 0; tt < NT; ++tt) {
        const s16x8 r12 = __builtin_shufflevector(vr[c % 3][2 * tt], vr[c % 3][2 * tt + 1], 0, 1,
                                                  2, 3, 4, 5, 6, 7);
        const V8 a = __builtin_bit_cast(V8, r12);
#pragma unroll
        for (int g = 0; g < QG; ++g) o[g][tt] = mfma32x32<T>(a, pb[g][c], o[g][tt]);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    vfrag(std::integral_constant<int, 0>{});
    vfrag(std::integral_constant<int, 1>{});
    static_for<4>(step);
  };

  // Slots: K tile t and V tile t live in slot (t - t_begin) % 3. Iteration t
  // is two intervals: (A) the leading group's MFMA phase (PV of V(t-1),
  // QK^T of K(t)) beside the trailing group's softmax of tile t-1, then (B)
  // the leading group's softmax of tile t beside the trailing group's MFMA
  // phase. Each group requests tiles during its softmax: the leading waves
  // K(t+2) in (B), into the slot of K(t-1), last read in iteration t-1, and
  // wait for K(t+1) at the end of it; the trailing waves V(t+1) in (A) of
  // iteration t+1, into the slot of V(t-2), and wait for it at the end of
  // their next MFMA phase. Every wait is before the barrier after which the
  // other group reads the tile. K(t_begin), K(t_begin+1) and V(t_begin) are
  // loaded up front.
  // barrier without the fence of __syncthreads (which would drain the DMA);
  // the empty asm keeps the compiler from moving LDS accesses across it
  auto bar = [] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // K(t_begin), K(t_begin + 1) (leading waves), V(t_begin) (trailing waves)
  // of the item, into slot 0, 1 and 0
  auto first_dma = [&] {
    if (t_begin < t_end) {
#pragma unroll
      for (int j = 0; j < NDMA; ++j) dma(j, t_begin, 0);
      if (lead && t_begin + 1 < t_end) {
#pragma unroll
        for (int j = 0; j < NDMA; ++j) dma(j, t_begin + 1, 1);
      }
    }
  };
  // Output staging, 32 rows x D per wave, apart from the K / V slots so the
  // next item's first tiles can land while this item's rows are written out
  typedef typename VecT<T>::v4 V4;
  constexpr int RBY = D * (int)sizeof(T), OCH = RBY / 16, ORPI = 64 / OCH; // row bytes, chunks, rows per pass
  __shared__ V8 stage_all[NW * 32 * OCH];
  char *const stg = reinterpret_cast<char *>(stage_all) + w * (32 * RBY);

  first_dma();
  for (;;) {
    __syncthreads(); // (its fence also drains the DMA and the q loads)
#pragma unroll
    for (int g = 0; g < QG; ++g) {
      m_run[g] = -INFINITY, l_run[g] = 0.f;
#pragma unroll
      for (int tt = 0; tt < NT; ++tt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[g][tt][r] = 0.f;
    }
    if (!lead) bar();
    int sc = 0; // slot of tile t
    for (int t = t_begin; t < t_end; ++t) {
      const int sp = sc == 0 ? kPrefillSlots - 1 : sc - 1; // slot of t-1 (and of t+2)
      const int sn = sc == kPrefillSlots - 1 ? 0 : sc + 1; // slot of t+1
      // At D 64 an iteration is mostly softmax: the matrix wave of a SIMD goes
      // first, so its MFMAs are not held up by the other group's VALU work
      // (bf16, us: 4 x 2048, 16 / 8 heads 58.9 -> 55.9, window 511 43.0 ->
      // 41.5, 1 x 6000, 16 / 1 heads 156.7 -> 147.7). At D 128 the MFMAs fill
      // the iteration themselves: 8 x 2048 160 -> 157, 4 x 2048 89 -> 90.
      if constexpr (D == 64) __builtin_amdgcn_s_setprio(1);
      if (t > t_begin) pv(sp);
      qk(sc);
      if constexpr (D == 64) __builtin_amdgcn_s_setprio(0);
      if (!lead) __builtin_amdgcn_s_waitcnt(0x0F70); // vmcnt(0): V(t) landed
      bar();
      const bool k2 = t + 2 < t_end;
      // K(t+2) into the slot of t-1 (leading waves), V(t+1) into the slot of
      // t+1 (trailing waves)
      const int dt = lead ? (k2 ? t + 2 : -1) : (t + 1 < t_end ? t + 1 : -1);
      const int ds = lead ? sp : sn;
      softmax(t, [&](int j) {
        if (dt >= 0) dma(j, dt, ds);
      });
      if (lead) {
        // K(t+1) landed; K(t+2), issued just now, may stay in flight
        if (k2) __builtin_amdgcn_s_waitcnt((NDMA & 0xF) | ((NDMA >> 4) << 14) | (0x7 << 4) | (0xF << 8));
        else __builtin_amdgcn_s_waitcnt(0x0F70);
      }
      bar();
      sc = sn;
    }
    if (t_begin < t_end) pv(sc == 0 ? kPrefillSlots - 1 : sc - 1);
    if (lead) bar();

    // The item's output rows, then the next item: its q rows are requested
    // now (q is dead after the last QK^T), its first K / V tiles once every
    // wave is past its last PV (the barrier below), after the staging reads.
    const int oqw = qw, oSq = Sq, ohq = hq, ohk = hk, o_tb = t_begin, o_te = t_end;
    const PackedSeq oseq = {seq_q, Sq, seq_k, Sk};
    T *orow = (T *)p.o + (int64_t)b * p.o_sb + (int64_t)hq * p.o_sh;
    if constexpr (PACKED) orow += (int64_t)seq_q * p.o_ss;
    int qt1 = 0, rest1 = 0;
    ++kitem;
    const bool more = next_item(kitem, qt1, rest1);
    if (more) {
      setup(qt1, rest1);
      load_q();
    }
    bar(); // every wave is done with the K / V slots

    // Epilogue: each wave stages its 32 x D output rows in LDS and reads
    // them back as whole 16-byte chunks, D / 8 lanes per output row (straight
    // from the accumulators each store would write 8 bytes into each of 32
    // rows: 4x the write requests).
#pragma unroll
    for (int g = 0; g < QG; ++g) {
      const float l = l_run[g] + __shfl_xor(l_run[g], 32, kWave);
      float inv = l > 0.f ? 1.f / l : 0.f;
      if constexpr (PACKED) { // rows that see nothing are 0, those whose scores are all -inf NaN
        const KeyRange kr = packed_keys(p, oqw + g * 32 + ql, oseq.Sq, oseq.Sk);
        inv = kr.lo < kr.hi ? 1.f / l : 0.f;
      }
      // register 4rg..4rg+3 of tile tt: dims tt*32 + rg*8 + h*4 + 0..3 of query ql,
      // i.e. half h of 16-byte chunk tt*4 + rg of row ql (chunks XOR-swizzled by row)
#pragma unroll
      for (int tt = 0; tt < NT; ++tt)
#pragma unroll
        for (int rg = 0; rg < 4; ++rg) {
          V4 pk;
#pragma unroll
          for (int i = 0; i < 4; ++i) pk[i] = from_f32<T>(o[g][tt][rg * 4 + i] * inv);
          const int ch = (tt * 4 + rg) ^ (ql % OCH);
          *reinterpret_cast<V4 *>(stg + ql * RBY + ch * 16 + h * 8) = pk;
        }
      V8 ov[32 / ORPI];
#pragma unroll
      for (int r = 0; r < 32 / ORPI; ++r) {
        const int row = r * ORPI + lane / OCH, c = lane % OCH;
        ov[r] = *reinterpret_cast<const V8 *>(stg + row * RBY + ((c ^ (row % OCH)) * 16));
      }
      // the DMA goes out after the staging reads: an LDS read issued behind
      // an LDS-DMA waits for it
      if (g == QG - 1 && more) first_dma();
#pragma unroll
      for (int r = 0; r < 32 / ORPI; ++r) {
        const int row = r * ORPI + lane / OCH, c = lane % OCH;
        const int qi = oqw + g * 32 + row;
        if (qi < oSq) *reinterpret_cast<V8 *>(orow + (int64_t)qi * p.o_ss + c * 8) = ov[r];
      }
      if constexpr (PACKED) { // (packed_row_again)
        float z = 0.f;
#pragma unroll
        for (int tt = 0; tt < NT; ++tt)
#pragma unroll
          for (int r = 0; r < 16; ++r) z = fmaf(o[g][tt][r], 0.f, z);
        // a NaN among the scores makes the row NaN anyway
        unsigned long long bad = __ballot(z != z && l == l && oqw + g * 32 + ql < oSq);
        bad = (bad | (bad >> 32)) & 0xffffffffull;
        if (bad) {
          const int qa = oqw + g * 32, qe = min(qa + 31, oSq - 1);
          const KeyRange ka = packed_keys(p, qa, oseq.Sq, oseq.Sk), ke = packed_keys(p, qe, oseq.Sq, oseq.Sk);
          const int k0 = oseq.k0;
          if (packed_odd_values<T, D>(p, ohk, k0 + o_tb * kKvTile, k0 + min(ke.lo, oseq.Sk)) ||
              packed_odd_values<T, D>(p, ohk, k0 + max(ka.hi, 0), k0 + min(o_te * kKvTile, oseq.Sk))) {
            vm_wait<0>(); // the rows above are written before
            for (; bad; bad &= bad - 1) {
              const int i = qa + __builtin_ctzll(bad);
              const KeyRange kr = packed_keys(p, i, oseq.Sq, oseq.Sk);
              packed_row_again<T, D>(p, oseq.q0 + i, k0 + kr.lo, k0 + kr.hi, ohq, ohk);
            }
          }
        }
      }
    }
    if (!more) break;
  }
}

// ---------------------------------------------------------------------------
// Prefill with few work items (a short prompt, a follow-up turn against a
// long cache): the keys are split inside the block, and over blocks where
// that still leaves CUs idle. A block is 32 queries of two heads of a KV head
// (64 queries of one head when the group size is odd), its 8 waves four key
// groups of two waves; group g takes the KT-key tiles g, g + 4, ... of the
// block's chunk of `ct` tiles, staged in its own two-slot LDS ring (the
// group's first wave fetches K, the second V). The groups' running (m, l, O)
// are merged through LDS at the end; with more than one chunk the merged fp32
// partial goes to the workspace, slot = row * nsmax + chunk, and
// attn_prefill_merge_kernel combines the chunks.
// What bounds it: attn_prefill_kernel gives a 128-query item all its keys, so
// 200 queries against 3001 cached keys ran 47 serial tiles on 16 of 256 CUs.
// Here a round of four 32-key tiles takes 1.1-1.45 us (LDS reads and a barrier
// per round; the DMA of the next round in flight beside it) and a block's
// start, merge and stores ~4 us. Splitting the keys in the block first keeps
// the partials small (fp32 rows are 520 bytes per chunk, written and read
// back): the same split over blocks alone would write four times as many. Two
// accumulators per score block (shorter MFMA chains) were no faster.
template <int D> constexpr int kSplitTile = D == 128 ? 32 : 64; // keys per tile (8 KB of K)
constexpr int kSplitGroups = 4;

template <typename T, int D>
__global__ __launch_bounds__(512) void attn_prefill_split_kernel(AttnArgs p, int hpb, int ct, int nsmax,
                                                                 float *__restrict__ ws_o,
                                                                 float *__restrict__ ws_ml) {
  typedef typename VecT<T>::v8 V8;
  constexpr int KT = kSplitTile<D>, NB = KT / 32; // 32-key blocks per tile
  constexpr int CPR = D / 8, NT = D / 32, NG = kSplitGroups;
  constexpr int TU = KT * CPR;                    // 16-byte units per K or V tile
  constexpr int KPI = 64 / CPR, NDMA = KT / KPI;  // keys per DMA instruction, instructions per tile
  constexpr int LDO = D + 4;                      // fp32 pitch of a merged row (odd in 16-byte units)
  constexpr int RING = 2 * NG * 2 * TU, MRG = 8 * 32 * LDO / 4;
  __shared__ V8 smem[RING > MRG ? RING : MRG];
  __shared__ float s_m[8][32], s_l[8][32];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = w >> 1, wu = w & 1, h = lane >> 5, ql = lane & 31;
  const int G = p.Hq / p.Hkv, QL = hpb == 2 ? 32 : 64;
  const int nqt = (p.Sq + QL - 1) / QL, nhg = p.Hq / hpb, npair = p.B * nhg, ipp = nqt * nsmax;
  // all items of a (batch, head group) pair on one XCD (XCD = blockIdx % 8)
  // when the pairs split evenly: their K / V rows stay in its L2
  int pair, r;
  if (npair % 8 == 0) {
    const int j = blockIdx.x / 8;
    pair = (j / ipp) * 8 + blockIdx.x % 8;
    r = j % ipp;
  } else {
    pair = blockIdx.x / ipp;
    r = blockIdx.x % ipp;
  }
  const int qt = nqt - 1 - r / nsmax, split = r % nsmax; // late (causal: heavy) query tiles first
  const int b = pair / nhg, hg = pair % nhg;
  const int hq = hg * hpb + (hpb == 2 ? wu : 0), hk = (hg * hpb) / G;
  const int q0 = qt * QL, q_last = (q0 + QL < p.Sq ? q0 + QL : p.Sq) - 1;
  const int qw = q0 + (hpb == 2 ? 0 : wu * 32);
  const int off = p.Sk - p.Sq;
  const KeyBand kb = key_band(q0, q_last, p.Sq, p.Sk, p.left, p.right, KT);
  const KeyBand chunk = key_chunk(kb, split, ct, nsmax);
  const int t0 = chunk.t_begin, t1 = chunk.t_end;
  if (t0 >= t1 && (split > 0 || nsmax > 1)) return; // (no key at all and one chunk: rows of zeros)
  const int niter = t0 < t1 ? (t1 - t0 + NG - 1) / NG : 0;

  // this wave's DMA: K tiles (first wave of the group) or V tiles (second)
  const bool kwave = wu == 0;
  const int64_t ss = kwave ? p.k_ss : p.v_ss;
  const char *src = kwave ? (const char *)((const T *)p.k + (int64_t)b * p.k_sb + (int64_t)hk * p.k_sh)
                          : (const char *)((const T *)p.v + (int64_t)b * p.v_sb + (int64_t)hk * p.v_sh);
  const int dkey = lane / CPR, dslot = lane % CPR;
  V8 *const gring = smem + g * (4 * TU); // [slot][K | V][TU]
  auto issue = [&](int i) {
    const int t = t0 + i * NG + g;
    if (t >= t1) return; // wave-uniform
    const char *tb = src + (int64_t)t * KT * ss * (int64_t)sizeof(T);
    const int kmax = p.Sk - 1 - t * KT; // keys past Sk read the last one (masked)
    V8 *dst = gring + (i & 1) * (2 * TU) + (kwave ? 0 : TU);
#pragma unroll
    for (int j = 0; j < NDMA; ++j) {
      const int key = j * KPI + dkey;
      const int ch = kwave ? dslot ^ (key & (CPR - 1)) : dslot ^ vswz<D>(key);
      const unsigned o = (unsigned)((min(key, kmax) * ss + ch * 8) * (int64_t)sizeof(T));
      __builtin_amdgcn_global_load_lds((const void *)(tb + o),
                                       (__attribute__((address_space(3))) void *)&dst[j * 64], 16, 0, 0);
    }
  };
  issue(0);

  // q rows, past Sq the last one (never stored); one round trip with the
  // first tiles, waited for here so that no wait for them sits in the loop
  const T *qp = (const T *)p.q + (int64_t)b * p.q_sb + (int64_t)hq * p.q_sh +
                (int64_t)min(qw + ql, p.Sq - 1) * p.q_ss;
  V8 qf[D / 16];
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) qf[ks] = *reinterpret_cast<const V8 *>(qp + ks * 16 + h * 8);
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) asm volatile("" ::"v"(qf[ks]));

  f32x16 o[NT];
#pragma unroll
  for (int tt = 0; tt < NT; ++tt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[tt][i] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;
  const float c2 = p.scale_log2;

  const unsigned gbase = (unsigned)(uintptr_t)(const __attribute__((address_space(3))) char *)gring;
  // V operand addresses within a tile (attn_prefill_kernel explains the layout)
  const int grp = lane >> 4, a4 = lane & 3, c4 = (lane >> 2) & 3, kl = 4 * (grp >> 1) + c4;
  unsigned vo[NT];
#pragma unroll
  for (int tt = 0; tt < NT; ++tt) {
    const int d0 = tt * 32 + 16 * (grp & 1) + 4 * a4;
    vo[tt] = TU * 16 + kl * D * 2 + (((d0 >> 3) ^ vswz<D>(kl)) << 4) + ((d0 & 7) << 1);
  }

  auto tile = [&](int t, int slot) {
    const unsigned base = gbase + slot * (2 * TU * 16);
    // S^T = K Q^T, fragments two steps ahead
    constexpr int KS = D / 16;
    f32x16 s[NB];
#pragma unroll
    for (int st = 0; st < NB; ++st)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[st][i] = 0.f;
    // step i reads two fragments: the two 32-key blocks of K step i, or K
    // steps 2i and 2i + 1 of a one-block tile
    constexpr int NS = KS * NB / 2;
    V8 kr[3][2];
    auto kfrag = [&](auto ii) {
      constexpr int i = decltype(ii)::value;
      static_for<2>([&](auto jj) {
        constexpr int j = decltype(jj)::value, ks = NB == 2 ? i : 2 * i + j;
        const unsigned a = base + (unsigned)((ql * CPR + ((ks * 2 + h) ^ (ql & (CPR - 1)))) * 16);
        kr[i % 3][j] = lds_read_b128<(NB == 2 ? j : 0) * 32 * D * 2, V8>(a);
      });
    };
    kfrag(std::integral_constant<int, 0>{});
    kfrag(std::integral_constant<int, 1>{});
    static_for<NS>([&](auto ii) {
      constexpr int i = decltype(ii)::value;
      if constexpr (i + 2 < NS) kfrag(std::integral_constant<int, i + 2>{});
      lds_wait_tied<(i + 2 < NS ? 2 : NS - 1 - i) * 2>(kr[i % 3]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        s[j % NB] = mfma32x32<T>(kr[i % 3][j], qf[NB == 2 ? i : 2 * i + j], s[j % NB]);
      __builtin_amdgcn_sched_barrier(0);
    });
    // online softmax, as attn_prefill_kernel: raw running max moved only by
    // more than 2^8, masking on band edges
    const int k0 = t * KT;
    if ((p.right >= 0 && k0 + KT - 1 > q0 + off + p.right) ||
        (p.left >= 0 && k0 < q_last + off - p.left) || k0 + KT > p.Sk) {
      const int qpos = qw + ql + off;
      int hi = p.Sk - 1;
      if (p.right >= 0) hi = min(hi, qpos + p.right);
      const int lo = p.left >= 0 ? max(qpos - p.left, 0) : 0;
      const int jb = k0 + h * 4;
      const int ca = max(lo - jb, 0), cb = min(hi - jb, KT - 1);
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
        const float e = __builtin_amdgcn_exp2f(fmaf(s[st][i], c2, -mc));
        s[st][i] = e;
        ps[i & 3] += e;
      }
    l_run = l_run * alpha + ((ps[0] + ps[1]) + (ps[2] + ps[3]));
    m_run = m_new;
    if (__any(move)) {
#pragma unroll
      for (int tt = 0; tt < NT; ++tt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[tt][i] *= alpha;
    }
    V8 pb[2 * NB];
#pragma unroll
    for (int c = 0; c < 2 * NB; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) pb[c][j] = from_f32<T>(s[c >> 1][(c & 1) * 8 + j]);
    // O^T += V^T P^T, one 16-key step ahead
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    constexpr int R = 2 * NT;
    s16x4 vr[2][R];
    auto vfrag = [&](auto cc) {
      constexpr int c = decltype(cc)::value;
#pragma unroll
      for (int tt = 0; tt < NT; ++tt) {
        vr[c % 2][2 * tt] = lds_read_tr16<c * 32 * D>(base + vo[tt]);
        vr[c % 2][2 * tt + 1] = lds_read_tr16<c * 32 * D + 16 * D>(base + vo[tt]);
      }
    };
    vfrag(std::integral_constant<int, 0>{});
    static_for<2 * NB>([&](auto cc) {
      constexpr int c = decltype(cc)::value;
      if constexpr (c + 1 < 2 * NB) vfrag(std::integral_constant<int, c + 1>{});
      lds_wait_tied<(c + 1 < 2 * NB ? R : 0)>(vr[c % 2]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int tt = 0; tt < NT; ++tt) {
        const s16x8 r12 = __builtin_shufflevector(vr[c % 2][2 * tt], vr[c % 2][2 * tt + 1], 0, 1, 2, 3, 4, 5, 6, 7);
        o[tt] = mfma32x32<T>(__builtin_bit_cast(V8, r12), pb[c], o[tt]);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // One barrier per iteration: past it every wave's share of this iteration's
  // tiles has landed and every wave is done with the other slot, which is
  // refilled while this iteration computes.
  for (int i = 0; i < niter; ++i) {
    __builtin_amdgcn_s_waitcnt(0x0F70); // vmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    issue(i + 1);
    if (t0 + i * NG + g < t1) tile(t0 + i * NG + g, i & 1);
  }
  __syncthreads(); // the ring is free

  // merge of the key groups
  float *const mo = reinterpret_cast<float *>(smem) + (w * 32 + ql) * LDO;
#pragma unroll
  for (int tt = 0; tt < NT; ++tt)
#pragma unroll
    for (int rg = 0; rg < 4; ++rg) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = o[tt][rg * 4 + e];
      *reinterpret_cast<f32x4 *>(mo + tt * 32 + rg * 8 + h * 4) = v;
    }
  const float l = l_run + __shfl_xor(l_run, 32, kWave);
  if (h == 0) s_m[w][ql] = m_run, s_l[w][ql] = l;
  __syncthreads();
  for (int idx = tid; idx < 64 * CPR; idx += 512) {
    const int row = idx / CPR, c = idx % CPR, u = row >> 5, rl = row & 31; // u: wave of the groups
    const int qi = q0 + (hpb == 2 ? 0 : u * 32) + rl, hr = hg * hpb + (hpb == 2 ? u : 0);
    if (qi >= p.Sq) continue;
    float mg[NG], mx = -INFINITY;
#pragma unroll
    for (int gg = 0; gg < NG; ++gg) mg[gg] = s_m[gg * 2 + u][rl], mx = fmaxf(mx, mg[gg]);
    const float ms = mx == -INFINITY ? 0.f : mx;
    float ls = 0.f, v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
#pragma unroll
    for (int gg = 0; gg < NG; ++gg) {
      const float a = __builtin_amdgcn_exp2f((mg[gg] - ms) * c2);
      ls += a * s_l[gg * 2 + u][rl];
      const float *q = reinterpret_cast<const float *>(smem) + ((gg * 2 + u) * 32 + rl) * LDO + c * 8;
      const f32x4 x = *reinterpret_cast<const f32x4 *>(q), y = *reinterpret_cast<const f32x4 *>(q + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += a * x[e], v[e + 4] += a * y[e];
    }
    if (nsmax == 1) {
      const float inv = ls > 0.f ? 1.f / ls : 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= inv;
      store8((T *)p.o + (int64_t)b * p.o_sb + (int64_t)qi * p.o_ss + (int64_t)hr * p.o_sh + c * 8, v);
    } else {
      const int64_t sl = (((int64_t)b * p.Hq + hr) * p.Sq + qi) * nsmax + split;
      f32x4 x, y;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = v[e], y[e] = v[e + 4];
      *reinterpret_cast<f32x4 *>(ws_o + sl * D + c * 8) = x;
      *reinterpret_cast<f32x4 *>(ws_o + sl * D + c * 8 + 4) = y;
      if (c == 0) ws_ml[sl * 2] = mx, ws_ml[sl * 2 + 1] = ls;
    }
  }
}

} // namespace tpp
