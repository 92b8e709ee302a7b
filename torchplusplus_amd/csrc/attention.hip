// Flash attention for gfx950: GQA/MQA/MHA, causal and sliding-window prefill,
// and split-KV decode against a KV cache.
//
// Contract: the flash_attn_func calls of the reference
// (torchpp/attention/gqa.py:128, swa.py:85-89, mha.py:84, mqa.py:87, ca.py:83):
//   O = softmax(Q K^T * scale + mask) V, fp32 softmax and accumulation,
//   scale = 1/sqrt(D) by default, query head h reads KV head h / (Hq/Hkv),
//   causal aligned bottom-right (key j visible to query i iff
//   j <= i + Sk - Sq), window (left, right) keeps
//   i + Sk - Sq - left <= j <= i + Sk - Sq + right (negative = unbounded),
//   a query with no visible key yields O = 0.
// Layout: q/o [B, S, H, D] and k/v [B, S, Hkv, D] with arbitrary batch/seq/
// head strides and a contiguous last dim (flash-attn's layout); the KV cache
// of the decode path is [B, Hkv, Lmax, D] through the same strides.
//
// Prefill kernel (D = 64 or 128): one wave = 32 queries of one head.
//  * S^T = K . Q^T with v_mfma_f32_32x32x16 (K tile from LDS as operand A,
//    the wave's Q kept in VGPRs as operand B), so every lane owns ONE query
//    and 32 of the 64 scores of a KV tile: the softmax max/sum is an in-lane
//    loop plus a single exchange with lane ^ 32.
//  * O^T += V^T . P^T: P never leaves registers. MFMA operands pair lane half
//    h and element j with a K index; choosing key(c, h, j) =
//    16c + 8(j/4) + 4h + j%4 for the c-th 16-key step makes the score
//    registers of S^T exactly the B operand, and the A operand two 8-byte LDS
//    reads of a transposed V tile.
//  * K and V^T tiles are staged through XOR-swizzled LDS (16-byte chunks for
//    K, 8-byte 4-key slots for V^T), double-buffered, one barrier per tile.
//  * A block is 4 waves over the query heads that share one KV head (GQA),
//    so a K/V tile in LDS serves up to 4 heads; causal/window tiles outside
//    the block's band are skipped, masks are evaluated only on band edges,
//    and the heaviest (latest) query tiles are dispatched first.
// Decode kernel: a block = (batch, KV head, split); each 16-lane DPP row
// (D/8 lanes) handles one key, all query heads of the group are scored
// against it, online softmax per lane, then log-sum-exp merges across rows,
// waves (LDS) and splits (in the last block, or a small merge kernel).
#include "attention_prefill.hpp"

#include <atomic>
#include <mutex>

namespace tpp {

// Optional fused decode prologue: the new token's raw QKV projection, QK
// RMSNorm weights and RoPE tables. When set, the decode kernel normalises and
// rotates q itself and appends the new key/value to the cache.
struct DecodeFuse {
  const void *qkv; // [B, (Hq + 2 Hkv) * D]
  const void *qw, *kw;
  const void *cos, *sin;
  int cs_dtype, ctx;
  float eps;
};

// Output projection + residual add folded into the decode attention (the
// OP instantiation): residual[B, E] <- T(residual + T(T(o) W^T)).
struct DecodeOproj {
  const void *w; // [E, Hq * D] (nn.Linear layout)
  void *resid;   // [B, E]
  int *ctr;      // counter region (XCD arrival / departure, chunk counters, error flag)
  float *part;   // [8][B][E] fp32 per-XCD partial projections
  int E;
};

// Combine the key chunks of every (batch, head, query) row: D / 4 lanes per
// row, the chunks' (m, l) and outputs read eight at a time.
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_prefill_merge_kernel(AttnArgs p, int QL, int ct, int nsmax,
                                                                 const float *__restrict__ ws_o,
                                                                 const float *__restrict__ ws_ml) {
  constexpr int LPR = D / 4, MG = 8;
  const int64_t row = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int d4 = threadIdx.x % LPR;
  if (row >= (int64_t)p.B * p.Hq * p.Sq) return;
  const int qi = (int)(row % p.Sq), hq = (int)(row / p.Sq % p.Hq), b = (int)(row / p.Sq / p.Hq);
  const int q0 = qi / QL * QL, q_last = (q0 + QL < p.Sq ? q0 + QL : p.Sq) - 1;
  const KeyBand kb = key_band(q0, q_last, p.Sq, p.Sk, p.left, p.right, kSplitTile<D>);
  const int ns = key_chunks(kb, ct, nsmax); // chunks written for this query tile
  float mu = -INFINITY, ls = 0.f, os[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < ns; s0 += MG) {
    float2 ml[MG];
    f32x4 ov[MG];
#pragma unroll
    for (int j = 0; j < MG; ++j) {
      const int64_t sl = row * nsmax + (s0 + j < ns ? s0 + j : ns - 1);
      ml[j] = *reinterpret_cast<const float2 *>(ws_ml + sl * 2);
      ov[j] = *reinterpret_cast<const f32x4 *>(ws_o + sl * D + d4 * 4);
    }
    float mx = mu;
#pragma unroll
    for (int j = 0; j < MG; ++j) mx = fmaxf(mx, ml[j].x);
    const float mn = mx == -INFINITY ? 0.f : mx;
    const float a = __builtin_amdgcn_exp2f((mu - mn) * p.scale_log2);
    ls *= a;
#pragma unroll
    for (int e = 0; e < 4; ++e) os[e] *= a;
#pragma unroll
    for (int j = 0; j < MG; ++j) {
      const float wgt = s0 + j < ns ? __builtin_amdgcn_exp2f((ml[j].x - mn) * p.scale_log2) : 0.f;
      ls += wgt * ml[j].y;
#pragma unroll
      for (int e = 0; e < 4; ++e) os[e] += wgt * ov[j][e];
    }
    mu = mx;
  }
  const float inv = ls > 0.f ? 1.f / ls : 0.f;
  typename VecT<T>::v4 pk;
#pragma unroll
  for (int e = 0; e < 4; ++e) pk[e] = from_f32<T>(os[e] * inv);
  *reinterpret_cast<typename VecT<T>::v4 *>((T *)p.o + (int64_t)b * p.o_sb + (int64_t)qi * p.o_ss +
                                            (int64_t)hq * p.o_sh + d4 * 4) = pk;
}

// Generic prefill (any D <= 256, any alignment): one wave per (b, query,
// head), keys streamed one at a time with a wave reduction. Slow; exists so
// that every head size flash-attn accepts still runs on the GPU.
template <typename T>
__global__ __launch_bounds__(64) void attn_generic_kernel(AttnArgs p, int D) {
  const int lane = threadIdx.x;
  const int64_t id = blockIdx.x; // (b, qi, hq)
  const int hq = (int)(id % p.Hq);
  const int qi = (int)((id / p.Hq) % p.Sq);
  const int b = (int)(id / ((int64_t)p.Hq * p.Sq));
  const int hk = hq / (p.Hq / p.Hkv);
  const int off = p.Sk - p.Sq;
  const T *qp = (const T *)p.q + b * p.q_sb + (int64_t)qi * p.q_ss + hq * p.q_sh;
  const T *kp = (const T *)p.k + b * p.k_sb + hk * p.k_sh;
  const T *vp = (const T *)p.v + b * p.v_sb + hk * p.v_sh;
  float qv[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    qv[i] = d < D ? to_f32(qp[d]) * p.scale_log2 : 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < p.Sk; ++j) {
    const int rel = j - (qi + off);
    if (p.right >= 0 && rel > p.right) break;
    if (p.left >= 0 && rel < -p.left) continue;
    float sdot = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      if (d < D) sdot += qv[i] * to_f32(kp[(int64_t)j * p.k_ss + d]);
    }
    sdot = wave_sum(sdot);
    const float mn = fmaxf(m, sdot);
    const float a = exp2f(m - mn), e = exp2f(sdot - mn);
    l = l * a + e;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      acc[i] = acc[i] * a + (d < D ? e * to_f32(vp[(int64_t)j * p.v_ss + d]) : 0.f);
    }
    m = mn;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  T *op = (T *)p.o + b * p.o_sb + (int64_t)qi * p.o_ss + hq * p.o_sh;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    if (d < D) op[d] = from_f32<T>(acc[i] * inv);
  }
}

// ---------------------------------------------------------------------------
// Decode: one query per sequence against keys [lo_b, L_b) of the cache.
// grid = (nsplit, Hkv, B), block = 256 (4 waves); G = Hq / Hkv <= 8.
// A wave takes KPW keys per pass (one per D/8-lane DPP row) and issues the
// K and V loads of kDecU passes before using any of them; the online
// softmax is updated once per batch of passes.
// ---------------------------------------------------------------------------
constexpr int kDecMaxG = 8;
constexpr int kDecU = 4; // key passes per load batch (two batches in flight)

constexpr int kDecMaxSplit = 256;
#ifndef TPP_DEC_INLINE_MERGE
#define TPP_DEC_INLINE_MERGE 1
#endif
constexpr bool kDecInlineMerge = TPP_DEC_INLINE_MERGE;
constexpr int64_t kDecCounterBytes = 65536; // counters region at the start of the workspace:
constexpr int64_t kDecOpCtrOffset = 32768;  // per-pair arrival counters below, the folded
                                            // projection's counters from here
#ifndef TPP_DEC_WAVES
#define TPP_DEC_WAVES 2048
#endif
constexpr int kDecWaves = TPP_DEC_WAVES; // split-KV target: waves per decode launch
#ifndef TPP_DEC_BIG_NW
#define TPP_DEC_BIG_NW 8
#endif
constexpr int kDecBigNW = TPP_DEC_BIG_NW; // waves per block when G <= 2

// RMSNorm (optional) + rotate-half RoPE of one head row held as 8 values per
// lane by LPK lanes (lane dp owns d = 8 dp .. 8 dp + 7), rounded to T at the
// same points as the unfused path (norm output, rotated output). The norm
// weights w and the table rows c, sn are passed in already loaded.
template <typename T, int LPK>
__device__ __forceinline__ void norm_rope_vals(float (&x)[8], bool norm, const float (&w)[8],
                                               float eps, const float (&c)[8],
                                               const float (&sn)[8], int dp) {
  constexpr int D = LPK * 8;
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
    ss = group_sum<LPK>(ss);
    const float inv = rsqrtf(ss / (float)D + eps);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = to_f32(from_f32<T>((x[j] * inv) * w[j]));
  }
  float pt[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) pt[j] = __shfl_xor(x[j], LPK / 2, kWave); // d +- D/2
  const float sgn = dp < LPK / 2 ? -1.f : 1.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = to_f32(from_f32<T>(x[j] * c[j] + sgn * pt[j] * sn[j]));
}

// 8 RoPE table entries from 32 loaded bytes (fp32: lo then hi 16 bytes;
// fp16 / bf16: the low 16 bytes), the table type a tpp_dtype code. All three
// readings are formed and one selected, with no branch: a branch would let the
// compiler sink the load of `hi` into it, and a load under a branch makes
// every later wait a wait for all loads in flight.
__device__ __forceinline__ void cs_vals(u32x4 lo, u32x4 hi, int cs_dtype, float (&v)[8]) {
  const f16x8 h = __builtin_bit_cast(f16x8, lo);
  const bf16x8 bh = __builtin_bit_cast(bf16x8, lo);
  const bool f32 = cs_dtype == TPP_F32, f16t = cs_dtype == TPP_F16;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = __uint_as_float(i < 4 ? lo[i & 3] : hi[i & 3]);
    const float b16 = f16t ? (float)h[i] : (float)bh[i];
    v[i] = f32 ? a : b16;
  }
}

// Folded output projection (OP): one workgroup per CU, 8 XCDs x 32, the XCD
// of a workgroup = its KV head (Hkv = 8), so XCD x holds every split of every
// sequence for query heads x G .. x G + G - 1, i.e. the K slice
// [x G D, (x + 1) G D) of the projection. Its workgroup j owns output
// columns [32 j, 32 j + 32). Constants of that layout:
constexpr int kOpXcds = 8, kOpPerXcd = 32, kOpCols = 32;
constexpr unsigned kOpSpinLimit = 1u << 20;
// counter region (ints, each counter on its own 128-byte line) at
// kDecOpCtrOffset of the workspace: arrive[8], depart[8], chunk[32], err
constexpr int kOpArrive = 0, kOpDepart = 8 * 32, kOpChunk = 16 * 32, kOpErr = 48 * 32;
static_assert(kAttnOprojCtrOffset == (size_t)kDecOpCtrOffset &&
                  kAttnOprojErrOffset == (size_t)kDecOpCtrOffset + kOpErr * sizeof(int),
              "counter and flag offsets shared with ffn.hip");

template <typename T>
__device__ __forceinline__ f32x4 mfma16x32(typename VecT<T>::v8 a, typename VecT<T>::v8 b, f32x4 c) {
  if constexpr (__is_same(T, bf16))
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// End of the OP kernel, after this workgroup published its split partial:
//  1. XCD-local sync: the workgroup counts itself in and waits until all 32
//     workgroups of its XCD (every split of every sequence for the XCD's KV
//     head) have published; the partials then sit in this XCD's L2. The wait
//     is bounded: if the workgroups were not all resident it gives up, sets
//     the error flag and the output is wrong (flagged).
//  2. Every workgroup merges the splits of all B sequences for the XCD's G
//     heads into LDS (the attention output, rounded to T like the unfused
//     path's output tensor), and workgroup j < B also stores sequence j's
//     rows to the output tensor.
//  3. Partial projection of output columns [32 j, 32 j + 32) over the XCD's
//     K slice with v_mfma_f32_16x16x32 (batch rows padded to 16), written
//     through to memory as fp32.
//  4. An agent-scope counter per column chunk finds the chunk's last XCD,
//     which sums the 8 partials in XCD order (fixed: bit-reproducible) and
//     updates the residual: T(residual + T(sum)).
template <typename T, int D, int G, int NW, int MG>
__device__ __forceinline__ void attn_decode_oproj_tail(const AttnArgs &p, const float *__restrict__ ws_o,
                                                       int nsplit, const DecodeOproj &op,
                                                       const T *s_w, T *s_o, f32x4 (*s_red)[64]) {
  typedef typename VecT<T>::v8 V8;
  constexpr int KO = G * D, UPR = KO / 8;
  const int lane = lane_id(), w = __builtin_amdgcn_readfirstlane(wave_id());
  const int x = blockIdx.x % kOpXcds, jb = blockIdx.x / kOpXcds;
  const int B = p.B, E = op.E;
  int *arrive = op.ctr + kOpArrive + x * 32;
  int *depart = op.ctr + kOpDepart + x * 32;
  int *chunkc = op.ctr + kOpChunk + jb * 32;
  int *err = op.ctr + kOpErr;
  T *resid = (T *)op.resid;
  __shared__ int s_last;
  // residual values of this workgroup's column chunk (used if it is the
  // chunk's last XCD), requested before the waits below
  const int e = threadIdx.x; // blockDim.x == 512 >= 16 * 32
  const int rb = e / kOpCols < B ? e / kOpCols : 0;
  const T rres = resid[(int64_t)rb * E + kOpCols * jb + e % kOpCols];

  // ---- 1. XCD-local sync (the partial stores and the weight DMA are done:
  // vmcnt(0); the counter lives in this XCD's L2, polled with an atomic add
  // of 0 from an asm move so the compiler keeps it an atomic)
  __builtin_amdgcn_s_waitcnt(0x0F70);
  __syncthreads();
  if (threadIdx.x == 0) {
    __hip_atomic_fetch_add(arrive, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    unsigned n = 0;
    int zero;
    asm volatile("v_mov_b32 %0, 0" : "=v"(zero));
    while (__hip_atomic_fetch_add(arrive, zero, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) < kOpPerXcd) {
      if (++n > kOpSpinLimit) {
        __hip_atomic_fetch_or(err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        break;
      }
      __builtin_amdgcn_s_sleep(1);
    }
    // the XCD's last workgroup past the wait resets both counters
    if (__hip_atomic_fetch_add(depart, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
        kOpPerXcd - 1) {
      __hip_atomic_store(arrive, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(depart, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  __syncthreads();

  // ---- 2. merge the splits: item = (batch row, head, 4 columns); rows past
  // B are zero (MFMA padding). Each split slot is D outputs, m, l, padding;
  // the splits are read in groups of MG (nsplit = 32 / B is a multiple), all
  // loads of a group before any use: one L2 round trip per group.
  for (int it = threadIdx.x; it < 16 * G * (D / 4); it += 64 * NW) {
    const int d4 = it % (D / 4), gi = (it / (D / 4)) % G, bb = it / (D / 4 * G);
    float r[4] = {0.f, 0.f, 0.f, 0.f};
    if (bb < B) {
      const float *sl = ws_o + ((int64_t)bb * p.Hq + x * G + gi) * nsplit * (D + 32);
      float mu = -INFINITY, ls = 0.f, os[4] = {0.f, 0.f, 0.f, 0.f};
      for (int s0 = 0; s0 < nsplit; s0 += MG) {
        float mv[MG], lv[MG];
        f32x4 ov[MG];
#pragma unroll
        for (int jj = 0; jj < MG; ++jj) {
          const float *q = sl + (int64_t)(s0 + jj) * (D + 32);
          const float2 ml = *reinterpret_cast<const float2 *>(q + D);
          mv[jj] = ml.x;
          lv[jj] = ml.y;
          ov[jj] = *reinterpret_cast<const f32x4 *>(q + 4 * d4);
        }
        float mx = mu;
#pragma unroll
        for (int jj = 0; jj < MG; ++jj) mx = fmaxf(mx, mv[jj]);
        const float mn = mx == -INFINITY ? 0.f : mx;
        const float a = mu == -INFINITY ? 0.f : exp2f(mu - mn);
        ls *= a;
#pragma unroll
        for (int c = 0; c < 4; ++c) os[c] *= a;
#pragma unroll
        for (int jj = 0; jj < MG; ++jj) {
          const float wgt = exp2f(mv[jj] - mn);
          ls += wgt * lv[jj];
#pragma unroll
          for (int c = 0; c < 4; ++c) os[c] += wgt * ov[jj][c];
        }
        mu = mx;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) r[c] = ls > 0.f ? os[c] / ls : 0.f;
    }
    T tv[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) tv[c] = from_f32<T>(r[c]);
    T *so = s_o + bb * (KO + 8) + gi * D + 4 * d4;
#pragma unroll
    for (int c = 0; c < 4; ++c) so[c] = tv[c];
    if (bb < B && bb == jb) {
      T *o = (T *)p.o + (int64_t)bb * p.o_sb + (int64_t)(x * G + gi) * p.o_sh + 4 * d4;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] = tv[c];
    }
  }
  __syncthreads();

  // ---- 3. partial projection: waves 0-3 output columns 32 j .. + 15,
  // waves 4-7 the next 16; wave w & 3 takes K steps (w & 3) G .. + G - 1 of 32
  const int t = w >> 2;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const int ks = (w & 3) * G + i;
    const int gu = ks * 4 + (lane >> 4);          // 16-byte unit of K
    const int wr = 16 * t + (lane & 15);          // weight row of the tile
    const V8 a = *reinterpret_cast<const V8 *>(s_o + (lane & 15) * (KO + 8) + gu * 8);
    const V8 bw = *reinterpret_cast<const V8 *>(s_w + wr * KO + (gu ^ (wr & (UPR - 1))) * 8);
    acc = mfma16x32<T>(a, bw, acc);
  }
  s_red[w][lane] = acc;
  __syncthreads();
  if ((w & 3) == 0) {
    f32x4 sum = s_red[w][lane];
#pragma unroll
    for (int i = 1; i < 4; ++i) sum += s_red[w + i][lane];
    // D layout: lane -> column lane & 15, batch rows 4 (lane >> 4) + i
    const int n = kOpCols * jb + 16 * t + (lane & 15);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = 4 * (lane >> 4) + i;
      if (b < B)
        __hip_atomic_store(op.part + ((int64_t)x * B + b) * E + n, sum[i], __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  // ---- 4. partial written through (vmcnt(0)); count this XCD in for the chunk
  __builtin_amdgcn_s_waitcnt(0x0F70);
  __syncthreads();
  if (threadIdx.x == 0) {
    const int old = __hip_atomic_fetch_add(chunkc, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = old == kOpXcds - 1;
    if (old == kOpXcds - 1) __hip_atomic_store(chunkc, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!s_last || e >= B * kOpCols) return;
  const int b = e / kOpCols, n = kOpCols * jb + e % kOpCols;
  float v[kOpXcds];
#pragma unroll
  for (int xx = 0; xx < kOpXcds; ++xx)
    v[xx] = __hip_atomic_load(op.part + ((int64_t)xx * B + b) * E + n, __ATOMIC_RELAXED,
                              __HIP_MEMORY_SCOPE_AGENT);
  float sum = 0.f;
#pragma unroll
  for (int xx = 0; xx < kOpXcds; ++xx) sum += v[xx];
  resid[(int64_t)b * E + n] = from_f32<T>(to_f32(rres) + to_f32(from_f32<T>(sum)));
}

// How a sequence's keys are dealt to the splits of its pair: whole batches of
// `stride` keys (a power of two) from key `lead`, the batch that holds the
// first visible key `lo`, `batches` of them per split. By the sequence's
// length: runs cut from the capacity left most splits empty where the cache
// has room to spare (bf16, 16 / 8 heads, D 128: 8 x 500 keys of 8192 14.9 ->
// 10.4 us, 1 x 900 13.7 -> 9.2 us, 32 / 8 heads 16 x 2000 of 4096 60.6 -> 41.1
// us; with the folded projection 8 x 2058 of 2304 22.0 -> 20.6 us). Dealing
// the batches to the splits in turn instead was 5% slower at 16000 keys.
struct SplitRun {
  int lo, lead, nbatch, batches;
  // splits that have a batch (the first `live`), at least one
  __host__ __device__ int live() const { return nbatch > 0 ? (nbatch + batches - 1) / batches : 1; }
};
__host__ __device__ inline SplitRun split_run(int L, int left, int stride, int nsplit, unsigned inv) {
  SplitRun r;
  r.lo = left >= 0 && L - 1 - left > 0 ? L - 1 - left : 0;
  r.lead = r.lo & ~(stride - 1);
  r.nbatch = L > r.lead ? (int)((unsigned)(L - r.lead + stride - 1) / (unsigned)stride) : 0;
  const int per = div_inv((unsigned)(r.nbatch + nsplit - 1), inv); // < 2^24 batches, nsplit <= 256
  r.batches = per > 0 ? per : 1;
  return r;
}

// In-kernel merge of a pair's splits, after this workgroup wrote its partial
// slots (`live` of the `nsplit` slots of a head hold keys).
template <typename T, int D>
__device__ __forceinline__ void decode_merge_splits(const AttnArgs &p, int b, int hk, int G, int nsplit,
                                                    int live, const float *__restrict__ ws_o,
                                                    int *__restrict__ counters) {
  // The last block of the pair to finish merges the splits. Every thread
  // waits for its partial stores to reach L2 (an explicit vmcnt(0): the
  // workgroup-scope fence of __syncthreads does not wait for global stores),
  // then one thread counts the block in with an atomic in L2; the block that
  // takes the count to `live` reads the other partials from the same L2.
  // Each partial slot is whole 128-byte lines written by one block only, and
  // a block reads other blocks' slots only here, so this CU's L1 (clean at
  // kernel start) holds no stale copy of them.
  __shared__ int s_last;
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0F70); // vmcnt(0)
  __syncthreads();
  const int pair = b * p.Hkv + hk;
  if (threadIdx.x == 0) {
    // agent scope: the counter is shared by workgroups (of one XCD); the
    // atomic is performed in that XCD's L2 either way
    const int old = __hip_atomic_fetch_add(&counters[pair], 1, __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_AGENT);
    s_last = old == live - 1;
    if (old == live - 1) // leave the counter at 0 for the next launch
      __hip_atomic_store(&counters[pair], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!s_last) return;
  for (int idx = threadIdx.x; idx < G * D; idx += blockDim.x) {
    const int gi = idx / D, d = idx % D;
    const float *sl = ws_o + (((int64_t)b * p.Hq + hk * G + gi) * nsplit) * (D + 32);
    // the partials in groups of MG splits: a group's loads all go out before
    // any is used (indices past nsplit read the last split and weigh 0), one
    // L2 round trip per group instead of two per split; groups after the
    // first rescale the running sums (online softmax)
    constexpr int MG = 8;
    float mu = -INFINITY, ls = 0.f, os = 0.f;
    for (int s0 = 0; s0 < live; s0 += MG) {
      float mv[MG], lv[MG], ov[MG];
#pragma unroll
      for (int j = 0; j < MG; ++j) {
        const int sp = s0 + j < live ? s0 + j : live - 1;
        const float *q = sl + (int64_t)sp * (D + 32);
        mv[j] = q[D];
        lv[j] = q[D + 1];
        ov[j] = q[d];
      }
      float mx = mu;
#pragma unroll
      for (int j = 0; j < MG; ++j)
        if (s0 + j < live) mx = fmaxf(mx, mv[j]);
      const float mn = mx == -INFINITY ? 0.f : mx;
      const float a = mu == -INFINITY ? 0.f : exp2f(mu - mn);
      ls *= a;
      os *= a;
#pragma unroll
      for (int j = 0; j < MG; ++j) {
        const float wgt = s0 + j < live ? exp2f(mv[j] - mn) : 0.f;
        ls += wgt * lv[j];
        os += wgt * ov[j];
      }
      mu = mx;
    }
    T *op = (T *)p.o + (int64_t)b * p.o_sb + (int64_t)(hk * G + gi) * p.o_sh;
    op[d] = from_f32<T>(ls > 0.f ? os / ls : 0.f);
  }
}

template <typename T, int D, int G, int NW, bool OP = false>
__global__ __launch_bounds__(64 * NW) void attn_decode_kernel(AttnArgs p, const int *__restrict__ seqlens,
                                                              int fixed_len, float *__restrict__ ws_o,
                                                              float *__restrict__ ws_ml, int nsplit,
                                                              unsigned nsplit_inv, unsigned hkv_inv,
                                                              DecodeFuse fz,
                                                              int *__restrict__ counters,
                                                              DecodeOproj op) {
  typedef typename VecT<T>::v8 V8;
  constexpr int LPK = D / 8;        // lanes per key
  constexpr int KPW = kWave / LPK;  // keys per wave pass
  constexpr int U = kDecU;
  __shared__ float red_m[NW][G], red_l[NW][G];
  __shared__ float red_o[NW][G][D];
  // OP: the workgroup's [32 x G D] projection weight tile (LDS-DMA at kernel
  // start, 16-byte units of a row XOR-swizzled by the row), the merged
  // attention output of the XCD's heads for 16 (padded) batch rows, and the
  // cross-wave reduction of the projection
  constexpr int KO = G * D;        // projection K slice of an XCD
  constexpr int UPR = KO / 8;      // 16-byte units per weight row
  __shared__ __attribute__((aligned(16))) T s_w[OP ? kOpCols * KO : 8];
  __shared__ __attribute__((aligned(16))) T s_o[OP ? 16 * (KO + 8) : 8];
  __shared__ f32x4 s_red[OP ? NW : 1][64];
  static_assert(!OP || (D == 128 && NW == 8 && G <= 2), "folded projection: D 128, 8 waves, G <= 2");

  // w through readfirstlane: the compiler then knows it (and every key index
  // derived from it) is wave-uniform, so the key loop's exits are scalar
  // branches rather than exec-mask updates with per-lane live-out copies
  const int lane = lane_id(), w = __builtin_amdgcn_readfirstlane(wave_id());
  const int row = lane / LPK, dp = lane % LPK;
  int split = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
  if (counters) {
    // one-dimensional grid; workgroups are dealt to the 8 XCDs round-robin
    // (XCD = blockIdx % 8): all splits of a (batch, KV head) pair share an
    // XCD, so their partials meet in that XCD's L2
    const int xcd = blockIdx.x % 8, slot = blockIdx.x / 8;
    const int group = div_inv(slot, nsplit_inv), pair = group * 8 + xcd;
    split = slot - group * nsplit;
    b = div_inv(pair, hkv_inv);
    hk = pair - b * p.Hkv;
  }
  const T *kp = (const T *)p.k + (int64_t)b * p.k_sb + (int64_t)hk * p.k_sh + dp * 8;
  const T *vp = (const T *)p.v + (int64_t)b * p.v_sb + (int64_t)hk * p.v_sh + dp * 8;
  // K/V rows of one batch of keys base + u*NW*KPW + row (u < U), each key
  // clamped to `last`: past the keys a block scores they read a finite cache
  // row whose scores compute_batch masks. Every batch is issued
  // unconditionally: with no load under a branch the compiler's count of
  // loads in flight stays exact, so scoring batch i waits for batch i only (a
  // conditional load makes it wait for everything in flight).
  constexpr int STRIDE = NW * KPW * U; // keys per block-wide batch
  auto load_batch = [&](int base, int last, V8 (&kr)[U], V8 (&vr)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key0 = base + u * NW * KPW + row;
      const int key = key0 < last ? key0 : last;
      kr[u] = ld_nt(reinterpret_cast<const V8 *>(kp + (int64_t)key * p.k_ss));
      vr[u] = ld_nt(reinterpret_cast<const V8 *>(vp + (int64_t)key * p.v_ss));
    }
  };
  // The split's keys: the sequence's batches in `nsplit` even runs (by its
  // length, not the cache's: a length far below the capacity still spreads
  // over all splits), from the window's first batch on. Splits without a batch
  // leave at once, except that the folded projection needs every workgroup.
  // The length is one scalar load ahead of the first K/V loads (0.4 us;
  // loading two batches of the capacity's split before the length was known
  // cost more wherever the sequence is short: 64 KB per batch and block). A
  // full cache pays for it: 1 x 4096 keys of 4096, 8 heads, 11.7 -> 12.0 us, 32
  // x 1000 of 1024, 16 heads, D 64, 23.8 -> 24.5 us.
  const int Lraw = seqlens ? seqlens[b] : fixed_len;
  const int L = Lraw < p.Sk ? (Lraw > 0 ? Lraw : 0) : p.Sk; // never read past the cache
  const SplitRun run = split_run(L, p.left, STRIDE, nsplit, nsplit_inv);
  const int64_t c0 = run.lead + (int64_t)split * run.batches * STRIDE;
  if (!OP && split > 0 && c0 >= L) return;
  const int first = (int)(c0 < L ? c0 : L) + w * KPW;
  const int last0 = L > 0 ? L - 1 : 0;
  // Three register sets: while one batch is scored the next two are in flight.
  V8 k0[U], v0[U], k1[U], v1[U], k2[U], v2[U];
  load_batch(first, last0, k0, v0);
  load_batch(first + STRIDE, last0, k1, v1);
  if constexpr (OP) {
    // the projection weight tile W[32 j .. 32 j + 31][x G D .. + G D) by
    // LDS-DMA (1 KB per wave instruction). Issued before the prologue loads,
    // whose first use waits for every load in flight anyway, so the compiler's
    // counted waits of the key loop are not disturbed by it.
    const int jb = blockIdx.x / kOpXcds;
    const T *wsrc = (const T *)op.w + (int64_t)(kOpCols * jb) * (p.Hq * D) + (int64_t)hk * KO;
    constexpr int NQ = kOpCols * KO * (int)sizeof(T) / (NW * 1024); // instructions per wave
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int unit = (w * NQ + q) * 64 + lane; // LDS 16-byte unit
      const int r = unit / UPR, lu = unit % UPR;
      const int gu = lu ^ (r & (UPR - 1));       // global unit stored at LDS unit lu
      __builtin_amdgcn_global_load_lds(
          (const void *)(wsrc + (int64_t)r * (p.Hq * D) + gu * 8),
          (__attribute__((address_space(3))) void *)(s_w + (w * NQ + q) * 64 * 8), 16, 0, 0);
    }
  }

  const int k_begin = (int)(c0 > run.lo ? (c0 < L ? c0 : L) : run.lo);
  int k_end = (int)(c0 + (int64_t)run.batches * STRIDE < L ? c0 + (int64_t)run.batches * STRIDE : L);
  // fused prologue: position L-1 is the new token; this block attends to it
  // from registers (if it falls in its run) and the cache loop stops before it
  const bool fused = fz.qkv != nullptr;
  const int pnew = L - 1;
  const bool own_new = fused && Lraw <= p.Sk && pnew >= k_begin && pnew < k_end;
  if (fused && k_end > pnew) k_end = pnew;
  const T *qkv_row = fused ? (const T *)fz.qkv + (int64_t)b * (p.Hq + 2 * p.Hkv) * D : nullptr;

  // Every load the prologue needs goes out next, unconditionally (an absent
  // operand reads a valid row instead, never used): the q rows of the group,
  // and when fused the norm weights, the RoPE rows at the new position and
  // the new token's K/V row. One memory round trip then covers all of them
  // and the first K/V batches, where a load under a branch, or a load whose
  // address depends on an earlier one, costs a round trip each.
  const T *qbase = fused ? qkv_row + (int64_t)hk * G * D
                         : (const T *)p.q + (int64_t)b * p.q_sb + (int64_t)(hk * G) * p.q_sh;
  const int64_t qstep = fused ? (int64_t)D : p.q_sh;
  V8 q_raw[G];
#pragma unroll
  for (int gi = 0; gi < G; ++gi) q_raw[gi] = *reinterpret_cast<const V8 *>(qbase + gi * qstep + dp * 8);
  const T *anyrow = qbase + dp * 8;
  const T *qw_src = fz.qw ? (const T *)fz.qw + dp * 8 : anyrow;
  const T *kw_src = fz.kw ? (const T *)fz.kw + dp * 8 : anyrow;
  const V8 qw_raw = *reinterpret_cast<const V8 *>(qw_src);
  const V8 kw_raw = *reinterpret_cast<const V8 *>(kw_src);
  const int pr = fused ? (pnew < 0 ? 0 : (pnew < fz.ctx ? pnew : fz.ctx - 1)) : 0;
  const int64_t cs_es = fz.cs_dtype == TPP_F32 ? 4 : 2;
  const char *c_src = fused ? (const char *)fz.cos + ((int64_t)pr * D + dp * 8) * cs_es
                            : (const char *)anyrow;
  const char *s_src = fused ? (const char *)fz.sin + ((int64_t)pr * D + dp * 8) * cs_es
                            : (const char *)anyrow;
  const int64_t cs_hi = fused && cs_es == 4 ? 16 : 0;
  const u32x4 c_lo = *reinterpret_cast<const u32x4 *>(c_src);
  const u32x4 c_hi = *reinterpret_cast<const u32x4 *>(c_src + cs_hi);
  const u32x4 s_lo = *reinterpret_cast<const u32x4 *>(s_src);
  const u32x4 s_hi = *reinterpret_cast<const u32x4 *>(s_src + cs_hi);
  const V8 knew_raw =
      *reinterpret_cast<const V8 *>(fused ? qkv_row + (int64_t)(p.Hq + hk) * D + dp * 8 : anyrow);
  const V8 vnew_raw = *reinterpret_cast<const V8 *>(
      fused ? qkv_row + (int64_t)(p.Hq + p.Hkv + hk) * D + dp * 8 : anyrow);

  float c[8], sn[8];
  cs_vals(c_lo, c_hi, fz.cs_dtype, c);
  cs_vals(s_lo, s_hi, fz.cs_dtype, sn);
  // q rounded to T after the fused QK-norm and RoPE, as the unfused path
  // stores it in its q tensor; scores by v_dot2 on T pairs accumulated in
  // fp32, scaled after the row reduction
  V8 qh[G];
#pragma unroll
  for (int gi = 0; gi < G; ++gi) {
    float qv[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) qv[j] = to_f32(q_raw[gi][j]);
    if (fused) {
      float wq[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) wq[j] = to_f32(qw_raw[j]);
      norm_rope_vals<T, LPK>(qv, fz.qw != nullptr, wq, fz.eps, c, sn, dp);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) qh[gi][j] = from_f32<T>(qv[j]);
  }
  const float qscale = p.scale_log2;
  // the new token's K (normalised, rotated) and V, computed here by every
  // wave and pinned (empty asm uses): left to the block that appends them
  // they would keep their loads in flight across the whole key loop, and the
  // registers the loop reuses would make every iteration wait for all loads
  float kf[8], vf[8];
  {
    float wk[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      kf[j] = to_f32(knew_raw[j]);
      vf[j] = to_f32(vnew_raw[j]);
      wk[j] = to_f32(kw_raw[j]);
    }
    norm_rope_vals<T, LPK>(kf, fz.kw != nullptr, wk, fz.eps, c, sn, dp);
#pragma unroll
    for (int j = 0; j < 8; ++j) asm volatile("" ::"v"(kf[j]), "v"(vf[j]));
  }
  float m[G], l[G], acc[G][8];
#pragma unroll
  for (int gi = 0; gi < G; ++gi) {
    m[gi] = -INFINITY;
    l[gi] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[gi][j] = 0.f;
  }
  auto compute_batch = [&](int base, const V8 (&kr)[U], const V8 (&vr)[U]) {
    float sc[U][G];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool ok = (unsigned)(base + u * NW * KPW + row - k_begin) < (unsigned)(k_end - k_begin);
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        float sdot = dot8<T>(qh[gi], kr[u], 0.f);
        sdot += dpp_f32<kDppQuadXor1>(sdot);
        sdot += dpp_f32<kDppQuadXor2>(sdot);
        if constexpr (LPK >= 8) sdot += dpp_f32<kDppRowHalfMirror>(sdot);
        if constexpr (LPK >= 16) sdot += dpp_f32<kDppRowMirror>(sdot);
        sc[u][gi] = ok ? sdot * qscale : -INFINITY;
      }
    }
#pragma unroll
    for (int gi = 0; gi < G; ++gi) {
      float mb = m[gi];
#pragma unroll
      for (int u = 0; u < U; ++u) mb = fmaxf(mb, sc[u][gi]);
      const float mu = mb == -INFINITY ? 0.f : mb;
      const float alpha = exp2f(m[gi] - mu);
      l[gi] *= alpha;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[gi][j] *= alpha;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float e = exp2f(sc[u][gi] - mu);
        l[gi] += e;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[gi][j] += e * to_f32(vr[u][j]);
      }
      m[gi] = mb;
    }
  };
  // Whole triples of batches in the loop (a single exit: with a break after
  // every batch the compiler merges the exits into one latch, whose state
  // then has a batch in flight, and waits for everything at the loop head),
  // the last one or two batches after it. Batches past the keys that a
  // triple loads are clamped rows and never scored.
  // this wave's keys: first + i*STRIDE + u*NW*KPW + row, scored iff in
  // [k_begin, k_end) (a window can start inside a batch)
  const int k_last = k_end > 0 ? k_end - 1 : 0;
  int nbat = k_begin < k_end && first < k_end ? (k_end - first + STRIDE - 1) / STRIDE : 0;
  int base = first;
  for (; nbat >= 3; nbat -= 3, base += 3 * STRIDE) {
    asm volatile("" ::: "memory");
    load_batch(base + 2 * STRIDE, k_last, k2, v2);
    asm volatile("" ::: "memory");
    compute_batch(base, k0, v0);
    asm volatile("" ::: "memory");
    load_batch(base + 3 * STRIDE, k_last, k0, v0);
    asm volatile("" ::: "memory");
    compute_batch(base + STRIDE, k1, v1);
    asm volatile("" ::: "memory");
    load_batch(base + 4 * STRIDE, k_last, k1, v1);
    asm volatile("" ::: "memory");
    compute_batch(base + 2 * STRIDE, k2, v2);
  }
  if (nbat >= 1) compute_batch(base, k0, v0);
  if (nbat >= 2) compute_batch(base + STRIDE, k1, v1);
  if (own_new && w == 0) {
    // the new key/value (normalised and rotated in the prologue): append both
    // to the cache (row 0 lanes) and fold the key into row 0's online softmax
    if (row == 0) {
      store8((T *)kp + (int64_t)pnew * p.k_ss, kf);
      store8((T *)vp + (int64_t)pnew * p.v_ss, vf);
    }
    V8 kh; // the key as the cache holds it
#pragma unroll
    for (int j = 0; j < 8; ++j) kh[j] = from_f32<T>(kf[j]);
#pragma unroll
    for (int gi = 0; gi < G; ++gi) {
      const float sdot = group_sum<LPK>(dot8<T>(qh[gi], kh, 0.f)) * qscale;
      if (row == 0) {
        const float mn = fmaxf(m[gi], sdot);
        const float a = exp2f(m[gi] - mn), e = exp2f(sdot - mn);
        l[gi] = l[gi] * a + e;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[gi][j] = acc[gi][j] * a + e * to_f32(from_f32<T>(vf[j]));
        m[gi] = mn;
      }
    }
  }
  // merge the KPW key rows of the wave (lanes with equal dp): at distance
  // SH = LPK .. 32 every lane gets its own and its partner's (m, l, acc) as an
  // unordered pair (v_permlane16/32_swap, or a row rotation by 8), and
  // combines them symmetrically, so both lanes of a pair get the same value
#pragma unroll
  for (int gi = 0; gi < G; ++gi) {
    auto merge_at = [&](auto pair_of) {
      float ma, mb, la, lb;
      pair_of(m[gi], ma, mb);
      pair_of(l[gi], la, lb);
      const float mn = fmaxf(ma, mb);
      const float mu = mn == -INFINITY ? 0.f : mn;
      const float a = exp2f(ma - mu), c = exp2f(mb - mu);
      l[gi] = la * a + lb * c;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float xa, xb;
        pair_of(acc[gi][j], xa, xb);
        acc[gi][j] = xa * a + xb * c;
      }
      m[gi] = mn;
    };
    if constexpr (LPK <= 8)
      merge_at([](float x, float &a, float &b) { a = x, b = dpp_f32<kDppRowRor8>(x); });
    if constexpr (LPK <= 16)
      merge_at([](float x, float &a, float &b) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
      });
    merge_at([](float x, float &a, float &b) {
      const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
      a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
    });
    if (row == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) red_o[w][gi][dp * 8 + j] = acc[gi][j];
      if (dp == 0) {
        red_m[w][gi] = m[gi];
        red_l[w][gi] = l[gi];
      }
    }
  }
  __syncthreads();
  const int live = run.live(); // splits with a batch (at least one)
  // merge the NW waves: thread -> (gi, d); write this split's partial, or the
  // final output when one split has all the keys
  for (int idx = threadIdx.x; idx < G * D; idx += blockDim.x) {
    const int gi = idx / D, d = idx % D;
    float mx = -INFINITY;
#pragma unroll
    for (int ww = 0; ww < NW; ++ww) mx = fmaxf(mx, red_m[ww][gi]);
    const float mu = mx == -INFINITY ? 0.f : mx;
    float ls = 0.f, os = 0.f;
#pragma unroll
    for (int ww = 0; ww < NW; ++ww) {
      const float c = exp2f(red_m[ww][gi] - mu);
      ls += red_l[ww][gi] * c;
      os += red_o[ww][gi][d] * c;
    }
    const int hq = hk * G + gi;
    if (!OP && live == 1) {
      T *op = (T *)p.o + (int64_t)b * p.o_sb + (int64_t)hq * p.o_sh;
      op[d] = from_f32<T>(ls > 0.f ? os / ls : 0.f);
      continue;
    }
    const int64_t slot = ((int64_t)b * p.Hq + hq) * nsplit + split;
    if (counters) {
      // slot = D partial outputs, m, l, padding: whole 128-byte lines
      float *sl = ws_o + slot * (D + 32);
      sl[d] = os;
      if (d == 0) sl[D] = mx, sl[D + 1] = ls;
    } else {
      ws_o[slot * D + d] = os;
      if (d == 0) ws_ml[slot * 2] = mx, ws_ml[slot * 2 + 1] = ls;
    }
  }
  if constexpr (OP) {
    // nsplit = 32 / B: 2, 4 or a multiple of 8
    if (nsplit == 2) attn_decode_oproj_tail<T, D, G, NW, 2>(p, ws_o, nsplit, op, s_w, s_o, s_red);
    else if (nsplit == 4) attn_decode_oproj_tail<T, D, G, NW, 4>(p, ws_o, nsplit, op, s_w, s_o, s_red);
    else attn_decode_oproj_tail<T, D, G, NW, 8>(p, ws_o, nsplit, op, s_w, s_o, s_red);
    return;
  }
  if (!counters || live == 1) return;
  decode_merge_splits<T, D>(p, b, hk, G, nsplit, live, ws_o, counters);
}

// ---------------------------------------------------------------------------
// Decode with two or more query heads per KV head, on the matrix cores. The
// VALU kernel above scores every head of the group against every key: at four
// heads it is bound by that work (3.2 TB/s of the cache, at eight 1.2 TB/s).
// Here the group's heads are the columns of S^T = K Q^T (32x32x16, at most 8
// of 32 columns used: still several times the rate the cache arrives at) and
// of O^T = V^T P^T. A block is 4 waves; each wave streams its own tiles of the
// split's run (K and V by LDS-DMA into a private slot, no barrier in the
// loop): the next K tile is requested as soon as this one's fragments are
// read, the next V tile after this one's. The probabilities keep their fp32
// bits: P is the sum of three parts in T, each what the ones ahead leave (8
// bits each in bf16, 11 in fp16), and the parts are columns 0-7, 8-15 and
// 16-23 of one product, summed in fp32 at the end. Two parts in two products
// lost a P below 2^-25 in fp16 and the last bits in bf16, in the same time
// (bf16 within 0.3 us either way, fp16 0.1-0.5 us faster). Waves, then splits,
// are merged as in the kernel above. Measured (bf16, the VALU kernel first): 16
// sequences of 2000 keys, 32 / 8 heads, D 128, 41.1 -> 26.1 us; 64 sequences of
// 64-4000 keys, 8 / 1 heads, 57.6 -> 22.3 us; 8 of 300-3000, 32 / 8 heads, D
// 64, 22.1 -> 12.0 us; two heads: 1 sequence of 900 keys, 16 / 8 heads, D 128,
// 9.1 -> 7.9 us, 32 of 100-4096 55.3 -> 52.1 us, 8 of 2058 16.9 -> 16.7 us.
// ---------------------------------------------------------------------------
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_decode_mfma_kernel(AttnArgs p, const int *__restrict__ seqlens,
                                                               int fixed_len, float *__restrict__ ws_o,
                                                               float *__restrict__ ws_ml, int nsplit,
                                                               unsigned nsplit_inv, unsigned hkv_inv,
                                                               int *__restrict__ counters) {
  typedef typename VecT<T>::v8 V8;
  constexpr int KT = kSplitTile<D>, NB = KT / 32, NW = 4, STRIDE = NW * KT;
  constexpr int CPR = D / 8, NT = D / 32, TU = KT * CPR;
  constexpr int KPI = 64 / CPR, NDMA = KT / KPI;
  constexpr int LDO = D + 4; // fp32 pitch of a wave's partial rows
  __shared__ V8 smem[NW * 2 * TU];
  __shared__ float s_m[NW][kDecMaxG], s_l[NW][kDecMaxG];
  constexpr int NP = 3; // parts of a probability
  static_assert(NP * kDecMaxG * LDO * 4 <= 2 * TU * 16 && kDecMaxG == 8 && NP * kDecMaxG <= 32,
                "a wave's partial rows fit its tile slot, its parts the columns");
  // fp16 parts are scaled by 2^15 (P is 1 at most) and by 2^11 more each: what
  // falls below the least half of the last one is under 2^-61 of P's largest
  constexpr bool H = !__is_same(T, bf16);
  constexpr float kScale0 = H ? 32768.f : 1.f, kScale1 = H ? 2048.f : 1.f;

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, ql = lane & 31, G = p.Hq / p.Hkv;
  int split = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
  if (counters) { // splits of a pair on one XCD, as above
    const int xcd = blockIdx.x % 8, slot = blockIdx.x / 8;
    const int group = div_inv(slot, nsplit_inv), pair = group * 8 + xcd;
    split = slot - group * nsplit;
    b = div_inv(pair, hkv_inv);
    hk = pair - b * p.Hkv;
  }
  const int Lraw = seqlens ? seqlens[b] : fixed_len;
  const int L = Lraw < p.Sk ? (Lraw > 0 ? Lraw : 0) : p.Sk; // never read past the cache
  const SplitRun run = split_run(L, p.left, STRIDE, nsplit, nsplit_inv);
  const int64_t c0 = run.lead + (int64_t)split * run.batches * STRIDE;
  if (split > 0 && c0 >= L) return;
  const int k_begin = (int)(c0 > run.lo ? (c0 < L ? c0 : L) : run.lo);
  const int k_end = (int)(c0 + (int64_t)run.batches * STRIDE < L ? c0 + (int64_t)run.batches * STRIDE : L);

  // LDS-DMA of this wave's tiles: keys past the run read its last one (finite,
  // masked)
  const char *ks = (const char *)((const T *)p.k + (int64_t)b * p.k_sb + (int64_t)hk * p.k_sh);
  const char *vs = (const char *)((const T *)p.v + (int64_t)b * p.v_sb + (int64_t)hk * p.v_sh);
  const int dkey = lane / CPR, dslot = lane % CPR;
  V8 *const ring = smem + w * (2 * TU);
  auto issue = [&](bool kt, int base) {
    const char *src = kt ? ks : vs;
    const int64_t ss = kt ? p.k_ss : p.v_ss;
#pragma unroll
    for (int j = 0; j < NDMA; ++j) {
      const int key = j * KPI + dkey;
      const int ch = kt ? dslot ^ (key & (CPR - 1)) : dslot ^ vswz<D>(key);
      __builtin_amdgcn_global_load_lds(
          (const void *)(src + ((int64_t)min(base + key, k_end - 1) * ss + ch * 8) * (int64_t)sizeof(T)),
          (__attribute__((address_space(3))) void *)(ring + (kt ? 0 : TU) + j * 64), 16, 0, kCpolNT);
    }
  };
  const int first = (int)(c0 < L ? c0 : L) + w * KT;
  const int n = first < k_end ? (k_end - first + STRIDE - 1) / STRIDE : 0; // this wave's tiles
  if (n > 0) {
    issue(true, first);
    issue(false, first);
  }
  // Query heads of the group as columns ql % 8 (past G the last head again),
  // once for each part of the probabilities (columns past the parts repeat the
  // last part): every lane of a head computes the same scores.
  const int head = ql % kDecMaxG, prt = ql / kDecMaxG;
  // this lane's part of eight probabilities x[8 half ..]: what the parts ahead
  // of it leave, cut (not rounded) to T, two values at a time
  const float off1 = prt > 0 ? -1.f : 0.f, off2 = prt > 1 ? -1.f : 0.f;
  const float sc1 = prt > 0 ? kScale1 : 1.f, sc2 = prt > 1 ? kScale1 : 1.f;
  const unsigned m1 = prt > 0 ? 0xffff0000u : 0u, m2 = prt > 1 ? 0xffff0000u : 0u;
  auto part_of = [&](const f32x16 &x, int half) {
    u32x4 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a = x[half * 8 + 2 * j], b = x[half * 8 + 2 * j + 1];
      if constexpr (H) {
        a *= kScale0, b *= kScale0;
        const auto h0 = __builtin_amdgcn_cvt_pkrtz(a, b);
        a = fmaf(off1, (float)h0[0], a) * sc1, b = fmaf(off1, (float)h0[1], b) * sc1;
        const auto h1 = __builtin_amdgcn_cvt_pkrtz(a, b);
        a = fmaf(off2, (float)h1[0], a) * sc2, b = fmaf(off2, (float)h1[1], b) * sc2;
        r[j] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(a, b));
      } else { // a bfloat16 is the upper half of a float
        a -= __uint_as_float(__float_as_uint(a) & m1), b -= __uint_as_float(__float_as_uint(b) & m1);
        a -= __uint_as_float(__float_as_uint(a) & m2), b -= __uint_as_float(__float_as_uint(b) & m2);
        r[j] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
      }
    }
    return __builtin_bit_cast(V8, r);
  };
  const T *qp = (const T *)p.q + (int64_t)b * p.q_sb + (int64_t)(hk * G + min(head, G - 1)) * p.q_sh;
  V8 qf[D / 16];
#pragma unroll
  for (int i = 0; i < D / 16; ++i) qf[i] = *reinterpret_cast<const V8 *>(qp + i * 16 + h * 8);
  // waited for here (with the first tiles): no wait for them inside the loop
#pragma unroll
  for (int i = 0; i < D / 16; ++i) asm volatile("" ::"v"(qf[i]));

  f32x16 o[NT];
#pragma unroll
  for (int tt = 0; tt < NT; ++tt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[tt][i] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;
  const float c2 = p.scale_log2;
  const unsigned base0 = (unsigned)(uintptr_t)(const __attribute__((address_space(3))) char *)ring;
  const int grp = lane >> 4, a4 = lane & 3, c4 = (lane >> 2) & 3, kl = 4 * (grp >> 1) + c4;
  unsigned vo[NT];
#pragma unroll
  for (int tt = 0; tt < NT; ++tt) {
    const int d0 = tt * 32 + 16 * (grp & 1) + 4 * a4;
    vo[tt] = base0 + TU * 16 + kl * D * 2 + (((d0 >> 3) ^ vswz<D>(kl)) << 4) + ((d0 & 7) << 1);
  }
  for (int i = 0; i < n; ++i) {
    const int kb = first + i * STRIDE;
    const bool more = i + 1 < n;
    vm_wait<NDMA>(); // this tile's K landed (its V may be in flight)
    constexpr int KS = D / 16, NS = KS * NB / 2;
    f32x16 s[NB];
#pragma unroll
    for (int st = 0; st < NB; ++st)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[st][r] = 0.f;
    V8 kr[3][2];
    auto kfrag = [&](auto ii) {
      constexpr int x = decltype(ii)::value;
      static_for<2>([&](auto jj) {
        constexpr int j = decltype(jj)::value, k = NB == 2 ? x : 2 * x + j;
        const unsigned a = base0 + (unsigned)((ql * CPR + ((k * 2 + h) ^ (ql & (CPR - 1)))) * 16);
        kr[x % 3][j] = lds_read_b128<(NB == 2 ? j : 0) * 32 * D * 2, V8>(a);
      });
    };
    kfrag(std::integral_constant<int, 0>{});
    kfrag(std::integral_constant<int, 1>{});
    static_for<NS>([&](auto ii) {
      constexpr int x = decltype(ii)::value;
      if constexpr (x + 2 < NS) kfrag(std::integral_constant<int, x + 2>{});
      lds_wait_tied<(x + 2 < NS ? 2 : NS - 1 - x) * 2>(kr[x % 3]);
      // every K fragment is in registers: the next K tile may land
      if constexpr (x == NS - 1) {
        asm volatile("" ::: "memory");
        if (more) issue(true, kb + STRIDE);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        s[j % NB] = mfma32x32<T>(kr[x % 3][j], qf[NB == 2 ? x : 2 * x + j], s[j % NB]);
      __builtin_amdgcn_sched_barrier(0);
    });
    if (kb < k_begin || kb + KT > k_end) {
      const int jb = kb + h * 4;
      const int ca = max(k_begin - jb, 0), cb = min(k_end - 1 - jb, KT - 1);
      const unsigned ninf = __float_as_uint(-INFINITY);
#pragma unroll
      for (int st = 0; st < NB; ++st) {
        const int l0 = max(ca - 32 * st, 0), h0 = min(cb - 32 * st, 31);
        const unsigned keep = l0 <= h0 ? ((2u << h0) - 1u) & ~((1u << l0) - 1u) : 0u;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const unsigned bm = (unsigned)__builtin_amdgcn_sbfe((int)keep, (r >> 2) * 8 + (r & 3), 1);
          s[st][r] = __uint_as_float((__float_as_uint(s[st][r]) & bm) | (ninf & ~bm));
        }
      }
    }
    float mx[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
#pragma unroll
    for (int st = 0; st < NB; ++st)
#pragma unroll
      for (int r = st == 0 ? 4 : 0; r < 16; ++r) mx[r & 3] = fmaxf(mx[r & 3], s[st][r]);
    float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
    mt = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
    const bool move = mt > m_run;
    const float m_new = move ? mt : m_run;
    const float mc = m_new == -INFINITY ? 0.f : m_new * c2;
    const float alpha = move ? __builtin_amdgcn_exp2f(m_run * c2 - mc) : 1.f;
    float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int st = 0; st < NB; ++st)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float e = __builtin_amdgcn_exp2f(fmaf(s[st][r], c2, -mc));
        s[st][r] = e;
        ps[r & 3] += e;
      }
    l_run = l_run * alpha + ((ps[0] + ps[1]) + (ps[2] + ps[3]));
    m_run = m_new;
    if (__any(move)) {
#pragma unroll
      for (int tt = 0; tt < NT; ++tt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[tt][r] *= alpha;
    }
    // this lane's part of each probability: what the parts ahead leave
    V8 pb[2 * NB];
#pragma unroll
    for (int c = 0; c < 2 * NB; ++c) pb[c] = part_of(s[c >> 1], c & 1);
    // this tile's V landed (the next K may be in flight)
    if (more) vm_wait<NDMA>();
    else vm_wait<0>();
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    constexpr int R = 2 * NT;
    s16x4 vr[2][R];
    auto vfrag = [&](auto cc) {
      constexpr int c = decltype(cc)::value;
#pragma unroll
      for (int tt = 0; tt < NT; ++tt) {
        vr[c % 2][2 * tt] = lds_read_tr16<c * 32 * D>(vo[tt]);
        vr[c % 2][2 * tt + 1] = lds_read_tr16<c * 32 * D + 16 * D>(vo[tt]);
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
        const s16x8 r12 = __builtin_shufflevector(vr[c % 2][2 * tt], vr[c % 2][2 * tt + 1], 0, 1, 2, 3, 4, 5, 6, 7);
        o[tt] = mfma32x32<T>(__builtin_bit_cast(V8, r12), pb[c], o[tt]);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  }

  // this wave's rows (its tile slot is drained), then the block's
  const float l = l_run + __shfl_xor(l_run, 32, kWave);
  float *const part = reinterpret_cast<float *>(ring);
  if (head < G && prt < NP) {
#pragma unroll
    for (int tt = 0; tt < NT; ++tt)
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = o[tt][rg * 4 + e];
        *reinterpret_cast<f32x4 *>(part + ql * LDO + tt * 32 + rg * 8 + h * 4) = v;
      }
    if (h == 0 && prt == 0) s_m[w][head] = m_run == -INFINITY ? m_run : m_run * c2, s_l[w][head] = l;
  }
  // An infinity in V: its products with the parts of P (which may be zero or
  // of opposite sign) sum to NaN where P times V is infinite. A wave with a
  // non-finite sum therefore redoes its sums with one product per key.
  bool odd = false;
#pragma unroll
  for (int tt = 0; tt < NT; ++tt)
#pragma unroll
    for (int r = 0; r < 16; ++r) odd |= !(fabsf(o[tt][r]) < INFINITY);
  if (__any(odd)) {
    for (int gi = 0; gi < G; ++gi) {
      const T *qr = (const T *)p.q + (int64_t)b * p.q_sb + (int64_t)(hk * G + gi) * p.q_sh;
      const float mg = __shfl(m_run, gi, kWave), mc = mg == -INFINITY ? 0.f : mg * c2;
      float acc[D / 64];
#pragma unroll
      for (int c = 0; c < D / 64; ++c) acc[c] = 0.f;
      for (int i = 0; i < n; ++i)
        for (int key = max(first + i * STRIDE, k_begin); key < min(first + i * STRIDE + KT, k_end); ++key) {
          const T *kr = (const T *)ks + (int64_t)key * p.k_ss, *vr = (const T *)vs + (int64_t)key * p.v_ss;
          float sd = 0.f;
#pragma unroll
          for (int c = 0; c < D / 64; ++c) sd += to_f32(qr[c * 64 + lane]) * to_f32(kr[c * 64 + lane]);
          const float e = __builtin_amdgcn_exp2f(fmaf(wave_sum(sd), c2, -mc));
#pragma unroll
          for (int c = 0; c < D / 64; ++c) acc[c] += e * to_f32(vr[c * 64 + lane]);
        }
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        part[gi * LDO + c * 64 + lane] = acc[c] * kScale0;
#pragma unroll
        for (int x = 1; x < NP; ++x) part[(x * kDecMaxG + gi) * LDO + c * 64 + lane] = 0.f;
      }
    }
  }
  __syncthreads();
  const int live = run.live();
  for (int idx = tid; idx < G * D; idx += 64 * NW) {
    const int gi = idx / D, d = idx % D;
    float mx = -INFINITY;
#pragma unroll
    for (int ww = 0; ww < NW; ++ww) mx = fmaxf(mx, s_m[ww][gi]);
    const float mu = mx == -INFINITY ? 0.f : mx;
    float ls = 0.f, os = 0.f;
#pragma unroll
    for (int ww = 0; ww < NW; ++ww) {
      const float c = exp2f(s_m[ww][gi] - mu);
      ls += s_l[ww][gi] * c;
      const float *pr = reinterpret_cast<const float *>(smem + ww * (2 * TU)) + gi * LDO + d;
      float sum = 0.f; // the least part first
#pragma unroll
      for (int x = NP - 1; x >= 0; --x) sum = sum * (1.f / kScale1) + pr[x * kDecMaxG * LDO];
      os += sum * (1.f / kScale0) * c;
    }
    const int hq = hk * G + gi;
    if (live == 1) {
      T *op = (T *)p.o + (int64_t)b * p.o_sb + (int64_t)hq * p.o_sh;
      op[d] = from_f32<T>(ls > 0.f ? os / ls : 0.f);
      continue;
    }
    const int64_t slot = ((int64_t)b * p.Hq + hq) * nsplit + split;
    if (counters) {
      float *sl = ws_o + slot * (D + 32);
      sl[d] = os;
      if (d == 0) sl[D] = mx, sl[D + 1] = ls;
    } else {
      ws_o[slot * D + d] = os;
      if (d == 0) ws_ml[slot * 2] = mx, ws_ml[slot * 2 + 1] = ls;
    }
  }
  if (!counters || live == 1) return;
  decode_merge_splits<T, D>(p, b, hk, G, nsplit, live, ws_o, counters);
}

// Merge the split partials of one (batch, KV head): grid (Hkv, B), 256
// threads, G query heads. A separate launch on purpose: publishing partials
// across blocks inside one kernel needs device-scope release/acquire fences,
// which on MI355X write back / invalidate the XCD's L2 (the 8 XCD L2s are not
// coherent) and cost far more than a kernel boundary.
template <typename T, int D, int G>
__global__ __launch_bounds__(G * D) void attn_decode_merge_kernel(AttnArgs p, const int *__restrict__ seqlens,
                                                                  int fixed_len, int stride,
                                                                  const float *__restrict__ ws_o,
                                                                  const float *__restrict__ ws_ml,
                                                                  int slots, unsigned slots_inv) {
  constexpr int PRE = 16; // partial outputs prefetched per thread
  __shared__ float s_w[G][kDecMaxSplit], s_l[G][kDecMaxSplit], s_inv[G];
  const int hk = blockIdx.x, b = blockIdx.y, lane = lane_id(), w = wave_id();
  const int gi = threadIdx.x / D, d = threadIdx.x % D;
  const int64_t s0 = ((int64_t)b * p.Hq + hk * G) * slots; // slot of (gi = 0, split 0)
  // this thread's partial outputs and the (m, l) pairs do not depend on the
  // length: load first (slots without keys hold anything and are not used)
  const float *po = ws_o + (s0 + (int64_t)gi * slots) * D + d;
  float pre[PRE];
#pragma unroll
  for (int j = 0; j < PRE; ++j) pre[j] = po[(int64_t)(j < slots ? j : 0) * D];
  for (int idx = threadIdx.x; idx < G * slots; idx += blockDim.x) {
    const int g2 = idx / slots, sp = idx % slots;
    const float *ml = ws_ml + (s0 + (int64_t)g2 * slots + sp) * 2;
    s_w[g2][sp] = ml[0];
    s_l[g2][sp] = ml[1];
  }
  // splits that had keys; with one, that split wrote the output itself
  const int Lraw = seqlens ? seqlens[b] : fixed_len;
  const int L = Lraw < p.Sk ? (Lraw > 0 ? Lraw : 0) : p.Sk;
  const int nsplit = split_run(L, p.left, stride, slots, slots_inv).live();
  __syncthreads();
  if (nsplit <= 1) return;
  const int nwave = blockDim.x / kWave;
  for (int g2 = w; g2 < G; g2 += nwave) { // one wave per query head
    float mx = -INFINITY;
    for (int sp = lane; sp < nsplit; sp += kWave) mx = fmaxf(mx, s_w[g2][sp]);
#pragma unroll
    for (int sh = 1; sh < kWave; sh <<= 1) mx = fmaxf(mx, __shfl_xor(mx, sh, kWave));
    const float mu = mx == -INFINITY ? 0.f : mx;
    float ls = 0.f;
    for (int sp = lane; sp < nsplit; sp += kWave) {
      const float wgt = exp2f(s_w[g2][sp] - mu);
      s_w[g2][sp] = wgt;
      ls += wgt * s_l[g2][sp];
    }
    ls = wave_sum(ls);
    if (lane == 0) s_inv[g2] = ls > 0.f ? 1.f / ls : 0.f;
  }
  __syncthreads();
  float os = 0.f;
#pragma unroll
  for (int j = 0; j < PRE; ++j) os += j < nsplit ? s_w[gi][j] * pre[j] : 0.f;
  for (int sp = PRE; sp < nsplit; ++sp) os += s_w[gi][sp] * po[(int64_t)sp * D];
  T *op = (T *)p.o + (int64_t)b * p.o_sb + (int64_t)(hk * G + gi) * p.o_sh;
  op[d] = from_f32<T>(os * s_inv[gi]);
}

static int check_attn(const char *name, const AttnArgs &a, int64_t D) {
  if (!a.q || !a.k || !a.v || !a.o) return set_error(TPP_E_INVALID, "%s: null pointer", name);
  if (a.B < 0 || a.Sq < 0 || a.Sk < 0 || a.Hq <= 0 || a.Hkv <= 0 || D <= 0)
    return set_error(TPP_E_INVALID, "%s: invalid shapes", name);
  if (a.Hq % a.Hkv != 0)
    return set_error(TPP_E_INVALID, "%s: Hq (%d) must be a multiple of Hkv (%d)", name, a.Hq,
                     a.Hkv);
  if (D > 256) return set_error(TPP_E_UNSUPPORTED, "%s: head_dim %lld > 256", name, (long long)D);
  return TPP_OK;
}

static bool strides16(const AttnArgs &a) {
  auto al = [](int64_t s) { return s % 8 == 0; };
  return aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.o) && al(a.q_sb) &&
         al(a.q_ss) && al(a.q_sh) && al(a.k_sb) && al(a.k_ss) && al(a.k_sh) && al(a.v_sb) &&
         al(a.v_ss) && al(a.v_sh) && al(a.o_sb) && al(a.o_ss) && al(a.o_sh);
}

// Prefill plan: the whole-chip kernel (one workgroup per CU looping over 8-wave
// work items), or the key-split kernel with `nsmax` chunks of `ct` tiles.
struct PrefillPlan {
  bool split;
  int hpb, ct, nsmax;
  int64_t blocks;
  size_t ws_bytes;
};

// Estimated times in us, from measurements of both kernels (bf16, B 1 - 4, Sq
// 17 - 4096, Sk 64 - 8000): the whole-chip kernel takes 6.5 us plus 1.55 (D =
// 128; 2.0 with every CU busy) or 1.2 (D = 64) per 64-key tile of its longest
// CU; a key-split block 4.2 us plus 1.1 (1.45 with most CUs busy) or 1.3 per
// round of four tiles, and several chunks a merge launch of 2.5 us + 0.55 us
// per MB of partials. The split kernel is taken where it is expected to be
// 10% faster at least (the margin covers the estimate's error), e.g. 230
// causal tokens of 16 heads 12.3 -> 8.6 us, 1000 tokens 32.4 -> 16.5 us, 200
// tokens against 3001 cached keys 80.4 -> 21.5 us (3 chunks), 33 against 8000
// 202 -> 19.7 us (11 chunks), 2 x 1000 tokens of 16 / 16 heads, D 64, in a
// window of 512 22.0 -> 17.1 us; left alone: 4 x 512 tokens (20.8 against 21.5
// us), 4096 tokens in a window of 512 (29 against 50 us).
static PrefillPlan plan_prefill(int64_t B, int64_t Sq, int64_t Sk, int64_t Hq, int64_t Hkv, int64_t D,
                                int left, int right, bool workspace) {
  PrefillPlan pl{};
  pl.nsmax = 1;
  const int64_t G = Hq / Hkv;
  const int cus = device_cu_count() > 0 ? device_cu_count() : 256;
  pl.hpb = G % 2 == 0 ? 2 : 1;
  const int64_t ql = 64 / pl.hpb, nqt = (Sq + ql - 1) / ql, npair = B * (Hq / pl.hpb);
  if (npair * nqt > 8 * (int64_t)cus || Sk > (1 << 30)) return pl;
  // tiles of `kt` keys per query tile of `len` queries: an upper bound (the
  // chunks are cut by it) and the average of the first, middle and last tile
  auto tiles = [&](int64_t len, int kt, double &most, double &mean) {
    const int64_t n = (Sq + len - 1) / len;
    auto at = [&](int64_t t) {
      const int64_t q0 = t * len, last = (q0 + len < Sq ? q0 + len : Sq) - 1;
      return key_band((int)q0, (int)last, (int)Sq, (int)Sk, left, right, kt);
    };
    const KeyBand f = at(0), m = at(n / 2), l = at(n - 1);
    mean = (double)((f.t_end - f.t_begin) + 2 * (m.t_end - m.t_begin) + (l.t_end - l.t_begin)) / 4;
    // bands move right with the query; bounded on both sides, a whole one also
    // has at most the tiles that its keys touch from where one can begin in a
    // tile (kt and len are powers of two: kt / len places, or one)
    int64_t top = l.t_end - f.t_begin;
    if (left >= 0 && right >= 0) {
      const int64_t keys = (len < Sq ? len : Sq) + left + right;
      int64_t touched = 0;
      for (int64_t q0 = 0; q0 < (kt > len ? kt : len); q0 += len) {
        const int64_t begin = (q0 + Sk - Sq - left) & (kt - 1), t = (begin + keys - 1) / kt + 1;
        touched = t > touched ? t : touched;
      }
      top = touched < top ? touched : top;
    }
    most = (double)top;
  };
  double most, mean;
  const int hpb8 = (G % 4 == 0) ? 4 : (G % 2 == 0) ? 2 : 1;
  const int64_t len8 = (8 / hpb8) * 32;
  tiles(len8, kKvTile, most, mean);
  const double items8 = (double)(B * (Hq / hpb8) * ((Sq + len8 - 1) / len8));
  const double per8 = D == 128 ? (items8 >= cus ? 2.0 : 1.55) : 1.2;
  const double whole = items8 * (4.5 + mean * per8) / cus > 4.5 + most * per8
                           ? 2.0 + items8 * (4.5 + mean * per8) / cus
                           : 6.5 + most * per8;
  tiles(ql, D == 128 ? kSplitTile<128> : kSplitTile<64>, most, mean);
  double best = 0.9 * whole;
  for (const int n : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
    int ct = ((int)(most + n - 1) / n + kSplitGroups - 1) / kSplitGroups * kSplitGroups;
    if (ct < kSplitGroups) ct = kSplitGroups;
    const int ns = most > ct ? (int)((most + ct - 1) / ct) : 1;
    const double parts = mean / ct > 1 ? mean / ct + (ns > 1 ? 0.5 : 0) : 1; // chunks per query tile
    const double blocks = (double)(npair * nqt) * (parts < ns ? parts : ns), load = blocks / cus;
    const double c = D == 128 ? (load >= 0.75 ? 1.45 : 1.1) : 1.3;
    const double longest = 4.2 + (most < ct ? (int)(most + kSplitGroups - 1) / kSplitGroups : ct / kSplitGroups) * c;
    const double each = 4.2 + (mean / (parts < ns ? parts : ns) / kSplitGroups + 0.4) * c;
    const double rounds = load <= 1 ? 1 : (load + 0.5 < ceil(load) ? load + 0.5 : ceil(load));
    const size_t ws = ns > 1 ? (size_t)(B * Hq * Sq * ns) * (size_t)(D + 2) * sizeof(float) : 0;
    const double t = 2.0 + (rounds * each > longest ? rounds * each : longest) +
                     (ns > 1 ? 2.5 + 0.55e-6 * (double)ws : 0.0);
    if (t < best && (ns == 1 || workspace)) {
      best = t;
      pl.split = true;
      pl.ct = ct, pl.nsmax = ns, pl.ws_bytes = ws;
      pl.blocks = npair * nqt * ns;
    }
    if (ct == kSplitGroups) break;
  }
  return pl;
}

template <typename T>
static int launch_prefill(const AttnArgs &a, int64_t D, void *ws, size_t ws_bytes, hipStream_t st,
                          const char *name) {
  if (a.B == 0 || a.Sq == 0) return TPP_OK;
  const int G = a.Hq / a.Hkv;
  // the tiled kernels address a 64-row K / V tile with 32-bit byte offsets
  const bool rows_fit = a.k_ss >= 0 && a.v_ss >= 0 && (int64_t)kKvTile * a.k_ss * 2 < (1LL << 31) &&
                        (int64_t)kKvTile * a.v_ss * 2 < (1LL << 31);
  if ((D == 64 || D == 128) && strides16(a) && rows_fit) {
    const PrefillPlan pl = plan_prefill(a.B, a.Sq, a.Sk, a.Hq, a.Hkv, D, a.left, a.right, ws != nullptr);
    if (pl.split) {
      if (pl.ws_bytes > ws_bytes)
        return set_error(TPP_E_WORKSPACE, "%s: workspace of %zu bytes required", name, pl.ws_bytes);
      const int64_t rows = (int64_t)a.B * a.Hq * a.Sq;
      float *wo = (float *)ws, *wml = wo + (pl.nsmax > 1 ? rows * pl.nsmax * D : 0);
      auto go = [&](auto dd) {
        constexpr int DD = decltype(dd)::value;
        attn_prefill_split_kernel<T, DD><<<dim3((unsigned)pl.blocks), dim3(512), 0, st>>>(
            a, pl.hpb, pl.ct, pl.nsmax, wo, wml);
        constexpr int rpb = 256 / (DD / 4); // rows per merge block
        if (pl.nsmax > 1)
          attn_prefill_merge_kernel<T, DD><<<dim3((unsigned)((rows + rpb - 1) / rpb)), dim3(256), 0, st>>>(
              a, 64 / pl.hpb, pl.ct, pl.nsmax, wo, wml);
      };
      if (D == 128) go(std::integral_constant<int, 128>{});
      else go(std::integral_constant<int, 64>{});
      return check_launch(name);
    }
    const int hpb = (G % 4 == 0) ? 4 : (G % 2 == 0) ? 2 : 1;
    constexpr int QG = kPrefillQG;
    constexpr int NW = kPrefillWaves;
    const int qt_len = (NW / hpb) * 32 * QG;
    const int64_t items =
        (int64_t)a.B * (a.Hq / hpb) * ((a.Sq + qt_len - 1) / qt_len);
    if (items > 0x7fffffffLL) return set_error(TPP_E_UNSUPPORTED, "%s: too large", name);
    // one workgroup per CU loops over the work items (more items than CUs)
    const int cus = device_cu_count();
    const int64_t blocks = (cus > 0 && items > cus) ? cus : items;
    if (D == 128)
      attn_prefill_kernel<T, 128, QG, NW><<<dim3((unsigned)blocks), dim3(64 * NW), 0, st>>>(a, hpb);
    else
      attn_prefill_kernel<T, 64, QG, NW><<<dim3((unsigned)blocks), dim3(64 * NW), 0, st>>>(a, hpb);
  } else {
    const int64_t blocks = (int64_t)a.B * a.Sq * a.Hq;
    if (blocks > 0x7fffffffLL) return set_error(TPP_E_UNSUPPORTED, "%s: too large", name);
    attn_generic_kernel<T><<<dim3((unsigned)blocks), dim3(64), 0, st>>>(a, (int)D);
  }
  return check_launch(name);
}

struct DecodePlan {
  int nsplit, nw;
  bool inline_merge; // the last split block merges (no merge kernel)
  size_t o_bytes, ml_bytes, ws_bytes;
};

// Partial-slot layout of a split plan: in-kernel merge (one padded slot per
// split) or merge kernel (D outputs, then m/l pairs; the counter region stays
// reserved and untouched, so a workspace shared with in-kernel-merge calls
// keeps its counters at zero).
static void use_merge_layout(DecodePlan &pl, size_t slots, int64_t D, bool inline_merge) {
  pl.inline_merge = inline_merge;
  if (inline_merge) {
    pl.o_bytes = slots * (size_t)(D + 32) * sizeof(float);
    pl.ml_bytes = 0;
  } else {
    pl.o_bytes = slots * (size_t)D * sizeof(float);
    pl.ml_bytes = slots * 2 * sizeof(float);
  }
}

// Split-KV plan: about one 8-wave block per CU; each sequence's load batches
// are dealt evenly to the splits of its (batch, KV head) pair on the device
// (split_run). One split needs no merge.
static DecodePlan plan_decode(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t Lmax) {
  DecodePlan pl{};
  const int64_t kpw = kWave / (D / 8);
  const int64_t pairs = B * Hkv > 0 ? B * Hkv : 1;
  pl.nw = (Hkv > 0 && Hq / Hkv <= 2) ? kDecBigNW : 4; // more query heads per KV head: more VGPRs
  const int64_t batch = pl.nw * kpw * kDecU; // keys per block-wide load batch
  // about kDecWaves waves, in whole load batches (a block's loop runs whole
  // batches: a chunk of part batches costs the same time with keys masked,
  // measured 18.3 -> 20.0 us at the model shape with 32-key granularity)
  int64_t want = (kDecWaves / pl.nw + pairs - 1) / pairs;
  int64_t chunk = (Lmax + want - 1) / want;
  chunk = ((chunk + batch - 1) / batch) * batch;
  if (chunk < batch) chunk = batch;
  while ((Lmax + chunk - 1) / chunk > kDecMaxSplit) chunk += batch;
  pl.nsplit = (int)((Lmax + chunk - 1) / chunk);
  if (pl.nsplit < 1) pl.nsplit = 1;
  pl.inline_merge = pl.nsplit > 1 && pairs % 8 == 0 && pairs * (int64_t)sizeof(int) <= kDecOpCtrOffset &&
                    kDecInlineMerge;
  const size_t slots = (size_t)(B * Hq * pl.nsplit);
  if (pl.nsplit == 1) {
    pl.o_bytes = pl.ml_bytes = 0;
    pl.ws_bytes = 16;
  } else {
    // The size is the in-kernel merge layout's whatever the mode, so a call
    // that falls back to the merge kernel (placement check below) fits too.
    // One arrival counter per (batch, KV head) pair in a fixed region at the
    // start (calls of every shape and mode keep partials out of it), then
    // slots of D partial outputs + m + l padded to whole 128-byte lines.
    pl.ws_bytes = kDecCounterBytes + slots * (size_t)(D + 32) * sizeof(float);
    use_merge_layout(pl, slots, D, pl.inline_merge);
  }
  return pl;
}

template <typename T, int D, int G>
static void launch_decode_g(const AttnArgs &a, dim3 grid, const int *seqlens, int L, float *ws_o,
                            float *ws_ml, int *counters, const DecodePlan &pl, const DecodeFuse &fz,
                            hipStream_t st) {
  const DecodeOproj none{};
  // The matrix-core kernel from two heads per KV head on; one head leaves its
  // products too little to do (64 sequences of 64-4000 keys, 8 / 8 heads, 88
  // us by the VALU kernel, 100 us by it). The fused prologue is the VALU
  // kernel's only.
  const bool mfma = G >= 2 && !fz.qkv;
  if (mfma) {
    attn_decode_mfma_kernel<T, D><<<grid, dim3(256), 0, st>>>(a, seqlens, L, ws_o, ws_ml, pl.nsplit,
                                                              inv_of(pl.nsplit), inv_of(a.Hkv), counters);
  } else {
    constexpr int NW = G <= 2 ? kDecBigNW : 4; // as plan_decode
    attn_decode_kernel<T, D, G, NW><<<grid, dim3(64 * NW), 0, st>>>(
        a, seqlens, L, ws_o, ws_ml, pl.nsplit, inv_of(pl.nsplit), inv_of(a.Hkv), fz, counters, none);
  }
  if (pl.nsplit > 1 && !counters)
    attn_decode_merge_kernel<T, D, G><<<dim3(a.Hkv, a.B), dim3(G * D), 0, st>>>(
        a, seqlens, L, mfma ? 4 * kSplitTile<D> : pl.nw * (kWave / (D / 8)) * kDecU, ws_o,
        ws_ml, pl.nsplit,
        inv_of(pl.nsplit));
}

template <typename T, int D>
static void launch_decode_d(const AttnArgs &a, int G, dim3 grid, const int *seqlens, int L,
                            float *ws_o, float *ws_ml, int *counters, const DecodePlan &pl,
                            const DecodeFuse &fz, hipStream_t st) {
  switch (G) {
  case 1: launch_decode_g<T, D, 1>(a, grid, seqlens, L, ws_o, ws_ml, counters, pl, fz, st); break;
  case 2: launch_decode_g<T, D, 2>(a, grid, seqlens, L, ws_o, ws_ml, counters, pl, fz, st); break;
  case 3: launch_decode_g<T, D, 3>(a, grid, seqlens, L, ws_o, ws_ml, counters, pl, fz, st); break;
  case 4: launch_decode_g<T, D, 4>(a, grid, seqlens, L, ws_o, ws_ml, counters, pl, fz, st); break;
  case 5: launch_decode_g<T, D, 5>(a, grid, seqlens, L, ws_o, ws_ml, counters, pl, fz, st); break;
  case 6: launch_decode_g<T, D, 6>(a, grid, seqlens, L, ws_o, ws_ml, counters, pl, fz, st); break;
  case 7: launch_decode_g<T, D, 7>(a, grid, seqlens, L, ws_o, ws_ml, counters, pl, fz, st); break;
  default: launch_decode_g<T, D, 8>(a, grid, seqlens, L, ws_o, ws_ml, counters, pl, fz, st); break;
  }
}

template <typename T>
static void launch_decode(const AttnArgs &a, int64_t D, int G, dim3 grid, const int *seqlens,
                          int L, float *ws_o, float *ws_ml, int *counters, const DecodePlan &pl,
                          const DecodeFuse &fz, hipStream_t st) {
  if (D == 128) launch_decode_d<T, 128>(a, G, grid, seqlens, L, ws_o, ws_ml, counters, pl, fz, st);
  else launch_decode_d<T, 64>(a, G, grid, seqlens, L, ws_o, ws_ml, counters, pl, fz, st);
}

} // namespace tpp

using namespace tpp;

static AttnArgs make_args(const void *q, const void *k, const void *v, void *o,
                          const int64_t *qs, const int64_t *ks, const int64_t *vs,
                          const int64_t *os, int64_t B, int64_t Sq, int64_t Sk, int64_t Hq,
                          int64_t Hkv, int64_t D, float scale, int left, int right) {
  AttnArgs a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.o = o;
  a.q_sb = qs[0], a.q_ss = qs[1], a.q_sh = qs[2];
  a.k_sb = ks[0], a.k_ss = ks[1], a.k_sh = ks[2];
  a.v_sb = vs[0], a.v_ss = vs[1], a.v_sh = vs[2];
  a.o_sb = os[0], a.o_ss = os[1], a.o_sh = os[2];
  a.B = (int)B, a.Sq = (int)Sq, a.Sk = (int)Sk, a.Hq = (int)Hq, a.Hkv = (int)Hkv;
  const float sc = scale > 0.f ? scale : 1.0f / sqrtf((float)D);
  a.scale_log2 = sc * kLog2e;
  a.left = left;
  a.right = right;
  return a;
}

extern "C" size_t tpp_attn_prefill_workspace_size(int64_t B, int64_t Sq, int64_t Sk, int64_t Hq,
                                                  int64_t Hkv, int64_t D, int causal,
                                                  int window_left, int window_right) {
  if (B < 1 || Sq < 1 || Sk < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv != 0 || (D != 64 && D != 128) ||
      B > 0x7fffffff || Sq > 0x7fffffff || Sk > 0x7fffffff)
    return 0;
  const int right = causal ? 0 : (window_right < 0 ? -1 : window_right);
  return plan_prefill(B, Sq, Sk, Hq, Hkv, D, window_left < 0 ? -1 : window_left, right, true).ws_bytes;
}

extern "C" int tpp_attn_prefill_chunks(int64_t B, int64_t Sq, int64_t Sk, int64_t Hq, int64_t Hkv, int64_t D,
                                       int causal, int window_left, int window_right, int32_t *dims,
                                       int32_t *ranges, int64_t capacity) {
  const char *name = "tpp_attn_prefill_chunks";
  if (!dims) return set_error(TPP_E_INVALID, "%s: null pointer argument", name);
  if (B < 1 || Sq < 1 || Sk < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv != 0 || B > 0x7fffffff || Sq > 0x7fffffff ||
      Sk > 0x7fffffff)
    return set_error(TPP_E_INVALID, "%s: invalid shapes", name);
  const int right = causal ? 0 : (window_right < 0 ? -1 : window_right), left = window_left < 0 ? -1 : window_left;
  dims[0] = dims[1] = dims[2] = dims[3] = 0;
  if (D != 64 && D != 128) return TPP_OK;
  const PrefillPlan pl = plan_prefill(B, Sq, Sk, Hq, Hkv, D, left, right, true);
  if (!pl.split) return TPP_OK;
  const int ql = 64 / pl.hpb, kt = D == 128 ? kSplitTile<128> : kSplitTile<64>;
  const int64_t nqt = (Sq + ql - 1) / ql, each = 1 + 2 * (int64_t)pl.nsmax;
  dims[0] = ql, dims[1] = kt, dims[2] = (int32_t)nqt, dims[3] = pl.nsmax;
  if (!ranges || capacity < nqt * each) return TPP_OK;
  for (int64_t t = 0; t < nqt; ++t, ranges += each) {
    const int64_t q0 = t * ql, last = (q0 + ql < Sq ? q0 + ql : Sq) - 1;
    const KeyBand kb = key_band((int)q0, (int)last, (int)Sq, (int)Sk, left, right, kt);
    ranges[0] = key_chunks(kb, pl.ct, pl.nsmax);
    for (int c = 0; c < pl.nsmax; ++c) {
      const KeyBand r = key_chunk(kb, c, pl.ct, pl.nsmax);
      ranges[1 + 2 * c] = r.t_begin, ranges[2 + 2 * c] = r.t_end;
    }
  }
  return TPP_OK;
}

extern "C" int tpp_attn_prefill_ws(const void *q, const void *k, const void *v, void *o,
                                   const int64_t *q_strides, const int64_t *k_strides,
                                   const int64_t *v_strides, const int64_t *o_strides, int64_t B,
                                   int64_t Sq, int64_t Sk, int64_t Hq, int64_t Hkv, int64_t D,
                                   float softmax_scale, int causal, int window_left,
                                   int window_right, int dtype, void *workspace, size_t ws_bytes,
                                   void *stream) {
  const char *name = "tpp_attn_prefill";
  if (!q_strides || !k_strides || !v_strides || !o_strides)
    return set_error(TPP_E_INVALID, "%s: null stride array", name);
  if (B > 0x7fffffff || Sq > 0x7fffffff || Sk > 0x7fffffff)
    return set_error(TPP_E_UNSUPPORTED, "%s: dimension too large", name);
  if (workspace && !aligned16(workspace))
    return set_error(TPP_E_WORKSPACE, "%s: the workspace must be 16-byte aligned", name);
  const int right = causal ? 0 : (window_right < 0 ? -1 : window_right);
  const int left = window_left < 0 ? -1 : window_left;
  AttnArgs a = make_args(q, k, v, o, q_strides, k_strides, v_strides, o_strides, B, Sq, Sk, Hq,
                         Hkv, D, softmax_scale, left, right);
  if (int e = check_attn(name, a, D)) return e;
  hipStream_t st = as_stream(stream);
  return TPP_DISPATCH_HALF(dtype, [&] { return launch_prefill<T>(a, D, workspace, ws_bytes, st, name); });
}

extern "C" int tpp_attn_prefill(const void *q, const void *k, const void *v, void *o,
                                const int64_t *q_strides, const int64_t *k_strides,
                                const int64_t *v_strides, const int64_t *o_strides, int64_t B,
                                int64_t Sq, int64_t Sk, int64_t Hq, int64_t Hkv, int64_t D,
                                float softmax_scale, int causal, int window_left,
                                int window_right, int dtype, void *stream) {
  return tpp_attn_prefill_ws(q, k, v, o, q_strides, k_strides, v_strides, o_strides, B, Sq, Sk, Hq,
                             Hkv, D, softmax_scale, causal, window_left, window_right, dtype, nullptr,
                             0, stream);
}

extern "C" size_t tpp_attn_decode_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                                                 int64_t Lmax) {
  return plan_decode(B, Hq, Hkv, D, Lmax).ws_bytes;
}

static int decode_impl(const char *name, AttnArgs &a, int64_t D, int64_t Lmax,
                       const int32_t *seqlens, const DecodeFuse &fz, int dtype, void *workspace,
                       size_t ws_bytes, void *stream, bool may_probe = true, int64_t len = -1) {
  if (int e = check_attn(name, a, D)) return e;
  if (a.B == 0) return TPP_OK;
  // the kernel reads cache row 0 even for empty sequences (clamped loads)
  if (Lmax < 1) return set_error(TPP_E_INVALID, "%s: the cache must hold at least one row", name);
  if (D != 64 && D != 128)
    return set_error(TPP_E_UNSUPPORTED, "%s: head_dim %lld not in {64, 128}", name, (long long)D);
  if (a.Hq / a.Hkv > kDecMaxG)
    return set_error(TPP_E_UNSUPPORTED, "%s: more than %d query heads per KV head", name,
                     kDecMaxG);
  if (!strides16(a)) return set_error(TPP_E_INVALID, "%s: 16-byte alignment required", name);
  DecodePlan pl = plan_decode(a.B, a.Hq, a.Hkv, D, Lmax);
  if (!workspace || ws_bytes < pl.ws_bytes || (uintptr_t)workspace % 128 != 0)
    return set_error(TPP_E_WORKSPACE, "%s: 128-byte aligned workspace of %zu bytes required",
                     name, pl.ws_bytes);
  hipStream_t st = as_stream(stream);
  if (pl.inline_merge && !xcd_grouping_holds(st, may_probe))
    use_merge_layout(pl, (size_t)a.B * a.Hq * pl.nsplit, D, false);
  int *counters = pl.inline_merge ? (int *)workspace : nullptr;
  float *ws_o = (float *)((char *)workspace + kDecCounterBytes);
  float *ws_ml = (float *)((char *)ws_o + pl.o_bytes);
  const dim3 grid = pl.inline_merge
                        ? dim3((unsigned)(pl.nsplit * a.Hkv * a.B))
                        : dim3((unsigned)pl.nsplit, (unsigned)a.Hkv, (unsigned)a.B);
  return TPP_DISPATCH_HALF(dtype, [&] {
    launch_decode<T>(a, D, a.Hq / a.Hkv, grid, seqlens, (int)(len < 0 ? Lmax : len), ws_o, ws_ml, counters, pl, fz,
                     st);
    return check_launch(name);
  });
}

extern "C" int tpp_attn_decode(const void *q, const void *k_cache, const void *v_cache, void *o,
                               const int64_t *q_strides, const int64_t *k_strides,
                               const int64_t *v_strides, const int64_t *o_strides,
                               const int32_t *seqlens, int64_t B, int64_t Hq, int64_t Hkv,
                               int64_t D, int64_t Lmax, float softmax_scale, int window_left,
                               int dtype, void *workspace, size_t ws_bytes, void *stream) {
  const char *name = "tpp_attn_decode";
  if (!q_strides || !k_strides || !v_strides || !o_strides)
    return set_error(TPP_E_INVALID, "%s: null stride array", name);
  if (B > 0xffff || Hkv > 0xffff || Lmax > 0x7fffffff)
    return set_error(TPP_E_UNSUPPORTED, "%s: dimension too large", name);
  AttnArgs a = make_args(q, k_cache, v_cache, o, q_strides, k_strides, v_strides, o_strides, B,
                         1, Lmax, Hq, Hkv, D, softmax_scale, window_left < 0 ? -1 : window_left,
                         0);
  DecodeFuse fz{};
  return decode_impl(name, a, D, Lmax, seqlens, fz, dtype, workspace, ws_bytes, stream);
}

// ---- allocation-free decode ------------------------------------------------
// tpp_attn_decode_noalloc runs the decode kernels on a file-scope device
// array instead of a caller workspace, for callers that cannot allocate. Each
// device holds its own copy of `scratch`; its address on a device comes from
// hipGetSymbolAddress at the first call with that device current (the host
// symbol itself is not a device address) and is kept per device. The first
// call also zeroes the arrival-counter region with a fill kernel on the
// caller's stream (every call leaves it at zero again). Calls on one device
// share the array: calls that overlap on one GPU race.
constexpr size_t kNoAllocScratchBytes = (size_t)4 << 20; // plans up to this many bytes
static __device__ __align__(256) unsigned char scratch[kNoAllocScratchBytes];
static void *g_scratch_ptr[64];
static std::mutex g_scratch_mu;

__global__ __launch_bounds__(256) void zero_words_kernel(int *__restrict__ p, int n) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) p[i] = 0;
}

static int noalloc_scratch(const char *name, hipStream_t st, void **out) {
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) {
    (void)hipGetLastError();
    return set_error(TPP_E_LAUNCH, "%s: no current device", name);
  }
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (!g_scratch_ptr[dev]) {
    void *ptr = nullptr;
    hipError_t e = hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch));
    if (e != hipSuccess || !ptr) {
      (void)hipGetLastError();
      return set_error(TPP_E_LAUNCH, "%s: hipGetSymbolAddress(scratch) failed: %s", name,
                       hipGetErrorString(e));
    }
    constexpr int words = (int)(kDecCounterBytes / 4);
    zero_words_kernel<<<dim3((words + 255) / 256), dim3(256), 0, st>>>((int *)ptr, words);
    if (int rc = check_launch(name)) return rc;
    g_scratch_ptr[dev] = ptr;
  }
  *out = g_scratch_ptr[dev];
  return TPP_OK;
}

extern "C" int tpp_attn_decode_noalloc(const void *q, const void *k_cache, const void *v_cache,
                                       void *o, const int64_t *q_strides,
                                       const int64_t *k_strides, const int64_t *v_strides,
                                       const int64_t *o_strides, const int32_t *seqlens,
                                       int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                                       int64_t Lmax, float softmax_scale, int window_left,
                                       int dtype, void *stream) {
  const char *name = "tpp_attn_decode_noalloc";
  if (!q_strides || !k_strides || !v_strides || !o_strides)
    return set_error(TPP_E_INVALID, "%s: null stride array", name);
  if (B > 0xffff || Hkv > 0xffff || Lmax > 0x7fffffff)
    return set_error(TPP_E_UNSUPPORTED, "%s: dimension too large", name);
  AttnArgs a = make_args(q, k_cache, v_cache, o, q_strides, k_strides, v_strides, o_strides, B,
                         1, Lmax, Hq, Hkv, D, softmax_scale, window_left < 0 ? -1 : window_left,
                         0);
  if (int e = check_attn(name, a, D)) return e;
  if (a.B == 0) return TPP_OK;
  const size_t need = plan_decode(B, Hq, Hkv, D, Lmax).ws_bytes;
  if (need > kNoAllocScratchBytes)
    return set_error(TPP_E_UNSUPPORTED,
                     "%s: this shape needs %zu bytes of scratch, more than the %zu-byte static "
                     "array (use tpp_attn_decode with a workspace)",
                     name, need, kNoAllocScratchBytes);
  void *ws = nullptr;
  if (int e = noalloc_scratch(name, as_stream(stream), &ws)) return e;
  DecodeFuse fz{};
  // no placement probe here (it reads back to the host): the in-kernel merge
  // is used once another decode call has verified the placement on this
  // device, the merge kernel until then
  return decode_impl(name, a, D, Lmax, seqlens, fz, dtype, ws, kNoAllocScratchBytes, stream,
                     false);
}

static int decode_fused(const char *name, const void *qkv, const void *q_norm_w, const void *k_norm_w,
                        const void *cos, const void *sin, int64_t ctx, int cs_dtype, float eps,
                        void *k_cache, void *v_cache, void *o, const int64_t *k_strides,
                        const int64_t *v_strides, const int64_t *o_strides, const int32_t *seqlens,
                        int64_t len, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t Lmax,
                        float softmax_scale, int window_left, int dtype, void *workspace,
                        size_t ws_bytes, void *stream) {
  if (!k_strides || !v_strides || !o_strides)
    return set_error(TPP_E_INVALID, "%s: null stride array", name);
  if (!qkv || !cos || !sin || (!seqlens && len < 0))
    return set_error(TPP_E_INVALID, "%s: qkv, cos, sin and seqlens are required", name);
  if (!aligned16(qkv) || !aligned16(cos) || !aligned16(sin) ||
      (q_norm_w && !aligned16(q_norm_w)) || (k_norm_w && !aligned16(k_norm_w)))
    return set_error(TPP_E_INVALID, "%s: 16-byte alignment required", name);
  if (cs_dtype != TPP_F16 && cs_dtype != TPP_BF16 && cs_dtype != TPP_F32)
    return set_error(TPP_E_UNSUPPORTED, "%s: cos/sin dtype", name);
  if (ctx <= 0 || ctx > 0x7fffffff) return set_error(TPP_E_INVALID, "%s: ctx", name);
  if (ctx < Lmax) // every cache position must have a table row (no clamping)
    return set_error(TPP_E_INVALID, "%s: cos/sin hold %lld positions, fewer than the cache length %lld",
                     name, (long long)ctx, (long long)Lmax);
  if (B > 0xffff || Hkv > 0xffff || Lmax > 0x7fffffff)
    return set_error(TPP_E_UNSUPPORTED, "%s: dimension too large", name);
  const int64_t qs[3] = {0, 0, 0};
  AttnArgs a = make_args(qkv, k_cache, v_cache, o, qs, k_strides, v_strides, o_strides, B, 1,
                         Lmax, Hq, Hkv, D, softmax_scale, window_left < 0 ? -1 : window_left, 0);
  DecodeFuse fz{qkv, q_norm_w, k_norm_w, cos, sin, cs_dtype, (int)ctx, eps};
  return decode_impl(name, a, D, Lmax, seqlens, fz, dtype, workspace, ws_bytes, stream, true, len);
}

extern "C" int tpp_attn_decode_fused(const void *qkv, const void *q_norm_w, const void *k_norm_w,
                                     const void *cos, const void *sin, int64_t ctx, int cs_dtype,
                                     float eps, void *k_cache, void *v_cache, void *o,
                                     const int64_t *k_strides, const int64_t *v_strides,
                                     const int64_t *o_strides, const int32_t *seqlens, int64_t B,
                                     int64_t Hq, int64_t Hkv, int64_t D, int64_t Lmax,
                                     float softmax_scale, int window_left, int dtype,
                                     void *workspace, size_t ws_bytes, void *stream) {
  return decode_fused("tpp_attn_decode_fused", qkv, q_norm_w, k_norm_w, cos, sin, ctx, cs_dtype, eps,
                      k_cache, v_cache, o, k_strides, v_strides, o_strides, seqlens, -1, B, Hq, Hkv, D,
                      Lmax, softmax_scale, window_left, dtype, workspace, ws_bytes, stream);
}

extern "C" int tpp_attn_decode_fused_at(const void *qkv, const void *q_norm_w, const void *k_norm_w,
                                        const void *cos, const void *sin, int64_t ctx, int cs_dtype,
                                        float eps, void *k_cache, void *v_cache, void *o,
                                        const int64_t *k_strides, const int64_t *v_strides,
                                        const int64_t *o_strides, int64_t position, int64_t B,
                                        int64_t Hq, int64_t Hkv, int64_t D, int64_t Lmax,
                                        float softmax_scale, int window_left, int dtype,
                                        void *workspace, size_t ws_bytes, void *stream) {
  const char *name = "tpp_attn_decode_fused_at";
  if (position < 0 || position >= Lmax)
    return set_error(TPP_E_INVALID, "%s: position %lld outside the cache", name, (long long)position);
  return decode_fused(name, qkv, q_norm_w, k_norm_w, cos, sin, ctx, cs_dtype, eps, k_cache, v_cache, o,
                      k_strides, v_strides, o_strides, nullptr, position + 1, B, Hq, Hkv, D, Lmax,
                      softmax_scale, window_left, dtype, workspace, ws_bytes, stream);
}

// ---- decode attention + output projection + residual add -------------------
// The OP kernel's plan: one workgroup per CU (Hkv = 8 KV heads x B sequences
// x 32 / B splits = 256), 128-key load batches dealt evenly to the splits by
// the sequence's length (some may hold no key). Workspace: the counters region (the projection's
// counters at kDecOpCtrOffset), the split partial slots, then the fp32
// per-XCD partial projections [8][B][E].
static bool oproj_shape(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t E) {
  return Hkv == kOpXcds && D == 128 && (Hq == 8 || Hq == 16) && E == kOpPerXcd * kOpCols &&
         (B == 1 || B == 2 || B == 4 || B == 8 || B == 16);
}

struct OprojPlan {
  int nsplit;
  size_t part_off, ws_bytes;
};

static OprojPlan plan_oproj(int64_t B, int64_t Hq, int64_t D, int64_t E) {
  OprojPlan pl{};
  pl.nsplit = (int)(kOpPerXcd / B);
  pl.part_off = (size_t)kDecCounterBytes + (size_t)(B * Hq * pl.nsplit) * (size_t)(D + 32) * sizeof(float);
  pl.ws_bytes = pl.part_off + (size_t)kOpXcds * B * E * sizeof(float);
  return pl;
}

extern "C" size_t tpp_attn_decode_oproj_workspace_size(int64_t B, int64_t Hq, int64_t Hkv,
                                                       int64_t D, int64_t Lmax, int64_t E) {
  const size_t plain = plan_decode(B, Hq, Hkv, D, Lmax).ws_bytes;
  if (!oproj_shape(B, Hq, Hkv, D, E) || Lmax < 1) return plain;
  const size_t op = plan_oproj(B, Hq, D, E).ws_bytes;
  return op > plain ? op : plain;
}

extern "C" int tpp_attn_decode_oproj(const void *qkv, const void *q_norm_w, const void *k_norm_w,
                                     const void *cos, const void *sin, int64_t ctx, int cs_dtype,
                                     float eps, void *k_cache, void *v_cache, void *o,
                                     const int64_t *k_strides, const int64_t *v_strides,
                                     const int32_t *seqlens, const void *w_o, void *residual,
                                     int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t Lmax,
                                     int64_t E, float softmax_scale, int window_left, int dtype,
                                     void *workspace, size_t ws_bytes, void *stream) {
  const char *name = "tpp_attn_decode_oproj";
  if (!w_o || !residual || !o) return set_error(TPP_E_INVALID, "%s: null pointer argument", name);
  if (!aligned16(w_o) || !aligned16(residual) || !aligned16(o))
    return set_error(TPP_E_INVALID, "%s: 16-byte alignment required", name);
  if (E <= 0 || B <= 0 || B > 16)
    return set_error(TPP_E_INVALID, "%s: need 1 <= B <= 16 and E > 0", name);
  const int64_t os[3] = {Hq * D, Hq * D, D}; // o: contiguous [B, 1, Hq, D]
  hipStream_t st = as_stream(stream);
  const size_t need = tpp_attn_decode_oproj_workspace_size(B, Hq, Hkv, D, Lmax, E);
  if (!workspace || ws_bytes < need || (uintptr_t)workspace % 128 != 0)
    return set_error(TPP_E_WORKSPACE, "%s: 128-byte aligned workspace of %zu bytes required", name,
                     need);
  const bool fold = oproj_shape(B, Hq, Hkv, D, E) && half_type(dtype) &&
                    device_cu_count() == kOpXcds * kOpPerXcd && xcd_grouping_holds(st, true);
  if (!fold) {
    // two launches: fused decode attention into o, then the projection GEMV
    // with the residual add
    if (int rc = tpp_attn_decode_fused(qkv, q_norm_w, k_norm_w, cos, sin, ctx, cs_dtype, eps,
                                       k_cache, v_cache, o, k_strides, v_strides, os, seqlens, B,
                                       Hq, Hkv, D, Lmax, softmax_scale, window_left, dtype,
                                       workspace, ws_bytes, stream))
      return rc;
    return tpp_gemv_fused(o, nullptr, 0.f, w_o, nullptr, residual, B, E, Hq * D, 0, dtype, stream);
  }
  if (!k_strides || !v_strides) return set_error(TPP_E_INVALID, "%s: null stride array", name);
  if (!qkv || !cos || !sin || !seqlens)
    return set_error(TPP_E_INVALID, "%s: qkv, cos, sin and seqlens are required", name);
  if (!aligned16(qkv) || !aligned16(cos) || !aligned16(sin) ||
      (q_norm_w && !aligned16(q_norm_w)) || (k_norm_w && !aligned16(k_norm_w)))
    return set_error(TPP_E_INVALID, "%s: 16-byte alignment required", name);
  if (cs_dtype != TPP_F16 && cs_dtype != TPP_BF16 && cs_dtype != TPP_F32)
    return set_error(TPP_E_UNSUPPORTED, "%s: cos/sin dtype", name);
  if (ctx < Lmax || ctx > 0x7fffffff)
    return set_error(TPP_E_INVALID, "%s: cos/sin hold %lld positions, fewer than the cache length %lld",
                     name, (long long)ctx, (long long)Lmax);
  if (Lmax < 1 || Lmax > 0x7fffffff) return set_error(TPP_E_INVALID, "%s: cache length", name);
  const int64_t qs[3] = {0, 0, 0};
  AttnArgs a = make_args(qkv, k_cache, v_cache, o, qs, k_strides, v_strides, os, B, 1, Lmax, Hq,
                         Hkv, D, softmax_scale, window_left < 0 ? -1 : window_left, 0);
  if (int rc = check_attn(name, a, D)) return rc;
  if (!strides16(a)) return set_error(TPP_E_INVALID, "%s: 16-byte alignment required", name);
  const OprojPlan pl = plan_oproj(B, Hq, D, E);
  DecodeFuse fz{qkv, q_norm_w, k_norm_w, cos, sin, cs_dtype, (int)ctx, eps};
  char *ws = (char *)workspace;
  DecodeOproj op{w_o, residual, (int *)(ws + kDecOpCtrOffset), (float *)(ws + pl.part_off), (int)E};
  float *ws_o = (float *)(ws + kDecCounterBytes);
  const dim3 grid(kOpXcds * kOpPerXcd), block(64 * kDecBigNW);
  return TPP_DISPATCH_HALF(dtype, [&] {
    if (Hq == 16)
      attn_decode_kernel<T, 128, 2, kDecBigNW, true><<<grid, block, 0, st>>>(
          a, seqlens, (int)Lmax, ws_o, nullptr, pl.nsplit, inv_of(pl.nsplit), inv_of(a.Hkv), fz, (int *)ws, op);
    else
      attn_decode_kernel<T, 128, 1, kDecBigNW, true><<<grid, block, 0, st>>>(
          a, seqlens, (int)Lmax, ws_o, nullptr, pl.nsplit, inv_of(pl.nsplit), inv_of(a.Hkv), fz, (int *)ws, op);
    return check_launch(name);
  });
}

extern "C" int tpp_attn_decode_oproj_sync_errors(void *workspace, int *out, void *stream) {
  const char *name = "tpp_attn_decode_oproj_sync_errors";
  if (!workspace || !out) return set_error(TPP_E_INVALID, "%s: null pointer", name);
  hipStream_t st = as_stream(stream);
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(st, &cs) != hipSuccess || cs != hipStreamCaptureStatusNone) {
    (void)hipGetLastError();
    return set_error(TPP_E_INVALID, "%s: not callable while the stream is being captured", name);
  }
  char *ctr = (char *)workspace + kDecOpCtrOffset;
  int flag = 0;
  if (hipMemcpyAsync(&flag, ctr + kOpErr * sizeof(int), sizeof(int), hipMemcpyDeviceToHost, st) !=
          hipSuccess ||
      hipStreamSynchronize(st) != hipSuccess) {
    (void)hipGetLastError();
    return set_error(TPP_E_LAUNCH, "%s: copy failed", name);
  }
  // a launch that gave up leaves the counters in an unknown state: zero them
  if (flag && (hipMemsetAsync(ctr, 0, (kOpErr + 32) * sizeof(int), st) != hipSuccess ||
               hipStreamSynchronize(st) != hipSuccess)) {
    (void)hipGetLastError();
    return set_error(TPP_E_LAUNCH, "%s: clearing the counters failed", name);
  }
  *out = flag;
  return TPP_OK;
}
