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
//  * few tiles: attn_prefill_split_kernel, tiles of 32 queries of two heads whose keys the
//    block's four pairs of waves share out. Each block finds its sequence by a scan of the
//    lengths, so it is one launch.
//  * else attn_prefill_kernel, one block a CU, 128 queries of two heads (or 64 of four, 256 of
//    one) a tile. Its static dealing of tiles to blocks wants them from the heaviest to the
//    lightest: packed_plan_kernel sorts them first.
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
  int sum = n;
#pragma unroll
  for (int sh = 1; sh < kWave; sh <<= 1) {
    const int o = __shfl_up(sum, sh, kWave);
    if (lane >= sh) sum += o;
  }
  if (lane == kWave - 1) s_sum[w] = sum;
  __syncthreads();
  for (int i = 0; i < w; ++i) sum += s_sum[i];
  s_at[tid] = sum - n;
  if (tid == 1023) plan[0] = min(sum, room);
  __syncthreads();
  each([&](const PackedSeq &s, int t, int bin) {
    const int at = atomicAdd(&s_at[bin], 1); // (the order inside a bin changes no result)
    if (at >= room) return;                   // (lengths that do not ascend)
    int32_t *it = plan + kPlanHead + at * kPlanItem;
    it[0] = s.q0, it[1] = t * QL, it[2] = s.Sq, it[3] = s.k0, it[4] = s.Sk;
  });
}

// How a call is cut: query heads of a tile, queries a tile, the most tiles there can be, and
// whether tiles are of the kernel that splits keys in the block.
struct PackedPlan {
  bool tiles, split;
  int hpb, QL;
  int64_t most;
};
static PackedPlan packed_plan(int64_t B, int64_t Nq, int64_t Hq, int64_t Hkv, int64_t D) {
  PackedPlan pl = {};
  if (D != 64 && D != 128) return pl;
  pl.tiles = true;
  const int64_t G = Hq / Hkv;
  const int cus = device_cu_count() > 0 ? device_cu_count() : 256;
  auto most = [&](int64_t QL) { return Nq / QL + (B + 2 < Nq ? B + 2 : Nq); };
  pl.hpb = G % 2 == 0 ? 2 : 1, pl.QL = 64 / pl.hpb;
  pl.split = most(pl.QL) * (Hq / pl.hpb) <= 2 * cus;
  if (!pl.split) {
    pl.hpb = G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1;
    pl.QL = kPrefillWaves / pl.hpb * 32;
  }
  pl.most = most(pl.QL);
  return pl;
}

} // namespace tpp

using namespace tpp;

extern "C" size_t tpp_attn_packed_workspace_size(int64_t B, int64_t Nq, int64_t Nk, int64_t Hq, int64_t Hkv, int64_t D) {
  if (B < 0 || Nq <= 0 || Hkv <= 0 || Hq <= 0) return 0;
  const PackedPlan pl = packed_plan(B, Nq, Hq, Hkv, D);
  return pl.tiles && !pl.split ? (size_t)(kPlanHead + pl.most * kPlanItem) * sizeof(int32_t) : 0;
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
  // a window that reaches past every key is none (and query + window stays below 2^31)
  auto window = [&](int x) { return x < 0 || x >= Nq + Nk ? -1 : x; };
  a.left = window(window_left), a.right = causal ? 0 : window(window_right);
  a.fill = fill;
  hipStream_t st = as_stream(stream);
  // the matrix-core kernels: whole 16-byte rows, a tile's rows by 32-bit byte offsets
  uint64_t low = (uint64_t)(uintptr_t)q | (uint64_t)(uintptr_t)k | (uint64_t)(uintptr_t)v | (uint64_t)(uintptr_t)o;
  for (const int64_t x : {a.q_ss, a.q_sh, a.k_ss, a.k_sh, a.v_ss, a.v_sh, a.o_ss, a.o_sh}) low |= (uint64_t)(x * 2);
  PackedPlan pl = packed_plan(B, Nq, Hq, Hkv, D);
  const bool fits = !(low & 15) && a.k_ss >= 0 && a.v_ss >= 0 && kKvTile * a.k_ss * 2 < (1LL << 31) &&
                    kKvTile * a.v_ss * 2 < (1LL << 31) && pl.most * Hq < (1LL << 31);
  if (!pl.tiles || !fits)
    return TPP_DISPATCH_HALF(dtype, [&] {
      packed_generic_kernel<T><<<dim3((unsigned)Nq, (unsigned)Hq), dim3(64), 0, st>>>(a, (int)D);
      return check_launch(name);
    });
  const int64_t items = pl.most * (Hq / pl.hpb);
  if (!pl.split) {
    if (!workspace || !aligned16(workspace) || ws_bytes < tpp_attn_packed_workspace_size(B, Nq, Nk, Hq, Hkv, D))
      return set_error(TPP_E_WORKSPACE, "%s: workspace missing, unaligned or too small", name);
    a.plan = (const int32_t *)workspace;
    packed_plan_kernel<<<dim3(1), dim3(1024), 0, st>>>(a, pl.QL, (int32_t *)workspace, (int)pl.most);
  }
  return TPP_DISPATCH_HALF(dtype, [&] {
    auto go = [&](auto dd) {
      constexpr int DD = decltype(dd)::value;
      if (pl.split) {
        attn_prefill_split_kernel<T, DD><<<dim3((unsigned)items), dim3(512), 0, st>>>(a, pl.hpb, (int)pl.most, 1, nullptr, nullptr);
      } else {
        const int cus = device_cu_count() > 0 ? device_cu_count() : 256;
        attn_prefill_kernel<T, DD, kPrefillQG, kPrefillWaves>
            <<<dim3((unsigned)(items < cus ? items : cus)), dim3(64 * kPrefillWaves), 0, st>>>(a, pl.hpb);
      }
    };
    if (D == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 64>{});
    return check_launch(name);
  });
}
