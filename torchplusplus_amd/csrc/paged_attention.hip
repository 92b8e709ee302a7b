// Attention of one new token a sequence over a cache held in pages:
//   o[b, h] = softmax_j(scale q[b, h] . K[j, h / G]) V[j, h / G],  j < seqlens[b],
// key j in row j % page_size of page block_tables[b, j / page_size] (and, in a window,
// j >= seqlens[b] - 1 - left). The positions of an entry that is no page (outside [0,
// pages)) are not seen. A row that sees nothing is 0, one whose scores are all -inf NaN.
#include "attn_row.hpp"
#include "tree_wave.hpp"

namespace tpp {

// TreeArgs with one token a sequence, {page, head, row} strides in k_s and v_s, and T = 1.
struct PagedArgs : TreeArgs {
  const int32_t *table;
  int64_t t_sb;
  int pages, lpage, left, lkt; // pages of 2^lpage rows; tiles of 2^lkt keys
  // of len positions: the first that is seen, the first tile's first, and the keys from there
  __device__ __forceinline__ int lowest(int len) const { return left >= 0 ? max(len - 1 - left, 0) : 0; }
  __device__ __forceinline__ int begin(int len) const { return lowest(len) >> lkt << lkt; }
  __device__ __forceinline__ int keys(int len) const { return max(len - begin(len), 1); } // (none: one split, of zeros)
  __device__ __forceinline__ int length(int b) const { return min(max(seqlens[b], 0), Lmax); }
};

// Any head size up to 256, any alignment: one wave per (sequence, head).
template <typename T> __global__ __launch_bounds__(64) void paged_generic_kernel(PagedArgs p, int D) {
  const int lane = lane_id(), h = blockIdx.x, b = blockIdx.y, hk = h / p.G;
  const int L = min(max(p.seqlens[b], 0), p.Lmax), lo = p.lowest(L);
  const int32_t *table = p.table + b * p.t_sb;
  AttnRow r;
  attn_row<T>(r, (const T *)p.q + b * p.q_s[0] + h * p.q_s[2], D, lo, L, p.scale_log2,
              [&](int j, const T *&k, const T *&v) {
                const int pg = __builtin_amdgcn_readfirstlane(table[j >> p.lpage]);
                if (pg < 0 || pg >= p.pages) return false;
                const int64_t row = j & ((1 << p.lpage) - 1);
                k = (const T *)p.k + pg * p.k_s[0] + hk * p.k_s[1] + row * p.k_s[2];
                v = (const T *)p.v + pg * p.v_s[0] + hk * p.v_s[1] + row * p.v_s[2];
                return true;
              });
  T *op = (T *)p.o + b * p.o_s[0] + h * p.o_s[2];
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (c * 64 + lane < D) op[c * 64 + lane] = from_f32<T>(r.out(c));
}

// ---------------------------------------------------------------------------
// Head sizes 64 and 128, 16-byte rows: TreeWave's products and softmax (tree_wave.hpp), the
// G query rows of a KV head in one group of 16 or two, a block's four waves over one split of
// the sequence's keys, each streaming its own tiles of 32 (D = 128) or 64 keys by LDS-DMA.
//
// A page holds whole groups of 16 keys and a DMA instruction brings 4 or 8 keys, so one page
// an instruction: its address is that page's, uniform, plus lane offsets fixed for the launch.
// The table's entries of a tile's groups are in the wave's first lanes; they come by LDS-DMA
// a tile ahead, between that tile's K and V (a load into registers was waited for at once, and
// K with it, where its value is carried around the loop).
//
// HBM bounds it where the cache is long: 32 sequences of 100 to 4096 positions, 146 MB, 30.0 us
// (4.9 TB/s), two of 60000 to 100000, 328 MB, 57 us (5.8); one of 700, 2.9 MB, is its launch and
// trips to memory, 6.9 us.
// ---------------------------------------------------------------------------
constexpr int kPagedDealt = 512; // sequences whose lengths a block looks at

// What tile keys kb .. are shown of: pages that exist, positions from the window's first on.
struct PagedShown {
  unsigned groups; // bit g: keys 16 g .. of the tile have a page
  int rel;         // the window's first key in the tile
  bool any;
  __device__ __forceinline__ unsigned word(int c) const {
    const unsigned two = groups >> (2 * c) & 3u, r = (unsigned)(rel - 32 * c);
    return ((two & 1 ? 0xffffu : 0u) | (two & 2 ? 0xffff0000u : 0u)) &
           (rel - 32 * c <= 0 ? ~0u : r >= 32u ? 0u : ~0u << r);
  }
};

// A sequence's splits: runs of `per` batches of 2^(lkt + 2) keys, `n` of them, the first the
// head's `at`-th.
struct PagedDeal {
  int b, at, n, per, batches;
};
// The splits are dealt to the sequences by their lengths: all of a head's keys into runs of one
// length, the least that makes `target` of them or fewer (or nearly: a sequence has one at
// least, and the search is short), each sequence's as even as its batches allow, and at most
// `most` of them, for one block to merge. Then every block has about the same to read, where
// one number of splits for all left the longest sequence's blocks reading when the others were
// done: 32 sequences of 100 to 4096 keys, 36.6 -> 29.9 us. By a whole wave, for split `e` of a
// head, or, FIND = false, for sequence `e` (b < 0: there is none).
// a / n rounded up, for a and n up to 2^20 (a table's positions are limited to so many batches):
// (a + n - 1/2) / n is 1 / (2 n) off a whole number at least, its error, 2^-22 of it, less.
// (An integer division is ~30 dependent instructions, and four stood ahead of the first key.)
__device__ __forceinline__ int div_up(int a, int n) {
  return (int)(((float)(a + n) - 0.5f) * __builtin_amdgcn_rcpf((float)n));
}
__device__ __forceinline__ PagedDeal paged_runs(int b, int at, int batches, int per) {
  PagedDeal d = {b, at, div_up(batches, per), 0, batches};
  d.per = div_up(batches, d.n);
  d.n = div_up(batches, d.per); // (evened out they may be fewer)
  return d;
}
template <bool FIND> __device__ __forceinline__ PagedDeal paged_deal(const PagedArgs &p, int target, int most, int e) {
  constexpr int U = kPagedDealt / kWave;
  const int lane = lane_id(), lb = p.lkt + 2;
  int nb[U], total = 0;
  float longest = 0.f; // (batches)
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int b = u * kWave + lane;
    nb[u] = 0;
    if (b < p.B) nb[u] = (int)(((unsigned)p.keys(p.length(b)) + (1u << lb) - 1) >> lb);
    longest = fmaxf(longest, (float)nb[u]);
  }
  int sum[U], per = 0;
  auto scan = [&](int div) { // running numbers of runs of `div` batches, their sum
    int before = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u * kWave >= p.B) break;
      sum[u] = wave_scan(div_up(nb[u], div)) + before;
      before = __builtin_amdgcn_readlane(sum[u], kWave - 1);
    }
    return before;
  };
  total = scan(1);
  longest = row16_max(longest);
  const int top = (int)fmaxf(fmaxf(readlane_f32(longest, 0), readlane_f32(longest, 16)),
                             fmaxf(readlane_f32(longest, 32), readlane_f32(longest, 48)));
  per = max(min(max((total + target - 1) / target, div_up(top, most)), top), 1);
  for (int i = 0; scan(per) > target && i < 6; ++i) per += (per + 7) / 8;
  PagedDeal d = {-1, 0, 0, 1, 0};
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (u * kWave >= p.B || d.b >= 0) break;
    const unsigned long long hit = __ballot(FIND ? sum[u] > e && u * kWave + lane < p.B : u * kWave + lane == e);
    if (!hit) continue;
    const int l = __builtin_ctzll(hit);
    const int batches = __builtin_amdgcn_readlane(nb[u], l), n = div_up(batches, per);
    d = paged_runs(u * kWave + l, __builtin_amdgcn_readlane(sum[u], l) - n, batches, per);
  }
  return d;
}

// Block (qt, hk) = blockIdx.x, split blockIdx.y of the head, or, undealt (target 0), the whole
// of sequence blockIdx.y; `slots` splits a head at most.
template <typename T, int D, int NC>
__global__ __launch_bounds__(256, 2) void paged_tile_kernel(PagedArgs p, float *__restrict__ ws_o,
                                                            float *__restrict__ ws_ml, int target, int most,
                                                            int slots, unsigned hkv_inv, unsigned g_inv,
                                                            unsigned *__restrict__ arrived) {
  typedef TreeTile<0, D> TT;
  typedef TreeWave<T, 0, D, NC> W;
  constexpr int KT = TT::KT, NW = 4, STRIDE = NW * KT, NDMA = TT::TILEB / 1024, C4 = D / 4, ROWS = 16 * NC;
  constexpr int KPI = 64 / TT::UPR, NG = KT / 16; // keys of a DMA instruction, groups of 16 keys
  constexpr int SLOT = 2 * TT::TILEB > ROWS * D * 4 ? 2 * TT::TILEB : ROWS * D * 4;
  constexpr int kRing = NW * SLOT, kMerge = NC == 1 ? tree_merge_lds<D> : 0;
  __shared__ __attribute__((aligned(16))) char smem[kRing > kMerge ? kRing : kMerge];
  __shared__ float s_m[NW][ROWS], s_l[NW][ROWS];
  __shared__ unsigned s_entry[NW][64];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int u4 = lane >> 4, l16 = lane & 15;
  TreeBlock k = {};
  k.qt = div_inv(blockIdx.x, hkv_inv), k.hk = blockIdx.x - k.qt * p.Hkv;
  PagedDeal d = {(int)blockIdx.y, 0, 1, 1 << 30, 1};
  if (target && p.B > 1) {
    d = paged_deal<true>(p, target, most, blockIdx.y);
    if (d.b < 0 || (int)blockIdx.y - d.at >= d.n) return; // (the whole block)
  } else if (target) {
    d.b = 0; // its query rows need not wait for its length
  }
  k.b = d.b, k.pair = d.b * p.Hkv + k.hk;
  const int rows = p.G;
  W wv;
  int row0[NC], row[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) row0[i] = k.qt * ROWS + i * 16, row[i] = min(row0[i] + l16, rows - 1);
  wv.ask(p, k.b, k.hk, g_inv, row);
  const int len = __builtin_amdgcn_readfirstlane(p.length(k.b));
  const int lowest = p.lowest(len), begin = p.begin(len);
  if (target && p.B == 1) {
    const int batches = (int)((unsigned)(p.keys(len) + STRIDE - 1) / (unsigned)STRIDE);
    d = paged_runs(0, 0, batches, max(div_up(batches, target), div_up(batches, most)));
    if ((int)blockIdx.y >= d.n) return; // (the whole block)
  }
  k.split = target ? blockIdx.y - d.at : 0, k.live = d.n;
  const int c0 = begin + k.split * d.per * STRIDE; // (below 2^31, as two tiles on)
  const int k_end = (int)min((int64_t)c0 + (int64_t)d.per * STRIDE, (int64_t)len);
  const int first = c0 + w * KT;
  const int n = first < k_end ? (k_end - first + STRIDE - 1) / STRIDE : 0; // this wave's tiles

  const char *ks = (const char *)p.k + (int64_t)k.hk * p.k_s[1] * 2, *vs = (const char *)p.v + (int64_t)k.hk * p.v_s[1] * 2;
  const int32_t *const table = p.table + (int64_t)k.b * p.t_sb;
  char *const ring = smem + w * SLOT;
  unsigned koff[NDMA], voff[NDMA];
#pragma unroll
  for (int j = 0; j < NDMA; ++j) {
    const int kr = lane / TT::UPR, key = j * KPI + kr, u = lane % TT::UPR;
    koff[j] = (unsigned)(kr * (int)p.k_s[2] * 2 + ((u ^ TT::ksw(key)) << 4));
    voff[j] = (unsigned)(kr * (int)p.v_s[2] * 2 + ((u ^ TT::vsw(key)) << 4));
  }
  // the page of group lane % NG of the tile at kb (past the last key: the last key's)
  auto entry = [&](int kb) { return table + (min((kb >> 4) + (lane & (NG - 1)), (len - 1) >> 4) >> (p.lpage - 4)); };
  const int pmask = (1 << p.lpage) - 1;
  auto issue = [&](const char *head, const int64_t (&st)[3], const unsigned (&off)[NDMA], int kb, int page, char *dst,
                   auto swizzle) {
    auto dma = [&](int j, auto place) {
      const char *src = head + (int64_t)__builtin_amdgcn_readlane(page, j * KPI / 16) * st[0] * 2 + place(kb + j * KPI);
      __builtin_amdgcn_global_load_lds((const void *)src, (__attribute__((address_space(3))) void *)(dst + j * 1024), 16,
                                       0, kCpolNT);
    };
    if (kb + KT <= len) {
#pragma unroll
      for (int j = 0; j < NDMA; ++j) dma(j, [&](int key) { return (int64_t)(key & pmask) * st[2] * 2 + off[j]; });
    } else { // keys past the last read its row (masked)
      const int kr = lane / TT::UPR, u = lane % TT::UPR;
#pragma unroll
      for (int j = 0; j < NDMA; ++j)
        dma(j, [&](int key) {
          return (int64_t)(min(key + kr, len - 1) & pmask) * st[2] * 2 + ((u ^ swizzle(j * KPI + kr)) << 4);
        });
    }
  };
  // entries that are no page read page 0 (and are hidden)
  auto real = [&](int page) { return page >= 0 && page < p.pages; };
  auto shown = [&](int page) { return (unsigned)__ballot(real(page)) & ((1u << NG) - 1u); };
  auto issue_k = [&](int kb, int page) {
    issue(ks, p.k_s, koff, kb, real(page) ? page : 0, ring, [](int r) { return TT::ksw(r); });
  };
  auto issue_v = [&](int kb, int page) {
    issue(vs, p.v_s, voff, kb, real(page) ? page : 0, ring + TT::TILEB, [](int r) { return TT::vsw(r); });
  };
  auto issue_entry = [&](int kb) {
    __builtin_amdgcn_global_load_lds((const void *)entry(kb), (__attribute__((address_space(3))) void *)s_entry[w], 4, 0, 0);
  };
  int page = 0; // of this tile's groups
  unsigned groups = 0;
  bool saw = false;
  if (n > 0) page = *entry(first);
  // (waits for the query rows, which have come when the entries have: no tile's loads ahead)
  wv.begin(len > 0 ? 1ull : 0ull, lds_addr(ring), lds_addr(ring) + TT::TILEB, 0);
  if (n > 0) {
    issue_k(first, page);
    issue_entry(first + STRIDE); // (past the last tile: the last entry)
    issue_v(first, page);
    groups = shown(page);
  }
  const unsigned entry_at = lds_addr(s_entry[w]) + 4 * lane;
  for (int it = 0; it < n; ++it) {
    const int kb = first + it * STRIDE;
    const bool more = it + 1 < n;
    PagedShown mask;
    mask.groups = groups, mask.rel = lowest - kb;
    mask.any = groups != (1u << NG) - 1u || kb < lowest;
    saw = saw || groups >> (max(lowest - kb, 0) >> 4); // (a group of keys ahead of the window is none)
    vm_wait<NDMA>(); // this tile's K and the next one's entries landed, its V may be in flight
    float next = lds_read_b32<0>(entry_at);
    wv.step(p, kb, len - 1, 0, 0,
            [&] { // (the entries came ahead of the K fragments, which were waited for)
              asm volatile("" : "+v"(next));
              if (!more) return;
              page = __float_as_int(next), groups = shown(page);
              issue_k(kb + STRIDE, page);
              issue_entry(kb + 2 * STRIDE);
            },
            [&] { // the next K, and the entries behind it, may be in flight
              if (more) vm_wait<NDMA + 1>();
              else vm_wait<0>();
            },
            [&] { if (more) issue_v(kb + STRIDE, page); }, mask);
  }

  // The wave's rows, then the block's: chunk c (4 values) of row r at c ^ r. A wave that sees
  // no key has a weight of 1 on nothing below every score, one that sees scores of -inf alone
  // none, above that: a row of all holes is 0, one of -inf (and holes) 0 / 0.
  f32x4 *const part = reinterpret_cast<f32x4 *>(ring);
  const bool odd = wv.end(p) && saw;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int r = i * 16 + l16;
#pragma unroll
    for (int tt = 0; tt < W::NT; ++tt)
      part[r * C4 + ((tt * 4 + u4) ^ (r & (C4 - 1)))] = saw ? wv.o[i][tt] : f32x4{0.f, 0.f, 0.f, 0.f};
    if (u4 == 0) {
      s_m[w][r] = !saw ? -3.4e38f : wv.m[i] == -INFINITY ? -3e38f : wv.top(p, i);
      s_l[w][r] = saw ? wv.l[i] : 1.f;
    }
  }
  if (n > 0 && __any(odd))
    wv.again(p, k.b, k.hk,
             [&](int j, const char *&kr, const char *&vr) {
               const int pg = table[j >> p.lpage];
               if (pg < 0 || pg >= p.pages || j < lowest) return false;
               kr = ks + ((int64_t)pg * p.k_s[0] + (int64_t)(j & pmask) * p.k_s[2]) * 2;
               vr = vs + ((int64_t)pg * p.v_s[0] + (int64_t)(j & pmask) * p.v_s[2]) * 2;
               return true;
             },
             0, first, STRIDE, n, k_end, len - 1, g_inv, row0, rows, [&](int i, int q, int d, float x) {
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
    float ls = 0.f;
    f32x4 os = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ww = 0; ww < NW; ++ww) {
      const float cf = __builtin_amdgcn_exp2f(s_m[ww][q] - mx);
      ls += s_l[ww][q] * cf;
      const f32x4 pr = reinterpret_cast<const f32x4 *>(smem + ww * SLOT)[q * C4 + (c ^ (q & (C4 - 1)))];
#pragma unroll
      for (int e = 0; e < 4; ++e) os[e] += pr[e] * cf;
    }
    if (k.live == 1) {
      T *op = W::row_of((T *)p.o, p.o_s, p, k.b, k.hk, r, 0);
      typename VecT<T>::v4 ov;
      const float inv = 1.f / ls;
#pragma unroll
      for (int e = 0; e < 4; ++e) ov[e] = from_f32<T>(os[e] * inv);
      *reinterpret_cast<typename VecT<T>::v4 *>(op + c * 4) = ov;
    } else {
      const int64_t slot = ((int64_t)k.hk * rows + r) * slots + blockIdx.y;
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
    if (arrived && k.live > 1)
      tree_merge_here<T, D>(p, k, rows, (int64_t)k.hk * rows * slots + d.at, slots, ws_o, ws_ml, g_inv, arrived, smem);
}

// The splits of every row, as tree_merge_kernel, a row block of one sequence and KV head each.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedArgs p, const float *__restrict__ ws_o,
                                                          const float *__restrict__ ws_ml, int target, int most, int slots) {
  constexpr int C4 = D / 4, RPB = 256 / (C4 * kMergeParts);
  __shared__ f32x4 s_o[RPB * kMergeParts * C4];
  __shared__ float s_ml[RPB * kMergeParts * 2];
  const int grp = threadIdx.x / C4, q = grp / kMergeParts, g0 = grp % kMergeParts, c = threadIdx.x % C4;
  const int r = min((int)blockIdx.x * RPB + q, p.G - 1), hk = blockIdx.y, b = blockIdx.z;
  const PagedDeal d = paged_deal<false>(p, target, most, b);
  if (d.n == 1) return; // written by the tile kernel
  const int64_t slot = ((int64_t)hk * p.G + r) * slots + d.at;
  TreeMerge<1> mg;
  mg.begin();
  for (int s0 = 0; s0 < d.n; s0 += kMergeParts * kMergeAhead) {
    mg.template load<D, false>(ws_o, ws_ml, slot, c, s0, g0, 1, d.n - 1);
    mg.add(s0, g0, 1, d.n);
  }
  s_o[grp * C4 + c] = mg.o[0];
  if (c == 0) s_ml[grp * 2] = mg.m[0], s_ml[grp * 2 + 1] = mg.l[0];
  __syncthreads();
  if (g0 || (int)blockIdx.x * RPB + q >= p.G) return;
  T *op = (T *)p.o + (int64_t)b * p.o_s[0] + (int64_t)(hk * p.G + r) * p.o_s[2];
  *reinterpret_cast<typename VecT<T>::v4 *>(op + c * 4) =
      tree_merge_parts<T>(s_o + q * kMergeParts * C4 + c, C4, s_ml + q * kMergeParts * 2);
}

// How a call is cut: groups of 16 query rows a block, blocks of them a KV head, splits that a
// head is to have (0: one a sequence), that one of its sequences, and that there can be.
struct PagedPlan {
  int nc, qtiles, target, most, slots;
};
static PagedPlan paged_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t Lmax) {
  PagedPlan pl = {0, 0, 0, 0, 0};
  if (D != 64 && D != 128) return pl;
  const int64_t G = Hq / Hkv, stride = 4 * (D == 128 ? 32 : 64);
  pl.nc = G > 16 ? 2 : 1;
  pl.qtiles = (int)((G + 16 * pl.nc - 1) / (16 * pl.nc));
  pl.slots = (int)B;
  const int cus = device_cu_count() > 0 ? device_cu_count() : 256;
  // With four blocks for each that can be resident the card deals sequences of like lengths well
  // itself (300 of 500 keys, 16 / 8 heads: 95 us, 120 at the copy's rate). A long one among so
  // many is one block a KV head, and the call waits for it: of 60000 beside 254 of 500, dealt,
  // 140 us (150), beside 299, undealt, 608 (168).
  if (B > kPagedDealt || B * Hkv * pl.qtiles >= 8 * cus || Lmax <= stride) return pl;
  // A block for three quarters of the CUs: four waves' tiles in flight are what a CU reads at
  // its best, a second block only has it read for two (bf16, us at 3/4, 1, 1.5 and 2 a CU: 100000
  // and 60000 keys, 32 / 4 heads, 57, 60, 72, 65; one of 60000, 16 / 8, 41, 42, 46, 44; eight of
  // 8000, 32 / 8, 44, 45, 51, 46; three of 300 to 9000, 16 / 8, 15.5, 16.1, 17.9, 17.4). Two a
  // sequence, where those are more, for the long ones to be split.
  int64_t t = 3 * (int64_t)cus / 4 / (Hkv * pl.qtiles);
  if (t < 1) t = 1;
  if (t < 2 * B) t = 2 * B;
  const int64_t most = B * ((Lmax + stride - 1) / stride);
  if (t > most) t = most;
  pl.target = (int)t;
  // A block that merges reads rows * splits sums of 4 (D + 2) bytes (one of 15741 keys, 32 / 4
  // heads: 16 with 32 splits, 17 with 48, 19 with 96, 30 with 123; of 40000, 8 / 1: 22 with 32, 20
  // with 48, 24 with 128).
  pl.most = pl.nc == 1 ? (int)(384 / G) : 1024;
  pl.slots = (int)(t + B); // (at most t runs of equal length, and a last one each)
  return pl;
}

} // namespace tpp

using namespace tpp;

extern "C" size_t tpp_attn_paged_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t Lmax) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Lmax <= 0) return 0;
  const PagedPlan pl = paged_plan(B, Hq, Hkv, D, Lmax);
  return pl.target ? (size_t)Hq * pl.slots * (D + 2) * sizeof(float) : 0;
}

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
  if (D > 256 || B > 65535 || Hq > 65535 || pages > 0x7fffffffLL || table_pages > ((1LL << 27) >> lpage))
    return set_error(TPP_E_UNSUPPORTED, "%s: head_dim above 256, or too many sequences, heads or pages", name);
  if (B == 0) return TPP_OK;
  if (!q || !o || !seqlens || (pages > 0 && (!k_pages || !v_pages)) || (table_pages > 0 && !block_tables))
    return set_error(TPP_E_INVALID, "%s: null pointer", name);
  PagedArgs a = {};
  a.q = q, a.k = k_pages, a.v = v_pages, a.o = o;
  a.q_s[0] = q_strides[0], a.q_s[2] = q_strides[1], a.o_s[0] = o_strides[0], a.o_s[2] = o_strides[1];
  for (int i = 0; i < 3; ++i) a.k_s[i] = k_strides[i], a.v_s[i] = v_strides[i];
  a.table = block_tables, a.t_sb = table_stride, a.seqlens = seqlens;
  a.B = (int)B, a.T = 1, a.Hq = (int)Hq, a.Hkv = (int)Hkv, a.G = (int)(Hq / Hkv);
  a.pages = (int)pages, a.lpage = lpage, a.Lmax = (int)(table_pages << lpage), a.lkt = D == 128 ? 5 : 6;
  const float sc = softmax_scale > 0.f ? softmax_scale : 1.f / sqrtf((float)D);
  a.scale_log2 = sc * 1.4426950408889634f;
  a.left = window_left < 0 ? -1 : window_left;
  hipStream_t st = as_stream(stream);
  // the matrix-core kernel: whole 16-byte rows, a DMA instruction's by 32-bit byte offsets
  uint64_t low = (uint64_t)(uintptr_t)q | (uint64_t)(uintptr_t)k_pages | (uint64_t)(uintptr_t)v_pages;
  uint64_t low_o = (uint64_t)(uintptr_t)o;
  for (int i = 0; i < 3; ++i) {
    low |= (uint64_t)(a.q_s[i] * 2) | (uint64_t)(a.k_s[i] * 2) | (uint64_t)(a.v_s[i] * 2);
    low_o |= (uint64_t)(a.o_s[i] * 2);
  }
  bool tiles = (D == 64 || D == 128) && !(low & 15) && !(low_o & 7) && pages > 0 && table_pages > 0 &&
               (uint64_t)a.G * (uint64_t)a.G < 1ull << 32;
  for (int64_t r : {a.k_s[2], a.v_s[2]}) tiles = tiles && r >= 0 && r < (1 << 23);
  if (!tiles)
    return TPP_DISPATCH_HALF(dtype, [&] {
      paged_generic_kernel<T><<<dim3((unsigned)Hq, (unsigned)B), dim3(64), 0, st>>>(a, (int)D);
      return check_launch(name);
    });
  const PagedPlan pl = paged_plan(B, Hq, Hkv, D, a.Lmax);
  float *ws_o = (float *)workspace, *ws_ml = nullptr;
  if (pl.target) {
    if (!workspace || ((uintptr_t)workspace & 127) || ws_bytes < tpp_attn_paged_workspace_size(B, Hq, Hkv, D, a.Lmax))
      return set_error(TPP_E_WORKSPACE, "%s: workspace missing, unaligned or too small", name);
    ws_ml = ws_o + (size_t)Hq * pl.slots * D;
  }
  // the merge by a pair's last block (one a pair)
  unsigned *arrived = pl.target && pl.nc == 1 ? arrival_words(st, B * Hkv) : nullptr;
  const dim3 grid((unsigned)(Hkv * pl.qtiles), (unsigned)pl.slots);
  const unsigned hinv = inv_of((int)Hkv), ginv = inv_of(a.G);
  return TPP_DISPATCH_HALF(dtype, [&] {
    auto go = [&](auto dd) {
      constexpr int DD = decltype(dd)::value;
      if (pl.nc == 1) paged_tile_kernel<T, DD, 1><<<grid, dim3(256), 0, st>>>(a, ws_o, ws_ml, pl.target, pl.most, pl.slots, hinv, ginv, arrived);
      else paged_tile_kernel<T, DD, 2><<<grid, dim3(256), 0, st>>>(a, ws_o, ws_ml, pl.target, pl.most, pl.slots, hinv, ginv, nullptr);
      if (pl.target && !arrived)
        paged_merge_kernel<T, DD><<<dim3((unsigned)((a.G + 256 / DD - 1) / (256 / DD)), (unsigned)Hkv, (unsigned)B), dim3(256), 0, st>>>(
            a, ws_o, ws_ml, pl.target, pl.most, pl.slots);
    };
    if (D == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 64>{});
    return check_launch(name);
  });
}
