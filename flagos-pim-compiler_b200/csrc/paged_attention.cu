// pim_paged_attention: attention of one new token per row over a paged KV cache, split over
// the cache's length and joined.
//
//   s_j = scale q . k_j,  p_j = exp(s_j - m) / sum_i exp(s_i - m),  o = sum_j p_j v_j,  j < lengths[row]
//
// Bound by the bytes of K and V, each of which is needed once: a query group shares one kv
// head, so the unit of work is (row, kv head, head tile of up to 16 query heads).
//
// Split.  Lengths are read on the device and differ, so no grid fits them: the units' keys
// are cut into tiles of 64 and the tiles of all units, in order, are dealt out evenly to as
// many CTAs as the GPU holds at once (CTA c takes [c T / G, (c + 1) T / G)).  A CTA walks its
// range unit by unit; units that lie in one CTA are written at once, a unit that spans several
// leaves a partial (max, sum, o) per CTA, of which a CTA has at most two: its first and its
// last.  A unit begun costs loads that wait and a join of the warps, about as much as two
// tiles, and is dealt out at that price (40 rows of 0 to 8192 keys x 64 heads over 8: 129.9 us
// without the charge, where one CTA drew ten short units and ended at 131 us, the others at 111;
// 121.4, 115.2, 115.8 and 117.1 with 1, 2, 3 and 5 tiles).  paged_finish_kernel joins the
// partials: which CTAs hold a unit follows from the lengths alone, so there are no tickets, no
// atomics and nothing that must be zero before a call, and the result does not depend on timing.
// Measured: 64 rows x 4096 keys x 32 heads 4.27 GB in 653 to 689 us on different GPUs, 6.2 to 6.5 TB/s;
// the ragged rows above 662 MB in 117 to 123 us, 5.4 to 5.7 TB/s (DRAM 71 % busy, tensor pipe 21 %, 8 warps
// an SM that mostly wait for their loads); what did not help there, at 116 us: a third CTA per SM with fewer registers (139 us),
// asking L2 for tiles ahead (134 to 145), loads that run on into the next unit (136), 32-byte
// loads (117), CTAs of 1 or 2 warps (119, 118).
//
// Short rows, and longer ones of few units, run in one launch instead, a CTA or a cluster of
// CTAs per unit: paged_whole_kernel, chosen in paged_layout().
//
// bf16: the products run on warp-level MMA (m16n8k16) straight from registers.  The order of
// the summed dims is free, so a lane takes the 16 bytes at dim 8 t + 32 i of key g (lane = 4 g +
// t) for K, which are two k-steps of its B fragment, and the query the same; for V it takes 16
// bytes at dim 8 g of keys 2t, 2t+1, 2t+8, 2t+9 and pairs two keys' elements with one byte
// permutation each.  Nothing goes through shared memory, every load is 16 bytes and
// 64 (K) or 128 (V) contiguous bytes a row.  The scores come out as (heads) x (keys), which is the
// layout that the second product's B fragment needs, so that one is taken as V^T P^T: 16 dims
// by 8 heads a tile.  P enters as three bf16 parts, each what is left of a probability rounded
// towards zero: 3 x 8 bits are all 24 of a float.  (Two
// parts: sums of p v that cancel are off by 2^-18 of their terms, and the 64 rows above take 1.7 %
// less.)  A step's products are summed from zero and added to the rest in fp32: see step(); that
// costs 0.6 % more.  The next tile's K loads start as soon as this one's scores are formed, its V
// loads once this one's V is paired, before the products that read the pairs (4 % behind them).
// tcgen05 would add staging in shared memory and TMEM for a product of 8 rows that the memory
// system bounds.
//
// fp32: a key's dims are spread over head_dim / 4 lanes; the partial dot products of several
// keys and heads are summed by one butterfly that leaves one score per lane.
//
// Weights: a key's probability needs its row's final max and sum, so the first kernel stores
// the scores and the second adds the probabilities (4 bytes per key and query head, written
// and read back mostly in L2).

#include <cooperative_groups.h>
#include <math.h>

#include "paged.cuh"

namespace pim {

struct PagedAttnArgs {
  PagedKV kv;
  const void* q;
  void* out;
  int64_t q_stride, out_stride;
  const int* lengths;
  int hq, group;    // query heads, and per kv head
  float scale_log2; // scale * log2(e): exponentials are powers of two
  float* weights;
  int64_t w_row_stride, w_head_stride;
  int* err;
  int head_tiles;   // of a kv head's query group
  int whole_warps;  // CTAs of so many warps for whole units (paged_whole_kernel); 0: split
  int cluster;      // CTAs that share a unit there
  int ctas;
  int64_t* cost;    // [rows + 1] cost of the units of the rows before, and of all
  float* part_stat; // [ctas][2][NH][2]  max, sum
  float* part_acc;  // [ctas][2][NH][HD]
  float* row_stat;  // [rows][hq][2]     of units that one CTA finished (with weights)
  float* scores;    // [rows][hq][score_stride] (with weights)
  int64_t score_stride; // slots of a row in `scores` (paged_whole_kernel: in shared memory)
};

constexpr int kTile = 64;          // keys of a tile
constexpr int kMaxCluster = 8;
constexpr int kUnitCost = 2;       // what a unit costs beside its tiles, in tiles: see the head of the file
constexpr int kSplitWarps = 4;     // of a CTA that walks a range of tiles
// CTAs of the splitting kernel per SM: what its registers allow with next to no spilling (fp32 of 128 dims with 4 or 8 heads
// 28 to 32 bytes, bf16 with 16 heads up to 8; the others none).
constexpr int paged_ctas_per_sm(bool bf16, int hd) { return bf16 && hd == 128 ? 2 : 3; }
constexpr int kFinishThreads = 128;
constexpr int kFinishKeys = 4 * kFinishThreads;  // keys whose weights one CTA adds to

__device__ __forceinline__ int row_length(const PagedAttnArgs& a, int row) {
  return min(max(a.lengths[row], 0), a.kv.slots());
}
__device__ __forceinline__ int row_tiles(const PagedAttnArgs& a, int row) {
  return (row_length(a, row) + kTile - 1) / kTile;
}
// What a row's unit counts for when the work is dealt out; its tiles are the last of it.
__device__ __forceinline__ int row_cost(const PagedAttnArgs& a, int row) {
  const int n = row_tiles(a, row);
  return n ? n + kUnitCost : 0;
}
// A share of a row's sum: 0 where no key had a score above -inf, NaN where a score was NaN.
__device__ __forceinline__ float quotient(float a, float sum) { return sum == 0.f ? 0.f : a / sum; }
// Off by at most 2 units in the last place, as exp2f is; results below 2^-126 come out 0 (the weights, by exp2f, have them).
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What one warp carries over a unit's keys: bf16 form (see the head of the file).
template <int HD, int NH>
struct MmaCore {
  using T = __nv_bfloat16;
  static constexpr bool kBf16 = true;
  static constexpr int kSub = 16;        // keys of one step of a warp
  static constexpr int KC = HD / 32;     // 16-byte pieces of a K row per lane
  static constexpr int VE = HD >= 64 ? 8 : HD / 8;  // dims of a V load
  static constexpr int VC = HD / (8 * VE);          // V loads of a row per lane
  static constexpr int NT = VC * VE / 2; // m-tiles of the output: 16 dims each
  static constexpr int HI = NH / 8;      // head rows of a lane: g (and g + 8)
  static constexpr int kParts = 1;       // states of a warp
  static constexpr int kPParts = 3;      // bf16 parts of a probability: 3 x 8 bits, all of a float
  uint4 q[HI][KC];
  uint4 kr[2][KC];
  uint32_t vr[4][VC][VE / 2];
  float acc[HI][NT][4];
  float m[HI], l[HI];
  int64_t at[2], at_next[2];
  int lim[2], lim_next[2];
  int page[2];
  int g, t;

  __device__ __forceinline__ void init(const PagedAttnArgs& a, int row, int head0, int nh) {
    const int lane = threadIdx.x % 32;
    g = lane / 4;
    t = lane % 4;
#pragma unroll
    for (int i = 0; i < HI; ++i) {
      const bool real = g + 8 * i < nh;
      const T* qr = static_cast<const T*>(a.q) + row * a.q_stride + (int64_t)(head0 + g + 8 * i) * HD;
#pragma unroll
      for (int c = 0; c < KC; ++c)
        q[i][c] = real ? *reinterpret_cast<const uint4*>(qr + 32 * c + 8 * t) : make_uint4(0, 0, 0, 0);
      m[i] = -INFINITY;
      l[i] = 0.f;
    }
#pragma unroll
    for (int h = 0; h < HI; ++h)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[h][n][e] = 0.f;
  }

  // Page ids of the 16 keys at key0 (two halves of 8, which never straddle a page).
  __device__ __forceinline__ void fetch_pages(const PagedAttnArgs& a, const int* trow, int key0, int end) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      page[i] = (int)ld4_if(trow + ((key0 + 8 * i) >> a.kv.ps_log2), key0 + 8 * i < end);
  }
  __device__ __forceinline__ void place(const PagedAttnArgs& a, int kvh, int key0, int end) {
    const int mask = (1 << a.kv.ps_log2) - 1;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      lim_next[i] = min(max(end - key0 - 8 * i, 0), 8);
      if ((unsigned)page[i] >= (unsigned)a.kv.num_pages) {
        if (lim_next[i] > 0) raise_flag(a.err);
        lim_next[i] = 0;
      }
      at_next[i] = page[i] * a.kv.page_stride + (((int64_t)kvh << a.kv.ps_log2) + ((key0 + 8 * i) & mask)) * HD;
    }
  }
  __device__ __forceinline__ void load_k(const PagedAttnArgs& a) {
    const T* kp = static_cast<const T*>(a.kv.k);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const int4 x = ld_once_if(reinterpret_cast<const int4*>(kp + at_next[i] + g * HD + 32 * c + 8 * t),
                                  g < lim_next[i]);
        kr[i][c] = make_uint4(x.x, x.y, x.z, x.w);
      }
  }
  __device__ __forceinline__ void load_v(const PagedAttnArgs& a) {
    const T* vp = static_cast<const T*>(a.kv.v);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = r / 2, key = 2 * t + r % 2;
#pragma unroll
      for (int c = 0; c < VC; ++c) {
        // a slot behind the length may hold anything, and 0 x NaN must not enter: it is not read, but zero
        const bool ok = key < lim[i];
        const T* p = vp + at[i] + key * HD + 64 * c + VE * g;
        if (VE == 8) {
          const int4 x = ld_once_if(reinterpret_cast<const int4*>(p), ok);
          vr[r][c][0] = x.x;
          vr[r][c][1] = x.y;
          vr[r][c][VE / 2 - 2] = x.z;
          vr[r][c][VE / 2 - 1] = x.w;
        } else {
          vr[r][c][0] = ld4_if(p, ok);
          vr[r][c][1] = ld4_if(p + 2, ok);
        }
      }
    }
  }
  __device__ __forceinline__ void advance() {
#pragma unroll
    for (int i = 0; i < 2; ++i) at[i] = at_next[i], lim[i] = lim_next[i];
  }

  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  // A float's upper 16 bits, as a float and of two floats side by side: what bf16 holds of them, rounded towards zero.
  static __device__ __forceinline__ float top(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
  static __device__ __forceinline__ uint32_t tops(float lo, float hi) {
    return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
  }

  // The step's keys key0 .. key0 + 15; next_k() and next_v() load the next step's once the registers are free.
  // `scores`: where the unit's first head has its scores, or nullptr.
  template <typename NextK, typename NextV>
  __device__ __forceinline__ void step(const PagedAttnArgs& a, float* scores, int nh, int key0, NextK&& next_k,
                                       NextV&& next_v) {
    float s[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const uint4 q1 = HI > 1 ? q[HI - 1][c] : make_uint4(0, 0, 0, 0);
        mma(s[i], q[0][c].x, q1.x, q[0][c].y, q1.y, kr[i][c].x, kr[i][c].y);
        mma(s[i], q[0][c].z, q1.z, q[0][c].w, q1.w, kr[i][c].z, kr[i][c].w);
      }
    }
    next_k();
    uint32_t part[kPParts][2][HI];
    float alpha[HI];
    bool grew = false;
#pragma unroll
    for (int h = 0; h < HI; ++h) {
      float best = -INFINITY;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& x = s[i][2 * h + e];
          x = 2 * t + e < lim[i] ? x * a.scale_log2 : -INFINITY;
          best = fmaxf(best, x);
        }
      if (scores && g + 8 * h < nh) {
        float* sp = scores + (g + 8 * h) * a.score_stride + key0 + 2 * t;
#pragma unroll
        for (int i = 0; i < 2; ++i) *reinterpret_cast<float2*>(sp + 8 * i) = make_float2(s[i][2 * h], s[i][2 * h + 1]);
      }
      best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
      best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
      const float mn = fmaxf(m[h], best);
      const float safe = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: every probability is 0, not NaN
      grew |= mn > m[h];
      alpha[h] = exp2_fast(m[h] - safe);
      m[h] = mn;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float p0 = exp2_fast(s[i][2 * h] - safe), p1 = exp2_fast(s[i][2 * h + 1] - safe);
        sum += p0 + p1;
        float r0 = p0, r1 = p1;
#pragma unroll
        for (int x = 0; x < kPParts; ++x) {
          part[x][i][h] = tops(r0, r1);
          // (at least 2^-30 of p, so that no part of a positive p is 0: an infinite V times 0 would be NaN, not infinite)
          r0 = fmaxf(r0 - top(r0), p0 * 0x1p-30f);
          r1 = fmaxf(r1 - top(r1), p1 * 0x1p-30f);
        }
      }
      l[h] = l[h] * alpha[h] + sum;
    }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int h = 0; h < HI; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // (column 2t + e is head 2t + e of the eight, whose lanes are 4 (2t + e) ..)
          const float f = __shfl_sync(0xffffffffu, alpha[h], 8 * t + 4 * e);
#pragma unroll
          for (int n = 0; n < NT; ++n) acc[h][n][e] *= f, acc[h][n][2 + e] *= f;
        }
    }
    uint32_t v[NT][4];
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
      for (int w = 0; w < VE / 2; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[c * VE / 2 + w][i] = __byte_perm(vr[i / 2 * 2][c][w], vr[i / 2 * 2 + 1][c][w], i % 2 ? 0x7632 : 0x5410);
    next_v();
    // A tile's products are summed from zero, the smallest part of P first, and added to the rest in fp32: the tensor cores'
    // own additions round towards zero, which over thousands of keys adds up to several times the error of nearest.
#pragma unroll
    for (int h = 0; h < HI; ++h)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = kPParts - 1; x >= 0; --x) mma(d, v[n][0], v[n][1], v[n][2], v[n][3], part[x][0][h], part[x][1][h]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[h][n][e] += d[e];
      }
  }

  // The state of part `warp` into shared memory: [parts][NH] max and sum, [parts][NH][HD] output.
  __device__ __forceinline__ void store(float* sm_m, float* sm_l, float* sm_acc, int warp) {
#pragma unroll
    for (int h = 0; h < HI; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      const int at = warp * NH + 8 * h;
      if (t == 0) sm_m[at + g] = m[h], sm_l[at + g] = l[h];
      // rows g and g + 8 of m-tile (c, w) are dims 8 VE c + VE g + 2 w and the next; this lane has heads 2t and 2t + 1
#pragma unroll
      for (int c = 0; c < VC; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int w = 0; w < VE / 2; w += 2) {
            const float(&x)[4] = acc[h][c * VE / 2 + w], (&y)[4] = acc[h][c * VE / 2 + w + 1];
            *reinterpret_cast<float4*>(sm_acc + (at + 2 * t + e) * HD + 8 * VE * c + VE * g + 2 * w) =
                make_float4(x[e], x[2 + e], y[e], y[2 + e]);
          }
    }
  }
};

// fp32 form.  A group of LPK lanes owns a key, NK keys a step; the NK * NH dot products of a
// group are summed over its lanes by a butterfly that halves the number of values a lane
// holds at each step, so one (key, head) is left per lane (or per LPK / N lanes).
template <int HD, int NH>
struct FmaCore {
  using T = float;
  static constexpr bool kBf16 = false;
  static constexpr int LPK = HD / 4;
  static constexpr int KG = 32 / LPK;
  static constexpr int NK = LPK / NH < 8 ? LPK / NH : 8;
  static constexpr int N = NK * NH;
  static constexpr int REP = LPK / N;   // lanes that hold the same score
  static constexpr int kSub = KG * NK;
  static constexpr int kParts = KG;
  float4 q[NH], acc[NH], k[NK], v[NK];
  float m, l;
  int page[NK];
  int64_t at[NK], at_next[NK];  // this lane's 16 bytes of each key; -1: no such key
  int grp, sl, head, key_of;    // this lane's score: head, and key within the group's NK

  __device__ __forceinline__ void init(const PagedAttnArgs& a, int row, int head0, int nh) {
    const int lane = threadIdx.x % 32;
    grp = lane / LPK;
    sl = lane % LPK;
    head = sl / REP % NH;
    key_of = sl / REP / NH;
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      q[h] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (h < nh)
        q[h] = *reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + row * a.q_stride +
                                                (int64_t)(head0 + h) * HD + 4 * sl);
      acc[h] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    m = -INFINITY;
    l = 0.f;
  }
  __device__ __forceinline__ void fetch_pages(const PagedAttnArgs& a, const int* trow, int key0, int end) {
#pragma unroll
    for (int u = 0; u < NK; ++u) {
      const int key = key0 + grp * NK + u;
      page[u] = (int)ld4_if(trow + (key >> a.kv.ps_log2), key < end);
    }
  }
  __device__ __forceinline__ void place(const PagedAttnArgs& a, int kvh, int key0, int end) {
#pragma unroll
    for (int u = 0; u < NK; ++u) {
      const int key = key0 + grp * NK + u;
      at_next[u] = -1;
      if (key < end) {
        if ((unsigned)page[u] < (unsigned)a.kv.num_pages)
          at_next[u] = page[u] * a.kv.page_stride +
                       (((int64_t)kvh << a.kv.ps_log2) + (key & ((1 << a.kv.ps_log2) - 1))) * HD + 4 * sl;
        else
          raise_flag(a.err);
      }
    }
  }
  static __device__ __forceinline__ float4 load(const void* pages, int64_t at) {
    const int4 x = ld_once_if(reinterpret_cast<const int4*>(static_cast<const float*>(pages) + at), at >= 0);
    return make_float4(__int_as_float(x.x), __int_as_float(x.y), __int_as_float(x.z), __int_as_float(x.w));
  }
  __device__ __forceinline__ void load_k(const PagedAttnArgs& a) {
#pragma unroll
    for (int u = 0; u < NK; ++u) k[u] = load(a.kv.k, at_next[u]);
  }
  __device__ __forceinline__ void load_v(const PagedAttnArgs& a) {
#pragma unroll
    for (int u = 0; u < NK; ++u) v[u] = load(a.kv.v, at[u]);
  }
  __device__ __forceinline__ void advance() {
#pragma unroll
    for (int u = 0; u < NK; ++u) at[u] = at_next[u];
  }
  template <typename NextK, typename NextV>
  __device__ __forceinline__ void step(const PagedAttnArgs& a, float* scores, int nh, int key0, NextK&& next_k,
                                       NextV&& next_v) {
    bool mine_ok = false;
#pragma unroll
    for (int u = 0; u < NK; ++u) mine_ok |= at[u] >= 0 && u == key_of;
    float s[N];
#pragma unroll
    for (int u = 0; u < NK; ++u)
#pragma unroll
      for (int h = 0; h < NH; ++h)
        s[u * NH + h] = fmaf(q[h].x, k[u].x, fmaf(q[h].y, k[u].y, fmaf(q[h].z, k[u].z, q[h].w * k[u].w)));
    next_k();
    int o = LPK / 2;
#pragma unroll
    for (int n = N; n > 1; n /= 2, o /= 2) {
      const bool up = sl & o;
#pragma unroll
      for (int i = 0; i < N / 2; ++i)
        if (i < n / 2) {
          const float give = up ? s[i] : s[i + n / 2];
          const float keep = up ? s[i + n / 2] : s[i];
          s[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    }
    float x = s[0];
#pragma unroll
    for (int r = REP / 2; r > 0; r /= 2) x += __shfl_xor_sync(0xffffffffu, x, r);
    x = mine_ok ? x * a.scale_log2 : -INFINITY;
    // (a key behind the end writes -inf behind the row's scores, within score_stride)
    if (scores && sl % REP == 0 && head < nh) scores[head * a.score_stride + key0 + grp * NK + key_of] = x;
    float top = x;
#pragma unroll
    for (int r = REP * NH; r < LPK; r *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, r));
    const float mn = fmaxf(m, top);
    const float safe = mn == -INFINITY ? 0.f : mn;
    const float alpha = exp2f(m - safe), p = exp2f(x - safe);
    const bool grew = mn > m;
    l = l * alpha + p;
    m = mn;
    const int base = grp * LPK;
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const float f = __shfl_sync(0xffffffffu, alpha, base + h * REP);
        acc[h].x *= f;
        acc[h].y *= f;
        acc[h].z *= f;
        acc[h].w *= f;
      }
    }
#pragma unroll
    for (int u = 0; u < NK; ++u)
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const float f = __shfl_sync(0xffffffffu, p, base + (u * NH + h) * REP);
        acc[h].x = fmaf(f, v[u].x, acc[h].x);
        acc[h].y = fmaf(f, v[u].y, acc[h].y);
        acc[h].z = fmaf(f, v[u].z, acc[h].z);
        acc[h].w = fmaf(f, v[u].w, acc[h].w);
      }
    next_v();
  }
  __device__ __forceinline__ void store(float* sm_m, float* sm_l, float* sm_acc, int warp) {
#pragma unroll
    for (int r = REP * NH; r < LPK; r *= 2) l += __shfl_xor_sync(0xffffffffu, l, r);
    const int part = warp * KG + grp;
    if (key_of == 0 && sl % REP == 0) sm_m[part * NH + head] = m, sm_l[part * NH + head] = l;
#pragma unroll
    for (int h = 0; h < NH; ++h) *reinterpret_cast<float4*>(sm_acc + (part * NH + h) * HD + 4 * sl) = acc[h];
  }
};

// One warp's keys of [begin, end) (begin a multiple of 64), the CTA's WARPS warps taking turns: page ids two steps
// ahead, the next step's K loads once this one's scores are formed, its V loads once this one's V was taken up.
template <int WARPS, typename Core>
__device__ __forceinline__ void walk(Core& core, const PagedAttnArgs& a, const int* trow, float* scores, int kvh, int nh,
                                     int begin, int end) {
  constexpr int STRIDE = Core::kSub * WARPS;
  int key0 = begin + (int)threadIdx.x / 32 * Core::kSub;
  if (key0 >= end) return;  // (the whole warp)
  core.fetch_pages(a, trow, key0, end);
  core.place(a, kvh, key0, end);
  core.load_k(a);
  core.advance();
  core.load_v(a);
  core.fetch_pages(a, trow, key0 + STRIDE, end);
  for (; key0 < end; key0 += STRIDE) {
    core.step(
        a, scores, nh, key0,
        [&] {
          core.place(a, kvh, key0 + STRIDE, end);
          core.fetch_pages(a, trow, key0 + 2 * STRIDE, end);
          core.load_k(a);
        },
        [&] {
          core.advance();
          core.load_v(a);
        });
  }
}

// The parts of a unit that a CTA's warps hold, brought together.
template <typename Core, int HD, int NH, int WARPS>
struct Joint {
  static constexpr int PARTS = WARPS * Core::kParts;
  float m[PARTS * NH], l[PARTS * NH];
  float top[NH], sum[NH];  // the unit's max (0 where there is none) and sum
  float none[NH];          // 1 where no key had a score above -inf
  alignas(16) float acc[PARTS * NH * HD];

  // Keys [begin, end) of the unit by the whole CTA; out(h, d, value before the division) for its heads.
  template <typename Out>
  __device__ __forceinline__ void run(const PagedAttnArgs& a, int row, int kvh, int head0, int nh, int begin, int end,
                                      float* scores, Out&& out) {
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    {
      Core core;
      core.init(a, row, head0, nh);
      walk<WARPS>(core, a, a.kv.table + row * a.kv.table_stride, scores, kvh, nh, begin, end);
      core.store(m, l, acc, warp);
    }
    __syncthreads();
    for (int h = warp; h < nh; h += WARPS) {  // a lane per part
      const float pm = lane < PARTS ? m[lane * NH + h] : -INFINITY;
      const float M = warp_max(pm);
      const float safe = M == -INFINITY ? 0.f : M;
      const float f = exp2f(pm - safe);
      const float L = warp_sum(lane < PARTS ? l[lane * NH + h] * f : 0.f);
      if (lane < PARTS) m[lane * NH + h] = f;
      if (lane == 0) top[h] = safe, sum[h] = L, none[h] = M == -INFINITY;
    }
    __syncthreads();
    for (int i = tid; i < nh * HD; i += WARPS * 32) {
      const int h = i / HD, d = i % HD;
      float A = 0.f;
#pragma unroll
      for (int w = 0; w < PARTS; ++w) A += acc[(w * NH + h) * HD + d] * m[w * NH + h];
      out(h, d, A);
    }
  }
};

// A CTA, or a cluster of a.cluster CTAs, per unit: rows short enough for it to walk, with their scores in shared memory
// where the weights are asked for.  One launch and no workspace: a cluster's CTAs take an equal part of the tiles each and
// join through one another's shared memory.
template <typename Core, int HD, int NH, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) paged_whole_kernel(PagedAttnArgs a) {
  using T = typename Core::T;
  constexpr int THREADS = WARPS * 32;
  extern __shared__ float sm_scores[];  // [NH][score_stride]
  __shared__ Joint<Core, HD, NH, WARPS> joint;
  __shared__ float sm_part[NH * HD], sm_stat[kMaxCluster][NH][2];  // this CTA's part; every CTA's max and sum
  const int tid = threadIdx.x;
  pdl_trigger();
  pdl_wait();
  const int units = a.kv.hkv * a.head_tiles, at = blockIdx.x / a.cluster, rank = blockIdx.x - at * a.cluster;
  const int row = at / units, unit = at - row * units;
  const int kvh = unit / a.head_tiles, ht = unit - kvh * a.head_tiles;
  const int head0 = kvh * a.group + ht * NH, nh = min(NH, a.group - ht * NH);
  const int len = row_length(a, row), tiles = (len + kTile - 1) / kTile;
  if (tid == 0 && len != a.lengths[row]) raise_flag(a.err);
  const int begin = rank * tiles / a.cluster * kTile, end = min(len, (rank + 1) * tiles / a.cluster * kTile);
  T* out = static_cast<T*>(a.out) + row * a.out_stride + (int64_t)head0 * HD;
  // (the scores of this CTA's keys: key `begin` is at sm_scores[0])
  joint.run(a, row, kvh, head0, nh, begin, end, a.weights ? sm_scores - begin : nullptr, [&](int h, int d, float A) {
    if (a.cluster > 1) {
      sm_part[h * HD + d] = A;
    } else {
      const float L = joint.sum[h];
      out[h * HD + d] = from_f<T>(quotient(A, L));
    }
  });
  if (a.cluster > 1) {
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    cluster.sync();
    for (int i = tid; i < a.cluster * nh; i += THREADS) {
      const int r = i / nh, h = i - r * nh;
      const auto* theirs = cluster.map_shared_rank(&joint, r);
      sm_stat[r][h][0] = theirs->none[h] ? -INFINITY : theirs->top[h];
      sm_stat[r][h][1] = theirs->sum[h];
    }
    __syncthreads();
    for (int i = rank * THREADS + tid; i < nh * HD; i += a.cluster * THREADS) {
      const int h = i / HD;
      float M = -INFINITY, L = 0.f, A = 0.f;
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r)
        if (r < a.cluster) M = fmaxf(M, sm_stat[r][h][0]);
      const float safe = M == -INFINITY ? 0.f : M;
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r)
        if (r < a.cluster) {
          const float f = exp2f(sm_stat[r][h][0] - safe);
          L += sm_stat[r][h][1] * f;
          A += cluster.map_shared_rank(sm_part, r)[i] * f;
        }
      out[i] = from_f<T>(quotient(A, L));
    }
    cluster.sync();  // (the others may still read this CTA's part; and joint's statistics become the unit's below)
    if (a.weights && tid < nh) {
      float M = -INFINITY, L = 0.f;
      for (int r = 0; r < a.cluster; ++r) M = fmaxf(M, sm_stat[r][tid][0]);
      const float safe = M == -INFINITY ? 0.f : M;
      for (int r = 0; r < a.cluster; ++r) L += sm_stat[r][tid][1] * exp2f(sm_stat[r][tid][0] - safe);
      joint.top[tid] = safe;
      joint.sum[tid] = L;
    }
    __syncthreads();
  }
  if (!a.weights) return;
  float* w = a.weights + row * a.w_row_stride + (int64_t)kvh * a.w_head_stride;
  for (int key = begin + tid; key < end; key += THREADS) {
    float p = 0.f;
    for (int h = 0; h < nh; ++h) {
      const float L = joint.sum[h];
      p += exp2f(sm_scores[h * a.score_stride + key - begin] - joint.top[h]) * quotient(1.f, L);
    }
    w[key] += p;
  }
}

template <typename Core, int HD, int NH>
__global__ void __launch_bounds__(kSplitWarps * 32, paged_ctas_per_sm(Core::kBf16, HD)) paged_attn_kernel(PagedAttnArgs a) {
  using T = typename Core::T;
  constexpr int THREADS = kSplitWarps * 32;
  __shared__ Joint<Core, HD, NH, kSplitWarps> joint;
  __shared__ int64_t sm_scan[kSplitWarps];
  __shared__ int sm_row;
  __shared__ int64_t sm_rest;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  pdl_trigger();
  pdl_wait();
  // where this CTA's range begins: thread i counts the cost of rows [i per, (i + 1) per)
  const int units = a.kv.hkv * a.head_tiles;
  const int per = (a.kv.rows + THREADS - 1) / THREADS;
  const int r0 = min(tid * per, a.kv.rows), r1 = min(r0 + per, a.kv.rows);
  int64_t mine = 0;
  for (int b = r0; b < r1; ++b) {
    if (blockIdx.x == 0 && row_length(a, b) != a.lengths[b]) raise_flag(a.err);
    mine += row_cost(a, b);
  }
  int64_t scan = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += y;
  }
  if (lane == 31) sm_scan[warp] = scan;
  __syncthreads();
  int64_t total = 0, before = scan - mine;
#pragma unroll
  for (int w = 0; w < kSplitWarps; ++w) {
    if (w < warp) before += sm_scan[w];
    total += sm_scan[w];
  }
  if (blockIdx.x == 0) {  // for the second kernel
    int64_t at = before * units;
    for (int b = r0; b < r1; ++b) {
      a.cost[b] = at;
      at += (int64_t)row_cost(a, b) * units;
    }
    if (tid == 0) a.cost[a.kv.rows] = total * units;
  }
  total *= units;
  const int64_t ctas = min((int64_t)a.ctas, total);  // none of them has an empty range
  if (blockIdx.x >= ctas) return;
  const int64_t lo = blockIdx.x * total / ctas, hi = (blockIdx.x + 1) * total / ctas;
  if (lo >= before * units && lo < (before + mine) * units) {
    int64_t at = before * units;
    int b = r0;
    for (;; ++b) {
      const int64_t n = (int64_t)row_cost(a, b) * units;
      if (lo < at + n) break;
      at += n;
    }
    sm_row = b;
    sm_rest = lo - at;
  }
  __syncthreads();
  int row = sm_row;
  int cost = row_cost(a, row);
  int unit = (int)(sm_rest / cost);
  int64_t at = sm_rest - (int64_t)unit * cost;  // within the unit
  bool first = true;
  for (int64_t left = hi - lo; left > 0;) {
    const int len = row_length(a, row), tiles = cost - kUnitCost;
    // the part of [at, at + left) that is tiles of this unit
    const int64_t stop = min(at + left, (int64_t)cost);
    const int tile = (int)max(at - kUnitCost, (int64_t)0), n = (int)(stop - kUnitCost) - tile;
    left -= stop - at;
    if (n > 0) {
      const int kvh = unit / a.head_tiles, ht = unit - kvh * a.head_tiles;
      const int head0 = kvh * a.group + ht * NH, nh = min(NH, a.group - ht * NH);
      const bool whole = n == tiles;
      // a partial that begins with the CTA's range is its slot 0, one that begins later its slot 1
      const int64_t slot = ((int64_t)blockIdx.x * 2 + (first ? 0 : 1)) * NH;
      first = false;
      const int64_t head_at = (int64_t)row * a.hq + head0;
      joint.run(a, row, kvh, head0, nh, tile * kTile, min(len, (tile + n) * kTile),
                a.scores ? a.scores + head_at * a.score_stride : nullptr, [&](int h, int d, float A) {
                  const float L = joint.sum[h];
                  if (whole) {
                    static_cast<T*>(a.out)[row * a.out_stride + (int64_t)(head0 + h) * HD + d] =
                        from_f<T>(quotient(A, L));
                  } else {
                    a.part_acc[(slot + h) * HD + d] = A;
                  }
                  if (d == 0 && (!whole || a.scores)) {
                    float* st = whole ? a.row_stat + (head_at + h) * 2 : a.part_stat + (slot + h) * 2;
                    st[0] = !whole && joint.none[h] ? -INFINITY : joint.top[h];
                    st[1] = L;
                  }
                });
      __syncthreads();
    }
    at = stop;
    if (at == cost && left > 0) {
      at = 0;
      if (++unit == units) {
        unit = 0;
        do ++row;
        while ((cost = row_cost(a, row)) == 0);  // (some of the range is left, so a row with some is)
      }
    }
  }
}

// The CTAs that hold a unit's tiles, the unit's cost being [start, start + kUnitCost + tiles) of `total`: first ..
// last, and the slot of the first one's part.
struct Holders {
  int first, last, first_slot;
};
__device__ __forceinline__ Holders holders(int64_t start, int tiles, int64_t total, int64_t ctas) {
  Holders h;
  const int64_t begin = start + kUnitCost, end = begin + tiles;
  h.first = (int)(((begin + 1) * ctas + total - 1) / total) - 1;  // the largest c with c total / ctas <= begin
  h.last = (int)((end * ctas + total - 1) / total) - 1;
  h.first_slot = h.first * total / ctas >= start ? 0 : 1;
  return h;
}

template <typename T, int HD, int NH>
__global__ void __launch_bounds__(kFinishThreads) paged_finish_kernel(PagedAttnArgs a, int join_ctas, int key_chunks) {
  constexpr int WARPS = kFinishThreads / 32;
  constexpr int G = HD / 4, PARTS = kFinishThreads / G;  // lanes of a part (16 bytes each), parts at a time
  __shared__ float sm_m[WARPS], sm_l[WARPS];
  __shared__ alignas(16) float sm_acc[PARTS][HD];
  __shared__ float sm_stat[32][2];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  pdl_trigger();
  pdl_wait();
  const bool join = (int)blockIdx.x < join_ctas;
  int row, head, chunk = 0;
  if (join) {
    row = blockIdx.x / a.hq;
    head = blockIdx.x - row * a.hq;
  } else {
    int r = blockIdx.x - join_ctas;
    chunk = r % key_chunks;
    r /= key_chunks;
    row = r / a.kv.hkv;
    head = (r - row * a.kv.hkv) * a.group;
    if (chunk * kFinishKeys >= row_length(a, row)) return;
  }
  const int tiles = row_tiles(a, row);
  if (tiles == 0) {  // nothing to attend to
    for (int d = tid; d < HD; d += kFinishThreads)
      static_cast<T*>(a.out)[row * a.out_stride + (int64_t)head * HD + d] = from_f<T>(0.f);
    return;
  }
  const int64_t before = a.cost[row], total = a.cost[a.kv.rows];
  auto holders_of = [&](int h) {
    const int unit = h / a.group * a.head_tiles + h % a.group / NH;
    return holders(before + (int64_t)unit * (tiles + kUnitCost), tiles, total, min((int64_t)a.ctas, total));
  };
  auto slot_of = [&](const Holders& p, int c) {
    return ((int64_t)c * 2 + (c == p.first ? p.first_slot : 0)) * NH;
  };
  if (join) {
    const Holders p = holders_of(head);
    if (p.first == p.last) return;  // written by its one CTA
    const int hl = head % a.group % NH;
    const int pg = tid / G, d4 = 4 * (tid % G);
    float m = -INFINITY, l = 0.f;
    for (int c = p.first + tid; c <= p.last; c += kFinishThreads) {
      const float2 st = *reinterpret_cast<const float2*>(a.part_stat + (slot_of(p, c) + hl) * 2);
      const float mn = fmaxf(m, st.x), safe = mn == -INFINITY ? 0.f : mn;
      l = l * exp2f(m - safe) + st.y * exp2f(st.x - safe);
      m = mn;
    }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float safe = 0.f;
    // The loads of FLY parts a thread are under way together: a unit of few and long rows lies in every CTA.
    auto add = [&](auto fly) {
      constexpr int kFly = decltype(fly)::value;
      for (int c0 = p.first + pg, round = 0; round * kFly * PARTS <= p.last - p.first; ++round, c0 += kFly * PARTS) {
        int4 v[kFly];
        float f[kFly];
#pragma unroll
        for (int u = 0; u < kFly; ++u) {
          const int c = c0 + u * PARTS;
          const int64_t at = slot_of(p, c) + hl;
          v[u] = ld_once_if(reinterpret_cast<const int4*>(a.part_acc + at * HD + d4), c <= p.last);
          f[u] = __uint_as_float(ld4_if(a.part_stat + at * 2, c <= p.last));
        }
        if (round == 0) {  // the unit's maximum and sum, beside the first loads
          const float M = warp_max(m), here = M == -INFINITY ? 0.f : M;
          l = warp_sum(l * exp2f(m - here));
          if (lane == 0) sm_m[warp] = M, sm_l[warp] = l;
          __syncthreads();
          float top = sm_m[0];
#pragma unroll
          for (int w = 1; w < WARPS; ++w) top = fmaxf(top, sm_m[w]);
          safe = top == -INFINITY ? 0.f : top;
        }
#pragma unroll
        for (int u = 0; u < kFly; ++u) {
          const float g = c0 + u * PARTS <= p.last ? exp2f(f[u] - safe) : 0.f;
          acc.x += __int_as_float(v[u].x) * g;
          acc.y += __int_as_float(v[u].y) * g;
          acc.z += __int_as_float(v[u].z) * g;
          acc.w += __int_as_float(v[u].w) * g;
        }
      }
    };
    if (p.last - p.first < PARTS) add(std::integral_constant<int, 1>());
    else add(std::integral_constant<int, 8>());
    *reinterpret_cast<float4*>(&sm_acc[pg][d4]) = acc;
    __syncthreads();
    for (int d = tid; d < HD; d += kFinishThreads) {
      float L = 0.f, A = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) L += sm_l[w] * exp2f(sm_m[w] - safe);
#pragma unroll
      for (int w = 0; w < PARTS; ++w) A += sm_acc[w][d];
      static_cast<T*>(a.out)[row * a.out_stride + (int64_t)head * HD + d] = from_f<T>(quotient(A, L));
    }
    return;
  }
  // the probabilities of this CTA's keys, summed over the group's heads in order; the scores of the first heads and
  // the weights are under way while the units' statistics are found
  constexpr int KEYS = kFinishKeys / kFinishThreads, AHEAD = 4;
  const int len = row_length(a, row), key0 = chunk * kFinishKeys + tid;
  float* w = a.weights + row * a.w_row_stride + (int64_t)(head / a.group) * a.w_head_stride;
  const float* sp = a.scores + ((int64_t)row * a.hq + head) * a.score_stride;
  float sum[KEYS], old[KEYS], x[AHEAD][KEYS];
#pragma unroll
  for (int u = 0; u < KEYS; ++u) {
    const int key = key0 + u * kFinishThreads;
    sum[u] = 0.f;
    old[u] = __uint_as_float(ld4_if(w + key, key < len));
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      x[i][u] = __uint_as_float(ld4_if(sp + i * a.score_stride + key, key < len && i < a.group));
  }
  for (int h0 = 0; h0 < a.group; h0 += 32) {
    const int nh = min(32, a.group - h0);
    __syncthreads();
    for (int i = warp; i < nh; i += WARPS) {  // a warp per head: the unit's max and sum
      const int h = head + h0 + i;
      const Holders p = holders_of(h);
      float m = -INFINITY, l = 0.f;
      if (p.first == p.last) {
        m = a.row_stat[((int64_t)row * a.hq + h) * 2];
        l = a.row_stat[((int64_t)row * a.hq + h) * 2 + 1];
      } else {
        const int hl = h % a.group % NH;
        for (int c0 = p.first + lane; c0 <= p.last; c0 += 32 * 4) {
          float x[4], y[4];  // (four parts under way)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float* st = a.part_stat + (slot_of(p, c0 + 32 * u) + hl) * 2;
            x[u] = __uint_as_float(ld4_if(st, c0 + 32 * u <= p.last));
            y[u] = __uint_as_float(ld4_if(st + 1, c0 + 32 * u <= p.last));
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (c0 + 32 * u > p.last) break;
            const float mn = fmaxf(m, x[u]), safe = mn == -INFINITY ? 0.f : mn;
            l = l * exp2f(m - safe) + y[u] * exp2f(x[u] - safe);
            m = mn;
          }
        }
        const float M = warp_max(m), safe = M == -INFINITY ? 0.f : M;
        l = warp_sum(l * exp2f(m - safe));
        m = safe;
      }
      if (lane == 0) sm_stat[i][0] = m, sm_stat[i][1] = quotient(1.f, l);
    }
    __syncthreads();
    for (int i0 = 0; i0 < nh; i0 += AHEAD) {
      if (h0 + i0 > 0) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
#pragma unroll
          for (int u = 0; u < KEYS; ++u)
            x[i][u] = __uint_as_float(ld4_if(sp + (h0 + i0 + i) * a.score_stride + key0 + u * kFinishThreads,
                                             key0 + u * kFinishThreads < len && i0 + i < nh));
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (i0 + i < nh) {
#pragma unroll
          for (int u = 0; u < KEYS; ++u) sum[u] += exp2f(x[i][u] - sm_stat[i0 + i][0]) * sm_stat[i0 + i][1];
        }
    }
  }
#pragma unroll
  for (int u = 0; u < KEYS; ++u)
    if (key0 + u * kFinishThreads < len) w[key0 + u * kFinishThreads] = old[u] + sum[u];
}

// Query heads of a tile: the smallest tile that holds the group, up to 16 (bf16) or 8 (fp32) heads.
static int head_tile(int dtype, int group) {
  if (dtype == PIM_BF16) return group <= 8 ? 8 : 16;
  return group <= 1 ? 1 : group <= 2 ? 2 : group <= 4 ? 4 : 8;
}

// CTAs of the first kernel: as many as are resident at once on the current device (148 SMs if
// there is none: the workspace of a call can be asked for anywhere).
static int paged_ctas(int dtype, int hd) {
  static int sms[64];
  const int per_sm = paged_ctas_per_sm(dtype == PIM_BF16, hd);
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    (void)cudaGetLastError();
    return 148 * per_sm;
  }
  if (!sms[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
      (void)cudaGetLastError();
      n = 148;
    }
    sms[dev] = n;
  }
  return sms[dev] * per_sm;
}

template <typename Core, int HD, int NH, int WARPS>
static cudaError_t launch_whole(const PagedAttnArgs& a, cudaStream_t st) {
  static ResidentCache cache;
  const size_t smem = a.weights ? (size_t)NH * a.score_stride * 4 : 0;
  cudaError_t e;
  if (resident_ctas(paged_whole_kernel<Core, HD, NH, WARPS>, WARPS * 32, smem, cache, &e) < 0) return e;
  const dim3 grid(a.kv.rows * a.kv.hkv * a.head_tiles * a.cluster);
  return a.cluster > 1 ? launch_pdl_cluster(paged_whole_kernel<Core, HD, NH, WARPS>, a.cluster, grid, dim3(WARPS * 32), smem,
                                            st, a)
                       : launch_pdl(paged_whole_kernel<Core, HD, NH, WARPS>, grid, dim3(WARPS * 32), smem, st, a);
}

template <typename Core, int HD, int NH>
static cudaError_t launch_paged(const PagedAttnArgs& a, cudaStream_t st) {
  using T = typename Core::T;
  if (a.whole_warps == 8) {
    // (the parts of 16 heads by 8 warps would not fit the static shared memory: see paged_layout())
    if constexpr (NH <= 8) return launch_whole<Core, HD, NH, 8>(a, st);
    return cudaErrorNotSupported;
  }
  if (a.whole_warps == 4) return launch_whole<Core, HD, NH, 4>(a, st);
  if (a.whole_warps == 2) return launch_whole<Core, HD, NH, 2>(a, st);
  if (a.whole_warps == 1) return launch_whole<Core, HD, NH, 1>(a, st);
  cudaError_t e = launch_pdl(paged_attn_kernel<Core, HD, NH>, dim3(a.ctas), dim3(kSplitWarps * 32), 0, st, a);
  if (e != cudaSuccess) return e;
  const int join = a.kv.rows * a.hq;
  const int chunks = a.weights ? ceil_div((int64_t)a.kv.max_pages << a.kv.ps_log2, kFinishKeys) : 0;
  const int64_t grid = join + (int64_t)a.kv.rows * a.kv.hkv * chunks;
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  return launch_pdl(paged_finish_kernel<T, HD, NH>, dim3((unsigned)grid), dim3(kFinishThreads), 0, st, a, join,
                    chunks ? chunks : 1);
}

template <int HD>
static cudaError_t paged_attention_hd(const PagedAttnArgs& a, int dtype, int nh, cudaStream_t st) {
  if (dtype == PIM_BF16)
    return nh == 8 ? launch_paged<MmaCore<HD, 8>, HD, 8>(a, st)
                   : launch_paged<MmaCore<HD, 16>, HD, 16>(a, st);
  if (nh == 1) return launch_paged<FmaCore<HD, 1>, HD, 1>(a, st);
  if (nh == 2) return launch_paged<FmaCore<HD, 2>, HD, 2>(a, st);
  if (nh == 4) return launch_paged<FmaCore<HD, 4>, HD, 4>(a, st);
  return launch_paged<FmaCore<HD, 8>, HD, 8>(a, st);
}

// nullptr, or what is wrong with the arguments.
static const char* paged_attention_error(const pim_paged_attention_args* a, int dtype) {
  if (!a) return "null arguments";
  if (!dtype_ok(dtype)) return "bad dtype";
  if (const char* e = paged_kv_error(a->kv, dtype)) return e;
  const int es = elem_bytes(dtype);
  if (!a->q || !a->out || !a->lengths) return "null q, out or lengths";
  if (a->kv.rows > 65535) return "more than 65535 rows";
  if (a->q_heads <= 0 || a->q_heads > 65535 || a->q_heads % a->kv.kv_heads)
    return "q_heads must be a multiple of kv_heads, at most 65535";
  if ((int64_t)a->kv.rows * a->q_heads > (1 << 27)) return "more than 2^27 rows times heads";
  const int64_t row = (int64_t)a->q_heads * a->kv.head_dim;
  if (a->q_stride < row || a->out_stride < row) return "q or out stride is less than a row";
  if (!aligned16(a->q) || !aligned16(a->out) || a->q_stride * es % 16 || a->out_stride * es % 16)
    return "q, out and their strides must be 16-byte aligned";
  if (!(a->scale >= 0.f) || isinf(a->scale)) return "bad scale";
  if (a->weights && (a->weights_head_stride < (int64_t)a->kv.max_pages * a->kv.page_size ||
                     a->weights_row_stride < a->weights_head_stride * a->kv.kv_heads))
    return "weights strides are less than a row's slots";
  return nullptr;
}

// The parts of the workspace, as byte offsets.
struct PagedLayout {
  int nh, tiles, ctas;
  bool whole;
  int whole_warps, cluster;
  int64_t score_stride, stat, acc, row_stat, scores, bytes;
};
static PagedLayout paged_layout(const pim_paged_attention_args* a, int dtype) {
  PagedLayout p;
  const int group = a->q_heads / a->kv.kv_heads;
  p.nh = head_tile(dtype, group);
  p.tiles = ceil_div(group, p.nh);
  p.ctas = paged_ctas(dtype, a->kv.head_dim);
  const int64_t slots = (int64_t)a->kv.max_pages * a->kv.page_size, units = (int64_t)a->kv.rows * a->kv.kv_heads * p.tiles;
  // Whole units in a CTA or a cluster save the second launch and the join, and lose where rows are long or units many.
  // "Slots" are the table's: lengths are on the device, so short rows of a wide table are split (1 row of 130 keys x 32
  // heads: 4.9 us in a table of 144 slots, 5.4 in 512 to 2048, 8.2 in 4096 and more).
  // Few units: 8 warps a CTA and the largest cluster that leaves every CTA an SM, up to 512 slots a CTA (fp32 256); one CTA
  // up to 256 slots, where a cluster gains nothing.  Device us by slots 256, 512, 1024, 2048, 4000:
  //   1 row x 8 heads x 4    clusters of 8  5.6  5.7  6.5  7.6  9.5   one CTA 5.6  7.5          split - 8.5  9.5  9.9 11.8
  //   1 row x 32 heads x 1   clusters of 4  5.4  6.3  7.4 12.1    -   one CTA 5.5  7.3 11.2     split 9.0 9.6  9.4 12.9 18.4
  //   8 rows x 8 heads x 8   clusters of 2  7.2  8.2 11.2 20.9    -   one CTA 6.0  7.9 13.9     split 11.5 11.9 13.0 18.4
  //   fp32 1 row x 4 heads   clusters of 8  5.6  5.9  6.4  8.0 11.3                             split   -   -  7.2  7.9  9.7
  // More units than SMs twice over: fewer warps a CTA, bf16 2 up to 256 slots (128 rows x 8 heads x 8: 22.6, 35.6, 60.8 us
  // at 128, 256, 512 against 38.6, 46.7, 61.7 split), fp32 4 up to 512 (64 x 8 x 4: 8.6, 16.6, 30.5, 56.7 at 128 .. 1024
  // against 17.3, 24.7, 34.7, 55.8).  More than the GPU holds at once: fewer still, as a warp has all the keys of 16 or 32 slots
  // and a CTA's warps wait for one another: bf16 1 up to 128 slots (123 rows x 32 heads of 10, 62, 126, 250 keys 14.8, 39.8,
  // 69.6, 127 us, with 2 23.0, 44.0, 70.5, 122; 40 x 16 of 10 4.6 and 6.4, 64 x 8 5.9 and 4.7), fp32 2 (128 x 8 x 4 of 10, 62,
  // 250 5.1, 9.8, 30.8, with 4 6.8, 10.9, 32.2), and 1 for many short ones (123 x 32 of 10, 62, 126 11.7, 33.0, 58.7, with 2
  // 18.5, 34.9, 57.6; 128 x 8 x 4 of 10 6.9 and 5.1).  A query group of several tiles would add to the same weights from several CTAs: it is
  // split.
  const bool bf16 = dtype == PIM_BF16, many = units > 2 * 148;
  p.whole_warps = !many ? (p.nh > 8 ? 4 : 8) : !bf16 && units <= 4 * 148 ? 4 : 2;
  if (bf16 ? units > 4 * 148 && slots <= 128 : units > 16 * 148 && slots <= 64) p.whole_warps = 1;
  p.cluster = 1;
  if (slots > 256)
    while (p.cluster < kMaxCluster && units * p.cluster * 2 * p.whole_warps <= 8 * 148) p.cluster *= 2;
  const int64_t most = p.cluster > 1 ? (bf16 ? 512 : 256) * p.cluster : many && bf16 ? 256 : 512;
  p.whole = slots <= (most > 512 || many ? most : 512) && (!a->weights || p.tiles == 1);
  p.score_stride = (slots + 63) / 64 * 64;
  if (p.whole) {
    p.score_stride = (p.score_stride / p.cluster + 127) / 64 * 64;  // a CTA's part is a tile more at most
    p.stat = p.acc = p.row_stat = p.scores = p.bytes = 0;
    return p;
  }
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  const int64_t parts = (int64_t)p.ctas * 2 * p.nh;
  p.stat = up(((int64_t)a->kv.rows + 1) * 8);
  p.acc = p.stat + up(parts * 2 * 4);
  p.row_stat = p.acc + up(parts * a->kv.head_dim * 4);
  p.scores = p.bytes = p.row_stat;
  if (a->weights) {
    const int64_t heads = (int64_t)a->kv.rows * a->q_heads;
    p.scores = p.row_stat + up(heads * 2 * 4);
    p.bytes = p.scores + heads * p.score_stride * 4;
  }
  return p;
}

}  // namespace pim

extern "C" int64_t pim_paged_attention_workspace_bytes(const pim_paged_attention_args* a, int32_t dtype) {
  using namespace pim;
  if (paged_attention_error(a, dtype)) return -1;
  return paged_layout(a, dtype).bytes;
}

extern "C" int pim_paged_attention(const pim_paged_attention_args* a, int32_t dtype, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  using namespace pim;
  if (const char* e = paged_attention_error(a, dtype)) {
    char msg[200];
    snprintf(msg, sizeof(msg), "pim_paged_attention: %s", e);
    return report_status(PIM_EINVAL, msg);
  }
  const PagedLayout p = paged_layout(a, dtype);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes || !aligned16(workspace)))
    return report_status(PIM_EINVAL, "pim_paged_attention: workspace too small or not 16-byte aligned");
  PagedAttnArgs d{};
  d.kv = to_dev(a->kv);
  d.q = a->q;
  d.out = a->out;
  d.q_stride = a->q_stride;
  d.out_stride = a->out_stride;
  d.lengths = a->lengths;
  d.hq = a->q_heads;
  d.group = a->q_heads / a->kv.kv_heads;
  const double scale = a->scale > 0.f ? a->scale : 1.0 / sqrt((double)a->kv.head_dim);
  d.scale_log2 = (float)(scale * 1.4426950408889634);  // log2(e)
  d.weights = a->weights;
  d.w_row_stride = a->weights_row_stride;
  d.w_head_stride = a->weights_head_stride;
  d.err = a->err_flag;
  d.head_tiles = p.tiles;
  d.ctas = p.ctas;
  d.whole_warps = p.whole ? p.whole_warps : 0;
  d.cluster = p.cluster;
  d.score_stride = p.score_stride;
  if (!p.whole) {
    char* ws = static_cast<char*>(workspace);
    d.cost = reinterpret_cast<int64_t*>(ws);
    d.part_stat = reinterpret_cast<float*>(ws + p.stat);
    d.part_acc = reinterpret_cast<float*>(ws + p.acc);
    if (a->weights) {
      d.row_stat = reinterpret_cast<float*>(ws + p.row_stat);
      d.scores = reinterpret_cast<float*>(ws + p.scores);
    }
  }
  const int hd = a->kv.head_dim;
  cudaStream_t st = (cudaStream_t)stream;
  return report_cuda(hd == 128  ? paged_attention_hd<128>(d, dtype, p.nh, st)
                     : hd == 64 ? paged_attention_hd<64>(d, dtype, p.nh, st)
                                : paged_attention_hd<32>(d, dtype, p.nh, st),
                     "pim_paged_attention");
}
