// pim_paged_evict: a paged cache cut down to a budget by accumulated attention weight.
//
// Per (row, kv head), over the n slots in use: a token that must stay (recent or sink) ranks
// above every weight; the budget largest stay, of equal ones the lower slot.  The selection
// is a radix select over 64-bit keys, the weight's bits in unsigned order above the complement
// of the slot: they are unique, so equal weights need no case of their own, and the bound of
// what stays is one key.  Passes of 11 + 11 + 10 bits (of the slot's too, where weights are
// equal) narrow it down until at most 256 keys share the bits fixed so far; those are ranked
// by counting.  The kept slots as bit words, scanned in slot order, then list the freed slots
// below the budget and the kept ones above it; there are equally many, and moving the i-th kept
// one into the i-th freed slot moves the fewest rows that any compaction can.  Sources lie at or
// above the budget and destinations below it, so the moves need no order.
//
// evict_select_kernel: one CTA per (row, head), keys in shared memory where they fit; it
// reads 8 bytes a slot and writes the state and the list of moves.  evict_cluster_kernel does the
// same by a cluster of CTAs where rows are long and few.  evict_move_kernel: moves
// the K and V rows, a grid over (row, head) x blocks of moves; bound by DRAM.
// Measured: 8 prompts of 1500 to 8190 slots x 32 heads cut to 2048 68 us, the selection 19 and the
// moves, 232 MB in rows of 256 bytes, 40 to 45 (5.2 to 5.8 TB/s); longer lists moved by the
// selecting CTA itself would take 84 -> 90 us, a single row's 36 -> 52.  16 rows x 8 heads one
// token over 1024: 3.8 us in one launch (9.9 with histograms and scans, 11.7 in two launches).

#include <cooperative_groups.h>

#include "paged.cuh"

namespace pim {

struct EvictArgs {
  PagedKV kv;
  const int *lengths, *positions;
  const float* weights;
  const int* slot_positions;
  float* weights_out;
  int *slot_positions_out, *lengths_out;
  int64_t row_stride, head_stride;
  int budget, recent, sink;
  int* err;
  int* counts;   // [rows * hkv] moves
  int2* moves;   // [rows * hkv][max_moves] (freed slot, kept slot)
  int max_moves;
  int64_t page_pieces;  // 16-byte pieces between pages
  int cluster;          // CTAs of a (row, head): evict_cluster_kernel
};

constexpr int kSelThreads = 512;
constexpr int kMaxSmemKeys = 48 * 1024;
constexpr int kChunkWords = kMaxSmemKeys / 32;
constexpr int kMoveThreads = 128;
constexpr int kFusedMoves = 128;  // see evict_rows()
constexpr int kFewEvicted = 8;
constexpr int kRankMost = 256;

// Unsigned key of the same order as the weight; NaN lowest.  -0 and +0 are equal.
__device__ __forceinline__ uint32_t order_key(float w) {
  w += 0.f;
  if (w != w) return 0;
  const uint32_t u = __float_as_uint(w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive prefix sum over the CTA (kSelThreads threads); *total: the sum.
__device__ __forceinline__ uint32_t cta_scan(uint32_t v, uint32_t* sm, uint32_t* total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) sm[warp] = x;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelThreads / 32; ++w) {
    if (w < warp) before += sm[w];
    all += sm[w];
  }
  *total = all;
  return x - v + before;
}

// Up to kWarpMoves moves of a unit's list by one warp.  Each lane finds one row (the freed or the
// kept slot of a move: one table entry), then all lanes copy 16-byte pieces (LPR of them are a K or
// V row), eight loads under way at a time, with the rows' places taken from the lanes that know them.
// (8 prompts cut from up to 8190 to 2048 slots x 32 heads, 232 MB of rows: 8 moves a warp and 128 threads a CTA
// 67.5 us with the selection, 16 and 256 72.7, 4 and 128 72.1.)
constexpr int kWarpMoves = 8;
template <int LPR>
__device__ __forceinline__ void move_rows(const EvictArgs& a, const int2* moves, int row, int head, int count) {
  constexpr int STEPS = kWarpMoves * 2 * LPR / 32, FLY = STEPS < 8 ? STEPS : 8;
  const int lane = threadIdx.x % 32, mine = lane % kWarpMoves;
  int64_t at = -1;  // in pieces
  if (mine < count) {
    const int2 mv = moves[mine];
    const int slot = lane < kWarpMoves ? mv.x : mv.y;
    const int page = a.kv.table[row * a.kv.table_stride + (slot >> a.kv.ps_log2)];
    if ((unsigned)page < (unsigned)a.kv.num_pages)
      at = page * a.page_pieces + (((int64_t)head << a.kv.ps_log2) + (slot & ((1 << a.kv.ps_log2) - 1))) * LPR;
    else
      raise_flag(a.err);
  }
  for (int s0 = 0; s0 < STEPS; s0 += FLY) {
    int4 v[FLY];
    int64_t to[FLY];
#pragma unroll
    for (int u = 0; u < FLY; ++u) {
      const int flat = (s0 + u) * 32 + lane, m = flat / (2 * LPR), r = flat % (2 * LPR), piece = r % LPR;
      const int64_t src = __shfl_sync(0xffffffffu, at, kWarpMoves + m);
      to[u] = __shfl_sync(0xffffffffu, at, m);
      const int4* p = static_cast<const int4*>(r < LPR ? a.kv.k : a.kv.v);
      if (src < 0) to[u] = -1;
      v[u] = ld_once_if(p + src + piece, to[u] >= 0);
    }
#pragma unroll
    for (int u = 0; u < FLY; ++u) {
      const int r = ((s0 + u) * 32 + lane) % (2 * LPR), piece = r % LPR;
      int4* p = static_cast<int4*>(r < LPR ? a.kv.k : a.kv.v);
      if (to[u] >= 0) p[to[u] + piece] = v[u];
    }
  }
}

// The state of the slots that are refilled and, with LPR, their K and V, by the selecting CTAs' `threads` threads, of which
// this is number t.
template <int LPR>
__device__ __forceinline__ void finish_moves(const EvictArgs& a, const int2* mv, int moved, int row, int head,
                                             int64_t base, const float* w, const int* sp, int t, int threads) {
  constexpr int FLY = 4;
  for (int i0 = t; i0 < moved; i0 += FLY * threads) {
    int2 m[FLY];
    uint32_t x[FLY], p[FLY];
#pragma unroll
    for (int u = 0; u < FLY; ++u) {
      const int i = i0 + u * threads;
      m[u].x = (int)ld4_if(&mv[i].x, i < moved);
      m[u].y = (int)ld4_if(&mv[i].y, i < moved);
    }
#pragma unroll
    for (int u = 0; u < FLY; ++u) {
      x[u] = ld4_if(w + m[u].y, i0 + u * threads < moved);
      p[u] = ld4_if(sp + m[u].y, i0 + u * threads < moved);
    }
#pragma unroll
    for (int u = 0; u < FLY; ++u)
      if (i0 + u * threads < moved) {
        a.weights_out[base + m[u].x] = __uint_as_float(x[u]);
        a.slot_positions_out[base + m[u].x] = (int)p[u];
      }
  }
  if constexpr (LPR > 0) {
    for (int m = t / 32 * kWarpMoves; m < moved; m += threads / 32 * kWarpMoves)
      move_rows<LPR>(a, mv + m, row, head, moved - m);
  }
}

// SMEM: the keys of a row fit the shared memory.  LPR: 0, or the CTA moves its rows itself.
template <bool SMEM, int LPR>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(EvictArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ uint32_t hist[2048];
  __shared__ uint32_t sm_keep[kChunkWords], sm_at[kChunkWords];
  __shared__ unsigned long long sm_near[kRankMost];
  __shared__ unsigned long long sm_bound;
  __shared__ uint32_t sm_scan[kSelThreads / 32];
  __shared__ uint32_t sm_bin, sm_above, sm_count;
  const int head = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  for (int i = tid; i < 2048; i += kSelThreads) hist[i] = 0;
  pdl_trigger();
  pdl_wait();
  const int want = a.lengths[row];
  const int64_t next = a.positions[row];
  const int n = min(max(want, 0), a.kv.slots());
  const int left = min(n, a.budget);
  if (head == 0 && tid == 0) {
    if (n != want) raise_flag(a.err);
    a.lengths_out[row] = left;
  }
  const int64_t base = row * a.row_stride + head * a.head_stride;
  const float* w = a.weights + base;
  const int* sp = a.slot_positions + base;
  const int unit = row * a.kv.hkv + head;
  const bool copy_w = a.weights_out != a.weights, copy_p = a.slot_positions_out != a.slot_positions;
  // (int64: a position near the type's ends less `recent` must not wrap)
  const int64_t from = next - a.recent;
  auto make_key = [&](float wt, int p) { return p >= from || p < a.sink ? 0xffffffffu : order_key(wt); };
  const bool evicts = n > a.budget, few = SMEM && LPR > 0 && n - a.budget <= kFewEvicted;
  __syncthreads();
  // one pass over the state, kLoads slots of a thread in flight: the kept part's copy, the keys and the first
  // histogram
  constexpr int kLoads = 8;
  for (int j = tid; j < n; j += kLoads * kSelThreads) {
    float wt[kLoads];
    int p[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      wt[u] = __uint_as_float(ld4_if(w + j + u * kSelThreads, j + u * kSelThreads < n));
      p[u] = (int)ld4_if(sp + j + u * kSelThreads, j + u * kSelThreads < n);
    }
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int i = j + u * kSelThreads;
      if (i < left) {
        if (copy_w) a.weights_out[base + i] = wt[u];
        if (copy_p) a.slot_positions_out[base + i] = p[u];
      }
      if (i < n && evicts) {
        const uint32_t k = make_key(wt[u], p[u]);
        if (SMEM) keys[i] = k;
        if (!few) atomicAdd(&hist[k >> 21], 1);
      }
    }
  }
  if (!evicts) {
    if (LPR == 0 && tid == 0) a.counts[unit] = 0;
    return;
  }
  if (few) {
    // A step's one or few tokens over the budget: that many rounds of a minimum, in place of the histograms and scans.
    // Of equal keys the higher slot goes.
    __shared__ uint2 sm_least[kSelThreads / 32];
    __shared__ int sm_gone[kFewEvicted];
    const int gone = n - a.budget;
    unsigned long long last = 0;  // (every packed key is above it: a slot's complement is not 0)
    __syncthreads();
    for (int r = 0; r < gone; ++r) {
      unsigned long long best = ~0ull;
      for (int j = tid; j < n; j += kSelThreads) {
        const unsigned long long x = (unsigned long long)keys[j] << 32 | (uint32_t)~j;
        if (x > last && x < best) best = x;
      }
      uint32_t hi = __reduce_min_sync(0xffffffffu, (uint32_t)(best >> 32));
      uint32_t lo = __reduce_min_sync(0xffffffffu, (uint32_t)(best >> 32) == hi ? (uint32_t)best : ~0u);
      if (lane == 0) sm_least[warp] = make_uint2(lo, hi);
      __syncthreads();
      const uint2 x = lane < kSelThreads / 32 ? sm_least[lane] : make_uint2(~0u, ~0u);
      hi = __reduce_min_sync(0xffffffffu, x.y);
      lo = __reduce_min_sync(0xffffffffu, x.y == hi ? x.x : ~0u);
      last = (unsigned long long)hi << 32 | lo;
      if (tid == 0) sm_gone[r] = (int)~lo;
      __syncthreads();
    }
    // the freed slots below the budget in order, and the kept ones above it
    int2* mv = a.moves + (int64_t)unit * a.max_moves;
    if (warp == 0) {
      const int mine = lane < gone ? sm_gone[lane] : n;
      int rank = 0;
      bool stays = lane < gone;  // slot budget + lane
      for (int i = 0; i < gone; ++i) {
        rank += sm_gone[i] < mine;
        if (sm_gone[i] == a.budget + lane) stays = false;
      }
      if (lane < gone && mine < a.budget) mv[rank].x = mine;
      const unsigned who = __ballot_sync(0xffffffffu, stays);
      if (stays) mv[__popc(who & ((1u << lane) - 1))].y = a.budget + lane;
      if (lane == 0) sm_count = __popc(who);
    }
    __syncthreads();
    finish_moves<LPR>(a, mv, (int)sm_count, row, head, base, w, sp, tid, kSelThreads);
    return;
  }
  auto key = [&](int j) { return SMEM ? keys[j] : make_key(w[j], sp[j]); };
  auto packed = [&](int j) { return (unsigned long long)key(j) << 32 | (uint32_t)~j; };
  // the budget-th largest packed key
  unsigned long long bound = 0;
  uint32_t need = a.budget;
  int shift = 64;
  for (int pass = 0;; ++pass) {
    const int bits = pass % 3 < 2 ? 11 : 10;
    if (pass) {
#pragma unroll 4
      for (int j = tid; j < n; j += kSelThreads) {
        const unsigned long long k = packed(j);
        if (k >> shift == bound >> shift) atomicAdd(&hist[(uint32_t)(k >> (shift - bits)) & ((1u << bits) - 1)], 1);
      }
    }
    shift -= bits;
    __syncthreads();
    // thread t owns the bins 2047 - 4t .. 2044 - 4t, so the scan runs from the largest bin down
    constexpr int OWN = 2048 / kSelThreads;
    uint32_t c[OWN], sum = 0, total;
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      sum += c[i] = hist[2047 - OWN * tid - i];
      hist[2047 - OWN * tid - i] = 0;
    }
    uint32_t above = cta_scan(sum, sm_scan, &total);
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      if (above < need && need <= above + c[i]) sm_bin = 2047 - OWN * tid - i, sm_above = above, sm_count = c[i];
      above += c[i];
    }
    __syncthreads();
    bound |= (unsigned long long)sm_bin << shift;
    need -= sm_above;
    if (sm_count <= kRankMost || shift == 0) break;
  }
  if (shift > 0) {  // rank those that share the bits fixed so far; with all fixed there is one
    __syncthreads();
    if (tid == 0) sm_count = 0;
    __syncthreads();
#pragma unroll 4
    for (int j = tid; j < n; j += kSelThreads) {
      const unsigned long long k = packed(j);
      if (k >> shift == bound >> shift) sm_near[atomicAdd(&sm_count, 1)] = k;
    }
    __syncthreads();
    const int near = (int)sm_count;
    if (tid < near) {
      const unsigned long long mine = sm_near[tid];
      uint32_t rank = 0;
      for (int i = 0; i < near; ++i) rank += sm_near[i] > mine;
      if (rank == need - 1) sm_bound = mine;
    }
    __syncthreads();
    bound = sm_bound;
  }
  int2* mv = a.moves + (int64_t)unit * a.max_moves;
  const int half = (n + 1) / 2;  // (at most half of the slots move: two lists fit the place of the keys)
  uint32_t moved_to = 0, moved_from = 0;
  for (int c0 = 0; c0 < n; c0 += kMaxSmemKeys) {  // (one round where SMEM)
    const int m = min(n - c0, kMaxSmemKeys), words = (m + 31) / 32;
#pragma unroll 4
    for (int i = warp; i < words; i += kSelThreads / 32) {
      const int j = c0 + 32 * i + lane;
      const uint32_t keep = __ballot_sync(0xffffffffu, j < n && packed(j < n ? j : 0) >= bound);
      if (lane == 0) sm_keep[i] = keep;
    }
    __syncthreads();
    // the slots of word i that a move frees (below the budget) or takes its row from (above it)
    auto freed = [&](int i) {
      const int b = a.budget - c0 - 32 * i;
      return b <= 0 ? 0u : ~sm_keep[i] & (b >= 32 ? ~0u : (1u << b) - 1);
    };
    auto taken = [&](int i) {
      const int b = a.budget - c0 - 32 * i;
      return b >= 32 ? 0u : sm_keep[i] & (b <= 0 ? ~0u : ~((1u << b) - 1));
    };
    const int per = (words + kSelThreads - 1) / kSelThreads;
    const int w0 = min(tid * per, words), w1 = min(w0 + per, words);
    uint32_t total, counts = 0;  // freed in the low, taken in the high half: at most kMaxSmemKeys < 2^16 of each
    for (int i = w0; i < w1; ++i) counts += __popc(freed(i)) + (__popc(taken(i)) << 16);
    uint32_t before = cta_scan(counts, sm_scan, &total);
    for (int i = w0; i < w1; ++i) {
      sm_at[i] = before;
      before += __popc(freed(i)) + (__popc(taken(i)) << 16);
    }
    __syncthreads();
#pragma unroll 4
    for (int i = warp; i < words; i += kSelThreads / 32) {  // a lane per slot
      const uint32_t f = freed(i), t = taken(i), lower = (1u << lane) - 1, at = sm_at[i];
      const int j = c0 + 32 * i + lane;
      if (f >> lane & 1) {
        const uint32_t to = moved_to + (at & 0xffff) + __popc(f & lower);
        if (SMEM) keys[to] = j;
        else mv[to].x = j;
      }
      if (t >> lane & 1) {
        const uint32_t src = moved_from + (at >> 16) + __popc(t & lower);
        if (SMEM) keys[half + src] = j;
        else mv[src].y = j;
      }
    }
    moved_to += total & 0xffff;
    moved_from += total >> 16;
    __syncthreads();
  }
  const int moved = (int)moved_from;  // as many as were freed: budget slots are kept in all
  if (LPR == 0 && tid == 0) a.counts[unit] = moved;
  if (SMEM) {
#pragma unroll 4
    for (int i = tid; i < moved; i += kSelThreads) mv[i] = make_int2((int)keys[i], (int)keys[half + i]);
  }
  __syncthreads();
  finish_moves<LPR>(a, mv, moved, row, head, base, w, sp, tid, kSelThreads);
}

// The same by a cluster of a.cluster CTAs per (row, head), for long rows of few units: each holds the keys of an equal part of
// the slots in its shared memory.  Histograms and minima are brought together through one another's shared memory, each
// CTA summing them for itself, so all of them find the same bound; lists start where those of the CTAs before end.
template <int LPR>
__global__ void __launch_bounds__(kSelThreads) evict_cluster_kernel(EvictArgs a) {
  extern __shared__ uint32_t keys[];  // of slots lo ..
  __shared__ alignas(16) uint32_t hist[2][2048];
  __shared__ uint32_t sm_keep[kChunkWords], sm_at[kChunkWords];
  __shared__ unsigned long long sm_near[kRankMost];  // the first CTA's: all keys to be ranked
  __shared__ unsigned long long sm_bound, sm_best[2];
  __shared__ uint32_t sm_scan[kSelThreads / 32];
  __shared__ uint32_t sm_bin, sm_above, sm_count, sm_near_count, sm_total;
  __shared__ int sm_gone[kFewEvicted];
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  const int size = a.cluster, head = blockIdx.x / size, rank = blockIdx.x - head * size, row = blockIdx.y;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  for (int i = tid; i < 2 * 2048; i += kSelThreads) hist[i / 2048][i % 2048] = 0;
  if (tid == 0) sm_near_count = 0;
  pdl_trigger();
  pdl_wait();
  const int want = a.lengths[row];
  const int64_t next = a.positions[row];
  const int n = min(max(want, 0), a.kv.slots());
  const int left = min(n, a.budget);
  if (head == 0 && rank == 0 && tid == 0) {
    if (n != want) raise_flag(a.err);
    a.lengths_out[row] = left;
  }
  const int part = ((n + size - 1) / size + 31) / 32 * 32;  // (whole words of the bit lists)
  const int lo = min(rank * part, n), m = min(part, n - lo);
  const int64_t base = row * a.row_stride + head * a.head_stride;
  const float* w = a.weights + base;
  const int* sp = a.slot_positions + base;
  const int unit = row * a.kv.hkv + head;
  const bool copy_w = a.weights_out != a.weights, copy_p = a.slot_positions_out != a.slot_positions;
  const int64_t from = next - a.recent;
  const bool evicts = n > a.budget, few = LPR > 0 && n - a.budget <= kFewEvicted;
  __syncthreads();
  constexpr int kLoads = 8;
  for (int j = tid; j < m; j += kLoads * kSelThreads) {
    float wt[kLoads];
    int p[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      wt[u] = __uint_as_float(ld4_if(w + lo + j + u * kSelThreads, j + u * kSelThreads < m));
      p[u] = (int)ld4_if(sp + lo + j + u * kSelThreads, j + u * kSelThreads < m);
    }
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int i = j + u * kSelThreads;
      if (i < m && lo + i < left) {
        if (copy_w) a.weights_out[base + lo + i] = wt[u];
        if (copy_p) a.slot_positions_out[base + lo + i] = p[u];
      }
      if (i < m && evicts) {
        const uint32_t k = p[u] >= from || p[u] < a.sink ? 0xffffffffu : order_key(wt[u]);
        keys[i] = k;
        if (!few) atomicAdd(&hist[0][k >> 21], 1);
      }
    }
  }
  if (!evicts) {  // (the whole cluster)
    if (LPR == 0 && rank == 0 && tid == 0) a.counts[unit] = 0;
    return;
  }
  int2* mv = a.moves + (int64_t)unit * a.max_moves;
  auto packed = [&](int j) { return (unsigned long long)keys[j] << 32 | (uint32_t)~(lo + j); };
  if (few) {
    __shared__ uint2 sm_least[kSelThreads / 32];
    const int gone = n - a.budget;
    unsigned long long last = 0;
    __syncthreads();
    for (int r = 0; r < gone; ++r) {
      unsigned long long best = ~0ull;
      for (int j = tid; j < m; j += kSelThreads) {
        const unsigned long long x = packed(j);
        if (x > last && x < best) best = x;
      }
      uint32_t hi = __reduce_min_sync(0xffffffffu, (uint32_t)(best >> 32));
      uint32_t low = __reduce_min_sync(0xffffffffu, (uint32_t)(best >> 32) == hi ? (uint32_t)best : ~0u);
      if (lane == 0) sm_least[warp] = make_uint2(low, hi);
      __syncthreads();
      if (warp == 0) {
        const uint2 x = lane < kSelThreads / 32 ? sm_least[lane] : make_uint2(~0u, ~0u);
        hi = __reduce_min_sync(0xffffffffu, x.y);
        low = __reduce_min_sync(0xffffffffu, x.y == hi ? x.x : ~0u);
        if (lane == 0) sm_best[r & 1] = (unsigned long long)hi << 32 | low;
      }
      cluster.sync();  // (the other of the two is still read until the next one)
      best = ~0ull;
      for (int c = 0; c < size; ++c) {
        const unsigned long long x = *cluster.map_shared_rank(&sm_best[r & 1], c);
        best = x < best ? x : best;
      }
      last = best;
      if (tid == 0) sm_gone[r] = (int)~(uint32_t)last;
    }
    cluster.sync();  // no CTA leaves while its minimum is read
    if (rank != 0) return;
    if (warp == 0) {
      const int mine = lane < gone ? sm_gone[lane] : n;
      int ahead = 0;
      bool stays = lane < gone;  // slot budget + lane
      for (int i = 0; i < gone; ++i) {
        ahead += sm_gone[i] < mine;
        if (sm_gone[i] == a.budget + lane) stays = false;
      }
      if (lane < gone && mine < a.budget) mv[ahead].x = mine;
      const unsigned who = __ballot_sync(0xffffffffu, stays);
      if (stays) mv[__popc(who & ((1u << lane) - 1))].y = a.budget + lane;
      if (lane == 0) sm_count = __popc(who);
    }
    __syncthreads();
    finish_moves<LPR>(a, mv, (int)sm_count, row, head, base, w, sp, tid, kSelThreads);
    return;
  }
  unsigned long long bound = 0;
  uint32_t need = a.budget;
  int shift = 64;
  for (int pass = 0;; ++pass) {
    const int bits = pass % 3 < 2 ? 11 : 10;
    if (pass) {
#pragma unroll 4
      for (int j = tid; j < m; j += kSelThreads) {
        const unsigned long long k = packed(j);
        if (k >> shift == bound >> shift)
          atomicAdd(&hist[pass & 1][(uint32_t)(k >> (shift - bits)) & ((1u << bits) - 1)], 1);
      }
    }
    shift -= bits;
    cluster.sync();
    constexpr int OWN = 2048 / kSelThreads;
    uint32_t c[OWN] = {}, sum = 0, total;
    for (int r = 0; r < size; ++r) {
      const uint4 x = *reinterpret_cast<const uint4*>(
          cluster.map_shared_rank(&hist[pass & 1][2048 - OWN * (tid + 1)], r));
      static_assert(OWN == 4, "a thread's bins are 16 bytes");
      c[0] += x.w;
      c[1] += x.z;
      c[2] += x.y;
      c[3] += x.x;
    }
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      sum += c[i];
      hist[(pass + 1) & 1][2047 - OWN * tid - i] = 0;  // (read last before the barrier above; filled behind cta_scan's)
    }
    uint32_t above = cta_scan(sum, sm_scan, &total);
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      if (above < need && need <= above + c[i]) sm_bin = 2047 - OWN * tid - i, sm_above = above, sm_count = c[i];
      above += c[i];
    }
    __syncthreads();
    bound |= (unsigned long long)sm_bin << shift;
    need -= sm_above;
    if (sm_count <= kRankMost || shift == 0) break;
  }
  if (shift > 0) {
    unsigned long long* near_keys = cluster.map_shared_rank(sm_near, 0);
    uint32_t* near_count = cluster.map_shared_rank(&sm_near_count, 0);
#pragma unroll 4
    for (int j = tid; j < m; j += kSelThreads) {
      const unsigned long long k = packed(j);
      if (k >> shift == bound >> shift) near_keys[atomicAdd(near_count, 1u)] = k;
    }
    cluster.sync();
    const int near = (int)*near_count;
    const unsigned long long mine = tid < near ? near_keys[tid] : 0;
    if (rank != 0 && tid < near) sm_near[tid] = mine;
    __syncthreads();
    if (tid < near) {
      uint32_t ahead = 0;
      for (int i = 0; i < near; ++i) ahead += sm_near[i] > mine;
      if (ahead == need - 1) sm_bound = mine;
    }
    __syncthreads();
    bound = sm_bound;
  }
  const int words = (m + 31) / 32;
#pragma unroll 4
  for (int i = warp; i < words; i += kSelThreads / 32) {
    const int j = 32 * i + lane;
    const uint32_t keep = __ballot_sync(0xffffffffu, j < m && packed(j < m ? j : 0) >= bound);
    if (lane == 0) sm_keep[i] = keep;
  }
  __syncthreads();
  auto freed = [&](int i) {
    const int b = a.budget - lo - 32 * i;
    return b <= 0 ? 0u : ~sm_keep[i] & (b >= 32 ? ~0u : (1u << b) - 1);
  };
  auto taken = [&](int i) {
    const int b = a.budget - lo - 32 * i;
    return b >= 32 ? 0u : sm_keep[i] & (b <= 0 ? ~0u : ~((1u << b) - 1));
  };
  const int per = (words + kSelThreads - 1) / kSelThreads;
  const int w0 = min(tid * per, words), w1 = min(w0 + per, words);
  uint32_t total, counts = 0;  // freed in the low, taken in the high half, as above
  for (int i = w0; i < w1; ++i) counts += __popc(freed(i)) + (__popc(taken(i)) << 16);
  uint32_t before = cta_scan(counts, sm_scan, &total);
  for (int i = w0; i < w1; ++i) {
    sm_at[i] = before;
    before += __popc(freed(i)) + (__popc(taken(i)) << 16);
  }
  if (tid == 0) sm_total = total;
  cluster.sync();
  int moved_to = 0, moved_from = 0, moved = 0;
  for (int r = 0; r < size; ++r) {
    const uint32_t x = *cluster.map_shared_rank(&sm_total, r);
    if (r < rank) moved_to += x & 0xffff, moved_from += x >> 16;
    moved += x >> 16;
  }
#pragma unroll 4
  for (int i = warp; i < words; i += kSelThreads / 32) {
    const uint32_t f = freed(i), t = taken(i), lower = (1u << lane) - 1, at = sm_at[i];
    const int j = lo + 32 * i + lane;
    if (f >> lane & 1) mv[moved_to + (at & 0xffff) + __popc(f & lower)].x = j;
    if (t >> lane & 1) mv[moved_from + (at >> 16) + __popc(t & lower)].y = j;
  }
  if (LPR == 0 && rank == 0 && tid == 0) a.counts[unit] = moved;
  cluster.sync();  // the whole list is there, and no CTA leaves while its total is read
  finish_moves<LPR>(a, mv, moved, row, head, base, w, sp, rank * kSelThreads + tid, size * kSelThreads);
}

template <int LPR>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(EvictArgs a) {
  constexpr int WARPS = kMoveThreads / 32;
  const int unit = blockIdx.x, row = unit / a.kv.hkv, head = unit - row * a.kv.hkv;
  pdl_trigger();
  pdl_wait();
  const int count = a.counts[unit];
  for (int64_t m = (int64_t)(blockIdx.y * WARPS + threadIdx.x / 32) * kWarpMoves; m < count;
       m += (int64_t)gridDim.y * WARPS * kWarpMoves)
    move_rows<LPR>(a, a.moves + (int64_t)unit * a.max_moves + m, row, head, count - (int)m);
}

static int64_t evict_max_moves(const pim_paged_evict_args* a) {
  const int64_t slots = (int64_t)a->kv.max_pages * a->kv.page_size;
  const int64_t over = slots - a->budget;
  return over <= 0 ? 0 : over < a->budget ? over : a->budget;
}

static const char* evict_error(const pim_paged_evict_args* a, int dtype) {
  if (!a) return "null arguments";
  if (!dtype_ok(dtype)) return "bad dtype";
  if (const char* e = paged_kv_error(a->kv, dtype)) return e;
  if (!a->lengths || !a->positions || !a->weights || !a->slot_positions || !a->weights_out || !a->slot_positions_out ||
      !a->lengths_out)
    return "null state";
  if (a->kv.rows > 65535 || (int64_t)a->kv.rows * a->kv.kv_heads > INT32_MAX) return "too many rows";
  if (a->lengths_out == a->lengths || a->lengths_out == a->positions) return "lengths_out must be an array of its own";
  if (a->budget < 1 || a->recent < 0 || a->sink < 0 || (int64_t)a->recent + a->sink > a->budget)
    return "budget must be at least 1 and at least recent + sink";
  if (a->state_head_stride < (int64_t)a->kv.max_pages * a->kv.page_size ||
      a->state_row_stride < a->state_head_stride * a->kv.kv_heads)
    return "state strides are less than a row's slots";
  return nullptr;
}

static int64_t evict_counts_bytes(const pim_paged_evict_args* a) {
  return ((int64_t)a->kv.rows * a->kv.kv_heads * 4 + 255) / 256 * 256;
}

template <bool SMEM, int LPR>
static cudaError_t launch_select(const EvictArgs& a, size_t smem, cudaStream_t st) {
  static ResidentCache cache;
  cudaError_t e;
  if (resident_ctas(evict_select_kernel<SMEM, LPR>, kSelThreads, smem, cache, &e) < 0) return e;
  return launch_pdl(evict_select_kernel<SMEM, LPR>, dim3(a.kv.hkv, a.kv.rows), dim3(kSelThreads), smem, st, a);
}

template <int LPR>
static cudaError_t launch_cluster(const EvictArgs& a, cudaStream_t st) {
  static ResidentCache cache;
  cudaError_t e;
  const int64_t slots = (int64_t)a.kv.max_pages << a.kv.ps_log2;
  const size_t smem = (size_t)(ceil_div(ceil_div(slots, a.cluster), 32) * 32) * 4;
  if (resident_ctas(evict_cluster_kernel<LPR>, kSelThreads, smem, cache, &e) < 0) return e;
  return launch_pdl_cluster(evict_cluster_kernel<LPR>, a.cluster, dim3(a.kv.hkv * a.cluster, a.kv.rows), dim3(kSelThreads),
                            smem, st, a);
}

template <int LPR>
static cudaError_t select_rows(EvictArgs a, cudaStream_t st) {
  const int64_t slots = (int64_t)a.kv.max_pages << a.kv.ps_log2, units = (int64_t)a.kv.rows * a.kv.hkv;
  // Long rows of few units in clusters, of CTAs that have an SM and 2048 slots each.  Device us by slots 4096, 8192, 16384, 32768
  // cut to a quarter, of one CTA and of clusters:  1 unit 10.4 14.1 21.1 35.4 and 11.5 12.7 15.4 17.4;  8 units 10.9 14.7 25.5 39.1
  // and 12.2 14.0 17.5 20.6;  32 units 15.5 18.1 28.0 51.6 and 13.8 19.1 24.9 33.6;  64 units 16.3 22.1 38.3 and 16.4 23.0 33.9;
  // 8 heads of 131000 to 16384, which one CTA reads anew at each pass, 338 and 35 (rows of 64 bytes; 53 with 256); 8 heads
  // one over 16384 8.7 and 5.5.
  // CTAs of 1024 slots: 1 unit - 14.9 15.5 17.4;  two an SM: 32 units - - 32.0 43.2.
  a.cluster = 1;
  if (slots >= 8192)
    while (a.cluster < 8 && units * a.cluster * 2 <= 148 && slots >= 4096 * a.cluster) a.cluster *= 2;
  if (a.cluster > 1 && ceil_div(slots, a.cluster) <= kMaxSmemKeys - 32) return launch_cluster<LPR>(a, st);
  return slots <= kMaxSmemKeys ? launch_select<true, LPR>(a, (size_t)slots * 4, st) : launch_select<false, LPR>(a, 0, st);
}

template <int LPR>
static cudaError_t evict_rows(const EvictArgs& a, cudaStream_t st) {
  // Where a unit cannot have more moves than the selecting CTA's warps do in one go, that CTA does them: a launch less.
  // That goes by the table, not by the lengths, which are on the device: 16 rows x 8 heads one over 1024 3.6 us in a table
  // of 1040 or 1152 slots, 9.5 in one of 2048 and more.
  if (a.max_moves <= kFusedMoves) return select_rows<LPR>(a, st);
  const cudaError_t e = select_rows<0>(a, st);
  if (e != cudaSuccess) return e;
  const int by = ceil_div(a.max_moves, kWarpMoves * kMoveThreads / 32);
  return launch_pdl(evict_move_kernel<LPR>, dim3(a.kv.rows * a.kv.hkv, by < 65535 ? by : 65535), dim3(kMoveThreads), 0,
                    st, a);
}

static cudaError_t evict(const EvictArgs& a, int row_bytes, cudaStream_t st) {
  switch (row_bytes) {
    case 64: return evict_rows<4>(a, st);
    case 128: return evict_rows<8>(a, st);
    case 256: return evict_rows<16>(a, st);
    default: return evict_rows<32>(a, st);
  }
}

}  // namespace pim

extern "C" int64_t pim_paged_evict_workspace_bytes(const pim_paged_evict_args* a, int32_t dtype) {
  using namespace pim;
  if (evict_error(a, dtype)) return -1;
  return evict_counts_bytes(a) + (int64_t)a->kv.rows * a->kv.kv_heads * evict_max_moves(a) * 8;
}

extern "C" int pim_paged_evict(const pim_paged_evict_args* a, int32_t dtype, void* workspace, int64_t workspace_bytes,
                               void* stream) {
  using namespace pim;
  if (const char* e = evict_error(a, dtype)) {
    char msg[200];
    snprintf(msg, sizeof(msg), "pim_paged_evict: %s", e);
    return report_status(PIM_EINVAL, msg);
  }
  if (!workspace || workspace_bytes < pim_paged_evict_workspace_bytes(a, dtype) || !aligned16(workspace))
    return report_status(PIM_EINVAL, "pim_paged_evict: workspace too small or not 16-byte aligned");
  EvictArgs d{};
  d.kv = to_dev(a->kv);
  d.lengths = a->lengths;
  d.positions = a->positions;
  d.weights = a->weights;
  d.slot_positions = a->slot_positions;
  d.weights_out = a->weights_out;
  d.slot_positions_out = a->slot_positions_out;
  d.lengths_out = a->lengths_out;
  d.row_stride = a->state_row_stride;
  d.head_stride = a->state_head_stride;
  d.budget = a->budget;
  d.recent = a->recent;
  d.sink = a->sink;
  d.err = a->err_flag;
  d.counts = static_cast<int*>(workspace);
  d.moves = reinterpret_cast<int2*>(static_cast<char*>(workspace) + evict_counts_bytes(a));
  d.max_moves = (int)evict_max_moves(a);
  d.page_pieces = a->kv.page_stride * elem_bytes(dtype) / 16;
  return report_cuda(evict(d, a->kv.head_dim * elem_bytes(dtype), (cudaStream_t)stream), "pim_paged_evict");
}
