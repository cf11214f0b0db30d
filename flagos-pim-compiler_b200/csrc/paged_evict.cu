// pim_paged_evict: a paged cache cut down to a budget by accumulated attention weight.
//
// Per (row, kv head), over the n slots in use: a token that must stay (recent or sink) ranks
// above every weight; the budget largest stay, of equal ones the lower slot.  The selection
// is a radix select: weights map to unsigned keys of the same order, three passes over
// 11 + 11 + 10 bits find the key of the budget-th largest and how many equal to it stay.
// A scan in slot order then lists the freed slots below the budget and the kept ones above
// it; there are equally many, and moving the i-th kept one into the i-th freed slot moves the
// fewest rows that any compaction can.  Sources lie at or above the budget and destinations
// below it, so the moves need no order.
//
// evict_select_kernel: one CTA per (row, head), keys in shared memory where they fit; it
// reads 8 bytes a slot and writes the state and the list of moves.  evict_move_kernel: moves
// the K and V rows, a grid over (row, head) x blocks of moves; bound by DRAM.

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
  int smem_keys;  // keys that fit the shared memory of the launch
};

constexpr int kSelThreads = 512;
constexpr int kMaxSmemKeys = 48 * 1024;
constexpr int kMoveThreads = 256;

// Unsigned key of the same order as the weight; NaN lowest.  -0 and +0 are equal.
__device__ __forceinline__ uint32_t order_key(float w) {
  w += 0.f;
  if (w != w) return 0;
  const uint32_t u = __float_as_uint(w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive prefix sum over the CTA (kSelThreads threads); *total: the sum.
__device__ __forceinline__ int cta_scan(int v, int* sm, int* total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) sm[warp] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelThreads / 32; ++w) {
    if (w < warp) before += sm[w];
    all += sm[w];
  }
  *total = all;
  return x - v + before;
}

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(EvictArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ int hist[2048];
  __shared__ int sm_scan[kSelThreads / 32];
  __shared__ int sm_bin, sm_above;
  const int head = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  pdl_trigger();
  pdl_wait();
  const int want = a.lengths[row];
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
  const int64_t from = (int64_t)a.positions[row] - a.recent;
  auto make_key = [&](float wt, int p) { return p >= from || p < a.sink ? 0xffffffffu : order_key(wt); };
  const bool evicts = n > a.budget, in_smem = n <= a.smem_keys;
  // one pass over the state, kLoads slots of a thread in flight: the kept part's copy and the keys
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
      if (i < n && evicts && in_smem) keys[i] = make_key(wt[u], p[u]);
    }
  }
  if (!evicts) {
    if (tid == 0 && a.max_moves > 0) a.counts[unit] = 0;
    return;
  }
  auto key = [&](int j) { return in_smem ? keys[j] : make_key(w[j], sp[j]); };
  // the budget-th largest key
  uint32_t prefix = 0;
  int need = a.budget, shift = 32;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int bits = pass < 2 ? 11 : 10, bins = 1 << bits;
    const uint32_t top = pass ? ~0u << shift : 0;  // bits fixed so far
    shift -= bits;
    for (int i = tid; i < 2048; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int j = tid; j < n; j += kSelThreads) {
      const uint32_t k = key(j);
      if ((k & top) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1);
    }
    __syncthreads();
    // thread t owns the bins 2047 - 4t .. 2044 - 4t, so the scan runs from the largest bin down
    constexpr int OWN = 2048 / kSelThreads;
    int c[OWN], sum = 0, total;
#pragma unroll
    for (int i = 0; i < OWN; ++i) sum += c[i] = hist[2047 - OWN * tid - i];
    int above = cta_scan(sum, sm_scan, &total);
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      if (above < need && need <= above + c[i]) sm_bin = 2047 - OWN * tid - i, sm_above = above;
      above += c[i];
    }
    __syncthreads();
    prefix |= (uint32_t)sm_bin << shift;
    need -= sm_above;
  }
  // prefix: the smallest key kept; `need` of those equal to it stay, the lowest slots first.
  // A thread owns consecutive slots (an odd number of them: no shared-memory bank conflicts).
  const int per = ((n + kSelThreads - 1) / kSelThreads) | 1;
  const int j0 = min((int64_t)tid * per, (int64_t)n), j1 = min(j0 + per, n);
  int total, eq = 0;
  for (int j = j0; j < j1; ++j) eq += key(j) == prefix;
  const int eq0 = cta_scan(eq, sm_scan, &total);
  int holes = 0, sources = 0, e = eq0;
  for (int j = j0; j < j1; ++j) {
    const uint32_t k = key(j);
    const bool keep = k > prefix || (k == prefix && e++ < need);
    holes += !keep && j < a.budget;
    sources += keep && j >= a.budget;
  }
  const int h0 = cta_scan(holes, sm_scan, &total);
  int moved;
  const int s0 = cta_scan(sources, sm_scan, &moved);
  int2* mv = a.moves + (int64_t)unit * a.max_moves;
  int hi = h0, si = s0;
  e = eq0;
  for (int j = j0; j < j1; ++j) {
    const uint32_t k = key(j);
    const bool keep = k > prefix || (k == prefix && e++ < need);
    if (!keep && j < a.budget) mv[hi++].x = j;
    if (keep && j >= a.budget) mv[si++].y = j;
  }
  if (tid == 0) a.counts[unit] = moved;
  __syncthreads();
  for (int i = tid; i < moved; i += kSelThreads) {
    const int2 m = mv[i];
    a.weights_out[base + m.x] = w[m.y];
    a.slot_positions_out[base + m.x] = sp[m.y];
  }
}

// Up to kWarpMoves moves of a unit's list by one warp.  Each lane finds one row (the freed or the
// kept slot of a move: one table entry), then all lanes copy 16-byte pieces, eight loads under
// way at a time, with the rows' places taken from the lanes that know them.
constexpr int kWarpMoves = 16;
template <typename T, int HD>
__device__ __forceinline__ void move_rows(const EvictArgs& a, const int2* moves, int row, int head, int count) {
  constexpr int LPR = HD * (int)sizeof(T) / 16;        // pieces of a K or V row
  constexpr int STEPS = kWarpMoves * 2 * LPR / 32, FLY = STEPS < 8 ? STEPS : 8;
  const int lane = threadIdx.x % 32, mine = lane % kWarpMoves;
  int64_t at = -1;
  if (mine < count) {
    const int2 mv = moves[mine];
    at = a.kv.at<HD>(row, lane < kWarpMoves ? mv.x : mv.y, head);
    if (at < 0) raise_flag(a.err);
  }
  for (int s0 = 0; s0 < STEPS; s0 += FLY) {
    int4 v[FLY];
    int64_t to[FLY];
#pragma unroll
    for (int u = 0; u < FLY; ++u) {
      const int flat = (s0 + u) * 32 + lane, m = flat / (2 * LPR), r = flat % (2 * LPR), piece = r % LPR;
      const int64_t src = __shfl_sync(0xffffffffu, at, kWarpMoves + m);
      to[u] = __shfl_sync(0xffffffffu, at, m);
      T* p = static_cast<T*>(r < LPR ? a.kv.k : a.kv.v);
      if (src < 0) to[u] = -1;
      v[u] = ld_once_if(reinterpret_cast<const int4*>(p + src) + piece, to[u] >= 0);
    }
#pragma unroll
    for (int u = 0; u < FLY; ++u) {
      const int r = ((s0 + u) * 32 + lane) % (2 * LPR), piece = r % LPR;
      T* p = static_cast<T*>(r < LPR ? a.kv.k : a.kv.v);
      if (to[u] >= 0) reinterpret_cast<int4*>(p + to[u])[piece] = v[u];
    }
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(EvictArgs a) {
  constexpr int WARPS = kMoveThreads / 32;
  const int unit = blockIdx.x, row = unit / a.kv.hkv, head = unit - row * a.kv.hkv;
  pdl_trigger();
  pdl_wait();
  const int count = a.counts[unit];
  for (int64_t m = (int64_t)(blockIdx.y * WARPS + threadIdx.x / 32) * kWarpMoves; m < count;
       m += (int64_t)gridDim.y * WARPS * kWarpMoves)
    move_rows<T, HD>(a, a.moves + (int64_t)unit * a.max_moves + m, row, head, count - (int)m);
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

static cudaError_t evict(EvictArgs& a, int hd, int dtype, cudaStream_t st) {
  static ResidentCache cache;
  a.smem_keys = (int)min((int64_t)kMaxSmemKeys, (int64_t)a.kv.max_pages << a.kv.ps_log2);
  cudaError_t e;
  if (resident_ctas(evict_select_kernel, kSelThreads, (size_t)a.smem_keys * 4, cache, &e) < 0) return e;
  e = launch_pdl(evict_select_kernel, dim3(a.kv.hkv, a.kv.rows), dim3(kSelThreads), (size_t)a.smem_keys * 4, st, a);
  if (e != cudaSuccess || a.max_moves == 0) return e;
  return dispatch_type_dim(dtype, hd, [&](auto t, auto d) {
    const int by = ceil_div(a.max_moves, kWarpMoves * kMoveThreads / 32);
    return launch_pdl(evict_move_kernel<decltype(t), decltype(d)::value>,
                      dim3(a.kv.rows * a.kv.hkv, by < 65535 ? by : 65535), dim3(kMoveThreads), 0, st, a);
  });
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
  return report_cuda(evict(d, a->kv.head_dim, dtype, (cudaStream_t)stream), "pim_paged_evict");
}
