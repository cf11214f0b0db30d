// pim_paged_append: rotary embedding of new tokens' q and k, and their K / V rows into the
// pages of their sequences.
//
// With (c, s) the cosine and sine of the token's position and a head's halves (x1, x2):
//   (x1, x2) -> (x1 c - x2 s, x2 c + x1 s)   for q and k,   v as it is,
// in fp32 from the stored values and rounded once (pim_projection's ROPE_KV rounds each
// product too, as the HF bf16 model does; here one rounding is left).  Nothing is reused:
// every element is read once and written once, so the kernel is bound by DRAM at
// prompt sizes and by the latency of its dependent loads at one token.  A thread owns the
// 16 bytes at dim d and the 16 bytes at d + head_dim / 2, which the rotation mixes, so
// nothing is exchanged between threads.  A token's row, slot and page are found once per
// CTA (one thread per token) and shared.
//
// Many tokens: a CTA takes whole tokens, a round of its threads after another (8 prompts of up to 2048
// tokens x 96 heads, 392 MB: 67.6 us, 5.8 TB/s, with 128 threads; 71 with 256; loads issued ahead of the
// rows and pages, or several rounds at once, cost registers and with them CTAs: 76 to 82 us).  Few: a CTA
// takes one round's pieces, so that a token is spread over several, and loads them before it knows where
// they go (one token x 96 heads: 2.8 us against 4.1).

#include "paged.cuh"

namespace pim {

constexpr int kAppendThreads = 128;
constexpr int kAppendTokens = 72;  // most tokens of a CTA (a token has at least 4 items)

struct AppendArgs {
  PagedKV kv;
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride, k_head_stride, v_head_stride;
  void* q_out;
  int64_t q_out_stride;
  const float *cos, *sin;
  int max_pos, hq, pair_order;
  int64_t tokens;
  const int *starts, *lengths, *positions;
  int *lengths_out, *positions_out;
  int* slot_positions;
  float* weights;
  int64_t state_row_stride, state_head_stride;
  int* err;
};

// Item (16-byte pair) r of a token: head r / CH (q's, then k's, then v's), dims (r % CH) V .. and half a head further.
template <typename T, int HD>
struct AppendItem {
  static constexpr int V = VecW<T>::n, HALF = HD / 2, CH = HALF / V;
  int head, c, h;
  bool is_q, is_v;
  __device__ __forceinline__ AppendItem(const AppendArgs& a, int r) {
    head = r / CH;
    c = r - head * CH;
    is_q = head < a.hq;
    is_v = head >= a.hq + a.kv.hkv;
    h = is_q ? head : is_v ? head - a.hq - a.kv.hkv : head - a.hq;
  }
  __device__ __forceinline__ const T* source(const AppendArgs& a, int64_t t) const {
    return is_q   ? static_cast<const T*>(a.q) + t * a.q_stride + (int64_t)h * HD
           : is_v ? static_cast<const T*>(a.v) + t * a.v_stride + h * a.v_head_stride
                  : static_cast<const T*>(a.k) + t * a.k_stride + h * a.k_head_stride;
  }
  __device__ __forceinline__ int first(const AppendArgs& a) const { return a.pair_order ? 2 * c * V : c * V; }
  __device__ __forceinline__ int second(const AppendArgs& a) const { return a.pair_order ? 2 * c * V + V : HALF + c * V; }
  // Rotates the pair and writes it to its q_out row or slot (page offset `at`).
  __device__ __forceinline__ void put(const AppendArgs& a, int64_t t, int row, int slot, int pos, int64_t at,
                                      const int4& r1, const int4& r2) const {
    T* dst = is_q ? static_cast<T*>(a.q_out) + t * a.q_out_stride + (int64_t)h * HD
                  : static_cast<T*>(is_v ? a.kv.v : a.kv.k) + at + ((int64_t)h << a.kv.ps_log2) * HD;
    float x1[V], x2[V];
    unpack(r1, x1, T());
    unpack(r2, x2, T());
    if (a.pair_order) {  // (1st, 2nd) of each pair were adjacent
      float y[2 * V];
#pragma unroll
      for (int e = 0; e < V; ++e) y[e] = x1[e], y[V + e] = x2[e];
#pragma unroll
      for (int e = 0; e < V; ++e) x1[e] = y[2 * e], x2[e] = y[2 * e + 1];
    }
    if (!is_v && a.cos) {
      const float* cp = a.cos + (int64_t)pos * HALF + c * V;
      const float* sp = a.sin + (int64_t)pos * HALF + c * V;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float cs = cp[e], sn = sp[e];
        const float o1 = x1[e] * cs - x2[e] * sn, o2 = x2[e] * cs + x1[e] * sn;
        x1[e] = o1;
        x2[e] = o2;
      }
    }
    *reinterpret_cast<int4*>(dst + c * V) = pack(x1, T());
    *reinterpret_cast<int4*>(dst + HALF + c * V) = pack(x2, T());
    if (is_v && c == 0 && a.weights) {
      const int64_t o = row * a.state_row_stride + h * a.state_head_stride + slot;
      a.slot_positions[o] = pos;
      a.weights[o] = 0.f;
    }
  }
};

// FEW: a CTA has one item per thread of the run [128 blockIdx.x, ..) of all tokens' items; else whole tokens.
template <typename T, int HD, bool FEW>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(AppendArgs a, int tokens_per_cta, int work_ctas) {
  using Item = AppendItem<T, HD>;
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x == 0 && threadIdx.x == 0 && a.starts && (a.starts[0] < 0 || a.starts[a.kv.rows] > a.tokens))
    raise_flag(a.err);
  if ((int)blockIdx.x >= work_ctas) {  // the rows' token counts, and the lengths after the call
    const int b = (blockIdx.x - work_ctas) * kAppendThreads + threadIdx.x;
    if (b < a.kv.rows) {
      int n = 1;
      if (a.starts) {
        const int64_t count = (int64_t)a.starts[b + 1] - a.starts[b];
        if (count < 0) raise_flag(a.err);
        n = (int)min(max(count, (int64_t)0), (int64_t)INT32_MAX);
      }
      const int len = a.lengths[b];
      if (a.lengths_out) a.lengths_out[b] = len + n;
      if (a.positions_out) a.positions_out[b] = (a.positions ? a.positions[b] : len) + n;
    }
    return;
  }
  __shared__ int s_row[kAppendTokens], s_slot[kAppendTokens], s_pos[kAppendTokens];
  __shared__ int64_t s_at[kAppendTokens];
  const int per = (a.hq + 2 * a.kv.hkv) * Item::CH;  // items of a token
  const int64_t begin = FEW ? (int64_t)blockIdx.x * kAppendThreads : 0;
  const int64_t t0 = FEW ? begin / per : (int64_t)blockIdx.x * tokens_per_cta;
  const int skip = FEW ? (int)(begin - t0 * per) : 0;  // items of token t0 that the CTA before has
  const int count = FEW ? (int)min((int64_t)kAppendThreads, a.tokens * per - begin)
                        : (int)min((int64_t)tokens_per_cta, a.tokens - t0) * per;
  const int nt = (skip + count + per - 1) / per;
  int4 r1, r2;
  if (FEW) {
    const int i = skip + threadIdx.x, ti = i / per;
    const Item item(a, i - ti * per);
    const T* src = item.source(a, t0 + ti);
    r1 = ld_once_if(reinterpret_cast<const int4*>(src + item.first(a)), (int)threadIdx.x < count);
    r2 = ld_once_if(reinterpret_cast<const int4*>(src + item.second(a)), (int)threadIdx.x < count);
  }
  if ((int)threadIdx.x < nt) {
    const int64_t t = t0 + threadIdx.x;
    int row = -1;
    int64_t off = 0;
    if (!a.starts) {
      row = (int)t;
    } else if (t >= a.starts[0] && t < a.starts[a.kv.rows]) {  // the last row that starts at or before t
      int lo = 0, hi = a.kv.rows - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (a.starts[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
      row = lo;
      off = t - a.starts[row];
    }
    int64_t at = -1, slot = 0, pos = 0;
    if (row >= 0) {
      slot = a.lengths[row] + off;
      pos = (a.positions ? a.positions[row] : a.lengths[row]) + off;
      if (slot >= 0 && slot < a.kv.slots() && (!a.cos || (pos >= 0 && pos < a.max_pos)))
        at = a.kv.at<HD>(row, (int)slot, 0);
      if (at < 0) raise_flag(a.err);
    }
    s_row[threadIdx.x] = row;
    s_slot[threadIdx.x] = (int)slot;
    s_pos[threadIdx.x] = (int)pos;
    s_at[threadIdx.x] = at;
  }
  __syncthreads();
  for (int n = threadIdx.x; n < count; n += kAppendThreads) {
    const int i = skip + n, ti = i / per;
    const int64_t at = s_at[ti], t = t0 + ti;
    if (at < 0) continue;
    const Item item(a, i - ti * per);
    if (!FEW) {
      const T* src = item.source(a, t);
      r1 = *reinterpret_cast<const int4*>(src + item.first(a));
      r2 = *reinterpret_cast<const int4*>(src + item.second(a));
    }
    item.put(a, t, s_row[ti], s_slot[ti], s_pos[ti], at, r1, r2);
  }
}

static cudaError_t append(const AppendArgs& a, int hd, int dtype, cudaStream_t st) {
  return dispatch_type_dim(dtype, hd, [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int HD = decltype(d)::value;
    const int per = (a.hq + 2 * a.kv.hkv) * (HD / 2 / VecW<T>::n);
    const int64_t items = a.tokens * per;
    const int tail = a.lengths_out || a.positions_out || a.starts ? ceil_div(a.kv.rows, kAppendThreads) : 0;
    // few: the items do not fill the GPU's threads
    if (items <= 2048 * 148) {
      const int work = ceil_div(items, kAppendThreads);
      if (work + tail == 0) return cudaSuccess;
      return launch_pdl(append_kernel<T, HD, true>, dim3(work + tail), dim3(kAppendThreads), 0, st, a, 0, work);
    }
    int tpc = 2 * kAppendThreads / per;  // tokens of a CTA: two rounds of its threads
    tpc = tpc < 1 ? 1 : tpc > 64 ? 64 : tpc;
    const int work = ceil_div(a.tokens, tpc);
    return launch_pdl(append_kernel<T, HD, false>, dim3(work + tail), dim3(kAppendThreads), 0, st, a, tpc, work);
  });
}

}  // namespace pim

extern "C" int pim_paged_append(const pim_paged_append_args* a, int32_t dtype, void* stream) {
  using namespace pim;
  auto bad = [](const char* what) {
    char msg[200];
    snprintf(msg, sizeof(msg), "pim_paged_append: %s", what);
    return report_status(PIM_EINVAL, msg);
  };
  if (!a) return bad("null arguments");
  if (!dtype_ok(dtype)) return bad("bad dtype");
  if (const char* e = paged_kv_error(a->kv, dtype)) return bad(e);
  const int es = elem_bytes(dtype), hd = a->kv.head_dim;
  if (a->tokens < 0 || a->tokens > (1 << 30)) return bad("bad number of tokens");
  if (!a->lengths || (a->tokens > 0 && (!a->k || !a->v))) return bad("null k, v or lengths");
  if (!a->starts && a->tokens != a->kv.rows) return bad("without starts there is one token per row");
  if ((a->q != nullptr) != (a->q_out != nullptr)) return bad("q and q_out go together");
  if (a->q && (a->q_heads <= 0 || a->q_heads > 65535)) return bad("bad q_heads");
  if ((a->rope_cos != nullptr) != (a->rope_sin != nullptr)) return bad("rope_cos and rope_sin go together");
  if (a->rope_cos && a->max_pos <= 0) return bad("bad max_pos");
  if ((a->slot_positions != nullptr) != (a->weights != nullptr)) return bad("slot_positions and weights go together");
  if (a->weights && (a->state_head_stride < (int64_t)a->kv.max_pages * a->kv.page_size ||
                     a->state_row_stride < a->state_head_stride * a->kv.kv_heads))
    return bad("state strides are less than a row's slots");
  if (a->lengths_out == a->lengths || (a->positions_out && a->positions_out == a->lengths) ||
      (a->positions_out && a->positions_out == a->positions) || (a->lengths_out && a->lengths_out == a->positions) ||
      (a->lengths_out && a->lengths_out == a->positions_out))
    return bad("lengths_out and positions_out must be arrays of their own");
  if (a->q && (a->q_stride < (int64_t)a->q_heads * hd || a->q_out_stride < (int64_t)a->q_heads * hd))
    return bad("q strides are less than a row");
  if (a->q && a->q == a->q_out && (a->pair_order || a->q_stride != a->q_out_stride))
    return bad("q in place needs the same stride and no pair_order");
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->q_out) || a->q_stride * es % 16 ||
      a->k_stride * es % 16 || a->v_stride * es % 16 || a->k_head_stride * es % 16 || a->v_head_stride * es % 16 ||
      a->q_out_stride * es % 16)
    return bad("q, k, v, q_out and their strides must be 16-byte aligned");
  AppendArgs d{};
  d.kv = to_dev(a->kv);
  d.q = a->q;
  d.k = a->k;
  d.v = a->v;
  d.q_stride = a->q_stride;
  d.k_stride = a->k_stride;
  d.v_stride = a->v_stride;
  d.k_head_stride = a->k_head_stride;
  d.v_head_stride = a->v_head_stride;
  d.q_out = a->q_out;
  d.q_out_stride = a->q_out_stride;
  d.cos = a->rope_cos;
  d.sin = a->rope_sin;
  d.max_pos = a->max_pos;
  d.hq = a->q ? a->q_heads : 0;
  d.pair_order = a->pair_order;
  d.tokens = a->tokens;
  d.starts = a->starts;
  d.lengths = a->lengths;
  d.positions = a->positions;
  d.lengths_out = a->lengths_out;
  d.positions_out = a->positions_out;
  d.slot_positions = a->slot_positions;
  d.weights = a->weights;
  d.state_row_stride = a->state_row_stride;
  d.state_head_stride = a->state_head_stride;
  d.err = a->err_flag;
  return report_cuda(append(d, hd, dtype, (cudaStream_t)stream), "pim_paged_append");
}
