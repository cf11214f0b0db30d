// pim_beam_select and pim_beam_reorder: one step of beam search over a paged cache.
//
// Selection.  With lse_w = log sum_t exp(x[w][t]) the candidates are
//   c(w, t) = score_w + x[w][t] - lse_w,
// and the best K over all beams and tokens come out, ties to the lowest w * vocab + t.
// Within a beam c falls with x, so each chunk of a beam's vocabulary only has to give its K
// largest logits: beam_partial_kernel reads every logit once, into registers, and leaves per
// chunk the sorted K largest (as 64-bit keys: the logit's order-preserving bits above the
// complement of its token, so keys are unique and equal logits rank by token) and the
// chunk's maximum and sum of exponentials.  K-th largest of a chunk: it is at least the K-th
// largest of the threads' maxima, and only K threads can hold values at or above that bound, so
// at most K * 16 keys are left to rank by counting.  beam_merge_kernel joins the sums to the
// beams' lse in fp64 (neighbouring candidates decide which tokens come out) and merges the
// sorted lists: K rounds of a maximum over the lists' heads.
//
// Reordering.  See pim_beam_reorder in pim_b200.h: the table entries of full pages follow
// the parent, the partly filled pages of an entry's beams are dealt out again, and the
// copies read pages of beams with children and write pages of beams without.

#include <math.h>

#include "paged.cuh"

namespace pim {

constexpr int kBeamThreads = 256;
constexpr int kBeamVals = 16;  // logits of a thread
constexpr int kBeamChunk = kBeamThreads * kBeamVals;
constexpr int kMaxBeams = 64;

struct BeamStats {
  float max;
  int count;   // entries of the chunk's list
  double sum;  // of exp(x - max) over the chunk's finite logits
};

struct BeamSelectArgs {
  const void* logits;
  int64_t stride;
  const float* scores;
  const int* done;
  float* scores_out;
  int *parents, *tokens, *done_out;
  int batch, beams, k, vocab, eos, pad, splits;
  BeamStats* stats;           // [batch * beams][splits]
  unsigned long long* lists;  // [batch * beams][splits][k]
};

// A logit's key: larger is better; 0 for a logit that is no candidate.
__device__ __forceinline__ unsigned long long beam_key(float x, int token) {
  if (!isfinite(x)) return 0;
  const uint32_t u = __float_as_uint(x + 0.f);
  const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
  return ((unsigned long long)o << 32) | (uint32_t)~token;
}
__device__ __forceinline__ float key_logit(unsigned long long key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int key_token(unsigned long long key) { return (int)~(uint32_t)key; }

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kBeamThreads) beam_partial_kernel(BeamSelectArgs a) {
  constexpr int V = VecW<T>::n;
  __shared__ unsigned long long sm_max[kBeamThreads];
  __shared__ unsigned long long sm_cand[kMaxBeams * kBeamVals];
  __shared__ unsigned long long sm_tau;
  __shared__ int sm_n;
  __shared__ float sm_m[kBeamThreads / 32];
  __shared__ double sm_s[kBeamThreads / 32];
  const int split = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  pdl_trigger();
  pdl_wait();
  if (a.done && a.done[row]) return;  // offers one candidate, which the merge adds
  const T* x = static_cast<const T*>(a.logits) + row * a.stride;
  const int base = split * kBeamChunk;
  float v[kBeamVals];
  // value i of this thread is token base + tok(i)
  auto tok = [&](int i) { return ALIGNED ? (i / V) * kBeamThreads * V + tid * V + i % V : i * kBeamThreads + tid; };
#pragma unroll
  for (int i = 0; i < kBeamVals; ++i) v[i] = -INFINITY;
  if (ALIGNED) {
    int4 raw[kBeamVals / V];
#pragma unroll
    for (int i = 0; i < kBeamVals / V; ++i)
      if (base + tok(i * V) < a.vocab) raw[i] = ld_once(reinterpret_cast<const int4*>(x + base + tok(i * V)));
#pragma unroll
    for (int i = 0; i < kBeamVals / V; ++i)
      if (base + tok(i * V) < a.vocab) {
        float f[V];
        unpack(raw[i], f, T());
#pragma unroll
        for (int e = 0; e < V; ++e) v[i * V + e] = f[e];
      }
  } else {
#pragma unroll
    for (int i = 0; i < kBeamVals; ++i)
      if (base + tok(i) < a.vocab) v[i] = to_f(x[base + tok(i)]);
  }
  unsigned long long mine = 0;
#pragma unroll
  for (int i = 0; i < kBeamVals; ++i) {
    if (!isfinite(v[i])) v[i] = -INFINITY;
    const unsigned long long k = beam_key(v[i], base + tok(i));
    mine = k > mine ? k : mine;
  }
  sm_max[tid] = mine;
  if (tid == 0) sm_n = 0, sm_tau = 1;
  const float wm = warp_max(mine ? key_logit(mine) : -INFINITY);
  if (lane == 0) sm_m[warp] = wm;
  __syncthreads();
  float m = sm_m[0];
#pragma unroll
  for (int w = 1; w < kBeamThreads / 32; ++w) m = fmaxf(m, sm_m[w]);
  // fp32 exponentials and a thread's 16 of them; the sum over threads in fp64
  float part = 0.f;
  if (m != -INFINITY) {
#pragma unroll
    for (int i = 0; i < kBeamVals; ++i) part += expf(v[i] - m);
  }
  double s = part;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) sm_s[warp] = s;
  // the k-th largest of the threads' maxima bounds the chunk's k-th largest from below
  int above = 0;
  for (int i = 0; i < kBeamThreads; ++i) above += sm_max[i] > mine;
  if (mine && above == a.k - 1) sm_tau = mine;
  __syncthreads();
  const unsigned long long tau = sm_tau;
  if (mine >= tau) {
#pragma unroll
    for (int i = 0; i < kBeamVals; ++i) {
      const unsigned long long k = beam_key(v[i], base + tok(i));
      if (k >= tau) sm_cand[atomicAdd(&sm_n, 1)] = k;  // at most k threads come here, with 16 keys each
    }
  }
  __syncthreads();
  const int n = sm_n, out = min(n, a.k);
  unsigned long long* list = a.lists + ((int64_t)row * a.splits + split) * a.k;
  for (int i = tid; i < n; i += kBeamThreads) {
    const unsigned long long k = sm_cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += sm_cand[j] > k;
    if (rank < a.k) list[rank] = k;
  }
  if (tid == 0) {
    BeamStats st;
    st.max = m;
    st.count = out;
    st.sum = 0;
    for (int w = 0; w < kBeamThreads / 32; ++w) st.sum += sm_s[w];
    a.stats[(int64_t)row * a.splits + split] = st;
  }
}

struct BeamBest {
  double score;   // -inf: none
  int64_t flat;   // beam * vocab + token
};
__device__ __forceinline__ bool better(const BeamBest& x, const BeamBest& y) {
  return x.score > y.score || (x.score == y.score && x.flat < y.flat);
}

constexpr int kMergeThreads = 256;

__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(BeamSelectArgs a) {
  extern __shared__ unsigned char sm_next[];  // [beams * splits] entries of each list that are taken
  __shared__ double sm_shift[kMaxBeams];      // score_w - lse_w; -inf: the beam offers nothing
  __shared__ int sm_done[kMaxBeams];
  __shared__ BeamBest sm_best[kMergeThreads / 32];
  __shared__ int sm_list[kMergeThreads / 32];
  const int b = blockIdx.x, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  pdl_trigger();
  pdl_wait();
  const int lists = a.beams * a.splits;
  for (int i = tid; i < lists; i += kMergeThreads) sm_next[i] = 0;
  for (int w = warp; w < a.beams; w += kMergeThreads / 32) {
    const int row = b * a.beams + w;
    const int done = a.done ? a.done[row] : 0;
    const float score = a.scores[row];
    double shift = score;
    if (!done) {
      float m = -INFINITY;
      for (int i = lane; i < a.splits; i += 32) m = fmaxf(m, a.stats[(int64_t)row * a.splits + i].max);
      m = warp_max(m);
      double s = 0;
      if (m != -INFINITY)
        for (int i = lane; i < a.splits; i += 32) {
          const BeamStats st = a.stats[(int64_t)row * a.splits + i];
          if (st.max != -INFINITY) s += st.sum * exp((double)st.max - (double)m);
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      shift = m == -INFINITY ? -INFINITY : (double)score - ((double)m + log(s));
    }
    if (lane == 0) {
      sm_shift[w] = isfinite(score) ? shift : -INFINITY;
      sm_done[w] = done;
    }
  }
  __syncthreads();
  // the head of list l
  auto head = [&](int l) {
    BeamBest c{-INFINITY, INT64_MAX};
    const int w = l / a.splits, split = l - w * a.splits, at = sm_next[l];
    if (sm_shift[w] == -INFINITY) return c;
    if (sm_done[w]) {
      if (split == 0 && at == 0) c.score = sm_shift[w], c.flat = (int64_t)w * a.vocab + a.pad;
      return c;
    }
    const int64_t list = (int64_t)(b * a.beams + w) * a.splits + split;
    if (at >= a.stats[list].count) return c;
    const unsigned long long k = a.lists[list * a.k + at];
    c.score = sm_shift[w] + (double)key_logit(k);
    c.flat = (int64_t)w * a.vocab + key_token(k);
    return c;
  };
  BeamBest mine{-INFINITY, INT64_MAX};
  int mine_list = -1;
  auto refresh = [&]() {
    mine = BeamBest{-INFINITY, INT64_MAX};
    for (int l = tid; l < lists; l += kMergeThreads) {
      const BeamBest c = head(l);
      if (better(c, mine)) mine = c, mine_list = l;
    }
  };
  refresh();
  for (int j = 0; j < a.k; ++j) {
    BeamBest best = mine;
    int from = mine_list;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      BeamBest other;
      other.score = __shfl_xor_sync(0xffffffffu, best.score, o);
      other.flat = __shfl_xor_sync(0xffffffffu, (long long)best.flat, o);
      const int of = __shfl_xor_sync(0xffffffffu, from, o);
      if (better(other, best)) best = other, from = of;
    }
    __syncthreads();
    if (lane == 0) sm_best[warp] = best, sm_list[warp] = from;
    __syncthreads();
    best = sm_best[0];
    from = sm_list[0];
#pragma unroll
    for (int w = 1; w < kMergeThreads / 32; ++w)
      if (better(sm_best[w], best)) best = sm_best[w], from = sm_list[w];
    const bool none = best.score == -INFINITY;
    const int parent = none ? 0 : (int)(best.flat / a.vocab);
    const int token = none ? a.pad : (int)(best.flat - (int64_t)parent * a.vocab);
    if (tid == 0) {
      const int64_t o = (int64_t)b * a.k + j;
      a.scores_out[o] = (float)best.score;
      a.parents[o] = parent;
      a.tokens[o] = token;
      if (a.done_out) a.done_out[o] = none || sm_done[parent] || (a.eos >= 0 && token == a.eos);
    }
    if (!none && from % kMergeThreads == tid) {
      sm_next[from]++;
      refresh();
    }
  }
}

struct BeamReorderArgs {
  char* pages;
  int64_t block_bytes, page_bytes;
  const int* table;
  int* table_out;
  int64_t table_stride;
  const int *lengths, *parents;
  int beams, num_blocks, max_pages, num_pages, ps_log2, hkv, row_bytes;
  int* err;
};

__global__ void __launch_bounds__(256) beam_reorder_kernel(BeamReorderArgs a) {
  __shared__ int sm_parent[kMaxBeams], sm_page[kMaxBeams], sm_first[kMaxBeams], sm_childless[kMaxBeams];
  __shared__ int sm_bad, sm_take;
  const int row = blockIdx.x, b = row / a.beams, j = row - b * a.beams, tid = threadIdx.x;
  pdl_trigger();
  pdl_wait();
  const int n = a.lengths[b], ps = 1 << a.ps_log2;
  const int full = n >> a.ps_log2, fill = n & (ps - 1);
  if (tid == 0) sm_bad = n < 0 || n > (int64_t)a.max_pages << a.ps_log2, sm_take = 0;
  __syncthreads();
  if (tid < a.beams) {
    const int p = a.parents[b * a.beams + tid];
    sm_parent[tid] = p;
    if (p < 0 || p >= a.beams) sm_bad = 1;
    if (!sm_bad && fill) {  // (a length out of range was seen before the barrier: `full` is an entry of the table)
      const int page = a.table[(int64_t)(b * a.beams + tid) * a.table_stride + full];
      sm_page[tid] = page;
      if (page < 0 || page >= a.num_pages) sm_bad = 1;
    }
  }
  __syncthreads();
  const bool bad = sm_bad;
  if (bad && tid == 0 && blockIdx.y == 0) raise_flag(a.err);
  if (tid < a.beams && !bad) {
    bool first = true, childless = true;
    for (int i = 0; i < a.beams; ++i) {
      if (i < tid && sm_parent[i] == sm_parent[tid]) first = false;
      if (sm_parent[i] == tid) childless = false;
    }
    sm_first[tid] = first;
    sm_childless[tid] = childless;
  }
  __syncthreads();
  const int parent = bad ? j : sm_parent[j];
  const bool copies = !bad && fill && !sm_first[j];
  if (copies && tid < a.beams) {  // the i-th further child takes the page of the i-th beam without a child
    int nth = 0, order = 0;
    for (int i = 0; i < j; ++i) nth += !sm_first[i];
    for (int i = 0; i < tid; ++i) order += sm_childless[i];
    if (sm_childless[tid] && order == nth) sm_take = tid;
  }
  __syncthreads();
  const int take = copies ? sm_take : parent;
  if (blockIdx.y == 0) {
    const int* mine = a.table + row * a.table_stride;
    const int* theirs = a.table + (int64_t)(b * a.beams + parent) * a.table_stride;
    for (int i = tid; i < a.max_pages; i += blockDim.x) {
      int page = bad || i > full || (i == full && !fill) ? mine[i] : theirs[i];
      if (!bad && fill && i == full) page = sm_page[take];
      a.table_out[row * a.table_stride + i] = page;
    }
  }
  if (!copies) return;
  const int per_head = fill * a.row_bytes / 16, head_pieces = a.row_bytes << a.ps_log2 >> 4;
  for (int blk = blockIdx.y; blk < a.num_blocks; blk += gridDim.y) {
    char* block = a.pages + blk * a.block_bytes;
    const int4* src = reinterpret_cast<const int4*>(block + sm_page[parent] * a.page_bytes);
    int4* dst = reinterpret_cast<int4*>(block + sm_page[take] * a.page_bytes);
    for (int i = tid; i < a.hkv * per_head; i += blockDim.x) {
      const int h = i / per_head, r = i - h * per_head;
      dst[(int64_t)h * head_pieces + r] = src[(int64_t)h * head_pieces + r];
    }
  }
}

static const char* beam_select_error(const pim_beam_select_args* a, int dtype) {
  if (!a) return "null arguments";
  if (!dtype_ok(dtype)) return "bad dtype";
  if (!a->logits || !a->scores || !a->scores_out || !a->parents || !a->tokens) return "null pointer";
  if (a->batch <= 0 || a->beams <= 0 || a->beams > kMaxBeams || a->beams_out <= 0 || a->beams_out > kMaxBeams)
    return "batch must be positive, beams and beams_out 1 to 64";
  if (a->vocab <= 0 || a->vocab > (1 << 22) || (int64_t)a->batch * a->beams > 65535)
    return "vocab must be 1 to 2^22, batch * beams at most 65535";
  if (a->logits_stride < a->vocab) return "logits_stride is less than vocab";
  if ((uintptr_t)a->logits % elem_bytes(dtype)) return "logits are not aligned to their type";
  if (a->eos < -1 || a->eos >= a->vocab || a->pad < 0 || a->pad >= a->vocab) return "eos or pad outside the vocabulary";
  if (a->scores_out == a->scores || (a->done && a->done_out == a->done))
    return "scores_out and done_out must be arrays of their own";
  return nullptr;
}

static int beam_splits(int vocab) { return ceil_div(vocab, kBeamChunk); }

static int64_t beam_stats_bytes(const pim_beam_select_args* a) {
  return (int64_t)a->batch * a->beams * beam_splits(a->vocab) * (int64_t)sizeof(BeamStats);
}

template <typename T>
static cudaError_t beam_select(const BeamSelectArgs& a, cudaStream_t st) {
  const bool aligned = aligned16(a.logits) && a.stride * sizeof(T) % 16 == 0 && a.vocab % VecW<T>::n == 0;
  const dim3 grid(a.splits, a.batch * a.beams);
  cudaError_t e = aligned ? launch_pdl(beam_partial_kernel<T, true>, grid, dim3(kBeamThreads), 0, st, a)
                          : launch_pdl(beam_partial_kernel<T, false>, grid, dim3(kBeamThreads), 0, st, a);
  if (e != cudaSuccess) return e;
  static ResidentCache cache;
  const size_t smem = ((size_t)a.beams * a.splits + 15) / 16 * 16;
  if (resident_ctas(beam_merge_kernel, kMergeThreads, smem, cache, &e) < 0) return e;
  return launch_pdl(beam_merge_kernel, dim3(a.batch), dim3(kMergeThreads), smem, st, a);
}

}  // namespace pim

extern "C" int64_t pim_beam_select_workspace_bytes(const pim_beam_select_args* a, int32_t dtype) {
  using namespace pim;
  if (beam_select_error(a, dtype)) return -1;
  return beam_stats_bytes(a) + (int64_t)a->batch * a->beams * beam_splits(a->vocab) * a->beams_out * 8;
}

extern "C" int pim_beam_select(const pim_beam_select_args* a, int32_t dtype, void* workspace, int64_t workspace_bytes,
                               void* stream) {
  using namespace pim;
  if (const char* e = beam_select_error(a, dtype)) {
    char msg[200];
    snprintf(msg, sizeof(msg), "pim_beam_select: %s", e);
    return report_status(PIM_EINVAL, msg);
  }
  if (!workspace || workspace_bytes < pim_beam_select_workspace_bytes(a, dtype) || !aligned16(workspace))
    return report_status(PIM_EINVAL, "pim_beam_select: workspace too small or not 16-byte aligned");
  BeamSelectArgs d{};
  d.logits = a->logits;
  d.stride = a->logits_stride;
  d.scores = a->scores;
  d.done = a->done;
  d.scores_out = a->scores_out;
  d.parents = a->parents;
  d.tokens = a->tokens;
  d.done_out = a->done_out;
  d.batch = a->batch;
  d.beams = a->beams;
  d.k = a->beams_out;
  d.vocab = a->vocab;
  d.eos = a->eos;
  d.pad = a->pad;
  d.splits = beam_splits(a->vocab);
  d.stats = static_cast<BeamStats*>(workspace);
  d.lists = reinterpret_cast<unsigned long long*>(static_cast<char*>(workspace) + beam_stats_bytes(a));
  return report_cuda(dtype == PIM_BF16 ? beam_select<__nv_bfloat16>(d, (cudaStream_t)stream)
                                       : beam_select<float>(d, (cudaStream_t)stream),
                     "pim_beam_select");
}

extern "C" int pim_beam_reorder(const pim_beam_reorder_args* a, int32_t dtype, void* stream) {
  using namespace pim;
  auto bad = [](const char* what) {
    char msg[200];
    snprintf(msg, sizeof(msg), "pim_beam_reorder: %s", what);
    return report_status(PIM_EINVAL, msg);
  };
  if (!a) return bad("null arguments");
  if (!dtype_ok(dtype)) return bad("bad dtype");
  if (!a->pages || !a->table || !a->table_out || !a->lengths || !a->parents) return bad("null pointer");
  if (a->table == a->table_out) return bad("table_out must be an array of its own");
  if (!page_geometry_ok(a->page_size, a->kv_heads, a->head_dim))
    return bad("page_size must be 8, 16, 32, 64, 128 or 256, head_dim 32, 64 or 128, kv_heads 1 to 65535");
  if (a->batch <= 0 || a->beams <= 0 || a->beams > kMaxBeams || (int64_t)a->batch * a->beams > (1 << 30))
    return bad("batch must be positive, beams 1 to 64");
  if (a->num_blocks <= 0 || a->max_pages <= 0 || a->num_pages <= 0 || a->table_stride < a->max_pages ||
      (int64_t)a->max_pages * a->page_size > (1 << 30))
    return bad("bad block or page counts");
  const int es = elem_bytes(dtype);
  const int64_t page = (int64_t)a->kv_heads * a->page_size * a->head_dim;
  if (a->page_stride < page || (a->num_blocks > 1 && a->block_stride < page)) return bad("strides are less than a page");
  if (!aligned16(a->pages) || a->page_stride * es % 16 || a->block_stride * es % 16)
    return bad("pages must be 16-byte aligned");
  BeamReorderArgs d{};
  d.pages = static_cast<char*>(a->pages);
  d.block_bytes = a->block_stride * es;
  d.page_bytes = a->page_stride * es;
  d.table = a->table;
  d.table_out = a->table_out;
  d.table_stride = a->table_stride;
  d.lengths = a->lengths;
  d.parents = a->parents;
  d.beams = a->beams;
  d.num_blocks = a->num_blocks;
  d.max_pages = a->max_pages;
  d.num_pages = a->num_pages;
  d.ps_log2 = ilog2(a->page_size);
  d.hkv = a->kv_heads;
  d.row_bytes = a->head_dim * es;
  d.err = a->err_flag;
  const int by = a->num_blocks < 65535 ? a->num_blocks : 65535;
  return report_cuda(launch_pdl(beam_reorder_kernel, dim3(a->batch * a->beams, by), dim3(256), 0, (cudaStream_t)stream, d),
                     "pim_beam_reorder");
}
