// pim_beam_select and pim_beam_reorder: one step of beam search over a paged cache.
//
// Selection.  With lse_w = log sum_t exp(x[w][t]) the candidates are
//   c(w, t) = score_w + x[w][t] - lse_w,
// and the best K over all beams and tokens come out, ties to the lowest w * vocab + t.
// Within a beam c falls with x, so each chunk of a beam's vocabulary only has to give its K
// largest logits: beam_partial_kernel reads every logit once, into registers, and leaves per
// chunk the sorted K largest (as 64-bit keys: the logit's order-preserving bits above the
// complement of its token, so keys are unique and equal logits rank by token) and the
// chunk's maximum and sum of exponentials.  beam_merge_kernel joins the sums to the beams' lse,
// merges each beam's lists with one warp and then the beams.  Exponentials and sums are fp64
// throughout: candidates of different beams that lie next to one another decide which tokens come
// out, and fp32's error (3e-7 in a row of equal logits) is the same for every term of such a row.
//
// The K largest of a chunk: if every warp's ceil(K / warps)-th largest lane maximum is at least
// tau, then K values are, so only those >= tau, a few times K of them, are collected and ranked
// by counting.  Finding tau costs one warp reduction per rank instead of a sort.  Where that
// collects too many, the K-th largest of the threads' (unique) 64-bit maxima is the bound, and
// only K threads can hold keys at or above it.
//
// Measured (the three kernels one after another): 4 beams of one prompt, 32000 bf16 logits, 32 layers' pages
// 13 us, three launches' latency; 32 x 8 beams 84 us, of which the page copies, 354 MB, take 63 (5.6 TB/s) and the pass
// over the logits 16; 8 x 16 beams of 131072 fp32 logits 65 us: the pass 29 us for 53 MB (20 with fp32 exponentials; bound by
// instructions, the 64-bit pipe's 11 a logit alone 10 us), the merge 11, the copies 25.
//
// Reordering.  See pim_beam_reorder in pim_b200.h: the table entries of full pages follow
// the parent, the partly filled pages of an entry's beams are dealt out again, and the
// copies read pages of beams with children and write pages of beams without.

#include <float.h>
#include <math.h>

#include "paged.cuh"

namespace pim {

constexpr int kBeamThreads = 256;
constexpr int kBeamChunk = kBeamThreads * 16;  // tokens of the smallest chunk (a thread holds 16 or 32 logits)
constexpr int kMaxBeams = 64;
constexpr int kMaxSplits = 128;

struct BeamStats {
  float max;   // -inf where there is no finite logit
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
  int chunk;  // tokens of a split: a multiple of 8
  int* err;
  BeamStats* stats;           // [batch * beams][splits]
  unsigned long long* lists;  // [batch * beams][splits][k]
};

// The bits of a logit in unsigned order; 0 for a logit that is no candidate.
__device__ __forceinline__ uint32_t logit_order(float x) {
  if (!isfinite(x)) return 0;
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 and +0 are equal
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float order_logit(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
// A candidate's key: larger is better.
__device__ __forceinline__ unsigned long long beam_key(uint32_t order, int token) {
  return ((unsigned long long)order << 32) | (uint32_t)~token;
}
__device__ __forceinline__ int key_token(unsigned long long key) { return (int)~(uint32_t)key; }

// sum + e^d for d <= 0 in 64 bits, by a table of 2^(j / 32) (P. T. P. Tang, "Table-driven implementation of the
// exponential function in IEEE floating-point arithmetic", ACM TOMS 15, 1989): d = (32 k + j) log(2) / 32 + r with
// |r| < 0.011, e^d = 2^k 2^(j / 32) e^r, and e^r by its series to r^6 / 6! (what is left is below 2^-57).  Below -700: 0.
// (8 x 16 beams of 131072 logits with the reordering: 66.5 us; 66.2 with 64 entries and 67.8 with 16, a term less and more.)
constexpr int kExpTable = 32;
__device__ __forceinline__ double add_exp(double sum, double d, const double* table) {
  constexpr double kRound = 6755399441055744.0;  // 1.5 x 2^52: a sum with it has a whole number in its low word
  const double z = fma(d, kExpTable * 1.4426950408889634074, kRound);
  const int n = __double2loint(z);
  const double r = fma(z - kRound, -0.69314718055994530942 / kExpTable, d);
  double e = fma(r, fma(r, fma(r, 1.0 / 720, 1.0 / 120), 1.0 / 24), 1.0 / 6);
  e = fma(r, fma(r, fma(r, e, 0.5), 1.0), 1.0);
  const double t = table[n & (kExpTable - 1)];
  const double scaled = __hiloint2double(__double2hiint(t) + (n >> 5) * (1 << 20), __double2loint(t));
  // (a negative number's upper word grows with its magnitude, up to -infinity's; -700's is 0xc085e000)
  return (uint32_t)__double2hiint(d) > 0xc085e000u ? sum : fma(scaled, e, sum);
}

// The larger of two; NaN if one is.
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// The largest of the lanes' 64-bit keys: two 32-bit warp reductions.
__device__ __forceinline__ unsigned long long warp_best(unsigned long long key) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(key >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(key >> 32) == hi ? (uint32_t)key : 0u);
  return ((unsigned long long)hi << 32) | lo;
}

constexpr int kBeamWarps = kBeamThreads / 32;
// Candidates that are ranked by counting; of more (warps that a mask leaves nothing set no bound, equal logits pass it
// together, sorted ones crowd in one warp) the exact bound is found first.  256 rows of 32000 bf16 logits: random ones
// 20.5 us, ascending 42, of which 1500 are kept 28.5.  (With the sums still in fp32, at 256 or 512 and at 2048: ascending 37
// and 492, 1500 kept 22.5 and 233, random 15.3.)
constexpr int kCountMost = 512;
template <typename T, bool ALIGNED, int kBeamVals>
__global__ void __launch_bounds__(kBeamThreads) beam_partial_kernel(BeamSelectArgs a) {
  constexpr int V = VecW<T>::n, kBeamCand = kMaxBeams * kBeamVals;
  __shared__ unsigned long long sm_cand[kBeamCand];
  __shared__ uint32_t sm_top[kBeamWarps], sm_low[kBeamWarps];
  __shared__ double sm_s[kBeamWarps], sm_exp[kExpTable];
  __shared__ unsigned long long sm_tau;
  __shared__ int sm_n;
  const int split = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  pdl_trigger();
  if (tid < kExpTable) sm_exp[tid] = exp2((double)tid / kExpTable);
  pdl_wait();
  if (a.done && a.done[row]) return;  // offers one candidate, which the merge adds
  const T* row_x = static_cast<const T*>(a.logits) + row * a.stride;
  const int base = split * a.chunk, size = min(a.chunk, a.vocab - base);
  float x[kBeamVals];  // -inf: no candidate
  // value i of this thread is token base + tok(i)
  auto tok = [&](int i) { return ALIGNED ? (i / V) * kBeamThreads * V + tid * V + i % V : i * kBeamThreads + tid; };
  if (ALIGNED) {
    constexpr int kNone = V == 8 ? (int)0xff80ff80u : (int)0xff800000u;  // -inf: two bf16, or a float
    int4 raw[kBeamVals / V];
#pragma unroll
    for (int i = 0; i < kBeamVals / V; ++i)
      raw[i] = ld_once_if(reinterpret_cast<const int4*>(row_x + base + tok(i * V)), tok(i * V) < size, kNone);
#pragma unroll
    for (int i = 0; i < kBeamVals / V; ++i) {
      float f[V];
      unpack(raw[i], f, T());
#pragma unroll
      for (int e = 0; e < V; ++e) x[i * V + e] = f[e];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kBeamVals; ++i) x[i] = tok(i) < size ? to_f(row_x[base + tok(i)]) : -INFINITY;
  }
  float mine_x = -INFINITY;
#pragma unroll
  for (int i = 0; i < kBeamVals; ++i) mine_x = max_or_nan(mine_x, x[i]);
  if (!(mine_x < INFINITY)) {  // there is a NaN or +inf: reported, and left out
    raise_flag(a.err);
    mine_x = -INFINITY;
#pragma unroll
    for (int i = 0; i < kBeamVals; ++i) {
      x[i] = fabsf(x[i]) < INFINITY ? x[i] : -INFINITY;
      mine_x = fmaxf(mine_x, x[i]);
    }
  }
  const uint32_t mine = logit_order(mine_x);
  const int rounds = (a.k + kBeamWarps - 1) / kBeamWarps;
  uint32_t cur = mine, low = 0;
  for (int r = 0; r < rounds; ++r) {
    low = __reduce_max_sync(0xffffffffu, cur);
    if (r == 0 && lane == 0) sm_top[warp] = low;
    const unsigned who = __ballot_sync(0xffffffffu, cur == low);
    if (lane == __ffs(who) - 1) cur = 0;
  }
  if (lane == 0) sm_low[warp] = low;
  if (tid == 0) sm_n = 0, sm_tau = 1;
  __syncthreads();
  uint32_t top = sm_top[0], tau = sm_low[0];
#pragma unroll
  for (int w = 1; w < kBeamWarps; ++w) top = max(top, sm_top[w]), tau = min(tau, sm_low[w]);
  tau = max(tau, 1u);  // (0: not a candidate)
  if (mine >= tau) {
    const float least = order_logit(tau == 1 ? logit_order(-FLT_MAX) : tau);
#pragma unroll
    for (int i = 0; i < kBeamVals; ++i)
      if (x[i] >= least) {
        const int at = atomicAdd(&sm_n, 1);
        if (at < kBeamCand) sm_cand[at] = beam_key(logit_order(x[i]), base + tok(i));
      }
  }
  // The sum in 64 bits: neighbouring candidates of different beams decide which tokens come out, and an error of the
  // exponential in 32 bits does not average out over a row of equal logits.
  const double m = top ? (double)order_logit(top) : 0.0;
  double s = 0;
#pragma unroll
  for (int i = 0; i < kBeamVals; ++i) s = add_exp(s, (double)x[i] - m, sm_exp);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  if (lane == 0) sm_s[warp] = s;
  __syncthreads();
  int n = sm_n;
  if (n > kCountMost) {  // too many at or above the bound: the exact one
    unsigned long long best = 0;
#pragma unroll
    for (int i = 0; i < kBeamVals; ++i) {
      const unsigned long long k = x[i] != -INFINITY ? beam_key(logit_order(x[i]), base + tok(i)) : 0;
      best = k > best ? k : best;
    }
    __syncthreads();
    sm_cand[tid] = best;
    __syncthreads();
    int above = 0;
    for (int i = 0; i < kBeamThreads; ++i) above += sm_cand[i] > best;
    if (best && above == a.k - 1) sm_tau = best;
    if (tid == 0) sm_n = 0;
    __syncthreads();
    const unsigned long long bound = sm_tau;
    if (best >= bound) {
#pragma unroll
      for (int i = 0; i < kBeamVals; ++i) {
        const unsigned long long k = x[i] != -INFINITY ? beam_key(logit_order(x[i]), base + tok(i)) : 0;
        if (k >= bound) sm_cand[atomicAdd(&sm_n, 1)] = k;  // at most k threads come here, with kBeamVals keys each
      }
    }
    __syncthreads();
    n = sm_n;
  }
  unsigned long long* list = a.lists + ((int64_t)row * a.splits + split) * a.k;
  for (int i = tid; i < n; i += kBeamThreads) {
    const unsigned long long k = sm_cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += sm_cand[j] > k;
    if (rank < a.k) list[rank] = k;
  }
  if (tid == 0) {
    BeamStats st;
    st.max = top ? (float)m : -INFINITY;
    st.count = min(n, a.k);
    st.sum = 0;
    for (int w = 0; w < kBeamWarps; ++w) st.sum += sm_s[w];
    a.stats[(int64_t)row * a.splits + split] = st;
  }
}

constexpr int kMergeThreads = 1024;  // (512, with fp32 sums: 4 x 16 beams and their reordering 25.2 us, 4 x 64 78; with 1024 21.4 and 63, fewer the same)
constexpr int kDeep = 4;  // keys of a list at hand

// Order-preserving bits of a finite double, never 0.
__device__ __forceinline__ unsigned long long score_order(double s) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(s + 0.0);
  return u >> 63 ? ~u : u | (1ull << 63);
}

// Q: lists of a lane (splits <= 32 Q).
template <int Q>
__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(BeamSelectArgs a) {
  __shared__ unsigned long long sm_keys[kMaxBeams * kMaxBeams];  // [beams][k], sorted, 0: none
  __shared__ double sm_shift[kMaxBeams];                         // score_w - log(sum of exp(x - max))
  __shared__ float sm_max[kMaxBeams];                            // largest logit; 0 for a beam that has ended
  __shared__ int sm_done[kMaxBeams];
  const int b = blockIdx.x, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  pdl_trigger();
  pdl_wait();
  for (int w = warp; w < a.beams; w += kMergeThreads / 32) {  // a warp per beam
    const int row = b * a.beams + w;
    const int done = a.done ? a.done[row] : 0;
    const float score = a.scores[row];
    if (lane == 0 && !(score < INFINITY)) raise_flag(a.err);
    unsigned long long* keys = sm_keys + w * a.k;
    // lane i merges lists i, i + 32, ..: the first kDeep keys of each are at hand
    unsigned long long key[Q][kDeep];
    int taken[Q], count[Q];
    float lm[Q];
    double ls[Q];
    const unsigned long long* lists = a.lists + (int64_t)row * a.splits * a.k;
    float m = -INFINITY;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int l = lane + 32 * q;
      taken[q] = count[q] = 0;
      lm[q] = -INFINITY;
      ls[q] = 0;
      if (l < a.splits) {
        const BeamStats st = a.stats[(int64_t)row * a.splits + l];
        lm[q] = st.max;
        ls[q] = st.sum;
        count[q] = done ? 0 : st.count;
      }
#pragma unroll
      for (int d = 0; d < kDeep; ++d) {
        const unsigned long long* p = lists + (int64_t)l * a.k + d;
        const bool there = l < a.splits && d < a.k;  // (a key behind the list's count is not written: dropped below)
        key[q][d] = ld4_if(p, there) | (unsigned long long)ld4_if(reinterpret_cast<const uint32_t*>(p) + 1, there) << 32;
      }
#pragma unroll
      for (int d = 0; d < kDeep; ++d) key[q][d] = d < count[q] ? key[q][d] : 0;
      m = fmaxf(m, lm[q]);
    }
    // (an ended beam's lists were not written, and are not looked at: its loads only ran beside its flag's)
    if (done || !isfinite(score)) {
      for (int j = lane; j < a.k; j += 32) keys[j] = j == 0 && isfinite(score) ? beam_key(0x80000000u, a.pad) : 0;
      if (lane == 0) sm_shift[w] = score, sm_max[w] = 0.f, sm_done[w] = done;
      continue;
    }
    m = warp_max(m);
    double s = 0;
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (lm[q] != -INFINITY) s += ls[q] * exp((double)lm[q] - (double)m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) {
      sm_shift[w] = m == -INFINITY ? 0.0 : (double)score - log(s);
      sm_max[w] = m;
      sm_done[w] = 0;
    }
    for (int j = 0; j < a.k; ++j) {
      unsigned long long mine = key[0][0];
#pragma unroll
      for (int q = 1; q < Q; ++q) mine = key[q][0] > mine ? key[q][0] : mine;
      const unsigned long long best = warp_best(mine);
      if (lane == 0) keys[j] = best;
      if (best == 0) continue;  // (the warp agrees)
#pragma unroll
      for (int q = 0; q < Q; ++q)
        if (key[q][0] == best) {  // keys are unique: one list of one lane
#pragma unroll
          for (int d = 0; d + 1 < kDeep; ++d) key[q][d] = key[q][d + 1];
          const int next = ++taken[q] + kDeep - 1;
          key[q][kDeep - 1] = next < count[q] ? lists[(int64_t)(lane + 32 * q) * a.k + next] : 0;
        }
    }
  }
  __syncthreads();
  if (warp != 0) return;
  // lane w merges the lists of beams w and w + 32; of equal scores the lower beam is first
  int at[2] = {0, 0};
  unsigned long long score[2];
  auto look = [&](int i) {
    const int w = lane + 32 * i;
    const unsigned long long k = w < a.beams && at[i] < a.k ? sm_keys[w * a.k + at[i]] : 0;
    // (the maximum is taken off first: at logits of 1e38 the sum's logarithm would be lost beside it)
    score[i] = k ? score_order(sm_shift[w] + ((double)order_logit((uint32_t)(k >> 32)) - (double)sm_max[w])) : 0;
  };
  look(0);
  look(1);
  for (int j = 0; j < a.k; ++j) {
    const unsigned long long best = warp_best(score[0] > score[1] ? score[0] : score[1]);
    const unsigned low = __ballot_sync(0xffffffffu, score[0] == best), high = __ballot_sync(0xffffffffu, score[1] == best);
    const int i = low ? 0 : 1, from = __ffs(low ? low : high) - 1;
    const int64_t o = (int64_t)b * a.k + j;
    if (best == 0) {
      if (lane == 0) {
        a.scores_out[o] = -INFINITY;
        a.parents[o] = 0;
        a.tokens[o] = a.pad;
        if (a.done_out) a.done_out[o] = 1;
      }
    } else if (lane == from) {
      const int w = lane + 32 * i, token = key_token(sm_keys[w * a.k + at[i]]);
      const unsigned long long u = best >> 63 ? best & ~(1ull << 63) : ~best;
      a.scores_out[o] = (float)__longlong_as_double((long long)u);
      a.parents[o] = w;
      a.tokens[o] = token;
      if (a.done_out) a.done_out[o] = sm_done[w] || (a.eos >= 0 && token == a.eos);
      ++at[i];
      look(i);
    }
    __syncwarp();
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

constexpr int kReorderThreads = 64;
static_assert(kReorderThreads >= kMaxBeams, "a thread per beam");
constexpr int kCopyPieces = 8 * kReorderThreads;

__global__ void __launch_bounds__(kReorderThreads) beam_reorder_kernel(BeamReorderArgs a) {
  // A beam's parent and partly filled page; the pages that further children are copied from and to.
  __shared__ int sm_parent[kMaxBeams], sm_page[kMaxBeams], sm_from[kMaxBeams], sm_to[kMaxBeams];
  __shared__ unsigned sm_further[kReorderThreads / 32], sm_childless[kReorderThreads / 32];
  const int row = blockIdx.x, b = row / a.beams, j = row - b * a.beams, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  pdl_trigger();
  pdl_wait();
  // (the length and the parents come together; only the partly filled pages wait for them)
  const int n = a.lengths[b], ps = 1 << a.ps_log2;
  const int p = tid < a.beams ? a.parents[b * a.beams + tid] : 0;
  const int full = n >> a.ps_log2, fill = n & (ps - 1);
  const bool n_ok = n >= 0 && n <= (int64_t)a.max_pages << a.ps_log2;
  // 16-byte pieces of the slots in use, kCopyPieces of them per step of a CTA
  const int per_head = fill * a.row_bytes / 16, head_pieces = a.row_bytes << a.ps_log2 >> 4;
  const int pieces = a.hkv * per_head, steps = (pieces + kCopyPieces - 1) / kCopyPieces;
  const int64_t per_copy = (int64_t)a.num_blocks * steps, cta = (int64_t)blockIdx.y * a.beams + j;
  if (blockIdx.y > 0 && (!n_ok || cta >= (a.beams - 1) * per_copy)) return;  // (made for full pages)
  int page = 0;
  if (tid < a.beams) {
    if (n_ok && fill) page = a.table[(int64_t)(b * a.beams + tid) * a.table_stride + full];
    sm_parent[tid] = p;
  }
  bool bad = __syncthreads_or(!n_ok || p < 0 || p >= a.beams);
  bool further = false, childless = tid < a.beams;
  if (tid < a.beams)
    for (int i = 0; i < a.beams; ++i) {
      further |= i < tid && sm_parent[i] == p;
      childless &= sm_parent[i] != tid;
    }
  const unsigned who = __ballot_sync(0xffffffffu, further), free = __ballot_sync(0xffffffffu, childless);
  if (lane == 0) sm_further[warp] = who, sm_childless[warp] = free;
  if (tid < a.beams) sm_page[tid] = page;
  bad |= (bool)__syncthreads_or(page < 0 || page >= a.num_pages);
  if (bad && tid == 0 && blockIdx.y == 0) raise_flag(a.err);
  // the i-th further child takes the page of the i-th beam without a child (there are equally many)
  auto before = [&](const unsigned* mask, int i) {
    int count = __popc(mask[i / 32] & ((1u << i % 32) - 1));
    for (int w = 0; w < i / 32; ++w) count += __popc(mask[w]);
    return count;
  };
  if (!bad && further) sm_from[before(sm_further, tid)] = sm_page[p];
  if (!bad && childless) sm_to[before(sm_childless, tid)] = page;
  __syncthreads();
  if (blockIdx.y == 0) {
    const int parent = bad ? j : sm_parent[j];
    const int* mine = a.table + row * a.table_stride;
    const int* theirs = a.table + (int64_t)(b * a.beams + parent) * a.table_stride;
    const bool copied = sm_further[j / 32] >> j % 32 & 1;
    for (int i = tid; i < a.max_pages; i += blockDim.x) {
      int at = bad || i > full || (i == full && !fill) ? mine[i] : theirs[i];
      if (!bad && fill && i == full && copied) at = sm_to[before(sm_further, j)];
      a.table_out[row * a.table_stride + i] = at;
    }
  }
  if (bad || !fill) return;
  int copies = 0;
#pragma unroll
  for (int w = 0; w < kReorderThreads / 32; ++w) copies += __popc(sm_further[w]);
  // All CTAs of the batch entry share its copies, eight pieces a thread in flight; neighbours work on different copies
  // (on one after the other 32 x 8 beams take 97 us with the selection instead of 83).
  for (int64_t item = cta; item < copies * per_copy; item += (int64_t)gridDim.y * a.beams) {
    const int rest = (int)(item / copies), c = (int)(item - (int64_t)rest * copies);
    const int blk = rest / steps, i0 = (rest - blk * steps) * kCopyPieces + tid;
    char* block = a.pages + blk * a.block_bytes;
    const int4* src = reinterpret_cast<const int4*>(block + sm_from[c] * a.page_bytes);
    int4* dst = reinterpret_cast<int4*>(block + sm_to[c] * a.page_bytes);
    int4 v[kCopyPieces / kReorderThreads];
    int64_t off[kCopyPieces / kReorderThreads];
#pragma unroll
    for (int u = 0; u < kCopyPieces / kReorderThreads; ++u) {
      const int i = i0 + u * kReorderThreads, h = i / per_head;
      off[u] = (int64_t)h * head_pieces + (i - h * per_head);
      v[u] = ld_once_if(src + off[u], i < pieces);
    }
#pragma unroll
    for (int u = 0; u < kCopyPieces / kReorderThreads; ++u)
      if (i0 + u * kReorderThreads < pieces) dst[off[u]] = v[u];
  }
}

static const char* beam_select_error(const pim_beam_select_args* a, int dtype) {
  if (!a) return "null arguments";
  if (!dtype_ok(dtype)) return "bad dtype";
  if (!a->logits || !a->scores || !a->scores_out || !a->parents || !a->tokens) return "null pointer";
  if (a->batch <= 0 || a->beams <= 0 || a->beams > kMaxBeams || a->beams_out <= 0 || a->beams_out > kMaxBeams)
    return "batch must be positive, beams and beams_out 1 to 64";
  if (a->vocab <= 0 || a->vocab > kMaxSplits * kBeamChunk || (int64_t)a->batch * a->beams > 65535)
    return "vocab must be 1 to 2^19, batch * beams at most 65535";
  if (a->logits_stride < a->vocab) return "logits_stride is less than vocab";
  if ((uintptr_t)a->logits % elem_bytes(dtype)) return "logits are not aligned to their type";
  if (a->eos < -1 || a->eos >= a->vocab || a->pad < 0 || a->pad >= a->vocab) return "eos or pad outside the vocabulary";
  if (a->scores_out == a->scores || (a->done && a->done_out == a->done))
    return "scores_out and done_out must be arrays of their own";
  return nullptr;
}

// Logits of a thread: 32 where that leaves two chunks for every SM, which halves the lists and the work beside the
// logits (8 x 16 beams of 131072 fp32 logits with the reordering: 65.7 us against 71.4; 32 x 8 of 32000 bf16: 85.2 against
// 89.2); else 16, for more CTAs.
static int beam_vals(const pim_beam_select_args* a) {
  return (int64_t)a->batch * a->beams * ceil_div(a->vocab, 2 * kBeamChunk) >= 2 * 148 ? 32 : 16;
}
static int beam_splits(const pim_beam_select_args* a) { return ceil_div(a->vocab, kBeamThreads * beam_vals(a)); }
// The splits' chunks are as good as equal: in a short last one most warps would have nothing, which leaves no bound, and
// every logit of it would be a candidate (256 rows of 26080 bf16 logits: see the figures at the head of the file).
static int beam_chunk(const pim_beam_select_args* a) { return (ceil_div(a->vocab, beam_splits(a)) + 7) / 8 * 8; }

static int64_t beam_stats_bytes(const pim_beam_select_args* a) {
  return (int64_t)a->batch * a->beams * beam_splits(a) * (int64_t)sizeof(BeamStats);
}

template <typename T, int VALS>
static cudaError_t beam_select(const BeamSelectArgs& a, cudaStream_t st) {
  // 16-byte loads where rows allow them; a vocabulary that leaves most warps of such a chunk empty is read by
  // element, which spreads it over all of them
  const bool aligned = aligned16(a.logits) && a.stride * sizeof(T) % 16 == 0 && a.vocab % VecW<T>::n == 0 &&
                       a.vocab >= kBeamThreads * VecW<T>::n;
  const dim3 grid(a.splits, a.batch * a.beams);
  const cudaError_t e = aligned ? launch_pdl(beam_partial_kernel<T, true, VALS>, grid, dim3(kBeamThreads), 0, st, a)
                                : launch_pdl(beam_partial_kernel<T, false, VALS>, grid, dim3(kBeamThreads), 0, st, a);
  if (e != cudaSuccess) return e;
  return a.splits <= 32 ? launch_pdl(beam_merge_kernel<1>, dim3(a.batch), dim3(kMergeThreads), 0, st, a)
                        : launch_pdl(beam_merge_kernel<kMaxSplits / 32>, dim3(a.batch), dim3(kMergeThreads), 0, st, a);
}

}  // namespace pim

extern "C" int64_t pim_beam_select_workspace_bytes(const pim_beam_select_args* a, int32_t dtype) {
  using namespace pim;
  if (beam_select_error(a, dtype)) return -1;
  return beam_stats_bytes(a) + (int64_t)a->batch * a->beams * beam_splits(a) * a->beams_out * 8;
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
  d.splits = beam_splits(a);
  d.chunk = beam_chunk(a);
  d.err = a->err_flag;
  d.stats = static_cast<BeamStats*>(workspace);
  d.lists = reinterpret_cast<unsigned long long*>(static_cast<char*>(workspace) + beam_stats_bytes(a));
  cudaStream_t st = (cudaStream_t)stream;
  const bool wide = beam_vals(a) == 32;
  return report_cuda(dtype == PIM_BF16 ? wide ? beam_select<__nv_bfloat16, 32>(d, st) : beam_select<__nv_bfloat16, 16>(d, st)
                     : wide            ? beam_select<float, 32>(d, st)
                                       : beam_select<float, 16>(d, st),
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
  if (page * es / 16 > (1 << 30)) return bad("a page of more than 16 GiB");
  // The copies follow from the parents and the lengths.  A CTA per step of those that half-filled pages and a third of the
  // beams give, at least as many as run at once and at most a few rounds of them: a thousand CTAs cost 1.1 us to launch,
  // with nothing to do too, and a step per CTA balances best (device us with a selection whose sums were fp32, at 24, 48 and
  // 96 CTAs an SM: 32 x 8 beams with 354 MB to copy 92, 87, 83; 16 x 12 beams with eight slots in use 17.5, 21.1, 26.4; at a
  // sixth of the full pages' steps 84 and 17.5).
  const int64_t steps = (int64_t)a->num_blocks * ceil_div(page * es / 16, kCopyPieces);
  if (steps > INT32_MAX) return bad("more than 2^31 steps of 8 KiB to copy a page of every block");
  const int rows = a->batch * a->beams;
  int64_t by = (steps + 5) / 6;
  const int64_t least = ceil_div(24 * 148, rows), most = ceil_div(96 * 148, rows);
  by = by < least ? least : by > most ? most : by;
  by = by < steps ? by : steps;
  return report_cuda(launch_pdl(beam_reorder_kernel, dim3(rows, (unsigned)by), dim3(kReorderThreads), 0,
                                (cudaStream_t)stream, d),
                     "pim_beam_reorder");
}
