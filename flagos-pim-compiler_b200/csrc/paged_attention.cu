// pim_paged_attention: attention of one new token per row over a paged KV cache.
//
//   s_j = scale q . k_j,  p_j = exp(s_j - m) / sum_i exp(s_i - m),  o = sum_j p_j v_j,  j < lengths[row]
//
// First form, right for every shape: a CTA per (row, kv head), its warps walk the keys of
// one query head after another with an online softmax; the keys' probabilities are found
// again in a second walk when the weights are asked for.

#include <math.h>

#include "paged.cuh"

namespace pim {

struct PagedAttnArgs {
  PagedKV kv;
  const void* q;
  void* out;
  int64_t q_stride, out_stride;
  const int* lengths;
  int group;  // query heads per kv head
  float scale;
  float* weights;
  int64_t w_row_stride, w_head_stride;
  int* err;
};

constexpr int kPagedWarps = 8;

template <typename T, int HD>
__global__ void __launch_bounds__(kPagedWarps * 32) paged_attn_simple_kernel(PagedAttnArgs a) {
  constexpr int DPL = HD / 32;  // dims of a lane
  const int h = blockIdx.x, row = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  __shared__ float sm_m[kPagedWarps], sm_l[kPagedWarps], sm_acc[kPagedWarps][HD];
  pdl_trigger();
  pdl_wait();
  const int want = a.lengths[row];
  const int len = min(max(want, 0), a.kv.slots());
  if (len != want && threadIdx.x == 0) raise_flag(a.err);
  const T* kp = static_cast<const T*>(a.kv.k);
  const T* vp = static_cast<const T*>(a.kv.v);
  for (int g = 0; g < a.group; ++g) {
    const int head = h * a.group + g;
    const T* qr = static_cast<const T*>(a.q) + row * a.q_stride + (int64_t)head * HD;
    float q[DPL], acc[DPL], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < DPL; ++e) q[e] = to_f(qr[lane + 32 * e]), acc[e] = 0.f;
    auto score = [&](int64_t at) {
      float d = 0.f;
#pragma unroll
      for (int e = 0; e < DPL; ++e) d = fmaf(q[e], to_f(kp[at + lane + 32 * e]), d);
      return warp_sum(d) * a.scale;
    };
    for (int j = warp; j < len; j += kPagedWarps) {
      const int64_t at = a.kv.at<HD>(row, j, h);
      if (at < 0) {
        if (lane == 0) raise_flag(a.err);
        continue;
      }
      const float s = score(at);
      const float mn = fmaxf(m, s);
      const float safe = mn == -INFINITY ? 0.f : mn;
      const float alpha = expf(m - safe), p = expf(s - safe);
#pragma unroll
      for (int e = 0; e < DPL; ++e) acc[e] = fmaf(p, to_f(vp[at + lane + 32 * e]), acc[e] * alpha);
      l = l * alpha + p;
      m = mn;
    }
    __syncthreads();
    if (lane == 0) sm_m[warp] = m, sm_l[warp] = l;
#pragma unroll
    for (int e = 0; e < DPL; ++e) sm_acc[warp][lane + 32 * e] = acc[e];
    __syncthreads();
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < kPagedWarps; ++w) M = fmaxf(M, sm_m[w]);
    const float safe = M == -INFINITY ? 0.f : M;
    for (int w = 0; w < kPagedWarps; ++w) L += sm_l[w] * expf(sm_m[w] - safe);
    for (int d = threadIdx.x; d < HD; d += blockDim.x) {
      float A = 0.f;
      for (int w = 0; w < kPagedWarps; ++w) A += sm_acc[w][d] * expf(sm_m[w] - safe);
      static_cast<T*>(a.out)[row * a.out_stride + (int64_t)head * HD + d] = from_f<T>(L > 0.f ? A / L : 0.f);
    }
    if (a.weights)
      for (int j = warp; j < len; j += kPagedWarps) {
        const int64_t at = a.kv.at<HD>(row, j, h);
        if (at < 0) continue;
        const float s = score(at);
        if (lane == 0) a.weights[row * a.w_row_stride + h * a.w_head_stride + j] += L > 0.f ? expf(s - safe) / L : 0.f;
      }
  }
}

static cudaError_t paged_attention(const PagedAttnArgs& a, int hd, int dtype, cudaStream_t st) {
  return dispatch_type_dim(dtype, hd, [&](auto t, auto d) {
    return launch_pdl(paged_attn_simple_kernel<decltype(t), decltype(d)::value>, dim3(a.kv.hkv, a.kv.rows),
                      dim3(kPagedWarps * 32), 0, st, a);
  });
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

}  // namespace pim

extern "C" int64_t pim_paged_attention_workspace_bytes(const pim_paged_attention_args* a, int32_t dtype) {
  if (pim::paged_attention_error(a, dtype)) return -1;
  return 0;
}

extern "C" int pim_paged_attention(const pim_paged_attention_args* a, int32_t dtype, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  using namespace pim;
  if (const char* e = paged_attention_error(a, dtype)) {
    char msg[200];
    snprintf(msg, sizeof(msg), "pim_paged_attention: %s", e);
    return report_status(PIM_EINVAL, msg);
  }
  const int64_t need = pim_paged_attention_workspace_bytes(a, dtype);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return report_status(PIM_EINVAL, "pim_paged_attention: workspace too small or not 16-byte aligned");
  PagedAttnArgs d{};
  d.kv = to_dev(a->kv);
  d.q = a->q;
  d.out = a->out;
  d.q_stride = a->q_stride;
  d.out_stride = a->out_stride;
  d.lengths = a->lengths;
  d.group = a->q_heads / a->kv.kv_heads;
  d.scale = a->scale > 0.f ? a->scale : (float)(1.0 / sqrt((double)a->kv.head_dim));
  d.weights = a->weights;
  d.w_row_stride = a->weights_row_stride;
  d.w_head_stride = a->weights_head_stride;
  d.err = a->err_flag;
  return report_cuda(paged_attention(d, a->kv.head_dim, dtype, (cudaStream_t)stream), "pim_paged_attention");
}
