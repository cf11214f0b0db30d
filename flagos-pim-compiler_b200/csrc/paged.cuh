// What the paged-cache kernels share: the pages and tables as a kernel sees them, and the
// checks of a pim_paged_kv (pim_b200.h).
#pragma once

#include <stdio.h>

#include <type_traits>

#include "pim_b200.h"
#include "pim_common.cuh"

namespace pim {

int report_status(int code, const char* msg);
int report_cuda(cudaError_t e, const char* what);

struct PagedKV {
  void* k;
  void* v;
  int64_t page_stride;
  const int* table;
  int64_t table_stride;
  int rows, max_pages, num_pages, ps_log2, hkv;

  __device__ __forceinline__ int slots() const { return max_pages << ps_log2; }
  // Element offset of (row's slot, head) in the K and in the V pages; -1 where the page id is out of range.
  // 64-bit: a pool passes 2^31 elements at a few hundred thousand slots.
  template <int HD>
  __device__ __forceinline__ int64_t at(int row, int slot, int head) const {
    const int page = table[row * table_stride + (slot >> ps_log2)];
    if ((unsigned)page >= (unsigned)num_pages) return -1;
    return page * page_stride + (((int64_t)head << ps_log2) + (slot & ((1 << ps_log2) - 1))) * HD;
  }
};

inline int ilog2(int v) {
  int n = 0;
  while ((1 << n) < v) ++n;
  return n;
}

inline bool page_geometry_ok(int page_size, int kv_heads, int head_dim) {
  const bool ps = page_size == 8 || page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128 ||
                  page_size == 256;
  return ps && kv_heads > 0 && kv_heads <= 65535 && (head_dim == 32 || head_dim == 64 || head_dim == 128);
}

inline bool dtype_ok(int dtype) { return dtype == PIM_F32 || dtype == PIM_BF16; }
inline int elem_bytes(int dtype) { return dtype == PIM_BF16 ? 2 : 4; }
inline bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

// nullptr, or what is wrong with the pages and tables.
inline const char* paged_kv_error(const pim_paged_kv& kv, int dtype) {
  if (!kv.k_pages || !kv.v_pages || !kv.table) return "null pages or table";
  if (!page_geometry_ok(kv.page_size, kv.kv_heads, kv.head_dim))
    return "page_size must be 8, 16, 32, 64, 128 or 256, head_dim 32, 64 or 128, kv_heads 1 to 65535";
  if (kv.rows <= 0 || kv.rows > (1 << 20) || kv.max_pages <= 0 || kv.num_pages <= 0) return "bad rows or page counts";
  if ((int64_t)kv.max_pages * kv.page_size > (1 << 30)) return "more than 2^30 slots a row";
  if (kv.table_stride < kv.max_pages) return "table_stride is less than max_pages";
  if (kv.page_stride < (int64_t)kv.kv_heads * kv.page_size * kv.head_dim) return "page_stride is less than a page";
  if (!aligned16(kv.k_pages) || !aligned16(kv.v_pages) || kv.page_stride * elem_bytes(dtype) % 16)
    return "pages must be 16-byte aligned";
  return nullptr;
}

inline PagedKV to_dev(const pim_paged_kv& kv) {
  PagedKV d;
  d.k = kv.k_pages;
  d.v = kv.v_pages;
  d.page_stride = kv.page_stride;
  d.table = kv.table;
  d.table_stride = kv.table_stride;
  d.rows = kv.rows;
  d.max_pages = kv.max_pages;
  d.num_pages = kv.num_pages;
  d.ps_log2 = ilog2(kv.page_size);
  d.hkv = kv.kv_heads;
  return d;
}

__device__ __forceinline__ void raise_flag(int* err) {
  if (err) atomicExch(err, 1);
}

// The kernel template for a dtype and head_dim: f(T(), std::integral_constant<int, HD>()).
template <typename F>
cudaError_t dispatch_type_dim(int dtype, int hd, F&& f) {
  if (dtype == PIM_BF16) {
    if (hd == 128) return f(__nv_bfloat16(), std::integral_constant<int, 128>());
    if (hd == 64) return f(__nv_bfloat16(), std::integral_constant<int, 64>());
    return f(__nv_bfloat16(), std::integral_constant<int, 32>());
  }
  if (hd == 128) return f(float(), std::integral_constant<int, 128>());
  if (hd == 64) return f(float(), std::integral_constant<int, 64>());
  return f(float(), std::integral_constant<int, 32>());
}

}  // namespace pim
