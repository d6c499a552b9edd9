// What the kernels of the paged KV cache share: where a token lies, and the host-side checks of the geometry.
#pragma once
#include "common.cuh"

namespace we {

struct PagedView {
  const int32_t* table;
  int64_t table_stride;
  int64_t plane_s, page_s, head_s, token_s;   // strides of kv in elements
  int32_t S, Hkv, page, page_shift, n_pages, max_pages;
  int32_t* status;
};

__device__ __forceinline__ void paged_report(const PagedView& v) {
  if (v.status != nullptr) atomicExch(v.status, WE_B200_ST_PAGE_RANGE);
}

// A count of tokens as the kernels use it: within [0, max_pages * page].
__device__ __forceinline__ int paged_count(const PagedView& v, int n) {
  const int cap = v.max_pages << v.page_shift;
  if (n < 0 || n > cap) {
    paged_report(v);
    return n < 0 ? 0 : cap;
  }
  return n;
}

// The page of block `b` of session `s`; -1 (reported) where the table names none of the pool.
__device__ __forceinline__ int paged_page(const PagedView& v, int s, int b) {
  const int pg = v.table[s * v.table_stride + b];
  if (pg < 0 || pg >= v.n_pages) {
    paged_report(v);
    return -1;
  }
  return pg;
}

inline int check_paged_geom(const we_b200_paged_geom& g) {
  if (g.dtype != WE_B200_BF16 && g.dtype != WE_B200_F16) return WE_B200_E_DTYPE;
  if (g.Dh != 64 && g.Dh != 128) return WE_B200_E_DTYPE;
  if (g.S < 1 || g.Hkv < 1 || g.n_pages < 1 || g.max_pages < 1) return WE_B200_E_SHAPE;
  if (g.page != 16 && g.page != 32 && g.page != 64 && g.page != 128 && g.page != 256) return WE_B200_E_SHAPE;
  if (g.plane_stride < 0 || g.page_stride < 0 || g.head_stride < 0 || g.token_stride < g.Dh || g.table_stride < 0)
    return WE_B200_E_SHAPE;
  if ((g.plane_stride | g.page_stride | g.head_stride | g.token_stride) & 7) return WE_B200_E_ALIGN;
  // token indexes and (session, head) units are 32-bit in the kernels
  if (static_cast<int64_t>(g.max_pages) * g.page > (1 << 30)) return WE_B200_E_LIMIT;
  if (static_cast<int64_t>(g.S) * g.Hkv > (1 << 20) || g.S > 65535 || g.Hkv > 65535) return WE_B200_E_LIMIT;
  return WE_B200_OK;
}

inline PagedView paged_view(const we_b200_paged_geom& g, const int32_t* table, int32_t* status) {
  PagedView v;
  v.table = table;
  v.table_stride = g.table_stride;
  v.plane_s = g.plane_stride;
  v.page_s = g.page_stride;
  v.head_s = g.head_stride;
  v.token_s = g.token_stride;
  v.S = g.S;
  v.Hkv = g.Hkv;
  v.page = g.page;
  v.page_shift = g.page == 16 ? 4 : g.page == 32 ? 5 : g.page == 64 ? 6 : g.page == 128 ? 7 : 8;
  v.n_pages = g.n_pages;
  v.max_pages = g.max_pages;
  v.status = status;
  return v;
}

}  // namespace we
