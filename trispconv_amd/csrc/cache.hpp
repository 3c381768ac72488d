// Attention of new rows over what their samples keep in pages.
//
// Sample b's lengths[b] = Lk positions lie in the pages of its row of the table;
// its Lq queries are the last of them.  What a query sees, and what comes out,
// is as for packed keys (attend.hpp), with the keys and values fetched page by
// page.  With a prefix of P pages every sample's first P R positions are those
// pages, and their keys are read for all queries at once.
#pragma once

#include "attend.hpp"
#include "pages.hpp"

namespace tsc {

struct CacheArgs : AttendArgs {
  PageTable pages;
  PageStrides k_at, v_at;
  const int32_t* prefix;  // its pages, or none
  int prefix_pages;
};

template <typename T>
int launch_cache(const CacheArgs& a, hipStream_t s);

namespace {

// The keys or values of one head in the pages of one row of the table.  Page
// numbers that there are not are cut to those there are.
template <typename T>
struct PagedRows {
  const T* base;  // of the head
  int64_t page, stride;
  const int32_t* ids;
  const PageTable* pages;
  __device__ __forceinline__ const T* row(int j) const {
    const uint32_t at = pages->page_of(j);
    const int id = min(max(ids[at], 0), pages->pages - 1);
    return base + id * page + (j - (int)at * pages->page_rows) * stride;
  }
};

// Positions of sample b.
__device__ __forceinline__ int kept(const CacheArgs& a, int b) {
  return static_cast<int>(min(max((int64_t)a.pages.lengths[b], (int64_t)0), a.pages.most()));
}

// The sample of query row t (the last whose offset is not behind it), -1 for none.
__device__ __forceinline__ int sample_of(const CacheArgs& a, int64_t t) {
  int lo = 0, hi = a.samples + 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.off_q[mid] <= t) lo = mid + 1;
    else hi = mid;
  }
  return lo - 1 < a.samples ? lo - 1 : -1;
}

// A wave per query and head.
template <typename T>
__global__ void __launch_bounds__(256) cache_row_kernel(CacheArgs a) {
  __shared__ float q_s[4][256];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  for (int64_t item = blockIdx.x * (int64_t)4 + wave; item < a.rows(); item += gridDim.x * (int64_t)4) {
    const int64_t t = item / a.q_heads;
    const int h = static_cast<int>(item % a.q_heads), hk = h / (a.q_heads / a.k_heads);
    const int b = sample_of(a, t);
    T* out = static_cast<T*>(a.out) + item * a.dim;
    float m = 0.f, l = 0.f, o[4] = {};
    if (b >= 0) {
      const int lk = kept(a, b), first = a.prefix_pages * a.pages.page_rows;
      const int p = static_cast<int>(max(t - a.off_q[b + 1] + lk, -(int64_t)1 << 30));
      int lo, hi, sink;
      seen_keys(p, lk, a.left, a.right, a.sinks, lo, hi, sink);
      const T* q = static_cast<const T*>(a.q) + t * a.q_row + h * a.q_head;
      PagedRows<T> k{static_cast<const T*>(a.k) + hk * a.k_at.head, a.k_at.page, a.k_at.row, nullptr, &a.pages};
      PagedRows<T> v{static_cast<const T*>(a.v) + hk * a.v_at.head, a.v_at.page, a.v_at.row, nullptr, &a.pages};
      if (first) {
        k.ids = v.ids = a.prefix;
        attend_row(a, q, k, v, min(lo, first), min(hi, first), sink, 0, 0, 0, first, q_s[wave], m, l, o);
      }
      k.ids = v.ids = a.pages.table + b * a.pages.table_row;
      float m2, l2, o2[4];
      attend_row(a, q, k, v, max(lo, first), hi, sink, 0, 0, first, lk, q_s[wave], m2, l2, o2);
      const float top = l == 0.f ? m2 : l2 == 0.f ? m : fmaxf(m, m2);
      const float f = l == 0.f ? 0.f : exp2f(m - top), f2 = l2 == 0.f ? 0.f : exp2f(m2 - top);
      l = f * l + f2 * l2;
#pragma unroll
      for (int u = 0; u < 4; ++u) o[u] = f * o[u] + f2 * o2[u];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int d = lane + u * kWave;
      if (d < a.dim) out[d] = from_f32<T>(l == 0.f ? 0.f : o[u] / l);
    }
  }
}

}  // namespace

template <typename T>
int launch_cache(const CacheArgs& a, hipStream_t s) {
  const int64_t blocks = std::min<int64_t>(ceil_div(a.rows(), 4), 1 << 20);
  cache_row_kernel<T><<<static_cast<unsigned>(blocks), 256, 0, s>>>(a);
  TSC_LAUNCH_CHECK("cache_attention");
  return 0;
}

}  // namespace tsc
