// RMS norm of query and key heads with the rotation by position, one pass.
//
// For a head vector x of D values (g the gain, 1 without one):
//   n = x / sqrt(mean(x^2) + eps) * g
// and with A position axes, F = (D/2) div A pairs per axis, pair i of axis a
// (pair a*F + i) turns by t = p[a] * base^(-i/F):
//   (u, w) -> (u cos t - w sin t, u sin t + w cos t);
// pairs from A*F on stay.  Pair j is (j, j + D/2), or (2j, 2j + 1) interleaved.
//
// The queries go to a tensor of their own, the keys too, or with the values
// (copied as they are) to the pages that hold what a sample keeps.
#include "pages.hpp"
#include "sequence.hpp"

#include <algorithm>
#include <cmath>

namespace tsc {
namespace {

struct RotateArgs {
  const void* q;
  int64_t q_row, q_head;
  const void* k;
  int64_t k_row, k_head;
  const void* pos;
  int64_t pos_row;
  int pos_float, axes;
  const void* q_gain;
  const void* k_gain;
  int gain_dtype;
  int q_gain_head, k_gain_head;  // 0, or D for a gain per head
  float eps;
  double log2_base;
  int interleaved;
  int64_t n;
  int q_heads, k_heads, dim;
  void* q_out;
  void* k_out;
  // the paged form: values and where keys and values go
  const void* v;
  int64_t v_row, v_head;
  void* k_pages;
  PageStrides k_at;
  void* v_pages;
  PageStrides v_at;
  PageTable pages;
  const int32_t* offsets;
};

// The page and its row that an input row goes to: it is one of the last rows of
// the sample whose offsets enclose it.  A page of -1: nowhere (a row of no
// sample, a position or a page that there is not).
struct Place {
  int32_t page, row;
};
// For a row r of [first, last] a lane, by the whole wave.
__device__ __forceinline__ Place place_of(const RotateArgs& a, int64_t first, int64_t last, int64_t r) {
  if (a.pages.samples == 0) return Place{-1, 0};
  const int64_t t[1] = {r};
  int at[1], end[1], length[1];
  const int begin = a.offsets[0];
  samples_of<1>(a.offsets, a.pages.lengths, a.pages.samples, first, last, t, at, end, length);
  // (an end past the last row is cut to it)
  const int64_t pos = (int64_t)length[0] - (min((int64_t)end[0], a.n) - r);
  if (r < begin || r >= end[0] || pos < 0 || pos >= a.pages.most()) return Place{-1, 0};
  const uint32_t p = a.pages.page_of(static_cast<uint32_t>(pos));
  const int32_t page = a.pages.table[at[0] * a.pages.table_row + p];
  if (page < 0 || page >= a.pages.pages) return Place{-1, 0};
  return Place{page, static_cast<int32_t>(pos - (int64_t)p * a.pages.page_rows)};
}

// Cosine and sine of position p times a pair's speed, base^(-i/F) / 2 pi turns.
// The angle is taken in 64 bits: positions reach thousands, and an f32 angle
// of a thousand radians is already 6e-5 off.  What is left after the whole
// turns fits f32.
__device__ __forceinline__ float2 turn_of(double p, double speed) {
  const double t = p * speed;
  float2 cs;
  sincospif(static_cast<float>(2.0 * (t - rint(t))), &cs.y, &cs.x);
  return cs;
}
__device__ __forceinline__ double speed_of(int i, int F, double log2_base) {
  return exp2(-log2_base * i / F) * 0.15915494309189535;
}

// N gains as f32.
template <int N>
__device__ __forceinline__ void load_gain(const void* p, int dtype, int64_t at, float g[N]) {
  auto as = [&](auto tag) {
    using G = decltype(tag);
    G e[N];
    __builtin_memcpy(e, static_cast<const G*>(p) + at, sizeof e);
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = to_f32(e[i]);
  };
  if (dtype == TSC_F32) as(float{});
  else if (dtype == TSC_F16) as(__half{});
  else as(__hip_bfloat16{});
}

// One row by one wave: lane l of a head (its pairs l and l + lp), group `sub` of
// `heads` heads at a time.
template <typename T, bool PAGED>
__device__ __forceinline__ void rotate_any_row(const RotateArgs& a, int64_t r, int lp, int half, int F, int sub,
                                               int l, int heads) {
  float2 cs[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int j = l + u * lp;
    cs[u] = make_float2(1.f, 0.f);
    if (j < half && F > 0 && j < a.axes * F) {
      const int64_t at = r * a.pos_row + j / F;
      const double p = a.pos_float ? static_cast<const float*>(a.pos)[at]
                                   : static_cast<const int32_t*>(a.pos)[at];
      cs[u] = turn_of(p, speed_of(j % F, F, a.log2_base));
    }
  }
  Place to{0, 0};
  if constexpr (PAGED) to = place_of(a, r, r, r);
  const int total = a.q_heads + a.k_heads;
  for (int h0 = 0; h0 < total; h0 += heads) {
    const int h = h0 + sub;
    const bool is_q = h < a.q_heads, in = h < total && (is_q || to.page >= 0);
    const int hh = is_q ? h : h - a.q_heads;
    const T* src = static_cast<const T*>(is_q ? a.q : a.k) +
                   (is_q ? r * a.q_row + hh * a.q_head : r * a.k_row + hh * a.k_head);
    T* dst;
    if (PAGED && !is_q) dst = static_cast<T*>(a.k_pages) + a.k_at.at(to.page, to.row, hh);
    else dst = static_cast<T*>(is_q ? a.q_out : a.k_out) + (r * (is_q ? a.q_heads : a.k_heads) + hh) * a.dim;
    const void* gain = is_q ? a.q_gain : a.k_gain;
    const int64_t gain_at = (int64_t)hh * (is_q ? a.q_gain_head : a.k_gain_head);
    float x[2][2] = {}, sum = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int j = l + u * lp;
      if (in && j < half) {
        x[u][0] = to_f32(src[a.interleaved ? 2 * j : j]);
        x[u][1] = to_f32(src[a.interleaved ? 2 * j + 1 : j + half]);
      }
      sum += x[u][0] * x[u][0] + x[u][1] * x[u][1];
    }
    for (int d = 1; d < lp; d <<= 1) sum += __shfl_xor(sum, d, kWave);
    const float inv = 1.f / sqrtf(sum / a.dim + a.eps);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int j = l + u * lp;
      if (!in || j >= half) continue;
      const int ia = a.interleaved ? 2 * j : j, ib = a.interleaved ? 2 * j + 1 : j + half;
      float p = x[u][0] * inv, q = x[u][1] * inv;
      if (gain) {
        p *= load_any(gain, a.gain_dtype, gain_at + ia);
        q *= load_any(gain, a.gain_dtype, gain_at + ib);
      }
      dst[ia] = from_f32<T>(p * cs[u].x - q * cs[u].y);
      dst[ib] = from_f32<T>(p * cs[u].y + q * cs[u].x);
    }
  }
  if constexpr (PAGED) {
    if (to.page < 0) return;
    for (int h = sub; h < a.k_heads; h += heads) {
      const T* src = static_cast<const T*>(a.v) + r * a.v_row + h * a.v_head;
      T* dst = static_cast<T*>(a.v_pages) + a.v_at.at(to.page, to.row, h);
      for (int d = l; d < a.dim; d += lp) dst[d] = src[d];
    }
  }
}

// A wave per row and turn; a head takes LP lanes (a power of two from D/2 up, at most
// 64), a lane its pairs l, l + 64.  Any size, stride and alignment.
template <typename T, bool PAGED>
__global__ void __launch_bounds__(256) rotate_any_kernel(RotateArgs a, int lp) {
  const int lane = threadIdx.x % kWave;
  const int half = a.dim / 2, F = half / a.axes;
  const int sub = lane / lp, l = lane % lp, heads = kWave / lp;
  for (int64_t r = blockIdx.x * (int64_t)4 + threadIdx.x / kWave; r < a.n; r += (int64_t)gridDim.x * 4)
    rotate_any_row<T, PAGED>(a, r, lp, half, F, sub, l, heads);
}

// The vector form: a workgroup takes kRows rows; its threads first share out the
// rows' angles (cosine and sine of every turning pair, to LDS: they are the
// same for every head of q and k), then the heads.  A head takes LANES lanes (a
// power of two; the last may idle), each two pieces of P elements: [l P,
// l P + P) of its first and of its second half, which are pairs with each other
// (or one after the other where pairs are neighbours), so that a pair never
// leaves its lane.  Bound by memory: each vector is read and written once.
// 500k rows of 12 + 12 heads of 64, bf16: 607 us, 5.07 TB/s (a large copy on
// this card: 4.86).  The paged form takes keys and values head by head, so that
// what it writes of a page lies together (4 x 60k rows of 12 + 12 + 12 heads of
// 64, f16: 470 us, 4.6 TB/s; row by row a quarter more, and
// another 25 us where each row searched for its sample by itself).
constexpr int kRows = 8, kMaxHalf = 128;

template <typename T, int P, int LANES, bool PAGED>
__global__ void __launch_bounds__(256) rotate_vector_kernel(RotateArgs a) {
  constexpr int HEADS = 256 / LANES, BYTES = P * sizeof(T);
  __shared__ Place place[PAGED ? kRows : 1];
  __shared__ __align__(16) float2 turn[kRows][kMaxHalf];
  __shared__ double speed[kMaxHalf];
  const int half = a.dim / 2, F = half / a.axes;
  if (threadIdx.x < half)
    speed[threadIdx.x] = F > 0 && (int)threadIdx.x < a.axes * F
                             ? speed_of(threadIdx.x % F, F, a.log2_base) : 0.0;
  __syncthreads();
  const int turning = a.q_heads + a.k_heads, total = turning + (PAGED ? a.k_heads : 0), l = threadIdx.x % LANES;
  const bool in = LANES == 1 || l * P < half;
  const float over = 1.f / a.dim;
  // the lane's elements of a head: [first, first + P) and [second, second + P)
  const int first = in ? (a.interleaved ? 2 * P * l : P * l) : 0, second = first + (a.interleaved ? P : half);
  for (int64_t r0 = blockIdx.x * (int64_t)kRows; r0 < a.n; r0 += (int64_t)gridDim.x * kRows) {
    const int rows = static_cast<int>(min((int64_t)kRows, a.n - r0));
    if constexpr (PAGED) {
      if (threadIdx.x >= 256 - kWave) {  // the last wave, which has the fewest angles
        const int r = min((int)threadIdx.x - (256 - kWave), rows - 1);
        place[r] = place_of(a, r0, r0 + rows - 1, r0 + r);
      }
    }
    for (int x = threadIdx.x; x < rows * half; x += 256) {
      const int r = x / half, j = x - r * half;
      float2 cs = make_float2(1.f, 0.f);
      if (j < a.axes * F) {
        const int64_t at = (r0 + r) * a.pos_row + j / F;
        const double p = a.pos_float ? static_cast<const float*>(a.pos)[at]
                                     : static_cast<const int32_t*>(a.pos)[at];
        cs = turn_of(p, speed[j]);
      }
      turn[r][j] = cs;
    }
    __syncthreads();
    for (int v = threadIdx.x / LANES; v < rows * total; v += HEADS) {
      int r, h;
      if (PAGED && v >= rows * a.q_heads) {
        // head by head: its rows lie one behind the other in their page
        const int u = v - rows * a.q_heads, n = rows == kRows ? u / kRows : u / rows;
        h = a.q_heads + n, r = u - n * rows;
      } else {
        const int n = PAGED ? a.q_heads : total;
        r = v / n, h = v - r * n;
      }
      const bool is_q = h < a.q_heads;
      const int hh = is_q ? h : h - a.q_heads;
      const int64_t row = r0 + r;
      if (PAGED && !is_q && place[r].page < 0) continue;
      T e[2 * P];
      if (PAGED && h >= turning) {
        const int hv = h - turning;
        const T* src = static_cast<const T*>(a.v) + row * a.v_row + hv * a.v_head;
        T* dst = static_cast<T*>(a.v_pages) + a.v_at.at(place[r].page, place[r].row, hv);
        if (in) {
          __builtin_memcpy(e, src + first, BYTES);
          __builtin_memcpy(e + P, src + second, BYTES);
          __builtin_memcpy(dst + first, e, BYTES);
          __builtin_memcpy(dst + second, e + P, BYTES);
        }
        continue;
      }
      const T* src = static_cast<const T*>(is_q ? a.q : a.k) +
                     (is_q ? row * a.q_row + hh * a.q_head : row * a.k_row + hh * a.k_head);
      T* dst;
      if (PAGED && !is_q) dst = static_cast<T*>(a.k_pages) + a.k_at.at(place[r].page, place[r].row, hh);
      else dst = static_cast<T*>(is_q ? a.q_out : a.k_out) + (row * (is_q ? a.q_heads : a.k_heads) + hh) * a.dim;
      float x[2 * P] = {}, sum = 0.f;
      if (in) {
        __builtin_memcpy(e, src + first, BYTES);
        __builtin_memcpy(e + P, src + second, BYTES);
#pragma unroll
        for (int i = 0; i < 2 * P; ++i) {
          x[i] = to_f32(e[i]);
          sum = __builtin_fmaf(x[i], x[i], sum);
        }
      }
#pragma unroll
      for (int d = 1; d < LANES; d <<= 1) sum += __shfl_xor(sum, d, kWave);
      if (!in) continue;
      const float inv = 1.f / sqrtf(sum * over + a.eps);
      const void* gain = is_q ? a.q_gain : a.k_gain;
      if (gain) {
        const int64_t at = (int64_t)hh * (is_q ? a.q_gain_head : a.k_gain_head);
        float g[2 * P];
        load_gain<P>(gain, a.gain_dtype, at + first, g);
        load_gain<P>(gain, a.gain_dtype, at + second, g + P);
#pragma unroll
        for (int i = 0; i < 2 * P; ++i) x[i] *= inv * g[i];
      } else {
#pragma unroll
        for (int i = 0; i < 2 * P; ++i) x[i] *= inv;
      }
      float y[2 * P];
      const float2* cs = &turn[r][P * l];
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          y[2 * i] = x[2 * i] * cs[i].x - x[2 * i + 1] * cs[i].y;
          y[2 * i + 1] = x[2 * i] * cs[i].y + x[2 * i + 1] * cs[i].x;
        }
      } else {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          y[i] = x[i] * cs[i].x - x[P + i] * cs[i].y;
          y[P + i] = x[i] * cs[i].y + x[P + i] * cs[i].x;
        }
      }
      round_to<T, 2 * P>(y, e);
      __builtin_memcpy(dst + first, e, BYTES);
      __builtin_memcpy(dst + second, e + P, BYTES);
    }
    __syncthreads();
  }
}

template <typename T, bool PAGED, int P, int LANES>
int launch_vector(const RotateArgs& a, const char* what, hipStream_t s) {
  const int64_t blocks = std::min<int64_t>(ceil_div(a.n, kRows), 16384);
  rotate_vector_kernel<T, P, LANES, PAGED><<<static_cast<unsigned>(blocks), 256, 0, s>>>(a);
  TSC_LAUNCH_CHECK(what);
  return 0;
}

template <typename T, bool PAGED, int P>
int launch_lanes(const RotateArgs& a, const char* what, hipStream_t s) {
  const int lanes = a.dim / 2 / P;
  if (lanes <= 1) return launch_vector<T, PAGED, P, 1>(a, what, s);
  if (lanes <= 2) return launch_vector<T, PAGED, P, 2>(a, what, s);
  if (lanes <= 4) return launch_vector<T, PAGED, P, 4>(a, what, s);
  if (lanes <= 8) return launch_vector<T, PAGED, P, 8>(a, what, s);
  if (lanes <= 16) return launch_vector<T, PAGED, P, 16>(a, what, s);
  return launch_vector<T, PAGED, P, 32>(a, what, s);
}

template <typename T, bool PAGED>
int launch_rotate(const RotateArgs& a, const char* what, hipStream_t s) {
  // half a head in whole pieces of 16 bytes, or 8 for 16-bit values; head
  // sizes that are neither (2, 6, 250) go value by value
  const int half = a.dim / 2;
  if (half % kPer16<T> == 0) return launch_lanes<T, PAGED, kPer16<T>>(a, what, s);
  if constexpr (kIs16<T>)
    if (half % 4 == 0) return launch_lanes<T, PAGED, 4>(a, what, s);
  int lp = 1;
  while (lp < kWave && lp < a.dim / 2) lp *= 2;
  // (a launch holds fewer than 2^32 threads, 2^26 waves)
  const int64_t blocks = std::min<int64_t>(ceil_div(a.n, 4), 1 << 20);
  rotate_any_kernel<T, PAGED><<<static_cast<unsigned>(blocks), 256, 0, s>>>(a, lp);
  TSC_LAUNCH_CHECK(what);
  return 0;
}

template <bool PAGED>
int launch(const RotateArgs& a, int dtype, const char* what, hipStream_t s) {
  switch (dtype) {
    case TSC_F32: return launch_rotate<float, PAGED>(a, what, s);
    case TSC_F16: return launch_rotate<__half, PAGED>(a, what, s);
    default: return launch_rotate<__hip_bfloat16, PAGED>(a, what, s);
  }
}

// What both forms ask of their arguments; 0 or an error code.
int check(const char* what, int dtype, int gain_dtype, int64_t n, int q_heads, int k_heads, int dim, int axes,
          double base, float eps) {
  TSC_REQUIRE(dtype_ok(dtype) && dtype_ok(gain_dtype), "%s: unknown dtype", what);
  TSC_REQUIRE(n >= 0 && n < (1ll << 31) && q_heads >= 0 && k_heads >= 0 && q_heads <= 65536 &&
                  k_heads <= 65536, "%s: invalid sizes", what);
  TSC_REQUIRE(dim >= 2 && dim <= 256 && dim % 2 == 0,
              "%s: head size %d is not an even number up to 256", what, dim);
  TSC_REQUIRE(axes >= 1 && axes <= 4, "%s: %d position axes, 1 to 4 are supported", what, axes);
  TSC_REQUIRE(base > 1.0 && eps >= 0.f, "%s: base must be over 1 and eps not negative", what);
  return 0;
}

}  // namespace
}  // namespace tsc

using namespace tsc;

extern "C" int tsc_norm_rotate_heads(const void* q, int64_t q_row, int64_t q_head, const void* k,
                                     int64_t k_row, int64_t k_head, const void* positions,
                                     int64_t pos_row, int32_t pos_float, int32_t axes,
                                     const void* q_gain, const void* k_gain, int32_t gain_dtype,
                                     int32_t q_gain_per_head, int32_t k_gain_per_head, float eps,
                                     double base, int32_t interleaved, int32_t dtype, int64_t n,
                                     int32_t q_heads, int32_t k_heads, int32_t dim, void* q_out,
                                     void* k_out, tsc_stream_t stream) {
  const char* what = "norm_rotate_heads";
  if (int rc = check(what, dtype, gain_dtype, n, q_heads, k_heads, dim, axes, base, eps)) return rc;
  if (n == 0 || q_heads + k_heads == 0) return 0;
  TSC_REQUIRE(positions && (!q_heads || (q && q_out)) && (!k_heads || (k && k_out)),
              "norm_rotate_heads: null pointer");
  const RotateArgs a{q, q_row, q_head, k, k_row, k_head, positions, pos_row, pos_float, axes,
                     q_gain, k_gain, gain_dtype, q_gain_per_head ? dim : 0, k_gain_per_head ? dim : 0,
                     eps, log2(base), interleaved, n, q_heads, k_heads, dim, q_out, k_out};
  return launch<false>(a, dtype, what, static_cast<hipStream_t>(stream));
}

extern "C" int tsc_norm_rotate_append(
    const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v,
    int64_t v_row, int64_t v_head, const void* positions, int64_t pos_row, int32_t pos_float, int32_t axes,
    const void* q_gain, const void* k_gain, int32_t gain_dtype, int32_t q_gain_per_head, int32_t k_gain_per_head,
    float eps, double base, int32_t interleaved, int32_t dtype, int64_t n, int32_t q_heads, int32_t k_heads,
    int32_t dim, void* k_pages, int64_t k_page, int64_t k_page_row, int64_t k_page_head, void* v_pages,
    int64_t v_page, int64_t v_page_row, int64_t v_page_head, int64_t pages, int64_t page_rows,
    const int32_t* table, int64_t table_row, int64_t table_pages, const int32_t* offsets, const int32_t* lengths,
    int32_t samples, void* q_out, tsc_stream_t stream) {
  const char* what = "norm_rotate_append";
  if (int rc = check(what, dtype, gain_dtype, n, q_heads, k_heads, dim, axes, base, eps)) return rc;
  PageTable t;
  if (int rc = t.set(what, table, table_row, table_pages, lengths, samples, pages, page_rows)) return rc;
  if (n == 0 || q_heads + k_heads == 0) return 0;
  TSC_REQUIRE(positions && offsets && (!q_heads || (q && q_out)), "%s: null pointer", what);
  TSC_REQUIRE(!k_heads || (k && v && (pages == 0 || (k_pages && v_pages))), "%s: null pointer", what);
  const RotateArgs a{q, q_row, q_head, k, k_row, k_head, positions, pos_row, pos_float, axes,
                     q_gain, k_gain, gain_dtype, q_gain_per_head ? dim : 0, k_gain_per_head ? dim : 0,
                     eps, log2(base), interleaved, n, q_heads, k_heads, dim, q_out, nullptr, v, v_row, v_head,
                     k_pages, {k_page, k_page_row, k_page_head}, v_pages, {v_page, v_page_row, v_page_head},
                     t, offsets};
  return launch<true>(a, dtype, what, static_cast<hipStream_t>(stream));
}
