// Attention of packed sequences in a sliding window, with sinks.
//
// Sample b owns queries [oq[b], oq[b+1]) and keys [ok[b], ok[b+1]); its Lq
// queries are the last of its Lk positions: query i stands at p = i + Lk - Lq
// and sees key j when 0 <= j < Lk, j <= p + right, and j >= p - left or
// j < sinks.  Per head (G query heads share a key head)
//   o = sum_j e^(s_j) v_j / sum_j e^(s_j),  s_j = scale q.k_j  over the seen j,
// and 0 where there is none.  The seen keys are two ranges:
//   [lo, hi) with lo = max(0, p - left), hi = min(Lk, p + right + 1), and
//   [0, min(sinks, lo, hi)).
// One pass over the keys with the running maximum m and sum l of the
// exponentials (f32): a new maximum rescales what is there by e^(m_old - m).
#include "common.hpp"

namespace tsc {
namespace {

struct AttendArgs {
  const void* q;
  int64_t q_row, q_head;
  const void* k;
  int64_t k_row, k_head;
  const void* v;
  int64_t v_row, v_head;
  const int32_t* off_q;
  const int32_t* off_k;
  int samples;
  int64_t n_q, n_k;
  int q_heads, k_heads, dim;
  int left, right, sinks;  // left, right: kNoLimit where there is none
  float scale_log2;        // scale * log2(e)
  void* out;
};

constexpr int kNoLimit = 0x7fffffff;

// [offsets[b], offsets[b+1]) cut to [0, n]: no value of the offsets leads out
// of the tensors.
__device__ __forceinline__ void sample_range(const int32_t* off, int b, int64_t n, int64_t& at,
                                             int& len) {
  const int64_t lo = min(max((int64_t)off[b], (int64_t)0), n);
  const int64_t hi = min(max((int64_t)off[b + 1], lo), n);
  at = lo;
  len = static_cast<int>(hi - lo);
}

// The seen keys of position p among lk: [lo, hi) and [0, sink).
__device__ __forceinline__ void seen_keys(int p, int lk, int left, int right, int sinks, int& lo,
                                          int& hi, int& sink) {
  const int64_t h = (int64_t)p + right + 1, l = (int64_t)p - left;
  hi = static_cast<int>(max((int64_t)0, min(h, (int64_t)lk)));
  lo = static_cast<int>(min((int64_t)lk, max(l, (int64_t)0)));
  sink = min(sinks, min(lo, hi));
}

// A wave per query and head: a lane scores every 64th key, then the lanes
// share out the D values and add the 64 keys' values one by one.  Reads no
// key that the query does not see.  Any size, stride and alignment.
template <typename T>
__global__ void __launch_bounds__(256) attend_rows_kernel(AttendArgs a) {
  __shared__ float q_s[4][256];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t item = blockIdx.x * (int64_t)4 + wave;
  if (item >= a.n_q * a.q_heads) return;
  const int64_t row = item / a.q_heads;
  const int h = static_cast<int>(item - row * a.q_heads), hk = h / (a.q_heads / a.k_heads);
  int64_t q0 = 0, k0 = 0;
  int lq = 0, lk = 0, b = 0;
  for (; b < a.samples; ++b) {
    sample_range(a.off_q, b, a.n_q, q0, lq);
    if (row >= q0 && row < q0 + lq) break;
  }
  if (b == a.samples) return;
  sample_range(a.off_k, b, a.n_k, k0, lk);
  const T* q = static_cast<const T*>(a.q) + row * a.q_row + h * a.q_head;
  const T* k = static_cast<const T*>(a.k) + k0 * a.k_row + hk * a.k_head;
  const T* v = static_cast<const T*>(a.v) + k0 * a.v_row + hk * a.v_head;
  for (int d = lane; d < a.dim; d += kWave) q_s[wave][d] = to_f32(q[d]);
  __builtin_amdgcn_wave_barrier();
  int lo, hi, sink;
  seen_keys(static_cast<int>(row - q0) + lk - lq, lk, a.left, a.right, a.sinks, lo, hi, sink);
  float m = -__builtin_inff(), l = 0.f, o[4] = {};
  for (int part = 0; part < 2; ++part) {
    const int from = part ? lo : 0, to = part ? hi : sink;
    for (int j0 = from; j0 < to; j0 += kWave) {
      const int j = j0 + lane;
      float s = -__builtin_inff();
      if (j < to) {
        float dot = 0.f;
        for (int d = 0; d < a.dim; ++d) dot += q_s[wave][d] * to_f32(k[j * a.k_row + d]);
        s = dot * a.scale_log2;
      }
      float top = s;
#pragma unroll
      for (int x = 1; x < kWave; x <<= 1) top = fmaxf(top, __shfl_xor(top, x, kWave));
      const float m_new = fmaxf(m, top);
      const float base = m_new == -__builtin_inff() ? 0.f : m_new;
      const float fix = exp2f(m - base), p = j < to ? exp2f(s - base) : 0.f;
      l *= fix;
      m = m_new;
#pragma unroll
      for (int u = 0; u < 4; ++u) o[u] *= fix;
      const int cnt = min(kWave, to - j0);
      for (int x = 0; x < cnt; ++x) {
        const float px = __shfl(p, x, kWave);
        l += px;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int d = lane + u * kWave;
          if (d < a.dim) o[u] += px * to_f32(v[(j0 + x) * a.v_row + d]);
        }
      }
    }
  }
  T* out = static_cast<T*>(a.out) + item * a.dim;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int d = lane + u * kWave;
    if (d < a.dim) out[d] = from_f32<T>(l == 0.f ? 0.f : o[u] / l);
  }
}

template <typename T>
int launch_attend(const AttendArgs& a, hipStream_t s) {
  const int64_t items = a.n_q * a.q_heads;
  attend_rows_kernel<T><<<static_cast<unsigned>(ceil_div(items, 4)), 256, 0, s>>>(a);
  TSC_LAUNCH_CHECK("window_attention");
  return 0;
}

}  // namespace
}  // namespace tsc

using namespace tsc;

extern "C" int64_t tsc_window_attention_workspace_bytes(int32_t samples, int64_t n_q, int64_t n_k,
                                                        int32_t q_heads, int32_t k_heads,
                                                        int32_t dim, int32_t left, int32_t right,
                                                        int32_t sinks, int32_t dtype) {
  return 0;
}

extern "C" int tsc_window_attention(const void* q, int64_t q_row, int64_t q_head, const void* k,
                                    int64_t k_row, int64_t k_head, const void* v, int64_t v_row,
                                    int64_t v_head, const int32_t* offsets_q,
                                    const int32_t* offsets_k, int32_t samples, int64_t n_q,
                                    int64_t n_k, int32_t q_heads, int32_t k_heads, int32_t dim,
                                    int32_t left, int32_t right, int32_t sinks, float scale,
                                    int32_t dtype, void* ws, int64_t ws_bytes, void* out,
                                    tsc_stream_t stream) {
  TSC_REQUIRE(dtype_ok(dtype), "window_attention: unknown dtype");
  TSC_REQUIRE(samples >= 0 && n_q >= 0 && n_k >= 0 && n_q < (1ll << 31) && n_k < (1ll << 31),
              "window_attention: invalid sizes");
  TSC_REQUIRE(q_heads > 0 && k_heads > 0 && q_heads % k_heads == 0 && q_heads <= 65535,
              "window_attention: %d query heads do not share %d key heads evenly", q_heads, k_heads);
  TSC_REQUIRE(dim >= 1 && dim <= 256, "window_attention: head size %d, 1 to 256 are supported", dim);
  TSC_REQUIRE(sinks >= 0, "window_attention: negative number of sinks");
  if (n_q == 0 || samples == 0) return 0;
  TSC_REQUIRE(q && out && offsets_q && offsets_k && (n_k == 0 || (k && v)),
              "window_attention: null pointer");
  const AttendArgs a{q, q_row, q_head, k, k_row, k_head, v, v_row, v_head, offsets_q, offsets_k,
                     samples, n_q, n_k, q_heads, k_heads, dim, left < 0 ? kNoLimit : left,
                     right < 0 ? kNoLimit : right, sinks, scale * 1.44269504f, out};
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TSC_F32: return launch_attend<float>(a, s);
    case TSC_F16: return launch_attend<__half>(a, s);
    default: return launch_attend<__hip_bfloat16>(a, s);
  }
}
