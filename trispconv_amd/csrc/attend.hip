// Entry points of the windowed attention: argument checks and how a call is
// cut into workgroups.
#include <algorithm>
#include <cmath>

#include "attend.hpp"

namespace tsc {
extern template int launch_attend<float>(const AttendArgs&, const Cut&, hipStream_t);
extern template int launch_attend<__half>(const AttendArgs&, const Cut&, hipStream_t);
extern template int launch_attend<__hip_bfloat16>(const AttendArgs&, const Cut&, hipStream_t);

namespace {

constexpr int kCus = 256;

Cut attend_cut(int64_t samples, int64_t n_q, int64_t n_k, int q_heads, int k_heads, int left, int right,
               int sinks, int rows_wide) {
  const int64_t group = q_heads / k_heads;
  auto tiles = [&](int64_t rows) { return n_q * group / rows + std::min(samples, n_q); };
  Cut c{1, tiles(rows_wide), 1};
  // Fewer workgroups than CUs: one wave each, 32 rows, and the keys that a
  // tile can see at most split so that there are about three per CU, but not
  // under 128 keys.
  if (c.tiles * k_heads < kCus) {
    c.wide = 0;
    c.tiles = tiles(32);
    int64_t span = n_k;
    if (left >= 0 && right >= 0) span = std::min<int64_t>(span, (int64_t)left + right + 32 + sinks);
    const int64_t most = std::max<int64_t>(1, span / 128);
    c.splits = static_cast<int>(std::min<int64_t>(most, std::max<int64_t>(1, 3 * kCus / (c.tiles * k_heads))));
  }
  return c;
}

// Scratch of a call: the splits' maxima, sums and values.
int64_t part_bytes(const Cut& c, int64_t rows, int dim) {
  return c.splits > 1 ? (align_up(c.splits * rows * 2, 4) + c.splits * rows * dim) * 4 : 0;
}

int rows_of_type(int dtype, int dim) {
  return dtype == TSC_F32 ? rows_of<float>(dim) : rows_of<__half>(dim);
}

}  // namespace
}  // namespace tsc

using namespace tsc;

extern "C" int64_t tsc_window_attention_workspace_bytes(int32_t samples, int64_t n_q, int64_t n_k,
                                                        int32_t q_heads, int32_t k_heads,
                                                        int32_t dim, int32_t left, int32_t right,
                                                        int32_t sinks, int32_t dtype) {
  if (!dtype_ok(dtype) || samples < 0 || n_q < 0 || n_k < 0 || q_heads <= 0 || k_heads <= 0 || dim < 1 ||
      dim > 256)
    return -1;
  const Cut c = attend_cut(samples, n_q, n_k, q_heads, k_heads, left, right, sinks, rows_of_type(dtype, dim));
  return part_bytes(c, n_q * q_heads, dim);
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
  TSC_REQUIRE(n_q * (q_heads / k_heads) < (1ll << 32) - 1024,
              "window_attention: over 2^32 rows of queries and the heads that share a key head");
  TSC_REQUIRE(dim >= 1 && dim <= 256, "window_attention: head size %d, 1 to 256 are supported", dim);
  TSC_REQUIRE(sinks >= 0, "window_attention: negative number of sinks");
  if (n_q == 0 || samples == 0) return 0;
  TSC_REQUIRE(q && out && offsets_q && offsets_k && (n_k == 0 || (k && v)),
              "window_attention: null pointer");
  TSC_REQUIRE(std::isfinite(scale), "window_attention: scale is not finite");
  const Cut c = attend_cut(samples, n_q, n_k, q_heads, k_heads, left, right, sinks, rows_of_type(dtype, dim));
  const int64_t need = part_bytes(c, n_q * q_heads, dim);
  TSC_REQUIRE(need == 0 || (ws && ws_bytes >= need), "window_attention: a workspace of %lld bytes is needed",
              static_cast<long long>(need));
  const AttendArgs a{q, q_row, q_head, k, k_row, k_head, v, v_row, v_head, offsets_q, offsets_k,
                     samples, n_q, n_k, q_heads, k_heads, dim, left < 0 ? kNoLimit : left,
                     right < 0 ? kNoLimit : right, sinks, scale == 0.f ? 1.f : fabsf(scale) * 1.44269504f,
                     scale > 0.f ? 1.f : scale < 0.f ? -1.f : 0.f, out, static_cast<float*>(ws)};
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TSC_F32: return launch_attend<float>(a, c, s);
    case TSC_F16: return launch_attend<__half>(a, c, s);
    default: return launch_attend<__hip_bfloat16>(a, c, s);
  }
}
