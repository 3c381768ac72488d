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

Cut attend_cut(int64_t samples, int64_t n_q, int64_t n_k, int q_heads, int k_heads, int dim, int elem,
               int left, int right, int sinks) {
  const int64_t group = q_heads / k_heads;
  auto tiles = [&](int64_t rows) { return n_q * group / rows + std::min(samples, n_q); };
  // keys that a tile can see at most
  int64_t span = n_k;
  if (left >= 0 && right >= 0) span = std::min<int64_t>(span, (int64_t)left + right + 32 + sinks);
  auto splits = [&](int64_t tiles, int64_t least) {  // about two workgroups per CU
    return static_cast<int>(std::max<int64_t>(1, std::min(span / least, 2 * kCus / (tiles * k_heads))));
  };
  // Samples of few rows (one new token each): workgroups of one wave and 32
  // rows, for four waves would share nothing.  When they leave CUs idle, the keys
  // are split, down to 128 (one token over 60k keys, 16 heads on 4: 28 us,
  // three workgroups per CU 35 us).
  if (n_q * group < 64 * samples) return Cut{0, tiles(32), splits(tiles(32), 128)};
  // 64 rows a wave for long walks: 8k voxels, 16 heads of 64, bf16, all seeing
  // one another: 303 us, with 32 rows 331 us; in a window of 1025 keys, four
  // scans of 60k: 435 us against 391 (the wider tile walks more that it masks)
  if (can_pair(padded_dim(dim), elem) && span >= 4096 && tiles(256) * k_heads >= 2 * kCus)
    return Cut{2, tiles(256), 1};
  // Fewer workgroups than CUs: the keys are split, down to 256 (2k voxels, 8
  // heads of 64, all seeing one another: 52 us, unsplit in lone waves 60 us)
  return Cut{1, tiles(128), tiles(128) * k_heads < kCus ? splits(tiles(128), 256) : 1};
}

// Scratch of a call: the splits' maxima, sums and values.
int64_t part_bytes(const Cut& c, int64_t rows, int dim) {
  return c.splits > 1 ? (align_up(c.splits * rows * 2, 4) + c.splits * rows * dim) * 4 : 0;
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
  if (n_q == 0 || samples == 0) return 0;
  const Cut c = attend_cut(samples, n_q, n_k, q_heads, k_heads, dim, dtype_bytes(dtype), left, right, sinks);
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
  // key numbers are 32-bit, and a walk looks up to a tile past the last
  TSC_REQUIRE(n_k < (1ll << 31) - 1024, "window_attention: over 2^31 - 1025 keys");
  TSC_REQUIRE(dim >= 1 && dim <= 256, "window_attention: head size %d, 1 to 256 are supported", dim);
  TSC_REQUIRE(sinks >= 0, "window_attention: negative number of sinks");
  if (n_q == 0 || samples == 0) return 0;
  TSC_REQUIRE(q && out && offsets_q && offsets_k && (n_k == 0 || (k && v)),
              "window_attention: null pointer");
  TSC_REQUIRE(std::isfinite(scale), "window_attention: scale is not finite");
  const Cut c = attend_cut(samples, n_q, n_k, q_heads, k_heads, dim, dtype_bytes(dtype), left, right, sinks);
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
