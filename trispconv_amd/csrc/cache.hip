// Entry points of the attention over pages: argument checks and how a call is
// cut into workgroups.
#include <algorithm>
#include <cmath>

#include "cache.hpp"

namespace tsc {
extern template int launch_cache<float>(const CacheArgs&, const CachePlan&, hipStream_t);
extern template int launch_cache<__half>(const CacheArgs&, const CachePlan&, hipStream_t);
extern template int launch_cache<__hip_bfloat16>(const CacheArgs&, const CachePlan&, hipStream_t);

namespace {

constexpr int kCus = 256;

// longest: positions a sample may have, prefix_rows of them shared.
CachePlan cache_plan(int64_t samples, int64_t n_q, int64_t longest, int64_t prefix_rows, int q_heads, int k_heads,
                     int dim, int elem, int left, int right, int sinks) {
  CachePlan p;
  const int64_t group = q_heads / k_heads, all = n_q * group, mean = all / samples;
  const int row_bytes = padded_dim(dim) * elem, kt = cache_keys(row_bytes);
  p.row_blocks = mean <= 16 ? 1 : mean <= 32 ? 2 : 4;
  while (p.row_blocks > cache_row_blocks(row_bytes)) p.row_blocks /= 2;
  // lists: of the rows that `tiles` are cut from; mean: rows of such a list
  auto cut = [&](int64_t keys, int64_t lists, int64_t mean) {
    CacheCut c;
    auto tiles = [&](int64_t rows) { return lists == 1 ? ceil_div(all, rows) : all / rows + std::min(lists, n_q); };
    if (sinks > 0) keys += kt;  // (a tile of their own)
    // workgroups that do something, and those that the CUs hold at once
    auto units = [&](int64_t rows) { return std::max<int64_t>(1, lists * ceil_div(mean, rows)) * k_heads; };
    if (mean <= 64) {
      const int64_t rows = 16 * p.row_blocks;
      c.tiles = tiles(rows);
      // Parts of 256 to 2048 keys (4096 where a workgroup has a CU to itself), one
      // round of workgroups where that allows it: 64 samples of up to 32k keys in
      // parts of 2048 276 us, of 512 321, of 8192 295; 24 windows of 4096 in one
      // round of 1024 27 us, in two of 768 30.  Up to 1024 keys by themselves are
      // not worth a join (14 us, in parts 17).
      const int per_cu = cache_per_cu(row_bytes);
      const int64_t want = std::max<int64_t>(1, per_cu * kCus / units(rows));
      int64_t chunk = std::min<int64_t>(std::max<int64_t>(ceil_div(keys, want), 256), 4096 / per_cu);
      if (!prefix_rows && keys <= 1024) chunk = keys;
      chunk = std::max(chunk, ceil_div(keys, kMostSplits / 2));
      c.chunk = static_cast<int>(align_up(std::max<int64_t>(chunk, 1), kt * cache_waves(row_bytes)));
      c.splits = static_cast<int>(std::max<int64_t>(1, ceil_div(keys, c.chunk)));
      return c;
    }
    // as attend_cut
    c.wave_rows = can_pair(padded_dim(dim), elem) && keys >= 4096 && units(256) >= 2 * kCus ? 2 : 1;
    const int64_t work = units(128 * c.wave_rows);
    c.tiles = tiles(128 * c.wave_rows);
    // One round of workgroups, of 512 keys and more (20k keys in 136 tiles, four
    // workgroups a CU: 141 us in seven parts, 166 in six, 239 in three); beside
    // the samples' own keys one a CU (a prefix of 32k keys in 8 tiles: 42 us in 32
    // parts, 45 in 64, 61 in 128)
    const bool beside = lists == 1 && prefix_rows && all / samples <= 64 && row_bytes <= 128;
    const int64_t per_cu = beside ? 1 : row_bytes <= 128 ? 4 / c.wave_rows : row_bytes <= 256 ? 2 : 1;
    const int64_t slots = per_cu * kCus;
    c.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({keys / 512, slots / work, kMostSplits / 2})));
    return c;
  };
  // keys that a tile of a sample's rows can see at most
  int64_t span = std::max<int64_t>(longest - prefix_rows, 0);
  if (left >= 0) span = std::min<int64_t>(span, (int64_t)left + n_q + sinks + kt);
  p.own = cut(span, samples, mean);
  if (prefix_rows) p.prefix = cut(prefix_rows, 1, all);
  p.own.first_split = p.prefix.splits;
  return p;
}

// Scratch of a call: the parts' references, sums and values.
int64_t part_bytes(const CachePlan& p, int64_t rows, int dim) {
  const int64_t s = p.splits();
  return s > 1 ? (align_up(s * rows * 2, 4) + s * rows * dim) * 4 : 0;
}

}  // namespace
}  // namespace tsc

using namespace tsc;

extern "C" int64_t tsc_cache_attention_workspace_bytes(int32_t samples, int64_t n_q, int64_t longest,
                                                       int64_t prefix_rows, int32_t q_heads, int32_t k_heads,
                                                       int32_t dim, int32_t left, int32_t right, int32_t sinks,
                                                       int32_t dtype) {
  if (!dtype_ok(dtype) || samples < 0 || n_q < 0 || longest < 0 || prefix_rows < 0 || q_heads <= 0 ||
      k_heads <= 0 || dim < 1 || dim > 256)
    return -1;
  if (n_q == 0 || samples == 0) return 0;
  return part_bytes(cache_plan(samples, n_q, longest, prefix_rows, q_heads, k_heads, dim, dtype_bytes(dtype), left,
                               right, sinks),
                    n_q * q_heads, dim);
}

extern "C" int tsc_cache_attention(const void* q, int64_t q_row, int64_t q_head, const void* k_pages,
                                   int64_t k_page, int64_t k_page_row, int64_t k_page_head, const void* v_pages,
                                   int64_t v_page, int64_t v_page_row, int64_t v_page_head, int64_t pages,
                                   int64_t page_rows, const int32_t* table, int64_t table_row, int64_t table_pages,
                                   const int32_t* offsets, const int32_t* lengths, int32_t samples,
                                   const int32_t* prefix, int64_t prefix_pages, int64_t n_q, int32_t q_heads,
                                   int32_t k_heads, int32_t dim, int32_t left, int32_t right, int32_t sinks,
                                   float scale, int32_t dtype, void* ws, int64_t ws_bytes, void* out,
                                   tsc_stream_t stream) {
  const char* what = "cache_attention";
  TSC_REQUIRE(dtype_ok(dtype), "%s: unknown dtype", what);
  TSC_REQUIRE(n_q >= 0 && n_q < (1ll << 31), "%s: invalid sizes", what);
  TSC_REQUIRE(q_heads > 0 && k_heads > 0 && q_heads % k_heads == 0 && q_heads <= 65535,
              "%s: %d query heads do not share %d key heads evenly", what, q_heads, k_heads);
  TSC_REQUIRE(n_q * (q_heads / k_heads) < (1ll << 32) - 1024,
              "%s: over 2^32 rows of queries and the heads that share a key head", what);
  TSC_REQUIRE(dim >= 1 && dim <= 256, "%s: head size %d, 1 to 256 are supported", what, dim);
  TSC_REQUIRE(sinks >= 0, "%s: negative number of sinks", what);
  TSC_REQUIRE(std::isfinite(scale), "%s: scale is not finite", what);
  CacheArgs a{};
  if (int rc = a.pages.set(what, table, table_row, table_pages, lengths, samples, pages, page_rows)) return rc;
  TSC_REQUIRE(prefix_pages >= 0 && prefix_pages <= table_pages, "%s: a prefix of %lld pages, the table has %lld",
              what, static_cast<long long>(prefix_pages), static_cast<long long>(table_pages));
  if (n_q == 0 || samples == 0) return 0;
  TSC_REQUIRE(q && out && offsets && (pages == 0 || (k_pages && v_pages)) && (prefix_pages == 0 || prefix),
              "%s: null pointer", what);
  const CachePlan p = cache_plan(samples, n_q, a.pages.most(), prefix_pages * page_rows, q_heads, k_heads, dim,
                                 dtype_bytes(dtype), left, right, sinks);
  const int64_t need = part_bytes(p, n_q * q_heads, dim);
  TSC_REQUIRE(need == 0 || (ws && ws_bytes >= need), "%s: a workspace of %lld bytes is needed", what,
              static_cast<long long>(need));
  if (pages == 0) a.pages.table_pages = 0, prefix_pages = 0;  // nothing is kept anywhere
  a.q = q, a.q_row = q_row, a.q_head = q_head;
  a.k = k_pages, a.k_at = {k_page, k_page_row, k_page_head};
  a.v = v_pages, a.v_at = {v_page, v_page_row, v_page_head};
  a.off_q = offsets, a.samples = samples, a.n_q = n_q;
  a.q_heads = q_heads, a.k_heads = k_heads, a.dim = dim;
  a.left = left < 0 ? kNoLimit : left, a.right = right < 0 ? kNoLimit : right, a.sinks = sinks;
  a.scale_log2 = scale == 0.f ? 1.f : fabsf(scale) * 1.44269504f;
  a.q_sign = scale > 0.f ? 1.f : scale < 0.f ? -1.f : 0.f;
  a.out = out, a.part = static_cast<float*>(ws);
  a.prefix = prefix, a.prefix_pages = static_cast<int>(prefix_pages);
  // (with 2^(l-1) < g <= 2^l: floor(2^32 (2^l - g) / g) + 1 and l - 1)
  const uint64_t g = q_heads / k_heads;
  int l = 0;
  while ((1ull << l) < g) ++l;
  a.group_mul = g == 1 ? 0 : static_cast<uint32_t>((((1ull << l) - g) << 32) / g + 1);
  a.group_shift = l - 1;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TSC_F32: return launch_cache<float>(a, p, s);
    case TSC_F16: return launch_cache<__half>(a, p, s);
    default: return launch_cache<__hip_bfloat16>(a, p, s);
  }
}
