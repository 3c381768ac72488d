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

// The form for many rows (of `lists` lists): 64 rows a wave or 32, and the parts,
// by what they cost by this account (in us): rounds of workgroups over the slots that the CUs have,
// each walking its part at what a key costs there; a round that leaves slots free
// gains up to 30%; more parts have more sums to write and join.  20k keys, 18
// tiles of 256 rows on 4 heads: 128 us in seven parts of one round, 155 in eight;
// 141 with 128 rows.  2 x 32k keys, 64 tiles: 615 us in two parts, 833 in one
// (half the slots), 671 with 128 rows.  Parts have 512 keys at least, which leaves
// CUs idle over short caches (4 x 17 rows, 16 heads on 4 of 64: 1000 keys 23 us in 16
// workgroups, 4000 keys 24; shorter parts are not measured).
CacheCut many_cut(int64_t rows, int64_t lists, int64_t heads, int64_t keys_of_row, int64_t keys_per_tile_row, int dim, int elem) {
  const int row_bytes = padded_dim(dim) * elem;
  CacheCut best;
  double least = 0;
  for (int w = can_pair(padded_dim(dim), elem) ? 2 : 1; w >= 1; --w) {
    const int per_cu = many_per_cu(row_bytes, w);
    const int64_t keys = keys_of_row + keys_per_tile_row * 128 * w;
    const double key = (w == 2 ? 0.0375 : row_bytes <= 128 ? 0.0336 : 0.0375 * row_bytes / 256) * (elem == 4 ? 4 : 1);
    // (lists of few tiles round up one by one; of many, some are shorter than others)
    const int64_t each = rows / lists, tile = 128 * w;
    const int64_t units = (each < 2 * tile ? lists * ceil_div(each, tile) : ceil_div(rows, tile)) * heads;
    for (int64_t parts = 1; parts == 1 || (parts <= keys / 512 && parts <= 16); ++parts) {
      const int64_t a_cu = ceil_div(units * parts, kCus), rest = a_cu % per_cu;
      const double rounds = a_cu / per_cu + (rest ? 0.7 + 0.3 * rest / per_cu : 0);
      const double us = rounds * (4 + keys * key / parts) +
                        (parts > 1 ? 6 + parts * rows * heads * (dim + 2) * 8 / 4e6 : 0);
      if (best.wave_rows && us >= least) continue;
      least = us, best.wave_rows = w, best.splits = static_cast<int>(parts);
    }
  }
  return best;
}

// longest: positions a sample may have, prefix_rows of them shared.
CachePlan cache_plan(int64_t samples, int64_t n_q, int64_t longest, int64_t prefix_rows, int q_heads, int k_heads,
                     int dim, int elem, int left, int right, int sinks) {
  CachePlan p;
  const int64_t group = q_heads / k_heads, all = n_q * group, mean = all / samples;
  const int row_bytes = padded_dim(dim) * elem, kt = cache_keys(row_bytes);
  p.row_blocks = mean <= 16 ? 1 : mean <= 32 ? 2 : 4;
  while (p.row_blocks > cache_row_blocks(row_bytes)) p.row_blocks /= 2;
  const int64_t rows = 16 * p.row_blocks;
  // own keys that rows of a sample can see at most: each of them, and with every
  // row more of the tile
  int64_t span = std::max<int64_t>(longest - prefix_rows, 0), per_row = 0;
  if (left >= 0) {
    const int64_t seen = (int64_t)left + sinks + kt + (right >= 0 ? right : n_q);
    if (seen < span) span = seen, per_row = right >= 0;
  }
  // Few rows against `keys`: parts of 256 to 2048 keys (4096 where a workgroup has
  // a CU to itself), one round of workgroups where that allows it: 64 samples of up
  // to 32k keys in parts of 2048 276 us, of 512 321, of 8192 295; 24 windows of
  // 4096 in one round of 1024 27 us, in two of 768 30.  Up to 1024 keys by
  // themselves are not worth a join (4 x 1000: 12 us, in parts 10 on the GPU, but the
  // host takes 16 with the second launch and the workspace).
  auto few = [&](int64_t keys, int64_t tiles, int64_t units) {
    CacheCut c;
    if (sinks > 0) keys += kt;  // (a tile of their own)
    const int per_cu = cache_per_cu(row_bytes);
    const int64_t slots = per_cu * kCus, lists = std::max<int64_t>(1, units * k_heads);
    const int64_t want = std::max<int64_t>(1, slots / lists);
    int64_t chunk = std::min<int64_t>(std::max<int64_t>(ceil_div(keys, want), 256), 4096 / per_cu);
    if (!prefix_rows && keys <= 1024) chunk = keys;
    // (and no more than 16 rounds are worth their parts' memory)
    chunk = std::max({chunk, ceil_div(keys, kMostSplits / 2), ceil_div(keys, std::max<int64_t>(1, 16 * slots / lists))});
    c.tiles = static_cast<int>(std::min<int64_t>(tiles, 1 << 30));  // (more than a launch takes)
    c.chunk = static_cast<int>(align_up(std::max<int64_t>(chunk, 1), kt * cache_waves(row_bytes)));
    c.splits = static_cast<int>(std::max<int64_t>(1, ceil_div(keys, c.chunk)));
    // (the table may have room for far more than is kept, in a captured step above all:
    // 4 x 4000 keys with room for 65536 each, 10.7 us, in parts of 2048 19.9)
    if (c.splits > 1 && c.splits <= want) c.chunk = -1;
    return c;
  };
  // One form for all samples, by their mean rows.  On the border, 4 samples of 16 and
  // of 17 rows, 16 heads on 4 of 64, over 300, 1000 and 4000 keys: bf16 16, 24 and 25
  // us, and 15, 23 and 24; f32 17, 32 and 44, and 31, 48 and 54 (a tile of 128 rows
  // half full).  Rows far from the mean pay for it: one sample of 2048 rows and 63 of
  // one over 32k keys take 1152 us, by themselves 333 and 365.
  if (mean <= 64) {
    // Tiles at most: those of every query by itself, or all rows' and one more a
    // sample; then an odd number, so that those that there are, the first, meet all
    // XCDs (4 samples of 4 rows over 8k keys, 16 heads on 4: 18.6 us, with 8 22.0; one
    // of 16 rows over 30k keys 31, with 8 41).
    const int64_t each = n_q * ceil_div(group, rows);
    p.own = few(span + per_row * rows, std::min(each, (all / rows + std::min(samples, n_q)) | 1),
                samples * ceil_div(mean, rows));
  } else {
    p.own = many_cut(all, samples, k_heads, span, per_row, dim, elem);
    p.own.tiles = static_cast<int>(std::min<int64_t>(all / (128 * p.own.wave_rows) + std::min(samples, n_q), 1 << 30));
  }
  if (prefix_rows && all <= 64) {
    p.prefix = few(prefix_rows, ceil_div(all, rows), ceil_div(all, rows));
  } else if (prefix_rows && mean <= 64 && row_bytes <= 128) {
    // beside the samples' own keys (cache_both_kernel), one workgroup a CU and 512
    // keys at least: 32k keys in 8 tiles 42 us in 32 parts, 45 in 64, 61 in 128
    p.prefix.wave_rows = 1, p.prefix.tiles = static_cast<int>(ceil_div(all, 128));
    p.prefix.splits = static_cast<int>(std::max<int64_t>(
        1, std::min<int64_t>({prefix_rows / 512, kCus / ((int64_t)p.prefix.tiles * k_heads), kMostSplits / 2})));
  } else if (prefix_rows) {
    p.prefix = many_cut(all, 1, k_heads, prefix_rows, 0, dim, elem);
    p.prefix.tiles = static_cast<int>(ceil_div(all, 128 * p.prefix.wave_rows));
  }
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
