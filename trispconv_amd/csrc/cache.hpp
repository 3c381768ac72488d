// Attention of new rows over what their samples keep in pages.
//
// Sample b's lengths[b] = Lk positions lie in the pages of its row of the table;
// its Lq queries are the last of them.  What a query sees, and what comes out,
// is as for packed keys (attend.hpp), with the keys and values fetched page by
// page.  With a prefix of P pages every sample's first P R positions are those
// pages: their keys are read once, for the queries of all samples (one list of
// rows), and the rest sample by sample.  A call is cut into parts, the prefix's
// and each sample's own keys in chunks of their own; a part leaves its reference
// score m, the sum l of the exponentials and the sums o of the values, and
//   out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.
#pragma once

#include "attend.hpp"
#include "pages.hpp"

namespace tsc {

struct CacheArgs : AttendArgs {
  PageTable pages;
  PageStrides k_at, v_at;
  const int32_t* prefix;  // its pages, or none
  int prefix_pages;
  // r / group for any 32-bit r without a division: with t = umulhi(r, group_mul),
  // (t + (r - t) / 2) >> group_shift; group_mul 0 for groups of one
  uint32_t group_mul;
  int group_shift;
  __host__ __device__ int prefix_rows() const { return prefix_pages * pages.page_rows; }
};

// How the prefix's or the samples' own keys are cut: tiles of query rows (at
// most), and parts of the keys, numbered from first_split on.
struct CacheCut {
  int tiles = 0, splits = 0, first_split = 0;
  int wave_rows = 0;  // rows of a workgroup of four waves in 128s, 0: the form for few rows
  int chunk = 0;      // that form's keys of a part; -1: a tile's shared out evenly, 256 at least
};
struct CachePlan {
  int row_blocks = 1;  // that form's rows of a tile in 16s
  CacheCut prefix, own;
  int splits() const { return prefix.splits + own.splits; }
};

template <typename T>
int launch_cache(const CacheArgs& a, const CachePlan& p, hipStream_t s);

// The form for few rows: keys of a wave's tile, waves of a workgroup and the
// tiles of K and V that each has in LDS, one in use and the others on their way.
// Two workgroups share a CU's LDS, so that one walks while the other begins or
// ends; rows of 256 bytes and more leave too few waves for that (32 x 16k keys,
// heads of 128, bf16: 147 us with one workgroup of four waves, 152 with two of two;
// heads of 64 in f32: 86 and 102; of 64 in bf16, 64 x 32k keys: 286 with one of
// eight, 276 with two of four).
constexpr int cache_per_cu(int row_bytes) { return row_bytes <= 192 ? 2 : 1; }
constexpr int cache_lds(int row_bytes) { return (152 << 10) / cache_per_cu(row_bytes) - (4 << 10); }
constexpr int cache_keys(int row_bytes) { return row_bytes <= 512 ? 32 : 16; }
constexpr int cache_tile(int row_bytes) { return 2 * cache_keys(row_bytes) * row_bytes; }
constexpr int cache_waves(int row_bytes) {
  const int most = cache_lds(row_bytes) / (2 * cache_tile(row_bytes));
  return most < 4 ? most : 4;
}
constexpr int cache_buffers(int row_bytes) {
  return cache_lds(row_bytes) / (cache_waves(row_bytes) * cache_tile(row_bytes));
}
// The form for many rows: key blocks of a tile and its buffers (8k rows, 16 heads of
// 64, bf16: 333 us with three, 364 with two; rows of 256 bytes have no room for
// more at two workgroups a CU, and halved tiles cost them 30%).
constexpr int many_key_blocks(int row_bytes) { return row_bytes <= 512 ? 2 : 1; }
constexpr int many_buffers(int row_bytes) { return row_bytes <= 192 ? 3 : 2; }
// Its workgroups a CU (row_blocks: 32s of rows a wave).
constexpr int many_per_cu(int row_bytes, int row_blocks) {
  return row_bytes <= 128 ? 4 - row_blocks : row_bytes <= 256 ? 2 : 1;
}
// Waves a SIMD that the compiler leaves registers for.  With two, a wave's half of the
// file holds the products' sums as well; a wave with all of it keeps them in the
// other half and moves them over and back for every tile (few rows, `values` a lane
// of a quarter: 8 samples of 16 rows over 32k keys, 16 heads on 4 of 64, bf16, 92 us,
// before 154; 4 x 1000 keys 11.4, before 12.1; four samples of 512 rows over 8k keys,
// heads of 128, f32, 1057 us, before 1097).  More do not fit (16 rows, heads of 256,
// bf16: 532 us, in half the file 2855).
constexpr int few_per_simd(int values) { return values <= 384 ? 2 : 1; }
constexpr int many_per_simd(int dim, int per_cu) { return dim <= 128 && per_cu < 2 ? 2 : per_cu; }
// Rows of a tile in 16s at most: queries and sums stay in the registers (8 samples of
// 16 rows over 32k keys, 16 heads on 4: of 128, bf16, 199 us in 32s, 203 in 64s; of 64,
// f32, 271 and 324; of 256, bf16, 532 in 32s, 636 in 16s).
constexpr int cache_row_blocks(int row_bytes) { return row_bytes <= 192 ? 4 : row_bytes <= 512 ? 2 : 1; }

namespace {

// c += a b for a 16x16 tile: lane l holds row (a) or column (b) l % 16, and of the
// sum's terms the 16 bytes' elements of its quarter l / 16, the same for a and b.
// c: lane l holds column l % 16, rows 4 (l / 16) + 0..3.
template <typename T>
__device__ __forceinline__ f32x4 mma16(int4v a, int4v b, f32x4 c) {
  if constexpr (std::is_same_v<T, __half>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                  0, 0);
  } else if constexpr (std::is_same_v<T, __hip_bfloat16>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                   0, 0, 0);
  } else {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
    return c;
  }
}

// 16 bytes per lane from an address of its own; otherwise as load_to_lds.
__device__ __forceinline__ void load_to_lds_from(const void* p, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(p), "s"(m0) : "memory");
}

// The larger of a lane's value and that of the lane 16 away in its half.
__device__ __forceinline__ float max_quarters(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

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

// A loaded value that is waited for here, and not at its first use: there the
// compiler would wait for all loads, those to LDS that it knows nothing of too.
template <typename V>
__device__ __forceinline__ void arrived(V& v) {
  asm volatile("" : "+v"(v));
}

// 64 page numbers from `from` on, a lane each.
struct PageIds {
  const int32_t* ids;
  int entries;  // of the table's row
  int pages, from, id;
  __device__ __forceinline__ void begin(const int32_t* ids_, int entries_, int pages_) {
    ids = ids_, entries = entries_, pages = pages_, from = -1, id = 0;
  }
  // Pages first to last (at most 63 further) are among them.
  __device__ __forceinline__ void seek(int first, int last) {
    if (from >= 0 && first >= from && last < from + kWave) return;
    from = first;
    id = min(max(ids[min(from + (int)(threadIdx.x % kWave), entries - 1)], 0), pages - 1);
    arrived(id);
  }
};

// Positions of sample b.
__device__ __forceinline__ int kept(const CacheArgs& a, int b) {
  return a.pages.cut(a.pages.lengths[b]);
}

// Tiles of `rows` query rows of all samples.
__device__ __forceinline__ int64_t count_tiles(const CacheArgs& a, int group, int rows) {
  const int lane = threadIdx.x % kWave;
  int64_t all = 0;
  for (int b0 = 0; b0 < a.samples; b0 += kWave) {
    int64_t at = 0;
    int len = 0;
    if (b0 + lane < a.samples) sample_range(a.off_q, b0 + lane, a.n_q, at, len);
    const uint32_t inc = wave_inclusive(static_cast<uint32_t>(((int64_t)len * group + rows - 1) / rows));
    all += __builtin_amdgcn_readlane(inc, kWave - 1);
  }
  return all;
}

// The sample and the tile of query rows within it of the x-th tile of all (as
// find_tile).  false: past the last.
__device__ __forceinline__ bool find_rows(const CacheArgs& a, int group, int rows, int x, int& b, int64_t& q0,
                                          int& lq, int& lk, int& tile) {
  const int lane = threadIdx.x % kWave;
  for (int b0 = 0; b0 < a.samples; b0 += kWave) {
    int64_t at = 0;
    int len = 0, keys = 0;
    if (b0 + lane < a.samples) {
      sample_range(a.off_q, b0 + lane, a.n_q, at, len);
      keys = kept(a, b0 + lane);
    }
    const uint32_t tiles = static_cast<uint32_t>(((int64_t)len * group + rows - 1) / rows);
    const uint32_t inc = wave_inclusive(tiles);
    const uint64_t past = __ballot(inc > static_cast<uint32_t>(x));
    if (past) {
      const int at_lane = __builtin_ctzll(past);
      b = b0 + at_lane;
      tile = x - __builtin_amdgcn_readlane(inc - tiles, at_lane);
      lq = __builtin_amdgcn_readlane(len, at_lane);
      lk = __builtin_amdgcn_readlane(keys, at_lane);
      q0 = __builtin_amdgcn_readlane(static_cast<int>(at), at_lane);
      return true;
    }
    x -= __builtin_amdgcn_readlane(inc, kWave - 1);
  }
  return false;
}

// The query rows of one sample, or of all of them, each with a position of its own.
struct CacheWalk : Walk {
  const CacheArgs* args;
  // The sample; -1: all, and lk is where their rows end: what the offsets name past
  // that is cut off, as sample_range does.  (The arguments' n_q instead takes
  // cache_tile_kernel scalar registers in the walk: 512 to 2 rows over 15k to 20k
  // keys 136 us, with lk 128.)
  int b;
  __device__ __forceinline__ int token(uint32_t r) const {
    r = min(r, rows - 1);
    const uint32_t t = __umulhi(r, args->group_mul);
    return static_cast<int>(args->group_mul ? (t + ((r - t) >> 1)) >> args->group_shift : r);
  }
  __device__ __forceinline__ int head(uint32_t r) const {
    return hk * group + static_cast<int>(min(r, rows - 1) - static_cast<uint32_t>(token(r)) * group);
  }
  __device__ __forceinline__ void seen(const AttendArgs& a, uint32_t r, int& lo, int& hi, int& sink) const {
    int p = token(r) + shift, keys = lk;
    if (b < 0) {
      const int64_t t = q0 + token(r);
      const int s = first_past(a.off_q, a.samples, t);
      keys = kept(*args, s);
      p = position(t, min(a.off_q[s + 1], lk), keys);
    }
    seen_keys(p, keys, a.left, a.right, a.sinks, lo, hi, sink);
  }
  __device__ __forceinline__ void bounds(const AttendArgs& a, uint32_t first, uint32_t last, int& lo_first,
                                         int& hi_first, int& lo_last, int& hi_last) const {
    int sink;
    seen(a, first, lo_first, hi_first, sink);
    seen(a, last, lo_last, hi_last, sink);
  }
  template <int N, int STEP>
  __device__ __forceinline__ void wave(const AttendArgs& a, uint32_t first, int col, int lo[N], int hi[N],
                                       int& lo_first, int& hi_first, int& lo_last, int& hi_last) const {
    if (b >= 0) {  // (later rows see later keys)
      int sink;
#pragma unroll
      for (int x = 0; x < N; ++x) seen(a, first + x * STEP + col, lo[x], hi[x], sink);
      lo_first = __builtin_amdgcn_readlane(lo[0], 0), hi_first = __builtin_amdgcn_readlane(hi[0], 0);
      lo_last = __builtin_amdgcn_readlane(lo[N - 1], STEP - 1), hi_last = __builtin_amdgcn_readlane(hi[N - 1], STEP - 1);
      return;
    }
    int at[N], end[N], length[N];
    int64_t t[N];
#pragma unroll
    for (int x = 0; x < N; ++x) t[x] = q0 + token(first + x * STEP + col);
    samples_of<N>(a.off_q, args->pages.lengths, a.samples, q0 + token(first), q0 + token(first + N * STEP - 1), t, at,
                  end, length);
    lo_first = hi_first = kNoLimit, lo_last = hi_last = 0;
#pragma unroll
    for (int x = 0; x < N; ++x) {
      int sink;
      const int keys = args->pages.cut(length[x]);
      seen_keys(position(t[x], min(end[x], lk), keys), keys, a.left, a.right, a.sinks, lo[x], hi[x], sink);
      lo_first = min(lo_first, lo[x]), lo_last = max(lo_last, lo[x]);
      hi_first = min(hi_first, hi[x]), hi_last = max(hi_last, hi[x]);
    }
#pragma unroll
    for (int x = 1; x < STEP; x <<= 1) {
      lo_first = min(lo_first, __shfl_xor(lo_first, x, kWave)), lo_last = max(lo_last, __shfl_xor(lo_last, x, kWave));
      hi_first = min(hi_first, __shfl_xor(hi_first, x, kWave)), hi_last = max(hi_last, __shfl_xor(hi_last, x, kWave));
    }
    lo_first = __builtin_amdgcn_readfirstlane(lo_first), lo_last = __builtin_amdgcn_readfirstlane(lo_last);
    hi_first = __builtin_amdgcn_readfirstlane(hi_first), hi_last = __builtin_amdgcn_readfirstlane(hi_last);
  }
  // Row t's position in a sample whose rows end at `end`.
  __device__ static __forceinline__ int position(int64_t t, int end, int keys) {
    return static_cast<int>(max(t - end + keys, -(int64_t)(1 << 30)));
  }
  // Takes the x-th tile of `tile_rows` rows (the prefix's: of all samples) and the
  // range of keys [from, to) of this part.  false: past the last tile.
  __device__ __forceinline__ bool begin(const CacheArgs& a, bool prefix, int tile_rows, int x, int& from, int& to) {
    args = &a;
    int tile = x;
    if (prefix) {
      int64_t last;
      sample_rows(a, q0, last);
      rows = static_cast<uint32_t>((last - q0) * group);
      b = -1, lk = static_cast<int>(last), shift = 0, from = 0, to = a.prefix_rows();
      if ((int64_t)tile * tile_rows >= rows) return false;
    } else {
      int lq;
      if (!find_rows(a, group, tile_rows, x, b, q0, lq, lk, tile)) return false;
      rows = static_cast<uint32_t>(lq) * group;
      shift = lk - lq, from = a.prefix_rows(), to = lk;
    }
    row0 = static_cast<uint32_t>(tile) * tile_rows;
    return true;
  }
  __device__ const int32_t* table() const {
    return b < 0 ? args->prefix : args->pages.table + b * args->pages.table_row;
  }
  __device__ int entries() const { return b < 0 ? args->prefix_pages : args->pages.table_pages; }
  // The key tiles of rows that see from lo_first on, up to hi_last at most: the
  // window's begin at a multiple of `align`.  Returns how many there are.
  __device__ __forceinline__ int place(int lo_first, int hi_last, int from, int to, int kt, int align) {
    start = lo_first / align * align;
    sink_end = min(args->sinks, hi_last);
    if (args->sinks > start) start = sink_end = 0;
    start = max(start, from), end = min(hi_last, to);
    sink_start = from, sink_end = min(sink_end, to);
    sink_tiles = max(sink_end - sink_start + kt - 1, 0) / kt;
    return sink_tiles + max(end - start + kt - 1, 0) / kt;
  }
  // The first key of the window's first tile that a row sees (as a sink, or in
  // its window): what lies before it in the tile is not read.
  __device__ int first_seen(int lo_first) const {
    return args->sinks > start ? start : max(start, min(lo_first, end - 1));
  }
};

template <typename T>
__device__ __forceinline__ PagedRows<T> paged_rows(const CacheArgs& a, const void* base, const PageStrides& at,
                                                   const CacheWalk& w) {
  return {static_cast<const T*>(base) + w.hk * at.head, at.page, at.row, w.table(), &a.pages};
}

// What 16-byte slot chunk c of row r of a V tile is stored in: the 16 lanes that
// read b64 pieces of four rows, twice (16 bits), and the 64 that read words of
// four rows four apart (f32), find them in different columns of 256 bytes.
template <int RB, bool F32>
__device__ __forceinline__ int v_slot16(int r, int c) {
  if constexpr (F32) return RB % 256 == 0 ? c ^ (4 * ((r >> 2) & 3)) : RB % 128 == 0 ? c ^ (4 * ((r >> 2) & 1)) : c;
  return RB % 256 == 0 ? c ^ (2 * (r & 7)) : RB % 128 == 0 ? c ^ (2 * ((r >> 1) & 3)) : c ^ (2 * ((r >> 2) & 1));
}

// Brings tiles of KT rows of one head's K and V into a wave's LDS, chunk by chunk
// in the order of the slots.  Rows before `first` or from `to` on are those
// nearest to them again, and chunks past the head's last are its first again (q
// is 0 there): nothing is read that no query sees, and every tile takes the
// same number of loads, which the waits count on.
template <typename T, int DP, int KT, bool ALIGNED>
struct PagedStager {
  static constexpr int RB = DP * sizeof(T), CH = RB / 16, ROUNDS = KT * CH / kWave;
  static constexpr int LOADS = 2 * ROUNDS;
  static_assert(KT * CH % kWave == 0, "whole instructions");
  const T* k;
  const T* v;
  PageStrides k_at, v_at;
  const PageTable* pages;
  PageIds ids;
  int dim;
  int page;           // whose first rows' addresses these are, -1: none
  const T* k_base;
  const T* v_base;
  uint32_t k_offset[ROUNDS], v_offset[ROUNDS];

  __device__ static int slot(int i) { return i * kWave + (int)(threadIdx.x % kWave); }
  __device__ static int row(int i) { return slot(i) / CH; }
  __device__ static int k_chunk(int i) { return k_slot<RB>(slot(i) / CH, slot(i) % CH); }
  __device__ static int v_chunk(int i) { return v_slot16<RB, !kIs16<T>>(slot(i) / CH, slot(i) % CH); }
  __device__ int there(int c) const { return c * kPer16<T> < dim ? c : 0; }

  __device__ __forceinline__ void begin(const CacheArgs& a, int hk, const int32_t* table, int entries) {
    k = static_cast<const T*>(a.k) + hk * a.k_at.head, v = static_cast<const T*>(a.v) + hk * a.v_at.head;
    k_at = a.k_at, v_at = a.v_at, pages = &a.pages, dim = a.dim;
    ids.begin(table, entries, a.pages.pages);
    page = -1, k_base = v_base = nullptr;
    if constexpr (ALIGNED) {
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i) {
        k_offset[i] = static_cast<uint32_t>(row(i) * k_at.row * sizeof(T)) + there(k_chunk(i)) * 16;
        v_offset[i] = static_cast<uint32_t>(row(i) * v_at.row * sizeof(T)) + there(v_chunk(i)) * 16;
      }
    }
  }
  // Asks for the page numbers from row j on.
  __device__ __forceinline__ void seek(int j) {
    const int p = __builtin_amdgcn_readfirstlane(pages->page_of(j));
    ids.seek(p, p);
  }
  __device__ __forceinline__ void load(char* tile, int j0, int first, int to) {
    const int j_first = first, j_last = min(j0 + KT, to) - 1;
    const int p_first = __builtin_amdgcn_readfirstlane(pages->page_of(j_first));
    const int p_last = __builtin_amdgcn_readfirstlane(pages->page_of(j_last));
    const uint32_t at = __builtin_amdgcn_readfirstlane(lds_address(tile));
    if (ALIGNED && p_first == p_last && j_first == j0 && j_last == j0 + KT - 1) {
      if (p_first != page) {
        page = p_first;
        ids.seek(page, page);
        const int64_t id = __builtin_amdgcn_readlane(ids.id, page - ids.from);
        k_base = k + id * k_at.page, v_base = v + id * v_at.page;
      }
      const int64_t r = j0 - page * pages->page_rows;
      const T* kp = k_base + r * k_at.row;
      const T* vp = v_base + r * v_at.row;
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i) load_to_lds(kp, k_offset[i], at + i * 1024);
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i) load_to_lds(vp, v_offset[i], at + KT * RB + i * 1024);
      return;
    }
    ids.seek(p_first, p_last);
#pragma unroll 2
    for (int i = 0; i < ROUNDS; ++i) {
      const int j = min(max(j0 + row(i), j_first), j_last), p = static_cast<int>(pages->page_of(j));
      const int64_t id = __shfl(ids.id, p - ids.from, kWave), r = j - p * pages->page_rows;
      const T* kp = k + id * k_at.page + r * k_at.row;
      const T* vp = v + id * v_at.page + r * v_at.row;
      if constexpr (ALIGNED) {
        load_to_lds_from(kp + there(k_chunk(i)) * kPer16<T>, at + i * 1024);
        load_to_lds_from(vp + there(v_chunk(i)) * kPer16<T>, at + KT * RB + i * 1024);
      } else {
        auto chunk = [&](const T* p, int c) {
          const int d = c * kPer16<T>;
          return d + kPer16<T> <= dim ? load16_unaligned(p + d) : load16_partial(p + d, dim - d);
        };
        *reinterpret_cast<int4v*>(tile + slot(i) * 16) = chunk(kp, k_chunk(i));
        *reinterpret_cast<int4v*>(tile + KT * RB + slot(i) * 16) = chunk(vp, v_chunk(i));
      }
    }
  }
};

// Few query rows (16 NR; rows past the last are copies of it) against many keys:
// the keys of a workgroup's chunk are shared out over its waves, each with tiles
// of its own in LDS and no barrier between them, and the waves' sums meet in LDS
// at the end.  Bound by memory: 64 samples of 14k to 33k keys, 16 heads on 4 of 64,
// bf16, 1.53 GB in 276 us, 5.5 TB/s (a large copy on this card: 4.87).  Small
// calls are bound by what comes before the first tile: arguments, offsets, page
// numbers and keys are dependent reads, 6 of the 11 us of 4 x 900 keys.
//
// Scores are kept transposed as in attend.hpp, S^T = K Q^T, in 16x16 tiles: a lane
// has four keys of one row per 16, which are, as they stand, the right operand of
// O^T = V^T e^S^T.  A row's reference is the largest of its first tile's scores and
// moves only when weights outgrow it (kMostWeight).  Weights of 16-bit tensors go
// into the product as two parts, value and remainder, which leave out 2^-16 of a
// bf16 weight and 2^-22 of an f16 one at most: errors against 64 bits are those of
// f32 weights (bf16 0.0017), with one part 0.0024.  The walk is bound by memory, and
// the products are idle.
template <typename T, int DP, int NR, bool ALIGNED>
__device__ __forceinline__ void cache_few(const CacheArgs& a, const CacheCut& cut, bool is_prefix, int splits,
                                          uint32_t id, char* lds) {
  constexpr int RB = DP * sizeof(T), KT = cache_keys(RB), WAVES = cache_waves(RB), KB = KT / 16;
  constexpr int STEPS = RB / 64, DB = DP / 16, TILE = cache_tile(RB), ROWS = 16 * NR, BUFFERS = cache_buffers(RB);
  using Stager = PagedStager<T, DP, KT, ALIGNED>;
  static_assert((BUFFERS - 1) * Stager::LOADS <= 63, "the wait counts to 63");
  static_assert(ROWS * DP * 4 <= BUFFERS * TILE, "a wave's sums take the place of its tiles");
  // lds: the waves' tiles, m and l of the waves' rows, a word a wave
  float* ml = reinterpret_cast<float*>(lds + WAVES * BUFFERS * TILE);
  const int lane = threadIdx.x % kWave, col = lane % 16, quarter = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  auto zero_others = [&] {
    if (splits > 1) return;  // (the join does it)
    int64_t first, last;
    sample_rows(a, first, last);
    if (first > 0 || last < a.n_q)
      zero_outside(static_cast<T*>(a.out), (int64_t)a.q_heads * a.dim, first, last, a.n_q);
  };

  // rows next to each other, then heads, then chunks
  const uint32_t rest = id / cut.tiles;
  const int split = rest / a.k_heads;
  CacheWalk w;
  w.group = a.q_heads / a.k_heads;
  w.hk = rest - split * a.k_heads;
  int from, to;
  if (!w.begin(a, is_prefix, ROWS, id - rest * cut.tiles, from, to)) return zero_others();
  const uint32_t row0 = w.row0;

  // rows past the last are copies of it
  int lo[NR], hi[NR], lo_min, hi_min, lo_max, hi_max;
  w.template wave<NR, 16>(a, row0, col, lo, hi, lo_min, hi_min, lo_max, hi_max);
  // the window's tiles begin where pages of whole tiles have theirs
  const int tiles = w.place(lo_min, hi_max, from, to, KT, a.pages.page_rows % KT == 0 ? KT : 1);
  // this chunk's tiles, and this wave's
  int chunk_tiles = cut.chunk / KT;
  if (cut.chunk < 0) {
    const float share = static_cast<float>(tiles) * __builtin_amdgcn_rcpf(static_cast<float>(cut.splits * WAVES));
    chunk_tiles = max(static_cast<int>(ceilf(share)) * WAVES, 256 / KT / WAVES * WAVES);
  }
  const int c0 = min(split * (int64_t)chunk_tiles, (int64_t)tiles);
  const int c1 = split == cut.splits - 1 ? tiles : min(c0 + chunk_tiles, tiles), each = (c1 - c0 + WAVES - 1) / WAVES;
  const int t0 = min(c0 + wave * each, c1), t1 = min(t0 + each, c1);
  auto item_of = [&](uint32_t r) { return (w.q0 + w.token(r)) * a.q_heads + w.head(r); };
  const int part = cut.first_split + split;
  if (c0 == c1 && splits > 1) {  // nothing to see here
    for (uint32_t r = threadIdx.x; r < ROWS; r += kWave * WAVES)
      if (row0 + r < w.rows) {
        const int64_t at = part * a.rows() + item_of(row0 + r);
        a.part[2 * at] = -__builtin_inff();
        a.part[2 * at + 1] = 0.f;
      }
    return;
  }

  int4v qf[NR][STEPS];
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    const uint32_t r = row0 + 16 * x + col;
    const T* q = static_cast<const T*>(a.q) + (w.q0 + w.token(r)) * a.q_row + w.head(r) * a.q_head;
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      const int d = (4 * st + quarter) * kPer16<T>;
      int4v y;
      if (d + kPer16<T> <= a.dim) y = load16_unaligned(q + d);
      else y = load16_partial(q + d, a.dim - d);
      if (a.q_sign != 1.f) {  // (as in attend_walk)
        T e[kPer16<T>];
        __builtin_memcpy(e, &y, 16);
#pragma unroll
        for (int i = 0; i < kPer16<T>; ++i) e[i] = from_f32<T>(to_f32(e[i]) * a.q_sign);
        __builtin_memcpy(&y, e, 16);
      }
      qf[x][st] = y;
    }
  }
  Stager stager;
  stager.begin(a, w.hk, w.table(), w.entries());
  char* mine = lds + wave * BUFFERS * TILE;
  auto place = [&](int t) { return t < w.sink_tiles ? w.sink_start + t * KT : w.start + (t - w.sink_tiles) * KT; };
  const int first_seen = w.first_seen(lo_min);
  auto stage = [&](int t, int buf) {
    const int j0 = place(t);
    stager.load(mine + buf * TILE, j0, t == w.sink_tiles ? first_seen : j0, t < w.sink_tiles ? w.sink_end : w.end);
  };
  if (t0 < t1) stager.seek(place(t0));  // (while the queries are on their way)
#pragma unroll
  for (int x = 0; x < NR; ++x)
#pragma unroll
    for (int st = 0; st < STEPS; ++st) arrived(qf[x][st]);
#pragma unroll
  for (int i = 0; i < BUFFERS - 1; ++i)
    if (t0 + i < t1) stage(t0 + i, i);
  zero_others();

  f32x4 o[NR][DB];
  float m[NR], l[NR];  // reference; this lane's share of the sum
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    m[x] = -__builtin_inff(), l[x] = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db) o[x][db] = f32x4(0.f);
  }
  const float c = a.scale_log2;
  for (int t = t0, buf = 0; t < t1; ++t, buf = buf + 1 == BUFFERS ? 0 : buf + 1) {
    if (t + BUFFERS - 1 < t1) {
      // (what was read from that buffer has arrived)
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      stage(t + BUFFERS - 1, buf == 0 ? BUFFERS - 1 : buf - 1);
    }
    // all but the tiles behind this one
    const int behind = min(t1 - 1 - t, BUFFERS - 1);
    for_each_index(
        [&](auto n) {
          if (behind == n) asm volatile("s_waitcnt vmcnt(%0)" : : "n"(ALIGNED ? n * Stager::LOADS : 0) : "memory");
        },
        std::make_integer_sequence<int, BUFFERS>{});
    const char* kt = mine + buf * TILE;
    const char* vt = kt + KT * RB;
    const int j0 = place(t), last = t < w.sink_tiles ? w.sink_end : w.end;
    f32x4 s[NR][KB];
#pragma unroll
    for (int x = 0; x < NR; ++x)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) s[x][kb] = f32x4(0.f);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        const int4v k = *reinterpret_cast<const int4v*>(kt + (16 * kb + col) * RB +
                                                        k_slot<RB>(16 * kb + col, 4 * st + quarter) * 16);
#pragma unroll
        for (int x = 0; x < NR; ++x) s[x][kb] = mma16<T>(k, qf[x][st], s[x][kb]);
      }
    const bool whole = j0 + KT <= min(last, hi_min) && (j0 >= lo_max || j0 + KT <= a.sinks);
    if (!whole) {
#pragma unroll
      for (int x = 0; x < NR; ++x)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = j0 + 16 * kb + 4 * quarter + i;
            const bool see = j < min(last, hi[x]) && (j >= lo[x] || j < a.sinks);
            s[x][kb][i] = see ? s[x][kb][i] : -__builtin_inff();
          }
    }
    // weights, and their sums; a new reference rescales what is there
    float p[NR][KB][4], sum[NR];
    auto weights = [&] {
#pragma unroll
      for (int x = 0; x < NR; ++x) {
        const float base = m[x] == -__builtin_inff() ? 0.f : m[x];
        sum[x] = 0.f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p[x][kb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][kb][i] - base, c, kLift<T>));
            sum[x] += p[x][kb][i];
          }
      }
    };
    bool over = false;
    weights();
#pragma unroll
    for (int x = 0; x < NR; ++x) over |= m[x] == -__builtin_inff() || sum[x] > kMostWeight<T>;
    if (__any(over)) {
#pragma unroll
      for (int x = 0; x < NR; ++x) {
        float top = m[x];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, s[x][kb][i]);
        top = max_halves(max_quarters(top));
        const float fix = m[x] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((m[x] - top) * c);
        m[x] = top;
        l[x] *= fix;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[x][db] *= fix;
      }
      weights();
    }
#pragma unroll
    for (int x = 0; x < NR; ++x) l[x] += sum[x];
    if constexpr (kIs16<T>) {
      static_assert(KB == 2, "a product of 32 keys");
      int4v ph[NR], pl[NR];  // the weights, and what their rounding leaves
#pragma unroll
      for (int x = 0; x < NR; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float u = p[x][i / 2][i % 2 * 2], v = p[x][i / 2][i % 2 * 2 + 1];
          ph[x][i] = pack2<T>(u, v);
          T e[2];
          const int both = ph[x][i];
          __builtin_memcpy(e, &both, 4);
          pl[x][i] = pack2<T>(u - to_f32(e[0]), v - to_f32(e[1]));
        }
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        int4v y;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = 16 * h + 4 * quarter + col / 4, d = 16 * db + 4 * (col % 4);
          const char* at = vt + r * RB + v_slot16<RB, false>(r, d / 8) * 16 + d % 8 * 2;
          const int2v z = __builtin_bit_cast(int2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                        (__attribute__((address_space(3))) short4v*)at));
          y[2 * h] = z[0], y[2 * h + 1] = z[1];
        }
#pragma unroll
        for (int x = 0; x < NR; ++x) {
          o[x][db] = mma16<T>(y, ph[x], o[x][db]);
          o[x][db] = mma16<T>(y, pl[x], o[x][db]);
        }
      }
    } else {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 16 * kb + 4 * quarter + i;
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            const int ch = 4 * db + col / 4;
            const float y = *reinterpret_cast<const float*>(vt + r * RB + v_slot16<RB, true>(r, ch) * 16 + col % 4 * 4);
#pragma unroll
            for (int x = 0; x < NR; ++x)
              o[x][db] = __builtin_amdgcn_mfma_f32_16x16x4f32(y, p[x][kb][i], o[x][db], 0, 0, 0);
          }
        }
    }
  }

  // the waves' sums meet
  float off = 0.f;  // NaN when one of them is not finite
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    l[x] += __shfl_xor(l[x], 16, kWave);
    l[x] += __shfl_xor(l[x], 32, kWave);
    off = __builtin_fmaf(l[x], 0.f, off);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i) off = __builtin_fmaf(o[x][db][i], 0.f, off);
    if (quarter == 0) {
      ml[2 * (wave * ROWS + 16 * x + col)] = m[x];
      ml[2 * (wave * ROWS + 16 * x + col) + 1] = l[x];
    }
  }
  int* odd = reinterpret_cast<int*>(ml + 2 * WAVES * ROWS);
  if (lane == 0) odd[wave] = 0;
  if (off != off) odd[wave] = 1;
  __syncthreads();
  int any = 0;
#pragma unroll
  for (int y = 0; y < WAVES; ++y) any |= odd[y];
  if (!any) {
    float* sums = reinterpret_cast<float*>(mine);
#pragma unroll
    for (int x = 0; x < NR; ++x) {
      float all = -__builtin_inff();
#pragma unroll
      for (int y = 0; y < WAVES; ++y) all = fmaxf(all, ml[2 * (y * ROWS + 16 * x + col)]);
      const float f = m[x] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((m[x] - all) * c);
#pragma unroll
      for (int db = 0; db < DB; ++db)
        *reinterpret_cast<f32x4*>(sums + (16 * x + col) * DP + 16 * db + 4 * quarter) = f * o[x][db];
    }
    __syncthreads();
    constexpr int PIECES = DP / 4;
    for (int x = threadIdx.x; x < ROWS * PIECES; x += kWave * WAVES) {
      const int r = x / PIECES, d = x % PIECES * 4;
      if (row0 + r >= w.rows || d >= a.dim) continue;
      float all = -__builtin_inff(), sum = 0.f;
#pragma unroll
      for (int y = 0; y < WAVES; ++y) all = fmaxf(all, ml[2 * (y * ROWS + r)]);
      f32x4 v = f32x4(0.f);
#pragma unroll
      for (int y = 0; y < WAVES; ++y) {
        const float my = ml[2 * (y * ROWS + r)], ly = ml[2 * (y * ROWS + r) + 1];
        sum += my == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((my - all) * c) * ly;
        v += *reinterpret_cast<const f32x4*>(lds + y * BUFFERS * TILE + (r * DP + d) * 4);
      }
      const int64_t item = item_of(row0 + r);
      const int cnt = min(4, a.dim - d);
      if (splits > 1) {
        const int64_t at = part * a.rows() + item;
        float* to = a.part + a.part_values(splits) + at * a.dim + d;
        if (d == 0) {
          a.part[2 * at] = sum == 0.f ? -__builtin_inff() : all * c - kLift<T>;
          a.part[2 * at + 1] = sum;
        }
        for (int i = 0; i < cnt; ++i) to[i] = v[i];
      } else {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        T* to = static_cast<T*>(a.out) + item * a.dim + d;
        for (int i = 0; i < cnt; ++i) to[i] = from_f32<T>(v[i] * inv);
      }
    }
    return;
  }
  // a value that is not finite, seen or not: key by key, of the seen ones only
  const PagedRows<T> kr = paged_rows<T>(a, a.k, a.k_at, w), vr = paged_rows<T>(a, a.v, a.v_at, w);
  const int s0 = min(w.sink_start + c0 * KT, w.sink_end), s1 = min(w.sink_start + c1 * KT, w.sink_end);
  const int w0 = w.start + max(c0 - w.sink_tiles, 0) * KT;
  const int w1 = min(w.start + max(c1 - w.sink_tiles, 0) * KT, w.end);
  float* q_s = reinterpret_cast<float*>(mine);
  for (int r = wave; r < ROWS && row0 + r < w.rows; r += WAVES) {
    int lo_r, hi_r, sink;
    w.seen(a, row0 + r, lo_r, hi_r, sink);
    const T* q = static_cast<const T*>(a.q) + (w.q0 + w.token(row0 + r)) * a.q_row + w.head(row0 + r) * a.q_head;
    float m_r, l_r, o_r[4];
    attend_row(a, q, kr, vr, lo_r, hi_r, sink, s0, s1, w0, w1, q_s, m_r, l_r, o_r);
    const int64_t item = item_of(row0 + r), at = part * a.rows() + item;
    if (splits > 1 && lane == 0) {
      a.part[2 * at] = l_r == 0.f ? -__builtin_inff() : m_r;
      a.part[2 * at + 1] = l_r;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int d = lane + u * kWave;
      if (d >= a.dim) continue;
      if (splits > 1) a.part[a.part_values(splits) + at * a.dim + d] = o_r[u];
      else static_cast<T*>(a.out)[item * a.dim + d] = from_f32<T>(l_r == 0.f ? 0.f : o_r[u] / l_r);
    }
  }
}

template <typename T, int DP, int NR, bool ALIGNED>
__global__ void __launch_bounds__(kWave* cache_waves(DP * sizeof(T)), few_per_simd(NR * DP))
    cache_few_kernel(CacheArgs a, CacheCut prefix, CacheCut own, int splits) {
  extern __shared__ __align__(16) char lds[];
  const uint32_t prefix_blocks = prefix.tiles * a.k_heads * prefix.splits;
  const bool is_prefix = blockIdx.x < prefix_blocks;
  cache_few<T, DP, NR, ALIGNED>(a, is_prefix ? prefix : own, is_prefix, splits,
                                blockIdx.x - (is_prefix ? 0 : prefix_blocks), lds);
}

// Tiles of K and V for attend_walk, from pages.  Rows of a tile that no query sees
// are those nearest to them again.
template <typename T, int DP, int KB, int WAVES, bool ALIGNED>
struct PagedTiles {
  static constexpr int TILE = 32 * KB * DP * (int)sizeof(T), KT = 32 * KB, BUFFERS = many_buffers(DP * sizeof(T));
  using K = Stager<T, DP, KB, WAVES, ALIGNED, false>;
  using V = Stager<T, DP, KB, WAVES, ALIGNED, true>;
  // rows that an instruction of the workgroup brings
  static constexpr int UNIT = K::SAME ? K::THREADS / K::CH : KT;
  static constexpr int LOADS = ALIGNED ? K::ROUNDS + V::ROUNDS : 0;
  static_assert((BUFFERS - 2) * LOADS <= 63, "the wait counts to 63");
  // (2 x 2048 rows over 32k keys, heads of 128, bf16: 1153 us, 1199 with the branch;
  // 1-2% slower for heads of 64, and those of 256 have no registers left)
  static constexpr bool STRAIGHT = kIs16<T> && DP == 128;
  static constexpr bool WIDE_PARTS = true;
  K k;
  V v;
  const CacheArgs* args;
  PageIds ids;
  const int32_t* table;
  int start, first;  // the window's first tile, and the first row of it that is seen
  __device__ __forceinline__ void begin(const CacheArgs& a, const CacheWalk& w, int lo_first, int wave) {
    args = &a, table = w.table();
    k.begin(static_cast<const T*>(a.k) + w.hk * a.k_at.head, a.k_at.row, a.dim, wave);
    v.begin(static_cast<const T*>(a.v) + w.hk * a.v_at.head, a.v_at.row, a.dim, wave);
    ids.begin(table, w.entries(), a.pages.pages);
    start = w.start, first = w.first_seen(lo_first);
  }
  // (where chunks are left out, a wave may have fewer loads)
  __device__ bool counted() const { return k.dim >= DP; }
  __device__ __forceinline__ void clear(char* tile) const {
    k.clear(tile);
    v.clear(tile + TILE);
  }
  __device__ __forceinline__ void load(char* tile, int j0, int end) {
    const PageTable& t = args->pages;
    const int j_first = j0 == start ? first : j0, j_last = min(j0 + KT, end) - 1;
    auto page_of = [&](int j) { return __builtin_amdgcn_readfirstlane(t.page_of(j)); };
    const int p_first = page_of(j_first), p_last = page_of(j_last);
    ids.seek(p_first, p_last);
    const uint32_t k_place = k.place(tile), v_place = v.place(tile + TILE);
    if (ALIGNED && j_first == j0 && j_last == j0 + KT - 1 && k.dim >= DP) {
      auto row_at = [&](int j, int p, const T*& kp, const T*& vp) {
        const int64_t id = __builtin_amdgcn_readlane(ids.id, p - ids.from), r = j - p * t.page_rows;
        kp = k.src + id * args->k_at.page + r * k.stride;
        vp = v.src + id * args->v_at.page + r * v.stride;
      };
      if (p_first == p_last) {
        const T* kp;
        const T* vp;
        row_at(j0, p_first, kp, vp);
        k.load_whole(k_place, kp);
        v.load_whole(v_place, vp);
        return;
      }
      if constexpr (K::SAME)
        if (t.page_rows % UNIT == 0 && j0 % UNIT == 0) {
#pragma unroll
          for (int i = 0; i < K::ROUNDS; ++i) {
            const T* kp;
            const T* vp;
            row_at(j0 + i * UNIT, page_of(j0 + i * UNIT), kp, vp);
            load_to_lds(kp, k.offset[0], k_place + i * WAVES * 1024);
            load_to_lds(vp, v.offset[0], v_place + i * WAVES * 1024);
          }
          return;
        }
    }
#pragma unroll 2
    for (int i = 0; i < K::ROUNDS; ++i) {
      const int j = min(max(j0 + K::row(k.slot(i)), j_first), j_last), p = static_cast<int>(t.page_of(j));
      const int64_t id = __shfl(ids.id, p - ids.from, kWave), r = j - p * t.page_rows;
      const T* kp = k.src + id * args->k_at.page + r * k.stride;
      const T* vp = v.src + id * args->v_at.page + r * v.stride;
      if constexpr (ALIGNED) {
        if (k.in(i)) load_to_lds_from(kp + K::chunk(k.slot(i)) * kPer16<T>, k_place + i * WAVES * 1024);
        if (v.in(i)) load_to_lds_from(vp + V::chunk(v.slot(i)) * kPer16<T>, v_place + i * WAVES * 1024);
      } else {
        k.load_chunk(tile, kp, i);
        v.load_chunk(tile + TILE, vp, i);
      }
    }
  }
  __device__ PagedRows<T> k_rows() const { return {k.src, args->k_at.page, k.stride, table, &args->pages}; }
  __device__ PagedRows<T> v_rows() const { return {v.src, args->v_at.page, v.stride, table, &args->pages}; }
};

// Many query rows: attend_walk's tiles, over pages.  lds: as attend_kernel's.  Bound
// as attend_walk is, by vector instructions and products that overlap little: 2 x
// 2048 rows over 32k keys, 16 heads on 4, bf16, 1123 us with heads of 128 (0.90
// PFLOP/s; a library product's rate on this card 1.13), 619 us with heads of 64 (0.82).
template <typename T, int DP, int RB, int KB, bool ALIGNED>
__device__ __forceinline__ void cache_many(const CacheArgs& a, const CacheCut& cut, bool is_prefix, int splits,
                                           char* lds) {
  constexpr int ROWS = 32 * RB * 4, KT = 32 * KB;
  using Tiles = PagedTiles<T, DP, KB, 4, ALIGNED>;
  if (splits == 1) {  // (the join does it otherwise)
    int64_t first, last;
    sample_rows(a, first, last);
    if (first > 0 || last < a.n_q)
      zero_outside(static_cast<T*>(a.out), (int64_t)a.q_heads * a.dim, first, last, a.n_q);
  }
  // Tiles that walk the same keys next to each other on one XCD (workgroups go
  // round the eight in turn), so that its L2 reads them once.  The tiles that
  // there are, not those that there might be, are shared out evenly: one more
  // than an XCD holds at once and all wait for it (8k rows, 16 heads on 4: 317 us,
  // with 65 for 64 places 467).
  CacheWalk w;
  w.group = a.q_heads / a.k_heads;
  const uint32_t there = is_prefix ? cut.tiles : min(count_tiles(a, w.group, ROWS), (int64_t)cut.tiles);
  const uint32_t units = there * a.k_heads;
  // Of the host's parts as many as make the fewest rounds of them (a_cu: a CU's).
  int parts = is_prefix ? cut.splits : 1;
  uint32_t a_cu = (units + 255) / 256;
  for (int n = 2; n <= cut.splits && !is_prefix; ++n) {
    const uint32_t next = (units * n + 255) / 256, per_cu = many_per_cu(DP * sizeof(T), RB);
    if ((next + per_cu - 1) / per_cu * parts < (a_cu + per_cu - 1) / per_cu * n) parts = n, a_cu = next;
  }
  const uint32_t blocks = units * parts, per = (blocks + 7) / 8;
  uint32_t id = blockIdx.x / 8 < per ? (blockIdx.x % 8) * per + blockIdx.x / 8 : blockIdx.x;
  if (id >= units * cut.splits) return;
  const bool idle = id >= blocks;  // a part that is not made says so
  if (idle) id -= blocks;
  const uint32_t rest = id / there;
  const int split = static_cast<int>(idle ? parts + rest / a.k_heads : rest % parts);
  w.hk = static_cast<int>(idle ? rest % a.k_heads : rest / parts);
  w.split = cut.first_split + split;
  w.splits = splits;
  int from, to;
  if (!w.begin(a, is_prefix, ROWS, static_cast<int>(id % there), from, to)) return;
  if (idle) {
    for (uint32_t r = w.row0 + threadIdx.x; r < w.row0 + ROWS && r < w.rows; r += kWave * 4) {
      const int64_t at = w.split * a.rows() + (w.q0 + w.token(r)) * a.q_heads + w.head(r);
      a.part[2 * at] = -__builtin_inff();
      a.part[2 * at + 1] = 0.f;
    }
    return;
  }
  int lo_first = 0, hi_first, lo_last, hi_last = to;
  // (the rows of all samples: every key of the prefix, most of them see it whole.  In
  // a window they walk it whole too: 64 samples of one row behind 32k shared keys, 16
  // heads on 4 of 64, a window of 4096, 45 us, without a shared prefix 31)
  if (!is_prefix) w.bounds(a, w.row0, w.row0 + ROWS - 1, lo_first, hi_first, lo_last, hi_last);
  const int tiles = w.place(lo_first, hi_last, from, to, KT, a.pages.page_rows % Tiles::UNIT == 0 ? KT : 1);
  const int each = (tiles + parts - 1) / parts;
  w.t0 = min(split * each, tiles);
  w.t1 = min(w.t0 + each, tiles);
  Tiles kv;
  kv.begin(a, w, lo_first, __builtin_amdgcn_readfirstlane(threadIdx.x / kWave));
  attend_walk<T, DP, RB, KB, 4>(a, w, kv, lds);
}

template <typename T, int DP, int RB, int KB, bool ALIGNED>
__global__ void __launch_bounds__(kWave * 4, many_per_simd(DP, many_per_cu(DP * sizeof(T), RB)))
    cache_tile_kernel(CacheArgs a, CacheCut cut, int is_prefix, int splits) {
  extern __shared__ __align__(16) char lds[];
  cache_many<T, DP, RB, KB, ALIGNED>(a, cut, is_prefix, splits, lds);
}

// Many rows against the prefix and few against each sample's own keys, side by
// side: either leaves CUs idle while it begins and ends (64 samples, 32k keys for
// all and 1000 of their own: 27 and 15 us one after the other).
template <typename T, int DP, int NR, bool ALIGNED>
__global__ void __launch_bounds__(kWave * 4, 2)
    cache_both_kernel(CacheArgs a, CacheCut prefix, CacheCut own, int splits, int prefix_blocks) {
  extern __shared__ __align__(16) char lds[];
  if ((int)blockIdx.x < prefix_blocks)
    cache_many<T, DP, 1, many_key_blocks(DP * sizeof(T)), ALIGNED>(a, prefix, true, splits, lds);
  else
    cache_few<T, DP, NR, ALIGNED>(a, own, false, splits, blockIdx.x - prefix_blocks, lds);
}
// Where both fit a CU twice.
template <typename T>
constexpr bool cache_both(int dp) {
  return dp * (int)sizeof(T) <= 128 && cache_waves(dp * sizeof(T)) == 4;
}

template <typename T, int DP>
constexpr int many_lds() {
  constexpr int RB = DP * sizeof(T), KB = many_key_blocks(RB);
  return many_buffers(RB) * 2 * 32 * KB * RB + 4 * DP * 4 + KB * 4;
}
template <typename T, int DP, int NR>
constexpr int few_lds() {
  constexpr int RB = DP * sizeof(T);
  return cache_waves(RB) * (cache_buffers(RB) * cache_tile(RB) + 16 * NR * 8 + 4);
}

template <typename T, int DP, int RB, bool ALIGNED>
int launch_many(const CacheArgs& a, const CacheCut& c, bool is_prefix, int splits, hipStream_t s) {
  constexpr int KB = many_key_blocks(DP * sizeof(T)), bytes = many_lds<T, DP>();
  auto kernel = &cache_tile_kernel<T, DP, RB, KB, ALIGNED>;
  if (bytes > 65536)
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void*>(kernel), bytes)) return rc;
  const int64_t blocks = align_up((int64_t)c.tiles * a.k_heads * c.splits, 8);
  TSC_REQUIRE(blocks * kWave * 4 < (1ll << 32), "cache_attention: too many tiles");
  kernel<<<static_cast<unsigned>(blocks), kWave * 4, bytes, s>>>(a, c, is_prefix, splits);
  TSC_LAUNCH_CHECK("cache_attention");
  return 0;
}

template <typename T, int DP, int NR, bool ALIGNED>
int launch_few(const CacheArgs& a, const CachePlan& p, hipStream_t s) {
  constexpr int WAVES = cache_waves(DP * sizeof(T)), bytes = few_lds<T, DP, NR>();
  auto kernel = &cache_few_kernel<T, DP, NR, ALIGNED>;
  if (bytes > 65536)
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void*>(kernel), bytes)) return rc;
  const CacheCut prefix = p.prefix.wave_rows ? CacheCut{} : p.prefix, own = p.own.wave_rows ? CacheCut{} : p.own;
  const int64_t blocks = ((int64_t)prefix.tiles * prefix.splits + (int64_t)own.tiles * own.splits) * a.k_heads;
  TSC_REQUIRE(blocks * kWave * WAVES < (1ll << 32), "cache_attention: too many tiles");
  kernel<<<static_cast<unsigned>(blocks), kWave * WAVES, bytes, s>>>(a, prefix, own, p.splits());
  TSC_LAUNCH_CHECK("cache_attention");
  return 0;
}

template <typename T, int DP, int NR, bool ALIGNED>
int launch_both(const CacheArgs& a, const CachePlan& p, hipStream_t s) {
  constexpr int bytes = std::max(many_lds<T, DP>(), few_lds<T, DP, NR>());
  auto kernel = &cache_both_kernel<T, DP, NR, ALIGNED>;
  if (bytes > 65536)
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void*>(kernel), bytes)) return rc;
  const int64_t first = align_up((int64_t)p.prefix.tiles * a.k_heads * p.prefix.splits, 8);
  const int64_t blocks = first + (int64_t)p.own.tiles * a.k_heads * p.own.splits;
  TSC_REQUIRE(blocks * kWave * 4 < (1ll << 32), "cache_attention: too many tiles");
  kernel<<<static_cast<unsigned>(blocks), kWave * 4, bytes, s>>>(a, p.prefix, p.own, p.splits(),
                                                                 static_cast<int>(first));
  TSC_LAUNCH_CHECK("cache_attention");
  return 0;
}

// The join for few parts: a wave per row, VALUES / 4 lanes for its values and as
// many parts at a time as that leaves room for.  (16k rows of 7 parts: a
// workgroup per row 25 us.)
constexpr int kFewParts = 16;

template <typename T, int LANES, int GROUPS>
__device__ __forceinline__ void join_row(const AttendArgs& a, int splits, int64_t item, int64_t step, int lane, int d) {
  const float* ml = a.part + 2 * item;
  const float* o = a.part + a.part_values(splits) + item * a.dim + d;
  float m = -__builtin_inff(), l = 0.f;
  f32x4 sum = f32x4(0.f);
#pragma unroll 4
  for (int s = lane / LANES; s < splits; s += GROUPS) {
    const float ms = ml[2 * s * step], ls = ml[2 * s * step + 1];
    f32x4 x = f32x4(0.f);
    const float* p = o + s * step * a.dim;
    if (d + 4 <= a.dim) __builtin_memcpy(&x, p, 16);
    else
      for (int i = 0; i < 3; ++i) x[i] = d + i < a.dim ? p[i] : 0.f;
    if (ls == 0.f) continue;  // (a part that saw nothing has no values)
    const float m_new = fmaxf(m, ms);
    const float f = m == -__builtin_inff() ? 0.f : exp2f(m - m_new), g = exp2f(ms - m_new);
    m = m_new, l = f * l + g * ls, sum = f * sum + g * x;
  }
#pragma unroll
  for (int x = LANES; x < kWave; x <<= 1) {
    const float mx = __shfl_xor(m, x, kWave), lx = __shfl_xor(l, x, kWave), m_new = fmaxf(m, mx);
    const float f = l == 0.f ? 0.f : exp2f(m - m_new), g = lx == 0.f ? 0.f : exp2f(mx - m_new);
    f32x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __shfl_xor(sum[i], x, kWave);
    m = m_new, l = f * l + g * lx;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = f * sum[i] + g * y[i];
  }
  if (lane >= LANES) return;
  int64_t first, last;
  sample_rows(a, first, last);
  // (a row of no sample has no parts: what was read for it means nothing)
  const bool none = l == 0.f || item < first * a.q_heads || item >= last * a.q_heads;
  T* out = static_cast<T*>(a.out) + item * a.dim;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (d + i < a.dim) out[d + i] = from_f32<T>(none ? 0.f : sum[i] / l);
}

template <typename T, int VALUES>
__global__ void __launch_bounds__(256) cache_join_kernel(AttendArgs a, int splits) {
  constexpr int LANES = VALUES / 4, GROUPS = kWave / LANES;
  const int64_t step = a.rows();
  const int lane = threadIdx.x % kWave, c = lane % LANES, d = 4 * c;
  for (int64_t item = blockIdx.x * (int64_t)4 + threadIdx.x / kWave; item < step; item += gridDim.x * (int64_t)4)
    join_row<T, LANES, GROUPS>(a, splits, item, step, lane, d);
}

template <typename T>
int launch_parts(const AttendArgs& a, int splits, hipStream_t s) {
  // (a launch holds fewer than 2^32 threads)
  if (splits > kFewParts && a.rows() < (1 << 20)) return launch_join<T>(a, splits, s);
  const unsigned blocks = static_cast<unsigned>(std::min<int64_t>(ceil_div(a.rows(), 4), 1 << 22));
  if (a.dim <= 64) cache_join_kernel<T, 64><<<blocks, 256, 0, s>>>(a, splits);
  else if (a.dim <= 128) cache_join_kernel<T, 128><<<blocks, 256, 0, s>>>(a, splits);
  else cache_join_kernel<T, 256><<<blocks, 256, 0, s>>>(a, splits);
  TSC_LAUNCH_CHECK("cache_attention_join");
  return 0;
}

// f<NR>() for the plan's rows of a tile, of those that there are.
template <int MOST, typename F>
int with_row_blocks(int row_blocks, F&& f) {
  if constexpr (MOST >= 4)
    if (row_blocks == 4) return f(std::integral_constant<int, 4>{});
  if constexpr (MOST >= 2)
    if (row_blocks == 2) return f(std::integral_constant<int, 2>{});
  return f(std::integral_constant<int, 1>{});
}

template <typename T, int DP, bool ALIGNED>
int launch_rows(const CacheArgs& a, const CachePlan& p, hipStream_t s) {
  constexpr int MOST = cache_row_blocks(DP * sizeof(T));
  const bool few = !p.own.wave_rows || (p.prefix.splits && !p.prefix.wave_rows);
  if (!p.own.wave_rows && p.prefix.wave_rows == 1 && cache_both<T>(DP))
    return with_row_blocks<MOST>(p.row_blocks, [&](auto nr) {
      if constexpr (cache_both<T>(DP)) return launch_both<T, DP, nr, ALIGNED>(a, p, s);
      return 0;
    });
  for (const CacheCut* c : {&p.prefix, &p.own}) {
    if (!c->splits || !c->wave_rows) continue;
    int rc = 0;
    if constexpr (can_pair(DP, sizeof(T)))
      if (c->wave_rows == 2) rc = launch_many<T, DP, 2, ALIGNED>(a, *c, c == &p.prefix, p.splits(), s);
    if (c->wave_rows == 1) rc = launch_many<T, DP, 1, ALIGNED>(a, *c, c == &p.prefix, p.splits(), s);
    if (rc) return rc;
  }
  if (!few) return 0;
  return with_row_blocks<MOST>(p.row_blocks, [&](auto nr) { return launch_few<T, DP, nr, ALIGNED>(a, p, s); });
}

template <typename T, bool ALIGNED>
int launch_dims(const CacheArgs& a, const CachePlan& p, hipStream_t s) {
  switch (padded_dim(a.dim)) {
    case 32: return launch_rows<T, 32, ALIGNED>(a, p, s);
    case 64: return launch_rows<T, 64, ALIGNED>(a, p, s);
    case 96: return launch_rows<T, 96, ALIGNED>(a, p, s);
    case 128: return launch_rows<T, 128, ALIGNED>(a, p, s);
    default: return launch_rows<T, 256, ALIGNED>(a, p, s);
  }
}

}  // namespace

template <typename T>
int launch_cache(const CacheArgs& a, const CachePlan& p, hipStream_t s) {
  const int64_t e = kPer16<T>;
  // 16-byte pieces at 16-byte addresses, rows of a tile within 32-bit offsets
  auto whole = [&](const void* base, const PageStrides& at) {
    return at.row >= 0 && at.row < (1 << 24) && at.row % e == 0 && at.page % e == 0 && at.head % e == 0 &&
           reinterpret_cast<uintptr_t>(base) % 16 == 0;
  };
  const bool aligned = a.dim % e == 0 && whole(a.k, a.k_at) && whole(a.v, a.v_at);
  if (int rc = aligned ? launch_dims<T, true>(a, p, s) : launch_dims<T, false>(a, p, s)) return rc;
  return p.splits() > 1 ? launch_parts<T>(a, p.splits(), s) : 0;
}

}  // namespace tsc
