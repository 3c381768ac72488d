// Where the rows that a sample keeps lie: pages of R rows each, in any order,
// and per sample the numbers of its pages (row b of the table).  Position t of
// sample b is row t % R of page table[b][t / R].
#pragma once

#include "common.hpp"

namespace tsc {

struct PageStrides {  // in elements
  int64_t page, row, head;
  __device__ __forceinline__ int64_t at(int64_t p, int64_t r, int64_t h) const { return p * page + r * row + h * head; }
};

struct PageTable {
  const int32_t* table = nullptr;
  int64_t table_row = 0;
  int32_t table_pages = 0;  // entries of a row of the table
  const int32_t* lengths = nullptr;
  int32_t samples = 0;
  int32_t pages = 0, page_rows = 1;
  // position / page_rows without a division: (umulhi(t, multiplier) + (t & whole)) >> shift
  // for t < 2^31, with whole all ones for pages of one row
  uint32_t multiplier = 0, whole = 0;
  int32_t shift = 0;

  // Positions that a row of the table has room for.
  __host__ __device__ int64_t most() const { return (int64_t)table_pages * page_rows; }
  __host__ __device__ __forceinline__ uint32_t page_of(uint32_t t) const {
    return (static_cast<uint32_t>(static_cast<uint64_t>(t) * multiplier >> 32) + (t & whole)) >> shift;
  }

  // A length as far as there is room for it.
  __device__ __forceinline__ int cut(int length) const {
    return static_cast<int>(min(max((int64_t)length, (int64_t)0), most()));
  }
  // The checked arguments of an entry point; 0 or an error code.
  int set(const char* what, const int32_t* table_, int64_t table_row_, int64_t table_pages_, const int32_t* lengths_,
          int32_t samples_, int64_t pages_, int64_t page_rows_) {
    TSC_REQUIRE(samples_ >= 0 && samples_ < 0x7fffffff, "%s: invalid number of samples", what);
    TSC_REQUIRE(pages_ >= 0 && pages_ < (1ll << 31), "%s: invalid number of pages", what);
    TSC_REQUIRE(page_rows_ >= 1 && page_rows_ <= 1 << 20, "%s: pages of %lld rows, 1 to 2^20 are supported", what,
                static_cast<long long>(page_rows_));
    // positions are 32-bit, and a walk looks up to a tile past the last
    TSC_REQUIRE(table_pages_ >= 0 && table_pages_ <= ((1ll << 31) - 1025) / page_rows_,
                "%s: a table row of %lld pages holds over 2^31 - 1025 positions", what,
                static_cast<long long>(table_pages_));
    TSC_REQUIRE(samples_ == 0 || (lengths_ && (table_pages_ == 0 || table_)), "%s: null pointer", what);
    table = table_, table_row = table_row_, table_pages = static_cast<int32_t>(table_pages_);
    lengths = lengths_, samples = samples_, pages = static_cast<int32_t>(pages_);
    page_rows = static_cast<int32_t>(page_rows_);
    // with 2^(l-1) < R <= 2^l, ceil(2^(31+l) / R) / 2^(31+l) is right below 2^31
    int l = 0;
    while ((1 << l) < page_rows) ++l;
    if (l == 0) multiplier = 0, whole = ~0u, shift = 0;
    else multiplier = static_cast<uint32_t>(ceil_div(1ll << (31 + l), page_rows)), whole = 0, shift = l - 1;
    return 0;
  }
};

// The first sample (the last at most) whose end, off[s + 1], is past row t, by the
// whole wave: 64 at a time.
__device__ __forceinline__ int first_past(const int32_t* off, int samples, int64_t t) {
  int from = 0, n = samples;
  while (n > 1) {
    const int step = (n + kWave - 1) / kWave, lane = threadIdx.x % kWave;
    const int s = min(from + (lane + 1) * step, from + n) - 1;  // the last of the lane's
    const uint64_t past = __ballot(off[s + 1] > t);
    const int l = past ? __builtin_ctzll(past) : kWave - 1;
    const int next = min(from + l * step, from + n - 1);
    n = min(step, from + n - next);
    from = next;
  }
  return from;
}

// The samples at[x] of N rows t[x] a lane, all from t_first to t_last, with their
// ends and lengths (as they are in `lengths`), by the whole wave: the sample of
// the first row, then how many samples' ends each row is past.
template <int N>
__device__ __forceinline__ void samples_of(const int32_t* off, const int32_t* lengths, int samples, int64_t t_first,
                                           int64_t t_last, const int64_t t[N], int at[N], int end[N], int length[N]) {
  const int lane = threadIdx.x % kWave;
  const int s0 = samples <= kWave ? 0 : first_past(off, samples, t_first);
#pragma unroll
  for (int x = 0; x < N; ++x) at[x] = s0;
  const int mine = min(s0 + lane, samples - 1);
  int ends = off[mine + 1], s = s0;
  const int length_mine = lengths[mine];
  for (;;) {
    int k = 0;
    for (; k < kWave && s + k < samples - 1; ++k) {
      const int e = __builtin_amdgcn_readlane(ends, k);
      if (e > t_last) break;
#pragma unroll
      for (int x = 0; x < N; ++x) at[x] += t[x] >= e;
    }
    if (k < kWave) break;
    s += kWave;
    ends = off[min(s + lane, samples - 1) + 1];
  }
#pragma unroll
  for (int x = 0; x < N; ++x) {
    end[x] = s == s0 ? __shfl(ends, at[x] - s0, kWave) : off[at[x] + 1];
    length[x] = s == s0 ? __shfl(length_mine, at[x] - s0, kWave) : lengths[at[x]];
  }
}

}  // namespace tsc
