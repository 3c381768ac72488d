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

}  // namespace tsc
