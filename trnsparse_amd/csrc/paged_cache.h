// A key and value cache in pages, as the kernels over it see it
// (paged_attention.hip, paged_cache.hip, paged_evict.hip).
//
// K and V pages are (pages, kv_heads, page_size, head_dim); row j of sequence b
// is row j % page_size of page table[b][j / page_size]. A table entry outside
// [0, pages) is a page of zeros that cannot be written: what the table holds is
// data of the device that the host does not see, so every lookup checks it.
// Page sizes are whole numbers of 16 rows: a piece of 16 rows lies in one page.
#pragma once

#include "common.h"

namespace tsp {
namespace paged {

constexpr int PIECE = 16;  // rows
constexpr uint32_t NO_PAGE = 0xffffffffu;

struct Table {
  const void* p;
  int64_t ld;      // entries between rows
  int64_t pages;   // below 2^31
  int wide;        // 1: entries are int64 (0: int32)
  int cols;
  int page_size;
  uint64_t recip;  // ceil(2^32 / (page_size / PIECE))
};
struct Pages {
  char* p;
  int64_t page, h, s;  // strides in bytes: page, head, row
};
// lengths of cached rows and of new ones (null: all of `most`) of each sequence, each of
// int64 (`wide`) or int32
struct Lengths {
  const void *p, *fresh;
  int wide, fresh_wide;
  int64_t slots, most;
};

// Loads from memory that no kernel of the launch writes, at an address that is
// the same for the whole wavefront: scalar loads, which the counters of the
// direct loads into LDS do not see.
template <typename I>
__device__ inline I load_const(const void* p, int64_t i) {
  return *(const __attribute__((address_space(4))) I*)(uintptr_t)((const I*)p + i);
}
__device__ inline int64_t index_at(const void* p, int wide, int64_t i) {
  return wide ? load_const<int64_t>(p, i) : (int64_t)load_const<int32_t>(p, i);
}
__device__ inline int64_t clamped(int64_t v, int64_t most) { return v < 0 ? 0 : v > most ? most : v; }
__device__ inline int64_t cached_rows(const Lengths& a, int64_t b) {
  return clamped(index_at(a.p, a.wide, b), a.slots);
}
__device__ inline int64_t new_rows(const Lengths& a, int64_t b) {
  return a.fresh ? clamped(index_at(a.fresh, a.fresh_wide, b), a.most) : a.most;
}

// The column of piece `i` (16 rows): i / (page_size / 16), by the reciprocal. Exact as
// long as slots * page_size is below 2^40 (checked by the host): with d = page_size / 16
// and recip = (2^32 + e) / d, e < d, the quotient is off by i e / (d 2^32) < 1 / d.
__device__ inline uint32_t column_of(const Table& t, uint32_t i) { return (uint32_t)((i * t.recip) >> 32); }
// The page of column `col` in the row of the table that starts at entry `row`.
__device__ inline uint32_t page_at(const Table& t, int64_t row, uint32_t col) {
  const int64_t id = index_at(t.p, t.wide, row + col);
  return id >= 0 && id < t.pages ? (uint32_t)id : NO_PAGE;
}
// The same where the lanes of a wavefront ask for different columns: an entry's
// halves as they are (int32 entries: the entry twice), and what page they name.
// Both without a branch, which would wait for other loads in flight.
__device__ inline u32x2 entry_of_lane(const Table& t, int64_t row, uint32_t col) {
  const uint32_t* p = (const uint32_t*)t.p + ((row + col) << t.wide);
  return u32x2{p[0], p[t.wide]};
}
__device__ inline uint32_t page_of_entry(const Table& t, u32x2 e) {
  const uint32_t bad = (uint32_t)(e.x >= (uint32_t)t.pages) | ((uint32_t)t.wide & (uint32_t)(e.y != 0));
  return e.x | (0u - bad);
}
__device__ inline uint32_t page_of_lane(const Table& t, int64_t row, uint32_t col) {
  return page_of_entry(t, entry_of_lane(t, row, col));
}

// Sum over the lanes before this one, and the total of the wavefront: within rows of
// 16 lanes by shifts, then the rows' totals to those behind them.
__device__ inline int wave_scan(int v, int& total) {
  int x = v;
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // lane 15 of a row to the next row, rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31 to rows 2 and 3
  total = __builtin_amdgcn_readlane(x, 63);
  return x - v;
}

// ------------------------------------------------------------------- host

inline int esize(int dtype) { return dtype == TSP_F32 ? 4 : 2; }

// Checks of a cache's sizes, pages and table; 0 or a status with a message.
int check_cache(const char* who, int dtype, int64_t batch, int64_t kv_heads, int64_t pages, int64_t page_size,
                int64_t head_dim, const void* table, int table_type, int64_t table_stride, int64_t columns);
// (`written`: the kernels write them, so their rows may not overlap)
int check_pages(const char* who, const char* name, const void* p, const int64_t* strides, int dtype, int64_t pages,
                int64_t kv_heads, int64_t page_size, int64_t head_dim, bool written);
int check_lengths(const char* who, int64_t batch, const void* lengths, int index_type, bool has_new);
int check_lengths_out(const char* who, int64_t batch, const void* out, const Lengths& l);
int check_weights(const char* who, const void* weights, const int64_t* strides, int64_t batch, int64_t kv_heads,
                  int64_t slots);

inline Table table_of(const void* table, int table_type, int64_t table_stride, int64_t columns, int64_t pages,
                      int64_t page_size) {
  const uint64_t d = (uint64_t)(page_size / PIECE);
  return Table{table, table_stride, pages, table_type == TSP_I64, (int)columns, (int)page_size,
               ((uint64_t(1) << 32) + d - 1) / d};
}
inline Lengths lengths_of(const void* lengths, const void* fresh, int index_type, int64_t slots, int64_t most) {
  const int wide = (index_type & ~TSP_NEW_OTHER) == TSP_I64;
  return Lengths{lengths, fresh, wide, index_type & TSP_NEW_OTHER ? !wide : wide, slots, most};
}
inline Pages pages_of(const void* p, const int64_t* s, int dtype) {
  const int64_t e = esize(dtype);
  return Pages{(char*)p, s[0] * e, s[1] * e, s[2] * e};
}

}  // namespace paged
}  // namespace tsp
