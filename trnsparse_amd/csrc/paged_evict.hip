// Eviction from a key and value cache in pages: a sequence of more than `budget`
// rows keeps, per key head, its last `recent` rows and of the others the budget -
// recent with the largest accumulated weights, moved to rows [0, budget) in their
// order. No counterpart in the reference, whose attention takes one sequence's K
// and V whole (trnsparse/ops.py:549-625).
//
// A unit is one (sequence, key head) pair. Its weights are ranked by keys: unsigned
// numbers in their order, NaN above all, one zero. Selecting finds the key of the
// last row that stays, by histograms of digits of 11, 11 and 10 bits (fewer where all
// rows with the digits so far stay), and lists the kept rows in order.
//   select_kernel   one workgroup to a unit does it all; rows of up to one part
//                   stay in its registers
//   digit and list kernels (few units of many rows): a workgroup to a part of 8192
//                   rows, the histograms of a unit's parts added up by whoever needs them
// move_kernel then moves the listed rows of K and V. A row goes to a place at or
// before its own, and the list rises: a workgroup that takes the list in order, and
// writes a part only once all of its rows are read, never writes over a row that is
// still to be read. Workgroups share no byte: each has one unit's K or V, a slice of
// its rows' bytes and, in launches of few units, a segment of the places. A row that
// comes from another segment's places could be overwritten before it is read; those
// are copied aside first (save_kernel), the rows from behind the budget never are.
#include "paged_cache.h"

namespace tsp {
namespace paged {
namespace {

struct EvictArgs {
  Pages Kp, Vp;
  Table t;
  Lengths len;
  void* out;
  float* W;
  int64_t wb, wh;
  int64_t units;
  int Hkv, D, esz;
  int budget, recent;
  u32x2* list;     // [unit][budget]: kept rows, page and row of it (and SAVED)
  int32_t* first;  // [unit]: the first kept row that moves
  char* spare;     // 16 bytes that writes to no page go to
  // few units of many rows
  int parts;       // of a unit's rows at most
  int segment;     // log2 of the places of a segment; 31: all are one
  struct Find* state;  // [2][unit]: the search after the first and the second digit
  uint32_t* hist;  // [3][unit][part][BINS]
  int32_t* count;  // [unit][part]: rows that stay whatever the last digit is
  float* kept;     // [unit][budget]: weights; null where they are in place
  char* saved;     // [unit][K, V][budget]: rows
};
constexpr uint32_t SAVED = 0x80000000u;  // with the row's number: the row is taken from `saved`

constexpr int ST = 1024, SPT = 8, PART = ST * SPT, BINS = 2048;  // threads that select, rows of one in a part and all's

__device__ inline uint32_t order_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);  // (one zero)
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A thread's N rows of a part, consecutive ones of one page; rows from `end` on are not read.
template <int N>
struct Part {
  static_assert(PIECE % N == 0, "one page");
  float v[N];
  __device__ inline void load(const float* w, int j, int end, bool aligned) {
    if (aligned && j + N <= end) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const f32x4 x = *(const f32x4*)(w + j + i);
        v[i] = x[0], v[i + 1] = x[1], v[i + 2] = x[2], v[i + 3] = x[3];
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = j + i < end ? w[j + i] : 0.f;
    }
  }
};

// The search for the key of the last row that stays: among the keys from lo on
// that share its digits so far it is the want-th from the largest, and the next
// digit begins at bit `shift`. Done: the rows of keys above `last` stay, and of
// those equal to it the first `equal` ones.
struct Find {
  uint32_t lo, last;
  int shift, want, equal, done;
  __device__ inline void start(int keep) {
    lo = 0, shift = 21, want = keep, equal = 0, last = 0xffffffffu;
    done = keep == 0;  // (no key is above a NaN's)
  }
  __device__ inline bool has(uint32_t k) const {
    return k >= lo && k - lo <= (shift == 21 ? 0xffffffffu : shift == 10 ? (1u << 21) - 1 : (1u << 10) - 1);
  }
};
struct Scratch {
  int sums[2][ST / 64];
  uint32_t pick[3];
  int first;
};
template <int N>
__device__ inline void add_digits(uint32_t* hist, const Find& f, const Part<N>& p, int j, int end) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t k = order_key(p.v[i]);
    if (j + i < end && f.has(k)) atomicAdd(&hist[(k - f.lo) >> f.shift], 1u);
  }
}
// The next digit, from the counts c0 and c1 of digits BINS - 1 - 2 tid and the one
// below: the one in which the count from the largest passes `want`.
__device__ inline void next_digit(Find& f, int c0, int c1, Scratch& x) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, d = BINS - 1 - 2 * tid;
  int total, before = wave_scan(c0 + c1, total);
  if (lane == 0) x.sums[0][wave] = total;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ST / 64; ++i) before += i < wave ? x.sums[0][i] : 0;
  if (before < f.want && f.want <= before + c0 + c1) {
    const bool second = f.want > before + c0;
    x.pick[0] = (uint32_t)(second ? d - 1 : d);
    x.pick[1] = (uint32_t)(f.want - before - (second ? c0 : 0));
    x.pick[2] = (uint32_t)(second ? c1 : c0);
  }
  __syncthreads();
  f.want = (int)x.pick[1];
  f.lo += x.pick[0] << f.shift;
  if (f.want == (int)x.pick[2]) {  // all with this digit stay
    f.last = f.lo - 1;             // (no key is zero: it would be a NaN's)
    f.done = 1;
  } else if (f.shift == 0) {
    f.last = f.lo;
    f.equal = f.want;
    f.done = 1;
  }
  f.shift = f.shift > 10 ? 10 : 0;
}

struct Unit {
  int64_t unit, b, h;
  int n, E, keep;  // rows, of which the first E may go and `keep` of those stay
  float* w;
  bool aligned, cut;
};
__device__ inline Unit unit_at(const EvictArgs& a, int64_t unit) {
  Unit u;
  u.unit = unit;
  u.b = (uint32_t)unit / (uint32_t)a.Hkv;  // (32 bits: there are at most 2^30)
  u.h = unit - u.b * a.Hkv;
  u.n = (int)cached_rows(a.len, u.b);
  u.cut = u.n > a.budget;
  u.E = u.n - a.recent;
  u.keep = a.budget - a.recent;  // (below E where rows are cut)
  u.w = a.W + u.b * a.wb + u.h * a.wh;
  u.aligned = ((uintptr_t)u.w & 15) == 0;
  return u;
}
__device__ inline void put_length(const EvictArgs& a, const Unit& u) {
  const int v = u.cut ? a.budget : u.n;
  if (u.h == 0 && threadIdx.x == 0) {
    if (a.len.wide)
      ((int64_t*)a.out)[u.b] = v;
    else
      ((int32_t*)a.out)[u.b] = v;
  }
}
// Bits of the thread's rows that are above the last key (or recent), and that equal it.
template <int N>
__device__ inline void sort_out(const Unit& u, const Find& f, const Part<N>& p, int j, uint32_t& above, uint32_t& same) {
  above = same = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t k = order_key(p.v[i]);
    if (j + i < u.n && (j + i >= u.E || k > f.last)) above |= 1u << i;
    if (j + i < u.E && f.equal > 0 && k == f.last) same |= 1u << i;
  }
}
// Page and row of row j (a thread's rows of a part lie in one page).
__device__ inline u32x2 spot_of_row(const EvictArgs& a, const Unit& u, int j) {
  const uint32_t col = column_of(a.t, (uint32_t)j / PIECE), row = (uint32_t)j - col * (uint32_t)a.t.page_size;
  return u32x2{j < u.n ? page_of_lane(a.t, u.b * a.t.ld, col) : NO_PAGE, row};
}
// Lists the part's kept rows behind the `base` kept ones before it, of the rows that
// equal the last key as far as they go (`equal_base` came before); counts on. Their
// weights go to `to`, which may be the weights themselves. `spot`: of row j. Returns
// the first of the thread's rows that goes, n for none: the rows behind it move.
template <int N>
__device__ inline int list_part(const EvictArgs& a, const Unit& u, const Find& f, Part<N>& p, int j, u32x2 spot, float* to,
                                int& base, int& equal_base, int turn, Scratch& x) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t above, same;
  sort_out(u, f, p, j, above, same);
  // both counts in one scan: at most PART of each
  int total, before = wave_scan(__builtin_popcount(same) << 16 | __builtin_popcount(above), total);
  if (lane == 0) x.sums[turn][wave] = total;
  // every row of this part is read before one is written
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(p.v[i]));
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int i = 0; i < ST / 64; ++i) {
    const int c = x.sums[turn][i];
    before += i < wave ? c : 0;
    all += c;
  }
  int e = equal_base + (before >> 16);  // equal ones before this thread's
  const int e0 = equal_base < f.equal ? equal_base : f.equal;
  int d = base + (before & 0xffff) + (e < f.equal ? e : f.equal) - e0, goes = u.n;
  u32x2* list = a.list + u.unit * a.budget;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    bool stays = above >> i & 1;
    if (same >> i & 1) stays = e++ < f.equal;
    const int q = j + i;
    if (!stays && q < goes) goes = q;
    // (weights that another stream writes meanwhile could make more rows stay than there are places)
    if (!stays || d >= a.budget) continue;
    const uint32_t aside = q < a.budget && (q >> a.segment) != (d >> a.segment) && spot.x != NO_PAGE ? SAVED : 0;
    list[d] = u32x2{spot.x, (spot.y + i) | aside};
    if (d != q || to != u.w) to[d] = p.v[i];
    ++d;
  }
  equal_base += all >> 16;
  base += (all & 0xffff) + (equal_base < f.equal ? equal_base : f.equal) - e0;
  return goes;
}

// N 8, or 16 where that keeps all rows in registers.
template <int N>
__global__ __launch_bounds__(ST) void select_kernel(const EvictArgs a) {
  constexpr int PART = ST * N;
  __shared__ uint32_t hist[BINS];
  __shared__ Scratch x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Unit u = unit_at(a, blockIdx.x);
  put_length(a, u);
  if (!u.cut) {
    if (tid == 0) a.first[u.unit] = a.budget;
    return;
  }
  // The rows of up to one part stay in registers; of more, each pass reads them
  // again, two parts ahead of the one that is worked on.
  const int n = u.n;
  const bool once = n <= PART;
  Part<N> held;
  held.load(u.w, tid * N, n, u.aligned);
  const u32x2 held_spot = spot_of_row(a, u, tid * N);
  auto each = [&](int end, auto&& f) {
    Part<N> even = held, odd;
    if (!once) odd.load(u.w, PART + tid * N, n, u.aligned);
    for (int j0 = 0; j0 < end; j0 += 2 * PART) {
      f(j0 + tid * N, even);
      if (once) break;
      even.load(u.w, j0 + 2 * PART + tid * N, n, u.aligned);
      if (j0 + PART < end) f(j0 + PART + tid * N, odd);
      odd.load(u.w, j0 + 3 * PART + tid * N, n, u.aligned);
    }
  };
  Find f;
  f.start(u.keep);
  for (int i = tid; i < BINS; i += ST) hist[i] = 0;
  if (tid == 0) x.first = n;
  __syncthreads();
  while (!f.done) {
    each(u.E, [&](int j, const Part<N>& p) { add_digits(hist, f, p, j, u.E); });
    __syncthreads();
    const int d = BINS - 1 - 2 * tid, c0 = (int)hist[d], c1 = (int)hist[d - 1];
    hist[d] = hist[d - 1] = 0;  // (for the next turn)
    next_digit(f, c0, c1, x);
  }
  __syncthreads();
  int base = 0, equal_base = 0, first = n, turn = 0;
  each(n, [&](int j, Part<N> p) {
    const int goes = list_part(a, u, f, p, j, j < PART ? held_spot : spot_of_row(a, u, j), u.w, base, equal_base, turn, x);
    first = goes < first ? goes : first;
    turn ^= 1;
  });
  // (the lowest lane with one has the wavefront's first)
  const uint64_t some = __builtin_amdgcn_ballot_w64(first < n);
  if (some) {
    const int low = __builtin_amdgcn_readlane(first, __builtin_ctzll(some));
    if (once) {
      if (lane == 0) atomicMin(&x.first, low);
    } else if (first < n) {  // (of several parts, any lane may)
      atomicMin(&x.first, first);
    }
  }
  __syncthreads();
  if (tid == 0) a.first[u.unit] = x.first < a.budget ? x.first : a.budget;
}

// ------------------------------------------------- few units of many rows

// The search after `turn` digits, from the one before and that digit's counts over the unit's
// parts; b0 and b1: the counts of this thread's two digits (next_digit) in the parts before `upto`.
__device__ inline Find find_after(const EvictArgs& a, const Unit& u, int turn, Scratch& x, int upto, int& b0, int& b1) {
  Find f;
  f.start(u.keep);
  b0 = b1 = 0;
  if (turn == 0) return f;
  if (turn > 1) f = a.state[(turn - 2) * a.units + u.unit];
  if (f.done) return f;
  const int parts = (u.E + PART - 1) / PART, d = BINS - 1 - 2 * (int)threadIdx.x;
  const uint32_t* hist = a.hist + ((int64_t)(turn - 1) * a.units + u.unit) * a.parts * BINS + d - 1;
  int c0 = 0, c1 = 0;
  for (int i = 0; i < parts; i += 8) {
    u32x2 c[8];
#pragma unroll
    for (int v = 0; v < 8; ++v) c[v] = *(const u32x2*)(hist + (int64_t)(i + v < parts ? i + v : parts - 1) * BINS);
#pragma unroll
    for (int v = 0; v < 8; ++v) {
      c0 += i + v < parts ? (int)c[v].y : 0;
      c1 += i + v < parts ? (int)c[v].x : 0;
      b0 += i + v < parts && i + v < upto ? (int)c[v].y : 0;
      b1 += i + v < parts && i + v < upto ? (int)c[v].x : 0;
    }
  }
  next_digit(f, c0, c1, x);
  return f;
}

// Counts of the next digit in one part of a unit; in the last turn, of the rows that stay
// whatever the last digit is, too.
__global__ __launch_bounds__(ST) void digit_kernel(const EvictArgs a, int turn) {
  __shared__ uint32_t hist[BINS];
  __shared__ Scratch x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, part = blockIdx.x % (uint32_t)a.parts;
  const Unit u = unit_at(a, blockIdx.x / (uint32_t)a.parts);
  if (turn == 0 && part == 0) put_length(a, u);
  const int end = turn < 2 ? u.E : u.n, j = part * PART + tid * SPT;
  if (!u.cut || part * PART >= end) return;
  Part<SPT> p;
  p.load(u.w, j, u.n, u.aligned);
  int b0, b1;
  const Find f = find_after(a, u, turn, x, 0, b0, b1);
  if (turn > 0 && part == 0 && tid == 0) a.state[(turn - 1) * a.units + u.unit] = f;
  if (turn == 2) {
    Find top = f;
    if (!f.done) top.last = f.lo + (1u << 10) - 1;  // above all keys that are still in question
    uint32_t above, same;
    sort_out(u, top, p, j, above, same);
    int total;
    wave_scan(__builtin_popcount(above), total);
    if (lane == 0) x.sums[1][wave] = total;
    __syncthreads();
    if (tid == 0) {
      int all = 0;
      for (int i = 0; i < ST / 64; ++i) all += x.sums[1][i];
      a.count[u.unit * a.parts + part] = all;
    }
  }
  if (f.done) return;
  for (int i = tid; i < BINS; i += ST) hist[i] = 0;
  __syncthreads();
  add_digits(hist, f, p, j, u.E);
  __syncthreads();
  uint32_t* to = a.hist + (((int64_t)turn * a.units + u.unit) * a.parts + part) * BINS;
  for (int i = tid; i < BINS; i += ST) to[i] = hist[i];
}
__global__ __launch_bounds__(ST) void list_kernel(const EvictArgs a) {
  __shared__ Scratch x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, part = blockIdx.x % (uint32_t)a.parts;
  const Unit u = unit_at(a, blockIdx.x / (uint32_t)a.parts);
  if (part == 0 && tid == 0) a.first[u.unit] = u.cut ? 0 : a.budget;
  const int j = part * PART + tid * SPT;
  if (!u.cut || part * PART >= u.n) return;
  Part<SPT> p;
  p.load(u.w, j, u.n, u.aligned);
  const u32x2 spot = spot_of_row(a, u, j);
  int above = 0;  // of the parts before: rows above the last key, and those that equal it
  for (int i = tid; i < part; i += ST) above += a.count[u.unit * a.parts + i];
  const bool done = a.state[a.units + u.unit].done;
  int b0, b1;
  const Find f = find_after(a, u, 3, x, part, b0, b1);
  int equal = 0;
  if (!done) {
    const int d = BINS - 1 - 2 * tid, last = (int)(f.lo & 1023);
    above += (d > last ? b0 : 0) + (d - 1 > last ? b1 : 0);
    equal = (d == last ? b0 : 0) + (d - 1 == last ? b1 : 0);
    if (f.equal == 0) above += equal, equal = 0;  // (all of them stay)
  }
  int above_w, equal_w;
  wave_scan(above, above_w);
  wave_scan(equal, equal_w);
  __syncthreads();
  if (lane == 0) x.sums[0][wave] = above_w, x.sums[1][wave] = equal_w;
  __syncthreads();
  int base = 0, equal_base = 0;
  for (int i = 0; i < ST / 64; ++i) {
    base += x.sums[0][i];
    equal_base += x.sums[1][i];
  }
  base += equal_base < f.equal ? equal_base : f.equal;
  __syncthreads();
  list_part(a, u, f, p, j, spot, a.kept + u.unit * a.budget, base, equal_base, 0, x);
}

// Copies aside the rows that come from another segment's places, and puts the kept
// weights in theirs: 2^lanes threads to a row (16 bytes each), SU rows to a thread,
// `per` workgroups to a unit's K or V. (8 units of 32768 places, a quarter of their rows
// copied: one row to a thread 30 us, eight 24.)
constexpr int SU = 8;
__global__ __launch_bounds__(256) void save_kernel(const EvictArgs a, uint32_t per, int lanes) {
  const uint32_t at = blockIdx.x % per;
  const int64_t x = blockIdx.x / per, unit = x >> 1, b = (uint32_t)unit / (uint32_t)a.Hkv, h = unit - b * a.Hkv;
  const int step = 256 >> lanes, d0 = (int)at * step * SU + (int)(threadIdx.x >> lanes);
  const int c = 16 * (int)(threadIdx.x & ((1u << lanes) - 1)), row = a.D * a.esz;
  if (a.first[unit] >= a.budget) return;
  u32x2 e[SU];
#pragma unroll
  for (int i = 0; i < SU; ++i) {
    const int d = d0 + i * step;
    e[i] = d < a.budget ? a.list[unit * a.budget + d] : u32x2{NO_PAGE, 0};
    if (a.kept && !(x & 1) && c == 0 && d < a.budget) a.W[b * a.wb + h * a.wh + d] = a.kept[unit * a.budget + d];
  }
  const Pages& p = x & 1 ? a.Vp : a.Kp;
#pragma unroll
  for (int i = 0; i < SU; ++i) {
    const uint32_t r = e[i].y & ~SAVED;
    if ((e[i].y & SAVED) && c < row && e[i].x < (uint32_t)a.t.pages && r < (uint32_t)a.t.page_size)
      *(u32x4*)(a.saved + (x * a.budget + d0 + i * step) * row + c) = *(const u32x4*)(p.p + e[i].x * p.page + h * p.h + r * p.s + c);
  }
}

// ----------------------------------------------------------------- moving

// LPR lanes (16 bytes each) to a row's slice, MU rows of a thread in a part of the
// list. The list's entries come two parts ahead, the rows one, in three sets of
// registers by turns. A thread without a row takes the last one's (and stores the
// same once more), one without a page the spare place, so that no branch keeps a
// wait from being counted.
constexpr int MT = 512, MU = 8;
struct Move {
  u32x2 from[MU];  // page and row
  u32x2 to[MU];    // the table's entry
  u32x4 v[MU];
};
template <int LPR, bool SEGMENTS>
__global__ __launch_bounds__(MT) void move_kernel(const EvictArgs a, uint32_t slices, uint32_t segments) {
  // the slices of a row in consecutive slots of one XCD
  const uint32_t xcd = blockIdx.x & 7, at8 = blockIdx.x >> 3, slice = at8 % slices, y = at8 / slices * 8 + xcd;
  const int64_t x = y / segments, unit = x >> 1;
  if (unit >= a.units) return;
  const int64_t b = (uint32_t)unit / (uint32_t)a.Hkv, h = unit - b * a.Hkv;
  // the places of this workgroup
  const int64_t s0 = (int64_t)(y - (uint32_t)x * segments) << a.segment, s1 = s0 + ((int64_t)1 << a.segment);
  const int first = a.first[unit] > s0 ? a.first[unit] : (int)s0, end = (int)(s1 < a.budget ? s1 : a.budget) - 1;
  if (first > end) return;
  const Pages& p = x & 1 ? a.Vp : a.Kp;
  const u32x2* list = a.list + unit * a.budget;
  const int64_t trow = b * a.t.ld;
  constexpr int RP = MT / LPR, PR = RP * MU;  // rows at once, and of a part
  const uint32_t row_bytes = (uint32_t)(a.D * a.esz);
  uint32_t c = 16 * (LPR * slice + threadIdx.x % LPR);
  c = c < row_bytes ? c : row_bytes - 16;
  char* base = p.p + h * p.h + c;
  const int at = threadIdx.x / LPR;
  auto place = [&](int d0, int u) {
    const int d = d0 + RP * u + at;
    return (uint32_t)(d < end ? d : end);
  };
  // A row's place, or the spare one. What the list holds is checked once more: places
  // that no row went to (as above) hold anything.
  const uint32_t pages = (uint32_t)a.t.pages, rows = (uint32_t)a.t.page_size;
  auto spot = [&](uint32_t page, uint32_t row) {
    const uint64_t none = 0 - (uint64_t)((page >= pages) | (row >= rows));
    const uint64_t there = (uint64_t)(base + (int64_t)(page & ~(uint32_t)none) * p.page + (row & ~(uint32_t)none) * p.s);
    return (u32x4*)((there & ~none) | ((uint64_t)a.spare & none));
  };
  auto look = [&](Move& m, int d0) {
#pragma unroll
    for (int u = 0; u < MU; ++u) {
      const uint32_t d = place(d0, u);
      m.from[u] = list[d];
      m.to[u] = entry_of_lane(a.t, trow, column_of(a.t, d / PIECE));
    }
  };
  auto load = [&](Move& m, int d0) {
#pragma unroll
    for (int u = 0; u < MU; ++u) {
      if constexpr (!SEGMENTS) {
        m.v[u] = *spot(m.from[u].x, m.from[u].y);
        continue;
      }
      const uint64_t aside = 0 - (uint64_t)(m.from[u].y >> 31);
      const uint64_t there = (uint64_t)spot(m.from[u].x, m.from[u].y & ~SAVED);
      const uint64_t kept = (uint64_t)(a.saved + (x * a.budget + place(d0, u)) * row_bytes + c);
      m.v[u] = *(const u32x4*)((there & ~aside) | (kept & aside));
    }
  };
  auto step = [&](Move& now, Move& next, Move& later, int d0) {
    look(later, d0 + 2 * PR);
    load(next, d0 + PR);
    // the rows of this part have arrived in every wavefront before one is written
#pragma unroll
    for (int u = 0; u < MU; ++u) asm volatile("" : "+v"(now.v[u]));
    asm volatile("s_barrier" ::: "memory");
#pragma unroll
    for (int u = 0; u < MU; ++u) {
      const uint32_t d = place(d0, u), r = d - column_of(a.t, d / PIECE) * (uint32_t)a.t.page_size;
      const uint32_t keep = 0u - (uint32_t)(now.from[u].x != NO_PAGE);
      *spot(page_of_entry(a.t, now.to[u]), r) = now.v[u] & keep;
    }
  };
  Move m0, m1, m2;
  look(m0, first);
  look(m1, first + PR);
  load(m0, first);
  for (int d0 = first;; d0 += 3 * PR) {
    step(m0, m1, m2, d0);
    if (d0 + PR > end) break;
    step(m1, m2, m0, d0 + PR);
    if (d0 + 2 * PR > end) break;
    step(m2, m0, m1, d0 + 2 * PR);
    if (d0 + 3 * PR > end) break;
  }
}

// Whether a unit's weights are searched by a workgroup to each part of them: four
// launches, which take less time than one workgroup's turns where these are many and
// the units leave CUs without one. The whole eviction with one workgroup to each unit
// and by parts, us: 8 units of 24576 rows 52 and 56, of 32768 60 and 56, of 49152 71 and
// 56; 32 of 49152 166 and 168; 64 of 65536 174 and 185, of 81920 196 and 197. Every part
// reads all parts' counts, so that the work grows with their square: up to 4096 parts of
// all units (one workgroup to a unit and by parts, a budget of 4096: 32 units of 2^19 rows
// 399 us and 235, of 2^20 741 and 667; 8 units of 2^21 1412 and 661, of 2^22 2773 and 2435;
// one of 2^23 5475 and 1445).
bool by_parts(int64_t units, int64_t slots) {
  return units < 128 && slots > (3 + units / 10) * PART && units * ceil_div(slots, PART) <= 4096;
}
// log2 of the places of a segment, 31 where all are one. Segments for 512 workgroups,
// none of less than 1024 places, where the chains of parts are too few to take the
// memory's rate (64 with slices of 64 bytes) and long: copying rows aside is traffic
// of its own. (8 units, head_dim 128 in 16 bits: 32768 places of 131072 rows 150 us,
// in segments 53 and 25 to copy; 8192 of 16384: 47.6 us and 45.6 the whole eviction.
// 32 units, 8192 of 16384: 69 us, 104 in segments.)
int segment_of(int64_t units, int64_t budget, int64_t row) {
  if (units * 2 * ceil_div(row, 64) > 64 || budget <= 8192) return 31;
  int s = 10;
  while (s < 31 && (int64_t(1) << s) * ceil_div(512, units * 2 * ceil_div(row, 128)) < budget) ++s;
  return s;
}
struct Space {  // of the workspace, in bytes from its start
  int64_t first, list, state, hist, count, kept, saved, end;
};
Space space_of(int64_t units, int64_t slots, int64_t budget, int64_t row) {
  auto up = [](int64_t v) { return ceil_div(v, 16) * 16; };
  Space s{};
  s.first = 16;
  s.list = s.first + up(4 * units);
  s.state = s.list + up(8 * units * budget);
  const int64_t parts = by_parts(units, slots) ? ceil_div(slots, PART) : 0;
  s.hist = s.state + (parts ? up(2 * units * (int64_t)sizeof(Find)) : 0);
  s.count = s.hist + 3 * units * parts * BINS * 4;
  s.kept = s.count + up(4 * units * parts);
  s.saved = s.kept + (parts ? up(4 * units * budget) : 0);
  s.end = s.saved + (segment_of(units, budget, row) < 31 ? units * 2 * budget * row : 0);
  return s;
}

}  // namespace
}  // namespace paged
}  // namespace tsp

using namespace tsp;

extern "C" int64_t tsp_paged_evict_workspace_size(int dtype, int64_t B, int64_t Hkv, int64_t slots, int64_t D,
                                                  int64_t budget) {
  const int64_t most = int64_t(1) << 30;
  if ((dtype != TSP_F32 && dtype != TSP_BF16 && dtype != TSP_F16) || B < 0 || Hkv < 1 || budget < 0 || slots < 0 ||
      B > most || Hkv > most || slots > most || D < 1 || D > 128 || B * Hkv > most)
    return fail(TSP_EINVAL, "tsp_paged_evict_workspace_size: bad sizes"), -1;
  return paged::space_of(B * Hkv, slots, budget < slots ? budget : slots, D * paged::esize(dtype)).end;
}

extern "C" int tsp_paged_evict(void* K_pages, const int64_t* kps, void* V_pages, const int64_t* vps, int dtype, int64_t B,
                               int64_t Hkv, int64_t pages, int64_t page_size, int64_t D, const void* table,
                               int table_type, int64_t table_stride, int64_t cols, const void* lengths, int index_type,
                               float* weights, const int64_t* ws, int64_t budget, int64_t recent, void* lengths_out,
                               void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "tsp_paged_evict";
  const hipStream_t st = (hipStream_t)stream;
  int rc = paged::check_cache(who, dtype, B, Hkv, pages, page_size, D, table, table_type, table_stride, cols);
  if (rc) return rc;
  if (recent < 0 || budget < recent) return fail(TSP_EINVAL, "%s: budget %lld, recent %lld", who, (long long)budget, (long long)recent);
  if ((rc = paged::check_lengths(who, B, lengths, index_type, false))) return rc;
  if (B == 0) return TSP_OK;
  const int64_t slots = cols * page_size;
  if (budget > slots) budget = slots;  // (nothing to evict: as for any budget that holds all)
  if (recent > budget) recent = budget;
  const paged::Lengths len = paged::lengths_of(lengths, nullptr, index_type, slots, 0);
  if ((rc = paged::check_lengths_out(who, B, lengths_out, len))) return rc;
  if (!weights && slots > 0) return fail(TSP_EINVAL, "%s: null weights", who);
  if ((rc = paged::check_weights(who, weights, ws, B, Hkv, slots))) return rc;
  if ((rc = paged::check_pages(who, "K_pages", K_pages, kps, dtype, pages, Hkv, page_size, D, true))) return rc;
  if ((rc = paged::check_pages(who, "V_pages", V_pages, vps, dtype, pages, Hkv, page_size, D, true))) return rc;
  if (pages > 0 && K_pages == V_pages) return fail(TSP_EINVAL, "%s: K_pages and V_pages are the same", who);
  const int64_t units = B * Hkv, row = D * paged::esize(dtype);
  const paged::Space sp = paged::space_of(units, slots, budget, row);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < sp.end) return fail(TSP_EINVAL, "%s: workspace too small or not 16-byte aligned", who);
  paged::EvictArgs a{};
  a.Kp = paged::pages_of(K_pages, kps, dtype);
  a.Vp = paged::pages_of(V_pages, vps, dtype);
  a.t = paged::table_of(table, table_type, table_stride, cols, pages, page_size);
  a.len = len;
  a.out = lengths_out;
  a.W = weights, a.wb = ws[0], a.wh = ws[1];
  a.units = units, a.Hkv = (int)Hkv, a.D = (int)D, a.esz = paged::esize(dtype);
  a.budget = (int)budget, a.recent = (int)recent;
  a.spare = (char*)workspace;
  a.first = (int32_t*)(a.spare + sp.first);
  a.list = (u32x2*)(a.spare + sp.list);
  a.segment = paged::segment_of(units, budget, row);
  const uint32_t segments = a.segment < 31 ? (uint32_t)ceil_div(budget, int64_t(1) << a.segment) : 1;
  // Slices of 256 bytes where these are no more bytes than slices of 128 (a line of the
  // cache) and give 192 workgroups; of 64 where those of 128 leave CUs without one. (The
  // eviction of units of 4096 rows to 2048, slices of 128 and 256 bytes, us: rows of 256
  // bytes, 64 units 34.6 and 37.2, 96 units 46.6 and 44.1, 256 units 122 and 117; rows of
  // 192 bytes, 256 units 119 and 97; of 384 bytes, 128 units 88 and 92. 32768 rows of 131072
  // in segments, 8 units: 105 and 101.)
  const bool parts = paged::by_parts(units, slots), thin = segments == 1 && units * 2 * ceil_div(row, 128) < 256;
  const bool broad = ceil_div(row, 128) % 2 == 0 && units * 2 * segments * ceil_div(row, 256) >= 192;
  const int64_t slices = ceil_div(row, broad ? 256 : thin ? 64 : 128), lanes = row > 256 ? 5 : row > 128 ? 4 : 3,
                per = ceil_div(budget, (256 >> lanes) * paged::SU);
  if (parts) {
    a.parts = (int)ceil_div(slots, paged::PART);
    a.state = (paged::Find*)(a.spare + sp.state);
    a.hist = (uint32_t*)(a.spare + sp.hist);
    a.count = (int32_t*)(a.spare + sp.count);
    a.kept = (float*)(a.spare + sp.kept);
  }
  a.saved = a.spare + sp.saved;
  const int64_t grid = ceil_div(units * 2 * segments, 8) * 8 * slices;
  if (grid > INT32_MAX || units * a.parts > INT32_MAX || units * 2 * per > INT32_MAX)
    return fail(TSP_EUNSUPPORTED, "%s: too large a grid", who);
  if (parts) {
    for (int turn = 0; turn < 3; ++turn)
      hipLaunchKernelGGL(paged::digit_kernel, dim3((unsigned)(units * a.parts)), dim3(paged::ST), 0, st, a, turn);
    hipLaunchKernelGGL(paged::list_kernel, dim3((unsigned)(units * a.parts)), dim3(paged::ST), 0, st, a);
  } else {
    // (the eviction of 8 units, head_dim 128 in 16 bits: 4096 of 16384 rows 37.9 us with 8
    // rows to a thread, 33.2 with 16; 8192 of 32768 56.5 and 62.9)
    if (slots > paged::PART && slots <= 2 * paged::PART)
      hipLaunchKernelGGL(paged::select_kernel<16>, dim3((unsigned)units), dim3(paged::ST), 0, st, a);
    else
      hipLaunchKernelGGL(paged::select_kernel<8>, dim3((unsigned)units), dim3(paged::ST), 0, st, a);
  }
  if (budget > 0 && (parts || segments > 1))
    hipLaunchKernelGGL(paged::save_kernel, dim3((unsigned)(units * 2 * per)), dim3(256), 0, st, a, (uint32_t)per, (int)lanes);
  if ((rc = check_launch("select launch"))) return rc;
  if (pages == 0 || budget == 0) return TSP_OK;
  const auto move = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(paged::MT), 0, st, a, (uint32_t)slices, segments);
  };
  if (segments > 1)
    broad ? move(paged::move_kernel<16, true>) : move(paged::move_kernel<8, true>);
  else if (broad)
    move(paged::move_kernel<16, false>);
  else
    thin ? move(paged::move_kernel<4, false>) : move(paged::move_kernel<8, false>);
  return check_launch("move launch");
}
