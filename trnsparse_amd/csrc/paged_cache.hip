// Writes to a key and value cache in pages: new tokens' rows, and the eviction
// that keeps a budget of rows. No counterpart in the reference, whose attention
// takes one sequence's K and V whole (trnsparse/ops.py:549-625).
#include "paged_cache.h"

namespace tsp {
namespace paged {

int check_cache(const char* who, int dtype, int64_t B, int64_t Hkv, int64_t pages, int64_t page_size, int64_t D,
                const void* table, int table_type, int64_t table_stride, int64_t cols) {
  if (dtype != TSP_F32 && dtype != TSP_BF16 && dtype != TSP_F16)
    return fail(TSP_EUNSUPPORTED, "%s: dtype %d not supported", who, dtype);
  if (B < 0 || Hkv < 1 || pages < 0 || page_size < 1 || D < 1 || cols < 0)
    return fail(TSP_EINVAL, "%s: bad sizes batch %lld kv_heads %lld pages %lld page_size %lld head_dim %lld columns %lld",
                who, (long long)B, (long long)Hkv, (long long)pages, (long long)page_size, (long long)D, (long long)cols);
  if (page_size % PIECE) return fail(TSP_EUNSUPPORTED, "%s: page_size %lld must be a multiple of 16", who, (long long)page_size);
  if (D > 128 || D % (16 / esize(dtype)) != 0)
    return fail(TSP_EUNSUPPORTED, "%s: head_dim %lld (at most 128, whole 16-byte pieces)", who, (long long)D);
  const int64_t most = int64_t(1) << 30;
  if (B > most || Hkv > most || pages > INT32_MAX || page_size > most || cols > most || cols * page_size > most ||
      B * Hkv > most || cols * page_size > (int64_t(1) << 40) / page_size - 1)
    return fail(TSP_EUNSUPPORTED, "%s: too many rows, pages or heads", who);
  if (table_type != TSP_I32 && table_type != TSP_I64) return fail(TSP_EINVAL, "%s: bad table type", who);
  if (B > 0 && cols > 0) {
    if (!table) return fail(TSP_EINVAL, "%s: null block table", who);
    if (table_stride < 0) return fail(TSP_EINVAL, "%s: negative stride of the block table", who);
  }
  return TSP_OK;
}

int check_pages(const char* who, const char* name, const void* p, const int64_t* s, int dtype, int64_t pages, int64_t D) {
  if (!s) return fail(TSP_EINVAL, "%s: no strides of %s", who, name);
  if (pages == 0) return TSP_OK;
  if (!p) return fail(TSP_EINVAL, "%s: null %s", who, name);
  const int64_t e = esize(dtype);
  if (((uintptr_t)p | (uint64_t)(s[0] * e) | (uint64_t)(s[1] * e) | (uint64_t)(s[2] * e)) & 15)
    return fail(TSP_EINVAL, "%s: %s and its strides must be whole 16-byte pieces", who, name);
  if (s[0] < 0 || s[1] < 0 || s[2] < D || s[2] * e >= (int64_t(1) << 24))
    return fail(TSP_EINVAL, "%s: strides of %s: %lld, %lld, %lld", who, name, (long long)s[0], (long long)s[1],
                (long long)s[2]);
  return TSP_OK;
}

int check_lengths(const char* who, int64_t B, const void* lengths, int index_type) {
  if (index_type != TSP_I32 && index_type != TSP_I64) return fail(TSP_EINVAL, "%s: bad index type", who);
  if (B > 0 && !lengths) return fail(TSP_EINVAL, "%s: null lengths", who);
  return TSP_OK;
}

int check_weights(const char* who, const void* w, const int64_t* s) {
  if (!w) return TSP_OK;
  if (!s) return fail(TSP_EINVAL, "%s: no strides of weights", who);
  if (((uintptr_t)w & 3) || s[0] < 0 || s[1] < 0) return fail(TSP_EINVAL, "%s: bad weights", who);
  return TSP_OK;
}

namespace {

// ---------------------------------------------------------------- append
// One thread to a 16-byte piece of a new row: K's, V's, then the zeros of the
// weights and the lengths. Bound by the rows' bytes, or by the launch.
struct AppendArgs {
  const char *K, *V;
  int64_t kb, kh, ks, vb, vh, vs;  // strides in bytes
  Pages Kp, Vp;
  Table t;
  Lengths len;
  void* out;  // lengths after
  float* W;
  int64_t wb, wh;
  int64_t B;
  uint32_t Hkv, N, chunks;  // chunks: 16-byte pieces of a row
};
__global__ __launch_bounds__(256) void append_kernel(const AppendArgs a, int64_t total) {
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (x < a.B) {
    const int64_t n = cached_rows(a.len, x) + new_rows(a.len, x), v = n < a.len.slots ? n : a.len.slots;
    if (a.len.wide)
      ((int64_t*)a.out)[x] = v;
    else
      ((int32_t*)a.out)[x] = (int32_t)v;
  }
  if (x >= total) return;
  // (batch, token, head, piece), the order of a projection's output
  const int64_t row = x / a.chunks, tok = row / a.Hkv;
  const uint32_t c = (uint32_t)(x - row * a.chunks), h = (uint32_t)(row - tok * a.Hkv);
  const int64_t b = tok / a.N, i = tok - b * a.N;
  const int64_t m = a.len.fresh ? clamped(a.len.wide ? ((const int64_t*)a.len.fresh)[b]
                                                     : (int64_t)((const int32_t*)a.len.fresh)[b], a.len.most)
                                : a.len.most;
  if (i >= m) return;
  const int64_t n = clamped(a.len.wide ? ((const int64_t*)a.len.p)[b] : (int64_t)((const int32_t*)a.len.p)[b], a.len.slots);
  const int64_t j = n + i;
  if (j >= a.len.slots) return;
  if (a.W && c == 0) a.W[b * a.wb + h * a.wh + j] = 0.f;
  const uint32_t col = (uint32_t)j / (uint32_t)a.t.page_size, r = (uint32_t)j - col * (uint32_t)a.t.page_size;
  const uint32_t page = page_of_lane(a.t, b * a.t.ld, col);
  if (page == NO_PAGE) return;
  const u32x4 k = *(const u32x4*)(a.K + b * a.kb + h * a.kh + i * a.ks + 16 * c);
  const u32x4 v = *(const u32x4*)(a.V + b * a.vb + h * a.vh + i * a.vs + 16 * c);
  *(u32x4*)(a.Kp.p + page * a.Kp.page + h * a.Kp.h + r * a.Kp.s + 16 * c) = k;
  *(u32x4*)(a.Vp.p + page * a.Vp.page + h * a.Vp.h + r * a.Vp.s + 16 * c) = v;
}

// -------------------------------------------------------------- eviction
// select_kernel, one workgroup to a (sequence, head) pair: the key (an unsigned
// number in the order of the weights, NaN above all) of the k-th largest of the
// rows that may go, by histograms of the keys' digits of 11, 11 and 10 bits, fewer
// where all rows with the digits so far stay; then one pass in the rows' order that
// lists the kept ones and moves their weights, each to a place at or before its own.
// move_kernel moves the listed rows of K and V to their places. A row goes to a
// place at or before its own, and the list rises: a workgroup that takes the list
// in order, and writes a part only once all of its rows are read, never writes
// over a row that is still to be read. Workgroups share no byte: each has one
// head's K or V and a slice of its rows.
struct EvictArgs {
  Pages Kp, Vp;
  Table t;
  Lengths len;
  void* out;
  float* W;
  int64_t wb, wh;
  int64_t B;
  int Hkv, D, esz;
  int budget, recent;
  u32x2* list;     // [batch][head][budget]: kept rows, page and row of it
  int32_t* first;  // [batch][head]: the first kept row that moves
  char* spare;     // 16 bytes
};

constexpr int ST = 1024, SPT = 8, PART = ST * SPT, BINS = 2048;  // threads of select_kernel, rows of one in a part

__device__ inline uint32_t order_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);  // (one zero)
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// sum over the lanes before this one, and the total of the wavefront
__device__ inline int wave_scan(int v, int lane, int& total) {
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  total = __builtin_amdgcn_readlane(x, 63);
  return x - v;
}

// A thread's rows of a part, consecutive ones; rows from `end` on are not read.
struct Part {
  float v[SPT];
  __device__ inline void load(const float* w, int j, int end, bool aligned) {
    if (aligned && j + SPT <= end) {
#pragma unroll
      for (int i = 0; i < SPT; i += 4) {
        const f32x4 x = *(const f32x4*)(w + j + i);
        v[i] = x[0], v[i + 1] = x[1], v[i + 2] = x[2], v[i + 3] = x[3];
      }
    } else {
#pragma unroll
      for (int i = 0; i < SPT; ++i) v[i] = j + i < end ? w[j + i] : 0.f;
    }
  }
};

__global__ __launch_bounds__(ST) void select_kernel(const EvictArgs a) {
  __shared__ uint32_t hist[BINS];
  __shared__ int sums[2][2][ST / 64];
  __shared__ uint32_t pick[3];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t unit = blockIdx.x, b = unit / a.Hkv, h = unit - b * a.Hkv;
  const int64_t n64 = cached_rows(a.len, b);
  if (h == 0 && tid == 0) {
    const int64_t v = n64 < a.budget ? n64 : a.budget;
    if (a.len.wide)
      ((int64_t*)a.out)[b] = v;
    else
      ((int32_t*)a.out)[b] = (int32_t)v;
  }
  const int n = (int)n64;
  if (n <= a.budget) {
    if (tid == 0) a.first[unit] = a.budget;
    return;
  }
  float* w = a.W + b * a.wb + h * a.wh;
  const bool aligned = ((uintptr_t)w & 15) == 0;
  const int E = n - a.recent;            // rows that may go
  const int keep = a.budget - a.recent;  // of those, the ones that stay (fewer than E)
  // The rows of up to one part stay in registers; of more, each pass reads them
  // again, two parts ahead of the one that is worked on.
  const bool once = n <= PART;
  Part held;
  held.load(w, tid * SPT, n, aligned);
  auto each = [&](int end, auto&& f) {
    Part even = held, odd;
    if (!once) odd.load(w, PART + tid * SPT, n, aligned);
    for (int j0 = 0; j0 < end; j0 += 2 * PART) {
      f(j0 + tid * SPT, even);
      if (once) break;
      even.load(w, j0 + 2 * PART + tid * SPT, n, aligned);
      if (j0 + PART < end) f(j0 + PART + tid * SPT, odd);
      odd.load(w, j0 + 3 * PART + tid * SPT, n, aligned);
    }
  };
  // `last`: the keys above it stay, and of those equal to it the first `equal` ones
  uint32_t last = 0xffffffffu;
  int equal = 0;
  if (keep > 0) {
    for (int i = tid; i < BINS; i += ST) hist[i] = 0;
    __syncthreads();
    uint32_t lo = 0, hi = 0xffffffffu;
    int want = keep;  // the place of the wanted key among those of [lo, hi], from the largest
    for (int shift = 21;; shift = shift > 10 ? shift - 11 : 0) {
      each(E, [&](int j, const Part& p) {
#pragma unroll
        for (int i = 0; i < SPT; ++i) {
          const uint32_t k = order_key(p.v[i]);
          if (j + i < E && k >= lo && k <= hi) atomicAdd(&hist[(k - lo) >> shift], 1u);
        }
      });
      __syncthreads();
      // two digits to a thread, from the largest; the one where the count passes `want`
      const int d = BINS - 1 - 2 * tid;
      const int c0 = (int)hist[d], c1 = (int)hist[d - 1];
      hist[d] = hist[d - 1] = 0;  // (for the next turn)
      int total, before = wave_scan(c0 + c1, lane, total);
      if (lane == 0) sums[0][0][wave] = total;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < ST / 64; ++i) before += i < wave ? sums[0][0][i] : 0;
      if (before < want && want <= before + c0 + c1) {
        const bool second = want > before + c0;
        pick[0] = (uint32_t)(second ? d - 1 : d);
        pick[1] = (uint32_t)(want - before - (second ? c0 : 0));
        pick[2] = (uint32_t)(second ? c1 : c0);
      }
      __syncthreads();
      want = (int)pick[1];
      lo += pick[0] << shift;
      hi = lo + (shift ? (1u << shift) - 1 : 0);
      if (want == (int)pick[2]) {  // all with this digit stay
        last = lo - 1;             // (no key is zero: it would be a NaN's)
        break;
      }
      if (shift == 0) {
        last = lo;
        equal = want;
        break;
      }
    }
  }
  __syncthreads();
  // the kept rows in order; those that equal the last one's key as far as they go
  u32x2* list = a.list + unit * a.budget;
  int base = 0, equal_base = 0, first = a.budget, turn = 0;
  each(n, [&](int j, Part p) {
    // (a thread's rows lie in one page)
    const uint32_t col = column_of(a.t, (uint32_t)j / PIECE), row = (uint32_t)j - col * (uint32_t)a.t.page_size;
    const uint32_t page = j < n ? page_of_lane(a.t, b * a.t.ld, col) : NO_PAGE;
    uint32_t above = 0, same = 0;
#pragma unroll
    for (int i = 0; i < SPT; ++i) {
      const uint32_t k = order_key(p.v[i]);
      if (j + i < n && (j + i >= E || (keep > 0 && k > last))) above |= 1u << i;
      if (j + i < E && keep > 0 && k == last) same |= 1u << i;
    }
    // both counts in one scan: at most PART of each
    int total, before = wave_scan(__builtin_popcount(same) << 16 | __builtin_popcount(above), lane, total);
    if (lane == 0) sums[turn][0][wave] = total;
    // every row of this part is read before one is written
#pragma unroll
    for (int i = 0; i < SPT; ++i) asm volatile("" : "+v"(p.v[i]));
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int i = 0; i < ST / 64; ++i) {
      const int c = sums[turn][0][i];
      before += i < wave ? c : 0;
      all += c;
    }
    turn ^= 1;
    int e = equal_base + (before >> 16);  // equal ones before this thread's
    const int e0 = equal_base < equal ? equal_base : equal;
    int d = base + (before & 0xffff) + (e < equal ? e : equal) - e0;
#pragma unroll
    for (int i = 0; i < SPT; ++i) {
      bool stays = above >> i & 1;
      if (same >> i & 1) stays = e++ < equal;
      if (!stays) continue;
      list[d] = u32x2{page, row + i};
      if (d != j + i) {
        w[d] = p.v[i];
        first = d < first ? d : first;
      }
      ++d;
    }
    equal_base += all >> 16;
    base += (all & 0xffff) + (equal_base < equal ? equal_base : equal) - e0;
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const int f = __shfl_xor(first, o, 64);
    first = f < first ? f : first;
  }
  if (lane == 0) sums[turn][1][wave] = first;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < ST / 64; ++i) first = sums[turn][1][i] < first ? sums[turn][1][i] : first;
    a.first[unit] = first;
  }
}

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
template <int LPR>
__global__ __launch_bounds__(MT) void move_kernel(const EvictArgs a, uint32_t slices) {
  // the slices of a row in consecutive slots of one XCD
  const uint32_t xcd = blockIdx.x & 7, at8 = blockIdx.x >> 3, slice = at8 % slices, x = at8 / slices * 8 + xcd;
  const int64_t unit = x >> 1;
  if (unit >= a.B * a.Hkv) return;
  const int64_t b = unit / a.Hkv, h = unit - b * a.Hkv;
  const int first = a.first[unit];
  if (first >= a.budget) return;
  const Pages& p = x & 1 ? a.Vp : a.Kp;
  const u32x2* list = a.list + unit * a.budget;
  const int64_t trow = b * a.t.ld;
  constexpr int RP = MT / LPR, PR = RP * MU;  // rows at once, and of a part
  const uint32_t row_bytes = (uint32_t)(a.D * a.esz);
  uint32_t c = 16 * (LPR * slice + threadIdx.x % LPR);
  c = c < row_bytes ? c : row_bytes - 16;
  char* base = p.p + h * p.h + c;
  const int at = threadIdx.x / LPR, end = a.budget - 1;
  auto place = [&](int d0, int u) {
    const int d = d0 + RP * u + at;
    return (uint32_t)(d < end ? d : end);
  };
  // a row's place, or the spare one
  auto spot = [&](uint32_t page, uint32_t row) {
    const uint64_t none = 0 - (uint64_t)(page == NO_PAGE);
    const uint64_t there = (uint64_t)(base + (int64_t)(page & ~(uint32_t)none) * p.page + row * p.s);
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
  auto load = [&](Move& m) {
#pragma unroll
    for (int u = 0; u < MU; ++u) {
      m.v[u] = *spot(m.from[u].x, m.from[u].y);
    }
  };
  auto step = [&](Move& now, Move& next, Move& later, int d0) {
    look(later, d0 + 2 * PR);
    load(next);
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
  load(m0);
  for (int d0 = first;; d0 += 3 * PR) {
    step(m0, m1, m2, d0);
    if (d0 + PR > end) break;
    step(m1, m2, m0, d0 + PR);
    if (d0 + 2 * PR > end) break;
    step(m2, m0, m1, d0 + 2 * PR);
    if (d0 + 3 * PR > end) break;
  }
}

// Workspace: 16 bytes that writes to no page go to, the units' first rows that
// move, then the lists.
int64_t list_at(int64_t B, int64_t Hkv) { return 16 + ceil_div(4 * B * Hkv, 16) * 16; }
int64_t list_bytes(int64_t B, int64_t Hkv, int64_t budget) { return list_at(B, Hkv) + 8 * B * Hkv * budget; }

}  // namespace
}  // namespace paged
}  // namespace tsp

using namespace tsp;

extern "C" int tsp_paged_append(const void* K, const int64_t* ks, const void* V, const int64_t* vs, void* K_pages,
                                const int64_t* kps, void* V_pages, const int64_t* vps, int dtype, int64_t B, int64_t Hkv,
                                int64_t N, int64_t pages, int64_t page_size, int64_t D, const void* table, int table_type,
                                int64_t table_stride, int64_t cols, const void* lengths, const void* new_lengths,
                                int index_type, void* lengths_out, float* weights, const int64_t* ws, void* stream) {
  const char* who = "tsp_paged_append";
  int rc = paged::check_cache(who, dtype, B, Hkv, pages, page_size, D, table, table_type, table_stride, cols);
  if (rc) return rc;
  if (N < 0 || N > (int64_t(1) << 30)) return fail(TSP_EINVAL, "%s: %lld tokens", who, (long long)N);
  if ((rc = paged::check_lengths(who, B, lengths, index_type))) return rc;
  if (B == 0) return TSP_OK;
  if (!lengths_out || lengths_out == lengths) return fail(TSP_EINVAL, "%s: lengths_out must be a place of its own", who);
  if ((rc = paged::check_pages(who, "K_pages", K_pages, kps, dtype, pages, D))) return rc;
  if ((rc = paged::check_pages(who, "V_pages", V_pages, vps, dtype, pages, D))) return rc;
  if ((rc = paged::check_weights(who, weights, ws))) return rc;
  const int64_t e = paged::esize(dtype);
  const int64_t* st[2] = {ks, vs};
  const void* pt[2] = {K, V};
  for (int i = 0; i < 2 && N > 0; ++i) {
    if (!pt[i] || !st[i]) return fail(TSP_EINVAL, "%s: null %s", who, i ? "V" : "K");
    if (((uintptr_t)pt[i] | (uint64_t)(st[i][0] * e) | (uint64_t)(st[i][1] * e) | (uint64_t)(st[i][2] * e)) & 15)
      return fail(TSP_EINVAL, "%s: %s and its strides must be whole 16-byte pieces", who, i ? "V" : "K");
  }
  paged::AppendArgs a{};
  if (N > 0) {
    a.K = (const char*)K, a.V = (const char*)V;
    a.kb = ks[0] * e, a.kh = ks[1] * e, a.ks = ks[2] * e;
    a.vb = vs[0] * e, a.vh = vs[1] * e, a.vs = vs[2] * e;
  }
  a.Kp = paged::pages_of(K_pages, kps, dtype);
  a.Vp = paged::pages_of(V_pages, vps, dtype);
  a.t = paged::table_of(table, table_type, table_stride, cols, pages, page_size);
  a.len = paged::Lengths{lengths, new_lengths, index_type == TSP_I64, cols * page_size, N};
  a.out = lengths_out;
  a.W = weights;
  if (weights) a.wb = ws[0], a.wh = ws[1];
  a.B = B, a.Hkv = (uint32_t)Hkv, a.N = (uint32_t)(N > 0 ? N : 1), a.chunks = (uint32_t)(D * e / 16);
  const int64_t total = cols > 0 ? B * N * Hkv * a.chunks : 0;
  const int64_t grid = ceil_div(total > B ? total : B, 256);
  if (grid > INT32_MAX) return fail(TSP_EUNSUPPORTED, "%s: too large a grid", who);
  hipLaunchKernelGGL(paged::append_kernel, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, a, total);
  return check_launch("append launch");
}

extern "C" int64_t tsp_paged_evict_workspace_size(int64_t B, int64_t Hkv, int64_t budget) {
  const int64_t most = int64_t(1) << 30;
  if (B < 0 || Hkv < 1 || budget < 0 || B > most || Hkv > most || budget > most || B * Hkv > most)
    return fail(TSP_EINVAL, "tsp_paged_evict_workspace_size: bad sizes"), -1;
  return paged::list_bytes(B, Hkv, budget);
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
  if ((rc = paged::check_lengths(who, B, lengths, index_type))) return rc;
  if (B == 0) return TSP_OK;
  const int64_t slots = cols * page_size;
  if (budget > slots) budget = slots;  // (nothing to evict: as for any budget that holds all)
  if (recent > budget) recent = budget;
  if (!lengths_out || lengths_out == lengths) return fail(TSP_EINVAL, "%s: lengths_out must be a place of its own", who);
  if (!weights) return fail(TSP_EINVAL, "%s: null weights", who);
  if ((rc = paged::check_weights(who, weights, ws))) return rc;
  if ((rc = paged::check_pages(who, "K_pages", K_pages, kps, dtype, pages, D))) return rc;
  if ((rc = paged::check_pages(who, "V_pages", V_pages, vps, dtype, pages, D))) return rc;
  if (pages > 0 && K_pages == V_pages) return fail(TSP_EINVAL, "%s: K_pages and V_pages are the same", who);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < paged::list_bytes(B, Hkv, budget)) return fail(TSP_EINVAL, "%s: workspace too small", who);
  paged::EvictArgs a{};
  a.Kp = paged::pages_of(K_pages, kps, dtype);
  a.Vp = paged::pages_of(V_pages, vps, dtype);
  a.t = paged::table_of(table, table_type, table_stride, cols, pages, page_size);
  a.len = paged::Lengths{lengths, nullptr, index_type == TSP_I64, slots, 0};
  a.out = lengths_out;
  a.W = weights, a.wb = ws[0], a.wh = ws[1];
  a.B = B, a.Hkv = (int)Hkv, a.D = (int)D, a.esz = paged::esize(dtype);
  a.budget = (int)budget, a.recent = (int)recent;
  a.spare = (char*)workspace;
  a.first = (int32_t*)(a.spare + 16);
  a.list = (u32x2*)(a.spare + paged::list_at(B, Hkv));
  // slices of 128 bytes, a line of the cache; of 64 where they leave CUs without one
  const int64_t units = B * Hkv * 2, row = D * a.esz;
  const bool thin = units * ceil_div(row, 128) < 256;
  const int64_t slices = ceil_div(row, thin ? 64 : 128), grid = ceil_div(units, 8) * 8 * slices;
  if (grid > INT32_MAX) return fail(TSP_EUNSUPPORTED, "%s: too large a grid", who);
  hipLaunchKernelGGL(paged::select_kernel, dim3((unsigned)(B * Hkv)), dim3(paged::ST), 0, st, a);
  if ((rc = check_launch("select launch"))) return rc;
  if (pages == 0 || budget == 0) return TSP_OK;
  if (thin)
    hipLaunchKernelGGL(paged::move_kernel<4>, dim3((unsigned)grid), dim3(paged::MT), 0, st, a, (uint32_t)slices);
  else
    hipLaunchKernelGGL(paged::move_kernel<8>, dim3((unsigned)grid), dim3(paged::MT), 0, st, a, (uint32_t)slices);
  return check_launch("move launch");
}
