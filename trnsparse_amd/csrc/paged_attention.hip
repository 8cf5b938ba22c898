// Attention of a chunk of new tokens over a key and value cache in pages
// (serving): sequence b has n = lengths[b] rows in its pages, the last m =
// new_lengths[b] of them the new tokens'. Query i of head h, key head hk = h / G:
//   O[b, h, i] = sum_j p_ij V[b, hk, j],  p_i = softmax_j(scale Q[b, h, i] . K[b, hk, j])
// over j < n - (m - 1 - i), and on request
//   W[b, hk, j] += sum over the heads of hk and the queries i of p_ij.
// No counterpart in the reference, whose attention is one sequence's over its
// whole K and V (trnsparse/ops.py:549-625).
//
// A unit is one (sequence, key head) pair; its rows are r = i G + g (token,
// head of the group), so that the keys which a run of rows sees end close
// together. Tiles, softmax and products: xattn_tiles.h.
//   wide    128 rows to a workgroup, a wavefront to 32; stages of keys that the
//           four wavefronts share in an LDS ring of two
//   narrow  up to 32 rows to a workgroup: every wavefront has all of them and
//           takes every fourth stage of 32 keys through LDS of its own. (40 rows as
//           two such workgroups, that read the keys twice: 40.9 us, wide 34.3.)
// The host does not see the lengths. It launches `items` workgroups for every
// unit; they find from the lengths how many tiles of rows each unit has and, where
// these are few, ranges of the keys (share_of), and the work is dealt to the
// first workgroups of the launch, the longest first (work_of); the others end.
// Ranges write their own normalised result and log-sum-exp in fp32, which
// combine_kernel joins in the ranges' order.
//
// The accumulated weights need the final log-sum-exp of every row. Up to 16 rows:
// the narrow kernel keeps its scores (4 bytes a pair, where reading K again is 2
// head_dim bytes a key), whose exponentials are added up afterwards. More: the
// scores are formed again, a wavefront having 32 keys as its own rows and the
// queries staged, so that a key's sum stays in its lane (weights_kernel). Either
// way a key's sum is added up in a fixed order: no atomics.
//
// What bounds them: narrow, the reads of K and V (64 sequences of up to 8192 keys, 8 key
// heads of 128, one token each: bf16 278 to 291 us by the lengths, 5.6 to 5.8 TB/s, fp32 550
// to 576, 5.7); wide, the matrix instructions with the softmax next to them rather than
// under them (2 x 2048 tokens over up to 10240 keys, 32 heads over 8 of 128 in bf16: 430 to
// 514 us, 1.01 to 1.03 PFLOP/s); small calls, the launch and one workgroup's chain of
// stages (4 sequences of up to 512 keys: 8.6 us). Tiles have 64 or 128 elements of a row:
// head_dim 16 to 32 reads as slowly as 64 (32 sequences of up to 8192 keys, 8 heads, one
// token: 46 us at 16 and 83 at 64 in bf16, 128 and 166 in fp32).
#include "lds_dma.h"
#include "paged_cache.h"
#include "xattn_fwd.h"

namespace tsp {
namespace xat {
int check_sizes(const char* who, int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t L, int64_t D);
}
namespace paged {
namespace {

using xat::Operand;
using xat::OUT_OF_RANGE;

struct Args {
  Operand Q;
  char* O;
  int64_t ob, oh, os;  // strides of O in bytes
  Pages K, V;
  Table t;
  Lengths len;
  int B, Hkv, G, R, D;       // R: rows of a unit
  int items;                 // workgroups of a unit at most
  int deal;                  // work goes to the launch's first workgroups, longest first (up to 64 sequences)
  int slots;                 // results of ranges that a unit has room for (0: keys stay whole)
  int own;                   // of which it takes this many whatever the other sequences have
  int places;                // and more as long as all tiles of a key head have this many workgroups (0: none)
  int least, step;           // a range's least keys, and what it is a multiple of
  int slot_rows;             // rows of one such result
  float *part, *plse;        // [unit][slot][row]: results, log-sum-exps (base 2)
  float* lse;                // [unit][R]: where the weights need them (else null), what scale_of makes of log-sum-exps
  float* scores;             // [unit][stage of 32 keys][sr][32], log2 units, of units of up to sr rows
  int sr;
  int stages;                // of a unit
  float scale_log2;
  float* W;
  int64_t wb, wh;
  int wsplits;               // parts of a unit's rows in weights_kernel; their sums:
  float* wpart;              // [part][unit][wkeys], where there are several
  int wkeys;
};

constexpr int MOST_RANGES = 64;  // of a unit's keys where the host chooses them
constexpr int TILE = 128;  // rows of a wide workgroup (a narrow one has all of its unit's)
struct Share {
  int n, m, rows, tiles, splits, chunk;
};
// What the workgroups of a unit of n cached and m new rows do; its keys may be in `share` ranges
// where there is room for them, and in more if a.own holds them.
__device__ inline Share share_of(const Args& a, int n, int m, int share) {
  Share s;
  s.n = n;
  s.m = m;
  s.rows = m * a.G;
  s.tiles = (s.rows + TILE - 1) / TILE;
  s.splits = 1;
  s.chunk = n > 0 ? n : 1;
  int k = s.tiles ? a.own / s.tiles : 0;
  if (share > 1 && s.tiles > 1) {
    const int room = a.slots / s.tiles, more = share < room ? share : room;
    k = k > more ? k : more;
  }
  const int most = (n + a.least - 1) / a.least;
  k = k < most ? k : most;
  if (k > 1) {
    s.chunk = ((n + k - 1) / k + a.step - 1) / a.step * a.step;
    s.splits = (n + s.chunk - 1) / s.chunk;
  }
  return s;
}
__device__ inline Share share_of(const Args& a, int64_t b, int share = 1) {
  return share_of(a, (int)cached_rows(a.len, b), (int)new_rows(a.len, b), share);
}
// A log-sum-exp (base 2) as the weights take it: of a row whose scores are all -inf,
// whose result is zero, such that every weight 2^(score - it) is zero too.
__device__ inline float scale_of(float lse) { return lse == -INFINITY ? INFINITY : lse; }
// Keys that a row's token sees.
__device__ inline int sees_of(const Share& s, int i) { return s.n - (s.m - 1 - i); }

__device__ inline bool unit_of(const Args& a, uint32_t block, int per_unit, uint32_t& unit, uint32_t& b, uint32_t& hk,
                               int& item) {
  int64_t u, i;
  if (!head_item(block, per_unit, (int64_t)a.B * a.Hkv, u, i)) return false;
  unit = (uint32_t)u;
  b = unit / (uint32_t)a.Hkv;
  hk = unit - b * (uint32_t)a.Hkv;
  item = (int)i;
  return true;
}

// The lengths of the lane's sequence, of up to 64 (none: zero).
struct Lane64 {
  int n, m;
};
__device__ inline Lane64 lane_lengths(const Args& a) {
  const int lane = threadIdx.x & 63;
  Lane64 l{0, 0};
  if (lane < a.B) {
    const auto at = [&](const void* p, int wide) {
      return wide ? ((const int64_t*)p)[lane] : (int64_t)((const int32_t*)p)[lane];
    };
    l.n = (int)clamped(at(a.len.p, a.len.wide), a.len.slots);
    l.m = (int)(a.len.fresh ? clamped(at(a.len.fresh, a.len.fresh_wide), a.len.most) : a.len.most);
  }
  return l;
}
// Ranges for the keys of every sequence such that all tiles have up to a.places workgroups
// (of up to 64 sequences, each in a lane).
__device__ inline int ranges_of(const Args& a, const Lane64& l) {
  if (!a.places) return 1;
  int total;
  wave_scan((l.m * a.G + TILE - 1) / TILE, total);
  const uint32_t n = total > 0 ? (uint32_t)a.places / (uint32_t)total : 1;
  return n < 4 ? 1 : (int)n;  // (fewer give less than joining them costs: 2 heads of 108 tiles 69 us whole, 72 in two)
}
// What a workgroup does: item `item` of the `wgs` that its unit has.
struct Work {
  uint32_t unit, b, hk;
  int item, wgs;
  Share s;
};
__device__ inline bool work_of(const Args& a, uint32_t block, Work& w) {
  if (!a.deal) {
    if (!unit_of(a, block, a.items, w.unit, w.b, w.hk, w.item)) return false;
    w.wgs = a.items;
    w.s = share_of(a, (int64_t)w.b);
    return true;
  }
  // A lane has one sequence: its workgroups for one key head, and how long the
  // first of them takes. The longest go first.
  const int lane = threadIdx.x & 63;
  const Lane64 l = lane_lengths(a);
  const int ranges = ranges_of(a, l);
  const Share v = share_of(a, l.n, l.m, ranges);
  const int rest = (a.R - v.rows + 255) / 256;  // (rows to clear)
  int wgs = v.tiles * v.splits;
  wgs = lane < a.B ? (wgs > rest ? wgs : rest) : 0;
  const int keys = v.chunk < l.n ? v.chunk : l.n, time = v.rows > 32 ? 4 * keys : keys;
  // Workgroups without work end before the places are found: they are most where a batch has
  // many sequences and few chunks. (64 sequences, 4 chunks of 256 tokens, 16 heads over 4 of
  // 128, up to 2048 keys: 105 us where all went through the loop over the sequences, 81 so.)
  int total, start = 0;
  wave_scan(wgs, total);
  int64_t hk, at;
  if (!sorted_item(block, total, a.Hkv, hk, at)) return false;
  const int p = (int)at;
  for (int j = 0; j < a.B; ++j) {
    const int wj = __builtin_amdgcn_readlane(wgs, j), tj = __builtin_amdgcn_readlane(time, j);
    start += tj > time || (tj == time && j < lane) ? wj : 0;
  }
  w.b = __builtin_amdgcn_readfirstlane(__builtin_ctzll(__builtin_amdgcn_ballot_w64(start <= p && p < start + wgs)));
  w.hk = (uint32_t)hk;
  w.unit = w.b * (uint32_t)a.Hkv + w.hk;
  w.item = p - __builtin_amdgcn_readlane(start, w.b);
  w.wgs = __builtin_amdgcn_readlane(wgs, w.b);
  w.s = share_of(a, __builtin_amdgcn_readlane(l.n, w.b), __builtin_amdgcn_readlane(l.m, w.b), ranges);
  return true;
}
// The sequence whose cache is the k-th longest (of up to 64, weighed with its new rows).
__device__ inline uint32_t longest_first(const Args& a, uint32_t k) {
  if (a.B < 2 || a.B > 64) return k;
  const int lane = threadIdx.x & 63;
  const Lane64 l = lane_lengths(a);
  const float work = lane < a.B ? (float)l.n * (float)l.m : -1.f;
  uint32_t rank = 0;
  for (int j = 0; j < a.B; ++j) {
    const float other = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(work), j));
    rank += other > work || (other == work && j < lane);
  }
  return __builtin_amdgcn_readfirstlane(__builtin_ctzll(__builtin_amdgcn_ballot_w64(lane < a.B && rank == k)));
}

__device__ inline const char* q_row(const Args& a, int64_t b, int64_t hk, int i, int g) {
  return a.Q.p + b * a.Q.b + (hk * a.G + g) * a.Q.h + i * a.Q.s;
}
__device__ inline char* o_row(const Args& a, int64_t b, int64_t hk, int i, int g) {
  return a.O + b * a.ob + (hk * a.G + g) * a.oh + i * a.os;
}

// Rows behind a sequence's new tokens are zero; the unit's workgroups share them.
__device__ inline void clear_rest(const Args& a, const Work& w, int esz) {
  const int c = 16 * (threadIdx.x & 31);
  for (int r = w.s.rows + w.item * 8 + (int)(threadIdx.x >> 5); r < a.R; r += 8 * w.wgs) {
    const int i = r / a.G, g = r - i * a.G;
    if (c < a.D * esz) *(u32x4*)(o_row(a, w.b, w.hk, i, g) + c) = u32x4{};
  }
}

// A buffer whose place and size are the same for the whole wavefront, in scalar registers.
__device__ inline dma::i32x4 buffer_at(const char* base, uint32_t bytes) {
  dma::i32x4 r = dma::make_rsrc(base, bytes);
  r.x = __builtin_amdgcn_readfirstlane(r.x);
  r.y = __builtin_amdgcn_readfirstlane(r.y);
  r.z = __builtin_amdgcn_readfirstlane(r.z);
  return r;
}

// A wavefront's rows of a stage: `ROWS` consecutive cached rows of one page.
template <typename T, int ROWS>
struct Loader {
  static constexpr int RPI = 64 / T::CPR, NI = ROWS / RPI;
  static_assert(NI >= 1 && ROWS == NI * RPI && PIECE % ROWS == 0, "whole instructions, one page");
  uint32_t off[NI];
  // `first`: the rows' place in the stage
  __device__ inline void init(int first, int lane, int64_t row_bytes, int D) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = RPI * i + lane / T::CPR, c = (lane % T::CPR) ^ T::swz(first + r);
      off[i] = c * T::CE < D ? (uint32_t)(r * row_bytes) + 16u * c : OUT_OF_RANGE;
    }
  }
  // The rows at `base` of which `rows` exist (none: all zero) into LDS dst.
  __device__ inline void issue(const char* base, int rows, int64_t row_bytes, int D, uint32_t dst) const {
    const uint32_t bytes = rows > 0 ? (uint32_t)((rows - 1) * row_bytes) + (uint32_t)(D * T::ESZ) : 0;
    const dma::i32x4 rs = buffer_at(base, bytes);
#pragma unroll
    for (int i = 0; i < NI; ++i) dma::buffer16(rs, off[i], dst + i * 1024);
  }
};

// Where the rows from key `key` on lie: looked up before a wait that takes in the scalar load.
struct Spot {
  uint32_t page;
  int row;
};
__device__ inline Spot spot_of(const Table& t, int64_t trow, int key, int end) {
  Spot s{NO_PAGE, 0};
  if (key < end) {
    const uint32_t col = column_of(t, (uint32_t)key / PIECE);
    s.page = page_at(t, trow, col);
    s.row = key - (int)col * t.page_size;
  }
  return s;
}
// Keeps the look-up before the wait that follows.
__device__ inline void settle(Spot& s) {
  s.page = __builtin_amdgcn_readfirstlane(s.page);
  asm volatile("" : "+s"(s.page));
}
// Rows [key, end) of the piece or part of one that starts at the spot.
template <typename L>
__device__ inline void fetch(const L& ld, const Pages& p, const char* head, const Spot& s, int key, int end, int most,
                             int D, uint32_t dst) {
  const int left = end - key, rows = s.page == NO_PAGE ? 0 : left < most ? left : most;
  const int64_t page = s.page == NO_PAGE ? 0 : s.page;
  ld.issue(head + page * p.page + s.row * p.s, rows, p.s, D, dst);
}

template <typename T>
struct Final {
  char* o;
  float* p;
  __device__ inline void put(int d, f32x4 v) const {
    if (p)
      *(f32x4*)(p + d) = v;
    else
      T::store4(o + d * T::ESZ, v);
  }
};

// ------------------------------------------------------------------- wide
template <typename T>
struct Wide {
  static constexpr int NT = T::ESZ == 2 ? 2 : 1, HK = 32 * NT, HBYTES = HK * T::ROWB, STAGE = 2 * HBYTES;
  static constexpr int LDS = 2 * STAGE, MINE = HK / 4;
  typedef Loader<T, MINE> Ld;

  static __device__ inline void run(const Args& a, const Work& wk, uint8_t* lds) {
    const Share& s = wk.s;
    const int64_t b = wk.b, hk = wk.hk;
    if (s.tiles == 0) return;
    const int split = wk.item / s.tiles;
    if (split >= s.splits) return;
    const int tile = s.tiles - 1 - (wk.item - split * s.tiles);  // the tiles that see most first
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
    const int r0 = tile * TILE + w * 32, r = r0 + (lane & 31);
    const bool live = r < s.rows, some = r0 < s.rows;
    const int i = live ? r / a.G : 0, g = live ? r - i * a.G : 0;
    typename T::Rows q;
    T::load(q, q_row(a, b, hk, i, g), live, a.D, h);

    const int c0 = split * s.chunk;
    const int tile_last = tile * TILE + TILE - 1 < s.rows ? tile * TILE + TILE - 1 : s.rows - 1;
    const int last = sees_of(s, tile_last / a.G);                   // keys that any row of the tile sees
    const int k1 = c0 + s.chunk < last ? c0 + s.chunk : last;
    const int sees = live ? sees_of(s, i) : 0;
    const int least = some ? sees_of(s, r0 / a.G) : 0;              // and that all rows of the wavefront see
    const int nst = k1 > c0 ? (k1 - c0 + HK - 1) / HK : 0;
    const char* Kh = a.K.p + hk * a.K.h;
    const char* Vh = a.V.p + hk * a.V.h;
    const int64_t trow = b * a.t.ld;
    Ld kl, vl;
    kl.init(MINE * w, lane, a.K.s, a.D);
    vl.init(MINE * w, lane, a.V.s, a.D);
    const typename T::Lane ln = T::lane_of(lane);
    const uint32_t lds0 = dma::lds_addr(lds), mine = w * (MINE * T::ROWB);
    auto key = [&](int st) { return c0 + st * HK + MINE * w; };
    auto issue = [&](int st, const Spot& sp) {
      const uint32_t at = lds0 + (st & 1) * STAGE + mine;
      fetch(kl, a.K, Kh, sp, key(st), k1, MINE, a.D, at);
      fetch(vl, a.V, Vh, sp, key(st), k1, MINE, a.D, at + HBYTES);
    };
    xat::RowState<T> x;
    x.clear();
    if (nst > 0) issue(0, spot_of(a.t, trow, key(0), k1));
    for (int st = 0; st < nst; ++st) {
      Spot sp = spot_of(a.t, trow, key(st + 1), k1);
      settle(sp);
      dma::wait_vm<0>();
      dma::barrier();
      if (st + 1 < nst) issue(st + 1, sp);
      if (!some) continue;
      const int at = c0 + st * HK;
      const uint32_t stage = lds0 + (st & 1) * STAGE;
      const int lim = least < k1 ? least : k1;
      // P as one 16-bit number, whose rounding is as large as the result's own: off by 2.3e-3
      // of the norm in bf16 and 2.9e-4 in fp16, as the sum of two, which the narrow kernel has,
      // 1.7e-3 and 2.1e-4. Two are half as many products again and registers that the
      // stages need: 2 x 2048 tokens 447 us and 610.
      xat::softmax_stage<T, NT, false>(x, q, stage, stage + HBYTES, ln, h, a.scale_log2, at + HK > lim,
                                       xat::keys_from(sees, k1, at), [] {});
    }
    const float l = xat::halves_sum(x.l), inv = l > 0.f || l != l ? 1.f / l : 0.f;
    if (!live) return;
    const bool whole = s.splits == 1;
    const int64_t at = ((int64_t)wk.unit * a.slots + wk.item) * a.slot_rows + (r - tile * TILE);
    const Final<T> out{o_row(a, b, hk, i, g), whole ? nullptr : a.part + at * a.D};
    T::quads(x.acc, h, [&](int d, f32x4 v) {
      if (d < a.D) out.put(d, v * inv);
    });
    if (h == 0) {
      const float e = x.m + __builtin_amdgcn_logf(l);
      if (!whole)
        a.plse[at] = e;
      else if (a.lse)
        a.lse[(int64_t)wk.unit * a.R + r] = scale_of(e);
    }
  }
};

// ----------------------------------------------------------------- narrow
template <typename T>
struct Narrow {
  static constexpr int NW = 4, HBYTES = 32 * T::ROWB, XLD = T::DP + 4;
  static constexpr int RING = NW * 2 * HBYTES, XB = NW * 32 * (XLD + 2) * 4, LDS = RING > XB ? RING : XB;
  typedef Loader<T, PIECE> Ld;
  static constexpr int NI = 2 * Ld::NI;  // instructions of a stage's K

  static __device__ inline void fence() { asm volatile("" ::: "memory"); }
  static __device__ inline void drained() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

  template <bool SCORES>
  static __device__ inline void run(const Args& a, const Work& wk, uint8_t* lds) {
    const Share& s = wk.s;
    const uint32_t unit = wk.unit, b = wk.b, hk = wk.hk;
    const int split = wk.item;
    if (s.rows == 0 || split >= s.splits) return;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
    const int l32 = lane & 31;
    const bool live = l32 < s.rows;
    const int i = live ? l32 / a.G : 0, g = live ? l32 - i * a.G : 0;
    const int k0 = split * s.chunk, k1 = k0 + s.chunk < s.n ? k0 + s.chunk : s.n;
    const int sees = live ? sees_of(s, i) : 0, lim = sees_of(s, 0);  // keys of this row, and keys that all rows see
    const int nst = k1 > k0 ? (k1 - k0 + 31) / 32 : 0, mine = nst > w ? (nst - w + NW - 1) / NW : 0;
    const char* Kh = a.K.p + hk * a.K.h;
    const char* Vh = a.V.p + hk * a.V.h;
    const int64_t trow = b * a.t.ld;
    // rows 16 and on of a stage are swizzled as the first 16 are
    static_assert(T::swz(16) == T::swz(0) && T::swz(19) == T::swz(3), "one set of offsets");
    Ld kl, vl;
    kl.init(0, lane, a.K.s, a.D);
    vl.init(0, lane, a.V.s, a.D);
    const uint32_t kst = dma::lds_addr(lds) + w * 2 * HBYTES, vst = kst + HBYTES;
    auto key = [&](int st) { return k0 + 32 * (st * NW + w); };
    struct Two {
      Spot p[2];
    };
    auto look = [&](int st) {
      Two t;
      t.p[0] = spot_of(a.t, trow, key(st), k1);
      t.p[1] = spot_of(a.t, trow, key(st) + PIECE, k1);
      return t;
    };
    auto issue = [&](const Ld& ld, const Pages& p, const char* head, int st, const Two& t, uint32_t dst) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        fetch(ld, p, head, t.p[j], key(st) + PIECE * j, k1, PIECE, a.D, dst + j * PIECE * T::ROWB);
    };
    Two now = look(0);
    if (mine > 0) {
      issue(kl, a.K, Kh, 0, now, kst);
      issue(vl, a.V, Vh, 0, now, vst);
    }
    typename T::Rows q;
    T::load(q, q_row(a, b, hk, i, g), live, a.D, h);
    const typename T::Lane ln = T::lane_of(lane);
    xat::RowState<T> x;
    x.clear();
    float* sc = nullptr;
    if constexpr (SCORES) sc = a.scores + ((int64_t)unit * a.stages * a.sr + l32) * 32 + 4 * h;
    for (int st = 0; st < mine; ++st) {
      const bool more = st + 1 < mine;
      const int at = key(st);
      Two next = look(st + 1);
      settle(next.p[0]);
      settle(next.p[1]);
      dma::wait_vm<NI>();  // K is there once only V's loads are out
      fence();
      f32x16 c[1];
      T::template scores<1>(c, kst, ln, q);
      drained();  // this wavefront's reads of K have returned: its place is free
      if (more) issue(kl, a.K, Kh, st + 1, next, kst);
      const bool check = at + 32 > (lim < k1 ? lim : k1);
      xat::weigh_stage<T, 1, true>(
          x, c, vst, ln, h, a.scale_log2, check, xat::keys_from(sees, k1, at),
          [&] {
            if constexpr (SCORES) {
              // four stores of every wavefront, its first row being there
              float* p = sc + (int64_t)(at / 32) * a.sr * 32;
              if (live) {
#pragma unroll
                for (int v = 0; v < 4; ++v)
                  *(f32x4*)(p + 8 * v) = f32x4{c[0][4 * v], c[0][4 * v + 1], c[0][4 * v + 2], c[0][4 * v + 3]} * a.scale_log2;
              }
            }
          },
          [&] {
            if (more)
              dma::wait_vm<NI + (SCORES ? 4 : 0)>();
            else
              dma::wait_vm<0>();
            fence();
          });
      drained();
      if (more) issue(vl, a.V, Vh, st + 1, next, vst);
    }
    join(a, s, unit, b, hk, split, x, lds, w, h, l32, live);
  }

  // m, l, acc of each row over the wavefronts, through LDS
  static __device__ inline void join(const Args& a, const Share& s, uint32_t unit, uint32_t b, uint32_t hk, int split,
                                     const xat::RowState<T>& x, uint8_t* lds, int w, int h, int l32, bool live) {
    const float l = xat::halves_sum(x.l);
    float* xo = (float*)lds;
    float* xm = xo + NW * 32 * XLD;
    float* xl = xm + NW * 32;
    __syncthreads();
    if (live) {
      T::quads(x.acc, h, [&](int d, f32x4 v) { *(f32x4*)(xo + (w * 32 + l32) * XLD + d) = v; });
      if (h == 0) {
        xm[w * 32 + l32] = x.m;
        xl[w * 32 + l32] = l;
      }
    }
    __syncthreads();
    constexpr int QPR = T::DP / 4;  // quads of a row
    for (int e = threadIdx.x; e < s.rows * QPR; e += 64 * NW) {
      const int row = e / QPR, d = 4 * (e % QPR), i = row / a.G, g = row - i * a.G;
      float m = -INFINITY;
#pragma unroll
      for (int j = 0; j < NW; ++j) m = fmaxf(m, xm[j * 32 + row]);
      float total = 0.f;
      f32x4 sum = f32x4{};
#pragma unroll
      for (int j = 0; j < NW; ++j) {
        const float lj = xl[j * 32 + row], mj = xm[j * 32 + row];
        // (a wavefront without keys for the row has m = -inf, l = 0; a NaN score leaves NaN in l)
        const float f = mj == -INFINITY ? (lj == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(mj - m);
        total += f * lj;
        sum += *(const f32x4*)(xo + (j * 32 + row) * XLD + d) * f;
      }
      const float inv = total > 0.f || total != total ? 1.f / total : 0.f, lse = m + __builtin_amdgcn_logf(total);
      const bool whole = s.splits == 1;
      const int64_t at = ((int64_t)unit * a.slots + split) * a.slot_rows + row;
      const Final<T> out{o_row(a, b, hk, i, g), whole ? nullptr : a.part + at * a.D};
      if (d < a.D) out.put(d, sum * inv);
      if (d == 0) {
        if (!whole)
          a.plse[at] = lse;
        else if (a.lse)
          a.lse[(int64_t)unit * a.R + row] = scale_of(lse);
      }
    }
  }
};

template <typename T>
constexpr int narrow_per_cu = Narrow<T>::LDS <= 80 * 1024 ? 2 : 1;

// Units of up to 32 rows each.
template <typename T, bool SCORES>
__global__ __launch_bounds__(256, narrow_per_cu<T>) void narrow_kernel(const Args a) {
  typedef Narrow<T> N;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[N::LDS];
  Work w;
  if (!work_of(a, blockIdx.x, w)) return;
  clear_rest(a, w, T::ESZ);
  N::template run<SCORES>(a, w, lds);
}
// Units of any number of rows, each narrow or wide by its own (wide where the
// narrow kernel's LDS would leave one workgroup to a CU: fp32 rows of 128).
template <typename T>
constexpr bool chunk_has_narrow = narrow_per_cu<T> == 2;
template <typename T, bool SCORES>
__global__ __launch_bounds__(256, 2) void chunk_kernel(const Args a) {
  typedef Wide<T> W;
  typedef Narrow<T> N;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[chunk_has_narrow<T> && N::LDS > W::LDS ? N::LDS : W::LDS];
  Work w;
  if (!work_of(a, blockIdx.x, w)) return;
  clear_rest(a, w, T::ESZ);
  if (SCORES && w.s.rows <= a.sr)
    N::template run<true>(a, w, lds);
  else if (chunk_has_narrow<T> && w.s.rows <= 32)
    N::template run<false>(a, w, lds);
  else
    W::run(a, w, lds);
}

// ---------------------------------------------------------------- joining
// One row: the ranges' results with weights 2^(lse_j - max lse); 32 lanes to a
// row, four values each. Returns the row's log-sum-exp.
template <typename T>
__device__ inline float combine_row(const Args& a, const Share& s, uint32_t unit, uint32_t b, uint32_t hk, int r) {
  const int lane = threadIdx.x & 31, d = 4 * lane;
  const int tile = r / TILE;
  const int64_t stride = (int64_t)s.tiles * a.slot_rows;  // of a row between ranges
  const int64_t at = ((int64_t)unit * a.slots + (s.tiles - 1 - tile)) * a.slot_rows + (r - tile * TILE);
  float m = -INFINITY, total = 0.f;
  f32x4 sum = f32x4{};
  for (int j0 = 0; j0 < s.splits; j0 += 32) {
    const float lse = j0 + lane < s.splits ? a.plse[at + (j0 + lane) * stride] : -INFINITY;
    float mx = lse;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    const float mn = fmaxf(m, mx);
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    total *= f;
    sum *= f;
    // (a range without keys for the row weighs nothing; a NaN goes on)
    const float wgt = lse == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(lse - mn);
    const int n = s.splits - j0 < 32 ? s.splits - j0 : 32;
    const float* p = a.part + (at + j0 * stride) * a.D + (d < a.D ? d : 0);
    for (int j = 0; j < n; j += 8) {
      f32x4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = j + u < n ? *(const f32x4*)(p + (j + u) * stride * a.D) : f32x4{};
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float wj = __shfl(wgt, (threadIdx.x & 32) + j + u, 64);  // (zero behind the last range)
        total += wj;
        sum += wj == 0.f ? f32x4{} : v[u] * wj;
      }
    }
  }
  const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
  const int i = r / a.G, g = r - i * a.G;
  if (d < a.D) T::store4(o_row(a, b, hk, i, g) + d * T::ESZ, sum * inv);
  return m + __builtin_amdgcn_logf(total);
}

// `per` workgroups to a unit, 8 rows of each at a time.
template <typename T>
__global__ __launch_bounds__(256) void combine_kernel(const Args a, int per) {
  const uint32_t unit = blockIdx.x / (uint32_t)per, part = blockIdx.x - unit * (uint32_t)per;
  const uint32_t b = unit / (uint32_t)a.Hkv, hk = unit - b * (uint32_t)a.Hkv;
  const Share s = share_of(a, (int64_t)b, a.places ? ranges_of(a, lane_lengths(a)) : 1);
  if (s.splits == 1) return;
  for (int r = (int)part * 8 + (int)(threadIdx.x >> 5); r < s.rows; r += 8 * per) {
    const float lse = combine_row<T>(a, s, unit, b, hk, r);
    if (a.lse && (threadIdx.x & 31) == 0) a.lse[(int64_t)unit * a.R + r] = scale_of(lse);
  }
}

// The weight of key k of a unit whose scores are kept (a key that a row does not
// see has a score of -inf).
__device__ inline float weight_of(const Args& a, const Share& s, uint32_t unit, const float* lse, int k) {
  const float* p = a.scores + ((int64_t)unit * a.stages + k / 32) * a.sr * 32 + k % 32;
  float sum = 0.f;
  for (int r = 0; r < s.rows; r += 4) {
    float c[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) c[u] = r + u < s.rows ? p[(r + u) * 32] : -INFINITY;
#pragma unroll
    for (int u = 0; u < 4; ++u) sum += c[u] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(c[u] - lse[r + u]);
  }
  return sum;
}

// After the narrow kernel: workgroups [0, cw) of a unit join its rows (where the
// keys were taken in ranges), the other `kw` add up the keys' weights, 256 keys
// at a time, from the scores and the rows' log-sum-exps.
template <typename T>
__global__ __launch_bounds__(256) void weigh_kernel(const Args a, int cw, int kw) {
  __shared__ float lse[36];  // (read four at a time)
  const uint32_t per = (uint32_t)(cw + kw), unit = blockIdx.x / per;
  const int part = (int)(blockIdx.x - unit * per);
  const uint32_t b = unit / (uint32_t)a.Hkv, hk = unit - b * (uint32_t)a.Hkv;
  const Share s = share_of(a, (int64_t)b);
  if (part < cw) {
    const int r = part * 8 + (int)(threadIdx.x >> 5);
    if (s.splits > 1 && r < s.rows) combine_row<T>(a, s, unit, b, hk, r);
    return;
  }
  if (s.splits > 1) {
    // 8 threads to a row, each with up to 8 of its ranges
    const int r = threadIdx.x >> 3, l8 = threadIdx.x & 7;
    float e[MOST_RANGES / 8], m = -INFINITY, total = 0.f;
    if (r < s.rows) {
      const int64_t at = (int64_t)unit * a.slots * a.slot_rows + r;
#pragma unroll
      for (int j = 0; j < MOST_RANGES / 8; ++j)
        e[j] = l8 + 8 * j < s.splits ? a.plse[at + (int64_t)(l8 + 8 * j) * a.slot_rows] : -INFINITY;
#pragma unroll
      for (int j = 0; j < MOST_RANGES / 8; ++j) m = fmaxf(m, e[j]);
      for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
#pragma unroll
      for (int j = 0; j < MOST_RANGES / 8; ++j) total += e[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(e[j] - m);
      for (int o = 4; o > 0; o >>= 1) total += __shfl_xor(total, o, 64);
      if (l8 == 0) lse[r] = m + __builtin_amdgcn_logf(total);
    }
  } else if ((int)threadIdx.x < s.rows) {
    lse[threadIdx.x] = a.lse[(int64_t)unit * a.R + threadIdx.x];
  }
  __syncthreads();
  float* w = a.W + b * a.wb + hk * a.wh;
  for (int k = (part - cw) * 256 + (int)threadIdx.x; k < s.n; k += 256 * kw) w[k] += weight_of(a, s, unit, lse, k);
}

// ------------------------------------------------- weights of many rows
// 32 keys to a wavefront as its own rows; the unit's rows staged 64 or 32 at a
// time with their log-sum-exps.
//   RW 1  128 keys to a workgroup, whose four wavefronts share the stages
//   RW 4  32 keys to a workgroup, every wavefront with every fourth stage of 32
//         rows through LDS of its own, their sums added at the end: four times as
//         many workgroups, each a quarter as long, for launches that have few; where
//         these would still be few and long, a workgroup takes a part of the rows only,
//         and add_kernel adds the parts' sums
template <typename T, int RW>
struct Weigh {
  static constexpr int NT = RW == 1 && T::ESZ == 2 ? 2 : 1, HR = 32 * NT, STAGE = HR * T::ROWB;
  static constexpr int KEYS = 128 / RW, RINGS = RW, LDS = RINGS * 2 * STAGE;
  static constexpr int RPI = 64 / T::CPR, MINE = RW == 1 ? HR / 4 : HR, NI = MINE / RPI;
};
template <typename T, int RW>
__global__ __launch_bounds__(256, (Weigh<T, RW>::LDS <= 72 * 1024 ? 2 : 1)) void weights_kernel(const Args a, int per) {
  typedef Weigh<T, RW> G;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[G::LDS];
  __shared__ __attribute__((aligned(256))) float lse[G::RINGS][2][64];  // of a stage's rows
  uint32_t unit, b, hk;
  int item;
  if constexpr (RW == 1) {
    if (!unit_of(a, blockIdx.x, per, unit, b, hk, item)) return;
  } else {
    // the few units' workgroups over all XCDs (one long sequence of two key heads next to
    // three of one token, each head on an XCD of its own: 78 us, 30 over all)
    const uint32_t p = blockIdx.x / (uint32_t)a.Hkv;
    hk = blockIdx.x - p * (uint32_t)a.Hkv;
    b = p / (uint32_t)per;
    item = (int)(p - b * (uint32_t)per);
  }
  b = longest_first(a, b);
  unit = b * (uint32_t)a.Hkv + hk;
  const Share s = share_of(a, (int64_t)b);  // (its lengths)
  const int part = RW == 1 ? 0 : item % a.wsplits, j0 = (RW == 1 ? item : item / a.wsplits) * G::KEYS;
  if (j0 >= s.n || s.rows == 0) return;
  float* W = a.W + b * a.wb + hk * a.wh;
  if (s.rows <= a.sr) {
    const int k = j0 + (int)threadIdx.x;
    if (part == 0 && (int)threadIdx.x < G::KEYS && k < s.n) W[k] += weight_of(a, s, unit, a.lse + (int64_t)unit * a.R, k);
    return;
  }
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int k0 = RW == 1 ? j0 + w * 32 : j0, j = k0 + (lane & 31);  // this wavefront's keys, this lane's
  const int ring = RW == 1 ? 0 : w, w4 = RW == 1 ? w : 0;
  const bool live = j < s.n;
  typename T::Rows k;
  {
    const uint32_t col = live ? column_of(a.t, (uint32_t)j / PIECE) : 0;
    const uint32_t page = live ? page_of_lane(a.t, b * a.t.ld, col) : NO_PAGE;
    const char* p = a.K.p + (page == NO_PAGE ? 0 : page) * a.K.page + hk * a.K.h + (j - (int)col * a.t.page_size) * a.K.s;
    T::load(k, p, live && page != NO_PAGE, a.D, h);
  }
  const int before = s.n - s.m;  // token i sees keys up to before + i
  int first = j0 > before ? (j0 - before) * a.G / G::HR : 0;  // the first stage with a row that sees a key
  int stages = (s.rows + G::HR - 1) / G::HR;
  if (RW > 1 && a.wsplits > 1) {
    const int most = (stages - first + a.wsplits - 1) / a.wsplits;
    first += part * most;
    stages = stages < first + most ? stages : first + most;
  }
  const int seen_by = (j > before ? j - before : 0) * a.G;          // the first row that sees this lane's key
  const int all_from = (k0 + 31 > before ? k0 + 31 - before : 0) * a.G;
  const char* Qh = a.Q.p + b * a.Q.b + hk * a.G * a.Q.h;
  const float* L = a.lse + (int64_t)unit * a.R;
  const typename T::Lane ln = T::lane_of(lane);
  const uint32_t lds0 = dma::lds_addr(lds) + ring * 2 * G::STAGE, mine = w4 * (G::MINE * T::ROWB);
  const uint32_t lse0 = dma::lds_addr(lse) + ring * 512;
  // A stage's rows through a buffer that begins with the first row's token, rows
  // behind the last as zeros; then their log-sum-exps. Where stages are whole
  // tokens, the rows' offsets are the same in all of them.
  const uint32_t qs = (uint32_t)a.Q.s, qh = (uint32_t)a.Q.h;
  const uint32_t group_recip = 0xffffffffu / (uint32_t)a.G + 1;
  uint32_t offs[G::NI];
  auto offset = [&](int u, int skip) {
    const int x = G::MINE * w4 + G::RPI * u + lane / T::CPR, c = (lane % T::CPR) ^ T::swz(x);
    // v / G of v below 64 + G: one or none from G = 64 on; below, by the reciprocal
    // ceil(2^32 / G), which is exact for v G < 2^32 (and passes 32 bits for G = 1)
    const uint32_t v = (uint32_t)(skip + x), G1 = (uint32_t)a.G;
    const uint32_t i = G1 >= 64 ? (uint32_t)(v >= G1) : G1 == 1 ? v : __umulhi(v, group_recip), g = v - i * G1;
    return c * T::CE < a.D ? i * qs + g * qh + 16u * c : OUT_OF_RANGE;
  };
  const bool even = G::HR % a.G == 0;
#pragma unroll
  for (int u = 0; u < G::NI; ++u) offs[u] = offset(u, 0);
  auto issue = [&](int st, int buf) {
    const int r0 = st * G::HR, i0 = r0 / a.G;
    const dma::i32x4 rs = buffer_at(Qh + i0 * a.Q.s, OUT_OF_RANGE);
    if (!even) {
#pragma unroll
      for (int u = 0; u < G::NI; ++u) offs[u] = offset(u, r0 - i0 * a.G);
    }
#pragma unroll
    for (int u = 0; u < G::NI; ++u) {
      const int x = G::MINE * w4 + G::RPI * u + lane / T::CPR;
      dma::buffer16(rs, r0 + x < s.rows ? offs[u] : OUT_OF_RANGE, lds0 + buf * G::STAGE + mine + u * 1024);
    }
    if (RW > 1 || w == 0) {
      const int left = s.rows - r0;
      const dma::i32x4 ls = buffer_at((const char*)(L + r0), 4u * (uint32_t)(left < G::HR ? left : G::HR));
      dma::buffer4(ls, 4u * (uint32_t)lane, lse0 + buf * 256);
    }
  };
  f32x4 sum = f32x4{};
  constexpr int STEP = RW;
  int st = RW == 1 ? first : first + (w + RW - first % RW) % RW;
  if (st < stages) issue(st, 0);
  for (int buf = 0; st < stages; st += STEP, buf ^= 1) {
    if constexpr (RW == 1) {
      dma::wait_vm<0>();
      dma::barrier();
      if (st + STEP < stages) issue(st + STEP, buf ^ 1);
    } else {
      if (st + STEP < stages) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage before has been read
        issue(st + STEP, buf ^ 1);
        dma::wait_vm<G::NI + 1>();
      } else {
        dma::wait_vm<0>();
      }
      asm volatile("" ::: "memory");
    }
    f32x16 c[G::NT];
    T::template scores<G::NT>(c, lds0 + buf * G::STAGE, ln, k);
    const int r0 = st * G::HR;
    // rows that do not see the key, and rows behind the last (zeros, which an
    // infinite key would turn into NaN)
    const bool check = r0 < all_from || r0 + G::HR > s.rows;
    auto add = [&](auto masked) {
#pragma unroll
      for (int t = 0; t < G::NT; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 e = *(const f32x4*)&lse[ring][buf][32 * t + 8 * q + 4 * h];
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            float p = __builtin_amdgcn_exp2f(__builtin_fmaf(c[t][4 * q + v], a.scale_log2, -e[v]));
            if constexpr (decltype(masked)::value) {
              const int r = r0 + 32 * t + 8 * q + 4 * h + v;
              if (r < seen_by || r >= s.rows) p = 0.f;
            }
            sum[v] += p;
          }
        }
    };
    if (check)
      add(std::true_type{});
    else
      add(std::false_type{});
  }
  float total = xat::halves_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
  if constexpr (RW > 1) {
    float* x = &lse[0][0][0];
    __syncthreads();
    if (h == 0) x[w * 32 + (lane & 31)] = total;
    __syncthreads();
    if (w) return;
    const int l32 = lane & 31;
    total = (x[l32] + x[32 + l32]) + (x[64 + l32] + x[96 + l32]);
  }
  if (!live || h) return;
  if (RW > 1 && a.wsplits > 1)
    a.wpart[((int64_t)part * a.B * a.Hkv + unit) * a.wkeys + j] = total;
  else
    W[j] += total;
}
// The sums of the parts of the rows, `per` workgroups to a unit.
__global__ __launch_bounds__(256) void add_kernel(const Args a, int per) {
  const uint32_t unit = blockIdx.x / (uint32_t)per, at = blockIdx.x - unit * (uint32_t)per;
  const uint32_t b = unit / (uint32_t)a.Hkv, hk = unit - b * (uint32_t)a.Hkv;
  const Share s = share_of(a, (int64_t)b);
  const int j = (int)(at * 256 + threadIdx.x);
  if (s.rows <= a.sr || j >= s.n) return;  // (up to sr rows have been added)
  const float* p = a.wpart + (int64_t)unit * a.wkeys + j;
  float sum = 0.f;
  for (int i = 0; i < a.wsplits; ++i) sum += p[(int64_t)i * a.B * a.Hkv * a.wkeys];
  a.W[b * a.wb + hk * a.wh + j] += sum;
}

// ------------------------------------------------------------------- host

struct Plan {
  bool narrow;
  int items, slots, own, places, least, step, slot_rows;
  int sr;
  bool again, few;  // weights from scores formed again, and by 32 keys to a workgroup
  int wsplits;      // whose rows are taken in so many parts
  int64_t part, lse, scores, wpart;  // floats
  int64_t floats() const { return part + lse + scores + wpart; }
};
Plan plan_of(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t keys, int64_t D, bool ragged, bool weights) {
  Plan p{};
  const int64_t G = Hq / Hkv, R = G * Sq, units = B * Hkv;
  const bool f32 = dtype == TSP_F32;
  p.narrow = R <= 32;
  const int64_t tiles = p.narrow ? 1 : ceil_div(R, TILE), wgs = units * tiles;
  // Ranges of keys: as many as bring the rounds of workgroups that fit the CUs
  // at once, each of its keys and of as much as `least` keys more (starting,
  // joining), to the shortest time.
  p.least = p.narrow ? (f32 ? 128 : 512) : (f32 ? 64 : 256);
  p.step = p.narrow ? 128 : 64;  // whole stages of all wavefronts
  p.slot_rows = (int)(p.narrow ? R : TILE);
  const int64_t room = p.narrow && f32 && D > 64 ? 256 : 512, most = ceil_div(keys > 0 ? keys : 1, p.least);
  int64_t n = 1, best = INT64_MAX;
  for (int64_t k = 1; k <= MOST_RANGES && k <= most; ++k) {
    const int64_t cost = ceil_div(wgs * k, room) * (ceil_div(keys, k) + p.least);
    if (cost < best) best = cost, n = k;
  }
  p.items = (int)(tiles * n);
  p.slots = n > 1 ? p.items : 0;
  if (ragged && !p.narrow && n == 1) {
    // sequences of few new tokens leave workgroups over, which take ranges
    const int64_t more = ceil_div(1024, units);
    p.slots = (int)(p.items < more ? p.items : more);
    if (p.slots < 2) p.slots = 0;
  }
  p.own = p.slots;
  if (ragged && !p.narrow && B <= 64 && tiles > 1 && tiles * Hkv <= 64) {
    // nor does a chunk of one sequence fill the CUs where key heads are few: as many ranges
    // as do, as far as there is room for their results (one chunk of 512 tokens, 8 heads of
    // one key head, next to 15 single tokens: 2048 keys 59 us and 32, 8192 keys 197 and 70;
    // with up to 64 tiles of a sequence for all key heads: 16 sequences of 8 key heads and 16
    // tiles, four chunks, 142 us without and 144 with; 4 sequences of one key head, one chunk
    // of 2000 tokens of 8 heads over 8192 keys, 144 without and 71 with)
    p.places = 512;
    int64_t room = ceil_div(2048, units), use = tiles * (most < MOST_RANGES ? most : MOST_RANGES);
    if (use > p.places / Hkv) use = p.places / Hkv;
    if (room > use) room = use;
    if (room > p.slots) p.slots = (int)room;
    if (p.slots < 2) p.places = 0;
  }
  auto pad = [](int64_t v) { return ceil_div(v, 64) * 64; };
  p.part = pad(p.slots * units * p.slot_rows * (D + 1));
  p.lse = weights ? pad(units * R) : 0;
  // scores of up to 16 rows are kept (with a chunk's workgroups, those of the
  // sequences that have so few). 24 sequences of 4096 keys, 8 key heads of 128 in 16 bits:
  // 20 rows 127 us kept and 129 formed again, 32 rows 170 and 130; fp32 is ahead up to
  // 20 rows (16 sequences, head_dim 64: 80 and 92) and even at 32.
  p.sr = (int)(!weights || (p.narrow ? R > 16 : !ragged || (f32 && D > 64)) ? 0 : R < 16 ? R : 16);
  p.scores = units * ceil_div(keys, 32) * p.sr * 32;
  p.again = weights && !(p.narrow && p.sr > 0);
  // (9 units of 1008 keys and up to 399 rows in fp32: 28 us with 128 keys to a workgroup)
  p.few = units * ceil_div(keys, 128) < 512;
  p.wsplits = 1;
  if (p.again && p.few) {
    // 1024 workgroups, of which in a ragged batch most end at once, each with 32 stages of
    // rows or more (4 sequences of two key heads, one of 10400 rows, 1300 keys: 96 us
    // without parts, 30 and the addition's 5)
    const int64_t n = ceil_div(ragged ? 4096 : 1024, units * ceil_div(keys > 0 ? keys : 1, 32)), most = ceil_div(R, 32) / 32;
    p.wsplits = (int)(n < most ? n : most);
    if (p.wsplits < 1) p.wsplits = 1;
  }
  p.wpart = p.wsplits > 1 ? p.wsplits * units * keys : 0;
  return p;
}

}  // namespace
}  // namespace paged
}  // namespace tsp

using namespace tsp;

extern "C" int64_t tsp_paged_attn_workspace_size(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t keys,
                                                 int64_t D, int ragged, int weights) {
  if (xat::check_sizes("tsp_paged_attn_workspace_size", dtype, B, Hq, Hkv, Sq, keys, D)) return -1;
  if (B * Hq * Sq == 0) return 0;
  const paged::Plan p = paged::plan_of(dtype, B, Hq, Hkv, Sq, keys, D, ragged != 0, weights != 0);
  return 4 * p.floats();
}

extern "C" int tsp_paged_attn_fwd(const void* Q, const int64_t* qs, const void* K_pages, const int64_t* kps,
                                  const void* V_pages, const int64_t* vps, int dtype, int64_t B, int64_t Hq, int64_t Hkv,
                                  int64_t Sq, int64_t pages, int64_t page_size, int64_t D, const void* table,
                                  int table_type, int64_t table_stride, int64_t cols, const void* lengths,
                                  const void* new_lengths, int index_type, double scale, void* O, const int64_t* os,
                                  float* weights, const int64_t* ws, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  const char* who = "tsp_paged_attn_fwd";
  const hipStream_t st = (hipStream_t)stream;
  int rc = paged::check_cache(who, dtype, B, Hkv, pages, page_size, D, table, table_type, table_stride, cols);
  if (rc) return rc;
  const int64_t keys = cols * page_size;
  if ((rc = xat::check_sizes(who, dtype, B, Hq, Hkv, Sq, keys, D))) return rc;
  if ((rc = paged::check_lengths(who, B, lengths, index_type, true))) return rc;
  if (!(scale > 1e-30) || !(scale < 1e30)) return fail(TSP_EINVAL, "%s: scale must be positive", who);
  if (B * Hq * Sq == 0) return TSP_OK;
  if ((rc = xat::check_operand(who, "Q", Q, qs, Sq, D, dtype))) return rc;
  if ((rc = xat::check_operand(who, "O", O, os, Sq, D, dtype))) return rc;
  if ((rc = paged::check_pages(who, "K_pages", K_pages, kps, dtype, pages, Hkv, page_size, D, false))) return rc;
  if ((rc = paged::check_pages(who, "V_pages", V_pages, vps, dtype, pages, Hkv, page_size, D, false))) return rc;
  if ((rc = paged::check_weights(who, weights, ws, B, Hkv, keys))) return rc;
  const bool weigh = weights && keys > 0;
  const paged::Plan p = paged::plan_of(dtype, B, Hq, Hkv, Sq, keys, D, new_lengths != nullptr, weigh);
  const int64_t need = 4 * p.floats();
  if (need > 0 && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need))
    return fail(TSP_EINVAL, "%s: workspace too small or not 16-byte aligned", who);
  paged::Args a{};
  a.Q = xat::operand(Q, qs, Sq, D, dtype);
  const xat::Operand o = xat::operand(O, os, Sq, D, dtype);
  a.O = (char*)O;
  a.ob = o.b, a.oh = o.h, a.os = o.s;
  a.K = paged::pages_of(K_pages, kps, dtype);
  a.V = paged::pages_of(V_pages, vps, dtype);
  a.t = paged::table_of(table, table_type, table_stride, cols, pages, page_size);
  a.len = paged::lengths_of(lengths, new_lengths, index_type, keys, Sq);
  a.B = (int)B, a.Hkv = (int)Hkv, a.G = (int)(Hq / Hkv), a.R = (int)(Hq / Hkv * Sq), a.D = (int)D;
  a.items = p.items, a.slots = p.slots, a.own = p.own, a.places = (int)(p.places / Hkv), a.least = p.least, a.step = p.step, a.slot_rows = p.slot_rows;
  const int64_t units = B * Hkv;
  a.part = (float*)workspace;
  a.plse = a.part + p.slots * units * p.slot_rows * D;
  if (weigh) {
    a.lse = (float*)workspace + p.part;
    a.scores = a.lse + p.lse;
    a.sr = p.sr;
    a.wsplits = p.wsplits, a.wpart = a.scores + p.scores, a.wkeys = (int)keys;
    a.stages = (int)ceil_div(keys, 32);
    a.W = weights, a.wb = ws[0], a.wh = ws[1];
    // a stage of queries is read at 32-bit offsets from its first token
    if ((double)(a.G - 1) * a.Q.h + 66.0 * a.Q.s + 512 >= 2147483632.0)
      return fail(TSP_EUNSUPPORTED, "%s: weights of query heads that lie 2 GiB apart", who);
  }
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  // (what the places are shared out to comes on top of a unit's own items)
  const int64_t grid = p.places ? head_grid(B * p.items + p.places / Hkv, Hkv) : head_grid(p.items, units);
  // (where all workgroups of tables that are filled alike start at once, dealing has no
  // certain gain: one token, 32 heads over 8 of 128, not dealt and dealt, us: 4 sequences of
  // up to 512 keys 9.0 and 9.5, 62 of 1024 36 and 40, of 4096 145 and 143, of 8192 286 and
  // 275; 15 of 128 tokens over 2048 keys 68 and 62; 24 of five tokens, 32 heads over 4, 32
  // and 33)
  a.deal = B <= 64 && (new_lengths || units * p.items >= 512);
  const int64_t wper = p.few ? ceil_div(keys, 32) * p.wsplits : ceil_div(keys, 128);
  const int64_t wgrid = !p.again ? 0 : p.few ? wper * units : head_grid(wper, units), aper = ceil_div(keys, 256);
  const int64_t joined = p.narrow || (int64_t)(p.slots / 2) * paged::TILE > a.R ? a.R : (int64_t)(p.slots / 2) * paged::TILE;
  int64_t cper = p.slots > 1 ? ceil_div(joined, 8) : 0;
  if (!p.narrow && new_lengths && cper > ceil_div(2048, units)) cper = ceil_div(2048, units);  // (most have few rows)
  // 1024 keys and more to a workgroup, as many as fill the CUs
  int64_t kper = ceil_div(2048, units);
  if (kper > ceil_div(keys, 1024)) kper = ceil_div(keys, 1024);
  if (kper < 1) kper = 1;
  if (grid > INT32_MAX || wgrid > INT32_MAX || units * (cper + kper) > INT32_MAX || units * aper > INT32_MAX)
    return fail(TSP_EUNSUPPORTED, "%s: too large a grid", who);
  return xat::with_tile(dtype, D, [&](auto tile) {
    typedef decltype(tile) T;
    const dim3 g((unsigned)grid), t(256);
    if (p.narrow && p.sr > 0)
      hipLaunchKernelGGL((paged::narrow_kernel<T, true>), g, t, 0, st, a);
    else if (p.narrow)
      hipLaunchKernelGGL((paged::narrow_kernel<T, false>), g, t, 0, st, a);
    else if (p.sr > 0)
      hipLaunchKernelGGL((paged::chunk_kernel<T, paged::chunk_has_narrow<T>>), g, t, 0, st, a);
    else
      hipLaunchKernelGGL((paged::chunk_kernel<T, false>), g, t, 0, st, a);
    int rc = check_launch("paged attention launch");
    if (rc) return rc;
    if (p.narrow && p.sr > 0) {
      hipLaunchKernelGGL((paged::weigh_kernel<T>), dim3((unsigned)(units * (cper + kper))), t, 0, st, a, (int)cper,
                         (int)kper);
      return check_launch("weights launch");
    }
    if (cper > 0) {
      hipLaunchKernelGGL((paged::combine_kernel<T>), dim3((unsigned)(units * cper)), t, 0, st, a, (int)cper);
      if ((rc = check_launch("combine launch"))) return rc;
    }
    if (p.again) {
      if (p.few)
        hipLaunchKernelGGL((paged::weights_kernel<T, 4>), dim3((unsigned)wgrid), t, 0, st, a, (int)wper);
      else
        hipLaunchKernelGGL((paged::weights_kernel<T, 1>), dim3((unsigned)wgrid), t, 0, st, a, (int)wper);
      if ((rc = check_launch("weights launch")) || p.wsplits == 1) return rc;
      hipLaunchKernelGGL(paged::add_kernel, dim3((unsigned)(units * aper)), t, 0, st, a, (int)aper);
      return check_launch("weights launch");
    }
    return TSP_OK;
  });
}
