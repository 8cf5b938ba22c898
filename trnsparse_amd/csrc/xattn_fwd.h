// Forward kernels of dense attention over strided operands: grouped key heads,
// a length for each batch entry, keys split over workgroups when there are few
// rows. Instantiated by cross_attention.hip and prefix_attention.hip.
//
// A unit is one (batch entry, key head) pair, or one key head alone where all
// batch entries share their keys; its rows are the (batch entry, query head of
// the group, query) triples that read those keys, so one pass over the keys
// serves them all.
//   wide    128 rows to a workgroup, a wavefront to 32 of them; stages of keys
//           shared by the four wavefronts through an LDS ring of two
//   narrow  up to 32 rows to a workgroup: every wavefront has all of them and
//           takes every fourth stage of 32 keys through LDS of its own, with no
//           workgroup barrier until the wavefronts' results are joined
// Either takes one of `nsplit` ranges of `chunk` keys. With one range it writes
// the rows' results; with more it writes each range's own normalised result
// and log-sum-exp in fp32, which combine_kernel joins in range order.
#pragma once

#include "tile_item.h"
#include "xattn_tiles.h"

namespace tsp {
namespace xat {

struct Operand {
  const char* p;
  int64_t b, h, s;  // strides in bytes: batch entry, head, row
};

struct FwdArgs {
  Operand Q, K, V;
  char* O;
  int64_t ob, oh, os;   // strides of O in bytes
  float* lse;           // (batch, heads, queries) natural log-sum-exp, or null
  float *part, *plse;   // partial results and log-sum-exps (base 2) of [split][row]; null with one range
  int64_t prows;        // rows of a partial result: batch * heads * queries
  const void* lengths;  // valid keys of each batch entry (null: all)
  int len64;            // lengths are int64 (else int32)
  int units_b;          // batch entries with keys of their own (1: shared)
  int Hkv, G, Sq, R, D; // R: rows of a unit
  int64_t L;            // keys
  int causal;           // query i sees keys below length - (Sq - 1 - i)
  int tiles, nsplit, split0;
  int64_t chunk;
  float scale_log2;
};

// What a workgroup takes: tile and range of a unit. The counts' product fits
// int32 (checked by the host), so 32-bit divisions do.
struct Item {
  uint32_t unit, ub, hk;
  int tile, split;
};
__device__ inline bool item_of(const FwdArgs& a, uint32_t block, int tiles, int nsplit, Item& x) {
  int64_t unit, item;
  if (!head_item(block, (int64_t)tiles * nsplit, (int64_t)a.units_b * a.Hkv, unit, item)) return false;
  const uint32_t i = (uint32_t)item, u = (uint32_t)unit;
  x.split = (int)(i / (uint32_t)tiles);
  x.tile = (int)(i - (uint32_t)x.split * (uint32_t)tiles);
  x.unit = u;
  x.ub = u / (uint32_t)a.Hkv;
  x.hk = u - x.ub * (uint32_t)a.Hkv;
  return true;
}

struct RowId {
  int64_t b, head, orow;
  int i;
};
__device__ inline RowId row_id(const FwdArgs& a, int64_t ub, int64_t hk, int r) {
  const uint32_t per = (uint32_t)(a.G * a.Sq), bb = (uint32_t)r / per, rem = (uint32_t)r - bb * per;
  const uint32_t g = rem / (uint32_t)a.Sq;
  RowId x;
  x.i = (int)(rem - g * (uint32_t)a.Sq);
  x.b = ub + bb;
  x.head = hk * a.G + g;
  x.orow = (x.b * a.Hkv * a.G + x.head) * a.Sq + x.i;
  return x;
}
__device__ inline int64_t unit_length(const FwdArgs& a, int64_t ub) {
  if (!a.lengths) return a.L;
  const int64_t n = a.len64 ? ((const int64_t*)a.lengths)[ub] : (int64_t)((const int32_t*)a.lengths)[ub];
  return n < 0 ? 0 : n > a.L ? a.L : n;
}

// The batch entry that is taken k-th when the longest go first, of up to 64 (a
// lane has one's length; ties by index). For launches of more workgroups than fit
// at once whose time goes with the length: a long entry that starts last would run
// alone. (4 x 32 heads of 128 over 8, 1024 rows x 700 to 1800 keys, bf16: forward
// 105.6 -> 99.0 us; 3 x 8 heads of 80, 257 rows x up to 383 keys, fp32: forward and
// backward 96 -> 89.) Of more than 64 entries each is a small part of the launch, and
// they go as they come.
__device__ inline uint32_t longest_first(const FwdArgs& a, uint32_t k) {
  if (!a.lengths || a.units_b < 2 || a.units_b > 64) return k;
  const int lane = threadIdx.x & 63;
  const bool on = lane < a.units_b;
  const int n = on ? (int)unit_length(a, lane) : -1;
  uint32_t rank = 0;
  for (int j = 0; j < a.units_b; ++j) {
    const int other = __builtin_amdgcn_readlane(n, j);
    rank += other > n || (other == n && j < lane);
  }
  return __builtin_amdgcn_readfirstlane(__builtin_ctzll(__builtin_amdgcn_ballot_w64(on && rank == k)));
}

// Results of one row (four values at d): final, or one range's part.
template <typename T>
struct RowOut {
  char* o;
  float* p;
  __device__ inline RowOut(const FwdArgs& a, const RowId& id, int split) {
    o = a.O + id.b * a.ob + id.head * a.oh + id.i * a.os;
    p = a.part ? a.part + ((int64_t)(a.split0 + split) * a.prows + id.orow) * a.D : nullptr;
  }
  __device__ inline void put(int d, f32x4 v) const {
    if (p)
      *(f32x4*)(p + d) = v;
    else
      T::store4(o + d * T::ESZ, v);
  }
};
__device__ inline void put_lse(const FwdArgs& a, const RowId& id, int split, float lse2) {
  if (a.part)
    a.plse[(int64_t)(a.split0 + split) * a.prows + id.orow] = lse2;
  else if (a.lse)
    a.lse[id.orow] = lse2 * 0.69314718055994531f;
}

// Keys of a row within the range that ends at k1, from key `at` of a stage.
__device__ inline int keys_from(int64_t sees, int64_t k1, int64_t at) {
  const int64_t n = (sees < k1 ? sees : k1) - at;
  return n < 0 ? 0 : n > 64 ? 64 : (int)n;
}

// KG 2: eight wavefronts, two for every 32 rows, each pair's stages in two halves
// (the first half's results joined with the second's through LDS at the end).
// P enters its product as one 16-bit number, which moves a result as far as its own
// rounding does: both together are off by 2.3e-3 of the norm in bf16 and 2.9e-4 in
// fp16, the rounding alone by 1.7e-3 and 2.1e-4. P as the sum of two such numbers
// leaves the rounding alone, for half as many products again on matrix cores that
// are what these workgroups wait for: 32 heads of 8192 x 8192 x 128 1413 us for
// 1020, 8 x 16 of 448 x 1500 x 64 55 for 43; a shared prefix of 8192 keys and 64
// sequences of one token 43 for 40, of 3001 and 24 of five tokens 31.5 for 28.3.
template <typename T, int NT, int KG>
struct Wide {
  static constexpr int HK = 32 * NT, HBYTES = HK * T::ROWB, STAGE = 2 * HBYTES;
  static constexpr int RING = KG * 2 * STAGE, XW = (16 * T::NU + 2) * 256, LDS = KG == 2 && 4 * XW > RING ? 4 * XW : RING;
  static __device__ inline void run(const FwdArgs& a, uint32_t block, uint8_t* lds) {
    Item it;
    if (!item_of(a, block, a.tiles, a.nsplit, it)) return;
    const int tile = it.tile, split = it.split;
    const int64_t ub = KG == 1 ? longest_first(a, it.ub) : it.ub, hk = it.hk;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int w = wave & 3, kg = wave >> 2;
    const int r = tile * 128 + w * 32 + (lane & 31);
    const bool live = r < a.R, some = tile * 128 + w * 32 < a.R;  // this row, a row of the wavefront's
    const RowId id = row_id(a, ub, hk, live ? r : 0);

    typename T::Rows q;
    T::load(q, a.Q.p + id.b * a.Q.b + id.head * a.Q.h + id.i * a.Q.s, live, a.D, h);

    const int64_t n = unit_length(a, ub);
    const int64_t c0 = split * a.chunk, k1 = c0 + a.chunk < n ? c0 + a.chunk : n;
    const int64_t sees = a.causal ? n - (a.Sq - 1 - id.i) : n;  // keys of this row
    const int all = k1 > c0 ? (int)ceil_div(k1 - c0, HK) : 0, turns = KG == 2 ? (all + 1) / 2 : all;
    const int nst = kg ? all - turns : turns;  // (no more than the first half's)
    const int64_t k0 = c0 + (int64_t)kg * turns * HK;
    const char* Kp = a.K.p + ub * a.K.b + hk * a.K.h;
    const char* Vp = a.V.p + ub * a.V.b + hk * a.V.h;
    Stager<T, HK, 4> ks, vs;
    ks.init(w, lane, a.K.s, a.D);
    vs.init(w, lane, a.V.s, a.D);
    const typename T::Lane ln = T::lane_of(lane);
    const uint32_t lds0 = dma::lds_addr(lds) + kg * 2 * STAGE;
    auto issue = [&](int s) {
      const uint32_t st = lds0 + (s & 1) * STAGE;
      ks.issue(Kp, k0 + (int64_t)s * HK, k1, a.K.s, a.D, st, w);
      vs.issue(Vp, k0 + (int64_t)s * HK, k1, a.V.s, a.D, st + HBYTES, w);
    };
    RowState<T> x;
    x.clear();
    if (nst > 0) issue(0);
    for (int s = 0; s < turns; ++s) {
      dma::wait_vm<0>();
      dma::barrier();
      if (s + 1 < nst) issue(s + 1);
      if (!some || (KG == 2 && s >= nst)) continue;
      const int64_t at = k0 + (int64_t)s * HK;
      const uint32_t st = lds0 + (s & 1) * STAGE;
      softmax_stage<T, NT, false>(x, q, st, st + HBYTES, ln, h, a.scale_log2, a.causal || at + HK > k1,
                           keys_from(sees, k1, at), [] {});
    }
    if constexpr (KG == 2) {
      float* xp = (float*)lds + w * (XW / 4) + lane;  // a register of the 64 lanes at a time
      __syncthreads();
      if (kg == 1) {
#pragma unroll
        for (int u = 0; u < T::NU; ++u)
#pragma unroll
          for (int v = 0; v < 16; ++v) xp[64 * (16 * u + v)] = x.acc[u][v];
        xp[64 * 16 * T::NU] = x.m;
        xp[64 * (16 * T::NU + 1)] = x.l;
      }
      __syncthreads();
      if (kg == 1) return;
      const float m1 = xp[64 * 16 * T::NU], l1 = xp[64 * (16 * T::NU + 1)], m = fmaxf(x.m, m1);
      // (a half without keys for the row has m = -inf and nothing to add)
      const float f0 = x.m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(x.m - m);
      const float f1 = m1 == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m1 - m);
#pragma unroll
      for (int u = 0; u < T::NU; ++u)
#pragma unroll
        for (int v = 0; v < 16; ++v) x.acc[u][v] = x.acc[u][v] * f0 + xp[64 * (16 * u + v)] * f1;
      x.l = x.l * f0 + l1 * f1;
      x.m = m;
    }
    const float l = halves_sum(x.l), inv = l > 0.f || l != l ? 1.f / l : 0.f;
    if (!live) return;
    const RowOut<T> out(a, id, split);
    T::quads(x.acc, h, [&](int d, f32x4 v) {
      if (d < a.D) out.put(d, v * inv);
    });
    if (h == 0) put_lse(a, id, split, x.m + __builtin_amdgcn_logf(l));
  }
};

// Four wavefronts, each with a stage of K and one of V of its own: the next
// stage's K is loaded while this one's softmax and V are worked on, its V while
// the next scores are. Half the LDS of a ring of two, so that two workgroups
// share a CU (16 bit; 128 wide fp32 has one): one streams while the other
// starts or joins its wavefronts (16 sequences of up to 1500 keys, 8 heads of
// 128: rings of two with one workgroup to a CU 21.7 us).
// P enters its product as the sum of two 16-bit numbers: the wavefront waits for
// memory here, not for the matrix cores (that case 24.0 us with cold caches, of one
// number 23.6; 64 sequences behind 8192 shared keys 51.1 and 50.2), and a result
// then is as near as its own rounding (of one number up to 1.5 times as far). A
// prefix that more than 32 rows share is Wide's: its part of a result is as Wide's.
template <typename T>
struct Narrow {
  static constexpr int NW = 4, HBYTES = 32 * T::ROWB, XLD = T::DP + 4;
  static constexpr int RING = NW * 2 * HBYTES, XB = NW * 32 * (XLD + 2) * 4, LDS = RING > XB ? RING : XB;
  typedef Stager<T, 32, 1> St;

  static __device__ inline void run(const FwdArgs& a, uint32_t block, uint8_t* lds) {
    Item it;
    if (!item_of(a, block, 1, a.nsplit, it)) return;
    const int split = it.split;
    const int64_t ub = it.ub, hk = it.hk;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int l32 = lane & 31;
    const bool live = l32 < a.R;
    const RowId id = row_id(a, ub, hk, live ? l32 : 0);

    const int64_t n = unit_length(a, ub);
    const int64_t k0 = split * a.chunk, k1 = k0 + a.chunk < n ? k0 + a.chunk : n;
    const int64_t sees = a.causal ? n - (a.Sq - 1 - id.i) : n;
    const int nst = k1 > k0 ? (int)ceil_div(k1 - k0, 32) : 0, mine = nst > w ? (nst - w + NW - 1) / NW : 0;
    const char* Kp = a.K.p + ub * a.K.b + hk * a.K.h;
    const char* Vp = a.V.p + ub * a.V.b + hk * a.V.h;
    St ks, vs;
    ks.init(0, lane, a.K.s, a.D);
    vs.init(0, lane, a.V.s, a.D);
    const uint32_t kst = dma::lds_addr(lds) + w * 2 * HBYTES, vst = kst + HBYTES;
    auto key = [&](int s) { return k0 + 32 * ((int64_t)s * NW + w); };
    if (mine > 0) {
      ks.issue(Kp, key(0), k1, a.K.s, a.D, kst, 0);
      vs.issue(Vp, key(0), k1, a.V.s, a.D, vst, 0);
    }
    typename T::Rows q;
    T::load(q, a.Q.p + id.b * a.Q.b + id.head * a.Q.h + id.i * a.Q.s, live, a.D, h);
    const typename T::Lane ln = T::lane_of(lane);
    RowState<T> x;
    x.clear();
    for (int s = 0; s < mine; ++s) {
      const bool more = s + 1 < mine;
      const int64_t at = key(s);
      dma::wait_vm<St::NI>();  // K is there once only V's loads are out
      fence();
      softmax_stage<T, 1, true>(x, q, kst, vst, ln, h, a.scale_log2, a.causal || at + 32 > k1, keys_from(sees, k1, at), [&] {
        drained();  // this wavefront's reads of K have returned: its place is free
        if (more) {
          ks.issue(Kp, key(s + 1), k1, a.K.s, a.D, kst, 0);
          dma::wait_vm<St::NI>();
        } else {
          dma::wait_vm<0>();
        }
        fence();
      });
      drained();
      if (more) vs.issue(Vp, key(s + 1), k1, a.V.s, a.D, vst, 0);
    }
    join(a, ub, hk, split, x, lds, w, h, l32, live);
  }

  // One range over two sets of keys, the first shared by the batch: for sets so
  // short that joining two results would cost more than reading the first again.
  static __device__ inline void run_joint(const FwdArgs& a, const FwdArgs& first, uint32_t block, uint8_t* lds) {
    Item it;
    if (!item_of(a, block, 1, 1, it)) return;
    const int64_t ub = it.ub, hk = it.hk;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int l32 = lane & 31;
    const bool live = l32 < a.R;
    const RowId id = row_id(a, ub, hk, live ? l32 : 0);

    const int64_t P = first.L, n = unit_length(a, ub), sees = a.causal ? n - (a.Sq - 1 - id.i) : n;
    const int np = (int)ceil_div(P, 32), nst = np + (int)ceil_div(n, 32), mine = nst > w ? (nst - w + NW - 1) / NW : 0;
    const char* Kp = a.K.p + ub * a.K.b + hk * a.K.h;
    const char* Vp = a.V.p + ub * a.V.b + hk * a.V.h;
    const char* Kf = first.K.p + hk * first.K.h;
    const char* Vf = first.V.p + hk * first.V.h;
    St ks, vs, kf, vf;
    ks.init(0, lane, a.K.s, a.D);
    vs.init(0, lane, a.V.s, a.D);
    kf.init(0, lane, first.K.s, a.D);
    vf.init(0, lane, first.V.s, a.D);
    const uint32_t kst = dma::lds_addr(lds) + w * 2 * HBYTES, vst = kst + HBYTES;
    auto stage = [&](int s) { return s * NW + w; };
    auto issue_k = [&](int s) {
      const int t = stage(s);
      if (t < np)
        kf.issue(Kf, 32 * (int64_t)t, P, first.K.s, a.D, kst, 0);
      else
        ks.issue(Kp, 32 * (int64_t)(t - np), n, a.K.s, a.D, kst, 0);
    };
    auto issue_v = [&](int s) {
      const int t = stage(s);
      if (t < np)
        vf.issue(Vf, 32 * (int64_t)t, P, first.V.s, a.D, vst, 0);
      else
        vs.issue(Vp, 32 * (int64_t)(t - np), n, a.V.s, a.D, vst, 0);
    };
    if (mine > 0) {
      issue_k(0);
      issue_v(0);
    }
    typename T::Rows q;
    T::load(q, a.Q.p + id.b * a.Q.b + id.head * a.Q.h + id.i * a.Q.s, live, a.D, h);
    const typename T::Lane ln = T::lane_of(lane);
    RowState<T> x;
    x.clear();
    for (int s = 0; s < mine; ++s) {
      const bool more = s + 1 < mine, own = stage(s) >= np;
      const int64_t at = 32 * (int64_t)(own ? stage(s) - np : stage(s)), end = own ? n : P;
      dma::wait_vm<St::NI>();
      fence();
      softmax_stage<T, 1, true>(x, q, kst, vst, ln, h, a.scale_log2, (own && a.causal) || at + 32 > end,
                          keys_from(own ? sees : P, end, at), [&] {
                            drained();
                            if (more) {
                              issue_k(s + 1);
                              dma::wait_vm<St::NI>();
                            } else {
                              dma::wait_vm<0>();
                            }
                            fence();
                          });
      drained();
      if (more) issue_v(s + 1);
    }
    join(a, ub, hk, 0, x, lds, w, h, l32, live);
  }

  static __device__ inline void fence() { asm volatile("" ::: "memory"); }
  static __device__ inline void drained() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

  // m, l, acc of each row over the wavefronts, through LDS
  static __device__ inline void join(const FwdArgs& a, int64_t ub, int64_t hk, int split, const RowState<T>& x, uint8_t* lds,
                                     int w, int h, int l32, bool live) {
    const float l = halves_sum(x.l);
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
    for (int e = threadIdx.x; e < a.R * QPR; e += 64 * NW) {
      const int row = e / QPR, d = 4 * (e % QPR);
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
      const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
      const RowId rid = row_id(a, ub, hk, row);
      if (d < a.D) RowOut<T>(a, rid, split).put(d, sum * inv);
      if (d == 0) put_lse(a, rid, split, m + __builtin_amdgcn_logf(total));
    }
  }
};

template <typename T>
struct Kernels {
  static constexpr int NT = T::ESZ == 2 ? 2 : 1;
  typedef Narrow<T> N;
  static constexpr int PER_CU = N::LDS <= 80 * 1024 ? 2 : 1;
};
template <typename T, int KG>
__global__ __launch_bounds__(256 * KG, 2 / KG) void fwd_wide(const FwdArgs a) {
  typedef Wide<T, Kernels<T>::NT, KG> W;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[W::LDS];
  W::run(a, blockIdx.x, lds);
}
template <typename T>
__global__ __launch_bounds__(256, Kernels<T>::PER_CU) void fwd_narrow(const FwdArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Kernels<T>::N::LDS];
  Kernels<T>::N::run(a, blockIdx.x, lds);
}
template <typename T>
__global__ __launch_bounds__(256, Kernels<T>::PER_CU) void fwd_joint(const FwdArgs a, const FwdArgs first) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Kernels<T>::N::LDS];
  Kernels<T>::N::run_joint(a, first, blockIdx.x, lds);
}
// Two sets of keys in one launch: the first `grid0` workgroups take the first.
// (Workgroups of eight wavefronts for either: 64 sequences behind 8192 keys 54
// us, of four 51.)
template <typename T>
__global__ __launch_bounds__(256, Kernels<T>::PER_CU) void fwd_two(const FwdArgs a, const FwdArgs b, uint32_t grid0,
                                                                   bool wide_a, bool wide_b) {
  typedef Wide<T, Kernels<T>::NT, 1> W;
  typedef typename Kernels<T>::N N;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[W::LDS > N::LDS ? W::LDS : N::LDS];
  const bool first = blockIdx.x < grid0;
  const FwdArgs& x = first ? a : b;
  const uint32_t block = first ? blockIdx.x : blockIdx.x - grid0;
  if (first ? wide_a : wide_b)
    W::run(x, block, lds);
  else
    N::run(x, block, lds);
}

// row = bh * S + i
__device__ inline void split_row(int64_t row, int64_t S, int64_t& bh, int64_t& i) {
  if (((row | S) >> 32) == 0) {
    const uint32_t q = (uint32_t)row / (uint32_t)S;
    bh = q;
    i = (uint32_t)row - q * (uint32_t)S;
  } else {
    bh = row / S;
    i = row - bh * S;
  }
}
struct CombineArgs {
  const float *part, *plse;
  int64_t prows;
  int nsplit, D, heads, Sq;
  char* O;
  int64_t ob, oh, os;
  float* lse;
};
// The ranges' results of every row in one: weights 2^(lse_j - max lse). Rows
// that no range has keys for are zero with a log-sum-exp of -inf. 32 lanes to a
// row, four values each.
template <typename T>
__global__ __launch_bounds__(256) void combine_kernel(const CombineArgs a) {
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, d = 4 * lane;
  if (row >= a.prows) return;
  // 32 ranges at a time, one to a lane: their weights against the largest so
  // far; then their parts, read without waiting for one another
  float m = -INFINITY, total = 0.f;
  f32x4 sum = f32x4{};
  for (int j0 = 0; j0 < a.nsplit; j0 += 32) {
    const float lse = j0 + lane < a.nsplit ? a.plse[(j0 + lane) * a.prows + row] : -INFINITY;
    float mx = lse;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    const float mn = fmaxf(m, mx);
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    total *= f;
    sum *= f;
    // (a range without keys weighs nothing; a NaN goes on)
    const float wgt = lse == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(lse - mn);
    const int n = a.nsplit - j0 < 32 ? a.nsplit - j0 : 32;
    const float* p = a.part + (j0 * a.prows + row) * a.D + (d < a.D ? d : 0);
#pragma unroll 8
    for (int j = 0; j < n; ++j) {
      const float wj = __shfl(wgt, (threadIdx.x & 32) + j, 64);
      const f32x4 v = *(const f32x4*)(p + j * a.prows * a.D);
      total += wj;
      sum += wj == 0.f ? f32x4{} : v * wj;
    }
  }
  const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
  int64_t bh, i, b, h;
  split_row(row, a.Sq, bh, i);
  split_row(bh, a.heads, b, h);
  if (d < a.D) T::store4(a.O + b * a.ob + h * a.oh + i * a.os + d * T::ESZ, sum * inv);
  if (d == 0 && a.lse) a.lse[row] = (m + __builtin_amdgcn_logf(total)) * 0.69314718055994531f;
}

// ------------------------------------------------------------------- host

// How one set of keys is gone over: narrow or wide, row tiles, key ranges.
struct Plan {
  bool narrow;
  int tiles, nsplit;
  int64_t chunk;
};
Plan fwd_plan(int dtype, int64_t units, int64_t rows, int64_t keys, int64_t wide_want,
              int64_t wide_least);
int launch_fwd(int dtype, const Plan& p, FwdArgs a, hipStream_t st);
int launch_fwd_joint(int dtype, FwdArgs a, const FwdArgs& first, hipStream_t st);
int launch_fwd_two(int dtype, const Plan& pa, FwdArgs a, const Plan& pb, FwdArgs b, hipStream_t st);
int launch_combine(int dtype, const CombineArgs& a, hipStream_t st);

// f(tile) for the operands' type and head_dim.
template <typename F>
int with_tile(int dtype, int64_t D, F&& f) {
  if (dtype == TSP_BF16)
    return D > 96 ? f(Tile16<__bf16, 128>{}) : D > 64 ? f(Tile16<__bf16, 128, 96>{}) : f(Tile16<__bf16, 64>{});
  if (dtype == TSP_F16)
    return D > 96 ? f(Tile16<_Float16, 128>{}) : D > 64 ? f(Tile16<_Float16, 128, 96>{}) : f(Tile16<_Float16, 64>{});
  return D > 96 ? f(Tile32<128>{}) : D > 64 ? f(Tile32<128, 96>{}) : f(Tile32<64>{});
}

// Checks of one strided operand; 0 or a status with a message.
int check_operand(const char* who, const char* name, const void* p, const int64_t* strides, int64_t rows, int64_t D,
                  int dtype);
inline int esize(int dtype) { return dtype == TSP_F32 ? 4 : 2; }
// One row's stride is not the caller's: a stage of it goes on behind the row, where
// offsets have to pass the end of the stage's buffer to read as zero.
inline int64_t row_stride(const int64_t* strides, int64_t rows, int64_t D) { return rows > 1 ? strides[2] : D; }
inline Operand operand(const void* p, const int64_t* strides, int64_t rows, int64_t D, int dtype) {
  const int e = esize(dtype);
  return Operand{(const char*)p, strides[0] * e, strides[1] * e, row_stride(strides, rows, D) * e};
}

}  // namespace xat
}  // namespace tsp
