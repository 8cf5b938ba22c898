// Cross attention backward for gfx950, from the forward's output O and its
// rows' log-sum-exps (cross_attention.hip). Per batch entry, query head and its
// key head, over keys j < key_lengths[b]:
//   D_i   = sum_d dO_id O_id
//   P_ij  = exp(scale Q_i . K_j - lse_i),  dS_ij = P_ij (dO_i . V_j - D_i)
//   dQ_i  = scale sum_j dS_ij K_j
//   dK_j  = scale sum_{g, i} dS_ij Q_i,  dV_j = sum_{g, i} P_ij dO_i
// with the sums of dK and dV over the query heads g of the key head's group.
// No counterpart in the reference, whose attention is one sequence's over
// itself (trnsparse/ops.py:360-473).
//
//   row_pass     128 rows of a unit to a workgroup (rows and units as in
//                xattn_fwd.h), a wavefront to 32 with their Q and dO in
//                registers; K and V stages stream through LDS.
//   column_pass  128 keys of a unit to a workgroup, a wavefront to 32 with
//                their K and V in registers; the Q and dO rows of all heads of
//                the group stream through LDS with their rows' two numbers,
//                log2(e) lse (less P_EXP) and D.
//   both_passes  the two as one launch: 16-bit types without FINE.
//   row_stats    leaves the rows' numbers ahead of both_passes, and in fp16
//                ahead of the separate passes too, with the largest |dO| and
//                |V| (else the row pass leaves the numbers for the column pass).
// S and dO V^T are formed in both passes (7 products instead of 5) so that
// neither adds across workgroups: results do not depend on any order of
// arrival. Where a pass has few workgroups its inner axis is split, each part
// writes fp32 and sum_parts adds them in order.
#include "xattn_fwd.h"

namespace tsp {
namespace xat {

int check_sizes(const char* who, int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t L, int64_t D);

namespace {

// P enters dV's product as 2^P_EXP P. In fp16 that fills the type's range: P of n
// keys is about 1 / n, and from 2^-14 down fp16 has a fixed step of 2^-24 (131072
// keys: dV off by 1.3e-3 of its norm as P itself, 2.9e-4 this way; its own
// rounding 2.1e-4). P <= 1, so 2^15 P stays finite.
template <typename T>
constexpr int P_EXP = T::SHORT_RANGE ? 15 : 0;

// And dS, in fp16, as c dS: the power of two that brings what dS can be to just
// below 2^15. |dS_ij| <= P_ij (|dO_i . V_j| + |D_i|) <= 2 head_dim max |dO| max
// |V|, whatever the scores. So no loss scale and no size of V takes dS out of
// fp16's range, and of many keys it keeps its digits (131072 keys: dQ and dK off
// by 7e-4 of their norms with dO near 1 alone; 3e-4 this way). The launch that
// finds the two sizes is 3 us of a small step (8 x 8 heads of 128 x 128 x 64 17.8 ->
// 20.7 us), 1 to 2 % of a large one.
__device__ inline float ds_scale(float dO, float V, int D) { return unit_scale(2.f * D * dO * V) * 16384.f; }

struct BwdArgs {
  FwdArgs f;           // Q, K, V, lengths and sizes; tiles, nsplit, chunk of the row pass
  Operand O, dO;
  Operand dQ, dK, dV;  // written
  const float* lse;
  float *stat;         // (2, rows): log2(e) lse - P_EXP, D
  float *gmax, *vmax;  // fp16: (units, tiles, 4) largest |dO| of 32 rows, (units, vparts) |V| of vkeys keys
  int vparts;
  int64_t vkeys;
  float *qpart;        // (nsplit, rows, D), null with one range
  float *kpart;        // (ksplit, 2, batch * kv_heads * keys, D), null with one range
  int ktiles, ksplit, per;  // column pass: key tiles, ranges of `per` stages
  float scale;
};

// Largest |V| of a unit's valid keys.
__device__ inline float largest_value(const BwdArgs& b, int64_t unit) {
  const int lane = threadIdx.x & 63;
  float mx = lane < b.vparts ? b.vmax[unit * b.vparts + lane] : 0.f;  // (at most 64 parts)
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  return mx;
}

// FINE: P and dS as sums of two 16-bit numbers (see fine() below). STATS: forms
// and leaves the rows' numbers itself (else row_stats has left them).
template <typename T, int NT, bool FINE, bool STATS>
struct RowPass {
  static constexpr int HK = 32 * NT, HBYTES = HK * T::ROWB, STAGE = 2 * HBYTES, LDS = 2 * STAGE;
  static __device__ inline void run(const BwdArgs& b, uint32_t block, uint8_t* lds);
};
template <typename T, int NT, bool FINE, bool STATS>
__device__ inline void RowPass<T, NT, FINE, STATS>::run(const BwdArgs& b, uint32_t block, uint8_t* lds) {
  const FwdArgs& a = b.f;
  Item it;
  if (!item_of(a, block, a.tiles, a.nsplit, it)) return;
  const int tile = it.tile, split = it.split;
  const int64_t ub = longest_first(a, it.ub), hk = it.hk, unit = ub * a.Hkv + hk;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, l32 = lane & 31;
  const int r = tile * 128 + w * 32 + l32;
  const bool live = r < a.R, some = tile * 128 + w * 32 < a.R;
  const RowId id = row_id(a, ub, hk, live ? r : 0);
  auto row_of = [&](const Operand& x) { return x.p + id.b * x.b + id.head * x.h + id.i * x.s; };

  const int64_t n = unit_length(a, ub);
  const int64_t k0 = split * a.chunk, k1 = k0 + a.chunk < n ? k0 + a.chunk : n;
  const int nst = k1 > k0 ? (int)ceil_div(k1 - k0, HK) : 0;
  const bool short_rows = FINE && a.nsplit == 1 && nst == 1;
  const char* Kp = a.K.p + ub * a.K.b + hk * a.K.h;
  const char* Vp = a.V.p + ub * a.V.b + hk * a.V.h;
  Stager<T, HK, 4> ks, vs;
  ks.init(w, lane, a.K.s, a.D);
  vs.init(w, lane, a.V.s, a.D);
  const typename T::Lane ln = T::lane_of(lane);
  const uint32_t lds0 = dma::lds_addr(lds);
  auto issue = [&](int s) {
    const uint32_t st = lds0 + (s & 1) * STAGE;
    ks.issue(Kp, k0 + (int64_t)s * HK, k1, a.K.s, a.D, st, w);
    vs.issue(Vp, k0 + (int64_t)s * HK, k1, a.V.s, a.D, st + HBYTES, w);
  };
  if (nst > 0) issue(0);
  typename T::Rows q, g;
  T::load(q, row_of(a.Q), live, a.D, h);
  T::load(g, row_of(b.dO), live, a.D, h);
  float Dr, rq, out_scale = b.scale;
  if constexpr (!STATS) {
    rq = live ? b.stat[id.orow] + P_EXP<T> : 0.f;
    Dr = live ? b.stat[a.prows + id.orow] : 0.f;
  } else {
    typename T::Rows o;
    T::load(o, row_of(b.O), live, a.D, h);
    Dr = halves_sum(T::dot(g, o));
    rq = live ? b.lse[id.orow] * LOG2E : 0.f;
    if (live && split == 0 && h == 0) {
      b.stat[id.orow] = rq - P_EXP<T>;
      if (!short_rows) b.stat[a.prows + id.orow] = Dr;
    }
  }
  float back = 1.f;  // of dS's scale
  if constexpr (T::SHORT_RANGE) {  // c P in place of P: one factor for a row
    const float c = ds_scale(halves_max(T::largest(g)), largest_value(b, unit), a.D);
    rq -= (float)((int)(__float_as_uint(c) >> 23) - 127);
    back = unit_scale(c);
    out_scale = b.scale * back;
  }
  f32x16 acc[T::NU];
#pragma unroll
  for (int u = 0; u < T::NU; ++u) acc[u] = f32x16{};
  for (int s = 0; s < nst; ++s) {
    dma::wait_vm<0>();
    dma::barrier();
    if (s + 1 < nst) issue(s + 1);
    if (!some) continue;
    const int keys = (int)(k1 - k0 - (int64_t)s * HK < HK ? k1 - k0 - (int64_t)s * HK : HK);
    const uint32_t st = lds0 + (s & 1) * STAGE;
    f32x16 sc[NT], dp[NT];
    T::template scores<NT>(sc, st, ln, q);
    T::template scores<NT>(dp, st + HBYTES, ln, g);
    if (short_rows) {
      // All of the row's keys are here: D = sum_j P_ij dP_ij, without the
      // rounding of O, which of few keys is as large as dS (7 keys in bf16: dQ
      // 1.6 times as far off as its own rounding, 1.4 this way).
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][v], a.scale_log2, -rq));
          if (32 * t + 8 * (v >> 2) + 4 * h + (v & 3) < keys) sum += p * dp[t][v];
        }
      Dr = halves_sum(sum) * back;
      if (live && h == 0) b.stat[a.prows + id.orow] = Dr;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v)
        sc[t][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][v], a.scale_log2, -rq)) * (dp[t][v] - Dr);
    if (keys < HK) {  // staged rows past the last key are zero, but their P is not
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (32 * t + 8 * (v >> 2) + 4 * h + (v & 3) >= keys) sc[t][v] = 0.f;
    }
    T::template product<NT, FINE>(acc, st, ln, sc);
  }
  if (!live) return;
  char* out = (char*)row_of(b.dQ);
  float* part = b.qpart ? b.qpart + ((int64_t)split * a.prows + id.orow) * a.D : nullptr;
  T::quads(acc, h, [&](int d, f32x4 v) {
    if (d >= a.D) return;
    if (part)
      *(f32x4*)(part + d) = v * out_scale;
    else
      T::store4(out + d * T::ESZ, v * out_scale);
  });
}

template <typename T, int NQ, bool FINE>
struct ColumnPass {
  static constexpr int HQ = 32 * NQ, HBYTES = HQ * T::ROWB, STAGE = 2 * HBYTES + 1024;  // Q, dO, two numbers of each row
  static constexpr int LDS = 2 * STAGE;
  static __device__ inline void run(const BwdArgs& b, uint32_t block, uint8_t* lds);
};
template <typename T, int NQ, bool FINE>
__device__ inline void ColumnPass<T, NQ, FINE>::run(const BwdArgs& b, uint32_t block, uint8_t* lds) {
  const FwdArgs& a = b.f;
  Item it;
  if (!item_of(a, block, b.ktiles, b.ksplit, it)) return;
  const int tile = it.tile, split = it.split;
  const int64_t unit = it.unit, ub = it.ub, hk = it.hk;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, l32 = lane & 31;
  const int64_t n = unit_length(a, ub);
  const int64_t key = (int64_t)tile * 128 + w * 32 + l32;
  const bool some = (int64_t)tile * 128 + w * 32 < n;

  const int spg = (int)ceil_div(a.Sq, HQ), total = a.G * spg;  // stages of a head, of the group
  const int s0 = split * b.per, s1 = s0 + b.per < total ? s0 + b.per : total;
  const int nst = (int64_t)tile * 128 < n && s1 > s0 ? s1 - s0 : 0;
  Stager<T, HQ, 4> qs, gs;
  qs.init(w, lane, a.Q.s, a.D);
  gs.init(w, lane, b.dO.s, a.D);
  const typename T::Lane ln = T::lane_of(lane);
  const uint32_t lds0 = dma::lds_addr(lds);
  auto issue = [&](int s) {
    const int g = (s0 + s) / spg, i0 = ((s0 + s) - g * spg) * HQ;
    const int64_t head = hk * a.G + g;
    const uint32_t st = lds0 + (s & 1) * STAGE;
    qs.issue(a.Q.p + ub * a.Q.b + head * a.Q.h, i0, a.Sq, a.Q.s, a.D, st, w);
    gs.issue(b.dO.p + ub * b.dO.b + head * b.dO.h, i0, a.Sq, b.dO.s, a.D, st + HBYTES, w);
    if (w < 2) {  // rows past the last one: both numbers zero, so a finite P meets dO = 0 and dS = 0
      const float* x = b.stat + w * a.prows + (ub * a.Hkv * a.G + head) * a.Sq + i0;
      const int left = a.Sq - i0;
      dma::buffer4(dma::make_rsrc(x, 4u * (left < HQ ? left : HQ)), 4u * lane, st + 2 * HBYTES + w * 256);
    }
  };
  if (nst > 0) issue(0);
  typename T::Rows k, v;
  T::load(k, a.K.p + ub * a.K.b + hk * a.K.h + key * a.K.s, key < n, a.D, h);
  T::load(v, a.V.p + ub * a.V.b + hk * a.V.h + key * a.V.s, key < n, a.D, h);
  constexpr float back = 1.f / (1 << P_EXP<T>);
  float cs = 1.f;  // makes dS of what P makes
  if constexpr (T::SHORT_RANGE) {  // one factor for the unit
    float mx = 0.f;
    for (int e = lane; e < a.tiles * 4; e += 64) mx = fmaxf(mx, b.gmax[unit * a.tiles * 4 + e]);
    mx = halves_max(mx);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    cs = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(ds_scale(mx, largest_value(b, unit), a.D) * back)));
  }
  f32x16 dk[T::NU], dv[T::NU];
#pragma unroll
  for (int u = 0; u < T::NU; ++u) dk[u] = dv[u] = f32x16{};
  for (int s = 0; s < nst; ++s) {
    dma::wait_vm<0>();
    dma::barrier();
    if (s + 1 < nst) issue(s + 1);
    if (!some) continue;
    const uint32_t st = lds0 + (s & 1) * STAGE;
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      const uint32_t at = st + 32 * t * T::ROWB;
      f32x16 sc[1], dp[1];
      T::template scores<1>(sc, at, ln, k);
      T::template scores<1>(dp, at + HBYTES, ln, v);
      typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t sa = st + 2 * HBYTES + 4 * (32 * t + 8 * x + 4 * h);
        const f32x4 rq = *(const lds_f32x4*)(uintptr_t)sa, Dr = *(const lds_f32x4*)(uintptr_t)(sa + 256);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[0][4 * x + e], a.scale_log2, -rq[e]));
          sc[0][4 * x + e] = p;
          const float ds = p * (dp[0][4 * x + e] - Dr[e]);
          dp[0][4 * x + e] = T::SHORT_RANGE ? ds * cs : ds;
        }
      }
      T::template product<1, FINE>(dv, at + HBYTES, ln, sc);
      T::template product<1, FINE>(dk, at, ln, dp);
    }
  }
  if (key >= a.L) return;
  const bool in = key < n;
  char* ok = (char*)b.dK.p + ub * b.dK.b + hk * b.dK.h + key * b.dK.s;
  char* ov = (char*)b.dV.p + ub * b.dV.b + hk * b.dV.h + key * b.dV.s;
  const int64_t krows = (int64_t)a.units_b * a.Hkv * a.L, row = unit * a.L + key;
  float* pk = b.kpart ? b.kpart + ((int64_t)split * 2 * krows + row) * a.D : nullptr;
  auto put = [&](const f32x16* acc, char* o, float* p, float f) {
    T::quads(acc, h, [&](int d, f32x4 x) {
      if (d >= a.D) return;
      const f32x4 y = in ? x * f : f32x4{};
      if (p)
        *(f32x4*)(p + d) = y;
      else
        T::store4(o + d * T::ESZ, y);
    });
  };
  put(dk, ok, pk, b.scale * (T::SHORT_RANGE ? unit_scale(cs) * back : 1.f));
  put(dv, ov, pk ? pk + krows * a.D : nullptr, back);
}

// (fp32 at 128: Q, dO and dQ alone take 192 registers of a lane)
template <typename T, int NT, bool FINE>
__global__ __launch_bounds__(256, T::ROWB > 256 || FINE ? 1 : 2) void row_pass(const BwdArgs b) {
  typedef RowPass<T, NT, FINE, !T::SHORT_RANGE> R;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[R::LDS];
  R::run(b, blockIdx.x, lds);
}
template <typename T, int NQ, bool FINE>
__global__ __launch_bounds__(256, T::ESZ == 4 || FINE ? 1 : 2) void column_pass(const BwdArgs b) {
  typedef ColumnPass<T, NQ, FINE> C;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[C::LDS];
  C::run(b, blockIdx.x, lds);
}
// Both passes in one launch, the column pass' workgroups (the longer) first:
// with lengths of their own the key tiles are never a whole number to a CU, and
// the row pass fills what they leave. bf16, 4 x 32 heads of 128 over 8, 1024 rows
// x 2048 keys: lengths of 700 to 1800 take 316 us this way, 359 as two launches;
// all of 2048, 474 and 469; 2 x 16 heads of 64, 2048 x 2048: 131 and 134.
template <typename T, int N>
__global__ __launch_bounds__(256, 2) void both_passes(const BwdArgs b, uint32_t columns) {
  typedef RowPass<T, N, false, false> R;
  typedef ColumnPass<T, N, false> C;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[C::LDS > R::LDS ? C::LDS : R::LDS];
  if (blockIdx.x < columns)
    C::run(b, blockIdx.x, lds);
  else
    R::run(b, blockIdx.x - columns, lds);
}

// The rows' two numbers ahead of the passes: 16 lanes to a row, 32 rows of a unit
// to a workgroup. fp16: also their largest |dO|, and behind those workgroups
// vparts for each unit's largest |V|.
template <typename T>
__global__ __launch_bounds__(256) void row_stats(const BwdArgs b) {
  static_assert(T::ESZ == 2, "8 elements to a lane");
  typedef typename T::elem vec8 __attribute__((ext_vector_type(8)));
  const FwdArgs& a = b.f;
  const uint32_t chunks = 4u * a.tiles, row_wgs = (uint32_t)a.units_b * a.Hkv * chunks;
  const int lane = threadIdx.x & 15, d = 8 * lane;
  float mx = 0.f;
  auto largest = [&](vec8 x) {
#pragma unroll
    for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf((float)x[e]));
  };
  if (blockIdx.x < row_wgs) {
    const uint32_t unit = blockIdx.x / chunks, chunk = blockIdx.x - unit * chunks;
    const uint32_t ub = unit / (uint32_t)a.Hkv, hk = unit - ub * (uint32_t)a.Hkv;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r = (int)chunk * 32 + 16 * k + (threadIdx.x >> 4);
      if (r >= a.R) continue;
      const RowId id = row_id(a, ub, hk, r);
      vec8 g = vec8{}, o = vec8{};
      if (d < a.D) {
        g = *(const vec8*)(b.dO.p + id.b * b.dO.b + id.head * b.dO.h + id.i * b.dO.s + 2 * d);
        o = *(const vec8*)(b.O.p + id.b * b.O.b + id.head * b.O.h + id.i * b.O.s + 2 * d);
      }
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += (float)g[e] * (float)o[e];
      if constexpr (T::SHORT_RANGE) largest(g);
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) sum += __shfl_xor(sum, x, 64);
      if (lane == 0) {
        b.stat[id.orow] = b.lse[id.orow] * LOG2E - P_EXP<T>;
        b.stat[a.prows + id.orow] = sum;
      }
    }
  } else if constexpr (T::SHORT_RANGE) {
    const uint32_t i = blockIdx.x - row_wgs, unit = i / (uint32_t)b.vparts, part = i - unit * (uint32_t)b.vparts;
    const uint32_t ub = unit / (uint32_t)a.Hkv, hk = unit - ub * (uint32_t)a.Hkv;
    const int64_t n = unit_length(a, ub), k0 = part * b.vkeys, k1 = k0 + b.vkeys < n ? k0 + b.vkeys : n;
    const char* V = a.V.p + ub * a.V.b + hk * a.V.h + 2 * d;
    if (d < a.D)
      for (int64_t k = k0 + (threadIdx.x >> 4); k < k1; k += 16) largest(*(const vec8*)(V + k * a.V.s));
  }
  if constexpr (T::SHORT_RANGE) {
    __shared__ float top[4];
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor(mx, x, 64));
    if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = mx;
    __syncthreads();
    if (threadIdx.x == 0)
      *(blockIdx.x < row_wgs ? b.gmax + blockIdx.x : b.vmax + (blockIdx.x - row_wgs)) =
          fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  }
}

// Sums of the parts of each result's rows in order, rounded once: 32 lanes to a
// row; blockIdx.y is the result (dQ, dK, dV; no rows where there is one part).
struct SumArgs {
  const float* part;
  int64_t rows, stride;  // floats between parts
  int nsplit, heads;
  int64_t S;
  Operand out;
};
struct SumsArgs {
  SumArgs of[3];
  int D;
};
template <typename T>
__global__ __launch_bounds__(256) void sum_parts(const SumsArgs all) {
  const SumArgs& a = all.of[blockIdx.y];
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int d = 4 * (threadIdx.x & 31);
  if (row >= a.rows || d >= all.D) return;
  f32x4 sum = f32x4{};
#pragma unroll 4
  for (int j = 0; j < a.nsplit; ++j) sum += *(const f32x4*)(a.part + j * a.stride + row * all.D + d);
  int64_t bh, i, b, h;
  split_row(row, a.S, bh, i);
  split_row(bh, a.heads, b, h);
  T::store4((char*)a.out.p + b * a.out.b + h * a.out.h + i * a.out.s + d * T::ESZ, sum);
}

struct BwdPlan {
  int tiles, nsplit, ktiles, ksplit, per, vparts;
  int64_t chunk, vkeys;
  int64_t stat, gmax, vmax, qpart, kpart;  // bytes
  int64_t bytes() const { return stat + gmax + vmax + qpart + kpart; }
};
// Ranges for 512 workgroups, where there are less than half of that. An fp32
// workgroup has a CU to itself, so one round of them is 256 and the ranges are as
// many as fit (2 x 8 heads of 512 x 512 x 128 108 us, for 512 workgroups 142; 12
// heads over 4 of 1000 x 200 x 64 52 and 66) - but not of a padded batch. Its
// lengths, which the host does not know, leave ranges empty, and one round then
// takes as long as its longest: with entries a quarter to all full, 3 x 6 heads of
// 700 x 900 x 96 take 190 to 210 us, in one round 279; 3 x 8 of 257 x 383 x 80 with
// an empty one 65 to 71 and 75. What a batch whose entries are all full pays for that: 2 x 8 heads of 512
// x 512 x 128 141 us for 109, 2 x 4 over 2 of 300 x 2000 x 128 160 for 126, 3 x 6 of
// 700 x 900 x 96 the same. Padded batches never take fewer ranges, so the workspace
// that does for them does for all.
BwdPlan bwd_plan(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t L, int64_t D, bool lengths) {
  BwdPlan p{};
  const int64_t G = Hq / Hkv, units = B * Hkv, stage = dtype == TSP_F32 ? 32 : 64;
  const auto ranges = [&](int64_t wgs) {
    if (wgs == 0 || wgs >= 256) return int64_t(1);
    return dtype == TSP_F32 && !lengths ? 256 / wgs : ceil_div(512, wgs);
  };
  p.tiles = (int)ceil_div(G * Sq, 128);
  int64_t n = ranges(units * p.tiles);
  const int64_t kst = ceil_div(L > 0 ? L : 1, stage);  // stages of keys
  if (n > kst / 2) n = kst / 2 > 1 ? kst / 2 : 1;
  p.chunk = ceil_div(kst, n) * stage;
  p.nsplit = (int)ceil_div(L > 0 ? L : 1, p.chunk);
  p.ktiles = (int)ceil_div(L, 128);
  const int64_t total = G * ceil_div(Sq, stage);
  n = ranges(units * p.ktiles);
  if (n > total / 2) n = total / 2 > 1 ? total / 2 : 1;
  p.per = (int)ceil_div(total, n);
  p.ksplit = (int)ceil_div(total, p.per > 0 ? p.per : 1);
  if (p.ksplit < 1) p.ksplit = 1;
  const int64_t rows = B * Hq * Sq, up = 255;
  p.stat = (2 * rows * 4 + up) & ~up;
  // the largest |V| of a unit in at most 64 parts, one to a lane of what reads them
  p.vkeys = ceil_div(L > 0 ? L : 1, 64);
  if (p.vkeys < 64) p.vkeys = 64;
  p.vparts = (int)ceil_div(L > 0 ? L : 1, p.vkeys);
  p.gmax = dtype == TSP_F16 ? (units * p.tiles * 16 + up) & ~up : 0;
  p.vmax = dtype == TSP_F16 ? (units * p.vparts * 4 + up) & ~up : 0;
  p.qpart = p.nsplit > 1 ? (p.nsplit * rows * D * 4 + up) & ~up : 0;
  p.kpart = p.ksplit > 1 ? p.ksplit * 2 * units * L * D * 4 : 0;
  return p;
}

template <typename T>
int sums(const BwdPlan& p, const BwdArgs& b, bool columns, hipStream_t st) {
  const FwdArgs& a = b.f;
  const int64_t units = (int64_t)a.units_b * a.Hkv;
  const int64_t krows = units * a.L, qsum = p.nsplit > 1 ? a.prows : 0, ksum = p.ksplit > 1 && columns ? krows : 0;
  const int64_t most = qsum > ksum ? qsum : ksum;
  if (most == 0) return TSP_OK;
  SumsArgs s{};
  s.D = a.D;
  s.of[0] = SumArgs{b.qpart, qsum, a.prows * a.D, p.nsplit, a.Hkv * a.G, a.Sq, b.dQ};
  s.of[1] = SumArgs{b.kpart, ksum, 2 * krows * a.D, p.ksplit, a.Hkv, a.L, b.dK};
  s.of[2] = SumArgs{b.kpart + krows * a.D, ksum, 2 * krows * a.D, p.ksplit, a.Hkv, a.L, b.dV};
  hipLaunchKernelGGL((sum_parts<T>), dim3((unsigned)ceil_div(most, 8), 3), dim3(256), 0, st, s);
  return check_launch("sum_parts launch");
}

// P and dS rounded to 16 bits move a gradient as far as the rounding of its
// result does: 1.41 times the error of that alone, of few rows or keys up to
// 1.6. A sum of two 16-bit numbers leaves the result's own, for 4 products in
// place of 3 in the row pass and 6 of 4 in the column pass. That is taken where
// the matrix cores are not what a step waits for: 2 x 16 heads of 256 x 512 x
// 128 45.9 us and 47.4 this way, 4 x 16 heads (2^30 products of the scores) 50.7
// and 59.8, 4 x 32 heads of 4096 x 32 x 128 293.5 and 293.6.
bool fine(int64_t rows, int64_t L, int64_t D) { return L <= 64 || rows * L <= (int64_t(1) << 29) / D; }

template <typename T, bool FINE>
int run_t(const BwdPlan& p, const BwdArgs& b, hipStream_t st) {
  const FwdArgs& a = b.f;
  const int64_t units = (int64_t)a.units_b * a.Hkv;
  constexpr int N = T::ESZ == 2 ? 2 : 1;
  const int64_t g1 = head_grid((int64_t)p.tiles * p.nsplit, units), g2 = b.dK.p ? head_grid((int64_t)p.ktiles * p.ksplit, units) : 0;
  if (g1 > INT32_MAX || g2 > INT32_MAX) return fail(TSP_EUNSUPPORTED, "tsp_cross_attn_bwd: too large a grid");
  int rc;
  if constexpr (T::ESZ == 2) {
    const bool both = !FINE && g2 > 0 && g1 + g2 <= INT32_MAX;
    if (both || T::SHORT_RANGE) {
      const int64_t g0 = units * (4 * p.tiles + (T::SHORT_RANGE ? p.vparts : 0));
      if (g0 > INT32_MAX) return fail(TSP_EUNSUPPORTED, "tsp_cross_attn_bwd: too large a grid");
      hipLaunchKernelGGL((row_stats<T>), dim3((unsigned)g0), dim3(256), 0, st, b);
      if ((rc = check_launch("row_stats launch"))) return rc;
    }
    if constexpr (!FINE)
      if (both) {
        hipLaunchKernelGGL((both_passes<T, N>), dim3((unsigned)(g1 + g2)), dim3(256), 0, st, b, (uint32_t)g2);
        if ((rc = check_launch("both_passes launch"))) return rc;
        return sums<T>(p, b, g2 > 0, st);
      }
  }
  hipLaunchKernelGGL((row_pass<T, N, FINE>), dim3((unsigned)g1), dim3(256), 0, st, b);
  if ((rc = check_launch("row_pass launch"))) return rc;
  if (g2 > 0) {
    hipLaunchKernelGGL((column_pass<T, N, FINE>), dim3((unsigned)g2), dim3(256), 0, st, b);
    if ((rc = check_launch("column_pass launch"))) return rc;
  }
  return sums<T>(p, b, g2 > 0, st);
}

// zeros in a strided result
struct ZeroArgs {
  Operand out;
  int64_t rows, S;
  int heads, bytes;  // of a row
};
__global__ __launch_bounds__(256) void zero_rows(const ZeroArgs a) {
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= a.rows) return;
  const int64_t i = row % a.S, bh = row / a.S;
  char* p = (char*)a.out.p + bh / a.heads * a.out.b + bh % a.heads * a.out.h + i * a.out.s;
  for (int d = 16 * (threadIdx.x & 31); d < a.bytes; d += 512) *(u32x4*)(p + d) = u32x4{};
}

}  // namespace
}  // namespace xat
}  // namespace tsp

using namespace tsp;

extern "C" int64_t tsp_cross_attn_bwd_workspace_size(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq,
                                                     int64_t L, int64_t D) {
  if (xat::check_sizes("tsp_cross_attn_bwd_workspace_size", dtype, B, Hq, Hkv, Sq, L, D)) return -1;
  if (B * Hq * Sq == 0) return 0;
  return xat::bwd_plan(dtype, B, Hq, Hkv, Sq, L, D, true).bytes();
}

extern "C" int tsp_cross_attn_bwd(const void* Q, const int64_t* qs, const void* K, const int64_t* ks, const void* V,
                                  const int64_t* vs, const void* O, const int64_t* os, const void* dO,
                                  const int64_t* gs, const float* lse, int dtype, int64_t B, int64_t Hq, int64_t Hkv,
                                  int64_t Sq, int64_t L, int64_t D, const void* key_lengths, int index_type,
                                  double scale, void* dQ, const int64_t* dqs, void* dK, const int64_t* dks, void* dV,
                                  const int64_t* dvs, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "tsp_cross_attn_bwd";
  const hipStream_t st = (hipStream_t)stream;
  int rc = xat::check_sizes(who, dtype, B, Hq, Hkv, Sq, L, D);
  if (rc) return rc;
  if (!(scale > 1e-30) || !(scale < 1e30)) return fail(TSP_EINVAL, "%s: scale must be positive", who);
  if (index_type != TSP_I32 && index_type != TSP_I64) return fail(TSP_EINVAL, "%s: bad index type", who);
  const bool rows = B * Hq * Sq > 0, keys = B * L > 0, cols = keys && (dK || dV);
  if (cols)
    if ((rc = xat::check_operand(who, "dK", dK, dks, L, D, dtype)) ||
        (rc = xat::check_operand(who, "dV", dV, dvs, L, D, dtype)))
      return rc;
  if (!rows) {  // no query: the keys' gradients are zero
    if (!cols) return TSP_OK;
    const int64_t n = B * Hkv * L;
    for (const xat::Operand& o : {xat::operand(dK, dks, L, D, dtype), xat::operand(dV, dvs, L, D, dtype)}) {
      const xat::ZeroArgs z{o, n, L, (int)Hkv, (int)(D * xat::esize(dtype))};
      if (ceil_div(n, 8) > INT32_MAX) return fail(TSP_EUNSUPPORTED, "%s: too many rows", who);
      hipLaunchKernelGGL(xat::zero_rows, dim3((unsigned)ceil_div(n, 8)), dim3(256), 0, st, z);
      if ((rc = check_launch("zero_rows launch"))) return rc;
    }
    return TSP_OK;
  }
  if ((rc = xat::check_operand(who, "Q", Q, qs, Sq, D, dtype)) || (rc = xat::check_operand(who, "O", O, os, Sq, D, dtype)) ||
      (rc = xat::check_operand(who, "dO", dO, gs, Sq, D, dtype)) ||
      (rc = xat::check_operand(who, "dQ", dQ, dqs, Sq, D, dtype)))
    return rc;
  if (keys)
    if ((rc = xat::check_operand(who, "K", K, ks, L, D, dtype)) || (rc = xat::check_operand(who, "V", V, vs, L, D, dtype)))
      return rc;
  if (!lse) return fail(TSP_EINVAL, "%s: null lse", who);
  const xat::BwdPlan p = xat::bwd_plan(dtype, B, Hq, Hkv, Sq, L, D, key_lengths != nullptr);
  if (!workspace || workspace_bytes < p.bytes())
    return fail(TSP_EINVAL, "%s: workspace too small", who);
  if (ceil_div(B * Hq * Sq, 8) > INT32_MAX || ceil_div(B * Hkv * L, 8) > INT32_MAX)
    return fail(TSP_EUNSUPPORTED, "%s: too many rows", who);
  const int64_t none[3] = {0, 0, 0};
  xat::BwdArgs b{};
  xat::FwdArgs& a = b.f;
  a.Q = xat::operand(Q, qs, Sq, D, dtype);
  a.K = xat::operand(K, keys ? ks : none, L, D, dtype);
  a.V = xat::operand(V, keys ? vs : none, L, D, dtype);
  b.O = xat::operand(O, os, Sq, D, dtype);
  b.dO = xat::operand(dO, gs, Sq, D, dtype);
  b.dQ = xat::operand(dQ, dqs, Sq, D, dtype);
  b.dK = xat::operand(dK, cols ? dks : none, L, D, dtype);
  b.dV = xat::operand(dV, cols ? dvs : none, L, D, dtype);
  b.lse = lse;
  b.stat = (float*)workspace;
  char* at = (char*)workspace + p.stat;
  if (p.gmax) b.gmax = (float*)at;
  at += p.gmax;
  if (p.vmax) b.vmax = (float*)at;
  at += p.vmax;
  if (p.qpart) b.qpart = (float*)at;
  if (p.kpart) b.kpart = (float*)(at + p.qpart);
  b.vparts = p.vparts, b.vkeys = p.vkeys;
  b.ktiles = p.ktiles, b.ksplit = p.ksplit, b.per = p.per;
  b.scale = (float)scale;
  a.prows = B * Hq * Sq;
  a.lengths = key_lengths;
  a.len64 = index_type == TSP_I64;
  a.units_b = (int)B;
  a.Hkv = (int)Hkv, a.G = (int)(Hq / Hkv), a.Sq = (int)Sq, a.R = (int)(Hq / Hkv * Sq), a.D = (int)D;
  a.L = L;
  a.tiles = p.tiles, a.nsplit = p.nsplit, a.chunk = p.chunk;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  using namespace xat;
  const bool two = fine(a.prows, L, D);
  return with_tile(dtype, D, [&](auto tile) {
    typedef decltype(tile) T;
    if constexpr (T::ESZ == 2)
      if (two) return run_t<T, true>(p, b, st);
    return run_t<T, false>(p, b, st);
  });
}
