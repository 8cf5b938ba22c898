// Tiles of the dense attention kernels (cross attention, shared-prefix
// attention): bf16, fp16 and fp32 rows of up to DP (64 or 128) elements in
// strided tensors, staged into LDS by direct loads and read as MFMA operands.
//
// Every product has 32 "own" rows of the wavefront as its B operand (row
// l32 = lane % 32 in registers) and 32 staged rows as its A operand:
//   scores  C[staged row][own row] = sum_d X[staged row][d] Y[own row][d];
//           element v of lane half h is staged row 8 (v / 4) + 4 h + v % 4
//   outer   acc[d][own row] += sum_r X[staged row r][d] p[r][own row], with p
//           the lane's own score elements (no cross-lane move), X read through
//           transpose reads (16 bit) or as rows (fp32)
// so a softmax row lives in two lanes (l32 and l32 + 32).
//
// A stage is filled from a buffer resource whose base is the stage's first
// row and whose size ends with the last row that exists: rows past it, and
// elements past head_dim, read as zero, so nothing behind a sequence's end
// reaches a product, and offsets stay within 32 bits at any sequence length.
#pragma once

#include "attention_tiles.h"
#include "common.h"
#include "lds_dma.h"

#include <type_traits>

namespace tsp {
namespace xat {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr uint32_t OUT_OF_RANGE = 0x7ffffff0u;  // past any stage's buffer size
constexpr int64_t MAX_ROW_BYTES = int64_t(1) << 24;  // row stride: 64 rows stay below OUT_OF_RANGE

__device__ inline f32x16 mfma16(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ inline f32x16 mfma16(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// max / sum over lanes l and l ^ 32, in every lane
__device__ inline float halves_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float halves_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The power of two that brings x > 0 into [1, 2); 1 for zero, infinity and NaN.
__device__ inline float unit_scale(float x) {
  const uint32_t e = __float_as_uint(x) >> 23;
  return e == 0 || e >= 254 ? 1.f : __uint_as_float((254u - e) << 23);
}

// ---------------------------------------------------------------- 16 bit
// DP: elements of a staged row; DC: elements that the products go over (the
// ones behind are zero in every operand). head_dim 80 and 96 in rows of 128.
template <typename E, int DP_, int DC = DP_>
struct Tile16 {
  typedef E elem;
  typedef E vec8 __attribute__((ext_vector_type(8)));
  typedef E vec4 __attribute__((ext_vector_type(4)));
  static constexpr int DP = DP_, ESZ = 2, CE = 8;  // CE: elements of a 16-byte chunk
  static constexpr bool SHORT_RANGE = std::is_same<E, _Float16>::value;  // of exponents: 2^-24 to 2^16
  static constexpr int ROWB = DP * 2, CPR = ROWB / 16, KS = DC / 16, NU = DC / 32;
  struct Rows {
    vec8 f[KS];
  };
  __host__ __device__ static constexpr int swz(int r) { return abw::swz<DP>(r); }

  static __device__ inline void load(Rows& x, const char* p, bool ok, int D, int h) {
#pragma unroll
    for (int s = 0; s < KS; ++s) x.f[s] = ok && 16 * s + 8 * h < D ? *(const vec8*)(p + 32 * s + 16 * h) : vec8{};
  }
  static __device__ inline float dot(const Rows& a, const Rows& b) {
    float t = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) t += (float)a.f[s][i] * (float)b.f[s][i];
    return t;
  }

  static __device__ inline float largest(const Rows& a) {
    float t = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) t = fmaxf(t, fabsf((float)a.f[s][i]));
    return t;
  }

  // LDS addresses of one stage, formed once per stage
  struct Lane {
    uint32_t row;     // l32 * ROWB + (swz(l32) ^ h) chunks
    uint32_t t0, t1;  // the two transpose reads
  };
  static __device__ inline Lane lane_of(int lane) {
    const abw::TrLane t = abw::tr_lane<DP>(lane);
    const int l32 = lane & 31, h = lane >> 5;
    return Lane{(uint32_t)(l32 * ROWB + ((swz(l32) ^ h) << 4)), (uint32_t)(t.off[0] + (t.xu << 6)),
                (uint32_t)(t.off[1] + (t.xu << 6))};
  }
  template <int NT>
  static __device__ inline void scores(f32x16* c, uint32_t st, const Lane& ln, const Rows& y) {
    const uint32_t rb = st + ln.row;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int t = 0; t < NT; ++t)
        c[t] = mfma16(__builtin_bit_cast(vec8, abw::lds_row(rb, ks, 32 * t * ROWB)), y.f[ks],
                      ks == 0 ? f32x16{} : c[t]);
  }
  // p in the element's type, the k order of the B operand
  template <int NT>
  struct Prob {
    vec8 b[NT][2];
  };
  template <int NT>
  static __device__ inline void pack(Prob<NT>& o, const f32x16* p) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        f32x8 x;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = p[t][8 * a + i];
        o.b[t][a] = __builtin_convertvector(x, vec8);
      }
  }
  // p less what pack() kept of it
  template <int NT>
  static __device__ inline void rest(f32x16* p, const Prob<NT>& kept) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v) p[t][v] -= (float)kept.b[t][v >> 3][v & 7];
  }
  // acc += X^T p, and X^T rest, of X's tile at st
  template <int NT>
  static __device__ inline void outer(f32x16* acc, uint32_t st, const Lane& ln, const Prob<NT>& p,
                                      const Prob<NT>* rest = nullptr) {
    const uint32_t t0 = st + ln.t0, t1 = st + ln.t1;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          const vec8 x = __builtin_bit_cast(vec8, abw::lds_trp(t0, t1, u, (32 * t + 16 * a) * ROWB));
          acc[u] = mfma16(x, p.b[t][a], acc[u]);
          if (rest) acc[u] = mfma16(x, rest->b[t][a], acc[u]);
        }
  }
  // acc += X^T p, with p in 16 bits or (TWICE) as the sum of two such numbers
  template <int NT, bool TWICE>
  static __device__ inline void product(f32x16* acc, uint32_t st, const Lane& ln, f32x16* p) {
    Prob<NT> a, b;
    pack<NT>(a, p);
    if constexpr (TWICE) {
      rest<NT>(p, a);
      pack<NT>(b, p);
    }
    outer<NT>(acc, st, ln, a, TWICE ? &b : nullptr);
  }
  // f(d, four consecutive values at d) over the lane's part of its own row
  template <typename F>
  static __device__ inline void quads(const f32x16* acc, int h, F&& f) {
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        f(32 * u + 8 * g + 4 * h, f32x4{acc[u][4 * g], acc[u][4 * g + 1], acc[u][4 * g + 2], acc[u][4 * g + 3]});
  }
  static __device__ inline void store4(char* p, f32x4 v) { *(vec4*)p = __builtin_convertvector(v, vec4); }
};

// ------------------------------------------------------------------ fp32
template <int DP_, int DC = DP_>
struct Tile32 {
  typedef float elem;
  static constexpr int DP = DP_, ESZ = 4, CE = 4;
  static constexpr bool SHORT_RANGE = false;
  static constexpr int ROWB = DP * 4, CPR = ROWB / 16, KT = DC / 8, NU = DC / 32;
  // output rows: element r of subtile u is d = NU r + u, so that one read of NU
  // floats feeds NU products; with three, d = 32 u + r and a read to each
  static constexpr bool TOGETHER = NU != 3;
  struct Rows {
    f32x4 f[KT];
  };
  __host__ __device__ static constexpr int swz(int r) { return r & 15; }

  static __device__ inline void load(Rows& x, const char* p, bool ok, int D, int h) {
#pragma unroll
    for (int t = 0; t < KT; ++t) x.f[t] = ok && 8 * t + 4 * h < D ? *(const f32x4*)(p + 32 * t + 16 * h) : f32x4{};
  }
  static __device__ inline float dot(const Rows& a, const Rows& b) {
    float s = 0.f;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) s += a.f[t][i] * b.f[t][i];
    return s;
  }
  struct Lane {
    uint32_t row, kx;  // chunk reads
    uint32_t h, col;   // row reads: 4 h rows down, the lane's first byte
  };
  static __device__ inline Lane lane_of(int lane) {
    const int l32 = lane & 31, h = lane >> 5;
    return Lane{(uint32_t)(l32 * ROWB), (uint32_t)((l32 & 15) ^ h), (uint32_t)h, (uint32_t)((TOGETHER ? NU : 1) * 4 * l32)};
  }
  typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
  typedef typename abf::VRow<TOGETHER ? NU : 4>::type vrow;
  typedef __attribute__((address_space(3))) float lds_float;
  typedef __attribute__((address_space(3))) vrow lds_vrow;
  template <int NT>
  static __device__ inline void scores(f32x16* c, uint32_t st, const Lane& ln, const Rows& y) {
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const f32x4 a = *(const lds_f32x4*)(uintptr_t)(st + ln.row + 32 * n * ROWB + (((2 * t) ^ ln.kx) << 4));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          c[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], y.f[t][i], t == 0 && i == 0 ? f32x16{} : c[n], 0, 0, 0);
      }
  }
  template <int NT>
  struct Prob {
    f32x16 b[NT];
  };
  template <int NT>
  static __device__ inline void pack(Prob<NT>& o, const f32x16* p) {
#pragma unroll
    for (int t = 0; t < NT; ++t) o.b[t] = p[t];
  }
  template <int NT>
  static __device__ inline void outer(f32x16* acc, uint32_t st, const Lane& ln, const Prob<NT>& p) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int s = 0; s < 16; ++s) {
        const uint32_t r = 8 * (s >> 2) + 4 * ln.h + (s & 3);  // row % 16 decides the slot, 32 t does not
        vrow a;
        if constexpr (TOGETHER) {
          a = *(const lds_vrow*)(uintptr_t)(st + (32 * t + r) * ROWB +
                                            ((((ln.col >> 4) ^ (r & 15)) << 4) | (ln.col & 15)));
        } else {
#pragma unroll
          for (int u = 0; u < NU; ++u)
            a[u] = *(const lds_float*)(uintptr_t)(st + (32 * t + r) * ROWB +
                                                  (((8 * u + (ln.col >> 4)) ^ (r & 15)) << 4 | (ln.col & 15)));
        }
#pragma unroll
        for (int u = 0; u < NU; ++u) acc[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[u], p.b[t][s], acc[u], 0, 0, 0);
      }
  }
  template <int NT, bool>
  static __device__ inline void product(f32x16* acc, uint32_t st, const Lane& ln, f32x16* p) {
    Prob<NT> a;
    pack<NT>(a, p);
    outer<NT>(acc, st, ln, a);
  }
  template <typename F>
  static __device__ inline void quads(const f32x16* acc, int h, F&& f) {
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int k = 0; k < NU; ++k) {
        f32x4 t;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          t[e] = TOGETHER ? acc[(4 * k + e) % NU][4 * a + (4 * k + e) / NU] : acc[k][4 * a + e];
        f(TOGETHER ? NU * (8 * a + 4 * h) + 4 * k : 32 * k + 8 * a + 4 * h, t);
      }
  }
  static __device__ inline void store4(char* p, f32x4 v) { *(f32x4*)p = v; }
};

// ------------------------------------------------------------- staging
// One wavefront's share of a stage of ROWS rows filled by NW wavefronts:
// NI instructions of 1 KiB, the byte offsets of its lanes computed once.
template <typename T, int ROWS, int NW>
struct Stager {
  static constexpr int RPI = 64 / T::CPR, NI = ROWS * T::ROWB / 1024 / NW;
  static_assert(NI >= 1 && ROWS * T::ROWB == NI * 1024 * NW, "whole instructions per wavefront");
  uint32_t off[NI];
  __device__ inline void init(int w, int lane, int64_t row_bytes, int D) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = RPI * (NI * w + i) + lane / T::CPR, c = (lane % T::CPR) ^ T::swz(r);
      off[i] = c * T::CE < D ? (uint32_t)(r * row_bytes) + 16u * c : OUT_OF_RANGE;
    }
  }
  // rows [row0, min(row0 + ROWS, n)) of the tensor at `base` into LDS `dst`; n > row0
  __device__ inline void issue(const char* base, int64_t row0, int64_t n, int64_t row_bytes, int D, uint32_t dst,
                               int w) const {
    const int64_t left = n - row0, rows = left < ROWS ? left : ROWS;
    const dma::i32x4 rs =
        dma::make_rsrc(base + row0 * row_bytes, (uint32_t)((rows - 1) * row_bytes) + (uint32_t)(D * T::ESZ));
#pragma unroll
    for (int i = 0; i < NI; ++i) dma::buffer16(rs, off[i], dst + (NI * w + i) * 1024);
  }
};

// ------------------------------------------------- online softmax, one stage
// acc, m, l of the lane's own row over the staged keys: acc = sum 2^(s - m) V,
// l = this lane half's part of sum 2^(s - m), s = log2(e) * scale * score. m
// follows the running maximum only when that has moved by more than 8 (log2
// units), so 2^(s - m) <= 2^8 and acc is rarely rescaled; acc / l does not
// depend on m. In fp16, m lies 7 below the maximum that it follows, so that
// 2^(s - m) <= 2^15 takes up the type's range: from 2^-14 down it has a fixed step
// of 2^-24, and the many keys of a long row that one key outweighs lose digits
// together (one of weight 1 and 524287 of 2^-20.4 in one range: results off by
// 23 u, u = 2^-11; by less than 1.6 u this way).
// `keys` (with check): the staged keys that this row sees.
template <typename T>
struct RowState {
  f32x16 acc[T::NU];
  float m, l;
  __device__ inline void clear() {
#pragma unroll
    for (int u = 0; u < T::NU; ++u) acc[u] = f32x16{};
    m = -INFINITY;
    l = 0.f;
  }
};
// `between` runs once the scores have left the K stage, before V is read.
template <typename T, int NT, bool TWICE, typename F>
__device__ inline void softmax_stage(RowState<T>& r, const typename T::Rows& q, uint32_t kst, uint32_t vst,
                                     const typename T::Lane& ln, int h, float scale_log2, bool check, int keys,
                                     F&& between) {
  f32x16 s[NT];
  T::template scores<NT>(s, kst, ln, q);
  between();
  if (check) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v)
        if (32 * t + 8 * (v >> 2) + 4 * h + (v & 3) >= keys) s[t][v] = -INFINITY;
  }
  float mx = s[0][0];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int v = 0; v < 16; ++v) mx = fmaxf(mx, s[t][v]);
  mx = halves_max(mx) * scale_log2 - (T::SHORT_RANGE ? 7.f : 0.f);
  const bool move = mx > r.m + 8.f;
  if (__builtin_amdgcn_ballot_w64(move) != 0) {
    const float f = move ? (r.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(r.m - mx)) : 1.f;
    r.m = move ? mx : r.m;
    r.l *= f;
#pragma unroll
    for (int u = 0; u < T::NU; ++u) r.acc[u] *= f;
  }
  const float base = r.m == -INFINITY ? 0.f : -r.m;  // scores of -inf give 0 either way
  float sum = 0.f;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      s[t][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][v], scale_log2, base));
      sum += s[t][v];
    }
  r.l += sum;
  T::template product<NT, TWICE>(r.acc, vst, ln, s);
}

}  // namespace xat
}  // namespace tsp
