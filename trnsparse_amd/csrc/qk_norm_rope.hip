// RMS norm of query and key heads and the rotation by their tokens' positions,
// in one pass, for gfx950. For a head vector x of D elements, weight w and the
// token's position t:
//   r = 1 / sqrt(mean_d x_d^2 + eps),  n_d = x_d r w_d
//   (y_a, y_b) = (n_a cos p - n_b sin p, n_b cos p + n_a sin p),  p = t f_j
// for the pair (a, b) of every frequency f_j, j < rot / 2: (j, j + rot / 2), or
// (2 j, 2 j + 1) interleaved; elements from rot on are not rotated. Backward:
// dn is dy rotated back, dw = sum_rows dn x r and
//   dx_d = r (w_d dn_d - x_d r (r / D sum_e x_e w_e dn_e)).
// No counterpart in the reference, whose attention takes Q and K as they are
// (trnsparse/ops.py:549-625).
//
// Bound by memory: x in and y out once (backward: x and dy in, dx out). 2 x 8192
// tokens with 32 + 8 heads of 128 in bf16 take 74 us forward (4.6 TB/s, where a
// copy runs at 5.1) and 123 + 5 us backward (4.1 TB/s). A row is held by a group
// of lanes, each with two chunks of CE elements that hold whole pairs (chunk t
// of either half, or two chunks in a row), so rotation needs no other lane and
// the sums a few lane moves. A wavefront's groups take consecutive heads of one
// token: they lie together in a projection's output, and each lane forms the
// angles of one pair for all of them (every lane its own chunk's: 77 and 128
// us; without the next rows' loads ahead 95 and 147). Angles are products in 64
// bits, reduced to half turns there: a position of 10^6 would leave an fp32
// product no correct digit after the point. Sums and norms are fp32; a result is
// rounded once.
//
// Weight gradients: every workgroup sums its tokens' rows in registers and
// writes one part; wgrad_kernel adds the parts in a fixed order, so results do
// not change from run to run. Those of fp32 rows are summed in fp64: a chain of
// fp32 sums left them off by up to 2.1 times 2^-24 of their norm (1.0 to 1.5 this
// way; 2 x 4096 tokens with 32 + 8 heads of 128 take 181 us for 178, forward and
// backward). Those of 16-bit rows, whose own rounding is 2^-11 or 2^-8, stay fp32.
#include "common.h"

#include <type_traits>

namespace {

template <typename E, int CE>
struct alignas(sizeof(E) * CE) Chunk {
  E v[CE];
};

__device__ inline float widen(float x) { return x; }
__device__ inline float widen(__bf16 x) { return (float)x; }
__device__ inline float widen(_Float16 x) { return (float)x; }

struct Rows {
  const char* p;
  int64_t b, h, s;  // strides in bytes
};
struct Side {  // the query or the key heads
  Rows x, y, g;   // x; y (forward: written) or dx (backward: written); dy
  const void* w;
  int H;
};
struct Args {
  Side side[2];
  const void* pos;
  int64_t pos_b, pos_s;  // strides in elements
  int pos64, w32;        // positions are int64; weights are fp32 (else the rows' type)
  const double* freq;
  int S, D, rot, interleaved, need_w;
  int64_t tokens;
  int parts;   // forward: wavefronts to a token
  float eps;
  float* wpart;  // (workgroups, 2, D)
};

// Where the two chunks of lane t's pair of chunks start, and the first of their
// frequencies (-1: not rotated).
struct Place {
  int a, b, j;
  bool on;
};
template <int CE>
__device__ inline Place place(const Args& g, int t) {
  Place p;
  p.on = 2 * CE * t < g.D;
  const int half = g.rot / 2;
  if (g.interleaved) {
    p.a = 2 * CE * t;
    p.b = p.a + CE;
    p.j = p.a < g.rot ? p.a / 2 : -1;
  } else if (CE * t < half) {
    p.a = CE * t;
    p.b = half + CE * t;
    p.j = CE * t;
  } else {
    p.a = g.rot + 2 * (CE * t - half);
    p.b = p.a + CE;
    p.j = -1;
  }
  return p;
}

template <int CE>
struct Angles {
  float c[CE], s[CE];
  // Lane l forms the angles of pairs l and (J = 2) l + 64; the lanes of a row
  // take theirs from there, by way of __shfl. Whole wavefronts call this.
  static __device__ inline void form(const Args& g, int lane, int64_t b, int64_t i, float* c, float* s, int rounds) {
    const int64_t at = b * g.pos_b + i * g.pos_s;
    const double t = g.pos64 ? (double)((const int64_t*)g.pos)[at] : (double)((const int32_t*)g.pos)[at];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      c[k] = 1.f;
      s[k] = 0.f;
      if (k < rounds && lane + 64 * k < g.rot / 2) {
        // less whole turns, 2 pi in two parts: adds at most 2^-50 up to 2^53 turns.
        // (The product itself is off by 2^-53 of the angle.)
        double angle = t * g.freq[lane + 64 * k];
        const double turns = __builtin_rint(angle * 0.15915494309189535);
        angle = __builtin_fma(-turns, 6.283185307179586477, angle);
        angle = __builtin_fma(-turns, 2.449293598294706414e-16, angle);
        // in half turns, and what 32 bits leave of them to first order: 2^-24 of a
        // half turn would move a result by more than its own rounding
        const double halves = angle * 0.31830988618379067154;
        const float head = (float)halves, rest = (float)((halves - head) * 3.14159265358979323846);
        float c0, s0;
        sincospif(head, &s0, &c0);
        c[k] = c0 - rest * s0;
        s[k] = s0 + rest * c0;
      }
    }
  }
  __device__ inline void take(const Args& g, const Place& p, const float* fc, const float* fs) {
#pragma unroll
    for (int e = 0; e < CE; ++e) {
      const int j = p.j + e, from = j & 63;
      const float c0 = __shfl(fc[0], from, 64), s0 = __shfl(fs[0], from, 64);
      c[e] = c0;
      s[e] = s0;
      if (g.rot > 128) {
        const float c1 = __shfl(fc[1], from, 64), s1 = __shfl(fs[1], from, 64);
        c[e] = j < 64 ? c0 : c1;
        s[e] = j < 64 ? s0 : s1;
      }
      if (!p.on || p.j < 0 || j >= g.rot / 2) {
        c[e] = 1.f;
        s[e] = 0.f;
      }
    }
  }
  // forward (dir = 1) or back (dir = -1), of the chunk pair x[0 .. 2 CE)
  __device__ inline void turn(float* x, bool interleaved, float dir) const {
    auto pair = [&](float& a, float& b, int e) {
      const float sn = dir * s[e], na = a * c[e] - b * sn, nb = b * c[e] + a * sn;
      a = na;
      b = nb;
    };
    if (interleaved) {
      if constexpr (CE == 1) {
        pair(x[0], x[1], 0);
      } else {
#pragma unroll
        for (int e = 0; e < CE; ++e) pair(x[2 * e], x[2 * e + 1], e);
      }
    } else {
#pragma unroll
      for (int e = 0; e < CE; ++e) pair(x[e], x[CE + e], e);
    }
  }
};

template <typename E, int CE>
__device__ inline void store2(char* row, const float* x, const Place& p) {
  if (!p.on) return;
  Chunk<E, CE> a, b;
#pragma unroll
  for (int e = 0; e < CE; ++e) {
    a.v[e] = (E)x[e];
    b.v[e] = (E)x[CE + e];
  }
  *(Chunk<E, CE>*)(row + p.a * sizeof(E)) = a;
  *(Chunk<E, CE>*)(row + p.b * sizeof(E)) = b;
}
template <typename E, int CE>
__device__ inline void load_weight(float* w, const void* p0, bool w32, const Place& p) {
#pragma unroll
  for (int e = 0; e < 2 * CE; ++e) {
    const int d = (e < CE ? p.a : p.b - CE) + e;
    w[e] = !p.on ? 0.f : w32 ? ((const float*)p0)[d] : widen(((const E*)p0)[d]);
  }
}
// Sum over the G lanes of a row, in every one of them: quads, their mirror
// images within 8 and 16 lanes, then the halves of 32 and 64.
template <int CTRL>
__device__ inline float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int G>
__device__ inline float lanes_sum(float v) {
  v += dpp<0xB1>(v);                           // lane ^ 1
  v += dpp<0x4E>(v);                           // lane ^ 2
  if constexpr (G >= 8) v += dpp<0x141>(v);    // mirrored within 8
  if constexpr (G >= 16) v += dpp<0x140>(v);   // mirrored within 16
  if constexpr (G >= 32) v += __shfl_xor(v, 16, 64);
  if constexpr (G >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}

// 1 / sqrt(x): the instruction's value, and for fp32 rows a Newton step from it
// (it is off by up to 2^-23, twice a result's rounding).
template <typename E>
__device__ inline float inv_sqrt(float x) {
  const float r = __builtin_amdgcn_rsqf(x);
  if constexpr (sizeof(E) == 2) return r;
  return r > 0.f && r < INFINITY ? __builtin_fmaf(0.5f * r, __builtin_fmaf(-x * r, r, 1.f), r) : r;
}

// A row's chunks as they lie in memory: loaded a step before they are used.
template <typename E, int CE, int J>
struct Raw {
  Chunk<E, CE> a[J], b[J];
  __device__ inline void load(const char* row, const Place* p, bool ok) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (ok && p[j].on) {
        a[j] = *(const Chunk<E, CE>*)(row + p[j].a * sizeof(E));
        b[j] = *(const Chunk<E, CE>*)(row + p[j].b * sizeof(E));
      } else {
        a[j] = b[j] = Chunk<E, CE>{};
      }
    }
  }
  __device__ inline void get(int j, float* x) const {
#pragma unroll
    for (int e = 0; e < CE; ++e) {
      x[e] = widen(a[j].v[e]);
      x[CE + e] = widen(b[j].v[e]);
    }
  }
};

// J chunk pairs to a lane, G lanes to a row. A wavefront takes one token (a
// `parts`-th of its heads), GW heads a step; the next step's rows load while
// this one's are worked on, the first ones while the angles are formed.
template <typename E, int CE, int J, int G>
__global__ __launch_bounds__(256) void norm_rope_fwd(const Args g) {
  constexpr int GW = 64 / G;  // rows a wavefront takes at once
  const int lane = threadIdx.x & 63, t0 = lane % G, grp = lane / G;
  const uint64_t item = (uint64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= (uint64_t)g.tokens * g.parts) return;
  const uint32_t tok = g.parts == 1 ? (uint32_t)item : (uint32_t)(item / (uint32_t)g.parts);
  const int part = (int)(item - (uint64_t)tok * g.parts);
  const uint32_t b = tok / (uint32_t)g.S, i = tok - b * (uint32_t)g.S;
  Place p[J];
#pragma unroll
  for (int j = 0; j < J; ++j) p[j] = place<CE>(g, t0 + j * G);
  auto head = [&](int step) { return (step * g.parts + part) * GW + grp; };
  auto rows_at = [&](const Rows& r, int hd) { return r.p + b * r.b + hd * r.h + i * r.s; };
  const int n[2] = {(g.side[0].H - part * GW + g.parts * GW - 1) / (g.parts * GW),
                    (g.side[1].H - part * GW + g.parts * GW - 1) / (g.parts * GW)};
  Raw<E, CE, J> cur;
  auto fetch = [&](int sd, int step) {
    const int hd = head(step);
    cur.load(rows_at(g.side[sd].x, hd), p, hd < g.side[sd].H);
  };
  fetch(n[0] > 0 ? 0 : 1, 0);
  Angles<CE> ang[J];
  float fc[2], fs[2];
  Angles<CE>::form(g, lane, b, i, fc, fs, g.rot > 128 ? 2 : 1);
#pragma unroll
  for (int j = 0; j < J; ++j) ang[j].take(g, p[j], fc, fs);
#pragma unroll
  for (int sd = 0; sd < 2; ++sd) {
    const Side& s = g.side[sd];
    float w[J][2 * CE];
#pragma unroll
    for (int j = 0; j < J; ++j) load_weight<E, CE>(w[j], s.w, g.w32, p[j]);
    for (int step = 0; step < n[sd]; ++step) {
      float x[J][2 * CE], ss = 0.f;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        cur.get(j, x[j]);
#pragma unroll
        for (int e = 0; e < 2 * CE; ++e) ss += x[j][e] * x[j][e];
      }
      if (step + 1 < n[sd])
        fetch(sd, step + 1);
      else if (sd == 0 && n[1] > 0)
        fetch(1, 0);
      const float r = inv_sqrt<E>(lanes_sum<G>(ss) / (float)g.D + g.eps);
      const int hd = head(step);
      char* out = (char*)rows_at(s.y, hd);
#pragma unroll
      for (int j = 0; j < J; ++j) {
#pragma unroll
        for (int e = 0; e < 2 * CE; ++e) x[j][e] *= r * w[j][e];
        ang[j].turn(x[j], g.interleaved, 1.f);
        if (hd < s.H) store2<E, CE>(out, x[j], p[j]);
      }
    }
  }
}

template <typename E, int CE, int J, int G>
__global__ __launch_bounds__(256) void norm_rope_bwd(const Args g) {
  constexpr int GW = 64 / G;
  typedef typename std::conditional<sizeof(E) == 4, double, float>::type W;  // weight gradients' sums
  __shared__ W sum[4][2][256];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t0 = lane % G, grp = lane / G;
  Place p[J];
  float w[2][J][2 * CE];
  W dw[2][J][2 * CE];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    p[j] = place<CE>(g, t0 + j * G);
#pragma unroll
    for (int sd = 0; sd < 2; ++sd) {
      load_weight<E, CE>(w[sd][j], g.side[sd].w, g.w32, p[j]);
#pragma unroll
      for (int e = 0; e < 2 * CE; ++e) dw[sd][j][e] = 0;
    }
  }
  const int n[2] = {(g.side[0].H + GW - 1) / GW, (g.side[1].H + GW - 1) / GW};
  const float invD = 1.f / (float)g.D;
  const uint32_t tokens = (uint32_t)g.tokens, stride = gridDim.x * 4;
  Raw<E, CE, J> cx, cg;
  auto fetch = [&](int sd, int step, uint32_t tok) {
    const uint32_t b = tok / (uint32_t)g.S, i = tok - b * (uint32_t)g.S;
    const Side& s = g.side[sd];
    const int hd = step * GW + grp;
    cx.load(s.x.p + b * s.x.b + hd * s.x.h + i * s.x.s, p, hd < s.H);
    cg.load(s.g.p + b * s.g.b + hd * s.g.h + i * s.g.s, p, hd < s.H);
  };
  const int first = n[0] > 0 ? 0 : 1;
  uint32_t tok = blockIdx.x * 4 + wv;
  if (tok < tokens) fetch(first, 0, tok);
  for (; tok < tokens; tok += stride) {
    const uint32_t b = tok / (uint32_t)g.S, i = tok - b * (uint32_t)g.S;
    Angles<CE> ang[J];
    float fc[2], fs[2];
    Angles<CE>::form(g, lane, b, i, fc, fs, g.rot > 128 ? 2 : 1);
#pragma unroll
    for (int j = 0; j < J; ++j) ang[j].take(g, p[j], fc, fs);
#pragma unroll
    for (int sd = 0; sd < 2; ++sd) {
      const Side& s = g.side[sd];
      for (int step = 0; step < n[sd]; ++step) {
        float x[J][2 * CE], d[J][2 * CE], ss = 0.f, sw = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          cx.get(j, x[j]);
          cg.get(j, d[j]);
        }
        if (step + 1 < n[sd])
          fetch(sd, step + 1, tok);
        else if (sd == 0 && n[1] > 0)
          fetch(1, 0, tok);
        else if (tok + stride < tokens)
          fetch(first, 0, tok + stride);
#pragma unroll
        for (int j = 0; j < J; ++j) {
          ang[j].turn(d[j], g.interleaved, -1.f);
#pragma unroll
          for (int e = 0; e < 2 * CE; ++e) {
            ss += x[j][e] * x[j][e];
            sw += x[j][e] * (w[sd][j][e] * d[j][e]);
          }
        }
        const float r = inv_sqrt<E>(lanes_sum<G>(ss) / (float)g.D + g.eps);
        // (r before the sums: r^3 alone leaves 32 bits for rows of 1e-13 or 1e13)
        const float c = r * (r * lanes_sum<G>(sw) * invD);
        const int hd = step * GW + grp;
        char* out = (char*)s.y.p + b * s.y.b + hd * s.y.h + i * s.y.s;
#pragma unroll
        for (int j = 0; j < J; ++j) {
#pragma unroll
          for (int e = 0; e < 2 * CE; ++e) {
            // (a lane without a row holds zeros, and r may be infinite there)
            const float u = x[j][e] * r;
            dw[sd][j][e] += hd < s.H ? (W)d[j][e] * (W)u : (W)0;
            x[j][e] = r * (w[sd][j][e] * d[j][e]) - u * c;
          }
          if (hd < s.H) store2<E, CE>(out, x[j], p[j]);
        }
      }
    }
  }
  if (!g.need_w) return;
  // ---- the wavefront's groups, then the four wavefronts, in a fixed order
#pragma unroll
  for (int sd = 0; sd < 2; ++sd)
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int e = 0; e < 2 * CE; ++e) {
        W v = dw[sd][j][e];
        for (int o = G; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
        if (grp == 0 && p[j].on) sum[wv][sd][(e < CE ? p[j].a : p[j].b - CE) + e] = v;
      }
  __syncthreads();
  for (int k = threadIdx.x; k < 2 * g.D; k += 256) {
    const int sd = k / g.D, d = k - sd * g.D;
    g.wpart[(int64_t)blockIdx.x * 2 * g.D + k] = (float)((sum[0][sd][d] + sum[1][sd][d]) + (sum[2][sd][d] + sum[3][sd][d]));
  }
}

// dw of 16 columns of (2, D): 64 threads to a column, then their sums in order,
// in fp64: as a chain of fp32 sums of up to 1024 parts they alone were off by 1.6
// times a result's rounding.
template <typename E>
__global__ __launch_bounds__(1024) void wgrad_kernel(const float* __restrict__ part, int n, int D, int w32, void* dwq,
                                                     void* dwk) {
  __shared__ double sum[64][17];
  const int c = threadIdx.x & 15, rg = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
  double v = 0.;
  if (col < 2 * D) {
#pragma unroll 8
    for (int k = rg; k < n; k += 64) v += part[(int64_t)k * 2 * D + col];
  }
  sum[rg][c] = v;
  __syncthreads();
  if (rg >= 4) return;
  double t = 0.;
#pragma unroll
  for (int k = 0; k < 16; ++k) t += sum[16 * rg + k][c];
  t += __shfl_xor(t, 16, 64);
  t += __shfl_xor(t, 32, 64);
  if (rg != 0 || col >= 2 * D) return;
  void* out = col < D ? dwq : dwk;
  const int d = col < D ? col : col - D;
  if (!out) return;
  if (w32)
    ((float*)out)[d] = (float)t;
  else
    ((E*)out)[d] = (E)(float)t;
}

// Workgroups of the backward (and parts of a weight gradient): four to a CU.
constexpr int MAX_WGS = 1024;

int bwd_wgs(int64_t tokens) {
  const int64_t n = tsp::ceil_div(tokens, 4);
  return (int)(n < 1 ? 1 : n < MAX_WGS ? n : MAX_WGS);
}

template <typename E, int CE, int J, int G>
int launch(const Args& a, bool back, hipStream_t st) {
  const int64_t grid = back ? bwd_wgs(a.tokens) : tsp::ceil_div(a.tokens * a.parts, 4);
  if (grid > INT32_MAX) return tsp::fail(TSP_EUNSUPPORTED, "qk_norm_rope: too many tokens");
  if (back)
    hipLaunchKernelGGL((norm_rope_bwd<E, CE, J, G>), dim3((unsigned)grid), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((norm_rope_fwd<E, CE, J, G>), dim3((unsigned)grid), dim3(256), 0, st, a);
  return tsp::check_launch("norm_rope launch");
}
template <typename E, int CE>
int launch_ce(Args a, bool back, hipStream_t st) {
  const int lanes = (a.D + 2 * CE - 1) / (2 * CE);
  // wavefronts to a token: all its heads at once while the chip is not full
  const int G = lanes <= 4 ? 4 : lanes <= 8 ? 8 : lanes <= 16 ? 16 : lanes <= 32 ? 32 : 64;
  const int most = (int)tsp::ceil_div(a.side[0].H > a.side[1].H ? a.side[0].H : a.side[1].H, 64 / G);
  const int64_t want = tsp::ceil_div(4096, a.tokens > 0 ? a.tokens : 1);
  a.parts = (int)(want < 1 ? 1 : want < most ? want : most < 1 ? 1 : most);
  if (lanes <= 4) return launch<E, CE, 1, 4>(a, back, st);
  if (lanes <= 8) return launch<E, CE, 1, 8>(a, back, st);
  if (lanes <= 16) return launch<E, CE, 1, 16>(a, back, st);
  if (CE == 4 || lanes <= 32) return launch<E, CE, 1, 32>(a, back, st);
  if constexpr (CE <= 2)
    if (CE == 2 || lanes <= 64) return launch<E, CE, 1, 64>(a, back, st);
  if constexpr (CE == 1) return launch<E, CE, 2, 64>(a, back, st);
  return TSP_EUNSUPPORTED;  // not reached: head_dim is at most 256
}

// The widest chunk of up to four elements that the pairing, the addresses and
// the strides allow. (Eight, 16 bytes of a 16-bit row, halve the loads but
// double a lane's registers: 86 us forward and 142 backward of 2 x 8192 tokens,
// 40 heads of 128, against 74 and 123.)
template <typename E>
int launch_e(const Args& a, bool back, hipStream_t st) {
  uint64_t all = 0;
  for (const Side& s : a.side)
    if (s.H > 0)
      for (const Rows* r : {&s.x, &s.y, &s.g}) all |= (uint64_t)(uintptr_t)r->p | r->b | r->h | r->s;
  auto fits = [&](int ce) {
    return a.D % (2 * ce) == 0 && (a.interleaved || a.rot / 2 % ce == 0) && all % (ce * sizeof(E)) == 0;
  };
  if (fits(4)) return launch_ce<E, 4>(a, back, st);
  if (fits(2)) return launch_ce<E, 2>(a, back, st);
  return launch_ce<E, 1>(a, back, st);
}

int run(int dtype, const Args& a, bool back, hipStream_t st) {
  if (dtype == TSP_F32) return launch_e<float>(a, back, st);
  if (dtype == TSP_BF16) return launch_e<__bf16>(a, back, st);
  return launch_e<_Float16>(a, back, st);
}

Rows rows(const void* p, const int64_t* s, int e) {
  if (!p || !s) return Rows{nullptr, 0, 0, 0};
  return Rows{(const char*)p, s[0] * e, s[1] * e, s[2] * e};
}

int fill(const char* who, Args& a, int dtype, int64_t B, int64_t Hq, int64_t Hk, int64_t S, int64_t D, const void* wq,
         const void* wk, int wdtype, const void* pos, int index_type, int64_t pos_b, int64_t pos_s, const double* freq,
         int64_t rot, int interleaved, double eps) {
  if (dtype != TSP_F32 && dtype != TSP_BF16 && dtype != TSP_F16)
    return tsp::fail(TSP_EUNSUPPORTED, "%s: dtype %d not supported", who, dtype);
  if (wdtype != dtype && wdtype != TSP_F32)
    return tsp::fail(TSP_EUNSUPPORTED, "%s: weights must have the rows' type or fp32", who);
  if (B < 0 || Hq < 0 || Hk < 0 || S < 0 || D < 2 || rot < 0 || rot > D || D % 2 || rot % 2)
    return tsp::fail(TSP_EINVAL, "%s: bad sizes batch %lld heads %lld, %lld tokens %lld head_dim %lld rotated %lld", who,
                     (long long)B, (long long)Hq, (long long)Hk, (long long)S, (long long)D, (long long)rot);
  if (D > 256) return tsp::fail(TSP_EUNSUPPORTED, "%s: head_dim %lld is over 256", who, (long long)D);
  if (S > INT32_MAX || Hq > INT32_MAX || Hk > INT32_MAX || B * S >= (int64_t(1) << 32) - (1 << 16))
    return tsp::fail(TSP_EUNSUPPORTED, "%s: too many rows", who);
  if (index_type != TSP_I32 && index_type != TSP_I64) return tsp::fail(TSP_EINVAL, "%s: bad index type", who);
  if (!(eps >= 0)) return tsp::fail(TSP_EINVAL, "%s: eps must not be negative", who);
  if (B * S * (Hq + Hk) > 0 && (!pos || !wq || !wk || (rot > 0 && !freq)))
    return tsp::fail(TSP_EINVAL, "%s: null operand", who);
  a.side[0].w = wq;
  a.side[1].w = wk;
  a.side[0].H = (int)Hq;
  a.side[1].H = (int)Hk;
  a.pos = pos;
  a.pos_b = pos_b;
  a.pos_s = pos_s;
  a.pos64 = index_type == TSP_I64;
  a.w32 = wdtype == TSP_F32;
  a.freq = freq;
  a.S = (int)S;
  a.D = (int)D;
  a.rot = (int)rot;
  a.interleaved = interleaved != 0;
  a.tokens = B * S;
  a.eps = (float)eps;
  return TSP_OK;
}

int need(const char* who, const char* name, int64_t heads, const void* p, const int64_t* s) {
  return heads > 0 && (!p || !s) ? tsp::fail(TSP_EINVAL, "%s: null %s", who, name) : TSP_OK;
}

}  // namespace

extern "C" int tsp_qk_norm_rope_fwd(const void* Q, const int64_t* qs, const void* K, const int64_t* ks, int dtype,
                                    int64_t B, int64_t Hq, int64_t Hk, int64_t S, int64_t D, const void* wq,
                                    const void* wk, int wdtype, const void* pos, int index_type, int64_t pos_b,
                                    int64_t pos_s, const double* freq, int64_t rot, int interleaved, double eps, void* Qo,
                                    const int64_t* qos, void* Ko, const int64_t* kos, void* stream) {
  const char* who = "tsp_qk_norm_rope_fwd";
  Args a{};
  int rc = fill(who, a, dtype, B, Hq, Hk, S, D, wq, wk, wdtype, pos, index_type, pos_b, pos_s, freq, rot, interleaved, eps);
  if (rc) return rc;
  if (a.tokens * (Hq + Hk) == 0) return TSP_OK;
  if ((rc = need(who, "Q", Hq, Q, qs)) || (rc = need(who, "K", Hk, K, ks)) || (rc = need(who, "Q result", Hq, Qo, qos)) ||
      (rc = need(who, "K result", Hk, Ko, kos)))
    return rc;
  const int e = dtype == TSP_F32 ? 4 : 2;
  a.side[0].x = rows(Q, qs, e);
  a.side[1].x = rows(K, ks, e);
  a.side[0].y = rows(Qo, qos, e);
  a.side[1].y = rows(Ko, kos, e);
  return run(dtype, a, false, (hipStream_t)stream);
}

extern "C" int64_t tsp_qk_norm_rope_bwd_workspace_size(int64_t B, int64_t S, int64_t D) {
  if (B < 0 || S < 0 || D < 2 || D > 256 || B * S >= (int64_t(1) << 32) - (1 << 16)) return -1;
  return (int64_t)bwd_wgs(B * S) * 2 * D * 4;
}

extern "C" int tsp_qk_norm_rope_bwd(const void* Q, const int64_t* qs, const void* K, const int64_t* ks, int dtype,
                                    int64_t B, int64_t Hq, int64_t Hk, int64_t S, int64_t D, const void* wq,
                                    const void* wk, int wdtype, const void* pos, int index_type, int64_t pos_b,
                                    int64_t pos_s, const double* freq, int64_t rot, int interleaved, double eps,
                                    const void* gQ, const int64_t* gqs, const void* gK, const int64_t* gks, void* dQ,
                                    const int64_t* dqs, void* dK, const int64_t* dks, void* dwq, void* dwk,
                                    void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "tsp_qk_norm_rope_bwd";
  Args a{};
  int rc = fill(who, a, dtype, B, Hq, Hk, S, D, wq, wk, wdtype, pos, index_type, pos_b, pos_s, freq, rot, interleaved, eps);
  if (rc) return rc;
  const hipStream_t st = (hipStream_t)stream;
  const int ew = wdtype == TSP_F32 ? 4 : 2, e = dtype == TSP_F32 ? 4 : 2;
  if (a.tokens * (Hq + Hk) == 0) {  // no row: the weights' gradients are zero
    for (void* w : {dwq, dwk})
      if (w && (rc = tsp::zero_fill(w, D * ew, st))) return rc;
    return TSP_OK;
  }
  if ((rc = need(who, "Q", Hq, Q, qs)) || (rc = need(who, "K", Hk, K, ks)) || (rc = need(who, "grad of Q", Hq, gQ, gqs)) ||
      (rc = need(who, "grad of K", Hk, gK, gks)) || (rc = need(who, "dQ", Hq, dQ, dqs)) ||
      (rc = need(who, "dK", Hk, dK, dks)))
    return rc;
  a.need_w = dwq || dwk;
  if (a.need_w && (!workspace || workspace_bytes < tsp_qk_norm_rope_bwd_workspace_size(B, S, D)))
    return tsp::fail(TSP_EINVAL, "%s: workspace too small", who);
  a.side[0].x = rows(Q, qs, e);
  a.side[1].x = rows(K, ks, e);
  a.side[0].g = rows(gQ, gqs, e);
  a.side[1].g = rows(gK, gks, e);
  a.side[0].y = rows(dQ, dqs, e);
  a.side[1].y = rows(dK, dks, e);
  a.wpart = (float*)workspace;
  if ((rc = run(dtype, a, true, st)) || !a.need_w) return rc;
  const dim3 grid((unsigned)tsp::ceil_div(2 * D, 16)), block(1024);
  const int n = bwd_wgs(a.tokens), w32 = wdtype == TSP_F32;
  if (dtype == TSP_BF16)
    hipLaunchKernelGGL((wgrad_kernel<__bf16>), grid, block, 0, st, a.wpart, n, (int)D, w32, dwq, dwk);
  else
    hipLaunchKernelGGL((wgrad_kernel<_Float16>), grid, block, 0, st, a.wpart, n, (int)D, w32, dwq, dwk);
  return tsp::check_launch("wgrad launch");
}
