// Cross attention forward for gfx950: queries of one sequence over the keys
// and values of another of any length, per batch entry b and query head h with
// key head h / (heads / kv_heads):
//   O[b, h, i] = sum_j p_ij V[b, hk, j],  p_i = softmax_j(scale Q[b, h, i] . K[b, hk, j])
// over keys j < key_lengths[b]; a row without keys is zero. No counterpart in
// the reference, whose attention is one sequence's over itself
// (trnsparse/ops.py:549-625). Kernels and their choice: xattn_fwd.h.
#include "xattn_fwd.h"

namespace tsp {
namespace xat {

int check_operand(const char* who, const char* name, const void* p, const int64_t* s, int64_t rows, int64_t D,
                  int dtype) {
  if (!p || !s) return fail(TSP_EINVAL, "%s: null %s", who, name);
  const int64_t e = esize(dtype), rs = row_stride(s, rows, D);
  if (((uintptr_t)p | (uint64_t)(s[0] * e) | (uint64_t)(s[1] * e) | (uint64_t)(rs * e)) & 15)
    return fail(TSP_EINVAL, "%s: %s and its strides must be whole 16-byte pieces", who, name);
  if (rs < D || rs * e >= MAX_ROW_BYTES)
    return fail(TSP_EINVAL, "%s: row stride %lld of %s is not in [%lld, %lld)", who, (long long)rs, name, (long long)D,
                (long long)(MAX_ROW_BYTES / e));
  return TSP_OK;
}

Plan fwd_plan(int dtype, int64_t units, int64_t rows, int64_t keys, int64_t wide_want, int64_t wide_least) {
  Plan p;
  p.narrow = rows <= 32;
  p.tiles = p.narrow ? 1 : (int)ceil_div(rows, 128);
  // Ranges of keys where the units and tiles are fewer than half of `want`
  // workgroups; none shorter than `least` keys, which is where a range costs as
  // much as the launch that joins the ranges. Narrow bf16 of 128, 300 / 1500 /
  // 4000 / 16000 keys of 32 units: 7.4 / 13.2 / 21.8 / 59 us, with 256 at
  // least 9.6 / 13.6 / 23.8 / 59; of 128 units 8.4 / 26 / 56 / 192, with one
  // range 8.4 / 25 / 55 / 197. In fp32 a stage of 32 keys is 3.4 us of matrix
  // instructions and a CU holds one workgroup: shorter ranges, fewer of them.
  const bool f32 = dtype == TSP_F32;
  const int64_t want = p.narrow ? (f32 ? 256 : 512) : wide_want, least = p.narrow ? (f32 ? 128 : 512) : wide_least;
  const int64_t wgs = units * p.tiles, step = p.narrow ? 128 : 64;
  int64_t n = wgs >= (p.narrow && f32 ? want : want / 2) ? 1 : ceil_div(want, wgs);
  if (n > ceil_div(keys, least)) n = ceil_div(keys, least);
  if (n > 32) n = 32;  // (8 heads on one key head, 16000 keys in fp32: 125 ranges 51 us, 32 36)
  if (n < 1) n = 1;
  p.chunk = ceil_div(ceil_div(keys > 0 ? keys : 1, n), step) * step;
  p.nsplit = (int)(keys > 0 ? ceil_div(keys, p.chunk) : 1);
  return p;
}

// Wide, 16 bit: one workgroup of eight wavefronts to a CU (fwd_wide<T, 2>) and
// ranges of 512 keys at least: 16 heads of 1500 x 1500 x 64 21.0 us, two
// workgroups of four with ranges of 256 34.7; 8 heads of 512 x 4000 x 128 29.3
// and 32.4; 2 x 8 of 512 x 512 x 128 14.3 and 18.4.
static Plan cross_plan(int dtype, int64_t units, int64_t rows, int64_t keys) {
  return dtype == TSP_F32 ? fwd_plan(dtype, units, rows, keys, 512, 64) : fwd_plan(dtype, units, rows, keys, 256, 512);
}

static void set_plan(FwdArgs& a, const Plan& p) {
  a.tiles = p.tiles;
  a.nsplit = p.nsplit;
  a.chunk = p.chunk;
}
static int64_t grid_of(const FwdArgs& a) {
  return head_grid((int64_t)a.tiles * a.nsplit, (int64_t)a.units_b * a.Hkv);
}

int launch_fwd(int dtype, const Plan& p, FwdArgs a, hipStream_t st) {
  set_plan(a, p);
  const int64_t grid = grid_of(a);
  if (grid > INT32_MAX) return fail(TSP_EUNSUPPORTED, "attention: too large a grid");
  return with_tile(dtype, a.D, [&](auto tile) {
    typedef decltype(tile) T;
    if (p.narrow)
      hipLaunchKernelGGL((fwd_narrow<T>), dim3((unsigned)grid), dim3(256), 0, st, a);
    else if (T::ESZ == 2 && grid <= 256)  // a CU has one workgroup at most
      hipLaunchKernelGGL((fwd_wide<T, T::ESZ == 2 ? 2 : 1>), dim3((unsigned)grid), dim3(T::ESZ == 2 ? 512 : 256), 0, st, a);
    else
      hipLaunchKernelGGL((fwd_wide<T, 1>), dim3((unsigned)grid), dim3(256), 0, st, a);
    return check_launch("attention launch");
  });
}

int launch_fwd_joint(int dtype, FwdArgs a, const FwdArgs& first, hipStream_t st) {
  a.tiles = a.nsplit = 1;
  const int64_t grid = grid_of(a);
  if (grid > INT32_MAX) return fail(TSP_EUNSUPPORTED, "attention: too large a grid");
  return with_tile(dtype, a.D, [&](auto tile) {
    typedef decltype(tile) T;
    hipLaunchKernelGGL((fwd_joint<T>), dim3((unsigned)grid), dim3(256), 0, st, a, first);
    return check_launch("attention launch");
  });
}

int launch_fwd_two(int dtype, const Plan& pa, FwdArgs a, const Plan& pb, FwdArgs b, hipStream_t st) {
  set_plan(a, pa);
  set_plan(b, pb);
  const int64_t ga = grid_of(a), gb = grid_of(b);
  if (ga + gb > INT32_MAX) return fail(TSP_EUNSUPPORTED, "attention: too large a grid");
  return with_tile(dtype, a.D, [&](auto tile) {
    typedef decltype(tile) T;
    hipLaunchKernelGGL((fwd_two<T>), dim3((unsigned)(ga + gb)), dim3(256), 0, st, a, b, (uint32_t)ga, !pa.narrow,
                       !pb.narrow);
    return check_launch("attention launch");
  });
}

int launch_combine(int dtype, const CombineArgs& a, hipStream_t st) {
  const int64_t grid = ceil_div(a.prows, 8);
  if (grid > INT32_MAX) return fail(TSP_EUNSUPPORTED, "attention: too many rows");
  const dim3 g((unsigned)grid), b(256);
  if (dtype == TSP_BF16)
    hipLaunchKernelGGL((combine_kernel<Tile16<__bf16, 128>>), g, b, 0, st, a);
  else if (dtype == TSP_F16)
    hipLaunchKernelGGL((combine_kernel<Tile16<_Float16, 128>>), g, b, 0, st, a);
  else
    hipLaunchKernelGGL((combine_kernel<Tile32<128>>), g, b, 0, st, a);
  return check_launch("combine launch");
}

// Sizes that every entry point takes; 0 or a status.
int check_sizes(const char* who, int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t L, int64_t D) {
  if (dtype != TSP_F32 && dtype != TSP_BF16 && dtype != TSP_F16)
    return fail(TSP_EUNSUPPORTED, "%s: dtype %d not supported", who, dtype);
  if (B < 0 || Hq < 0 || Sq < 0 || L < 0 || D < 1 || Hkv < 1 || Hq % Hkv != 0)
    return fail(TSP_EINVAL, "%s: bad sizes batch %lld heads %lld / %lld queries %lld keys %lld head_dim %lld", who,
                (long long)B, (long long)Hq, (long long)Hkv, (long long)Sq, (long long)L, (long long)D);
  if (D > 128 || D % (16 / esize(dtype)) != 0)
    return fail(TSP_EUNSUPPORTED, "%s: head_dim %lld (at most 128, whole 16-byte pieces)", who, (long long)D);
  // rows of a unit and keys are counted in 32 bits, tiles past the last included
  const int64_t most = int64_t(1) << 30;
  if (Sq > most || Hq > most || B > most || L > most || Hq * Sq > most || B * Hq > most || B * Hq * Sq > most * 256)
    return fail(TSP_EUNSUPPORTED, "%s: too many rows or keys", who);
  return TSP_OK;
}

}  // namespace xat
}  // namespace tsp

using namespace tsp;

extern "C" int64_t tsp_cross_attn_workspace_size(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t L,
                                                 int64_t D) {
  if (xat::check_sizes("tsp_cross_attn_workspace_size", dtype, B, Hq, Hkv, Sq, L, D)) return -1;
  if (B * Hq * Sq == 0) return 0;
  const xat::Plan p = xat::cross_plan(dtype, B * Hkv, Hq / Hkv * Sq, L);
  return p.nsplit > 1 ? p.nsplit * B * Hq * Sq * (D + 1) * 4 : 0;
}

extern "C" int tsp_cross_attn_fwd(const void* Q, const int64_t* qs, const void* K, const int64_t* ks, const void* V,
                                  const int64_t* vs, int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq,
                                  int64_t L, int64_t D, const void* key_lengths, int index_type, double scale, void* O,
                                  const int64_t* os, float* lse, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  const char* who = "tsp_cross_attn_fwd";
  int rc = xat::check_sizes(who, dtype, B, Hq, Hkv, Sq, L, D);
  if (rc) return rc;
  if (B * Hq * Sq == 0) return TSP_OK;
  if ((rc = xat::check_operand(who, "Q", Q, qs, Sq, D, dtype))) return rc;
  if ((rc = xat::check_operand(who, "O", O, os, Sq, D, dtype))) return rc;
  if (L > 0) {
    if ((rc = xat::check_operand(who, "K", K, ks, L, D, dtype))) return rc;
    if ((rc = xat::check_operand(who, "V", V, vs, L, D, dtype))) return rc;
  }
  if (!(scale > 1e-30) || !(scale < 1e30)) return fail(TSP_EINVAL, "%s: scale must be positive", who);
  if (index_type != TSP_I32 && index_type != TSP_I64) return fail(TSP_EINVAL, "%s: bad index type", who);
  const int64_t need = tsp_cross_attn_workspace_size(dtype, B, Hq, Hkv, Sq, L, D);
  if (need > 0 && (!workspace || workspace_bytes < need)) return fail(TSP_EINVAL, "%s: workspace too small", who);
  const int64_t none[3] = {0, 0, 0};
  const xat::Plan p = xat::cross_plan(dtype, B * Hkv, Hq / Hkv * Sq, L);
  xat::FwdArgs a{};
  a.Q = xat::operand(Q, qs, Sq, D, dtype);
  a.K = xat::operand(K, L > 0 ? ks : none, L, D, dtype);
  a.V = xat::operand(V, L > 0 ? vs : none, L, D, dtype);
  const xat::Operand o = xat::operand(O, os, Sq, D, dtype);
  a.O = (char*)O;
  a.ob = o.b, a.oh = o.h, a.os = o.s;
  a.lse = lse;
  a.prows = B * Hq * Sq;
  if (p.nsplit > 1) {
    a.part = (float*)workspace;
    a.plse = a.part + p.nsplit * a.prows * D;
  }
  a.lengths = key_lengths;
  a.len64 = index_type == TSP_I64;
  a.units_b = (int)B;
  a.Hkv = (int)Hkv, a.G = (int)(Hq / Hkv), a.Sq = (int)Sq, a.R = (int)(Hq / Hkv * Sq), a.D = (int)D;
  a.L = L;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  if ((rc = xat::launch_fwd(dtype, p, a, (hipStream_t)stream))) return rc;
  if (p.nsplit == 1) return TSP_OK;
  const xat::CombineArgs c{a.part, a.plse, a.prows, p.nsplit, a.D, (int)Hq, a.Sq, a.O, a.ob, a.oh, a.os, lse};
  return xat::launch_combine(dtype, c, (hipStream_t)stream);
}
