// Attention of new tokens over a prefix that all sequences of a batch share and
// each sequence's own keys behind it (serving):
//   O[b, h, i] = sum_j p_j V_j over the prefix keys of key head hk = h / group
//   and b's own keys j < lengths[b] - (Sq - 1 - i), p = softmax_j(scale Q . K_j)
// No counterpart in the reference, whose attention is one sequence's over
// itself (trnsparse/ops.py:549-625).
//
// The rows of all sequences that read one key head form one unit for the
// prefix, so it is read once for the batch; every sequence's own keys are a
// unit of their own. Both parts are ranges of the same softmax and are joined
// by their log-sum-exps (xattn_fwd.h).
#include "xattn_fwd.h"

namespace tsp {
namespace xat {
int check_sizes(const char* who, int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t L, int64_t D);

namespace {
struct PrefixPlan {
  bool joint;  // both sets in one pass of each sequence, nothing to join
  Plan shared, own;
  int nsplit;
};
PrefixPlan prefix_plan(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t P, int64_t S) {
  const int64_t G = Hq / Hkv;
  PrefixPlan p{};
  // 16 sequences on 8 key heads of 128, bf16, 512 + 512 keys: 12.1 us in one
  // pass, 13.9 joined; 1024 + 512: 17.8 and 15.0. fp32, 16 key heads of 128, 64 +
  // 64 keys: 10.1 and 13.9; 256 + 256: 24.1 and 14.8.
  p.joint = P > 0 && S > 0 && G * Sq <= 32 && P + S <= (dtype == TSP_F32 ? 256 : 1024);
  if (p.joint) return p;
  // (64 sequences, 32 heads on 8 key heads, 8192 + up to 1024 keys: the prefix
  // in ranges for 128 workgroups 38.1 us, for 96 42.1, 192 40.8, 256 46.1; each
  // range writes and reads back a result of every row)
  const int64_t least = dtype == TSP_F32 ? 64 : 256;
  if (P > 0) p.shared = fwd_plan(dtype, Hkv, B * G * Sq, P, 128, least);
  if (S > 0) p.own = fwd_plan(dtype, B * Hkv, G * Sq, S, 512, least);
  p.nsplit = p.shared.nsplit + p.own.nsplit;
  return p;
}
// Bytes of workspace: none where one range has all keys (and writes the result),
// an fp32 result and log-sum-exp of every row for each of more.
int64_t part_bytes(const PrefixPlan& p, int64_t rows, int64_t D) {
  return p.nsplit > 1 ? p.nsplit * rows * (D + 1) * 4 : 0;
}
}  // namespace
}  // namespace xat
}  // namespace tsp

using namespace tsp;

extern "C" int64_t tsp_prefix_attn_workspace_size(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t P,
                                                  int64_t S, int64_t D) {
  if (xat::check_sizes("tsp_prefix_attn_workspace_size", dtype, B, Hq, Hkv, Sq, P > S ? P : S, D)) return -1;
  if (P < 0 || S < 0) return fail(TSP_EINVAL, "tsp_prefix_attn_workspace_size: negative length"), -1;
  if (B * Hq * Sq == 0) return 0;
  return xat::part_bytes(xat::prefix_plan(dtype, B, Hq, Hkv, Sq, P, S), B * Hq * Sq, D);
}

extern "C" int tsp_prefix_attn_fwd(const void* Q, const int64_t* qs, const void* PK, const int64_t* pks, const void* PV,
                                   const int64_t* pvs, const void* K, const int64_t* ks, const void* V,
                                   const int64_t* vs, int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq,
                                   int64_t P, int64_t S, int64_t D, const void* lengths, int index_type, double scale,
                                   void* O, const int64_t* os, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "tsp_prefix_attn_fwd";
  const hipStream_t st = (hipStream_t)stream;
  if (P < 0 || S < 0) return fail(TSP_EINVAL, "%s: negative length", who);
  int rc = xat::check_sizes(who, dtype, B, Hq, Hkv, Sq, P > S ? P : S, D);
  if (rc) return rc;
  if (B * Hq * Sq == 0) return TSP_OK;
  if (B * Hq / Hkv * Sq > (int64_t(1) << 30)) return fail(TSP_EUNSUPPORTED, "%s: too many rows on a key head", who);
  if ((rc = xat::check_operand(who, "Q", Q, qs, Sq, D, dtype))) return rc;
  if ((rc = xat::check_operand(who, "O", O, os, Sq, D, dtype))) return rc;
  if (P > 0) {
    if ((rc = xat::check_operand(who, "prefix K", PK, pks, P, D, dtype))) return rc;
    if ((rc = xat::check_operand(who, "prefix V", PV, pvs, P, D, dtype))) return rc;
  }
  if (S > 0) {
    if ((rc = xat::check_operand(who, "K", K, ks, S, D, dtype))) return rc;
    if ((rc = xat::check_operand(who, "V", V, vs, S, D, dtype))) return rc;
  }
  if (!(scale > 1e-30) || !(scale < 1e30)) return fail(TSP_EINVAL, "%s: scale must be positive", who);
  if (index_type != TSP_I32 && index_type != TSP_I64) return fail(TSP_EINVAL, "%s: bad index type", who);
  const xat::PrefixPlan p = xat::prefix_plan(dtype, B, Hq, Hkv, Sq, P, S);
  const int64_t rows = B * Hq * Sq, need = xat::part_bytes(p, rows, D);
  if (need > 0 && (!workspace || workspace_bytes < need)) return fail(TSP_EINVAL, "%s: workspace too small", who);
  xat::FwdArgs a{};
  a.Q = xat::operand(Q, qs, Sq, D, dtype);
  const xat::Operand o = xat::operand(O, os, Sq, D, dtype);
  a.O = (char*)O;
  a.ob = o.b, a.oh = o.h, a.os = o.s;
  a.prows = rows;
  if (p.nsplit > 1) {
    a.part = (float*)workspace;
    a.plse = a.part + p.nsplit * rows * D;
  }
  a.Hkv = (int)Hkv, a.G = (int)(Hq / Hkv), a.Sq = (int)Sq, a.D = (int)D;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  xat::FwdArgs sh = a, own = a;
  if (P > 0) {
    sh.K = xat::operand(PK, pks, P, D, dtype);
    sh.V = xat::operand(PV, pvs, P, D, dtype);
    sh.units_b = 1;
    sh.R = (int)(B * Hq / Hkv * Sq);
    sh.L = P;
  }
  if (S > 0) {
    own.K = xat::operand(K, ks, S, D, dtype);
    own.V = xat::operand(V, vs, S, D, dtype);
    own.lengths = lengths;
    own.len64 = index_type == TSP_I64;
    own.units_b = (int)B;
    own.R = (int)(Hq / Hkv * Sq);
    own.L = S;
    own.causal = Sq > 1;
    own.split0 = p.shared.nsplit;
  }
  if (p.joint) return xat::launch_fwd_joint(dtype, own, sh, st);
  if (P > 0 && S > 0)
    rc = xat::launch_fwd_two(dtype, p.shared, sh, p.own, own, st);
  else if (P > 0)
    rc = xat::launch_fwd(dtype, p.shared, sh, st);
  else if (S > 0)
    rc = xat::launch_fwd(dtype, p.own, own, st);
  if (rc || p.nsplit == 1) return rc;
  const xat::CombineArgs c{a.part, a.plse, rows, p.nsplit, a.D, (int)Hq, a.Sq, a.O, a.ob, a.oh, a.os, nullptr};
  return xat::launch_combine(dtype, c, st);
}
