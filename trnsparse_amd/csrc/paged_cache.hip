// Writes of new tokens' rows into a key and value cache in pages, and the checks
// of a cache's operands. No counterpart in the reference, whose attention takes
// one sequence's K and V whole (trnsparse/ops.py:549-625).
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
