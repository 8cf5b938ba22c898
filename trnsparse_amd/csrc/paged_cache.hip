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

// Whether rows of `row` elements lie apart, `n` dimensions of them: each dimension's stride
// passes the extent of those of smaller strides. (Rows that interleave in other ways without
// an overlap are no views of a tensor by slices and transpositions.)
static bool lie_apart(const int64_t* size, const int64_t* stride, int n, int64_t row) {
  bool done[3] = {};
  __int128 extent = row;
  for (int k = 0; k < n; ++k) {
    int at = -1;
    for (int i = 0; i < n; ++i)
      if (!done[i] && (at < 0 || stride[i] < stride[at])) at = i;
    done[at] = true;
    if (size[at] == 0) return true;
    if (size[at] == 1) continue;
    if (stride[at] < extent) return false;
    extent += (__int128)stride[at] * (size[at] - 1);
  }
  return true;
}

int check_pages(const char* who, const char* name, const void* p, const int64_t* s, int dtype, int64_t pages, int64_t Hkv,
                int64_t page_size, int64_t D, bool written) {
  if (!s) return fail(TSP_EINVAL, "%s: no strides of %s", who, name);
  if (pages == 0) return TSP_OK;
  if (!p) return fail(TSP_EINVAL, "%s: null %s", who, name);
  const int64_t e = esize(dtype);
  if (((uintptr_t)p | (uint64_t)(s[0] * e) | (uint64_t)(s[1] * e) | (uint64_t)(s[2] * e)) & 15)
    return fail(TSP_EINVAL, "%s: %s and its strides must be whole 16-byte pieces", who, name);
  if (s[0] < 0 || s[1] < 0 || s[2] < D || s[2] * e >= (int64_t(1) << 24))
    return fail(TSP_EINVAL, "%s: strides of %s: %lld, %lld, %lld", who, name, (long long)s[0], (long long)s[1],
                (long long)s[2]);
  const int64_t size[3] = {pages, Hkv, page_size};
  if (written && !lie_apart(size, s, 3, D))
    return fail(TSP_EINVAL, "%s: rows of %s, which are written, overlap: strides %lld, %lld, %lld", who, name,
                (long long)s[0], (long long)s[1], (long long)s[2]);
  return TSP_OK;
}

int check_lengths(const char* who, int64_t B, const void* lengths, int index_type, bool has_new) {
  const int type = has_new ? index_type & ~TSP_NEW_OTHER : index_type;
  if (type != TSP_I32 && type != TSP_I64) return fail(TSP_EINVAL, "%s: bad index type", who);
  if (B > 0 && !lengths) return fail(TSP_EINVAL, "%s: null lengths", who);
  return TSP_OK;
}

// Workgroups of a sequence read its lengths while another writes the one after.
int check_lengths_out(const char* who, int64_t B, const void* out, const Lengths& l) {
  const auto meets = [&](const void* p, int wide) {
    const char *a = (const char*)out, *b = (const char*)p;
    return p && a < b + B * (wide ? 8 : 4) && b < a + B * (l.wide ? 8 : 4);
  };
  if (!out || meets(l.p, l.wide) || meets(l.fresh, l.fresh_wide))
    return fail(TSP_EINVAL, "%s: lengths_out must be a place of its own", who);
  return TSP_OK;
}

int check_weights(const char* who, const void* w, const int64_t* s, int64_t B, int64_t Hkv, int64_t slots) {
  if (!w) return TSP_OK;
  if (!s) return fail(TSP_EINVAL, "%s: no strides of weights", who);
  if (((uintptr_t)w & 3) || s[0] < 0 || s[1] < 0) return fail(TSP_EINVAL, "%s: bad weights", who);
  const int64_t size[2] = {B, Hkv};
  if (!lie_apart(size, s, 2, slots))
    return fail(TSP_EINVAL, "%s: rows of weights, which are written, overlap: strides %lld, %lld", who, (long long)s[0],
                (long long)s[1]);
  return TSP_OK;
}

namespace {

// A workgroup to `tokens` new tokens of one sequence, all heads, a thread to a piece
// of 16 bytes of K's row and V's, AU of them at a time. Workgroups behind a sequence's
// new tokens end at once. Bound by the launch (64 sequences, a token of 8 heads of 128 in
// 16 bits each: 3.6 us) or by the rows' bytes, read and written (four prompts of 1024 to
// 2047 tokens next to 12 single ones, 50 MB: 12.5 us, 4.0 TB/s).
struct AppendArgs {
  const char *K, *V;
  int64_t kb, kh, ks, vb, vh, vs;  // strides in bytes
  Pages Kp, Vp;
  Table t;
  Lengths len;
  void* out;  // lengths after
  float* W;
  int64_t wb, wh;
  uint32_t Hkv, chunks, pieces;  // pieces of a row, and of a token's rows
  uint32_t tokens, per;          // of a workgroup, workgroups of a sequence
};
constexpr int AU = 4;
__global__ __launch_bounds__(256) void append_kernel(const AppendArgs a) {
  const uint32_t b = blockIdx.x / a.per, part = blockIdx.x - b * a.per;
  const int64_t n = cached_rows(a.len, b), m = new_rows(a.len, b);
  if (part == 0 && threadIdx.x == 0) {
    const int64_t v = n + m < a.len.slots ? n + m : a.len.slots;
    if (a.len.wide)
      ((int64_t*)a.out)[b] = v;
    else
      ((int32_t*)a.out)[b] = (int32_t)v;
  }
  const int64_t i0 = (int64_t)part * a.tokens, room = a.len.slots - n, last = m < room ? m : room;
  const int64_t left = last - i0;
  if (left <= 0) return;
  // (both below 2^32: a workgroup has 2^11 pieces, or one token)
  const uint32_t total = (uint32_t)(left < a.tokens ? left : a.tokens) * a.pieces;
  const char* K = a.K + b * a.kb;
  const char* V = a.V + b * a.vb;
  for (uint32_t p0 = threadIdx.x; p0 < total; p0 += 256 * AU) {
    u32x4 k[AU], v[AU];
    uint32_t head[AU], c[AU], row[AU];
    u32x2 entry[AU];
#pragma unroll
    for (int u = 0; u < AU; ++u) {
      const uint32_t p = p0 + 256 * u < total ? p0 + 256 * u : total - 1;  // (the last piece, once more)
      const uint32_t tok = p / a.pieces, rest = p - tok * a.pieces;
      head[u] = rest / a.chunks;
      c[u] = 16 * (rest - head[u] * a.chunks);
      const int64_t i = i0 + tok;
      row[u] = (uint32_t)(n + i);
      entry[u] = entry_of_lane(a.t, b * a.t.ld, column_of(a.t, row[u] / PIECE));
      k[u] = *(const u32x4*)(K + head[u] * a.kh + i * a.ks + c[u]);
      v[u] = *(const u32x4*)(V + head[u] * a.vh + i * a.vs + c[u]);
    }
#pragma unroll
    for (int u = 0; u < AU; ++u) {
      if (a.W && c[u] == 0) a.W[b * a.wb + head[u] * a.wh + row[u]] = 0.f;
      const uint32_t page = page_of_entry(a.t, entry[u]);
      if (page == NO_PAGE) continue;
      const uint32_t r = row[u] - column_of(a.t, row[u] / PIECE) * (uint32_t)a.t.page_size;
      *(u32x4*)(a.Kp.p + page * a.Kp.page + head[u] * a.Kp.h + r * a.Kp.s + c[u]) = k[u];
      *(u32x4*)(a.Vp.p + page * a.Vp.page + head[u] * a.Vp.h + r * a.Vp.s + c[u]) = v[u];
    }
  }
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
  if ((rc = paged::check_lengths(who, B, lengths, index_type, true))) return rc;
  if (B == 0) return TSP_OK;
  const paged::Lengths len = paged::lengths_of(lengths, new_lengths, index_type, cols * page_size, N);
  if ((rc = paged::check_lengths_out(who, B, lengths_out, len))) return rc;
  if ((rc = paged::check_pages(who, "K_pages", K_pages, kps, dtype, pages, Hkv, page_size, D, true))) return rc;
  if ((rc = paged::check_pages(who, "V_pages", V_pages, vps, dtype, pages, Hkv, page_size, D, true))) return rc;
  if ((rc = paged::check_weights(who, weights, ws, B, Hkv, cols * page_size))) return rc;
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
  a.len = len;
  a.out = lengths_out;
  a.W = weights;
  if (weights) a.wb = ws[0], a.wh = ws[1];
  a.Hkv = (uint32_t)Hkv, a.chunks = (uint32_t)(D * e / 16), a.pieces = a.Hkv * a.chunks;
  if (Hkv > (int64_t(1) << 26)) return fail(TSP_EUNSUPPORTED, "%s: too many heads", who);
  a.tokens = a.pieces < 2048 ? 2048 / a.pieces : 1;
  a.per = (uint32_t)(N > 0 ? ceil_div(N, a.tokens) : 1);
  if (B * a.per > INT32_MAX) return fail(TSP_EUNSUPPORTED, "%s: too large a grid", who);
  hipLaunchKernelGGL(paged::append_kernel, dim3((unsigned)(B * a.per)), dim3(256), 0, (hipStream_t)stream, a);
  return check_launch("append launch");
}
