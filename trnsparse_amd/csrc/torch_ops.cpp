// PyTorch operator library over the C ABI: torch.ops.trnsparse_hip.*
//
// The reference reaches its device kernels through Python-level dispatch
// (trnsparse/ops.py:67-73, 204-209, 255-260, 500-505, 535-540 call into
// trnsparse/nki/dispatch.py). Here the same seam is a set of registered
// operators, so the kernels are visible to the dispatcher: torch.compile
// traces them through their Meta implementations (shapes and dtypes only),
// they run on the current HIP stream (graph capture records them like any
// other op), and C++ callers can use them without Python.
//
// Each operator allocates its outputs (and any workspace) with torch, takes
// device pointers and strides from contiguous tensors, calls one entry point
// of libtrnsparse_hip.so and turns a non-zero status into an exception
// carrying tsp_last_error(). The Python layer (trnsparse_amd/hip/dispatch.py)
// keeps the planning and caching (row orders, CSR windows and column plans,
// the attention backward's column plan) and the autograd wrappers.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <algorithm>
#include <string>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "trnsparse_hip.h"

namespace {

void check(int status, const char* who) {
  TORCH_CHECK(status == TSP_OK, who, " failed with status ", status, ": ", tsp_last_error());
}

void* stream_of(const at::Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return TSP_F32;
    case at::kDouble: return TSP_F64;
    case at::kBFloat16: return TSP_BF16;
    default: TORCH_CHECK(false, "trnsparse_hip: dtype ", t, " not supported");
  }
  return -1;
}

int index_code(at::ScalarType t) {
  TORCH_CHECK(t == at::kInt || t == at::kLong, "trnsparse_hip: index dtype ", t, " not supported");
  return t == at::kInt ? TSP_I32 : TSP_I64;
}

// a tensor the kernels may read: on `dev`, contiguous
void need(const at::Tensor& t, const at::Tensor& like, const char* name) {
  TORCH_CHECK(t.device() == like.device(), "trnsparse_hip: ", name, " is on ", t.device(), ", expected ",
              like.device());
  TORCH_CHECK(t.is_contiguous(), "trnsparse_hip: ", name, " must be contiguous");
}

const void* opt_ptr(const c10::optional<at::Tensor>& t) { return t.has_value() ? t->data_ptr() : nullptr; }

// The operators are public (C++ callers and torch.ops users reach them
// without the Python layer), and the kernels trust every size they are
// given: each operator checks that its tensors match the sizes, dtypes and
// index widths it passes on, so a mismatched call raises here instead of
// launching a kernel that reads or writes past a buffer.
void need_dtype(const at::Tensor& t, at::ScalarType dt, const char* op, const char* name) {
  TORCH_CHECK(t.scalar_type() == dt, op, ": ", name, " has dtype ", t.scalar_type(), ", expected ", dt);
}

void need_numel(const at::Tensor& t, int64_t n, const char* op, const char* name) {
  TORCH_CHECK(t.numel() == n, op, ": ", name, " has ", t.numel(), " elements, expected ", n);
}

void need_2d(const at::Tensor& t, int64_t rows, int64_t cols, const char* op, const char* name) {
  TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols, op, ": ", name, " has shape ", t.sizes(),
              ", expected [", rows, ", ", cols, "]");
}

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A BSR pattern of an m x n matrix in b x b blocks: int64 row pointers over
// the block rows, int64 column indices and (nnzb, b, b) blocks.
void need_bsr(const at::Tensor& blocks, const at::Tensor& rp, const at::Tensor& ci, int64_t m, int64_t n,
              int64_t b, const char* op) {
  TORCH_CHECK(m >= 0 && n >= 0 && b > 0, op, ": bad sizes m=", m, " n=", n, " block_size=", b);
  need_dtype(rp, at::kLong, op, "block_row_ptrs");
  need_dtype(ci, at::kLong, op, "block_col_indices");
  need_numel(rp, cdiv(m, b) + 1, op, "block_row_ptrs");
  TORCH_CHECK(blocks.dim() == 3 && blocks.size(1) == b && blocks.size(2) == b, op, ": blocks has shape ",
              blocks.sizes(), ", expected [nnzb, ", b, ", ", b, "]");
  need_numel(ci, blocks.size(0), op, "block_col_indices");
}

// ------------------------------------------------------------------- BSR

at::Tensor bsr_spmm(const at::Tensor& blocks, const at::Tensor& rp, const at::Tensor& ci,
                    const c10::optional<at::Tensor>& row_order, int64_t m, int64_t n, int64_t block_size,
                    const at::Tensor& B, at::ScalarType out_dtype) {
  for (auto* p : {&rp, &ci}) need(*p, B, "pattern");
  need(blocks, B, "blocks");
  TORCH_CHECK(B.dim() == 2 && B.stride(1) == 1, "bsr_spmm: B must be 2-D with unit column stride");
  need_bsr(blocks, rp, ci, m, n, block_size, "bsr_spmm");
  need_dtype(blocks, B.scalar_type(), "bsr_spmm", "blocks (the dtype of B)");
  TORCH_CHECK(B.size(0) >= n, "bsr_spmm: B has ", B.size(0), " rows, expected at least n = ", n);
  TORCH_CHECK(B.stride(0) >= B.size(1), "bsr_spmm: B's row stride ", B.stride(0), " is below its ", B.size(1),
              " columns");
  if (row_order.has_value() && row_order->numel()) {
    need(*row_order, B, "row_order");
    need_dtype(*row_order, at::kInt, "bsr_spmm", "row_order");
    TORCH_CHECK(row_order->numel() >= cdiv(m, block_size), "bsr_spmm: row_order has ", row_order->numel(),
                " entries for ", cdiv(m, block_size), " block rows");
  }
  const int64_t ncols = B.size(1);
  auto C = at::empty({m, ncols}, B.options().dtype(out_dtype));
  const int32_t* order = row_order.has_value() && row_order->numel() ? row_order->data_ptr<int32_t>() : nullptr;
  check(tsp_bsr_spmm(blocks.data_ptr(), dtype_code(blocks.scalar_type()), rp.data_ptr<int64_t>(),
                     ci.data_ptr<int64_t>(), blocks.size(0), block_size, m, n, B.data_ptr(), B.stride(0), ncols,
                     C.data_ptr(), ncols, dtype_code(out_dtype), order, stream_of(B)),
        "tsp_bsr_spmm");
  return C;
}

at::Tensor bsr_spmm_meta(const at::Tensor& blocks, const at::Tensor&, const at::Tensor&,
                         const c10::optional<at::Tensor>&, int64_t m, int64_t, int64_t, const at::Tensor& B,
                         at::ScalarType out_dtype) {
  return at::empty({m, B.size(1)}, B.options().dtype(out_dtype));
}

// (block_rows, col_ptrs, col_block_ids, col_block_rows, col_order)
typedef std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> ColPlan;

ColPlan bsr_col_plan_empty(const at::Tensor& ci, int64_t nbc) {
  const int64_t nnzb = ci.numel();
  return ColPlan(at::empty({nnzb}, ci.options()), at::empty({nbc + 1}, ci.options()), at::empty({nnzb}, ci.options()),
                 at::empty({nnzb}, ci.options()), at::empty({nbc > 0 ? nbc : 1}, ci.options().dtype(at::kInt)));
}

ColPlan bsr_col_plan(const at::Tensor& rp, const at::Tensor& ci, int64_t n_block_cols) {
  need(rp, ci, "block_row_ptrs");
  need(ci, ci, "block_col_indices");
  need_dtype(rp, at::kLong, "bsr_col_plan", "block_row_ptrs");
  need_dtype(ci, at::kLong, "bsr_col_plan", "block_col_indices");
  TORCH_CHECK(rp.numel() >= 1 && n_block_cols >= 0, "bsr_col_plan: bad sizes");
  const int64_t nnzb = ci.numel(), mb = rp.numel() - 1;
  ColPlan out = bsr_col_plan_empty(ci, n_block_cols);
  const int64_t wsb = tsp_bsr_col_plan_workspace_size(nnzb, mb, n_block_cols);
  TORCH_CHECK(wsb >= 0, "tsp_bsr_col_plan_workspace_size failed for ", nnzb, " blocks, ", n_block_cols,
              " block columns: ", tsp_last_error());
  at::Tensor ws;
  if (wsb > 0) ws = at::empty({wsb}, ci.options().dtype(at::kByte));
  check(tsp_bsr_col_plan(rp.data_ptr<int64_t>(), ci.data_ptr<int64_t>(), mb, n_block_cols, nnzb,
                         std::get<0>(out).data_ptr<int64_t>(), std::get<1>(out).data_ptr<int64_t>(),
                         std::get<2>(out).data_ptr<int64_t>(), std::get<3>(out).data_ptr<int64_t>(),
                         std::get<4>(out).data_ptr<int32_t>(), wsb > 0 ? ws.data_ptr() : nullptr, wsb, stream_of(ci)),
        "tsp_bsr_col_plan");
  return out;
}

ColPlan bsr_col_plan_meta(const at::Tensor&, const at::Tensor& ci, int64_t n_block_cols) {
  return bsr_col_plan_empty(ci, n_block_cols);
}

at::Tensor bsr_sddmm(const at::Tensor& G, const at::Tensor& B, const at::Tensor& block_rows,
                     const at::Tensor& block_col_indices, int64_t m, int64_t n, int64_t block_size) {
  need(G, G, "dC");
  need(B, G, "B");
  need(block_rows, G, "block_rows");
  need(block_col_indices, G, "block_col_indices");
  TORCH_CHECK(m >= 0 && n >= 0 && block_size > 0, "bsr_sddmm: bad sizes");
  TORCH_CHECK(G.dim() == 2 && G.size(0) == m, "bsr_sddmm: grad_out has shape ", G.sizes(), ", expected [", m,
              ", N]");
  need_2d(B, n, G.size(1), "bsr_sddmm", "B");
  need_dtype(B, G.scalar_type(), "bsr_sddmm", "B (the dtype of grad_out)");
  need_dtype(block_rows, at::kLong, "bsr_sddmm", "block_rows");
  need_dtype(block_col_indices, at::kLong, "bsr_sddmm", "block_col_indices");
  need_numel(block_rows, block_col_indices.numel(), "bsr_sddmm", "block_rows");
  const int64_t nnzb = block_col_indices.numel(), ncols = G.size(1);
  auto out = at::empty({nnzb, block_size, block_size}, G.options());
  check(tsp_bsr_sddmm(G.data_ptr(), ncols, m, B.data_ptr(), ncols, n, ncols, block_rows.data_ptr<int64_t>(),
                      block_col_indices.data_ptr<int64_t>(), nnzb, block_size, dtype_code(G.scalar_type()),
                      out.data_ptr(), stream_of(G)),
        "tsp_bsr_sddmm");
  return out;
}

at::Tensor bsr_sddmm_meta(const at::Tensor& G, const at::Tensor&, const at::Tensor&,
                          const at::Tensor& block_col_indices, int64_t, int64_t, int64_t block_size) {
  return at::empty({block_col_indices.size(0), block_size, block_size}, G.options());
}

at::Tensor bsr_spmm_t(const at::Tensor& blocks, const at::Tensor& cp, const at::Tensor& cbid, const at::Tensor& crow,
                      const at::Tensor& col_order, int64_t m, int64_t n, int64_t block_size, const at::Tensor& G) {
  for (auto* p : {&blocks, &cp, &cbid, &crow, &col_order}) need(*p, G, "pattern");
  TORCH_CHECK(m >= 0 && n >= 0 && block_size > 0, "bsr_spmm_t: bad sizes");
  TORCH_CHECK(G.dim() == 2 && G.size(0) == m, "bsr_spmm_t: grad_out has shape ", G.sizes(), ", expected [", m,
              ", N]");
  // (a padded grad_out is passed as its first N columns: the row stride stays)
  const int64_t ldg = m > 1 ? G.stride(0) : G.size(1);
  TORCH_CHECK((G.size(1) <= 1 || G.stride(1) == 1) && ldg >= G.size(1),
              "bsr_spmm_t: grad_out must have unit column stride and rows that do not overlap");
  // (the 128x128-tile kernels read whole rows of the stride, the last one too)
  TORCH_CHECK(G.numel() == 0 || m * ldg <= (int64_t)(G.storage().nbytes() / G.element_size()) - G.storage_offset(),
              "bsr_spmm_t: grad_out's storage ends inside the padding of its last row");
  TORCH_CHECK(blocks.dim() == 3 && blocks.size(1) == block_size && blocks.size(2) == block_size,
              "bsr_spmm_t: blocks has shape ", blocks.sizes());
  need_dtype(blocks, G.scalar_type(), "bsr_spmm_t", "blocks (the dtype of grad_out)");
  for (auto* p : {&cp, &cbid, &crow}) need_dtype(*p, at::kLong, "bsr_spmm_t", "column view");
  need_numel(cp, cdiv(n, block_size) + 1, "bsr_spmm_t", "col_ptrs");
  need_numel(cbid, blocks.size(0), "bsr_spmm_t", "col_block_ids");
  need_numel(crow, blocks.size(0), "bsr_spmm_t", "col_block_rows");
  if (col_order.numel()) {
    need_dtype(col_order, at::kInt, "bsr_spmm_t", "col_order");
    TORCH_CHECK(col_order.numel() >= cdiv(n, block_size), "bsr_spmm_t: col_order has ", col_order.numel(),
                " entries for ", cdiv(n, block_size), " block columns");
  }
  const int64_t ncols = G.size(1), nbc = cp.numel() - 1;
  auto out = at::empty({n, ncols}, G.options());
  // The entry point refuses null lists, and those of a pattern without blocks
  // have no storage: col_ptrs stands in for them (nothing reads an empty list).
  const bool stored = blocks.size(0) > 0;
  check(tsp_bsr_spmm_t(blocks.data_ptr(), dtype_code(blocks.scalar_type()), cp.data_ptr<int64_t>(),
                       (stored ? cbid : cp).data_ptr<int64_t>(), (stored ? crow : cp).data_ptr<int64_t>(), nbc,
                       block_size, m, n, G.data_ptr(), ldg, ncols, out.data_ptr(), ncols,
                       col_order.numel() ? col_order.data_ptr<int32_t>() : nullptr, stream_of(G)),
        "tsp_bsr_spmm_t");
  return out;
}

at::Tensor bsr_spmm_t_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                           const at::Tensor&, int64_t, int64_t n, int64_t, const at::Tensor& G) {
  return at::empty({n, G.size(1)}, G.options());
}

// ------------------------------------------------------------------- CSR

// A CSR matrix of m rows and n columns whose values share the dense
// operand's dtype, with one index dtype for both index arrays.
void need_csr(const at::Tensor& values, const at::Tensor& cols, const at::Tensor& ptrs, int64_t m, int64_t n,
              const at::Tensor& dense, const char* op) {
  TORCH_CHECK(m >= 0 && n >= 0, op, ": bad sizes m=", m, " n=", n);
  need_dtype(values, dense.scalar_type(), op, "values (the dtype of the dense operand)");
  index_code(cols.scalar_type());
  need_dtype(ptrs, cols.scalar_type(), op, "row_ptrs (the dtype of col_indices)");
  need_numel(ptrs, m + 1, op, "row_ptrs");
  need_numel(cols, values.numel(), op, "col_indices");
}

at::Tensor csr_spmv(const at::Tensor& values, const at::Tensor& cols, const at::Tensor& ptrs,
                    const at::Tensor& windows, int64_t m, int64_t n, const at::Tensor& x, double alpha,
                    const c10::optional<at::Tensor>& y, double beta) {
  for (auto* p : {&values, &cols, &ptrs, &windows}) need(*p, x, "matrix");
  need(x, x, "x");
  if (y.has_value()) need(*y, x, "y");
  need_csr(values, cols, ptrs, m, n, x, "csr_spmv");
  need_numel(x, n, "csr_spmv", "x");
  if (y.has_value()) {
    need_dtype(*y, x.scalar_type(), "csr_spmv", "y (the dtype of x)");
    need_numel(*y, m, "csr_spmv", "y");
  }
  need_dtype(windows, at::kLong, "csr_spmv", "windows");
  TORCH_CHECK(windows.numel() >= tsp_csr_plan_size(m, values.numel()), "csr_spmv: windows has ", windows.numel(),
              " entries, tsp_csr_plan_size gives ", tsp_csr_plan_size(m, values.numel()));
  auto out = at::empty({m}, x.options());
  check(tsp_csr_spmv(values.data_ptr(), dtype_code(values.scalar_type()), cols.data_ptr(), ptrs.data_ptr(),
                     index_code(cols.scalar_type()), m, n, values.numel(), windows.data_ptr<int64_t>(), x.data_ptr(),
                     alpha, opt_ptr(y), beta, out.data_ptr(), stream_of(x)),
        "tsp_csr_spmv");
  return out;
}

at::Tensor csr_spmv_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t m,
                         int64_t, const at::Tensor& x, double, const c10::optional<at::Tensor>&, double) {
  return at::empty({m}, x.options());
}

// The geometry is the 10 host values of tsp_csr_colplan_geometry as an int
// list (not a tensor: a CPU tensor beside device tensors cannot be traced
// by torch.compile's fake tensors).
at::Tensor csr_colplan_spmv(const at::Tensor& plan, at::IntArrayRef geometry, const at::Tensor& values,
                            const at::Tensor& cols, const at::Tensor& ptrs, int64_t m, int64_t n, const at::Tensor& x,
                            double alpha, const c10::optional<at::Tensor>& y, double beta) {
  need(plan, x, "plan");
  for (auto* p : {&values, &cols, &ptrs}) need(*p, x, "matrix");
  need(x, x, "x");
  if (y.has_value()) need(*y, x, "y");
  TORCH_CHECK(geometry.size() == 10,
              "csr_colplan_spmv: geometry must be the 10 int64 host values of tsp_csr_colplan_geometry");
  const int64_t* geom = geometry.data();
  need_csr(values, cols, ptrs, m, n, x, "csr_colplan_spmv");
  need_dtype(x, at::kFloat, "csr_colplan_spmv", "x");
  need_numel(x, n, "csr_colplan_spmv", "x");
  if (y.has_value()) {
    need_dtype(*y, at::kFloat, "csr_colplan_spmv", "y");
    need_numel(*y, m, "csr_colplan_spmv", "y");
  }
  TORCH_CHECK(plan.nbytes() >= (size_t)geom[6], "csr_colplan_spmv: plan holds ", plan.nbytes(),
              " bytes, the geometry needs ", geom[6]);
  auto out = at::empty({m}, x.options());
  at::Tensor work = at::empty({geom[8]}, x.options().dtype(at::kByte));
  check(tsp_csr_colplan_spmv(plan.data_ptr(), dtype_code(x.scalar_type()), m, n, values.numel(), geom,
                             values.data_ptr(), cols.data_ptr(), ptrs.data_ptr(), index_code(cols.scalar_type()),
                             x.data_ptr(), alpha, opt_ptr(y), beta, out.data_ptr(), work.data_ptr(), stream_of(x)),
        "tsp_csr_colplan_spmv");
  return out;
}

at::Tensor csr_colplan_spmv_meta(const at::Tensor&, at::IntArrayRef, const at::Tensor&, const at::Tensor&,
                                 const at::Tensor&, int64_t m, int64_t, const at::Tensor& x, double,
                                 const c10::optional<at::Tensor>&, double) {
  return at::empty({m}, x.options());
}

at::Tensor csr_spmm(const at::Tensor& values, const at::Tensor& cols, const at::Tensor& ptrs, int64_t m, int64_t n,
                    const at::Tensor& X, double alpha, const c10::optional<at::Tensor>& Y, double beta) {
  for (auto* p : {&values, &cols, &ptrs}) need(*p, X, "matrix");
  need(X, X, "X");
  if (Y.has_value()) need(*Y, X, "Y");
  need_csr(values, cols, ptrs, m, n, X, "csr_spmm");
  TORCH_CHECK(X.dim() == 2 && X.size(0) == n, "csr_spmm: X has shape ", X.sizes(), ", expected [", n, ", N]");
  const int64_t ncols = X.size(1);
  if (Y.has_value()) {
    need_dtype(*Y, X.scalar_type(), "csr_spmm", "Y (the dtype of X)");
    need_2d(*Y, m, ncols, "csr_spmm", "Y");
  }
  auto out = at::empty({m, ncols}, X.options());
  check(tsp_csr_spmm(values.data_ptr(), dtype_code(values.scalar_type()), cols.data_ptr(), ptrs.data_ptr(),
                     index_code(cols.scalar_type()), m, n, values.numel(), X.data_ptr(), ncols, ncols, alpha,
                     opt_ptr(Y), ncols, beta, out.data_ptr(), ncols, stream_of(X)),
        "tsp_csr_spmm");
  return out;
}

at::Tensor csr_spmm_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t m, int64_t,
                         const at::Tensor& X, double, const c10::optional<at::Tensor>&, double) {
  return at::empty({m, X.size(1)}, X.options());
}

// -------------------------------------------------------------- screened

at::Tensor screened_workspace(const at::Tensor& diag, int64_t m) {
  const int64_t bytes = tsp_screened_workspace_size(m, dtype_code(diag.scalar_type()));
  TORCH_CHECK(bytes >= 0, "tsp_screened_workspace_size failed: ", tsp_last_error());
  return at::empty({bytes > 0 ? bytes : 1}, diag.options().dtype(at::kByte));
}

at::Tensor screened_spmm(const at::Tensor& A, const at::Tensor& diag, const at::Tensor& B, double threshold_sqrt) {
  need(A, B, "A");
  need(diag, B, "diag_integrals");
  need(B, B, "B");
  TORCH_CHECK(A.dim() == 2 && A.size(0) == A.size(1), "screened_spmm: A has shape ", A.sizes(), ", expected square");
  const int64_t m = A.size(0);
  TORCH_CHECK(B.dim() == 2 && B.size(0) == m, "screened_spmm: B has shape ", B.sizes(), ", expected [", m, ", N]");
  need_dtype(A, B.scalar_type(), "screened_spmm", "A (the dtype of B)");
  TORCH_CHECK(diag.dim() == 1, "screened_spmm: diag_integrals must be 1-D");
  need_numel(diag, m, "screened_spmm", "diag_integrals");
  const int64_t ncols = B.size(1);
  auto C = at::empty({m, ncols}, B.options());
  auto ws = screened_workspace(diag, m);
  check(tsp_screened_spmm(A.data_ptr(), dtype_code(A.scalar_type()), A.size(1), diag.data_ptr(),
                          dtype_code(diag.scalar_type()), threshold_sqrt, m, B.data_ptr(), ncols, ncols, C.data_ptr(),
                          ncols, ws.data_ptr(), stream_of(B)),
        "tsp_screened_spmm");
  return C;
}

at::Tensor screened_spmm_meta(const at::Tensor& A, const at::Tensor&, const at::Tensor& B, double) {
  return at::empty({A.size(0), B.size(1)}, B.options());
}

std::tuple<at::Tensor, at::Tensor> screened_spmm_backward(const at::Tensor& A, const at::Tensor& diag,
                                                          const at::Tensor& B, double threshold_sqrt,
                                                          const at::Tensor& dC, bool need_a, bool need_b) {
  need(A, dC, "A");
  need(diag, dC, "diag_integrals");
  need(B, dC, "B");
  need(dC, dC, "grad_out");
  TORCH_CHECK(A.dim() == 2 && A.size(0) == A.size(1), "screened_spmm_backward: A has shape ", A.sizes(),
              ", expected square");
  const int64_t m = A.size(0);
  TORCH_CHECK(dC.dim() == 2 && dC.size(0) == m, "screened_spmm_backward: grad_out has shape ", dC.sizes(),
              ", expected [", m, ", N]");
  need_2d(B, m, dC.size(1), "screened_spmm_backward", "B");
  need_dtype(A, dC.scalar_type(), "screened_spmm_backward", "A (the dtype of grad_out)");
  need_dtype(B, dC.scalar_type(), "screened_spmm_backward", "B (the dtype of grad_out)");
  TORCH_CHECK(diag.dim() == 1, "screened_spmm_backward: diag_integrals must be 1-D");
  need_numel(diag, m, "screened_spmm_backward", "diag_integrals");
  const int64_t ncols = dC.size(1);
  // a gradient that is not asked for comes back empty (no kernel runs for it)
  auto dA = need_a ? at::empty({m, m}, A.options()) : at::empty({0}, A.options());
  auto dB = need_b ? at::empty({m, ncols}, B.options()) : at::empty({0}, B.options());
  auto ws = screened_workspace(diag, m);
  check(tsp_screened_spmm_backward(A.data_ptr(), dtype_code(A.scalar_type()), m, diag.data_ptr(),
                                   dtype_code(diag.scalar_type()), threshold_sqrt, m, B.data_ptr(), ncols, ncols,
                                   dC.data_ptr(), ncols, need_a ? dA.data_ptr() : nullptr, m,
                                   need_b ? dB.data_ptr() : nullptr, ncols, ws.data_ptr(), stream_of(dC)),
        "tsp_screened_spmm_backward");
  return {dA, dB};
}

std::tuple<at::Tensor, at::Tensor> screened_spmm_backward_meta(const at::Tensor& A, const at::Tensor&,
                                                               const at::Tensor& B, double, const at::Tensor& dC,
                                                               bool need_a, bool need_b) {
  const int64_t m = A.size(0);
  return {need_a ? at::empty({m, m}, A.options()) : at::empty({0}, A.options()),
          need_b ? at::empty({m, dC.size(1)}, B.options()) : at::empty({0}, B.options())};
}

// ------------------------------------------------------------- attention

at::ScalarType stat_dtype(const at::Tensor& Q) { return Q.scalar_type() == at::kDouble ? at::kDouble : at::kFloat; }

std::tuple<at::Tensor, at::Tensor, at::Tensor> bsa_fwd(const at::Tensor& Q, const at::Tensor& K, const at::Tensor& V,
                                                       const at::Tensor& rp, const at::Tensor& ci, int64_t block_size,
                                                       double scale, bool return_stats) {
  for (auto* p : {&K, &V, &rp, &ci}) need(*p, Q, "operand");
  need(Q, Q, "Q");
  TORCH_CHECK(Q.dim() == 3 && K.sizes() == Q.sizes() && V.sizes() == Q.sizes(),
              "bsa_fwd: Q, K, V must be (heads, seq, head_dim) of one shape");
  TORCH_CHECK(block_size > 0, "bsa_fwd: block_size must be positive");
  for (auto* p : {&K, &V}) need_dtype(*p, Q.scalar_type(), "bsa_fwd", "K and V (the dtype of Q)");
  const int64_t H = Q.size(0), S = Q.size(1), D = Q.size(2), Mt = S / block_size;
  need_dtype(rp, at::kLong, "bsa_fwd", "block_row_ptrs");
  need_dtype(ci, at::kLong, "bsa_fwd", "block_col_indices");
  TORCH_CHECK(rp.numel() >= Mt + 1, "bsa_fwd: block_row_ptrs has ", rp.numel(), " entries, expected at least ",
              Mt + 1);
  auto O = at::empty_like(Q);
  at::Tensor rmax, rden;
  if (return_stats) {
    rmax = at::empty({H, Mt, block_size}, Q.options().dtype(stat_dtype(Q)));
    rden = at::empty({H, Mt, block_size}, Q.options().dtype(stat_dtype(Q)));
  } else {
    rmax = at::empty({0}, Q.options().dtype(stat_dtype(Q)));
    rden = at::empty({0}, Q.options().dtype(stat_dtype(Q)));
  }
  check(tsp_bsa_fwd(Q.data_ptr(), K.data_ptr(), V.data_ptr(), dtype_code(Q.scalar_type()), H, S, D,
                    rp.data_ptr<int64_t>(), ci.data_ptr<int64_t>(), block_size, scale, O.data_ptr(),
                    return_stats ? rmax.data_ptr() : nullptr, return_stats ? rden.data_ptr() : nullptr, stream_of(Q)),
        "tsp_bsa_fwd");
  return {O, rmax, rden};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> bsa_fwd_meta(const at::Tensor& Q, const at::Tensor&, const at::Tensor&,
                                                            const at::Tensor&, const at::Tensor&, int64_t block_size,
                                                            double, bool return_stats) {
  const int64_t H = Q.size(0), Mt = Q.size(1) / block_size;
  auto so = Q.options().dtype(stat_dtype(Q));
  if (!return_stats) return {at::empty_like(Q), at::empty({0}, so), at::empty({0}, so)};
  return {at::empty_like(Q), at::empty({H, Mt, block_size}, so), at::empty({H, Mt, block_size}, so)};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> bsa_bwd(
    const at::Tensor& Q, const at::Tensor& K, const at::Tensor& V, const at::Tensor& O, const at::Tensor& dO,
    const at::Tensor& rp, const at::Tensor& ci, const at::Tensor& cp, const at::Tensor& crow, int64_t n_block_cols,
    int64_t block_size, double scale, const at::Tensor& row_max, const at::Tensor& row_denom, const at::Tensor& plan,
    int64_t n_items, int64_t n_splits, int64_t n_partials) {
  for (auto* p : {&K, &V, &O, &dO, &rp, &ci, &cp, &crow, &row_max, &row_denom, &plan}) need(*p, Q, "operand");
  need(Q, Q, "Q");
  TORCH_CHECK(Q.dim() == 3, "bsa_bwd: operands must be (heads, seq, head_dim)");
  TORCH_CHECK(block_size > 0, "bsa_bwd: block_size must be positive");
  for (auto* p : {&K, &V, &O, &dO}) {
    TORCH_CHECK(p->sizes() == Q.sizes(), "bsa_bwd: K, V, O and grad_out must have Q's shape ", Q.sizes());
    need_dtype(*p, Q.scalar_type(), "bsa_bwd", "K, V, O and grad_out (the dtype of Q)");
  }
  const int64_t H = Q.size(0), S = Q.size(1), D = Q.size(2), Mt = S / block_size;
  for (auto* p : {&rp, &ci, &cp, &crow}) need_dtype(*p, at::kLong, "bsa_bwd", "mask views");
  TORCH_CHECK(rp.numel() >= Mt + 1, "bsa_bwd: block_row_ptrs has ", rp.numel(), " entries, expected at least ",
              Mt + 1);
  TORCH_CHECK(n_block_cols >= 0, "bsa_bwd: negative n_block_cols");
  need_numel(cp, n_block_cols + 1, "bsa_bwd", "col_ptrs");
  // the column view covers the stored blocks of the block rows below Mt
  TORCH_CHECK(crow.numel() <= std::max<int64_t>(ci.numel(), 1), "bsa_bwd: col_block_rows has ", crow.numel(),
              " entries, more than the mask's ", ci.numel(), " blocks");
  for (auto* p : {&row_max, &row_denom}) {
    need_dtype(*p, stat_dtype(Q), "bsa_bwd", "row_max and row_denom");
    need_numel(*p, H * Mt * block_size, "bsa_bwd", "row_max and row_denom");
  }
  need_dtype(plan, at::kInt, "bsa_bwd", "plan");
  TORCH_CHECK(n_items >= 0 && n_splits >= 0 && n_partials >= 0, "bsa_bwd: negative plan counts");
  TORCH_CHECK(plan.numel() >= 4 + 4 * n_items + 4 * n_splits, "bsa_bwd: plan has ", plan.numel(),
              " entries, its header counts need ", 4 + 4 * n_items + 4 * n_splits);
  auto dQ = at::empty_like(Q), dK = at::empty_like(Q), dV = at::empty_like(Q);
  const int64_t wsb = tsp_bsa_bwd_workspace_size(H, S, D, n_partials);
  TORCH_CHECK(wsb >= 0, "tsp_bsa_bwd_workspace_size failed: ", tsp_last_error());
  auto ws = at::empty({wsb > 0 ? wsb : 1}, Q.options().dtype(at::kByte));
  check(tsp_bsa_bwd(Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(), dO.data_ptr(), dtype_code(Q.scalar_type()),
                    H, S, D, rp.data_ptr<int64_t>(), ci.data_ptr<int64_t>(), cp.data_ptr<int64_t>(),
                    crow.data_ptr<int64_t>(), n_block_cols, block_size, scale, row_max.data_ptr(),
                    row_denom.data_ptr(), dQ.data_ptr(), dK.data_ptr(), dV.data_ptr(), plan.data_ptr<int32_t>(),
                    n_items, n_splits, n_partials, ws.data_ptr(), stream_of(Q)),
        "tsp_bsa_bwd");
  return {dQ, dK, dV};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> bsa_bwd_meta(
    const at::Tensor& Q, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
    const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t, int64_t, double,
    const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t, int64_t, int64_t) {
  return {at::empty_like(Q), at::empty_like(Q), at::empty_like(Q)};
}

// ------------------------------------- attention over strided operands

int attn_dtype(at::ScalarType t, const char* who) {
  TORCH_CHECK(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf, who, ": dtype ", t, " not supported");
  return t == at::kFloat ? TSP_F32 : t == at::kHalf ? TSP_F16 : TSP_BF16;
}

// head_dim as the kernels take it: whole 16-byte pieces
int64_t piece_dim(const at::Tensor& t) {
  const int64_t ce = 16 / t.element_size();
  return (t.size(-1) + ce - 1) / ce * ce;
}

// A (batch, heads, rows, head_dim) operand as the kernels take it: t itself
// where its strides and address are whole 16-byte pieces and its rows lie
// apart, else a contiguous copy (head_dim padded with zeros).
at::Tensor attn_operand(const at::Tensor& t) {
  const int64_t ce = 16 / t.element_size(), D = t.size(3), Dp = piece_dim(t);
  if (D != Dp) return at::constant_pad_nd(t, {0, Dp - D}).contiguous();
  bool ok = (t.stride(3) == 1 || D == 1) && (uintptr_t)t.data_ptr() % 16 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) <= 1 || t.stride(i) % ce == 0);
  ok = ok && (t.size(2) <= 1 || (t.stride(2) >= D && t.stride(2) * t.element_size() < (1 << 24)));
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

struct Strides {
  int64_t s[3];
  explicit Strides(const at::Tensor& t) {
    for (int i = 0; i < 3; ++i) s[i] = t.size(i) <= 1 ? (i == 2 ? t.size(3) : 0) : t.stride(i);
  }
};

// A result of the operand's shape with head_dim Dp, in the operand's order of
// heads and rows.
at::Tensor attn_like(const at::Tensor& t, int64_t Dp) {
  const int64_t B = t.size(0), H = t.size(1), S = t.size(2);
  if (H > 1 && S > 1 && t.stride(2) > t.stride(1)) return at::empty({B, S, H, Dp}, t.options()).transpose(1, 2);
  return at::empty({B, H, S, Dp}, t.options());
}
at::Tensor attn_trim(const at::Tensor& t, int64_t D) { return t.size(3) == D ? t : t.narrow(3, 0, D).contiguous(); }

void need_4d(const at::Tensor& t, const at::Tensor& Q, const char* who, const char* name) {
  TORCH_CHECK(t.device() == Q.device(), who, ": ", name, " is on ", t.device(), ", expected ", Q.device());
  TORCH_CHECK(t.dim() == 4, who, ": ", name, " must be (batch, heads, rows, head_dim)");
  need_dtype(t, Q.scalar_type(), who, name);
  TORCH_CHECK(t.size(3) == Q.size(3), who, ": head_dim of ", name, " is ", t.size(3), ", expected ", Q.size(3));
}

const void* lengths_ptr(const c10::optional<at::Tensor>& t, int64_t B, const at::Tensor& Q, const char* who, int& code) {
  code = TSP_I64;
  if (!t.has_value()) return nullptr;
  need(*t, Q, "lengths");
  code = index_code(t->scalar_type());
  TORCH_CHECK(t->dim() == 1 && t->numel() == B, who, ": lengths must be (batch,)");
  return t->data_ptr();
}

struct Workspace {
  at::Tensor t;  // none when no byte is needed
  Workspace(int64_t bytes, const at::Tensor& like, const char* who) {
    TORCH_CHECK(bytes >= 0, who, " failed: ", tsp_last_error());
    if (bytes > 0) t = at::empty({bytes}, like.options().dtype(at::kByte));
  }
  void* ptr() const { return t.defined() ? t.data_ptr() : nullptr; }
};

void cross_shapes(const at::Tensor& Q, const at::Tensor& K, const at::Tensor& V, const char* who) {
  need_4d(Q, Q, who, "Q");
  need_4d(K, Q, who, "K");
  need_4d(V, Q, who, "V");
  TORCH_CHECK(K.sizes() == V.sizes() && K.size(0) == Q.size(0), who, ": Q ", Q.sizes(), ", K ", K.sizes(), " and V ",
              V.sizes(), " do not belong together");
  TORCH_CHECK(Q.size(3) >= 1 && Q.size(3) <= 128, who, ": head_dim ", Q.size(3), " is not in 1 .. 128");
  TORCH_CHECK(K.size(1) > 0 && Q.size(1) % K.size(1) == 0, who, ": ", Q.size(1), " query heads do not divide over ",
              K.size(1), " key heads");
}

// the result, and with `lse` its rows' log-sum-exps
at::Tensor cross_forward(const at::Tensor& Q_, const at::Tensor& K_, const at::Tensor& V_,
                         const c10::optional<at::Tensor>& key_lengths, double scale, at::Tensor* lse) {
  const char* who = "cross_attn_fwd";
  const c10::DeviceGuard guard(Q_.device());
  cross_shapes(Q_, K_, V_, who);
  const int code = attn_dtype(Q_.scalar_type(), who);
  const auto Q = attn_operand(Q_), K = attn_operand(K_), V = attn_operand(V_);
  const int64_t B = Q.size(0), Hq = Q.size(1), Sq = Q.size(2), D = Q.size(3), Hk = K.size(1), L = K.size(2);
  int icode;
  const void* lens = lengths_ptr(key_lengths, B, Q, who, icode);
  auto O = attn_like(Q_, D);
  if (lse) *lse = at::empty({B, Hq, Sq}, Q.options().dtype(at::kFloat));
  const int64_t wsb = tsp_cross_attn_workspace_size(code, B, Hq, Hk, Sq, L, D);
  const Workspace ws(wsb, Q, who);
  check(tsp_cross_attn_fwd(Q.data_ptr(), Strides(Q).s, K.data_ptr(), Strides(K).s, V.data_ptr(), Strides(V).s, code, B,
                           Hq, Hk, Sq, L, D, lens, icode, scale, O.data_ptr(), Strides(O).s,
                           lse ? lse->data_ptr<float>() : nullptr, ws.ptr(), wsb, stream_of(Q)),
        "tsp_cross_attn_fwd");
  return attn_trim(O, Q_.size(3));
}

std::tuple<at::Tensor, at::Tensor> cross_attn_fwd(const at::Tensor& Q, const at::Tensor& K, const at::Tensor& V,
                                                  const c10::optional<at::Tensor>& key_lengths, double scale,
                                                  bool return_lse) {
  at::Tensor lse;
  auto O = cross_forward(Q, K, V, key_lengths, scale, return_lse ? &lse : nullptr);
  if (!return_lse) lse = at::empty({0}, Q.options().dtype(at::kFloat));
  return {O, lse};
}

std::tuple<at::Tensor, at::Tensor> cross_attn_fwd_meta(const at::Tensor& Q, const at::Tensor&, const at::Tensor&,
                                                       const c10::optional<at::Tensor>&, double, bool return_lse) {
  auto lo = Q.options().dtype(at::kFloat);
  auto lse = return_lse ? at::empty({Q.size(0), Q.size(1), Q.size(2)}, lo) : at::empty({0}, lo);
  return {Q.size(3) == piece_dim(Q) ? attn_like(Q, Q.size(3)) : at::empty(Q.sizes(), Q.options()), lse};
}

// dK and dV come back empty when they are not asked for
std::tuple<at::Tensor, at::Tensor, at::Tensor> cross_attn_bwd(const at::Tensor& Q_, const at::Tensor& K_,
                                                              const at::Tensor& V_, const at::Tensor& O_,
                                                              const at::Tensor& dO_, const at::Tensor& lse,
                                                              const c10::optional<at::Tensor>& key_lengths, double scale,
                                                              bool need_kv) {
  const char* who = "cross_attn_bwd";
  const c10::DeviceGuard guard(Q_.device());
  cross_shapes(Q_, K_, V_, who);
  need_4d(O_, Q_, who, "O");
  need_4d(dO_, Q_, who, "grad_out");
  TORCH_CHECK(O_.sizes() == Q_.sizes() && dO_.sizes() == Q_.sizes(), who, ": O and grad_out must have Q's shape");
  const int code = attn_dtype(Q_.scalar_type(), who);
  const auto Q = attn_operand(Q_), K = attn_operand(K_), V = attn_operand(V_), O = attn_operand(O_),
             dO = attn_operand(dO_);
  const int64_t B = Q.size(0), Hq = Q.size(1), Sq = Q.size(2), D = Q.size(3), Hk = K.size(1), L = K.size(2);
  need(lse, Q, "lse");
  need_dtype(lse, at::kFloat, who, "lse");
  need_numel(lse, B * Hq * Sq, who, "lse");
  int icode;
  const void* lens = lengths_ptr(key_lengths, B, Q, who, icode);
  auto dQ = attn_like(Q_, D);
  auto dK = need_kv ? attn_like(K_, D) : at::empty({0, 0, 0, D}, K.options());
  auto dV = need_kv ? attn_like(V_, D) : at::empty({0, 0, 0, D}, V.options());
  const int64_t wsb = tsp_cross_attn_bwd_workspace_size(code, B, Hq, Hk, Sq, L, D);
  const Workspace ws(wsb, Q, who);
  check(tsp_cross_attn_bwd(Q.data_ptr(), Strides(Q).s, K.data_ptr(), Strides(K).s, V.data_ptr(), Strides(V).s,
                           O.data_ptr(), Strides(O).s, dO.data_ptr(), Strides(dO).s, lse.data_ptr<float>(), code, B, Hq,
                           Hk, Sq, L, D, lens, icode, scale, dQ.data_ptr(), Strides(dQ).s,
                           need_kv ? dK.data_ptr() : nullptr, Strides(dK).s, need_kv ? dV.data_ptr() : nullptr,
                           Strides(dV).s, ws.ptr(), wsb, stream_of(Q)),
        "tsp_cross_attn_bwd");
  const int64_t d = Q_.size(3);
  return {attn_trim(dQ, d), attn_trim(dK, d), attn_trim(dV, d)};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> cross_attn_bwd_meta(const at::Tensor& Q, const at::Tensor& K,
                                                                   const at::Tensor& V, const at::Tensor&,
                                                                   const at::Tensor&, const at::Tensor&,
                                                                   const c10::optional<at::Tensor>&, double,
                                                                   bool need_kv) {
  auto like = [&](const at::Tensor& t, bool need) {
    if (!need) return at::empty({0, 0, 0, t.size(3)}, t.options());
    return t.size(3) == piece_dim(t) ? attn_like(t, t.size(3)) : at::empty(t.sizes(), t.options());
  };
  return {like(Q, true), like(K, need_kv), like(V, need_kv)};
}

at::Tensor prefix_attn_fwd(const at::Tensor& Q_, const at::Tensor& PK_, const at::Tensor& PV_, const at::Tensor& K_,
                           const at::Tensor& V_, const c10::optional<at::Tensor>& lengths, double scale) {
  const char* who = "prefix_attn_fwd";
  const c10::DeviceGuard guard(Q_.device());
  cross_shapes(Q_, K_, V_, who);
  TORCH_CHECK(PK_.dim() == 3 && PK_.sizes() == PV_.sizes() && PK_.size(0) == K_.size(1), who, ": prefix_K ",
              PK_.sizes(), " and prefix_V ", PV_.sizes(), " must be (kv_heads, prefix, head_dim)");
  const int code = attn_dtype(Q_.scalar_type(), who);
  const auto pk4 = PK_.unsqueeze(0), pv4 = PV_.unsqueeze(0);
  need_4d(pk4, Q_, who, "prefix K");
  need_4d(pv4, Q_, who, "prefix V");
  const auto Q = attn_operand(Q_), K = attn_operand(K_), V = attn_operand(V_), PK = attn_operand(pk4),
             PV = attn_operand(pv4);
  const int64_t B = Q.size(0), Hq = Q.size(1), Sq = Q.size(2), D = Q.size(3), Hk = K.size(1), S = K.size(2);
  const int64_t P = PK.size(2);
  int icode;
  const void* lens = lengths_ptr(lengths, B, Q, who, icode);
  auto O = attn_like(Q_, D);
  const int64_t wsb = tsp_prefix_attn_workspace_size(code, B, Hq, Hk, Sq, P, S, D);
  const Workspace ws(wsb, Q, who);
  check(tsp_prefix_attn_fwd(Q.data_ptr(), Strides(Q).s, PK.data_ptr(), Strides(PK).s, PV.data_ptr(), Strides(PV).s,
                            K.data_ptr(), Strides(K).s, V.data_ptr(), Strides(V).s, code, B, Hq, Hk, Sq, P, S, D, lens,
                            icode, scale, O.data_ptr(), Strides(O).s, ws.ptr(), wsb, stream_of(Q)),
        "tsp_prefix_attn_fwd");
  return attn_trim(O, Q_.size(3));
}

at::Tensor prefix_attn_fwd_meta(const at::Tensor& Q, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                const at::Tensor&, const c10::optional<at::Tensor>&, double) {
  return Q.size(3) == piece_dim(Q) ? attn_like(Q, Q.size(3)) : at::empty(Q.sizes(), Q.options());
}

// ------------------------------------ a key and value cache in pages

// The pages, the table and the lengths of a call, checked.
struct PagedArgs {
  int code, tcode, icode;
  int64_t B, Hk, pages, page_size, D, cols, slots, tstride;
  const void *table, *lens, *fresh = nullptr;
  int64_t ks[3], vs[3];
  at::Tensor held[3];  // the table and the lengths as the kernels take them, where these are copies

  static void page_strides(const at::Tensor& t, int64_t* s) {
    for (int i = 0; i < 3; ++i) s[i] = t.size(i) <= 1 ? (i == 2 ? t.size(3) : 0) : t.stride(i);
  }
  void need_pages(const at::Tensor& t, const at::Tensor& like, const char* who, const char* name, bool written) const {
    TORCH_CHECK(t.device() == like.device(), who, ": ", name, " is on ", t.device(), ", expected ", like.device());
    need_dtype(t, like.scalar_type(), who, name);
    TORCH_CHECK(t.dim() == 4, who, ": ", name, " must be (pages, kv_heads, page_size, head_dim)");
    const int64_t ce = 16 / t.element_size();
    TORCH_CHECK(t.size(2) > 0 && t.size(2) % 16 == 0, who, ": page_size ", t.size(2), " must be a multiple of 16");
    TORCH_CHECK(t.size(3) >= 1 && t.size(3) <= 128 && t.size(3) % ce == 0, who, ": head_dim ", t.size(3),
                " must be at most 128 and a multiple of ", ce);
    bool ok = (t.stride(3) == 1 || t.size(3) == 1) && (t.numel() == 0 || (uintptr_t)t.data_ptr() % 16 == 0);
    for (int i = 0; i < 3; ++i)
      ok = ok && (t.size(i) <= 1 || (t.stride(i) % ce == 0 && t.stride(i) >= (i == 2 ? t.size(3) : written ? 1 : 0)));
    TORCH_CHECK(ok, who, ": ", name, " needs unit stride over head_dim and other strides of whole 16-byte pieces, got ",
                t.strides(), written ? " (and is written: its rows lie apart)" : "");
  }
  PagedArgs(const at::Tensor& K, const at::Tensor& V, const at::Tensor& table_, const at::Tensor& lengths,
            const c10::optional<at::Tensor>& new_lengths, const at::Tensor& like, bool written, const char* who) {
    code = attn_dtype(like.scalar_type(), who);
    need_pages(K, like, who, "K_pages", written);
    need_pages(V, like, who, "V_pages", written);
    TORCH_CHECK(K.sizes() == V.sizes(), who, ": K_pages ", K.sizes(), " and V_pages ", V.sizes(), " do not belong together");
    TORCH_CHECK(!written || K.numel() == 0 || K.data_ptr() != V.data_ptr(), who, ": K_pages and V_pages are the same");
    pages = K.size(0), Hk = K.size(1), page_size = K.size(2), D = K.size(3);
    TORCH_CHECK(Hk > 0, who, ": no key heads");
    page_strides(K, ks);
    page_strides(V, vs);
    TORCH_CHECK(table_.device() == like.device(), who, ": block_table is on ", table_.device());
    TORCH_CHECK(table_.dim() == 2, who, ": block_table must be (batch, columns)");
    tcode = index_code(table_.scalar_type());
    B = table_.size(0), cols = table_.size(1), slots = cols * page_size;
    const at::Tensor* t = &table_;
    if (cols > 1 && table_.stride(1) != 1) t = &(held[0] = table_.contiguous());
    table = t->data_ptr();
    tstride = B > 1 ? t->stride(0) : cols;
    lens = lengths_of(lengths, "lengths", like, who, held[1]);
    icode = index_code(lengths.scalar_type());
    if (new_lengths.has_value()) {
      fresh = lengths_of(*new_lengths, "new_lengths", like, who, held[2]);
      if (index_code(new_lengths->scalar_type()) != icode) icode |= TSP_NEW_OTHER;
    }
  }
  const void* lengths_of(const at::Tensor& l, const char* name, const at::Tensor& like, const char* who, at::Tensor& kept) const {
    TORCH_CHECK(l.device() == like.device(), who, ": ", name, " is on ", l.device(), ", expected ", like.device());
    TORCH_CHECK(l.dim() == 1 && l.numel() == B, who, ": ", name, " must be (batch,)");
    kept = l.contiguous();
    return kept.data_ptr();
  }
};

// accumulated weights (batch, kv_heads, slots)
const int64_t* need_weights(const at::Tensor& w, const PagedArgs& p, const at::Tensor& like, const char* who, int64_t* s) {
  TORCH_CHECK(w.device() == like.device(), who, ": weights are on ", w.device());
  need_dtype(w, at::kFloat, who, "weights");
  TORCH_CHECK(w.dim() == 3 && w.size(0) == p.B && w.size(1) == p.Hk && w.size(2) == p.slots, who, ": weights ", w.sizes(),
              " must be (batch, kv_heads, slots) = (", p.B, ", ", p.Hk, ", ", p.slots, ")");
  for (int i = 0; i < 2; ++i) {
    s[i] = w.size(i) <= 1 ? 0 : w.stride(i);
    TORCH_CHECK(w.size(i) <= 1 || w.stride(i) >= 1, who, ": weights are written: their rows lie apart");
  }
  TORCH_CHECK(w.size(2) <= 1 || w.stride(2) == 1, who, ": weights need unit stride over slots");
  return s;
}

// What an operator writes in place counts as written (before it is: a tensor that may
// not be written is refused).
void written(std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts) t->unsafeGetTensorImpl()->bump_version();
}

at::Tensor paged_attn_fwd(const at::Tensor& Q_, const at::Tensor& K, const at::Tensor& V, const at::Tensor& table,
                          const at::Tensor& lengths, const c10::optional<at::Tensor>& new_lengths, double scale,
                          const c10::optional<at::Tensor>& weights) {
  const char* who = "paged_attn_fwd";
  const c10::DeviceGuard guard(Q_.device());
  need_4d(Q_, Q_, who, "Q");
  const PagedArgs p(K, V, table, lengths, new_lengths, Q_, false, who);
  TORCH_CHECK(Q_.size(0) == p.B && Q_.size(3) == p.D && Q_.size(1) % p.Hk == 0, who, ": Q ", Q_.sizes(), ", K_pages ",
              K.sizes(), " and block_table ", table.sizes(), " do not belong together");
  int64_t ws2[2];
  if (weights.has_value()) need_weights(*weights, p, Q_, who, ws2);
  const auto Q = attn_operand(Q_);
  const int64_t Hq = Q.size(1), Sq = Q.size(2);
  auto O = attn_like(Q_, p.D);
  const int64_t wsb = tsp_paged_attn_workspace_size(p.code, p.B, Hq, p.Hk, Sq, p.slots, p.D, new_lengths.has_value(),
                                                    weights.has_value());
  const Workspace ws(wsb, Q, who);
  if (weights.has_value()) written({&*weights});
  check(tsp_paged_attn_fwd(Q.data_ptr(), Strides(Q).s, K.data_ptr(), p.ks, V.data_ptr(), p.vs, p.code, p.B, Hq, p.Hk, Sq,
                           p.pages, p.page_size, p.D, p.table, p.tcode, p.tstride, p.cols, p.lens, p.fresh,
                           p.icode, scale, O.data_ptr(), Strides(O).s,
                           weights.has_value() ? weights->data_ptr<float>() : nullptr, ws2, ws.ptr(), wsb, stream_of(Q)),
        "tsp_paged_attn_fwd");
  return O;
}

at::Tensor paged_attn_fwd_meta(const at::Tensor& Q, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                               const at::Tensor&, const c10::optional<at::Tensor>&, double,
                               const c10::optional<at::Tensor>&) {
  return attn_like(Q, Q.size(3));
}

// t, or a copy of it where it may share bytes with a tensor that is written (by the spans of both).
at::Tensor apart_from(const at::Tensor& t, std::initializer_list<const at::Tensor*> written) {
  const auto end_of = [](const at::Tensor& x) {
    int64_t last = 1;
    for (int64_t i = 0; i < x.dim(); ++i) last += (x.size(i) - 1) * x.stride(i);
    return (const char*)x.data_ptr() + last * x.element_size();
  };
  if (t.numel() == 0) return t;
  for (const at::Tensor* w : written)
    if (w->numel() > 0 && (const char*)t.data_ptr() < end_of(*w) && (const char*)w->data_ptr() < end_of(t))
      return t.clone(at::MemoryFormat::Contiguous);
  return t;
}

at::Tensor paged_append(const at::Tensor& K_, const at::Tensor& V_, const at::Tensor& Kp, const at::Tensor& Vp,
                        const at::Tensor& table, const at::Tensor& lengths, const c10::optional<at::Tensor>& new_lengths,
                        const c10::optional<at::Tensor>& weights) {
  const char* who = "paged_append";
  const c10::DeviceGuard guard(Kp.device());
  const PagedArgs p(Kp, Vp, table, lengths, new_lengths, Kp, true, who);
  need_4d(K_, Kp, who, "K");
  need_4d(V_, Kp, who, "V");
  TORCH_CHECK(K_.sizes() == V_.sizes() && K_.size(0) == p.B && K_.size(1) == p.Hk, who, ": K ", K_.sizes(), ", V ",
              V_.sizes(), ", K_pages ", Kp.sizes(), " and block_table ", table.sizes(), " do not belong together");
  int64_t ws2[2];
  if (weights.has_value()) need_weights(*weights, p, Kp, who, ws2);
  // (new rows that stand in the pages are read before any are written)
  const auto K = apart_from(attn_operand(K_), {&Kp, &Vp}), V = apart_from(attn_operand(V_), {&Kp, &Vp});
  auto out = at::empty({p.B}, lengths.options());
  written({&Kp, &Vp});
  if (weights.has_value()) written({&*weights});
  check(tsp_paged_append(K.data_ptr(), Strides(K).s, V.data_ptr(), Strides(V).s, Kp.data_ptr(), p.ks, Vp.data_ptr(), p.vs,
                         p.code, p.B, p.Hk, K.size(2), p.pages, p.page_size, p.D, p.table, p.tcode, p.tstride,
                         p.cols, p.lens, p.fresh, p.icode, out.data_ptr(),
                         weights.has_value() ? weights->data_ptr<float>() : nullptr, ws2, stream_of(Kp)),
        "tsp_paged_append");
  return out;
}

at::Tensor paged_append_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                             const at::Tensor&, const at::Tensor& lengths, const c10::optional<at::Tensor>&,
                             const c10::optional<at::Tensor>&) {
  return at::empty(lengths.sizes(), lengths.options());
}

at::Tensor paged_evict(const at::Tensor& Kp, const at::Tensor& Vp, const at::Tensor& weights, const at::Tensor& table,
                       const at::Tensor& lengths, int64_t budget, int64_t recent) {
  const char* who = "paged_evict";
  const c10::DeviceGuard guard(Kp.device());
  const PagedArgs p(Kp, Vp, table, lengths, c10::nullopt, Kp, true, who);
  int64_t ws2[2];
  need_weights(weights, p, Kp, who, ws2);
  TORCH_CHECK(0 <= recent && recent <= budget, who, ": recent ", recent, " is not in 0 .. budget ", budget);
  auto out = at::empty({p.B}, lengths.options());
  const int64_t wsb = tsp_paged_evict_workspace_size(p.code, p.B, p.Hk, p.slots, p.D, budget);
  const Workspace ws(wsb, Kp, who);
  written({&Kp, &Vp, &weights});
  check(tsp_paged_evict(Kp.data_ptr(), p.ks, Vp.data_ptr(), p.vs, p.code, p.B, p.Hk, p.pages, p.page_size, p.D,
                        p.table, p.tcode, p.tstride, p.cols, p.lens, p.icode, weights.data_ptr<float>(), ws2,
                        budget, recent, out.data_ptr(), ws.ptr(), wsb, stream_of(Kp)),
        "tsp_paged_evict");
  return out;
}

at::Tensor paged_evict_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                            const at::Tensor& lengths, int64_t, int64_t) {
  return at::empty(lengths.sizes(), lengths.options());
}

// --------------------------------- norm and rotation of query and key heads

// t with unit stride over head_dim (a contiguous copy where it has another)
at::Tensor unit_rows(const at::Tensor& t) {
  return t.stride(3) == 1 || t.size(3) == 1 ? t : t.clone(at::MemoryFormat::Contiguous);
}

struct RopeArgs {
  int code, wcode, icode;
  int64_t pos_b, pos_s, rot;
  RopeArgs(const at::Tensor& Q, const at::Tensor& K, const at::Tensor& wq, const at::Tensor& wk, const at::Tensor& pos,
           const at::Tensor& freq, const char* who) {
    need_4d(Q, Q, who, "Q");
    need_4d(K, Q, who, "K");
    code = attn_dtype(Q.scalar_type(), who);
    const int64_t B = Q.size(0), S = Q.size(2), D = Q.size(3);
    TORCH_CHECK(K.size(0) == B && K.size(2) == S, who, ": K must have Q's batch and tokens");
    for (auto* w : {&wq, &wk}) {
      need(*w, Q, "weight");
      TORCH_CHECK(w->dim() == 1 && w->numel() == D, who, ": weights must be (head_dim,)");
      TORCH_CHECK(w->scalar_type() == wq.scalar_type() &&
                      (w->scalar_type() == Q.scalar_type() || w->scalar_type() == at::kFloat),
                  who, ": weights must both have Q's dtype or both be float32");
    }
    wcode = attn_dtype(wq.scalar_type(), who);
    TORCH_CHECK(pos.device() == Q.device(), who, ": positions are on ", pos.device(), ", expected ", Q.device());
    icode = index_code(pos.scalar_type());
    TORCH_CHECK((pos.dim() == 1 && pos.size(0) == S) || (pos.dim() == 2 && pos.size(0) == B && pos.size(1) == S), who,
                ": positions must be (tokens,) or (batch, tokens)");
    pos_b = pos.dim() == 2 ? pos.stride(0) : 0;
    pos_s = pos.stride(pos.dim() - 1);
    need(freq, Q, "inv_freq");
    need_dtype(freq, at::kDouble, who, "inv_freq");
    TORCH_CHECK(freq.dim() == 1, who, ": inv_freq must be (rot / 2,)");
    rot = 2 * freq.numel();
  }
};

std::tuple<at::Tensor, at::Tensor> qk_norm_rope_fwd(const at::Tensor& Q_, const at::Tensor& K_, const at::Tensor& wq,
                                                    const at::Tensor& wk, const at::Tensor& pos, const at::Tensor& freq,
                                                    double eps, bool interleaved) {
  const c10::DeviceGuard guard(Q_.device());
  const RopeArgs r(Q_, K_, wq, wk, pos, freq, "qk_norm_rope_fwd");
  const auto Q = unit_rows(Q_), K = unit_rows(K_);
  auto Qo = at::empty(Q.sizes(), Q.options()), Ko = at::empty(K.sizes(), K.options());
  check(tsp_qk_norm_rope_fwd(Q.data_ptr(), Strides(Q).s, K.data_ptr(), Strides(K).s, r.code, Q.size(0), Q.size(1),
                             K.size(1), Q.size(2), Q.size(3), wq.data_ptr(), wk.data_ptr(), r.wcode, pos.data_ptr(),
                             r.icode, r.pos_b, r.pos_s, freq.data_ptr<double>(), r.rot, interleaved, eps, Qo.data_ptr(),
                             Strides(Qo).s, Ko.data_ptr(), Strides(Ko).s, stream_of(Q)),
        "tsp_qk_norm_rope_fwd");
  return {Qo, Ko};
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope_fwd_meta(const at::Tensor& Q, const at::Tensor& K, const at::Tensor&,
                                                         const at::Tensor&, const at::Tensor&, const at::Tensor&, double,
                                                         bool) {
  return {at::empty(Q.sizes(), Q.options()), at::empty(K.sizes(), K.options())};
}

// a weight gradient that is not asked for comes back empty
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> qk_norm_rope_bwd(
    const at::Tensor& Q_, const at::Tensor& K_, const at::Tensor& wq, const at::Tensor& wk, const at::Tensor& pos,
    const at::Tensor& freq, double eps, bool interleaved, const at::Tensor& gQ_, const at::Tensor& gK_,
    bool need_weights) {
  const char* who = "qk_norm_rope_bwd";
  const c10::DeviceGuard guard(Q_.device());
  const RopeArgs r(Q_, K_, wq, wk, pos, freq, who);
  need_4d(gQ_, Q_, who, "grad_Q");
  need_4d(gK_, Q_, who, "grad_K");
  TORCH_CHECK(gQ_.sizes() == Q_.sizes() && gK_.sizes() == K_.sizes(), who, ": gradients must have the results' shapes");
  const auto Q = unit_rows(Q_), K = unit_rows(K_), gQ = unit_rows(gQ_), gK = unit_rows(gK_);
  auto dQ = attn_like(Q_, Q.size(3)), dK = attn_like(K_, K.size(3));
  auto dwq = need_weights ? at::empty_like(wq) : at::empty({0}, wq.options());
  auto dwk = need_weights ? at::empty_like(wk) : at::empty({0}, wk.options());
  const int64_t wsb = tsp_qk_norm_rope_bwd_workspace_size(Q.size(0), Q.size(2), Q.size(3));
  const Workspace ws(need_weights ? wsb : 0, Q, who);
  check(tsp_qk_norm_rope_bwd(Q.data_ptr(), Strides(Q).s, K.data_ptr(), Strides(K).s, r.code, Q.size(0), Q.size(1),
                             K.size(1), Q.size(2), Q.size(3), wq.data_ptr(), wk.data_ptr(), r.wcode, pos.data_ptr(),
                             r.icode, r.pos_b, r.pos_s, freq.data_ptr<double>(), r.rot, interleaved, eps, gQ.data_ptr(),
                             Strides(gQ).s, gK.data_ptr(), Strides(gK).s, dQ.data_ptr(), Strides(dQ).s, dK.data_ptr(),
                             Strides(dK).s, need_weights ? dwq.data_ptr() : nullptr,
                             need_weights ? dwk.data_ptr() : nullptr, ws.ptr(), wsb, stream_of(Q)),
        "tsp_qk_norm_rope_bwd");
  return {dQ, dK, dwq, dwk};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> qk_norm_rope_bwd_meta(
    const at::Tensor& Q, const at::Tensor& K, const at::Tensor& wq, const at::Tensor& wk, const at::Tensor&,
    const at::Tensor&, double, bool, const at::Tensor&, const at::Tensor&, bool need_weights) {
  return {attn_like(Q, Q.size(3)), attn_like(K, K.size(3)), need_weights ? at::empty_like(wq) : at::empty({0}, wq.options()),
          need_weights ? at::empty_like(wk) : at::empty({0}, wk.options())};
}

// ----------------------------------------------- operators with gradients
//
// cross_attention and qk_norm_rope carry their gradients themselves, in C++: a
// small training step is bound by the host (forward and backward of 333 tokens
// took 140 us through a Python autograd function, 27 of them kernels).

namespace ag = torch::autograd;

// The registered operator `name`, of f's type: below autograd the calls go
// through the dispatcher, so that tracing reaches the Meta implementations.
template <typename F>
auto op_of(const char* name, F*) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

bool wants_grad(std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  return std::any_of(ts.begin(), ts.end(), [](const at::Tensor* t) { return t->defined() && t->requires_grad(); });
}

// Forward-mode derivatives are not formed. An input with a tangent need not
// require a gradient, and below autograd its tangent would be lost: refused.
void no_tangents(const char* who, std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), who, " has no forward-mode derivatives: an input has a "
                "tangent");
}

// A captured backward joins the stream on which its leaves' gradient
// accumulators were made. One that an eager graph (or a hook) of the same leaves
// keeps alive belongs to a stream outside the capture, and joining that ends the
// process: refused here, before anything of the step is recorded. Inputs that are
// leaves: any other stream. Inputs that the capture has made of leaves: the default
// stream, which no capture can take in (a side stream's accumulators, as a data
// parallel wrapper keeps them, wait for the captured work and so come into the
// capture); their graph is followed as far as it was made on the captured stream.
void capture_owns(const char* who, std::initializer_list<const at::Tensor*> ts) {
  if ((*ts.begin())->key_set().has(c10::DispatchKey::Python)) return;  // traced: no stream
  const at::Device dev = (*ts.begin())->device();
  const hipStream_t st = c10::hip::getCurrentHIPStream(dev.index()).stream();
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (!st || hipStreamIsCapturing(st, &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
  const c10::impl::VirtualGuardImpl impl(dev.type());
  const c10::Stream here = impl.getStream(dev), outside = impl.getDefaultStream(dev);
  auto refuse_if = [&](bool held) {
    TORCH_CHECK(!held, who, ": an input that needs its gradient, or what it comes from, is held by an autograd graph or "
                "hook made on another stream than the one being captured; release it before the capture, or call "
                "under torch.no_grad()");
  };
  std::vector<ag::Node*> todo;
  std::unordered_set<ag::Node*> seen;
  auto add = [&](ag::Node* n) {
    if (n && seen.insert(n).second) todo.push_back(n);
  };
  for (const at::Tensor* t : ts) {
    if (!t->requires_grad()) continue;
    if (!t->is_leaf()) {
      add(t->grad_fn().get());
      continue;
    }
    const auto acc = ag::impl::try_get_grad_accumulator(*t);
    const auto made = acc ? acc->stream() : c10::nullopt;
    refuse_if(made && *made != here);
  }
  while (!todo.empty()) {
    ag::Node* n = todo.back();
    todo.pop_back();
    const auto made = n->stream();
    refuse_if(made && *made == outside && dynamic_cast<ag::AccumulateGrad*>(n));
    if (!made || *made == here)
      for (const ag::Edge& e : n->next_edges()) add(e.function.get());
  }
}

void first_order(const char* who, const ag::variable_list& grads) {
  TORCH_CHECK(!at::GradMode::is_enabled(), who, " has no second derivatives: backward with create_graph=False");
  for (const at::Tensor& g : grads) no_tangents(who, {&g});
}

at::Tensor cross_attention(const at::Tensor& Q, const at::Tensor& K, const at::Tensor& V,
                           const c10::optional<at::Tensor>& key_lengths, double scale) {
  return cross_forward(Q, K, V, key_lengths, scale, nullptr);
}

at::Tensor cross_attention_meta(const at::Tensor& Q, const at::Tensor& K, const at::Tensor& V,
                                const c10::optional<at::Tensor>& key_lengths, double scale) {
  return std::get<0>(cross_attn_fwd_meta(Q, K, V, key_lengths, scale, false));
}

struct CrossAttention : public ag::Function<CrossAttention> {
  static at::Tensor forward(ag::AutogradContext* ctx, const at::Tensor& Q, const at::Tensor& K, const at::Tensor& V,
                            const c10::optional<at::Tensor>& key_lengths, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = op_of("trnsparse_hip::cross_attn_fwd", &cross_attn_fwd);
    auto [O, lse] = op.call(Q, K, V, key_lengths, scale, true);
    ctx->save_for_backward({Q, K, V, O, lse, key_lengths.has_value() ? *key_lengths : at::Tensor()});
    ctx->saved_data["scale"] = scale;
    return O;
  }
  static ag::variable_list backward(ag::AutogradContext* ctx, const ag::variable_list& grads) {
    first_order("cross_attention", grads);
    const auto s = ctx->get_saved_variables();
    const bool need_kv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    static const auto op = op_of("trnsparse_hip::cross_attn_bwd", &cross_attn_bwd);
    auto [dQ, dK, dV] = op.call(s[0], s[1], s[2], s[3], grads[0], s[4],
                                s[5].defined() ? c10::optional<at::Tensor>(s[5]) : c10::nullopt,
                                ctx->saved_data["scale"].toDouble(), need_kv);
    if (!need_kv) dK = dV = at::Tensor();
    return {dQ, dK, dV, at::Tensor(), at::Tensor()};
  }
};

at::Tensor cross_attention_autograd(const at::Tensor& Q, const at::Tensor& K, const at::Tensor& V,
                                    const c10::optional<at::Tensor>& key_lengths, double scale) {
  no_tangents("cross_attention", {&Q, &K, &V});
  if (wants_grad({&Q, &K, &V})) {
    capture_owns("cross_attention", {&Q, &K, &V});
    return CrossAttention::apply(Q, K, V, key_lengths, scale);
  }
  at::AutoDispatchBelowADInplaceOrView below;
  static const auto op = op_of("trnsparse_hip::cross_attention", &cross_attention);
  return op.call(Q, K, V, key_lengths, scale);
}

at::Tensor prefix_attn_autograd(const at::Tensor& Q, const at::Tensor& PK, const at::Tensor& PV, const at::Tensor& K,
                                const at::Tensor& V, const c10::optional<at::Tensor>& lengths, double scale) {
  no_tangents("shared_prefix_attention", {&Q, &PK, &PV, &K, &V});
  at::AutoDispatchBelowADInplaceOrView below;
  static const auto op = op_of("trnsparse_hip::prefix_attn_fwd", &prefix_attn_fwd);
  return op.call(Q, PK, PV, K, V, lengths, scale);
}

// The operators of the paged cache have no gradients: an input that needs one is
// refused, and what they write in place counts as written.
void no_gradients(const char* who, std::initializer_list<const at::Tensor*> ts) {
  no_tangents(who, ts);
  TORCH_CHECK(!wants_grad(ts), who, " has no gradients: call it under torch.no_grad()");
}
const at::Tensor& or_none(const c10::optional<at::Tensor>& t) {
  static const at::Tensor none;
  return t.has_value() ? *t : none;
}

at::Tensor paged_attn_autograd(const at::Tensor& Q, const at::Tensor& K, const at::Tensor& V, const at::Tensor& table,
                               const at::Tensor& lengths, const c10::optional<at::Tensor>& new_lengths, double scale,
                               const c10::optional<at::Tensor>& weights) {
  no_gradients("paged_attention", {&Q, &K, &V, &or_none(weights)});
  at::AutoDispatchBelowADInplaceOrView below;
  static const auto op = op_of("trnsparse_hip::paged_attn_fwd", &paged_attn_fwd);
  return op.call(Q, K, V, table, lengths, new_lengths, scale, weights);
}

at::Tensor paged_append_autograd(const at::Tensor& K, const at::Tensor& V, const at::Tensor& Kp, const at::Tensor& Vp,
                                 const at::Tensor& table, const at::Tensor& lengths,
                                 const c10::optional<at::Tensor>& new_lengths, const c10::optional<at::Tensor>& weights) {
  no_gradients("paged_cache_append", {&K, &V, &Kp, &Vp, &or_none(weights)});
  at::AutoDispatchBelowADInplaceOrView below;
  static const auto op = op_of("trnsparse_hip::paged_append", &paged_append);
  return op.call(K, V, Kp, Vp, table, lengths, new_lengths, weights);
}

at::Tensor paged_evict_autograd(const at::Tensor& Kp, const at::Tensor& Vp, const at::Tensor& weights,
                                const at::Tensor& table, const at::Tensor& lengths, int64_t budget, int64_t recent) {
  no_gradients("paged_cache_evict", {&Kp, &Vp, &weights});
  at::AutoDispatchBelowADInplaceOrView below;
  static const auto op = op_of("trnsparse_hip::paged_evict", &paged_evict);
  return op.call(Kp, Vp, weights, table, lengths, budget, recent);
}

struct QKNormRope : public ag::Function<QKNormRope> {
  static ag::variable_list forward(ag::AutogradContext* ctx, const at::Tensor& Q, const at::Tensor& K,
                                   const at::Tensor& wq, const at::Tensor& wk, const at::Tensor& pos,
                                   const at::Tensor& freq, double eps, bool interleaved) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = op_of("trnsparse_hip::qk_norm_rope_fwd", &qk_norm_rope_fwd);
    auto [q, k] = op.call(Q, K, wq, wk, pos, freq, eps, interleaved);
    ctx->save_for_backward({Q, K, wq, wk, pos, freq});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    return {q, k};
  }
  static ag::variable_list backward(ag::AutogradContext* ctx, const ag::variable_list& grads) {
    first_order("qk_norm_rope", grads);
    const auto s = ctx->get_saved_variables();
    const bool need_w = ctx->needs_input_grad(2) || ctx->needs_input_grad(3);
    auto grad = [&](int i) {  // a result that was not used
      return grads[i].defined() ? grads[i] : at::zeros(s[i].sizes(), s[i].options());
    };
    static const auto op = op_of("trnsparse_hip::qk_norm_rope_bwd", &qk_norm_rope_bwd);
    auto [dQ, dK, dwq, dwk] = op.call(s[0], s[1], s[2], s[3], s[4], s[5], ctx->saved_data["eps"].toDouble(),
                                      ctx->saved_data["interleaved"].toBool(), grad(0), grad(1), need_w);
    if (!need_w) dwq = dwk = at::Tensor();
    return {dQ, dK, dwq, dwk, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

std::tuple<at::Tensor, at::Tensor> qk_norm_rope_autograd(const at::Tensor& Q, const at::Tensor& K, const at::Tensor& wq,
                                                         const at::Tensor& wk, const at::Tensor& pos,
                                                         const at::Tensor& freq, double eps, bool interleaved) {
  no_tangents("qk_norm_rope", {&Q, &K, &wq, &wk, &freq});
  TORCH_CHECK(!wants_grad({&freq}), "qk_norm_rope has no gradient of inv_freq: pass inv_freq.detach()");
  if (wants_grad({&Q, &K, &wq, &wk})) {
    capture_owns("qk_norm_rope", {&Q, &K, &wq, &wk});
    auto r = QKNormRope::apply(Q, K, wq, wk, pos, freq, eps, interleaved);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  static const auto op = op_of("trnsparse_hip::qk_norm_rope", &qk_norm_rope_fwd);
  return op.call(Q, K, wq, wk, pos, freq, eps, interleaved);
}

}  // namespace

TORCH_LIBRARY(trnsparse_hip, m) {
  m.def("bsr_spmm(Tensor blocks, Tensor block_row_ptrs, Tensor block_col_indices, Tensor? row_order, int m, int n, "
        "int block_size, Tensor B, ScalarType out_dtype) -> Tensor");
  m.def("bsr_col_plan(Tensor block_row_ptrs, Tensor block_col_indices, int n_block_cols) -> (Tensor, Tensor, Tensor, "
        "Tensor, Tensor)");
  m.def("bsr_sddmm(Tensor grad_out, Tensor B, Tensor block_rows, Tensor block_col_indices, int m, int n, "
        "int block_size) -> Tensor");
  m.def("bsr_spmm_t(Tensor blocks, Tensor col_ptrs, Tensor col_block_ids, Tensor col_block_rows, Tensor col_order, "
        "int m, int n, int block_size, Tensor grad_out) -> Tensor");
  m.def("csr_spmv(Tensor values, Tensor col_indices, Tensor row_ptrs, Tensor windows, int m, int n, Tensor x, "
        "float alpha, Tensor? y, float beta) -> Tensor");
  m.def("csr_colplan_spmv(Tensor plan, int[] geometry, Tensor values, Tensor col_indices, Tensor row_ptrs, int m, "
        "int n, Tensor x, float alpha, Tensor? y, float beta) -> Tensor");
  m.def("csr_spmm(Tensor values, Tensor col_indices, Tensor row_ptrs, int m, int n, Tensor X, float alpha, "
        "Tensor? Y, float beta) -> Tensor");
  m.def("screened_spmm(Tensor A, Tensor diag_integrals, Tensor B, float threshold_sqrt) -> Tensor");
  m.def("screened_spmm_backward(Tensor A, Tensor diag_integrals, Tensor B, float threshold_sqrt, Tensor grad_out, "
        "bool need_a, bool need_b) -> (Tensor, Tensor)");
  m.def("bsa_fwd(Tensor Q, Tensor K, Tensor V, Tensor block_row_ptrs, Tensor block_col_indices, int block_size, "
        "float scale, bool return_stats) -> (Tensor, Tensor, Tensor)");
  m.def("bsa_bwd(Tensor Q, Tensor K, Tensor V, Tensor O, Tensor dO, Tensor block_row_ptrs, Tensor block_col_indices, "
        "Tensor col_ptrs, Tensor col_block_rows, int n_block_cols, int block_size, float scale, Tensor row_max, "
        "Tensor row_denom, Tensor plan, int n_items, int n_splits, int n_partials) -> (Tensor, Tensor, Tensor)");
  m.def("cross_attn_fwd(Tensor Q, Tensor K, Tensor V, Tensor? key_lengths, float scale, bool return_lse) -> "
        "(Tensor, Tensor)");
  m.def("cross_attn_bwd(Tensor Q, Tensor K, Tensor V, Tensor O, Tensor grad_out, Tensor lse, Tensor? key_lengths, "
        "float scale, bool need_kv) -> (Tensor, Tensor, Tensor)");
  m.def("prefix_attn_fwd(Tensor Q, Tensor prefix_K, Tensor prefix_V, Tensor K, Tensor V, Tensor? lengths, "
        "float scale) -> Tensor");
  m.def("paged_attn_fwd(Tensor Q, Tensor K_pages, Tensor V_pages, Tensor block_table, Tensor lengths, "
        "Tensor? new_lengths, float scale, Tensor(a!)? weights) -> Tensor");
  m.def("paged_append(Tensor K, Tensor V, Tensor(a!) K_pages, Tensor(b!) V_pages, Tensor block_table, Tensor lengths, "
        "Tensor? new_lengths, Tensor(c!)? weights) -> Tensor");
  m.def("paged_evict(Tensor(a!) K_pages, Tensor(b!) V_pages, Tensor(c!) weights, Tensor block_table, Tensor lengths, "
        "int budget, int recent) -> Tensor");
  m.def("qk_norm_rope_fwd(Tensor Q, Tensor K, Tensor q_weight, Tensor k_weight, Tensor positions, Tensor inv_freq, "
        "float eps, bool interleaved) -> (Tensor, Tensor)");
  m.def("qk_norm_rope_bwd(Tensor Q, Tensor K, Tensor q_weight, Tensor k_weight, Tensor positions, Tensor inv_freq, "
        "float eps, bool interleaved, Tensor grad_Q, Tensor grad_K, bool need_weights) -> (Tensor, Tensor, Tensor, "
        "Tensor)");
  m.def("cross_attention(Tensor Q, Tensor K, Tensor V, Tensor? key_lengths, float scale) -> Tensor");
  m.def("qk_norm_rope(Tensor Q, Tensor K, Tensor q_weight, Tensor k_weight, Tensor positions, Tensor inv_freq, "
        "float eps, bool interleaved) -> (Tensor, Tensor)");
}

// the "CUDA" dispatch key is the GPU key of PyTorch-ROCm
TORCH_LIBRARY_IMPL(trnsparse_hip, CUDA, m) {
  m.impl("bsr_spmm", &bsr_spmm);
  m.impl("bsr_col_plan", &bsr_col_plan);
  m.impl("bsr_sddmm", &bsr_sddmm);
  m.impl("bsr_spmm_t", &bsr_spmm_t);
  m.impl("csr_spmv", &csr_spmv);
  m.impl("csr_colplan_spmv", &csr_colplan_spmv);
  m.impl("csr_spmm", &csr_spmm);
  m.impl("screened_spmm", &screened_spmm);
  m.impl("screened_spmm_backward", &screened_spmm_backward);
  m.impl("bsa_fwd", &bsa_fwd);
  m.impl("bsa_bwd", &bsa_bwd);
  m.impl("cross_attn_fwd", &cross_attn_fwd);
  m.impl("cross_attn_bwd", &cross_attn_bwd);
  m.impl("prefix_attn_fwd", &prefix_attn_fwd);
  m.impl("paged_attn_fwd", &paged_attn_fwd);
  m.impl("paged_append", &paged_append);
  m.impl("paged_evict", &paged_evict);
  m.impl("qk_norm_rope_fwd", &qk_norm_rope_fwd);
  m.impl("qk_norm_rope_bwd", &qk_norm_rope_bwd);
  m.impl("cross_attention", &cross_attention);
  m.impl("qk_norm_rope", &qk_norm_rope_fwd);
}

TORCH_LIBRARY_IMPL(trnsparse_hip, AutogradCUDA, m) {
  m.impl("cross_attention", &cross_attention_autograd);
  m.impl("prefix_attn_fwd", &prefix_attn_autograd);
  m.impl("paged_attn_fwd", &paged_attn_autograd);
  m.impl("paged_append", &paged_append_autograd);
  m.impl("paged_evict", &paged_evict_autograd);
  m.impl("qk_norm_rope", &qk_norm_rope_autograd);
}

TORCH_LIBRARY_IMPL(trnsparse_hip, Meta, m) {
  m.impl("bsr_spmm", &bsr_spmm_meta);
  m.impl("bsr_col_plan", &bsr_col_plan_meta);
  m.impl("bsr_sddmm", &bsr_sddmm_meta);
  m.impl("bsr_spmm_t", &bsr_spmm_t_meta);
  m.impl("csr_spmv", &csr_spmv_meta);
  m.impl("csr_colplan_spmv", &csr_colplan_spmv_meta);
  m.impl("csr_spmm", &csr_spmm_meta);
  m.impl("screened_spmm", &screened_spmm_meta);
  m.impl("screened_spmm_backward", &screened_spmm_backward_meta);
  m.impl("bsa_fwd", &bsa_fwd_meta);
  m.impl("bsa_bwd", &bsa_bwd_meta);
  m.impl("cross_attn_fwd", &cross_attn_fwd_meta);
  m.impl("cross_attn_bwd", &cross_attn_bwd_meta);
  m.impl("prefix_attn_fwd", &prefix_attn_fwd_meta);
  m.impl("paged_attn_fwd", &paged_attn_fwd_meta);
  m.impl("paged_append", &paged_append_meta);
  m.impl("paged_evict", &paged_evict_meta);
  m.impl("qk_norm_rope_fwd", &qk_norm_rope_fwd_meta);
  m.impl("qk_norm_rope_bwd", &qk_norm_rope_bwd_meta);
  m.impl("cross_attention", &cross_attention_meta);
  m.impl("qk_norm_rope", &qk_norm_rope_fwd_meta);
}
