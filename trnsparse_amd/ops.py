"""Sparse operations: the public API of the compute path.

Signatures, defaults, error behaviour and results follow the reference
(trnsparse/ops.py). Each hot op checks `_use_hip()` exactly where the
reference checked `_use_nki()` (ops.py:67-73, 204-209, 255-260, 500-505,
535-540, 618-623) and then calls the HIP dispatch layer
(`trnsparse_amd.hip.dispatch`), which drives the gfx950 kernels through
the C ABI. With the "pytorch" backend selected the in-file torch code runs:
it restates the reference's torch path operation for operation (same loop
order and accumulation dtype), so both backends answer the same question.

`spmv` also crosses the seam here; in the reference it is always
`torch.sparse_csr_tensor @ x` (ops.py:30-48).
"""

from __future__ import annotations

import math

import torch

from .backend import _use_hip
from .formats import BSRMatrix, COOMatrix, CSRMatrix


def _as_torch_csr(A: CSRMatrix) -> torch.Tensor:
    """torch.sparse_csr_tensor view of a CSRMatrix (reference ops.py:25-27)."""
    return torch.sparse_csr_tensor(A.row_ptrs, A.col_indices, A.values, size=A.shape)


# --------------------------------------------------------------------- CSR


def spmv(
    A: CSRMatrix,
    x: torch.Tensor,
    alpha: float = 1.0,
    y: torch.Tensor | None = None,
    beta: float = 0.0,
) -> torch.Tensor:
    """y = alpha * A @ x + beta * y  (reference ops.py:30-48).

    alpha scales the product after the row sums; `y` is read only when it is
    given and beta != 0, and is never modified (a new tensor is returned).
    """
    m, n = A.shape
    assert x.shape[0] == n, f"Dimension mismatch: A is {A.shape}, x is {x.shape}"
    if _use_hip():
        from .hip.dispatch import hip_spmv

        return hip_spmv(A, x, alpha, y, beta)
    result = alpha * (_as_torch_csr(A) @ x)
    if y is not None and beta != 0.0:
        result = result + beta * y
    return result


def spmm(
    A: CSRMatrix,
    B: torch.Tensor,
    alpha: float = 1.0,
    C: torch.Tensor | None = None,
    beta: float = 0.0,
) -> torch.Tensor:
    """C = alpha * A @ B + beta * C  (reference ops.py:51-78)."""
    m, n = A.shape
    assert B.shape[0] == n, f"Dimension mismatch: A is {A.shape}, B is {B.shape}"
    if _use_hip():
        from .hip.dispatch import hip_spmm

        return hip_spmm(A, B, alpha, C, beta)
    result = alpha * (_as_torch_csr(A) @ B)
    if C is not None and beta != 0.0:
        result = result + beta * C
    return result


def spmv_symmetric(A: CSRMatrix, x: torch.Tensor, alpha: float = 1.0, uplo: str = "upper") -> torch.Tensor:
    """Symmetric SpMV from one stored triangle (reference ops.py:81-104):
    alpha * (A @ x + S^T @ x) with S the entries off the diagonal (duplicates
    summed); `uplo` is accepted and unused, as there. On the HIP backend with
    A on the GPU: S^T is built once on the device (transpose by a stable sort
    of (col, row), cached on A) and the two products run as CSR SpMVs, the
    second accumulating into the first."""
    m, n = A.shape
    assert m == n, "Matrix must be square for symmetric SpMV"
    if _use_hip() and A.values.is_cuda:
        from .hip.dispatch import hip_spmv

        St = _strict_transpose(A)
        y = hip_spmv(A, x, alpha)
        return hip_spmv(St, x, alpha, y, 1.0)
    counts = A.row_ptrs[1:] - A.row_ptrs[:-1]
    rows = torch.repeat_interleave(torch.arange(m, device=counts.device), counts)
    cols = A.col_indices
    strict = rows != cols
    strict_t = torch.sparse_coo_tensor(
        torch.stack([rows[strict], cols[strict]]), A.values[strict], size=A.shape
    ).coalesce()
    return alpha * (_as_torch_csr(A) @ x + strict_t.t() @ x)


def _strict_transpose(A: CSRMatrix) -> CSRMatrix:
    """CSR of the transpose of A's off-diagonal entries (duplicates summed),
    on A's device; cached on A keyed by the identity and version of its
    tensors."""
    key = tuple((t.data_ptr(), t._version) for t in (A.values, A.col_indices, A.row_ptrs))
    hit = getattr(A, "_strict_t", None)
    if hit is not None and hit[0] == key:
        return hit[1]
    from .hip import formats as hf

    coo = A.to_coo()
    keep = coo.row_indices != coo.col_indices
    vals, cols, rp = hf.coo_sum_to_csr(coo.values[keep], coo.col_indices[keep], coo.row_indices[keep],
                                       (A.shape[1], A.shape[0]))
    St = CSRMatrix(values=vals, col_indices=cols, row_ptrs=rp, shape=(A.shape[1], A.shape[0]))
    try:
        # the source tensors ride along, so a new tensor cannot take a freed
        # one's address (and key) while this entry lives
        A._strict_t = (key, St, (A.values, A.col_indices, A.row_ptrs))
    except AttributeError:
        pass
    return St


def sparse_add(A: CSRMatrix, B: CSRMatrix, alpha: float = 1.0, beta: float = 1.0) -> CSRMatrix:
    """C = alpha*A + beta*B on the union pattern (reference ops.py:107-132).

    Entries sorted by (row, col), one per distinct coordinate with its
    duplicates summed (explicit zeros kept). On the HIP backend with A and
    B on the GPU the coalesce runs on the device (`tsp_csr_sum`: each row's
    entries of A then B, stably sorted by column, runs summed); the values
    are scaled by torch first, as in the reference."""
    assert A.shape == B.shape, f"Shape mismatch: {A.shape} vs {B.shape}"
    if _use_hip() and A.values.is_cuda and B.values.is_cuda and A.values.dtype == B.values.dtype:
        from .hip import formats as hf

        if A.values.dtype in hf.DEVICE_DTYPES:
            # (x * 1.0 is x bit for bit, so a unit factor is not applied)
            av = A.values if alpha == 1.0 else alpha * A.values
            bv = B.values if beta == 1.0 else beta * B.values
            vals, cols, rp = hf.csr_sum(av, A.col_indices, A.row_ptrs, bv, B.col_indices, B.row_ptrs, A.shape)
            return CSRMatrix(values=vals, col_indices=cols, row_ptrs=rp, shape=A.shape)
    ca, cb = A.to_coo(), B.to_coo()
    idx = torch.stack(
        [torch.cat([ca.row_indices, cb.row_indices]), torch.cat([ca.col_indices, cb.col_indices])]
    )
    vals = torch.cat([alpha * ca.values, beta * cb.values])
    csr = torch.sparse_coo_tensor(idx, vals, size=A.shape).coalesce().to_sparse_csr()
    return CSRMatrix(values=csr.values(), col_indices=csr.col_indices(), row_ptrs=csr.crow_indices(), shape=A.shape)


def sparse_scale(A: CSRMatrix, alpha: float) -> CSRMatrix:
    """B = alpha * A (reference ops.py:135-142)."""
    return CSRMatrix(
        values=alpha * A.values,
        col_indices=A.col_indices.clone(),
        row_ptrs=A.row_ptrs.clone(),
        shape=A.shape,
    )


def sparse_transpose(A: CSRMatrix) -> CSRMatrix:
    """CSR of A^T (reference ops.py:145-154). On the HIP backend with A on
    the GPU: a stable device sort of the entries by column with the rows
    carried along (`tsp_csr_transpose`), the same order as the reference's
    sort by (col, row)."""
    if _use_hip() and A.values.is_cuda:
        from .hip import formats as hf

        if A.values.dtype in hf.DEVICE_DTYPES:
            vals, cols, rp = hf.csr_transpose(A.values, A.col_indices, A.row_ptrs, A.shape)
            return CSRMatrix(values=vals, col_indices=cols, row_ptrs=rp, shape=(A.shape[1], A.shape[0]))
    coo = A.to_coo()
    return COOMatrix(
        values=coo.values, row_indices=coo.col_indices, col_indices=coo.row_indices, shape=(A.shape[1], A.shape[0])
    ).to_csr()


def nnz_per_row(A: CSRMatrix) -> torch.Tensor:
    """Stored entries per row (reference ops.py:157-159)."""
    return A.row_ptrs[1:] - A.row_ptrs[:-1]


# --------------------------------------------------------------------- BSR


def _bsr_spmm_pytorch(A: BSRMatrix, B: torch.Tensor, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Torch semantics of bsr_spmm (reference ops.py:162-192).

    For each block row i and stored block idx (indptr order), with column
    block j: out[i*b:(i+1)*b] += blocks[idx] @ B[j*b:(j+1)*b]. `out` has
    A's dtype unless `out_dtype` asks otherwise, in which case the block
    products are formed in `out_dtype` from upcast operands.
    """
    m, n = A.shape
    _, k = B.shape
    b = A.block_size
    m_pad = ((m + b - 1) // b) * b
    n_pad = ((n + b - 1) // b) * b
    mb = m_pad // b
    if B.shape[0] != n:
        raise AssertionError(f"Dimension mismatch: A is {A.shape}, B is {B.shape}")
    if n_pad != n:
        B_p = torch.zeros(n_pad, k, dtype=B.dtype, device=B.device)
        B_p[:n, :] = B
        B = B_p
    odt = out_dtype or A.dtype
    blocks = A.blocks if odt == A.dtype else A.blocks.to(odt)
    if odt != B.dtype and out_dtype is not None:
        B = B.to(odt)
    out = torch.zeros(m_pad, k, dtype=odt, device=B.device)
    ptrs = A.block_row_ptrs.tolist()
    cols = A.block_col_indices.tolist()
    for i in range(mb):
        for idx in range(ptrs[i], ptrs[i + 1]):
            j = cols[idx]
            out[i * b : (i + 1) * b] += blocks[idx] @ B[j * b : (j + 1) * b]
    return out[:m]


def bsr_spmm(A: BSRMatrix, B: torch.Tensor, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Block-sparse x dense: C = A @ B  (reference ops.py:195-210).

    `out_dtype` (an addition; default A.dtype as in the reference) lets bf16
    operands produce an fp32 result, accumulated in fp32.
    """
    if B.shape[0] != A.shape[1]:
        raise AssertionError(f"Dimension mismatch: A is {A.shape}, B is {B.shape}")
    if _use_hip():
        from .hip.dispatch import hip_bsr_spmm

        return hip_bsr_spmm(A, B, out_dtype=out_dtype)
    return _bsr_spmm_pytorch(A, B, out_dtype=out_dtype)


# ---------------------------------------------------------------- screened


def screened_mask(diag_integrals: torch.Tensor, threshold: float) -> torch.Tensor:
    """mask[i, j] = Q_i*Q_j > sqrt(threshold), Q = sqrt(|diag|) (reference ops.py:273-276).

    The product and the compare run in diag's dtype: torch casts the Python
    float sqrt(threshold) to that dtype before comparing.
    """
    Q = torch.sqrt(torch.abs(diag_integrals))
    return (Q.unsqueeze(-1) * Q.unsqueeze(0)) > math.sqrt(threshold)


def screened_spmm(
    A: torch.Tensor,
    diag_integrals: torch.Tensor,
    B: torch.Tensor,
    threshold: float,
) -> torch.Tensor:
    """Schwarz-screened dense matmul C = (A * mask) @ B  (reference ops.py:213-277).

    mask[i, j] = sqrt(|d_i|) * sqrt(|d_j|) > sqrt(threshold). On the HIP
    backend the mask is applied while A tiles are staged (no mask tensor)
    and 128x128 tiles whose bound cannot pass are skipped.
    """
    assert diag_integrals.dim() == 1, f"diag_integrals must be 1-D; got shape {diag_integrals.shape}"
    M, K = A.shape
    assert diag_integrals.shape[0] == M == K, (
        "screened_spmm requires square A with diag_integrals of matching length; "
        f"got A shape {A.shape}, diag_integrals shape {diag_integrals.shape}"
    )
    if _use_hip():
        from .hip.dispatch import hip_screened_spmm

        return hip_screened_spmm(A, diag_integrals, B, threshold)
    mask = screened_mask(diag_integrals, threshold)
    return (A * mask.to(A.dtype)) @ B


# --------------------------------------------------------------- attention


def _block_sparse_attn_pytorch(Q, K, V, mask_bsr, scale: float, return_stats: bool = False):
    """Two-pass block-sparse attention, torch semantics (reference ops.py:280-357).

    Pass 1 stores per stored block the row max and stable exp-sum of
    score = (Q_m @ K_j^T) * scale; they are reduced to row_max / row_denom
    (row_denom clamped at 1e-12; empty block rows get row_max 0 and zero
    output); pass 2 accumulates exp(score - row_max) / row_denom @ V_j.
    Stats and output are in Q's dtype, as in the reference.
    """
    seq_len, head_dim = Q.shape
    b = mask_bsr.block_size
    M_tiles = seq_len // b
    ptrs = mask_bsr.block_row_ptrs.tolist()
    cols = mask_bsr.block_col_indices.tolist()
    n_blocks = len(cols)
    dev = Q.device

    tile_max = torch.full((n_blocks, b), float("-inf"), dtype=Q.dtype, device=dev)
    tile_sumexp = torch.zeros((n_blocks, b), dtype=Q.dtype, device=dev)
    for m in range(M_tiles):
        q_block = Q[m * b : (m + 1) * b]
        for idx in range(ptrs[m], ptrs[m + 1]):
            c = cols[idx]
            score = (q_block @ K[c * b : (c + 1) * b].T) * scale
            tile_max[idx] = score.max(dim=1).values
            tile_sumexp[idx] = torch.exp(score - tile_max[idx].unsqueeze(1)).sum(dim=1)

    row_max = torch.full((seq_len,), float("-inf"), dtype=Q.dtype, device=dev)
    row_denom = torch.zeros(seq_len, dtype=Q.dtype, device=dev)
    for m in range(M_tiles):
        s, e = ptrs[m], ptrs[m + 1]
        if s == e:
            row_max[m * b : (m + 1) * b] = 0.0
            continue
        row_max[m * b : (m + 1) * b] = tile_max[s:e].max(dim=0).values
        rm = row_max[m * b : (m + 1) * b]
        for idx in range(s, e):
            row_denom[m * b : (m + 1) * b] += tile_sumexp[idx] * torch.exp(tile_max[idx] - rm)
    row_denom = row_denom.clamp(min=1e-12)

    out = torch.zeros(seq_len, head_dim, dtype=Q.dtype, device=dev)
    for m in range(M_tiles):
        s, e = ptrs[m], ptrs[m + 1]
        if s == e:
            continue
        q_block = Q[m * b : (m + 1) * b]
        rm = row_max[m * b : (m + 1) * b].unsqueeze(1)
        rd = row_denom[m * b : (m + 1) * b].unsqueeze(1)
        for idx in range(s, e):
            c = cols[idx]
            score = (q_block @ K[c * b : (c + 1) * b].T) * scale
            out[m * b : (m + 1) * b] += (torch.exp(score - rm) / rd) @ V[c * b : (c + 1) * b]

    if return_stats:
        return out, row_max[: M_tiles * b].view(M_tiles, b), row_denom[: M_tiles * b].view(M_tiles, b)
    return out


def _block_sparse_attn_backward(Q, K, V, O, dO, mask_bsr, scale, row_max=None, row_denom=None):
    """Tiled softmax-attention backward (reference ops.py:360-473).

    D = rowsum(dO * O); per stored block P = exp(score - row_max)/row_denom,
    dS = P * (dO @ V_j^T - D); dQ += dS @ K_j * scale, dK_j += dS^T @ Q *
    scale, dV_j += P^T @ dO. Stats are recomputed when not supplied.
    """
    seq_len, head_dim = Q.shape
    b = mask_bsr.block_size
    M_tiles = seq_len // b
    ptrs = mask_bsr.block_row_ptrs.tolist()
    cols = mask_bsr.block_col_indices.tolist()
    dev = Q.device
    D = (dO * O).sum(dim=-1)

    if row_max is not None and row_denom is not None:
        rmax = row_max.reshape(-1)
        rden = row_denom.reshape(-1)
    else:
        rmax = torch.full((seq_len,), float("-inf"), dtype=Q.dtype, device=dev)
        rden = torch.zeros(seq_len, dtype=Q.dtype, device=dev)
        for m in range(M_tiles):
            s, e = ptrs[m], ptrs[m + 1]
            if s == e:
                rmax[m * b : (m + 1) * b] = 0.0
                continue
            q_block = Q[m * b : (m + 1) * b]
            rm = rmax[m * b : (m + 1) * b]
            for idx in range(s, e):
                c = cols[idx]
                score = (q_block @ K[c * b : (c + 1) * b].T) * scale
                rm = torch.maximum(rm, score.max(dim=1).values)
            rmax[m * b : (m + 1) * b] = rm
        for m in range(M_tiles):
            s, e = ptrs[m], ptrs[m + 1]
            if s == e:
                continue
            q_block = Q[m * b : (m + 1) * b]
            rm = rmax[m * b : (m + 1) * b]
            for idx in range(s, e):
                c = cols[idx]
                score = (q_block @ K[c * b : (c + 1) * b].T) * scale
                rden[m * b : (m + 1) * b] += torch.exp(score - rm.unsqueeze(1)).sum(dim=1)
        rden = rden.clamp(min=1e-12)

    dQ = torch.zeros_like(Q)
    dK = torch.zeros_like(K)
    dV = torch.zeros_like(V)
    for m in range(M_tiles):
        s, e = ptrs[m], ptrs[m + 1]
        if s == e:
            continue
        q_block = Q[m * b : (m + 1) * b]
        do_block = dO[m * b : (m + 1) * b]
        d_block = D[m * b : (m + 1) * b]
        rm = rmax[m * b : (m + 1) * b].unsqueeze(1)
        rd = rden[m * b : (m + 1) * b].unsqueeze(1)
        for idx in range(s, e):
            c = cols[idx]
            k_block = K[c * b : (c + 1) * b]
            v_block = V[c * b : (c + 1) * b]
            score = (q_block @ k_block.T) * scale
            P = torch.exp(score - rm) / rd
            dS = P * (do_block @ v_block.T - d_block.unsqueeze(1))
            dQ[m * b : (m + 1) * b] += dS @ k_block * scale
            dK[c * b : (c + 1) * b] += dS.T @ q_block * scale
            dV[c * b : (c + 1) * b] += P.T @ do_block
    return dQ, dK, dV


class _AttnTiledFunction(torch.autograd.Function):
    """Autograd wrapper of tiled attention (reference ops.py:476-546).

    Forward runs the HIP kernel (or the torch two-pass spec) and saves
    Q, K, V, O and the row stats; backward runs the HIP backward kernels (or
    the tiled torch backward on the "pytorch" backend).
    Q/K/V are (seq, d) or batched (..., seq, d) sharing one mask. The mask
    itself is passed (not its tensors, as the reference's pattern stand-in
    at ops.py:488-498 does): the device copies of its pattern and the row
    order are cached on it, so repeated calls copy nothing to the device and
    a HIP graph can capture a forward + backward step.
    """

    @staticmethod
    def forward(ctx, Q, K, V, mask_bsr, scale):
        handle = mask_bsr
        if _use_hip():
            from .hip.dispatch import hip_block_sparse_attention

            out, row_max, row_denom = hip_block_sparse_attention(Q, K, V, handle, scale, return_stats=True)
        else:
            out, row_max, row_denom = _attn_pytorch_batched(Q, K, V, handle, scale, return_stats=True)
        ctx.save_for_backward(Q, K, V, out, row_max, row_denom)
        ctx.handle = handle
        ctx.scale = scale
        return out

    @staticmethod
    def backward(ctx, dO):
        Q, K, V, O, row_max, row_denom = ctx.saved_tensors
        if _use_hip():
            from .hip.dispatch import hip_block_sparse_attention_backward

            dQ, dK, dV = hip_block_sparse_attention_backward(
                Q, K, V, O, dO.contiguous(), ctx.handle, ctx.scale, row_max, row_denom
            )
            return dQ, dK, dV, None, None
        lead = Q.shape[:-2]
        S, D = Q.shape[-2:]
        q, k, v, o, do = (t.reshape(math.prod(lead), S, D) for t in (Q, K, V, O, dO))
        rm = row_max.reshape(q.shape[0], -1).to(Q.dtype)
        rd = row_denom.reshape(q.shape[0], -1).to(Q.dtype)
        grads = [
            _block_sparse_attn_backward(q[h], k[h], v[h], o[h], do[h], ctx.handle, ctx.scale, rm[h], rd[h])
            for h in range(q.shape[0])
        ]
        dQ, dK, dV = (torch.stack([g[i] for g in grads]).reshape(*lead, S, D) for i in range(3))
        return dQ, dK, dV, None, None


def _attn_pytorch_batched(Q, K, V, mask_bsr, scale, return_stats=False):
    if Q.dim() == 2:
        return _block_sparse_attn_pytorch(Q, K, V, mask_bsr, scale, return_stats=return_stats)
    lead = Q.shape[:-2]
    S, D = Q.shape[-2:]
    q, k, v = (t.reshape(math.prod(lead), S, D) for t in (Q, K, V))
    res = [_block_sparse_attn_pytorch(q[h], k[h], v[h], mask_bsr, scale, return_stats=return_stats) for h in range(q.shape[0])]
    if not return_stats:
        return torch.stack(res).reshape(*lead, S, D)
    out = torch.stack([r[0] for r in res]).reshape(*lead, S, D)
    rmax = torch.stack([r[1] for r in res]).reshape(*lead, *res[0][1].shape)
    rden = torch.stack([r[2] for r in res]).reshape(*lead, *res[0][2].shape)
    return out, rmax, rden


def block_sparse_attention_tiled(
    Q: torch.Tensor,
    K: torch.Tensor,
    V: torch.Tensor,
    mask_bsr: BSRMatrix,
    scale: float | None = None,
) -> torch.Tensor:
    """Block-sparse softmax attention over the stored blocks of `mask_bsr`
    (reference ops.py:549-625).

    Q, K, V: (seq_len, head_dim), or (..., seq_len, head_dim) with leading
    batch/head dims sharing one mask (an addition; each head is the 2-D
    op). Only the mask's pattern is used. `scale` defaults to
    head_dim**-0.5. Rows of an empty block row produce zeros. When any input
    requires grad the call goes through `_AttnTiledFunction`.
    """
    head_dim = Q.shape[-1]
    if scale is None:
        scale = head_dim**-0.5
    if torch.is_grad_enabled() and (Q.requires_grad or K.requires_grad or V.requires_grad):
        return _AttnTiledFunction.apply(Q, K, V, mask_bsr, scale)
    if _use_hip():
        from .hip.dispatch import hip_block_sparse_attention

        return hip_block_sparse_attention(Q, K, V, mask_bsr, scale)
    return _attn_pytorch_batched(Q, K, V, mask_bsr, scale)


# ------------------------------------------- attention between sequences
#
# Operators that a decoder layer has next to block_sparse_attention_tiled: no
# counterpart in the reference.


def _default_scale(Q: torch.Tensor) -> float:
    d = Q.shape[-1] if Q.dim() else 0
    return d**-0.5 if d else 1.0  # (an empty head_dim is refused)


def _check_heads(who: str, Q, K, V, lengths, scale: float) -> None:
    """Shapes and types of (batch, heads, rows, head_dim) operands. The HIP
    operators refuse the same calls themselves (csrc/torch_ops.cpp)."""
    q, k, v, dt = Q.shape, K.shape, V.shape, Q.dtype
    if not (len(q) == len(k) == len(v) == 4):
        raise RuntimeError(f"{who}: Q, K, V must be (batch, heads, rows, head_dim), got {tuple(q)}, {tuple(k)}, {tuple(v)}")
    if k != v or k[0] != q[0] or k[3] != q[3]:
        raise RuntimeError(f"{who}: Q {tuple(q)}, K {tuple(k)} and V {tuple(v)} do not belong together")
    if k[1] == 0 or q[1] % k[1]:
        raise RuntimeError(f"{who}: {q[1]} query heads do not divide over {k[1]} key heads")
    if K.dtype != dt or V.dtype != dt or not dt.is_floating_point:
        raise RuntimeError(f"{who}: Q, K, V must have one floating dtype, got {dt}, {K.dtype}, {V.dtype}")
    if not 1 <= q[3] <= 128:
        raise RuntimeError(f"{who}: head_dim {q[3]} is not in 1 .. 128")
    if not 1e-30 < scale < 1e30:
        raise RuntimeError(f"{who}: scale must be positive, got {scale}")
    if lengths is not None:
        if lengths.dtype not in (torch.int32, torch.int64) or lengths.shape != q[:1]:
            raise RuntimeError(f"{who}: lengths must be ({q[0]},) of int32 or int64, got {tuple(lengths.shape)} of "
                               f"{lengths.dtype}")


def _masked_softmax(S: torch.Tensor) -> torch.Tensor:
    """Softmax over the last dimension; a row of -inf alone gives zeros."""
    m = S.amax(-1, keepdim=True).detach()
    P = torch.exp(S - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    total = P.sum(-1, keepdim=True)
    return P / torch.where(total == 0, torch.ones_like(total), total)


def _wide(t: torch.Tensor) -> torch.Tensor:
    return t.float() if t.dtype in (torch.bfloat16, torch.float16) else t


def _attn_parts_pytorch(Q, parts, scale):
    """Grouped-head attention over several sets of keys in one softmax. Each
    part is (K, V, seen): K, V (batch, kv_heads, keys, head_dim) and seen a
    mask broadcast to (batch, 1, queries, keys) or None. What no query sees is
    zeroed first: masked rows may hold anything."""
    B, H, N, D = Q.shape
    Hk = parts[0][0].shape[1]
    G = H // Hk
    q = _wide(Q).reshape(B, Hk, G * N, D)
    scores, values = [], []
    for K, V, seen in parts:
        k, v = _wide(K), _wide(V)
        if seen is not None:
            some = seen.any(2).unsqueeze(-1)  # (batch, 1, keys, 1)
            k, v = torch.where(some, k, torch.zeros_like(k)), torch.where(some, v, torch.zeros_like(v))
        s = (q @ k.transpose(2, 3)) * scale
        if seen is not None:
            s = s.view(B, H, N, -1).masked_fill(~seen, float("-inf")).view(B, Hk, G * N, -1)
        scores.append(s)
        values.append(v)
    if sum(s.shape[-1] for s in scores) == 0:
        return Q.masked_fill(torch.ones_like(Q, dtype=torch.bool), 0.0)  # (whatever Q holds)
    P = _masked_softmax(torch.cat(scores, -1))
    O = P.new_zeros(B, Hk, G * N, D)
    at = 0
    for s, v in zip(scores, values):
        O = O + P[..., at : at + s.shape[-1]] @ v
        at += s.shape[-1]
    return O.reshape(B, H, N, D).to(Q.dtype)


def cross_attention(
    Q: torch.Tensor,
    K: torch.Tensor,
    V: torch.Tensor,
    key_lengths: torch.Tensor | None = None,
    scale: float | None = None,
) -> torch.Tensor:
    """Softmax attention of one sequence's queries over another's keys.

    Q (batch, heads, queries, head_dim); K, V (batch, kv_heads, keys,
    head_dim) of any other length, heads a multiple of kv_heads: query head h
    reads key head h // (heads // kv_heads). `key_lengths` (batch,) int32 or
    int64 gives each sample's number of valid keys (values are taken into
    [0, keys]); what stands in K and V behind them is not read, and its
    gradient is zero. A sample without keys gives zeros. `scale` defaults to
    head_dim**-0.5 and lies in (1e-30, 1e30); head_dim is at most 128.

    float32, bfloat16 and float16 on the HIP backend, accumulated in float32.
    Operands may be strided views (heads of a projection's output); the result
    has Q's order of heads and rows (contiguous where head_dim is not whole
    16-byte pieces). Differentiable in Q, K and V.
    """
    if scale is None:
        scale = _default_scale(Q)
    if _use_hip():
        from .hip.dispatch import hip_cross_attention

        return hip_cross_attention(Q, K, V, key_lengths, scale)
    _check_heads("cross_attention", Q, K, V, key_lengths, scale)
    seen = None
    if key_lengths is not None:
        at = torch.arange(K.shape[2], device=Q.device)
        seen = (at < key_lengths.to(Q.device).view(-1, 1, 1, 1)).expand(-1, 1, Q.shape[2], -1)
        if Q.shape[2] == 0:
            return Q * 1
    return _attn_parts_pytorch(Q, [(K, V, seen)], scale)


def shared_prefix_attention(
    Q: torch.Tensor,
    prefix_K: torch.Tensor,
    prefix_V: torch.Tensor,
    K: torch.Tensor,
    V: torch.Tensor,
    lengths: torch.Tensor | None = None,
    scale: float | None = None,
) -> torch.Tensor:
    """Attention of new tokens over a prefix that the whole batch shares and
    each sequence's own tokens behind it (serving: no gradients).

    Q (batch, heads, queries, head_dim), the new tokens: one, or a few in
    order. prefix_K, prefix_V (kv_heads, prefix, head_dim), read once for the
    batch. K, V (batch, kv_heads, keys, head_dim), each sequence's cache, whose
    first lengths[b] rows hold its own tokens, the new ones last (None: all
    rows; values are taken into [0, keys]); rows behind them are not read.
    Query i sees the prefix and own tokens j < lengths[b] - (queries - 1 - i);
    a query that sees nothing gives zeros. What stands in V of a token that only
    some queries see has to be finite: the others weigh it with zero. Types,
    heads, scale, strides and the result's order as in `cross_attention`.
    """
    who = "shared_prefix_attention"
    if scale is None:
        scale = _default_scale(Q)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (Q, prefix_K, prefix_V, K, V)):
        raise RuntimeError(f"{who} has no gradients: call it under torch.no_grad()")
    if _use_hip():
        from .hip.dispatch import hip_shared_prefix_attention

        return hip_shared_prefix_attention(Q, prefix_K, prefix_V, K, V, lengths, scale)
    _check_heads(who, Q, K, V, lengths, scale)
    want = (K.shape[1], K.shape[3])
    if prefix_K.dim() != 3 or prefix_K.shape != prefix_V.shape or (prefix_K.shape[0], prefix_K.shape[2]) != want:
        raise RuntimeError(f"{who}: prefix_K {tuple(prefix_K.shape)} and prefix_V {tuple(prefix_V.shape)} must be "
                           f"({want[0]}, prefix, {want[1]})")
    if not (prefix_K.dtype == prefix_V.dtype == Q.dtype):
        raise RuntimeError(f"{who}: the prefix must have Q's dtype {Q.dtype}")
    B, _, N, _ = Q.shape
    if Q.numel() == 0:
        return Q * 1
    n = K.shape[2] if lengths is None else lengths.to(Q.device).clamp(0, K.shape[2]).view(-1, 1)
    last = n - N + 1 + torch.arange(N, device=Q.device)  # own keys each query sees
    seen = torch.arange(K.shape[2], device=Q.device) < last.expand(B, N).view(B, 1, N, 1)
    shared = (prefix_K.expand(B, -1, -1, -1), prefix_V.expand(B, -1, -1, -1), None)
    return _attn_parts_pytorch(Q, [shared, (K, V, seen)], scale)


# A key and value cache in pages: what the three operators share.


_dispatch = None


def _hip():
    """hip.dispatch, imported by the first call that needs it (an import statement
    costs every call about 0.5 us)."""
    global _dispatch
    if _dispatch is None:
        from .hip import dispatch

        _dispatch = dispatch
    return _dispatch


def _no_gradients(who: str, *tensors) -> None:
    """The HIP operators refuse the same (csrc/torch_ops.cpp)."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{who} has no gradients: call it under torch.no_grad()")


def _apart(t) -> bool:
    """Whether no two elements of a view share memory: every dimension's stride passes the
    extent of those of smaller strides."""
    extent = 1
    for stride, size in sorted((t.stride(i), t.shape[i]) for i in range(t.dim()) if t.shape[i] > 1):
        if stride < extent:
            return False
        extent += stride * (size - 1)
    return True


def _check_cache(who: str, K_pages, V_pages, block_table, lengths, new_lengths, weights, written=()) -> None:
    """Shapes and types of a paged cache, and that the rows of what is `written` lie
    apart. The HIP operators refuse the same calls themselves (csrc/torch_ops.cpp,
    csrc/paged_cache.hip)."""
    k, dt = K_pages.shape, K_pages.dtype
    if len(k) != 4 or V_pages.shape != k or V_pages.dtype != dt or not dt.is_floating_point:
        raise RuntimeError(f"{who}: K_pages {tuple(k)} of {dt} and V_pages {tuple(V_pages.shape)} of {V_pages.dtype} must "
                           "be (pages, kv_heads, page_size, head_dim) of one floating dtype")
    if k[1] == 0 or k[2] == 0 or k[2] % 16:
        raise RuntimeError(f"{who}: page_size {k[2]} must be a multiple of 16, kv_heads {k[1]} at least 1")
    if not 1 <= k[3] <= 128 or k[3] * K_pages.element_size() % 16:
        raise RuntimeError(f"{who}: head_dim {k[3]} must be at most 128 and whole 16-byte pieces")
    whole = (torch.int32, torch.int64)
    if block_table.dim() != 2 or block_table.dtype not in whole:
        raise RuntimeError(f"{who}: block_table must be (batch, columns) of int32 or int64")
    B, cols = block_table.shape
    for name, t in (("lengths", lengths), ("new_lengths", new_lengths)):
        if t is not None and (t.shape != (B,) or t.dtype not in whole):
            raise RuntimeError(f"{who}: {name} must be ({B},) of int32 or int64, got {tuple(t.shape)} of {t.dtype}")
    if weights is not None and (weights.shape != (B, k[1], cols * k[2]) or weights.dtype != torch.float32):
        raise RuntimeError(f"{who}: weights must be ({B}, {k[1]}, {cols * k[2]}) of float32, got {tuple(weights.shape)} of "
                           f"{weights.dtype}")
    if any(t is not None and t.numel() and not _apart(t) for t in written):
        raise RuntimeError(f"{who}: rows of pages or weights, which are written, overlap")


def _page_rows(K_pages, block_table, slots):
    """Of the given slots (batch, kv_heads, n) or (n,): pages and rows to index
    (pages, kv_heads, page_size, head_dim) with, and whether a page is there."""
    pages, Hk, size, _ = K_pages.shape
    B = block_table.shape[0]
    slots = slots.expand(B, Hk, slots.shape[-1])
    table = block_table.to(K_pages.device).long()
    page = table.gather(1, (slots // size).reshape(B, -1)).view(slots.shape)
    there = (page >= 0) & (page < pages)
    heads = torch.arange(Hk, device=K_pages.device).view(1, Hk, 1).expand(slots.shape)
    return (torch.where(there, page, torch.zeros_like(page)), heads, slots % size), there


def _read_rows(pages, at, there):
    if pages.shape[0] == 0:
        return pages.new_zeros(*there.shape, pages.shape[3])
    return torch.where(there.unsqueeze(-1), pages[at], torch.zeros((), dtype=pages.dtype, device=pages.device))


def paged_attention(
    Q: torch.Tensor,
    K_pages: torch.Tensor,
    V_pages: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    new_lengths: torch.Tensor | None = None,
    scale: float | None = None,
    weights: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of a chunk of new tokens of every sequence over its cache in
    pages, the new tokens' own rows included (serving: no gradients).

    K_pages, V_pages (pages, kv_heads, page_size, head_dim); page_size is a
    multiple of 16, head_dim at most 128 and whole 16-byte pieces. block_table
    (batch, columns) int32 or int64: row j of sequence b is row j % page_size of
    page block_table[b, j // page_size]; an entry outside [0, pages) is a page
    of zeros. lengths (batch,) int32 or int64: the rows that each sequence has
    (taken into [0, slots], slots = columns * page_size). Its last
    new_lengths[b] rows are the new tokens' (None: as many as Q has; taken into
    [0, queries]), whose queries are Q[b, :, :new_lengths[b]] of Q (batch,
    heads, queries, head_dim). Query i sees the rows j < lengths[b] -
    (new_lengths[b] - 1 - i), heads are grouped as in `cross_attention`. Results
    of queries behind new_lengths[b], or that see no row, are zero. What stands
    in V of a row that only some of the new tokens see has to be finite: the
    others weigh it with zero.

    With `weights` (batch, kv_heads, slots) float32, the softmax weight of every
    row, summed over the key head's query heads and the new tokens, is added to
    it: what `paged_cache_evict` goes by.

    The HIP kernels sum and normalise in float32; in 16 bits the softmax weights enter
    the product with V as sums of two 16-bit numbers where a sequence has at most 32 rows
    to a key head (new tokens times query heads over it), as one where it has more.

    Types, scale, strides of Q and the result's order as in `cross_attention`;
    pages and weights may be views with unit stride over the last dimension and
    (pages) other strides of whole 16-byte pieces. head_dim**-0.5 is the default
    scale.
    """
    who = "paged_attention"
    if scale is None:
        scale = _default_scale(Q)
    if _use_hip():
        return _hip().hip_paged_attention(Q, K_pages, V_pages, block_table, lengths, new_lengths, scale, weights)
    _no_gradients(who, Q, K_pages, V_pages, weights)
    _check_cache(who, K_pages, V_pages, block_table, lengths, new_lengths, weights, (weights,))
    B, cols = block_table.shape
    _, Hk, size, D = K_pages.shape
    if Q.dim() != 4 or Q.shape[0] != B or Q.shape[3] != D or Q.shape[1] % Hk or Q.dtype != K_pages.dtype:
        raise RuntimeError(f"{who}: Q {tuple(Q.shape)} of {Q.dtype} does not belong to K_pages {tuple(K_pages.shape)} of "
                           f"{K_pages.dtype} and block_table {tuple(block_table.shape)}")
    if not 1e-30 < scale < 1e30:
        raise RuntimeError(f"{who}: scale must be positive, got {scale}")
    H, N, L, dev = Q.shape[1], Q.shape[2], cols * size, Q.device
    if Q.numel() == 0 or L == 0:
        return torch.zeros_like(Q)
    j, i = torch.arange(L, device=dev), torch.arange(N, device=dev)
    n = lengths.to(dev).long().clamp(0, L).view(B, 1)
    m = torch.full_like(n, N) if new_lengths is None else new_lengths.to(dev).long().clamp(0, N).view(B, 1)
    sees = torch.where(i < m, n - (m - 1 - i), torch.zeros_like(n))  # (batch, queries)
    seen = j < sees.view(B, 1, N, 1)
    at, there = _page_rows(K_pages, block_table, j)
    K, V = (_wide(_read_rows(p, at, there & (j < n).view(B, 1, L))) for p in (K_pages, V_pages))
    G = H // Hk
    q = torch.where((i < m).view(B, 1, N, 1), _wide(Q), torch.zeros((), dtype=_wide(Q).dtype, device=dev))
    S = (q.reshape(B, Hk, G * N, D) @ K.transpose(2, 3)) * scale
    P = _masked_softmax(S.view(B, H, N, L).masked_fill(~seen, float("-inf")).view(B, Hk, G * N, L))
    if weights is not None:
        weights += P.sum(2).to(weights.dtype)
    return (P @ V).reshape(B, H, N, D).to(Q.dtype)


def paged_cache_append(
    K: torch.Tensor,
    V: torch.Tensor,
    K_pages: torch.Tensor,
    V_pages: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    new_lengths: torch.Tensor | None = None,
    weights: torch.Tensor | None = None,
) -> torch.Tensor:
    """Writes new tokens' keys and values behind the rows that a cache in pages
    has (`paged_attention`), in place, and returns the new lengths.

    K, V (batch, kv_heads, tokens, head_dim) in the pages' dtype, strided views
    allowed: row i < new_lengths[b] (None: all) becomes row lengths[b] + i of
    sequence b. Rows past the table's columns, or in a page that is not there,
    are left out. K and V may be rows of the pages themselves: they are read before
    any is written. `weights` (batch, kv_heads, slots), where given, is set to zero at
    the new rows. A page that is written stands once in block_table, and
    K_pages and V_pages lie apart.
    """
    who = "paged_cache_append"
    if _use_hip():
        return _hip().hip_paged_cache_append(K, V, K_pages, V_pages, block_table, lengths, new_lengths, weights)
    _no_gradients(who, K, V, K_pages, V_pages, weights)
    _check_cache(who, K_pages, V_pages, block_table, lengths, new_lengths, weights, (K_pages, V_pages, weights))
    B, cols = block_table.shape
    _, Hk, size, D = K_pages.shape
    if K.dim() != 4 or K.shape != V.shape or (K.shape[0], K.shape[1], K.shape[3]) != (B, Hk, D):
        raise RuntimeError(f"{who}: K {tuple(K.shape)} and V {tuple(V.shape)} must be ({B}, {Hk}, tokens, {D})")
    if K.dtype != K_pages.dtype or V.dtype != K_pages.dtype:
        raise RuntimeError(f"{who}: K and V must have the pages' dtype {K_pages.dtype}")
    if K_pages.numel() and K_pages.data_ptr() == V_pages.data_ptr():
        raise RuntimeError(f"{who}: K_pages and V_pages are the same")
    N, L, dev = K.shape[2], cols * size, K_pages.device
    n = lengths.to(dev).long().clamp(0, L)
    m = torch.full_like(n, N) if new_lengths is None else new_lengths.to(dev).long().clamp(0, N)
    held = [p.untyped_storage().data_ptr() for p in (K_pages, V_pages)]
    K, V = (t.clone() if t.untyped_storage().data_ptr() in held else t for t in (K, V))
    for b in range(B):
        new = min(int(m[b]), L - int(n[b]))
        if new <= 0:
            continue
        slots = int(n[b]) + torch.arange(new, device=dev)
        (page, head, row), there = _page_rows(K_pages, block_table[b : b + 1], slots)
        for pages, rows in ((K_pages, K), (V_pages, V)):
            pages[page[there], head[there], row[there]] = rows[b : b + 1, :, :new].to(dev)[there]
        if weights is not None:
            weights[b, :, int(n[b]) : int(n[b]) + new] = 0
    return (n + m).clamp_max(L).to(lengths.dtype).to(lengths.device)


def paged_cache_evict(
    K_pages: torch.Tensor,
    V_pages: torch.Tensor,
    weights: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    budget: int,
    recent: int = 0,
) -> torch.Tensor:
    """Cuts every sequence of a cache in pages (`paged_attention`) that has more
    than `budget` rows down to it, in place, and returns the new lengths.

    Each key head of such a sequence keeps its last `recent` rows (at most
    `budget`) and, of the others, the budget - recent with the largest
    accumulated `weights` (batch, kv_heads, slots) float32; of equal weights the
    first rows, a NaN counts as above all numbers. The kept rows of K_pages,
    V_pages and weights move to rows [0, budget) in their order; what stands
    behind them is left as it was. Heads keep rows of their own. A sequence of
    at most `budget` rows stays as it is. A page of a cut sequence's rows stands
    once in block_table, and K_pages and V_pages lie apart.
    """
    who = "paged_cache_evict"
    if _use_hip():
        return _hip().hip_paged_cache_evict(K_pages, V_pages, weights, block_table, lengths, budget, recent)
    _no_gradients(who, K_pages, V_pages, weights)
    _check_cache(who, K_pages, V_pages, block_table, lengths, None, weights, (K_pages, V_pages, weights))
    if not 0 <= recent <= budget:
        raise RuntimeError(f"{who}: recent {recent} is not in 0 .. budget {budget}")
    if K_pages.numel() and K_pages.data_ptr() == V_pages.data_ptr():
        raise RuntimeError(f"{who}: K_pages and V_pages are the same")
    B, cols = block_table.shape
    L, dev = cols * K_pages.shape[2], K_pages.device
    n = lengths.to(dev).long().clamp(0, L)
    for b in range(B):
        rows = int(n[b])
        if rows <= budget:
            continue
        heavy = weights[b, :, : rows - recent].sort(dim=-1, descending=True, stable=True).indices[:, : budget - recent]
        last = torch.arange(rows - recent, rows, device=dev).expand(heavy.shape[0], recent)
        kept = torch.cat([heavy.sort(-1).values, last], 1)
        source, there = _page_rows(K_pages, block_table[b : b + 1], kept.unsqueeze(0))
        (page, head, row), room = _page_rows(K_pages, block_table[b : b + 1], torch.arange(budget, device=dev))
        for pages in (K_pages, V_pages):
            pages[page[room], head[room], row[room]] = _read_rows(pages, source, there)[room]
        weights[b, :, :budget] = weights[b].gather(1, kept)
    return n.clamp_max(budget).to(lengths.dtype).to(lengths.device)


def rope_frequencies(rot_dim: int, theta: float = 10000.0, device=None) -> torch.Tensor:
    """The angles per position of `qk_norm_rope`: theta**(-2 j / rot_dim) for
    j < rot_dim / 2, in float64."""
    if rot_dim < 0 or rot_dim % 2:
        raise RuntimeError(f"rope_frequencies: rot_dim {rot_dim} must be even")
    j = torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device)
    return float(theta) ** (-j / max(rot_dim, 1))


def _rope_join(a, b, rest, interleaved):
    pairs = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([pairs, rest], -1)


def _norm_rope_pytorch(x, w, cos, sin, rot, eps, interleaved):
    X, W = _wide(x), _wide(w)
    n = X * torch.rsqrt((X * X).mean(-1, keepdim=True) + eps) * W
    if interleaved:
        a, b = n[..., 0:rot:2], n[..., 1:rot:2]
    else:
        a, b = n[..., : rot // 2], n[..., rot // 2 : rot]
    cos, sin = cos.to(n.dtype), sin.to(n.dtype)
    return _rope_join(a * cos - b * sin, b * cos + a * sin, n[..., rot:], interleaved).to(x.dtype)


def qk_norm_rope(
    Q: torch.Tensor,
    K: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    eps: float = 1e-6,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every query and key head and its rotation by its token's
    position: what goes into an attention's Q and K, in one pass over both.

    Q (batch, heads, tokens, head_dim) and K (batch, kv_heads, tokens,
    head_dim), strided views allowed; the results are contiguous, as
    `block_sparse_attention_tiled` takes them. Every head vector is divided by
    sqrt(mean square + eps) and multiplied by q_weight / k_weight (head_dim,),
    in Q's dtype or float32. Its first rot = 2 * len(inv_freq) elements are
    then rotated in pairs, (j, j + rot / 2) or with `interleaved` (2 j, 2 j +
    1), by the angle positions * inv_freq[j] formed in float64
    (`rope_frequencies`); the rest stay. positions (tokens,) or (batch, tokens)
    are int32 or int64.

    float32, bfloat16 and float16 on the HIP backend, head_dim even and at most
    256; squares are summed in float32, whose range they have to stay in.
    Differentiable in Q, K and the weights; the HIP backend refuses an inv_freq
    that requires a gradient.
    """
    if _use_hip():
        from .hip.dispatch import hip_qk_norm_rope

        return hip_qk_norm_rope(Q, K, q_weight, k_weight, positions, inv_freq, eps, interleaved)
    who = "qk_norm_rope"
    if Q.dim() != 4 or K.dim() != 4 or (K.shape[0], K.shape[2], K.shape[3]) != (Q.shape[0], Q.shape[2], Q.shape[3]):
        raise RuntimeError(f"{who}: Q {tuple(Q.shape)} and K {tuple(K.shape)} must be (batch, heads, tokens, head_dim)")
    B, _, S, D = Q.shape
    if Q.dtype != K.dtype or not Q.is_floating_point():
        raise RuntimeError(f"{who}: Q and K must have one floating dtype, got {Q.dtype} and {K.dtype}")
    if q_weight.shape != (D,) or k_weight.shape != (D,) or q_weight.dtype != k_weight.dtype:
        raise RuntimeError(f"{who}: weights must be ({D},) of one dtype")
    if q_weight.dtype not in (Q.dtype, torch.float32):
        raise RuntimeError(f"{who}: weights must be {Q.dtype} or torch.float32, got {q_weight.dtype}")
    if D % 2 or not 2 <= D <= 256:
        raise RuntimeError(f"{who}: head_dim {D} must be even and at most 256")
    if inv_freq.dim() != 1 or not inv_freq.is_floating_point() or 2 * inv_freq.numel() > D:
        raise RuntimeError(f"{who}: inv_freq must be up to {D // 2} floating values")
    if positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) not in ((S,), (B, S)):
        raise RuntimeError(f"{who}: positions must be ({S},) or ({B}, {S}) of int32 or int64")
    if not eps >= 0:
        raise RuntimeError(f"{who}: eps must not be negative")
    angle = (positions.to(Q.device).double().unsqueeze(-1) * inv_freq.to(Q.device).double()).expand(B, S, -1).unsqueeze(1)
    cos, sin, rot = angle.cos(), angle.sin(), 2 * inv_freq.numel()
    return tuple(_norm_rope_pytorch(x, w, cos, sin, rot, eps, interleaved) for x, w in ((Q, q_weight), (K, k_weight)))
