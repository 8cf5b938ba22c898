"""The decoder layer's C entry points with operands of one row, whose row stride
is anything: results are those of ordinary strides."""

from __future__ import annotations

import ctypes

import pytest
import torch

from trnsparse_amd.hip import _lib

pytestmark = pytest.mark.gpu


def _strides(t, row):
    """(batch, head, row) strides, that of a single row replaced by `row`."""
    s = list(t.stride()[:3])
    if t.size(2) == 1 and row is not None:
        s[2] = row
    return (ctypes.c_int64 * 3)(*s)


def _cross(q, k, v, dO, row):
    """Forward and backward through the C ABI."""
    lib = _lib.load()
    code = _lib.TSP_F32 if q.dtype == torch.float32 else _lib.TSP_BF16 if q.dtype == torch.bfloat16 else _lib.TSP_F16
    B, H, N, D = q.shape
    Hk, L = k.shape[1], k.shape[2]
    size = (code, B, H, Hk, N, L, D)
    ws = torch.empty(1 + max(lib.tsp_cross_attn_workspace_size(*size), lib.tsp_cross_attn_bwd_workspace_size(*size)),
                     dtype=torch.uint8, device="cuda")
    o, dq, dk, dv = (torch.full_like(t, 7.0) for t in (q, q, k, v))
    lse = torch.empty(B, H, N, device="cuda")
    arg = lambda t: (t.data_ptr(), _strides(t, row))  # noqa: E731
    st = torch.cuda.current_stream().cuda_stream
    tail = (None, _lib.TSP_I64, D**-0.5)
    assert lib.tsp_cross_attn_fwd(*arg(q), *arg(k), *arg(v), *size, *tail, *arg(o), lse.data_ptr(), ws.data_ptr(),
                                  ws.numel(), st) == 0, lib.tsp_last_error()
    assert lib.tsp_cross_attn_bwd(*arg(q), *arg(k), *arg(v), *arg(o), *arg(dO), lse.data_ptr(), *size, *tail, *arg(dq),
                                  *arg(dk), *arg(dv), ws.data_ptr(), ws.numel(), st) == 0, lib.tsp_last_error()
    torch.cuda.synchronize()
    return o, dq, dk, dv


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N,L,H", [(1, 70, 4), (1, 1, 2), (5, 1, 2), (1, 9000, 600)])
def test_stride_of_a_single_row_is_not_used(hip_backend, N, L, H, dt):
    """One query or one key may come with any row stride: none, one below
    head_dim, one whose 63rd multiple passes 2^32 bytes."""
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda h, n: torch.randn(1, h, n, 64, device="cuda", generator=g).to(dt)  # noqa: E731
    args = (r(H, N), r(2, L), r(2, L), r(H, N))
    want = _cross(*args, None)
    for row in (0, 8, 1 << 26, 5):
        assert all(torch.equal(a, b) for a, b in zip(_cross(*args, row), want)), row


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("P,S", [(1, 1), (1, 2000), (2000, 1)])
def test_prefix_of_single_rows(hip_backend, P, S, dt):
    lib = _lib.load()
    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda b, h, n: torch.randn(b, h, n, 64, device="cuda", generator=g).to(dt)  # noqa: E731
    q, pk, pv, k, v = r(3, 4, 1), r(1, 2, P), r(1, 2, P), r(3, 2, S), r(3, 2, S)
    size = (_lib.TSP_F32 if dt == torch.float32 else _lib.TSP_BF16, 3, 4, 2, 1, P, S, 64)
    ws = torch.empty(1 + lib.tsp_prefix_attn_workspace_size(*size), dtype=torch.uint8, device="cuda")
    outs = []
    for row in (None, 0, 8, 1 << 26, 5):
        o = torch.full_like(q, 7.0)
        arg = lambda t: (t.data_ptr(), _strides(t, row))  # noqa: E731,B023
        assert lib.tsp_prefix_attn_fwd(*arg(q), *arg(pk), *arg(pv), *arg(k), *arg(v), *size, None, _lib.TSP_I64, 0.125,
                                       *arg(o), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        outs.append(o)
    assert all(torch.equal(o, outs[0]) for o in outs)
