"""The operators around attention on the CPU: the "pytorch" backend against
the float64 oracle, their gradients against differences, and refusals (on the
host, before any device work)."""

from __future__ import annotations

import pytest
import torch

import trnsparse_amd as ts
from oracle import layer

F64 = torch.float64


def heads(B, H, Hk, N, L, D, dt=F64, seed=0):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(B, h, n, D, generator=g, dtype=F64).to(dt) for h, n in ((H, N), (Hk, L), (Hk, L)))


@pytest.mark.parametrize("size", [(2, 4, 2, 3, 7, 16), (1, 1, 1, 1, 1, 5), (3, 6, 2, 2, 0, 8), (2, 2, 1, 0, 4, 8)])
def test_cross_attention(pytorch_backend, size):
    Q, K, V = heads(*size)
    r = layer.attention(Q, K, V, size[-1] ** -0.5)
    torch.testing.assert_close(ts.cross_attention(Q, K, V), r["O"], rtol=1e-12, atol=1e-12)


def test_cross_attention_without_keys(pytorch_backend):
    Q, K, V = heads(2, 2, 2, 3, 0, 8)
    Q[0, 0, 0, 0] = float("inf")
    Q.requires_grad_()
    O = ts.cross_attention(Q, K, V)
    assert (O == 0).all() and (torch.autograd.grad(O.sum(), Q)[0] == 0).all()


def test_cross_attention_lengths(pytorch_backend):
    Q, K, V = heads(4, 4, 2, 3, 9, 8)
    lengths = torch.tensor([0, 1, 9, 20])
    K[0], V[1, :, 1:], K[1, :, 1:] = float("nan"), float("inf"), float("nan")
    O = ts.cross_attention(Q, K, V, lengths, scale=0.3)
    r = layer.attention(Q, K, V, 0.3, layer.lengths_seen(lengths, 3, 9))
    torch.testing.assert_close(O, r["O"], rtol=1e-12, atol=1e-12)
    assert (O[0] == 0).all()


def test_cross_attention_gradients(pytorch_backend):
    """Against the formula and against differences."""
    Q, K, V = (t.requires_grad_() for t in heads(2, 4, 2, 3, 5, 4))
    lengths = torch.tensor([3, 0])
    f = lambda q, k, v: ts.cross_attention(q, k, v, lengths)  # noqa: E731
    assert torch.autograd.gradcheck(f, (Q, K, V))
    O = f(Q, K, V)
    dO = torch.randn(O.shape, dtype=F64, generator=torch.Generator().manual_seed(1))
    r = layer.attention(Q, K, V, 0.5, layer.lengths_seen(lengths, 3, 5), dO)
    for got, want in zip(torch.autograd.grad(O, (Q, K, V), dO), ("dQ", "dK", "dV")):
        torch.testing.assert_close(got, r[want], rtol=1e-11, atol=1e-12)


@pytest.mark.parametrize("N", [1, 4])
def test_shared_prefix_attention(pytorch_backend, N):
    Q, K, V = heads(4, 4, 2, N, 6, 8)
    _, pK, pV = (t[0] for t in heads(1, 2, 2, 1, 5, 8, seed=1))
    lengths = torch.tensor([0, 2, 6, 50])
    K[0], V[1, :, 2:] = float("nan"), float("inf")
    seen = torch.cat([torch.ones(4, N, 5, dtype=torch.bool), layer.lengths_seen(lengths, N, 6, causal=True)], 2)
    for P in (5, 0):
        k = torch.cat([pK[:, :P].expand(4, -1, -1, -1), K], 2)
        v = torch.cat([pV[:, :P].expand(4, -1, -1, -1), V], 2)
        r = layer.attention(Q, k, v, 8**-0.5, seen[..., 5 - P:])
        O = ts.shared_prefix_attention(Q, pK[:, :P], pV[:, :P], K, V, lengths)
        torch.testing.assert_close(O, r["O"], rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [8, 4, 0])
def test_qk_norm_rope(pytorch_backend, interleaved, rot):
    """Against the formula, its gradients and differences."""
    g = torch.Generator().manual_seed(2)
    Q, K = (torch.randn(2, h, 3, 8, dtype=F64, generator=g).requires_grad_() for h in (3, 2))
    wq, wk = (torch.randn(8, dtype=F64, generator=g).requires_grad_() for _ in range(2))
    f = ts.rope_frequencies(rot, 100.0)
    for pos in (torch.tensor([0, 5, 70000]), torch.tensor([[1, 2, 3], [9, -4, 0]], dtype=torch.int32)):
        fn = lambda *t: ts.qk_norm_rope(*t, pos, f, 1e-3, interleaved)  # noqa: E731
        outs = fn(Q, K, wq, wk)
        dys = [torch.randn(o.shape, dtype=F64, generator=g) for o in outs]
        dQ, dK, dwq, dwk = torch.autograd.grad(outs, (Q, K, wq, wk), dys)
        for x, w, o, dy, dx, dw in ((Q, wq, outs[0], dys[0], dQ, dwq), (K, wk, outs[1], dys[1], dK, dwk)):
            r = layer.norm_rope(x, w, pos, f, 1e-3, interleaved, dy)
            for got, want in ((o, r["y"]), (dx, r["dx"]), (dw, r["dw"])):
                torch.testing.assert_close(got, want, rtol=1e-11, atol=1e-11)
        assert torch.autograd.gradcheck(fn, (Q, K, wq, wk))


def test_rope_frequencies():
    f = ts.rope_frequencies(64, 500.0)
    assert f.dtype == F64 and f.shape == (32,) and f[0] == 1 and abs(f[16] - 500.0**-0.5) < 1e-15
    with pytest.raises(RuntimeError):
        ts.rope_frequencies(7)


def refusals(dt=F64, other=torch.float32, dev="cpu"):
    Q, K, V = (t.to(dev) for t in heads(2, 4, 2, 3, 5, 8, dt))
    p, i = K[0], lambda *v: torch.tensor(v, device=dev)
    x, s, n = ts.cross_attention, ts.shared_prefix_attention, ts.qk_norm_rope
    wide = [torch.zeros(1, 1, 2, 129, dtype=dt, device=dev) for _ in range(3)]
    R = V[:, :, :3]  # Q's tokens
    w, pos, f = torch.ones(8, dtype=dt, device=dev), torch.arange(3, device=dev), ts.rope_frequencies(8, device=dev)
    odd, big = (torch.zeros(1, 1, 3, d, dtype=dt, device=dev) for d in (7, 258))
    ones, narrow = torch.ones(258, dtype=dt, device=dev), w.to(torch.bfloat16)
    return [
        (x, (Q[0], K, V)), (x, (Q, K, V[:, :, :4])), (x, (Q[:1], K, V)), (x, (Q[..., :4], K, V)), (x, (Q[:, :3], K, V)),
        (x, (Q, K[:, :0], V[:, :0])), (x, (Q.to(other), K, V)), (x, (Q.int(), K.int(), V.int())),
        (x, (Q, K, V, None, 0.0)), (x, (Q, K, V, None, -1.0)), (x, (Q, K, V, None, float("nan"))),
        (x, (Q, K, V, None, float("inf"))), (x, (Q, K, V, i(1))), (x, (Q, K, V, i(1.0, 2.0))),
        (x, (Q, K, V, i(1, 1).int().view(2, 1))), (x, tuple(wide)), (x, (Q[..., :0], K[..., :0], V[..., :0])),
        (s, (Q, p[:1], p[:1], K, V)), (s, (Q, p, p[:, :2], K, V)), (s, (Q, p[..., :4], p[..., :4], K, V)),
        (s, (Q, K, V, K, V)), (s, (Q, p.to(other), p.to(other), K, V)), (s, (Q.clone().requires_grad_(), p, p, K, V)),
        (s, (Q, p, p, K, V, i(1, 2, 3))), (s, (Q, p, p, K, V, None, 0.0)),
        (n, (Q[0], R[0], w, w, pos, f)), (n, (Q, R[:, :, :2], w, w, pos, f)), (n, (Q, R.to(other), w, w, pos, f)),
        (n, (Q, R, w[:4], w, pos, f)), (n, (Q, R, w, narrow, pos, f)), (n, (Q, R, narrow, narrow, pos, f)),
        (n, (odd, odd, w[:7], w[:7], pos, f[:2])), (n, (big, big, ones, ones, pos, f)),
        (n, (Q, R, w, w, pos, ts.rope_frequencies(10, device=dev))), (n, (Q, R, w, w, pos, f.view(2, 2))),
        (n, (Q, R, w, w, pos, pos)), (n, (Q, R, w, w, pos.float(), f)), (n, (Q, R, w, w, pos[:2], f)),
        (n, (Q, R, w, w, pos.view(1, 3), f)), (n, (Q, R, w, w, pos, f, -1.0)), (n, (Q, R, w, w, pos, f, float("nan"))),
    ]


@pytest.mark.parametrize("i", range(len(refusals())))
def test_refusals(pytorch_backend, i):
    f, args = refusals()[i]
    with pytest.raises(RuntimeError):
        f(*args)


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(refusals())))
def test_refusals_on_the_gpu(hip_backend, i):
    """The HIP operators refuse the same calls, on the host."""
    f, args = refusals(torch.float32, torch.float16, "cuda")[i]
    with pytest.raises(RuntimeError):
        f(*args)


def test_c_abi_refusals():
    """Sizes, alignment, strides, scale and workspace are checked on the host
    (dummy pointers: nothing is dereferenced)."""
    import ctypes

    from trnsparse_amd.hip import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built (run __graft_entry__.build())")
    lib = _lib.load()
    st = lambda *v: (ctypes.c_int64 * 3)(*v)  # noqa: E731
    d, good = 256, st(64 * 64, 64, 64)

    def call(Q=d, qs=good, K=d, ks=good, V=d, vs=good, dt=_lib.TSP_BF16, B=1, H=2, Hk=2, N=64, L=64, D=64, it=1, scale=0.1,
             O=d, ws=d, wsb=1 << 40):
        return lib.tsp_cross_attn_fwd(Q, qs, K, ks, V, vs, dt, B, H, Hk, N, L, D, None, it, scale, O, good, None, ws, wsb,
                                      None)

    assert call(dt=_lib.TSP_F64) == -2 and b"dtype" in lib.tsp_last_error()
    assert call(H=3) == -1 and call(Hk=0) == -1 and call(N=-1) == -1 and call(L=-5) == -1
    assert call(D=136) == -2 and call(D=60) == -2 and call(D=0) == -1
    assert call(Q=None) == -1 and call(V=None) == -1 and call(O=None) == -1
    assert call(K=264) == -1 and call(ks=st(64 * 64, 64, 68)) == -1  # pieces of 16 bytes
    assert call(vs=st(64 * 64, 64, 0)) == -1  # rows on top of each other
    assert call(ks=st(0, 0, 1 << 24)) == -1  # rows 32 MiB apart
    assert call(scale=0.0) == -1 and call(scale=float("nan")) == -1 and call(it=5) == -1
    assert call(scale=1e-40) == -1  # zero in fp32
    assert call(H=2048, Hk=2048, N=1 << 20) == -2 and call(L=1 << 31) == -2 and call(B=1 << 31) == -2
    assert call(L=100000, ws=None) == -1 and b"workspace" in lib.tsp_last_error()
    assert call(L=100000, wsb=16) == -1
    assert call(B=0) == 0 and call(N=0) == 0  # nothing to do
    assert lib.tsp_prefix_attn_fwd(d, good, d, good, d, good, d, good, d, good, 2, 1, 2, 2, 64, 64, -1, 64, None, 1, 0.1,
                                   d, good, d, 1 << 40, None) == -1
    assert lib.tsp_prefix_attn_fwd(d, good, d, good, d, good, d, good, d, good, 2, 1, 2, 2, 64, 64, 64, 64, None, 1, 0.1,
                                   d, good, None, 0, None) == -1 and b"workspace" in lib.tsp_last_error()
    assert lib.tsp_prefix_attn_workspace_size(7, 1, 2, 2, 1, 8, 8, 64) == -1
