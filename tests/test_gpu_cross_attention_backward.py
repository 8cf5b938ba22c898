"""GPU parity of cross_attention's gradients against the float64 oracle.

Bounds, elementwise against the oracle's scales (oracle/layer.py: aQ, aK, aV,
products of absolute values along each gradient's own path), u = eps / 2 of the
operands' type, e = 2^-24. Every gradient is rounded once (u). P and dS are
rounded to the type before their products (u each). O, from which D = dO . O
is formed, is rounded to the type (u of rowsum |dO| A, part of the scale): in
all 3 u (fp32: u of the result, the rest below). The fp32 steps: P = exp(s -
lse) with s off by (D + 4) e smax and lse by as much and (2 L + 64) e (sum and
logarithm) and 4 e |lse|; dO V^T and D, sums of D products, D e of their
scale, and again for their rounding when subtracted; the sums over L keys or
R = G N rows, one e a term.
fp16 gradients below its normal range are off by half a step, 2^-25, and so are
the terms of P and dS there, which are formed with dO near 1: 2^-25 sum |K| (or
|Q|) scale max |dO|.
"""

from __future__ import annotations

import pytest
import torch

import trnsparse_amd as ts
from oracle import layer
from test_gpu_cross_attention import BF, E, F32, HF, make

pytestmark = pytest.mark.gpu


def check_backward(Q, K, V, lengths=None, scale=None, dO=None, seed=50):
    B, H, N, D = Q.shape
    L, G = K.shape[2], H // K.shape[1]
    sc = scale or D**-0.5
    if dO is None:
        g = torch.Generator(device="cuda").manual_seed(seed)
        dO = torch.randn(B, N, H, D, device="cuda", generator=g).to(Q.dtype).transpose(1, 2)
    leaves = [t.detach().requires_grad_() for t in (Q, K, V)]
    O = ts.cross_attention(*leaves, lengths, scale)
    grads = torch.autograd.grad(O, leaves, dO)
    torch.cuda.synchronize()
    with torch.no_grad():
        assert torch.equal(O, ts.cross_attention(Q, K, V, lengths, scale))
    seen = None if lengths is None else layer.lengths_seen(lengths, N, L)
    r = layer.attention(Q, K, V, sc, seen, dO)
    lse = r["lse"][r["lse"].isfinite()]
    u = torch.finfo(Q.dtype).eps / 2
    inner = 2 * (D + 4) * r["smax"] + 2 * L + 64 + (4 * float(lse.abs().max()) if lse.numel() else 0) + 2 * D
    base = (3 * u if Q.dtype != F32 else u) + E * inner
    ok = torch.ones(B, 1, L, 1) if lengths is None else layer.lengths_seen(lengths, 1, L).view(B, 1, L, 1).double()
    low = 2.0**-25 if Q.dtype == HF else 0.0
    sumK = (K.double().cpu().nan_to_num(0, 0, 0).abs() * ok).sum(2, keepdim=True).repeat_interleave(G, 1) * sc
    sumQ = Q.double().cpu().abs().reshape(B, H // G, G * N, D).sum(2, keepdim=True) * sc
    top = 2 * float(dO.abs().max())
    sumK, sumQ = sumK * top, sumQ * top
    sumG = dO.double().cpu().abs().reshape(B, H // G, G * N, D).sum(2, keepdim=True)
    for got, like, k, terms, extra in zip(grads, (Q, K, V), ("Q", "K", "V"), (L, G * N, G * N), (sumK, sumQ, sumG)):
        assert got.shape == like.shape and got.dtype == like.dtype
        far = (got.double().cpu() - r["d" + k]).abs() - ((base + E * terms) * r["a" + k] + low * (1 + extra))
        assert not got.isnan().any() and (far.numel() == 0 or far.max() <= 1e-30), ("d" + k, float(far.max()))
    return grads, r


SIZES = [
    (1, 1, 1, 1, 1, 64), (2, 4, 2, 1, 37, 64), (1, 8, 2, 3, 1500, 128), (2, 6, 2, 5, 130, 40), (1, 4, 2, 17, 33, 96),
    (1, 3, 3, 128, 128, 128), (2, 2, 1, 129, 257, 128), (1, 6, 3, 70, 300, 80), (1, 2, 2, 300, 511, 16),
    (1, 1, 1, 600, 40, 8), (2, 4, 4, 64, 100, 120), (1, 2, 2, 40, 90, 7), (1, 4, 1, 200, 1, 64), (1, 1, 1, 2000, 130, 64),
]


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("size", SIZES)
def test_sizes(hip_backend, size, dt):
    check_backward(*make(*size, dt))


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("N,heads", [(1, (4, 2)), (140, (4, 2)), (300, (2, 2))])
def test_lengths(hip_backend, dt, N, heads):
    """Padded batches: gradients behind the length are zero, whatever stands there."""
    L = 300
    lengths = torch.tensor([0, 1, 64, 127, 300, 999], device="cuda")
    Q, K, V = make(6, *heads, N, L, 64, dt, seed=1)
    K, V = K.clone(), V.clone()
    for b, n in enumerate(lengths.clamp(0, L).tolist()):
        K[b, :, n:], V[b, :, n:] = float("inf"), float("nan")
    (dQ, dK, dV), _ = check_backward(Q, K, V, lengths)
    assert (dQ[0] == 0).all()
    for b, n in enumerate(lengths.clamp(0, L).tolist()):
        assert (dK[b, :, n:] == 0).all() and (dV[b, :, n:] == 0).all()


@pytest.mark.parametrize("dt", [BF, F32])
def test_empty(hip_backend, dt):
    for N, L in ((0, 9), (5, 0)):
        Q, K, V = (t.requires_grad_() for t in make(2, 4, 2, N, L, 64, dt, strided=False))
        grads = torch.autograd.grad(ts.cross_attention(Q, K, V), (Q, K, V), torch.ones_like(Q))
        assert all((g == 0).all() and g.shape == t.shape for g, t in zip(grads, (Q, K, V)))


@pytest.mark.parametrize("dt", [BF, F32])
def test_broadcast_and_views(hip_backend, dt):
    """One encoder's states for the whole batch: their gradient is the sum over
    it; other orders and offsets of the operands and of the gradient."""
    B, H, Hk, N, L, D = 3, 4, 2, 50, 70, 64
    Q, K, V = make(B, H, Hk, N, L, D, dt, seed=4, strided=False)
    g = torch.Generator(device="cuda").manual_seed(5)
    dO = torch.randn(B, H, N, D, device="cuda", generator=g).to(dt)
    k1 = K[:1].clone().requires_grad_()
    v1 = V[:1].clone().requires_grad_()
    O = ts.cross_attention(Q, k1.expand(B, -1, -1, -1), v1.expand(B, -1, -1, -1))
    dk1, dv1 = torch.autograd.grad(O, (k1, v1), dO)
    full = [t.clone().requires_grad_() for t in (Q, K[:1].expand(B, -1, -1, -1), V[:1].expand(B, -1, -1, -1))]
    want = torch.autograd.grad(ts.cross_attention(*full), full, dO)
    assert torch.equal(dk1, want[1].sum(0, keepdim=True)) and torch.equal(dv1, want[2].sum(0, keepdim=True))

    def odd(t):
        b = torch.zeros(*t.shape[:3], D + 3, dtype=dt, device="cuda")
        b[..., 1 : D + 1] = t
        return b[..., 1 : D + 1]

    base = [t.detach().requires_grad_() for t in (Q, K, V)]
    want = torch.autograd.grad(ts.cross_attention(*base), base, dO)
    for f in (odd, lambda t: t.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)):
        leaves = [f(t.detach()).requires_grad_() for t in (Q, K, V)]
        got = torch.autograd.grad(ts.cross_attention(*leaves), leaves, f(dO))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_parts_of_the_gradients(hip_backend):
    """Only Q, or only V, requires a gradient."""
    Q, K, V = make(2, 4, 2, 60, 90, 64, F32, seed=6)
    dO = torch.ones_like(Q)
    leaves = [t.detach().requires_grad_() for t in (Q, K, V)]
    dQ, _, dV = torch.autograd.grad(ts.cross_attention(*leaves), leaves, dO)
    q, v = Q.detach().requires_grad_(), V.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(ts.cross_attention(q, K, V), q, dO)[0], dQ)
    assert torch.equal(torch.autograd.grad(ts.cross_attention(Q, K, v), v, dO)[0], dV)


def test_against_differences(hip_backend):
    """fp32 gradients against central differences of the loss sum O W: step h
    has truncation h^2 M / 6 and rounding 2^-24 |loss terms| / h; with h = 2^-7
    and entries near 1 both stay below 2e-3."""
    Q, K, V = make(1, 2, 1, 4, 6, 16, F32, seed=7, strided=False)
    W = torch.randn(Q.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(8))
    leaves = [t.detach().requires_grad_() for t in (Q, K, V)]
    grads = torch.autograd.grad((ts.cross_attention(*leaves) * W).sum(), leaves)
    h = 2.0**-7
    for i in range(3):
        for at in ((0, 0, 0, 0), (0, -1, 3, 5), (0, 0, -1, 15)):
            vals = []
            for sgn in (1, -1):
                ts_ = [t.detach().clone() for t in (Q, K, V)]
                ts_[i][at] += sgn * h
                vals.append((ts.cross_attention(*ts_) * W).double().sum())
            assert abs((vals[0] - vals[1]) / (2 * h) - grads[i][at]) <= 2e-3


def test_repeats_are_equal(hip_backend):
    Q, K, V = (t.detach().requires_grad_() for t in make(2, 8, 2, 300, 500, 128, BF, seed=9))
    first = None
    for _ in range(3):
        grads = torch.autograd.grad(ts.cross_attention(Q, K, V), (Q, K, V), torch.ones_like(Q))
        first = first or grads
        assert all(torch.equal(a, b) for a, b in zip(first, grads))


@pytest.mark.parametrize("size", [2.0**-16, 2.0**-8, 2.0**10])
@pytest.mark.parametrize("N", [3, 200])
def test_fp16_gradients_of_any_size(hip_backend, size, N):
    """fp16 gradients far below 1 (an unscaled loss) and far above (a scaled
    one): dS is formed with dO brought near 1, so what is lost is the rounding of
    the results alone. Same bounds; rows of dO of different sizes in one tile."""
    g = torch.Generator(device="cuda").manual_seed(60)
    Q, K, V = make(2, 4, 2, N, 700, 64, HF, seed=10)
    dO = size * torch.randn(2, 4, N, 64, device="cuda", generator=g)
    dO = (dO * 2.0 ** -(torch.arange(N, device="cuda") % 5).view(N, 1)).to(HF)
    check_backward(Q, K, V, dO=dO)
    check_backward(Q, K, V, dO=torch.zeros_like(dO))


# Steps of 2^29 products of the scores and more in 16 bits: both passes in one
# launch, P and dS as one number each. With ranges of keys and of queries that are
# added (one head; one row tile), 65 to 96 elements, 64, odd edges.
LARGE = [(2, 8, 2, 401, 701, 128), (4, 8, 8, 300, 721, 80), (2, 16, 16, 513, 520, 64), (1, 1, 1, 2103, 2001, 128),
         (1, 8, 1, 16, 33000, 128)]


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("size", LARGE)
def test_large_steps(hip_backend, size, dt):
    B, H, _, N, L, D = size
    assert B * H * N * L * D >= 2**29
    (dQ, _, _), r = check_backward(*make(*size, dt, seed=11))
    # the queries' gradient alone takes the row pass alone: within two results'
    # bounds (3 u of the scale each, and the fp32 steps) of the one beside it
    Q, K, V = make(*size, dt, seed=11)
    g = torch.Generator(device="cuda").manual_seed(50)
    dO = torch.randn(B, N, H, D, device="cuda", generator=g).to(dt).transpose(1, 2)
    q = Q.detach().requires_grad_()
    alone = torch.autograd.grad(ts.cross_attention(q, K, V), q, dO)[0]
    u = torch.finfo(dt).eps / 2
    assert ((alone.double() - dQ.double()).abs().cpu() <= 8 * u * r["aQ"] + 2.0**-22).all()


@pytest.mark.parametrize("dt", [BF, HF])
def test_large_steps_with_lengths(hip_backend, dt):
    L = 1300
    lengths = torch.tensor([0, 1, 640, 1299, 1300, 5000], device="cuda", dtype=torch.int32)
    Q, K, V = make(6, 4, 2, 300, L, 64, dt, seed=12)
    K, V = K.clone(), V.clone()
    for b, n in enumerate(lengths.clamp(0, L).tolist()):
        K[b, :, n:], V[b, :, n:] = float("inf"), float("nan")
    (dQ, dK, dV), _ = check_backward(Q, K, V, lengths)
    assert (dQ[0] == 0).all()
    for b, n in enumerate(lengths.clamp(0, L).tolist()):
        assert (dK[b, :, n:] == 0).all() and (dV[b, :, n:] == 0).all()


@pytest.mark.parametrize("size", [2.0**-16, 2.0**10])
def test_large_fp16_gradients_of_any_size(hip_backend, size):
    N = 400
    g = torch.Generator(device="cuda").manual_seed(61)
    Q, K, V = make(2, 8, 2, N, 1400, 64, HF, seed=13)
    dO = size * torch.randn(2, 8, N, 64, device="cuda", generator=g)
    dO = (dO * 2.0 ** -(torch.arange(N, device="cuda") % 5).view(N, 1)).to(HF)
    check_backward(Q, K, V, dO=dO)
    check_backward(Q, K, V, dO=torch.zeros_like(dO))


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("B", [2, 64, 65])
def test_many_lengths(hip_backend, B, dt):
    """Entries of equal and of different lengths, as many as are taken longest
    first and more."""
    lengths = torch.arange(B, device="cuda") * 37 % 5 * 40
    check_backward(*make(B, 4, 2, 45, 150, 24, dt, seed=14), lengths)
