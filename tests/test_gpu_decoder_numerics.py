"""Errors of the decoder layer's operators as a whole, and operands of unusual
size, against the float64 oracle.

Elementwise bounds against sums of absolute values do not cancel where results
do, and with many keys hold for any result. Here the 2-norm of a gradient's
error is held against the gradient's own, u = eps / 2 of the operands' type. A
rounding moves each element by up to u of itself, evenly spread: u / sqrt(3) of
the norm, and a product's terms, rounded independently and of random signs, move
it as much. A gradient is rounded itself, from P or dS rounded to the type;
dS also takes up the rounding of O in D (u / sqrt(3) of |dO| |O|, |O| <= |V|):
three of them in quadrature are u. A quarter more is for what a draw of
thousands of elements leaves to chance and for the fp32 steps.
"""

from __future__ import annotations

import pytest
import torch

import trnsparse_amd as ts
from oracle import layer
import test_gpu_qk_norm_rope as norm_rope
from test_gpu_cross_attention import BF, E, F32, HF, make
from test_gpu_cross_attention_backward import LARGE

NORM = 1.25  # of u


def gradient_errors(Q, K, V, dO):
    """The 2-norms of dQ's, dK's and dV's errors over the gradients' own, in u."""
    leaves = [t.detach().requires_grad_() for t in (Q, K, V)]
    grads = torch.autograd.grad(ts.cross_attention(*leaves), leaves, dO)
    torch.cuda.synchronize()
    r = layer.attention(Q, K, V, Q.shape[3] ** -0.5, None, dO)
    u = torch.finfo(Q.dtype).eps / 2
    return {k: float((g.double().cpu() - r[k]).norm() / r[k].norm()) / u for k, g in zip(("dQ", "dK", "dV"), grads)}


def step(size, dt, seed=15):
    """Operands and a gradient large enough for fp16 results in the normal range."""
    Q, K, V = make(*size, dt, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    return Q, K, V, (2.0**8 * torch.randn(Q.shape, device="cuda", generator=g)).to(dt)


def test_the_norm_notices_a_missing_range():
    """A range of 128 of 33000 keys left out of one head's dQ, in the oracle."""
    g = torch.Generator().manual_seed(19)
    Q, dO, K, V = (torch.randn(n, 128, generator=g, dtype=torch.float64) for n in (16, 16, 33000, 33000))
    p = (Q @ K.t() * 128**-0.5).softmax(1)
    dp = dO @ V.t()
    ds = p * (dp - (p * dp).sum(1, keepdim=True))
    dQ = ds @ K
    ds[:, 640:768] = 0
    assert (ds @ K - dQ).norm() > 10 * NORM * 2.0**-8 * dQ.norm()  # bf16's bound


def check_fp16_gradients(Q, K, V, dO):
    """Elementwise, on the bounds of test_gpu_cross_attention_backward but for
    what fp16 cannot hold: P enters as 2^15 P, dS with its bound 2 D max |dO| max
    |V| at 2^14 or more, so a term below the normal range is off by 2^-40, or by
    2^-39 of that bound. O below the normal range is off by 2^-25, so D by 2^-25
    sum |dO|, which weighs rows of K with P of sum 1, and of Q with P <= 1. A
    gradient past fp16's range is infinite: both sides are clamped to it."""
    leaves = [t.requires_grad_() for t in (Q, K, V)]
    grads = torch.autograd.grad(ts.cross_attention(*leaves), leaves, dO)
    torch.cuda.synchronize()
    N, D, L, sc, top = Q.shape[2], Q.shape[3], K.shape[2], Q.shape[3] ** -0.5, torch.finfo(HF).max
    r = layer.attention(Q, K, V, sc, None, dO)
    inner = 2 * (D + 4) * r["smax"] + 2 * L + 64 + 4 * float(r["lse"].abs().max()) + 2 * D
    dS = 2.0**-39 * 2 * D * float(dO.abs().max()) * float(V.detach().abs().max()) * sc
    off = 2.0**-25 * float(dO.abs().sum(3).max()) * sc
    size = lambda t: t.detach().double().cpu().abs()  # noqa: E731
    col = lambda t: size(t).sum(2, keepdim=True)  # noqa: E731
    lows = (dS * col(K) + off * size(K).amax(2, keepdim=True), (dS + off) * col(Q), 2.0**-40 * col(dO))
    for got, k, terms, low in zip(grads, "QKV", (L, N, N), lows):
        bound = (3 * 2.0**-11 + E * (inner + terms)) * r["a" + k] + 2.0**-25 + low
        far = (got.double().cpu().clamp(-top, top) - r["d" + k].clamp(-top, top)).abs() - bound
        assert not got.isnan().any() and far.max() <= 0, ("d" + k, float(far.max()))


# (batch, heads, kv_heads, queries, keys, head_dim): many keys, with few queries
# (P and dS as sums of two numbers) and with more
MANY_KEYS = [(1, 1, 1, 32, 131072, 64), (1, 2, 1, 64, 131072, 64), (1, 1, 1, 8, 524288, 64), (1, 2, 1, 64, 33000, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("size", MANY_KEYS)
def test_many_keys(hip_backend, size, dt):
    """P and dS of many keys are small: fp16 keeps their digits all the same."""
    e = gradient_errors(*step(size, dt))
    assert max(e.values()) <= NORM, e


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("size", LARGE + [(2, 4, 2, 70, 90, 64), (1, 4, 2, 200, 300, 96)])
def test_steps(hip_backend, size, dt):
    """Both passes in one launch and apart, keys and queries in ranges; the
    queries' gradient alone, from the row pass alone."""
    Q, K, V, dO = step(size, dt)
    e = gradient_errors(Q, K, V, dO)
    assert max(e.values()) <= NORM, e
    q = Q.detach().requires_grad_()
    alone = torch.autograd.grad(ts.cross_attention(q, K, V), q, dO)[0].double()
    leaves = [t.detach().requires_grad_() for t in (Q, K, V)]
    dQ = torch.autograd.grad(ts.cross_attention(*leaves), leaves, dO)[0].double()
    assert (alone - dQ).norm() <= 2 * NORM * torch.finfo(dt).eps / 2 * dQ.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("value,grad", [(3000.0, 1.0), (65504.0, 2.0**-6), (2.0**-24, 1.0), (0.0, 1.0)])
@pytest.mark.parametrize("H,N,L", [(2, 3, 2), (2, 40, 50), (2, 200, 700), (16, 400, 1500)])
def test_values_of_any_size(hip_backend, H, N, L, value, grad):
    """fp16: dO V^T and dS of large values pass 65504 where the gradients do not.
    Two keys of opposite values share each row's weight."""
    g = torch.Generator(device="cuda").manual_seed(17)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    Q, K, V = 1 + 0.1 * r(1, H, N, 64), 0.1 * r(1, H, L, 64), 0.1 * value * r(1, H, L, 64)
    K[:, :, :2] += 1.5
    V[:, :, 0], V[:, :, 1] = value, -value
    dO = torch.full((1, H, N, 64), grad, device="cuda")
    dO[:, :, ::2] = -grad
    check_fp16_gradients(*(t.clamp(-65504, 65504).to(HF) for t in (Q, K, V)), dO.to(HF))


@pytest.mark.gpu
@pytest.mark.parametrize("at", [(5,), (0, 32, 64, 96), (524287,)])
@pytest.mark.parametrize("H,N", [(512, 1), (16, 4100), (1, 1)])
def test_one_key_outweighs_many(hip_backend, H, N, at):
    """fp16: the many keys of a long row weigh 2^-20.4 each beside a few of 1, and
    half of all or a tenth together. All of one weight, its rounding is theirs: u
    of the result, whose own rounding (u / sqrt(3) of its norm) comes on top."""
    L, D = 524288, 64
    K = torch.zeros(1, 1, L, D, dtype=HF, device="cuda")
    K[0, 0, list(at), 0] = 1
    Q = torch.zeros(1, H, N, D, dtype=HF, device="cuda")
    Q[..., 0] = 14.109375
    g = torch.Generator(device="cuda").manual_seed(18)
    V = (1 + torch.rand(1, 1, L, D, device="cuda", generator=g)).to(HF)
    O = ts.cross_attention(Q, K.expand(1, H, L, D), V.expand(1, H, L, D), scale=1.0)
    want = layer.attention(Q[:, :1, :1], K, V, 1.0)["O"]
    assert (O == O[:, :1, :1]).all()
    far = (O[:, :1, :1].double().cpu() - want).norm() / want.norm()
    assert far <= (1 + 3**-0.5) * 2.0**-11, float(far) * 2**11


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("size,eps", [(1e15, 1e-6), (1e-13, 0.0), (1e-16, 1e-30)])
def test_norms_of_any_size(hip_backend, size, eps, dt):
    """Rows whose inverse norm's third power leaves 32 bits, on the bounds of
    test_gpu_qk_norm_rope."""
    Q, K, *rest = norm_rope.make(2, 4, 2, 30, 128, dt)
    Q, K = ((size * t.float()).to(dt) for t in (Q, K))
    f, pos = ts.rope_frequencies(128, device="cuda"), torch.arange(30, device="cuda")
    norm_rope.check(Q, K, *rest, pos, f, eps)


@pytest.mark.gpu
def test_zero_rows_and_a_small_eps(hip_backend):
    """A row of zeros has the gradient w dn / sqrt(eps)."""
    Q, K, *rest = norm_rope.make(2, 4, 2, 30, 128, F32)
    f, pos = ts.rope_frequencies(128, device="cuda"), torch.arange(30, device="cuda")
    norm_rope.check(torch.zeros_like(Q), K, *rest, pos, f, 1e-28)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(11, 64, 16, 1, 128, 128), (2, 64, 8, 554, 128, 128), (1, 128, 16, 1, 96, 96),
                                  (2, 32, 8, 4096, 128, 128)])
def test_weight_gradients_in_fp32(hip_backend, size):
    """The 2-norm of a weight gradient's error. A term dn x r takes about eight
    roundings to 24 bits (cosine and sine, two products and their sum, r, x r, the
    workgroup's part, the result), 2^-24 / sqrt(3) each at most: 1.63 times 2^-24.
    Sums of the terms in 24 bits would add to it with their number."""
    *shape, rot = size
    Q, K, wq, wk, gQ, gK = norm_rope.make(*shape, F32, seed=21)
    g = torch.Generator(device="cuda").manual_seed(22)
    pos = torch.randint(0, 4_000_000, (shape[0], shape[3]), device="cuda", generator=g)
    f = ts.rope_frequencies(rot, device="cuda")
    leaves = [t.detach().requires_grad_() for t in (Q, K, wq, wk)]
    grads = torch.autograd.grad(ts.qk_norm_rope(*leaves, pos, f), leaves[2:], (gQ, gK))
    for got, x, w, dy in zip(grads, (Q, K), (wq, wk), (gQ, gK)):
        want = layer.norm_rope(x, w, pos, f, 1e-6, False, dy)["dw"]
        assert (got.double().cpu() - want).norm() <= 1.75 * 2.0**-24 * want.norm()
