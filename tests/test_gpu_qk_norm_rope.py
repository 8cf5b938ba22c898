"""GPU parity of qk_norm_rope and its gradients against the float64 oracle.

Bounds against the oracle's scales, u = eps / 2 of the result's type, e =
2^-24: the result's rounding gives u of itself; the fp32 steps before it: a sum
of D squares (relative error D e / 2 in r, once more where r^3 enters), the
reciprocal root, the angle's cosine and sine (4 e absolute each: e pi for its
rounding to fp32 half turns, an ulp of the function), and a handful of
products: (2 D + 32) e covers them. Weight gradients add sums over R rows, at
most R e more of their scale.
"""

from __future__ import annotations

import pytest
import torch

import trnsparse_amd as ts
from oracle import layer

pytestmark = pytest.mark.gpu

E = 2.0**-24
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def make(B, H, Hk, S, D, dt, wdt=None, seed=0):
    """Views of a fused projection's output."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    fused = torch.randn(B, S, H + 2 * Hk, D, device="cuda", generator=g).to(dt)
    Q, K = fused[:, :, :H].transpose(1, 2), fused[:, :, H : H + Hk].transpose(1, 2)
    wq, wk = (1 + 0.2 * torch.randn(2, D, device="cuda", generator=g)).to(wdt or dt)
    gQ, gK = (torch.randn(B, h, S, D, device="cuda", generator=g).to(dt) for h in (H, Hk))
    return Q, K, wq, wk, gQ, gK


def check(Q, K, wq, wk, gQ, gK, pos, f, eps=1e-6, interleaved=False):
    leaves = [t.detach().requires_grad_() for t in (Q, K, wq, wk)]
    outs = ts.qk_norm_rope(*leaves, pos, f, eps, interleaved)
    grads = torch.autograd.grad(outs, leaves, (gQ, gK))
    with torch.no_grad():
        again = ts.qk_norm_rope(Q, K, wq, wk, pos, f, eps, interleaved)
    D, R = Q.shape[3], Q.shape[0] * Q.shape[2]
    tiny = 2.0**-25 if Q.dtype == HF else 0.0
    for i, (x, w, dy) in enumerate(((Q, wq, gQ), (K, wk, gK))):
        assert outs[i].is_contiguous() and torch.equal(outs[i], again[i])
        assert outs[i].shape == x.shape and grads[i].shape == x.shape and grads[i].dtype == x.dtype
        r = layer.norm_rope(x, w, pos, f, eps, interleaved, dy)
        u, uw = torch.finfo(x.dtype).eps / 2, torch.finfo(w.dtype).eps / 2
        for got, k, un, steps, low in ((outs[i], "y", u, 2 * D + 32, tiny), (grads[i], "dx", u, 2 * D + 32, tiny),
                                       (grads[2 + i], "dw", uw, 2 * D + 32 + R * x.shape[1], 2.0**-25 if w.dtype == HF else 0.0)):
            far = (got.double().cpu() - r[k]).abs() - (un * r[k].abs() + steps * E * (1 + un) * r["a" + k] + low)
            assert far.numel() == 0 or far.max() <= 0, (k, i, float(far.max()))
    return outs, grads


# (batch, heads, kv_heads, tokens, head_dim, rot): every chunk width, one token
# and many, more heads than a wavefront takes at once, heads that leave lanes idle
SIZES = [
    (1, 1, 1, 1, 2, 2), (3, 32, 8, 1, 128, 128), (2, 4, 2, 65, 64, 64), (1, 9, 3, 333, 80, 40), (2, 3, 1, 17, 96, 96),
    (1, 5, 5, 33, 128, 64), (2, 2, 2, 40, 40, 20), (1, 2, 1, 30, 120, 60), (1, 3, 2, 21, 256, 256), (1, 2, 1, 9, 250, 126),
    (1, 2, 2, 50, 6, 4), (2, 7, 1, 12, 16, 0), (1, 16, 16, 1000, 64, 32),
]


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_sizes(hip_backend, size, interleaved, dt):
    *s, rot = size
    pos = torch.arange(s[3], device="cuda")
    check(*make(*s, dt), pos, ts.rope_frequencies(rot, device="cuda"), interleaved=interleaved)


@pytest.mark.parametrize("dt", [BF, F32])
def test_far_positions(hip_backend, dt):
    """Positions of their own for each sequence, past 2^31 and negative."""
    pos = torch.tensor([[0, 1, 4_000_000, 2**31 + 7, 2**40], [-1, -70000, 5, 5, 131071]], device="cuda")
    check(*make(2, 4, 2, 5, 64, dt), pos, ts.rope_frequencies(64, device="cuda"))
    check(*make(2, 4, 2, 5, 64, dt), pos.clamp(-70000, 2**30).int(), ts.rope_frequencies(64, 1e6, device="cuda"))


@pytest.mark.parametrize("dt", [BF, HF])
def test_float32_weights(hip_backend, dt):
    pos = torch.arange(70, device="cuda")
    check(*make(1, 4, 2, 70, 128, dt, wdt=F32), pos, ts.rope_frequencies(128, device="cuda"))


@pytest.mark.parametrize("dt", [BF, F32])
def test_views(hip_backend, dt):
    """Orders and strides do not change the results; unaligned rows hold the bounds; positions may be strided too."""
    Q, K, wq, wk, gQ, gK = make(2, 4, 2, 30, 64, dt)
    f = ts.rope_frequencies(64, device="cuda")
    pos = torch.arange(120, device="cuda").view(2, 60)
    want = ts.qk_norm_rope(Q.contiguous(), K.contiguous(), wq, wk, pos[:, ::2].contiguous(), f)

    def odd(t):
        b = torch.zeros(*t.shape[:3], 67, dtype=dt, device="cuda")
        b[..., 1:65] = t
        return b[..., 1:65]

    for fn in (lambda t: t, lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)):
        got = ts.qk_norm_rope(fn(Q), fn(K), wq, wk, pos[:, ::2], f)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # An unaligned view is read in narrower chunks, so its D squares are added
    # in another order: the sums of two orders differ by up to D e of the sum,
    # and so may the last bit of a result. Both are held to the bounds above.
    check(odd(Q), odd(K), wq, wk, odd(gQ), gK.transpose(2, 3).contiguous().transpose(2, 3), pos[:, ::2], f)
    same = Q[:, :1].expand(-1, 4, -1, -1)  # one head for all: a stride of zero
    assert torch.equal(ts.qk_norm_rope(same, K, wq, wk, pos[:, ::2], f)[0],
                       ts.qk_norm_rope(same.contiguous(), K, wq, wk, pos[:, ::2], f)[0])


def test_zero_rows_and_no_rows(hip_backend):
    """A zero head vector stays zero (eps holds the norm); no tokens, no heads."""
    f, pos = ts.rope_frequencies(64, device="cuda"), torch.arange(4, device="cuda")
    Q, K, wq, wk, gQ, gK = make(1, 2, 1, 4, 64, BF)
    Q = Q.clone()
    Q[0, 1, 2] = 0
    (q, _), _ = check(Q, K, wq, wk, gQ, gK, pos, f)
    assert (q[0, 1, 2] == 0).all()
    leaves = [t.detach().requires_grad_() for t in (Q[:, :, :0], K[:, :, :0], wq, wk)]
    outs = ts.qk_norm_rope(*leaves, pos[:0], f)
    grads = torch.autograd.grad(outs, leaves, [torch.zeros_like(o) for o in outs])
    assert outs[0].shape == (1, 2, 0, 64) and (grads[2] == 0).all() and (grads[3] == 0).all()
    q, k = ts.qk_norm_rope(Q, K[:, :0], wq, wk, pos, f)
    assert k.shape == (1, 0, 4, 64) and torch.equal(q, ts.qk_norm_rope(Q, K, wq, wk, pos, f)[0])


def test_one_result_used(hip_backend):
    """A gradient of one result alone, and frozen weights."""
    Q, K, wq, wk, gQ, _ = make(1, 2, 2, 40, 64, F32)
    f, pos = ts.rope_frequencies(64, device="cuda"), torch.arange(40, device="cuda")
    q = Q.detach().requires_grad_()
    out = ts.qk_norm_rope(q, K, wq, wk, pos, f)[0]
    (dq,) = torch.autograd.grad(out, (q,), gQ)
    r = layer.norm_rope(Q, wq, pos, f, 1e-6, False, gQ)
    assert (dq.double().cpu() - r["dx"]).abs().max() <= 1e-5 * r["dx"].abs().max()


def test_weight_gradients_repeat(hip_backend):
    args = make(2, 8, 2, 3000, 128, BF, seed=3)
    f, pos = ts.rope_frequencies(128, device="cuda"), torch.arange(3000, device="cuda")
    leaves = [t.detach().requires_grad_() for t in args[:4]]
    first = None
    for _ in range(3):
        grads = torch.autograd.grad(ts.qk_norm_rope(*leaves, pos, f), leaves, args[4:])
        first = first or grads
        assert all(torch.equal(a, b) for a, b in zip(first, grads))


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("size", [(1, 2, 1, 9001, 64, 64), (3, 5, 2, 1801, 128, 32), (2, 1, 3, 4999, 20, 10), (1, 9, 1, 4200, 256, 200)])
def test_long_sequences(hip_backend, size, dt):
    """More tokens than the backward's wavefronts: each takes several in turn."""
    *s, rot = size
    pos = torch.arange(s[0] * s[3], device="cuda").view(s[0], s[3])
    check(*make(*s, dt, seed=3), pos, ts.rope_frequencies(rot, device="cuda"), interleaved=s[4] == 20)
