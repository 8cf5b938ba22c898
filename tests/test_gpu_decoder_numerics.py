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
from test_gpu_cross_attention import BF, HF, make

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


# (batch, heads, kv_heads, queries, keys, head_dim): many keys, with few queries
# (P and dS as sums of two numbers) and with more
MANY_KEYS = [(1, 1, 1, 32, 131072, 64), (1, 2, 1, 64, 131072, 64), (1, 1, 1, 8, 524288, 64), (1, 2, 1, 64, 33000, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("size", MANY_KEYS)
def test_many_keys(hip_backend, size, dt):
    """P of many keys is small: fp16 keeps its digits all the same."""
    e = gradient_errors(*step(size, dt))
    assert e["dV"] <= NORM, e
