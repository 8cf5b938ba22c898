"""GPU parity of shared_prefix_attention against the float64 oracle, on the
bounds of test_gpu_cross_attention (L: prefix and own keys together)."""

from __future__ import annotations

import pytest
import torch

import trnsparse_amd as ts
from oracle import layer
from test_gpu_cross_attention import BF, F32, HF, tol

pytestmark = pytest.mark.gpu


def make(B, H, Hk, N, P, S, D, dt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dt)  # noqa: E731
    return r(B, N, H, D).transpose(1, 2), r(Hk, P, D), r(Hk, P, D), r(B, Hk, S, D), r(B, Hk, S, D)


def check(Q, pK, pV, K, V, lengths=None, scale=None):
    B, H, N, D = Q.shape
    P, S = pK.shape[1], K.shape[2]
    O = ts.shared_prefix_attention(Q, pK, pV, K, V, lengths, scale)
    torch.cuda.synchronize()
    assert O.shape == Q.shape and O.dtype == Q.dtype
    n = torch.full((B,), S) if lengths is None else lengths
    seen = torch.cat([torch.ones(B, N, P, dtype=torch.bool), layer.lengths_seen(n, N, S, causal=True)], 2)
    allK = torch.cat([pK.expand(B, -1, -1, -1), K], 2)
    allV = torch.cat([pV.expand(B, -1, -1, -1), V], 2)
    r = layer.attention(Q, allK, allV, scale or D**-0.5, seen)
    far = (O.double().cpu() - r["O"]).abs() - tol(Q.dtype, D, P + S, r["smax"]) * r["A"]
    assert not O.isnan().any() and far.max() <= 1e-30, float(far.max())
    return O


# (batch, heads, kv_heads, queries, prefix, keys, head_dim)
SIZES = [
    (1, 1, 1, 1, 1, 1, 64), (4, 4, 4, 1, 512, 256, 64), (3, 8, 2, 1, 3001, 700, 128), (9, 8, 1, 5, 70, 33, 128),
    (2, 6, 2, 12, 100, 40, 40), (40, 8, 2, 1, 900, 64, 64), (2, 4, 2, 40, 300, 130, 128), (2, 4, 4, 200, 65, 300, 96),
    (1, 2, 2, 3, 200, 3, 20),
]


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("size", SIZES)
def test_sizes(hip_backend, size, dt):
    check(*make(*size, dt))


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("N", [1, 4, 40])
@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_lengths(hip_backend, dt, N, itype):
    """Caches filled to 0, 1, fewer than the new tokens, a tile's edge, all,
    outside [0, keys]; what stands behind them is infinite or NaN."""
    S = 260
    lengths = torch.tensor([0, 1, 3, 32, 129, 260, 9999, -1], dtype=itype, device="cuda")
    Q, pK, pV, K, V = make(8, 4, 2, N, 75, S, 64, dt, seed=1)
    for b, n in enumerate(lengths.clamp(0, S).tolist()):
        K[b, :, n:], V[b, :, n:] = float("inf"), float("nan")
    check(Q, pK, pV, K, V, lengths)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("N", [1, 3, 50])
def test_empty_parts(hip_backend, dt, N):
    Q, pK, pV, K, V = make(3, 4, 2, N, 90, 80, 64, dt, seed=2)
    lengths = torch.tensor([0, 2, 80], device="cuda")
    check(Q, pK[:, :0], pV[:, :0], K, V, lengths)  # no prefix: the first sequence sees nothing
    O = ts.shared_prefix_attention(Q, pK[:, :0], pV[:, :0], K, V, lengths)
    assert (O[0] == 0).all()
    check(Q, pK, pV, K[:, :, :0], V[:, :, :0])  # nothing but the prefix
    none = ts.shared_prefix_attention(Q, pK[:, :0], pV[:, :0], K[:, :, :0], V[:, :, :0])
    assert (none == 0).all()


def test_matches_cross_attention(hip_backend):
    """With one token and no prefix it is cross_attention over the caches."""
    Q, pK, pV, K, V = make(4, 8, 2, 1, 5, 500, 128, F32, seed=3)
    lengths = torch.tensor([1, 100, 499, 500], device="cuda")
    a = ts.shared_prefix_attention(Q, pK[:, :0], pV[:, :0], K, V, lengths)
    torch.testing.assert_close(a, ts.cross_attention(Q, K, V, lengths), rtol=1e-5, atol=1e-6)


def test_views_and_slices_of_a_cache(hip_backend):
    """The prefix as a slice of longer buffers, caches in (batch, row, head) order."""
    Q, pK, pV, K, V = make(3, 4, 2, 2, 200, 64, 64, BF, seed=4)
    want = ts.shared_prefix_attention(Q, pK, pV, K, V)
    turn = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    long = lambda t: torch.cat([t, t.new_full((2, 50, 64), float("nan"))], 1)[:, :200]  # noqa: E731
    assert torch.equal(ts.shared_prefix_attention(Q, long(pK), long(pV), turn(K), turn(V)), want)
    assert torch.equal(ts.shared_prefix_attention(Q, turn(pK[None])[0], pV, K, V), want)


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("size", [(64, 16, 8, 1, 2100, 500, 128), (24, 32, 4, 5, 3001, 300, 80), (33, 12, 3, 40, 700, 400, 64)])
def test_full_grids(hip_backend, size, dt):
    """A prefix in wide workgroups, in several ranges, next to many sequences."""
    check(*make(*size, dt))
