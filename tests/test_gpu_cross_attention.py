"""GPU parity of cross_attention against the float64 oracle.

Bounds, elementwise against A = P |V| (oracle/layer.py), u = eps / 2 of the
operands' type and e = 2^-24: P is rounded to the type before its product with
V (u A; not in fp32) and the result once (u |O| <= u A). In fp32, a score of D
products differs by at most (D + 4) e smax, entering P twice (itself and its
sum): 2 (D + 4) e smax A; the sums over L keys, the exponentials and the
joining of key ranges add at most (2 L + 64) e A.
"""

from __future__ import annotations

import pytest
import torch

import trnsparse_amd as ts
from oracle import layer
from trnsparse_amd.hip import _lib

pytestmark = pytest.mark.gpu

E = 2.0**-24
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def tol(dt, D, L, smax):
    u = torch.finfo(dt).eps / 2
    return (2 * u if dt != F32 else u) + E * (2 * (D + 4) * smax + 2 * L + 64)


def make(B, H, Hk, N, L, D, dt, seed=0, strided=True):
    """Heads as views of projections' outputs, K and V of one."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    if not strided:
        return tuple(torch.randn(B, h, n, D, device="cuda", generator=g).to(dt) for h, n in ((H, N), (Hk, L), (Hk, L)))
    Q = torch.randn(B, N, H, D, device="cuda", generator=g).to(dt).transpose(1, 2)
    kv = torch.randn(B, L, 2, Hk, D, device="cuda", generator=g).to(dt)
    return Q, kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)


def check_forward(Q, K, V, lengths=None, scale=None):
    B, H, N, D = Q.shape
    L = K.shape[2]
    O = ts.cross_attention(Q, K, V, lengths, scale)
    torch.cuda.synchronize()
    assert O.shape == Q.shape and O.dtype == Q.dtype and O.device == Q.device
    seen = None if lengths is None else layer.lengths_seen(lengths, N, L)
    r = layer.attention(Q, K, V, scale or D**-0.5, seen)
    far = (O.double().cpu() - r["O"]).abs() - tol(Q.dtype, D, L, r["smax"]) * r["A"]
    assert not O.isnan().any() and far.max() <= 1e-30, float(far.max())
    return O, r


# (batch, heads, kv_heads, queries, keys, head_dim): single tokens, few and
# many rows, whole and broken tiles and key ranges, every head_dim class
SIZES = [
    (1, 1, 1, 1, 1, 64), (2, 4, 4, 1, 37, 64), (3, 8, 2, 1, 1500, 128), (1, 2, 1, 1, 6000, 128), (2, 6, 2, 5, 130, 40),
    (1, 8, 1, 4, 32, 128), (1, 4, 2, 17, 33, 96), (2, 4, 4, 33, 64, 64), (1, 3, 3, 128, 128, 128),
    (2, 2, 1, 129, 257, 128), (1, 6, 3, 70, 1000, 80), (1, 2, 2, 300, 511, 16), (1, 1, 1, 257, 3000, 8),
    (2, 16, 4, 64, 100, 120), (1, 2, 2, 1, 300, 100), (1, 2, 2, 40, 90, 7),
]


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("size", SIZES)
def test_sizes(hip_backend, size, dt):
    check_forward(*make(*size, dt))


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("N,heads", [(1, (8, 2)), (50, (2, 2)), (140, (4, 2))])
@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_lengths(hip_backend, dt, N, heads, itype):
    """Padded batches: lengths of 0, 1, a tile's edge, all, and outside [0, keys];
    rows behind the length hold infinities and NaN."""
    L = 700
    lengths = torch.tensor([0, 1, 32, 64, 127, 700, 9999, -3], dtype=itype, device="cuda")
    Q, K, V = make(8, *heads, N, L, 64, dt, seed=1)
    K, V = K.clone(), V.clone()
    for b, n in enumerate(lengths.clamp(0, L).tolist()):
        K[b, :, n:], V[b, :, n:] = float("nan"), float("inf")
    O, _ = check_forward(Q, K, V, lengths)
    assert (O[0] == 0).all() and (O[7] == 0).all()


@pytest.mark.parametrize("dt", [BF, HF, F32])
def test_no_keys_and_no_queries(hip_backend, dt):
    Q, K, V = make(2, 4, 2, 5, 0, 64, dt, strided=False)
    assert (ts.cross_attention(Q, K, V) == 0).all()
    Q, K, V = make(2, 4, 2, 0, 9, 64, dt, strided=False)
    assert ts.cross_attention(Q, K, V).shape == (2, 4, 0, 64)
    Q, K, V = make(0, 4, 2, 3, 9, 64, dt, strided=False)
    assert ts.cross_attention(Q, K, V).shape == (0, 4, 3, 64)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("N", [1, 200])
def test_large_scores(hip_backend, dt, N):
    """Scores that rise along the keys by hundreds: the running maximum moves
    at every stage, and a late key takes all of the weight."""
    Q, K, V = make(1, 2, 2, N, 900, 64, dt, seed=2)
    K = K * (1 + torch.arange(900, device="cuda").view(1, 1, -1, 1) / 20).to(dt)
    check_forward(Q, K.to(dt), V, scale=1.0)


def test_infinite_scores(hip_backend):
    """A key of +inf score makes its row NaN as in the definition, other rows
    stay; a key of -inf score has no weight."""
    Q, K, V = make(1, 1, 1, 3, 80, 64, F32, seed=3, strided=False)
    Q[0, 0, :, 0], Q[0, 0, 1, 0] = 1.0, -1.0
    K[0, 0, 70, 0] = float("inf")
    O = ts.cross_attention(Q, K, V)
    assert O[0, 0, 0].isnan().all() and O[0, 0, 2].isnan().all()
    keep = torch.arange(80, device="cuda") != 70
    r = layer.attention(Q[:, :, 1:2], K[:, :, keep], V[:, :, keep], 64**-0.5)
    assert (O[:, :, 1:2].double().cpu() - r["O"]).abs().max() <= 1e-5


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("N", [1, 150])
def test_views(hip_backend, dt, N):
    """Orders, offsets and strides: the result does not depend on them."""
    B, H, Hk, L, D = 2, 4, 2, 130, 64
    Q, K, V = make(B, H, Hk, N, L, D, dt, seed=4, strided=False)
    want = ts.cross_attention(Q, K, V)

    def odd(t):  # unaligned: one element into a wider buffer
        b = torch.zeros(*t.shape[:3], D + 3, dtype=dt, device="cuda")
        b[..., 1 : D + 1] = t
        return b[..., 1 : D + 1]

    def turned(t):  # rows outermost
        return t.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)

    def column(t):  # head_dim not innermost
        return t.transpose(2, 3).contiguous().transpose(2, 3)

    for f in (odd, turned, column):
        assert torch.equal(ts.cross_attention(f(Q), f(K), f(V)), want), f.__name__
    one = K[:1].expand(B, -1, -1, -1)  # one encoder's states for the batch
    same = ts.cross_attention(Q, one.contiguous(), V)
    assert torch.equal(ts.cross_attention(Q, one, V), same)
    row = V[:, :, :1].expand(-1, -1, L, -1)  # a stride of zero over rows
    assert torch.equal(ts.cross_attention(Q, K, row), ts.cross_attention(Q, K, row.contiguous()))


def test_far_offsets(hip_backend):
    """Keys whose byte offsets pass 2^32 in a batch entry of its own."""
    L, D, width = 70000, 64, 1 << 15  # 64 KiB between rows: 4.6 GB
    buf = torch.zeros(L, width, dtype=BF, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(5)
    K = buf[:, :D].view(1, 1, L, D)
    V = buf[:, D : 2 * D].view(1, 1, L, D)
    K[0, 0, -300:] = torch.randn(300, D, device="cuda", generator=g).to(BF)
    V[0, 0, -300:] = torch.randn(300, D, device="cuda", generator=g).to(BF)
    for N in (1, 40):
        Q = 4 * torch.randn(1, 1, N, D, device="cuda", generator=g).to(BF)
        check_forward(Q, K, V)
        near = ts.cross_attention(Q, K.contiguous(), V.contiguous())
        assert torch.equal(ts.cross_attention(Q, K, V), near)


def test_lse(hip_backend):
    """The operator's log-sum-exp, natural, -inf for a row without keys."""
    for N, L in ((1, 900), (150, 333)):
        Q, K, V = make(2, 4, 2, N, L, 64, F32, seed=6)
        lens = torch.tensor([L // 2, 0], device="cuda")
        _, lse = _lib.ops().cross_attn_fwd(Q, K, V, lens, 0.125, True)
        r = layer.attention(Q, K, V, 0.125, layer.lengths_seen(lens, N, L))
        assert (lse[1] == -float("inf")).all()
        # a score's error, the sum's and the rounding of the result
        bound = E * ((64 + 4) * r["smax"] + 2 * L + 64 + 4 * r["lse"][0].abs().max())
        assert (lse[0].double().cpu() - r["lse"][0]).abs().max() <= bound


def test_repeats_are_equal(hip_backend):
    Q, K, V = make(3, 8, 2, 1, 2000, 128, BF, seed=7)
    one = ts.cross_attention(Q, K, V)
    for _ in range(3):
        assert torch.equal(ts.cross_attention(Q, K, V), one)


def test_host_operands(hip_backend):
    Q, K, V = make(1, 2, 2, 9, 50, 64, F32, seed=8)
    want = ts.cross_attention(Q, K, V)
    got = ts.cross_attention(Q.cpu(), K.cpu(), V.cpu(), torch.tensor([50]))
    assert got.device.type == "cpu" and torch.equal(got, want.cpu())


def test_other_stream(hip_backend):
    s = torch.cuda.Stream()
    Q, K, V = make(2, 8, 2, 1, 1500, 128, BF, seed=9)
    want = ts.cross_attention(Q, K, V)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ts.cross_attention(Q, K, V)
    s.synchronize()
    assert torch.equal(got, want)


def test_float64_is_refused(hip_backend):
    Q, K, V = (t.double() for t in make(1, 2, 2, 3, 4, 64, F32))
    with pytest.raises(RuntimeError, match="not supported"):
        ts.cross_attention(Q, K, V)


# More workgroups than CUs, of four wavefronts each in 16 bits too; more narrow
# ones than fit at once; units that do not divide over the XCDs.
FULL = [(3, 32, 32, 300, 100, 64), (2, 40, 8, 700, 333, 128), (5, 21, 21, 290, 70, 90), (70, 24, 8, 2, 150, 128)]


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("size", FULL)
def test_full_grids(hip_backend, size, dt):
    check_forward(*make(*size, dt, seed=20))


@pytest.mark.parametrize("dt", [BF, F32])
def test_full_grid_with_lengths(hip_backend, dt):
    L = 300
    lengths = torch.tensor([0, 1, 63, 64, 299, 400], device="cuda")
    Q, K, V = make(6, 16, 16, 400, L, 64, dt, seed=21)
    K, V = K.clone(), V.clone()
    for b, n in enumerate(lengths.clamp(0, L).tolist()):
        K[b, :, n:], V[b, :, n:] = float("nan"), float("inf")
    O, _ = check_forward(Q, K, V, lengths)
    assert (O[0] == 0).all()
