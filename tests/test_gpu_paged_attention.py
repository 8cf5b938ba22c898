"""GPU parity of paged_attention against the float64 oracle.

Results: the bounds of test_gpu_cross_attention (`tol`). Accumulated weights, e =
2^-24, R rows (query heads of a key head times new tokens): every weight is
2^(s - lse) of scores within (D + 4) e smax and a log-sum-exp of such scores and a
sum over L keys; s and lse, at most smax + ln L in size, are scaled and rounded a
few times (8 e each, the exponential's argument); the exponentials, logarithms and
the joining of key ranges add 64 e; the sum over R rows and the addition to what
was there R + 2 roundings.
"""

from __future__ import annotations

import math

import pytest
import torch

import trnsparse_amd as ts
from oracle import layer
from test_gpu_cross_attention import BF, E, F32, HF, tol

pytestmark = pytest.mark.gpu


def wtol(D, L, R, smax):
    return E * (2 * (D + 4) * smax + 8 * (smax + math.log(max(L, 1))) + L + R + 66)


def make(B, H, Hk, N, cols, size, D, dt, seed=0, extra=3):
    """Q as heads of a projection, scattered pages, more of them than the table names."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dt)  # noqa: E731
    table = torch.randperm(B * cols + extra, device="cuda", generator=g)[: B * cols].view(B, cols).int()
    return r(B, N, H, D).transpose(1, 2), r(B * cols + extra, Hk, size, D), r(B * cols + extra, Hk, size, D), table


def check(Q, kp, vp, table, lengths, new=None, weights=True, scale=None):
    B, H, N, D = Q.shape
    Hk, L = kp.shape[1], table.shape[1] * kp.shape[2]
    w = torch.rand(B, Hk, L, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9)) if weights else None
    before = w.clone() if weights else None
    O = ts.paged_attention(Q, kp, vp, table, lengths, new, scale, w)
    torch.cuda.synchronize()
    assert O.shape == Q.shape and O.dtype == Q.dtype
    r = layer.attention(Q, layer.paged_rows(kp, table), layer.paged_rows(vp, table), scale or D**-0.5,
                        layer.chunk_seen(lengths, new, N, L))
    far = (O.double().cpu() - r["O"]).abs() - tol(Q.dtype, D, L, r["smax"]) * r["A"]
    assert not O.isnan().any() and (O.numel() == 0 or far.max() <= 1e-30), float(far.max())
    if weights:
        assert torch.equal(ts.paged_attention(Q, kp, vp, table, lengths, new, scale), O)  # the same without them
        off = (w.double() - before.double()).cpu() - r["W"]
        far = off.abs() - wtol(D, L, H // Hk * N, r["smax"]) * r["W"] - E * (before.double().cpu() + r["W"])
        assert L == 0 or far.max() <= 1e-30, float(far.max())
        for b, n in enumerate(lengths.clamp(0, L).tolist()):
            assert torch.equal(w[b, :, n:], before[b, :, n:])
    return O


# (batch, heads, kv_heads, queries, columns, page_size, head_dim)
SIZES = [
    (1, 1, 1, 1, 1, 16, 64), (4, 4, 4, 1, 9, 16, 64), (3, 8, 2, 1, 12, 64, 128), (2, 6, 2, 5, 5, 48, 40),
    (1, 8, 1, 4, 2, 256, 128), (2, 12, 4, 3, 40, 16, 96), (2, 4, 2, 17, 6, 32, 80), (1, 3, 3, 33, 7, 16, 64),
    (2, 8, 2, 40, 8, 32, 128), (1, 9, 3, 70, 3, 112, 120), (3, 4, 1, 129, 10, 16, 16), (1, 2, 2, 300, 20, 16, 128),
]


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("size", SIZES)
def test_sizes(hip_backend, size, dt):
    Q, kp, vp, table = make(*size, dt)
    L = size[4] * size[5]
    g = torch.Generator().manual_seed(1)
    check(Q, kp, vp, table, torch.randint(min(size[3], L), L + 1, (size[0],), generator=g).cuda())


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("N,heads", [(1, (8, 2)), (4, (4, 4)), (50, (4, 2)), (140, (2, 2))])
@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_lengths(hip_backend, dt, N, heads, itype):
    """Caches of 0 rows, 1, fewer than the new tokens, a tile's edge, all, outside
    [0, slots]; new tokens none, one, some, all, outside; what stands behind is NaN
    and infinite, in pages of the table and of nobody."""
    size, cols = 16, 20
    L = size * cols
    lengths = torch.tensor([0, 1, 3, 32, 129, L, 9999, -1, 64, 200], dtype=itype, device="cuda")
    new = torch.tensor([N, 1, N, 1, N, N, 9999, 3, 0, -7], dtype=itype, device="cuda")
    Q, kp, vp, table = make(10, *heads, N, cols, size, 64, dt, seed=1)
    table = table.to(itype)
    for b, n in enumerate(lengths.clamp(0, L).tolist()):
        for c in range(cols):
            at = max(0, min(size, n - c * size))
            kp[table[b, c], :, at:], vp[table[b, c], :, at:] = float("inf"), float("nan")
    named = torch.zeros(len(kp), dtype=torch.bool, device="cuda")
    named[table.view(-1).long()] = True
    kp[~named], vp[~named] = float("nan"), float("inf")
    Q[:, :, N - 1] = torch.where((new >= N).view(-1, 1, 1), Q[:, :, N - 1], float("nan"))  # behind the new tokens
    O = check(Q, kp, vp, table, lengths, new)
    assert (O[0] == 0).all() and (O[7] == 0).all() and (O[8] == 0).all() and (O[9] == 0).all()
    full = torch.where(lengths > 0, lengths, 0)
    Q = torch.nan_to_num(Q, nan=0.5)
    check(Q, kp, vp, table, full)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("N", [1, 3, 60])
def test_bad_pages(hip_backend, dt, N):
    """Table entries outside [0, pages) are pages of zeros, in either index type."""
    Q, kp, vp, table = make(4, 4, 2, N, 8, 32, 64, dt, seed=2)
    table = table.long()
    table[0, 2], table[1, 0], table[1, 7], table[2] = -1, len(kp), -(2**31), 2**31 - 1
    lengths = torch.tensor([200, 256, 100, 3], device="cuda")
    O = check(Q, kp, vp, table, lengths)
    assert (O[2] == 0).all()
    assert torch.equal(ts.paged_attention(Q, kp, vp, table.int(), lengths), O)
    far = table.clone()
    far[0, 2], far[1, 0] = 2**40 + 1, -(2**40) + 1  # in range in their low halves alone
    assert torch.equal(ts.paged_attention(Q, kp, vp, far, lengths), O)
    none = ts.paged_attention(Q, kp[:0], vp[:0], table, lengths)
    assert (none == 0).all()
    assert (ts.paged_attention(Q, kp, vp, table[:, :0], lengths) == 0).all()


@pytest.mark.parametrize("N", [1, 40])
def test_empty(hip_backend, N):
    Q, kp, vp, table = make(3, 4, 2, N, 2, 16, 64, BF)
    lengths = torch.tensor([5, 3, 1], device="cuda")
    assert ts.paged_attention(Q[:0], kp, vp, table[:0], lengths[:0]).shape == (0, 4, N, 64)
    assert ts.paged_attention(Q[:, :, :0], kp, vp, table, lengths).shape == (3, 4, 0, 64)
    w = torch.ones(3, 2, 0, device="cuda")
    assert (ts.paged_attention(Q, kp, vp, table[:, :0], lengths, None, None, w) == 0).all()


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("N", [1, 36])
def test_views(hip_backend, dt, N):
    """Pages in (page, row, head) order, K and V interleaved, a slice of a wider
    table, weights as a slice, Q in another order of heads."""
    Q, kp, vp, table = make(3, 8, 2, N, 5, 32, 64, dt, seed=4)
    lengths = torch.tensor([160, 37, 90], device="cuda")
    w = torch.zeros(3, 2, 160, device="cuda")
    want = ts.paged_attention(Q, kp, vp, table, lengths, weights=w)
    turn = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    both = torch.stack([kp, vp], 1)
    wide = torch.cat([table, torch.full_like(table, -1)], 1)
    w2 = torch.zeros(4, 3, 200, device="cuda")
    sl = w2[:3, 1:, 7:167]
    for k, v, t in ((turn(kp), vp, table), (turn(kp), turn(vp), wide[:, :5]), (both[:, 0], both[:, 1], table)):
        assert torch.equal(ts.paged_attention(Q, k, v, t, lengths), want)
    assert torch.equal(ts.paged_attention(turn(Q), kp, vp, table, lengths, weights=sl), want)
    assert torch.equal(sl, w) and w2.count_nonzero() == sl.count_nonzero()  # nothing written around the slice
    odd = torch.zeros(3, 8, N, 67, dtype=dt, device="cuda")[..., 1:65]  # not whole pieces: copied
    odd.copy_(Q)
    assert torch.equal(ts.paged_attention(odd, kp, vp, table, lengths), want)
    assert torch.equal(ts.paged_attention(Q, kp, vp, table.t().contiguous().t(), lengths), want)  # columns not in a row


def test_equals_shared_prefix_attention(hip_backend):
    """Over the same rows it is shared_prefix_attention without a prefix."""
    Q, kp, vp, table = make(4, 8, 2, 3, 16, 32, 128, F32, seed=3)
    lengths = torch.tensor([3, 100, 499, 512], device="cuda")
    K, V = (layer.paged_rows(p, table).cuda() for p in (kp, vp))
    none = K[0, :, :0]
    want = ts.shared_prefix_attention(Q, none, none, K, V, lengths)
    torch.testing.assert_close(ts.paged_attention(Q, kp, vp, table, lengths), want, rtol=1e-5, atol=1e-6)


def test_pages_shared_by_sequences(hip_backend):
    """A common beginning in pages that several tables name; weights are each
    sequence's own."""
    Q, kp, vp, table = make(3, 4, 2, 1, 6, 16, 64, BF, seed=5)
    table[1, :3], table[2, :3] = table[0, :3], table[0, :3]
    check(Q, kp, vp, table, torch.tensor([50, 70, 96], device="cuda"))


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("size", [
    (2, 8, 4, 1, 400, 16, 128),   # keys in ranges, few rows
    (1, 16, 2, 4, 70, 64, 128),   # ranges, full rows of a wavefront
    (2, 4, 2, 90, 60, 32, 64),    # ranges of whole tiles
    (40, 4, 4, 1, 12, 16, 64),    # many sequences
])
def test_ranges(hip_backend, size, dt):
    """Keys in ranges that are joined; lengths far below what the table has room for."""
    Q, kp, vp, table = make(*size, dt, seed=6)
    B, N, L = size[0], size[3], size[4] * size[5]
    check(Q, kp, vp, table, torch.full((B,), L, device="cuda"))
    lengths = torch.arange(B, device="cuda") * 37 + N
    check(Q, kp, vp, table, lengths)


@pytest.mark.parametrize("dt", [BF, F32])
def test_mixed_batch(hip_backend, dt):
    """Chunks of a prompt next to single tokens, in tables that allow for many more rows."""
    Q, kp, vp, table = make(9, 8, 2, 150, 90, 16, 64, dt, seed=7)
    new = torch.tensor([1, 150, 1, 9, 0, 40, 1, 149, 1], device="cuda")
    lengths = torch.tensor([1440, 1440, 1, 600, 600, 40, 900, 149, 33], device="cuda")
    check(Q, kp, vp, table, lengths, new)
    check(Q[:2], kp, vp, table[:2], lengths[:2], new[:2])  # few sequences: ranges of both kinds


@pytest.mark.parametrize("dt", [BF, HF, F32])
def test_large_scores_and_one_that_outweighs(hip_backend, dt):
    """Scores far apart: one key takes nearly all of the weight, the others add up."""
    Q, kp, vp, table = make(2, 4, 2, 3, 20, 32, 64, dt, seed=8)
    lengths = torch.tensor([640, 333], device="cuda")
    kp[table[0, 0], :, 0] = Q[0, ::2, 0] * 2
    kp[table[1, 3], :, 5] = -Q[1, ::2, 2] * 2
    check(Q, kp, vp, table, lengths, scale=0.5)


def test_far_pages(hip_backend):
    """Pages whose bytes lie past 2^32 from the pool's start."""
    pages, Hk, size, D = 70000, 4, 64, 128  # 4.6 GB each
    g = torch.Generator(device="cuda").manual_seed(9)
    kp = torch.zeros(pages, Hk, size, D, dtype=BF, device="cuda")
    vp = torch.zeros(pages, Hk, size, D, dtype=BF, device="cuda")
    table = torch.tensor([[69999, 0, 65536, 3], [1, 69998, 65535, 40000]], device="cuda")
    for p in table.view(-1).tolist():
        kp[p], vp[p] = (torch.randn(Hk, size, D, device="cuda", generator=g).to(BF) for _ in range(2))
    lengths = torch.tensor([256, 201], device="cuda")
    small = torch.arange(8, device="cuda").view(2, 4)
    ks, vs = kp[table.view(-1)], vp[table.view(-1)]
    for N in (1, 40):
        Q = torch.randn(2, 8, N, D, device="cuda", generator=g).to(BF)
        a, b = torch.zeros(2, Hk, 256, device="cuda"), torch.zeros(2, Hk, 256, device="cuda")
        assert torch.equal(ts.paged_attention(Q, kp, vp, table, lengths, weights=a),
                           ts.paged_attention(Q, ks, vs, small, lengths, weights=b))
        assert torch.equal(a, b) and float(a.sum()) > 0
    w = torch.rand(2, Hk, 256, device="cuda", generator=g)
    w2 = w.clone()
    K = torch.randn(2, Hk, 9, D, device="cuda", generator=g).to(BF)
    for k, v, t, x in ((kp, vp, table, w), (ks, vs, small, w2)):
        n = ts.paged_cache_append(K, K * 2, k, v, t, lengths - 20)
        ts.paged_cache_evict(k, v, x, t, n, 100, 30)
    assert torch.equal(w, w2) and torch.equal(kp[table.view(-1)], ks) and torch.equal(vp[table.view(-1)], vs)


def test_repeated_calls_are_equal(hip_backend):
    """No order of summation depends on timing."""
    Q, kp, vp, table = make(3, 8, 2, 45, 60, 32, 128, BF, seed=10)
    lengths, new = torch.tensor([1900, 1000, 300], device="cuda"), torch.tensor([45, 1, 30], device="cuda")
    outs = []
    for _ in range(4):
        w = torch.zeros(3, 2, 1920, device="cuda")
        outs.append((ts.paged_attention(Q, kp, vp, table, lengths, new, weights=w), w))
    assert all(torch.equal(o, outs[0][0]) and torch.equal(w, outs[0][1]) for o, w in outs)


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("R", [(8, 4), (8, 5), (4, 16), (3, 21), (13, 5)])  # 32, 40, 64, 63, 65 rows of a key head
def test_rows_around_a_tile(hip_backend, dt, R):
    """Units of one and two tiles of 32 rows, alone and next to others in one launch."""
    G, N = R
    Q, kp, vp, table = make(6, 2 * G, 2, N, 50, 16, 128, dt, seed=11)
    lengths = torch.tensor([800, 64, 5, 333, N, 799], device="cuda")
    check(Q, kp, vp, table, lengths)
    check(Q, kp, vp, table, lengths, torch.tensor([N, N, 3, 1, N - 1, 0], device="cuda"))
    Q, kp, vp, table = make(6, 2 * G, 2, N + 70, 50, 16, 128, dt, seed=12)
    check(Q, kp, vp, table, lengths.clamp_min(90), torch.tensor([N, N + 70, N, 1, N - 1, 0], device="cuda"))


@pytest.mark.parametrize("dt", [BF, F32])
def test_a_chunk_of_one_tile_next_to_few_rows(hip_backend, dt):
    """One tile of 128 rows at most, of which some sequences have two narrow ones."""
    Q, kp, vp, table = make(3, 4, 1, 20, 3, 16, 64, dt, seed=13)
    check(Q, kp, vp, table, torch.tensor([48, 20, 30], device="cuda"), torch.tensor([12, 20, 9], device="cuda"))
    Q, kp, vp, table = make(70, 4, 1, 20, 3, 16, 64, dt, seed=14)  # more than 64 sequences
    new = torch.arange(70, device="cuda") % 21
    check(Q, kp, vp, table, (new + torch.arange(70, device="cuda") % 29).clamp_max(48), new)


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("heads,N,cols", [((4, 2), 3, 4), ((8, 2), 6, 4), ((8, 2), 6, 400), ((2, 2), 50, 10), ((16, 16), 140, 40)])
@pytest.mark.parametrize("mixed", [False, True])
def test_rows_of_scores_that_are_all_minus_infinity(hip_backend, dt, heads, N, cols, mixed):
    """Their result is zero, and they weigh nothing; the rows beside them as ever."""
    Q, kp, vp, table = make(3, *heads, N, cols, 16, 64, dt, seed=4)
    L = 16 * cols
    kp = kp.abs() + 0.125
    lengths = torch.tensor([L, L - 5, N], device="cuda")
    new = torch.tensor([N, max(N - 20, 1), 1], device="cuda") if mixed else None
    clean = Q.clone()
    clean[:, 1, 1::2] = 0
    Q[:, 1, 1::2] = float("-inf")
    gone = torch.zeros(3, heads[0], N, 1, dtype=torch.bool, device="cuda")
    gone[:, 1, 1::2] = True
    w = torch.zeros(3, heads[1], L, device="cuda")
    O = ts.paged_attention(Q, kp, vp, table, lengths, new, None, w)
    assert not (O * gone).any() and not w.isnan().any()
    # the rows of equal scores that stand in their places weigh 1 / (keys seen) each
    whole = ts.paged_attention(clean, kp, vp, table, lengths, new, None, torch.zeros_like(w))
    assert torch.equal(O.masked_fill(gone, 0), whole.masked_fill(gone, 0))
    seen = layer.chunk_seen(lengths.cpu(), None if new is None else new.cpu(), N, L)
    each = (seen[:, 1::2].double() / seen[:, 1::2].sum(-1, keepdim=True).clamp(min=1)).sum(1)
    r = layer.attention(clean, layer.paged_rows(kp, table), layer.paged_rows(vp, table), 64**-0.5, seen)
    r["W"][:, 1 // (heads[0] // heads[1])] -= each  # head 1's key head
    far = (w.double().cpu() - r["W"]).abs() - wtol(64, L, heads[0] // heads[1] * N, r["smax"]) * r["W"]
    assert far.max() <= 1e-15, float(far.max())


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("size", [(1, 8, 1, 300, 20, 16, 64), (2, 4, 1, 1100, 72, 16, 128), (3, 16, 2, 513, 9, 64, 40), (1, 7, 1, 900, 57, 16, 80)])
@pytest.mark.parametrize("mixed", [False, True])
def test_weights_of_many_rows_and_few_keys(hip_backend, size, dt, mixed):
    """The rows of a key head in parts, next to sequences of none, one and few rows."""
    Q, kp, vp, table = make(*size, dt, seed=6)
    B, N, L = size[0], size[3], size[4] * size[5]
    lengths = torch.tensor([L, N - 7, L - 33], device="cuda")[:B]
    new = torch.tensor([N - 5, 1, 0] if B < 3 else [1, N - 3, 0], device="cuda")[:B] if mixed else None
    check(Q, kp, vp, table, lengths, new)


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("size", [(4, 8, 1, 200, 80, 16, 64), (9, 4, 2, 130, 24, 64, 128), (33, 2, 1, 80, 40, 48, 40), (2, 12, 3, 70, 20, 128, 96)])
def test_one_chunk_of_few_key_heads(hip_backend, size, dt):
    """Its keys in as many ranges as fill the CUs; with several chunks, in fewer or none."""
    Q, kp, vp, table = make(*size, dt, seed=7)
    B, N, L = size[0], size[3], size[4] * size[5]
    g = torch.Generator().manual_seed(8)
    lengths = torch.randint(N, L + 1, (B,), generator=g).cuda()
    lengths[B - 1] = L
    for chunks in (1, (B + 1) // 2, B):
        new = torch.ones(B, dtype=torch.int64, device="cuda")
        new[B - chunks :] = N - torch.arange(chunks, device="cuda")
        check(Q, kp, vp, table, lengths, new)
        assert torch.equal(ts.paged_attention(Q, kp, vp, table, lengths, new), ts.paged_attention(Q, kp, vp, table, lengths, new))


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("B", [63, 64, 65, 130])
@pytest.mark.parametrize("heads,N", [((4, 1), 70), ((6, 3), 12)])
def test_batches_of_many_sequences(hip_backend, dt, B, heads, N):
    """Chunks next to single tokens and to sequences of none, over caches in several ranges, on
    both sides of the 64 sequences that a wavefront deals out (one to a lane)."""
    Q, kp, vp, table = make(B, *heads, N, 70, 16, 64, dt, seed=15)
    g = torch.Generator().manual_seed(16)
    new = torch.ones(B, dtype=torch.int64)
    new[::9], new[5::17], new[B - 1] = N, 0, N - 1
    lengths = torch.randint(N, 1121, (B,), generator=g)
    lengths[::9], lengths[3] = 1120 - torch.arange(len(lengths[::9])), 0
    check(Q, kp, vp, table, lengths.cuda(), new.cuda())


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("G", [63, 64, 65, 96])
@pytest.mark.parametrize("size", [(2, 1, 1, 7, 16, 64), (3, 2, 3, 9, 48, 40), (8, 1, 2, 64, 128, 64)])
def test_weights_of_many_heads_to_a_key_head(hip_backend, dt, G, size):
    """A token's rows fill whole stages of the weights' rows, or more; 32 keys to a workgroup
    and (the last size) 128."""
    B, Hk, N, cols, ps, D = size
    Q, kp, vp, table = make(B, G * Hk, Hk, N, cols, ps, D, dt, seed=17)
    L = cols * ps
    lengths = torch.tensor([L, N, L - 31, L // 2, 0, L - 1, 77, 1][:B], device="cuda")
    check(Q, kp, vp, table, lengths)
    check(Q, kp, vp, table, lengths, torch.tensor([1, N, N, 0, 1, N, 1, N][:B], device="cuda"))


@pytest.mark.parametrize("dt,D", [(BF, 8), (HF, 24), (F32, 4), (F32, 12)])
@pytest.mark.parametrize("N,heads", [(1, (4, 2)), (5, (8, 2)), (50, (6, 3))])
def test_smallest_head_dims(hip_backend, dt, D, N, heads):
    """A row of one 16-byte piece, and of three."""
    Q, kp, vp, table = make(3, *heads, N, 9, 32, D, dt, seed=18)
    lengths = torch.tensor([288, 51, N], device="cuda")
    check(Q, kp, vp, table, lengths)
    check(Q, kp, vp, table, lengths, torch.tensor([1, N, max(N - 2, 0)], device="cuda"))


@pytest.mark.parametrize("N", [1, 40])
def test_one_pool_for_both_and_one_page_for_all(hip_backend, N):
    """Pages are only read here: K and V may be one tensor, and pages a view of stride zero."""
    Q, kp, vp, table = make(3, 4, 2, N, 5, 32, 64, BF, seed=19)
    lengths = torch.tensor([160, 40, 99], device="cuda")
    check(Q, kp, kp, table, lengths)
    one = kp[3:4].expand(len(kp), -1, -1, -1)
    want = check(Q, one, vp, table, lengths)
    assert torch.equal(ts.paged_attention(Q, one.contiguous(), vp, table, lengths), want)
    same = table[:1].expand(3, -1)  # one row of the table for all sequences
    check(Q, kp, vp, same, lengths)
