"""GPU parity of paged_cache_append and paged_cache_evict: every value is a copy
of one that was there, so results are equal to the oracle's bit for bit."""

from __future__ import annotations

import pytest
import torch

import trnsparse_amd as ts
from oracle import layer
from test_gpu_paged_attention import BF, F32, HF, make

pytestmark = pytest.mark.gpu


def same(got, want):
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        torch.testing.assert_close(a.cpu(), b.cpu(), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("size", [(1, 1, 1, 1, 16, 64), (5, 3, 7, 6, 48, 40), (3, 8, 40, 9, 16, 128), (2, 2, 300, 3, 128, 8)])
@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_append(hip_backend, size, dt, itype):
    B, Hk, N, cols, ps, D = size
    K, kp, vp, table = make(B, Hk, Hk, N, cols, ps, D, dt)
    V = torch.randn_like(K)
    L = cols * ps
    table[B - 1, cols - 1] = -1  # a page that is not there
    for lengths in ([0, 1, ps - 1, L, L - 1], [L // 2, -9, L + 9, ps, 0]):
        lengths = torch.tensor(lengths[:B], dtype=itype, device="cuda")
        for new in (None, torch.tensor([N, 0, 1, -1, 9999][:B], dtype=itype, device="cuda")):
            w = torch.rand(B, Hk, L, device="cuda")
            want = layer.paged_append(K, V, kp, vp, table, lengths, new, w)
            after = ts.paged_cache_append(K, V, kp, vp, table, lengths, new, w)
            assert after.dtype == itype
            same((kp, vp, w, after), want)
            ts.paged_cache_append(V, K, kp, vp, table, lengths, new)  # without weights, other values
            same((w,), (want[2],))


def test_append_views(hip_backend):
    """New rows that are not whole pieces apart; pages in (page, row, head) order;
    mixed index types."""
    K, kp, vp, table = make(3, 2, 2, 5, 4, 16, 64, BF)
    odd = torch.zeros(3, 2, 5, 67, dtype=BF, device="cuda")[..., 1:65]
    odd.copy_(K)
    lengths, new = torch.tensor([0, 14, 60], device="cuda"), torch.tensor([5, 2, 5], dtype=torch.int32, device="cuda")
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (kp, vp)]
    want = layer.paged_append(K, K, kp, vp, table, lengths, new)
    after = ts.paged_cache_append(odd, odd, *turned, table, lengths, new)
    same((*turned, after), (want[0], want[1], want[3]))
    with pytest.raises(RuntimeError):  # written rows on top of each other
        ts.paged_cache_append(K, K, kp[:1].expand(9, -1, -1, -1), vp[:1].expand(9, -1, -1, -1), table, lengths)
    with pytest.raises(RuntimeError):
        ts.paged_cache_append(K, K, kp[..., 1:], vp[..., 1:], table, lengths)


# (batch, kv_heads, columns, page_size, head_dim, budget, recent)
EVICT = [
    (1, 1, 1, 16, 64, 1, 0), (4, 2, 8, 16, 64, 40, 9), (3, 3, 5, 48, 80, 100, 100), (2, 8, 12, 64, 128, 333, 41),
    (5, 2, 40, 16, 40, 77, 0), (2, 1, 9, 256, 16, 2000, 300), (2, 2, 600, 16, 8, 4000, 17), (3, 2, 4, 16, 128, 63, 3),
]


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("size", EVICT)
@pytest.mark.parametrize("kind", ["random", "ties", "equal"])
def test_evict(hip_backend, size, dt, kind):
    B, Hk, cols, ps, D, budget, recent = size
    _, kp, vp, table = make(B, Hk, Hk, 1, cols, ps, D, dt)
    L = cols * ps
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn(B, Hk, L, device="cuda", generator=g)
    w = {"random": w.exp(), "ties": (3 * w).round(), "equal": torch.zeros_like(w)}[kind]
    lengths = torch.tensor([L, L - 1, budget, budget + 1, 0][:B], device="cuda").int()
    want = layer.paged_evict(kp, vp, w, table, lengths, budget, recent)
    after = ts.paged_cache_evict(kp, vp, w, table, lengths, budget, recent)
    assert after.dtype == torch.int32
    same((kp, vp, w, after), want)


def test_evict_special_weights(hip_backend):
    """Infinities, NaN of either sign, zeros of either sign, subnormal and negative weights."""
    _, kp, vp, table = make(2, 3, 3, 1, 4, 64, 32, F32)
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.randn(2, 3, 256, device="cuda", generator=g)
    for i, x in enumerate((float("inf"), float("-inf"), float("nan"), 0.0, -0.0, 1e-45, -1e-45, 1e-40, 3e38)):
        w[:, :, i::17] = x
    w[1, 0, 5::31] = -torch.tensor(float("nan"))
    w[1, 1], w[1, 2] = float("nan"), float("-inf")
    lengths = torch.tensor([256, 200], device="cuda")
    for budget, recent in ((9, 0), (30, 4), (120, 60)):
        k, v, x = kp.clone(), vp.clone(), w.clone()
        want = layer.paged_evict(k, v, x, table, lengths, budget, recent)
        same((k, v, x, ts.paged_cache_evict(k, v, x, table, lengths, budget, recent)), want)


def test_evict_to_nothing_and_bad_pages(hip_backend):
    _, kp, vp, table = make(3, 2, 2, 1, 8, 16, 64, BF)
    table[0, 1], table[1, 6], table[2] = -1, 10**6, 10**6
    w = torch.rand(3, 2, 128, device="cuda")
    lengths = torch.tensor([128, 120, 99], device="cuda")
    for budget, recent in ((50, 20), (0, 0)):
        want = layer.paged_evict(kp, vp, w, table, lengths, budget, recent)
        after = ts.paged_cache_evict(kp, vp, w, table, lengths, budget, recent)
        same((kp, vp, w, after), want)
    k0 = kp[:0]
    want = layer.paged_evict(k0, k0, w, table, lengths, 7, 2)
    same((w,), (layer.paged_evict(k0, k0, w, table, lengths, 128, 2)[2],))
    after = ts.paged_cache_evict(k0, vp[:0], w, table, lengths, 7, 2)
    same((w, after), (want[2], want[3]))
    assert ts.paged_cache_evict(kp, vp, w[..., :0], table[:, :0], lengths, 7).tolist() == [0, 0, 0]


@pytest.mark.parametrize("dt,size", [
    (BF, (2, 4, 300, 128, 128, 9000, 700)), (F32, (1, 2, 2200, 16, 64, 30000, 0)), (HF, (20, 8, 40, 32, 96, 501, 60)),
    (BF, (3, 1, 130, 256, 8, 300, 300)), (F32, (4, 2, 1100, 16, 40, 17000, 5)), (BF, (1, 1, 1300, 64, 128, 80000, 100)),
    (HF, (40, 8, 12, 64, 64, 300, 17)), (BF, (130, 1, 300, 64, 16, 9000, 100)),
])
@pytest.mark.parametrize("kind", ["random", "ties", "special"])
def test_evict_long(hip_backend, dt, size, kind):
    """Many parts of a row list and of the weights, against the "pytorch" backend."""
    B, Hk, cols, ps, D, budget, recent = size
    _, kp, vp, table = make(B, Hk, Hk, 1, cols, ps, D, dt)
    L = cols * ps
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.randn(B, Hk, L, device="cuda", generator=g).exp()
    w[:, :, ::3] = 0.0
    if kind == "ties":
        w = (w * 2).round()
    if kind == "special":
        table[0, 2], table[-1, cols // 2] = -1, len(kp)
        w[0, 0], w[-1, -1, ::2] = float("nan"), float("-inf")
        w[:, :, 1::7], w[:, :, 5::11] = float("inf"), -1.0
    lengths = torch.randint(budget - 50, L + 1, (B,), device="cuda", generator=g)
    lengths[0] = L
    k, v, x = kp.clone(), vp.clone(), w.clone()
    ts.set_backend("pytorch")
    want = ts.paged_cache_evict(k, v, x, table, lengths, budget, recent)
    ts.set_backend("hip")
    after = ts.paged_cache_evict(kp, vp, w, table, lengths, budget, recent)
    same((kp, vp, w, after), (k, v, x, want))


def test_evict_again_and_again(hip_backend):
    """One row over the budget at a time, as a decoding loop does."""
    _, kp, vp, table = make(2, 2, 2, 1, 4, 16, 64, BF)
    w = torch.rand(2, 2, 64, device="cuda")
    lengths = torch.tensor([41, 41], device="cuda")
    for i in range(12):
        want = layer.paged_evict(kp, vp, w, table, lengths, 40, 8)
        n = ts.paged_cache_evict(kp, vp, w, table, lengths, 40, 8)
        same((kp, vp, w, n), want)
        K = torch.full((2, 2, 1, 64), float(i), dtype=BF, device="cuda")
        lengths = ts.paged_cache_append(K, K, kp, vp, table, n, weights=w)
        w[:, :, 40] = torch.rand(2, 2, device="cuda")


@pytest.mark.parametrize("kind", ["random", "ties", "special"])
@pytest.mark.parametrize("size", [(20, 4, 3200, 16, 8, 300, 20), (1, 2, 220, 256, 64, 20000, 3000), (3, 1, 800, 64, 40, 51000, 0),
                                  (1, 1, 1000, 128, 16, 8192, 8192)])
def test_evict_by_parts(hip_backend, size, kind):
    """Weights searched part by part, rows moved in one list or in segments."""
    test_evict_long(hip_backend, BF, size, kind)


@pytest.mark.parametrize("cols", [64, 1000])
@pytest.mark.parametrize("step", [1 << 23, 1 << 12, 5])
@pytest.mark.parametrize("more", [-30, 0, 30])
def test_evict_where_the_search_ends(hip_backend, cols, step, more):
    """Two weights that differ in the first, the second or the last digit of the search; the
    budget takes some of the larger ones, all of them, or some of the smaller too."""
    _, kp, vp, table = make(2, 2, 2, 1, cols, 64, 16, BF)
    L, recent = cols * 64, 100
    g = torch.Generator(device="cuda").manual_seed(5)
    large = torch.zeros(2, 2, L, dtype=torch.bool, device="cuda")
    count = L // 5
    for b in range(2):
        for h in range(2):
            large[b, h, torch.randperm(L - recent - 77 * b, device="cuda", generator=g)[:count]] = True
    w = (torch.full((2, 2, L), 0x3F800000, dtype=torch.int32, device="cuda") + large.int() * step).view(torch.float32)
    lengths = torch.tensor([L, L - 77], device="cuda")
    k, v, x = kp.clone(), vp.clone(), w.clone()
    ts.set_backend("pytorch")
    want = ts.paged_cache_evict(k, v, x, table, lengths, count + more + recent, recent)
    ts.set_backend("hip")
    after = ts.paged_cache_evict(kp, vp, w, table, lengths, count + more + recent, recent)
    same((kp, vp, w, after), (k, v, x, want))


@pytest.mark.parametrize("cols", [16384, 16385])
def test_evict_at_the_most_parts(hip_backend, cols):
    """The longest caches of 8 units that are searched by parts, and the shortest that are not."""
    test_evict_long(hip_backend, BF, (2, 4, cols, 256, 8, 5000, 300), "ties")
