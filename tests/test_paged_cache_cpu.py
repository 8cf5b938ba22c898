"""The operators of a key and value cache in pages on the CPU: the "pytorch"
backend against the row-by-row oracle, bad pages, refusals (on the host, before
any device work), and what torch.compile traces with."""

from __future__ import annotations

import pytest
import torch

import trnsparse_amd as ts
from oracle import layer
from trnsparse_amd.hip import _lib

F64 = torch.float64


def make(B=3, H=4, Hk=2, N=3, cols=4, size=16, D=8, dt=F64, seed=0, pages=None):
    """Q, new K and V, pages (one more than the table names), a table of scattered pages."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=F64).to(dt)  # noqa: E731
    pages = B * cols + 1 if pages is None else pages
    table = torch.randperm(max(pages, B * cols), generator=g)[: B * cols].view(B, cols)
    return r(B, H, N, D), r(B, Hk, N, D), r(B, Hk, N, D), r(pages, Hk, size, D), r(pages, Hk, size, D), table


def attend(Q, kp, vp, table, lengths, new=None, weights=None, scale=0.4):
    N, L = Q.shape[2], table.shape[1] * kp.shape[2]
    seen = layer.chunk_seen(lengths, new, N, L)
    r = layer.attention(Q, layer.paged_rows(kp, table), layer.paged_rows(vp, table), scale, seen)
    O = ts.paged_attention(Q, kp, vp, table, lengths, new, scale, weights)
    torch.testing.assert_close(O, r["O"], rtol=1e-12, atol=1e-12)
    return O, r


@pytest.mark.parametrize("N", [1, 3, 20])
def test_attention(pytorch_backend, N):
    Q, _, _, kp, vp, table = make(B=4, N=N)
    attend(Q, kp, vp, table, torch.tensor([0, 1, 64, 99]))
    attend(Q, kp, vp, table.int(), torch.tensor([N, 16, 17, -5]).int(), torch.tensor([N, 1, 0, 3]).int())
    O, _ = attend(Q, kp, vp, table, torch.tensor([5, 5, 64, 33]), torch.tensor([99, -2, 0, 1]))
    assert (O[1] == 0).all() and (O[2] == 0).all() and (O[3, :, 1:] == 0).all()


def test_attention_weights(pytorch_backend):
    Q, _, _, kp, vp, table = make(N=5)
    lengths, new = torch.tensor([64, 2, 30]), torch.tensor([5, 4, 1])
    before = torch.rand(3, 2, 64)
    w = before.clone()
    _, r = attend(Q, kp, vp, table, lengths, new, w)
    torch.testing.assert_close(w.double(), before.double() + r["W"], rtol=1e-6, atol=1e-6)
    assert torch.equal(w[1, :, 2:], before[1, :, 2:])  # rows behind the length stay as they were


def test_rows_behind_the_length_are_not_read(pytorch_backend):
    Q, _, _, kp, vp, table = make(N=2)
    lengths = torch.tensor([64, 17, 3])
    want = ts.paged_attention(Q, kp, vp, table, lengths)
    kp2, vp2 = kp.clone(), vp.clone()
    for b, n in enumerate(lengths.tolist()):
        for j in range(n, 64):
            kp2[table[b, j // 16], :, j % 16], vp2[table[b, j // 16], :, j % 16] = float("nan"), float("inf")
    assert torch.equal(ts.paged_attention(Q, kp2, vp2, table, lengths), want)


def test_bad_pages(pytorch_backend):
    """Entries outside [0, pages) read as zeros and are not written."""
    Q, K, V, kp, vp, table = make(N=6)
    table[0, 1], table[1, 0], table[2] = -1, 10**9, 13
    lengths = torch.tensor([40, 20, 12])
    O, r = attend(Q, kp, vp, table, lengths)
    assert (O[2] == 0).all()
    before = lengths - 6
    want = layer.paged_append(K, V, kp, vp, table, before)
    after = ts.paged_cache_append(K, V, kp, vp, table, before)
    assert torch.equal(after, lengths) and torch.equal(kp, want[0]) and torch.equal(vp, want[1])
    w = torch.rand(3, 2, 64)
    want = layer.paged_evict(kp, vp, w, table, lengths, 10, 4)
    after = ts.paged_cache_evict(kp, vp, w, table, lengths, 10, 4)
    for got, x in zip((kp, vp, w, after), want):
        assert torch.equal(got, x)


def test_no_pages_at_all(pytorch_backend):
    Q, K, V, kp, vp, table = make(pages=0)
    lengths, w = torch.tensor([3, 50, 64]), torch.rand(3, 2, 64)
    assert (ts.paged_attention(Q, kp, vp, table, lengths) == 0).all()
    assert torch.equal(ts.paged_cache_append(K, V, kp, vp, table, lengths), torch.tensor([6, 53, 64]))
    want = layer.paged_evict(kp, vp, w, table, lengths, 9, 0)
    assert torch.equal(ts.paged_cache_evict(kp, vp, w, table, lengths, 9), want[3]) and torch.equal(w, want[2])
    empty = table[:, :0]
    assert (ts.paged_attention(Q, kp, vp, empty, lengths) == 0).all()


@pytest.mark.parametrize("new", [None, [3, 0, 2], [99, -1, 1]])
def test_append(pytorch_backend, new):
    _, K, V, kp, vp, table = make()
    new = None if new is None else torch.tensor(new)
    for lengths in ([0, 15, 47], [62, 64, 63], [-4, 16, 1000]):
        lengths = torch.tensor(lengths)
        w = torch.rand(3, 2, 64)
        want = layer.paged_append(K, V, kp, vp, table, lengths, new, w)
        after = ts.paged_cache_append(K, V, kp, vp, table, lengths, new, w)
        for got, x in zip((kp, vp, w, after), want):
            assert torch.equal(got, x)


@pytest.mark.parametrize("budget,recent", [(0, 0), (1, 0), (1, 1), (20, 0), (20, 7), (20, 20), (63, 5), (64, 2), (500, 400)])
def test_evict(pytorch_backend, budget, recent):
    _, _, _, kp, vp, table = make()
    lengths = torch.tensor([64, 21, 5])
    w = torch.randint(0, 6, (3, 2, 64)).float()  # many ties
    w[0, 0, ::5], w[0, 1, 3], w[1, 0, :2] = float("inf"), float("nan"), -0.0
    want = layer.paged_evict(kp, vp, w, table, lengths, budget, recent)
    after = ts.paged_cache_evict(kp, vp, w, table, lengths, budget, recent)
    for got, x in zip((kp, vp, w, after), want):
        torch.testing.assert_close(got, x, rtol=0, atol=0, equal_nan=True)


def test_a_run_of_them(pytorch_backend):
    """Tokens go in one at a time, are attended to and evicted by their weights:
    what the cache holds in the end is what stands at the kept places."""
    B, Hk, D, budget, recent = 2, 2, 8, 24, 8
    g = torch.Generator().manual_seed(3)
    Q, K, V, kp, vp, table = make(B=B, N=1, cols=3)
    lengths, w = torch.zeros(B, dtype=torch.int64), torch.zeros(B, Hk, 48)
    for _ in range(40):
        q, k, v = (torch.randn(B, h, 1, D, generator=g, dtype=F64) for h in (4, Hk, Hk))
        lengths = ts.paged_cache_append(k, v, kp, vp, table, lengths, weights=w)
        before = w.clone()
        O, r = attend(q, kp, vp, table, lengths, weights=w, scale=D**-0.5)
        torch.testing.assert_close((w - before).sum(-1), torch.full((B, Hk), 2.0), rtol=1e-5, atol=1e-5)  # 2 heads a key head
        if int(lengths.max()) == 32:
            lengths = ts.paged_cache_evict(kp, vp, w, table, lengths, budget, recent)
            assert (lengths == budget).all()
            assert torch.equal(layer.paged_rows(kp, table)[:, :, budget - 1 : budget], k)  # the newest is the last
    assert (lengths == 24).all()


def refusals(dt=F64, other=torch.float32, dev="cpu"):
    Q, K, V, kp, vp, t = (x.to(dev) for x in make(dt=dt))
    i = lambda *v: torch.tensor(v, device=dev)  # noqa: E731
    n, w = i(5, 6, 7), torch.zeros(3, 2, 64, device=dev)
    a, p, e = ts.paged_attention, ts.paged_cache_append, ts.paged_cache_evict
    grad = lambda x: x.clone().requires_grad_()  # noqa: E731
    wide = torch.zeros(2, 2, 16, 136, dtype=dt, device=dev)
    thin = torch.zeros(13, 2, 16, 1, dtype=dt, device=dev)
    caches = [
        (kp[0], vp[0], t, n), (kp, vp[:5], t, n), (kp, vp.to(other), t, n), (kp.int(), vp.int(), t, n),
        (kp[:, :, :15], vp[:, :, :15], t, n), (kp[:, :, :0], vp[:, :, :0], t, n), (kp[:, :0], vp[:, :0], t, n),
        (wide, wide.clone(), t, n), (thin, thin.clone(), t, n), (kp, vp, t[0], n), (kp, vp, t.float(), n),
        (kp, vp, t, n[:2]), (kp, vp, t, n.float()), (kp, vp, t, n.view(3, 1)),
    ]
    calls = [(a, (Q, *c)) for c in caches] + [(p, (K, V, *c)) for c in caches] + \
            [(e, (c[0], c[1], w, c[2], c[3], 4)) for c in caches]
    more = [
        (a, (Q[0], kp, vp, t, n)), (a, (Q[:2], kp, vp, t, n)), (a, (Q[..., :4], kp, vp, t, n)), (a, (Q[:, :3], kp, vp, t, n)),
        (a, (Q.to(other), kp, vp, t, n)), (a, (Q, kp, vp, t, n, i(1, 2))), (a, (Q, kp, vp, t, n, i(1.0, 2.0, 3.0))),
        (a, (Q, kp, vp, t, n, None, 0.0)), (a, (Q, kp, vp, t, n, None, float("nan"))),
        (a, (Q, kp, vp, t, n, None, float("inf"))), (a, (Q, kp, vp, t, n, None, 0.1, w[:, :, :63])),
        (a, (Q, kp, vp, t, n, None, 0.1, w.double())), (a, (Q, kp, vp, t, n, None, 0.1, w[:2])),
        (a, (grad(Q), kp, vp, t, n)), (a, (Q, grad(kp), vp, t, n)), (a, (Q, kp, vp, t, n, None, 0.1, grad(w))),
        (p, (K[0], V[0], kp, vp, t, n)), (p, (K[:2], V[:2], kp, vp, t, n)), (p, (K, V[:, :, :2], kp, vp, t, n)),
        (p, (K[:, :1], V[:, :1], kp, vp, t, n)), (p, (K.to(other), V, kp, vp, t, n)), (p, (K, V, kp, vp, t, n, i(1, 2))),
        (p, (K, V, kp, vp, t, n, i(1.0, 2.0, 3.0))), (p, (K, V, kp, vp, t, n, None, w[..., :48])), (p, (K, V, kp, kp, t, n)),
        (p, (grad(K), V, kp, vp, t, n)), (p, (K, V, grad(kp), vp, t, n)),
        (e, (kp, vp, w[..., :48], t, n, 4)), (e, (kp, vp, w.double(), t, n, 4)), (e, (kp, vp, w, t, n, -1)),
        (e, (kp, vp, w, t, n, 4, 5)), (e, (kp, vp, w, t, n, 4, -1)), (e, (kp, kp, w, t, n, 4)), (e, (kp, grad(vp), w, t, n, 4)),
    ]
    return calls + more


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


built = pytest.mark.skipif(not (_lib.LIB_PATH.exists() and _lib.OPS_PATH.exists()),
                           reason="library not built (run __graft_entry__.build())")


@built
def test_c_abi_refusals():
    """Sizes, alignment, strides and workspaces are checked on the host (dummy
    pointers: nothing is dereferenced)."""
    import ctypes

    lib = _lib.load()
    st = lambda *v: (ctypes.c_int64 * len(v))(*v)  # noqa: E731
    d, q3, k3 = 256, st(64 * 64, 64, 64), st(2 * 16 * 64, 16 * 64, 64)
    big = dict(dt=_lib.TSP_BF16, B=1, Hk=2, P=8, size=16, D=64, t=d, tt=1, ts=4, cols=4, n=d, it=1)

    def attend(Q=d, O=d, kp=d, ks=k3, H=2, N=64, scale=0.1, w=None, ws=d, wsb=1 << 40, **kw):
        c = {**big, **kw}
        return lib.tsp_paged_attn_fwd(Q, q3, kp, ks, d, k3, c["dt"], c["B"], H, c["Hk"], N, c["P"], c["size"], c["D"],
                                      c["t"], c["tt"], c["ts"], c["cols"], c["n"], None, c["it"], scale, O, q3, w,
                                      st(128, 64) if w else None, ws, wsb, None)

    def append(K=d, kp=d, ks=k3, N=3, out=512, **kw):
        c = {**big, **kw}
        return lib.tsp_paged_append(K, q3, d, q3, kp, ks, d, k3, c["dt"], c["B"], c["Hk"], N, c["P"], c["size"], c["D"],
                                    c["t"], c["tt"], c["ts"], c["cols"], c["n"], None, c["it"], out, None, None, None)

    def evict(kp=d, vp=4096, ks=k3, w=d, budget=8, recent=2, out=512, ws=d, wsb=1 << 40, **kw):
        c = {**big, **kw}
        return lib.tsp_paged_evict(kp, ks, vp, k3, c["dt"], c["B"], c["Hk"], c["P"], c["size"], c["D"], c["t"], c["tt"],
                                   c["ts"], c["cols"], c["n"], c["it"], w, st(128, 64), budget, recent, out, ws, wsb, None)

    for call in (attend, append, evict):
        assert call(dt=_lib.TSP_F64) == -2 and b"dtype" in lib.tsp_last_error()
        assert call(size=24) == -2 and b"page_size" in lib.tsp_last_error()
        assert call(D=60) == -2 and call(D=136) == -2 and call(D=0) == -1 and call(Hk=0) == -1 and call(size=0) == -1
        assert call(cols=-1) == -1 and call(P=-1) == -1 and call(t=None) == -1 and call(tt=7) == -1 and call(ts=-1) == -1
        assert call(cols=1 << 27) == -2 and call(P=1 << 31) == -2 and call(size=1 << 21, cols=1) == -2
        assert call(n=None) == -1 and call(it=9) == -1
        assert call(kp=None) == -1 and call(kp=264) == -1  # pieces of 16 bytes
        assert call(ks=st(2048, 1024, 68)) == -1 and call(ks=st(2048, 1024, 0)) == -1 and call(ks=st(-2048, 1024, 64)) == -1
        assert call(ks=st(2048, 1024, 1 << 24)) == -1  # rows 32 MiB apart
    assert attend(B=0) == 0 and attend(N=0) == 0 and append(B=0) == 0 and evict(B=0) == 0
    assert attend(H=3) == -1 and attend(N=-1) == -1 and attend(Q=None) == -1 and attend(O=None) == -1 and attend(Q=8) == -1
    assert attend(scale=0.0) == -1 and attend(scale=float("nan")) == -1 and attend(scale=1e-40) == -1
    assert attend(cols=4096, ws=None) == -1 and b"workspace" in lib.tsp_last_error()
    assert attend(w=d, wsb=16) == -1 and b"workspace" in lib.tsp_last_error()
    assert append(K=None) == -1 and append(K=8) == -1 and append(N=-1) == -1 and append(out=None) == -1 and append(out=d) == -1
    assert evict(w=None) == -1 and evict(recent=9) == -1 and evict(recent=-1) == -1 and evict(out=d) == -1
    assert evict(vp=d) == -1 and evict(ws=None) == -1 and evict(wsb=16) == -1
    assert lib.tsp_paged_attn_workspace_size(7, 1, 2, 2, 1, 64, 64, 0, 0) == -1
    size = lambda *v: lib.tsp_paged_evict_workspace_size(_lib.TSP_BF16, *v)  # noqa: E731
    assert size(1, 0, 64, 64, 5) == -1 and size(2, 3, 64, 64, -1) == -1 and size(2, 3, 64, 64, 5) >= 8 * 30
    assert size(1, 2, 1 << 17, 64, 1 << 15) >= 2 * 2 * 2 * 64 * (1 << 15)  # rows copied aside


SCHEMAS = {
    "paged_attn_fwd": "(Tensor Q, Tensor K_pages, Tensor V_pages, Tensor block_table, Tensor lengths, Tensor? new_lengths, "
                      "float scale, Tensor(a!)? weights) -> Tensor",
    "paged_append": "(Tensor K, Tensor V, Tensor(a!) K_pages, Tensor(b!) V_pages, Tensor block_table, Tensor lengths, "
                    "Tensor? new_lengths, Tensor(c!)? weights) -> Tensor",
    "paged_evict": "(Tensor(a!) K_pages, Tensor(b!) V_pages, Tensor(c!) weights, Tensor block_table, Tensor lengths, "
                   "int budget, int recent) -> Tensor",
}


@built
@pytest.mark.parametrize("name", SCHEMAS)
def test_schema(name):
    assert str(getattr(_lib.ops(), name).default._schema) == f"trnsparse_hip::{name}{SCHEMAS[name]}"


@built
def test_meta_shapes():
    ops, m = _lib.ops(), lambda *s, dt=torch.bfloat16: torch.empty(*s, dtype=dt, device="meta")  # noqa: E731
    Q, kp, t, n = m(2, 70, 8, 64).transpose(1, 2), m(9, 2, 16, 64), m(2, 4, dt=torch.int32), m(2, dt=torch.int32)
    O = ops.paged_attn_fwd(Q, kp, kp, t, n, None, 0.1, None)
    assert O.shape == Q.shape and O.stride() == Q.stride() and O.dtype == Q.dtype
    for out in (ops.paged_append(m(2, 2, 5, 64), m(2, 2, 5, 64), kp, kp, t, n, None, None),
                ops.paged_evict(kp, kp, m(2, 2, 64, dt=torch.float32), t, n, 8, 2)):
        assert out.shape == (2,) and out.dtype == torch.int32


@built
def test_c_abi_types_of_lengths():
    """new_lengths may be of the other type than lengths; an eviction has none."""
    import ctypes

    lib, d, B = _lib.load(), 256, 0
    s3, bf = (ctypes.c_int64 * 3)(2048, 1024, 64), _lib.TSP_BF16
    for it, rc in ((0, 0), (1, 0), (2, 0), (3, 0), (4, -1), (9, -1), (-1, -1)):
        assert lib.tsp_paged_attn_fwd(d, s3, d, s3, d, s3, bf, B, 2, 2, 1, 8, 16, 64, d, 1, 4, 4, d, d, it, 0.1, d, s3,
                                      None, None, None, 0, None) == rc
        assert lib.tsp_paged_append(d, s3, d, s3, d, s3, 4096, s3, bf, B, 2, 1, 8, 16, 64, d, 1, 4, 4, d, d, it, 512,
                                    None, None, None) == rc
        assert lib.tsp_paged_evict(d, s3, 4096, s3, bf, B, 2, 8, 16, 64, d, 1, 4, 4, d, it, d, s3, 8, 2, 512, None, 0,
                                   None) == (rc if it < 2 else -1)


def overlapping(dt=F64, dev="cpu"):
    """Calls whose written pages or weights have rows that share memory, though no stride is zero."""
    Q, K, V, kp, vp, t = (x.to(dev) for x in make(dt=dt))
    n, w = torch.tensor([5, 6, 7], device=dev), torch.zeros(3, 2, 64, device=dev)
    pool = torch.zeros(8192, dtype=dt, device=dev)
    a, p, e = ts.paged_attention, ts.paged_cache_append, ts.paged_cache_evict
    calls = []
    for strides in ((256, 8, 8), (8, 128, 8), (128, 128, 8), (256, 120, 8), (256, 64, 16), (16, 8, 104)):
        bad = pool.as_strided((13, 2, 16, 8), (*strides, 1))
        calls += [(p, (K, V, bad, vp, t, n)), (p, (K, V, kp, bad, t, n)), (e, (bad, vp, w, t, n, 4)), (e, (kp, bad, w, t, n, 4))]
    for strides in ((64, 64), (128, 1), (4, 128), (96, 64), (32, 64)):
        bad = torch.zeros(512, device=dev).as_strided((3, 2, 64), (*strides, 1))
        calls += [(a, (Q, kp, vp, t, n, None, 0.1, bad)), (p, (K, V, kp, vp, t, n, None, bad)), (e, (kp, vp, bad, t, n, 4))]
    return calls


@pytest.mark.parametrize("i", range(len(overlapping())))
def test_written_rows_that_overlap_are_refused(pytorch_backend, i):
    f, args = overlapping()[i]
    with pytest.raises(RuntimeError, match="overlap"):
        f(*args)


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(overlapping())))
@pytest.mark.parametrize("dev", ["cuda", "cpu"])
def test_written_rows_that_overlap_are_refused_on_the_gpu(hip_backend, i, dev):
    f, args = overlapping(torch.float32, dev)[i]
    # (the GPU's copy of a host view may have strides that are refused by another check)
    with pytest.raises(RuntimeError, match="overlap|lie apart" if dev == "cuda" else "overlap|lie apart|unit stride"):
        f(*args)


def apart(dt=F64, dev="cpu"):
    """Views of pages and weights whose rows lie apart, in any order of dimensions."""
    _, _, _, kp, vp, _ = (x.to(dev) for x in make(dt=dt))
    both, more = torch.stack([kp, vp], 1), torch.zeros(26, 4, 48, 24, dtype=dt, device=dev)
    w = torch.zeros(3, 2, 64, device=dev)
    turn = lambda x, *d: x.permute(*d).contiguous().permute(*(d.index(i) for i in range(len(d))))  # noqa: E731
    pages = [(kp, vp), (turn(kp, 0, 2, 1, 3), turn(vp, 2, 0, 1, 3)), (turn(kp, 1, 2, 0, 3), turn(vp, 2, 1, 0, 3)),
             (both[:, 0], both[:, 1]), (more[::2, 1::2, ::3, 8:16], more[1::2, ::2, 16:32, :8])]
    weights = [w, turn(w, 1, 0, 2), torch.zeros(5, 4, 99, device=dev)[::2, 1::2, 5:69]]
    return pages, weights


def run_apart(dt, dev):
    _, K, V, kp, vp, t = (x.to(dev) for x in make(dt=dt))
    n, g = torch.tensor([5, 46, 61], device=dev), torch.Generator().manual_seed(4)
    w0 = torch.rand(3, 2, 64, generator=g).to(dev)
    first = layer.paged_append(K, V, kp, vp, t, n, None, w0)
    want = layer.paged_evict(*first[:3], t, first[3], 20, 4)
    pages, weights = apart(dt, dev)
    for k, v in pages:
        for w in weights:
            k.copy_(kp), v.copy_(vp), w.copy_(w0)
            after = ts.paged_cache_append(K, V, k, v, t, n, None, w)
            assert all(torch.equal(x.cpu(), y) for x, y in zip((k, v, w, after), first))
            after = ts.paged_cache_evict(k, v, w, t, after, 20, 4)
            assert all(torch.equal(x.cpu(), y) for x, y in zip((k, v, w, after), want))


def test_views_that_lie_apart(pytorch_backend):
    run_apart(F64, "cpu")


@pytest.mark.gpu
def test_views_that_lie_apart_on_the_gpu(hip_backend):
    run_apart(torch.float32, "cuda")


@built
def test_c_abi_written_rows_that_overlap():
    import ctypes

    lib = _lib.load()
    st = lambda *v: (ctypes.c_int64 * len(v))(*v)  # noqa: E731
    d, good, bf = 256, st(2048, 1024, 64), _lib.TSP_BF16
    for bad in (st(2048, 64, 64), st(64, 1024, 64), st(2048, 1016, 64), st(1 << 62, 512, 64), st(2048, 512, 128)):
        for k, v in ((bad, good), (good, bad)):
            assert lib.tsp_paged_append(d, good, d, good, d, k, 4096, v, bf, 1, 2, 1, 8, 16, 64, d, 1, 4, 4, d, None, 1, 512,
                                        None, None, None) == -1 and b"overlap" in lib.tsp_last_error()
            assert lib.tsp_paged_evict(d, k, 4096, v, bf, 1, 2, 8, 16, 64, d, 1, 4, 4, d, 1, d, st(128, 64), 8, 2, 512, d,
                                       1 << 40, None) == -1 and b"overlap" in lib.tsp_last_error()
    for bad in (st(128, 63), st(64, 64), st(64, 1), st(1 << 62, 0)):
        assert lib.tsp_paged_attn_fwd(d, good, d, good, d, good, bf, 2, 2, 2, 1, 8, 16, 64, d, 1, 4, 4, d, None, 1, 0.1, d,
                                      good, d, bad, d, 1 << 40, None) == -1 and b"overlap" in lib.tsp_last_error()
        assert lib.tsp_paged_evict(d, good, 4096, good, bf, 2, 2, 8, 16, 64, d, 1, 4, 4, d, 1, d, bad, 8, 2, 512, d, 1 << 40,
                                   None) == -1 and b"overlap" in lib.tsp_last_error()


def run_append_of_cached_rows(dt, dev):
    """New rows that are views of the pages: of rows that other sequences, other heads or the
    other cache's rows overwrite, and of the very rows that they move by one."""
    _, _, _, kp, vp, t = make(B=3, N=1, cols=4, dt=dt, seed=21)
    n = torch.tensor([3, 20, 33])
    order = t[:, 0].tolist()
    for new in (None, torch.tensor([9, 2, 0])):
        for sources in (lambda k, v: (k[t[0, 0]][None], v[t[0, 0]][None]), lambda k, v: (v[t[1, 1]][None], k[t[0, 0]][None]),
                        lambda k, v: (k[order[0]][None], k[order[0]][None])):
            k, v, table = kp.clone().to(dev), vp.clone().to(dev), t.to(dev)
            a, b = (x.expand(3, -1, -1, -1)[:, :, :12] for x in sources(k, v))
            want = layer.paged_append(a.cpu().clone(), b.cpu().clone(), kp, vp, t, n, new)
            after = ts.paged_cache_append(a, b, k, v, table, n.to(dev), None if new is None else new.to(dev))
            assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1]) and torch.equal(after.cpu(), want[3])
        k, v = kp.clone().to(dev), vp.clone().to(dev)  # one pool of pages, whose first one's rows go to another
        pool = torch.stack([k, v], 1)
        a, b = pool[:3, 0, :, 2:14], pool[:3, 1, :, 2:14]
        want = layer.paged_append(a.cpu().clone(), b.cpu().clone(), kp, vp, t, n, new)
        after = ts.paged_cache_append(a, b, pool[:, 0], pool[:, 1], t.to(dev), n.to(dev), None if new is None else new.to(dev))
        assert torch.equal(pool[:, 0].cpu(), want[0]) and torch.equal(pool[:, 1].cpu(), want[1])


def test_append_of_cached_rows(pytorch_backend):
    run_append_of_cached_rows(F64, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("dev", ["cuda", "cpu"])
def test_append_of_cached_rows_on_the_gpu(hip_backend, dev):
    run_append_of_cached_rows(torch.float32, dev)


@built
def test_c_abi_workspaces_are_aligned():
    """Results of ranges and scores are read 16 bytes at a time."""
    import ctypes

    lib, d = _lib.load(), 256
    s3, w2, bf = (ctypes.c_int64 * 3)(2048, 1024, 64), (ctypes.c_int64 * 2)(65536, 32768), _lib.TSP_BF16
    for ws in (260, 264, 258):
        for w in (None, d):
            assert lib.tsp_paged_attn_fwd(d, s3, d, s3, d, s3, bf, 1, 2, 2, 1, 8, 16, 64, d, 1, 2048, 2048, d, None, 1, 0.1, d,
                                          s3, w, w2, ws, 1 << 40, None) == -1 and b"aligned" in lib.tsp_last_error()
        assert lib.tsp_paged_evict(d, s3, 4096, s3, bf, 1, 2, 8, 16, 64, d, 1, 2048, 2048, d, 1, d, w2, 8, 2, 512, ws, 1 << 40,
                                   None) == -1 and b"aligned" in lib.tsp_last_error()


@built
@pytest.mark.parametrize("it", [0, 1, 2, 3])
def test_c_abi_lengths_out_is_apart(it):
    """It is written while other workgroups of the sequence still read lengths and new_lengths."""
    import ctypes

    lib, d, n, new, B = _lib.load(), 256, 4096, 8192, 3
    s3, w2, bf = (ctypes.c_int64 * 3)(2048, 1024, 64), (ctypes.c_int64 * 2)(128, 64), _lib.TSP_BF16
    out = 8 if it & 1 else 4
    held = (out, 12 - out if it & 2 else out)
    for p, size in ((n, held[0]), (new, held[1])):
        for at in (p, p + size, p + (B - 1) * size, p + B * size - 4, p - (B - 1) * out, p - 4):
            assert lib.tsp_paged_append(d, s3, d, s3, d, s3, 512, s3, bf, B, 2, 1, 8, 16, 64, d, 1, 4, 4, n, new, it, at,
                                        None, None, None) == -1 and b"lengths_out" in lib.tsp_last_error(), (p, at)
            if p == n and it < 2:
                assert lib.tsp_paged_evict(d, s3, 512, s3, bf, B, 2, 8, 16, 64, d, 1, 4, 4, n, it, d, w2, 8, 2, at, d, 1 << 40,
                                           None) == -1 and b"lengths_out" in lib.tsp_last_error(), at
        for at in (p + B * size, p - B * out):  # (the next check's message)
            assert lib.tsp_paged_append(d, s3, d, s3, None, s3, 512, s3, bf, B, 2, 1, 8, 16, 64, d, 1, 4, 4, n, new, it, at,
                                        None, None, None) == -1 and b"null K_pages" in lib.tsp_last_error(), (p, at)


def run_no_columns(dt, dev):
    """Sequences without room for a row, weights of no elements included."""
    Q, K, V, kp, vp, t = (x.to(dev) for x in make(dt=dt))
    t, n, w = t[:, :0], torch.tensor([0, 5, -3], device=dev), torch.ones(3, 2, 0, device=dev)
    before = kp.clone(), vp.clone()
    for weights in (None, w):
        assert ts.paged_cache_append(K, V, kp, vp, t, n, None, weights).tolist() == [0, 0, 0]
        assert (ts.paged_attention(Q, kp, vp, t, n, None, None, weights) == 0).all()
    for budget in (0, 7):
        assert ts.paged_cache_evict(kp, vp, w, t, n, budget).tolist() == [0, 0, 0]
    assert torch.equal(kp, before[0]) and torch.equal(vp, before[1])


def test_no_columns(pytorch_backend):
    run_no_columns(F64, "cpu")


@pytest.mark.gpu
def test_no_columns_on_the_gpu(hip_backend):
    run_no_columns(torch.float32, "cuda")


@built
def test_c_abi_null_weights_of_no_columns():
    """A tensor without elements has no address; with columns, null weights are refused."""
    import ctypes

    lib, d = _lib.load(), 256
    s3, w2 = (ctypes.c_int64 * 3)(2048, 1024, 64), (ctypes.c_int64 * 2)(0, 0)
    for cols, message in ((0, b"null K_pages"), (4, b"null weights")):
        assert lib.tsp_paged_evict(None, s3, 512, s3, _lib.TSP_BF16, 1, 2, 8, 16, 64, d, 1, cols, cols, 1024, 1, None, w2, 8,
                                   2, 4096, d, 1 << 40, None) == -1 and message in lib.tsp_last_error()


@built
def test_evict_workspace_of_very_long_caches():
    """Counts by parts, which every part reads, are kept only where the parts are few: the
    workspace (and the work) of the longest caches does not grow with their square."""
    lib = _lib.load()
    for units, slots in ((1, 1 << 30), (8, 1 << 30), (100, 1 << 28), (8, (1 << 22) + 1), (32, (1 << 20) + 1)):
        size = lib.tsp_paged_evict_workspace_size(_lib.TSP_BF16, units, 1, slots, 64, 5)
        assert 0 < size < 1 << 16, (units, slots, size)
    assert lib.tsp_paged_evict_workspace_size(_lib.TSP_BF16, 8, 1, 1 << 22, 64, 5) >= 4096 * 3 * 2048 * 4
