"""The operators of a paged cache together, as a server uses them: prompts in by
chunks, tokens one at a time, sequences that come and go, eviction; captured and
replayed, from several streams and threads, traced."""

from __future__ import annotations

import threading

import pytest
import torch

import trnsparse_amd as ts
from oracle import layer
from test_gpu_graphs import _capture
from test_gpu_paged_attention import BF, F32, HF, check, make
from trnsparse_amd.hip import _lib

pytestmark = pytest.mark.gpu

H, Hk, D, SIZE = 8, 2, 64, 16


def rand(g, *shape, dt=F32):
    return torch.randn(*shape, device="cuda", generator=g).to(dt)


def test_chunks_and_tokens_equal_the_whole(hip_backend):
    """A prompt taken in by chunks, then tokens one at a time, all rotated by their
    positions, equals attention over the whole sequence in float64."""
    B, cols = 3, 12
    g = torch.Generator(device="cuda").manual_seed(1)
    total = torch.tensor([150, 77, 31], device="cuda")
    T = int(total.max())
    q, k, v = rand(g, B, H, T, D), rand(g, B, Hk, T, D), rand(g, B, Hk, T, D)
    w, freq = 1 + 0.1 * rand(g, D), ts.rope_frequencies(D, device="cuda")
    q, k = ts.qk_norm_rope(q, k, w, w, torch.arange(T, device="cuda"), freq)
    _, kp, vp, table = make(B, H, Hk, 1, cols, SIZE, D, F32)
    out, lengths = torch.zeros_like(q), torch.zeros(B, dtype=torch.int32, device="cuda")
    at = 0
    for n in (64, 33, 20, 1, 1, 17, 1, 13):
        new = (total - at).clamp(0, n).int()
        lengths = ts.paged_cache_append(k[:, :, at : at + n], v[:, :, at : at + n], kp, vp, table, lengths, new)
        out[:, :, at : at + n] = ts.paged_attention(q[:, :, at : at + n], kp, vp, table, lengths, new)
        at += n
    assert at == T and torch.equal(lengths, total.int())
    want = layer.attention(q, k, v, D**-0.5, layer.chunk_seen(total, total, T, T))["O"]
    assert (out.double().cpu() - want).norm() <= 1e-5 * want.norm()  # (of 150 keys: test_gpu_paged_attention's bound is 4e-5)


@pytest.mark.parametrize("dt", [BF, F32])
def test_decoding_with_eviction(hip_backend, dt):
    """Sequences decode with a budget of rows; at each step results and weights are the
    oracle's over what the cache then holds."""
    B, cols, budget, recent = 3, 5, 48, 16
    g = torch.Generator(device="cuda").manual_seed(2)
    _, kp, vp, table = make(B, H, Hk, 1, cols, SIZE, D, dt)
    lengths, w = torch.tensor([3, 40, 0], device="cuda"), torch.zeros(B, Hk, cols * SIZE, device="cuda")
    for step in range(30):
        n = 5 if step % 7 == 0 else 1
        k, v = rand(g, B, Hk, n, D, dt=dt), rand(g, B, Hk, n, D, dt=dt)
        lengths = ts.paged_cache_append(k, v, kp, vp, table, lengths, weights=w)
        for b, m in enumerate(lengths.tolist()):
            assert (w[b, :, m - n : m] == 0).all()
            rows = layer.paged_rows(kp, table)[b, :, m - n : m]
            assert torch.equal(rows, k[b].cpu())
        Q = rand(g, B, n, H, D, dt=dt).transpose(1, 2)
        check(Q, kp, vp, table, lengths)
        ts.paged_attention(Q, kp, vp, table, lengths, weights=w)
        want = layer.paged_evict(kp, vp, w, table, lengths, budget, recent)
        lengths = ts.paged_cache_evict(kp, vp, w, table, lengths, budget, recent)
        torch.cuda.synchronize()
        for got, x in zip((kp, vp, w, lengths), want):
            assert torch.equal(got.cpu(), x)
        assert int(lengths.max()) <= budget
    assert (lengths == torch.tensor([48, 48, 48], device="cuda")).sum() >= 1


def _step(s, budget):
    """One decoding step on static buffers: append, attend, evict, lengths in place."""
    n = ts.paged_cache_append(s["k"], s["v"], s["kp"], s["vp"], s["table"], s["lengths"], s["new"], s["w"])
    O = ts.paged_attention(s["q"], s["kp"], s["vp"], s["table"], n, s["new"], weights=s["w"])
    s["lengths"].copy_(ts.paged_cache_evict(s["kp"], s["vp"], s["w"], s["table"], n, budget, budget // 4))
    return O


def _state(seed, dt, N, cols=40, B=4):
    g = torch.Generator(device="cuda").manual_seed(seed)
    _, kp, vp, table = make(B, H, Hk, 1, cols, SIZE, D, dt, seed=seed)
    return {"q": rand(g, B, H, N, D, dt=dt), "k": rand(g, B, Hk, N, D, dt=dt), "v": rand(g, B, Hk, N, D, dt=dt), "kp": kp,
            "vp": vp, "table": table, "lengths": torch.tensor([0, 9, 300, 510], device="cuda")[:B].clone(),
            "new": torch.tensor([N, 1, N, max(N - 1, 1)], device="cuda")[:B].clone(),
            "w": torch.zeros(B, Hk, cols * SIZE, device="cuda")}


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("N", [1, 6, 60])
def test_graph_of_a_step(hip_backend, dt, N):
    """A captured step replayed as the sequences grow and are cut: lengths, tables and
    caches are read at every replay; eager work and synchronizations in between."""
    budget = 400
    s, e = _state(3, dt, N), _state(3, dt, N)
    graph, (out,) = _capture(lambda: _step(s, budget))
    for name, t in _state(3, dt, N).items():
        s[name].copy_(t)
    g = torch.Generator(device="cuda").manual_seed(4)
    for turn in range(5):
        for name in ("q", "k", "v"):
            x = rand(g, *s[name].shape, dt=dt)
            s[name].copy_(x), e[name].copy_(x)
        if turn == 2:  # a sequence ends, another takes its pages
            for t in (s, e):
                t["lengths"][3] = 2
                t["table"][3] = t["table"][3].flip(0)
        graph.replay()
        torch.cuda.synchronize()
        want = _step(e, budget)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for name in ("kp", "vp", "w", "lengths"):
            assert torch.equal(s[name], e[name]), name


def test_graph_of_a_long_eviction(hip_backend):
    """The eviction by parts and segments, captured and replayed on other weights."""
    B, cols, budget = 2, 1300, 9000
    _, kp, vp, table = make(B, Hk, Hk, 1, cols, SIZE, 16, BF, seed=5)
    w, lengths = torch.zeros(B, Hk, cols * SIZE, device="cuda"), torch.tensor([cols * SIZE, 15000], device="cuda")
    graph, (after,) = _capture(lambda: ts.paged_cache_evict(kp, vp, w, table, lengths, budget, 70))
    g = torch.Generator(device="cuda").manual_seed(6)
    for _ in range(4):
        x = rand(g, *w.shape).exp()
        w.copy_(x)
        k, v, y = kp.clone(), vp.clone(), x.clone()
        graph.replay()
        torch.cuda.synchronize()
        n = ts.paged_cache_evict(k, v, y, table, lengths, budget, 70)
        torch.cuda.synchronize()
        assert torch.equal(kp, k) and torch.equal(vp, v) and torch.equal(w, y) and torch.equal(after, n)


def test_graph_of_an_eviction_by_parts(hip_backend):
    B, cols, budget = 1, 3300, 9000
    _, kp, vp, table = make(B, Hk, Hk, 1, cols, SIZE, 16, BF, seed=5)
    w, lengths = torch.zeros(B, Hk, cols * SIZE, device="cuda"), torch.tensor([cols * SIZE - 7], device="cuda")
    graph, (after,) = _capture(lambda: ts.paged_cache_evict(kp, vp, w, table, lengths, budget, 70))
    g = torch.Generator(device="cuda").manual_seed(6)
    for _ in range(4):
        x = rand(g, *w.shape).exp().round()
        w.copy_(x)
        k, v, y = kp.clone(), vp.clone(), x.clone()
        graph.replay()
        torch.cuda.synchronize()
        n = ts.paged_cache_evict(k, v, y, table, lengths, budget, 70)
        torch.cuda.synchronize()
        assert torch.equal(kp, k) and torch.equal(vp, v) and torch.equal(w, y) and torch.equal(after, n)


def test_two_graphs_and_streams(hip_backend):
    """Two captured steps replayed at the same time: each has workspaces of its own."""
    states = [_state(7 + i, BF, 3) for i in range(2)]
    eager = [_state(7 + i, BF, 3) for i in range(2)]
    graphs = [_capture(lambda s=s: _step(s, 200)) for s in states]
    for i, s in enumerate(states):
        for name, t in _state(7 + i, BF, 3).items():
            s[name].copy_(t)
    streams = [torch.cuda.Stream() for _ in states]
    torch.cuda.synchronize()
    for _ in range(4):
        for (graph, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        want = [_step(e, 200) for e in eager]
        torch.cuda.synchronize()
        for (_, (out,)), w, s, e in zip(graphs, want, states, eager):
            assert torch.equal(out, w) and torch.equal(s["w"], e["w"]) and torch.equal(s["kp"], e["kp"])


def test_two_threads_two_streams(hip_backend):
    states, eager = [_state(11 + i, BF, 1) for i in range(2)], [_state(11 + i, BF, 1) for i in range(2)]
    want = [[_step(e, 300) for _ in range(15)] for e in eager]
    torch.cuda.synchronize()
    bad = []

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            outs = [_step(states[i], 300) for _ in range(15)]
            torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(outs, want[i])):
                bad.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    assert all(torch.equal(s[n], e[n]) for s, e in zip(states, eager) for n in ("kp", "vp", "w", "lengths"))


def test_operands_on_the_host(hip_backend):
    """Tables and lengths from the host, and a whole cache there: written ones come back."""
    dev = _state(13, F32, 2, cols=6)
    dev["lengths"] %= 90
    host = {n: t.cpu() for n, t in dev.items()}
    want = _step(dev, 60)
    got = _step(host, 60)
    torch.cuda.synchronize()
    assert got.device.type == "cpu" and torch.equal(got, want.cpu())
    for n in ("kp", "vp", "w", "lengths"):
        assert torch.equal(host[n], dev[n].cpu()), n
    O = ts.paged_attention(dev["q"], dev["kp"], dev["vp"], host["table"], host["lengths"], host["new"].int())
    assert torch.equal(O, ts.paged_attention(dev["q"], dev["kp"], dev["vp"], dev["table"], dev["lengths"], dev["new"]))


def test_no_gradients_and_versions(hip_backend):
    """What is written counts as written; gradients and tangents are refused."""
    import torch.autograd.forward_ad as fw

    s = _state(14, F32, 2)
    before = [s[n]._version for n in ("kp", "vp", "w")]
    _step(s, 100)
    assert all(s[n]._version > b for n, b in zip(("kp", "vp", "w"), before))
    ops = _lib.ops()
    q = s["q"].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradients"):
        ops.paged_attn_fwd(q, s["kp"], s["vp"], s["table"], s["lengths"], None, 0.1, None)
    with torch.no_grad():
        ops.paged_attn_fwd(q, s["kp"], s["vp"], s["table"], s["lengths"], None, 0.1, None)
    with fw.dual_level(), pytest.raises(RuntimeError, match="tangent"):
        ts.paged_attention(fw.make_dual(s["q"], s["q"]), s["kp"], s["vp"], s["table"], s["lengths"])
    with pytest.raises(RuntimeError, match="not supported"):  # (a type that the pytorch backend takes)
        ts.paged_attention(s["q"].double(), s["kp"].double(), s["vp"].double(), s["table"], s["lengths"])


def test_traced_and_compiled(hip_backend):
    """torch.compile reaches the operators whole, writes in place included, and the public
    functions by graph breaks; results equal eager calls."""
    ops = _lib.ops()

    def whole(s):
        n = ops.paged_append(s["k"], s["v"], s["kp"], s["vp"], s["table"], s["lengths"], None, s["w"])
        O = ops.paged_attn_fwd(s["q"] * 2.0, s["kp"], s["vp"], s["table"], n, None, 0.125, s["w"]) + 1.0
        return O, ops.paged_evict(s["kp"], s["vp"], s["w"], s["table"], n, 50, 10) + 1

    def public(s):
        n = ts.paged_cache_append(s["k"], s["v"], s["kp"], s["vp"], s["table"], s["lengths"], None, s["w"])
        O = ts.paged_attention(s["q"] * 2.0, s["kp"], s["vp"], s["table"], n, None, 0.125, s["w"]) + 1.0
        return O, ts.paged_cache_evict(s["kp"], s["vp"], s["w"], s["table"], n, 50, 10) + 1

    for f, full in ((whole, True), (public, False)):
        a, b = _state(15, F32, 2), _state(15, F32, 2)
        want = f(a)
        got = torch.compile(f, fullgraph=full, backend="aot_eager")(b)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert all(torch.equal(a[n], b[n]) for n in ("kp", "vp", "w"))


def test_inference_mode(hip_backend):
    """Caches made in and out of inference mode; one made in it is not written outside."""
    a, b = _state(16, F32, 2), _state(16, F32, 2)
    want = _step(a, 100)
    with torch.inference_mode():
        c = _state(16, F32, 2)
        assert torch.equal(_step(b, 100), want) and torch.equal(_step(c, 100), want)
    kept = c["kp"].clone()
    with pytest.raises(RuntimeError, match="[Ii]nference"):
        ts.paged_cache_append(c["k"] + 1, c["v"], c["kp"], c["vp"], c["table"], c["lengths"])
    assert torch.equal(c["kp"], kept)


@pytest.mark.parametrize("host", [False, True])
def test_public_refusal_of_gradients(hip_backend, host):
    """Whichever operand asks for one, on the GPU or not; nothing is written."""
    s = _state(17, F32, 2)
    if host:
        s = {n: t.cpu() if isinstance(t, torch.Tensor) else t for n, t in s.items()}
    calls = {
        "paged_attention": (lambda a: ts.paged_attention(a["q"], a["kp"], a["vp"], a["table"], a["lengths"], None, None, a["w"]),
                            ("q", "kp", "vp", "w")),
        "paged_cache_append": (lambda a: ts.paged_cache_append(a["k"], a["v"], a["kp"], a["vp"], a["table"], a["lengths"], None, a["w"]),
                               ("k", "v", "kp", "vp", "w")),
        "paged_cache_evict": (lambda a: ts.paged_cache_evict(a["kp"], a["vp"], a["w"], a["table"], a["lengths"], 20, 5),
                              ("kp", "vp", "w")),
    }
    for name, (call, operands) in calls.items():
        for n in operands:
            a = {m: t.clone() if isinstance(t, torch.Tensor) else t for m, t in s.items()}
            a[n].requires_grad_()
            with pytest.raises(RuntimeError, match=f"{name} has no gradients"):
                call(a)
            assert all(torch.equal(a[m].detach(), s[m]) for m in ("kp", "vp", "w"))


@pytest.mark.parametrize("types", [(torch.int32, torch.int64), (torch.int64, torch.int32), (torch.int64, torch.int64)])
def test_lengths_past_32_bits(hip_backend, types):
    """Lengths and numbers of new tokens are taken into their ranges as they are, whatever
    the other's type: not by their low halves."""
    far = [2**31, 2**32 + 1, 2**32, -(2**32) + 1, 2]
    near = torch.tensor([3, 3, 3, 0, 2], device="cuda")
    s = _state(18, F32, 3, cols=6, B=4)
    g = torch.Generator(device="cuda").manual_seed(19)
    q, k, v = rand(g, 5, H, 3, D), rand(g, 5, Hk, 3, D), rand(g, 5, Hk, 3, D)
    table = torch.cat([s["table"][:3], s["table"][:2].flip(0)])
    values = torch.tensor(far, device="cuda")
    n = torch.tensor([70, 71, 72, 73, 74], device="cuda")
    n64, n32 = (n, n.int())
    lengths = n64 if types[0] == torch.int64 else n32
    new = values if types[1] == torch.int64 else near.int()
    want = ts.paged_attention(q, s["kp"], s["vp"], table, n64, near)
    assert torch.equal(ts.paged_attention(q, s["kp"], s["vp"], table, lengths, new), want)
    assert (want[3] == 0).all() and (want[4, :, 2] == 0).all() and (want[:3] != 0).any(-1).all()
    table = s["table"][:, :5].reshape(5, 4)  # (every page once)
    n = torch.tensor([40, 41, 42, 43, 44], device="cuda")
    a, b = ([x.clone() for x in (s["kp"], s["vp"])] for _ in range(2))
    after = ts.paged_cache_append(k, v, *a, table, n.to(types[0]), new)
    assert after.dtype == types[0] and after.tolist() == [43, 44, 45, 43, 46]
    ts.paged_cache_append(k, v, *b, table, n, near)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    if types[0] == torch.int64:  # lengths themselves past 32 bits: as many rows as there is room for, or none
        n = torch.tensor([2**32 + 40, -(2**32) + 41, 42, 43, 44], device="cuda")
        assert ts.paged_cache_append(k, v, *a, table, n, new).tolist() == [64, 3, 45, 43, 46]


@pytest.mark.parametrize("B,cols,budget", [(2, 1700, 9000), (3, 1700, 8000), (2, 2600, 40000)])
def test_graph_of_long_evictions_of_several_sequences(hip_backend, B, cols, budget):
    """Weights searched by parts, rows moved in segments and (8000) in one list, captured and
    replayed on other weights and lengths, one of them below the budget."""
    _, kp, vp, table = make(B, Hk, Hk, 1, cols, SIZE, 16, BF, seed=7)
    L = cols * SIZE
    w, lengths = torch.zeros(B, Hk, L, device="cuda"), torch.full((B,), L, device="cuda")
    graph, (after,) = _capture(lambda: ts.paged_cache_evict(kp, vp, w, table, lengths, budget, 70))
    g = torch.Generator(device="cuda").manual_seed(8)
    for i in range(5):
        x = rand(g, *w.shape).exp()
        w.copy_(x.round() if i % 2 else x)
        lengths.copy_(torch.randint(budget, L + 1, (B,), device="cuda", generator=g))
        lengths[i % B] = budget - i
        k, v, y = kp.clone(), vp.clone(), w.clone()
        graph.replay()
        torch.cuda.synchronize()
        ts.set_backend("pytorch")
        n = ts.paged_cache_evict(k, v, y, table, lengths, budget, 70)
        ts.set_backend("hip")
        torch.cuda.synchronize()
        assert torch.equal(kp, k) and torch.equal(vp, v) and torch.equal(w, y) and torch.equal(after, n)


@pytest.mark.parametrize("dt", [BF, F32])
def test_the_longest_cache(hip_backend, dt):
    """2^30 rows of one sequence, of which three pages are there. All scores are zero, so that
    every key weighs 1 / n and sums of them are exact: results tell which rows were read."""
    cols, n, d = 1 << 26, 1 << 30, 16
    table = torch.full((1, cols), -1, dtype=torch.int32, device="cuda")
    table[0, 0], table[0, cols // 2 + 1], table[0, cols - 1] = 2, 0, 1
    g = torch.Generator(device="cuda").manual_seed(20)
    kp = torch.zeros(3, 1, SIZE, d, dtype=dt, device="cuda")
    vp = torch.randint(-64, 65, (3, 1, SIZE, d), device="cuda", generator=g).to(dt)
    lengths = torch.tensor([n - 3], device="cuda")
    k, v = rand(g, 1, 1, 5, d, dt=dt), torch.ones(1, 1, 5, d, dtype=dt, device="cuda")
    last = vp[1].clone()
    lengths = ts.paged_cache_append(torch.zeros_like(k), v, kp, vp, table, lengths)
    assert lengths.tolist() == [n] and torch.equal(vp[1, :, :13], last[:, :13]) and (vp[1, :, 13:] == 1).all()
    q = rand(g, 1, 2, 40, d, dt=dt)
    total = vp[:, 0].double().sum((0, 1))
    O = ts.paged_attention(q[:, :, :1], kp, vp, table, lengths)
    assert torch.equal(O[0, :, 0].double(), (total / n).to(dt).double().expand(2, -1))
    # Query i of 40 does not see the last 39 - i rows, which lie in the last page and before it.
    # e a rounding of float32: the ranges that have a page hold whole numbers over their number of
    # keys (4 e), and are joined by weights 2^(lse - largest lse) over their sum. An lse is a log2
    # of about 2^24, from 16 to 32, where half a step is 2^-20 = 16 e; logarithm and rounding
    # make it 48 e at most, so that weights and their sum are off by 48 ln 2 < 34 e each.
    O = ts.paged_attention(q, kp, vp, table, lengths)
    pages = [vp[2, 0].double().sum(0), vp[0, 0].double().sum(0)]
    for i in range(40):
        parts = torch.stack([*pages, vp[1, 0, : 16 - min(39 - i, 16)].double().sum(0)]) / (n - 39 + i)
        off = (O[0, :, i].double() - parts.sum(0)).abs()
        far = off - (2 * 34 + 8) * 2.0**-24 * parts.abs().sum(0) - torch.finfo(dt).eps / 2 * parts.sum(0).abs()
        assert far.max() <= 0, (i, float(far.max()))
    w = torch.zeros(1, 1, n, device="cuda")
    O = ts.paged_attention(q[:, :, :1], kp, vp, table, lengths, weights=w)
    assert bool((w == 2.0 / n).all())
    places = [3, 17, n // 2 + 20, n - 30, n - 12]
    w.zero_()
    w[0, 0, places] = torch.arange(1.0, 6.0, device="cuda")
    kept = sorted(places + [j for j in range(20) if j not in places][:11]) + list(range(n - 4, n))
    rows = {0: vp[2, 0].clone(), cols // 2 + 1: vp[0, 0].clone(), cols - 1: vp[1, 0].clone()}
    want = torch.stack([rows[j // SIZE][j % SIZE] if j // SIZE in rows else torch.zeros_like(last[0, 0]) for j in kept[:SIZE]])
    weights = w[0, 0, kept]
    assert ts.paged_cache_evict(kp, vp, w, table, lengths, 20, 4).tolist() == [20]
    assert torch.equal(vp[2, 0], want) and torch.equal(w[0, 0, :20], weights)
