"""The operators of a decoder layer together, as a model uses them: a training
step (norm and rotation, block-sparse self attention, cross attention) and a
serving loop (norm and rotation of the new token, its cache, attention behind a
shared prefix), captured and replayed, traced, from several streams.

fp32 runs are held to the same chain in float64 on the "pytorch" backend. Each
operator is within (4 D + 4 L) e of its error scale (D = 64, L <= 384, e =
2^-24: about 1e-4) and the scales of random data are within a few times the
values, so relative 2-norms stay below 1e-3 through three operators and back.
"""

from __future__ import annotations

import threading

import pytest
import torch

import trnsparse_amd as ts
from oracle import layer
from test_gpu_graphs import _capture, _grads_replay_match, _replays_match
from trnsparse_amd import workloads as W
from trnsparse_amd.hip import _lib

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
B, H, Hk, S, L, D = 2, 4, 4, 384, 200, 64


def _layer(p, x, enc, pos, lengths, mask):
    """x (B, S, E) through self attention and cross attention to enc (B, L, E)."""
    b, s, e = x.shape
    qkv = (x @ p["qkv"]).view(b, s, 3 * H, D)
    q, k, v = qkv[:, :, :H].transpose(1, 2), qkv[:, :, H : 2 * H].transpose(1, 2), qkv[:, :, 2 * H :].transpose(1, 2)
    q, k = ts.qk_norm_rope(q, k, p["wq"], p["wk"], pos, p["freq"])
    h = ts.block_sparse_attention_tiled(q, k, v.contiguous(), mask)
    x = x + h.transpose(1, 2).reshape(b, s, e) @ p["o"]
    q2 = (x @ p["q2"]).view(b, s, H, D).transpose(1, 2)
    kv = (enc @ p["kv2"]).view(b, -1, 2, H, D)
    c = ts.cross_attention(q2, kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2), lengths)
    return x + c.transpose(1, 2).reshape(b, s, e)


def _setup(dt, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    e = H * D
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    p = {"qkv": r(e, 3 * e) / e**0.5, "o": r(e, e) / e**0.5, "q2": r(e, e) / e**0.5, "kv2": r(e, 2 * e) / e**0.5,
         "wq": 1 + 0.1 * r(D), "wk": 1 + 0.1 * r(D)}
    p = {k: t.to(dt).to(dev).requires_grad_() for k, t in p.items()}
    p["freq"] = ts.rope_frequencies(D, device=dev)
    x, enc, dy = (t.to(dt).to(dev) for t in (r(B, S, e), r(B, L, e), r(B, S, e)))
    return p, x.requires_grad_(), enc.requires_grad_(), dy


def test_training_step(hip_backend):
    mask = W.bsr_from_block_mask(torch.tril(torch.ones(3, 3)).bool(), 128)
    lengths = torch.tensor([L, 77])
    pos = torch.arange(S)
    res = {}
    for dt, dev in ((F32, "cuda"), (torch.float64, "cpu")):
        ts.set_backend("hip" if dev == "cuda" else "pytorch")
        try:
            p, x, enc, dy = _setup(dt, dev)
            y = _layer(p, x, enc, pos.to(dev), lengths.to(dev), mask)
            leaves = [x, enc] + [p[k] for k in ("qkv", "o", "q2", "kv2", "wq", "wk")]
            res[dev] = [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
        finally:
            ts.set_backend("hip")
    for got, want in zip(res["cuda"], res["cpu"]):
        got = got.double().cpu()
        assert (got - want).norm() <= 1e-3 * want.norm()
    enc_grad = res["cuda"][2]
    assert (enc_grad[1, 77:] == 0).all()  # padded encoder states get none


def test_training_step_in_16_bits(hip_backend):
    """bf16 and fp16 steps run and give finite gradients everywhere."""
    mask = W.bsr_from_block_mask(torch.tril(torch.ones(3, 3)).bool(), 128)
    for dt in (BF, HF):
        p, x, enc, dy = _setup(dt, "cuda")
        y = _layer(p, x, enc, torch.arange(S, device="cuda"), torch.tensor([L, 77], device="cuda"), mask)
        grads = torch.autograd.grad(y, [x, enc, p["wq"], p["kv2"]], dy)
        assert all(t.isfinite().all() for t in (y, *grads))


def _serve(q, k, v, w, freq, prefix, cache, lengths, steps, P):
    """`steps` new tokens of every sequence, one at a time, behind the prefix."""
    outs = []
    for i in range(steps):
        qi, ki = ts.qk_norm_rope(q[:, :, i : i + 1], k[:, :, i : i + 1], w, w, (P + lengths).unsqueeze(1), freq)
        at = lengths.view(-1, 1, 1, 1).expand(-1, k.shape[1], 1, D)
        cache[0].scatter_(2, at, ki)
        cache[1].scatter_(2, at, v[:, :, i : i + 1])
        lengths += 1
        outs.append(ts.shared_prefix_attention(qi, *prefix, *cache, lengths))
    return torch.cat(outs, 2)


def test_serving_loop(hip_backend):
    """Token by token behind a shared prefix equals attention over the whole
    sequences, and all new tokens checked at once equals token by token."""
    nb, nh, nk, P, steps, room = 3, 8, 2, 130, 5, 40
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    pk, pv, w, freq = r(nk, P, D), r(nk, P, D), 1 + 0.1 * r(D), ts.rope_frequencies(D, device="cuda")
    zero = torch.zeros(1, 0, P, D, device="cuda")
    pk = ts.qk_norm_rope(zero, pk[None], w, w, torch.arange(P, device="cuda"), freq)[1][0]
    cache = [r(nb, nk, room, D), r(nb, nk, room, D)]
    start = torch.tensor([0, 7, 30], device="cuda")
    q, k, v = r(nb, nh, steps, D), r(nb, nk, steps, D), r(nb, nk, steps, D)
    lengths = start.clone()
    out = _serve(q, k, v, w, freq, (pk, pv), cache, lengths, steps, P)
    # the same in float64, over prefix and cache as they now are
    posn = P + start.view(-1, 1) + torch.arange(steps, device="cuda")
    qr = layer.norm_rope(q, w, posn, freq, 1e-6, False)["y"]
    seen = torch.cat([torch.ones(nb, steps, P, dtype=torch.bool), layer.lengths_seen(lengths, steps, room, causal=True)], 2)
    keys, vals = (torch.cat([a.expand(nb, -1, -1, -1), c], 2) for a, c in ((pk, cache[0]), (pv, cache[1])))
    want = layer.attention(qr, keys, vals, D**-0.5, seen)["O"]
    assert (out.double().cpu() - want).norm() <= 1e-4 * want.norm()
    qa, _ = ts.qk_norm_rope(q, k, w, w, posn, freq)
    once = ts.shared_prefix_attention(qa, pk, pv, *cache, lengths)
    assert (once - out).norm() <= 1e-5 * out.norm()


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("P", [100, 3000])
def test_graph_of_a_decoding_step(hip_backend, dt, P):
    """One captured step, replayed as the sequences grow: lengths, positions and
    caches are read at every replay."""
    nb, nh, nk, room = 4, 8, 2, 900
    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dt)  # noqa: E731
    pk, pv, w, freq = r(nk, P, D), r(nk, P, D), r(D), ts.rope_frequencies(D, device="cuda")
    first = [r(nb, nk, room, D), r(nb, nk, room, D)]
    q, k, v = r(nb, nh, 1, D), r(nb, nk, 1, D), r(nb, nk, 1, D)
    enc = r(nb, nk, 333, D)
    encl = torch.tensor([333, 1, 0, 64], device="cuda")
    cache, lengths = [t.clone() for t in first], torch.tensor([0, 3, 500, 800], device="cuda")

    def step():
        o = _serve(q, k, v, w, freq, (pk, pv), cache, lengths, 1, P)
        return o, ts.cross_attention(o, enc, enc, encl)

    start = lengths.clone()
    graph, outs = _capture(step)
    for t, f in zip(cache, first):
        t.copy_(f)
    lengths.copy_(start)
    ecache, elen = [t.clone() for t in first], start.clone()
    for _ in range(4):
        for t in (q, k, v):
            t.copy_(r(*t.shape))
        encl.add_(7)
        graph.replay()
        torch.cuda.synchronize()
        o = _serve(q, k, v, w, freq, (pk, pv), ecache, elen, 1, P)
        want = (o, ts.cross_attention(o, enc, enc, encl))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)) and torch.equal(lengths, elen)


def test_graphs_that_share_nothing(hip_backend):
    """Two captured calls that split their keys, replayed in turn and at the same
    time on two streams: each has its own workspace."""
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF)  # noqa: E731
    sets = [(r(1, 4, 1, D), r(1, 4, 5000, D), r(1, 4, 5000, D)) for _ in range(2)]
    want = [ts.cross_attention(*s) for s in sets]
    graphs = [_capture(lambda s=s: ts.cross_attention(*s)) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        for (graph, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out[0], w) for (_, out), w in zip(graphs, want))


@pytest.mark.parametrize("dt", [BF, HF, F32])
def test_graph_cross_attention_backward(hip_backend, dt):
    g = torch.Generator(device="cuda").manual_seed(4)
    for shapes in (((2, 4, 70, D), (2, 2, 300, D)), ((1, 2, 500, 128), (1, 2, 600, 128))):
        leaves = [torch.randn(s, device="cuda", generator=g).to(dt).requires_grad_(True)
                  for s in (shapes[0], shapes[1], shapes[1])]
        lengths = torch.arange(1, shapes[0][0] + 1, device="cuda") * 150
        _grads_replay_match(lambda q, k, v: ts.cross_attention(q, k, v, lengths), leaves, shapes[0], dt, 5)


@pytest.mark.parametrize("dt", [BF, F32])
def test_graph_qk_norm_rope(hip_backend, dt):
    g = torch.Generator(device="cuda").manual_seed(6)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dt)  # noqa: E731
    f, pos = ts.rope_frequencies(D, device="cuda"), torch.arange(300, device="cuda")
    sets = [(r(2, 4, 300, D), r(2, 2, 300, D), r(D), r(D)) for _ in range(4)]
    _replays_match(lambda: ts.qk_norm_rope(*sets[0], pos, f), sets[0], sets[1:],
                   lambda *t: ts.qk_norm_rope(*t, pos, f))
    leaves = [r(2, 4, 300, D).requires_grad_(True), r(D).requires_grad_(True)]
    _grads_replay_match(lambda q, w: ts.qk_norm_rope(q, sets[1][1], w, w, pos, f)[0], leaves, (2, 4, 300, D), dt, 7)


def test_capture_beside_an_eager_graph(hip_backend):
    """A training step is not captured while an eager graph of the same leaves
    lives: refused before it records anything; released, it is captured."""
    g = torch.Generator(device="cuda").manual_seed(10)
    Q, K, V = (torch.randn(1, 2, 40, D, device="cuda", generator=g).requires_grad_() for _ in range(3))
    w, pos, f = torch.ones(D, device="cuda"), torch.arange(40, device="cuda"), ts.rope_frequencies(D, device="cuda")
    for fn in (lambda: ts.cross_attention(Q, K, V), lambda: ts.qk_norm_rope(Q, K, w, w, pos, f)[0]):
        held = fn()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="release it before the capture"):
            with torch.cuda.graph(graph):
                fn()
        with torch.no_grad(), torch.cuda.graph(torch.cuda.CUDAGraph()):
            fn()  # (no gradients: nothing to join)
        want = torch.autograd.grad(held, Q, torch.ones_like(held))[0]
        del held
        ones = torch.ones_like(want)
        graph, (got,) = _capture(lambda: torch.autograd.grad(fn(), Q, ones)[0])
        for _ in range(2):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


def test_two_threads_two_streams(hip_backend):
    """Calls from two threads, each on its own stream, do not disturb each other."""
    g = torch.Generator(device="cuda").manual_seed(8)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF)  # noqa: E731
    sets = [(r(2, 8, 1, D), r(2, 2, 3000, D), r(2, 2, 3000, D)) for _ in range(2)]
    want = [ts.cross_attention(*s) for s in sets]
    torch.cuda.synchronize()
    bad = []

    def run(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(30):
                got = ts.cross_attention(*sets[i])
                st.synchronize()
                if not torch.equal(got, want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_no_second_derivatives(hip_backend):
    Q, K, V = (torch.randn(1, 2, 5, D, device="cuda", requires_grad=True) for _ in range(3))
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(ts.cross_attention(Q, K, V).sum(), Q, create_graph=True)
    w = torch.ones(D, device="cuda")
    out = ts.qk_norm_rope(Q, K, w, w, torch.arange(5, device="cuda"), ts.rope_frequencies(D, device="cuda"))
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(out[0].sum(), Q, create_graph=True)


def test_traced_and_compiled(hip_backend):
    """torch.compile reaches the operators whole (with their gradients) and the
    public functions by graph breaks; results equal eager calls."""
    ops = _lib.ops()
    g = torch.Generator(device="cuda").manual_seed(9)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    Q, K, V = r(1, 4, 20, D), r(1, 2, 30, D), r(1, 2, 30, D)
    w, pos, f = r(D), torch.arange(20, device="cuda"), ts.rope_frequencies(D, device="cuda")

    def whole(q, k, v):
        q2, _ = ops.qk_norm_rope(q, q, w, w, pos, f, 1e-6, False)
        return ops.cross_attention(q2 * 2.0, k, v, None, 0.125) + 1.0

    def public(q, k, v):
        q2, _ = ts.qk_norm_rope(q, q, w, w, pos, f)
        return ts.cross_attention(q2 * 2.0, k, v, None, 0.125) + 1.0

    want = whole(Q, K, V)
    assert torch.equal(torch.compile(whole, fullgraph=True, backend="aot_eager")(Q, K, V), want)
    assert torch.equal(torch.compile(public, backend="aot_eager")(Q, K, V), want)
    leaves = [t.clone().requires_grad_() for t in (Q, K, V)]
    a = torch.autograd.grad(public(*leaves).sum(), leaves)
    b = torch.autograd.grad(torch.compile(public, backend="aot_eager")(*leaves).sum(), leaves)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
