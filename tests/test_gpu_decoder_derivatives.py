"""Derivatives of the decoder layer's operators that they do not have are refused,
not answered with zeros; those that they have also trace whole."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import trnsparse_amd as ts
from test_gpu_graphs import _capture
from trnsparse_amd.hip import _lib

pytestmark = pytest.mark.gpu

D = 64


def _operators():
    """(call, inputs that could carry a derivative)"""
    g = torch.Generator(device="cuda").manual_seed(12)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    pos, f = torch.arange(5, device="cuda"), ts.rope_frequencies(D, device="cuda")
    heads = (r(2, 4, 5, D), r(2, 2, 5, D))
    return [
        (ts.cross_attention, (*heads, r(2, 2, 5, D))),
        (lambda *t: ts.qk_norm_rope(*t[:4], pos, t[4])[0], (*heads, r(D), r(D), f)),
        (ts.shared_prefix_attention, (heads[0], r(2, 7, D), r(2, 7, D), heads[1], r(2, 2, 5, D))),
    ]


@pytest.mark.parametrize("which", range(3))
def test_forward_mode_is_refused(hip_backend, which):
    """No operator has forward-mode derivatives: an input with a tangent is
    refused, whichever it is, not answered with a tangent of zero."""
    fn, inputs = _operators()[which]
    want = fn(*inputs)
    with fwAD.dual_level():
        assert torch.equal(fn(*inputs), want)
        for i in range(len(inputs)):
            args = list(inputs)
            args[i] = fwAD.make_dual(inputs[i], torch.ones_like(inputs[i]))
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    fn(*args)
    ones = tuple(torch.ones_like(t) for t in inputs)
    for call in (lambda: torch.func.jvp(fn, inputs, ones), lambda: torch.func.vjp(fn, *inputs),
                 lambda: torch.func.grad(lambda q: fn(q, *inputs[1:]).sum())(inputs[0])):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("which", range(2))
def test_forward_mode_of_a_gradient_is_refused(hip_backend, which):
    fn, inputs = _operators()[which]
    q = inputs[0].clone().requires_grad_()
    out = fn(q, *inputs[1:])
    with fwAD.dual_level():
        dual = fwAD.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, q, dual)


def test_frequencies_have_no_gradient(hip_backend):
    """inv_freq that asks for a gradient is refused, in either float type and
    whatever else asks for one; under no_grad it is taken."""
    fn, inputs = _operators()[1]
    for f in (inputs[4], inputs[4].float()):
        for q in (inputs[0], inputs[0].clone().requires_grad_()):
            with pytest.raises(RuntimeError, match="inv_freq"):
                fn(q, *inputs[1:4], f.clone().requires_grad_())
        with torch.no_grad():
            fn(*inputs[:4], f.clone().requires_grad_())


def test_capture_from_leaves_that_an_eager_graph_holds(hip_backend):
    """The operators' inputs come from a fused projection within the capture:
    an eager graph of its leaves is found there too, and refused before anything
    is recorded; one of other leaves does not matter, and released, the step is
    captured."""
    g = torch.Generator(device="cuda").manual_seed(14)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x, W, other = r(1, 40, 32), r(32, 6 * D).requires_grad_(), r(D).requires_grad_()
    pos, f = torch.arange(40, device="cuda"), ts.rope_frequencies(D, device="cuda")

    def heads():
        q, k, v = ((x @ W).view(1, 40, 6, D)[:, :, 2 * i : 2 * i + 2].transpose(1, 2) for i in range(3))
        return q, k, v

    for fn in (lambda: ts.cross_attention(*heads()), lambda: ts.qk_norm_rope(*heads()[:2], other, other, pos, f)[0]):
        held = fn()
        with pytest.raises(RuntimeError, match="release it before the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                fn()
        ones = torch.ones_like(held)
        want = torch.autograd.grad(held, W, ones)[0]
        del held
        apart = (r(D).requires_grad_() * 2).sum()
        graph, (got,) = _capture(lambda: torch.autograd.grad(fn(), W, ones)[0])
        for _ in range(2):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
        del apart


def test_fullgraph_with_gradients(hip_backend):
    """The operators trace whole with their gradients, in one graph."""
    ops = _lib.ops()
    g = torch.Generator(device="cuda").manual_seed(13)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    w, pos, f = r(D), torch.arange(20, device="cuda"), ts.rope_frequencies(D, device="cuda")

    def whole(q, k, v, wq):
        q2, k2 = ops.qk_norm_rope(q, k, wq, w, pos, f, 1e-6, False)
        return ops.cross_attention(q2 * 2.0, k2, v, None, 0.125) + 1.0

    leaves = [t.requires_grad_() for t in (r(1, 4, 20, D), r(1, 2, 20, D), r(1, 2, 20, D), r(D))]
    out = whole(*leaves)
    want = torch.autograd.grad(out, leaves, torch.ones_like(out))
    traced = torch.compile(whole, fullgraph=True, backend="aot_eager")(*leaves)
    got = torch.autograd.grad(traced, leaves, torch.ones_like(out))
    assert torch.equal(traced, out) and all(torch.equal(a, b) for a, b in zip(got, want))
