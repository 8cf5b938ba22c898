"""Schemas and Meta implementations of the decoder layer's registered operators
(csrc/torch_ops.cpp): what torch.compile traces with. No GPU."""

from __future__ import annotations

import pytest
import torch

from trnsparse_amd.hip import _lib

if not (_lib.LIB_PATH.exists() and _lib.OPS_PATH.exists()):
    pytest.skip("library not built (run __graft_entry__.build())", allow_module_level=True)

SCHEMAS = {
    "cross_attn_fwd": "(Tensor Q, Tensor K, Tensor V, Tensor? key_lengths, float scale, bool return_lse) -> "
                      "(Tensor, Tensor)",
    "cross_attn_bwd": "(Tensor Q, Tensor K, Tensor V, Tensor O, Tensor grad_out, Tensor lse, Tensor? key_lengths, "
                      "float scale, bool need_kv) -> (Tensor, Tensor, Tensor)",
    "prefix_attn_fwd": "(Tensor Q, Tensor prefix_K, Tensor prefix_V, Tensor K, Tensor V, Tensor? lengths, float scale) "
                       "-> Tensor",
    "qk_norm_rope_fwd": "(Tensor Q, Tensor K, Tensor q_weight, Tensor k_weight, Tensor positions, Tensor inv_freq, "
                        "float eps, bool interleaved) -> (Tensor, Tensor)",
    "qk_norm_rope_bwd": "(Tensor Q, Tensor K, Tensor q_weight, Tensor k_weight, Tensor positions, Tensor inv_freq, "
                        "float eps, bool interleaved, Tensor grad_Q, Tensor grad_K, bool need_weights) -> (Tensor, "
                        "Tensor, Tensor, Tensor)",
    "cross_attention": "(Tensor Q, Tensor K, Tensor V, Tensor? key_lengths, float scale) -> Tensor",
    "qk_norm_rope": "(Tensor Q, Tensor K, Tensor q_weight, Tensor k_weight, Tensor positions, Tensor inv_freq, "
                    "float eps, bool interleaved) -> (Tensor, Tensor)",
}


@pytest.mark.parametrize("name", SCHEMAS)
def test_schema(name):
    assert str(getattr(_lib.ops(), name).default._schema) == f"trnsparse_hip::{name}{SCHEMAS[name]}"


def meta(*shape, dt=torch.bfloat16):
    return torch.empty(*shape, dtype=dt, device="meta")


def test_attention_shapes_and_orders():
    ops = _lib.ops()
    Q = meta(2, 70, 8, 64).transpose(1, 2)  # heads of a projection
    K = meta(2, 2, 90, 64)
    O, lse = ops.cross_attn_fwd(Q, K, K, None, 0.1, True)
    assert O.shape == Q.shape and O.stride() == Q.stride() and lse.shape == (2, 8, 70) and lse.dtype == torch.float32
    assert ops.cross_attention(Q, K, K, None, 0.1).stride() == Q.stride()
    dQ, dK, dV = ops.cross_attn_bwd(Q, K, K, O, O, lse, None, 0.1, True)
    assert dQ.stride() == Q.stride() and dK.shape == dV.shape == K.shape and dK.is_contiguous()
    assert ops.cross_attn_bwd(Q, K, K, O, O, lse, None, 0.1, False)[1].numel() == 0
    odd = meta(1, 2, 5, 7)  # head_dim padded within: contiguous results
    assert ops.cross_attention(odd, odd, odd, None, 0.1).shape == odd.shape
    assert ops.prefix_attn_fwd(Q, meta(2, 40, 64), meta(2, 40, 64), K, K, None, 0.1).stride() == Q.stride()


def test_norm_rope_shapes():
    ops = _lib.ops()
    Q, K = meta(2, 70, 8, 64).transpose(1, 2), meta(2, 2, 70, 64)
    w, pos, f = meta(64), meta(70, dt=torch.int64), meta(32, dt=torch.float64)
    for op in (ops.qk_norm_rope, ops.qk_norm_rope_fwd):
        q, k = op(Q, K, w, w, pos, f, 1e-6, False)
        assert q.shape == Q.shape and q.is_contiguous() and k.shape == K.shape and k.dtype == K.dtype
    dQ, dK, dwq, dwk = ops.qk_norm_rope_bwd(Q, K, w, w, pos, f, 1e-6, False, q, k, True)
    assert dQ.stride() == Q.stride() and dK.shape == K.shape and dwq.shape == dwk.shape == (64,)
    assert ops.qk_norm_rope_bwd(Q, K, w, w, pos, f, 1e-6, False, q, k, False)[2].numel() == 0
