"""The language-model operators in the graph builder, the DSL and the Python
binding, as far as they go without a device."""
import ctypes

import numpy as np
import pytest

from tysor_b200 import native
from tysor_b200.graph import GraphBuilder
from tysor_b200.programs import random_parameters, student_lm
from tysor_b200.runtime import CudaContext, DeviceBuffer

SOURCE = """
layer model(q: tensor[float32], k: tensor[float32], v: tensor[float32], pos: tensor[float32], n: tensor[float32], ids: tensor[float32], best: tensor[float32]):
    norm = LayerNorm(8, 0.001)
    q = rope_axes(norm(q), pos, 10000.0, 1, 3, True)
    a = window_attention(q, k, v, 4, 1, n, True)
    h = flatten_heads(a)
    loss = distill_loss(h, ids, best, 2.0)
    return loss
"""


def test_the_dsl_lowers_the_operators():
    from tysor_b200 import frontend
    g = frontend.lower(SOURCE)
    assert [n.op for n in g.nodes if n.kind in ("call", "ctor")] == [
        "LayerNorm", "rope_axes", "window_attention", "flatten_heads", "distill_loss"]
    text = g.to_text()
    for op in ("ctor", "call"):
        assert f"node {op}" in text


def test_the_builder_refuses_unknown_constructors():
    b = GraphBuilder()
    with pytest.raises(ValueError, match="unknown layer constructor"):
        b.ctor("GroupNorm", 8)


def test_student_lm_has_its_parameters():
    g = student_lm(layers=2, d_model=64, n_heads=4, n_kv_heads=2, hidden=96, vocab=50, sections=(2, 3, 3))
    p = random_parameters(g)
    norms = [n for n in p if n.startswith("layernorm_")]
    assert len(norms) == 2 * 5 and all(p[n].shape == (64,) for n in norms)
    assert g.objective == "loss"
    with pytest.raises(ValueError, match="pairs of a head"):
        student_lm(d_model=64, n_heads=4, sections=(8, 8))


def test_a_null_context_is_an_error():
    lib = native.lib()
    one = (ctypes.c_int64 * 1)(1)
    calls = [
        ("layer_norm", [None] * 5 + [1, 1, 1e-5]), ("layer_norm_backward", [None] * 7 + [1, 1, False]),
        ("rope_axes", [None] * 3 + [1, 1, 1, one, 1, 1e4, False]),
        ("rope_axes_backward", [None] * 3 + [1, 1, 1, one, 1, 1e4, False, False]),
        ("window_attention", [None] * 7 + [1] * 6 + [0, 0, 1.0, False]),
        ("window_attention_backward", [None] * 11 + [1] * 6 + [0, 0, 1.0, False, False]),
        ("distill_loss", [None] * 5 + [1, 1, 1, 1.0]), ("distill_loss_backward", [None] * 6 + [1, 1, 1, 1.0, False]),
    ]
    for name, args in calls:
        assert not getattr(lib, "tysor_cuda_dispatch_" + name)(None, *args), name
        assert native.last_error() == "null context"
    assert not lib.tysor_cuda_buffer_wrap(None, None, 1)
    assert native.last_error() == "null context"


def test_wrap_refuses_what_it_cannot_see_as_floats():
    class Face:
        def __init__(self, a, **over):
            self.__cuda_array_interface__ = {"shape": a.shape, "typestr": a.dtype.str, "data": (a.ctypes.data, False),
                                             "strides": a.strides, "version": 3, **over}

    with pytest.raises(ValueError, match="float32"):
        DeviceBuffer.wrap(None, Face(np.zeros(4)))
    with pytest.raises(ValueError, match="contiguous"):
        DeviceBuffer.wrap(None, Face(np.zeros((4, 6), np.float32)[:, :3]))
    with pytest.raises(ValueError, match="contiguous"):
        DeviceBuffer.wrap(None, Face(np.zeros((4, 6), np.float32).T))
