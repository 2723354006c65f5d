"""rotary, decay_attention and token_logprobs in the graph builder, the DSL and
the Python binding, as far as they go without a device, and their 64-bit
restatements against differences and against each other."""
import numpy as np
import pytest

import linear_reference as R
from tysor_b200 import frontend, native
from tysor_b200.programs import linear_lm, random_parameters

SOURCE = """
layer model(q: tensor[float32], k: tensor[float32], v: tensor[float32], pos: tensor[float32], d: tensor[float32], n: tensor[float32], ids: tensor[float32]):
    q = rotary(q, pos, 10000.0, 4, False, True)
    k = rotary(k, pos, 10000.0, 4, True, 3, 8.0, 4096.0, 1.0, 32.0, 1.2, True)
    a = flatten_heads(decay_attention(q, k, v, d, n, True))
    loss = token_logprobs(a, ids, 1.0) + token_entropy(a, 1.0)
    return loss
"""


def test_the_dsl_lowers_the_operators():
    g = frontend.lower(SOURCE)
    assert [n.op for n in g.nodes if n.kind == "call"] == [
        "rotary", "rotary", "decay_attention", "flatten_heads", "token_logprobs", "token_entropy"]
    assert "decay_attention" in g.to_text()


def test_linear_lm_has_its_parameters():
    g = linear_lm(layers=3, d_model=64, n_heads=4, n_kv_heads=2, hidden=96, vocab=50, rotary_dim=8)
    p = random_parameters(g)
    assert sum(n.startswith("linear_") for n in p) == 3 * 7 and sum(n.startswith("embedding_") for n in p) == 1
    assert g.objective == "loss"


def test_a_null_context_is_an_error():
    lib = native.lib()
    calls = [
        ("rotary", [None] * 3 + [1, 1, 1, 8, 8, False, 1e4, 0] + [1.0] * 5 + [False]),
        ("rotary_backward", [None] * 3 + [1, 1, 1, 8, 8, False, 1e4, 0] + [1.0] * 5 + [False, False]),
        ("decay_attention", [None] * 8 + [1] * 6 + [1.0, False]),
        ("decay_attention_backward", [None] * 12 + [1] * 6 + [1.0, False, False]),
        ("token_logprobs", [None] * 7 + [1, 8, 1, 0, 1.0]), ("token_logprobs_backward", [None] * 7 + [1, 8, 1, 1.0, False]),
    ]
    for name, args in calls:
        assert not getattr(lib, "tysor_cuda_dispatch_" + name)(None, *args), name
        assert native.last_error() == "null context"


@pytest.mark.parametrize("seq_major", [False, True])
def test_the_restated_recurrence_and_its_gradients(seq_major):
    rng = np.random.default_rng(0)
    b, h, kv, s, dk, dv = 2, 4, 2, 9, 5, 3
    q, k, v, do = (rng.standard_normal((b, s, n, d) if seq_major else (b, n, s, d))
                   for n, d in ((h, dk), (kv, dk), (kv, dv), (h, dv)))
    decay, state, dnew = np.array([0.0, 0.1, 2.0, np.inf]), rng.standard_normal((b, h, dk, dv)), rng.standard_normal((b, h, dk, dv))
    n = np.array([9, 4])
    r = R.decay_attention(q, k, v, decay, state, n, 0.3, seq_major, do, dnew)
    for i in range(b):
        for j in range(h):
            x = state[i, j].copy()
            for t in range(n[i]):
                qt, kt, vt, ot = ((a[i, t, m] if seq_major else a[i, m, t]) for a, m in
                                  ((q, j), (k, j // 2), (v, j // 2), (r["out"], j)))
                x = np.exp(-decay[j]) * x + np.outer(kt, vt)
                np.testing.assert_allclose(ot, 0.3 * qt @ x, atol=1e-12)
            np.testing.assert_allclose(r["new_state"][i, j], x, atol=1e-12)
    args = dict(q=q, k=k, v=v, state=state)
    for name, grad in (("q", "dq"), ("k", "dk"), ("v", "dv"), ("state", "dstate")):
        d = rng.standard_normal(args[name].shape)
        ends = []
        for sign in (1, -1):
            a = dict(args, **{name: args[name] + sign * d})
            w = R.decay_attention(a["q"], a["k"], a["v"], decay, a["state"], n, 0.3, seq_major)
            ends.append((w["out"] * do).sum() + (w["new_state"] * dnew).sum())
        np.testing.assert_allclose((ends[0] - ends[1]) / 2, (r[grad] * d).sum(), rtol=1e-10, atol=1e-10)


def test_the_restated_rotary_scalings():
    plain = R.rotary_rates(8, 100.0, 0, 1.0, 0.0, 0.0, 0.0)
    np.testing.assert_allclose(R.rotary_rates(8, 100.0, 1, 4.0, 0.0, 0.0, 0.0), plain / 4)
    for kind in (2, 3):
        r = R.rotary_rates(8, 100.0, kind, 4.0, 200.0, 1.0, 8.0)
        turns = 200.0 * plain / (2 * np.pi)
        assert (r[turns >= 8.0] == plain[turns >= 8.0]).all() and np.allclose(r[turns <= 1.0], plain[turns <= 1.0] / 4)
        assert ((r >= plain / 4) & (r <= plain)).all() and (np.diff(r) < 0).all()
