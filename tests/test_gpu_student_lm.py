"""The language-model operators together, as a program uses them: the student
language model (programs.student_lm) through the graph executor against the
same model in 64 bits (torch on the CPU, exact gradients), and the operators'
gradients in --backward mode.

Bars: values 1e-5 and gradients 3e-5 of the tensor's norm, the strict
matmuls' own (each product loses up to 1.4e-6 to the tensor core's rounding
toward zero, and a gradient chains a dozen of them)."""
import numpy as np
import pytest

from tysor_b200.graph import GraphBuilder
from tysor_b200.programs import random_parameters, student_lm
from tysor_b200.runtime import CudaGraphExecutor

import lm_reference as R

pytestmark = pytest.mark.gpu

CFG = dict(layers=2, batch=3, seq=150, d_model=256, n_heads=4, n_kv_heads=2, hidden=384, vocab=500, window=40, sinks=3,
           sections=(8, 12, 12), temperature=2.0)
TOP = 9


def data(seed=0):
    rng = np.random.default_rng(seed)
    b, s, v = CFG["batch"], CFG["seq"], CFG["vocab"]
    lengths = np.array([s, 61, 0], np.float32)
    ids = rng.integers(0, v, b * s).astype(np.float32)
    pos = (np.arange(s)[None, None] + rng.integers(0, 30, (b, 3, s))).astype(np.float32)
    tid = np.stack([rng.permutation(v)[:TOP] for _ in range(b * s)]).astype(np.float32)
    tid[rng.random((b * s, TOP)) < 0.2] = -1
    for i in range(b):
        tid.reshape(b, s, TOP)[i, int(lengths[i]):] = -1
    teacher = (2 * rng.standard_normal((b * s, TOP))).astype(np.float32)
    return dict(ids=ids, positions=pos, lengths=lengths, teacher_ids=tid, teacher=teacher)


def reference(graph, inputs, params):
    """Loss terms and gradients of every parameter, in float64 with torch's autograd."""
    import torch
    P = {n: torch.tensor(a, dtype=torch.float64, requires_grad=True) for n, a in params.items()}
    c = CFG
    b, s, hd = c["batch"], c["seq"], c["d_model"] // c["n_heads"]
    half = hd // 2
    ctor = iter([n for n in graph.nodes if n.kind == "ctor"])
    emb = P[f"embedding_{next(ctor).output}_weight"]
    axis = np.repeat(np.arange(3), c["sections"])
    angle = torch.tensor(np.moveaxis(inputs["positions"].astype(np.float64)[:, axis], 1, 2)
                         * 10000.0 ** (-np.arange(half) / half))[:, :, None]
    seen = torch.tensor(R.visible(np.zeros(b), inputs["lengths"], b, s, s, c["window"], c["sinks"]))[:, None]

    def norm(x, n):
        m = x.mean(1, keepdim=True)
        d = (x - m) / ((x - m).pow(2).mean(1, keepdim=True) + 1e-5).sqrt()
        return d * P[f"layernorm_{n.output}_gain"] + P[f"layernorm_{n.output}_bias"]

    def lin(x, n):
        return x @ P[f"linear_{n.output}_weight"]

    def turn(x):
        l, h = x[..., :half], x[..., half:]
        return torch.cat((l * angle.cos() - h * angle.sin(), l * angle.sin() + h * angle.cos()), -1)

    x = emb[torch.tensor(inputs["ids"].astype(np.int64))]
    for _ in range(c["layers"]):
        n1, qp, kp, vp, op, n2, gp, up, dp, _act = (next(ctor) for _ in range(10))
        hn = norm(x, n1)
        group = c["n_heads"] // c["n_kv_heads"]
        q = turn(lin(hn, qp).reshape(b, s, c["n_heads"], hd)).transpose(1, 2)
        k = turn(lin(hn, kp).reshape(b, s, c["n_kv_heads"], hd)).transpose(1, 2).repeat_interleave(group, 1)
        v = lin(hn, vp).reshape(b, s, c["n_kv_heads"], hd).transpose(1, 2).repeat_interleave(group, 1)
        w = (q @ k.transpose(2, 3) / hd ** 0.5).masked_fill(~seen, -1e300)
        o = (torch.softmax(w, -1) * seen) @ v
        h = x + lin(o.transpose(1, 2).reshape(b * s, -1), op)
        hn2 = norm(h, n2)
        x = h + lin(torch.nn.functional.silu(lin(hn2, gp)) * lin(hn2, up), dp)
    logits = norm(x, next(ctor)) @ emb.T
    t = c["temperature"]
    tid = torch.tensor(inputs["teacher_ids"].astype(np.int64))
    here = tid >= 0
    best = torch.tensor(inputs["teacher"].astype(np.float64)) / t
    log_p = torch.log_softmax(best.masked_fill(~here, -1e300), 1)
    log_q = torch.log_softmax(logits / t, 1).gather(1, tid.clamp_min(0))
    loss = t * t * torch.where(here, log_p.exp() * (log_p - log_q), 0.0).sum(1)
    grads = torch.autograd.grad(loss.sum(), list(P.values()))
    return loss.detach().numpy(), dict(zip(P, (g.numpy() for g in grads)))


def off(got, want):
    got, want = np.asarray(got, np.float64).reshape(-1), np.asarray(want, np.float64).reshape(-1)
    return float(np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-300))


def shapes():
    b, s = CFG["batch"], CFG["seq"]
    return {"ids": [b * s], "positions": [b, 3, s], "lengths": [b], "teacher_ids": [b * s, TOP], "teacher": [b * s, TOP]}


def test_student_lm_trains_as_in_64_bits(cuda_ctx):
    lr, steps = 0.002, 3
    g = student_lm(**CFG, lr=lr, iterations=steps)
    inputs, params = data(), random_parameters(g, std=0.05)
    ex = CudaGraphExecutor(cuda_ctx, g, shapes(), inputs, params)
    mine = {n: a.astype(np.float64) for n, a in params.items()}
    for step in range(steps):  # the first step runs eagerly, the others replay its captured graph
        want, grads = reference(g, inputs, mine)
        loss = ex.train(1, lr)[0]
        assert abs(loss - want.sum()) <= 1e-5 * abs(want.sum()), step
        for n in grads:
            assert off(ex.parameter_grad(n), np.asarray(grads[n])) < 3e-5, (step, n)
            mine[n] = mine[n] - lr * grads[n]
            assert off(ex.parameter(n), mine[n]) < 1e-5, (step, n)
    per_row = ex.value(g.outputs[0]).data
    padded = (inputs["teacher_ids"] < 0).all(1)
    assert padded.any() and not per_row[padded].any()
    ex.close()


def test_student_lm_runs_and_captured_steps_repeat(cuda_ctx):
    g = student_lm(**CFG)
    inputs, params = data(1), random_parameters(g, std=0.05)
    results = []
    for capture in (True, False, True):
        ex = CudaGraphExecutor(cuda_ctx, g, shapes(), inputs, params)
        ex.set_capture(capture)
        results.append((ex.train(4, 1e-3), ex.parameters()))
        ex.close()
    for losses, p in results[1:]:
        assert losses == results[0][0]
        assert all(np.array_equal(p[n], results[0][1][n]) for n in p)
    # Two executors of one context in turn: each has its own workspace.
    a = CudaGraphExecutor(cuda_ctx, g, shapes(), inputs, params)
    b = CudaGraphExecutor(cuda_ctx, g, shapes(), data(2), params)
    got = []
    for _ in range(4):
        got.append(a.train(1, 1e-3)[0])
        b.train(1, 1e-3)
    assert got == results[0][0]
    a.close()
    b.close()
    # --run: the constant weights of an inference graph.
    ex = CudaGraphExecutor(cuda_ctx, g, shapes(), inputs)
    out = ex.run()
    assert out.shape == [CFG["batch"] * CFG["seq"], 1] and np.isfinite(out.data).all()
    ex.close()


@pytest.mark.parametrize("same", [False, True])
def test_backward_mode_reports_exact_gradients(cuda_ctx, same):
    """--backward on the operators alone, one value read as keys and values among them."""
    b = GraphBuilder()
    x, k, v, pos = b.param("x"), b.param("k"), b.param("v"), b.param("pos")
    n = b.apply(b.ctor("LayerNorm", 32, 1e-5), x)
    q = b.call("rope_axes", n, pos, 100.0, 6, 10)
    b.ret(b.call("window_attention", q, k, k if same else v, 5, 1))
    g = b.build()
    rng = np.random.default_rng(4)
    data = {n: rng.standard_normal(s).astype(np.float32) for n, s in
            (("x", (2, 4, 20, 32)), ("k", (2, 2, 20, 32)), ("v", (2, 2, 20, 32)))}
    data["pos"] = rng.integers(0, 99, (2, 2, 20)).astype(np.float32)
    ex = CudaGraphExecutor(cuda_ctx, g, {n: list(a.shape) for n, a in data.items()}, data)
    got = {n: t.data for n, t in ex.backward()}
    ex.close()
    flat = data["x"].reshape(-1, 32)
    norm = R.layer_norm(flat, None, None, 1e-5)["y"].reshape(data["x"].shape)
    qq = R.rope_axes(norm, data["pos"], (6, 10), 100.0, False)
    ones = np.ones(qq.shape)
    vv = data["k"] if same else data["v"]
    r = R.window_attention(qq, data["k"], vv, None, None, 5, 1, 32 ** -0.5, False, ones)
    dn = R.rope_axes(r["dq"], data["pos"], (6, 10), 100.0, False, back=True)
    dx = R.layer_norm(flat, None, None, 1e-5, dn.reshape(-1, 32))["dx"]
    assert off(got["x_grad"], dx) < 3e-5
    assert off(got["k_grad"], r["dk"] + r["dv"] if same else r["dk"]) < 3e-5
    if not same:
        assert off(got["v_grad"], r["dv"]) < 3e-5
    assert not got["pos_grad"].any()


def test_graph_refusals(cuda_ctx):
    from tysor_b200.native import NativeError

    def plan(message, shapes, make):
        b = GraphBuilder()
        p = {n: b.param(n) for n in shapes}
        b.ret(make(b, p))
        ex = CudaGraphExecutor(cuda_ctx, b.build(), shapes)
        with pytest.raises(NativeError, match=message):
            ex.run()
        ex.close()

    x, kv = [1, 2, 8, 16], [1, 1, 8, 16]
    plan("rank 4", {"q": x, "k": kv, "v": [1, 1, 9, 16]},
         lambda b, p: b.call("window_attention", p["q"], p["k"], p["v"], 4, 0))
    plan("one length", {"q": x, "k": kv, "v": kv, "n": [2]},
         lambda b, p: b.call("window_attention", p["q"], p["k"], p["v"], 4, 0, p["n"]))
    plan("window >= 0", {"q": x, "k": kv, "v": kv},
         lambda b, p: b.call("window_attention", p["q"], p["k"], p["v"], -1, 0))
    plan("1 to 128 values", {"q": [1, 1, 2, 130], "k": [1, 1, 2, 130], "v": [1, 1, 2, 130]},
         lambda b, p: b.call("window_attention", p["q"], p["k"], p["v"], 0, 0))
    plan("heads of 16", {"x": [1, 2, 8, 18], "p": [1, 2, 8]},
         lambda b, p: b.call("rope_axes", p["x"], p["p"], 1e4, 4, 4))
    plan("positions", {"x": x, "p": [1, 8]}, lambda b, p: b.call("rope_axes", p["x"], p["p"], 1e4, 4, 4))
    plan("1 to 8 sections", {"x": x, "p": [1, 8]}, lambda b, p: b.call("rope_axes", p["x"], p["p"], 1e4))
    plan("ids and teacher", {"z": [4, 30], "i": [4, 3], "t": [4, 2]},
         lambda b, p: b.call("distill_loss", p["z"], p["i"], p["t"], 1.0))
    plan("temperature", {"z": [4, 30], "i": [4, 3], "t": [4, 3]},
         lambda b, p: b.call("distill_loss", p["z"], p["i"], p["t"], 0.0))
    plan("hidden size mismatch", {"x": [4, 30]}, lambda b, p: b.apply(b.ctor("LayerNorm", 31), p["x"]))
