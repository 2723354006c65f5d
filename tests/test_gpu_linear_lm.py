"""rotary, decay_attention and token_logprobs together, as a program uses them:
the linear-attention language model (programs.linear_lm) through the graph
executor against the same model in 64 bits (torch on the CPU, exact
gradients), serving it token by token through the dispatch calls, and the
operators in graphs that a caller captures.

Bars as for the student model: values 1e-5 and gradients 3e-5 of the tensor's
norm, the strict matmuls' own."""
import numpy as np
import pytest

import linear_reference as R
from test_gpu_lm_ops import Lib
from test_gpu_student_lm import off
from tysor_b200.graph import GraphBuilder
from tysor_b200.programs import linear_lm, random_parameters
from tysor_b200.runtime import CudaContext, CudaGraphExecutor, DeviceBuffer

pytestmark = pytest.mark.gpu

CFG = dict(layers=2, batch=3, seq=150, d_model=256, n_heads=4, n_kv_heads=2, hidden=384, vocab=500, rotary_dim=48,
           scaling=(3, 8.0, 64.0, 1.0, 8.0, 1.2), temperature=0.9, entropy_weight=0.05)


def data(seed=0):
    rng = np.random.default_rng(seed)
    b, s, v = CFG["batch"], CFG["seq"], CFG["vocab"]
    lengths = np.array([s, 61, 0], np.float32)
    sampled = rng.integers(0, v, (b * s, 1)).astype(np.float32)
    for i in range(b):
        sampled.reshape(b, s)[i, int(lengths[i]):] = -1
    return dict(ids=rng.integers(0, v, b * s).astype(np.float32), lengths=lengths, sampled=sampled,
                positions=(np.arange(s)[None] + rng.integers(0, 900, (b, 1))).astype(np.float32),
                decay=np.array([0.7, 0.1, 0.01, 0.0], np.float32),
                advantage=rng.standard_normal((b * s, 1)).astype(np.float32))


def shapes():
    b, s = CFG["batch"], CFG["seq"]
    return {"ids": [b * s], "positions": [b, s], "lengths": [b], "decay": [CFG["n_heads"]], "sampled": [b * s, 1],
            "advantage": [b * s, 1]}


def reference(graph, inputs, params):
    """Loss terms and gradients of every parameter, in float64 with torch's autograd."""
    import torch
    P = {n: torch.tensor(a, dtype=torch.float64, requires_grad=True) for n, a in params.items()}
    c = CFG
    b, s, hd, r = c["batch"], c["seq"], c["d_model"] // c["n_heads"], c["rotary_dim"]
    ctor = iter([n for n in graph.nodes if n.kind == "ctor"])
    emb = P[f"embedding_{next(ctor).output}_weight"]
    rate = R.rotary_rates(r // 2, 10000.0, *c["scaling"][:5])
    angle = torch.tensor(inputs["positions"].astype(np.float64)[..., None] * rate)[:, :, None]
    n = torch.tensor(inputs["lengths"].astype(np.int64))[:, None, None, None]
    i, j = torch.arange(s)[:, None], torch.arange(s)[None]
    rate_h = torch.tensor(inputs["decay"].astype(np.float64))[None, :, None, None]
    weight = torch.exp(-rate_h * (i - j).clamp_min(0)) * ((j <= i) & (i < n) & (j < n))

    def norm(x, n):
        m = x.mean(1, keepdim=True)
        d = (x - m) / ((x - m).pow(2).mean(1, keepdim=True) + 1e-5).sqrt()
        return d * P[f"layernorm_{n.output}_gain"] + P[f"layernorm_{n.output}_bias"]

    def lin(x, n):
        return x @ P[f"linear_{n.output}_weight"]

    def turn(x):
        l, h = x[..., 0:r:2], x[..., 1:r:2]
        t = torch.stack((l * angle.cos() - h * angle.sin(), l * angle.sin() + h * angle.cos()), -1) * c["scaling"][5]
        return torch.cat((t.flatten(-2), x[..., r:]), -1)

    x = emb[torch.tensor(inputs["ids"].astype(np.int64))]
    group = c["n_heads"] // c["n_kv_heads"]
    for _ in range(c["layers"]):
        n1, qp, kp, vp, op, n2, gp, up, dp, _act = (next(ctor) for _ in range(10))
        hn = norm(x, n1)
        q = turn(lin(hn, qp).reshape(b, s, c["n_heads"], hd)).transpose(1, 2)
        k = turn(lin(hn, kp).reshape(b, s, c["n_kv_heads"], hd)).transpose(1, 2).repeat_interleave(group, 1)
        v = lin(hn, vp).reshape(b, s, c["n_kv_heads"], hd).transpose(1, 2).repeat_interleave(group, 1)
        o = ((q @ k.transpose(2, 3)) * weight) @ v / hd ** 0.5
        h = x + lin(o.transpose(1, 2).reshape(b * s, -1), op)
        hn2 = norm(h, n2)
        x = h + lin(torch.nn.functional.silu(lin(hn2, gp)) * lin(hn2, up), dp)
    logits = norm(x, next(ctor)) @ emb.T
    lp = torch.log_softmax(logits / c["temperature"], 1)
    ids = torch.tensor(inputs["sampled"].astype(np.int64))
    given = torch.where(ids >= 0, lp.gather(1, ids.clamp_min(0)), 0.0)
    entropy = -(lp.exp() * lp).sum(1, keepdim=True)
    loss = -(given * torch.tensor(inputs["advantage"].astype(np.float64)) + c["entropy_weight"] * entropy)
    grads = torch.autograd.grad(loss.sum(), list(P.values()))
    return loss.detach().numpy(), dict(zip(P, (g.numpy() for g in grads)))


def test_linear_lm_trains_as_in_64_bits(cuda_ctx):
    lr, steps = 0.002, 3
    g = linear_lm(**CFG, lr=lr, iterations=steps)
    inputs, params = data(), random_parameters(g, std=0.05)
    ex = CudaGraphExecutor(cuda_ctx, g, shapes(), inputs, params)
    mine = {n: a.astype(np.float64) for n, a in params.items()}
    for step in range(steps):  # the first step runs eagerly, the others replay its captured graph
        want, grads = reference(g, inputs, mine)
        ex.train(1, lr)
        assert off(ex.value(g.outputs[0]).data, want) < 1e-5, step
        for n in grads:
            assert off(ex.parameter_grad(n), np.asarray(grads[n])) < 3e-5, (step, n)
            mine[n] = mine[n] - lr * grads[n]
            assert off(ex.parameter(n), mine[n]) < 1e-5, (step, n)
    ex.close()


def test_linear_lm_runs_and_captured_steps_repeat(cuda_ctx):
    g = linear_lm(**CFG)
    inputs, params = data(1), random_parameters(g, std=0.05)
    results = []
    for capture in (True, False):
        ex = CudaGraphExecutor(cuda_ctx, g, shapes(), inputs, params)
        ex.set_capture(capture)
        results.append((ex.train(4, 1e-3), ex.parameters()))
        ex.close()
    assert results[0][0] == results[1][0]
    assert all(np.array_equal(results[1][1][n], a) for n, a in results[0][1].items())
    ex = CudaGraphExecutor(cuda_ctx, g, shapes(), inputs)
    out = ex.run()
    assert out.shape == [CFG["batch"] * CFG["seq"], 1] and np.isfinite(out.data).all()
    ex.close()


@pytest.mark.parametrize("same", [False, True])
def test_backward_mode_reports_exact_gradients(cuda_ctx, same):
    # `same`: one value as queries, keys and values.
    b, s, h, hd = 2, 70, 2, 16
    rng = np.random.default_rng(4)
    gb = GraphBuilder("m")
    q, k, v, pos, decay, ids = (gb.param(n) for n in ("q", "k", "v", "pos", "decay", "ids"))
    if same:
        k = v = q
    turned = gb.call("rotary", q, pos, 10000.0, 8, False, True) if not same else q
    a = gb.call("decay_attention", turned, turned if same else k, turned if same else v, decay, True)
    gb.ret(gb.binary("+", gb.call("token_logprobs", a, ids, 1.0), gb.call("token_entropy", a, 2.0)))
    g = gb.build()
    x = {n: rng.standard_normal((b, s, h, hd)).astype(np.float32) for n in "qkv"}
    x["pos"] = np.tile(np.arange(s, dtype=np.float32), (b, 1))
    x["decay"] = np.array([0.3, 0.01], np.float32)
    x["ids"] = rng.integers(0, hd, (b * s * h, 1)).astype(np.float32)
    ex = CudaGraphExecutor(cuda_ctx, g, {n: list(a.shape) for n, a in x.items()}, x)
    grads = {n: t.data.reshape(x[n[:-5]].shape) for n, t in ex.backward()}
    ex.close()
    plain = (0, 1.0, 0.0, 0.0, 0.0, 1.0)
    turn = (lambda t, back=False: t.astype(np.float64)) if same else \
        (lambda t, back=False: R.rotary(t, x["pos"], 8, False, 10000.0, plain, True, back))
    qq, kk, vv = turn(x["q"]), (x["q"] if same else x["k"]), (x["q"] if same else x["v"])
    out = R.decay_attention(qq, kk, vv, x["decay"], None, None, hd ** -0.5, True)["out"].reshape(-1, hd)
    one = np.ones(b * s * h)
    dz = R.token_logprobs(out, x["ids"], 0, 1.0, dout=one[:, None])["grad"] + R.token_logprobs(out, None, 0, 2.0, dentropy=one)["grad"]
    w = R.decay_attention(qq, kk, vv, x["decay"], None, None, hd ** -0.5, True, dz.reshape(b, s, h, hd))
    dq = turn(w["dq"], True)
    if same:
        assert off(grads["q_grad"], dq + w["dk"] + w["dv"]) < 3e-5
    else:
        assert off(grads["q_grad"], dq) < 3e-5 and off(grads["k_grad"], w["dk"]) < 3e-5
        assert off(grads["v_grad"], w["dv"]) < 3e-5
    assert not grads["decay_grad"].any() and not grads["pos_grad"].any()


def test_graph_refusals(cuda_ctx):
    def run(shapes, build):
        gb = GraphBuilder("m")
        gb.ret(build(gb, [gb.param(n) for n in shapes]))
        ex = CudaGraphExecutor(cuda_ctx, gb.build(), shapes)
        try:
            ex.run()
        finally:
            ex.close()

    x = {"x": [2, 4, 6, 8], "p": [2, 6]}
    for args, match in (((1e4, 7, False), "even number"), ((1e4, 10, False), "even number"), ((1e4, 0, False), "2 to 512"),
                        ((-1.0, 8, False), "theta"), ((1e4, 8, False, 2, 1.0, 8.0, 2.0, 1.0, 1.0), "low < high"),
                        ((1e4, 8, False, 2), "rotary expects"), ((1e4, 8, False, True), "positions")):
        with pytest.raises(RuntimeError, match=match):
            run(x, lambda gb, v: gb.call("rotary", *v, *args))
    d = {"q": [2, 4, 6, 8], "k": [2, 2, 6, 8], "v": [2, 2, 6, 5], "d": [4]}
    run(d, lambda gb, v: gb.call("decay_attention", *v))
    for over, match in (({"k": [2, 3, 6, 8], "v": [2, 3, 6, 5]}, "divide"), ({"k": [2, 2, 5, 8]}, "one length"),
                        ({"v": [2, 4, 6, 5]}, "one length"), ({"d": [3]}, "one decay"), ({"v": [2, 2, 6, 129]}, "1 to 128")):
        with pytest.raises(RuntimeError, match=match):
            run({**d, **over}, lambda gb, v: gb.call("decay_attention", *v))
    z = {"z": [6, 9], "i": [5]}
    for args, match in (((1.0,), "ids of"), ((0.0,), "ids of")):
        with pytest.raises(RuntimeError, match=match):
            run(z, lambda gb, v: gb.call("token_logprobs", *v, *args))
    with pytest.raises(RuntimeError, match="temperature"):
        run({"z": [6, 9]}, lambda gb, v: gb.call("token_entropy", *v, 0.0))


def test_a_decay_that_would_need_a_gradient_is_refused(cuda_ctx):
    # It has none, so that a graph which trains it, or asks for its inputs' gradients, would go on without.
    b, s, h, d = 2, 8, 4, 16
    shapes = {"x": [b, s, h, d], "r": [1, h]}
    data = {"x": np.ones((b, s, h, d), np.float32), "r": np.ones((1, h), np.float32)}

    def graph(decay):
        gb = GraphBuilder("m")
        x, r = gb.param("x"), gb.param("r")
        q = gb.apply(gb.ctor("LayerNorm", d), x)
        loss = gb.let("loss", gb.call("decay_attention", q, x, x, decay(gb, r), True))
        gb.ret(loss)
        gb.train(objective="loss", lr=0.1, iterations=1)
        return CudaGraphExecutor(cuda_ctx, gb.build(), shapes, data)

    direct, scaled = (lambda gb, r: r), (lambda gb, r: gb.binary("*", r, 0.5))
    trained = lambda gb, r: gb.apply(gb.ctor("linear", h, h, False), r)
    for decay, train, backward in ((direct, True, True), (scaled, True, False), (trained, False, False)):
        for call, works in ((lambda ex: ex.train(1, 0.1), train), (lambda ex: ex.backward(), backward),
                            (lambda ex: ex.run(), True)):
            ex = graph(decay)
            if works:
                call(ex)
            else:
                with pytest.raises(RuntimeError, match="no gradient for decay"):
                    call(ex)
            ex.close()


def test_serving_token_by_token(cuda_ctx):
    # A prompt, then one token at a time over the state: rotary on q and k, decay attention, an output
    # projection, and the answers' log probabilities.
    lib = Lib(cuda_ctx)
    b, h, d, s, prompt, vocab = 3, 4, 64, 24, 17, 300
    rng = np.random.default_rng(5)
    q, k, v = (rng.standard_normal((b, s, h, d)).astype(np.float32) for _ in range(3))
    w = (rng.standard_normal((h * d, vocab)) * (h * d) ** -0.5).astype(np.float32)
    pos = (np.arange(s)[None] + np.array([[0], [5000], [90000]])).astype(np.float32)
    decay = np.array([0.5, 0.05, 0.005, 0.0], np.float32)
    scaling = (2, 4.0, 1000.0, 1.0, 16.0, 1.1)
    bw, bd, state = lib.put(w), lib.put(decay), lib.zeros(b * h * d * d)
    got = []
    for at, n in [(0, prompt)] + [(t, 1) for t in range(prompt, s)]:
        bp = lib.put(pos[:, at:at + n])
        turned = []
        for t in (q, k):
            y = lib.zeros(b * n * h * d)
            lib.ok("rotary", lib.put(t[:, at:at + n]), bp, y, b, h, n, d, 32, True, 10000.0, *scaling, True)
            turned.append(y)
        out, z, ids = lib.zeros(b * n * h * d), lib.zeros(b * n * vocab), lib.put(np.full(b * n, 7, np.float32))
        lib.ok("decay_attention", *turned, lib.put(v[:, at:at + n]), bd, state, None, out, state, b, h, h, n, d, d, 0.125, True)
        lib.ok("matmul", out, bw, z, b * n, vocab, h * d)
        lp, ent, ti, tl = lib.zeros(b * n), lib.zeros(b * n), lib.zeros(b * n * 3), lib.zeros(b * n * 3)
        lib.ok("token_logprobs", z, ids, lp, ent, ti, tl, None, b * n, vocab, 1, 3, 1.0)
        got.append([lp.read().reshape(b, n), ent.read().reshape(b, n), tl.read().reshape(b, n, 3), ti.read().reshape(b, n, 3)])
    lp, ent, tl, ti = (np.concatenate(x, 1) for x in zip(*got))
    tq, tk = (R.rotary(t, pos, 32, True, 10000.0, scaling, True) for t in (q, k))
    o = R.decay_attention(tq, tk, v, decay, None, None, 0.125, True)["out"].reshape(b * s, -1)
    want = R.token_logprobs(o @ w, np.full((b * s, 1), 7.0), 3, 1.0)
    for a, n in ((lp, "out"), (ent, "entropy"), (tl, "top_logprobs")):
        assert abs(a.reshape(-1) - want[n].reshape(-1)).max() < 1e-4, n
    # Equal but for neighbours that 64 bits tell apart and 32 do not.
    gap = want["top_logprobs"][:, :-1] - want["top_logprobs"][:, 1:]
    clear = (gap > 1e-4).all(1)
    assert clear.mean() > 0.9 and np.array_equal(ti.reshape(-1, 3)[clear][:, :2], want["top_ids"][clear][:, :2])


def test_calls_in_a_captured_graph_and_on_a_waiting_stream():
    import torch
    ctx = CudaContext(0)
    lib = Lib(ctx)
    stream = torch.cuda.ExternalStream(lib.lib.tysor_cuda_context_stream(ctx.handle))
    b, s, h, d, vocab = 2, 200, 4, 64, 5000
    gen = torch.Generator("cuda").manual_seed(3)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    x = {"q": normal(b, s, h, d), "k": normal(b, s, 2, d), "v": normal(b, s, 2, d), "dout": normal(b, s, h, d),
         "pos": torch.arange(s, device="cuda").float().repeat(b, 1), "decay": torch.tensor([0.5, 0.1, 0.01, 0.0], device="cuda"),
         "z": normal(b * s, vocab), "ids": torch.randint(0, vocab, (b * s, 1), generator=gen, device="cuda").float()}
    x.update({n: torch.zeros_like(x[m]) for n, m in (("turned", "q"), ("out", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v"), ("g", "z"))})
    x.update({n: torch.zeros(b * s, w, device="cuda") for n, w in (("lp", 1), ("ent", 1), ("ti", 8), ("tl", 8), ("st", 2))})
    torch.cuda.synchronize()
    w = {n: DeviceBuffer.wrap(ctx, t) for n, t in x.items()}

    def calls():
        lib.ok("rotary", w["q"], w["pos"], w["turned"], b, h, s, d, 32, False, 10000.0, 0, 1.0, 0.0, 0.0, 0.0, 1.0, True)
        args = (b, h, 2, s, d, d, 0.125, True)
        lib.ok("decay_attention", w["turned"], w["k"], w["v"], w["decay"], None, None, w["out"], None, *args)
        lib.ok("decay_attention_backward", w["turned"], w["k"], w["v"], w["decay"], None, None, w["dout"], None, w["dq"],
               w["dk"], w["dv"], None, *args, False)
        lib.ok("token_logprobs", w["z"], w["ids"], w["lp"], w["ent"], w["ti"], w["tl"], w["st"], b * s, vocab, 1, 8, 1.0)
        lib.ok("token_logprobs_backward", w["z"], w["ids"], w["st"], w["ent"], w["lp"], w["ent"], w["g"], b * s, vocab, 1,
               1.0, False)

    results = ("turned", "out", "dq", "dk", "dv", "g", "lp", "ent", "ti", "tl")
    calls()
    ctx.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        calls()
    for seed in (4, 5):  # the graph's calls on new values, and the same calls by themselves
        gen.manual_seed(seed)
        for n in ("q", "k", "v", "dout", "z"):
            x[n].copy_(normal(*x[n].shape))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        stream.synchronize()
        first = {n: x[n].clone() for n in results}
        torch.cuda.synchronize()
        calls()
        ctx.synchronize()
        assert all(torch.equal(first[n], x[n]) for n in results)
    del graph
    for buf in w.values():
        buf.free()
    ctx.close()
