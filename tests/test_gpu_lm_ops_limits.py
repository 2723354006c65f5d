"""The language-model operators where their numbers or sizes end: inputs near
either end of fp32's range, scores that leave nothing of a softmax but its
greatest, sizes next to a hardware limit, and buffers whose owners let go of them.

Tolerances as in test_gpu_lm_ops.py (u = 2^-24): a score is off by at most 56u of
sum |q||k| * scale, a probability by as much relative, sums of values by 60u more;
gradients chain two such products.  Where the scores are of size 8 on average
over a row that is 510u for an output and three times as much for a gradient.
"""
import os
import subprocess
import sys

import numpy as np
import pytest

import lm_reference as R
from test_gpu_lm_ops import U, Lib, attention_inputs, lib, near, near_norm, run_attention  # noqa: F401

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


# ---- layer norm ----------------------------------------------------------------------


def norm_gradients(*widths):
    """Forward and gradients of each width in turn, in a process of its own."""
    from tysor_b200.runtime import CudaContext
    lib = Lib(CudaContext(0))
    for width in widths:
        rows = 3
        rng = np.random.default_rng(width)
        x, dy = (rng.standard_normal((rows, width)).astype(np.float32) for _ in range(2))
        gain = (1 + 0.1 * rng.standard_normal(width)).astype(np.float32)
        want = R.layer_norm(x, gain, None, 1e-5, dy)
        bx, bg, by = lib.put(x), lib.put(gain), lib.put(dy)
        y, stats, dx, dg, db = (lib.zeros(s, 7.0) for s in (x.shape, (rows, 2), x.shape, width, width))
        lib.ok("layer_norm", bx, bg, None, y, stats, rows, width, 1e-5)
        lib.ok("layer_norm_backward", bx, bg, stats, by, dx, dg, db, rows, width, False)
        # A row's mean is near 0 and its spread near 1: 40u of each value, four times that in dx.
        near(y.read(), want["y"], 120 * U, "y", 1.0)
        near(dx.read(), want["dx"], 480 * U, "dx", 1.0)
        near(dg.read(), want["dgain"], 240 * U, "dgain", 1.0)
        near(db.read(), want["dbias"], 40 * U, "dbias", 1.0)
    lib.ctx.close()


@pytest.mark.parametrize("widths", [(6112, 6144, 6116), (6113, 6143), (6144, 6148), (6145,)],
                         ids=lambda w: "-".join(map(str, w)))
def test_layer_norm_gradients_next_to_48_kb(widths):
    """The column sums of 6113 to 6144 values pass 48 KB of shared memory only
    together with the kernel's own; what an earlier call of the process asked for
    must not matter."""
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([os.path.dirname(HERE), HERE]))
    r = subprocess.run([sys.executable, "-c", f"import test_gpu_lm_ops_limits as t; t.norm_gradients(*{widths})"],
                       cwd=HERE, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


# ---- attention -----------------------------------------------------------------------

@pytest.mark.parametrize("dout_size,v_size", [(1e-31, 4.0), (1e-34, 1.0), (1e-3, 1e-31), (4e-16, 4e-16), (1e-24, 1e-12)])
@pytest.mark.parametrize("dims", [(1, 2, 1, 270, 270, 64), (1, 2, 2, 140, 140, 128)], ids=["64", "128"])
def test_window_attention_gradients_of_small_values(lib, dims, dout_size, v_size):
    """dP = dO.V^T far below 1: only the products of both sizes are small, and
    dq and dk follow them in proportion."""
    q, k, v, dout = attention_inputs(31, *dims, False)
    v, dout = v * np.float32(v_size), dout * np.float32(dout_size)
    scale = dims[5] ** -0.5
    want = R.window_attention(q, k, v, None, None, 100, 3, scale, False, dout)
    got = run_attention(lib, q, k, v, dout, None, None, dims, 100, 3, scale, False)
    near_norm(got["out"], want["out"], 510 * U, "out")
    for n in ("dq", "dk", "dv"):
        near_norm(got[n], want[n], 3 * 510 * U, n, want.get("size_" + n, np.zeros(1)))


@pytest.mark.parametrize("size", [1e-16, 1e-18])
def test_window_attention_of_small_inputs(lib, size):
    """All inputs small, the scale argument keeping the scores ordinary."""
    dims = (1, 2, 1, 270, 270, 64)
    q, k, v, dout = (t * np.float32(size) for t in attention_inputs(11, *dims, False))
    scale = 64 ** -0.5 / size / size
    want = R.window_attention(q, k, v, None, None, 100, 3, scale, False, dout)
    got = run_attention(lib, q, k, v, dout, None, None, dims, 100, 3, scale, False)
    near_norm(got["out"], want["out"], 510 * U, "out")
    # dP is about 1e-31 or 1e-35 here: its terms' size counts, as everywhere.
    for n in ("dq", "dk", "dv"):
        near_norm(got[n], want[n], 3 * 510 * U, n, want.get("size_" + n, np.zeros(1)))


@pytest.mark.parametrize("dims", [(1, 2, 1, 1, 700, 64), (2, 4, 1, 1, 5000, 128), (1, 9, 1, 1, 900, 33), (1, 2, 1, 3, 600, 64)],
                         ids=lambda c: "x".join(map(str, c)))
def test_window_attention_of_a_few_rows_over_values_near_the_greatest(lib, dims):
    """An output is a mean of values, which fits fp32 wherever they do."""
    q, k, v, _ = attention_inputs(37, *dims, False)
    k *= np.float32(0.1)  # many keys of similar weight
    v = np.clip(v, -1, 1) * np.float32(2.0 ** 127)
    scale = dims[5] ** -0.5
    want = R.window_attention(q, k, v, None, None, 0, 0, scale, False)
    got = run_attention(lib, q, k, v, None, None, None, dims, 0, 0, scale, False, backward=False)
    near_norm(got["out"], want["out"], 510 * U, "out")
    near(got["stats"][..., 1] / want["stats"][..., 1], np.ones(want["stats"].shape[:-1]), 510 * U, "sums")


def test_window_attention_of_many_keys_of_large_values(lib):
    """Values below 2^100 whose sum over a long cache passes fp32 before the division."""
    dims = (1, 1, 1, 9, 1 << 15, 64)
    q, k, v, _ = attention_inputs(41, *dims, False)
    q *= np.float32(0.01)
    v = (np.abs(v) % 1 + 1) * np.float32(2.0 ** 99)
    want = R.window_attention(q, k, v, None, None, 0, 0, 0.125, False)
    got = run_attention(lib, q, k, v, None, None, None, dims, 0, 0, 0.125, False, backward=False)
    # Scores of 0.01: what counts is the mean, taken over the keys one by one.  Each
    # rounds it by at most 2u, with either sign: 2u sqrt(32768 / 3) = 210u together.
    near_norm(got["out"], want["out"], 510 * U, "out")


LARGE = [(1, 2, 1, 150, 150, 64, 0, 0), (1, 2, 2, 270, 270, 128, 60, 3), (1, 4, 1, 1, 500, 64, 0, 0), (1, 1, 1, 9, 2000, 80, 0, 0)]


@pytest.mark.parametrize("dims", LARGE, ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("size", [300.0, 3000.0, 1e5])
def test_window_attention_of_scores_that_leave_one_key(lib, dims, size):
    """Scores from 1e5 to 1e11: each row's greatest takes all the weight (rows whose
    two greatest lie within 2^-18 of the terms' size are left out of the
    comparison, what fp32 makes of their scores being either's), its output is
    that key's value, and the gradients of the scores are 0."""
    batch, heads, kv_heads, q_len, k_len, dim, window, sinks = dims
    q, k, v, dout = attention_inputs(43, *dims[:6], False)
    q, k = q * np.float32(size), k * np.float32(size)
    scale = dim ** -0.5
    kk, s = np.repeat(k, heads // kv_heads, 1).astype(np.float64), None
    s = np.einsum("bhqd,bhkd->bhqk", q.astype(np.float64), kk) * scale
    terms = np.einsum("bhqd,bhkd->bhqk", np.abs(q).astype(np.float64), np.abs(kk)) * scale
    s = np.where(R.visible(None, None, batch, q_len, k_len, window, sinks)[:, None], s, -np.inf)
    two = np.sort(s, -1)[..., -2:] if k_len > 1 else None
    clear = (two[..., 1] - two[..., 0] > 2.0 ** -18 * terms.max(-1) + 30) | ~np.isfinite(two[..., 0])
    assert clear.mean() > 0.98
    dout[~clear] = 0  # and out of the gradients
    want = R.window_attention(q, k, v, None, None, window, sinks, scale, False, dout)
    got = run_attention(lib, q, k, v, dout, None, None, dims[:6], window, sinks, scale, False)
    near_norm(got["out"][clear], want["out"][clear], 64 * U, "out")
    near((got["stats"][..., 0] / want["stats"][..., 0])[clear], np.ones(int(clear.sum())), 2.0 ** -16, "greatest")
    near_norm(got["dv"], want["dv"], 3 * 64 * U, "dv")
    for n in ("dq", "dk"):
        assert np.isfinite(got[n]).all()
        near_norm(got[n], want[n], 3 * 64 * U, n, want["size_" + n])


def test_window_attention_of_one_large_key(lib):
    """A key many times larger than the others: rows that see it weigh it alone or
    not at all, the others are as without it."""
    dims = (1, 2, 1, 400, 400, 64)
    q, k, v, dout = attention_inputs(47, *dims, False)
    k[:, :, 70] *= np.float32(1e7)
    want = R.window_attention(q, k, v, None, None, 50, 2, 0.125, False, dout)
    got = run_attention(lib, q, k, v, dout, None, None, dims, 50, 2, 0.125, False)
    near_norm(got["out"], want["out"], 510 * U, "out")
    # The terms of dS cancel where one key has all the weight: their own size counts.
    for n in ("dq", "dk", "dv"):
        near_norm(got[n], want[n], 3 * 510 * U, n, want.get("size_" + n, np.zeros(1)))


@pytest.mark.parametrize("dims", [(2, 2, 1, 20, 20, 32), (2, 4, 1, 1, 30, 64)], ids=["tiles", "one"])
def test_window_attention_of_lengths_that_are_not_whole(lib, dims):
    batch, heads, kv_heads, q_len, k_len, dim = dims
    q, k, v, dout = attention_inputs(5, *dims, False)
    clean = run_attention(lib, q, k, v, dout, None, None, dims, 8, 0, 0.2, False, backward=False)
    first = float(k_len - q_len)
    for starts, lengths in (([first, first], [k_len, k_len - 0.5]), ([first, -0.5], [k_len, k_len]),
                            ([first, 0.25], [k_len, k_len]), ([first, first], [k_len, 1e-30])):
        bufs = [lib.put(t) for t in (q, k, v)]
        out = lib.zeros(q.shape, 5.0)
        lib.ok("window_attention", *bufs, lib.put(np.float32(starts)), lib.put(np.float32(lengths)), out, None, *dims,
               8, 0, 0.2, False)
        with pytest.raises(lib.native.NativeError, match="start or length out of range"):
            lib.ctx.synchronize()
        got = out.read().reshape(q.shape)
        assert np.array_equal(got[0], clean["out"][0]) and not got[1].any()


@pytest.mark.parametrize("dims", [(2, 4, 2, 257, 257, 64, 60, 2), (1, 2, 1, 5, 3000, 128, 0, 0), (2, 8, 2, 1, 1500, 64, 0, 0),
                                  (1, 2, 1, 700, 700, 128, 0, 0)], ids=lambda c: "x".join(map(str, c)))
def test_window_attention_statistics(lib, dims):
    """The greatest score and the sum apart: the one is off by at most 56u of the
    terms of a score, the other by as much relative twice (the greatest's and the
    others'), and the sum's 60u."""
    batch, heads, kv_heads, q_len, k_len, dim, window, sinks = dims
    q, k, v, _ = attention_inputs(53, *dims[:6], False)
    scale = dim ** -0.5
    want = R.window_attention(q, k, v, None, None, window, sinks, scale, False)["stats"]
    got = run_attention(lib, q, k, v, None, None, None, dims[:6], window, sinks, scale, False, backward=False)["stats"]
    kk = np.repeat(np.abs(k), heads // kv_heads, 1).astype(np.float64)
    terms = (np.einsum("bhqd,bhkd->bhqk", np.abs(q).astype(np.float64), kk) * scale).max(-1)
    assert np.all(np.abs(got[..., 0] - want[..., 0]) <= 56 * U * terms + 2 * U * np.abs(want[..., 0]))
    assert np.all(np.abs(got[..., 1] / want[..., 1] - 1) <= 2 * 56 * U * terms + 60 * U)


@pytest.mark.parametrize("dims", [(1, 2, 1, 1, 60, 32), (1, 2, 1, 40, 40, 32)], ids=["one", "tiles"])
def test_window_attention_of_the_greatest_scale(lib, dims):
    """2^127 on inputs so small that their scores are ordinary, and nothing above."""
    q, k, v, _ = attention_inputs(79, *dims, False)
    q, k = q * np.float32(2.0 ** -64), k * np.float32(2.0 ** -66)
    want = R.window_attention(q, k, v, None, None, 0, 0, 2.0 ** 127, False)
    got = run_attention(lib, q, k, v, None, None, None, dims, 0, 0, 2.0 ** 127, False, backward=False)
    near_norm(got["out"], want["out"], 510 * U, "out")
    bufs = [lib.put(t) for t in (q, k, v)]
    lib.refused("at most 2^127", "window_attention", *bufs, None, None, lib.zeros(q.shape), None, *dims, 0, 0, 3e38, False)


@pytest.mark.parametrize("dims", [(3, 4, 2, 1, 1, 33, 26, 4), (1, 2, 1, 300, 300, 64, 1, 0), (2, 2, 2, 140, 140, 128, 20, 1)],
                         ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("size", [1.0, 300.0])
def test_window_attention_of_rows_that_see_one_key(lib, dims, size):
    """Their output is that key's value, and their scores have no gradients at all."""
    q, k, v, dout = attention_inputs(83, *dims[:6], False)
    q, k = q * np.float32(size), k * np.float32(size)
    window, sinks = dims[6:]
    lengths = np.full(dims[0], dims[4], np.float32)
    lengths[-1] = 1
    starts = np.zeros(dims[0], np.float32)
    want = R.window_attention(q, k, v, starts, lengths, window, sinks, 0.1, False, dout)
    for accumulate in (False, True):
        got = run_attention(lib, q, k, v, dout, starts, lengths, dims[:6], window, sinks, 0.1, False, accumulate=accumulate)
        fill = 5.0 if accumulate else 0.0
        near_norm(got["out"][:, :, 0], want["out"][:, :, 0], 64 * U, "out")
        assert np.array_equal(got["dq"][:, :, 0], np.full_like(got["dq"][:, :, 0], fill))
        assert np.array_equal(got["dk"][-1], np.full_like(got["dk"][-1], fill))
        if (window, sinks) == (1, 0) or dims[4] == 1:
            assert np.array_equal(got["dq"], np.full_like(got["dq"], fill))
            assert np.array_equal(got["dk"], np.full_like(got["dk"], fill))
            near_norm(got["dv"] - fill, want["dv"], 64 * U, "dv", 1.0 if accumulate else 0.0)


@pytest.mark.parametrize("which", ["q", "k"])
def test_window_attention_of_one_key_that_is_no_number(lib, which):
    """... but a score that is NaN has NaN for its probability and all that follows."""
    dims = (1, 2, 1, 30, 30, 16)
    q, k, v, dout = attention_inputs(89, *dims, False)
    (q if which == "q" else k)[:, :, 0] = np.nan
    got = run_attention(lib, q, k, v, dout, None, None, dims, 5, 0, 0.25, False)
    assert np.isnan(got["out"][:, :, 0]).all() and np.isnan(got["dq"][:, :, 0]).all()
    assert np.isnan(got["dk"][:, :, 0]).all() and np.isnan(got["dv"][:, :, 0]).all()
    assert np.isfinite(got["out"][:, :, 5:]).all() and np.isfinite(got["dq"][:, :, 5:]).all()


# ---- memory --------------------------------------------------------------------------


def stream_of(lib):
    import torch
    return torch.cuda.ExternalStream(lib.lib.tysor_cuda_context_stream(lib.ctx.handle))


def test_a_wrapped_buffer_is_freed_after_its_last_use(lib):
    """Its owner may give the memory back as soon as the buffer is gone."""
    import torch
    x, y = (torch.ones(16384, 2048, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    bx, by = (lib.Buffer.wrap(lib.ctx, t) for t in (x, y))
    for free in (bx.free, by.free):
        again = [lib.Buffer.wrap(lib.ctx, t) for t in (x, y)]
        for _ in range(200):  # 45 us each
            lib.ok("layer_norm", again[0], None, None, again[1], None, 16384, 2048, 1e-5)
        assert not stream_of(lib).query()
        free()
        assert stream_of(lib).query()


def rope_inputs(lib, seed, sections=(8, 8)):
    rng = np.random.default_rng(seed)
    half = sum(sections)
    x = rng.standard_normal((1, 2, 40, 2 * half)).astype(np.float32)
    pos = rng.integers(0, 900, (1, len(sections), 40)).astype(np.float32)
    keep = np.asarray(sections, np.int64)
    return x, pos, keep, (lib.put(x), lib.put(pos)), lib.zeros(x.shape)


def test_rope_tables_come_in_the_order_of_their_stream(lib):
    """The first call of a theta copies its table on the context's own stream: it
    neither waits for the caller's nor could be overtaken by the kernel."""
    import torch
    x, pos, keep, ins, y = rope_inputs(lib, 61)
    caller = torch.cuda.default_stream()
    waits = []
    for i in range(4):
        theta = 777.0 + i
        with torch.cuda.stream(caller):
            torch.cuda._sleep(1_000_000_000)  # half a second
        lib.ok("rope_axes", *ins, y, 1, 2, 40, keep.ctypes.data_as(lib.native.I64P), 2, theta, False)
        lib.ok("rope", ins[0], y, 2, 40, 16, theta)
        waits.append(caller.query())
        caller.synchronize()
    assert not any(waits[1:])  # the first call also loads its kernels, which waits for all streams
    lib.ok("rope_axes", *ins, y, 1, 2, 40, keep.ctypes.data_as(lib.native.I64P), 2, 778.0, False)
    size = float(np.sqrt(x[..., :16].astype(np.float64) ** 2 + x[..., 16:].astype(np.float64) ** 2).max())
    near(y.read(), R.rope_axes(x, pos, (8, 8), 778.0, False), 8 * U, "y", size)


def test_rope_tables_in_a_capture(lib):
    """A call that would have to make its table is refused, and the capture goes on."""
    import torch
    x, pos, keep, ins, y = rope_inputs(lib, 67)
    args = (*ins, y, 1, 2, 40, keep.ctypes.data_as(lib.native.I64P), 2)
    lib.ok("rope_axes", *args, 900.0, False)
    want = y.read()
    lib.ctx.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream_of(lib)):
        graph.capture_begin()
        lib.refused("while the context's stream is captured", "rope_axes", *args, 901.0, False)
        lib.refused("while the context's stream is captured", "rope", ins[0], y, 2, 40, 16, 901.0)
        lib.ok("rope_axes", *args, 900.0, False)
        graph.capture_end()
        y.write(np.zeros(want.size, np.float32))
        graph.replay()
    assert np.array_equal(y.read(), want)
    lib.ok("rope_axes", *args, 901.0, False)
    del graph


def test_a_workspace_that_a_graph_uses_is_kept():
    """A captured call, larger ones after it (whose workspace takes the place of
    the graph's), and its replay; a call that would have to grow it in a capture is
    refused."""
    import torch
    from tysor_b200.runtime import CudaContext
    lib = Lib(CudaContext(0))
    dims = (1, 2, 1, 200, 200, 64)
    q, k, v, _ = attention_inputs(71, *dims, False)
    ins, out = [lib.put(t) for t in (q, k, v)], lib.zeros(q.shape)
    args = (*ins, None, None, out, None, *dims, 50, 2, 0.125, False)
    large = (1, 2, 1, 3000, 3000, 64)
    more = [lib.put(t) for t in attention_inputs(73, *large, False)]
    big = (*more[:3], None, None, more[3], None, *large, 50, 2, 0.125, False)
    lib.ok("window_attention", *args)
    want = out.read()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream_of(lib)):
        graph.capture_begin()
        lib.refused("workspace cannot grow", "window_attention", *big)
        lib.ok("window_attention", *args)
        graph.capture_end()
        lib.ok("window_attention", *big)
        held = torch.full((1 << 24,), float("nan"), device="cuda")  # takes freed memory, if any was
        out.write(np.zeros(want.size, np.float32))
        graph.replay()
        torch.cuda.current_stream().synchronize()
    assert np.array_equal(out.read(), want) and bool(held.isnan().all())
    del graph
    lib.ctx.close()


# ---- graphs --------------------------------------------------------------------------


def test_graphs_refuse_sizes_that_no_kernel_counts(cuda_ctx):
    """A reshape whose sizes are negative in pairs has the right product."""
    from tysor_b200.graph import GraphBuilder
    from tysor_b200.native import NativeError
    from tysor_b200.runtime import CudaGraphExecutor

    def plan(message, shapes, make):
        b = GraphBuilder()
        p = {n: b.param(n) for n in shapes}
        b.ret(make(b, p))
        ex = CudaGraphExecutor(cuda_ctx, b.build(), shapes)
        with pytest.raises(NativeError, match=message):
            ex.run()
        ex.close()

    x = [1, 2, 8, 16]
    for sizes in ((-1, -2, 8, 16), (1, -2, -8, 16), (1, -2, 8, -16)):
        plan("sizes from 1", {"x": x}, lambda b, p: (lambda q: b.call("window_attention", q, q, q, 0, 0))(
            b.call("reshape", p["x"], *sizes)))
        plan("sizes from 1|heads of 16", {"x": x, "p": [1, 1, 8]}, lambda b, p: b.call(
            "rope_axes", b.call("reshape", p["x"], *sizes), p["p"], 1e4, 8))
    plan("finite eps", {"x": [4, 30]}, lambda b, p: b.apply(b.ctor("LayerNorm", 30, 1e39), p["x"]))
