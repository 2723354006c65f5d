"""rotary, decay_attention and token_logprobs through the C ABI against their
formulas in 64 bits (linear_reference.py), forward and backward.

Tolerances (u = 2^-24, half a step of fp32), fixed from the arithmetic:

* rotary: as rope_axes (8u of the pair's length), and the amplitude's product
  with sine and cosine: 10u.
* decay_attention: products of two rows come from halves of 11 bits each (4u an
  operand, 3 operands), and 16 + 24 + 12 + 16 instructions add them up, each of
  which may lose a whole step (2u) of a sum that is no larger than the result's
  own order; the state is rounded once per 64 tokens more, at random.  Together
  128u of the result's norm; a single value may be off by more of itself, 512u of
  the tensor's greatest.  Token by token, 2 roundings a token at random for up to
  1000 tokens: less.
* token_logprobs: (z - max) / T is rounded twice at a size of up to 40 where it
  counts (80u), the sum over the width has at most 100 terms a thread and 16 levels
  of 2 steps each (240u with ex2's), its logarithm is of up to 20 (40u): 400u.
  Gradients have as much relative to the row's greatest.
"""
import numpy as np
import pytest

import linear_reference as R
from test_gpu_lm_ops import Lib, U, near

pytestmark = pytest.mark.gpu


@pytest.fixture
def lib(cuda_ctx):
    return Lib(cuda_ctx)


PLAIN = (0, 1.0, 0.0, 0.0, 0.0, 1.0)
SCALINGS = [PLAIN, (1, 4.0, 0.0, 0.0, 0.0, 1.0), (2, 8.0, 4096.0, 1.0, 4.0, 0.75), (3, 32.0, 2048.0, 1.0, 32.0, 1.35),
            (2, 0.5, 100.0, 0.0, 8.0, -2.0)]


# ---- rotary --------------------------------------------------------------------------


@pytest.mark.parametrize("batch,heads,seq,head_dim,rotary_dim", [
    (1, 1, 1, 2, 2), (1, 3, 5, 7, 4), (2, 4, 33, 64, 64), (2, 4, 33, 128, 64), (1, 5, 17, 90, 90), (3, 2, 9, 80, 24),
    (1, 16, 300, 128, 128), (1, 2, 3, 512, 512), (1, 2, 3, 1000, 512), (1, 70000, 1, 8, 8), (2, 3, 40, 12, 8),
    (2, 3, 9, 12, 4), (1, 6, 300, 128, 44), (1, 5, 17, 14, 12)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("scaling", SCALINGS)
def test_rotary(lib, batch, heads, seq, head_dim, rotary_dim, interleaved, scaling):
    rng = np.random.default_rng(seq + head_dim)
    for seq_major in (False, True):
        shape = (batch, seq, heads, head_dim) if seq_major else (batch, heads, seq, head_dim)
        x, dy, old = (rng.standard_normal(shape).astype(np.float32) for _ in range(3))
        pos = rng.integers(0, 1 << 22, (batch, seq)).astype(np.float32)
        args = (batch, heads, seq, head_dim, rotary_dim, interleaved, 10000.0, *scaling, seq_major)
        ref = (rotary_dim, interleaved, 10000.0, scaling, seq_major)
        bx, by, bp, out, dx = lib.put(x), lib.put(dy), lib.put(pos), lib.zeros(x.size, 9.0), lib.put(old)
        size = 1.5 * max(abs(x).max(), abs(dy).max()) * abs(scaling[5])
        lib.ok("rotary", bx, bp, out, *args)
        near(out.read(), R.rotary(x, pos, *ref), 10 * U, "y", size)
        lib.ok("rotary", bx, None, out, *args)
        near(out.read(), R.rotary(x, None, *ref), 10 * U, "y by place", size)
        want = R.rotary(dy, pos, *ref, back=True)
        lib.ok("rotary_backward", by, bp, dx, *args, True)
        near(dx.read(), old + want, 12 * U, "dx added", size)
        lib.ok("rotary_backward", by, bp, dx, *args, False)
        near(dx.read(), want, 10 * U, "dx", size)


def test_rotary_of_all_pairs_is_rope_axes(lib):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((2, 3, 64, 32)).astype(np.float32)
    pos = rng.integers(0, 5000, (2, 64)).astype(np.float32)
    bx, a, b = lib.put(x), lib.zeros(x.size), lib.zeros(x.size)
    import ctypes
    lib.ok("rotary", bx, lib.put(pos), a, 2, 3, 64, 32, 32, False, 10000.0, *PLAIN, False)
    lib.ok("rope_axes", bx, lib.put(pos[:, None]), b, 2, 3, 64, (ctypes.c_int64 * 1)(16), 1, 10000.0, False)
    assert np.array_equal(a.read(), b.read())


def test_rotary_turns_back_and_its_gradient_is_a_difference(lib):
    # Linear in x: a difference over any step is the derivative.
    rng = np.random.default_rng(2)
    args = (2, 3, 20, 48, 32, True, 500.0, 3, 16.0, 512.0, 0.5, 16.0, 1.25, True)
    x, d, dy = (rng.standard_normal((2, 20, 3, 48)).astype(np.float32) for _ in range(3))
    pos = lib.put(rng.integers(0, 9000, (2, 20)).astype(np.float32))
    y, y2, dx = (lib.zeros(x.size) for _ in range(3))
    lib.ok("rotary", lib.put(x + d), pos, y, *args)
    lib.ok("rotary", lib.put(x), pos, y2, *args)
    lib.ok("rotary_backward", lib.put(dy), pos, dx, *args, False)
    step = (y.read().astype(np.float64) - y2.read()) @ dy.reshape(-1).astype(np.float64)
    got = dx.read().astype(np.float64) @ ((x + d).astype(np.float64) - x).reshape(-1)
    assert abs(step - got) <= 60 * U * np.linalg.norm(dy) * (np.linalg.norm(x) + np.linalg.norm(d)) * 1.25


@pytest.mark.parametrize("rotary_dim", [64, 44, 10])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_off_16_byte_boundaries(lib, rotary_dim, interleaved):
    rng = np.random.default_rng(rotary_dim)
    x = rng.standard_normal((2, 3, 7, 64)).astype(np.float32)
    want = R.rotary(x, None, rotary_dim, interleaved, 10000.0, PLAIN, False)
    for a, b in ((0, 1), (1, 0), (2, 2), (3, 1)):
        base, out = lib.put(np.concatenate([np.zeros(a, np.float32), x.reshape(-1)])), lib.zeros(b + x.size + 1, 9.0)
        view = [lib.Buffer(lib.ctx, lib.lib.tysor_cuda_buffer_view(p.handle, o, x.size), x.size)
                for p, o in ((base, a), (out, b))]
        lib.ok("rotary", view[0], None, view[1], 2, 3, 7, 64, rotary_dim, interleaved, 10000.0, *PLAIN, False)
        got = out.read()
        near(got[b:-1], want, 10 * U, "y", 1.5 * abs(x).max())
        assert (got[:b] == 9.0).all() and got[-1] == 9.0


def test_rotary_refusals(lib):
    x, y = lib.zeros(64), lib.zeros(64)
    pos = lib.zeros(2)

    def bad(message, *args, x=x, y=y):
        lib.refused(message, "rotary", x, pos, y, *args)

    bad("even number", 1, 4, 2, 8, 7, False, 1e4, *PLAIN, False)
    bad("even number", 1, 4, 2, 8, 10, False, 1e4, *PLAIN, False)
    bad("2 to 512 values", 1, 4, 2, 8, 0, False, 1e4, *PLAIN, False)
    bad("2 to 512 values", 1, 1, 1, 1024, 514, False, 1e4, *PLAIN, False)
    bad("theta", 1, 4, 2, 8, 8, False, 0.0, *PLAIN, False)
    bad("theta", 1, 4, 2, 8, 8, False, float("nan"), *PLAIN, False)
    bad("scalings 0 to 3", 1, 4, 2, 8, 8, False, 1e4, 4, 1.0, 1.0, 1.0, 2.0, 1.0, False)
    bad("factor", 1, 4, 2, 8, 8, False, 1e4, 1, 0.0, 1.0, 1.0, 2.0, 1.0, False)
    bad("original length", 1, 4, 2, 8, 8, False, 1e4, 2, 2.0, 0.0, 1.0, 2.0, 1.0, False)
    bad("low < high", 1, 4, 2, 8, 8, False, 1e4, 2, 2.0, 64.0, 2.0, 2.0, 1.0, False)
    bad("low < high", 1, 4, 2, 8, 8, False, 1e4, 3, 2.0, 64.0, 0.0, 2.0, 1.0, False)
    bad("amplitude", 1, 4, 2, 8, 8, False, 1e4, 0, 1.0, 0.0, 0.0, 0.0, float("inf"), False)
    bad("input buffer holds 64", 1, 5, 2, 8, 8, False, 1e4, *PLAIN, False)
    bad("positions buffer holds 2", 1, 2, 3, 8, 8, False, 1e4, *PLAIN, False)
    bad("out overlaps input", 1, 4, 2, 8, 8, False, 1e4, *PLAIN, False, y=x)
    bad("up to 2^30", 1 << 31, 1, 1, 8, 8, False, 1e4, *PLAIN, False)
    lib.ok("rotary", x, pos, y, 0, 4, 2, 8, 8, False, 1e4, *PLAIN, False)


# ---- decay attention -----------------------------------------------------------------


def close(got, want, what, tol=128 * U, most=512 * U):
    got, want = np.asarray(got, np.float64).reshape(-1), np.asarray(want, np.float64).reshape(-1)
    assert got.shape == want.shape and np.isfinite(got).all(), what
    err = np.linalg.norm(got - want)
    assert err <= tol * np.linalg.norm(want), (what, err / max(np.linalg.norm(want), 1e-300), tol)
    if got.size:
        assert abs(got - want).max() <= most * abs(want).max(), (what, abs(got - want).max(), abs(want).max())


def rates(heads, rng):
    d = 2.0 ** -(0.5 + 11.0 * (np.arange(heads) + rng.random(heads)) / heads)
    return d.astype(np.float32)


def decay_data(rng, batch, heads, kv, seq, dk, dv, seq_major, state):
    def of(h, d):
        return (batch, seq, h, d) if seq_major else (batch, h, seq, d)

    def normal(shape, std=1.0):
        return (std * rng.standard_normal(shape)).astype(np.float32)

    t = dict(q=normal(of(heads, dk)), k=normal(of(kv, dk)), v=normal(of(kv, dv)), decay=rates(heads, rng), state=None,
             lengths=None, dout=normal(of(heads, dv), 1e-3), dnew=None)
    if state:
        t["state"], t["dnew"] = normal((batch, heads, dk, dv), 3.0), normal((batch, heads, dk, dv), 1e-3)
    return t


NAMES = ("q", "k", "v", "decay", "state", "lengths")


def decay_run(lib, t, scale, seq_major, accumulate=None, need=("out", "new_state", "dq", "dk", "dv", "dstate")):
    """Forward and backward; `accumulate`: what the gradients hold before."""
    sl, hl = (1, 2) if seq_major else (2, 1)
    shape = (t["q"].shape[0], t["q"].shape[hl], t["k"].shape[hl], t["q"].shape[sl], t["q"].shape[3], t["v"].shape[3],
             scale, seq_major)
    states = shape[0] * shape[1] * shape[4] * shape[5]
    buf = [lib.put(t[n]) for n in NAMES]
    out, new = lib.zeros(t["dout"].size, 7.0), lib.zeros(states, 7.0)
    lib.ok("decay_attention", *buf, out, new, *shape)
    r = {"out": out.read(), "new_state": new.read()}
    if "dq" in need:
        grads = {n: lib.zeros(s, 7.0 if accumulate is None else accumulate)
                 for n, s in (("dq", t["q"].size), ("dk", t["k"].size), ("dv", t["v"].size), ("dstate", states))}
        lib.ok("decay_attention_backward", *buf, lib.put(t["dout"]), lib.put(t["dnew"]), *grads.values(), *shape,
               accumulate is not None)
        r.update({n: g.read() for n, g in grads.items()})
    return r


SHAPES = [(1, 1, 1, 1, 1, 1), (2, 2, 1, 1, 128, 128), (1, 1, 1, 2, 3, 5), (1, 2, 2, 5, 128, 128), (2, 3, 3, 17, 33, 40),
          (1, 2, 2, 63, 64, 64), (1, 2, 2, 64, 64, 128), (1, 2, 1, 65, 128, 64), (2, 4, 2, 130, 80, 48),
          (1, 3, 1, 200, 16, 112), (2, 6, 2, 333, 80, 48), (1, 2, 2, 700, 128, 128), (3, 2, 2, 100, 127, 1),
          (1, 2, 2, 129, 1, 127), (1, 4, 4, 1000, 64, 64), (1, 1, 1, 3000, 32, 32),
          # Several steps of 64 tokens a block: more heads than SMs, and long sequences in segments.
          (5, 32, 8, 200, 128, 128), (10, 16, 16, 300, 64, 48), (3, 50, 50, 150, 33, 90), (1, 16, 16, 2500, 128, 128),
          (1, 8, 4, 4200, 64, 112)]


@pytest.mark.parametrize("batch,heads,kv,seq,dk,dv", SHAPES)
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("seq_major", [False, True])
def test_decay_attention(lib, batch, heads, kv, seq, dk, dv, state, seq_major):
    rng = np.random.default_rng(seq * 7 + dk)
    t = decay_data(rng, batch, heads, kv, seq, dk, dv, seq_major, state)
    scale = float(np.float32(dk ** -0.5))
    want = R.decay_attention(t["q"], t["k"], t["v"], t["decay"], t["state"], None, scale, seq_major, t["dout"], t["dnew"])
    got = decay_run(lib, t, scale, seq_major)
    for n in got:
        close(got[n], want[n], n)
    added = decay_run(lib, t, scale, seq_major, accumulate=0.25)
    for n in ("dq", "dk", "dv", "dstate"):
        near(added[n], 0.25 + want[n], 4 * U, n + " added", 0.25 + 128 * abs(want[n]).max())


@pytest.mark.parametrize("batch,heads,kv,seq,dk,dv", [(4, 2, 1, 1, 64, 64), (4, 3, 3, 70, 80, 48), (5, 4, 2, 300, 64, 128),
                                                      (5, 2, 2, 129, 33, 20), (5, 3, 3, 2300, 48, 64),
                                                      (4, 6, 2, 1500, 80, 40)])
@pytest.mark.parametrize("seq_major", [False, True])
def test_decay_attention_of_padded_batches(lib, batch, heads, kv, seq, dk, dv, seq_major):
    rng = np.random.default_rng(seq)
    t = decay_data(rng, batch, heads, kv, seq, dk, dv, seq_major, True)
    n = rng.integers(0, seq + 1, batch)
    n[:3] = seq, 0, min(seq, 64)
    t["lengths"] = n.astype(np.float32)
    want = R.decay_attention(t["q"], t["k"], t["v"], t["decay"], t["state"], n, 0.125, seq_major, t["dout"], t["dnew"])
    # Whatever the rows behind the ends hold, nothing reads it.
    for name in ("q", "k", "v", "dout"):
        a = np.moveaxis(t[name], 1, 2) if not seq_major else t[name]
        for b in range(batch):
            a[b, n[b]:] = np.array([np.nan, np.inf, -np.inf], np.float32)[b % 3]
    got = decay_run(lib, t, 0.125, seq_major)
    for name in got:
        close(got[name], want[name], name)
    for name in ("out", "dq", "dk", "dv"):
        a = got[name].reshape(want[name].shape)
        a = a if seq_major else np.moveaxis(a, 1, 2)
        assert all(not a[b, n[b]:].any() for b in range(batch)), name


@pytest.mark.parametrize("seq", [1, 40, 150, 1100])
def test_decay_attention_at_the_ends_of_the_decays(lib, seq):
    rng = np.random.default_rng(3)
    t = decay_data(rng, 1, 6, 6, seq, 64, 64, False, True)
    t["decay"] = np.array([0.0, 1e-7, 3e-3, 2.0, 60.0, np.inf], np.float32)
    want = R.decay_attention(t["q"], t["k"], t["v"], t["decay"], t["state"], None, 1.0, False, t["dout"], t["dnew"])
    got = decay_run(lib, t, 1.0, False)
    for n in got:
        a, w = got[n].reshape(want[n].shape), want[n]
        for h in range(6):
            if w[0, h].any():
                close(a[0, h], w[0, h], (n, h))
            else:
                assert not a[0, h].any()


@pytest.mark.parametrize("parts", [[200], [1, 1, 198], [64, 64, 72], [63, 2, 70, 65], [1] * 8 + [192]])
def test_decay_attention_in_parts_is_the_whole(lib, parts):
    # A prompt in chunks and single tokens over a state kept in place.
    rng = np.random.default_rng(4)
    t = decay_data(rng, 2, 4, 2, 200, 80, 96, True, True)
    want = R.decay_attention(t["q"], t["k"], t["v"], t["decay"], t["state"], None, 0.1, True)
    state, decay = lib.put(t["state"]), lib.put(t["decay"])
    at, outs = 0, []
    for n in parts:
        q, k, v = (lib.put(t[x][:, at:at + n]) for x in ("q", "k", "v"))
        out = lib.zeros(2 * n * 4 * 96)
        lib.ok("decay_attention", q, k, v, decay, state, None, out, state, 2, 4, 2, n, 80, 96, 0.1, True)
        outs.append(out.read().reshape(2, n, 4, 96))
        at += n
    close(np.concatenate(outs, 1), want["out"], "out")
    close(state.read(), want["new_state"], "state")


@pytest.mark.parametrize("apart", [("q",), ("dout",), ("v", "dq"), ("dk", "dv"), ("q", "k", "v", "dout", "dq", "dk", "dv")])
@pytest.mark.parametrize("seq", [9, 70, 1700])
def test_decay_attention_of_rows_off_16_byte_boundaries(lib, seq, apart):
    # Of the gradients' three scans some then take whole pieces and some do not.
    rng = np.random.default_rng(seq)
    t = decay_data(rng, 1, 4, 2, seq, 64, 72, False, True)
    want = R.decay_attention(t["q"], t["k"], t["v"], t["decay"], t["state"], None, 0.125, False, t["dout"], t["dnew"])

    def place(name, a):
        if name not in apart:
            return lib.put(a)
        base = lib.put(np.concatenate([np.zeros(1, np.float32), a.reshape(-1)]))
        place.held.append(base)
        return lib.Buffer(lib.ctx, lib.lib.tysor_cuda_buffer_view(base.handle, 1, a.size), a.size)

    place.held = []
    buf = {n: place(n, t[n]) for n in ("q", "k", "v", "decay", "state", "dout")}
    grads = {n: place(n, np.full(t[n[1:]].shape, 7.0, np.float32)) for n in ("dq", "dk", "dv")}
    grads["dstate"] = lib.zeros(t["state"].size)
    lib.ok("decay_attention_backward", buf["q"], buf["k"], buf["v"], buf["decay"], buf["state"], None, buf["dout"],
           lib.put(t["dnew"]), *grads.values(), 1, 4, 2, seq, 64, 72, 0.125, False, False)
    for n in grads:
        close(grads[n].read(), want[n], n)


@pytest.mark.parametrize("seq", [20, 700, 3000])
def test_decay_attention_replaces_its_state(lib, seq):
    # Sequences of any length among them empty ones, whose last segments end before the first begin.
    rng = np.random.default_rng(seq)
    t = decay_data(rng, 4, 3, 3, seq, 128, 64, True, True)
    n = np.array([seq, 0, min(seq, 65), 1])
    t["lengths"] = n.astype(np.float32)
    want = R.decay_attention(t["q"], t["k"], t["v"], t["decay"], t["state"], n, 0.1, True)
    buf = [lib.put(t[x]) for x in NAMES]
    for _ in range(5):
        buf[4].write(t["state"])
        out = lib.zeros(t["dout"].size)
        lib.ok("decay_attention", *buf, out, buf[4], 4, 3, 3, seq, 128, 64, 0.1, True)
        close(out.read(), want["out"], "out")
        close(buf[4].read(), want["new_state"], "state")


@pytest.mark.parametrize("seq,dim", [(12, 64), (300, 64), (300, 128)])
def test_decay_attention_gradients_are_differences(lib, seq, dim):
    # The outputs are linear in each input: differences over whole steps.
    rng = np.random.default_rng(5)
    t = decay_data(rng, 2, 4, 2, seq, dim, dim, False, True)
    got = decay_run(lib, t, 0.1, False)

    def value(t):
        r = decay_run(lib, t, 0.1, False, need=())
        return [r["out"].astype(np.float64) @ t["dout"].reshape(-1), r["new_state"].astype(np.float64) @ t["dnew"].reshape(-1)]

    for name, grad in (("q", "dq"), ("k", "dk"), ("v", "dv"), ("state", "dstate")):
        d = rng.standard_normal(t[name].shape).astype(np.float32)
        ahead, behind = dict(t), dict(t)
        ahead[name], behind[name] = t[name] + d, t[name] - d
        a, b = value(ahead), value(behind)
        step = (sum(a) - sum(b)) / 2
        along = got[grad].astype(np.float64) @ d.reshape(-1)
        # Off by 128u of the outputs' norms times the gradients', and as much of the gradient's own.
        r = decay_run(lib, t, 0.1, False, need=())
        size = 3 * sum(np.linalg.norm(r[n]) * np.linalg.norm(t[w]) for n, w in (("out", "dout"), ("new_state", "dnew")))
        assert abs(step - along) <= 128 * U * (size + np.linalg.norm(got[grad]) * np.linalg.norm(d)), name


@pytest.mark.parametrize("seq,where", [(5, 2), (200, 70), (200, 127), (1000, 500)])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_decay_attention_spreads_what_is_not_finite_forward_alone(lib, seq, where, value):
    rng = np.random.default_rng(6)
    for name in ("q", "k", "v"):
        t = decay_data(rng, 1, 2, 2, seq, 64, 48, False, True)
        clean = R.decay_attention(t["q"], t["k"], t["v"], t["decay"], t["state"], None, 0.1, False)
        t[name][0, 0, where, 3] = value
        r = decay_run(lib, t, 0.1, False, need=())
        out = r["out"].reshape(clean["out"].shape)
        new = r["new_state"].reshape(clean["new_state"].shape)
        close(out[0, 0, :where], clean["out"][0, 0, :where], "before")
        close(out[0, 1], clean["out"][0, 1], "the other head")
        close(new[0, 1], clean["new_state"][0, 1], "the other state")
        if name == "q":
            assert not np.isfinite(out[0, 0, where]).any()
            close(out[0, 0, where + 1:], clean["out"][0, 0, where + 1:], "after")
            close(new[0, 0], clean["new_state"][0, 0], "state")
        elif name == "k":
            assert not np.isfinite(out[0, 0, where:]).any() and not np.isfinite(new[0, 0, 3]).any()
        else:
            assert not np.isfinite(out[0, 0, where:, 3]).any()
            other = np.arange(48) != 3
            close(out[0, 0][:, other], clean["out"][0, 0][:, other], "other columns")
            close(new[0, 0][:, other], clean["new_state"][0, 0][:, other], "other columns' state")


@pytest.mark.parametrize("seq", [7, 150])
@pytest.mark.parametrize("qk,v", [(1e-16, 1e-16), (1e16, 1e-20), (1e-35, 1e30), (1e12, 1e12), (1e-12, 1e25)])
def test_decay_attention_of_large_and_small_values(lib, seq, qk, v):
    rng = np.random.default_rng(7)
    t = decay_data(rng, 1, 2, 2, seq, 64, 64, False, False)
    t["q"] = (t["q"] / np.float32(qk)).astype(np.float32)
    t["k"] = (t["k"] * np.float32(qk)).astype(np.float32)
    t["v"] = (t["v"] * np.float32(v)).astype(np.float32)
    with np.errstate(all="ignore"):
        want = R.decay_attention(t["q"], t["k"], t["v"], t["decay"], None, None, 0.1, False)
    r = decay_run(lib, t, 0.1, False, need=())
    close(r["out"], want["out"], "out")
    if qk * v > 1e-30:  # normal numbers of fp32
        close(r["new_state"], want["new_state"], "state")


def test_decay_attention_of_rows_of_unlike_sizes(lib):
    # Each token's own factor: a row's result is near relative to its own terms.
    rng = np.random.default_rng(8)
    t = decay_data(rng, 1, 2, 2, 256, 64, 64, False, False)
    size = (10.0 ** rng.integers(-6, 7, (1, 2, 256, 1))).astype(np.float32)
    t["q"] = t["q"] * size
    want = R.decay_attention(t["q"], t["k"], t["v"], t["decay"], None, None, 0.1, False)
    out = decay_run(lib, t, 0.1, False, need=())["out"].reshape(want["out"].shape)
    close(out / size, want["out"] / size, "out")


def test_decay_attention_repeats_bit_by_bit_and_empty_calls(lib):
    rng = np.random.default_rng(9)
    t = decay_data(rng, 2, 4, 2, 500, 64, 64, True, True)
    a, b = (decay_run(lib, t, 0.1, True) for _ in range(2))
    assert all(np.array_equal(a[n], b[n]) for n in a)
    e = decay_data(rng, 2, 4, 2, 0, 8, 8, True, True)
    r = decay_run(lib, e, 0.1, True)
    assert np.array_equal(r["new_state"], e["state"].reshape(-1)) and r["out"].size == 0
    assert np.allclose(r["dstate"], e["dnew"].reshape(-1), rtol=2 * U)
    one = lib.put(np.zeros(8, np.float32))
    lib.ok("decay_attention", one, one, one, one, None, None, lib.zeros(1), None, 0, 2, 2, 4, 8, 8, 0.1, False)


def test_decay_attention_refusals(lib):
    x, y, d, s = lib.zeros(256), lib.zeros(256), lib.zeros(2), lib.zeros(2 * 64)

    def bad(message, *shape, q=x, out=y, state=None, new=None):
        lib.refused(message, "decay_attention", q, x, x, d, state, None, out, new, *shape)

    bad("divide the query heads", 1, 2, 3, 4, 8, 8, 0.1, False)
    bad("divide the query heads", 1, 2, 0, 4, 8, 8, 0.1, False)
    bad("1 to 128", 1, 1, 1, 1, 129, 8, 0.1, False)
    bad("1 to 128", 1, 1, 1, 1, 8, 0, 0.1, False)
    bad("2^29", 1, 2, 2, (1 << 29) + 1, 8, 8, 0.1, False)
    bad("2^31 - 1", 1 << 20, 1 << 20, 1 << 20, 1, 8, 8, 0.1, False)
    for scale in (0.0, -1.0, float("nan"), float("inf"), 2.0 ** 61):
        bad("scale", 1, 2, 2, 4, 8, 8, scale, False)
    bad("q buffer holds 256", 1, 2, 2, 17, 8, 8, 0.1, False)
    bad("state buffer holds 128", 1, 2, 2, 4, 8, 16, 0.1, False, state=s)
    bad("out overlaps q", 1, 2, 2, 4, 8, 8, 0.1, False, out=x)
    bad("new_state overlaps q", 1, 2, 2, 4, 8, 8, 0.1, False, new=x)
    part = lib.Buffer(lib.ctx, lib.lib.tysor_cuda_buffer_view(s.handle, 0, 128), 128)
    lib.ok("decay_attention", x, x, x, d, s, None, y, part, 1, 2, 2, 4, 8, 8, 0.1, False)  # the same memory
    base = lib.zeros(300)
    odd = lib.Buffer(lib.ctx, lib.lib.tysor_cuda_buffer_view(base.handle, 1, 128), 128)
    bad("16-byte boundary", 1, 2, 2, 4, 8, 8, 0.1, False, state=odd)
    lib.refused("null buffer", "decay_attention", x, x, x, None, None, None, y, None, 1, 2, 2, 4, 8, 8, 0.1, False)
    # Bad values are found on the device.
    for value in (-1.0, float("nan")):
        lib.ok("decay_attention", x, x, x, lib.put(np.array([0.1, value], np.float32)), None, None, y, None, 1, 2, 2, 4, 8,
               8, 0.1, False)
        with pytest.raises(RuntimeError, match="Decay below 0"):
            lib.ctx.synchronize()
    for n in (-1.0, 0.5, 5.0, float("nan"), float("inf")):
        lib.ok("decay_attention", x, x, x, d, None, lib.put(np.array([n], np.float32)), y, None, 1, 2, 2, 4, 8, 8, 0.1, False)
        with pytest.raises(RuntimeError, match="length out of range"):
            lib.ctx.synchronize()
        assert not y.read(64).any()


# ---- log probabilities ---------------------------------------------------------------


def logprob_run(lib, z, ids, top, temperature, dout=None, dentropy=None, old=None):
    rows, width = z.shape
    given = 0 if ids is None else ids.shape[1]
    bz, bi = lib.put(z), lib.put(ids)
    out, ent, stats = lib.zeros(rows * given), lib.zeros(rows), lib.zeros((rows, 2))
    ti, tl = (lib.zeros(rows * top), lib.zeros(rows * top)) if top else (None, None)
    lib.ok("token_logprobs", bz, bi, out if given else None, ent, ti, tl, stats, rows, width, given, top, temperature)
    r = {"out": out.read(), "entropy": ent.read(), "stats": stats.read()}
    if top:
        r.update(top_ids=ti.read(), top_logprobs=tl.read())
    grad = lib.zeros(z.size, 3.0) if old is None else lib.put(old)
    lib.ok("token_logprobs_backward", bz, bi, stats, ent, lib.put(dout), lib.put(dentropy), grad, rows, width, given,
           temperature, old is not None)
    r["grad"] = grad.read().reshape(z.shape)
    return r


def logprob_check(lib, z, ids, top, temperature, dout=None, dentropy=None):
    want = R.token_logprobs(z, ids, top, temperature, dout, dentropy)
    got = logprob_run(lib, z, ids, top, temperature, dout, dentropy)
    if top:
        assert np.array_equal(got["top_ids"], want["top_ids"].reshape(-1))
        same(got["top_logprobs"], want["top_logprobs"], 400 * U)
    for n in ("out", "entropy"):
        same(got[n], want[n], 400 * U)
    np.testing.assert_allclose(got["stats"].reshape(-1, 2)[:, 1], want["stats"][:, 1], rtol=400 * U)
    assert np.array_equal(got["stats"].reshape(-1, 2)[:, 0], want["stats"][:, 0].astype(np.float32), equal_nan=True)
    for i in range(z.shape[0]):
        near(got["grad"][i], want["grad"][i], 400 * U, "grad", 1e-30) if np.isfinite(want["grad"][i]).all() else \
            np.testing.assert_array_equal(np.isnan(got["grad"][i]), True)
    if dout is not None:
        old = np.full(z.shape, 0.5, np.float32)
        added = logprob_run(lib, z, ids, 0, temperature, dout, dentropy, old)["grad"]
        assert np.array_equal(added, (got["grad"] + old).astype(np.float32), equal_nan=True) or \
            np.nanmax(abs(added - (got["grad"].astype(np.float64) + 0.5))) <= 2 * U * (0.5 + np.nanmax(abs(got["grad"])))
    return got


def same(got, want, tol):
    got, want = np.asarray(got, np.float64).reshape(-1), np.asarray(want, np.float64).reshape(-1)
    assert got.shape == want.shape
    fine = np.isfinite(want)
    np.testing.assert_array_equal(got[~fine], want[~fine])
    np.testing.assert_allclose(got[fine], want[fine], rtol=4 * U, atol=tol)


@pytest.mark.parametrize("rows,width,given,top", [
    (1, 1, 1, 1), (3, 2, 1, 2), (2, 5, 3, 4), (4, 31, 1, 0), (3, 255, 2, 20), (5, 1000, 1, 128), (2, 1001, 128, 5),
    (3, 4096, 1, 64), (2, 4097, 0, 1), (40, 3001, 1, 7), (700, 513, 1, 3), (2, 32000, 4, 20), (1, 128003, 1, 128),
    (3, 65537, 16, 33), (1, 100, 2, 128), (160, 9000, 1, 20)])
@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_token_logprobs(lib, rows, width, given, top, temperature):
    rng = np.random.default_rng(width + top)
    z = (2.5 * rng.standard_normal((rows, width))).astype(np.float32)
    ids = rng.integers(-1, width, (rows, given)).astype(np.float32) if given else None
    dout = rng.standard_normal((rows, given)).astype(np.float32) if given else None
    logprob_check(lib, z, ids, top, temperature, dout, rng.standard_normal(rows).astype(np.float32))


@pytest.mark.parametrize("width", [40, 5000, 40001])
def test_token_logprobs_of_masked_rows(lib, width):
    rng = np.random.default_rng(width)
    z = (2.5 * rng.standard_normal((8, width))).astype(np.float32)
    z[0] = -np.inf                      # nothing is left
    z[1, 3:] = -np.inf                  # fewer than `top`
    z[2, rng.random(width) < 0.9] = -np.inf
    z[3, 1:] = -np.inf                  # one token
    z[4, :width // 2] = -np.inf
    z[5] = -1e38                        # all alike
    z[6, 5] = 3e38                      # one far above
    ids = np.tile(np.array([0, 2, width - 1, -1], np.float32), (8, 1))
    dout = rng.standard_normal((8, 4)).astype(np.float32)
    got = logprob_check(lib, z, ids, 6, 1.0, dout, rng.standard_normal(8).astype(np.float32))
    assert np.array_equal(got["top_ids"].reshape(8, 6)[5], np.arange(6))


@pytest.mark.parametrize("width", [300, 20011, 131072])
@pytest.mark.parametrize("order", ["equal", "rising", "falling", "two values", "zeros of both signs", "one thread's"])
def test_token_logprobs_best_tokens_of_hard_rows(lib, width, order):
    i = np.arange(width, dtype=np.float32)
    z = {"equal": 0 * i, "rising": i / width, "falling": -i / width, "two values": (i % 7 == 3).astype(np.float32),
         "zeros of both signs": np.where(i % 2 == 0, np.float32(-0.0), np.float32(0.0)),
         "one thread's": np.where(i % 1024 < 16, i, -i).astype(np.float32) / width}[order].astype(np.float32)
    rows = np.stack([z, np.roll(z, 5), z[::-1]])
    for top in (1, 20, 128):
        logprob_check(lib, np.ascontiguousarray(rows), np.zeros((3, 1), np.float32), top, 1.0)


def test_token_logprobs_of_rows_that_are_not_finite(lib):
    rng = np.random.default_rng(11)
    for width in (9, 3000, 70000):
        z = rng.standard_normal((5, width)).astype(np.float32)
        z[1, width // 2] = np.nan
        z[2, width - 1] = np.inf
        z[3, :] = np.nan
        z[4, 0], z[4, 1:] = np.nan, -np.inf
        ids = np.tile(np.array([1, -1], np.float32), (5, 1))
        logprob_check(lib, z, ids, 5, 1.0, np.ones((5, 2), np.float32), np.ones(5, np.float32))


def test_token_logprobs_given_twice_and_differences(lib):
    rng = np.random.default_rng(12)
    z = rng.standard_normal((3, 50)).astype(np.float32)
    ids = np.array([[4, 4, 7, 4], [0, 49, 0, -1], [-1, -1, -1, -1]], np.float32)
    dout = rng.standard_normal((3, 4)).astype(np.float32)
    dh = rng.standard_normal(3).astype(np.float32)
    got = logprob_check(lib, z, ids, 0, 1.3, dout, dh)
    d = rng.standard_normal(z.shape)
    # Central differences in 64 bits of the formulas themselves: their error is of the step's square.
    h = 1e-4
    a, b = (R.token_logprobs((z + s * h * d), ids, 0, 1.3) for s in (1, -1))
    step = sum(((a[n] - b[n]) * w).sum() for n, w in (("out", dout), ("entropy", dh))) / (2 * h)
    assert abs(step - (got["grad"].astype(np.float64) * d).sum()) <= 1e-5 * np.abs(got["grad"]).sum()
    for one in ("dout", "dentropy"):  # each alone
        logprob_check(lib, z, ids, 0, 1.3, **{one: dout if one == "dout" else dh})


def test_token_logprobs_at_the_ends_of_the_temperatures(lib):
    rng = np.random.default_rng(13)
    z = rng.standard_normal((3, 700)).astype(np.float32)
    for t in (2.0 ** -60, 1e-3, 50.0, 2.0 ** 60):
        want, got = R.token_logprobs(z, None, 5, t), logprob_run(lib, z, None, 5, t)
        assert np.array_equal(got["top_ids"], want["top_ids"].reshape(-1))
        np.testing.assert_allclose(got["top_logprobs"], want["top_logprobs"].reshape(-1), rtol=4 * U, atol=400 * U)
        same(got["entropy"], want["entropy"], 400 * U)


def test_token_logprobs_refusals(lib):
    z, o, e, s = lib.zeros(64), lib.zeros(8), lib.zeros(8), lib.zeros(16)
    ids = lib.zeros(8)

    def bad(message, rows, width, given, top, t, out=o, ids=ids, stats=s, top_ids=None):
        lib.refused(message, "token_logprobs", z, ids, out, e, top_ids, None, stats, rows, width, given, top, t)

    bad("width of 1 to 2^24", 8, 0, 1, 0, 1.0)
    bad("width of 1 to 2^24", 0, (1 << 24) + 1, 1, 0, 1.0)
    bad("up to 2^31 - 1 rows", 1 << 31, 8, 1, 0, 1.0)
    bad("up to 128 given", 8, 8, 129, 0, 1.0)
    bad("up to 128 best", 8, 8, 1, 129, 1.0)
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-30):
        bad("temperature", 8, 8, 1, 0, t)
    bad("logits buffer holds 64", 9, 8, 0, 0, 1.0)
    bad("null buffer", 8, 8, 1, 0, 1.0, out=None)
    bad("null buffer", 8, 8, 1, 0, 1.0, ids=None)
    bad("null buffer", 8, 8, 1, 1, 1.0)
    bad("out overlaps ids", 8, 8, 1, 0, 1.0, out=ids)
    bad("stats buffer holds 8", 8, 8, 1, 0, 1.0, stats=lib.zeros(8))
    lib.refused("null buffer", "token_logprobs_backward", z, ids, None, None, o, None, lib.zeros(64), 8, 8, 1, 1.0, False)
    lib.refused("null buffer", "token_logprobs_backward", z, ids, s, None, o, e, lib.zeros(64), 8, 8, 1, 1.0, False)
    lib.refused("grad overlaps logits", "token_logprobs_backward", z, ids, s, e, o, e, z, 8, 8, 1, 1.0, False)
    for v in (8.0, float("nan"), float("inf")):
        lib.ok("token_logprobs", z, lib.put(np.full(8, v, np.float32)), o, e, None, None, s, 8, 8, 1, 0, 1.0)
        with pytest.raises(RuntimeError, match="index out of range"):
            lib.ctx.synchronize()
        assert not o.read().any()
    lib.ok("token_logprobs", z, ids, o, None, None, None, None, 0, 8, 1, 0, 1.0)
