"""The language-model operators through the C ABI against their formulas in
64 bits (lm_reference.py): layer_norm, rope_axes, window_attention and
distill_loss, forward and backward.

Tolerances (u = 2^-24, half a step of fp32), fixed from the arithmetic:

* layer_norm: a row's mean and variance are sums of at most 16 values per
  thread and 11 levels of a tree, 27u of the terms' size each (rows held in
  shared memory: 28 additions to growing sums, 14u of the whole, and 2 + 5 + 8
  for a quad, a warp and 16 warps: 29u); rstd has half
  the variance's error; three more roundings: 40u of the largest |n * gain|.
* rope_axes: the angle's fraction of a turn is rounded to fp32 (at most 2^-25
  of half a turn, 2^-25 pi in the angle), the sine and cosine are within 2
  steps, each product and sum half a step: 8u of the pair's length.
* window_attention: a score is a dot product of at most 128 terms, formed in
  at most 3 * 8 + 4 additions that may each lose a whole step (2u): 56u of
  sum |q||k| * scale, which for unit normal inputs is at most 8 on average
  over a row: 450u in a score and as much relative in a probability; the
  values' sums add 60u.  Gradients chain two such products more.
* distill_loss: a sum over the width has at most 100 terms per thread and
  16 levels; (z - max) / T * log2(e) is rounded three times at a size of
  up to 40 where exp of it still counts: 240u of the sum, T^2 times that in
  the loss, and as much relative in the gradient.
"""
import ctypes

import numpy as np
import pytest

import lm_reference as R

U = 2.0 ** -24
pytestmark = pytest.mark.gpu


class Lib:
    def __init__(self, ctx):
        from tysor_b200 import native
        from tysor_b200.runtime import DeviceBuffer
        self.ctx, self.lib, self.native, self.Buffer = ctx, native.lib(), native, DeviceBuffer

    def put(self, a):
        return None if a is None else self.Buffer.from_array(self.ctx, a)

    def zeros(self, shape, value=0.0):
        return self.Buffer.from_array(self.ctx, np.full(shape, value, np.float32))

    def call(self, name, *args):
        h = [a.handle if isinstance(a, self.Buffer) else a for a in args]
        return bool(getattr(self.lib, "tysor_cuda_dispatch_" + name)(self.ctx.handle, *h))

    def ok(self, name, *args):
        self.native.check(self.call(name, *args), name)

    def refused(self, message, name, *args):
        assert not self.call(name, *args)
        assert message in self.native.last_error()


@pytest.fixture
def lib(cuda_ctx):
    return Lib(cuda_ctx)


def near(got, want, tol, what="", floor=0.0):
    """Largest difference over the largest value wanted (or `floor`)."""
    got, want = np.asarray(got, np.float64).reshape(-1), np.asarray(want, np.float64).reshape(-1)
    assert got.shape == want.shape
    fine = np.isfinite(want)
    assert np.array_equal(fine, np.isfinite(got)), what
    assert np.array_equal(got[~fine], want[~fine]), what
    if fine.any():
        size = max(float(np.abs(want[fine]).max()), floor, 1e-300)
        err = float(np.abs(got[fine] - want[fine]).max()) / size
        assert err <= tol, (what, err, tol)


def near_norm(got, want, tol, what="", size=0.0):
    """The difference's norm, at most tol times the wanted values', plus 56u
    times `size`, the terms' whose difference they are."""
    got, want = np.asarray(got, np.float64).reshape(-1), np.asarray(want, np.float64).reshape(-1)
    assert np.isfinite(got).all(), what
    bar = tol * np.linalg.norm(want) + 56 * U * np.linalg.norm(size)
    err = np.linalg.norm(got - want)
    assert err <= bar, (what, err, bar)


# ---- layer norm ----------------------------------------------------------------------


@pytest.mark.parametrize("rows,width", [(1, 1), (3, 2), (5, 31), (2, 128), (7, 129), (33, 512), (4, 513), (9, 1001),
                                        (6, 1024), (700, 2048), (3, 2052), (5, 4096), (3, 8190), (2, 8192), (3, 8196),
                                        (2, 16384), (2, 16385), (3, 20000), (1300, 64),
                                        (300, 8200), (151, 16384), (150, 14340), (2, 57340), (2, 57348)])
@pytest.mark.parametrize("shift", [0.0, 100.0])
def test_layer_norm(lib, rows, width, shift):
    rng = np.random.default_rng(rows * 100003 + width)
    x = (rng.standard_normal((rows, width)) * 1.5 + shift).astype(np.float32)
    gain = (1 + 0.1 * rng.standard_normal(width)).astype(np.float32)
    bias = (0.1 * rng.standard_normal(width)).astype(np.float32)
    dy = rng.standard_normal((rows, width)).astype(np.float32)
    want = R.layer_norm(x, gain, bias, 1e-5, dy)
    bx, bg, bb, by = lib.put(x), lib.put(gain), lib.put(bias), lib.put(dy)
    y, stats, dx = lib.zeros(x.shape, 7.0), lib.zeros((rows, 2), 7.0), lib.zeros(x.shape, 7.0)
    dg, db = lib.zeros(width, 7.0), lib.zeros(width, 7.0)
    lib.ok("layer_norm", bx, bg, bb, y, stats, rows, width, 1e-5)
    lib.ok("layer_norm_backward", bx, bg, stats, by, dx, dg, db, rows, width, False)
    # A mean far from 0 is rounded at its own size, which the narrow spread
    # around it enlarges: |mean| / spread times as much.
    spread = max(float(np.min(x.std(1))), 0.05) if width > 1 else 1.0
    tol = 40 * U * (1 + (abs(shift) + 2) / spread)
    if width > 1:
        near(y.read(), want["y"], tol, "y", 1.0)
        near(dx.read(), want["dx"], 4 * tol, "dx", float(want["stats"][:, 1].max()))
        # Sums over the rows: their terms' errors and (rows / 592 + 40) roundings.
        near(dg.read(), want["dgain"], 2 * tol + (rows / 592 + 40) * U, "dgain", float(rows) ** 0.5 * 3)
    near(db.read(), want["dbias"], (rows / 592 + 40) * U, "dbias", float(rows) ** 0.5 * 3)
    near(stats.read().reshape(rows, 2)[:, 0], want["stats"][:, 0], 30 * U, "mean", 1.0)
    # accumulate adds to what is there; the statistics may be left out.
    before = dx.read()
    lib.ok("layer_norm_backward", bx, bg, stats, by, dx, dg, None, rows, width, True)
    np.testing.assert_allclose(dx.read(), 2 * before, rtol=4 * U, atol=0)
    again = lib.zeros(x.shape)
    lib.ok("layer_norm", bx, bg, bb, again, None, rows, width, 1e-5)
    assert np.array_equal(again.read(), y.read())


def test_layer_norm_without_gain_and_of_no_rows(lib):
    rng = np.random.default_rng(5)
    x, dy = (rng.standard_normal((6, 96)).astype(np.float32) for _ in range(2))
    want = R.layer_norm(x, None, None, 1e-6, dy)
    bx, by, y, stats, dx = lib.put(x), lib.put(dy), lib.zeros(x.shape), lib.zeros((6, 2)), lib.zeros(x.shape)
    lib.ok("layer_norm", bx, None, None, y, stats, 6, 96, 1e-6)
    lib.ok("layer_norm_backward", bx, None, stats, by, dx, None, None, 6, 96, False)
    near(y.read(), want["y"], 120 * U, "y")
    near(dx.read(), want["dx"], 480 * U, "dx")
    dg, db = lib.zeros(96, 3.0), lib.zeros(96, 3.0)
    empty = lib.zeros(0)
    lib.ok("layer_norm", empty, None, None, empty, None, 0, 96, 1e-6)
    lib.ok("layer_norm_backward", empty, None, empty, empty, empty, dg, db, 0, 96, False)
    assert not dg.read().any() and not db.read().any()


def test_layer_norm_rows_do_not_meet(lib):
    """A row with NaN or infinities leaves the others as they are; a constant
    row has rstd 1 / sqrt(eps) and output bias."""
    rng = np.random.default_rng(6)
    x = rng.standard_normal((8, 260)).astype(np.float32)
    y = lib.zeros(x.shape)
    lib.ok("layer_norm", lib.put(x), None, None, y, None, 8, 260, 1e-5)
    clean = y.read().reshape(8, 260)
    x[2, 5], x[4, 7], x[6] = np.nan, np.inf, 3.25
    lib.ok("layer_norm", lib.put(x), None, None, y, None, 8, 260, 1e-5)
    got = y.read().reshape(8, 260)
    keep = [0, 1, 3, 5, 7]
    assert np.array_equal(got[keep], clean[keep])
    assert np.isnan(got[2]).all() and np.isnan(got[4]).all() and not got[6].any()


def test_layer_norm_refusals(lib):
    x, y, s = lib.zeros(64), lib.zeros(64), lib.zeros(8)
    lib.refused("width of at least 1", "layer_norm", x, None, None, y, None, 4, 0, 1e-5)
    lib.refused("finite eps", "layer_norm", x, None, None, y, None, 4, 16, -1.0)
    lib.refused("finite eps", "layer_norm", x, None, None, y, None, 4, 16, float("nan"))
    lib.refused("input buffer holds 64", "layer_norm", x, None, None, y, None, 5, 16, 1e-5)
    lib.refused("out overlaps input", "layer_norm", x, None, None, x, None, 4, 16, 1e-5)
    lib.refused("out overlaps stats", "layer_norm", x, None, None, y, y, 4, 16, 1e-5)
    lib.refused("null buffer", "layer_norm_backward", x, None, None, y, s, None, None, 4, 16, False)
    view = lib.Buffer(lib.ctx, lib.lib.tysor_cuda_buffer_view(s.handle, 1, 2), 2)
    lib.refused("8-byte boundary", "layer_norm", x, None, None, y, view, 1, 16, 1e-5)


# ---- rotary positions -------------------------------------------------------------------


def sections_ptr(sections):
    from tysor_b200 import native
    a = np.asarray(sections, np.int64)
    return a, a.ctypes.data_as(native.I64P)


@pytest.mark.parametrize("batch,heads,seq,sections", [(1, 1, 1, (1,)), (1, 16, 1, (16, 24, 24)), (2, 3, 5, (2, 3, 1)),
                                                      (3, 4, 77, (8, 12, 12)), (1, 2, 130, (5, 6)), (2, 8, 33, (32,)),
                                                      (1, 1, 9, (1, 1, 1, 1, 1, 1, 1, 1)), (1, 40, 3, (40, 88)),
                                                      (1, 70001, 1, (1,))])
@pytest.mark.parametrize("seq_major", [False, True])
def test_rope_axes(lib, batch, heads, seq, sections, seq_major):
    rng = np.random.default_rng(seq * 31 + heads)
    half = sum(sections)
    shape = (batch, seq, heads, 2 * half) if seq_major else (batch, heads, seq, 2 * half)
    x = rng.standard_normal(shape).astype(np.float32)
    pos = rng.integers(0, 2000000, (batch, len(sections), seq)).astype(np.float32)
    pos[0, 0, 0] = 0
    keep, ptr = sections_ptr(sections)
    bx, bp, y = lib.put(x), lib.put(pos), lib.zeros(shape, 9.0)
    lib.ok("rope_axes", bx, bp, y, batch, heads, seq, ptr, len(sections), 10000.0, seq_major)
    size = float(np.sqrt(x[..., :half].astype(np.float64) ** 2 + x[..., half:].astype(np.float64) ** 2).max())
    near(y.read(), R.rope_axes(x, pos, sections, 10000.0, seq_major), 8 * U, "y", size)
    dx = lib.zeros(shape, 9.0)
    lib.ok("rope_axes_backward", bx, bp, dx, batch, heads, seq, ptr, len(sections), 10000.0, seq_major, False)
    want = R.rope_axes(x, pos, sections, 10000.0, seq_major, back=True)
    near(dx.read(), want, 8 * U, "dx", size)
    lib.ok("rope_axes_backward", bx, bp, dx, batch, heads, seq, ptr, len(sections), 10000.0, seq_major, True)
    near(dx.read(), 2 * want, 8 * U, "accumulated", 2 * size)


def test_rope_axes_of_equal_positions_is_rope(lib):
    """Positions 0, 1, 2, ... on every axis turn as rope does (whose angles are
    formed in 32 bits: half a step of an angle up to 63, 2^-19, each way)."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((2, 3, 64, 32)).astype(np.float32)
    pos = np.broadcast_to(np.arange(64, dtype=np.float32), (2, 3, 64))
    keep, ptr = sections_ptr((4, 6, 6))
    bx, y, z = lib.put(x), lib.zeros(x.shape), lib.zeros(x.shape)
    lib.ok("rope_axes", bx, lib.put(pos), y, 2, 3, 64, ptr, 3, 10000.0, False)
    lib.ok("rope", bx, z, 6, 64, 16, 10000.0)
    near(y.read(), z.read(), 2.0 ** -18, "rope")


def test_rope_axes_refusals(lib):
    x, p, y = lib.zeros(64), lib.zeros(16), lib.zeros(64)
    keep, ptr = sections_ptr((2, 2))
    lib.refused("1 to 8 axes", "rope_axes", x, p, y, 1, 1, 8, ptr, 0, 10000.0, False)
    lib.refused("1 to 8 axes", "rope_axes", x, p, y, 1, 1, 8, ptr, 9, 10000.0, False)
    lib.refused("1 to 8 axes", "rope_axes", x, p, y, 1, 1, 8, None, 2, 10000.0, False)
    lib.refused("finite theta", "rope_axes", x, p, y, 1, 1, 8, ptr, 2, 0.0, False)
    lib.refused("positions buffer holds 16", "rope_axes", x, p, y, 1, 0, 9, ptr, 2, 10000.0, False)
    lib.refused("out overlaps input", "rope_axes", x, p, x, 1, 1, 8, ptr, 2, 10000.0, False)
    lib.refused("sizes overflow", "rope_axes", x, p, y, 1 << 30, 1 << 30, 1 << 30, ptr, 2, 10000.0, False)
    keep, ptr = sections_ptr((2, 0))
    lib.refused("1 to 65536 pairs", "rope_axes", x, p, y, 1, 1, 8, ptr, 2, 10000.0, False)


# ---- attention -----------------------------------------------------------------------------


def attention_inputs(seed, batch, heads, kv_heads, q_len, k_len, dim, seq_major):
    rng = np.random.default_rng(seed)
    qs = (batch, q_len, heads, dim) if seq_major else (batch, heads, q_len, dim)
    ks = (batch, k_len, kv_heads, dim) if seq_major else (batch, kv_heads, k_len, dim)
    return [rng.standard_normal(s).astype(np.float32) for s in (qs, ks, ks, qs)]


def run_attention(lib, q, k, v, dout, starts, lengths, dims, window, sinks, scale, seq_major, backward=True,
                  accumulate=False, fill=5.0):
    batch, heads, kv_heads, q_len, k_len, dim = dims
    shape = (batch, heads, kv_heads, q_len, k_len, dim, window, sinks, scale, seq_major)
    bq, bk, bv, bd = (lib.put(t) for t in (q, k, v, dout))
    bs, bl = lib.put(starts), lib.put(lengths)
    out, stats = lib.zeros(q.shape, fill), lib.zeros((batch, heads, q_len, 2), fill)
    lib.ok("window_attention", bq, bk, bv, bs, bl, out, stats, *shape)
    r = {"out": out.read(), "stats": stats.read().reshape(batch, heads, q_len, 2)}
    if backward:
        dq, dk, dv = lib.zeros(q.shape, fill), lib.zeros(k.shape, fill), lib.zeros(v.shape, fill)
        lib.ok("window_attention_backward", bq, bk, bv, bs, bl, out, stats, bd, dq, dk, dv, *shape, accumulate)
        r.update(dq=dq.read(), dk=dk.read(), dv=dv.read())
    return {n: t.reshape(q.shape if n in ("out", "dq") else k.shape if n in ("dk", "dv") else t.shape)
            for n, t in r.items()}


def compare_attention(got, want, backward=True):
    tol = 510 * U
    near_norm(got["out"], want["out"], tol, "out")
    near(got["out"], want["out"], 4 * tol, "out")
    # The greatest score alone and the sum: absolute errors of single scores.
    live = np.isfinite(want["stats"][..., 0])
    assert np.array_equal(live, np.isfinite(got["stats"][..., 0]))
    assert np.array_equal(got["stats"][~live], want["stats"][~live])
    near(got["stats"][live], want["stats"][live], 2 * tol, "stats")
    if backward:
        # dS = P (dP - delta): both are dot products of at most 128 terms in at
        # most 28 additions, 56u of their terms' size off each, however small
        # their difference (0 for a row that sees one key).
        for n in ("dq", "dk", "dv"):
            size = want.get("size_" + n, np.zeros(1))
            near_norm(got[n], want[n], 3 * tol, n, size)
            near(got[n], want[n], 8 * tol, n, float(size.max()))


CASES = [  # batch, heads, kv_heads, q_len, k_len, dim, window, sinks
    (1, 1, 1, 1, 1, 1, 0, 0), (1, 2, 1, 3, 3, 3, 1, 0), (2, 4, 2, 17, 17, 33, 4, 2), (1, 2, 2, 64, 64, 64, 0, 0),
    (1, 2, 1, 65, 65, 65, 16, 1), (2, 2, 1, 127, 127, 16, 40, 4), (1, 4, 2, 128, 128, 128, 0, 0),
    (1, 3, 3, 129, 129, 80, 128, 0), (2, 4, 1, 257, 257, 128, 64, 130), (1, 5, 1, 300, 300, 40, 129, 7),
    (1, 2, 1, 513, 513, 128, 100, 1), (1, 1, 1, 400, 400, 112, 1000, 4), (1, 2, 2, 385, 385, 96, 1, 3),
    (2, 4, 2, 1, 50, 128, 0, 0), (3, 8, 2, 1, 700, 128, 64, 4), (1, 4, 4, 1, 1500, 64, 0, 0), (2, 6, 2, 5, 333, 72, 50, 2),
    (1, 16, 1, 2, 2100, 128, 0, 0), (1, 2, 1, 40, 900, 128, 300, 4), (1, 2, 1, 200, 130, 32, 0, 0),
    (1, 1, 1, 150, 1000, 65, 0, 0), (2, 20, 4, 3, 260, 33, 30, 1),
    # Few query tiles over many keys: their key tiles are cut into segments.
    (1, 5, 1, 5, 3000, 128, 0, 0), (2, 3, 1, 30, 4001, 64, 0, 0), (1, 2, 1, 1300, 1300, 40, 0, 0),
    # More than eight rows of a key head, straight from the cache.
    (2, 9, 1, 1, 900, 64, 0, 0), (1, 40, 2, 1, 1300, 128, 300, 5), (1, 8, 2, 5, 700, 33, 0, 0), (1, 33, 1, 2, 130, 80, 20, 3),
    (1, 2, 2, 130, 2500, 72, 1500, 140), (1, 1, 1, 1100, 600, 128, 0, 0), (1, 8, 2, 600, 600, 33, 70, 5),
]


@pytest.mark.parametrize("seq_major", [False, True])
@pytest.mark.parametrize("dims", CASES, ids=lambda c: "x".join(map(str, c)))
def test_window_attention(lib, dims, seq_major):
    batch, heads, kv_heads, q_len, k_len, dim, window, sinks = dims
    q, k, v, dout = attention_inputs(sum(dims), *dims[:6], seq_major)
    scale = dim ** -0.5
    want = R.window_attention(q, k, v, None, None, window, sinks, scale, seq_major, dout)
    got = run_attention(lib, q, k, v, dout, None, None, dims[:6], window, sinks, scale, seq_major)
    compare_attention(got, want)
    lib.ctx.synchronize()


@pytest.mark.parametrize("dims", [(4, 4, 2, 150, 150, 64, 30, 2), (3, 2, 1, 260, 260, 128, 0, 0),
                                  (5, 4, 1, 1, 300, 128, 40, 3), (3, 8, 8, 1, 700, 64, 0, 0),
                                  (4, 2, 1, 70, 290, 40, 64, 1)], ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("seq_major", [False, True])
def test_window_attention_of_padded_sequences(lib, dims, seq_major):
    """Each sequence has a length of its own (full, one, none, ...); what lies
    behind it holds NaN and infinities and reaches no result."""
    batch, heads, kv_heads, q_len, k_len, dim, window, sinks = dims
    q, k, v, dout = attention_inputs(sum(dims), *dims[:6], seq_major)
    rng = np.random.default_rng(1)
    lengths = rng.integers(1, k_len + 1, batch).astype(np.float32)
    lengths[0], lengths[1], lengths[2] = k_len, 1, 0
    starts = np.zeros(batch, np.float32) if q_len == k_len else lengths - q_len  # partly negative
    for b in range(batch):
        n = int(lengths[b])
        for t, bad in ((k, np.nan), (v, np.inf)):
            rows = t[b] if seq_major else np.swapaxes(t[b], 0, 1)
            rows[n:] = bad
        live = starts[b] + np.arange(q_len)
        dead = (live < 0) | (live >= n)
        for t in (q, dout):
            (t[b] if seq_major else np.swapaxes(t[b], 0, 1))[dead] = np.nan
    scale = dim ** -0.5
    want = R.window_attention(q, k, v, starts, lengths, window, sinks, scale, seq_major, dout)
    got = run_attention(lib, q, k, v, dout, starts, lengths, dims[:6], window, sinks, scale, seq_major)
    compare_attention(got, want)
    lib.ctx.synchronize()


@pytest.mark.parametrize("dims", [(1, 2, 1, 200, 200, 64, 20, 2), (1, 2, 2, 300, 300, 128, 0, 0),
                                  (1, 4, 1, 1, 400, 128, 16, 2)], ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_window_attention_of_values_that_are_not_finite(lib, dims, bad):
    """A key that a row does not see takes no part in it, whatever it holds:
    rows before it and rows whose window has passed it stay as they are."""
    batch, heads, kv_heads, q_len, k_len, dim, window, sinks = dims
    q, k, v, dout = attention_inputs(7, *dims[:6], False)
    scale = dim ** -0.5
    at = 150 if q_len > 1 else 100
    want = R.window_attention(q, k, v, None, None, window, sinks, scale, False, dout)
    seen = R.visible(None, None, batch, q_len, k_len, window, sinks)[0, :, at]
    k[:, :, at], v[:, :, at] = bad, bad
    got = run_attention(lib, q, k, v, dout, None, None, dims[:6], window, sinks, scale, False)
    for n in ("out", "dq"):
        near_norm(got[n][:, :, ~seen], want[n][:, :, ~seen], 3 * 510 * U, n)
        assert not np.isfinite(got[n][:, :, seen]).all() or not seen.any()
    # Keys that only rows without it see.
    reached = R.visible(None, None, batch, q_len, k_len, window, sinks)[0][seen].any(0)
    for n in ("dk", "dv"):
        near(got[n][:, :, ~reached], want[n][:, :, ~reached], 8 * 510 * U, n, float(np.abs(want[n]).max()))


@pytest.mark.parametrize("size", [1e-12, 1e4, 1e20])
def test_window_attention_of_any_size(lib, size):
    """Inputs far from 1, tokens of very different sizes among them: the scale
    argument keeps the scores ordinary, the sizes pass through."""
    dims = (1, 2, 1, 270, 270, 64)
    q, k, v, dout = attention_inputs(11, *dims, False)
    k[:, :, 40] *= 1e3
    v[:, :, 200] *= 1e4
    q, k, v, dout = (t * np.float32(size) for t in (q, k, v, dout))
    scale = 64 ** -0.5 / size / size / 1e2
    if scale < 2.0 ** -126:  # subnormal: fp32 holds it to 2^-149 only, 0.6% of 1.25e-43, so the call is refused
        bufs = [lib.put(t) for t in (q, k, v)]
        lib.refused("finite scale", "window_attention", *bufs, None, None, lib.zeros(q.shape), None, *dims, 100, 3,
                    scale, False)
        return
    want = R.window_attention(q, k, v, None, None, 100, 3, scale, False, dout)
    got = run_attention(lib, q, k, v, dout, None, None, dims, 100, 3, scale, False)
    tol = 510 * U * 10  # scores up to ten times as large
    for n in ("out", "dq", "dk", "dv"):
        near_norm(got[n], want[n], tol, n)


@pytest.mark.parametrize("which,size", [("qk", 2.0 ** -70), ("v", 2.0 ** 126), ("q0", 2.0 ** 90)])
def test_window_attention_at_the_ends_of_the_range(lib, which, size):
    """Queries and keys so small that a score is below fp32's least value (every
    visible key then counts the same), values near fp32's greatest, and a query
    of zeros beside ones so large that no score of theirs fits fp32."""
    dims = (1, 2, 1, 270, 270, 64)
    q, k, v, dout = attention_inputs(13, *dims, False)
    if which == "qk":
        q, k = q * np.float32(size), k * np.float32(size)
    elif which == "v":
        v = np.clip(v, -1, 1) * np.float32(size)
        dout *= np.float32(2.0 ** -100)
    else:
        q, k = q * np.float32(size), k * np.float32(size)
        q[:, :, 77] = 0
    want = R.window_attention(q, k, v, None, None, 100, 3, 0.125, False, dout)
    got = run_attention(lib, q, k, v, dout, None, None, dims, 100, 3, 0.125, False)
    if which == "q0":  # only the row of zeros has a value to compare
        near_norm(got["out"][:, :, 77], want["out"][:, :, 77], 510 * U, "out")
        return
    near_norm(got["out"], want["out"], 510 * U, "out")
    # The terms of dS cancel where all probabilities are alike: their own size counts.
    for n in ("dq", "dk", "dv"):
        near_norm(got[n], want[n], 3 * 510 * U, n, want.get("size_" + n, np.zeros(1)))


@pytest.mark.parametrize("dim", [64, 128])
def test_window_attention_of_many_short_items(lib, dim):
    """More work items than blocks, of one to three key tiles each: a block's
    items follow one another through the pipeline."""
    dims = (3, 40, 8, 384, 384, dim)
    q, k, v, dout = attention_inputs(17, *dims, True)
    lengths = np.array([384, 100, 257], np.float32)
    starts = np.zeros(3, np.float32)
    want = R.window_attention(q, k, v, starts, lengths, 60, 2, dim ** -0.5, True, dout)
    for _ in range(3):
        got = run_attention(lib, q, k, v, dout, starts, lengths, dims, 60, 2, dim ** -0.5, True)
        compare_attention(got, want)


def test_window_attention_gradients_against_differences(lib):
    """A few coordinates of each gradient against central differences of the
    64-bit forward: a step h leaves h^2 / 6 of the third derivative (about 1),
    1e-6 here, above the kernel's own error."""
    dims = (2, 4, 2, 37, 37, 24)
    q, k, v, dout = attention_inputs(3, *dims, True)
    got = run_attention(lib, q, k, v, dout, None, None, dims, 9, 2, 0.3, True)

    def loss(t):
        o = R.window_attention(t[0], t[1], t[2], None, None, 9, 2, 0.3, True)["out"]
        return float((o * dout.astype(np.float64)).sum())

    rng = np.random.default_rng(0)
    h = 1e-3
    for i, name in enumerate(("dq", "dk", "dv")):
        base = [q.astype(np.float64), k.astype(np.float64), v.astype(np.float64)]
        for _ in range(12):
            at = tuple(rng.integers(0, n) for n in base[i].shape)
            held = base[i][at]
            base[i][at] = held + h
            up = loss(base)
            base[i][at] = held - h
            down = loss(base)
            base[i][at] = held
            assert abs((up - down) / (2 * h) - got[name][at]) < 2e-5 * max(1.0, abs(got[name][at]))


def test_window_attention_accumulates_and_repeats(lib):
    dims = (2, 4, 2, 140, 140, 64)
    q, k, v, dout = attention_inputs(5, *dims, False)
    a = run_attention(lib, q, k, v, dout, None, None, dims, 50, 2, 0.125, False)
    b = run_attention(lib, q, k, v, dout, None, None, dims, 50, 2, 0.125, False)
    c = run_attention(lib, q, k, v, dout, None, None, dims, 50, 2, 0.125, False, accumulate=True, fill=1.5)
    for n in a:
        assert np.array_equal(a[n], b[n]), n  # the same bits every time
    for n in ("dq", "dk", "dv"):
        np.testing.assert_allclose(c[n], a[n] + 1.5, rtol=4 * U, atol=4 * U * 1.5)


@pytest.mark.parametrize("dims,window,sinks", [((3, 2, 1, 150, 2200, 64), 0, 0), ((2, 4, 1, 5, 3000, 128), 1100, 20)])
def test_window_attention_of_segments_that_are_empty_or_not_finite(lib, dims, window, sinks):
    """Sequences too short to fill their segments, and rows that meet a NaN."""
    batch, heads, kv_heads, q_len, k_len, dim = dims
    q, k, v, dout = attention_inputs(23, *dims, False)
    lengths = np.array([k_len, 700, 0], np.float32)[:batch]
    starts = np.array([k_len - q_len, 690, -3], np.float32)[:batch]
    want = R.window_attention(q, k, v, starts, lengths, window, sinks, 0.1, False, dout)
    got = run_attention(lib, q, k, v, dout, starts, lengths, dims, window, sinks, 0.1, False)
    compare_attention(got, want)
    k[0, :, k_len - 3] = np.nan  # seen by the last queries of the first sequence
    got = run_attention(lib, q, k, v, dout, starts, lengths, dims, window, sinks, 0.1, False)
    seen = R.visible(starts, lengths, batch, q_len, k_len, window, sinks)[:, :, k_len - 3]
    assert seen[0].sum() == 3
    for n in ("out", "dq"):
        assert np.isnan(got[n][0, :, seen[0]]).all()
        near_norm(got[n][0, :, ~seen[0]], want[n][0, :, ~seen[0]], 3 * 510 * U, n)
        near_norm(got[n][1:], want[n][1:], 3 * 510 * U, n)


def test_window_attention_far_offsets(lib):
    """A cache whose offsets pass 2^31 values: 17 million keys of 128, the rows
    at its end."""
    import torch
    keys, dim = (1 << 24) + 9, 128
    cache = torch.zeros((1, 1, keys, dim), device="cuda")
    q, k, v, dout = attention_inputs(9, 1, 2, 1, 1, 40, dim, False)
    cache[0, 0, -40:] = torch.from_numpy(k[0, 0]).cuda()
    torch.cuda.synchronize()
    kv = lib.Buffer.wrap(lib.ctx, cache)
    vv = cache.clone()
    torch.cuda.synchronize()
    bv = lib.Buffer.wrap(lib.ctx, vv)
    out = lib.zeros(q.shape)
    want = R.window_attention(q, k, k, None, None, 32, 0, 0.1, False)
    for q_len in (1,):
        lib.ok("window_attention", lib.put(q), kv, bv, None, None, out, None, 1, 2, 1, q_len, keys, dim, 32, 0, 0.1,
               False)
    near_norm(out.read(), want["out"], 510 * U, "out")


def test_window_attention_bad_lengths_are_errors(lib):
    dims = (2, 2, 1, 20, 20, 32)
    q, k, v, dout = attention_inputs(5, *dims, False)
    clean = run_attention(lib, q, k, v, dout, None, None, dims, 8, 0, 0.2, False)
    for starts, lengths in (([0, 0], [20, 21]), ([0, 0], [20, -1]), ([0, 0], [20, np.nan]), ([0, np.inf], [20, 20]),
                            ([0, 2e9], [20, 20])):
        bufs = [lib.put(t) for t in (q, k, v)]
        out = lib.zeros(q.shape, 5.0)
        lib.ok("window_attention", *bufs, lib.put(np.float32(starts)), lib.put(np.float32(lengths)), out, None, *dims,
               8, 0, 0.2, False)
        with pytest.raises(lib.native.NativeError, match="start or length out of range"):
            lib.ctx.synchronize()
        got = out.read().reshape(q.shape)
        assert np.array_equal(got[0], clean["out"][0]) and not got[1].any()


def test_window_attention_refusals(lib):
    q, k, v, out = (lib.zeros(4096) for _ in range(4))
    ok = (1, 2, 1, 16, 16, 32, 4, 1, 0.1, False)

    def bad(message, *shape):
        lib.refused(message, "window_attention", q, k, v, None, None, out, None, *shape)

    bad("must divide", 1, 3, 2, 16, 16, 32, 4, 1, 0.1, False)
    bad("must divide", 1, 2, 0, 16, 16, 32, 4, 1, 0.1, False)
    bad("1 to 128 values", 1, 2, 1, 16, 16, 129, 4, 1, 0.1, False)
    bad("1 to 128 values", 1, 2, 1, 16, 16, 0, 4, 1, 0.1, False)
    bad("finite scale", 1, 2, 1, 16, 16, 32, 4, 1, 0.0, False)
    bad("finite scale", 1, 2, 1, 16, 16, 32, 4, 1, float("inf"), False)
    bad("q buffer holds 4096", 1, 2, 1, 65, 16, 32, 4, 1, 0.1, False)
    bad("k buffer holds 4096", 1, 2, 1, 16, 129, 32, 4, 1, 0.1, False)
    bad("sizes overflow", 1 << 29, 1 << 20, 1, 1 << 29, 1, 32, 4, 1, 0.1, False)
    bad("up to 2^29", (1 << 29) + 1, 2, 1, 16, 16, 32, 4, 1, 0.1, False)
    lib.refused("out overlaps q", "window_attention", q, k, v, None, None, q, None, *ok)
    lib.refused("lengths buffer holds 0", "window_attention", q, k, v, None, lib.zeros(0), out, None, *ok)
    lib.refused("null buffer", "window_attention_backward", q, k, v, None, None, out, None, q, k, v, out, *ok, False)
    empty = lib.zeros(0)
    lib.ok("window_attention", empty, empty, empty, None, None, empty, None, 0, 2, 1, 16, 16, 32, 4, 1, 0.1, False)
    # No keys at all: every row is empty.
    lib.ok("window_attention", q, empty, empty, None, None, out, None, 1, 2, 1, 16, 0, 32, 4, 1, 0.1, False)
    assert not out.read(1024).any()


# ---- distillation ------------------------------------------------------------------------------


def distill_inputs(rows, width, top, seed=0):
    rng = np.random.default_rng(seed)
    z = (2 * rng.standard_normal((rows, width))).astype(np.float32)
    ids = np.stack([rng.permutation(width)[:top] for _ in range(rows)]).astype(np.float32)
    teacher = (3 * rng.standard_normal((rows, top))).astype(np.float32)
    dloss = rng.standard_normal(rows).astype(np.float32)
    return z, ids, teacher, dloss


def run_distill(lib, z, ids, teacher, dloss, t, accumulate=False, fill=5.0):
    rows, width = z.shape
    top = ids.shape[1]
    bz, bi, bt = lib.put(z), lib.put(ids), lib.put(teacher)
    loss, stats, grad = lib.zeros(rows, fill), lib.zeros((rows, 2), fill), lib.zeros(z.shape, fill)
    lib.ok("distill_loss", bz, bi, bt, loss, stats, rows, width, top, t)
    lib.ok("distill_loss_backward", bz, bi, bt, stats, lib.put(dloss), grad, rows, width, top, t, accumulate)
    return {"loss": loss.read(), "stats": stats.read().reshape(rows, 2), "grad": grad.read().reshape(z.shape)}


def compare_distill(got, want, t):
    near(got["loss"], want["loss"], 240 * U * max(1.0, t * t), "loss", 1.0)
    near(got["stats"][:, 0], want["stats"][:, 0], 0.0, "max")
    assert np.all(np.abs(got["stats"][:, 1] / want["stats"][:, 1] - 1) <= 240 * U)
    near(got["grad"], want["grad"], 240 * U, "grad")


@pytest.mark.parametrize("rows,width,top", [(1, 1, 1), (2, 3, 2), (5, 64, 7), (3, 1001, 64), (4, 4096, 1), (2, 32000, 64),
                                            (7, 50257, 20), (1, 128003, 300), (600, 515, 8), (9, 2050, 1024)])
@pytest.mark.parametrize("t", [1.0, 2.5])
def test_distill_loss(lib, rows, width, top, t):
    z, ids, teacher, dloss = distill_inputs(rows, width, top, rows + width)
    want = R.distill_loss(z, ids, teacher, t, dloss)
    got = run_distill(lib, z, ids, teacher, dloss, t)
    compare_distill(got, want, t)
    acc = run_distill(lib, z, ids, teacher, dloss, t, accumulate=True, fill=0.25)
    np.testing.assert_allclose(acc["grad"], got["grad"] + 0.25, rtol=0, atol=8 * U * (1 + np.abs(got["grad"]).max()))
    lib.ctx.synchronize()


def test_distill_loss_of_absent_and_repeated_entries(lib):
    z, ids, teacher, dloss = distill_inputs(8, 300, 6)
    ids[1, 2:] = -1                      # fewer entries
    ids[2] = -1                          # none
    ids[3, 4], ids[3, 5] = ids[3, 0], ids[3, 0]   # the same id three times
    teacher[4, 1] = -np.inf              # an entry of no weight
    teacher[5] = -np.inf                 # nothing left
    teacher[1, 3] = np.nan               # behind an absent id
    z[2, 7] = np.nan                     # a padded row may hold anything
    want = R.distill_loss(np.where(np.isnan(z), 0, z), ids, teacher, 2.0, dloss)
    got = run_distill(lib, z, ids, teacher, dloss, 2.0)
    keep = np.arange(8) != 2
    compare_distill({n: v[keep] for n, v in got.items()}, {n: v[keep] for n, v in want.items()}, 2.0)
    assert got["loss"][2] == 0 and not got["grad"][2].any() and got["loss"][5] == 0 and not got["grad"][5].any()
    # The largest and smallest finite logits; a -inf logit has probability 0.
    z[0, :3] = (3e38, -3e38, -np.inf)
    ids[0] = (0, 5, 6, 7, 8, 9)
    want = R.distill_loss(z[:1], ids[:1], teacher[:1], 2.0, dloss[:1])
    got = run_distill(lib, z[:1], ids[:1], teacher[:1], dloss[:1], 2.0)
    compare_distill(got, want, 2.0)


@pytest.mark.parametrize("width", [1, 20, 700, 40000])
def test_distill_loss_of_many_entries(lib, width):
    """The most entries a row may have, ids in any order and many times."""
    rng = np.random.default_rng(width)
    z = (2 * rng.standard_normal((3, width))).astype(np.float32)
    ids = rng.integers(-1, width, (3, 1024)).astype(np.float32)
    ids[2] = rng.integers(0, min(width, 3), 1024)
    teacher = (3 * rng.standard_normal((3, 1024))).astype(np.float32)
    dloss = rng.standard_normal(3).astype(np.float32)
    want = R.distill_loss(z, ids, teacher, 2.0, dloss)
    got = run_distill(lib, z, ids, teacher, dloss, 2.0)
    near(got["loss"], want["loss"], 240 * U * 4, "loss", 1.0)
    # q and the entries' p cancel: both are at most 1, p sums up to 1024 terms of
    # them (at most 1024u / 2 off, in order), times T dloss.
    near(got["grad"], want["grad"], (240 + 512) * U, "grad", float(2 * np.abs(dloss).max()))
    again = run_distill(lib, z, ids, teacher, dloss, 2.0)
    assert np.array_equal(got["grad"], again["grad"])


def test_distill_loss_of_entries_that_are_no_numbers(lib):
    """A teacher's NaN makes its own row's loss NaN, absent entries beside it
    notwithstanding, and no other row's."""
    z, ids, teacher, dloss = distill_inputs(5, 300, 6)
    clean = run_distill(lib, z, ids, teacher, dloss, 2.0)
    ids[1, 3:] = -1
    teacher[1, 0], teacher[3, 2] = np.nan, np.inf
    got = run_distill(lib, z, ids, teacher, dloss, 2.0)
    assert np.isnan(got["loss"][[1, 3]]).all()
    keep = [0, 2, 4]
    for n in ("loss", "grad", "stats"):
        assert np.array_equal(got[n][keep], clean[n][keep]), n
    lib.ctx.synchronize()


def test_distill_gradient_against_differences(lib):
    z, ids, teacher, dloss = distill_inputs(4, 30, 5)
    got = run_distill(lib, z, ids, teacher, dloss, 1.5)["grad"]
    h = 1e-4
    for r in range(4):
        for c in (0, int(ids[r, 0]), 29):
            up, down = z.astype(np.float64), z.astype(np.float64)
            up[r, c] += h
            down[r, c] -= h
            d = (R.distill_loss(up, ids, teacher, 1.5)["loss"] - R.distill_loss(down, ids, teacher, 1.5)["loss"])[r]
            assert abs(d / (2 * h) * dloss[r] - got[r, c]) < 1e-6


def test_distill_bad_ids_are_errors(lib):
    z, ids, teacher, dloss = distill_inputs(3, 40, 4)
    for bad in (40.0, 1e9, np.nan, np.inf):
        broken = ids.copy()
        broken[1, 2] = bad
        with pytest.raises(lib.native.NativeError, match="index out of range"):
            run_distill(lib, z, broken, teacher, dloss, 1.0)
        lib.ctx.synchronize()  # reported once


def test_distill_refusals(lib):
    z, e, out, s = lib.zeros(400), lib.zeros(40), lib.zeros(10), lib.zeros(20)
    lib.refused("1 to 1024 entries", "distill_loss", z, e, e, out, s, 10, 40, 0, 1.0)
    lib.refused("1 to 1024 entries", "distill_loss", z, e, e, out, s, 10, 40, 1025, 1.0)
    lib.refused("width of 1", "distill_loss", z, e, e, out, s, 10, 0, 4, 1.0)
    for t in (0.0, -1.0, float("nan"), float("inf")):
        lib.refused("finite temperature", "distill_loss", z, e, e, out, s, 10, 40, 4, t)
    for t in (2.0 ** -61, 2.0 ** 61):
        lib.refused("from 2^-60 to 2^60", "distill_loss", z, e, e, out, s, 10, 40, 4, t)
    lib.refused("teacher buffer holds 10", "distill_loss", z, e, out, out, s, 10, 40, 4, 1.0)
    lib.refused("grad overlaps logits", "distill_loss_backward", z, e, e, s, None, z, 10, 40, 4, 1.0, False)
    lib.ok("distill_loss", z, e, e, out, None, 0, 40, 4, 1.0)


# ---- views -------------------------------------------------------------------------------------


def odd(lib, a, keep):
    """The values of `a` in a view that starts one float into its buffer."""
    flat = np.concatenate([np.full(1, 3.0, np.float32), np.asarray(a, np.float32).reshape(-1), np.full(1, 3.0, np.float32)])
    base = lib.put(flat)
    keep.append(base)
    return lib.Buffer(lib.ctx, lib.lib.tysor_cuda_buffer_view(base.handle, 1, flat.size - 2), flat.size - 2)


def untouched(keep):
    return all(b.read().reshape(-1)[[0, -1]].tolist() == [3.0, 3.0] for b in keep)


@pytest.mark.parametrize("dims", [(1, 4, 2, 140, 140, 64), (2, 4, 2, 1, 900, 128)], ids=["tiles", "one"])
def test_window_attention_on_odd_views(lib, dims):
    q, k, v, dout = attention_inputs(29, *dims, True)
    want = R.window_attention(q, k, v, None, None, 50, 3, 0.1, True, dout)
    keep = []
    bq, bk, bv, bd = (odd(lib, t, keep) for t in (q, k, v, dout))
    out, dq, dk, dv = (odd(lib, np.full(t.shape, 9.0), keep) for t in (q, q, k, v))
    stats = lib.zeros((dims[0], dims[1], dims[3], 2))
    shape = (*dims, 50, 3, 0.1, True)
    lib.ok("window_attention", bq, bk, bv, None, None, out, stats, *shape)
    lib.ok("window_attention_backward", bq, bk, bv, None, None, out, stats, bd, dq, dk, dv, *shape, False)
    got = {n: b.read().reshape(want[n].shape) for n, b in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv))}
    got["stats"] = stats.read().reshape(want["stats"].shape)
    compare_attention(got, want)
    assert untouched(keep)


def test_other_operators_on_odd_views(lib):
    rng = np.random.default_rng(31)
    keep = []
    x, dy = (rng.standard_normal((5, 256)).astype(np.float32) for _ in range(2))
    gain, bias = (rng.standard_normal(256).astype(np.float32) for _ in range(2))
    want = R.layer_norm(x, gain, bias, 1e-5, dy)
    bx, by, bg, bb = (odd(lib, t, keep) for t in (x, dy, gain, bias))
    y, dx, dg, db = (odd(lib, np.full(t.shape, 9.0), keep) for t in (x, x, gain, bias))
    stats = lib.zeros((5, 2))
    lib.ok("layer_norm", bx, bg, bb, y, stats, 5, 256, 1e-5)
    lib.ok("layer_norm_backward", bx, bg, stats, by, dx, dg, db, 5, 256, False)
    tol = 40 * U * 4  # as in test_layer_norm, means of about 0 over a spread of about 1
    near(y.read(), want["y"], tol, "y", 1.0)
    near(dx.read(), want["dx"], 4 * tol, "dx", 1.0)
    near(dg.read(), want["dgain"], 4 * tol, "dgain", 1.0)
    near(db.read(), want["dbias"], 4 * tol, "dbias", 1.0)

    section, ptr = sections_ptr((4, 8))
    heads = rng.standard_normal((2, 3, 7, 24)).astype(np.float32)
    pos = rng.integers(0, 5000, (2, 2, 7)).astype(np.float32)
    out = odd(lib, np.full(heads.shape, 9.0), keep)
    lib.ok("rope_axes", odd(lib, heads, keep), odd(lib, pos, keep), out, 2, 3, 7, ptr, 2, 10000.0, False)
    near(out.read(), R.rope_axes(heads, pos, (4, 8), 10000.0, False), 8 * U * 2, "rope_axes", 1.0)

    z, ids, teacher, dloss = distill_inputs(6, 1000, 9)
    want = R.distill_loss(z, ids, teacher, 2.0, dloss)
    bz, bi, bt, bd = (odd(lib, t, keep) for t in (z, ids, teacher, dloss))
    loss, grad, stats = odd(lib, np.full(6, 9.0), keep), odd(lib, np.full(z.shape, 9.0), keep), lib.zeros((6, 2))
    lib.ok("distill_loss", bz, bi, bt, loss, stats, 6, 1000, 9, 2.0)
    lib.ok("distill_loss_backward", bz, bi, bt, stats, bd, grad, 6, 1000, 9, 2.0, False)
    compare_distill({"loss": loss.read(), "stats": stats.read().reshape(6, 2), "grad": grad.read().reshape(z.shape)},
                    want, 2.0)
    assert untouched(keep)


# ---- wrapped memory ----------------------------------------------------------------------------


def test_wrapped_tensors(lib):
    """The operators on another library's tensors, without a copy, after other
    work on the caller's stream."""
    import torch
    x = torch.randn(64, 96, device="cuda")
    y = torch.empty_like(x)
    stream = torch.cuda.ExternalStream(lib.lib.tysor_cuda_context_stream(lib.ctx.handle))
    x.mul_(2.0)
    stream.wait_stream(torch.cuda.current_stream())
    lib.ok("layer_norm", lib.Buffer.wrap(lib.ctx, x), None, None, lib.Buffer.wrap(lib.ctx, y), None, 64, 96, 1e-5)
    torch.cuda.current_stream().wait_stream(stream)
    near(y.cpu().numpy(), R.layer_norm(x.cpu().numpy(), None, None, 1e-5)["y"], 120 * U)
    with pytest.raises(ValueError, match="float32"):
        lib.Buffer.wrap(lib.ctx, x.double())
    with pytest.raises(ValueError, match="contiguous"):
        lib.Buffer.wrap(lib.ctx, x.t())
    host = np.zeros(4, np.float32)
    assert not lib.lib.tysor_cuda_buffer_wrap(lib.ctx.handle, host.ctypes.data, 4)
    assert "not on the context's device" in lib.native.last_error()
    assert not lib.lib.tysor_cuda_buffer_wrap(lib.ctx.handle, x.data_ptr() + 2, 4)
    assert not lib.lib.tysor_cuda_buffer_wrap(lib.ctx.handle, None, 4)
    empty = lib.Buffer.wrap(lib.ctx, torch.empty((0, 4), device="cuda"))
    assert empty.count == 0
