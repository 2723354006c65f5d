"""decay_attention where tokens' rows differ in size, value by value against its formulas in 64 bits
(linear_reference.py): what a token sees, not what else its 64 tokens or its head's other columns hold,
says how far a result may be off.

Tolerance, fixed from the arithmetic, relative to the same sums over absolute values (u = 2^-24): three
operands of two halves (4u each), 68 instructions that may each lose a step (2u) of what they have added,
a fade of e^-x whose exponent is rounded (xu, x below 88, where fp32 ends), two roundings a step of the state
(8 steps at most); or one by one two roundings a token and sum, of which 64 in a row have one sign once
in 2^64.  Together below 256u.  Where one by one the tokens are up to 1100 more than 64 follow one another
at random: 256u still holds eight times their root."""
import numpy as np
import pytest

import linear_reference as R
from test_gpu_linear_ops import decay_data, decay_run
from test_gpu_lm_ops import Lib, U

pytestmark = pytest.mark.gpu

BAR = 256 * U
RATES = np.array([0.0, 0.01, 0.3, 2.0], np.float32)


@pytest.fixture
def lib(cuda_ctx):
    return Lib(cuda_ctx)


def wanted(t, scale, seq_major):
    """The results, and the same sums over absolute values."""
    def of(t):
        return R.decay_attention(t["q"], t["k"], t["v"], t["decay"], t["state"], None, scale, seq_major, t["dout"], t["dnew"])

    return of(t), of({n: a if a is None else abs(a) for n, a in t.items()})


def within(got, want, size, name):
    off = abs(got.reshape(want.shape).astype(np.float64) - want)
    bad = ~(off <= BAR * size + 2.0 ** -120)
    assert not bad.any(), f"{name}: {(off / (size + 1e-300)).max() / U:.0f}u, {bad.sum()} values, first {np.argwhere(bad)[0]}"


# ---- the state -----------------------------------------------------------------------


@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 80), (33, 20)])
@pytest.mark.parametrize("power", [10, 20, 30, 40, 50])
@pytest.mark.parametrize("where", [5, 63, 90])
def test_a_large_key_beside_small_values_leaves_their_columns_as_they_are(lib, dk, dv, power, where):
    # The key's size reaches the state only by what it is multiplied with.  `batch` 40 leaves a head's
    # tokens to one block; 1 shares them out.
    for batch in (1, 40):
        rng = np.random.default_rng(power + where)
        t = decay_data(rng, batch, 4, 4, 200, dk, dv, False, True)
        t["decay"] = RATES
        t["k"][:, :, where] *= np.float32(2.0 ** power)
        t["v"][:, :, where, 1::3] = 0
        t["v"][:, :, where, 2::3] *= np.float32(2.0 ** -power)
        got = decay_run(lib, t, 0.125, False, need=())
        t["dout"], t["dnew"] = None, None
        want = R.decay_attention(t["q"], t["k"], t["v"], RATES, t["state"], None, 0.125, False)
        size = R.decay_attention(abs(t["q"]), abs(t["k"]), abs(t["v"]), RATES, abs(t["state"]), None, 0.125, False)
        within(got["new_state"], want["new_state"], size["new_state"], (batch, "new_state"))
        later = (where // 64 + 1) * 64
        within(got["out"].reshape(want["out"].shape)[:, :, later:], want["out"][:, :, later:], size["out"][:, :, later:],
               (batch, "out"))


def test_a_state_that_a_large_token_has_left_again(lib):
    # 18 steps in one block: the token fades and what is left has its own size again.
    rng = np.random.default_rng(2)
    t = decay_data(rng, 8, 20, 20, 1100, 16, 16, True, True)
    t["decay"] = np.resize(np.array([0.0, 0.02, 0.05, 0.2], np.float32), 20)
    t["k"][:, 70] *= np.float32(2.0 ** 40)
    t["v"][:, 70] *= np.float32(2.0 ** -20)
    got = decay_run(lib, t, 0.25, True, need=())
    want = R.decay_attention(t["q"], t["k"], t["v"], t["decay"], t["state"], None, 0.25, True)
    size = R.decay_attention(abs(t["q"]), abs(t["k"]), abs(t["v"]), t["decay"], abs(t["state"]), None, 0.25, True)
    within(got["new_state"], want["new_state"], size["new_state"], "new_state")
    within(got["out"].reshape(want["out"].shape)[:, 128:], want["out"][:, 128:], size["out"][:, 128:], "out")


# ---- what the tokens of 64 hold, beside one another -----------------------------------

# Whose row stands in the key's place of the products that give a result, and whose in the value's.
KEYS = {"out": "k", "dq": "v", "dv": "q", "dk": "dout"}


def sized_run(lib, t, names):
    want, size = wanted(t, 0.125, False)
    got = decay_run(lib, t, 0.125, False)
    for n in names:
        within(got[n], want[n], size[n], n)


def sized_data(seed, seq, dk, dv, batch=1):
    t = decay_data(np.random.default_rng(seed), batch, 4, 2, seq, dk, dv, False, True)
    t["decay"] = RATES
    t["dout"] *= 1000
    t["dnew"] *= 1000
    return t


@pytest.mark.parametrize("result", list(KEYS))
@pytest.mark.parametrize("seq,where", [(23, 11), (24, 11), (64, 0), (64, 63), (200, 40), (200, 100), (700, 300)])
@pytest.mark.parametrize("power", [10, 16, 24, 32, 40, 50, -20, -50])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 80)])
def test_a_large_or_small_key_leaves_other_tokens_as_they_are(lib, result, seq, where, power, dk, dv):
    t = sized_data(seq + power + 50, seq, dk, dv)
    t[KEYS[result]][:, :, where] *= np.float32(2.0 ** power)
    sized_run(lib, t, [result])


@pytest.mark.parametrize("seq", [100, 700])
@pytest.mark.parametrize("spread", [8, 20, 40, 70])
def test_keys_of_all_sizes(lib, seq, spread):
    for result, key in KEYS.items():
        t = sized_data(spread, seq, 80, 64)
        size = np.random.default_rng(seq).integers(-spread // 2, spread // 2 + 1, t[key].shape[:3] + (1,))
        t[key] *= (2.0 ** size).astype(np.float32)
        sized_run(lib, t, [result])


@pytest.mark.parametrize("result", list(KEYS))
def test_keys_that_have_faded(lib, result):
    # Behind rows of zeros a token sees only what has faded: 40 tokens at e^-1.5 are 2^-86.
    t = sized_data(4, 200, 64, 64)
    t["decay"] = np.array([0.01, 0.3, 1.0, 1.5], np.float32)
    t["state"] = t["dnew"] = None
    t[KEYS[result]][:, :, 10:50] = 0
    t[KEYS[result]][:, :, 70:120] = 0
    sized_run(lib, t, [result])


@pytest.mark.parametrize("seq", [64, 200])
@pytest.mark.parametrize("power", [12, 20, 40, 55])
def test_a_large_key_beside_small_values_within_its_64_tokens(lib, seq, power):
    for result, value in (("out", "v"), ("dq", "k"), ("dv", "dout"), ("dk", "q")):
        t = sized_data(power, seq, 64, 64)
        for where in (9, 30):
            t[KEYS[result]][:, :, where] *= np.float32(2.0 ** power)
            t[value][:, :, where, where % 3::3] = 0
            t[value][:, :, where, where % 3 + 1::3] *= np.float32(2.0 ** -power)
        sized_run(lib, t, [result])


VALUES = {"out": "v", "dq": "k", "dv": "dout", "dk": "q"}


@pytest.mark.parametrize("result", list(VALUES))
@pytest.mark.parametrize("seq,where", [(23, 11), (24, 11), (64, 0), (64, 63), (200, 40), (200, 100), (700, 300)])
@pytest.mark.parametrize("power", [10, 16, 24, 32, 40, 50, -20, -50])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 80)])
def test_a_large_or_small_value_leaves_other_tokens_as_they_are(lib, result, seq, where, power, dk, dv):
    t = sized_data(seq + power + 50, seq, dk, dv)
    t[VALUES[result]][:, :, where] *= np.float32(2.0 ** power)
    sized_run(lib, t, [result])


@pytest.mark.parametrize("seq", [100, 700])
@pytest.mark.parametrize("spread", [8, 20, 40, 70])
@pytest.mark.parametrize("dims", [(80, 64), (33, 70)])
def test_rows_of_all_sizes(lib, seq, spread, dims):
    for name in ("q", "k", "v", "dout"):
        t = sized_data(spread, seq, *dims)
        size = np.random.default_rng(seq).integers(-spread // 2, spread // 2 + 1, t[name].shape[:3] + (1,))
        t[name] *= (2.0 ** size).astype(np.float32)
        sized_run(lib, t, ["out", "new_state", "dq", "dk", "dv", "dstate"])


@pytest.mark.parametrize("seq", [24, 200])
def test_large_keys_with_small_values_and_small_ones_with_large(lib, seq):
    # The products are alike: nothing needs to go token by token, and nothing may be lost.
    for keys, values in (("k", "v"), ("q", "dout")):
        t = sized_data(seq, seq, 64, 80)
        size = (2.0 ** np.random.default_rng(seq).integers(-25, 26, t[keys].shape[:3] + (1,))).astype(np.float32)
        t[keys] *= size
        t[values] /= size
        sized_run(lib, t, ["out", "new_state", "dq", "dk", "dv", "dstate"])


@pytest.mark.parametrize("power", [-20, 20])
def test_columns_of_all_sizes(lib, power):
    # A column that is small in all tokens keeps its own digits.
    t = sized_data(1, 200, 64, 64)
    size = (2.0 ** np.linspace(0, power, 64)).astype(np.float32)
    t["v"] *= size
    sized_run(lib, t, ["out", "new_state"])
    t = sized_data(2, 200, 64, 64)
    t["k"] *= size
    sized_run(lib, t, ["dq"])


@pytest.mark.parametrize("size", [2.0 ** -62, 2.0 ** -55, 2.0 ** -40, 2.0 ** 50])
def test_products_near_the_ends_of_fp32(lib, size):
    # Down to where the products of key and value leave fp32's normal numbers (2^-126), and up.
    t = sized_data(3, 200, 64, 64)
    t["state"] = None
    t["k"] *= np.float32(size)
    t["v"] *= np.float32(size)
    t["q"] *= np.float32(min(1.0 / size, 2.0 ** 55))
    want = R.decay_attention(t["q"], t["k"], t["v"], RATES, None, None, 0.125, False)
    much = R.decay_attention(abs(t["q"]), abs(t["k"]), abs(t["v"]), RATES, None, None, 0.125, False)
    got = decay_run(lib, t, 0.125, False, need=())
    within(got["out"], want["out"], much["out"], "out")


@pytest.mark.parametrize("seq_major", [False, True])
@pytest.mark.parametrize("dims", [(64, 64), (128, 80), (33, 70)])
def test_rows_of_all_sizes_in_padded_batches(lib, dims, seq_major):
    rng = np.random.default_rng(7)
    t = decay_data(rng, 5, 4, 2, 300, *dims, seq_major, True)
    t["decay"] = RATES
    n = np.array([300, 0, 64, 65, 190])
    t["lengths"] = n.astype(np.float32)
    for name in ("q", "k", "v", "dout"):
        t[name] *= (2.0 ** rng.integers(-15, 16, t[name].shape[:3] + (1,))).astype(np.float32)

    def of(a):
        return R.decay_attention(a["q"], a["k"], a["v"], RATES, a["state"], n, 0.125, seq_major, a["dout"], a["dnew"])

    want, size = of(t), of({m: a if a is None else abs(a) for m, a in t.items()})
    for name in ("q", "k", "v", "dout"):
        a = t[name] if seq_major else np.moveaxis(t[name], 1, 2)
        for b in range(5):
            a[b, n[b]:] = (np.nan, np.inf, -np.inf, 1e30, 1e-30)[b]
    got = decay_run(lib, t, 0.125, seq_major)
    for m in got:
        within(got[m], want[m], size[m], m)


@pytest.mark.parametrize("seq", [23, 200, 700])
@pytest.mark.parametrize("size", [2.0 ** 50, 2.0 ** 55, 2.0 ** 57])
def test_large_products_that_fp32_holds(lib, size, seq):
    # Outputs up to 2^123 with queries of 1: what stands between must not leave fp32's range either.
    t = sized_data(5, seq, 64, 64)
    t["dnew"] = None
    t["state"] *= np.float32(size * size)
    t["k"] *= np.float32(size)
    t["v"] *= np.float32(size)
    t["dout"] *= np.float32(1e-3 / size)  # dq = dout S: 2^63
    sized_run(lib, t, ["out", "new_state", "dq"])
    t = sized_data(6, seq, 64, 64)
    t["state"] = None
    t["q"] *= np.float32(size)
    t["dout"] *= np.float32(1e-3 * size)
    t["dnew"] *= np.float32(1e-3 * size * size)
    sized_run(lib, t, ["dk", "dv", "dstate"])
