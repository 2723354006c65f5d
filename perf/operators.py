"""Workloads of the language-model operators: layer normalisation, rotary
positions over several axes, sliding-window attention with sinks, and
distillation from a teacher's top logits.

`listed()` and `draw()` give cases, `prepare()` a case's data on the GPU,
`run()` one pass in elementary torch operations, or with `own` through the C
ABI of libtysor_cuda, and `exact()` the same results in 64 bits.
"""
import math

import numpy as np
import torch

own = False

_context = None


def _ctx():
    """The process's context of the library, made at its first use."""
    global _context
    if _context is None:
        from tysor_b200.runtime import CudaContext
        _context = CudaContext(torch.cuda.current_device())
    return _context


# ---- cases -------------------------------------------------------------------


def _attention(name, batch, heads, kv_heads, q_len, k_len, head_dim, window, sinks, ragged, seq_major, train):
    c = dict(op="window_attention", batch=batch, heads=heads, kv_heads=kv_heads, q_len=q_len, k_len=k_len,
             head_dim=head_dim, window=window, sinks=sinks, ragged=ragged, seq_major=seq_major, train=train)
    return dict(c, name=name) if name else c


def _norm(name, rows, width, train):
    c = dict(op="layer_norm", rows=rows, width=width, train=train)
    return dict(c, name=name) if name else c


def _rope(name, batch, heads, seq, sections, seq_major, train):
    c = dict(op="rope_axes", batch=batch, heads=heads, seq=seq, sections=sections, seq_major=seq_major, train=train)
    return dict(c, name=name) if name else c


def _distill(name, rows, width, top, temperature, train):
    c = dict(op="distill_loss", rows=rows, width=width, top=top, temperature=temperature, train=train)
    return dict(c, name=name) if name else c


def listed():
    return [
        # One new token of four sequences over caches of up to 32768 keys, all of them visible.
        _attention("attention_one_token_32k", 4, 16, 4, 1, 32768, 128, 0, 0, True, True, False),
        # One new token of 32 sequences that keep a window of 1024 keys and four first tokens.
        _attention("attention_one_token_window", 32, 16, 4, 1, 4096, 128, 1024, 4, True, True, False),
        # The decoder block's attention (8 x 2048, 16 heads over 4, 128 wide) without gradients.
        _attention("attention_block_forward", 8, 16, 4, 2048, 2048, 128, 512, 4, False, False, False),
        # A training step on one long sequence.
        _attention("attention_train_8k", 1, 16, 4, 8192, 8192, 128, 1024, 4, False, True, True),
        # A padded batch of short odd sequences and a head width that fills no tile.
        _attention("attention_train_ragged", 3, 6, 2, 777, 777, 80, 200, 3, True, False, True),
        # The norm of a few new tokens.
        _norm("norm_16x2048_forward", 16, 2048, False),
        # The norm of the decoder block's training step.
        _norm("norm_16384x2048_train", 16384, 2048, True),
        # An odd width, whose rows start at no 16-byte boundary.
        _norm("norm_1023x1001_train", 1023, 1001, True),
        # The positions of one new token.
        _rope("rope_one_token", 1, 16, 1, "16,24,24", False, False),
        # The block's queries with (time, height, width) positions, forward and backward.
        _rope("rope_block_train", 8, 16, 2048, "16,24,24", False, True),
        # A training batch's logits against a teacher's 64 best of 32000.
        _distill("distill_8192x32000_train", 8192, 32000, 64, 2.0, True),
        # The loss of a few rows over a large odd vocabulary.
        _distill("distill_7x128003_forward", 7, 128003, 20, 1.0, False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("window_attention", "window_attention", "layer_norm", "rope_axes", "distill_loss"))
    train = rng.random() < 0.6
    if op == "window_attention":
        kv_heads = rng.choice((1, 2, 3, 4, 8))
        heads = kv_heads * rng.choice((1, 2, 4, 5))
        head_dim = rng.choice((16, 32, 33, 40, 64, 72, 80, 96, 112, 128))
        window = rng.choice((0, _log(rng, 16, 4096)))
        sinks = rng.choice((0, 1, 4, 17))
        if rng.random() < 0.35:  # a few new tokens over a cache
            batch, k_len = _log(rng, 1, 32), _log(rng, 16, 65536)
            while batch * kv_heads * k_len * head_dim > 1 << 27:
                k_len = (k_len + 1) // 2
            q_len, train = rng.choice((1, 1, 2, 5)), False
        else:
            batch, k_len = _log(rng, 1, 8), _log(rng, 1, 8192)
            while batch * heads * k_len * k_len > 240_000_000:
                k_len = (k_len + 1) // 2
            q_len = k_len
        return _attention("", batch, heads, kv_heads, q_len, k_len, head_dim, window, sinks, rng.random() < 0.5,
                          rng.random() < 0.5, train)
    if op == "layer_norm":
        rows, width = _log(rng, 1, 65536), _log(rng, 8, 16384)
        while rows * width > 1 << 27:
            rows = (rows + 1) // 2
        return _norm("", rows, width, train)
    if op == "rope_axes":
        sections = ",".join(str(rng.randint(1, 32)) for _ in range(rng.randint(1, 4)))
        batch, heads, seq = _log(rng, 1, 8), _log(rng, 1, 32), _log(rng, 1, 16384)
        while batch * heads * seq * 2 * _half(sections) > 1 << 26:
            seq = (seq + 1) // 2
        return _rope("", batch, heads, seq, sections, rng.random() < 0.5, train)
    rows, width = _log(rng, 1, 8192), _log(rng, 64, 160000)
    while rows * width > 260_000_000:
        rows = (rows + 1) // 2
    return _distill("", rows, width, rng.randint(1, 64), rng.choice((1.0, 2.0, 3.5)), train)


def _half(sections):
    return sum(int(s) for s in sections.split(","))


# ---- data --------------------------------------------------------------------


def prepare(case, seed):
    state = _PREPARE[case["op"]](case, torch.Generator("cuda").manual_seed(int(seed)))
    state["case"] = case
    if own:
        _take(state)
    return state


def _normal(gen, *shape, std=1.0):
    return torch.randn(shape, generator=gen, device="cuda") * std


def _prepare_attention(c, gen):
    def of(n, h):
        return (c["batch"], n, h, c["head_dim"]) if c["seq_major"] else (c["batch"], h, n, c["head_dim"])

    s = {"q": _normal(gen, *of(c["q_len"], c["heads"])), "k": _normal(gen, *of(c["k_len"], c["kv_heads"])),
         "v": _normal(gen, *of(c["k_len"], c["kv_heads"])), "starts": None, "lengths": None}
    if c["ragged"]:
        # Each sequence's keys: the first fills the cache, the last of a padded training batch is empty.
        low = 1 if c["q_len"] < c["k_len"] else 0
        n = torch.randint(low, c["k_len"] + 1, (c["batch"],), generator=gen, device="cuda")
        n[0] = c["k_len"]
        if c["batch"] > 1 and not low:
            n[-1] = 0
        s["lengths"] = n.float()
        s["starts"] = (n - c["q_len"]).float() if low else torch.zeros_like(s["lengths"])
    if c["train"]:
        s["dout"] = _normal(gen, *of(c["q_len"], c["heads"]), std=1e-3)
    return s


def _prepare_norm(c, gen):
    s = {"x": _normal(gen, c["rows"], c["width"], std=1.5) + 0.5, "gain": 1 + _normal(gen, c["width"], std=0.02),
         "bias": _normal(gen, c["width"], std=0.02)}
    if c["train"]:
        s["dy"] = _normal(gen, c["rows"], c["width"], std=1e-3)
    return s


def _prepare_rope(c, gen):
    axes = c["sections"].count(",") + 1
    shape = (c["batch"], c["seq"], c["heads"]) if c["seq_major"] else (c["batch"], c["heads"], c["seq"])
    # Text and video tokens mixed: a common offset and small coordinates on each axis.
    place = torch.randint(0, 60, (c["batch"], axes, c["seq"]), generator=gen, device="cuda")
    place += torch.arange(c["seq"], device="cuda") + torch.randint(0, 100000, (1,), generator=gen, device="cuda")
    s = {"x": _normal(gen, *shape, 2 * _half(c["sections"])), "positions": place.float()}
    if c["train"]:
        s["dy"] = _normal(gen, *s["x"].shape)
    return s


def _prepare_distill(c, gen):
    logits = _normal(gen, c["rows"], c["width"], std=2.0)
    teacher, ids = (logits + _normal(gen, c["rows"], c["width"])).topk(c["top"], dim=1)
    # Some rows come with fewer entries, the last of several with none (a padded position).
    keep = torch.randint(1, c["top"] + 1, (c["rows"], 1), generator=gen, device="cuda")
    if c["rows"] > 1:
        keep[-1] = 0
    ids = ids.masked_fill(torch.arange(c["top"], device="cuda") >= keep, -1)
    s = {"logits": logits, "ids": ids.float(), "teacher": teacher.contiguous()}
    if c["train"]:
        s["dloss"] = torch.rand(c["rows"], generator=gen, device="cuda") / c["rows"]
    return s


_PREPARE = {"window_attention": _prepare_attention, "layer_norm": _prepare_norm, "rope_axes": _prepare_rope,
            "distill_loss": _prepare_distill}


# ---- the plain form ----------------------------------------------------------


def run(state):
    return (_CALL if own else _PLAIN)[state["case"]["op"]](state)


def _grouped(t, c, heads, seq_major):
    """[batch, kv_heads, rows, head_dim] of a tensor whose heads share keys in groups."""
    t = t.transpose(1, 2) if seq_major else t
    return t.reshape(c["batch"], c["kv_heads"], -1, c["head_dim"])


def _ungrouped(t, c, heads, seq_major):
    t = t.reshape(c["batch"], heads, -1, c["head_dim"])
    return t.transpose(1, 2).contiguous() if seq_major else t


def _plain_attention(s):
    c = s["case"]
    scale, group, major = 1.0 / math.sqrt(c["head_dim"]), c["heads"] // c["kv_heads"], c["seq_major"]
    q, k, v = (_grouped(s[n], c, c["heads"], major) for n in ("q", "k", "v"))
    j = torch.arange(c["k_len"], device="cuda")
    ends = s["lengths"] if c["ragged"] else torch.full((c["batch"],), float(c["k_len"]), device="cuda")
    first = s["starts"] if c["ragged"] else ends - c["q_len"]
    at = (first[:, None] + torch.arange(c["q_len"], device="cuda"))[:, :, None]
    seen = (j <= at) & (at < ends[:, None, None])
    if c["window"]:
        seen &= (at - j < c["window"]) | (j < c["sinks"])
    hidden = ~seen.repeat(1, group, 1)[:, None]
    p = torch.matmul(q, k.transpose(2, 3)).mul_(scale).masked_fill_(hidden, -math.inf)
    top = p.amax(3, keepdim=True)
    p.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(3, keepdim=True)
    p.div_(total.masked_fill(total == 0, 1.0))
    out = torch.matmul(p, v)
    stats = torch.cat((top, total), 3).reshape(c["batch"], c["heads"], c["q_len"], 2)
    result = [_ungrouped(out, c, c["heads"], major), stats]
    if c["train"]:
        g = _grouped(s["dout"], c, c["heads"], major)
        dv = torch.matmul(p.transpose(2, 3), g)
        ds = torch.matmul(g, v.transpose(2, 3)).sub_((g * out).sum(3, keepdim=True)).mul_(p).mul_(scale)
        dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(2, 3), q)
        result += [_ungrouped(dq, c, c["heads"], major), _ungrouped(dk, c, c["kv_heads"], major),
                   _ungrouped(dv, c, c["kv_heads"], major)]
    return result


_EPS = 1e-5


def _plain_norm(s):
    x = s["x"]
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + _EPS)
    n = d * rstd
    result = [n * s["gain"] + s["bias"], torch.cat((mean, rstd), 1)]
    if s["case"]["train"]:
        dy = s["dy"]
        g = dy * s["gain"]
        dx = (g - g.mean(1, keepdim=True) - n * (g * n).mean(1, keepdim=True)) * rstd
        result += [dx, (dy * n).sum(0), dy.sum(0)]
    return result


_THETA = 10000.0


def _plain_rope(s):
    c = s["case"]
    half = _half(c["sections"])
    axis = torch.from_numpy(_axis_of(c["sections"])).cuda()
    # Angles of far positions need 64 bits.
    rate = torch.exp(torch.arange(half, device="cuda", dtype=torch.float64) * (-math.log(_THETA) / half))
    angle = s["positions"].double()[:, axis].transpose(1, 2) * rate
    angle = angle[:, :, None] if c["seq_major"] else angle[:, None]
    cos, sin = angle.cos().float(), angle.sin().float()

    def turn(x, sin):
        a, b = x[..., :half], x[..., half:]
        return torch.cat((a * cos - b * sin, a * sin + b * cos), 3)

    return [turn(s["x"], sin)] + ([turn(s["dy"], -sin)] if c["train"] else [])


def _axis_of(sections):
    """The axis that turns each pair."""
    n = [int(v) for v in sections.split(",")]
    return np.repeat(np.arange(len(n)), n)


def _plain_distill(s):
    c = s["case"]
    t = c["temperature"]
    z = s["logits"]
    top = z.amax(1, keepdim=True)
    e = ((z - top) / t).exp()
    total = e.sum(1, keepdim=True)
    ids = s["ids"].long()
    here = ids >= 0
    w = s["teacher"].masked_fill(~here, -math.inf)
    best = w.amax(1, keepdim=True)
    w = ((w - best.masked_fill(best == -math.inf, 0.0)) / t).exp()
    mass = w.sum(1, keepdim=True)
    p = w / mass.masked_fill(mass == 0, 1.0)
    student = (z.gather(1, ids.clamp_min(0)) - top) / t - total.log()
    own_log = (s["teacher"] - best.masked_fill(best == -math.inf, 0.0)) / t - mass.masked_fill(mass == 0, 1.0).log()
    loss = t * t * torch.where(p > 0, p * (own_log - student), 0.0).sum(1)
    result = [loss, torch.cat((top, total), 1)]
    if c["train"]:
        scale = torch.where(mass[:, 0] > 0, t * s["dloss"], 0.0)[:, None]
        grad = e.mul_(scale / total)
        result.append(grad.scatter_add_(1, ids.clamp_min(0), p * -scale))
    return result


_PLAIN = {"window_attention": _plain_attention, "layer_norm": _plain_norm, "rope_axes": _plain_rope,
          "distill_loss": _plain_distill}


# ---- the library's calls -----------------------------------------------------


def _take(state):
    """The buffers that a program of the library keeps: its inputs, and its outputs' memory."""
    from tysor_b200.runtime import DeviceBuffer

    c, ctx = state["case"], _ctx()
    out = {}
    if c["op"] == "window_attention":
        out = {"out": torch.empty_like(state["q"]),
               "stats": torch.empty((c["batch"], c["heads"], c["q_len"], 2), device="cuda")}
        if c["train"]:
            out.update({"dq": torch.empty_like(state["q"]), "dk": torch.empty_like(state["k"]),
                        "dv": torch.empty_like(state["v"])})
    elif c["op"] == "layer_norm":
        out = {"y": torch.empty_like(state["x"]), "stats": torch.empty((c["rows"], 2), device="cuda")}
        if c["train"]:
            out.update({"dx": torch.empty_like(state["x"]), "dgain": torch.empty_like(state["gain"]),
                        "dbias": torch.empty_like(state["bias"])})
    elif c["op"] == "rope_axes":
        out = {"y": torch.empty_like(state["x"])}
        if c["train"]:
            out["dx"] = torch.empty_like(state["x"])
        state["sections"] = np.array([int(v) for v in c["sections"].split(",")], np.int64)
    else:
        out = {"loss": torch.empty(c["rows"], device="cuda"), "stats": torch.empty((c["rows"], 2), device="cuda")}
        if c["train"]:
            out["grad"] = torch.empty_like(state["logits"])
    state["out"] = out
    # The library works on its own stream: the inputs are ready there from here on.
    torch.cuda.current_stream().synchronize()
    tensors = {n: t for n, t in list(state.items()) + list(out.items()) if isinstance(t, torch.Tensor)}
    state["buffers"] = {n: DeviceBuffer.wrap(ctx, t) for n, t in tensors.items()}
    state["handle"] = {n: b.handle for n, b in state["buffers"].items()}


def _call_attention(s):
    from tysor_b200 import native

    c, h, o = s["case"], s["handle"], s["out"]
    lib, ctx = native.lib(), _ctx().handle
    shape = (c["batch"], c["heads"], c["kv_heads"], c["q_len"], c["k_len"], c["head_dim"], c["window"], c["sinks"],
             1.0 / math.sqrt(c["head_dim"]), c["seq_major"])
    starts, lengths = h.get("starts"), h.get("lengths")
    native.check(lib.tysor_cuda_dispatch_window_attention(ctx, h["q"], h["k"], h["v"], starts, lengths, h["out"],
                                                          h["stats"], *shape))
    if not c["train"]:
        return [o["out"], o["stats"]]
    native.check(lib.tysor_cuda_dispatch_window_attention_backward(
        ctx, h["q"], h["k"], h["v"], starts, lengths, h["out"], h["stats"], h["dout"], h["dq"], h["dk"], h["dv"],
        *shape, False))
    return [o["out"], o["stats"], o["dq"], o["dk"], o["dv"]]


def _call_norm(s):
    from tysor_b200 import native

    c, h, o = s["case"], s["handle"], s["out"]
    lib, ctx = native.lib(), _ctx().handle
    native.check(lib.tysor_cuda_dispatch_layer_norm(ctx, h["x"], h["gain"], h["bias"], h["y"], h["stats"], c["rows"],
                                                    c["width"], _EPS))
    if not c["train"]:
        return [o["y"], o["stats"]]
    native.check(lib.tysor_cuda_dispatch_layer_norm_backward(ctx, h["x"], h["gain"], h["stats"], h["dy"], h["dx"],
                                                             h["dgain"], h["dbias"], c["rows"], c["width"], False))
    return [o["y"], o["stats"], o["dx"], o["dgain"], o["dbias"]]


def _call_rope(s):
    from tysor_b200 import native

    c, h, o = s["case"], s["handle"], s["out"]
    lib, ctx = native.lib(), _ctx().handle
    sections = s["sections"].ctypes.data_as(native.I64P)
    shape = (c["batch"], c["heads"], c["seq"], sections, len(s["sections"]), _THETA, c["seq_major"])
    native.check(lib.tysor_cuda_dispatch_rope_axes(ctx, h["x"], h["positions"], h["y"], *shape))
    if not c["train"]:
        return [o["y"]]
    native.check(lib.tysor_cuda_dispatch_rope_axes_backward(ctx, h["dy"], h["positions"], h["dx"], *shape, False))
    return [o["y"], o["dx"]]


def _call_distill(s):
    from tysor_b200 import native

    c, h, o = s["case"], s["handle"], s["out"]
    lib, ctx = native.lib(), _ctx().handle
    shape = (c["rows"], c["width"], c["top"], c["temperature"])
    native.check(lib.tysor_cuda_dispatch_distill_loss(ctx, h["logits"], h["ids"], h["teacher"], h["loss"], h["stats"],
                                                      *shape))
    if not c["train"]:
        return [o["loss"], o["stats"]]
    native.check(lib.tysor_cuda_dispatch_distill_loss_backward(ctx, h["logits"], h["ids"], h["teacher"], h["stats"],
                                                               h["dloss"], h["grad"], *shape, False))
    return [o["loss"], o["stats"], o["grad"]]


_CALL = {"window_attention": _call_attention, "layer_norm": _call_norm, "rope_axes": _call_rope,
         "distill_loss": _call_distill}


# ---- the work ----------------------------------------------------------------


def work(case):
    c = case
    if c["op"] == "window_attention":
        # Full lengths: the visible pairs of one head, and the keys that some query sees.
        first = c["k_len"] - c["q_len"]
        pairs, low = 0, c["k_len"]
        for r in range(c["q_len"]):
            at = first + r
            begin = max(0, at - c["window"] + 1) if c["window"] else 0
            pairs += at + 1 - begin + min(c["sinks"], begin)
            low = min(low, begin)
        keys = c["k_len"] - low + min(c["sinks"], low)
        q = c["batch"] * c["heads"] * c["q_len"] * c["head_dim"]
        kv = c["batch"] * c["kv_heads"] * keys * c["head_dim"]
        rows = c["batch"] * c["heads"] * c["q_len"]
        part = _mean_part(c)
        values, flops = 2 * q + 2 * kv * part + 2 * rows, 4.0 * c["head_dim"]
        if c["train"]:
            # The output's gradient, and the gradients of queries, keys and values.
            values, flops = values + 2 * q + 2 * kv * part, 14.0 * c["head_dim"]
        return {"bytes": 4.0 * values, "flops": flops * pairs * c["batch"] * c["heads"] * part}
    if c["op"] == "layer_norm":
        n = c["rows"] * c["width"]
        if c["train"]:
            return {"bytes": 4.0 * (4 * n + 4 * c["width"] + 2 * c["rows"]), "flops": 20.0 * n}
        return {"bytes": 4.0 * (2 * n + 2 * c["width"] + 2 * c["rows"]), "flops": 8.0 * n}
    if c["op"] == "rope_axes":
        n = c["batch"] * c["heads"] * c["seq"] * 2 * _half(c["sections"])
        p = c["batch"] * c["seq"] * (c["sections"].count(",") + 1)
        passes = 2 if c["train"] else 1
        return {"bytes": 4.0 * (2 * passes * n + p), "flops": 3.0 * passes * n}
    n = c["rows"] * c["width"]
    if c["train"]:
        return {"bytes": 4.0 * (2 * n + 2 * c["rows"] * c["top"] + 4 * c["rows"]), "flops": 8.0 * n}
    return {"bytes": 4.0 * (n + 2 * c["rows"] * c["top"] + 3 * c["rows"]), "flops": 4.0 * n}


def _mean_part(c):
    """The share of a full batch that a ragged one has, on average (its first sequence is full)."""
    return (1 + 0.5 * (c["batch"] - 1)) / c["batch"] if c["ragged"] and not c["window"] else 1.0


# ---- in 64 bits --------------------------------------------------------------


def exact(case, seed):
    global own
    held, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = held
    return _EXACT[case["op"]](s, case)


def _exact_attention(s, c):
    names = ("q", "k", "v")
    q, k, v = (s[n].double().requires_grad_(c["train"]) for n in names)
    qh, kh, vh = ((t.permute(0, 2, 1, 3) if c["seq_major"] else t) for t in (q, k, v))
    qh = qh.unflatten(1, (c["kv_heads"], -1))
    score = torch.einsum("bgrqd,bgkd->bgrqk", qh, kh) / c["head_dim"] ** 0.5
    if c["ragged"]:
        begin, end = s["starts"].double(), s["lengths"].double()
    else:
        begin = torch.full((c["batch"],), c["k_len"] - c["q_len"], device="cuda", dtype=torch.float64)
        end = torch.full_like(begin, c["k_len"])
    place = begin.view(-1, 1, 1) + torch.arange(c["q_len"], device="cuda").view(1, -1, 1)
    key = torch.arange(c["k_len"], device="cuda").view(1, 1, -1)
    hidden = (key > place) | (place >= end.view(-1, 1, 1))
    if c["window"]:
        hidden |= (key <= place - c["window"]) & (key >= c["sinks"])
    hidden = hidden[:, None, None]
    nothing = hidden.all(-1, keepdim=True)
    masked = torch.where(hidden, -math.inf, score)
    weight = torch.softmax(torch.where(nothing, 0.0, masked), -1) * ~nothing
    out = torch.einsum("bgrqk,bgkd->bgrqd", weight, vh).flatten(1, 2)
    with torch.no_grad():
        best = masked.amax(-1)
        total = torch.where(nothing[..., 0], 0.0, (torch.logsumexp(masked, -1) - best).exp())
        stats = torch.stack((best, total), -1).flatten(1, 2)
    out = out.permute(0, 2, 1, 3) if c["seq_major"] else out
    result = [out.detach().contiguous(), stats]
    if c["train"]:
        result += [g.contiguous() for g in torch.autograd.grad(out, (q, k, v), s["dout"].double())]
    return result


def _exact_norm(s, c):
    x, gain, bias = (s[n].double().requires_grad_(c["train"]) for n in ("x", "gain", "bias"))
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    y = (x - mean) / (var + _EPS).sqrt() * gain + bias
    result = [y.detach(), torch.cat((mean, 1 / (var + _EPS).sqrt()), 1).detach()]
    if c["train"]:
        result += list(torch.autograd.grad(y, (x, gain, bias), s["dy"].double()))
    return result


def _exact_rope(s, c):
    half = _half(c["sections"])
    rate = _THETA ** (-np.arange(half) / half)
    place = s["positions"].double().permute(0, 2, 1)[:, :, torch.from_numpy(_axis_of(c["sections"])).cuda()]
    turn = torch.polar(torch.ones_like(place), place * torch.from_numpy(rate).cuda())
    turn = turn.unsqueeze(2 if c["seq_major"] else 1)

    def go(t, by):
        z = torch.complex(t[..., :half].double(), t[..., half:].double()) * by
        return torch.cat((z.real, z.imag), -1)

    return [go(s["x"], turn)] + ([go(s["dy"], turn.conj())] if c["train"] else [])


def _exact_distill(s, c):
    t = c["temperature"]
    z = s["logits"].double().requires_grad_(c["train"])
    log_q = torch.log_softmax(z / t, 1)
    ids = s["ids"].long()
    absent = ids < 0
    empty = absent.all(1, keepdim=True)
    w = torch.where(absent & ~empty, -math.inf, s["teacher"].double()) / t
    log_p = torch.log_softmax(w, 1)
    p = torch.where(absent, 0.0, log_p.exp())
    term = torch.where(absent, 0.0, log_p - torch.gather(log_q, 1, torch.where(absent, 0, ids)))
    loss = (p * term).sum(1) * t ** 2
    with torch.no_grad():
        best = z.amax(1)
        stats = torch.stack((best, (torch.logsumexp(z / t, 1) - best / t).exp()), 1)
    result = [loss.detach(), stats]
    if c["train"]:
        result += list(torch.autograd.grad(loss, (z,), s["dloss"].double()))
    return result


_EXACT = {"window_attention": _exact_attention, "layer_norm": _exact_norm, "rope_axes": _exact_rope,
          "distill_loss": _exact_distill}
