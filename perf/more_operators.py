"""Workloads of further language-model operators: rotary positions in either
layout, on part of a head, scaled for long contexts; linear attention with a
decay for each head; and the log probabilities of given tokens, with entropy
and best alternatives.

`listed()` and `draw()` give cases, `prepare()` a case's data on the GPU,
`run()` one pass in elementary torch operations, or with `own` through the C
ABI of libtysor_cuda, and `exact()` the same results in 64 bits.
"""
import math

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


def _rotary(name, batch, heads, seq, head_dim, rotary_dim, interleaved, scaling, seq_major, train):
    c = dict(op="rotary", batch=batch, heads=heads, seq=seq, head_dim=head_dim, rotary_dim=rotary_dim,
             interleaved=interleaved, scaling=scaling, seq_major=seq_major, train=train)
    return dict(c, name=name) if name else c


def _decay(name, batch, heads, kv_heads, seq, key_dim, value_dim, ragged, state, seq_major, train):
    c = dict(op="decay_attention", batch=batch, heads=heads, kv_heads=kv_heads, seq=seq, key_dim=key_dim,
             value_dim=value_dim, ragged=ragged, state=state, seq_major=seq_major, train=train)
    return dict(c, name=name) if name else c


def _logprobs(name, rows, width, given, top, temperature, masked, train):
    c = dict(op="token_logprobs", rows=rows, width=width, given=given, top=top, temperature=temperature,
             masked=masked, train=train)
    return dict(c, name=name) if name else c


def listed():
    return [
        # The positions of one new token of 32 sequences, half of each head turned.
        _rotary("rotary_one_token", 32, 16, 1, 128, 64, True, "log_turns", True, False),
        # The decoder block's queries (8 x 2048, 16 heads, 128 wide), forward and backward.
        _rotary("rotary_block_train", 8, 16, 2048, 128, 64, True, "turns", True, True),
        # A long prompt of odd head widths.
        _rotary("rotary_prompt_odd", 1, 5, 16385, 90, 90, False, "linear", False, False),
        # One new token of 32 sequences: the states read, turned over and written.
        _decay("decay_one_token", 32, 16, 16, 1, 128, 128, False, True, True, False),
        # The decoder block's attention (8 x 2048, 16 heads over 4, 128 wide) as a prompt, its states kept.
        _decay("decay_block_prompt", 8, 16, 4, 2048, 128, 128, False, True, True, False),
        # A prompt of 65536 tokens.
        _decay("decay_prompt_64k", 1, 4, 4, 65536, 128, 128, False, True, False, False),
        # A training step on one long sequence.
        _decay("decay_train_8k", 1, 16, 16, 8192, 128, 128, False, False, True, True),
        # A padded batch of short odd sequences, heads that share keys, widths that fill no tile.
        _decay("decay_train_ragged", 3, 6, 2, 777, 80, 48, True, True, False, True),
        # The reward's step of a training batch: the sampled tokens' log probabilities, entropy and gradients.
        _logprobs("logprobs_8192x32000_train", 8192, 32000, 1, 0, 1.0, False, True),
        # A prompt scored, each token with the 20 best alternatives.
        _logprobs("logprobs_2048x32000_top20", 2048, 32000, 1, 20, 1.0, False, False),
        # One new token of 32 sequences, some of the vocabulary ruled out.
        _logprobs("logprobs_32x32000_top8", 32, 32000, 1, 8, 0.7, True, False),
        # A few rows over a large odd vocabulary.
        _logprobs("logprobs_7x128003_top5", 7, 128003, 4, 5, 1.0, False, False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


_SCALINGS = ("plain", "linear", "turns", "log_turns")


def draw(rng):
    op = rng.choice(("rotary", "decay_attention", "decay_attention", "token_logprobs", "token_logprobs"))
    train = rng.random() < 0.5
    if op == "rotary":
        head_dim = rng.choice((32, 64, 80, 90, 96, 128, 128, 192, 256))
        rotary_dim = 2 * rng.randint(1, head_dim // 2) if rng.random() < 0.5 else head_dim
        batch, heads, seq = _log(rng, 1, 32), _log(rng, 1, 32), _log(rng, 1, 16384)
        while batch * heads * seq * head_dim > 1 << 25:
            seq = (seq + 1) // 2
        return _rotary("", batch, heads, seq, head_dim, rotary_dim, rng.random() < 0.5, rng.choice(_SCALINGS),
                       rng.random() < 0.5, train)
    if op == "decay_attention":
        kv_heads = rng.choice((1, 2, 3, 4, 8, 16))
        heads = kv_heads * rng.choice((1, 1, 2, 4))
        key_dim, value_dim = rng.choice(((128, 128), (128, 128), (64, 64), (64, 128), (80, 96), (33, 40), (16, 112)))
        state = rng.random() < 0.5
        if rng.random() < 0.3:  # new tokens of sequences under way
            batch, seq, train, state = _log(rng, 1, 64), rng.choice((1, 1, 1, 2, 5)), False, True
        else:
            batch, seq = _log(rng, 1, 8), _log(rng, 1, 65536)
            while batch * heads * seq > (1 << 17 if train else 1 << 18):
                seq = (seq + 1) // 2
        return _decay("", batch, heads, kv_heads, seq, key_dim, value_dim, rng.random() < 0.4, state,
                      rng.random() < 0.5, train)
    rows, width = _log(rng, 1, 8192), _log(rng, 256, 160000)
    while rows * width > 260_000_000:
        rows = (rows + 1) // 2
    top = 0 if train else rng.choice((0, 1, 5, 20, 64))
    return _logprobs("", rows, width, rng.choice((1, 1, 1, 2, 16)), top, rng.choice((1.0, 0.7, 1.5)),
                     rng.random() < 0.5, train)


# ---- data --------------------------------------------------------------------


def prepare(case, seed):
    state = _PREPARE[case["op"]](case, torch.Generator("cuda").manual_seed(int(seed)))
    state["case"] = case
    if own:
        _take(state)
    return state


def _normal(gen, *shape, std=1.0):
    return torch.randn(shape, generator=gen, device="cuda") * std


def _heads_of(c, heads, dim):
    return (c["batch"], c["seq"], heads, dim) if c["seq_major"] else (c["batch"], heads, c["seq"], dim)


def _prepare_rotary(c, gen):
    # Each sequence goes on from somewhere in a long context.
    first = torch.randint(0, 100000, (c["batch"], 1), generator=gen, device="cuda")
    s = {"x": _normal(gen, *_heads_of(c, c["heads"], c["head_dim"])),
         "positions": (first + torch.arange(c["seq"], device="cuda")).float()}
    if c["train"]:
        s["dy"] = _normal(gen, *s["x"].shape)
    return s


def _prepare_decay(c, gen):
    dims = (c["heads"], c["key_dim"], c["value_dim"])
    s = {"q": _normal(gen, *_heads_of(c, c["heads"], c["key_dim"])),
         "k": _normal(gen, *_heads_of(c, c["kv_heads"], c["key_dim"])),
         "v": _normal(gen, *_heads_of(c, c["kv_heads"], c["value_dim"])), "lengths": None, "state": None}
    # From heads that forget within two tokens to ones that remember thousands.
    place = (torch.arange(c["heads"], device="cuda") + torch.rand(c["heads"], generator=gen, device="cuda"))
    s["decay"] = torch.exp2(-0.5 - 11.0 * place / c["heads"])
    if c["ragged"]:
        # The first sequence is full, the last of several empty.
        n = torch.randint(1, c["seq"] + 1, (c["batch"],), generator=gen, device="cuda")
        n[0] = c["seq"]
        if c["batch"] > 2:
            n[-1] = 0
        s["lengths"] = n.float()
    if c["state"]:
        s["state"] = _normal(gen, c["batch"], *dims, std=4.0)
    if c["train"]:
        s["dout"] = _normal(gen, *_heads_of(c, c["heads"], c["value_dim"]), std=1e-3)
        if c["state"]:
            s["dnew_state"] = _normal(gen, c["batch"], *dims, std=1e-4)
    return s


def _prepare_logprobs(c, gen):
    logits = _normal(gen, c["rows"], c["width"], std=2.5)
    if c["masked"]:
        # What a grammar rules out, another share in each row.
        share = 0.9 * torch.rand(c["rows"], 1, generator=gen, device="cuda")
        logits.masked_fill_(torch.rand(c["rows"], c["width"], generator=gen, device="cuda") < share, -math.inf)
    # Sampled tokens: the greatest of the logits with Gumbel noise.
    noise = torch.rand(c["rows"], c["width"], generator=gen, device="cuda").clamp_(1e-7, 1.0 - 1e-7)
    noise.log_().neg_().log_().neg_().mul_(c["temperature"]).add_(logits)
    ids = noise.topk(c["given"], 1).indices if c["given"] > 1 else noise.argmax(1, keepdim=True)
    if c["rows"] > 1:
        ids[-1, -1] = -1  # a padded position
    s = {"logits": logits, "ids": ids.float()}
    if c["train"]:
        s["dout"] = _normal(gen, c["rows"], c["given"]) / c["rows"]
        s["dentropy"] = torch.rand(c["rows"], generator=gen, device="cuda") * (-0.01 / c["rows"])
    return s


_PREPARE = {"rotary": _prepare_rotary, "decay_attention": _prepare_decay, "token_logprobs": _prepare_logprobs}


# ---- the plain form ----------------------------------------------------------


def run(state):
    return (_CALL if own else _PLAIN)[state["case"]["op"]](state)


_THETA = 10000.0
# A context eight times as long as the 4096 tokens trained on; pairs that turn fewer than `low` times over those
# keep an eighth of their rate, those of more than `high` all of it.  The turned part grows by 0.1 ln 8 + 1.
_SCALE = {"plain": (0, 1.0, 0.0, 0.0, 0.0, 1.0), "linear": (1, 8.0, 0.0, 0.0, 0.0, 1.0),
          "turns": (2, 8.0, 4096.0, 1.0, 4.0, 1.0), "log_turns": (3, 8.0, 4096.0, 1.0, 32.0, 0.1 * math.log(8.0) + 1.0)}


def _plain_rotary(s):
    c = s["case"]
    kind, factor, context, low, high, amplitude = _SCALE[c["scaling"]]
    half = c["rotary_dim"] // 2
    # Angles of far positions need 64 bits.
    rate = torch.exp(torch.arange(half, device="cuda", dtype=torch.float64) * (-math.log(_THETA) / half))
    keep = torch.zeros_like(rate) if kind else torch.ones_like(rate)
    if kind >= 2:
        turns = context * rate / (2.0 * math.pi)
        if kind == 3:
            keep = (turns.log() - math.log(low)) / (math.log(high) - math.log(low))
        else:
            keep = (turns - low) / (high - low)
        keep = keep.clamp(0.0, 1.0)
    rate = rate * (keep + (1.0 - keep) / factor)
    angle = s["positions"].double()[:, :, None] * rate
    angle = angle[:, :, None] if c["seq_major"] else angle[:, None]
    cos, sin = (angle.cos() * amplitude).float(), (angle.sin() * amplitude).float()

    def turn(x, sin):
        part = x[..., :2 * half]
        y = x.clone()
        if c["interleaved"]:
            a, b = part[..., 0::2], part[..., 1::2]
            y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * cos - b * sin, a * sin + b * cos
        else:
            a, b = part[..., :half], part[..., half:]
            y[..., :half], y[..., half:2 * half] = a * cos - b * sin, a * sin + b * cos
        return y

    return [turn(s["x"], sin)] + ([turn(s["dy"], -sin)] if c["train"] else [])


_STEP = 256  # tokens that the plain form takes at once


def _plain_decay(s):
    c = s["case"]
    batch, heads, seq, group = c["batch"], c["heads"], c["seq"], c["heads"] // c["kv_heads"]
    scale = 1.0 / math.sqrt(c["key_dim"])

    def by_head(t, repeat):
        t = t.transpose(1, 2) if c["seq_major"] else t
        return t.repeat_interleave(repeat, 1) if repeat > 1 else t

    def back(t, shared):
        t = t.unflatten(1, (c["kv_heads"], group)).sum(2) if shared else t
        return t.transpose(1, 2).contiguous() if c["seq_major"] else t.contiguous()

    q, k, v = by_head(s["q"], 1), by_head(s["k"], group), by_head(s["v"], group)
    n = s["lengths"].long() if c["ragged"] else torch.full((batch,), seq, device="cuda")
    # Tokens that count up to and with each place; rows behind a sequence's end add nothing.
    place = torch.minimum(torch.arange(1, seq + 1, device="cuda"), n[:, None])
    live = (torch.arange(seq, device="cuda") < n[:, None])[:, None, :, None]
    if c["ragged"]:
        q, k, v = q * live, k * live, v * live
    rate = s["decay"].double()

    def weight(steps):  # decay over `steps` [batch, ...] tokens, by head
        view = rate.view(1, heads, *([1] * (steps.dim() - 1)))
        return torch.exp(-view * steps.unsqueeze(1)).float()

    def chunk(t):
        at = place[:, t:t + _STEP]
        before = place[:, t - 1:t] if t else torch.zeros_like(at[:, :1])
        within = weight((at[:, :, None] - at[:, None, :]).clamp_min(0))
        within = within * torch.ones(at.shape[1], at.shape[1], device="cuda").tril_()
        since, left = weight(at - before)[..., None], weight(at[:, -1:] - at)[..., None]
        return within, since, left, weight(at[:, -1:] - before)[..., None]

    state = s["state"] if c["state"] else torch.zeros(batch, heads, c["key_dim"], c["value_dim"], device="cuda")
    outs, states = [], []
    for t in range(0, seq, _STEP):
        e = slice(t, t + _STEP)
        within, since, left, whole = chunk(t)
        states.append(state)
        score = torch.matmul(q[:, :, e], k[:, :, e].transpose(2, 3)).mul_(within)
        outs.append((torch.matmul(score, v[:, :, e]) + torch.matmul(q[:, :, e], state) * since) * scale)
        state = state * whole + torch.matmul((k[:, :, e] * left).transpose(2, 3), v[:, :, e])
    result = [back(torch.cat(outs, 2), False)]
    if c["state"]:
        result.append(state)
    if not c["train"]:
        return result
    g = by_head(s["dout"], 1)
    g = g * live if c["ragged"] else g
    later = s["dnew_state"] if c["state"] else torch.zeros_like(state)
    dq, dk, dv = [], [], []
    for t in reversed(range(0, seq, _STEP)):
        e = slice(t, t + _STEP)
        within, since, left, whole = chunk(t)
        score = torch.matmul(q[:, :, e], k[:, :, e].transpose(2, 3)).mul_(within)
        dscore = torch.matmul(g[:, :, e], v[:, :, e].transpose(2, 3)).mul_(within)
        dq.append((torch.matmul(dscore, k[:, :, e])
                   + torch.matmul(g[:, :, e], states[t // _STEP].transpose(2, 3)) * since) * scale)
        dk.append(torch.matmul(dscore.transpose(2, 3), q[:, :, e]) * scale
                  + torch.matmul(v[:, :, e], later.transpose(2, 3)) * left)
        dv.append(torch.matmul(score.transpose(2, 3), g[:, :, e]) * scale
                  + torch.matmul(k[:, :, e], later) * left)
        later = later * whole + torch.matmul((q[:, :, e] * since).transpose(2, 3), g[:, :, e]) * scale
    dq, dk, dv = (torch.cat(d[::-1], 2) for d in (dq, dk, dv))
    if c["ragged"]:
        dk, dv = dk * live, dv * live
    result += [back(dq, False), back(dk, True), back(dv, True)]
    if c["state"]:
        result.append(later)
    return result


def _plain_logprobs(s):
    c = s["case"]
    t = c["temperature"]
    z = s["logits"]
    top = z.amax(1, keepdim=True)
    y = (z - top) / t
    e = y.exp()
    total = e.sum(1, keepdim=True)
    # A token of probability 0 adds nothing to the entropy.
    y.masked_fill_(e == 0, 0.0)
    entropy = total.log() - (e * y).sum(1, keepdim=True) / total
    ids = s["ids"].long()
    here = ids >= 0
    at = ids.clamp_min(0)
    given = torch.where(here, (z.gather(1, at) - top) / t - total.log(), 0.0)
    result = [given, entropy[:, 0], torch.cat((top, total), 1)]
    if c["top"]:
        # Equal logits in the order of their ids.
        best, which = z.sort(dim=1, descending=True, stable=True)
        best = best[:, :c["top"]]
        none = best == -math.inf
        result += [torch.where(none, -1, which[:, :c["top"]]).float(),
                   torch.where(none, -math.inf, (best - top) / t - total.log())]
    if c["train"]:
        d = torch.where(here, s["dout"], 0.0)
        p = e.div_(total)
        log_p = y.sub_(total.log())
        grad = p * (-d.sum(1, keepdim=True) - s["dentropy"][:, None] * (log_p + entropy))
        result.append(grad.scatter_add_(1, at, d).div_(t))
    return result


_PLAIN = {"rotary": _plain_rotary, "decay_attention": _plain_decay, "token_logprobs": _plain_logprobs}


# ---- the library's calls -----------------------------------------------------


def _take(state):
    """The buffers that a program of the library keeps: its inputs, and its outputs' memory."""
    from tysor_b200.runtime import DeviceBuffer

    c, ctx = state["case"], _ctx()
    if c["op"] == "rotary":
        out = {"y": torch.empty_like(state["x"])}
        if c["train"]:
            out["dx"] = torch.empty_like(state["x"])
    elif c["op"] == "decay_attention":
        out = {"out": torch.empty(_heads_of(c, c["heads"], c["value_dim"]), device="cuda")}
        if c["state"]:
            out["new_state"] = torch.empty_like(state["state"])
        if c["train"]:
            out.update({"d" + n: torch.empty_like(state[n]) for n in ("q", "k", "v")})
            if c["state"]:
                out["dstate"] = torch.empty_like(state["state"])
    else:
        def rows(*more):
            return torch.empty(c["rows"], *more, device="cuda")

        out = {"out": rows(c["given"]), "entropy": rows(), "stats": rows(2)}
        if c["top"]:
            out.update({"top_ids": rows(c["top"]), "top_logprobs": rows(c["top"])})
        if c["train"]:
            out["grad"] = torch.empty_like(state["logits"])
    state["out"] = out
    # The library works on its own stream: the inputs are ready there from here on.
    torch.cuda.current_stream().synchronize()
    tensors = {n: t for n, t in list(state.items()) + list(out.items()) if isinstance(t, torch.Tensor)}
    state["buffers"] = {n: DeviceBuffer.wrap(ctx, t) for n, t in tensors.items()}
    state["handle"] = {n: b.handle for n, b in state["buffers"].items()}


def _call_rotary(s):
    from tysor_b200 import native

    c, h, o = s["case"], s["handle"], s["out"]
    lib, ctx = native.lib(), _ctx().handle
    shape = (c["batch"], c["heads"], c["seq"], c["head_dim"], c["rotary_dim"], c["interleaved"], _THETA,
             *_SCALE[c["scaling"]], c["seq_major"])
    native.check(lib.tysor_cuda_dispatch_rotary(ctx, h["x"], h["positions"], h["y"], *shape))
    if not c["train"]:
        return [o["y"]]
    native.check(lib.tysor_cuda_dispatch_rotary_backward(ctx, h["dy"], h["positions"], h["dx"], *shape, False))
    return [o["y"], o["dx"]]


def _call_decay(s):
    from tysor_b200 import native

    c, h, o = s["case"], s["handle"], s["out"]
    lib, ctx = native.lib(), _ctx().handle
    shape = (c["batch"], c["heads"], c["kv_heads"], c["seq"], c["key_dim"], c["value_dim"],
             1.0 / math.sqrt(c["key_dim"]), c["seq_major"])
    given = (h["q"], h["k"], h["v"], h["decay"], h.get("state"), h.get("lengths"))
    native.check(lib.tysor_cuda_dispatch_decay_attention(ctx, *given, h["out"], h.get("new_state"), *shape))
    result = [o["out"]] + ([o["new_state"]] if c["state"] else [])
    if not c["train"]:
        return result
    native.check(lib.tysor_cuda_dispatch_decay_attention_backward(
        ctx, *given, h["dout"], h.get("dnew_state"), h["dq"], h["dk"], h["dv"], h.get("dstate"), *shape, False))
    return result + [o["dq"], o["dk"], o["dv"]] + ([o["dstate"]] if c["state"] else [])


def _call_logprobs(s):
    from tysor_b200 import native

    c, h, o = s["case"], s["handle"], s["out"]
    lib, ctx = native.lib(), _ctx().handle
    native.check(lib.tysor_cuda_dispatch_token_logprobs(
        ctx, h["logits"], h["ids"], h["out"], h["entropy"], h.get("top_ids"), h.get("top_logprobs"), h["stats"],
        c["rows"], c["width"], c["given"], c["top"], c["temperature"]))
    result = [o["out"], o["entropy"], o["stats"]] + ([o["top_ids"], o["top_logprobs"]] if c["top"] else [])
    if not c["train"]:
        return result
    native.check(lib.tysor_cuda_dispatch_token_logprobs_backward(
        ctx, h["logits"], h["ids"], h["stats"], h["entropy"], h["dout"], h["dentropy"], h["grad"], c["rows"],
        c["width"], c["given"], c["temperature"], False))
    return result + [o["grad"]]


_CALL = {"rotary": _call_rotary, "decay_attention": _call_decay, "token_logprobs": _call_logprobs}


# ---- the work ----------------------------------------------------------------


def work(case):
    c = case
    passes = 2 if c["train"] else 1
    if c["op"] == "rotary":
        n = c["batch"] * c["heads"] * c["seq"]
        return {"bytes": 4.0 * (2 * passes * n * c["head_dim"] + c["batch"] * c["seq"]),
                "flops": 3.0 * passes * n * c["rotary_dim"]}
    if c["op"] == "decay_attention":
        # The share of a padded batch's rows that hold tokens, on average.
        rest = max(c["batch"] - (2 if c["batch"] > 2 else 1), 0)
        tokens = c["seq"] * ((1 + 0.5 * rest) if c["ragged"] else c["batch"])
        rows = c["batch"] * c["seq"]
        wide = c["heads"] * c["key_dim"] + c["kv_heads"] * (c["key_dim"] + c["value_dim"])  # q, k, v of a token
        out = c["heads"] * c["value_dim"]
        states = c["batch"] * c["heads"] * c["key_dim"] * c["value_dim"] * (2 * passes if c["state"] else 0)
        product = 2.0 * tokens * c["heads"] * c["key_dim"] * c["value_dim"]
        if c["train"]:
            # Also the output's gradient, and those of q, k and v; the states of either direction, five products.
            return {"bytes": 4.0 * (tokens * (wide + out) + rows * (out + wide) + states), "flops": 7.0 * product}
        return {"bytes": 4.0 * (tokens * wide + rows * out + states), "flops": 2.0 * product}
    n, rows = c["rows"] * c["width"], c["rows"]
    small = rows * (2 * c["given"] + 2 * c["top"] + 3)
    if c["train"]:
        return {"bytes": 4.0 * (2 * n + small + rows * (c["given"] + 1)), "flops": 11.0 * n}
    return {"bytes": 4.0 * (n + small), "flops": 6.0 * n}


# ---- in 64 bits --------------------------------------------------------------


def exact(case, seed):
    global own
    held, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = held
    return _EXACT[case["op"]](s, case)


def _exact_rotary(s, c):
    kind, factor, context, low, high, amplitude = _SCALE[c["scaling"]]
    pairs = c["rotary_dim"] // 2
    rates = []
    for i in range(pairs):
        rate = _THETA ** (-i / pairs)
        share = 1.0
        if kind == 1:
            share = 0.0
        elif kind:
            turns = context * rate / (2.0 * math.pi)
            share = (turns - low) / (high - low) if kind == 2 else math.log(turns / low) / math.log(high / low)
            share = min(max(share, 0.0), 1.0)
        rates.append(rate * share + rate / factor * (1.0 - share))
    place = s["positions"].double().unsqueeze(-1) * torch.tensor(rates, device="cuda", dtype=torch.float64)
    by = torch.polar(torch.full_like(place, amplitude), place).unsqueeze(2 if c["seq_major"] else 1)

    def go(t, by):
        t = t.double()
        head, tail = t[..., :2 * pairs], t[..., 2 * pairs:]
        two = head.unflatten(-1, (pairs, 2) if c["interleaved"] else (2, pairs))
        two = two if c["interleaved"] else two.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(two.contiguous()) * by)
        z = z if c["interleaved"] else z.transpose(-1, -2)
        return torch.cat((z.flatten(-2), tail), -1)

    return [go(s["x"], by)] + ([go(s["dy"], by.conj())] if c["train"] else [])


_ROWS = 2048  # output rows of a head that the exact form takes at once, without gradients


def _exact_decay(s, c):
    batch, heads, share = c["batch"], c["heads"], c["heads"] // c["kv_heads"]
    kept = {n: t.double() for n, t in s.items() if isinstance(t, torch.Tensor)}

    def view(t, b, h):
        return t[b, :, h] if c["seq_major"] else t[b, h]

    out = torch.zeros(_heads_of(c, heads, c["value_dim"]), device="cuda", dtype=torch.float64)
    new_state = torch.zeros(batch, heads, c["key_dim"], c["value_dim"], device="cuda", dtype=torch.float64)
    grads = {n: torch.zeros_like(kept[n]) for n in ("q", "k", "v")} if c["train"] else {}
    dstate = torch.zeros_like(new_state)
    for b in range(batch):
        n = int(s["lengths"][b]) if c["ragged"] else c["seq"]
        for h in range(heads):
            q, k, v = (view(kept[x], b, h // share if x != "q" else h)[:n] for x in ("q", "k", "v"))
            start = kept["state"][b, h] if c["state"] else torch.zeros_like(new_state[b, h])
            rate = kept["decay"][h]
            at = torch.arange(n, device="cuda", dtype=torch.float64)
            if c["train"]:
                q, k, v, start = (t.detach().clone().requires_grad_() for t in (q, k, v, start))
            parts = []
            for i in range(0, n, max(n, 1) if c["train"] else _ROWS):
                j = n if c["train"] else min(i + _ROWS, n)
                gap = at[i:j, None] - at[None, :j]
                kernel = torch.where(gap >= 0, torch.exp(-rate * gap.clamp_min(0)), 0.0)
                part = ((q[i:j] @ k[:j].T) * kernel) @ v[:j]
                part = part + torch.exp(-rate * (at[i:j, None] + 1)) * (q[i:j] @ start)
                parts.append(part / c["key_dim"] ** 0.5)
            last = (k * torch.exp(-rate * (n - 1 - at))[:, None]).T @ v + torch.exp(-rate * n) * start
            new_state[b, h] = last.detach()
            if n:
                whole = torch.cat(parts)
                view(out, b, h)[:n] = whole.detach()
            if c["train"]:
                loss = (last * kept["dnew_state"][b, h]).sum() if c["state"] else (last * 0.0).sum()
                if n:
                    loss = loss + (whole * view(kept["dout"], b, h)[:n]).sum()
                found = torch.autograd.grad(loss, (q, k, v, start), allow_unused=n == 0)
                for x, g in zip(("q", "k", "v", None), found):
                    if x is None:
                        dstate[b, h] = g
                    elif n:
                        view(grads[x], b, h // share if x != "q" else h)[:n] += g
    result = [out] + ([new_state] if c["state"] else [])
    if c["train"]:
        result += [grads["q"], grads["k"], grads["v"]] + ([dstate] if c["state"] else [])
    return result


def _exact_logprobs(s, c):
    t = c["temperature"]
    ids = s["ids"].long()
    absent = ids < 0
    pieces = []
    step = max(1, (1 << 26) // c["width"])
    for r in range(0, c["rows"], step):
        e = slice(r, r + step)
        z = s["logits"][e].double().requires_grad_(c["train"])
        lp = torch.log_softmax(z / t, 1)
        possible = lp > -math.inf
        given = torch.where(absent[e], 0.0, lp.gather(1, torch.where(absent[e], 0, ids[e])))
        entropy = -(lp.exp() * torch.where(possible, lp, 0.0)).sum(1)
        with torch.no_grad():
            best = z.amax(1)
            piece = [given.detach(), entropy.detach(),
                     torch.stack((best, (torch.logsumexp(z / t, 1) - best / t).exp()), 1)]
            if c["top"]:
                # Stable: equal logits stay in the order of their ids.
                which = torch.argsort(-s["logits"][e], dim=1, stable=True)[:, :c["top"]]
                value = lp.gather(1, which)
                piece += [torch.where(value > -math.inf, which, -1).double(), value]
        if c["train"]:
            loss = (given * s["dout"][e]).sum() + (entropy * s["dentropy"][e]).sum()
            g = torch.autograd.grad(loss, z)[0]
            piece.append(torch.where(possible, g, 0.0).detach())
        pieces.append(piece)
    return [torch.cat(p) for p in zip(*pieces)]


_EXACT = {"rotary": _exact_rotary, "decay_attention": _exact_decay, "token_logprobs": _exact_logprobs}
