"""64-bit restatements of rotary, decay_attention and token_logprobs (numpy),
straight from their formulas."""
import numpy as np


def rotary_rates(half, theta, scaling, factor, original_len, low, high):
    base = np.float64(theta) ** (-np.arange(half) / half)
    keep = np.ones(half) if scaling == 0 else np.zeros(half)
    if scaling >= 2:
        of = (lambda t: t) if scaling == 2 else np.log
        turns = original_len * base / (2 * np.pi)
        keep = np.clip((of(turns) - of(np.float64(low))) / (of(np.float64(high)) - of(np.float64(low))), 0.0, 1.0)
    return base if scaling == 0 else base * (keep + (1 - keep) / factor)


def rotary(x, positions, rotary_dim, interleaved, theta, scaling, seq_major, back=False):
    """x [B, H, S, D] or [B, S, H, D]; positions [B, S] or None; scaling the six last arguments."""
    half = rotary_dim // 2
    b, s = x.shape[0], x.shape[1 if seq_major else 2]
    place = np.tile(np.arange(s), (b, 1)) if positions is None else positions
    angle = place.astype(np.float64)[..., None] * rotary_rates(half, theta, *scaling[:5])
    angle = angle[:, :, None] if seq_major else angle[:, None]
    by = scaling[5] * np.exp((-1j if back else 1j) * angle)
    y = x.astype(np.float64)
    lo, hi = (slice(0, rotary_dim, 2), slice(1, rotary_dim, 2)) if interleaved else (slice(0, half), slice(half, rotary_dim))
    z = (y[..., lo] + 1j * y[..., hi]) * by
    y[..., lo], y[..., hi] = z.real, z.imag
    return y


def decay_attention(q, k, v, decay, state, lengths, scale, seq_major, dout=None, dnew=None):
    """The formulas token against token; rows behind a sequence's end are not read."""
    if seq_major:
        q, k, v = (np.swapaxes(t, 1, 2) for t in (q, k, v))
        dout = None if dout is None else np.swapaxes(dout, 1, 2)
    batch, heads, seq, dk = q.shape
    group, dv = heads // k.shape[1], v.shape[3]
    out, new = np.zeros((batch, heads, seq, dv)), np.zeros((batch, heads, dk, dv))
    g = {"dq": np.zeros(q.shape), "dk": np.zeros(k.shape), "dv": np.zeros(v.shape), "dstate": np.zeros(new.shape)}
    for b in range(batch):
        n = seq if lengths is None else int(lengths[b])
        gap = np.arange(n)[:, None] - np.arange(n)[None]
        for h in range(heads):
            qq, kk, vv = (t[b, i, :n].astype(np.float64) for t, i in ((q, h), (k, h // group), (v, h // group)))
            s0 = np.zeros((dk, dv)) if state is None else state[b, h].astype(np.float64)
            rate = np.float64(decay[h])

            def power(steps):  # the present token counts 1 whatever the decay
                with np.errstate(invalid="ignore"):
                    return np.where(steps == 0, 1.0, np.exp(-rate * steps))

            w = np.where(gap >= 0, power(np.maximum(gap, 0)), 0.0)
            since, left, whole = power(np.arange(1, n + 1))[:, None], power(n - 1 - np.arange(n))[:, None], power(np.float64(n))
            out[b, h, :n] = scale * (((qq @ kk.T) * w) @ vv + since * (qq @ s0))
            new[b, h] = whole * s0 + (kk * left).T @ vv
            if dout is None:
                continue
            dd = dout[b, h, :n].astype(np.float64)
            end = np.zeros((dk, dv)) if dnew is None else dnew[b, h].astype(np.float64)
            p, dp = (qq @ kk.T) * w, (dd @ vv.T) * w
            g["dq"][b, h, :n] = scale * (dp @ kk + since * (dd @ s0.T))
            g["dk"][b, h // group, :n] += scale * (dp.T @ qq) + left * (vv @ end.T)
            g["dv"][b, h // group, :n] += scale * (p.T @ dd) + left * (kk @ end)
            g["dstate"][b, h] = whole * end + scale * ((qq * since).T @ dd)
    r = {"out": out, "new_state": new}
    if dout is not None:
        r.update(g)
    if seq_major:
        r = {n: t if n.endswith("state") else np.swapaxes(t, 1, 2) for n, t in r.items()}
    return r


def token_logprobs(logits, ids, top, temperature, dout=None, dentropy=None):
    t = float(temperature)
    z = logits.astype(np.float64)
    rows, width = z.shape
    given = 0 if ids is None else ids.shape[1]
    r = {"out": np.zeros((rows, given)), "entropy": np.zeros(rows), "top_ids": np.full((rows, top), -1.0),
         "top_logprobs": np.full((rows, top), -np.inf), "stats": np.zeros((rows, 2)), "grad": np.zeros(z.shape)}
    for i in range(rows):
        m = z[i].max()
        here = [] if ids is None else [(e, int(ids[i, e])) for e in range(given) if ids[i, e] >= 0]
        if not m < np.inf:  # NaN or +inf
            r["stats"][i] = r["entropy"][i] = r["top_logprobs"][i] = r["grad"][i] = np.nan
            for e, _ in here:
                r["out"][i, e] = np.nan
            continue
        if m == -np.inf:
            r["stats"][i] = m, 0.0
            for e, _ in here:
                r["out"][i, e] = -np.inf
            continue
        y = (z[i] - m) / t
        e = np.exp(y)
        lp = y - np.log(e.sum())
        p = e / e.sum()
        some = e > 0
        r["stats"][i] = m, e.sum()
        r["entropy"][i] = -(p[some] * lp[some]).sum()
        for at, token in here:
            r["out"][i, at] = lp[token]
        best = np.lexsort((np.arange(width), -logits[i]))[:top]
        best = best[logits[i, best] > -np.inf]
        r["top_ids"][i, :len(best)] = best
        r["top_logprobs"][i, :len(best)] = lp[best]
        d = np.zeros(width)
        if dout is not None:
            for at, token in here:
                d[token] += float(dout[i, at])
        total = d.sum()
        if dentropy is not None:
            d[some] -= float(dentropy[i]) * p[some] * (lp[some] + r["entropy"][i])
        r["grad"][i] = (d - p * total) / t
    return r
