"""64-bit restatements of the language-model operators (numpy), straight from
their formulas."""
import numpy as np


def layer_norm(x, gain, bias, eps, dy=None):
    x = x.astype(np.float64)
    mean = x.mean(1, keepdims=True)
    rstd = 1.0 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    n = (x - mean) * rstd
    gain = np.ones(x.shape[1]) if gain is None else gain.astype(np.float64)
    y = n * gain + (0.0 if bias is None else bias.astype(np.float64))
    out = {"y": y, "stats": np.concatenate([mean, rstd], 1)}
    if dy is not None:
        dy = dy.astype(np.float64)
        g = dy * gain
        out["dx"] = rstd * (g - g.mean(1, keepdims=True) - n * (g * n).mean(1, keepdims=True))
        out["dgain"], out["dbias"] = (dy * n).sum(0), dy.sum(0)
    return out


def rope_axes(x, positions, sections, theta, seq_major, back=False):
    """x [B, H, S, 2 half] or [B, S, H, 2 half]; positions [B, axes, S]."""
    half = sum(sections)
    axis = np.repeat(np.arange(len(sections)), sections)
    rate = np.float64(theta) ** (-np.arange(half) / half)
    angle = np.moveaxis(positions.astype(np.float64)[:, axis], 1, 2) * rate
    angle = angle[:, :, None] if seq_major else angle[:, None]
    z = (x[..., :half].astype(np.float64) + 1j * x[..., half:]) * np.exp((-1j if back else 1j) * angle)
    return np.concatenate([z.real, z.imag], -1)


def visible(starts, lengths, batch, q_len, k_len, window, sinks):
    """[batch, q_len, k_len]: whether a row sees a key."""
    n = np.full(batch, k_len) if lengths is None else np.asarray(lengths).astype(np.int64)
    first = np.full(batch, k_len - q_len) if starts is None else np.asarray(starts).astype(np.int64)
    p = first[:, None, None] + np.arange(q_len)[None, :, None]
    j = np.arange(k_len)[None, None]
    seen = (p >= 0) & (p < n[:, None, None]) & (j <= p)
    if window:
        seen &= (p - j < window) | (j < sinks)
    return seen


def window_attention(q, k, v, starts, lengths, window, sinks, scale, seq_major, dout=None):
    if seq_major:
        q, k, v = (np.swapaxes(t, 1, 2) for t in (q, k, v))
        dout = None if dout is None else np.swapaxes(dout, 1, 2)
    batch, heads, q_len, dim = q.shape
    kv_heads, k_len = k.shape[1:3]
    group = heads // kv_heads
    seen = visible(starts, lengths, batch, q_len, k_len, window, sinks)
    out = np.zeros(q.shape)
    stats = np.zeros((batch, heads, q_len, 2))
    dq, dk, dv = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
    size_q, size_k = np.zeros(q.shape), np.zeros(k.shape)
    for b in range(batch):
        any_row = seen[b].any(0)
        live = seen[b].any(1)
        for h in range(heads):
            # Keys and rows that take part in nothing are left out, whatever they hold.
            kk = np.where(any_row[:, None], k[b, h // group], 0.0).astype(np.float64)
            vv = np.where(any_row[:, None], v[b, h // group], 0.0).astype(np.float64)
            qq = np.where(live[:, None], q[b, h], 0.0).astype(np.float64)
            s = np.where(seen[b], (qq @ kk.T) * scale, -np.inf)
            m = s.max(1, initial=-np.inf)
            e = np.exp(s - np.where(live, m, 0.0)[:, None])
            l = e.sum(1)
            p = e / np.where(live, l, 1.0)[:, None]
            o = p @ vv
            out[b, h], stats[b, h, :, 0], stats[b, h, :, 1] = o, m, l
            if dout is not None:
                g = np.where(live[:, None], dout[b, h], 0.0).astype(np.float64)
                ds = p * (g @ vv.T - (g * o).sum(1, keepdims=True)) * scale
                dq[b, h] = ds @ kk
                dk[b, h // group] += ds.T @ qq
                dv[b, h // group] += p.T @ g
                # The size of the terms whose difference dS is.
                terms = p * (np.abs(g) @ np.abs(vv).T + (np.abs(g) * np.abs(o)).sum(1, keepdims=True)) * scale
                size_q[b, h] = terms @ np.abs(kk)
                size_k[b, h // group] += terms.T @ np.abs(qq)
    r = {"out": out, "stats": stats}
    if dout is not None:
        r.update(dq=dq, dk=dk, dv=dv, size_dq=size_q, size_dk=size_k)
    if seq_major:
        r = {n: t if n == "stats" else np.swapaxes(t, 1, 2) for n, t in r.items()}
    return r


def distill_loss(logits, ids, teacher, temperature, dloss=None):
    t = float(temperature)
    z = logits.astype(np.float64)
    rows, width = z.shape
    top = z.max(1, keepdims=True)
    e = np.exp((z - top) / t)
    total = e.sum(1, keepdims=True)
    loss, grad = np.zeros(rows), np.zeros(z.shape)
    for r in range(rows):
        here = (ids[r] >= 0) & (teacher[r] > -np.inf)
        if not here.any():
            continue
        w = teacher[r, here].astype(np.float64) / t
        log_p = w - w.max() - np.log(np.exp(w - w.max()).sum())
        at = ids[r, here].astype(np.int64)
        log_q = (z[r, at] - top[r, 0]) / t - np.log(total[r, 0])
        p = np.exp(log_p)
        loss[r] = t * t * (p * (log_p - log_q)).sum()
        if dloss is not None:
            g = e[r] / total[r, 0]
            np.subtract.at(g, at, p)
            grad[r] = t * float(dloss[r]) * g
    out = {"loss": loss, "stats": np.concatenate([top, total], 1)}
    if dloss is not None:
        out["grad"] = grad
    return out
