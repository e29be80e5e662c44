"""The batched serving operators from their definitions, in 64 bits on the host (numpy), a row at a time."""
import math

import numpy as np


def f64(x):
    return x.detach().cpu().double().numpy() if hasattr(x, "detach") else np.asarray(x, np.float64)


def norm_rotate(x, w, p, rot, halves, theta, eps):
    """x [heads, D] at position p -> (result, sum of the magnitudes that enter each element)."""
    x = np.array(x, np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * f64(w)
    out, mag = x.copy(), np.abs(x)
    i = np.arange(rot // 2)
    angle = p * float(theta) ** (-2.0 * i / rot) if rot else np.zeros(0)
    a, b = (i, i + rot // 2) if halves else (2 * i, 2 * i + 1)
    cos, sin = np.cos(angle), np.sin(angle)
    out[:, a] = x[:, a] * cos - x[:, b] * sin
    out[:, b] = x[:, b] * cos + x[:, a] * sin
    mag[:, a] = mag[:, b] = np.abs(x[:, a]) + np.abs(x[:, b])
    return out, mag


def places(offsets, lens, n_rows):
    """(row, sequence, position) of every row of the batch."""
    for s in range(len(lens)):
        n = offsets[s + 1] - offsets[s]
        for i in range(n):
            t = offsets[s] + i
            if 0 <= t < n_rows:
                yield t, s, lens[s] - n + i


def attention(q, k, v, offsets, lens, pages, prefix_pages, prefix_len, n_heads, scale, out):
    """q [rows, H D], k and v [n_pages, ps, Hkv, D] -> out (a copy of `out` with the batch's rows written)."""
    q, k, v, out = f64(q), f64(k), f64(v), f64(out).copy()
    _, ps, Hkv, D = k.shape
    G, cap = n_heads // Hkv, len(pages[0]) * ps
    for t, s, p in places(offsets, lens, len(q)):
        end = min(p + 1, max(cap, min(prefix_len, p + 1)))
        if end <= 0:
            out[t] = 0
            continue
        j = np.arange(end)
        page = np.array([prefix_pages[x // ps] if x < prefix_len else pages[s][x // ps] for x in j])
        kk, vv = k[page, j % ps], v[page, j % ps]  # [end, Hkv, D]
        for h in range(n_heads):
            x = kk[:, h // G] @ q[t, h * D:(h + 1) * D] * scale
            w = np.exp(x - x.max())
            out[t, h * D:(h + 1) * D] = (w / w.sum()) @ vv[:, h // G]
    return out


def verify(target, draft, ids, u, draws, offsets, out, accepted):
    """Copies of out and accepted with the batch's entries written."""
    p_all, q_all = f64(target), None if draft is None else f64(draft)
    ids, u, draws, out, accepted = np.asarray(ids), f64(u), f64(draws), np.array(out), np.array(accepted)
    V = p_all.shape[1]
    for s in range(len(offsets) - 1):
        lo, hi = offsets[s], offsets[s + 1]
        accepted[s] = 0
        if hi <= lo:
            continue
        a = 0
        for r in range(lo, hi - 1):
            x = ids[r]
            if not (0 <= x < V and u[r] * (1.0 if q_all is None else q_all[r, x]) < p_all[r, x]):
                break
            a += 1
        r = lo + a
        p = np.where(p_all[r] > 0, p_all[r], 0.0)
        w = p.copy()
        if r < hi - 1:
            if q_all is None:
                if 0 <= ids[r] < V:
                    w[ids[r]] = 0
            else:
                with np.errstate(invalid="ignore"):
                    w = p - q_all[r]
                w = np.where(w > 0, w, 0.0)
            if not math.fsum(w) > 0:
                w = p
        out[lo:hi] = -1
        out[lo:lo + a] = ids[lo:lo + a]
        some = np.flatnonzero(w > 0)
        if len(some):
            total, run, tok = math.fsum(w), 0.0, some[-1]
            for i in some:
                run += w[i]
                if run > draws[r] * total:
                    tok = i
                    break
            out[r] = tok
        accepted[s] = a
    return out, accepted
