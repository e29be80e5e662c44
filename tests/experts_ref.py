"""A layer of experts from its definitions, in 64 bits on the host (numpy), and how far an fp32 result may be from them.

Bars of a product over K values, with u = 2^-24 half a step of fp32.  An activation in two fp16 parts is off by at most
2^-22 of itself (half a step of fp16, 2^-11, twice) or, where the second part is subnormal, by 2^-25 with the row's largest
at 2^14 or more: 2^-39 of the largest.  The integers of the weights and their products are exact; sums are rounded once or
twice per matrix instruction of 16 values and once or twice per scale of 16 or 32: fewer than K / 4 + 16 roundings of
partial sums that are at most S = sum |x w| (Q4_K: with |w| = d sc q + dmin mn, its two sums).
  * worst: (2^-22 + (K / 4 + 16) u) S + 2^-39 K max|x| max|w|
  * typical: roundings are independent and partial sums of centred products about their root sum of squares Q, so the errors'
    root mean square stays below (2^-22 + 2 sqrt(K / 4 + 16) u) Q.  One fp16 part instead of two would give 2^-11 / sqrt(12) Q,
    which is 50 times as much at K = 2048.
SiLU(g) u: |u| 1.1 times g's error, |silu(g)| times u's, and (|g| + 8) 2^-23 of the result for exp2, its argument and 1 / x."""
import numpy as np

import oracle as orc

U = 2.0 ** -24


def f64(x):
    return x.detach().cpu().double().numpy() if hasattr(x, "detach") else np.asarray(x, np.float64)


def weights(fmt, raw, E, N, K):
    """([E, N, K] values, their magnitudes as the kernels add them up), both float64."""
    raw = np.ascontiguousarray(raw).reshape(-1)
    if fmt == "fp16":
        w = raw.view(np.float16).astype(np.float64).reshape(E, N, K)
    else:
        w = orc.dequantize(fmt, raw, E * N * K).astype(np.float64).reshape(E, N, K)
    mag = np.abs(w)
    if fmt == "q4_k":  # d sc q + dmin mn = w + 2 dmin mn
        b = raw.reshape(-1, 144)
        dmin = b[:, 2:4].copy().view(np.float16).astype(np.float64)
        s = b[:, 4:16].astype(np.int64)
        mn = np.concatenate([s[:, 4:8] & 63, (s[:, 8:] >> 4) | ((s[:, 4:8] >> 6) << 4)], 1)
        mag = np.abs(w + 2 * np.repeat(dmin * mn, 32, 1).reshape(E, N, K))
        mag = np.maximum(mag, np.abs(w))
    return w, mag


def group(ids, E):
    """offsets, rows, slots of ids [M, k]."""
    flat = np.asarray(ids).reshape(-1)
    members = [np.flatnonzero(flat == e) for e in range(E)]
    order = np.concatenate(members) if len(flat) else np.zeros(0, np.int64)
    offsets = np.cumsum([0] + [len(m) for m in members])
    rows, slots = np.full(len(flat), -1), np.full(len(flat), -1)
    rows[:len(order)] = order
    slots[order] = np.arange(len(order))
    return offsets, rows, slots


def route(logits, k, sigmoid, bias, normalize, scale):
    """ids, weights, and the smallest gap between a choice's score and the next one's, relative (ties excepted)."""
    z = f64(logits)
    M, E = z.shape
    ids, w = np.full((M, k), -1), np.zeros((M, k))
    for t in range(M):
        x = np.where(np.isnan(z[t]), -np.inf, z[t])
        some = np.flatnonzero(x > -np.inf)
        if not len(some):
            continue
        v = x[some]
        with np.errstate(over="ignore", invalid="ignore"):
            top = v.max()
            e = np.where(v == top, 1.0, np.exp(v - top))
            s = 1 / (1 + np.exp(-v)) if sigmoid else e / e.sum()
        key = v if bias is None else s + f64(bias)[some]
        key = np.where(np.isnan(key), -np.inf, key)
        best = np.lexsort((some, -key))
        best = best[key[best] > -np.inf][:k]
        ids[t, :len(best)] = some[best]
        p = s[best]
        if normalize:
            p = p / p.sum() if p.sum() > 0 else 0 * p
        w[t, :len(best)] = p * scale
    return ids, w


class Product:
    """x [R, K] rows (already gathered) times w [N, K]: the result and its two bars."""

    def __init__(self, x, w, mag):
        x = f64(x)
        K = x.shape[1]
        ax = np.abs(x)
        self.want = x @ w.T
        S, Q = ax @ mag.T, np.sqrt((x * x) @ (mag * mag).T)
        n = K / 4 + 16
        self.worst = (2.0 ** -22 + n * U) * S + 2.0 ** -39 * K * ax.max(1, initial=0)[:, None] * mag.max(1)[None]
        self.rms = (2.0 ** -22 + 2 * np.sqrt(n) * U) * Q


def silu(g):
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-g))


class Swiglu:
    def __init__(self, x, gate, up):
        g, u = Product(x, *gate), Product(x, *up)
        s = silu(g.want)
        self.want = s * u.want
        own = (np.abs(g.want) + 8) * 2 * U * np.abs(self.want)
        self.worst = 1.1 * (np.abs(u.want) + u.worst) * g.worst + np.abs(s) * u.worst + own
        self.rms = np.sqrt((1.1 * u.want * g.rms) ** 2 + (s * u.rms) ** 2) + own


def check(got, ref, name=""):
    """Every element within the worst bar, the errors' root mean square within the typical one."""
    got = f64(got)
    assert got.shape == ref.want.shape, (name, got.shape, ref.want.shape)
    err = np.abs(got - ref.want)
    assert np.isfinite(got).all(), name
    assert (err <= ref.worst + 1e-300).all(), (name, float((err / (ref.worst + 1e-300)).max()))
    if err.size:
        a, b = np.sqrt((err ** 2).mean()), np.sqrt((ref.rms ** 2).mean())
        assert a <= b, (name, a / b)
