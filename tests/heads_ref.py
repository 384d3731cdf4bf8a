"""The heads' operators in 64 bits and whole numbers, on numpy arrays."""

from __future__ import annotations

import math

import numpy as np

M64 = (1 << 64) - 1


def mix(z):
    """SplitMix64's finaliser on uint64 arrays."""
    z = z ^ (z >> np.uint64(30))
    z = z * np.uint64(0xBF58476D1CE4E5B9)
    z = z ^ (z >> np.uint64(27))
    z = z * np.uint64(0x94D049BB133111EB)
    return z ^ (z >> np.uint64(31))


def kept(seed, drop, elements):
    """Which elements (their numbers) stay."""
    e = np.asarray(elements, np.uint64)
    with np.errstate(over="ignore"):
        key = mix(np.array([seed], np.uint64) ^ np.uint64(0x9E3779B97F4A7C15))
        w = mix(key ^ ((e >> np.uint64(1)) * np.uint64(0xD6E8FEB86659FD93)))
    bits = np.where(e & np.uint64(1), w >> np.uint64(32), w & np.uint64(0xFFFFFFFF))
    return bits >= np.uint64(min(int(np.rint(drop * 2.0 ** 32)), 2 ** 32 - 1))


def tokens(ids, sizes, n_tokens, drop=0.0, seed=0):
    """(rows, columns) tokens, -1 where a position takes nothing. sizes None: one shared
    vocabulary."""
    n, t = ids.shape
    f = ids.astype(np.float64)
    first = np.zeros(t) if sizes is None else np.concatenate([[0], np.cumsum(sizes)[:-1]])
    most = np.full(t, n_tokens) if sizes is None else np.asarray(sizes)
    with np.errstate(invalid="ignore"):
        ok = (f >= 0) & (f < most) & (f == np.floor(f))
    if drop:
        ok &= kept(seed, drop, np.arange(n * t)).reshape(n, t)
    return np.where(ok, np.where(ok, f, 0) + first, -1).astype(np.int64)


def embed(table, tok, scale, pooled):
    """Values, and the sums of the magnitudes that went into them."""
    rows = np.where((tok >= 0)[..., None], table.astype(np.float64)[np.maximum(tok, 0)], 0.0)
    if pooled:
        return rows.sum(1) * scale, np.abs(rows).sum(1) * abs(scale)
    return rows * scale, np.abs(rows) * abs(scale)


def embed_grad(grad, tok, n_tokens, scale, pooled):
    """The same of the table's gradient, and how many positions each token has."""
    n, t = tok.shape
    g = grad.astype(np.float64)
    g = np.repeat(g[:, None], t, 1) if pooled else g.reshape(n, t, -1)
    at = tok >= 0
    out = np.zeros((n_tokens, g.shape[-1]))
    mag = np.zeros_like(out)
    np.add.at(out, tok[at], g[at])
    np.add.at(mag, tok[at], np.abs(g[at]))
    return out * scale, mag * abs(scale), np.bincount(tok[at], minlength=n_tokens)


ONE = 1 << 45


def _options_row(opt, i, v):
    t, k, p, m = (np.asarray(o).reshape(-1) for o in opt)
    t, k, p, m = (o[i if o.size > 1 else 0] for o in (t, k, p, m))
    t, p, m = (float(np.float32(x)) for x in (t, p, m))
    k = int(k) if t > 0.0 else 1  # (NaN: 1)
    k = v if k <= 0 else min(k, v)
    p = 1.0 if not p < 1.0 else max(p, 0.0)
    m = min(m, 1.0) if m > 0.0 else 0.0
    return t, k, p, m


def sample(logits, uniforms, temperature, top_k, top_p, min_p):
    """Classes and log-probabilities, weights in Python's whole numbers."""
    n, v = logits.shape
    ids = np.full(n, -1, np.int64)
    logp = np.full(n, -np.inf)
    for i in range(n):
        t, k, p, m = _options_row((temperature, top_k, top_p, min_p), i, v)
        x = logits[i].astype(np.float64)
        x[np.isnan(x)] = -np.inf
        top = x.max()
        if top == -np.inf:
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            z = np.where(x == top, 0.0, (x - top) / t if t > 0.0 else -np.inf)
        w = [int(a) for a in np.rint(np.exp(z) * ONE)]
        order = sorted(range(v), key=lambda j: (-x[j], j))[:k]
        total = sum(w[j] for j in order)
        most = max(1, -(-int(p * 2 ** 31) * total // 2 ** 31))
        stay, before = set(), 0
        for j in order:
            if before < most and w[j] >= m * ONE:
                stay.add(j)
            before += w[j]
        total = sum(w[j] for j in stay)
        u = float(uniforms[i])
        u31 = min(int(u * 2 ** 31), 2 ** 31 - 1) if u > 0 else 0
        target, cum = u31 * total >> 31, 0
        for j in range(v):
            if j in stay:
                cum += w[j]
                if cum > target:
                    ids[i], logp[i] = j, z[j] - math.log(total / ONE)
                    break
    return ids, logp
