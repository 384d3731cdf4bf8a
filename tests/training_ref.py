"""The training heads' operators in 64 bits and whole numbers, on numpy arrays."""

from __future__ import annotations

import numpy as np

import heads_ref

ULP = 2.0 ** -24  # half a step of float32, relative


def norm_parts(x, eps):
    """(h, 1 / sqrt(variance + eps)) of rows."""
    x = x.astype(np.float64)
    c = x - x.mean(-1, keepdims=True)
    r = 1.0 / np.sqrt((c * c).mean(-1, keepdims=True) + float(np.float32(eps)))
    return c * r, r


def layer_norm(x, w, b, eps):
    """Values, and how far float32 may be from them. A sum over a row is a tree of at most 44
    additions a path (32 cells a lane, 10 levels of lanes, the division): a mean is off by 44
    half steps of the mean magnitude. What is left of the mean is taken out, so h is off by
    its own differences' rounding, by the 44 of the rest (of a mean magnitude of at most 1 in
    units of 1 / r), by the variance's (44 + 4) / 2 and by 6 roundings of what is done to it:
    together below 64 half steps of |h| + 1."""
    h, _ = norm_parts(x, eps)
    w = np.ones(x.shape[-1]) if w is None else w.astype(np.float64)
    b = np.zeros(x.shape[-1]) if b is None else b.astype(np.float64)
    y = h * w + b
    return y, ULP * (64 * (np.abs(h) + 1) * np.abs(w) + 2 * (np.abs(y) + np.abs(b)))


def layer_norm_grad(g, x, w, eps, groups=512):
    """((dx, off), (dw, off), (db, off)). The means over a row are trees as above, 48 half steps
    of their terms' magnitudes; h is off by 64 of |h| + 1, the statistics kept in float32 among
    them, r by 30. A weight's sum is a chain over the rows of a workgroup, in turn (a group of
    lanes has at most one in 512 of a few thousand rows, or one in 64 of up to 600 wide ones) and
    then side by side (at most 64 groups, of which wide rows have one), and exact from there
    on."""
    g, n = g.astype(np.float64), x.shape[0]
    w = np.ones(x.shape[-1]) if w is None else w.astype(np.float64)
    h, r = norm_parts(x, eps)
    d = g * w
    a, b = d.mean(-1, keepdims=True), (d * h).mean(-1, keepdims=True)
    dx = r * (d - a - h * b)
    am = np.abs(d).mean(-1, keepdims=True)
    bm = (np.abs(d) * (np.abs(h) + 1)).mean(-1, keepdims=True)
    off = r * ULP * 128 * (np.abs(d) + am + (np.abs(h) + 1) * bm)
    terms = -(-n // groups) + 64 + 2
    dw, db = (g * h).sum(0), g.sum(0)
    off_w = ULP * (64 + terms) * (np.abs(g) * (np.abs(h) + 1)).sum(0)
    return (dx, off), (dw, off_w), (db, ULP * terms * np.abs(g).sum(0))


def route(ids, n_experts):
    """order, place, starts of an id matrix."""
    f = ids.astype(np.float64).reshape(-1)
    with np.errstate(invalid="ignore"):
        ok = (f >= 0) & (f < n_experts) & (f == np.floor(f))
    key = np.where(ok, np.where(ok, f, 0), n_experts).astype(np.int64)
    order = np.argsort(key, kind="stable")
    row = np.empty(key.size, np.int64)
    row[order] = np.arange(key.size)
    place = np.where(ok, row, -1 - row)
    starts = np.concatenate([[0], np.cumsum(np.bincount(key, minlength=n_experts + 1)[:-1])])
    return order.astype(np.int32), place.astype(np.int32).reshape(ids.shape), starts.astype(
        np.int32)


def from_experts(y, place, weights):
    """Values and the sums of the magnitudes that went into them; rows 2-d, place (n, k)."""
    ok = (place >= 0)[..., None]
    rows = np.where(ok, y[np.maximum(place, 0)].astype(np.float64), 0.0)
    if weights is not None:
        rows = rows * weights.astype(np.float64)[..., None]
    return rows.sum(1), np.abs(rows).sum(1)


def from_experts_grad(g, y, place, weights):
    """dy, dweights and the sums of the magnitudes of the latter's products."""
    n, k = place.shape
    g = g.astype(np.float64)
    ok = (place >= 0)[..., None]
    w = np.ones((n, k)) if weights is None else weights.astype(np.float64)
    part = np.where(ok, g[:, None] * w[..., None], 0.0)
    dy = np.empty((n * k, g.shape[1]))
    dy[np.where(place >= 0, place, -1 - place).reshape(-1)] = part.reshape(n * k, -1)
    rows = np.where(ok, y[np.maximum(place, 0)].astype(np.float64), 0.0)
    prod = rows * g[:, None]
    return dy, prod.sum(2), np.abs(prod).sum(2)


# ---- AdamW. Values of the 8-bit floats: the exponent field of 30 or 14 is the block's.
def byte_values(code, field, square):
    code = code.astype(np.int64)
    size = code if square else code & 0x7F
    e, f = size >> 3, size & 7
    top, least = (30, 29) if square else (14, 13)
    big = np.maximum(field.astype(np.int64), 1).repeat(256) - 127
    v = np.where(e > 0, np.ldexp(1.0 + f / 8.0, e - top + big), np.ldexp(f / 8.0, big - least))
    v = np.where(size == (0xFF if square else 0x7F), np.nan, v)
    return v if square or not code.size else np.where(code & 0x80, -v, v)


def to_bytes(x, random, square):
    """Codes and exponent fields of float32 values in blocks of 256; random: 16 bits each."""
    x = np.ascontiguousarray(x, np.float32)
    bits = x.view(np.uint32) & np.uint32(0x7FFFFFFF)
    finite = bits < 0x7F800000
    field = (np.where(finite, bits, 0) >> 23).reshape(-1, 256).max(1)
    top, least = (30, 29) if square else (14, 13)
    big = np.maximum(field.astype(np.int64), 1).repeat(256) - 127
    mag = np.where(finite, np.abs(x), 0).astype(np.float64)
    e = np.maximum(np.frexp(mag)[1] - 1, big - least)
    q = np.ldexp(mag, 3 - e)  # in units of the last place
    low = np.floor(q)
    up = np.rint((q - low) * 2.0 ** 20) + random.astype(np.float64) * 16 >= 2.0 ** 20
    units = (low + up).astype(np.int64)
    # a number of units below 8 is subnormal, and 16 of them are 8 of the next exponent
    code = units + ((e - (big - least)) << 3) * (units > 0)
    if square:
        code = np.where((code == 0) & (mag > 0), 1, code)
    code = np.where(finite, code, 0xFF if square else 0x7F)
    if not square:
        code = code | (np.signbit(x).astype(np.int64) << 7)
    return code.astype(np.uint8), field.astype(np.uint8)


def random_words(seed, n):
    """32 bits a cell, those that dropout draws."""
    e = np.arange(n, dtype=np.uint64)
    with np.errstate(over="ignore"):
        key = heads_ref.mix(np.array([seed & heads_ref.M64], np.uint64) ^
                            np.uint64(0x9E3779B97F4A7C15))
        w = heads_ref.mix(key ^ ((e >> np.uint64(1)) * np.uint64(0xD6E8FEB86659FD93)))
    return np.where(e & np.uint64(1), w >> np.uint64(32), w & np.uint64(0xFFFFFFFF))


def adamw(w, g, m, s, t, lr, betas, eps, decay):
    """(w, off), (m, off), (s, off) of step t in 64 bits, and how far float32 may be: 5
    roundings of a moment's terms (its factors among them), and of the step a further 12."""
    b1, b2 = betas
    w, g, m, s = (a.astype(np.float64) for a in (w, g, m, s))
    mm, ss = np.abs(b1 * m) + np.abs((1 - b1) * g), b2 * s + (1 - b2) * g * g
    m = b1 * m + (1 - b1) * g
    size, root = lr / (1 - b1 ** t), 1 / np.sqrt(1 - b2 ** t)
    den = np.sqrt(ss) * root + float(np.float32(eps))
    out = w * (1 - lr * decay) - size * m / den
    off = ULP * (3 * np.abs(w) + np.abs(out) + 20 * size * mm / den)
    return (out, off), (m, 5 * ULP * mm + 2.0 ** -148), (ss, 5 * ULP * ss + 2.0 ** -148)
