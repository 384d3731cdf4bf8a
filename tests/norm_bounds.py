"""How far layer norm's float32 sums may be from their values, from the lanes and cells that a
row of a width has."""

from __future__ import annotations

import math

import numpy as np

import training_ref as ref

# widths up to these have so many lanes a row, of so many cells each
SHAPES = [(32, 4, 8), (64, 8, 8), (128, 16, 8), (256, 16, 16), (512, 64, 8), (1024, 64, 16),
          (2048, 256, 8), (4096, 256, 16), (8192, 512, 16), (16_384, 512, 32), (32_768, 512, 64)]
CHAIN = 1024  # rows that a lane adds up in float32 at most


def _shape(dim):
    return next(s[1:] for s in SHAPES if dim <= s[0])


def path(dim):
    """Roundings on the way of a cell into its row's mean: a lane's cells in turn, its levels of
    lanes, and the division by a rounded 1 / dim."""
    lanes, cells = _shape(dim)
    return cells + int(math.log2(lanes)) + 2


def parts(n, dim):
    """(workgroups, rows that one holds at once) of the weights' sums."""
    lanes, _ = _shape(dim)
    rows = max(256 // lanes, 1)
    if dim <= 4096 and n <= 2 * rows:
        return 1, rows
    most = 1024 if dim <= 256 else 512 if dim <= 4096 else 256 if dim <= 16_384 else 64
    turns = max(-(-n // rows), 1)
    return min(turns, most, max(turns // (8 if rows == 1 else 4), 128)), rows


def weight_path(n, dim):
    """Roundings on the way of a row's term into a weight's sum, up to the part of its workgroup:
    the rows of a lane in turn, then a quarter of the rows that a workgroup holds at once, and
    two levels of those four."""
    groups, rows = parts(n, dim)
    return min(-(-n // (groups * rows)), CHAIN) + (rows // 4 + 2 if rows > 1 else 0)


def layer_norm_grad(g, x, w, eps):
    """((dx, off), (dw, off), (db, off)) as training_ref gives the values. In half steps of
    float32, with p a row's path: a mean is off by p of its terms' mean magnitude and what is
    left of it by as many of the differences', so h by p + 3 (of a mean magnitude of at most 1)
    and by 2 |h|, and r by (p + 5) / 2 + 3: h by less than (p + 9) (|h| + 1) with the kept
    statistics' rounding. Terms of mean(d h) are off by that and by p + 6, the result by its
    product with h and 4 roundings more: below 3 p + 30 of the magnitudes together. A weight's
    sum takes its path, one rounding of the product and what h is off by."""
    (dx, _), (dw, _), (db, _) = ref.layer_norm_grad(g, x, w, eps)
    g = np.abs(g.astype(np.float64))
    n, dim = x.shape
    p, length = path(dim), weight_path(n, dim)
    h, r = ref.norm_parts(x, eps)
    size = np.abs(h) + 1
    d = g if w is None else g * np.abs(w.astype(np.float64))
    off = r * ref.ULP * (3 * p + 30) * (d + d.mean(-1, keepdims=True) +
                                        size * (d * size).mean(-1, keepdims=True))
    return ((dx, off), (dw, ref.ULP * (p + 9 + length + 1) * (g * size).sum(0)),
            (db, ref.ULP * length * g.sum(0)))
