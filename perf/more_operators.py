"""Workloads of training heads on a model's outputs: vectors normalised, rows handed to experts
by their ids and brought back, and the step that learns their parameters.

  norm          layer norm over a row's cells
  norm_grad     its gradients: of the rows, and of the weight and bias, summed over all rows
  route         positions of an id matrix (leaf ids, codes) in the order of their ids
  experts       the same, the rows copied in that order, and what experts give for them brought
                back, weighted and summed
  experts_grad  the gradients of both copies and of the weights
  adamw         an AdamW step of many parameters at once, moments in 32 bits or in 8
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
CHUNK = 1 << 26  # elements of one intermediate of the plain forms
M64 = (1 << 64) - 1
GOLDEN, STEP = 0x9E3779B97F4A7C15, 0xD6E8FEB86659FD93
MIX1, MIX2 = 0xBF58476D1CE4E5B9, 0x94D049BB133111EB
BLOCK = 256  # cells of a parameter whose 8-bit moments share an exponent
BETAS, EPS, DECAY = (0.9, 0.999), 1e-8, 0.01
NORM_EPS = 1e-5


# --------------------------------------------------------------------- cases
def _norm(name, kind, **kw):
    c = {"name": name, "kind": kind, "rows": 1, "dim": 64, "type": "float32",
         "weight": "float32"}
    c.update(kw)
    return c


def _experts(name, kind, **kw):
    c = {"name": name, "kind": kind, "rows": 1, "columns": 2, "experts": 8, "dim": 64,
         "type": "float32", "ids": "int32", "skew": 0.0, "missing": 0.0}
    c.update(kw)
    return c


def _adamw(name, **kw):
    c = {"name": name, "kind": "adamw", "tensors": 1, "cells": 4096, "type": "float32",
         "even": False, "bits": 32, "step": 100, "lr": 1e-3}
    c.update(kw)
    return c


def listed():
    return [
        # One row's vector in a service.
        _norm("norm_row", "norm"),
        # A batch of wide vectors on their way to the next product.
        _norm("norm_batch", "norm", rows=32_768, dim=4096, type="bfloat16", weight="bfloat16"),
        # The gradient of a head's training batch: 100k rows of 64 cells, the weight in float32.
        _norm("norm_grad_vectors", "norm_grad", rows=100_000, type="bfloat16"),
        # An odd width, and the gradient of norm_batch.
        _norm("norm_grad_odd", "norm_grad", rows=20_001, dim=1023),
        _norm("norm_grad_batch", "norm_grad", rows=32_768, dim=4096, type="bfloat16",
              weight="bfloat16"),
        # A few rows in a service, each to the experts of its leaves in two trees of depth 3.
        _experts("experts_rows", "experts", rows=4, experts=15, ids="float32"),
        # The ids of 2M rows in one tree of depth 8: rows by leaf.
        _experts("route_leaves", "route", rows=2_000_000, columns=1, experts=511,
                 ids="float32"),
        # A training batch of vectors, two of 64 experts a row, some experts frequent; then
        # the backward pass of an odd one, some positions without an expert.
        _experts("experts_batch", "experts", rows=65_536, experts=64, dim=1024,
                 type="bfloat16", skew=0.8),
        _experts("experts_grad_odd", "experts_grad", rows=30_001, columns=4, experts=200,
                 dim=515, ids="int64", missing=0.05),
        # The parameters of a small head: a table of leaves' vectors and a few layers.
        _adamw("adamw_head", tensors=12, cells=4000),
        # Large ones: 8 tables of 8M cells, and 60 tensors of 2M cells with moments in 8 bits,
        # which are read as float32 values afterwards, as what stores or watches them does.
        _adamw("adamw_tables", tensors=8, cells=8_000_000, even=True),
        _adamw("adamw_8bit", tensors=60, cells=2_000_000, even=True, type="bfloat16", bits=8),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "norm_grad", "route", "experts", "experts_grad",
                       "adamw", "adamw", "adamw"])
    dtype = rng.choice(sorted(TYPES))
    if kind in ("norm", "norm_grad"):
        # (the gradient of one cell is 0, of two a term of eps alone)
        dim = _log_int(rng, 3, 32_768)
        return _norm("", kind, dim=dim, type=dtype, weight=rng.choice([dtype, "float32"]),
                     rows=_log_int(rng, 1, min(2_000_000, (128 << 20) // dim)))
    if kind == "adamw":
        tensors = _log_int(rng, 1, 200)
        # (a tensor's cells are up to four times these)
        return _adamw("", tensors=tensors, cells=_log_int(rng, 4, (16 << 20) // tensors),
                      even=rng.random() < 0.3, type=dtype, bits=rng.choice([8, 32]), step=rng.choice([0, 1, 10, 10_000]),
                      lr=rng.choice([1e-4, 1e-3, 1e-2]))
    columns = rng.choice([1, 2, 2, 4, 8])
    rows, dim = _log_int(rng, 1, 2_000_000 // columns), 1
    if kind != "route":
        dim = _log_int(rng, 1, 4096)
        rows = max(1, min(rows, (64 << 20) // (columns * dim)))
    return _experts("", kind, rows=rows, columns=columns, experts=_log_int(rng, 2, 1024),
                    dim=dim, type=dtype, ids=rng.choice(["int32", "int64", "float32"]),
                    skew=rng.choice([0.0, 0.8, 1.5]), missing=rng.choice([0.0, 0.05]))


# -------------------------------------------------------------------- inputs
def _randn(shape, g, dtype, scale=1.0):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).mul_(scale).to(dtype)


def _prepare_norm(case, g, st):
    n, d, dt, wt = case["rows"], case["dim"], TYPES[case["type"]], TYPES[case["weight"]]
    # vectors with means and lengths of their own
    x = torch.randn((n, d), generator=g, device=DEV)
    x.mul_(torch.rand((n, 1), generator=g, device=DEV).add_(0.5))
    st["x"] = x.add_(torch.randn((n, 1), generator=g, device=DEV)).to(dt)
    st["w"] = _randn((d,), g, torch.float32, 0.2).add_(1.0).to(wt)
    st["b"] = _randn((d,), g, wt, 0.1)
    if case["kind"] == "norm_grad":
        st["g"] = _randn((n, d), g, dt)
        # what the forward pass has kept: each row's mean and 1 / sqrt(variance + eps)
        st["stats"] = torch.empty((n, 2), device=DEV)
        for b in range(0, n, max(1, CHUNK // d)):
            x = st["x"][b:b + max(1, CHUNK // d)].double()
            mean = x.mean(1, keepdim=True)
            var = (x - mean).square().mean(1)
            st["stats"][b:b + x.shape[0], 0] = mean[:, 0].float()
            st["stats"][b:b + x.shape[0], 1] = torch.rsqrt(var + NORM_EPS).float()


def _prepare_experts(case, g, st):
    n, k, e, d = case["rows"], case["columns"], case["experts"], case["dim"]
    dt = TYPES[case["type"]]
    p = torch.arange(1, e + 1, device=DEV, dtype=torch.float64) ** -case["skew"]
    u = torch.rand((n, k), generator=g, device=DEV, dtype=torch.float64)
    rank = torch.searchsorted(torch.cumsum(p / p.sum(), 0), u).clamp_(max=e - 1)
    ids = torch.randperm(e, generator=g, device=DEV)[rank]
    if case["missing"]:
        ids[torch.rand((n, k), generator=g, device=DEV) < case["missing"]] = -1
    st["ids"] = ids.to(getattr(torch, case["ids"])).contiguous()
    if case["kind"] == "route":
        return
    st["weights"] = torch.softmax(torch.randn((n, k), generator=g, device=DEV), 1)
    st["y"] = _randn((n * k, d), g, dt)
    if case["kind"] == "experts":
        st["x"] = _randn((n, d), g, dt)
        return
    st["g"], st["gs"] = _randn((n, d), g, dt), _randn((n * k, d), g, dt)
    if own:
        from ferrisboost_amd import heads

        st["routes"] = heads.Routes(st["ids"], e)
    else:
        st["routes"] = _plain_route(st)


def _sizes(case):
    """Cells of each parameter, and where its moments begin in all of them."""
    rng = random.Random(case["tensors"] * 1_000_003 + case["cells"])
    n = [case["cells"] if case["even"] else
         max(1, int(case["cells"] * 4.0 ** rng.uniform(-1.0, 1.0)))
         for _ in range(case["tensors"])]
    first = [0]
    for s in n:
        first.append(first[-1] + -(-s // BLOCK) * BLOCK)
    return n, first


def _prepare_adamw(case, g, st):
    n, first = _sizes(case)
    dt, total = TYPES[case["type"]], first[-1]
    st.update(n=n, first=first, step=case["step"], seed=st["key"])
    pad = torch.zeros(total, dtype=torch.bool, device=DEV)
    for s, a, b in zip(n, first, first[1:]):
        pad[a + s:b] = True
    # parameters in one buffer, gradients of sizes that differ from tensor to tensor, and
    # moments as if such gradients had been averaged
    w = torch.randn(total, generator=g, device=DEV).mul_(0.05)
    grad = torch.randn(total, generator=g, device=DEV)
    mean = torch.randn(total, generator=g, device=DEV).mul_(0.2)
    square = torch.rand(total, generator=g, device=DEV).add_(0.5)
    for i, (a, b) in enumerate(zip(first, first[1:])):
        size = 10.0 ** (-2 - i % 4)
        grad[a:b].mul_(size)
        mean[a:b].mul_(size)
        square[a:b].mul_(size * size)
    if case["step"] == 0:
        mean.zero_()
        square.zero_()
    for x in (w, grad, mean, square):
        x[pad] = 0.0
    st["grad"] = grad.to(dt)
    st["param"] = w.to(dt)
    del grad
    if dt != torch.float32:
        st["master"] = st["param"].float() + (w - st["param"].float()) * 0.5
    del w
    if case["bits"] == 8:
        half = torch.full((total,), 0x8000, dtype=torch.int32, device=DEV)
        st["mean"], em = _encode(mean, half, False)
        st["square"], es = _encode(square, half, True)
        st["scales"] = torch.stack((em, es))
    else:
        st["mean"], st["square"] = mean, square
    if own:
        from ferrisboost_amd import heads

        cut = lambda x: [x[a:a + s] for a, s in zip(first, n)]  # noqa: E731
        st["params"], st["grads"] = cut(st["param"]), cut(st["grad"])
        opt = heads.AdamW(st["params"], lr=case["lr"], betas=BETAS, eps=EPS, weight_decay=DECAY,
                          bits=case["bits"], seed=st["seed"])
        kept = {"step": st["step"], "mean": st["mean"], "square": st["square"]}
        if case["bits"] == 8:
            kept["scales"] = st["scales"]
        if dt != torch.float32:
            kept["masters"] = cut(st["master"])
        opt.load_state_dict(kept)
        st["optimizer"] = opt
        for k in ("mean", "square", "scales", "master"):
            st.pop(k, None)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    st = {"case": case, "key": (seed * 0x5851F42D4C957F2D + 12345) & (M64 >> 1)}
    if case["kind"] in ("norm", "norm_grad"):
        _prepare_norm(case, g, st)
    elif case["kind"] == "adamw":
        _prepare_adamw(case, g, st)
    else:
        _prepare_experts(case, g, st)
    return st


# --------------------------------------------------------------- plain forms
def _plain_norm(st):
    x, w, b = st["x"], st["w"].float(), st["b"].float()
    n, d = x.shape
    out = torch.empty_like(x)
    step = max(1, CHUNK // d)
    for r in range(0, n, step):
        c = x[r:r + step].float()
        c = c - c.mean(1, keepdim=True)
        c = c * torch.rsqrt(c.square().mean(1, keepdim=True) + NORM_EPS)
        out[r:r + step] = (c * w + b).to(x.dtype)
    return out


def _plain_norm_grad(st):
    x, g, stats, w = st["x"], st["g"], st["stats"], st["w"].float()
    n, d = x.shape
    dx = torch.empty_like(x)
    # over all rows in 64 bits
    dw = torch.zeros(d, dtype=torch.float64, device=DEV)
    db = torch.zeros(d, dtype=torch.float64, device=DEV)
    step = max(1, CHUNK // d)
    for r in range(0, n, step):
        gr, rstd = g[r:r + step].float(), stats[r:r + step, 1:]
        h = (x[r:r + step].float() - stats[r:r + step, :1]) * rstd
        dw += (gr * h).sum(0, dtype=torch.float64)
        db += gr.sum(0, dtype=torch.float64)
        gr = gr * w
        a, c = gr.mean(1, keepdim=True), (gr * h).mean(1, keepdim=True)
        dx[r:r + step] = ((gr - a - h * c) * rstd).to(x.dtype)
    return dx, dw.to(st["w"].dtype), db.to(st["w"].dtype)


def _plain_route(st):
    case = st["case"]
    e = case["experts"]
    ids = st["ids"].reshape(-1).to(torch.int64)
    ids = torch.where((ids >= 0) & (ids < e), ids, e)  # those without an expert come last
    order = torch.sort(ids, stable=True).indices
    row = torch.empty_like(order)
    row[order] = torch.arange(order.numel(), device=DEV)
    place = torch.where(ids < e, row, -1 - row).to(torch.int32).reshape(st["ids"].shape)
    starts = torch.searchsorted(ids[order], torch.arange(e + 1, device=DEV))
    return {"order": order.to(torch.int32), "place": place, "starts": starts.to(torch.int32)}


def _plain_to(x, routes, columns):
    held = torch.arange(routes["order"].numel(), device=DEV) < routes["starts"][-1]
    return x[routes["order"] // columns] * held[:, None].to(x.dtype)


def _plain_from(y, place, weights):
    n, k = place.shape
    out = torch.empty((n, y.shape[1]), dtype=y.dtype, device=DEV)
    step = max(1, CHUNK // (k * y.shape[1]))
    for b in range(0, n, step):
        at = place[b:b + step].long()
        rows = y[at.clamp(min=0)].float() * (at >= 0).unsqueeze(2)
        if weights is not None:
            rows = rows * weights[b:b + step].unsqueeze(2)
        out[b:b + step] = rows.sum(1).to(y.dtype)
    return out


def _plain_experts(st):
    routes = _plain_route(st)
    rows = _plain_to(st["x"], routes, st["case"]["columns"])
    return {**routes, "rows": rows, "out": _plain_from(st["y"], routes["place"], st["weights"])}


def _plain_experts_grad(st):
    y, g, place, weights = st["y"], st["g"], st["routes"]["place"], st["weights"]
    n, k = place.shape
    dy = torch.zeros_like(y)
    dw = torch.empty_like(weights)
    step = max(1, CHUNK // (k * y.shape[1]))
    for b in range(0, n, step):
        at = place[b:b + step].long()
        ok = (at >= 0).unsqueeze(2)
        gr = g[b:b + step].float().unsqueeze(1)
        rows = y[at.clamp(min=0)].float() * ok
        dw[b:b + step] = (rows * gr).sum(2)
        part = gr * (weights[b:b + step].unsqueeze(2) * ok)
        dy[torch.where(at >= 0, at, -1 - at)] = part.to(y.dtype)
    return dy, dw, _plain_from(st["gs"], place, None)


def _srl(x, n):
    """x >> n of the 64 bits as they stand."""
    return (x >> n) & ((1 << (64 - n)) - 1)


def _s64(v):
    return v - (1 << 64) if v >> 63 else v


def _mix_int(z):
    z = ((z ^ (z >> 30)) * MIX1) & M64
    z = ((z ^ (z >> 27)) * MIX2) & M64
    return z ^ (z >> 31)


def _bits(seed, begin, end):
    """32 bits of each of the elements begin..end-1 (begin even): half a 64-bit word each."""
    c = torch.arange(begin >> 1, (end + 1) >> 1, device=DEV, dtype=torch.int64)
    z = (c * _s64(STEP)) ^ _s64(_mix_int((seed & M64) ^ GOLDEN))
    z = (z ^ _srl(z, 30)) * _s64(MIX1)
    z = (z ^ _srl(z, 27)) * _s64(MIX2)
    z = z ^ _srl(z, 31)
    return torch.stack((z & 0xFFFFFFFF, _srl(z, 32)), 1).reshape(-1)[:end - begin]


def _encode(x, r, square):
    """Moments (float32, whole blocks) as 8-bit floats under each block's largest exponent,
    rounded up with the probability of what is cut off (r: 16 bits a cell): a sign, 4 bits of
    exponent and 3 of the mantissa, or for squares 5 and 3. Codes and exponents."""
    top = 30 if square else 14
    bits = x.view(torch.int32) & 0x7FFFFFFF
    field = torch.where(bits < 0x7F800000, bits >> 23, 0).reshape(-1, BLOCK).amax(1)
    power = torch.ldexp(torch.ones((), dtype=torch.float64, device=DEV),
                        (top - field.clamp(min=1)).to(torch.int64))
    y = (x.abs().double().reshape(-1, BLOCK) * power[:, None]).float().reshape(-1)
    code = (y.view(torch.int32) + (r << 4)) >> 20
    if square:
        code = torch.where(x > 0, code.clamp(min=1), code)
    code = torch.where(bits < 0x7F800000, code, 0xFF if square else 0x7F)
    if not square:
        code = code | ((x.view(torch.int32) < 0).to(torch.int32) << 7)
    return code.to(torch.uint8), field.to(torch.uint8)


def _decode(code, field, square):
    """What codes stand for, in 64 bits."""
    top = 30 if square else 14
    c = code.to(torch.int32)
    size = c if square else c & 0x7F
    v = (size << 20).view(torch.float32).double()
    power = torch.ldexp(torch.ones((), dtype=torch.float64, device=DEV),
                        field.to(torch.int64).clamp(min=1) - top)
    v = (v.reshape(-1, BLOCK) * power[:, None]).reshape(-1)
    v = torch.where(size == (0xFF if square else 0x7F), math.nan, v)
    return v if square else torch.where(c >= 0x80, -v, v)


def _plain_adamw(st):
    case = st["case"]
    st["step"] += 1
    t, lr = st["step"], case["lr"]
    (b1, b2), small = BETAS, case["type"] != "float32"
    size, root = lr / (1.0 - b1 ** t), math.sqrt(1.0 - b2 ** t)
    most = CHUNK // BLOCK * BLOCK
    parts = [(i, min(i + most, b)) for a, b in zip(st["first"], st["first"][1:])
             for i in range(a, b, most)]
    for a, b in parts:
        g = st["grad"][a:b].float()
        if case["bits"] == 8:
            s = st["scales"][:, a // BLOCK:b // BLOCK]
            g = g.double()
            m = _decode(st["mean"][a:b], s[0], False) * b1 + g * (1.0 - b1)
            v = _decode(st["square"][a:b], s[1], True) * b2 + g * g * (1.0 - b2)
            m, v = m.float(), v.float()
            r = _bits(st["seed"] + t, a, b)
            st["mean"][a:b], s[0] = _encode(m, (r & 0xFFFF).to(torch.int32), False)
            st["square"][a:b], s[1] = _encode(v, (r >> 16).to(torch.int32), True)
        else:
            m = st["mean"][a:b].mul_(b1).add_(g * (1.0 - b1))
            v = st["square"][a:b].mul_(b2).add_(g * g * (1.0 - b2))
        w = st["master" if small else "param"][a:b]
        w.mul_(1.0 - lr * DECAY).sub_(m / (v.sqrt() / root + EPS) * size)
        if small:
            st["param"][a:b] = w.to(st["param"].dtype)
    if case["bits"] == 8:
        mean, square = (torch.empty(st["first"][-1], device=DEV) for _ in range(2))
        for a, b in parts:
            s = st["scales"][:, a // BLOCK:b // BLOCK]
            mean[a:b] = _decode(st["mean"][a:b], s[0], False).float()
            square[a:b] = _decode(st["square"][a:b], s[1], True).float()
    else:
        mean, square = st["mean"], st["square"]
    return {"param": st["param"], "mean": mean, "square": square}


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        return {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "route": _plain_route,
                "experts": _plain_experts, "experts_grad": _plain_experts_grad,
                "adamw": _plain_adamw}[kind](state)
    from ferrisboost_amd import heads

    if kind == "norm":
        return heads.layer_norm(state["x"], state["w"], state["b"], eps=NORM_EPS)
    if kind == "norm_grad":
        return heads.layer_norm_grad(state["g"], state["x"], state["stats"], state["w"])
    if kind == "adamw":
        state["optimizer"].step(state["grads"])
        mean, square = state["optimizer"].moments()
        return {"param": state["param"], "mean": mean, "square": square}
    if kind == "experts_grad":
        routes = state["routes"]
        dy, dw = heads.from_experts_grad(state["g"], state["y"], routes, state["weights"])
        return dy, dw, heads.from_experts(state["gs"], routes)
    routes = heads.Routes(state["ids"], case["experts"])
    out = {"order": routes.order, "place": routes.place, "starts": routes.starts}
    if kind == "experts":
        out["rows"] = heads.to_experts(state["x"], routes)
        out["out"] = heads.from_experts(state["y"], routes, state["weights"])
    return out


# ------------------------------------------------------------ needed work
def work(case):
    kind, size = case["kind"], TYPES[case["type"]].itemsize
    if kind == "adamw":
        n = sum(_sizes(case)[0])
        # parameter and gradient, the float32 copy of a 16-bit parameter, two moments; those of
        # 8 bits are read once more, as float32 values
        cell = 3 * size + (8 if size == 2 else 0) + (4 + 2 + 8 if case["bits"] == 8 else 16)
        return {"bytes": n * cell, "flops": 14 * n}
    n, d = case["rows"], case["dim"]
    if kind == "norm":
        return {"bytes": 2 * n * d * size, "flops": 8 * n * d}
    if kind == "norm_grad":
        return {"bytes": n * (3 * d * size + 8), "flops": 14 * n * d}
    k = case["columns"]
    ids = n * k * getattr(torch, case["ids"]).itemsize
    if kind == "route":
        return {"bytes": ids + 8 * n * k, "flops": n * k}
    if kind == "experts":
        return {"bytes": ids + 12 * n * k + (2 * n + 2 * n * k) * d * size,
                "flops": 2 * n * k * d}
    return {"bytes": 12 * n * k + (2 * n + 3 * n * k) * d * size, "flops": 4 * n * k * d}


# ------------------------------------------------------- results in 64 bits
def _exact_norm(case, st):
    n, d = case["rows"], case["dim"]
    w, b = st["w"].double(), st["b"].double()
    if case["kind"] == "norm":
        out = torch.empty((n, d), dtype=torch.float64, device=DEV)
    else:
        out = [torch.empty((n, d), dtype=torch.float64, device=DEV)]
        dw, db = torch.zeros_like(w), torch.zeros_like(w)
    step = max(1, CHUNK // (2 * d))
    for r in range(0, n, step):
        x = st["x"][r:r + step].double()
        mean = x.sum(1, keepdim=True) / d
        var = (x - mean).pow(2).sum(1, keepdim=True) / d
        h = (x - mean) / (var + NORM_EPS).sqrt()
        if case["kind"] == "norm":
            out[r:r + step] = torch.addcmul(b, h, w)
            continue
        g = st["g"][r:r + step].double()
        dw += (g * h).sum(0)
        db += g.sum(0)
        # the gradient of sum(g * (h * w + b)) by x, from dh = g * w
        dh = g * w
        dvar = (dh * (x - mean)).sum(1, keepdim=True) * (-0.5) * (var + NORM_EPS).pow(-1.5)
        dc = dh / (var + NORM_EPS).sqrt() + dvar * 2.0 * (x - mean) / d
        out[0][r:r + step] = dc - dc.sum(1, keepdim=True) / d
    return out if case["kind"] == "norm" else (out[0], dw, db)


def _exact_experts(case, st):
    n, k, e, d = case["rows"], case["columns"], case["experts"], case["dim"]
    ids = st["ids"].double().cpu().numpy().reshape(-1)
    known = (ids >= 0) & (ids < e)
    key = np.where(known, ids, e).astype(np.int64)
    order = np.lexsort((np.arange(n * k), key))
    row = np.argsort(order, kind="stable")
    place = np.where(known, row, -1 - row).reshape(n, k)
    counts = np.bincount(key, minlength=e + 1)[:e]
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV)  # noqa: E731
    out = {"order": dev(order.astype(np.int32)), "place": dev(place.astype(np.int32)),
           "starts": dev(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))}
    if case["kind"] == "route":
        return out
    at, ok = dev(row.reshape(n, k)), dev(known.reshape(n, k))

    def back(y, weights):
        sums = torch.zeros((n, d), dtype=torch.float64, device=DEV)
        for j in range(k):
            rows = y[at[:, j]].double().masked_fill_(~ok[:, j:j + 1], 0.0)
            sums += rows if weights is None else rows * weights[:, j:j + 1].double()
        return sums

    if case["kind"] == "experts":
        rows = torch.zeros((n * k, d), dtype=torch.float64, device=DEV)
        for j in range(k):
            rows[at[:, j]] = st["x"].double().masked_fill_(~ok[:, j:j + 1], 0.0)
        return {**out, "rows": rows, "out": back(st["y"], st["weights"])}
    dy = torch.zeros((n * k, d), dtype=torch.float64, device=DEV)
    dw = torch.zeros((n, k), dtype=torch.float64, device=DEV)
    g = st["g"].double()
    for j in range(k):
        dy[at[:, j]] = (g * st["weights"][:, j:j + 1].double()).masked_fill_(~ok[:, j:j + 1], 0.0)
        dots = (st["y"][at[:, j]].double() * g).sum(1)
        dw[:, j] = dots.masked_fill_(~ok[:, j], 0.0)
    return dy, dw, back(st["gs"], None)


def _np_bits(seed, begin, end):
    """_bits() in numpy's unsigned words."""
    key = (seed & M64) ^ GOLDEN
    key = ((key ^ (key >> 30)) * MIX1) & M64
    key = ((key ^ (key >> 27)) * MIX2) & M64
    z = np.arange(begin // 2, (end + 1) // 2, dtype=np.uint64)
    z *= np.uint64(STEP)
    z ^= np.uint64(key ^ (key >> 31))
    z ^= z >> np.uint64(30)
    z *= np.uint64(MIX1)
    z ^= z >> np.uint64(27)
    z *= np.uint64(MIX2)
    z ^= z >> np.uint64(31)
    out = np.empty(2 * z.size, np.uint64)
    out[::2], out[1::2] = z & np.uint64(0xFFFFFFFF), z >> np.uint64(32)
    return out[:end - begin]


def _np_values(code, field, square):
    code = code.astype(np.int64)
    mag = code & (0xFF if square else 0x7F)
    e, f = mag >> 3, mag & 7
    v = np.where(e > 0, np.ldexp(8.0 + f, e - 1), f).astype(np.float64)
    # (field: of the largest cell, whose code's exponent is 30 or 14)
    v = np.ldexp(v, (np.maximum(field.astype(np.int64), 1) - 127 - (29 if square else 13) - 3)
                 .repeat(BLOCK))
    return np.where(code >= 0x80, -v, v) if not square else v


def _np_rounded(x, r, square):
    """Moments as their 8-bit floats stand for them: x between two neighbours of the grid goes
    to the upper one when the part behind the lower and the random one reach 1 together."""
    x = x.astype(np.float32).astype(np.float64)
    mag = np.abs(x).reshape(-1, BLOCK)
    high = np.maximum(np.frexp(mag.max(1))[1] - 1, -126)  # the largest one's exponent
    high[mag.max(1) == 0] = -126
    e = np.maximum(np.frexp(mag)[1] - 1, (high - (29 if square else 13))[:, None])
    q = np.ldexp(mag, 3 - e)
    low = np.floor(q)
    part = np.rint((q - low) * 2.0 ** 20) + 16.0 * r.reshape(-1, BLOCK).astype(np.float64)
    low += part >= 2.0 ** 20
    if square:
        low = np.where((low == 0) & (mag > 0), 1.0, low)
    return np.copysign(np.ldexp(low, e - 3).reshape(-1), x)


def _exact_adamw(case, st):
    total, t = st["first"][-1], case["step"] + 1
    if total > 20_000_000 and case["bits"] == 8:
        return None
    (b1, b2), lr = BETAS, case["lr"]
    g = st["grad"].double()
    if case["bits"] == 8:
        field = st["scales"].cpu().numpy()
        gn = g.cpu().numpy()
        m = b1 * _np_values(st["mean"].cpu().numpy(), field[0], False) + (1.0 - b1) * gn
        v = b2 * _np_values(st["square"].cpu().numpy(), field[1], True) + (1.0 - b2) * gn ** 2
        r = _np_bits(st["seed"] + t, 0, total)
        mean = torch.from_numpy(_np_rounded(m, r & np.uint64(0xFFFF), False)).to(DEV)
        square = torch.from_numpy(_np_rounded(v, r >> np.uint64(16), True)).to(DEV)
        m, v = torch.from_numpy(m).to(DEV), torch.from_numpy(v).to(DEV)
    else:
        mean = m = b1 * st["mean"].double() + (1.0 - b1) * g
        square = v = b2 * st["square"].double() + (1.0 - b2) * g * g
    w = st["param" if case["type"] == "float32" else "master"].double()
    step = (m / (1.0 - b1 ** t)) / ((v / (1.0 - b2 ** t)).sqrt() + EPS)
    return {"param": w - lr * (step + DECAY * w), "mean": mean, "square": square}


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    if case["kind"] in ("norm", "norm_grad"):
        return _exact_norm(case, st)
    return _exact_adamw(case, st) if case["kind"] == "adamw" else _exact_experts(case, st)
