"""Workloads of the heads on a model's outputs: vectors learned for leaves and categorical
codes, dropout while they are learned, and classes drawn from predicted margins.

  embed    rows of a table looked up by id (leaf ids of a model's trees, category codes), each
           column with its own part of the table; as they are or summed over a row's columns
  grad     the gradient of that table
  dropout  elementwise, forward and backward, from (seed, element) alone
  sample   one class a row from logits and given uniform numbers, with temperature, top-k,
           top-p and min-p
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
CHUNK = 1 << 27  # elements of one intermediate of the plain forms
M64 = (1 << 64) - 1
GOLDEN, STEP = 0x9E3779B97F4A7C15, 0xD6E8FEB86659FD93
MIX1, MIX2 = 0xBF58476D1CE4E5B9, 0x94D049BB133111EB
ONE = float(1 << 45)  # the weight of a row's largest logit


# --------------------------------------------------------------------- cases
def _table(name, kind, **kw):
    c = {"name": name, "kind": kind, "rows": 1, "columns": 1, "size": 511, "dim": 64,
         "type": "float32", "ids": "int32", "pooled": True, "scale": 1.0, "drop": 0.0,
         "missing": 0.0, "skew": 0.0}
    c.update(kw)
    return c


def _dropout(name, **kw):
    c = {"name": name, "kind": "dropout", "rows": 1, "dim": 64, "type": "float32", "drop": 0.1}
    c.update(kw)
    return c


def _sample(name, **kw):
    c = {"name": name, "kind": "sample", "rows": 1, "classes": 4, "type": "float32",
         "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "masked": 0.0,
         "spread": 2.0}
    c.update(kw)
    return c


def listed():
    return [
        # One row scored by a service: the leaves of 100 trees of depth 8 summed to one vector.
        _table("embed_row", "embed", rows=1, columns=100),
        # A batch of a head's training: 100k rows, 100 trees of depth 8 (511 nodes a tree), the
        # ids as the device's leaf prediction writes them, one in ten trees of a row left out.
        _table("embed_leaves", "embed", rows=100_000, columns=100, type="bfloat16",
               ids="float32", drop=0.1),
        # Vectors of 20 columns of 500 categories side by side, 2M rows, some codes unseen.
        _table("embed_categories", "embed", rows=2_000_000, columns=20, size=500, dim=8,
               pooled=False, missing=0.05, skew=1.2),
        # A step on a few rows: the table's gradient is mostly zeros.
        _table("grad_rows", "grad", rows=64, columns=100, dim=16),
        # The backward pass of embed_leaves.
        _table("grad_leaves", "grad", rows=100_000, columns=100, type="bfloat16",
               ids="float32", drop=0.1),
        # One column of many tokens, a few of them frequent, and wide vectors.
        _table("grad_tokens", "grad", rows=32_768, columns=1, size=50_000, dim=1024,
               type="bfloat16", ids="int64", pooled=False, scale=32.0, skew=1.1),
        # Dropout of a small batch's vectors, and of a large one's with an odd width.
        _dropout("dropout_rows", rows=64, dim=64),
        _dropout("dropout_batch", rows=100_000, dim=1023, type="bfloat16"),
        # The four classes of the multiclass workload, 500k rows.
        _sample("sample_classes", rows=500_000, classes=4, temperature=0.7),
        # A categorical column of 500 codes drawn for 20k rows, its rare codes left out.
        _sample("sample_codes", rows=20_000, classes=500, top_k=50, top_p=0.9, masked=0.02),
        # One row over a large set of classes, then a batch of them.
        _sample("sample_row", rows=1, classes=50_000, type="bfloat16", temperature=0.8,
                top_p=0.95),
        _sample("sample_wide", rows=256, classes=131_071, type="bfloat16", temperature=0.8,
                top_k=200, top_p=0.95, min_p=0.02),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "grad", "dropout", "sample", "grad", "sample"])
    dtype = rng.choice(sorted(TYPES))
    if kind in ("embed", "grad"):
        columns = rng.choice([1, _log_int(rng, 2, 400)])
        size = _log_int(rng, 2, 60_000) if columns == 1 else _log_int(rng, 2, 1000)
        dim = _log_int(rng, 1, 1024)
        pooled = rng.random() < 0.5
        # ids times width up to the largest listed one's, and the table up to 64M cells
        dim = max(1, min(dim, (64 << 20) // (size * columns)))
        most = min(4_000_000, (320 << 20) // (columns * dim))
        rows = _log_int(rng, 1, max(1, most))
        return _table("", kind, rows=rows, columns=columns, size=size, dim=dim, type=dtype,
                      ids=rng.choice(["int32", "int64", "float32"]), pooled=pooled,
                      scale=rng.choice([1.0, 0.25, math.sqrt(dim)]),
                      drop=rng.choice([0.0, 0.0, 0.1, 0.5]),
                      missing=rng.choice([0.0, 0.05]), skew=rng.choice([0.0, 0.8, 1.2]))
    if kind == "dropout":
        dim = _log_int(rng, 1, 2048)
        return _dropout("", rows=_log_int(rng, 1, 100_000_000 // dim), dim=dim, type=dtype,
                        drop=rng.choice([0.0, 0.05, 0.1, 0.5, 0.9]))
    classes = _log_int(rng, 2, 200_000)
    return _sample("", rows=_log_int(rng, 1, max(1, min(1_000_000, 32_000_000 // classes))),
                   classes=classes, type=dtype, temperature=rng.choice([0.0, 0.5, 0.8, 1.0, 1.5]),
                   top_k=rng.choice([0, 0, 1, _log_int(rng, 1, classes)]),
                   top_p=rng.choice([1.0, 1.0, 0.95, 0.5]), min_p=rng.choice([0.0, 0.0, 0.05]),
                   masked=rng.choice([0.0, 0.1, 0.6]), spread=rng.choice([1.0, 2.0, 4.0]))


# -------------------------------------------------------------------- inputs
def _ids(case, g):
    """Ids of every column: uniform, or frequent ones in a shuffled order (a column's ids
    taken with probability falling as rank^-skew); some are missing (-1)."""
    n, t, size = case["rows"], case["columns"], case["size"]
    if case["skew"]:
        p = torch.arange(1, size + 1, device=DEV, dtype=torch.float64) ** -case["skew"]
        cum = torch.cumsum(p / p.sum(), 0)
        rank = torch.empty((n, t), dtype=torch.int64, device=DEV)
        step = max(1, CHUNK // t)
        for b in range(0, n, step):
            u = torch.rand((min(step, n - b), t), generator=g, device=DEV, dtype=torch.float64)
            rank[b:b + step] = torch.searchsorted(cum, u).clamp_(max=size - 1)
        ids = torch.randperm(size, generator=g, device=DEV)[rank]
    else:
        ids = torch.randint(0, size, (n, t), generator=g, device=DEV)
        if size % 2 == 1 and size > 1:
            # a full binary tree's leaves are some half of its nodes
            leaf = torch.randperm(size, generator=g, device=DEV)[: size // 2 + 1]
            ids = leaf[ids % leaf.numel()]
    if case["missing"]:
        ids[torch.rand((n, t), generator=g, device=DEV) < case["missing"]] = -1
    return ids.to(getattr(torch, case["ids"])).contiguous()


def _seeded(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def prepare(case, seed):
    g = _seeded(seed)
    kind = case["kind"]
    st = {"case": case}
    key = (seed * 0x5851F42D4C957F2D + 12345) & M64
    if kind in ("embed", "grad"):
        dt = TYPES[case["type"]]
        n, t, d = case["rows"], case["columns"], case["dim"]
        st.update(ids=_ids(case, g), key=key, n_tokens=t * case["size"])
        st["first"] = torch.arange(t, device=DEV, dtype=torch.int64) * case["size"]
        if kind == "embed":
            st["table"] = torch.randn((t * case["size"], d), generator=g, device=DEV,
                                      dtype=torch.float32).to(dt)
        else:
            shape = (n, d) if case["pooled"] else (n, t, d)
            st["g"] = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dt)
        if own:
            import ferrisboost_amd as fb

            st["vocabulary"] = fb.heads.Vocabulary([case["size"]] * t, device=DEV)
    elif kind == "dropout":
        shape = (case["rows"], case["dim"])
        dt = TYPES[case["type"]]
        st.update(key=key,
                  x=torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dt),
                  g=torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dt))
    else:
        n, v = case["rows"], case["classes"]
        # margins: a trend over the classes in a shuffled order, noise, and masked classes
        base = -case["spread"] * torch.log(torch.arange(1, v + 1, device=DEV,
                                                        dtype=torch.float32))
        base = base[torch.randperm(v, generator=g, device=DEV)]
        x = torch.randn((n, v), generator=g, device=DEV, dtype=torch.float32)
        x = x.mul_(case["spread"]).add_(0.5 * base)
        if case["masked"]:
            x[torch.rand((n, v), generator=g, device=DEV) < case["masked"]] = -math.inf
        st.update(logits=x.to(TYPES[case["type"]]),
                  u=torch.rand(n, generator=g, device=DEV, dtype=torch.float32))
    return st


# --------------------------------------------------------------- plain forms
def _srl(x, n):
    """x >> n of the 64 bits as they stand."""
    return (x >> n) & ((1 << (64 - n)) - 1)


def _s64(v):
    return v - (1 << 64) if v >> 63 else v


def _mix_int(z):
    z = ((z ^ (z >> 30)) * MIX1) & M64
    z = ((z ^ (z >> 27)) * MIX2) & M64
    return z ^ (z >> 31)


def _kept(key, drop, begin, end):
    """Which of the elements begin..end-1 stay: half a 64-bit word each."""
    c = torch.arange(begin >> 1, (end + 1) >> 1, device=DEV, dtype=torch.int64)
    z = (c * _s64(STEP)) ^ _s64(_mix_int(key ^ GOLDEN))
    z = (z ^ _srl(z, 30)) * _s64(MIX1)
    z = (z ^ _srl(z, 27)) * _s64(MIX2)
    z = z ^ _srl(z, 31)
    bits = torch.stack((z & 0xFFFFFFFF, _srl(z, 32)), 1).reshape(-1)
    bits = bits[begin - ((begin >> 1) << 1):][: end - begin]
    return bits >= int(round(drop * 4294967296.0))


def _tokens(st, b, e):
    """Tokens of rows b..e-1 and which count: ids of their column, not dropped."""
    case = st["case"]
    t = case["columns"]
    ids = st["ids"][b:e].to(torch.int64)
    ok = (ids >= 0) & (ids < case["size"])
    if case["drop"]:
        ok &= _kept(st["key"], case["drop"], b * t, e * t).reshape(e - b, t)
    return (ids + st["first"]) * ok, ok


def _plain_embed(st):
    case = st["case"]
    n, t, d = case["rows"], case["columns"], case["dim"]
    s = case["scale"] / (1.0 - case["drop"])
    shape = (n, d) if case["pooled"] else (n, t, d)
    out = torch.empty(shape, dtype=st["table"].dtype, device=DEV)
    step = max(1, CHUNK // (t * d))
    for b in range(0, n, step):
        e = min(b + step, n)
        tok, ok = _tokens(st, b, e)
        rows = st["table"][tok].float() * ok.unsqueeze(-1)
        if case["pooled"]:
            rows = rows.sum(1)
        out[b:e] = (rows * s).to(out.dtype)
    return out


def _plain_grad(st):
    case = st["case"]
    n, t, d = case["rows"], case["columns"], case["dim"]
    s = case["scale"] / (1.0 - case["drop"])
    # in 64 bits: a frequent id sums a large part of all rows
    acc = torch.zeros((st["n_tokens"], d), dtype=torch.float64, device=DEV)
    step = max(1, CHUNK // (t * d))
    for b in range(0, n, step):
        e = min(b + step, n)
        tok, ok = _tokens(st, b, e)
        g = st["g"][b:e].double()
        if case["pooled"]:
            g = g.unsqueeze(1).expand(e - b, t, d)
        g = g * ok.unsqueeze(-1)
        acc.index_add_(0, tok.reshape(-1), g.reshape(-1, d))
    return (acc * s).to(st["g"].dtype)


def _plain_dropout(st):
    case = st["case"]
    n = case["rows"] * case["dim"]
    s = 1.0 / (1.0 - case["drop"])
    kept = torch.empty(n, dtype=torch.bool, device=DEV)
    for b in range(0, n, CHUNK):
        kept[b:b + CHUNK] = _kept(st["key"], case["drop"], b, min(b + CHUNK, n))
    kept = kept.reshape(case["rows"], case["dim"])
    zero = torch.zeros((), device=DEV)
    return [torch.where(kept, st[k].float() * s, zero).to(st[k].dtype) for k in ("x", "g")]


def _share(part, total):
    """ceil(part * total / 2^31) of whole numbers, part at most 2^31, total below 2^63."""
    hi, lo = total >> 31, total & 0x7FFFFFFF
    return part * hi + ((part * lo + 0x7FFFFFFF) >> 31)


def _plain_sample(st):
    case = st["case"]
    n, v = case["rows"], case["classes"]
    ids = torch.empty(n, dtype=torch.int64, device=DEV)
    logp = torch.empty(n, dtype=torch.float32, device=DEV)
    step = max(1, CHUNK // (4 * v))
    top_p, min_p = (float(np.float32(case[k])) for k in ("top_p", "min_p"))
    temperature = float(np.float32(case["temperature"]))
    for b in range(0, n, step):
        x = st["logits"][b:b + step].double()
        top = x.max(1, keepdim=True).values
        if temperature > 0.0:
            z = (x - top) / temperature
        else:
            z = torch.where(x == top, 0.0, -math.inf)
        w = torch.where(x == -math.inf, 0.0, torch.round(torch.exp(z) * ONE)).to(torch.int64)
        # by falling logit, equal ones by class
        order = torch.sort(x, dim=1, descending=True, stable=True).indices
        k = 1 if temperature <= 0.0 else case["top_k"] or v
        ws = torch.gather(w, 1, order)
        ws[:, k:] = 0
        most = _share(int(top_p * (1 << 31)), ws.sum(1, keepdim=True)).clamp_(min=1)
        before = torch.cumsum(ws, 1) - ws
        ws = ws * ((before < most) & (ws >= min_p * ONE))
        w = torch.zeros_like(w).scatter_(1, order, ws)
        cum = torch.cumsum(w, 1)
        total = cum[:, -1:]
        r = (st["u"][b:b + step].double() * (1 << 31)).to(torch.int64).unsqueeze(1)
        hi, lo = total >> 31, total & 0x7FFFFFFF
        at = r * hi + ((r * lo) >> 31)
        got = torch.searchsorted(cum, at, right=True).clamp_(max=v - 1)
        none = total == 0
        lp = torch.gather(z, 1, got) - torch.log(total.double() / ONE)
        ids[b:b + step] = torch.where(none, -1, got)[:, 0]
        logp[b:b + step] = torch.where(none, -math.inf, lp)[:, 0].float()
    return ids, logp


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        return {"embed": _plain_embed, "grad": _plain_grad, "dropout": _plain_dropout,
                "sample": _plain_sample}[kind](state)
    from ferrisboost_amd import heads

    if kind == "embed":
        return heads.embed(state["table"], state["ids"], state["vocabulary"],
                           scale=case["scale"], pooled=case["pooled"], drop=case["drop"],
                           seed=state["key"])
    if kind == "grad":
        return heads.embed_grad(state["g"], state["ids"], state["vocabulary"],
                                scale=case["scale"], pooled=case["pooled"], drop=case["drop"],
                                seed=state["key"])
    if kind == "dropout":
        return [heads.dropout(state[k], case["drop"], state["key"]) for k in ("x", "g")]
    return heads.sample(state["logits"], state["u"], temperature=case["temperature"],
                        top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"])


# ------------------------------------------------------------ needed work
def work(case):
    kind = case["kind"]
    if kind == "dropout":
        n = case["rows"] * case["dim"]
        return {"bytes": 4 * n * TYPES[case["type"]].itemsize, "flops": 2 * n}
    size = TYPES[case["type"]].itemsize
    if kind == "sample":
        n, v = case["rows"], case["classes"]
        return {"bytes": n * (v * size + 4 + 12), "flops": 4 * n * v}
    n, t, d, v = case["rows"], case["columns"], case["dim"], case["columns"] * case["size"]
    ids = n * t * getattr(torch, case["ids"]).itemsize
    rows = n * d * size if case["pooled"] else n * t * d * size
    table = (v if kind == "grad" else min(v, n * t)) * d * size
    return {"bytes": ids + rows + table, "flops": n * t * d}


# ------------------------------------------------------- results in 64 bits
def _np_kept(key, drop, n):
    """_kept() of elements 0..n-1 in numpy's unsigned words."""
    out = np.empty(n, bool)
    limit = np.uint64(int(round(drop * 2.0 ** 32)))
    base = key ^ GOLDEN
    base = ((base ^ (base >> 30)) * MIX1) & M64
    base = ((base ^ (base >> 27)) * MIX2) & M64
    base ^= base >> 31
    for b in range(0, n, 1 << 22):
        e = min(b + (1 << 22), n)
        z = np.arange(b // 2, (e + 1) // 2, dtype=np.uint64)
        z *= np.uint64(STEP)
        z ^= np.uint64(base)
        z ^= z >> np.uint64(30)
        z *= np.uint64(MIX1)
        z ^= z >> np.uint64(27)
        z *= np.uint64(MIX2)
        z ^= z >> np.uint64(31)
        out[b:e:2] = (z & np.uint64(0xFFFFFFFF)) >= limit
        out[b + 1:e:2] = (z >> np.uint64(32))[: (e - b) // 2] >= limit
    return out


def _exact_table(case, st):
    n, t, d, size = case["rows"], case["columns"], case["dim"], case["size"]
    s = case["scale"] / (1.0 - case["drop"])
    keep = torch.ones((n, t), dtype=torch.bool, device=DEV)
    if case["drop"]:
        keep = torch.from_numpy(_np_kept(st["key"], case["drop"], n * t)).to(DEV).reshape(n, t)
    embed = case["kind"] == "embed"
    shape = (n, d) if case["pooled"] else (n, t, d)
    out = torch.zeros(shape if embed else (t * size, d), dtype=torch.float64, device=DEV)
    for c in range(t):
        ids = st["ids"][:, c].long()
        at = torch.nonzero(keep[:, c] & (ids >= 0) & (ids < size))[:, 0]
        tok = ids[at] + c * size
        for b in range(0, at.numel(), max(1, CHUNK // (4 * d))):
            a, k = at[b:b + max(1, CHUNK // (4 * d))], tok[b:b + max(1, CHUNK // (4 * d))]
            if not embed:
                g = st["g"][a] if case["pooled"] else st["g"][a, c]
                out.index_add_(0, k, g.double())
            elif case["pooled"]:
                out[a] += st["table"][k].double()
            else:
                out[a, c] = st["table"][k].double()
    return out.mul_(s)


def _exact_sample(case, st):
    """Row by row: the classes sorted, filters as prefixes of that order, the draw by class."""
    n, v = case["rows"], case["classes"]
    x = st["logits"].double().cpu().numpy()
    u = st["u"].double().cpu().numpy()
    temp, top_p, min_p = (float(np.float32(case[k])) for k in ("temperature", "top_p", "min_p"))
    ids = np.full(n, -1, np.int64)
    logp = np.full(n, -np.inf)
    step = max(1, (1 << 23) // v)
    for b in range(0, n, step):
        xb = x[b:b + step]
        top = xb.max(1, keepdims=True)
        with np.errstate(invalid="ignore"):
            z = (xb - top) / temp if temp > 0.0 else np.where(xb == top, 0.0, -np.inf)
        z[xb == -np.inf] = -np.inf
        w = np.rint(np.exp(z) * ONE)
        order = np.argsort(-xb, 1, kind="stable")
        ws = np.take_along_axis(w, order, 1).astype(np.uint64)
        k = 1 if temp <= 0.0 else (case["top_k"] or v)
        ws[:, k:] = 0
        after = np.cumsum(ws, 1)
        sums = [int(a) for a in after[:, -1]]
        part = int(top_p * 2 ** 31)
        most = np.array([max(1, -(-part * a // 2 ** 31)) for a in sums], np.uint64)[:, None]
        ws[(after - ws >= most) | (ws.astype(np.float64) < min_p * ONE)] = 0
        kept = np.zeros_like(ws)
        np.put_along_axis(kept, order, ws, 1)
        cum = np.cumsum(kept, 1)
        for i in range(xb.shape[0]):
            total = int(cum[i, -1])
            if not total:
                continue
            at = int(u[b + i] * 2 ** 31) * total >> 31
            j = int(np.searchsorted(cum[i], np.uint64(at), side="right"))
            ids[b + i] = j
            logp[b + i] = z[i, j] - math.log(total / ONE)
    return torch.from_numpy(ids).to(DEV), torch.from_numpy(logp).to(DEV)


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "dropout":
        n = case["rows"] * case["dim"]
        keep = torch.from_numpy(_np_kept(st["key"], case["drop"], n)).to(DEV)
        keep = keep.reshape(case["rows"], case["dim"])
        return [(st[k].double() / (1.0 - case["drop"])).masked_fill_(~keep, 0.0)
                for k in ("x", "g")]
    if kind == "sample":
        return _exact_sample(case, st)
    return _exact_table(case, st)
