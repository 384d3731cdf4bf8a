"""Heads on a model's outputs, for programs that go on in torch.

A model answers with leaf ids (predict(pred_leaf=True), FBH_PREDICT_LEAF on the
device) and class margins, and its rows hold categorical codes. What follows them:

  embed / embed_grad  vectors learned for ids: rows of a table looked up by id, as they
                      are or summed over a row's columns, and the table's gradient
  dropout             while they are learned, from (seed, element) alone: no mask
  sample              classes drawn from margins (Model.sample does it on host arrays)
  layer_norm          a row's cells to mean 0 and variance 1, with its gradients
  Routes, to_experts, from_experts
                      rows by their ids (a tree's leaves, say, each with a model of its own)
                      and back, weighted, with the gradients
  AdamW               the step of all parameters at once, moments in 32 bits or in 8

    model = fb.train({"objective": "multi:softprob", "num_class": 4, ...}, X, label=y)
    leaves = torch.from_numpy(model.predict(X, pred_leaf=True)).cuda()
    voc = model.leaf_vocabulary()
    table = torch.zeros(voc.n_tokens, 64, device="cuda", requires_grad=True)
    h = fb.heads.embed(table, leaves, voc, pooled=True, drop=0.1, seed=step)
    h = fb.heads.dropout(h, 0.1, seed=step + 1)
    h = fb.heads.layer_norm(h, gain, bias)
    loss = torch.nn.functional.cross_entropy(h @ W, labels)
    loss.backward()
    optimizer.step()                           # fb.heads.AdamW([table, gain, bias, W], lr=1e-3)
    classes, log_probs = fb.heads.sample(h @ W, torch.rand(len(h), device="cuda"), top_p=0.9)

Tensors are torch tensors on one gfx950 device; torch must be imported before the
package's first call, so that both share one HIP runtime. Kernels are hand-written HIP
behind the C ABI of include/fbhip.h, enqueued on torch's current stream of the tensors'
device; nothing waits, results are the same in every call, and all of it can be captured
into a graph. A tensor that is not contiguous is copied first. embed, dropout, layer_norm,
to_experts and from_experts take part in autograd, in reverse mode; tensors with a tangent of
forward mode are refused. What embed_grad, layer_norm_grad, from_experts_grad and sample give
has no gradient. Bad arguments are ValueErrors, device failures RuntimeErrors.
"""

from __future__ import annotations

import functools
import operator
import struct
from collections.abc import Mapping

import numpy as np

from . import _native as N

__all__ = ["Vocabulary", "embed", "embed_grad", "dropout", "sample", "layer_norm",
           "layer_norm_grad", "Routes", "to_experts", "from_experts", "from_experts_grad", "AdamW"]

_torch = None
_L = None
_CELLS: dict = {}
_IDS: dict = {}
_raw_stream = None
_forward_ad = None
_Tensor = _strided = None
# fbh_embed and fbh_sample_options (include/fbhip.h), packed in one call: a small
# operation's time is its host time.
_EMBED = struct.Struct("QIIIIIIPPdQfI")
_OPTIONS = struct.Struct("PPPPfiff")
_NORM = struct.Struct("QIIIf")                 # fbh_norm
_ADAMW = struct.Struct("IfdddPQQPPPP")         # fbh_adamw
_MOST = float(np.finfo(np.float32).max)
_dtype_of, _shape_of = operator.attrgetter("dtype"), operator.attrgetter("shape")


def _need_torch():
    """torch, once it is known to share this package's HIP runtime."""
    global _torch, _L, _raw_stream, _forward_ad, _Tensor, _strided
    if _torch is not None:
        return _torch
    import torch

    N.hip()
    with open("/proc/self/maps") as f:
        runtimes = {line.split()[-1] for line in f if "libamdhip64.so" in line}
    if len(runtimes) > 1:
        raise N.BackendError(
            "torch was imported after the package's first call and has brought a HIP runtime of "
            "its own; import torch first")
    _CELLS.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    _IDS.update({torch.int32: 0, torch.int64: 1, torch.float32: 2})
    # the current stream's handle, as torch.cuda.current_stream() wraps it
    _raw_stream = torch._C._cuda_getCurrentRawStream
    _forward_ad = torch.autograd.forward_ad
    _Tensor, _strided = torch.Tensor, torch.strided
    _L = N.hip()
    _torch = torch
    return torch


def _no_tangent(x, what: str):
    if _forward_ad._current_level >= 0 and _forward_ad.unpack_dual(x).tangent is not None:
        raise ValueError(f"{what} has a tangent: forward-mode derivatives are not available")


def _dense(x, what: str):
    if x.layout is not _strided or x.is_nested:
        raise ValueError(f"{what} must be dense, got "
                         f"{'a nested tensor' if x.is_nested else x.layout}")


def _device_tensor(x, what: str, on: int | None = None):
    """x, contiguous, after checking that it is a dense tensor on a GPU, that of `on` where the
    call has one already. (Each look at a tensor takes some 40 ns of a small call's 7 us.)"""
    if not isinstance(x, _Tensor):
        raise ValueError(f"{what} must be a torch tensor, got {type(x).__name__}")
    if _forward_ad._current_level >= 0:
        _no_tangent(x, what)
    if x.layout is not _strided or x.is_nested:
        _dense(x, what)
    dev = x.get_device()
    if dev != on:
        if dev < 0:
            raise ValueError(f"{what} must be on a GPU, it is on {x.device}")
        if on is not None:
            raise ValueError(f"{what} is on {x.device}, the call's other tensors on cuda:{on}")
    return x if x.is_contiguous() else x.contiguous()


def _cells(x, what: str) -> int:
    code = _CELLS.get(x.dtype)
    if code is None:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, got {x.dtype}")
    return code


def _beside(x, other, what: str):
    if x.get_device() != other.get_device():
        raise ValueError(f"{what} is on {x.device}, the call's other tensors on {other.device}")
    return x


def _whole(v, what: str) -> int:
    if type(v) is int:
        return v
    try:
        if _torch is not None and isinstance(v, _torch.Tensor) and v.numel() != 1:
            raise ValueError
        whole = int(v)
        if whole != v and not isinstance(v, str):
            raise ValueError
        return whole
    except (OverflowError, TypeError, ValueError):
        raise ValueError(f"{what} must be a whole number, got {v!r}") from None


def _number(v, what: str) -> float:
    if type(v) is float:
        return v
    try:
        if _torch is not None and isinstance(v, _torch.Tensor) and v.numel() != 1:
            raise ValueError
        return float(v)
    except (OverflowError, TypeError, ValueError):
        raise ValueError(f"{what} must be a number, got {v!r}") from None


def _list(v, what: str) -> list:
    try:
        return list(v)
    except TypeError:
        raise ValueError(f"{what} must be a list, got {type(v).__name__}") from None


def _seed(seed) -> int:
    seed = _whole(seed, "seed")
    if not 0 <= seed < 1 << 64:
        raise ValueError(f"seed must be in 0..=2^64 - 1, got {seed}")
    return seed


def _drop(drop) -> float:
    drop = _number(drop, "drop")
    if not 0.0 <= drop < 1.0:
        raise ValueError(f"drop must be in [0, 1), got {drop}")
    return drop


def _scale(scale) -> float:
    scale = _number(scale, "scale")
    if not abs(scale) <= _MOST:
        raise ValueError(f"scale must be a finite float32, got {scale}")
    return scale


class _Kept:
    """Device memory that an object keeps for its calls: copies of it have been used on no
    stream yet."""

    def _tensors(self):
        raise NotImplementedError

    def _used_on(self, stream: int):
        """Keeps that memory from the allocator until the work now on this stream, the current
        one, has passed, also when the object is dropped before."""
        if stream not in self._streams:
            for x in self._tensors():
                x.record_stream(_torch.cuda.current_stream(x.device))
            self._streams.add(stream)

    def __setstate__(self, state):
        self.__dict__.update(state, _streams=set())


class Vocabulary(_Kept):
    """The table rows of several columns' ids: column t's ids 0 .. sizes[t] - 1 are rows
    first[t] .. first[t] + sizes[t] - 1 of a table of n_tokens rows (a model's trees:
    Model.leaf_vocabulary(); categorical columns: their numbers of codes). It may be copied,
    stored and used on any stream of its device; a captured graph reads it at every replay,
    so it has to live as long as the graph does."""

    def __init__(self, sizes, device="cuda:0"):
        torch = _need_torch()
        sizes = np.asarray(sizes)
        if sizes.ndim != 1 or sizes.size == 0 or sizes.dtype.kind not in "iu":
            raise ValueError("sizes must be a list of whole numbers, one for each column")
        if sizes.size > 32768:
            raise ValueError(f"at most 32768 columns, got {sizes.size}")
        if (sizes < 0).any():
            raise ValueError("sizes must not be negative")
        if (sizes >= 1 << 31).any():  # (and their sum is below 2^46)
            raise ValueError("a column has at most 2^31 - 1 ids")
        first = np.concatenate([[0], np.cumsum(sizes, dtype=np.int64)])
        if not 1 <= first[-1] < 1 << 31:
            raise ValueError(f"a table has 1 to 2^31 - 1 rows, these columns {first[-1]}")
        self.sizes = sizes.astype(np.int64)
        self.n_tokens = int(first[-1])
        self.n_columns = int(sizes.size)
        self.most_ids = int(sizes.max())
        self.first = torch.from_numpy(first.astype(np.int32)).to(device)
        if self.first.device.type != "cuda":
            raise ValueError(f"device must be a GPU, got {device!r}")
        self._streams = set()

    def _tensors(self):
        return (self.first,)

    def __repr__(self):
        return (f"Vocabulary({self.n_columns} columns, {self.n_tokens} tokens, "
                f"{self.first.device})")


def _positions(ids, vocabulary, pooled: bool, n_tokens: int, dim: int, cells: int, scale: float,
               drop: float, seed: int):
    """The call's fbh_embed (None without columns), and the leading shape of its vectors."""
    code = _IDS.get(ids.dtype)
    if code is None:
        raise ValueError(f"ids must be int32, int64 or float32, got {ids.dtype}")
    shape = tuple(ids.shape)
    if pooled or vocabulary is not None:
        if not shape:
            raise ValueError("ids must have a last axis of columns")
        columns = shape[-1]
        if vocabulary is not None:
            if columns != vocabulary.n_columns:
                raise ValueError(f"ids have {columns} columns, the vocabulary "
                                 f"{vocabulary.n_columns}")
            _beside(vocabulary.first, ids, "the vocabulary")
        n_rows = 1
        for s in shape[:-1]:
            n_rows *= s
    else:
        n_rows, columns = ids.numel(), 1
    if max(columns, dim, n_tokens) >> 32:
        raise ValueError(f"{columns} columns, {n_tokens} table rows and {dim} cells: all must be "
                         "below 2^32")
    # (the address that the tensor has now: a copied or unpickled vocabulary has one of its own)
    first, most = (0, 0) if vocabulary is None else (vocabulary.first.data_ptr(),
                                                     vocabulary.most_ids)
    # (a call without columns or positions launches nothing)
    e = _EMBED.pack(n_rows, columns, dim, n_tokens, code, cells, pooled, ids.data_ptr(), first,
                    drop, seed, scale, most) if columns else None
    return e, shape[:-1] if pooled else shape


def _embed(table, ids, vocabulary, scale, pooled, drop, seed):
    e, lead = _positions(ids, vocabulary, pooled, table.shape[0], table.shape[1],
                         _cells(table, "table"), scale, drop, seed)
    out = table.new_empty(lead + (table.shape[1],))
    if e is None:
        return out.zero_()
    dev = table.get_device()
    stream = _raw_stream(dev)
    if vocabulary is not None:
        vocabulary._used_on(stream)
    rc = _L.fbh_embed_rows(dev, e, table.data_ptr(), out.data_ptr(), stream)
    if rc:
        N.check_hip(rc)
    return out


@functools.lru_cache(maxsize=None)
def _functions():
    torch = _torch

    class Embed(torch.autograd.Function):
        @staticmethod
        def forward(ctx, table, ids, vocabulary, scale, pooled, drop, seed):
            ctx.save_for_backward(ids)
            ctx.rest = (vocabulary if vocabulary is not None else table.shape[0], scale, pooled,
                        drop, seed)
            return _embed(table, ids, vocabulary, scale, pooled, drop, seed)

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad):
            tokens, scale, pooled, drop, seed = ctx.rest
            return (embed_grad(grad, ctx.saved_tensors[0], tokens, scale=scale, pooled=pooled,
                               drop=drop, seed=seed),) + (None,) * 6

    class Dropout(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, drop, seed, first):
            ctx.rest = (drop, seed, first)
            return _dropout(x, drop, seed, first)

        @staticmethod
        def backward(ctx, grad):
            return (dropout(grad, *ctx.rest),) + (None,) * 3

    class LayerNorm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, bias, a):
            out, stats = _layer_norm(a, x, weight, bias, True)
            ctx.save_for_backward(x, stats, weight)
            ctx.a = a
            ctx.mark_non_differentiable(stats)
            return out, stats

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad, _):
            x, stats, weight = ctx.saved_tensors
            return _layer_norm_grad(ctx.a, _device_tensor(grad, "grad"), x, stats, weight,
                                    ctx.needs_input_grad[:3]) + (None,)

    class ToExperts(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, routes, place, *size):
            ctx.routes, ctx.size = routes, size
            ctx.save_for_backward(place)
            return _to_experts(x, routes, place, *size)

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad):
            (place,) = ctx.saved_tensors
            dx = _from_experts(_device_tensor(grad, "grad"), ctx.routes, place, None, *ctx.size)
            return dx, None, None, None, None

    class FromExperts(torch.autograd.Function):
        @staticmethod
        def forward(ctx, y, weights, routes, place, *size):
            ctx.routes, ctx.size = routes, size
            ctx.save_for_backward(y if weights is not None and weights.requires_grad else None,
                                  weights, place)
            return _from_experts(y, routes, place, weights, *size)

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad):
            y, weights, place = ctx.saved_tensors
            return _from_experts_grad(_device_tensor(grad, "grad"), y, ctx.routes, place, weights,
                                      *ctx.needs_input_grad[:2], *ctx.size) + (None,) * 4

    return Embed, Dropout, LayerNorm, ToExperts, FromExperts


def embed(table, ids, vocabulary: Vocabulary | None = None, *, scale: float = 1.0,
          pooled: bool = False, drop: float = 0.0, seed: int = 0):
    """Rows of `table` (n_tokens, dim) by id, times `scale`: (*ids.shape, dim), or with
    pooled=True summed over the last axis of ids, in float32 and rounded once.

    ids are int32, int64, or float32 as predict(pred_leaf=True) gives leaf ids. With a
    vocabulary the last axis of ids are its columns, each with its own part of the table;
    without, every id is a table row. An id outside its column (-1 for a missing or unseen
    code, say) gives zeros. drop > 0 leaves out each id of the call with that probability,
    drawn from `seed` and the id's place in `ids`, and scales the others by 1 / (1 - drop):
    whole trees, or whole columns, of a row."""
    torch = _need_torch()
    table = _device_tensor(table, "table")
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError(f"table must be (tokens, cells), got shape {tuple(table.shape)}")
    if vocabulary is not None and not isinstance(vocabulary, Vocabulary):
        raise ValueError(f"vocabulary must be a Vocabulary, got {type(vocabulary).__name__}")
    if vocabulary is not None and vocabulary.n_tokens != table.shape[0]:
        raise ValueError(f"table has {table.shape[0]} rows, the vocabulary "
                         f"{vocabulary.n_tokens} tokens")
    ids = _device_tensor(ids, "ids", table.get_device())
    args = (table, ids, vocabulary, _scale(scale), bool(pooled), _drop(drop), _seed(seed))
    if table.requires_grad and torch.is_grad_enabled():
        return _functions()[0].apply(*args)
    return _embed(*args)


def embed_grad(grad, ids, tokens, *, scale: float = 1.0, pooled: bool = False,
               drop: float = 0.0, seed: int = 0):
    """The gradient of embed()'s table, (n_tokens, dim) in grad's type: `grad` is the
    gradient of embed()'s output, `tokens` its vocabulary or, without one, the number of
    table rows, and the rest embed()'s arguments. Sums are taken in a fixed order (the
    positions sorted by token), parts of at most 3072 in float32 and the parts in float64,
    and rounded once. (embed() calls this in
    backward(); a captured training step can call it by itself.)"""
    _need_torch()
    grad = _device_tensor(grad, "grad")
    ids = _device_tensor(ids, "ids", grad.get_device())
    vocabulary = tokens if isinstance(tokens, Vocabulary) else None
    n_tokens = vocabulary.n_tokens if vocabulary is not None else _whole(
        tokens, "tokens, other than a vocabulary,")
    if not 1 <= n_tokens < 1 << 31:
        raise ValueError(f"a table has 1 to 2^31 - 1 rows, got {n_tokens}")
    if grad.dim() < 1 or grad.shape[-1] < 1:
        raise ValueError(f"grad must have a last axis of cells, got shape {tuple(grad.shape)}")
    e, lead = _positions(ids, vocabulary, bool(pooled), n_tokens, grad.shape[-1],
                         _cells(grad, "grad"), _scale(scale), _drop(drop), _seed(seed))
    if tuple(grad.shape[:-1]) != lead:
        raise ValueError(f"grad has shape {tuple(grad.shape)}, expected {lead} vectors")
    out = grad.new_empty((n_tokens, grad.shape[-1]))
    if e is None:
        return out.zero_()
    dev = grad.get_device()
    size = _L.fbh_embed_grad_bytes(e)
    work = grad.new_empty(size, dtype=_torch.uint8)
    stream = _raw_stream(dev)
    if vocabulary is not None:
        vocabulary._used_on(stream)
    rc = _L.fbh_embed_grad(dev, e, grad.data_ptr(), out.data_ptr(), work.data_ptr(), size, stream)
    if rc:
        N.check_hip(rc)
    return out


def _dropout(x, drop, seed, first):
    out = _torch.empty_like(x)
    dev = x.get_device()
    rc = _L.fbh_dropout(dev, x.data_ptr(), out.data_ptr(), x.numel(), _cells(x, "x"), drop, seed,
                        first, _raw_stream(dev))
    if rc:
        N.check_hip(rc)
    return out


def dropout(x, drop: float, seed: int, first: int = 0):
    """x / (1 - drop) where an element stays, 0 where it is dropped (with probability
    `drop`), whatever it holds. An element's fate depends on `seed` and its number alone
    (counted in row-major order from `first`), so the gradient of a call, which
    backward() takes, is dropout() of the output's gradient with the same arguments, and
    nothing is stored for it. Use another seed for another layer or step."""
    torch = _need_torch()
    x = _device_tensor(x, "x")
    _cells(x, "x")
    first = _whole(first, "first")
    if not 0 <= first < 1 << 63:
        raise ValueError(f"first must be in 0..=2^63 - 1, got {first}")
    args = (x, _drop(drop), _seed(seed), first)
    if x.requires_grad and torch.is_grad_enabled():
        return _functions()[1].apply(*args)
    return _dropout(*args)


def _option(value, what: str, lead, like, dtype):
    """The tensor of one value a row that `value` is, or None."""
    if not isinstance(value, _Tensor) or value.dim() == 0:
        return None
    v = _device_tensor(value, what, like.get_device())
    if tuple(v.shape) != lead:
        raise ValueError(f"{what} must have shape {lead}, got {tuple(v.shape)}")
    if v.dtype != dtype:
        raise ValueError(f"{what} must be {dtype}, got {v.dtype}")
    return v


@functools.lru_cache(maxsize=256, typed=True)
def _packed_numbers(temperature, top_k, top_p, min_p) -> bytes:
    return _OPTIONS.pack(0, 0, 0, 0, *check_options(temperature, top_k, top_p, min_p))


def check_options(temperature, top_k, top_p, min_p) -> tuple[float, int, float, float]:
    """The options of sample() as one set of numbers."""
    return (_temperature(temperature), _top_k(top_k), _share("top_p", top_p),
            _share("min_p", min_p))


def _temperature(v) -> float:
    v = _number(v, "temperature")
    if not 0.0 <= v <= _MOST:
        raise ValueError(f"temperature must be a finite float32, not negative, got {v}")
    return v


def _top_k(v) -> int:
    k = _whole(v, "top_k")
    if isinstance(v, bool) or k != v or k < 0:
        raise ValueError(f"top_k must be a whole number, 0 (all) or more, got {v!r}")
    return min(k, 0x7FFFFFFF)


def _share(what: str, v) -> float:
    v = _number(v, what)
    if not 0.0 <= v <= 1.0:
        raise ValueError(f"{what} must be in [0, 1], got {v}")
    return v


def check_uniforms(uniforms, n: int) -> np.ndarray:
    """Uniform numbers of n rows as float32: what they were given as has to be in [0, 1), and
    those that float32 rounds to 1 are the largest number below it."""
    u = np.asarray(uniforms)
    if u.dtype.kind != "f":
        u = u.astype(np.float64)
    if u.shape != (n,):
        raise ValueError(f"uniforms must have one value for each of {n} rows, got shape "
                         f"{u.shape}")
    if not ((u >= 0.0) & (u < 1.0)).all():
        raise ValueError("uniforms must be in [0, 1)")
    return np.minimum(u.astype(np.float32), np.float32(1.0 - 2.0 ** -24))


def sample(logits, uniforms, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One class for every row of `logits` (..., classes), from a uniform float32 number
    in [0, 1) a row: (classes int64, log_probs float32), each of shape (...).

    Weights are exp(logit / temperature). Ordered by falling logit (equal ones by class),
    the first top_k classes stay (0: all), of those the shortest prefix that holds top_p
    of their weight, and of those the ones with at least min_p times the largest weight.
    The class is the first, by number, at which the running share of what stays exceeds
    the row's uniform number; log_probs is the logarithm of its own share. temperature 0
    takes the largest logit. Each option is a number, or a tensor of one a row (float32;
    top_k int32), whose values the device reads: there 0 or less, and NaN, are
    temperature 0, no top_k, top_p 0 (NaN: 1) and min_p 0, and at an infinite temperature
    all classes weigh the same.

    Logits of -inf or NaN are masked; a row with no others gets class -1 and -inf. At most
    262144 classes. Weights are held as whole numbers of 2^-45 of the largest one, so the
    drawn classes are the same wherever and however often they are drawn."""
    torch = _need_torch()
    logits = _device_tensor(logits, "logits")
    cells = _cells(logits, "logits")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= 262144:
        raise ValueError(f"logits must be (..., 1 to 262144 classes), got shape "
                         f"{tuple(logits.shape)}")
    lead = tuple(logits.shape[:-1])
    uniforms = _device_tensor(uniforms, "uniforms", logits.get_device())
    if uniforms.dtype != torch.float32 or tuple(uniforms.shape) != lead:
        raise ValueError(f"uniforms must be float32 of shape {lead}, got {uniforms.dtype} of "
                         f"{tuple(uniforms.shape)}")
    f32 = torch.float32
    given = (temperature, top_k, top_p, min_p)
    if all(type(v) is float or type(v) is int for v in given):
        o = _packed_numbers(*given)
    else:
        rows = [_option(v, w, lead, logits, torch.int32 if w == "top_k" else f32)
                for v, w in zip(given, ("temperature", "top_k", "top_p", "min_p"))]
        numbers = check_options(*(off if r is not None else v
                                  for v, r, off in zip(given, rows, (1.0, 0, 1.0, 0.0))))
        o = _OPTIONS.pack(*(0 if r is None else r.data_ptr() for r in rows), *numbers)
    classes = logits.new_empty(lead, dtype=torch.int64)
    log_probs = logits.new_empty(lead, dtype=f32)
    dev, n, v = logits.get_device(), classes.numel(), logits.shape[-1]
    size = _L.fbh_sample_bytes(n, v) if v > 1024 else 0
    work = logits.new_empty(size, dtype=torch.uint8) if size else None
    rc = _L.fbh_sample_classes(dev, logits.data_ptr(), n, v, cells, uniforms.data_ptr(), o,
                               classes.data_ptr(), log_probs.data_ptr(),
                               work.data_ptr() if size else None, size, _raw_stream(dev))
    if rc:
        N.check_hip(rc)
    return classes, log_probs


# ------------------------------------------------------------------- layer norm
def _eps(eps) -> float:
    eps = _number(eps, "eps")
    if not 2.0 ** -126 <= eps <= _MOST:
        raise ValueError(f"eps must be a positive normal float32, got {eps}")
    return eps


def _norm_of(x, weight, eps: float) -> bytes:
    """The call's fbh_norm, after checking x and weight."""
    shape = x.shape
    dim = shape[-1] if shape else 0
    if not 1 <= dim <= 32768:
        raise ValueError(f"x must be (..., 1 to 32768 cells), got shape {tuple(shape)}")
    kind = 0
    if weight is not None:
        if weight.shape != (dim,):
            raise ValueError(f"weight must have shape ({dim},), got {tuple(weight.shape)}")
        kind = _cells(weight, "weight")
    return _NORM.pack(x.numel() // dim, dim, _cells(x, "x"), kind, eps)


def _layer_norm(a: bytes, x, weight, bias, stats: bool):
    out = _torch.empty_like(x)
    kept = x.new_empty(x.shape[:-1] + (2,), dtype=_torch.float32) if stats else None
    dev = x.get_device()
    rc = _L.fbh_layer_norm(dev, a, x.data_ptr(), 0 if weight is None else weight.data_ptr(),
                           0 if bias is None else bias.data_ptr(), out.data_ptr(),
                           kept.data_ptr() if stats else 0, _raw_stream(dev))
    if rc:
        N.check_hip(rc)
    return out, kept


def layer_norm(x, weight=None, bias=None, *, eps: float = 1e-5, stats: bool = False):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last axis of `x` (up to
    32768 cells), computed in float32 and rounded once. weight and bias are of x's type or any
    other of the three, both of the same; bias needs a weight. With stats=True also what
    layer_norm_grad() takes: each row's mean and 1 / sqrt(variance + eps), (..., 2) float32."""
    torch = _need_torch()
    x = _device_tensor(x, "x")
    dev = x.get_device()
    if weight is not None:
        weight = _device_tensor(weight, "weight", dev)
    a = _norm_of(x, weight, _eps(eps))
    if bias is not None:
        if weight is None:
            raise ValueError("a bias needs a weight")
        bias = _device_tensor(bias, "bias", dev)
        if bias.dtype != weight.dtype or bias.shape != weight.shape:
            raise ValueError(f"bias is {bias.dtype} of {tuple(bias.shape)}, weight "
                             f"{weight.dtype} of {tuple(weight.shape)}")
    if torch.is_grad_enabled() and (x.requires_grad or
                                    (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        out = _functions()[2].apply(x, weight, bias, a)
    else:
        out = _layer_norm(a, x, weight, bias, stats)
    return out if stats else out[0]


def _layer_norm_grad(a: bytes, grad, x, stats, weight, wanted):
    dx = _torch.empty_like(x) if wanted[0] else None
    dw = _torch.empty_like(weight) if wanted[1] else None
    db = _torch.empty_like(weight) if wanted[2] else None
    size = _L.fbh_layer_norm_grad_bytes(a) if wanted[1] or wanted[2] else 0
    work = grad.new_empty(size, dtype=_torch.uint8) if size else None
    at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    dev = x.get_device()
    rc = _L.fbh_layer_norm_grad(dev, a, grad.data_ptr(), x.data_ptr(), stats.data_ptr(),
                                at(weight), at(dx), at(dw), at(db), at(work), size,
                                _raw_stream(dev))
    if rc:
        N.check_hip(rc)
    return dx, dw, db


def layer_norm_grad(grad, x, stats, weight=None):
    """The gradients of layer_norm()'s x, weight and bias for `grad`, that of its output:
    (dx, dweight, dbias), the last two in weight's type and None without one. x, weight and
    `stats` are those of the call layer_norm(..., stats=True). Sums over rows are taken in a
    fixed order, a workgroup's in float32 (at most 1024 rows one after the other) and theirs in
    float64, and rounded once.
    (layer_norm() does this in backward(); a captured training step can call it by itself.)"""
    torch = _need_torch()
    x = _device_tensor(x, "x")
    dev = x.get_device()
    grad = _device_tensor(grad, "grad", dev)
    stats = _device_tensor(stats, "stats", dev)
    if weight is not None:
        weight = _device_tensor(weight, "weight", dev)
    a = _norm_of(x, weight, 1.0)
    if grad.shape != x.shape or grad.dtype != x.dtype:
        raise ValueError(f"grad is {grad.dtype} of {tuple(grad.shape)}, x {x.dtype} of "
                         f"{tuple(x.shape)}")
    if stats.dtype != torch.float32 or stats.shape != x.shape[:-1] + (2,):
        raise ValueError(f"stats must be float32 of {tuple(x.shape[:-1]) + (2,)}, got "
                         f"{stats.dtype} of {tuple(stats.shape)}")
    both = weight is not None
    return _layer_norm_grad(a, grad, x, stats, weight, (True, both, both))


# ------------------------------------------------------------------- experts
class Routes(_Kept):
    """The positions of an id matrix `ids` (..., columns) in the order of their ids, each id
    from 0 to n_experts - 1 an expert (at most 1024): a tree's leaves, say, or a router's
    choices. An id that is anything else (-1) has no expert; ids are int32, int64, or float32
    as predict(pred_leaf=True) gives leaf ids. All columns have the same experts: for leaves of
    several trees add each tree's first token, Vocabulary.first, to its column.

    order   positions (row * columns + column) by expert, equal ones in their order, those
            without an expert behind all others; int32
    place   the row in that order of every position, of ids' shape, or -1 - row of one without
            an expert; int32
    starts  expert e's rows are starts[e] .. starts[e + 1] - 1; int32, n_experts + 1 values

    It is used with to_experts() and from_experts(), on any stream of its device that has
    waited for the one that made it."""

    def __init__(self, ids, n_experts: int):
        torch = _need_torch()
        ids = _device_tensor(ids, "ids")
        code = _IDS.get(ids.dtype)
        if code is None:
            raise ValueError(f"ids must be int32, int64 or float32, got {ids.dtype}")
        if ids.dim() < 1:
            raise ValueError("ids must have a last axis of columns")
        n_experts = _whole(n_experts, "n_experts")
        if not 1 <= n_experts <= 1024:
            raise ValueError(f"n_experts must be in 1..=1024, got {n_experts}")
        n = ids.numel()
        if n >> 31:
            raise ValueError(f"at most 2^31 - 1 positions, got {n}")
        self.n_experts = n_experts
        self.order = ids.new_empty(n, dtype=torch.int32)
        self.place = ids.new_empty(ids.shape, dtype=torch.int32)
        self.starts = ids.new_empty(n_experts + 1, dtype=torch.int32)
        dev = ids.get_device()
        size = _L.fbh_route_bytes(n, n_experts)
        work = ids.new_empty(size, dtype=torch.uint8) if size else None
        stream = _raw_stream(dev)
        rc = _L.fbh_route(dev, ids.data_ptr(), code, n, n_experts, self.order.data_ptr(),
                          self.place.data_ptr(), self.starts.data_ptr(),
                          work.data_ptr() if size else 0, size, stream)
        if rc:
            N.check_hip(rc)
        self._streams = {stream}

    def _tensors(self):
        return self.order, self.place, self.starts

    def __repr__(self):
        return f"Routes({tuple(self.place.shape)} ids, {self.n_experts} experts)"


def _routes(routes, like):
    if not isinstance(routes, Routes):
        raise ValueError(f"routes must be Routes, got {type(routes).__name__}")
    return _beside(routes.place, like, "the routes")


def _rows_of(x, what: str, lead):
    """The cells of a row of x, whose leading shape is `lead`: 1 to 32768."""
    shape = x.shape
    dim = shape[-1] if shape else 0
    if not 1 <= dim <= 32768 or shape[:-1] != lead:
        raise ValueError(f"{what} must have shape {tuple(lead)} and a last axis of 1 to 32768 "
                         f"cells, got {tuple(shape)}")
    return dim


def _to_experts(x, routes, place, dim: int, cells: int):
    n = place.numel()
    out = x.new_empty((n, dim))
    if n:
        dev = x.get_device()
        stream = _raw_stream(dev)
        routes._used_on(stream)
        columns = place.shape[-1]
        rc = _L.fbh_to_experts(dev, x.data_ptr(), place.data_ptr(), n // columns, columns, dim,
                               cells, out.data_ptr(), stream)
        if rc:
            N.check_hip(rc)
    return out


def to_experts(x, routes: Routes):
    """The rows of `x` (..., cells), with the leading shape of the routes' ids, in the order of
    the routes: (positions, cells). Expert e's are rows starts[e] .. starts[e + 1] - 1; rows
    behind the last expert's are zeros."""
    torch = _need_torch()
    x = _device_tensor(x, "x")
    place = _routes(routes, x)
    dim, cells = _rows_of(x, "x", place.shape[:-1]), _cells(x, "x")
    if x.requires_grad and torch.is_grad_enabled():
        return _functions()[3].apply(x, routes, place, dim, cells)
    return _to_experts(x, routes, place, dim, cells)


def _from_experts(y, routes, place, weights, dim: int, cells: int):
    shape = place.shape
    out = y.new_empty(shape[:-1] + (dim,))
    n = place.numel()
    if not n:
        return out.zero_()
    dev = y.get_device()
    stream = _raw_stream(dev)
    routes._used_on(stream)
    rc = _L.fbh_from_experts(dev, y.data_ptr(), place.data_ptr(),
                             0 if weights is None else weights.data_ptr(), n // shape[-1],
                             shape[-1], dim, cells, out.data_ptr(), stream)
    if rc:
        N.check_hip(rc)
    return out


def _weights(weights, place):
    weights = _device_tensor(weights, "weights", place.get_device())
    if weights.dtype is not _torch.float32 or weights.shape != place.shape:
        raise ValueError(f"weights must be float32 of {tuple(place.shape)}, got {weights.dtype} of "
                         f"{tuple(weights.shape)}")
    return weights


def from_experts(y, routes: Routes, weights=None):
    """What experts have given for the rows of to_experts(), `y` (positions, cells), back at
    its rows: for each, the sum over its columns of weights[..., column] * the position's row
    of y, in float32 and rounded once. weights (the shape of ids, float32) may be None: 1. A
    position without an expert gives nothing, whatever its row of y and its weight hold."""
    torch = _need_torch()
    y = _device_tensor(y, "y")
    place = _routes(routes, y)
    dim, cells = _rows_of(y, "y", (place.numel(),)), _cells(y, "y")
    if weights is not None:
        weights = _weights(weights, place)
    if (y.requires_grad or (weights is not None and weights.requires_grad)) and (
            torch.is_grad_enabled()):
        return _functions()[4].apply(y, weights, routes, place, dim, cells)
    return _from_experts(y, routes, place, weights, dim, cells)


def _from_experts_grad(grad, y, routes, place, weights, want_y: bool, want_weights: bool,
                       dim: int, cells: int):
    n = place.numel()
    dy = grad.new_empty((n, dim)) if want_y else None
    dw = _torch.empty_like(weights) if want_weights else None
    if n and (want_y or want_weights):
        dev = grad.get_device()
        stream = _raw_stream(dev)
        routes._used_on(stream)
        columns = place.shape[-1]
        rc = _L.fbh_from_experts_grad(
            dev, grad.data_ptr(), 0 if y is None else y.data_ptr(), place.data_ptr(),
            0 if weights is None else weights.data_ptr(), n // columns, columns, dim, cells,
            dy.data_ptr() if want_y else 0, dw.data_ptr() if want_weights else 0, stream)
        if rc:
            N.check_hip(rc)
    return dy, dw


def from_experts_grad(grad, y, routes: Routes, weights=None):
    """The gradients of from_experts()'s y and weights for `grad`, that of its output: (dy,
    dweights), the second None without weights. Rows of dy without an expert are zeros.
    (from_experts() does this in backward(); a captured training step can call it by itself.
    to_experts()'s gradient is from_experts() without weights.)"""
    _need_torch()
    grad = _device_tensor(grad, "grad")
    place = _routes(routes, grad)
    dim, cells = _rows_of(grad, "grad", place.shape[:-1]), _cells(grad, "grad")
    y = _device_tensor(y, "y", grad.get_device())
    if y.shape != (place.numel(), dim) or y.dtype is not grad.dtype:
        raise ValueError(f"y must be {grad.dtype} of {(place.numel(), dim)}, got {y.dtype} of "
                         f"{tuple(y.shape)}")
    if weights is not None:
        weights = _weights(weights, place)
    return _from_experts_grad(grad, y, routes, place, weights, True, weights is not None, dim,
                              cells)


# ------------------------------------------------------------------- AdamW
@functools.lru_cache(maxsize=64)
def _adamw_tensors(n: int) -> struct.Struct:
    """n of fbh_adamw_tensor."""
    return struct.Struct("PPPQQfI" * n)


class AdamW(_Kept):
    """AdamW over `params`, all in one step: for gradient g of a cell w at step t,

        m = beta1 m + (1 - beta1) g,  s = beta2 s + (1 - beta2) g^2
        w = w (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(s / (1 - beta2^t)) + eps)

    in float32. params are contiguous tensors of one device; one of 16 bits has a float32 copy
    in `masters`, which is what the steps move and round into it (call take_params() after
    writing into such a parameter). weight_decay is a number, or a list of one for each
    parameter; lr a number, or a float32 tensor of one value on the device, in memory that is no
    parameter's, which a step reads when it runs. Both are attributes that may be set between
    steps. The steps are counted on the device too, so a captured step goes on at each replay (and
    the optimizer and that lr have to live as long as the graph). Steps of one optimizer follow one
    another: on another stream only when that has waited.

    bits=32 keeps m and s in float32, bits=8 in a byte each and an exponent for 256 cells:
    small floats with 3 bits behind the point, rounded up or down at random (from `seed`, the
    step and the cell, so the same in every run) with the new value as their mean, as a step
    moves s by less than half the distance of its neighbours. What is not finite is NaN then.

    The state of all parameters is flat: parameter i's cells are first[i] .. first[i] + n - 1
    of mean and square, first[i] a multiple of 256 and what lies between zeros."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay=0.01, *, bits: int = 32, seed: int = 0):
        torch = _need_torch()
        self.params = [params] if isinstance(params, torch.Tensor) else _list(params, "params")
        if not self.params:
            raise ValueError("no parameters")
        betas = tuple(_number(b, "betas must be two numbers in [0, 1): each")
                      for b in _list(betas, "betas must be two numbers in [0, 1): they"))
        if len(betas) != 2 or not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"betas must be two numbers in [0, 1), got {betas}")
        if bits not in (8, 32):
            raise ValueError(f"bits must be 8 or 32, got {bits!r}")
        self.lr, self.betas, self.eps, self.bits = lr, betas, _eps(eps), int(bits)
        self.seed = _seed(seed)
        self._parts = None
        self.weight_decay = weight_decay
        self.first, at, spans = [], 0, []
        for i, p in enumerate(self.params):
            self._check(i, p)
            self.first.append(at)
            at += -(-p.numel() // 256) * 256
            if p.numel():
                spans.append((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()))
        if at > 1 << 42:
            raise ValueError(f"at most 2^42 cells, got {at}")
        spans.sort()
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("parameters overlap in memory")
        self._sizes = [p.numel() for p in self.params]
        self._types = [p.dtype for p in self.params]
        # an fbh_adamw_tensor a parameter, whose addresses are filled in at each step
        self._parts = [x for i, p in enumerate(self.params) for x in
                       (0, 0, 0, self._sizes[i], self.first[i], self._decays[i],
                        _CELLS[p.dtype])]
        self._lr()
        like = self.params[0]
        cell = torch.float32 if bits == 32 else torch.uint8
        self.mean, self.square = (torch.zeros(at, dtype=cell, device=like.device)
                                  for _ in range(2))
        self.scales = (torch.zeros((2, at // 256), dtype=torch.uint8, device=like.device)
                       if bits == 8 else None)
        self.masters = [None if p.dtype == torch.float32 else p.detach().float()
                        for p in self.params]
        self._clock = torch.zeros(4, dtype=torch.int64, device=like.device)
        self._clock[1:3] = 0x3FF0000000000000  # 1.0
        self._streams = {_raw_stream(like.get_device())}

    # the learning rate's tensor and the stream that the last step has kept it for
    _lr_used = (None, None)

    def __setstate__(self, state):
        super().__setstate__({**state, "_lr_used": (None, None)})

    @property
    def weight_decay(self) -> tuple:
        """Each parameter's weight decay; it is set as a number or a list of one for each."""
        return self._decays

    @weight_decay.setter
    def weight_decay(self, value):
        n = len(self.params)
        decays = tuple(_number(d, "weight_decay") for d in value) if (
            isinstance(value, (list, tuple))) else (_number(value, "weight_decay"),) * n
        if len(decays) != n or not all(0.0 <= d <= _MOST for d in decays):
            raise ValueError(f"weight_decay must be a number, not negative, or a list of {n}")
        self._decays = decays
        if self._parts is not None:
            parts = list(self._parts)  # (a copy of the optimizer shares the list)
            parts[5::7] = decays
            self._parts = parts

    def _check(self, i: int, p):
        if not isinstance(p, _torch.Tensor):
            raise ValueError(f"parameter {i} must be a torch tensor, got {type(p).__name__}")
        _no_tangent(p, f"parameter {i}")
        _dense(p, f"parameter {i}")
        if not p.is_cuda:
            raise ValueError(f"parameter {i} must be on a GPU, it is on {p.device}")
        _cells(p, f"parameter {i}")
        _beside(p, self.params[0], f"parameter {i}")
        if not p.is_contiguous():
            raise ValueError(f"parameter {i} must be contiguous")

    def _tensors(self):
        return [x for x in (self.mean, self.square, self.scales, self._clock, *self.masters)
                if x is not None]

    def _lr(self):
        """The learning rate as a number, and the address of one on the device or 0."""
        lr = self.lr
        if isinstance(lr, _Tensor):
            _device_tensor(lr, "lr", self.params[0].get_device())
            if lr.dtype != _torch.float32 or lr.numel() != 1:
                raise ValueError(f"lr must be one float32, got {lr.dtype} of {tuple(lr.shape)}")
            return 0.0, lr.data_ptr()
        lr = _number(lr, "lr")
        if not 0.0 <= lr <= _MOST:
            raise ValueError(f"lr must be a finite float32, not negative, got {lr}")
        return lr, 0

    def _packed(self) -> bytes:
        """The call's fbh_adamw."""
        lr, lr_at = self._lr()
        return _ADAMW.pack(self.bits, self.eps, *self.betas, lr, lr_at, self.seed,
                           self.mean.numel(), self.mean.data_ptr(), self.square.data_ptr(),
                           0 if self.scales is None else self.scales.data_ptr(),
                           self._clock.data_ptr())

    def _gradient(self, i: int, p, g):
        """The gradient of parameter i, checked and contiguous."""
        if g is None:
            raise ValueError(f"parameter {i} has no gradient")
        g = _device_tensor(g, f"gradient {i}")
        if g.dtype != p.dtype or g.shape != p.shape or g.device != p.device:
            raise ValueError(f"gradient {i} is {g.dtype} of {tuple(g.shape)} on {g.device}, "
                             f"its parameter {p.dtype} of {tuple(p.shape)} on {p.device}")
        return g

    def step(self, grads=None):
        """One step, in place, with the parameters' .grad or with `grads`, a list of one for
        each parameter, of its shape and type. Every parameter needs one, in memory that is no
        parameter's."""
        params = self.params
        grads = [p.grad for p in params] if grads is None else _list(grads, "grads")
        if len(grads) != len(params):
            raise ValueError(f"{len(grads)} gradients for {len(params)} parameters")
        # (a small step's time is what the host takes for these)
        T = _torch.Tensor
        dev = self.mean.get_device()
        devices = [dev] * len(params)
        try:
            plain = (_forward_ad._current_level < 0 and all(type(g) is T for g in grads) and
                     list(map(T.get_device, grads)) == devices and
                     all(map(T.is_contiguous, grads)) and
                     list(map(_dtype_of, grads)) == self._types and
                     list(map(_shape_of, grads)) == list(map(_shape_of, params)))
            at = list(map(T.data_ptr, grads)) if plain else None
        except RuntimeError:  # (sparse ones have no address)
            plain = False
        if not plain:
            for i, p in enumerate(params):
                _no_tangent(p, f"parameter {i}")
            grads = [self._gradient(i, p, g) for i, (p, g) in enumerate(zip(params, grads))]
            at = list(map(T.data_ptr, grads))
        if not (list(map(_dtype_of, params)) == self._types and
                list(map(T.numel, params)) == self._sizes and
                list(map(T.get_device, params)) == devices and all(map(T.is_contiguous, params))):
            raise ValueError("a parameter has changed its type, size or place")
        parts = self._parts
        parts[0::7] = map(T.data_ptr, params)
        parts[1::7] = at
        parts[2::7] = [0 if w is None else w.data_ptr() for w in self.masters]
        stream = _raw_stream(dev)
        self._used_on(stream)
        lr = self.lr
        if isinstance(lr, T) and (self._lr_used[0] is not lr or self._lr_used[1] != stream):
            lr.record_stream(_torch.cuda.current_stream(lr.device))
            self._lr_used = lr, stream
        rc = _L.fbh_adamw_step(dev, self._packed(), _adamw_tensors(len(params)).pack(*parts),
                               len(params), stream)
        if rc:
            N.check_hip(rc)
        _torch.autograd.graph.increment_version(params)

    def zero_grad(self):
        """Drops the parameters' gradients."""
        for p in self.params:
            p.grad = None

    def moments(self):
        """(mean, square) of all parameters, flat, as float32: with bits=32 the state itself,
        with bits=8 new tensors of what it stands for. split() cuts them by parameter."""
        if self.bits == 32:
            return self.mean, self.square
        out = [self.mean.new_empty(self.mean.numel(), dtype=_torch.float32) for _ in range(2)]
        dev = self.mean.get_device()
        stream = _raw_stream(dev)
        self._used_on(stream)
        rc = _L.fbh_adamw_moments(dev, self._packed(), out[0].data_ptr(), out[1].data_ptr(),
                                  stream)
        if rc:
            N.check_hip(rc)
        return out[0], out[1]

    def split(self, flat):
        """A flat tensor's parts as views in the parameters' shapes."""
        if not isinstance(flat, _Tensor) or flat.shape != self.mean.shape:
            raise ValueError(f"flat must be a tensor of {tuple(self.mean.shape)}, as moments() "
                             f"gives")
        return [flat[a:a + n].view(p.shape)
                for a, n, p in zip(self.first, self._sizes, self.params)]

    def take_params(self):
        """Sets the float32 copies of 16-bit parameters to what these hold now."""
        for i, p in enumerate(self.params):
            _no_tangent(p, f"parameter {i}")
        self._used_on(_raw_stream(self.mean.get_device()))
        with _torch.no_grad():
            for p, w in zip(self.params, self.masters):
                if w is not None:
                    w.copy_(p)

    def state_dict(self) -> dict:
        """What load_state_dict() takes: the steps done (waits for the device) and the state's
        own tensors, of which what stores them later makes copies. The numbers that the
        optimizer was made with or given since (lr, betas, eps, weight_decay) are not in it."""
        clock = self._clock.cpu()
        return {"step": int(clock[0]), "decays": clock[1:3].view(_torch.float64).tolist(),
                "bits": self.bits, "sizes": list(self._sizes), "seed": self.seed,
                "mean": self.mean, "square": self.square, "scales": self.scales,
                "masters": list(self.masters)}

    def load_state_dict(self, state: dict):
        """Takes up a state of as many parameters of the same sizes, copying it. "decays" (the
        betas' powers) follow from "step" where they are missing, "masters" from the
        parameters; without "sizes", the parameters' numbers of cells, only their padded sum
        is checked, and without "seed" the optimizer keeps its own."""
        if not isinstance(state, Mapping):
            raise ValueError(f"a state must be a dict, got {type(state).__name__}")
        missing = {"step", "mean", "square"} | ({"scales"} if self.bits == 8 else set())
        missing -= state.keys()
        if missing:
            raise ValueError(f"the state has no {', '.join(sorted(missing))}")
        step = _whole(state["step"], "step")
        if not 0 <= step < 1 << 62:
            raise ValueError(f"step must be in 0..=2^62 - 1, got {step}")
        if state.get("bits", self.bits) != self.bits:
            raise ValueError(f"the state has {state['bits']} bits, the optimizer {self.bits}")
        sizes = state.get("sizes")
        if sizes is not None and _list(sizes, "sizes") != self._sizes:
            raise ValueError(f"the state is one of parameters of {list(sizes)} cells, these have "
                             f"{self._sizes}")
        seed = self.seed if state.get("seed") is None else _seed(state["seed"])
        decays = state.get("decays")
        decays = [b ** step for b in self.betas] if decays is None else [
            _number(d, "decays must be two numbers in [0, 1]: each")
            for d in _list(decays, "decays must be two numbers in [0, 1]: they")]
        if len(decays) != 2 or not all(0.0 <= d <= 1.0 for d in decays):
            raise ValueError(f"decays must be two numbers in [0, 1], got {decays}")
        masters = state.get("masters")
        if masters is None:
            masters = [None if w is None else p for p, w in zip(self.params, self.masters)]
        masters = _list(masters, "masters")
        if len(masters) != len(self.masters):
            raise ValueError(f"{len(masters)} masters for {len(self.masters)} parameters")
        pairs = [("mean", self.mean, state["mean"]), ("square", self.square, state["square"])]
        if self.bits == 8:
            pairs.append(("scales", self.scales, state["scales"]))
        pairs += [(f"master {i}", to, m) for i, (to, m) in enumerate(zip(self.masters, masters))
                  if to is not None]
        for what, to, x in pairs:
            if not isinstance(x, _torch.Tensor) or x.shape != to.shape or (
                    x.dtype != to.dtype and not what.startswith("master")):
                raise ValueError(f"{what} must be {to.dtype} of {tuple(to.shape)}")
            _no_tangent(x, what)
        self._used_on(_raw_stream(self.mean.get_device()))
        with _torch.no_grad():
            for _, to, x in pairs:
                to.copy_(x)
            words = struct.unpack("4q", struct.pack("qddq", step, *decays, 0))
            self._clock.copy_(_torch.tensor(words, dtype=_torch.int64))
        self.seed = seed

    def __repr__(self):
        return (f"AdamW({len(self.params)} parameters, {sum(self._sizes)} cells, {self.bits} "
                f"bits)")
