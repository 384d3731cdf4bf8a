"""Heads on a model's outputs, for programs that go on in torch.

A model answers with leaf ids (predict(pred_leaf=True), FBH_PREDICT_LEAF on the
device) and class margins, and its rows hold categorical codes. What follows them:

  embed / embed_grad  vectors learned for ids: rows of a table looked up by id, as they
                      are or summed over a row's columns, and the table's gradient
  dropout             while they are learned, from (seed, element) alone: no mask
  sample              classes drawn from margins (Model.sample does it on host arrays)

    model = fb.train({"objective": "multi:softprob", "num_class": 4, ...}, X, label=y)
    leaves = torch.from_numpy(model.predict(X, pred_leaf=True)).cuda()
    voc = model.leaf_vocabulary()
    table = torch.zeros(voc.n_tokens, 64, device="cuda", requires_grad=True)
    h = fb.heads.embed(table, leaves, voc, pooled=True, drop=0.1, seed=step)
    h = fb.heads.dropout(h, 0.1, seed=step + 1)
    classes, log_probs = fb.heads.sample(h @ W, torch.rand(len(h), device="cuda"), top_p=0.9)

Tensors are torch tensors on one gfx950 device; torch must be imported before the
package's first call, so that both share one HIP runtime. Kernels are hand-written HIP
behind the C ABI of include/fbhip.h, enqueued on torch's current stream of the tensors'
device; nothing waits, results are the same in every call, and all of it can be captured
into a graph. A tensor that is not contiguous is copied first. embed and dropout take
part in autograd, in reverse mode; tensors with a tangent of forward mode are refused. What
embed_grad and sample give has no gradient. Bad arguments are ValueErrors, device failures
RuntimeErrors.
"""

from __future__ import annotations

import functools
import struct

import numpy as np

from . import _native as N

__all__ = ["Vocabulary", "embed", "embed_grad", "dropout", "sample"]

_torch = None
_L = None
_CELLS: dict = {}
_IDS: dict = {}
_raw_stream = None
_forward_ad = None
# fbh_embed and fbh_sample_options (include/fbhip.h), packed in one call: a small
# operation's time is its host time.
_EMBED = struct.Struct("QIIIIIIPPdQfI")
_OPTIONS = struct.Struct("PPPPfiff")
_MOST = float(np.finfo(np.float32).max)


def _need_torch():
    """torch, once it is known to share this package's HIP runtime."""
    global _torch, _L, _raw_stream, _forward_ad
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
    _L = N.hip()
    _torch = torch
    return torch


def _device_tensor(x, what: str):
    if not isinstance(x, _torch.Tensor):
        raise ValueError(f"{what} must be a torch tensor, got {type(x).__name__}")
    if _forward_ad._current_level >= 0 and _forward_ad.unpack_dual(x).tangent is not None:
        raise ValueError(f"{what} has a tangent: forward-mode derivatives are not available")
    if not x.is_cuda:
        raise ValueError(f"{what} must be on a GPU, it is on {x.device}")
    return x if x.is_contiguous() else x.contiguous()


def _cells(x, what: str) -> int:
    code = _CELLS.get(x.dtype)
    if code is None:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, got {x.dtype}")
    return code


def _beside(x, other, what: str):
    if x.device != other.device:
        raise ValueError(f"{what} is on {x.device}, the call's other tensors on {other.device}")
    return x


def _whole(v, what: str) -> int:
    try:
        return int(v)
    except (OverflowError, TypeError, ValueError):
        raise ValueError(f"{what} must be a whole number, got {v!r}") from None


def _seed(seed) -> int:
    seed = _whole(seed, "seed")
    if not 0 <= seed < 1 << 64:
        raise ValueError(f"seed must be in 0..=2^64 - 1, got {seed}")
    return seed


def _drop(drop) -> float:
    drop = float(drop)
    if not 0.0 <= drop < 1.0:
        raise ValueError(f"drop must be in [0, 1), got {drop}")
    return drop


def _scale(scale) -> float:
    scale = float(scale)
    if not abs(scale) <= _MOST:
        raise ValueError(f"scale must be a finite float32, got {scale}")
    return scale


class Vocabulary:
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

    def _used_on(self, stream: int):
        """Keeps the offsets' memory from the allocator until the work now on this stream, the
        current one, has passed, also when the vocabulary is dropped before."""
        if stream not in self._streams:
            self.first.record_stream(_torch.cuda.current_stream(self.first.device))
            self._streams.add(stream)

    def __setstate__(self, state):
        # (a copy's tensor has not been used on any stream yet)
        self.__dict__.update(state, _streams=set())

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

    return Embed, Dropout


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
    ids = _beside(_device_tensor(ids, "ids"), table, "ids")
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
    ids = _beside(_device_tensor(ids, "ids"), grad, "ids")
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
    if not isinstance(value, _torch.Tensor) or value.dim() == 0:
        return None
    v = _beside(_device_tensor(value, what), like, what)
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
    v = float(v)
    if not 0.0 <= v <= _MOST:
        raise ValueError(f"temperature must be a finite float32, not negative, got {v}")
    return v


def _top_k(v) -> int:
    k = _whole(v, "top_k")
    if isinstance(v, bool) or k != v or k < 0:
        raise ValueError(f"top_k must be a whole number, 0 (all) or more, got {v!r}")
    return min(k, 0x7FFFFFFF)


def _share(what: str, v) -> float:
    v = float(v)
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
    uniforms = _beside(_device_tensor(uniforms, "uniforms"), logits, "uniforms")
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
