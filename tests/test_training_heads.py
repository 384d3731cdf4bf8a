"""The training heads' checks of arguments, sizes and definitions, which need no device."""

from __future__ import annotations

import copy
import pickle
import struct

import numpy as np
import pytest
import torch

import heads_ref
import training_ref as ref
from ferrisboost_amd import _native as N
from ferrisboost_amd import heads


def _norm(**kw):
    v = {"n_rows": 4, "dim": 8, "dtype": 0, "weight_type": 0, "eps": 1e-5, **kw}
    return heads._NORM.pack(*v.values())


@pytest.mark.parametrize("bad, msg", [
    ({"dtype": 3}, "cell type"), ({"weight_type": 3}, "weight type"), ({"dim": 0}, "dim must"),
    ({"dim": 32769}, "dim must"), ({"n_rows": 1 << 60}, "cells"), ({"eps": 0.0}, "eps"),
    ({"eps": 1e-40}, "eps"), ({"eps": float("inf")}, "eps"), ({"eps": float("nan")}, "eps"),
    ({"eps": -1.0}, "eps")])
def test_layer_norm_refusals_of_the_c_abi(bad, msg):
    L, a = N.hip(), _norm(**bad)
    with pytest.raises(ValueError, match=msg):
        N.check_hip(L.fbh_layer_norm(0, a, 64, None, None, 64, None, None))
    with pytest.raises(ValueError, match=msg):
        N.check_hip(L.fbh_layer_norm_grad(0, a, 64, 64, 64, None, 72, None, None, None, 0, None))
    assert L.fbh_layer_norm_grad_bytes(a) == 0


def test_layer_norm_null_arguments_and_workspace():
    L, a = N.hip(), _norm(n_rows=1000)
    for args in ((None, None, None, 64, None), (64, None, None, None, None)):
        with pytest.raises(ValueError, match="null"):
            N.check_hip(L.fbh_layer_norm(0, a, *args, None))
    with pytest.raises(ValueError, match="null"):
        N.check_hip(L.fbh_layer_norm_grad(0, a, 64, 64, None, None, 64, None, None, None, 0, None))
    for dx in (64, 128):
        with pytest.raises(ValueError, match="must not be grad or x"):
            N.check_hip(L.fbh_layer_norm_grad(0, a, 64, 128, 64, None, dx, None, None, None, 0,
                                              None))
    need = L.fbh_layer_norm_grad_bytes(a)
    assert need > 0
    for work, size, msg in ((64, need - 1, "workspace"), (None, 0, "workspace"),
                            (72, need, "aligned")):
        with pytest.raises(ValueError, match=msg):
            N.check_hip(L.fbh_layer_norm_grad(0, a, 64, 64, 64, None, None, 64, None, work, size,
                                              None))


@pytest.mark.parametrize("n", [0, 1, 63, 5000, 1 << 20, 1 << 25])
@pytest.mark.parametrize("dim", [1, 3, 8, 33, 256, 257, 4096, 4097, 16_384, 16_385, 32_768])
def test_layer_norm_workspace_is_bounded(n, dim):
    """At most 1024 parts of two float32 vectors, fewer of wider ones (32 MiB but for the
    widest rows, which take 4 bytes a row besides), and no more parts than rows; none for a
    few rows."""
    got = N.hip().fbh_layer_norm_grad_bytes(_norm(n_rows=n, dim=dim))
    rows = 4 * n + 16 if dim > 16_384 else 0
    assert got <= min(32 << 20, 8 * dim * max(n, 1)) + rows
    assert got >= 8 * dim or (got == 0 and n <= 128 and dim <= 4096)


def test_experts_refusals_of_the_c_abi():
    L = N.hip()

    def route(n=10, e=4, ids=64, kind=0, order=64, place=64, starts=64, work=64, size=1 << 30):
        N.check_hip(L.fbh_route(0, ids, kind, n, e, order, place, starts, work, size, None))

    for kw, msg in [({"n": 1 << 31}, "positions"), ({"e": 0}, "n_experts"),
                    ({"e": 1025}, "n_experts"), ({"ids": None}, "null"), ({"kind": 3}, "id type"),
                    ({"order": None}, "null"), ({"place": None}, "null"),
                    ({"starts": None}, "null"), ({"n": 5000, "work": None}, "workspace"),
                    ({"n": 5000, "size": 8}, "workspace"), ({"n": 5000, "work": 66}, "aligned")]:
        with pytest.raises(ValueError, match=msg):
            route(**kw)
    assert L.fbh_route_bytes(4096, 1024) == 0 < L.fbh_route_bytes(4097, 1)
    assert L.fbh_route_bytes(1 << 31, 4) == L.fbh_route_bytes(5000, 1025) == 0
    # a counter an expert and at least 1024 positions, and one an expert
    for n in (4097, 1 << 19, (1 << 19) + 1, 1 << 25, (1 << 31) - 1):
        for e in (1, 1024):
            assert L.fbh_route_bytes(n, e) <= 4 * (e + 1) * (n // 1024 + 2)
    bad = [({"n": 1 << 31}, "positions"), ({"k": 0}, "columns"), ({"dim": 0}, "dim must"),
           ({"dim": 32_769}, "dim must"), ({"dtype": 3}, "cell type"), ({"place": None}, "null"),
           ({"x": None}, "null")]
    for kw, msg in bad:
        v = {"n": 4, "k": 2, "dim": 8, "dtype": 0, "place": 64, "x": 64, **kw}
        shape = (v["n"], v["k"], v["dim"], v["dtype"])
        with pytest.raises(ValueError, match=msg):
            N.check_hip(L.fbh_to_experts(0, v["x"], v["place"], *shape, 64, None))
        with pytest.raises(ValueError, match=msg):
            N.check_hip(L.fbh_from_experts(0, v["x"], v["place"], None, *shape, 64, None))
        with pytest.raises(ValueError, match=msg):
            N.check_hip(L.fbh_from_experts_grad(0, v["x"], 64, v["place"], None, *shape, 64, None,
                                                None))
    with pytest.raises(ValueError, match="null"):
        N.check_hip(L.fbh_from_experts_grad(0, 64, None, 64, None, 4, 2, 8, 0, None, 64, None))


def _adamw(**kw):
    v = {"bits": 8, "eps": 1e-8, "beta1": 0.9, "beta2": 0.999, "lr": 1e-3, "lr_at": 0, "seed": 0,
         "n": 512, "mean": 64, "square": 64, "scales": 64, "clock": 64, **kw}
    return heads._ADAMW.pack(*v.values())


def _tensor(**kw):
    v = {"param": 64, "grad": 64, "master": 64, "n": 256, "first": 0, "decay": 0.0, "dtype": 2,
         **kw}
    return struct.pack("PPPQQfI", *v.values())


@pytest.mark.parametrize("bad, msg", [
    ({"bits": 16}, "bits"), ({"eps": 0.0}, "eps"), ({"eps": float("nan")}, "eps"),
    ({"beta1": 1.0}, "betas"), ({"beta2": -0.1}, "betas"), ({"beta2": float("nan")}, "betas"),
    ({"lr": -1.0}, "lr"), ({"lr": float("inf")}, "lr"), ({"n": 100}, "multiple of 256"),
    ({"n": 1 << 43}, "multiple of 256"), ({"mean": 0}, "moments"), ({"square": 72}, "moments"),
    ({"scales": 0}, "scales"), ({"clock": 0}, "clock"), ({"clock": 68}, "clock")])
def test_adamw_refusals_of_the_c_abi(bad, msg):
    L, a = N.hip(), _adamw(**bad)
    with pytest.raises(ValueError, match=msg):
        N.check_hip(L.fbh_adamw_step(0, a, _tensor(), 1, None))
    with pytest.raises(ValueError, match=msg):
        N.check_hip(L.fbh_adamw_moments(0, a, 64, 64, None))


def test_adamw_tensor_refusals_of_the_c_abi():
    L = N.hip()
    for bad, msg in [({"param": 0}, "null"), ({"grad": 0}, "null"), ({"master": 0}, "null"),
                     ({"dtype": 3}, "cell type"), ({"first": 128}, "outside"),
                     ({"first": 512}, "outside"), ({"n": 513}, "outside"),
                     ({"first": 1 << 63}, "outside"), ({"n": 1 << 63}, "outside"),
                     ({"decay": -1.0}, "weight_decay"), ({"decay": float("nan")}, "weight_decay")]:
        with pytest.raises(ValueError, match=msg):
            N.check_hip(L.fbh_adamw_step(0, _adamw(), _tensor(**bad), 1, None))
    with pytest.raises(ValueError, match="null"):
        N.check_hip(L.fbh_adamw_step(0, _adamw(), None, 1, None))
    with pytest.raises(ValueError, match="32 bits"):
        N.check_hip(L.fbh_adamw_moments(0, _adamw(bits=32), 64, 64, None))
    with pytest.raises(ValueError, match="null"):
        N.check_hip(L.fbh_adamw_moments(0, _adamw(), 64, None, None))


@pytest.mark.parametrize("tensors, msg", [
    # (256 cells of float32: 1024 bytes each)
    ([(0x1000, 0x9000), (0x13FC, 0xA000)], "parameters overlap"),
    ([(0x1400, 0x9000), (0x3000, 0xA000), (0x1001, 0xB000)], "parameters overlap"),
    ([(0x1000, 0x9000), (0x1000, 0xA000)], "parameters overlap"),
    ([(0x1000, 0x1000)], "gradient overlaps"),
    ([(0x1000, 0x3000), (0x3000, 0x1000)], "gradient overlaps"),
    ([(0x1000, 0x9000), (0x3000, 0x33FF)], "gradient overlaps"),
    ([(0x1000, 0x9000), (0x3000, 0x0C01), (0x5000, 0xA000)], "gradient overlaps")])
def test_adamw_refuses_overlapping_tensors(tensors, msg):
    packed = b"".join(_tensor(param=p, grad=g, first=256 * i, dtype=0)
                      for i, (p, g) in enumerate(tensors))
    with pytest.raises(ValueError, match=msg):
        N.check_hip(N.hip().fbh_adamw_step(0, _adamw(n=1024), packed, len(tensors), None))


def test_structs_have_the_header_s_sizes():
    """8-byte fields first and 4-byte ones in pairs: no padding but the norm's last word."""
    assert heads._ADAMW.size == 88 and len(_tensor()) == 48
    assert heads._NORM.size == 24


def test_tensors_must_be_on_a_gpu():
    x, ids = torch.zeros(4, 8), torch.zeros((4, 1), dtype=torch.int32)
    w = torch.ones(8)
    for call in (lambda: heads.layer_norm(x, w, w), lambda: heads.layer_norm_grad(x, x, x),
                 lambda: heads.Routes(ids, 4), lambda: heads.AdamW([x])):
        with pytest.raises(ValueError, match="on a GPU"):
            call()
    for call in (lambda: heads.layer_norm(np.zeros(3)), lambda: heads.Routes([1, 2], 4),
                 lambda: heads.AdamW([[1.0]])):
        with pytest.raises(ValueError, match="torch tensor"):
            call()
    with pytest.raises(ValueError, match="no parameters"):
        heads.AdamW([])


def test_eps():
    for bad in (0.0, -1e-5, float("nan"), float("inf"), 1e-39, 1e39):
        with pytest.raises(ValueError, match="eps"):
            heads._eps(bad)
    assert heads._eps(2.0 ** -126) == 2.0 ** -126


@pytest.mark.parametrize("kw, msg", [
    ({"betas": (0.9,)}, "betas"), ({"betas": (0.9, 1.0)}, "betas"), ({"betas": (-0.1, 0.9)}, "betas"),
    ({"bits": 4}, "bits"), ({"eps": 0.0}, "eps"), ({"seed": -1}, "seed"),
    ({"weight_decay": -0.1}, "weight_decay"), ({"weight_decay": [0.1, 0.1]}, "weight_decay"),
    ({"weight_decay": float("nan")}, "weight_decay")])
def test_adamw_refusals(kw, msg):
    with pytest.raises(ValueError, match=msg):
        heads.AdamW([torch.zeros(3)], **kw)


def test_tensors_with_a_tangent_are_refused():
    import torch.autograd.forward_ad as fwd

    x = torch.ones(4, 8)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: heads.layer_norm(d), lambda: heads.layer_norm_grad(x, d, x),
                     lambda: heads.Routes(d, 4)):
            with pytest.raises(ValueError, match="has a tangent"):
                call()


def test_copied_routes_have_been_used_on_no_stream():
    r = object.__new__(heads.Routes)
    r.n_experts, r._streams = 3, {0, 77}
    r.order, r.place, r.starts = (torch.arange(4, dtype=torch.int32) for _ in range(3))
    for v in (copy.copy(r), copy.deepcopy(r), pickle.loads(pickle.dumps(r))):
        assert v._streams == set() and torch.equal(v.place, r.place)
    assert r._streams == {0, 77}


# ------------------------------------------------- the definitions by themselves
def test_gradient_of_the_norm_s_definition_against_differences():
    """Central differences of doubles, with 1e-5: step^2 times the third derivative (below 10^4
    for rows of 7 cells of variance 0.1 and more) and 2^-53 of values of some 10 over the step,
    together below 1e-5."""
    rng = np.random.default_rng(1)
    x, g, w = rng.normal(size=(3, 7)), rng.normal(size=(3, 7)), rng.normal(size=7)
    (dx, _), (dw, _), (db, _) = ref.layer_norm_grad(g, x, w, 1e-5)
    for want, arg in ((dx, 0), (dw, 1), (db, 2)):
        args = [x, w, np.zeros(7)]
        for at in np.ndindex(want.shape):
            got = 0.0
            for s in (1, -1):
                moved = [a.copy() for a in args]
                moved[arg][at] += s * 1e-5
                got += s * (ref.layer_norm(*moved, 1e-5)[0] * g).sum() / 2e-5
            assert abs(got - want[at]) < 1e-5


def test_gradient_of_the_experts_definition_against_differences():
    """Linear in y and in the weights: differences are exact but for roundings."""
    rng = np.random.default_rng(2)
    ids = rng.integers(-1, 4, (5, 3))
    _, place, _ = ref.route(ids, 4)
    y, g, w = rng.normal(size=(15, 6)), rng.normal(size=(5, 6)), rng.normal(size=(5, 3))
    dy, dw, _ = ref.from_experts_grad(g, y, place, w)
    for want, arg in ((dy, 0), (dw, 1)):
        for at in np.ndindex(want.shape):
            moved = [y.copy(), w.copy()]
            moved[arg][at] += 1.0
            got = ((ref.from_experts(moved[0], place, moved[1])[0] -
                    ref.from_experts(y, place, w)[0]) * g).sum()
            assert abs(got - want[at]) < 1e-12


def test_random_words_are_those_of_dropout():
    n = 1001
    words = ref.random_words((1 << 64) - 5, n)
    for drop in (0.25, 0.5):
        assert np.array_equal(words >= round(drop * 2 ** 32),
                              heads_ref.kept((1 << 64) - 5, drop, np.arange(n)))


@pytest.mark.parametrize("square", [False, True])
def test_bytes_and_their_values(square):
    """Values of a byte are kept by every random number; others go to one of the two around
    them, up as often as the part that is cut off says."""
    field = np.full(1, 130, np.uint8)
    top = 0xF0 if square else 0x70  # the largest one's exponent
    codes = np.arange(256, dtype=np.uint8)
    codes = codes[codes < top + 8] if square else codes[(codes & 0x7F) < top + 8]
    block = np.zeros(256, np.uint8)
    block[:codes.size] = codes
    block[-1] = top  # (keeps the exponent)
    v = ref.byte_values(block, field, square).astype(np.float32)
    for r in (0, 1, 0x8000, 0xFFFF):
        got, f = ref.to_bytes(v, np.full(256, r), square)
        assert f[0] == 130 and np.array_equal(got, block)
    x = np.zeros(256, np.float32)
    x[0], x[1] = 8.0, 1.0 + 1 / 32  # a quarter between 1 and 1 + 1 / 8
    ups = 0
    for r in range(0, 1 << 16, 64):
        got, f = ref.to_bytes(x, np.full(256, r), square)
        value = ref.byte_values(got, f, square)[1]
        assert value in (1.0, 1.125)
        ups += value == 1.125
    assert ups == 256  # of 1024
    x[2], x[3] = np.nan, np.inf
    got, f = ref.to_bytes(x, np.zeros(256), square)
    assert f[0] == 130 and np.isnan(ref.byte_values(got, f, square)[2:4]).all()
    if square:
        x[4] = 1e-30
        got, f = ref.to_bytes(x, np.zeros(256), True)
        assert got[4] == 1
