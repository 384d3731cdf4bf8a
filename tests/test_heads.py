"""The heads' checks of arguments, which need no device."""

from __future__ import annotations

import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from ferrisboost_amd import _native as N
from ferrisboost_amd import heads


def _embed(**kw):
    e = N.Embed()
    e.n_rows, e.n_columns, e.dim, e.n_tokens, e.ids, e.scale = 4, 3, 8, 10, 64, 1.0
    for k, v in kw.items():
        setattr(e, k, v)
    return e


@pytest.mark.parametrize("bad, msg", [
    ({"dtype": 3}, "cell type"), ({"id_type": 3}, "id type"), ({"dim": 0}, "dim must"),
    ({"dim": 32769}, "dim must"), ({"n_columns": 0}, "no columns"),
    ({"n_columns": 32769, "first": 64}, "32768 columns"), ({"n_tokens": 0}, "n_tokens"),
    ({"n_tokens": 1 << 31}, "n_tokens"), ({"ids": None}, "null"), ({"drop": 1.0}, "drop"),
    ({"drop": -0.1}, "drop"), ({"drop": float("nan")}, "drop"),
    ({"n_rows": 1 << 60}, "positions")])
def test_embed_refusals_of_the_c_abi(bad, msg):
    L = N.hip()
    e = _embed(**bad)
    with pytest.raises(ValueError, match=msg):
        N.check_hip(L.fbh_embed_rows(0, C.byref(e), 64, 64, None))
    with pytest.raises(ValueError, match=msg):
        N.check_hip(L.fbh_embed_grad(0, C.byref(e), 64, 64, 64, 1 << 40, None))
    assert L.fbh_embed_grad_bytes(C.byref(e)) == 0


def test_gradient_workspace():
    L = N.hip()
    e = _embed()
    need = L.fbh_embed_grad_bytes(C.byref(e))
    assert need > 0
    with pytest.raises(ValueError, match="workspace"):
        N.check_hip(L.fbh_embed_grad(0, C.byref(e), 64, 64, 64, need - 1, None))
    with pytest.raises(ValueError, match="aligned"):
        N.check_hip(L.fbh_embed_grad(0, C.byref(e), 64, 64, 72, need, None))
    big = _embed(n_rows=1 << 31)
    with pytest.raises(ValueError, match="positions"):
        N.check_hip(L.fbh_embed_grad(0, C.byref(big), 64, 64, 64, 1 << 50, None))


def test_dropout_and_sampling_refusals_of_the_c_abi():
    L = N.hip()
    for args, msg in [((None, 64, 4, 0, 0.5), "null"), ((64, 64, 4, 7, 0.5), "cell type"),
                      ((64, 64, 4, 0, 1.0), "drop"), ((64, 64, 1 << 36, 0, 0.5), "2\\^35")]:
        with pytest.raises(ValueError, match=msg):
            N.check_hip(L.fbh_dropout(0, *args, 1, 0, None))
    o = N.SampleOptions()
    for v, dt, u, msg in [(0, 0, 64, "n_classes"), (262145, 0, 64, "n_classes"),
                          (5, 9, 64, "cell type"), (5, 0, None, "null")]:
        with pytest.raises(ValueError, match=msg):
            N.check_hip(L.fbh_sample_classes(0, 64, 2, v, dt, u, C.byref(o), 64, None, None, 0,
                                             None))
    need = L.fbh_sample_bytes(2, 100_000)
    assert need > 0 and L.fbh_sample_bytes(2, 1000) == L.fbh_sample_bytes(5000, 100_000) == 0
    with pytest.raises(ValueError, match="workspace"):
        N.check_hip(L.fbh_sample_classes(0, 64, 2, 100_000, 0, 64, C.byref(o), 64, None, 64,
                                         need - 1, None))
    with pytest.raises(ValueError, match="aligned"):
        N.check_hip(L.fbh_sample_classes(0, 64, 2, 100_000, 0, 64, C.byref(o), 64, None, 68,
                                         need, None))
    o.top_ks = 64
    with pytest.raises(ValueError, match="each row"):
        N.check_hip(L.fbh_sample_classes_host(0, 64, 2, 5, 64, C.byref(o), 64, None))


def test_tensors_must_be_on_a_gpu():
    x = torch.zeros(4, 8)
    ids = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: heads.embed(x, ids), lambda: heads.embed_grad(x, ids, 4),
                 lambda: heads.dropout(x, 0.1, 0), lambda: heads.sample(x, x[:, 0])):
        with pytest.raises(ValueError, match="on a GPU"):
            call()
    with pytest.raises(ValueError, match="torch tensor"):
        heads.dropout(np.zeros(3, np.float32), 0.1, 0)
    with pytest.raises(ValueError, match="must be a GPU"):
        heads.Vocabulary([3, 4], device="cpu")


@pytest.mark.parametrize("sizes", [[], [[1, 2]], [1.5], [3, -1], [0, 0], [1 << 30, 1 << 30],
                                   [1] * 32769])
def test_vocabulary_refusals(sizes):
    with pytest.raises(ValueError):
        heads.Vocabulary(sizes)


@pytest.mark.parametrize("bad", [
    {"temperature": -1.0}, {"temperature": float("nan")}, {"temperature": 1e39}, {"top_k": -1},
    {"top_k": 2.5}, {"top_k": True}, {"top_p": 1.01}, {"top_p": float("nan")}, {"min_p": -0.1}])
def test_sampling_options(bad):
    with pytest.raises(ValueError, match=next(iter(bad))):
        heads.check_options(**{**{"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0},
                               **bad})


def test_torch_after_the_first_call_is_refused():
    """The package's library has loaded the system's HIP runtime by then, and torch brings
    its own: pointers of one mean nothing to the other."""
    code = ("from ferrisboost_amd import _native as N, heads\n"
            "N.hip()\n"
            "try:\n"
            "    heads.Vocabulary([1])\n"
            "except RuntimeError as e:\n"
            "    print('refused:', e)\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True,
                         timeout=300)
    assert "refused:" in out.stdout and "import torch first" in out.stdout, (out.stdout,
                                                                            out.stderr[-500:])
