"""Calls of the heads that their documentation allows and their ordinary use does not make.

Tolerances are those of tests/test_gpu_heads.py unless a test says otherwise."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import heads_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def heads():
    import ferrisboost_amd as fb

    if not fb.device_available(0):
        pytest.fail("no gfx950 device: the GPU suite needs an MI355X")
    return fb.heads


def test_few_rows_of_many_classes_behind_a_full_launch(heads):
    """2^21 + 5 rows of 16,385 classes: the last launch's 5 rows have no workspace."""
    n, v, tail = (1 << 21) + 5, 16_385, 9
    x = torch.full((n, v), float("-inf"), dtype=torch.bfloat16, device="cuda")  # 69 GB
    rng = np.random.default_rng(1)
    x[-tail:] = torch.from_numpy(rng.normal(size=(tail, v)).astype(np.float32)).cuda()
    u = torch.zeros(n, device="cuda")
    u[-tail:] = torch.from_numpy(rng.random(tail).astype(np.float32)).cuda()
    last = x[-tail:].float().cpu().numpy()
    top_p = torch.full((n,), 0.9, device="cuda")
    for kw, opt in [({"top_p": 0.9}, (1.0, 0, 0.9, 0.0)), ({}, (1.0, 0, 1.0, 0.0)),
                    ({"top_p": top_p}, (1.0, 0, 0.9, 0.0))]:
        c, lp = heads.sample(x, u, **kw)
        want, want_lp = ref.sample(last, u[-tail:].cpu().numpy(), *opt)
        assert np.array_equal(c[-tail:].cpu().numpy(), want)
        got = lp[-tail:].cpu().numpy().astype(np.float64)
        assert (np.abs(got - want_lp) <= np.abs(want_lp) * 2.0 ** -24 + 2.0 ** -45).all()
        assert (c[:-tail] == -1).all() and (lp[:-tail] == float("-inf")).all()
