"""Calls of the training heads that their documentation allows and few programs make."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def heads():
    import ferrisboost_amd as fb

    if not fb.device_available(0):
        pytest.fail("no gfx950 device: the GPU suite needs an MI355X")
    return fb.heads


def test_a_copy_s_weight_decay_moves_no_other_weights(heads):
    import copy

    p = torch.ones(300, device="cuda")
    opt = heads.AdamW([p], lr=0.5, weight_decay=0.0)
    c = copy.copy(opt)
    c.weight_decay = 0.5
    opt.step([torch.zeros_like(p)])
    assert (p == 1.0).all()
    c.step([torch.zeros_like(p)])
    assert (p == 0.75).all()


def test_parameters_that_left_the_device(heads):
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    opt = heads.AdamW([p])
    p.data = p.data.cpu()
    with pytest.raises(ValueError, match="on a GPU"):
        opt.step([torch.zeros(300)])
    with pytest.raises(ValueError, match="changed its type, size or place"):
        opt.step([torch.zeros(300, device="cuda")])
    assert opt.state_dict()["step"] == 0
