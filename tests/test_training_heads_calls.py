"""Calls of the training heads that need no device: what they refuse, and what they leave to
others that share their tensors."""

from __future__ import annotations

import copy
import pickle
import struct

import numpy as np
import pytest
import torch

from ferrisboost_amd import _native as N
from ferrisboost_amd import heads


def _optimizer(sizes=(3, 300), bits=32, **kw):
    """An optimizer of float32 parameters on the host, which can do everything but step."""
    heads._need_torch()
    opt = object.__new__(heads.AdamW)
    opt.params = [torch.zeros(n) for n in sizes]
    opt.lr, opt.betas, opt.eps, opt.bits, opt.seed = 0.1, (0.9, 0.999), 1e-8, bits, 0
    opt._parts, opt.weight_decay = None, kw.pop("weight_decay", 0.1)
    blocks = [-(-n // 256) for n in sizes]
    opt.first = [256 * sum(blocks[:i]) for i in range(len(sizes))]
    opt._sizes, opt._types = list(sizes), [torch.float32] * len(sizes)
    opt._parts = [x for i, n in enumerate(sizes)
                  for x in (0, 0, 0, n, opt.first[i], opt.weight_decay[i], 0)]
    opt.mean, opt.square = (torch.zeros(256 * sum(blocks),
                                        dtype=torch.uint8 if bits == 8 else torch.float32)
                            for _ in range(2))
    opt.scales = torch.zeros((2, sum(blocks)), dtype=torch.uint8) if bits == 8 else None
    opt.masters = [None] * len(sizes)
    opt._clock = torch.tensor([0, 0x3FF0000000000000, 0x3FF0000000000000, 0])
    opt._streams = set()
    for k, v in kw.items():
        setattr(opt, k, v)
    return opt


@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))])
def test_weight_decay_of_a_copy_is_its_own(how):
    """What a step packs for the first one stays, whichever of the two is set."""
    opt = _optimizer()
    c = how(opt)
    c.weight_decay = 0.75
    assert opt.weight_decay == (0.1, 0.1) and opt._parts[5::7] == [0.1, 0.1]
    assert c.weight_decay == (0.75, 0.75) and c._parts[5::7] == [0.75, 0.75]
    opt.weight_decay = [0.5, 0.25]
    assert opt._parts[5::7] == [0.5, 0.25] and c._parts[5::7] == [0.75, 0.75]


def test_parameters_that_left_the_optimizer_s_device():
    """Parameters and gradients moved together: the state has not."""
    opt = _optimizer()

    class On0:
        @staticmethod
        def get_device():
            return 0

    opt.mean = On0()
    with pytest.raises(ValueError, match="on a GPU"):
        opt.step([torch.ones_like(p) for p in opt.params])


def test_a_parameter_with_a_tangent_is_refused():
    """A step would move its value and leave its tangent as it was."""
    import torch.autograd.forward_ad as fwd

    opt = _optimizer()
    with fwd.dual_level():
        d = fwd.make_dual(opt.params[1], torch.ones_like(opt.params[1]))
        opt.params[1] = d
        with pytest.raises(ValueError, match="parameter 1 has a tangent"):
            opt.step([torch.ones_like(p) for p in opt.params])
        with pytest.raises(ValueError, match="parameter 0 has a tangent"):
            heads.AdamW([d])
        mean = fwd.make_dual(opt.mean, torch.ones_like(opt.mean))
        with pytest.raises(ValueError, match="mean has a tangent"):
            opt.load_state_dict({"step": 0, "mean": mean, "square": opt.square})


@pytest.mark.parametrize("call, msg", [
    (lambda o: heads._eps(None), "eps must be a number"),
    (lambda o: heads._drop("half"), "drop must be a number"),
    (lambda o: heads._scale([1.0, 2.0]), "scale must be a number"),
    (lambda o: heads._scale(10 ** 400), "scale must be a number"),
    (lambda o: heads.check_options(None, 0, 1.0, 0.0), "temperature must be a number"),
    (lambda o: heads.check_options(1.0, 0, torch.ones(2), 0.0), "top_p must be a number"),
    (lambda o: heads.AdamW([torch.zeros(3)], betas=0.9), "betas must be two numbers"),
    (lambda o: heads.AdamW([torch.zeros(3)], betas=(0.9, None)), "betas must be two numbers"),
    (lambda o: heads.AdamW([torch.zeros(3)], eps=None), "eps must be a number"),
    (lambda o: heads.AdamW(3), "params must be"),
    (lambda o: setattr(o, "weight_decay", np.array([0.1, 0.1])), "weight_decay must be"),
    (lambda o: setattr(o, "weight_decay", None), "weight_decay must be"),
    (lambda o: setattr(o, "weight_decay", [0.1, None]), "weight_decay must be"),
    (lambda o: (setattr(o, "lr", None), o._lr()), "lr must be a number"),
    (lambda o: o.step(5), "grads must be a list"),
    (lambda o: o.load_state_dict(None), "a state must be a dict"),
    (lambda o: o.load_state_dict({"step": 0, "mean": o.mean, "square": o.square, "decays": 1.0}),
     "decays must be two numbers"),
    (lambda o: o.load_state_dict({"step": 0, "mean": o.mean, "square": o.square, "masters": 1}),
     "masters must be a list")])
def test_arguments_of_another_kind_are_value_errors(call, msg):
    with pytest.raises(ValueError, match=msg):
        call(_optimizer())


@pytest.mark.parametrize("sparse", [
    lambda x: x.to_sparse(), lambda x: x.to_sparse_csr(),
    lambda x: torch.nested.nested_tensor([x[0], x[1]])])
def test_tensors_that_are_not_dense_are_refused(sparse):
    x = sparse(torch.ones(4, 3))
    for call in (lambda: heads.layer_norm(x), lambda: heads.dropout(x, 0.5, 1),
                 lambda: heads.AdamW([x])):
        with pytest.raises(ValueError, match="must be dense"):
            call()


def test_sparse_gradients_are_refused():
    """What an embedding with sparse=True leaves in .grad, say."""
    opt = _optimizer()
    grads = [torch.ones(3), torch.ones(300).to_sparse()]
    opt.mean = grads[0]  # (on the gradients' device, as it is on a GPU)
    with pytest.raises(ValueError, match="gradient 1 must be dense"):
        opt._gradient(1, opt.params[1], grads[1])
    with pytest.raises(ValueError, match="gradient"):
        opt.step(grads)


@pytest.mark.parametrize("v", [2.5, 1e-3, np.float32(7.25), torch.tensor(0.5), -0.1,
                               torch.tensor([1, 2])])
def test_whole_numbers_have_no_fraction(v):
    with pytest.raises(ValueError, match="n must be a whole number"):
        heads._whole(v, "n")
    assert heads._whole(3.0, "n") == heads._whole(np.int64(3), "n") == 3
    assert heads._whole(torch.tensor(3), "n") == heads._whole(True, "n") + 2 == 3


# 100 rows of 8 float32: 3200 bytes; their statistics 800, weights 32
ROWS, CELLS = 100, 8


@pytest.mark.parametrize("over", ["dx", "out", "stats"])
@pytest.mark.parametrize("shift", [-3196, -4, 4, 3196])
def test_layer_norm_outputs_that_overlap_an_input_in_part(over, shift):
    """Rows would be read after others have been written over them."""
    L, a = N.hip(), heads._NORM.pack(ROWS, CELLS, 0, 0, 1e-5)
    x, g = 0x10000, 0x20000
    if over == "dx":
        for dx, msg in ((x + shift, "dx must not"), (g + shift, "dx must not")):
            with pytest.raises(ValueError, match=msg):
                N.check_hip(L.fbh_layer_norm_grad(0, a, g, x, 0x30000, None, dx, None, None, None,
                                                  0, None))
    elif over == "out":
        with pytest.raises(ValueError, match="out must be x or apart"):
            N.check_hip(L.fbh_layer_norm(0, a, x, None, None, x + shift, None, None))
    else:
        at = x + (shift if shift > 0 else shift % 800 - 800)
        with pytest.raises(ValueError, match="stats must not"):
            N.check_hip(L.fbh_layer_norm(0, a, x, None, None, 0x30000, at, None))
        with pytest.raises(ValueError, match="stats must not"):
            N.check_hip(L.fbh_layer_norm(0, a, x, None, None, x, at, None))


def test_layer_norm_outputs_that_overlap_weights_or_statistics():
    L, a = N.hip(), heads._NORM.pack(ROWS, CELLS, 0, 0, 1e-5)
    x, g, out = 0x10000, 0x20000, 0x30000
    for w, b in ((out + 3196, None), (out - 28, None), (0x40000, out)):
        with pytest.raises(ValueError, match="out must not overlap a weight"):
            N.check_hip(L.fbh_layer_norm(0, a, x, w, b, out, None, None))
    for stats, w in ((out - 796, None), (out + 3196, None), (0x40000, out + 3196)):
        with pytest.raises(ValueError, match="dx must not"):
            N.check_hip(L.fbh_layer_norm_grad(0, a, g, x, stats, w, out, None, None, None, 0,
                                              None))


def test_states_of_other_sizes_are_refused():
    """Sizes of the same padded total: moments would land in other cells."""
    for sizes, other in (((300, 100), (100, 300)), ((1,), (256,)), ((300, 5), (300, 6))):
        a, b = _optimizer(sizes), _optimizer(other)
        assert a.mean.shape == b.mean.shape
        state = a.state_dict()
        assert state["sizes"] == list(sizes)
        with pytest.raises(ValueError, match="parameters of"):
            b.load_state_dict(state)
        with pytest.raises(ValueError, match="sizes must be a list"):
            b.load_state_dict({**state, "sizes": 3})


def test_states_hold_their_seed():
    for bits in (8, 32):
        state = _optimizer(bits=bits, seed=2 ** 64 - 1).state_dict()
        assert state["seed"] == 2 ** 64 - 1
        for bad in (-1, 1 << 64, "none"):
            with pytest.raises(ValueError, match="seed"):
                _optimizer(bits=bits).load_state_dict({**state, "seed": bad})


def test_learning_rates_on_the_device_are_kept_for_a_step_s_stream(monkeypatch):
    """Each tensor that is set, on each stream that reads it: also one that is replaced while a
    step of its stream is still to come."""
    recorded = []

    class Native:
        @staticmethod
        def fbh_adamw_step(*args):
            return 0

    opt = _optimizer()
    now = [5]
    monkeypatch.setattr(heads, "_raw_stream", lambda device: now[0])
    monkeypatch.setattr(heads, "_L", Native)
    monkeypatch.setattr(torch.Tensor, "record_stream",
                        lambda self, stream: recorded.append((float(self), stream)))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: now[0])
    monkeypatch.setattr(heads.AdamW, "_used_on", lambda self, stream: None)
    monkeypatch.setattr(heads.AdamW, "_lr", lambda self: (0.0, 64))
    grads = [torch.ones_like(p) for p in opt.params]

    def step(o=opt):
        o.step(grads)

    step()
    assert not recorded  # (a number)
    opt.lr = torch.tensor([1.0])
    step()
    step()
    assert recorded == [(1.0, 5)]
    now[0] = 6
    step()
    opt.lr = torch.tensor([2.0])
    step()
    assert recorded == [(1.0, 5), (1.0, 6), (2.0, 6)]
    for c in (copy.copy(opt), copy.deepcopy(opt)):
        step(c)
        assert recorded.pop() == (2.0, 6) and len(recorded) == 3


def _step_arguments(params, lr_at, n=256):
    """fbh_adamw and float32 tensors of n cells for the C entry."""
    a = heads._ADAMW.pack(32, 1e-8, 0.9, 0.999, 0.0, lr_at, 0, 256 * len(params), 0x100000,
                          0x200000, 0, 0x300000)
    return a, b"".join(struct.pack("PPPQQfI", p, 0x400000, 0, n, 256 * i, 0.0, 0)
                       for i, p in enumerate(params)), len(params)


@pytest.mark.parametrize("lr_at", [0x1000, 0x13FC, 0x3004, 0x0FFD, 0x33FF])
def test_a_learning_rate_in_a_parameter_s_memory_is_refused(lr_at):
    """Some cells would be stepped by what it was and some by what it becomes."""
    with pytest.raises(ValueError, match="learning rate overlaps a parameter"):
        N.check_hip(N.hip().fbh_adamw_step(0, *_step_arguments([0x1000, 0x3000], lr_at), None))


def test_split_takes_a_flat_tensor_of_the_state_s_size():
    opt = _optimizer()
    assert [v.shape for v in opt.split(opt.mean)] == [p.shape for p in opt.params]
    for bad in (torch.zeros(5), torch.zeros(opt.mean.numel() + 1), opt.mean[None], None, [0.0]):
        with pytest.raises(ValueError, match="flat must be a tensor"):
            opt.split(bad)
