"""Calls of the training heads that their documentation allows and few programs make."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import norm_bounds
import training_ref as ref

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


def test_sparse_gradients_are_refused(heads):
    table = torch.nn.Embedding(50, 8, sparse=True, device="cuda")
    bias = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    opt = heads.AdamW([bias, table.weight])
    before = table.weight.detach().clone()
    (table(torch.tensor([3, 4, 3], device="cuda")) + bias).sum().backward()
    assert table.weight.grad.is_sparse
    with pytest.raises(ValueError, match="gradient 1 must be dense"):
        opt.step()
    assert opt.state_dict()["step"] == 0 and torch.equal(table.weight, before)
    with pytest.raises(ValueError, match="gradient 1 must be dense"):
        opt.step([bias.grad, table.weight.grad.to_dense().to_sparse_csr()])
    table.weight.grad = table.weight.grad.to_dense()
    opt.step()
    moved = (table.weight != before).any(1)
    assert moved[3] and moved[4]
    with pytest.raises(ValueError, match="x must be dense"):
        heads.layer_norm(before.to_sparse())
    with pytest.raises(ValueError, match="x must be dense"):
        heads.layer_norm(before.to_sparse_csr())


@pytest.mark.parametrize("bits", [32, 8])
def test_states_of_other_sizes_are_refused(heads, bits):
    """Of parameters whose padded sizes add up to the same."""
    a = heads.AdamW([torch.ones(n, device="cuda") for n in (300, 100)], bits=bits)
    b = heads.AdamW([torch.ones(n, device="cuda") for n in (100, 300)], bits=bits)
    a.step([torch.ones_like(p) for p in a.params])
    with pytest.raises(ValueError, match="parameters of"):
        b.load_state_dict(a.state_dict())
    assert b.state_dict()["step"] == 0 and (b.mean == 0).all()
    state = a.state_dict()
    del state["sizes"]  # (one that was stored before states held them)
    heads.AdamW([torch.ones(n, device="cuda") for n in (300, 100)],
                bits=bits).load_state_dict(state)


def test_a_resumed_run_rounds_as_the_first_one_would(heads):
    """Moments of 8 bits are rounded by bits of the seed, which a state brings with it."""
    grads = [torch.randn(3000, device="cuda") for _ in range(6)]
    p = torch.randn(3000, device="cuda")
    opt = heads.AdamW([p], lr=0.01, bits=8, seed=77)
    for g in grads[:3]:
        opt.step([g])
    q = p.clone()
    again = heads.AdamW([q], lr=0.01, bits=8)
    again.load_state_dict(opt.state_dict())
    assert again.seed == 77
    for g in grads[3:]:
        opt.step([g])
        again.step([g])
    assert torch.equal(p, q) and torch.equal(opt.mean, again.mean)
    assert torch.equal(opt.square, again.square) and torch.equal(opt.scales, again.scales)
    old = opt.state_dict()
    del old["seed"]  # (one that was stored before states held it)
    other = heads.AdamW([q], bits=8, seed=5)
    other.load_state_dict(old)
    assert other.seed == 5


def test_a_learning_rate_that_is_replaced_while_a_stream_still_reads_it(heads):
    """Its memory is not given out again before the stream has passed the step."""
    p = torch.randn(3000, device="cuda")
    q, grad = p.clone(), torch.randn(3000, device="cuda")
    heads.AdamW([q], lr=0.25).step([grad])
    opt = heads.AdamW([p], lr=0.1)
    a = torch.zeros(1 << 28, device="cuda")  # 1 GiB
    b = torch.empty_like(a)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):  # (its state has been used there before)
        opt.lr = 0.0
        opt.step([torch.zeros_like(p)])
    opt.load_state_dict({**opt.state_dict(), "step": 0, "decays": [1.0, 1.0]})
    opt.mean.zero_()
    opt.square.zero_()
    opt.lr = torch.full((1,), 0.25, device="cuda")
    at = opt.lr.data_ptr()
    s.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(200):  # some 80 ms
            b.copy_(a)
        opt.step([grad])
        done = s.record_event()
    opt.lr = 0.1
    del opt
    others = [torch.zeros(1, device="cuda") for _ in range(600)]
    assert not done.query()  # (else the rest says nothing)
    assert at not in {o.data_ptr() for o in others}
    s.synchronize()
    assert torch.equal(p, q)


def _off(got, want, off):
    """Half a step of got's type more than `off`, in numpy's doubles."""
    info = torch.finfo(got.dtype)
    return np.abs(got.cpu().double().numpy() - want) <= (
        off * (1 + info.eps) + np.abs(want) * info.eps / 2 + info.smallest_normal * info.eps / 2)


# 1024 parts of a weight's sums, 781 and 512; 128 of some rows and of all
@pytest.mark.parametrize("n, dim", [(200_000, 64), (300_001, 7), (100_000, 64), (30_000, 1000),
                                    (6000, 130), (70_000, 260), (3001, 4100)])
def test_layer_norm_gradients_of_many_rows(heads, n, dim):
    rng = np.random.default_rng([n, dim])
    x = torch.from_numpy(rng.normal(size=(n, dim)).astype(np.float32) +
                         rng.normal(size=(n, 1)).astype(np.float32)).cuda()
    g = torch.from_numpy(rng.normal(size=(n, dim)).astype(np.float32)).cuda()
    w = torch.from_numpy((1 + rng.normal(size=dim) / 2).astype(np.float32)).cuda()
    _, stats = heads.layer_norm(x, w, stats=True)
    got = heads.layer_norm_grad(g, x, stats, w)
    want = norm_bounds.layer_norm_grad(g.cpu().numpy(), x.cpu().numpy(), w.cpu().numpy(), 1e-5)
    for a, (value, off), what in zip(got, want, ("dx", "dw", "db")):
        assert _off(a, value, off).all(), what


@pytest.mark.parametrize("n, dim", [(1 << 19, 16_386), (1 << 21, 4098), (1 << 29, 4)])
def test_weights_sums_of_any_number_of_rows(heads, n, dim):
    """Equal terms, whose float32 sum is off the same way at each addition, by a half step of the
    sum at most, and the rounding of the result. (In a chain of 8192 rows, as there would be, sums
    of this number are off by 1.2e-4.)"""
    c = float(np.float32(1.9545904397964478))
    x = torch.full((n, dim), c, device="cuda")  # up to 34 GB
    x[:, dim // 2:] = -c
    stats = torch.zeros((n, 2), device="cuda")  # mean 0, deviation 1
    stats[:, 1] = 1.0
    w = torch.ones(dim, device="cuda")
    _, dw, db = heads._layer_norm_grad(heads._norm_of(x, w, 1.0), x, x, stats, w,
                                       (False, True, True))
    del x
    sign = torch.where(torch.arange(dim, device="cuda") < dim // 2, 1.0, -1.0).double()
    off = ref.ULP * (norm_bounds.weight_path(n, dim) + 1) * n
    assert float((db.double() - sign * (n * c)).abs().max()) <= off * c
    assert float((dw.double() - n * c * c).abs().max()) <= off * c * c
    torch.cuda.empty_cache()


def test_gradients_to_experts_rows_beyond_2_31_cells(heads):
    n, k, dim = 600_001, 2, 2048
    g = torch.Generator(device="cuda").manual_seed(4)
    ids = torch.randint(-1, 64, (n, k), device="cuda", generator=g)
    r = heads.Routes(ids, 64)
    x = torch.randn(n, dim, device="cuda", dtype=torch.bfloat16, generator=g)
    w = torch.rand(n, k, device="cuda", generator=g)
    y = heads.to_experts(x, r)
    dy, dw = heads.from_experts_grad(x, y, r, w)
    end = int(r.starts[-1])
    assert end * dim > (1 << 31) + 1000 * dim
    far = (1 << 31) // dim
    at = torch.cat([torch.arange(0, 100), torch.arange(far - 50, far + 50),
                    torch.arange(end - 100, end)]).cuda()
    position = r.order[at].long()
    row = position // k
    want = (w.view(-1)[position][:, None] * x[row].float()).bfloat16()
    assert torch.equal(dy[at], want) and (dy[end:] == 0).all()
    # (a lane's products in turn, a piece more, 6 levels of lanes)
    dots = (x[row].double() * y[at].double()).sum(1)
    assert ((dw.view(-1)[position] - dots).abs() <= dots * ref.ULP * (dim / 64 + 8 + 7)).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_small_weight_decay_is_not_rounded(heads, bits):
    """Without a gradient a step is one product that is taken from the weight: the result is off
    by half a step of the weight, and by what the product itself is, 3 half steps of it."""
    rng = np.random.default_rng(3)
    w = np.concatenate([rng.uniform(1, 2, 60_000), rng.normal(size=20_000)]).astype(np.float32)
    for lr, decay in ((1e-5, 0.01), (1e-6, 0.3), (1e-3, 0.1), (0.5, 0.125)):
        p = torch.from_numpy(w).cuda()
        heads.AdamW([p], lr=lr, weight_decay=decay, bits=bits).step([torch.zeros_like(p)])
        part = lr * float(np.float32(decay)) * w.astype(np.float64)
        want = w - part
        off = np.spacing(np.abs(want).astype(np.float32)).astype(np.float64) / 2
        got = p.cpu().double().numpy()
        assert (np.abs(got - want) <= off + 4 * ref.ULP * np.abs(part)).all(), (lr, decay)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinite_weights_decay_to_themselves(heads, bits, dtype):
    """As those of masked classes may be."""
    inf = float("inf")
    for decay in (0.0, 0.25):
        p = torch.tensor([inf, -inf, 1.0, float("nan"), -2.0], device="cuda").to(dtype)
        opt = heads.AdamW([p], lr=0.5, weight_decay=decay, bits=bits)
        opt.step([torch.zeros_like(p)])
        keep = 1 - 0.5 * decay
        assert p.tolist()[:3] == [inf, -inf, keep] and p[3].isnan() and float(p[4]) == -2 * keep


def test_leaves_of_two_trees_have_experts_of_their_own(heads):
    """As a program with an expert a leaf numbers them: by the vocabulary."""
    rng = np.random.default_rng(11)
    voc = heads.Vocabulary([15, 15, 7])
    leaves = rng.integers(7, 15, (400, 2)).astype(np.float32)
    ids = torch.from_numpy(leaves).cuda() + voc.first[:2]
    routes = heads.Routes(ids, int(voc.sizes[:2].sum()))
    starts = routes.starts.tolist()
    assert starts[-1] == 800 and len(starts) == 31
    order = routes.order.cpu().numpy()
    for expert, (a, b) in enumerate(zip(starts, starts[1:])):
        want = np.flatnonzero(leaves[:, expert // 15] == expert % 15) * 2 + expert // 15
        assert np.array_equal(order[a:b], want)
