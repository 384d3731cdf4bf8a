"""Calls of the heads that their documentation allows and their ordinary use does not make.

Tolerances are those of tests/test_gpu_heads.py unless a test says otherwise."""

from __future__ import annotations

import copy
import io
import pickle

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


def test_copied_and_stored_vocabularies(heads):
    """A copy has a tensor of its own, which the kernels read also when the first one's
    memory holds something else."""
    rng = np.random.default_rng(2)
    voc = heads.Vocabulary([9, 4, 30])
    table = torch.randn(43, 12, device="cuda")
    ids = torch.from_numpy(rng.integers(-1, 30, (700, 3))).cuda()
    want = heads.embed(table, ids, voc, pooled=True)
    grad = heads.embed_grad(want, ids, voc, pooled=True)
    stored = io.BytesIO()
    torch.save({"vocabulary": voc}, stored)
    stored.seek(0)
    copies = [copy.deepcopy(voc), pickle.loads(pickle.dumps(voc)),
              torch.load(stored, weights_only=False)["vocabulary"], copy.copy(voc)]
    for c in copies[:3]:
        assert c.first.data_ptr() != voc.first.data_ptr()
    first, voc = voc.first, None
    first.zero_()
    for c in copies[:3]:
        assert torch.equal(heads.embed(table, ids, c, pooled=True), want)
        assert torch.equal(heads.embed_grad(want, ids, c, pooled=True), grad)
    first.copy_(copies[0].first)
    assert torch.equal(heads.embed(table, ids, copies[3], pooled=True), want)


@pytest.mark.parametrize("backward", [False, True])
def test_a_vocabulary_dropped_while_a_stream_still_reads_it(heads, backward):
    """Its memory is not given out again before the stream has passed the call."""
    voc = heads.Vocabulary([50, 60])
    table = torch.randn(110, 8, device="cuda")
    ids = torch.randint(0, 50, (4000, 2), device="cuda")
    want = heads.embed(table, ids, voc, pooled=True)
    if backward:
        grad, want = want, heads.embed_grad(want, ids, voc, pooled=True)
    a = torch.zeros(1 << 28, device="cuda")  # 1 GiB
    b = torch.empty_like(a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(200):  # some 80 ms
            b.copy_(a)
        got = (heads.embed_grad(grad, ids, voc, pooled=True) if backward
               else heads.embed(table, ids, voc, pooled=True))
        done = s.record_event()
    at = voc.first.data_ptr()
    del voc
    others = [torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(64)]
    assert not done.query()  # (else the rest says nothing)
    assert at not in [o.data_ptr() for o in others]
    s.synchronize()
    assert torch.equal(got, want)


def _sampled(got, want):
    """Classes as they must be, log-probabilities to half a step."""
    (c, lp), (want_c, want_p) = got, want
    assert np.array_equal(c.cpu().numpy(), want_c)
    none, got_p = want_c < 0, lp.cpu().numpy().astype(np.float64)
    assert np.array_equal(got_p[none], want_p[none])
    tol = np.abs(want_p[~none]) * 2.0 ** -24 + 2.0 ** -45
    assert (np.abs(got_p[~none] - want_p[~none]) <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("v", [1, 2, 3, 4, 5, 6, 7, 8, 9, 40, 64, 90, 300, 1000, 3000, 20_000])
def test_infinite_temperatures(heads, v, dtype):
    """Rows of an infinite temperature beside others, whatever kernel takes them: all that
    stays weighs the same, ranks still go by logit."""
    rng = np.random.default_rng(v)
    n = 40 if v <= 3000 else 8
    x = torch.from_numpy((rng.normal(size=(n, v)) * 3).astype(np.float32)).to(dtype).cuda()
    u = torch.from_numpy(rng.random(n).astype(np.float32)).cuda()
    t = np.where(np.arange(n) % 4 == 3, np.float32(0.5), np.float32(np.inf))
    k = rng.choice([0, 1, 2, max(1, v // 2), v], n).astype(np.int32)
    p = rng.choice([0.0, 0.3, 0.9, 1.0], n).astype(np.float32)
    d_t, d_k, d_p = (torch.from_numpy(o).cuda() for o in (t, k, p))
    host = x.float().cpu().numpy()
    for kw, opt in [({}, (t, 0, 1.0, 0.0)), ({"top_k": d_k}, (t, k, 1.0, 0.0)),
                    ({"top_p": d_p}, (t, 0, p, 0.0)),
                    ({"top_k": d_k, "top_p": d_p, "min_p": 1.0}, (t, k, p, 1.0))]:
        _sampled(heads.sample(x, u, temperature=d_t, **kw),
                 ref.sample(host, u.cpu().numpy(), *opt))
    # masked classes stay masked: the same as equal logits at temperature 1
    x[torch.from_numpy(rng.random((n, v)) < 0.3).cuda()] = float("-inf")
    x[0] = float("-inf")
    flat = np.where(x.float().cpu().numpy() == -np.inf, -np.inf, 0.0)
    inf = torch.full((n,), float("inf"), device="cuda")
    _sampled(heads.sample(x, u, temperature=inf),
             ref.sample(flat, u.cpu().numpy(), 1.0, 0, 1.0, 0.0))
    # and next to plus infinity, finite logits weigh nothing
    x[:, v // 2] = float("inf")
    _sampled(heads.sample(x, u, temperature=inf),
             (np.full(n, v // 2), np.zeros(n)))


def test_a_model_takes_uniform_doubles(heads):
    """Model.sample's default kind of uniform numbers: also ones that float32 rounds to 1."""
    import ferrisboost_amd as fb
    from helpers import product_params

    rng = np.random.default_rng(3)
    x = rng.normal(size=(2000, 4)).astype(np.float32)
    m = fb.train(product_params({"objective": "multi:softprob", "num_class": 3, "max_depth": 3}),
                 x, np.digitize(x[:, 0], [-0.5, 0.5]).astype(np.float32), num_boost_round=3)
    u = rng.random(2000)
    u[:3] = [1 - 2.0 ** -30, 1 - 2.0 ** -53, 0.0]
    near = np.minimum(u.astype(np.float32), np.float32(1 - 2.0 ** -24))
    assert np.array_equal(m.sample(x, u), m.sample(x, near))
    assert m.sample(x, u)[0] == 2
    u[5] = 1.0
    with pytest.raises(ValueError, match="in \\[0, 1\\)"):
        m.sample(x, u)


def test_tangents_are_refused_and_their_level_is_not(heads):
    import torch.autograd.forward_ad as fwd

    x = torch.randn(50, 8, device="cuda")
    ids = torch.arange(50, device="cuda")
    u = torch.rand(50, device="cuda")
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: heads.embed(d, ids), lambda: heads.embed_grad(d, ids, 50),
                     lambda: heads.dropout(d, 0.5, 1), lambda: heads.sample(d, u)):
            with pytest.raises(ValueError, match="has a tangent"):
                call()
        assert torch.equal(heads.embed(x, ids), x)
        y = heads.dropout(x.requires_grad_(), 0.5, 1)
        (g,) = torch.autograd.grad(y.sum(), x)
    assert torch.equal(g, heads.dropout(torch.ones_like(x), 0.5, 1))


def test_scales_of_any_finite_size(heads):
    """Positions that take nothing stay zeros up to the largest scale; beyond it the call is
    refused."""
    table = torch.full((4, 8), 2.0 ** -100, device="cuda")
    ids = torch.tensor([[0, -1], [-1, 3], [4, 9]], device="cuda")
    most = float(np.finfo(np.float32).max)
    for scale in (most, -most, 1e-45, 0.0):
        one = torch.tensor(np.float32(scale)) * 2.0 ** -100
        out = heads.embed(table, ids, scale=scale).cpu()
        assert (out[0, 0] == one).all() and (out[1, 1] == one).all()
        assert (out[0, 1] == 0).all() and (out[1, 0] == 0).all() and (out[2] == 0).all()
    grad = torch.ones(3, 2, 8, device="cuda")
    for scale, drop in ((float("inf"), 0.0), (float("nan"), 0.0), (1e39, 0.0), (most, 0.5)):
        with pytest.raises(ValueError, match="finite"):
            heads.embed(table, ids, scale=scale, drop=drop)
        with pytest.raises(ValueError, match="finite"):
            heads.embed_grad(grad, ids, 4, scale=scale, drop=drop)


# (positions of one id, table rows, width, distance of the ones): sorted through memory, in
# buckets, in runs of a few chunks, by columns in chunks of rows, in one chunk, and wide
LONG_RUNS = [(1 << 20, 70_000, 4, 256), (65_536, 5000, 256, 256), (65_536, 5000, 3, 256),
             (208, 5000, 8, 16), (208, 5000, 260, 16), (1 << 22, 9, 4, 16_384),
             (1 << 21, 1000, 2, 16_384), (16_384, 5, 4, 2048), (16_384, 700, 1, 2048),
             (70_000, 9, 256, 16_384), (140_000, 2, 33, 16_384)]


@pytest.mark.parametrize("n, v, dim, every", LONG_RUNS)
def test_sums_of_frequent_ids(heads, n, v, dim, every):
    """2^24, then ones so far apart that every part of the sum is a whole number below 2^24
    or has no other addend: joined in more bits than float32 the sum is exact and rounded
    once, in float32 each of the ones would be lost."""
    x = torch.zeros(n, dim, device="cuda")
    x[::every] = 1.0
    x[0] = 2.0 ** 24
    x[:, ::2] *= -1
    ones = -(-n // every) - 1
    want = torch.full((dim,), float(np.float32(2 ** 24 + ones)))
    want[::2] *= -1
    for token in (0, v - 1):
        ids = torch.full((n,), token, device="cuda")
        got = heads.embed_grad(x, ids, v).cpu()
        assert torch.equal(got[token], want), (got[token][:4], want[:4])
        got[token] = 0
        assert (got == 0).all()


def _close(got, want, magnitude, terms, dtype):
    info = torch.finfo(dtype)
    tol = (np.abs(want) * info.eps / 2 + info.smallest_normal * info.eps / 2
           + magnitude * ((np.maximum(terms, 1) + 1) * 2.0 ** -24 * (1 + info.eps)))
    bad = ~(np.abs(got.detach().cpu().double().numpy() - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4].tolist(), want[bad][:4])


# (rows, columns, table rows, width): few rows and many (both summing kernels), gradients in
# buckets, in several passes, of a table that columns of their own would take whole, and odd
SHARED = [(1, 2, 5, 3), (3, 33, 40, 16), (300, 7, 2000, 33), (9000, 7, 300, 8),
          (1999, 33, 70_000, 5), (20_011, 7, 900, 12), (40_000, 2, 100_000, 20),
          (30_000, 33, 1000, 1), (5000, 33, 600_000, 2)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, t, v, dim", SHARED)
def test_columns_that_share_one_table(heads, n, t, v, dim, dtype):
    """Sums over columns without a vocabulary, by autograd and by the explicit call."""
    rng = np.random.default_rng([n, t, v])
    table = torch.from_numpy(rng.normal(size=(v, dim)).astype(np.float32)).to(dtype).cuda()
    ids = rng.integers(-1, v + 1, (n, t))
    ids[:, 0] = np.minimum(rng.pareto(0.5, n), v - 1).astype(np.int64)  # frequent ones
    d_ids = torch.from_numpy(ids).cuda()
    for drop in (0.0, 0.25):
        tok = ref.tokens(ids, None, v, drop, 5)
        s = 1.5 / (1.0 - drop)
        leaf = table.clone().requires_grad_()
        out = heads.embed(leaf, d_ids, scale=1.5, pooled=True, drop=drop, seed=5)
        want, mag = ref.embed(table.double().cpu().numpy(), tok, s, True)
        _close(out, want, mag, t, dtype)
        grad = torch.from_numpy(rng.normal(size=(n, dim)).astype(np.float32)).to(dtype).cuda()
        out.backward(grad)
        want, mag, terms = ref.embed_grad(grad.double().cpu().numpy(), tok, v, s, True)
        _close(leaf.grad, want, mag, terms[:, None], dtype)
        got = heads.embed_grad(grad, d_ids, v, scale=1.5, pooled=True, drop=drop, seed=5)
        assert torch.equal(got, leaf.grad)


@pytest.mark.parametrize("rows, sizes, dim, pooled, dtype", [
    (40_000, [1000] * 90 + [7, 0, 400], 1024, True, torch.bfloat16),   # 3 groups of columns
    (70_001, [1000, 3, 0, 1000, 500, 8], 20_000, True, torch.float32),  # a column each
    (140_000, [0, 1024, 0], 32_768, True, torch.float16),              # all ids in one column
    (33_000, [900] * 200, 515, False, torch.float16)])                 # 2, an odd width
def test_columns_whose_parts_take_more_than_one_workspace(heads, rows, sizes, dim, pooled, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows)
    voc = heads.Vocabulary(sizes)
    ids = torch.stack([torch.randint(-1, max(s, 1), (rows,), generator=g, device="cuda")
                       for s in sizes], 1).int()
    shape = (rows, dim) if pooled else (rows, len(sizes), dim)
    grad = torch.randn(shape, generator=g, device="cuda", dtype=dtype)
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = heads.embed_grad(grad, ids, voc, pooled=pooled, scale=0.5)
    out = got.numel() * got.element_size()
    parts = max(1 << 30, rows * dim // 2)  # (at least a column's)
    assert torch.cuda.max_memory_allocated() - before <= out + parts + 8 * ids.numel() + (16 << 20)
    first = np.concatenate([[0], np.cumsum(sizes)])
    info = torch.finfo(dtype)
    for t, s in enumerate(sizes):  # a column at a time, in doubles
        at = ((ids[:, t] >= 0) & (ids[:, t] < s)).nonzero()[:, 0]
        tok = ids[at, t].long()
        x = (grad if pooled else grad[:, t])[at].double()
        want = torch.zeros(s, dim, dtype=torch.float64, device="cuda").index_add_(0, tok, x) * 0.5
        mag = torch.zeros_like(want).index_add_(0, tok, x.abs()) * 0.5
        terms = torch.bincount(tok, minlength=s)[:, None] if s else torch.zeros(0, 1, device="cuda")
        tol = (want.abs() * info.eps / 2 + info.smallest_normal * info.eps / 2
               + mag * ((terms + 1) * 2.0 ** -24 * (1 + info.eps)))
        assert ((got[first[t]:first[t + 1]].double() - want).abs() <= tol).all(), t
    assert torch.equal(got, heads.embed_grad(grad, ids, voc, pooled=pooled, scale=0.5))



def test_vocabularies_of_another_type(heads):
    table, ids = torch.zeros(4, 8, device="cuda"), torch.zeros(3, 1, device="cuda")
    for voc in (4, [4], "4"):
        with pytest.raises(ValueError, match="must be a Vocabulary"):
            heads.embed(table, ids, voc)
    with pytest.raises(ValueError, match="whole number"):
        heads.embed_grad(table, ids, [4])


def test_classes_of_margins_that_are_no_numbers(heads):
    """A row whose margins are all NaN has class -1, in binary models (one margin) too."""
    import ferrisboost_amd as fb
    from helpers import product_params

    rng = np.random.default_rng(4)
    x = rng.normal(size=(900, 3)).astype(np.float32)
    y = (x[:, 0] > 0).astype(np.float32)
    u = rng.random(900)
    for params, outputs in (({}, 1), ({"objective": "multi:softprob", "num_class": 2}, 2)):
        m = fb.train(product_params({"max_depth": 2, **params}), x, y, num_boost_round=2)
        base = np.zeros((900, outputs), np.float32)
        base[5], base[6, -1], base[7, -1] = np.nan, np.inf, -np.inf
        c, lp = m.sample(x, u, base_margin=base if outputs > 1 else base[:, 0],
                         return_log_probs=True)
        assert list(c[5:8]) == [-1, 1, 0] and list(lp[5:8]) == [-np.inf, 0, 0]
        assert (np.delete(c, 5) >= 0).all()
