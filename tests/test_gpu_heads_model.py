"""The heads beside the models whose outputs they take: margins as embeddings of leaf
values, leaf gradients as the sums that a tree's leaves hold, classes drawn from
multi:softprob and binary:logistic models, and a run of all of them together."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import heads_ref as ref
from helpers import product_params

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fb():
    import ferrisboost_amd as fb

    if not fb.device_available(0):
        pytest.fail("no gfx950 device: the GPU suite needs an MI355X")
    return fb


def _rows(n, seed, nf=9):
    rng = np.random.default_rng(seed)
    x = rng.normal(size=(n, nf)).astype(np.float32)
    x[rng.random(x.shape) < 0.05] = np.nan
    z = np.nan_to_num(x[:, 0]) - np.nan_to_num(x[:, 1]) * np.nan_to_num(x[:, 2])
    return x, z + 0.3 * rng.normal(size=n)


@pytest.fixture(scope="module")
def classes(fb):
    x, z = _rows(6000, 1)
    y = np.digitize(z, [-1.0, 0.0, 1.0]).astype(np.float32)
    m = fb.train(product_params({"objective": "multi:softprob", "num_class": 4, "max_depth": 4}),
                 x, y, num_boost_round=6)
    return m, x, y


def test_margins_are_embeddings_of_leaf_values(fb):
    x, z = _rows(5000, 2)
    m = fb.train(product_params({"max_depth": 5, "eta": 0.3}), x, (z > 0).astype(np.float32),
                 num_boost_round=15)
    for kw in ({}, {"iteration_range": (3, 11)}):
        leaves = m.predict(x, pred_leaf=True, **kw)
        voc = m.leaf_vocabulary(**kw)
        b, e = kw.get("iteration_range", (0, m.num_trees))
        values = np.concatenate([t["leaf_value"] for t in m.trees()[b:e]]).astype(np.float32)
        assert voc.n_tokens == values.size and voc.n_columns == leaves.shape[1] == e - b
        out = fb.heads.embed(torch.from_numpy(values[:, None]).cuda(),
                             torch.from_numpy(leaves).cuda(), voc, pooled=True)
        want = m.predict(x, output_margin=True, **kw).astype(np.float64) - m.base_margin
        # both sum e - b leaf values in float32, the margin after the intercept
        mag = np.abs(values).max() * (e - b) + abs(m.base_margin)
        assert np.abs(out.cpu().numpy()[:, 0] - want).max() <= 2 * (e - b + 1) * 2.0 ** -24 * mag
    with pytest.raises(ValueError, match="no trees"):
        m.leaf_vocabulary(iteration_range=(4, 4))


def test_a_margin_gradient_by_leaf(fb):
    """The gradient of leaf values is the rows' gradients summed by leaf: the hessians of a
    squared-error tree's leaves are their row counts."""
    x, z = _rows(9000, 3)
    m = fb.train(product_params({"objective": "reg:squarederror", "max_depth": 6}), x,
                 z.astype(np.float32), num_boost_round=4)
    voc = m.leaf_vocabulary()
    leaves = torch.from_numpy(m.predict(x, pred_leaf=True)).cuda()
    counts = fb.heads.embed_grad(torch.ones(9000, 1, device="cuda"), leaves, voc, pooled=True)
    want = np.concatenate([np.where(t["is_leaf"] == 1, t["sum_hess"], 0) for t in m.trees()])
    assert np.array_equal(counts.cpu().numpy()[:, 0], want)


@pytest.mark.parametrize("kw", [{}, {"temperature": 0.5}, {"top_k": 2}, {"top_p": 0.7},
                                {"temperature": 2.0, "min_p": 0.3}, {"temperature": 0.0}])
def test_classes_of_a_model(classes, kw):
    m, x, _ = classes
    rng = np.random.default_rng(5)
    u = rng.random(x.shape[0]).astype(np.float32)
    got, lp = m.sample(x, u, return_log_probs=True, **kw)
    opt = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, **kw}
    want, want_p = ref.sample(m.predict(x, output_margin=True), u, **opt)
    assert got.dtype == np.int64 and np.array_equal(got, want)
    assert (np.abs(lp - want_p) <= np.abs(want_p) * 2.0 ** -24 + 2.0 ** -45).all()
    assert np.array_equal(m.sample(x, u, **kw), want)
    if kw.get("temperature") == 0.0:
        assert np.array_equal(got, m.predict(x).argmax(1))


def test_classes_of_a_binary_model_and_refusals(fb, classes):
    x, z = _rows(3000, 7)
    m = fb.train(product_params({"max_depth": 3}), x, (z > 0).astype(np.float32),
                 num_boost_round=5)
    u = np.random.default_rng(1).random(3000).astype(np.float32)
    got = m.sample(x, u)
    margin = m.predict(x, output_margin=True)
    want, _ = ref.sample(np.stack([np.zeros_like(margin), margin], 1), u, 1.0, 0, 1.0, 0.0)
    assert np.array_equal(got, want)
    assert m.sample(x[:0], u[:0]).shape == (0,)
    for bad, msg in [((u[:5],), "one value for each"), ((u + 1.0,), "in \\[0, 1\\)"),
                     ((np.full(3000, np.nan, np.float32),), "in \\[0, 1\\)")]:
        with pytest.raises(ValueError, match=msg):
            m.sample(x, *bad)
    with pytest.raises(ValueError, match="top_p"):
        m.sample(x, u, top_p=2.0)
    r = fb.train(product_params({"objective": "reg:squarederror", "max_depth": 3}), x,
                 z.astype(np.float32), num_boost_round=2)
    with pytest.raises(ValueError, match="no classes"):
        r.sample(x, u)
    back = fb.Model.from_json(m.to_json())
    assert np.array_equal(back.sample(x, u), got)


def test_large_host_samples(classes):
    m, x, _ = classes
    x = np.resize(x, (150_000, x.shape[1]))
    u = np.random.default_rng(2).random(150_000).astype(np.float32)
    a = m.sample(x, u, top_p=0.9)
    assert np.array_equal(a[:6000], m.sample(x[:6000], u[:6000], top_p=0.9))


def _within(got, want, magnitude, terms):
    """float32 sums of `terms` values, scaled and rounded: see tests/test_gpu_heads.py."""
    tol = np.abs(want) * 2.0 ** -24 + 1e-45 + magnitude * (np.maximum(terms, 1) + 1) * 2.0 ** -24
    return (np.abs(got.detach().cpu().double().numpy() - want) <= tol * (1 + 1e-6)).all()


def test_a_head_on_a_models_leaves(fb, classes):
    """Leaf vectors, dropout and a product to class logits, trained for some steps, each
    stage and each gradient checked; then classes drawn from the logits."""
    m, x, y = classes
    n, d = x.shape[0], 16
    voc = m.leaf_vocabulary()
    ids = m.predict(x, pred_leaf=True)
    leaves = torch.from_numpy(ids).cuda()
    g = torch.Generator(device="cuda").manual_seed(1)
    table = (0.1 * torch.randn(voc.n_tokens, d, generator=g, device="cuda")).requires_grad_()
    weight = torch.randn(d, 4, generator=g, device="cuda").requires_grad_()
    target = torch.from_numpy(y).cuda().long()
    t = leaves.shape[1]
    for step in range(3):
        h = fb.heads.embed(table, leaves, voc, pooled=True, drop=0.1, seed=2 * step)
        h.retain_grad()
        z = fb.heads.dropout(h, 0.2, 2 * step + 1)
        z.retain_grad()
        torch.nn.functional.cross_entropy(z @ weight, target).backward()

        tok = ref.tokens(ids, voc.sizes, voc.n_tokens, 0.1, 2 * step)
        want, mag = ref.embed(table.detach().cpu().double().numpy(), tok, 1 / 0.9, True)
        assert _within(h, want, mag, t)
        stay = torch.from_numpy(ref.kept(2 * step + 1, 0.2, np.arange(n * d))).cuda().reshape(n, d)
        scale = torch.tensor(np.float32(1 / 0.8), device="cuda")
        zero = torch.zeros((), device="cuda")
        assert torch.equal(z, torch.where(stay, h * scale, zero))
        assert torch.equal(h.grad, torch.where(stay, z.grad * scale, zero))
        want, mag, terms = ref.embed_grad(h.grad.cpu().double().numpy(), tok, voc.n_tokens,
                                          1 / 0.9, True)
        assert _within(table.grad, want, mag, terms[:, None])
        with torch.no_grad():
            table -= 0.5 * table.grad
            weight -= 0.5 * weight.grad
        table.grad = weight.grad = None
    with torch.no_grad():
        logits = fb.heads.embed(table, leaves, voc, pooled=True) @ weight
        u = torch.rand(n, generator=g, device="cuda")
        c, lp = fb.heads.sample(logits, u, temperature=0.8, top_p=0.9)
    want, _ = ref.sample(logits.cpu().numpy(), u.cpu().numpy(), 0.8, 0, 0.9, 0.0)
    assert np.array_equal(c.cpu().numpy(), want) and (lp <= 0).all()
