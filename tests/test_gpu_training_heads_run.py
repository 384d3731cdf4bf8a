"""The training heads together, as a program that trains on a model's leaves uses them: eager,
captured into graphs, on other streams."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import training_ref as ref

pytestmark = pytest.mark.gpu

EPS = 1e-5


@pytest.fixture(scope="module")
def heads():
    import ferrisboost_amd as fb

    if not fb.device_available(0):
        pytest.fail("no gfx950 device: the GPU suite needs an MI355X")
    return fb.heads


@pytest.fixture(scope="module")
def leaves():
    """A small model's leaf ids of 700 rows, its trees' nodes, and the labels."""
    import ferrisboost_amd as fb
    from helpers import product_params

    rng = np.random.default_rng(5)
    x = rng.normal(size=(700, 6)).astype(np.float32)
    y = np.digitize(x[:, 0] + x[:, 1], [-0.6, 0.6]).astype(np.float32)
    m = fb.train(product_params({"objective": "multi:softprob", "num_class": 3, "max_depth": 3}),
                 x, y, num_boost_round=4)
    return m.predict(x, pred_leaf=True), m.leaf_vocabulary(), torch.from_numpy(y).long()


def _parameters(voc, dim, experts, seed=0):
    g = torch.Generator().manual_seed(seed)
    shapes = {"table": (voc.n_tokens, dim), "experts": (experts, dim, dim), "gain": (dim,),
              "bias": (dim,), "out": (dim, 3)}
    p = {k: torch.randn(s, generator=g) * (0.3 if len(s) > 1 else 0.1) for k, s in shapes.items()}
    p["gain"] += 1.0
    return p


def _experts_products(rows, starts, weight):
    """Each expert's product on its rows."""
    return torch.cat([rows[a:b] @ w for a, b, w in zip(starts, starts[1:], weight)]
                     + [rows[starts[-1]:] * 0])


def _forward(heads, p, ids, voc, chosen, experts):
    """Vectors of a row's leaves, through the experts of two of them, normalised, to classes."""
    h = heads.embed(p["table"], ids, voc, pooled=True, drop=0.1, seed=3)
    routes = heads.Routes(chosen, experts)
    rows = heads.to_experts(h, routes)
    y = _experts_products(rows, routes.starts.tolist(), p["experts"])
    weights = torch.softmax(h[:, :2], 1)
    h = h + heads.from_experts(y, routes, weights)
    return heads.layer_norm(h, p["gain"], p["bias"], eps=EPS) @ p["out"]


def _forward_64(p, ids, voc, chosen, experts):
    """The same in doubles, from torch's elementary operations on the host."""
    import heads_ref

    tok = torch.from_numpy(heads_ref.tokens(ids.cpu().numpy(), voc.sizes, voc.n_tokens, 0.1, 3))
    rows = p["table"][tok.clamp(min=0)] * (tok >= 0).unsqueeze(-1)
    h = rows.sum(1) / 0.9
    weights = torch.softmax(h[:, :2], 1)
    c = chosen.cpu().long()
    add = torch.zeros_like(h)
    for j in range(c.shape[1]):
        ok = (c[:, j] >= 0) & (c[:, j] < experts)
        y = torch.stack([h[i] @ p["experts"][c[i, j]] if ok[i] else h[i] * 0
                         for i in range(len(h))])
        add = add + weights[:, j:j + 1] * y
    h = h + add
    d = h - h.mean(1, keepdim=True)
    h = d / (d.square().mean(1, keepdim=True) + EPS).sqrt()
    return (h * p["gain"] + p["bias"]) @ p["out"]


def test_a_head_s_gradients_and_its_training(heads, leaves):
    """Gradients of a loss through all of the operators, against doubles: seven operators,
    the products and the softmax among them, each off by at most 128 half steps of float32 of
    the magnitudes that it adds up, which are at most 4 times as large (in the 2-norm) as their
    sums: 2^-24 * 7 * 128 * 4. Then steps on it run, and move every parameter."""
    ids, voc, labels = leaves
    ids = torch.from_numpy(ids).cuda()
    labels = labels.cuda()
    experts = 15
    chosen = ids[:, :2].contiguous()
    chosen[:30, 1] = -1  # without an expert
    start = _parameters(voc, 24, experts)
    p = {k: v.cuda().requires_grad_() for k, v in start.items()}
    loss = torch.nn.functional.cross_entropy(_forward(heads, p, ids, voc, chosen, experts), labels)
    loss.backward()
    q = {k: v.double().requires_grad_() for k, v in start.items()}
    want = torch.nn.functional.cross_entropy(_forward_64(q, ids, voc, chosen, experts),
                                             labels.cpu())
    want.backward()
    bound = ref.ULP * 7 * 128 * 4
    assert abs(float(loss) - float(want)) <= bound * float(want)
    for k in p:
        off = (p[k].grad.cpu().double() - q[k].grad).norm() / q[k].grad.norm()
        assert off <= bound, (k, float(off))
    for bits in (32, 8):
        opt = heads.AdamW(list(p.values()), lr=1e-2, bits=bits, weight_decay=[0.0] * 5)
        before = {k: v.detach().clone() for k, v in p.items()}
        for _ in range(3):
            opt.zero_grad()
            torch.nn.functional.cross_entropy(_forward(heads, p, ids, voc, chosen, experts),
                                              labels).backward()
            opt.step()
        for k, v in p.items():
            assert torch.isfinite(v).all() and not torch.equal(v, before[k])


def _step(heads, s):
    """One training step by the explicit gradients, as a program captures it: a table's vectors
    through a norm and weighted experts (the identity) towards a target."""
    voc, r = s["voc"], None
    h = heads.embed(s["table"], s["ids"], voc, pooled=True, drop=0.1, seed=7)
    y, stats = heads.layer_norm(h, s["gain"], s["bias"], eps=EPS, stats=True)
    r = heads.Routes(s["chosen"], 9)
    rows = heads.to_experts(y, r)
    out = heads.from_experts(rows, r, s["weights"])
    grad = out - s["target"]
    d_rows, d_weights = heads.from_experts_grad(grad, rows, r, s["weights"])
    dy = heads.from_experts(d_rows, r)
    dh, d_gain, d_bias = heads.layer_norm_grad(dy, h, stats, s["gain"])
    d_table = heads.embed_grad(dh, s["ids"], voc, pooled=True, drop=0.1, seed=7)
    s["opt"].step([d_table, d_gain, d_bias])
    return [out, d_weights, dh, r.order, r.place, r.starts]


def _setup(heads, n, dim, bits, dtype, lr):
    g = torch.Generator(device="cuda").manual_seed(n + dim)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    voc = heads.Vocabulary([40, 7, 300])
    s = {"voc": voc, "ids": torch.randint(-1, 40, (n, 3), generator=g, device="cuda"),
         "chosen": torch.randint(-1, 9, (n, 2), generator=g, device="cuda", dtype=torch.int32),
         "weights": torch.rand((n, 2), generator=g, device="cuda"),
         "table": rand(voc.n_tokens, dim).to(dtype), "target": rand(n, dim).to(dtype),
         "gain": torch.ones(dim, device="cuda"), "bias": torch.zeros(dim, device="cuda")}
    s["opt"] = heads.AdamW([s["table"], s["gain"], s["bias"]], lr=lr, bits=bits, seed=5)
    return s


@pytest.mark.parametrize("n, dim, bits, dtype", [
    (1, 8, 32, torch.float32), (300, 24, 8, torch.float32), (5000, 33, 8, torch.bfloat16),
    (9000, 1024, 32, torch.bfloat16), (700, 9000, 8, torch.float16)])
def test_captured_training_steps(heads, n, dim, bits, dtype):
    """Replays go on as eager steps do, bit by bit: counts of steps, random bits and learning
    rates are the device's. Eager work and synchronisation come between the replays."""
    lr, lr2 = (torch.full((1,), 0.01, device="cuda") for _ in range(2))
    a, b = _setup(heads, n, dim, bits, dtype, lr), _setup(heads, n, dim, bits, dtype, lr2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _step(heads, a)
    torch.cuda.current_stream().wait_stream(s)
    _step(heads, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(heads, a)
    for i in range(5):
        lr.fill_(0.01 / (i + 1))
        lr2.fill_(0.01 / (i + 1))
        graph.replay()
        want = _step(heads, b)
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y), i
        for k in ("table", "gain", "bias"):
            assert torch.equal(a[k], b[k]), (i, k)
        for x, y in zip(a["opt"]._tensors(), b["opt"]._tensors()):
            assert torch.equal(x, y), i
        # an eager call on the same state and other work in between
        if i % 2:
            _step(heads, a)
            _step(heads, b)
        torch.randn(1000, 1000, device="cuda") @ torch.randn(1000, 1000, device="cuda")
        torch.cuda.synchronize()


@pytest.mark.parametrize("sizes", [[300_000_0, 5], [70] * 150, [1 << 22, 3, 1 << 20]])
def test_captured_steps_of_many_and_large_parameters(heads, sizes):
    """Several launches a step, and the clock in a launch of its own."""
    g = torch.Generator(device="cuda").manual_seed(1)
    make = lambda: [torch.randn(n, generator=g, device="cuda") for n in sizes]  # noqa: E731
    p = make()
    q = [x.clone() for x in p]
    grads = make()
    a, b = heads.AdamW(p, bits=8, lr=0.1), heads.AdamW(q, bits=8, lr=0.1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step(grads)
    assert a.state_dict()["step"] == 0
    for i in range(4):
        graph.replay()
        b.step(grads)
        torch.cuda.synchronize()
        assert a.state_dict()["step"] == b.state_dict()["step"] == i + 1
        for x, y in zip(p + a._tensors(), q + b._tensors()):
            assert torch.equal(x, y)
        for x in grads:
            x.mul_(0.5)
    assert int(a._clock[3]) == 0


def test_on_another_stream(heads):
    """Tensors and routes of a stream of its own, read by a second one that waits for it."""
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    x = torch.randn(4000, 96, device="cuda")
    ids = torch.randint(-1, 7, (4000, 2), device="cuda")
    r = heads.Routes(ids, 7)
    want = heads.from_experts(heads.layer_norm(heads.to_experts(x, r)), r)
    for u in (s, t):
        u.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        r2 = heads.Routes(ids, 7)
        rows = heads.layer_norm(heads.to_experts(x, r2))
    t.wait_stream(s)
    with torch.cuda.stream(t):
        got = heads.from_experts(rows, r2)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("what", ["routes", "optimizer"])
def test_dropped_while_a_stream_still_reads_it(heads, what):
    """Their memory is not given out again before the stream has passed the call."""
    x = torch.randn(3000, 64, device="cuda")
    ids = torch.randint(0, 5, (3000, 1), device="cuda")
    grad = torch.randn_like(x)
    if what == "routes":
        kept = heads.Routes(ids, 5)
        call = lambda k: heads.to_experts(x, k)  # noqa: E731
        want = call(kept)
    else:
        y = x.clone()
        kept, want = heads.AdamW([x], lr=0.1, bits=8), y

        def call(k):
            k.step([grad])
            return x

        heads.AdamW([y], lr=0.1, bits=8).step([grad])
    at = [k.data_ptr() for k in kept._tensors()]
    sizes = [(k.shape, k.dtype) for k in kept._tensors()]
    a = torch.zeros(1 << 28, device="cuda")  # 1 GiB
    b = torch.empty_like(a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(200):  # some 80 ms
            b.copy_(a)
        got = call(kept)
        done = s.record_event()
    del kept
    others = [torch.zeros(z, dtype=t, device="cuda") for z, t in sizes for _ in range(16)]
    assert not done.query()  # (else the rest says nothing)
    assert not set(at) & {o.data_ptr() for o in others}
    s.synchronize()
    assert torch.equal(got, want)


def test_refusals(heads):
    x = torch.randn(4, 6, device="cuda")
    w, ids = torch.ones(6, device="cuda"), torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    r = heads.Routes(ids, 3)
    rows = heads.to_experts(x, r)
    _, stats = heads.layer_norm(x, stats=True)
    for call, msg in [
            (lambda: heads.layer_norm(x.double()), "float32, float16 or bfloat16"),
            (lambda: heads.layer_norm(x, w[:5]), "shape"),
            (lambda: heads.layer_norm(x, w.view(1, 6)), "shape"),
            (lambda: heads.layer_norm(x, w.cpu()), "on a GPU"),
            (lambda: heads.layer_norm(x, w.double()), "float32, float16 or bfloat16"),
            (lambda: heads.layer_norm(x, w, w.half()), "bias is"),
            (lambda: heads.layer_norm(x, None, w), "needs a weight"),
            (lambda: heads.layer_norm(x, eps=0.0), "eps"),
            (lambda: heads.layer_norm(torch.zeros(2, 0, device="cuda")), "32768 cells"),
            (lambda: heads.layer_norm(torch.zeros(2, 32_769, device="cuda")), "32768 cells"),
            (lambda: heads.layer_norm(torch.tensor(1.0, device="cuda")), "32768 cells"),
            (lambda: heads.layer_norm_grad(x[:3], x, stats, w), "grad is"),
            (lambda: heads.layer_norm_grad(x.half(), x, stats, w), "grad is"),
            (lambda: heads.layer_norm_grad(x, x, stats[:3], w), "stats must"),
            (lambda: heads.layer_norm_grad(x, x, stats.half(), w), "stats must"),
            (lambda: heads.Routes(ids.double(), 3), "int32, int64 or float32"),
            (lambda: heads.Routes(ids, 0), "n_experts"), (lambda: heads.Routes(ids, 1025), "n_exp"),
            (lambda: heads.Routes(ids, None), "whole number"),
            (lambda: heads.Routes(ids[0, 0], 3), "last axis"),
            (lambda: heads.to_experts(x, ids), "must be Routes"),
            (lambda: heads.to_experts(x[:3], r), "must have shape"),
            (lambda: heads.to_experts(x.double(), r), "float32, float16 or bfloat16"),
            (lambda: heads.from_experts(rows[:7], r), "must have shape"),
            (lambda: heads.from_experts(rows, r, w), "weights must"),
            (lambda: heads.from_experts(rows, r, torch.ones(4, 2, device="cuda").half()),
             "weights must"),
            (lambda: heads.from_experts_grad(x[:2], rows, r), "must have shape"),
            (lambda: heads.from_experts_grad(x, rows.half(), r), "y must"),
            (lambda: heads.AdamW([x, x]), "overlap"), (lambda: heads.AdamW([x, x[1]]), "overlap"),
            (lambda: heads.AdamW([x.t()]), "contiguous"),
            (lambda: heads.AdamW([x.double()]), "float32, float16 or bfloat16"),
            (lambda: heads.AdamW([x, w.cpu()]), "on a GPU"),
            (lambda: heads.AdamW([x], lr=-1.0), "lr must"),
            (lambda: heads.AdamW([x], lr=torch.ones(2, device="cuda")), "lr must"),
            (lambda: heads.AdamW([x], lr=torch.ones(1, device="cuda").half()), "lr must")]:
        with pytest.raises(ValueError, match=msg):
            call()
    opt = heads.AdamW([x, w])
    kept = x.clone()
    for grads, msg in [([x], "1 gradients for 2"), ([x, None], "no gradient"),
                       ([x, x], "gradient 1 is"), ([x.half(), w], "gradient 0 is"),
                       ([x.cpu(), w], "on a GPU"), ([x, 1.0], "torch tensor")]:
        with pytest.raises(ValueError, match=msg):
            opt.step(grads)
    opt.lr = float("nan")
    with pytest.raises(ValueError, match="lr must"):
        opt.step([x, w])
    opt.lr = 0.1
    v = torch.nn.Parameter(torch.ones(6, device="cuda"))
    other = heads.AdamW([v])
    v.data = torch.ones(7, device="cuda")
    with pytest.raises(ValueError, match="changed"):
        other.step([torch.ones(7, device="cuda")])
    v.data = torch.ones(6, device="cuda").half()
    with pytest.raises(ValueError, match="changed"):
        other.step([torch.ones(6, device="cuda").half()])
    state = opt.state_dict()
    assert state["step"] == 0 and torch.equal(x, kept)
    for bad, msg in [({"step": -1}, "step"), ({"bits": 8}, "bits"), ({"decays": [1.0]}, "decays"),
                     ({"decays": [1.0, 2.0]}, "decays"), ({"mean": state["mean"][:5]}, "mean must"),
                     ({"square": state["square"].half()}, "square must"),
                     ({"masters": [None]}, "masters")]:
        with pytest.raises(ValueError, match=msg):
            opt.load_state_dict({**state, **bad})
