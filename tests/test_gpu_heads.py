"""The heads on a model's outputs against their definitions in 64 bits.

Tolerances. A cell is rounded once to its type, by half a step: |value| * eps / 2 (and half
the type's smallest subnormal). Sums of m terms in float32 in any order are off by at most
(m - 1) * 2^-24 times the sum of their magnitudes (to first order), the scaling by 2^-23 more
(the factor's own rounding and the product's). Dropout and sampling have no tolerance but
for log-probabilities: float32's half step, and 2^-50 for the doubles that they are made of.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import heads_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def heads():
    import ferrisboost_amd as fb

    if not fb.device_available(0):
        pytest.fail("no gfx950 device: the GPU suite needs an MI355X")
    return fb.heads


def _host(x):
    return x.detach().cpu().to(torch.float64).numpy()


def _close(got, want, magnitude, terms, dtype, where=""):
    info = torch.finfo(dtype)
    tol = (np.abs(want) * info.eps / 2 + info.smallest_normal * info.eps / 2
           + magnitude * ((np.maximum(terms, 1) + 1) * 2.0 ** -24 * (1 + info.eps)))
    g = _host(got)
    with np.errstate(invalid="ignore"):
        bad = ~((np.abs(g - want) <= tol) | (g == want) | (np.isnan(g) & np.isnan(want)))
    assert not bad.any(), (where, np.argwhere(bad)[:4].tolist(), g[bad][:4], want[bad][:4])


def _cells(rng, shape, dtype):
    x = torch.from_numpy(rng.normal(size=shape).astype(np.float32)).to(TYPES[dtype])
    return x.cuda()


def _draw_ids(rng, n, t, sizes, kind, skew):
    cols = []
    for s in sizes:
        if skew:
            c = np.minimum((rng.pareto(0.8, n)).astype(np.int64), max(s - 1, 0))
        else:
            c = rng.integers(0, max(s, 1), n)
        cols.append(c)
    ids = np.stack(cols, 1) if t else np.zeros((n, 0), np.int64)
    ids[rng.random(ids.shape) < 0.05] = -1
    ids[rng.random(ids.shape) < 0.02] = 1 << 20  # beyond every column
    dt = {"i32": np.int32, "i64": np.int64, "f32": np.float32}[kind]
    ids = ids.astype(dt)
    if kind == "f32" and ids.size > 8:
        ids.flat[1], ids.flat[3], ids.flat[5] = np.nan, 0.5, np.inf
    if kind == "i64" and ids.size > 8:
        ids.flat[1], ids.flat[3] = (1 << 32) + 1, -(1 << 40)
    return ids


# (rows, columns' sizes, dim): one id to long lists, widths around the 16-byte pieces, a
# column without ids, few rows and many (both summing kernels), columns beyond one stage
TABLES = [
    (1, [7], 1), (1, [3, 0, 5], 3), (2, [511] * 100, 64), (5, [9, 1, 300], 17),
    (64, [2] * 9, 8), (333, [50, 3, 1000], 5), (1000, [40] * 33, 16), (70, [5] * 600, 127),
    (4097, [31, 77], 33), (9000, [100, 28], 260), (40, [12] * 7, 1100), (30_000, [17] * 5, 2),
    (1, [10_000], 2048),
    (900, [1500] * 80, 20),  # many positions, sorted through memory
    # columns summed chunk by chunk: one chunk, several, uneven ones, wide vectors
    (3000, [40] * 33, 64), (20_000, [511, 3, 0, 200], 24), (140_000, [9], 7),
    (70_001, [31, 1000], 3), (9000, [1024, 5] * 4, 600), (66_000, [2, 1], 1),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", TABLES, ids=lambda c: f"{c[0]}x{len(c[1])}x{c[2]}")
def test_embed_and_its_gradient(heads, case, dtype):
    n, sizes, dim = case
    rng = np.random.default_rng([n, len(sizes), dim])
    voc = heads.Vocabulary(sizes)
    table = _cells(rng, (voc.n_tokens, dim), dtype)
    t64 = _host(table)
    for k, (kind, drop, scale, pooled) in enumerate(
            [("i32", 0.0, 1.0, True), ("f32", 0.25, 0.5, True), ("i64", 0.0, 3.0, False),
             ("i32", 0.5, 1.0, False)]):
        ids = _draw_ids(rng, n, len(sizes), sizes, kind, skew=k % 2 == 1)
        seed = 12345 + k + (k << 60)
        tok = ref.tokens(ids, sizes, voc.n_tokens, drop, seed)
        d_ids = torch.from_numpy(ids).cuda()
        kw = dict(scale=scale, pooled=pooled, drop=drop, seed=seed)
        s = scale / (1.0 - drop)
        out = heads.embed(table, d_ids, voc, **kw)
        want, mag = ref.embed(t64, tok, s, pooled)
        assert out.shape == want.shape and out.dtype == table.dtype
        _close(out, want, mag, len(sizes) if pooled else 1, table.dtype, ("embed", kw))
        grad = _cells(rng, want.shape, dtype)
        dt = heads.embed_grad(grad, d_ids, voc, **kw)
        want, mag, terms = ref.embed_grad(_host(grad), tok, voc.n_tokens, s, pooled)
        assert dt.shape == table.shape and dt.dtype == table.dtype
        _close(dt, want, mag, terms[:, None], table.dtype, ("grad", kw))


@pytest.mark.parametrize("n, v, dim, skew", [
    (1, 1, 1, False), (7, 3, 4, False), (4096, 50_000, 32, True), (32_768, 300, 1024, True),
    (100_000, 5, 24, False), (20_000, 70_000, 7, True), (300_000, 260, 3, True),
    (65_537, 16_777_217, 1, False), (70_000, 3000, 20, True), (200_000, 100_000, 5, False),
    (66_000, 70_000, 260, True), (5000, 600_000, 3, False), (65_536, 1_048_576, 2, True),
    (65_536, 1_048_577, 2, True), (9000, 262_143, 3, True), (9000, 262_144, 1, False),
    (300, 1024, 5, True), (16_384, 700, 4, True), (16_385, 700, 4, False)])
def test_one_vocabulary(heads, n, v, dim, skew):
    """Flat ids without a vocabulary: one to four radix passes, runs over many chunks."""
    rng = np.random.default_rng(n + v)
    ids = np.minimum(rng.pareto(0.5, n).astype(np.int64), v - 1) if skew else rng.integers(
        -1, v, n)
    d_ids = torch.from_numpy(ids).cuda()
    grad = _cells(rng, (n, dim), "f32")
    got = heads.embed_grad(grad, d_ids, v, scale=2.0)
    want, mag, terms = ref.embed_grad(_host(grad), ids[:, None], v, 2.0, False)
    _close(got, want, mag, terms[:, None], torch.float32)
    for _ in range(2):  # the same bits again
        assert torch.equal(got, heads.embed_grad(grad, d_ids, v, scale=2.0))


def test_a_row_does_not_depend_on_the_rows_beside_it(heads):
    rng = np.random.default_rng(3)
    voc = heads.Vocabulary([60] * 50)
    table = _cells(rng, (voc.n_tokens, 48), "f32")
    ids = torch.from_numpy(rng.integers(0, 60, (20_000, 50))).cuda()
    many = heads.embed(table, ids, voc, pooled=True)
    for n in (1, 3, 700):
        assert torch.equal(many[:n], heads.embed(table, ids[:n], voc, pooled=True))


def test_masked_cells_may_hold_anything(heads):
    """Table rows that nothing refers to, rows of dropped and missing positions, and
    dropped elements give and take nothing, whatever they hold."""
    rng = np.random.default_rng(4)
    voc = heads.Vocabulary([4, 4])
    table = _cells(rng, (8, 16), "f32")
    table[0] = float("nan")
    table[7] = float("inf")
    ids = torch.from_numpy(rng.integers(1, 3, (5000, 2))).cuda()
    ids[::3, 0] = -1
    ids[1::3, 1] = 4
    for pooled in (True, False):
        assert torch.isfinite(heads.embed(table, ids, voc, pooled=pooled)).all()
    grad = _cells(rng, (5000, 2, 16), "f32")
    grad[::3, 0] = float("nan")
    grad[1::3, 1] = float("-inf")
    assert torch.isfinite(heads.embed_grad(grad, ids, voc)).all()
    x = torch.full((4099,), float("nan"), device="cuda")
    out = heads.dropout(x, 0.5, 9)
    stay = torch.from_numpy(ref.kept(9, 0.5, np.arange(4099))).cuda()
    assert torch.equal(torch.isnan(out), stay) and (out[~stay] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 255, 4096, 8193, 100_003])
def test_dropout(heads, n, dtype):
    rng = np.random.default_rng(n)
    whole = _cells(rng, n + 3, dtype)
    for drop in (0.0, 0.1, 0.5, 0.999):
        scale = torch.tensor(np.float32(1.0 / (1.0 - drop)))
        for skip in (0, 1, 3):  # and unaligned parts, numbered as in the whole
            for first in (skip, (1 << 33) + 1 + skip):
                x = whole[skip:skip + n]
                out = heads.dropout(x, drop, 77, first)
                stay = torch.from_numpy(ref.kept(77, drop, first + np.arange(n)))
                want = torch.where(stay, (x.cpu().float() * scale), torch.zeros(())).to(x.dtype)
                assert torch.equal(out.cpu(), want), (drop, skip, first)


def test_dropout_rates(heads):
    x = torch.ones(1 << 22, device="cuda")
    for seed in (0, 1, 2 ** 64 - 1):
        for drop in (0.1, 0.5):
            share = (heads.dropout(x, drop, seed) == 0).double().mean().item()
            # five standard deviations of 2^22 draws
            assert abs(share - drop) < 5 * (drop * (1 - drop)) ** 0.5 / 2 ** 11
    a, b = (heads.dropout(x, 0.5, s) != 0 for s in (1, 2))
    assert abs((a == b).double().mean().item() - 0.5) < 5 * 0.5 / 2 ** 11
    assert abs((a[1:] == a[:-1]).double().mean().item() - 0.5) < 5 * 0.5 / 2 ** 11


def test_strides_and_streams(heads):
    """Inputs that are not contiguous, and calls on a stream of the caller's."""
    rng = np.random.default_rng(6)
    voc = heads.Vocabulary([20, 30])
    wide = _cells(rng, (50, 40), "bf16")
    table = wide[:, 3:27]
    ids = torch.from_numpy(rng.integers(0, 20, (2, 900)).astype(np.int32)).cuda().t()
    want = heads.embed(table.contiguous(), ids.contiguous(), voc, pooled=True)
    assert torch.equal(heads.embed(table, ids, voc, pooled=True), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = heads.embed(table, ids, voc, pooled=True)
        g = heads.embed_grad(got, ids, voc, pooled=True)
        d = heads.dropout(wide.t(), 0.5, 3)
    s.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(g, heads.embed_grad(want, ids, voc, pooled=True))
    assert torch.equal(d, heads.dropout(wide.t().contiguous(), 0.5, 3))


def test_autograd(heads):
    """backward() gives the gradients of the explicit calls, also of an expanded one."""
    rng = np.random.default_rng(7)
    voc = heads.Vocabulary([9, 11])
    table = _cells(rng, (20, 6), "f32").requires_grad_()
    ids = torch.from_numpy(rng.integers(0, 9, (500, 2))).cuda()
    h = heads.embed(table, ids, voc, pooled=True, drop=0.2, seed=1, scale=1.5)
    y = heads.dropout(h, 0.3, 2)
    y.sum().backward()
    g = heads.dropout(torch.ones_like(y), 0.3, 2)
    g = heads.embed_grad(g, ids, voc, pooled=True, drop=0.2, seed=1, scale=1.5)
    assert torch.equal(table.grad, g)
    # against differences: the sum is linear in each cell
    with torch.no_grad():
        for cell in ((0, 0), (13, 5), (19, 2)):
            up, down = table.detach().clone(), table.detach().clone()
            up[cell] += 8.0
            down[cell] -= 8.0
            f = [heads.dropout(heads.embed(t, ids, voc, pooled=True, drop=0.2, seed=1, scale=1.5),
                               0.3, 2).double().sum().item() for t in (up, down)]
            # 3000 outputs of at most 2 * 16 * 2.7, each off by 2^-24 of that and twice more
            assert abs((f[0] - f[1]) / 16 - g[cell].item()) < 3000 * 90 * 3 * 2.0 ** -24 / 16


def test_a_captured_step(heads):
    """Forward, gradient, dropout and sampling in one graph, replayed on new inputs with
    eager work between."""
    rng = np.random.default_rng(8)
    voc = heads.Vocabulary([30] * 6)
    table = _cells(rng, (180, 32), "bf16")
    ids = torch.from_numpy(rng.integers(0, 30, (3000, 6)).astype(np.int32)).cuda()
    u = torch.rand(3000, device="cuda")

    def step():
        h = heads.dropout(heads.embed(table, ids, voc, pooled=True, drop=0.1, seed=3), 0.1, 4)
        return h, heads.embed_grad(h, ids, voc, pooled=True), heads.sample(h, u, top_k=5)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, g, (c, p) = step()
    for k in range(4):
        ids.copy_(torch.from_numpy(rng.integers(-1, 30, (3000, 6)).astype(np.int32)))
        u.uniform_()
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert torch.equal(h, want[0]) and torch.equal(g, want[1]), k
        assert torch.equal(c, want[2][0]) and torch.equal(p, want[2][1]), k


def _check_sample(heads, x, u, t, k, p, m):
    dev = [torch.from_numpy(o).cuda() if isinstance(o, np.ndarray) else o for o in (t, k, p, m)]
    c, lp = heads.sample(x, u, temperature=dev[0], top_k=dev[1], top_p=dev[2], min_p=dev[3])
    want_c, want_p = ref.sample(x.cpu().float().numpy(), u.cpu().numpy(), t, k, p, m)
    bad = np.nonzero(c.cpu().numpy() != want_c)[0]
    assert bad.size == 0, (bad[:5], c[bad[:5]], want_c[bad[:5]])
    got = lp.cpu().numpy().astype(np.float64)
    none = want_c < 0
    assert np.array_equal(got[none], want_p[none])
    tol = np.abs(want_p[~none]) * 2.0 ** -24 + 2.0 ** -45
    assert (np.abs(got[~none] - want_p[~none]) <= tol).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n, v", [(1, 1), (300, 2), (200, 3), (130, 4), (300, 5), (64, 6), (77, 7),
                                  (257, 8), (40, 9), (33, 16), (20, 17), (50, 33), (40, 64),
                                  (40, 65), (9, 128), (9, 129), (13, 256), (10, 400), (30, 500),
                                  (11, 1000), (6, 1024), (6, 1025), (9, 2048), (7, 2049),
                                  (3, 16_384), (3, 16_385), (2, 131_071), (1, 262_144),
                                  (129, 16_400)])
def test_sample(heads, n, v, dtype):
    rng = np.random.default_rng([n, v])
    x = rng.normal(size=(n, v)) * 3
    x[rng.random(x.shape) < 0.1] = -np.inf
    x[rng.random(x.shape) < 0.02] = np.nan
    if n > 2:
        x[1] = -np.inf  # nothing left
    if n > 4:
        x[2] = 0.25     # all alike
        x[3, : (v + 1) // 2] = np.inf
        x[4] = np.where(rng.random(v) < 0.5, 0.0, -0.0)
    x = torch.from_numpy(x.astype(np.float32)).to(TYPES[dtype]).cuda()
    u = torch.from_numpy(rng.random(n).astype(np.float32)).cuda()
    u[0] = 0.0
    if n > 1:
        u[-1] = 1.0 - 2.0 ** -24
    for t, k, p, m in [(1.0, 0, 1.0, 0.0), (0.7, max(1, v // 3), 1.0, 0.0), (1.3, 0, 0.9, 0.0),
                       (1.0, 3, 0.5, 0.0), (1.0, 0, 1.0, 0.1), (0.9, min(50, v), 0.95, 0.02),
                       (0.0, 0, 1.0, 0.0), (1.0, v, 0.0, 0.0), (1e-30, 0, 0.3, 0.5),
                       (1e30, 5, 0.99, 1.0)]:
        _check_sample(heads, x, u, t, k, p, m)


@pytest.mark.parametrize("v", [4, 8, 40, 90, 300, 1000, 3000, 20_000])
def test_sample_options_of_each_row(heads, v):
    rng = np.random.default_rng(v)
    n = 64 if v <= 3000 else 12
    x = torch.from_numpy((rng.normal(size=(n, v)) * 2).astype(np.float32)).cuda()
    u = torch.from_numpy(rng.random(n).astype(np.float32)).cuda()
    t = rng.choice([0.0, 0.5, 1.0, 2.0, -1.0, np.nan], n).astype(np.float32)
    k = rng.choice([-3, 0, 1, 2, v // 2, v, 10 * v], n).astype(np.int32)
    p = rng.choice([0.0, 0.3, 0.9, 1.0, 7.0, -1.0, np.nan], n).astype(np.float32)
    m = rng.choice([0.0, 0.05, 1.0, 3.0, -2.0, np.nan], n).astype(np.float32)
    _check_sample(heads, x, u, t, k, p, m)


@pytest.mark.parametrize("v", [8, 48, 120, 700, 5000, 40_000])
def test_sample_of_ties_and_far_logits(heads, v):
    """Cuts that fall among equal logits, and among ones beyond the range of weights."""
    rng = np.random.default_rng(v)
    n = 24
    x = rng.integers(0, 3, (n, v)).astype(np.float32)
    x[: n // 2, 5:] -= rng.choice([0.0, 50.0, 1e9], (n // 2, v - 5)).astype(np.float32)
    x[n // 2, 3:] = -1e30  # all but three far below
    u = torch.from_numpy(rng.random(n).astype(np.float32)).cuda()
    for dtype in ("f32", "bf16"):
        d = torch.from_numpy(x).to(TYPES[dtype]).cuda()
        for k, p in [(7, 1.0), (0, 0.4), (v // 2, 0.7), (v - 1, 1.0), (4, 0.999)]:
            _check_sample(heads, d, u, 1.0, k, p, 0.0)


def test_sample_follows_the_distribution(heads):
    """2^20 draws of one row: each class' share within five standard deviations."""
    x = torch.tensor([0.0, 1.0, -1.0, 2.0, -np.inf, 0.5], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    n = 1 << 20
    c, _ = heads.sample(x.expand(n, 6), torch.rand(n, generator=g, device="cuda"))
    p = torch.softmax(x.double(), 0).cpu().numpy()
    share = np.bincount(c.cpu().numpy(), minlength=6) / n
    assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / n)).all()


def test_beyond_32_bits(heads):
    """More than 2^32 cells, tables beyond the reach of buffer loads, and more rows than one
    launch takes."""
    n = (1 << 32) + 4099
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    out = heads.dropout(x, 0.5, 11)
    for at in (0, (1 << 31) - 7, (1 << 32) - 33, n - 4100):
        part = slice(at, min(at + 4100, n))
        stay = ref.kept(11, 0.5, np.arange(part.start, part.stop))
        assert np.array_equal(out[part].float().cpu().numpy(), np.where(stay, 2.0, 0.0))
        assert torch.equal(heads.dropout(x[part], 0.5, 11, at), out[part])
    del x, out
    rows, dim = 40_000_003, 32
    table = torch.zeros((rows, dim), dtype=torch.bfloat16, device="cuda")
    table[:, 0] = torch.arange(rows, device="cuda") % 128
    last = torch.arange(rows - 200_000, rows, device="cuda").reshape(-1, 10)
    want = (last % 128).float().sum(1)
    pooled = heads.embed(table.float(), last, pooled=True)
    assert torch.equal(pooled[:, 0], want) and (pooled[:, 1:] == 0).all()
    assert torch.equal(heads.embed(table, last, pooled=True)[:, 0], want.bfloat16())
    ids = torch.arange(rows - 1, -1, -1, dtype=torch.int32, device="cuda").repeat(4)
    out = heads.embed(table, ids)  # 2^32 cells and more
    assert out.numel() > 1 << 32 and torch.equal(out[-1], table[0])
    assert torch.equal(out[:rows:10_007], table.flip(0)[::10_007])
    assert torch.equal(out[3 * rows::10_007], table.flip(0)[::10_007])
    g = heads.embed_grad(out, ids, rows)  # four positions a row, a chunk's rows far apart
    assert torch.equal(g[::9973], (4 * table[::9973].float()).bfloat16())
    del table, out, g, ids
    u = torch.rand(2_500_000, device="cuda")
    x = torch.randn(2_500_000, 70, device="cuda")
    c, p = heads.sample(x, u, top_k=9)
    at = slice((1 << 21) - 50, (1 << 21) + 50)
    c2, p2 = heads.sample(x[at], u[at], top_k=9)
    assert torch.equal(c[at], c2) and torch.equal(p[at], p2) and (c >= 0).all()
    want, _ = ref.sample(x[-40:].cpu().numpy(), u[-40:].cpu().numpy(), 1.0, 9, 1.0, 0.0)
    assert np.array_equal(c[-40:].cpu().numpy(), want)


def test_captured_calls_with_much_lds(heads):
    """A gradient whose workgroups take more LDS than a kernel has without asking."""
    rng = np.random.default_rng(9)
    voc = heads.Vocabulary([1000, 900])
    ids = torch.from_numpy(rng.integers(0, 1000, (40_000, 2))).cuda()
    grad = _cells(rng, (40_000, 2, 40), "bf16")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g = heads.embed_grad(grad, ids, voc)
    for _ in range(3):
        ids.copy_(torch.from_numpy(rng.integers(-1, 950, (40_000, 2))))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(g, heads.embed_grad(grad, ids, voc))


def test_captured_large_calls(heads):
    """Calls of several launches that hand counters and lists to one another."""
    rng = np.random.default_rng(10)
    flat = torch.from_numpy(rng.integers(0, 3000, 70_000)).cuda()
    few = torch.from_numpy(rng.integers(0, 5000, 3000)).cuda()
    grad = _cells(rng, (70_000, 12), "f32")
    x = _cells(rng, (3, 40_000), "bf16") * 3
    u = torch.rand(3, device="cuda")

    def step():
        return (heads.embed_grad(grad, flat, 3000), heads.embed_grad(grad[:3000], few, 5000),
                *heads.sample(x, u, top_p=0.9), *heads.sample(x, u))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(4):
        flat.random_(0, 3000)
        few.random_(-1, 5000)
        x.normal_()
        u.uniform_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_empty_calls(heads):
    voc = heads.Vocabulary([3, 4])
    table = torch.ones(7, 5, device="cuda")
    ids = torch.zeros(0, 2, dtype=torch.int32, device="cuda")
    assert heads.embed(table, ids, voc, pooled=True).shape == (0, 5)
    assert heads.embed(table, ids, voc).shape == (0, 2, 5)
    assert (heads.embed_grad(torch.ones(0, 5, device="cuda"), ids, voc, pooled=True) == 0).all()
    for v in (3, 300_000):  # one vocabulary, in one pass and in several
        g = heads.embed_grad(torch.ones(0, 5, device="cuda"), ids[:, 0], v)
        assert g.shape == (v, 5) and (g == 0).all()
    none = torch.zeros(3, 0, dtype=torch.int64, device="cuda")
    assert (heads.embed(table, none, pooled=True) == 0).all()
    assert (heads.embed_grad(torch.ones(3, 5, device="cuda"), none, 7, pooled=True) == 0).all()
    assert heads.dropout(torch.ones(0, 4, device="cuda"), 0.5, 1).shape == (0, 4)
    c, p = heads.sample(torch.ones(0, 9, device="cuda"), torch.ones(0, device="cuda"))
    assert c.shape == (0,) and p.shape == (0,)
