"""The training heads against their definitions in 64 bits.

Tolerances: training_ref derives how far float32 may be from each value; a cell is then rounded
once to its type, by half a step, |value| * eps / 2 (and half the type's smallest subnormal).
Orders, places and the 8-bit moments have no tolerance."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import training_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


@pytest.fixture(scope="module")
def heads():
    import ferrisboost_amd as fb

    if not fb.device_available(0):
        pytest.fail("no gfx950 device: the GPU suite needs an MI355X")
    return fb.heads


def _host(x):
    return x.detach().cpu().to(torch.float64).numpy()


def _near(got, want, off, where=""):
    info = torch.finfo(got.dtype)
    off = off * (1 + info.eps) + np.abs(want) * info.eps / 2 + info.smallest_normal * info.eps / 2
    g = _host(got)
    assert g.shape == want.shape, (where, g.shape, want.shape)
    with np.errstate(invalid="ignore"):
        bad = ~((np.abs(g - want) <= off) | (g == want) | (np.isnan(g) & np.isnan(want)))
    assert not bad.any(), (where, bad.sum(), np.argwhere(bad)[:4].tolist(), g[bad][:4],
                           want[bad][:4], (off * np.ones_like(want))[bad][:4])


def _cells(rng, shape, dtype, scale=1.0, shift=0.0):
    x = torch.from_numpy((rng.normal(size=shape) * scale + shift).astype(np.float32))
    return x.to(TYPES[dtype]).cuda()


# ------------------------------------------------------------------- layer norm
# every number of lanes and cells a lane, full and one more, odd and tiny widths
NORMS = [(1, 1), (7, 1), (300, 2), (5, 3), (64, 7), (130, 8), (65, 31), (64, 32), (33, 33),
         (1000, 64), (17, 100), (31, 128), (16, 129), (700, 255), (16, 256), (5, 257), (9, 511),
         (4, 512), (3, 513), (6000, 130), (3, 1000), (5, 1024), (2, 1025), (1, 2047), (600, 2048),
         (3, 2049), (2, 4095), (4, 4096), (1, 4097), (3, 8192), (2, 8193), (520, 16384),
         (1, 16385), (530, 20001), (2, 32767), (3, 32768)]


@pytest.mark.parametrize("dtype, weight", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"),
                                           ("bf16", "f32"), ("f32", "bf16"), ("f16", None)])
@pytest.mark.parametrize("n, dim", NORMS)
def test_layer_norm_and_its_gradients(heads, n, dim, dtype, weight):
    rng = np.random.default_rng([n, dim])
    x = _cells(rng, (n, dim), dtype) * _cells(rng, (n, 1), dtype) + _cells(rng, (n, 1), dtype)
    w = None if weight is None else _cells(rng, dim, weight, 0.5, 1.0).requires_grad_()
    b = None if weight is None else _cells(rng, dim, weight).requires_grad_()
    g = _cells(rng, (n, dim), dtype)
    x.requires_grad_()
    y = heads.layer_norm(x, w, b, eps=EPS)
    hx, hw, hb = _host(x), None if w is None else _host(w), None if b is None else _host(b)
    _near(y, *ref.layer_norm(hx, hw, hb, EPS), "y")
    y.backward(g)
    dx, dw, db = ref.layer_norm_grad(_host(g), hx, hw, EPS)
    _near(x.grad, *dx, "dx")
    y2, stats = heads.layer_norm(x.detach(), w, b, eps=EPS, stats=True)
    assert torch.equal(y, y2)
    got = heads.layer_norm_grad(g, x.detach(), stats, w)
    assert torch.equal(got[0], x.grad)
    if weight is None:
        assert got[1:] == (None, None)
        return
    _near(w.grad, *dw, "dw")
    _near(b.grad, *db, "db")
    assert torch.equal(got[1], w.grad) and torch.equal(got[2], b.grad)


def test_layer_norm_rows_far_from_zero(heads):
    """The mean's own rounding is taken out: cells of 1000 +- 1 keep theirs."""
    rng = np.random.default_rng(1)
    for dim in (30, 500, 3000, 9000):
        x = _cells(rng, (40, dim), "f32", 1.0, 1000.0)
        g = _cells(rng, (40, dim), "f32")
        y, stats = heads.layer_norm(x, stats=True)
        _near(y, *ref.layer_norm(_host(x), None, None, EPS))
        (dx, off), _, _ = ref.layer_norm_grad(_host(g), _host(x), None, EPS)
        _near(heads.layer_norm_grad(g, x, stats)[0], dx, off)


@pytest.mark.parametrize("dim", [1, 40, 200, 1500, 12_000, 30_000])
def test_layer_norm_of_constant_and_broken_rows(heads, dim):
    """A constant row is the bias; NaN and infinity stay in their row, and in the weights' sums."""
    x = torch.randn(9, dim, device="cuda")
    x[1], x[3] = 5.0, 0.0
    w, b = torch.randn(dim, device="cuda"), torch.randn(dim, device="cuda")
    y, stats = heads.layer_norm(x, w, b, stats=True)
    assert torch.equal(y[1], b) and torch.equal(y[3], b)
    g = torch.randn_like(x)
    dx, dw, db = heads.layer_norm_grad(g, x, stats, w)
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all()
    x2 = x.clone()
    x2[2, dim // 2], x2[6, 0] = float("nan"), float("inf")
    y2, stats2 = heads.layer_norm(x2, w, b, stats=True)
    dx2, dw2, db2 = heads.layer_norm_grad(g, x2, stats2, w)
    bad = [2, 6]
    good = [i for i in range(9) if i not in bad]
    assert torch.equal(y2[good], y[good]) and torch.equal(dx2[good], dx[good])
    assert torch.isnan(y2[bad]).all() and torch.isnan(dw2).all() and torch.equal(db2, db)


def test_layer_norm_rows_do_not_depend_on_their_neighbours(heads):
    x = torch.randn(5000, 200, device="cuda", dtype=torch.bfloat16)
    y = heads.layer_norm(x)
    for n in (1, 3, 77):
        assert torch.equal(heads.layer_norm(x[:n]), y[:n])


def test_gradients_of_broadcast_and_strided_inputs(heads):
    """Copies of one cell, of one row, and transposed ones: their gradients are summed, or laid
    out, as those of what they are views of."""
    rng = np.random.default_rng(9)
    x, g = _cells(rng, (40, 60), "f32"), _cells(rng, (40, 60), "f32")
    w, b = _cells(rng, 60, "f32"), _cells(rng, 60, "f32")

    def grads(make, *leaves):
        leaves = [a.detach().clone().requires_grad_() for a in leaves]
        return torch.autograd.grad(heads.layer_norm(*make(*leaves)), leaves, g)

    base = grads(lambda *a: a, x, w, b)
    got = grads(lambda x, w, b: (x.t(), w, b), x.t().contiguous(), w, b)
    assert torch.equal(got[0].t(), base[0]) and torch.equal(got[1], base[1])
    one = grads(lambda *a: a, x[:1].expand(40, 60).contiguous(), w, b)
    got = grads(lambda x, w, b: (x.expand(40, 60), w, b), x[:1], w, b)
    assert torch.equal(got[0], one[0].sum(0, keepdim=True)) and torch.equal(got[1], one[1])
    one = grads(lambda *a: a, x, w[:1].expand(60).contiguous(), b)
    got = grads(lambda x, w, b: (x, w.expand(60), b), x, w[:1], b)
    assert torch.equal(got[1], one[1].sum(0, keepdim=True))
    # experts: one weight for all, rows of a transposed output, an expanded gradient
    ids = torch.from_numpy(rng.integers(-1, 5, (40, 2))).cuda()
    r = heads.Routes(ids, 5)
    y = _cells(rng, (80, 60), "f32").requires_grad_()
    v = torch.tensor(0.5, device="cuda", requires_grad=True)
    out = heads.from_experts(y, r, v.expand(40, 2))
    out.backward(g[:, :1].expand(40, 60))
    dy, dw = heads.from_experts_grad(g[:, :1].expand(40, 60).contiguous(), y.detach(), r,
                                     torch.full((40, 2), 0.5, device="cuda"))
    assert torch.equal(y.grad, dy) and torch.equal(v.grad, dw.sum())
    t = y.detach().t().contiguous().requires_grad_()
    heads.from_experts(t.t(), r, torch.full((40, 2), 0.5, device="cuda")).backward(
        g[:, :1].expand(40, 60))
    assert torch.equal(t.grad.t(), dy)


@pytest.mark.parametrize("dim", [3, 31, 100, 1000, 5000, 12_000, 30_000])
def test_layer_norm_of_equal_cells_with_a_tiny_eps(heads, dim):
    """What rounding leaves of a variance of 0 may be below it, never a NaN: cells are off from
    their mean by at most 46 half steps of it, and by 46 of that once it is taken out."""
    x = torch.full((64, dim), 1.0, device="cuda") * (torch.rand(64, 1, device="cuda") * 1000 + 0.1)
    for eps in (2.0 ** -126, 1e-30, 1e-12):
        y, stats = heads.layer_norm(x, eps=eps, stats=True)
        assert torch.isfinite(y).all() and torch.isfinite(stats).all()
        off = x.abs().max().double() * (46 * 2.0 ** -24) ** 2 * stats[:, 1:].double()
        assert (y.double().abs() <= off * 1.01).all()


@pytest.mark.parametrize("n, dim", [(700, 3), (700, 33), (300, 513), (40, 4097), (300, 16_385)])
def test_layer_norm_in_place(heads, n, dim):
    """The C entry allows an output over its input."""
    from ferrisboost_amd import _native as N

    x = torch.randn(n, dim, device="cuda")
    want = heads.layer_norm(x)
    a = heads._norm_of(x, None, EPS)
    N.check_hip(heads._L.fbh_layer_norm(0, a, x.data_ptr(), None, None, x.data_ptr(), None,
                                        heads._raw_stream(0)))
    assert torch.equal(x, want)


def test_layer_norm_shapes(heads):
    """Leading axes, no rows, slices that no 16-byte piece begins at, transposed tensors."""
    x = torch.randn(3, 4, 50, device="cuda")
    y, stats = heads.layer_norm(x, stats=True)
    assert y.shape == x.shape and stats.shape == (3, 4, 2)
    assert torch.equal(y.view(12, 50), heads.layer_norm(x.view(12, 50)))
    assert torch.equal(heads.layer_norm(x[1, 2]), y[1, 2])
    t = torch.randn(50, 12, device="cuda").t()
    assert torch.equal(heads.layer_norm(t), heads.layer_norm(t.contiguous()))
    flat = torch.randn(1 + 7 * 333, device="cuda", dtype=torch.float16)
    odd = flat[1:].view(7, 333)
    assert torch.equal(heads.layer_norm(odd), heads.layer_norm(odd.clone()))
    none = torch.zeros(0, 50, device="cuda")
    w = torch.ones(50, device="cuda")
    y, stats = heads.layer_norm(none, w, w, stats=True)
    dx, dw, db = heads.layer_norm_grad(none, none, stats, w)
    assert y.shape == dx.shape == (0, 50) and (dw == 0).all() and (db == 0).all()
    wide = torch.zeros(0, 30_000, device="cuda")
    _, stats = heads.layer_norm(wide, stats=True)
    w = torch.ones(30_000, device="cuda")
    assert (heads.layer_norm_grad(wide, wide, stats, w)[1] == 0).all()


def test_layer_norm_of_more_than_2_31_cells(heads):
    n, dim = 70_001, 32_000
    x = torch.randn(64, dim, device="cuda", dtype=torch.bfloat16).repeat(n // 64 + 1, 1)[:n]
    y, stats = heads.layer_norm(x, stats=True)
    assert torch.equal(y[:64], y[-64 - n % 64:-(n % 64)])
    _near(y[-3:], *ref.layer_norm(_host(x[-3:]), None, None, EPS))
    dx = heads.layer_norm_grad(y, x, stats)[0]
    (want, off), _, _ = ref.layer_norm_grad(_host(y[-3:]), _host(x[-3:]), None, EPS)
    _near(dx[-3:], want, off)


def test_layer_norm_gradient_against_differences(heads):
    """Along a direction, of a sum in doubles: halves of the differences of float32 outputs,
    each off by at most 2^-24 * 64 * (|h| + 1) * |g|, divided by the step, and by the third
    derivative's part, below step^2 * 8 of the sum of |g| here (cells of unit size)."""
    rng = np.random.default_rng(2)
    x, u, g = (_cells(rng, (20, 90), "f32") for _ in range(3))
    y, stats = heads.layer_norm(x, stats=True)
    dx = heads.layer_norm_grad(g, x, stats)[0]
    step = 2.0 ** -6
    high, low = heads.layer_norm(x + step * u), heads.layer_norm(x - step * u)
    got = float(((high.double() - low.double()) * g.double()).sum()) / (2 * step)
    off = float((g.double().abs() * (y.double().abs() + 1)).sum())
    assert abs(got - float((dx.double() * u.double()).sum())) <= off * (
        64 * ref.ULP / step + 8 * step ** 2)


# ------------------------------------------------------------------- experts
def _ids(rng, shape, e, kind, skew):
    ids = rng.integers(0, e, shape) if not skew else np.minimum(
        rng.pareto(0.7, shape).astype(np.int64), e - 1)
    ids[rng.random(shape) < 0.04] = -1
    ids[rng.random(shape) < 0.02] = e
    ids = ids.astype({"i32": np.int32, "i64": np.int64, "f32": np.float32}[kind])
    if kind == "f32" and ids.size > 8:
        ids.flat[1], ids.flat[3], ids.flat[5], ids.flat[6] = np.nan, 0.5, np.inf, -0.0
    if kind == "i64" and ids.size > 8:
        ids.flat[1], ids.flat[3] = 1 << 32, -(1 << 40)
    return ids


def _check_routes(r, ids, e):
    order, place, starts = ref.route(ids, e)
    assert np.array_equal(r.starts.cpu().numpy(), starts)
    assert np.array_equal(r.place.cpu().numpy(), place)
    assert np.array_equal(r.order.cpu().numpy(), order)
    return place


@pytest.mark.parametrize("kind", ["i32", "i64", "f32"])
@pytest.mark.parametrize("n, k, e", [
    (1, 1, 1), (1, 2, 1024), (2, 1, 2), (3, 33, 7), (63, 1, 3), (64, 1, 64), (65, 1, 63),
    (255, 2, 255), (256, 2, 256), (1000, 1, 511), (2048, 2, 8), (4097, 1, 1023), (8191, 1, 64),
    (8193, 1, 1024), (16_384, 1, 200), (16_385, 1, 200), (30_000, 4, 1000), (65_537, 1, 1),
    (700_001, 2, 300), (5_000_000, 1, 1024)])
def test_routes(heads, n, k, e, kind):
    rng = np.random.default_rng([n, k, e])
    for skew in (False, True):
        ids = _ids(rng, (n, k), e, kind, skew)
        _check_routes(heads.Routes(torch.from_numpy(ids).cuda(), e), ids, e)


def test_routes_of_one_expert_and_of_none(heads):
    for n in (1, 500, 5000, 300_000):
        for value in (0, 3, -1, 9):
            ids = np.full((n, 1), value, np.int32)
            r = heads.Routes(torch.from_numpy(ids).cuda(), 5)
            _check_routes(r, ids, 5)
    for shape in ((0, 3), (0,), (4, 0), (2, 0, 5)):
        r = heads.Routes(torch.zeros(shape, dtype=torch.int64, device="cuda"), 4)
        assert r.order.shape == (0,) and r.place.shape == shape and r.starts.tolist() == [0] * 5
    x = torch.randn(4, 7, device="cuda")
    r = heads.Routes(torch.zeros((4, 0), dtype=torch.int32, device="cuda"), 4)
    rows = heads.to_experts(x, r)
    assert rows.shape == (0, 7) and (heads.from_experts(rows, r) == 0).all()
    assert heads.from_experts(rows, r).shape == (4, 7)
    dy, dw = heads.from_experts_grad(x, rows, r, torch.zeros(4, 0, device="cuda"))
    assert dy.shape == (0, 7) and dw.shape == (4, 0)


ROWS = [(1, 1, 1, 1), (1, 2, 8, 64), (3, 8, 5, 3), (5, 33, 9, 17), (64, 1, 3, 7), (67, 3, 20, 8),
        (300, 2, 11, 9), (1000, 4, 64, 5), (77, 2, 6, 515), (129, 5, 9, 1024), (9, 9, 4, 4100),
        (2000, 2, 100, 31), (5, 2, 3, 32_768)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n, k, e, dim", ROWS)
def test_rows_to_experts_and_back(heads, n, k, e, dim, dtype):
    rng = np.random.default_rng([n, k, e, dim])
    ids = _ids(rng, (n, k), e, "i64", False)
    r = heads.Routes(torch.from_numpy(ids).cuda(), e)
    order, place, starts = ref.route(ids, e)
    x = _cells(rng, (n, dim), dtype).requires_grad_()
    rows = heads.to_experts(x, r)
    want = _host(x)[order // k]
    want[starts[-1]:] = 0
    assert np.array_equal(_host(rows), want)
    gs = _cells(rng, (n * k, dim), dtype)
    rows.backward(gs)
    dx, mag = ref.from_experts(_host(gs), place, None)
    _near(x.grad, dx, (k + 1) * ref.ULP * mag)
    # NaN where no expert is
    y = _cells(rng, (n * k, dim), dtype)
    y[starts[-1]:] = float("nan")
    w = torch.from_numpy(rng.random((n, k)).astype(np.float32)).cuda()
    g = _cells(rng, (n, dim), dtype)
    for weights in (None, w.clone().requires_grad_()):
        y = y.detach().requires_grad_()
        out = heads.from_experts(y, r, weights)
        hw = None if weights is None else _host(weights)
        want, mag = ref.from_experts(_host(y), place, hw)
        _near(out, want, (k + 2) * ref.ULP * mag)
        out.backward(g)
        dy, dw, mag = ref.from_experts_grad(_host(g), _host(y), place, hw)
        _near(y.grad, dy, ref.ULP * np.abs(dy))
        got = heads.from_experts_grad(g, y.detach(), r, weights)
        assert torch.equal(got[0], y.grad)
        if weights is None:
            assert got[1] is None
            continue
        # a lane's products in turn (a 64th of them and a piece more), 6 levels of lanes
        _near(weights.grad, dw, (dim / 64 + 8 + 7) * ref.ULP * mag)
        assert torch.equal(got[1], weights.grad)


def test_positions_without_an_expert_take_any_weight(heads):
    """NaN and infinity there reach neither outputs nor gradients."""
    rng = np.random.default_rng(8)
    for k in (1, 2, 5):
        ids = torch.from_numpy(rng.integers(-1, 4, (500, k))).cuda()
        ids[7] = -1  # a row of none
        r = heads.Routes(ids, 4)
        y = torch.randn(500 * k, 70, device="cuda")
        g = torch.randn(500, 70, device="cuda")
        w = torch.rand(500, k, device="cuda")
        bad = torch.where(ids < 0, torch.tensor(float("nan"), device="cuda"), w)
        bad[7] = float("inf")
        assert torch.equal(heads.from_experts(y, r, bad), heads.from_experts(y, r, w))
        got, want = (heads.from_experts_grad(g, y, r, a) for a in (bad, w))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert (want[1][ids < 0] == 0).all() and (heads.from_experts(y, r, bad)[7] == 0).all()


def test_experts_leading_axes_and_odd_addresses(heads):
    rng = np.random.default_rng(3)
    ids = torch.from_numpy(rng.integers(-1, 6, (3, 5, 2))).cuda()
    flat = torch.randn(1 + 15 * 33, device="cuda", dtype=torch.bfloat16)
    x = flat[1:].view(3, 5, 33)
    r = heads.Routes(ids, 6)
    rows = heads.to_experts(x, r)
    flat_r = heads.Routes(ids.view(15, 2), 6)
    assert torch.equal(rows, heads.to_experts(x.clone().view(15, 33), flat_r))
    out = heads.from_experts(rows, r)
    assert out.shape == x.shape
    kept = (ids >= 0).sum(-1, keepdim=True)
    assert torch.equal(out, x * kept)
    t = torch.randn(33, 15, device="cuda").t()
    assert torch.equal(heads.to_experts(t, flat_r), heads.to_experts(t.contiguous(), flat_r))


def test_experts_of_more_than_2_31_cells(heads):
    n, k, dim = 600_001, 2, 2048
    ids = torch.randint(-1, 64, (n, k), device="cuda")
    r = heads.Routes(ids, 64)
    x = torch.randn(n, dim, device="cuda", dtype=torch.bfloat16)
    rows = heads.to_experts(x, r)
    at = r.place[-5:].long()
    for i in range(5):
        for j in range(k):
            a = int(at[i, j])
            want = x[n - 5 + i] if a >= 0 else torch.zeros_like(x[0])
            assert torch.equal(rows[a if a >= 0 else -1 - a], want)
    out = heads.from_experts(rows, r)
    assert torch.equal(out[-100:], x[-100:] * (ids[-100:] >= 0).sum(1, keepdim=True))
    w = torch.rand(n, k, device="cuda")
    dy, dw = heads.from_experts_grad(x, rows, r, w)
    assert torch.equal(dy[-1], rows[-1] * 0 if int(r.starts[-1]) < n * k else dy[-1])
    want = (x[-50:].double().square().sum(1, keepdim=True) * (ids[-50:] >= 0))
    assert ((dw[-50:] - want).abs() <= want * (dim / 64 + 15) * ref.ULP * 1.01).all()


# ------------------------------------------------------------------- AdamW
SIZES = [[1], [3, 1], [255, 256, 257, 1], [0, 1000, 0, 4096, 5], [4097, 20_000, 33], [70_001],
         [17] * 130, [0]]
BETAS = (0.9, 0.999)


def _state(opt):
    return [_host(a) if a is not None else None for a in opt.moments()]


def _adam_case(heads, sizes, dtype, bits, **kw):
    rng = np.random.default_rng([len(sizes), sizes[0], bits])
    params = [_cells(rng, s, dtype) for s in sizes]
    opt = heads.AdamW(params, bits=bits, **kw)
    return rng, params, opt


def _check_step(opt, params, grads, before, t, lr, decays, eps=1e-8, seed=0):
    """One step's parameters, copies and state against those before."""
    total = opt.mean.numel()
    flat = {k: np.zeros(total) for k in "gm"}
    (m, s), weights, codes = before
    got_m, got_s = (a.cpu().numpy() for a in opt.moments())
    words = ref.random_words(seed + t, total)
    for i, p in enumerate(params):
        a, n = opt.first[i], p.numel()
        part = slice(a, a + n)
        flat["g"][part] = _host(grads[i]).reshape(-1)
        (w, off), (mi, off_m), (si, off_s) = ref.adamw(
            weights[i].reshape(-1), flat["g"][part], m[part], s[part], t, lr, opt.betas, eps,
            decays[i])
        new = p if p.dtype == torch.float32 else opt.masters[i]
        _near(new.reshape(-1), w, off, ("w", i))
        if p.dtype != torch.float32:
            # (NaN in both, where a square's byte was not finite)
            assert np.array_equal(_host(p), _host(opt.masters[i].to(p.dtype)), equal_nan=True)
        if opt.bits == 32:
            _near(opt.mean[part], mi, off_m, ("m", i))
            _near(opt.square[part], si, off_s, ("s", i))
    if opt.bits == 8:
        b1, b2 = opt.betas
        with np.errstate(over="ignore", invalid="ignore"):
            m = (b1 * m + (1 - b1) * flat["g"]).astype(np.float32)
            s = (b2 * s + (1 - b2) * flat["g"] ** 2).astype(np.float32)
        cm, fm = ref.to_bytes(m, words & np.uint64(0xFFFF), False)
        cs, fs = ref.to_bytes(s, words >> np.uint64(16), True)
        assert np.array_equal(opt.scales[0].cpu().numpy(), fm)
        assert np.array_equal(opt.scales[1].cpu().numpy(), fs)
        assert np.array_equal(opt.mean.cpu().numpy(), cm)
        assert np.array_equal(opt.square.cpu().numpy(), cs)
        assert np.array_equal(got_m, ref.byte_values(cm, fm, False).astype(np.float32),
                              equal_nan=True)
        assert np.array_equal(got_s, ref.byte_values(cs, fs, True).astype(np.float32),
                              equal_nan=True)


def _before(opt, params):
    weights = [_host(p if p.dtype == torch.float32 else w) for p, w in zip(params, opt.masters)]
    if opt.bits == 32:
        return _state(opt), weights, None
    sc = opt.scales.cpu().numpy()
    return [ref.byte_values(opt.mean.cpu().numpy(), sc[0], False),
            ref.byte_values(opt.square.cpu().numpy(), sc[1], True)], weights, None


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
def test_adamw_steps(heads, sizes, dtype, bits):
    decays = [0.1 * (i % 3) for i in range(len(sizes))]
    rng, params, opt = _adam_case(heads, sizes, dtype, bits, lr=0.01, weight_decay=decays,
                                  seed=77)
    for t in range(1, 5):
        grads = [_cells(rng, s, dtype, 10.0 ** (i % 5 - 2)) for i, s in enumerate(sizes)]
        before = _before(opt, params)
        opt.step(grads)
        _check_step(opt, params, grads, before, t, 0.01, decays, seed=77)
    # cells between parameters stay zeros
    mean, square = opt.moments()
    held = torch.zeros(mean.numel(), dtype=torch.bool, device="cuda")
    for a, p in zip(opt.first, params):
        held[a:a + p.numel()] = True
    assert (mean[~held] == 0).all() and (square[~held] == 0).all()
    assert [tuple(v.shape) for v in opt.split(mean)] == [tuple(p.shape) for p in params]
    assert opt.state_dict()["step"] == 4


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_adamw_bytes_of_any_size(heads, dtype):
    """Gradients over the whole range of their type in one block, zeros, and blocks of
    subnormals: moments of 8 bits agree with the definition bit by bit."""
    rng = np.random.default_rng(5)
    n = 256 * 40
    p = torch.randn(n, device="cuda").to(TYPES[dtype])
    opt = heads.AdamW([p], lr=0.0, eps=1e-30, weight_decay=0.0, bits=8, seed=2 ** 64 - 3)
    for t in range(1, 8):
        g = rng.normal(size=n) * 2.0 ** rng.uniform(-40, 10, n)
        g[:256] = 0
        g[256:512] = 1e-38 * rng.normal(size=256)
        g[512:768] *= 1e20
        g[768:1024] *= 1e-30
        g[1024:1280] *= 2.0 ** rng.uniform(-60, 60, 256)
        grad = torch.from_numpy(g.astype(np.float32)).to(TYPES[dtype]).cuda()
        before = _before(opt, [p])
        opt.step([grad])
        _check_step(opt, [p], [grad], before, t, 0.0, [0.0], eps=1e-30, seed=2 ** 64 - 3)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_cells_that_are_not_finite_stay_alone(heads, bits):
    p = torch.randn(2000, device="cuda")
    q = p.clone()
    a, b = (heads.AdamW([x], lr=0.1, bits=bits) for x in (p, q))
    for _ in range(3):
        g = torch.randn(2000, device="cuda")
        b.step([g])
        g = g.clone()
        g[5], g[300], g[301] = float("nan"), float("inf"), -float("inf")
        a.step([g])
    bad = torch.tensor([5, 300, 301], device="cuda")
    assert torch.isnan(p[bad]).all()
    if bits == 8:
        assert torch.isnan(a.moments()[0][bad]).all() and torch.isnan(a.moments()[1][bad]).all()
    p[bad], q[bad] = 0.0, 0.0
    ok = torch.ones(2000, dtype=torch.bool, device="cuda")
    ok[bad] = False
    if bits == 32:
        assert torch.equal(p, q)
        assert torch.equal(a.mean[:2000][ok], b.mean[:2000][ok])
    else:  # (the exponents of the two blocks may differ: nothing else is NaN)
        assert torch.isfinite(p).all() and torch.isfinite(a.moments()[0][:2000][ok]).all()
        assert torch.equal(p[512:], q[512:]) and torch.equal(a.mean[512:], b.mean[512:])


def test_adamw_rounding_follows_the_mean(heads):
    """Moments of 8 bits over many cells: the sum of what a step of the square takes, 0.1 % of
    it, arrives. Each cell's rounding is a variable of its own in [0, step) with the right
    mean, so the sum of N of them has a deviation of at most step / 2 * sqrt(N): 6 of these."""
    n = 1 << 20
    p = torch.zeros(n, device="cuda")
    opt = heads.AdamW([p], lr=0.0, bits=8, seed=9)
    opt.step([torch.full((n,), 2.0, device="cuda")])
    s0 = opt.moments()[1].double()
    opt.step([torch.zeros(n, device="cuda")])
    s1 = opt.moments()[1].double()
    want = (s0 * 0.999).float().double().sum()
    step = float(s0.max()) / 8
    assert abs(float(s1.sum() - want)) <= 6 * step / 2 * n ** 0.5 + n * step * 2.0 ** -16
    assert 0 < int((s1 != s0).sum()) < n


def test_adamw_learning_rates_on_the_device(heads):
    x = torch.randn(3000, device="cuda")
    p, q = x.clone(), x.clone()
    lr = torch.tensor([0.5], device="cuda")
    a, b = heads.AdamW([p], lr=lr), heads.AdamW([q], lr=0.5)
    for v in (0.5, 0.25, 0.0):
        g = torch.randn(3000, device="cuda")
        lr.fill_(v)
        b.lr = v
        a.step([g])
        b.step([g])
        assert torch.equal(p, q)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_state_is_stored_and_taken_up(heads, bits, tmp_path):
    rng, params, opt = _adam_case(heads, [300, 5, 4096], "bf16", bits, lr=0.01, seed=3)
    grads = [[_cells(rng, p.shape, "bf16") for p in params] for _ in range(6)]
    for g in grads[:3]:
        opt.step(g)
    torch.save({"opt": opt.state_dict(), "params": params}, tmp_path / "s.pt")
    held = torch.load(tmp_path / "s.pt", weights_only=True)
    again = heads.AdamW([p.cuda() for p in held["params"]], lr=0.01, bits=bits, seed=3)
    again.load_state_dict(held["opt"])
    for g in grads[3:]:
        opt.step(g)
        again.step(g)
    for x, y in zip(params + [opt.mean, opt.square] + opt.masters,
                    again.params + [again.mean, again.square] + again.masters):
        assert torch.equal(x, y)
    assert again.state_dict()["step"] == 6
    # 16-bit parameters that were written into, taken up
    with torch.no_grad():
        params[0].fill_(3.0)
    opt.take_params()
    assert (opt.masters[0] == 3.0).all()


def test_adamw_gradients_of_backward(heads):
    """.grad by default; strided gradients; saved tensors notice the step."""
    w = torch.nn.Parameter(torch.randn(8, 6, device="cuda"))
    opt = heads.AdamW(w, lr=0.1, weight_decay=0.0)
    x = torch.randn(4, 8, device="cuda", requires_grad=True)  # (so that the product saves w)
    before = w.detach().clone()
    y = (x @ w).square().sum()
    y.backward(retain_graph=True)
    opt.step()
    assert torch.allclose((before - w).abs(), torch.full_like(w, 0.1), atol=1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
    opt.zero_grad()
    assert w.grad is None
    with pytest.raises(ValueError, match="no gradient"):
        opt.step()
    g = torch.randn(6, 8, device="cuda").t()
    v = w.detach().clone()
    other = heads.AdamW([v], lr=0.1, weight_decay=0.0)
    other.load_state_dict(opt.state_dict())
    opt.step([g])
    other.step([g.contiguous()])
    assert torch.equal(v, w)


def test_adamw_parameters_at_odd_addresses(heads):
    """Slices whose cells no 16-byte piece begins at, and cells beside them left alone."""
    for dtype in ("f32", "f16", "bf16"):
        flat = torch.full((5000,), 7.0, device="cuda", dtype=TYPES[dtype])
        grad = torch.randn(5000, device="cuda").to(TYPES[dtype])
        spans = [(1, 4), (6, 1003), (1005, 1006), (1009, 4999)]
        parts = [flat[a:b] for a, b in spans]
        copies = [p.clone() for p in parts]
        a, b = heads.AdamW(parts, lr=0.1, bits=8), heads.AdamW(copies, lr=0.1, bits=8)
        for _ in range(2):
            a.step([grad[i:j] for i, j in spans])
            b.step([grad[i:j].clone() for i, j in spans])
        for p, c in zip(parts, copies):
            assert torch.equal(p, c)
        left = torch.ones(5000, dtype=torch.bool)
        for i, j in spans:
            left[i:j] = False
        assert (flat.cpu()[left] == 7.0).all()


def test_adamw_of_more_than_2_32_bytes(heads):
    n = (1 << 31) + 4097
    p = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    g = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    g[-5:] = 1.0
    g[:5] = 1.0
    opt = heads.AdamW([p, torch.zeros(3, device="cuda")], lr=0.5, bits=8, weight_decay=0.0)
    opt.step([g, torch.ones(3, device="cuda")])
    # m / (1 - b1) = 1 and s / (1 - b2) = 1 but for roundings of 3 * 2^-24, then to bfloat16
    for part in (p[:5], p[-5:], opt.params[1]):
        assert (part.float() + 0.5).abs().max() <= 0.5 * 2.0 ** -8
    assert int((p != 0).sum()) == 10 and int((opt.square != 0).sum()) == 13


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_copies(heads, bits):
    """A copy has parameters and a state of its own and goes on as the first one would."""
    import copy
    import pickle

    p = [torch.randn(900, device="cuda"), torch.randn(5, device="cuda").bfloat16()]
    grads = [[torch.randn_like(x) for x in p] for _ in range(4)]
    opt = heads.AdamW(p, lr=0.1, bits=bits)
    opt.step(grads[0])
    copies = [copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))]
    for g in grads[1:]:
        opt.step(g)
    for c in copies:
        assert c.params[0].data_ptr() != p[0].data_ptr()
        for g in grads[1:]:
            c.step(g)
        for x, y in zip(opt.params + opt._tensors(), c.params + c._tensors()):
            assert torch.equal(x, y)
    shared = copy.copy(opt)
    shared.step(grads[0])
    assert opt.state_dict()["step"] == 5 and shared.params[0] is p[0]


def test_adamw_weight_decay_between_steps(heads):
    p = [torch.ones(300, device="cuda"), torch.ones(7, device="cuda")]
    zeros = [torch.zeros_like(x) for x in p]
    opt = heads.AdamW(p, lr=0.5, weight_decay=0.0)
    opt.step(zeros)
    assert (p[0] == 1.0).all() and opt.weight_decay == (0.0, 0.0)
    opt.weight_decay = [0.5, 0.25]
    opt.step(zeros)
    assert (p[0] == 0.75).all() and (p[1] == 0.875).all()
    for bad in ([0.1], -1.0, float("inf")):
        with pytest.raises(ValueError, match="weight_decay"):
            opt.weight_decay = bad
    assert opt.weight_decay == (0.5, 0.25)


def test_adamw_states_without_parts(heads):
    opt = heads.AdamW([torch.zeros(5, device="cuda").half()], bits=8)
    state = opt.state_dict()
    for k in ("step", "mean", "square", "scales"):
        with pytest.raises(ValueError, match=f"has no {k}"):
            opt.load_state_dict({a: b for a, b in state.items() if a != k})
    opt.params[0].fill_(2.0)
    opt.load_state_dict({k: state[k] for k in ("step", "mean", "square", "scales")})
    assert (opt.masters[0] == 2.0).all()


def test_adamw_8_bit_moments_near_the_end_of_the_range(heads):
    """A mean of 2^128, which rounding up gives, that a beta near 1 keeps beyond float32: its
    cells are NaN. 2^127 (1 - 2^-30) is 2^127 as a float, whose exponent field is 254."""
    n = 256
    p = torch.zeros(n, device="cuda")
    opt = heads.AdamW([p], lr=0.0, betas=(1.0 - 2.0 ** -30, 0.999), bits=8)
    state = opt.state_dict()
    state["mean"][:3] = torch.tensor([0x78, 0xF8, 0x70], dtype=torch.uint8)
    state["scales"][0] = 254
    opt.load_state_dict(state)
    opt.step([torch.zeros(n, device="cuda")])
    m = opt.moments()[0]
    assert torch.isnan(m[:2]).all() and float(m[2]) == 2.0 ** 127
    assert (m[3:] == 0).all() and int(opt.scales[0, 0]) == 254


def test_adamw_gradients_in_parameters_memory(heads):
    """A gradient that is another parameter, or one moved onto another's memory later, is
    refused before anything moves; neighbours in one buffer are not."""
    flat = torch.randn(4, 256, device="cuda")
    p, q, g, h = flat
    opt = heads.AdamW([p, q], lr=0.1)
    before = flat.clone()
    for grads in ([q, p], [g, flat.view(-1)[255:511]], [p, h]):
        with pytest.raises(ValueError, match="overlaps a parameter"):
            opt.step(grads)
    moved = [torch.nn.Parameter(torch.zeros(256, device="cuda")) for _ in range(2)]
    other = heads.AdamW(moved)
    moved[1].data = moved[0].data
    with pytest.raises(ValueError, match="parameters overlap"):
        other.step([g, h])
    assert torch.equal(flat, before) and opt.state_dict()["step"] == 0
    opt.step([h, g])
    assert torch.equal(flat[2:], before[2:]) and (flat[:2] != before[:2]).all()
    assert opt.state_dict()["step"] == 1
