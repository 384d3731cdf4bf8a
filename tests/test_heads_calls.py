"""Calls of the heads that their documentation allows and their ordinary use does not make,
as far as they need no device."""

from __future__ import annotations

import copy
import ctypes as C
import pickle

import numpy as np
import pytest
import torch

from ferrisboost_amd import _native as N
from ferrisboost_amd import heads
from test_host_rules import run_cpp


def test_a_sampling_call_keeps_to_its_workspace(tmp_path):
    """Launches of a call cover its rows, and take tiles only where the call's workspace
    (whose size is asked for with the whole call's rows) holds them: not the last 1 to 128
    rows of a call that takes several launches."""
    run_cpp(tmp_path, """
    const uint64_t launch = 1ull << 21;
    for (uint64_t n : std::vector<uint64_t>{1ull, 5ull, 128ull, 129ull, 4096ull, launch - 1, launch, launch + 1,
                       launch + 128, launch + 129, 3 * launch, 3 * launch + 77, 1ull << 40})
        for (uint32_t v : {1u, 1024u, 16384u, 16385u, 262144u}) {
            const uint64_t held = sample_tiled_rows(n, v);
            CHECK(held == (n <= 128 && v > 16384 ? n : 0));
            uint64_t next = 0;
            sample_launches(n, v, [&](uint64_t r, uint64_t rows, bool tiled) {
                CHECK(r == next && rows >= 1 && rows <= launch);
                CHECK(!tiled || r + rows <= held);
                CHECK(tiled == (held > 0));
                next = r + rows;
            });
            CHECK(next == n);
        }""")


def _vocabulary(sizes):
    """A vocabulary in host memory, for what happens before a device is asked for."""
    voc = object.__new__(heads.Vocabulary)
    first = np.concatenate([[0], np.cumsum(sizes)])
    voc.sizes, voc.n_tokens, voc.n_columns = np.asarray(sizes), int(first[-1]), len(sizes)
    voc.most_ids, voc.first = max(sizes), torch.from_numpy(first.astype(np.int32))
    return voc


def test_a_copied_vocabulary_gives_the_address_of_its_own_tensor():
    heads._need_torch()
    voc = _vocabulary([3, 4])
    ids = torch.zeros((5, 2), dtype=torch.int32)
    for v in (voc, copy.copy(voc), copy.deepcopy(voc), pickle.loads(pickle.dumps(voc)),
              copy.deepcopy({"a": [voc]})["a"][0]):
        e, lead = heads._positions(ids, v, True, 7, 8, 0, 1.0, 0.0, 0)
        assert heads._EMBED.unpack(e)[8] == v.first.data_ptr() and lead == (5,)


@pytest.mark.parametrize("dtype", [np.float16, np.float32, np.float64, np.longdouble, np.int64])
def test_uniforms_are_checked_as_they_are_given(dtype):
    """Numbers below 1 that float32 rounds to 1 are legal; 1 itself is not."""
    below = np.nextafter(dtype(1), dtype(0)) if dtype is not np.int64 else 0
    u = np.array([0, below, 0], dtype)
    got = heads.check_uniforms(u, 3)
    assert got.dtype == np.float32 and got.max() < 1 and got[0] == 0
    assert got[1] == min(np.float32(below), np.nextafter(np.float32(1), np.float32(0)))
    with pytest.raises(ValueError, match="in \\[0, 1\\)"):
        heads.check_uniforms(np.array([0, 1], dtype), 2)
    if dtype is not np.int64:
        for bad in (-below, np.nan, np.inf):
            with pytest.raises(ValueError, match="in \\[0, 1\\)"):
                heads.check_uniforms(np.array([bad], dtype), 1)
    with pytest.raises(ValueError, match="one value for each of 4 rows"):
        heads.check_uniforms(u, 4)


def test_uniforms_of_a_list_and_of_doubles_near_one():
    assert (heads.check_uniforms([0.25, 1 - 2.0 ** -30, 1 - 2.0 ** -24], 3)
            == np.float32([0.25, 1 - 2.0 ** -24, 1 - 2.0 ** -24])).all()
    assert heads.check_uniforms([], 0).shape == (0,)


def test_tensors_with_a_tangent_are_refused():
    """Outputs without one would read as derivatives of zero."""
    import torch.autograd.forward_ad as fwd

    x, ids = torch.ones(4, 8), torch.zeros(4, dtype=torch.int32)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: heads.embed(d, ids), lambda: heads.embed_grad(d, ids, 4),
                     lambda: heads.dropout(d, 0.5, 1), lambda: heads.sample(d, x[:, 0]),
                     lambda: heads.embed(torch.nn.Parameter(x) * d, ids)):
            with pytest.raises(ValueError, match="has a tangent"):
                call()
        with pytest.raises(ValueError, match="on a GPU"):  # a level by itself changes nothing
            heads.dropout(x, 0.5, 1)


@pytest.mark.parametrize("scale, drop", [(float("inf"), 0.0), (float("nan"), 0.0),
                                         (-float("inf"), 0.5), (3e38, 0.5), (-2e38, 0.9),
                                         (1e30, 1 - 2.0 ** -53)])
def test_scales_that_are_not_finite_are_refused(scale, drop):
    """Positions that take nothing would be zero times infinity."""
    e = N.Embed()
    e.n_rows, e.n_columns, e.dim, e.n_tokens, e.ids = 4, 3, 8, 10, 64
    e.scale, e.drop = scale, drop
    L = N.hip()
    with pytest.raises(ValueError, match="finite"):
        N.check_hip(L.fbh_embed_rows(0, C.byref(e), 64, 64, None))
    with pytest.raises(ValueError, match="finite"):
        N.check_hip(L.fbh_embed_grad(0, C.byref(e), 64, 64, 64, 1 << 40, None))
    assert L.fbh_embed_grad_bytes(C.byref(e)) == 0


@pytest.mark.parametrize("scale", [float("inf"), float("nan"), 1e39, -1e300])
def test_scales_beyond_float32(scale):
    with pytest.raises(ValueError, match="finite float32"):
        heads._scale(scale)


@pytest.mark.parametrize("sizes", [[1 << 62] * 3 + [(1 << 62) + 5], [1 << 31], [3, 1 << 40],
                                   np.array([2 ** 63, 2 ** 63 - 1, 2], np.uint64)])
def test_sizes_whose_sum_is_beyond_64_bits(sizes):
    with pytest.raises(ValueError, match="at most 2\\^31 - 1 ids"):
        heads.Vocabulary(sizes)


@pytest.mark.parametrize("value", [float("inf"), float("nan"), None, "many"])
def test_whole_numbers(value):
    for check in (heads._seed, heads._top_k):
        with pytest.raises(ValueError, match="whole number"):
            check(value)
    assert heads._seed(2 ** 64 - 1) == 2 ** 64 - 1 and heads._top_k(5.0) == 5
    assert heads._top_k(1 << 40) == 0x7FFFFFFF


def test_sizes_beyond_32_bits_are_value_errors():
    """(tensors of one element, expanded)"""
    heads._need_torch()
    wide = torch.zeros((1, 1), dtype=torch.int32).expand(2, 1 << 32)
    ids = torch.zeros((2, 3), dtype=torch.int32)
    for args in ((wide, None, True, 5, 8), (ids, None, False, 1 << 32, 1),
                 (ids, None, False, 1, 1 << 32)):
        with pytest.raises(ValueError, match="below 2\\^32"):
            heads._positions(*args, 0, 1.0, 0.0, 0)


def _columns(rows, columns, ids, dim, dtype, pooled=1):
    e = N.Embed()
    e.n_rows, e.n_columns, e.dim, e.n_tokens, e.most_ids = rows, columns, dim, columns * ids, ids
    e.ids, e.first, e.scale, e.dtype, e.pooled = 64, 64, 1.0, dtype, pooled
    return e


@pytest.mark.parametrize("rows, columns, ids, dim, dtype", [
    (1_000_000, 400, 1000, 160, 2), (100_000, 100, 511, 64, 2), (40_000, 96, 1000, 1024, 2),
    (9000, 32_768, 1024, 512, 0), (1 << 29, 1, 1024, 64, 0), (1 << 29, 1, 7, 32_768, 0),
    (65_536, 20, 1024, 32_768, 1), (70_000, 3, 1024, 32_768, 0)])
def test_workspace_of_column_gradients_is_bounded(rows, columns, ids, dim, dtype):
    """2 bytes a position (chunks are rounded up to 64 rows), and parts of 1 GiB or an eighth
    of an f32 vector a row, with two bytes of counts a vector. 1M rows of 400 columns of 1000 ids, 160 cells,
    took 16 GB."""
    got = N.hip().fbh_embed_grad_bytes(C.byref(_columns(rows, columns, ids, dim, dtype)))
    # (at most a chunk for 64 rows and one more)
    parts = max(1 << 30, rows * dim // 2)
    assert got <= 2 * (2 * rows + 64) * columns + parts + parts // (2 * dim) + 4096
    assert got >= 2 * rows * columns


@pytest.mark.parametrize("n, tokens, dim", [(1 << 20, 50_000, 64), (60_000, 50_000, 1024),
                                            ((1 << 31) - 1, 1 << 30, 1), (1 << 25, 4096, 32_768)])
def test_workspace_of_sorted_gradients(n, tokens, dim):
    e = _columns(n, 1, tokens, dim, 0)
    e.first, e.most_ids = None, 0
    got = N.hip().fbh_embed_grad_bytes(C.byref(e))
    assert 16 * n <= got <= 17 * n + n * dim // 2 + 16 * dim + (1 << 20)


@pytest.mark.parametrize("columns", [1 << 31, (1 << 32) - 1024, (1 << 32) - 1])
def test_rows_of_too_many_columns_to_sum_are_refused(columns):
    """The summing kernels' steps over a row would pass 2^32 and never end."""
    e = _columns(3, 1, 4, 8, 0)
    e.first, e.n_columns, e.most_ids = None, columns, 0
    with pytest.raises(ValueError, match="2147483647 columns"):
        N.check_hip(N.hip().fbh_embed_rows(0, C.byref(e), 64, 64, None))


def test_a_copied_vocabulary_has_been_used_on_no_stream():
    """Also one that was stored without the streams it had been used on."""
    voc = _vocabulary([3, 4])
    voc._streams = {0, 77}
    for v in (copy.copy(voc), copy.deepcopy(voc), pickle.loads(pickle.dumps(voc))):
        assert v._streams == set() and torch.equal(v.first, voc.first)
    assert voc._streams == {0, 77}
    del voc._streams
    assert pickle.loads(pickle.dumps(voc))._streams == set()
