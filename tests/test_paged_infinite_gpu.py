"""Attention over pages where values are infinite or NaN: held in pages and as given, in few and in many query rows, whole
and in parts, against the definition in 64 bits."""

from __future__ import annotations

import pytest
import torch

from paged_helpers import D, Paged, close

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def _held(c, s, t, dim, x, what="v"):
    """Held position t of sequence s gets x in a dimension."""
    page, off = c.place(int(c.active[s]), t)
    getattr(c, what)[page, :, off, dim] = x


def _check(c, splits, many, starts="own"):
    want, bound, written = c.attention64(weights_bf16=many)
    got = c.run(splits, starts)[0].double()
    want, bound, got = want[written], bound[written], got[written]
    there = want.isfinite()
    close(got[there], want[there], bound[there])
    same = (got == want) | (got.isnan() & want.isnan())
    assert same[~there].all(), f"{int((~same[~there]).sum())} of {int((~there).sum())}"
    return got, want


@pytest.mark.parametrize("page", [16, 4, 1])
@pytest.mark.parametrize("splits", [1, 2, 3, 7])
@pytest.mark.parametrize("chunk,ratio", [([1], 1), ([1], 5), ([3], 2), ([40], 2), ([200], 1)])
def test_infinities_among_held_values(gpu, page, splits, chunk, ratio):
    """They reach their own dimensions alone, as the sum's definition has it: an infinity however small its weight is,
    NaN where both signs meet; and those of a chunk's own tokens the rows that see them."""
    c = Paged(31 + page, [300], chunk, 2, ratio, page, 16)
    n = 300
    for t, dim, x in ((0, 3, INF), (299, 5, -INF), (130, 7, INF), (40, 7, -INF), (77, 9, NAN), (31, 11, INF), (32, 11, INF),
                      (200, 127, INF), (5, 64, -INF)):
        _held(c, 0, t, dim, x)
    own = c.q[:, (c.H + c.kv) * D:]
    own[chunk[0] // 2, 20], own[chunk[0] // 2, D + 3] = INF, -INF
    many = chunk[0] * ratio > 16
    got, want = _check(c, splits, many)
    assert got.reshape(-1, c.H, D)[:, :, 5].eq(-INF).all() and got.reshape(-1, c.H, D)[:, :, 0].isfinite().all()
    # behind a score far below the others (2^-200 of the largest weight)
    c = Paged(32, [n], chunk, 1, ratio, page, 16)
    c.q[:, :c.H * D] = 4.0
    c.k[c.k.isfinite()] = 0
    low = -200.0 / (4.0 * D * c.scale * 1.4427)
    for t in range(64):
        page_, off = c.place(int(c.active[0]), t)
        c.k[page_, :, off] = low
    c.q[:, c.H * D:(c.H + 1) * D] = 0
    _held(c, 0, 10, 2, INF)
    got, want = _check(c, splits, many)
    assert got.reshape(-1, c.H, D)[:, :, 2].eq(INF).all() and want.isfinite().any()


@pytest.mark.parametrize("starts", ["own", None])
def test_single_tokens_over_infinities(gpu, starts):
    c = Paged(33, [40, 0, 700], [1, 1, 1], 3, 2, 16, 16)
    _held(c, 0, 39, 1, INF)
    _held(c, 2, 0, 2, -INF)
    c.q[1, (c.H + c.kv) * D + 4] = INF  # the second sequence's own value, its only one
    for splits in (1, 4):
        _check(c, splits, False, starts)


@pytest.mark.parametrize("splits", [1, 2, 5])
@pytest.mark.parametrize("chunk", [[1], [7], [50]])
def test_scales_that_are_not_finite(gpu, splits, chunk):
    """int8 vectors without a scale (NaN, as the kernels write them; infinite, as a caller may) make their dimensions what
    code x scale is, NaN for a code of 0."""
    c = Paged(36, [90], chunk, 2, 2, 16, 8)
    page, off = c.place(int(c.active[0]), 70)
    c.vs[page, 1, off] = NAN
    c.v[page, 0, off, ::3] = 0
    c.vs[page, 0, off] = INF
    got, want = _check(c, splits, chunk[0] * 2 > 16)
    rows = got.reshape(-1, c.H, D)
    assert rows[:, 2:].isnan().all() and rows[:, :2, ::3].isnan().all() and rows[:, :2].isinf().any()
