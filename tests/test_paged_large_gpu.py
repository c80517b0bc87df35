"""Attention over pages where values are the type's largest, or very small: held in pages and as given, in few and in many
query rows, whole and in parts, against the definition in 64 bits."""

from __future__ import annotations

import pytest
import torch

from paged_helpers import BF, D, Paged, close, held_q8

pytestmark = pytest.mark.gpu
TOP = torch.finfo(BF).max


def _check(c, splits, many, starts="own"):
    want, bound, written = c.attention64(weights_bf16=many)
    got = c.run(splits, starts)[0].double()
    want, bound, got = want[written], bound[written], got[written]
    close(got, want, bound)
    return got, want


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("splits", [1, 2, 5])
@pytest.mark.parametrize("held,chunk,ratio", [(2, [1], 1), (700, [1], 4), (5000, [1], 1), (30, [6], 2), (0, [300], 1),
                                              (700, [90], 2), (3000, [20], 1)])
def test_the_types_largest_values_stay_finite(gpu, bits, splits, held, chunk, ratio):
    """A mean of values up to the type's largest is no larger: sums over many keys of nearly equal weight, with scores
    that are level and that rise by less than 8 behind the first."""
    for rise in (0.0, 5.0):
        c = Paged(34 + held, [held], chunk, 1, ratio, 16, 16)
        for t in range(held):
            page, off = c.place(int(c.active[0]), t)
            c.k[page, :, off] = 0
            c.k[page, :, off, 0] = rise * min(t, 40) / 40
            c.v[page, :, off, :64], c.v[page, :, off, 64:96], c.v[page, :, off, 96:] = TOP, -TOP, TOP / 3
        c.q[:, :c.H * D] = 0
        c.q[:, :c.H * D:D] = 8.0
        c.q[:, c.H * D:(c.H + 1) * D] = 0
        c.q[:, c.H * D] = rise
        own = c.q[:, (c.H + 1) * D:]
        own[:, :64], own[:, 64:96], own[:, 96:] = TOP, -TOP, TOP / 3
        if bits == 8:
            (c.k, c.ks), (c.v, c.vs), c.bits = held_q8(c.k.nan_to_num(0)), held_q8(c.v.nan_to_num(0)), 8
        got, _ = _check(c, splits, chunk[0] * ratio > 16)
        assert got.isfinite().all()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("held,chunk", [(5000, [1]), (5000, [9]), (900, [60])])
def test_small_values_keep_their_digits(gpu, bits, held, chunk):
    """Values around 2^-70 under weights that are small for the large ones' sake."""
    c = Paged(35, [held], chunk, 1, 2, 16, bits, v_std=2.0 ** -71)
    c.q[:, (c.H + 1) * D:] = (c.q[:, (c.H + 1) * D:].float() * 2.0 ** -70).to(BF)
    for splits in (1, 4):
        _check(c, splits, chunk[0] * 2 > 16)
