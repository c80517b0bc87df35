"""What the beam search's entry points refuse and say of their sizes, on the CPU."""

from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("eos", [-2, 64, 2 ** 40])
def test_select_refuses_end_tokens_outside_the_vocabulary(eos):
    from kernels.cuda_ext import ext

    lib, p = ext._lib, torch.zeros(4096).data_ptr()
    a = dict(logits=p, ld=64, n=2, beams=4, V=64, groups=p, slots=3, score=p, finished=p, made=None, norm=None, norm_len=0,
             pad=3, eos=eos, parent=p, token=p, total=p, work=p, work_bytes=8 * (16 + 32), stream=None)
    assert lib.cohere_dec_beam_select_eos(*a.values()) == 1 and b"end token" in lib.cohere_last_error()
    a.update(eos=63, n=0)
    assert lib.cohere_dec_beam_select_eos(*a.values()) == 0


@pytest.mark.parametrize("V", [8, 16384, 16392, 100008, 4200000])
@pytest.mark.parametrize("B", [1, 4, 16])
def test_select_work_is_enough_for_fewer_rows(V, B):
    """A workspace sized for the most rows serves every smaller call: no fewer bytes for more rows, also where longer
    stretches a workgroup leave fewer parts."""
    from kernels.cuda_ext import ext

    sizes = [ext.dec_beam_select_work(rows, V, B) for rows in range(1, 600)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:]))
    part = 16 + 8 * B
    for rows, size in zip(range(1, 600), sizes):  # parts of 2048 logits up to 255 stretches of 16384 in all, of 16384 behind
        parts = -(-V // (2048 if rows * -(-V // 16384) < 256 else 16384))
        assert size >= rows * parts * part
    assert sizes[0] == -(-V // (2048 if -(-V // 16384) < 256 else 16384)) * part
