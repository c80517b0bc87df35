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
