"""dec_beam_select with one workspace for batches of every size."""

from __future__ import annotations

import pytest
import torch

from paged_helpers import BF, select64

pytestmark = pytest.mark.gpu


def test_one_workspace_for_all_batches(gpu):
    """Sized for 300 rows and used for 300, 256, 255, 8 and 1: on both sides of the change of the parts' length."""
    from kernels.cuda_ext import ext

    V, g = 16384, torch.Generator().manual_seed(0)
    work = torch.empty(ext.dec_beam_select_work(300, V, 1), dtype=torch.uint8).cuda()
    x = (3 * torch.randn(300, V, generator=g)).to(BF)
    score, finished = -torch.rand(300, 1, generator=g), torch.zeros(300, 1, dtype=torch.uint8)
    for n in (300, 256, 255, 8, 1):
        groups = torch.arange(n, dtype=torch.int32)
        parent, token = torch.zeros(n, 1, dtype=torch.int32).cuda(), torch.zeros(n, 1, dtype=torch.int64).cuda()
        total = torch.zeros(n, 1).cuda()
        ext.dec_beam_select(x[:n].cuda(), groups.cuda(), score.cuda(), finished.cuda(), None, None, 2, parent, token, total,
                            work)
        want = select64(x[:n], groups, score, finished, None, None, 2)
        assert torch.equal(token.cpu(), want[1]) and torch.equal(parent.cpu(), want[0])
        err = (total.cpu().double() - want[2]).abs()
        assert (err <= 2.0 ** -24 * want[2].abs() * (1 + 2.0 ** -20) + 2.0 ** -32).all()
