"""dec_beam_select with one workspace for batches of every size; dec_beam_advance at the ends of its rows."""

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


def test_advance_at_positions_that_out_does_not_have(gpu):
    """Positions below zero and behind the last one: the state moves on, and no row's tokens change."""
    from kernels.cuda_ext import ext

    G, B, OUT, width = 3, 2, 6, 256
    groups = torch.arange(G, dtype=torch.int32).cuda()
    parent, token = torch.zeros(G, B, dtype=torch.int32).cuda(), torch.full((G, B), 9).cuda()
    total = torch.full((G, B), -1.0).cuda()
    pos = torch.tensor([-40, -40, 5, 5, 3, 3], dtype=torch.int32)
    guard = torch.full((G * B + 16, OUT), 7).cuda()  # rows of other memory around out
    tok, score = torch.zeros(G * B, dtype=torch.int64).cuda(), torch.zeros(G, B).cuda()
    ended, made = torch.zeros(G, B, dtype=torch.uint8).cuda(), torch.zeros(G, B, dtype=torch.int32).cuda()
    done, limit = torch.zeros(G, dtype=torch.uint8).cuda(), torch.full((G,), 100, dtype=torch.int32).cuda()
    emb, ptab = torch.ones(16, width, dtype=BF).cuda(), torch.ones(8, width, dtype=BF).cuda()
    ln = torch.ones(width, dtype=BF).cuda()
    x, h = (torch.empty(G * B, width, dtype=BF).cuda() for _ in range(2))
    pos_d = pos.cuda()
    ext.dec_beam_advance(groups, parent, token, total, G, tok, pos_d, None, score, ended, made, done, limit, guard[8:-8], 3,
                         False, emb, ptab, ln, ln, 1e-5, ln, ln, 1e-5, x, h, None)
    want = torch.full((G * B + 16, OUT), 7)
    want[8 + 4:8 + 6, 4] = 9
    assert torch.equal(guard.cpu(), want) and torch.equal(pos_d.cpu(), pos + 1)
