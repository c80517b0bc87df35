"""Beam search's selection, reordering and advance against the definitions in 64 bits: parents and tokens are whole
numbers and have to be equal, as has everything that is moved."""

from __future__ import annotations

import math

import pytest
import torch

from paged_helpers import BF, reorder64, same_bits, select64

pytestmark = pytest.mark.gpu


def _select(logits, groups, score, finished, made=None, norm=None, pad=2, ld=None):
    from kernels.cuda_ext import ext

    n, (G, B), V = len(groups), score.shape, logits.shape[1]
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    x = torch.full((n * B, ld or V), float("nan"), dtype=BF).cuda()[:, :V]
    x.copy_(logits)
    parent = torch.full((n, B), -7, dtype=torch.int32).cuda()
    token = torch.full((n, B), -7, dtype=torch.int64).cuda()
    total = torch.full((n, B), float("nan")).cuda()
    work = torch.empty(ext.dec_beam_select_work(n * B, V, B), dtype=torch.uint8).cuda()
    ext.dec_beam_select(x, dev(groups), dev(score), dev(finished), dev(made), dev(norm), pad, parent, token, total, work)
    torch.cuda.synchronize()
    return parent.cpu(), token.cpu(), total.cpu()


def _same(args, **kw):
    """Parents and tokens equal; totals are rounded once to fp32, 2^-24 of them, after an error of 2^-32 in all.

    Candidates of different beams may have totals that are equal but for the roundings of their sums (rows of the same
    logits in another order): which of them comes first is then the sums' affair, on either side. The exponentials are off
    by 6e-11 of themselves at most, so a logarithm of their sum by 6e-11; a sum of V of them in 64 bits adds V 2^-53, below
    2e-11 up to V = 131072, and the reference as much: ranks (norms are at most 1) within 2e-10 may change places. Of one
    beam's candidates the logits decide, and then the index."""
    got = _select(*args, **kw)
    kw.pop("ld", None)
    ranks = []
    want = select64(*args[:4], *(kw.get(k) for k in ("made", "norm")), kw.get("pad", 2), ranks)
    for i in ((got[0] != want[0]) | (got[1] != want[1])).any(1).nonzero().flatten().tolist():
        at = got[0][i].long() * ranks[i].shape[1] + got[1][i]
        assert len(set(at.tolist())) == len(at) and (got[1][i] < ranks[i].shape[1]).all()
        flat = torch.from_numpy(ranks[i].reshape(-1))
        here, there = flat[at], flat[want[0][i].long() * ranks[i].shape[1] + want[1][i]]
        assert torch.equal(here.isinf(), there.isinf())
        assert torch.equal(at[here.isinf()], (want[0][i].long() * ranks[i].shape[1] + want[1][i])[here.isinf()])
        assert ((here - there).abs()[~here.isinf()] <= 2e-10).all()
        for b in range(ranks[i].shape[0]):
            own = here[got[0][i] == b], got[1][i][got[0][i] == b]
            assert all(x > y or (x == y and s < t) for x, y, s, t in zip(own[0], own[0][1:], own[1], own[1][1:]))
    inf = torch.isinf(want[2])
    assert torch.equal(got[2][inf].double(), want[2][inf])
    err = (got[2].double() - want[2]).abs()[~inf]
    assert (err <= 2.0 ** -24 * want[2].abs()[~inf] * (1 + 2.0 ** -20) + 2.0 ** -32).all()
    return got


def _inputs(seed, n, B, V, G=None, ended=0.2, std=3.0):
    g = torch.Generator().manual_seed(seed)
    G = G or n + 2
    groups = torch.randperm(G, generator=g)[:n].to(torch.int32)
    logits = (std * torch.randn(n * B, V, generator=g)).to(BF)
    score = -30 * torch.rand(G, B, generator=g)
    finished = (torch.rand(G, B, generator=g) < ended).to(torch.uint8)
    made = torch.randint(0, 40, (G, B), generator=g, dtype=torch.int32)
    return [logits, groups, score, finished], made


@pytest.mark.parametrize("B", [1, 2, 3, 4, 5, 8, 11, 16])
@pytest.mark.parametrize("n,V", [(1, 16), (3, 64), (2, 2048), (5, 2056), (1, 16384), (40, 8200), (2, 100008)])
def test_select(gpu, n, B, V):
    print(f"select n={n} B={B} V={V}", flush=True)
    a, made = _inputs(n * B + V, n, B, V)
    _same(a)
    norm = torch.arange(33).clamp_min(1).double().pow(-0.7).float()
    _same(a, made=made, norm=norm, ld=V + 8)


@pytest.mark.parametrize("B", [1, 4, 16])
@pytest.mark.parametrize("V", [16, 4096, 20000])
def test_select_ties_go_to_the_lowest_index(gpu, B, V):
    """Equal logits, all or many of them, across lanes, waves and workgroups, and -0 beside 0."""
    a, _ = _inputs(B + V, 2, B, V, ended=0.0)
    a[0][:] = 0.0
    a[0][1::2, ::3] = -0.0
    a[2][:] = -1.0  # beams of equal scores: b decides
    got = _same(a)
    assert got[1].tolist() == [list(range(B))] * 2 and (got[0] == 0).all()
    a[0][:, -5:] = 1.5
    a[0][:, V // 2] = 1.5
    _same(a)
    a[0] = (torch.randint(0, 3, a[0].shape) / 4).to(BF)
    _same(a)


def test_select_masked_rows(gpu):
    """Masks that leave nothing, one token or a few; NaN and infinities among the logits; beams of score -inf."""
    for B in (1, 3, 8, 16):
        a, made = _inputs(B, 6, B, 4096, ended=0.1)
        x = a[0].reshape(6, B, -1)
        x[0] = -math.inf
        x[1, :, 3:] = -math.inf
        x[2, 0] = -math.inf
        x[2, 0, 77] = -50.0
        x[3, :, ::7] = float("nan")
        x[4, 0, 100:104] = math.inf
        x[4, -1, :] = float("nan")
        x[5] = torch.finfo(BF).min
        _same(a)
        a[2][a[1][1].long(), 1:] = -math.inf
        a[2][a[1][2].long()] = float("nan")
        a[2][a[1][5].long(), 0] = -math.inf
        _same(a, made=made, norm=torch.tensor([1.0, 0.5, 0.25]))


def test_select_many_rows(gpu):
    """As many rows as take long stretches a workgroup: masks, equal logits, NaN and infinities there too."""
    for B in (3, 4, 13):
        n = 300 // B
        a, made = _inputs(B, n, B, 16400)
        x = a[0].reshape(n, B, -1)
        x[0] = -math.inf
        x[1, :, 5:] = -math.inf
        x[2, 0, :16380] = -math.inf
        x[3, :, ::7] = float("nan")
        x[4, 0, 100:104] = math.inf
        x[5] = 0.25
        x[6] = (torch.randint(0, 3, x[6].shape, generator=torch.Generator().manual_seed(1)) / 4).to(BF)
        x[7, -1, 4096:] = float("nan")
        x[8, :, :] = -math.inf
        x[8, 0, 4096:4104] = 1.0  # one lane's
        x[9, :, 512:1024] = 8.0
        _same(a)
        _same(a, made=made, norm=torch.tensor([1.0, 0.5, 0.25]))


def test_select_ended_beams(gpu):
    """Groups whose beams have all ended keep them in order of their scores; pad at the ends of the vocabulary."""
    for pad in (0, 5, 63):
        a, _ = _inputs(pad, 3, 8, 64, ended=1.1)
        a[2] = a[2].sort(1, descending=True).values
        got = _same(a, pad=pad)
        assert torch.equal(got[0], torch.arange(8, dtype=torch.int32).repeat(3, 1)) and (got[1] == pad).all()
        a[3][:, ::2] = 0
        _same(a, pad=pad)


def test_select_groups_out_of_range(gpu):
    a, _ = _inputs(4, 4, 4, 512)
    a[1][0], a[1][2] = -1, a[2].shape[0]
    got = _same(a)
    assert got[0][0].tolist() == [0, 1, 2, 3] and (got[2][2] == -math.inf).all()


def test_select_close_candidates(gpu):
    """Candidates of different beams whose totals differ by 1e-8: in 32 bits they would be equal."""
    g = torch.Generator().manual_seed(0)
    V, tried = 16384, 0
    for seed in range(20):
        logits = (2 * torch.randn(2, V, generator=g)).to(BF)
        l = logits.double()
        lse = torch.logsumexp(l, 1)
        top = l.max(1).values
        # the second beam's best lands just above or below the first's: scores are fp32, so the gap is what they leave
        score = torch.zeros(1, 2)
        score[0, 0] = -0.001 * seed
        score[0, 1] = float(score[0, 0].double() + (top[0] - lse[0]) - (top[1] - lse[1]))
        gap = float(score[0, 0].double() + top[0] - lse[0] - (score[0, 1].double() + top[1] - lse[1]))
        tried += 1e-9 < abs(gap) < 1e-6
        _same([logits, torch.zeros(1, dtype=torch.int32), score, torch.zeros(1, 2, dtype=torch.uint8)])
    assert tried >= 10


def test_select_captured(gpu):
    """A captured call replayed with new logits, eager work between."""
    from kernels.cuda_ext import ext

    a, made = _inputs(1, 3, 4, 8192)
    dev = [t.cuda() for t in a]
    parent, token = torch.zeros(3, 4, dtype=torch.int32).cuda(), torch.zeros(3, 4, dtype=torch.int64).cuda()
    total = torch.zeros(3, 4).cuda()
    work = torch.empty(ext.dec_beam_select_work(12, 8192, 4), dtype=torch.uint8).cuda()

    def call():
        ext.dec_beam_select(*dev, None, None, 2, parent, token, total, work)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(4):
        a[0] = (3 * torch.randn(12, 8192, generator=torch.Generator().manual_seed(i))).to(BF)
        dev[0].copy_(a[0].cuda())
        work.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        want = select64(*a, None, None, 2)
        assert torch.equal(parent.cpu(), want[0]) and torch.equal(token.cpu(), want[1])
        torch.randn(1000, device="cuda").sum()


@pytest.mark.parametrize("bits", [16, 8, 0])
@pytest.mark.parametrize("B", [1, 2, 4, 5, 8, 16])
@pytest.mark.parametrize("P,n_held", [(1, [0, 1, 40]), (16, [15, 16, 37]), (4, [3, 40, 41]), (64, [5, 40, 0])])
def test_reorder(gpu, bits, B, P, n_held):
    from kernels.cuda_ext import ext

    print(f"reorder bits={bits} B={B} P={P}", flush=True)
    if bits == 0 and P != 1:
        return
    g = torch.Generator().manual_seed(B * P)
    G, OUT, L, kv = 5, 43, 2, 3
    W = 48 // P + 1
    groups = torch.tensor([3, 0, 4], dtype=torch.int32)
    parent = torch.randint(0, B, (3, B), generator=g, dtype=torch.int32)
    parent[1, 0], parent[1, B - 1] = B, -1  # rows left as they are
    if B > 1:
        parent[2] = torch.roll(torch.arange(B, dtype=torch.int32), 1)  # every beam moves
    held = torch.zeros(G, dtype=torch.int32)
    held[groups.long()] = torch.tensor(n_held, dtype=torch.int32)
    n = held.repeat_interleave(B)
    pages = G * B * W + 1
    table = torch.randperm(pages, generator=g)[:G * B * W].reshape(G * B, W).to(torch.int32)
    table[3 * B, min(n_held[0] // P, W - 1)] = pages  # an absent page: nothing is copied from or to it
    tokens = torch.randint(0, 10 ** 12, (G * B, OUT), generator=g)
    states = torch.randint(-5, 5, (G * B, 2), generator=g, dtype=torch.int32)
    k = v = ks = vs = None
    if bits == 16:
        k, v = (torch.randn(L, pages, kv, P, 128, generator=g).to(BF) for _ in range(2))
    elif bits == 8:
        k, v = (torch.randint(-127, 128, (L, pages, kv, P, 128), generator=g, dtype=torch.int8) for _ in range(2))
        ks, vs = (torch.rand(L, pages, kv, P, generator=g) for _ in range(2))
    for done in (None, torch.tensor([1, 0, 0, 0, 1], dtype=torch.uint8)):
        state = [None if t is None else t.cuda() for t in (table, tokens, states, k, v, ks, vs)]
        ext.dec_beam_reorder(groups.cuda(), parent.cuda(), n.cuda(), None if done is None else done.cuda(), *state)
        want = reorder64(groups, parent, n, done, P, table, tokens, states, k, v, ks, vs)
        for got, w in zip(state, want):
            assert same_bits(None if got is None else got.cpu(), w)


def test_reorder_parts_and_groups_out_of_range(gpu):
    """Absent tables, tokens and states; groups out of range; more positions than the table and the tokens have."""
    from kernels.cuda_ext import ext

    g = torch.Generator().manual_seed(0)
    groups = torch.tensor([1, -1, 2], dtype=torch.int32)
    parent = torch.tensor([[1, 0], [1, 0], [1, 1]], dtype=torch.int32)
    n = torch.full((4,), 100, dtype=torch.int32)
    table = torch.randint(0, 9, (4, 3), generator=g, dtype=torch.int32)
    tokens = torch.randint(0, 9, (4, 7), generator=g)
    k, v = (torch.randn(1, 9, 1, 16, 128, generator=g).to(BF) for _ in range(2))
    for use in ((1, 1), (1, 0), (0, 1), (0, 0)):
        state = [table if use[0] else None, tokens if use[1] else None, None] + ([k, v] if use[0] else [None, None])
        dev = [None if t is None else t.cuda() for t in state] + [None, None]
        ext.dec_beam_reorder(groups.cuda(), parent.cuda(), n.cuda(), None, *dev)
        want = reorder64(groups, parent, n, None, 16 if use[0] else 1, *state, None, None)
        for got, w in zip(dev, want):
            assert same_bits(None if got is None else got.cpu(), w)


@pytest.mark.parametrize("by_length", [False, True])
@pytest.mark.parametrize("B,width", [(1, 256), (4, 512), (5, 1024), (16, 264)])
def test_advance(gpu, B, width, by_length):
    """The state after a step, and embeddings equal to dec_embed's."""
    from kernels.cuda_ext import ext

    g = torch.Generator().manual_seed(B)
    G, OUT, V, eos, dummy = 7, 20, 64, 3, 6
    groups = torch.tensor([5, 0, 6, 2, 3, 6, 1], dtype=torch.int32)
    n = len(groups)
    parent = torch.randint(0, B, (n, B), generator=g, dtype=torch.int32)
    token = torch.randint(0, V, (n, B), generator=g)
    total = -10 * torch.rand(n, B, generator=g)
    tok, pos = torch.randint(0, V, (G * B,), generator=g), torch.randint(0, 18, (G,), generator=g).repeat_interleave(B).int()
    score, made = -9 * torch.rand(G, B, generator=g), torch.randint(0, 9, (G, B), generator=g, dtype=torch.int32)
    finished = (torch.rand(G, B, generator=g) < 0.3).to(torch.uint8)
    done = torch.zeros(G, dtype=torch.uint8)
    limit = pos.reshape(G, B)[:, 0] + 5
    out = torch.randint(0, V, (G * B, OUT), generator=g)
    done[0] = 1  # keeps its state
    token[0, 0] = eos  # group 5: the best ends
    finished[5, parent[0, 0]] = 0
    limit[2] = pos[2 * B] + 1  # at its limit
    token[4] = eos  # group 3: all end
    total[6] = -math.inf  # group 1: no candidate
    limit = limit.int()
    emb, ptab = (torch.randn(r, width, generator=g).to(BF) for r in (V, 19))
    w0, b0, w1, b1 = (torch.randn(width, generator=g).to(BF) for _ in range(4))
    dev = [t.cuda() for t in (groups, parent, token, total)]
    state = [t.cuda() for t in (tok, pos, score, finished, made, done, limit, out)]
    held = torch.full_like(state[1], -3) if B != 4 else None
    x, h = (torch.empty(n * B, width, dtype=BF).cuda() for _ in range(2))
    flags = torch.zeros(G, dtype=torch.uint8).pin_memory()
    norms = [t.cuda() for t in (w0, b0, w1, b1)]
    ext.dec_beam_advance(*dev, dummy, *state[:2], held, *state[2:], eos, by_length, emb.cuda(), ptab.cuda(), norms[0], norms[1], 1e-5, norms[2],
                         norms[3], 1e-6, x, h, flags)
    torch.cuda.synchronize()
    w = [t.clone() for t in (tok, pos, score, finished, made, done, out)]
    for i, gr in enumerate(groups.tolist()):
        if gr == dummy or done[gr]:
            continue
        ends = []
        for b in range(B):
            r, q = gr * B + b, int(parent[i, b])
            was = bool(finished[gr, q])
            p = int(pos[r]) + 1
            w[0][r], w[1][r], w[2][gr, b], w[6][r, p] = token[i, b], p, total[i, b], token[i, b]
            ends.append(was or int(token[i, b]) == eos or float(total[i, b]) == -math.inf)
            w[3][gr, b], w[4][gr, b] = ends[-1], made[gr, q] + (not was)
        w[5][gr] = all(ends) or (not by_length and ends[0]) or p >= int(limit[gr])
    for got, want in zip(state[:6] + state[7:], w):
        assert torch.equal(got.cpu(), want)
    if held is not None:
        moved = w[1] != pos
        assert torch.equal(held.cpu(), torch.where(moved, w[1] + 1, torch.full_like(w[1], -3)))
    assert torch.equal(flags.bool(), w[5].bool() & ~done.bool())
    rows = (groups.long()[:, None] * B + torch.arange(B)).reshape(-1).int().cuda()
    x1, h1 = torch.empty_like(x), torch.empty_like(h)
    ext.dec_embed(rows, state[0], state[1].clamp_max(18), emb.cuda(), ptab.cuda(), norms[0], norms[1], 1e-5, norms[2],
                  norms[3], 1e-6, x1, h1)
    assert torch.equal(x, x1) and torch.equal(h, h1)
