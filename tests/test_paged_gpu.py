"""Attention of chunks of new tokens over caches in pages, and their reading back, against the definitions in 64 bits.
What the pages hold is whole: it has to be equal."""

from __future__ import annotations

import pytest
import torch

from paged_helpers import BF, D, Paged, close, same_bits

pytestmark = pytest.mark.gpu


def _check(c, splits=1, starts="own", **kw):
    if starts is None:
        got = c.run(splits, None)
    else:
        got = c.run(splits)
    want, bound, written = c.attention64(**kw)
    close(got[0][written], want[written], bound[written])
    assert (got[0][~written] == 7).all()
    for a, b in zip(got[1:], c.appended()):
        assert same_bits(a, b)
    return got


@pytest.mark.parametrize("ratio", [1, 2, 3, 4, 5, 8, 16, 17])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("page,held", [(1, [0, 1, 5]), (16, [15, 16, 17, 0, 200]), (4, [3, 4, 63, 64, 65]), (256, [255, 256, 257])])
def test_single_tokens(gpu, bits, ratio, page, held):
    print(f"paged single bits={bits} ratio={ratio} page={page}", flush=True)
    c = Paged(page * 100 + ratio, held, [1] * len(held), 2, ratio, page, bits, pad=8)
    _check(c, weights_bf16=ratio > 16)
    _check(c, starts=None, weights_bf16=ratio > 16)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("splits", [2, 3, 4, 5, 16, 64])
def test_splits(gpu, bits, splits):
    print(f"paged splits={splits} bits={bits}", flush=True)
    c = Paged(splits, [0, 7, 300, 1500], [1, 1, 1, 1], 3, 2, 16, bits)
    _check(c, splits)
    c = Paged(splits, [0, 700, 30, 9], [3, 5, 0, 70], 2, 3, 8, bits, front=2, back=3)
    _check(c, splits, weights_bf16=True)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("kv,ratio", [(1, 1), (2, 3), (3, 8), (1, 17)])
@pytest.mark.parametrize("page,held,chunk", [
    (16, [0, 0, 0, 0], [1, 15, 16, 17]), (1, [3, 0, 40], [2, 33, 0]), (64, [64, 100, 0, 513], [64, 0, 129, 1]),
    (8, [1, 130], [200, 65]), (256, [300], [257]), (32, [31, 33, 0], [0, 0, 1])])
def test_chunks(gpu, bits, kv, ratio, page, held, chunk):
    print(f"paged chunk bits={bits} kv={kv} ratio={ratio} page={page} held={held} chunk={chunk}", flush=True)
    c = Paged(kv * 10 + ratio + page, held, chunk, kv, ratio, page, bits, front=1, back=2, pad=16)
    _check(c, weights_bf16=True)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("chunk", [[1, 1, 1], [40, 1, 90]])
def test_absent_pages(gpu, bits, chunk):
    """Entries of -1, of the number of pages and of 2^31 - 1: their positions are neither read nor written."""
    c = Paged(3, [70, 33, 64], chunk, 2, 2, 16, bits, absent=((0, 1), (0, 4), (1, 0), (1, 2), (2, 3), (2, 4)))
    _check(c, weights_bf16=True)
    _check(c, 4, weights_bf16=True)


@pytest.mark.parametrize("chunk", [1, 50])
def test_slots_and_positions_out_of_range(gpu, chunk):
    """Slots out of range and negative positions get zeros and write nothing; positions behind the table's last page are
    attended as given and not kept."""
    c = Paged(5, [20, 30, 40, 16], [chunk] * 4, 2, 1, 16, 16, extra_slots=2)
    c.active[0], c.active[1] = -1, c.table.shape[0]
    c.n[c.active[2].long()] = -1
    c.table = c.table[:, :2].contiguous()
    got = _check(c, weights_bf16=True)
    assert (got[0][:3 * chunk] == 0).all()
    c.n[c.active[3].long()] = 2 ** 31 - 1 - chunk
    _check(c, 2, weights_bf16=True)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("ratio,chunk", [(1, 9), (2, 100), (1, 300)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_later_tokens_never_show(gpu, bits, ratio, chunk, what):
    """NaN and infinities in the keys and values of a token reach its own row and later ones only."""
    c = Paged(8, [21], [chunk], 1, ratio, 16, bits)
    clean = c.run()[0]
    at = chunk * 2 // 3
    c.q[at, c.H * D:] = what
    got = c.run()[0]
    assert torch.equal(got[:at], clean[:at])
    assert not torch.isfinite(got[at:].float()).any()


@pytest.mark.parametrize("bits", [16, 8])
def test_rising_and_extreme_scores(gpu, bits):
    """Scores that rise along the keys by thousands, and rows whose scores are all very low."""
    for chunk in ([1], [80]):
        c = Paged(9, [400], chunk, 1, 2, 16, 16)
        ramp = torch.linspace(-40, 40, 400)
        for t in range(400):
            page, off = c.place(int(c.active[0]), t)
            c.k[page, :, off] = ramp[t].to(BF)
        c.q[:, :c.H * D] = 8.0
        if bits == 8:
            from paged_helpers import held_q8
            k, v = c.k.nan_to_num(), c.v.nan_to_num()
            (c.k, c.ks), (c.v, c.vs), c.bits = held_q8(k), held_q8(v), 8
        _check(c, weights_bf16=True)
        _check(c, 3, weights_bf16=True)
        c.q[:, :c.H * D] = -1000.0
        _check(c, weights_bf16=True)


def test_infinite_scores(gpu):
    """A key whose score is +inf makes its rows NaN, as the formula does; -inf keys weigh nothing."""
    c = Paged(10, [40], [1], 1, 1, 16, 16)
    page, off = c.place(int(c.active[0]), 3)
    c.k[page, 0, off] = 0
    c.k[page, 0, off, 0] = float("inf")
    c.q[0, 0] = -1.0
    want = c.attention64()
    got = c.run()[0]
    close(got, want[0], want[1])
    c.q[0, 0] = 1.0
    assert c.run()[0].isnan().all()


@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_q8_vectors_without_a_scale(gpu, what):
    """A vector with a NaN or an infinity reads back as NaN throughout; the smallest and largest magnitudes do not
    overflow."""
    from kernels.cuda_ext import ext

    c = Paged(11, [0], [4], 1, 1, 16, 8)
    c.q[0, D + 5] = what
    c.q[1, D:] = 2.0 ** -133
    c.q[2, D:] = 3.3e38
    c.q[3, D:] = 0
    out, k, v, ks, vs = c.run()
    kv = torch.empty(4, 2 * D, dtype=BF).cuda()
    s = c.active.repeat(4).cuda()
    ext.dec_gather_paged_q8(s, torch.arange(4, dtype=torch.int32).cuda(), c.table.cuda(), k[None].cuda(), v[None].cuda(),
                            ks[None].cuda(), vs[None].cuda(), kv)
    kv = kv.cpu().float()
    assert kv[0, :D].isnan().all()
    assert (kv[1].abs() <= 2.0 ** -126).all() and torch.isfinite(kv[1:]).all()
    assert ((kv[2] - 3.3e38).abs() <= 3.3e38 / 128).all() and (kv[3] == 0).all()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("layers,kv,page,rows", [(1, 1, 1, 5), (3, 2, 4, 70), (8, 8, 16, 700), (2, 3, 256, 9)])
def test_gather(gpu, bits, layers, kv, page, rows):
    from kernels.cuda_ext import ext

    g = torch.Generator().manual_seed(rows)
    pages, slots, W = 11, 4, 3
    shape = (layers, pages, kv, page, D)
    table = torch.randint(-1, pages + 1, (slots, W), generator=g, dtype=torch.int32)
    slot = torch.randint(-1, slots + 1, (rows,), generator=g, dtype=torch.int32)
    pos = torch.randint(-2, W * page + 2, (rows,), generator=g, dtype=torch.int32)
    if bits == 16:
        k, v = (torch.randn(*shape, generator=g).to(BF) for _ in range(2))
        sc = []
    else:
        k, v = (torch.randint(-127, 128, shape, generator=g, dtype=torch.int8) for _ in range(2))
        sc = [torch.rand(*shape[:-1], generator=g) for _ in range(2)]
    kv_out = torch.full((rows, layers * 2 * kv * D + 8), 7.0, dtype=BF).cuda()
    fn = ext.dec_gather_paged if bits == 16 else ext.dec_gather_paged_q8
    fn(slot.cuda(), pos.cuda(), table.cuda(), k.cuda(), v.cuda(), *(x.cuda() for x in sc), kv_out[:, :-8])
    got = kv_out.cpu()
    assert (got[:, -8:] == 7).all()
    got = got[:, :-8].reshape(rows, layers, 2, kv, D)
    for r in range(rows):
        s, t = int(slot[r]), int(pos[r])
        want = torch.zeros(layers, 2, kv, D)
        if 0 <= s < slots and 0 <= t < W * page and 0 <= int(table[s, t // page]) < pages:
            p = int(table[s, t // page])
            for z, x in enumerate((k, v)):
                y = x[:, p, :, t % page].float()
                want[:, z] = y if bits == 16 else y * sc[z][:, p, :, t % page].unsqueeze(-1)
        assert torch.equal(got[r], want.to(BF)), f"row {r}"


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("chunk", [[1, 1], [70, 3]])
def test_offsets_beyond_32_bits(gpu, bits, chunk):
    """Pages whose offsets pass 2^32 elements."""
    from kernels.cuda_ext import ext

    P, kv, held = 256, 4, [300, 511]
    c = Paged(12, held, chunk, kv, 1, P, bits)
    far = (2 ** 32 + 2 ** 26) // (kv * P * D)  # the pages lie from here on
    big = [torch.empty(far + c.pages, *x.shape[1:], dtype=x.dtype, device="cuda") if x is not None else None
           for x in (c.k, c.v, c.ks, c.vs)]
    for b, x in zip(big, (c.k, c.v, c.ks, c.vs)):
        if x is not None:
            b[far:] = x.cuda()
    table = torch.where(c.table >= 0, c.table + far, c.table)
    out = torch.empty(c.rows, c.H * D, dtype=BF, device="cuda")
    args = (table.cuda(), c.n.cuda(), c.scale, 1, None, out)
    q = c.q.contiguous().cuda()
    if bits == 16:
        ext.dec_attention_paged(c.active.cuda(), c.starts.cuda(), q, *big[:2], *args)
    else:
        ext.dec_attention_paged_q8(c.active.cuda(), c.starts.cuda(), q, *big, *args)
    want, bound, _ = c.attention64(weights_bf16=True)
    close(out.cpu(), want, bound)
    for b, x in zip(big, c.appended()):
        if x is not None:
            assert same_bits(b[far:].cpu(), x)


def test_calls_repeat_captured_and_on_another_stream(gpu):
    """The same bits on another stream, in a captured graph over several replays with eager work between, and when the
    positions move between replays."""
    from kernels.cuda_ext import ext

    c = Paged(13, [100, 40, 0], [1, 1, 1], 4, 2, 16, 8)
    dev = [t.cuda() for t in (c.active, c.q.contiguous(), c.k, c.v, c.ks, c.vs, c.table, c.n)]
    active, q, k, v, ks, vs, table, n = dev
    out = torch.zeros(3, c.H * D, dtype=BF, device="cuda")
    part = torch.empty(3 * c.H * 4 * 130, device="cuda")

    def call():
        ext.dec_attention_paged_q8(active, None, q, k, v, ks, vs, table, n, c.scale, 4, part, out)

    call()
    torch.cuda.synchronize()
    first = out.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out.zero_()
        call()
    s.synchronize()
    assert torch.equal(out, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(4):
        n.copy_(c.n.cuda() - i)
        out.zero_()
        call()
        want = out.clone()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        torch.randn(1000, device="cuda").sum()


def test_long_context(gpu):
    """Hundreds of pages in many parts, few query rows, against one part."""
    c = Paged(14, [9000], [2], 1, 4, 64, 16)
    _check(c, 32)
    _check(c, 1)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("ratio", [2, 17, 40])
def test_splits_without_starts(gpu, bits, ratio):
    """A row a sequence in several parts, of few and of many heads to a key head."""
    c = Paged(ratio, [0, 7, 300, 1500], [1, 1, 1, 1], 1, ratio, 16, bits)
    for splits in (2, 5, 16):
        _check(c, splits, starts=None, weights_bf16=ratio > 16)


@pytest.mark.parametrize("ratio", [2, 8])
@pytest.mark.parametrize("copies", [12, 13, 30])
def test_many_sequences(gpu, ratio, copies):
    """60 to 150 sequences, some without a row, in both kernels."""
    c = Paged(copies, [0, 5, 33, 64, 17] * copies, [3, 0, 20, 1, 7] * copies, 1, ratio, 16, 16, front=2, back=3)
    _check(c, weights_bf16=True)
    _check(c, 3, weights_bf16=True)


@pytest.mark.parametrize("scale", [0.0, -0.07, 1e-30])
def test_scales(gpu, scale):
    """Scales that turn the order of the scores round, or leave nothing of it."""
    for chunk, splits in (([1, 1], 1), ([1, 1], 3), ([90, 20], 1), ([90, 20], 4)):
        c = Paged(15, [300, 0], chunk, 2, 2, 16, 16)
        c.scale = scale
        _check(c, splits, weights_bf16=True)


@pytest.mark.parametrize("bits", [16, 8])
def test_parts_of_a_tiles_own_number(gpu, bits):
    """So many sequences that parts have to be long: some have several, some one, some no row."""
    c = Paged(16, [1700, 0, 90, 800] * 8, [18, 17, 0, 40] * 8, 8, 1, 16, bits)
    for splits in (2, 5):
        _check(c, splits, weights_bf16=True)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("page", [16, 2])
def test_many_chunks_at_once(gpu, bits, page):
    """So many workgroups that each has one group of waves (the tests of few chunks have two)."""
    c = Paged(18, [100, 0, 260] * 20, [17, 20, 0] * 20, 8, 2, page, bits)
    _check(c, weights_bf16=True)


def test_chunks_captured_while_positions_move(gpu):
    """A captured chunk whose sequences have other numbers of parts in every replay, its workspace left as it was."""
    from kernels.cuda_ext import ext

    c = Paged(17, [900, 300, 0], [60, 30, 50], 2, 2, 16, 16)
    starts, active, q, k, v, table, n = (t.cuda() for t in (c.starts, c.active, c.q.contiguous(), c.k.nan_to_num(),
                                                            c.v.nan_to_num(), c.table, c.n))
    out = torch.zeros(c.rows, c.H * D, dtype=BF, device="cuda")
    part = torch.full((c.rows * c.H * 6 * 130,), float("nan"), device="cuda")

    def call(splits=6):
        ext.dec_attention_paged(active, starts, q, k, v, table, n, c.scale, splits, part, out)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    slots = c.active.long()
    for held in ([900, 300, 0], [0, 0, 0], [10, 299, 0], [860, 0, 0], [900, 300, 0]):
        now = c.n.clone()
        now[slots] = torch.tensor(held, dtype=torch.int32)
        n.copy_(now.cuda())
        out.zero_()
        part.fill_(float("nan"))
        call()
        want = out.clone()
        part.fill_(-3.0)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        torch.randn(1000, device="cuda").sum()


def test_two_streams_at_once(gpu):
    """Calls on two streams, each with its own cache and workspace, beside each other."""
    from kernels.cuda_ext import ext

    runs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for i, chunk in enumerate(([1, 1, 1], [33, 80, 7])):
        c = Paged(18 + i, [500, 40, 7], chunk, 4, 2, 16, 16)
        t = [x.cuda() for x in (c.active, c.starts, c.q.contiguous(), c.k, c.v, c.table, c.n)]
        out = torch.zeros(c.rows, c.H * D, dtype=BF, device="cuda")
        part = torch.empty(c.rows * c.H * 4 * 130, device="cuda")
        runs.append((c, t, part, out))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (c, t, part, out) in zip(streams, runs):
            with torch.cuda.stream(s):
                ext.dec_attention_paged(*t, c.scale, 4, part, out)
    torch.cuda.synchronize()
    for c, _, _, out in runs:
        want, bound, _ = c.attention64(weights_bf16=True)
        close(out.cpu(), want, bound)
