"""Attention over caches in 4 bits, their filling and reading back, against the definitions in 64 bits. Codes and maxima
are whole: they have to be equal."""

from __future__ import annotations

import pytest
import torch

from q4_helpers import BF, assert_rounded, attention64, codes64, filled, pack, value64

pytestmark = pytest.mark.gpu


def _case(seed, self_attn, rows, KV, ratio, T, lengths, q_std=1.5, poison=True, pad=0):
    """Inputs on the CPU: a slot per row and one more, in another order; keys past a slot's length are poisoned (any
    codes, NaN maxima)."""
    g = torch.Generator().manual_seed(seed)
    S, H = rows + 1, KV * ratio
    k4, ks = filled(g, S, KV, T)
    v4, vs = filled(g, S, KV, T, 0.5)
    active = torch.randperm(S, generator=g)[:rows].to(torch.int32)
    n = torch.zeros(S, dtype=torch.int32)
    n[active.long()] = torch.tensor(lengths, dtype=torch.int32)
    if poison:
        dead = torch.arange(T)[None, :] >= n[:, None]
        for m in (ks, vs):
            m.masked_fill_(dead[:, None, :, None], float("nan"))
    cols = (H + (2 * KV if self_attn else 0)) * 128
    q = (q_std * torch.randn(rows, cols + pad, generator=g)).to(BF)
    return active, q[:, :cols], k4, v4, ks, vs, n, H


def _run(self_attn, active, q, k4, v4, ks, vs, n, H, splits=1, scale=128 ** -0.5):
    from kernels.cuda_ext import ext

    dev = [t.cuda() for t in (active, k4, v4, ks, vs, n)]
    qd = torch.empty(q.shape[0], q.stride(0), dtype=BF).cuda()[:, :q.shape[1]]
    qd.copy_(q)
    out = torch.full((q.shape[0], H * 128), float("nan"), dtype=BF).cuda()
    part = torch.full((q.shape[0] * H * splits * 130,), float("nan")).cuda() if splits > 1 else None
    active_d, k, v, km, vm, nd = dev
    ext.dec_attention_q4(self_attn, active_d, qd, k, v, km, vm, nd, scale, splits, part, out)
    torch.cuda.synchronize()
    return out.cpu(), k.cpu(), v.cpu(), km.cpu(), vm.cpu()


def _close(got, want, bound):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {float((err / bound)[bad].max()):.3f} x bound"


@pytest.mark.parametrize("ratio", [1, 2, 3, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("self_attn", [False, True])
@pytest.mark.parametrize("T,lengths", [(1, [0, 0]), (5, [0, 1, 4]), (129, [127, 128, 63, 64, 65]),
                                       (700, [511, 512, 513, 699, 0, 1])])
def test_attention(gpu, self_attn, ratio, T, lengths):
    print(f"attention_q4 self={self_attn} ratio={ratio} T={T}", flush=True)
    if not self_attn:
        lengths = [x + 1 if x == T - 1 else x for x in lengths]
    a = _case(T + ratio, self_attn, len(lengths), 2, ratio, T, lengths, pad=8)
    want, bound = attention64(self_attn, *a[:7], 128 ** -0.5, a[7])
    out, k4, v4, ks, vs = _run(self_attn, *a)
    _close(out, want, bound)
    _appended(self_attn, a, k4, v4, ks, vs)


def _appended(self_attn, a, k4, v4, ks, vs):
    """The caches hold the new tokens' codes and maxima at n, and elsewhere the bytes that were there."""
    active, q, k0, v0, ks0, vs0, n, H = a
    k0, v0, ks0, vs0 = (t.clone() for t in (k0, v0, ks0, vs0))
    KV, T = k0.shape[1], k0.shape[2]
    if self_attn:
        for r in range(q.shape[0]):
            s = int(active[r])
            if 0 <= s < k0.shape[0] and 0 <= int(n[s]) < T:
                c, m = codes64(q[r, H * 128:].reshape(2, KV, 128))
                k0[s, :, n[s]], v0[s, :, n[s]] = pack(c)
                ks0[s, :, n[s]], vs0[s, :, n[s]] = m.to(BF)
    for got, want in ((k4, k0), (v4, v0), (ks, ks0), (vs, vs0)):
        bits = (lambda t: t.view(torch.int16) if t.dtype == BF else t)
        assert torch.equal(bits(got), bits(want))


@pytest.mark.parametrize("splits", [2, 3, 64])
@pytest.mark.parametrize("self_attn,ratio", [(False, 1), (True, 1), (False, 4), (True, 3), (True, 12)])
def test_attention_split(gpu, self_attn, ratio, splits):
    print(f"attention_q4 split self={self_attn} ratio={ratio} splits={splits}", flush=True)
    lengths = [0, 1, 2, 63, 64, 700, 1299]
    a = _case(splits, self_attn, len(lengths), 1, ratio, 1300, lengths)
    want, bound = attention64(self_attn, *a[:7], 128 ** -0.5, a[7])
    out, k4, v4, ks, vs = _run(self_attn, *a, splits=splits)
    _close(out, want, bound)
    _appended(self_attn, a, k4, v4, ks, vs)
    again = _run(self_attn, *a, splits=splits)[0]
    assert torch.equal(again.view(torch.int16), out.view(torch.int16))


@pytest.mark.parametrize("self_attn", [False, True])
def test_attention_rows_out_of_range(gpu, self_attn):
    """Slots and lengths that no cache has: zeros, nothing written; lengths beyond T read T keys (cross)."""
    print(f"attention_q4 out of range self={self_attn}", flush=True)
    T = 40
    active, q, k4, v4, ks, vs, n, H = _case(5, self_attn, 6, 2, 2, T, [7, 7, 7, 7, 7, 7], poison=False)
    n[active[1].long()], n[active[2].long()], n[active[3].long()] = -1, T, 2 ** 31 - 1
    active[4], active[5] = -1, 7
    a = (active, q, k4, v4, ks, vs, n, H)
    want, bound = attention64(self_attn, *a[:7], 0.1, H)
    out, *caches = _run(self_attn, *a, scale=0.1)
    _close(out, want, bound)
    assert not out[[1, 4, 5]].float().any() and (not self_attn or not out[[2, 3]].float().any())
    _appended(self_attn, a, *caches)


@pytest.mark.parametrize("q_std,scale", [(0.0, 1.0), (1e-30, 1.0), (1e30, 1e-31), (1.0, 0.0), (1.0, -0.3), (20.0, 0.3)])
def test_attention_magnitudes(gpu, q_std, scale):
    """Queries of any magnitude (all zero, tiny, huge), scales of zero and below, one key far above the others."""
    print(f"attention_q4 q_std={q_std} scale={scale}", flush=True)
    a = _case(11, False, 4, 2, 1, 300, [300, 1, 17, 299], q_std=q_std)
    want, bound = attention64(False, *a[:7], scale, a[7])
    out = _run(False, *a, scale=scale)[0]
    _close(out, want, bound)


@pytest.mark.parametrize("ratio", [1, 4])
@pytest.mark.parametrize("slope", [0.002, 0.02, 0.3, -0.02])
def test_attention_scores_that_rise(gpu, slope, ratio):
    """Scores that rise (or fall) key by key, slowly and fast: the softmax base moves seldom, often or at every step."""
    print(f"attention_q4 slope={slope} ratio={ratio}", flush=True)
    T = 900
    active, q, k4, v4, ks, vs, n, H = _case(17, False, 3, 2, ratio, T, [900, 899, 130], poison=False)
    g = torch.Generator().manual_seed(4)
    u = torch.randn(128, generator=g)
    k = 0.3 * torch.randn(4, 2, T, 128, generator=g) + (slope * torch.arange(T))[None, None, :, None] * u / 4
    c, m = codes64(k.to(BF))
    q = (u.repeat(3, H) * 2 + 0.1 * torch.randn(3, H * 128, generator=g)).to(BF)
    a = (active, q, pack(c), v4, m.to(BF), vs, n, H)
    want, bound = attention64(False, *a[:7], 128 ** -0.5, H)
    for splits in (1, 3):
        _close(_run(False, *a, splits=splits)[0], want, bound)


def test_attention_nonfinite_stays_in_its_row(gpu):
    """A NaN or infinity in a row's query, key or value makes that row's heads NaN, and no other's."""
    active, q, k4, v4, ks, vs, n, H = _case(3, True, 5, 2, 1, 64, [10, 20, 30, 40, 50])
    q[0, 3] = float("nan")                      # head 0's query
    q[1, H * 128 + 128 + 5] = float("inf")      # key of head 1, its score +inf
    q[1, 128 + 5] = 1.0
    q[2, (H + 2) * 128 + 7] = float("nan")      # value of head 0
    ks[active[3].long(), 1, 12, 2] = float("nan")  # a cached key of head 1
    out = _run(True, active, q, k4, v4, ks, vs, n, H)[0].reshape(5, 2, 128)
    nan = out.isnan().any(-1)
    assert nan.tolist() == [[True, False], [False, True], [True, False], [False, True], [False, False]]
    held = _run(True, active, q, k4, v4, ks, vs, n, H)[3]
    assert held[active[1].long(), 1, 20].isnan().tolist() == [True, False, False, False]


def test_attention_far_slots(gpu):
    """Caches of more than 2^32 bytes of codes: the last slot's keys."""
    from kernels.cuda_ext import ext

    S, KV, T, n = 5, 4, 1 << 22, 130
    k4, v4 = (torch.zeros(S, KV, T, 64, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(S, KV, T, 4, dtype=BF, device="cuda") for _ in range(2))
    assert k4.numel() > 2 ** 32
    active, q, a, b, am, bm, _, H = _case(9, True, 1, KV, 1, n + 1, [n], poison=False)
    for big, small in ((k4, a), (v4, b), (ks, am), (vs, bm)):
        big[S - 1, :, :n + 1] = small[int(active[0])].cuda()
    last = torch.full((1,), S - 1, dtype=torch.int32)
    out = torch.empty(1, H * 128, dtype=BF, device="cuda")
    nd = torch.full((S,), n, dtype=torch.int32, device="cuda")
    ext.dec_attention_q4(True, last.cuda(), q.cuda(), k4, v4, ks, vs, nd, 128 ** -0.5, 1, None, out)
    want, bound = attention64(True, torch.zeros(1), q, *(t[int(active[0])][None] for t in (a, b, am, bm)),
                              torch.tensor([n]), 128 ** -0.5, H)
    _close(out.cpu(), want, bound)
    got = torch.empty(1, 2 * KV * 128, dtype=BF, device="cuda")
    ext.dec_gather_kv_q4(last.cuda(), nd[:1], k4[None], v4[None], ks[None], vs[None], got)
    c, m = codes64(q[0, H * 128:].reshape(2 * KV, 128))
    assert torch.equal(got.cpu().reshape(2 * KV, 128), (c * (m / 7).repeat_interleave(32, -1)).to(BF))


# ---- filling and reading back -----------------------------------------------------------------------------------------

def _edge_vectors(g, count):
    """Vectors where codes can go wrong: halves of a step (x = m / 2, m / 14 ..), zero groups, powers of two, the smallest
    and the largest bf16 values, one value alone."""
    x = torch.randn(count, 4, 32, generator=g).to(BF)
    m = torch.tensor([1.0, 1.75, 14 / 8, 7 / 4, 3.5, 1e-38, 9.2e-41, 3.3e38, 2.0 ** 64, 2.0 ** -64, 1.9921875, 0.0])
    for i in range(0, count, 2):
        top = m[(i // 2) % len(m)]
        k = torch.randint(-14, 15, (4, 32), generator=g)
        x[i] = (k * (top.double() / 14)).to(BF)  # every code boundary, as far as bf16 holds it
        x[i, :, 0] = top.to(BF)
    x[1] = 0
    x[min(3, count - 1), 2] = 0
    x[min(3, count - 1), 2, 31] = -2.0
    return x.reshape(count, 128)


@pytest.mark.parametrize("L,KV,T,rows", [(1, 1, 1, 1), (2, 3, 50, 7), (8, 8, 33, 61), (3, 2, 376, 375),
                                         (8, 8, 120, 301), (1, 1, 5500, 16411), (1, 3, 3100, 8200)])
def test_scatter_and_gather(gpu, L, KV, T, rows):
    from kernels.cuda_ext import ext
    from kernels.stream_decoder import dequantize_q4, quantize_q4

    print(f"scatter_q4 L={L} KV={KV} T={T} rows={rows}", flush=True)
    g = torch.Generator().manual_seed(rows)
    S = 3
    where = torch.randperm(S * T, generator=g)[:rows]
    slot, frame = (where // T).to(torch.int32), (where % T).to(torch.int32)
    bad = {}
    if rows > 6:
        bad = {0: (-1, 0), 2: (S, 0), 3: (0, T), 5: (1, -1)}
        for i, (s, t) in bad.items():
            slot[i], frame[i] = s, t
    kv = _edge_vectors(g, rows * L * 2 * KV).reshape(rows, -1)
    wide = torch.zeros(rows, kv.shape[1] + 16, dtype=BF)
    wide[:, :kv.shape[1]] = kv
    caches = [torch.full((L, S, KV, T, 64), 0x5a, dtype=torch.uint8) for _ in range(2)] + \
             [torch.full((L, S, KV, T, 4), -3.0, dtype=BF) for _ in range(2)]
    want = [t.clone() for t in caches]
    c, m = codes64(kv.reshape(rows, L, 2, KV, 128))
    good = torch.tensor([i for i in range(rows) if i not in bad])
    at = (slice(None), slot[good].long(), slice(None), frame[good].long())
    for which in range(2):
        want[which][at] = pack(c[good, :, which])  # (rows, L, KV, ..)
        want[2 + which][at] = m[good, :, which].to(BF)
    dev = [t.cuda() for t in caches]
    ext.dec_scatter_kv_q4(wide.cuda()[:, :kv.shape[1]], slot.cuda(), frame.cuda(), *dev)
    for got, w in zip(dev, want):
        assert torch.equal(got.cpu(), w)
    codes, maxima = quantize_q4(kv.reshape(rows, L, 2, KV, 128))
    assert torch.equal(codes, pack(c)) and torch.equal(maxima, m.to(BF))
    back = torch.full((rows, kv.shape[1] + 8), 7.0, dtype=BF, device="cuda")
    ext.dec_gather_kv_q4(slot.cuda(), frame.cuda(), *dev, back[:, :kv.shape[1]])
    value = value64(pack(c), m).reshape(rows, -1)
    value[list(bad)] = 0
    assert torch.equal(back[:, :kv.shape[1]].cpu(), value.to(BF))
    assert torch.equal(back[:, kv.shape[1]:].cpu(), torch.full((rows, 8), 7.0, dtype=BF))
    assert_rounded(dequantize_q4(codes, maxima).to(BF), value64(codes, maxima), torch.zeros_like(c) + 2.0 ** -140)


@pytest.mark.parametrize("exponent", [0, -140, -100, -64, 64, 120])
def test_scatter_every_significand(gpu, exponent):
    """Codes for every pair of a maximum's and a value's significand, values down to 2^-6 of the maximum (every tie of a
    code among them), at magnitudes from the smallest to the largest."""
    from kernels.cuda_ext import ext

    print(f"scatter_q4 significands, 2^{exponent}", flush=True)
    g = torch.Generator().manual_seed(exponent + 200)
    m = torch.arange(128, 256, dtype=torch.float64).repeat_interleave(7 * 5)  # (groups): 5 sets of 31 cover 128 and more
    shift = torch.arange(7).repeat_interleave(5).repeat(128)
    x = (128 + (torch.arange(31)[None, :] + 31 * (torch.arange(len(m)) % 5)[:, None]) % 128).double()
    x = torch.minimum(x * 2.0 ** -shift[:, None], m[:, None]) * (1 - 2 * torch.randint(0, 2, x.shape, generator=g))
    v = torch.cat((m[:, None], x), 1) * 2.0 ** (exponent - 7)
    v = v.to(BF)[:len(m) // 8 * 8].reshape(-1, 2 * 128)
    rows = v.shape[0]
    dev = [torch.zeros(1, 1, 1, rows, w, dtype=t, device="cuda") for w, t in ((64, torch.uint8), (64, torch.uint8), (4, BF),
                                                                             (4, BF))]
    slot, frame = torch.zeros(rows, dtype=torch.int32), torch.arange(rows, dtype=torch.int32)
    ext.dec_scatter_kv_q4(v.cuda(), slot.cuda(), frame.cuda(), *dev)
    c, top = codes64(v.reshape(rows, 2, 128))
    for which in range(2):
        assert torch.equal(dev[which][0, 0, 0].cpu(), pack(c[:, which]))
        assert torch.equal(dev[2 + which][0, 0, 0].cpu(), top[:, which].to(BF))


def test_scatter_nonfinite(gpu):
    from kernels.cuda_ext import ext
    from kernels.stream_decoder import quantize_q4

    kv = torch.randn(1, 2 * 128).to(BF)
    kv[0, 5], kv[0, 40], kv[0, 130] = float("nan"), float("-inf"), float("inf")
    dev = [torch.zeros(1, 1, 1, 1, 64, dtype=torch.uint8, device="cuda") for _ in range(2)] + \
          [torch.zeros(1, 1, 1, 1, 4, dtype=BF, device="cuda") for _ in range(2)]
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    ext.dec_scatter_kv_q4(kv.cuda(), zero, zero, *dev)
    codes, maxima = quantize_q4(kv.reshape(2, 128))
    assert torch.equal(torch.stack((dev[0].cpu().flatten(), dev[1].cpu().flatten())), codes)
    got = torch.stack((dev[2].cpu().flatten(), dev[3].cpu().flatten()))
    assert got.isnan().tolist() == [[True, True, False, False], [True, False, False, False]]
    assert torch.equal(got.nan_to_num(0), maxima.nan_to_num(0))


# ---- together ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("captured", [False, True])
def test_steps_together(gpu, captured):
    """Cross caches filled, then steps that append, attend to themselves and to the audio, on a stream of their own; the
    captured step is replayed with other tokens, and matches the eager one and the definition at every step."""
    from kernels.cuda_ext import ext

    g = torch.Generator().manual_seed(1)
    S, KV, ratio, T, F = 4, 2, 2, 12, 21
    H, rows, scale = KV * ratio, 3, 128 ** -0.5
    frames = [21, 1, 8]
    slots = [2, 0, 3]
    kv = torch.randn(sum(frames), 2 * KV * 128, generator=g).to(BF)
    slot_of = torch.tensor([s for s, f in zip(slots, frames) for _ in range(f)], dtype=torch.int32)
    frame_of = torch.tensor([t for f in frames for t in range(f)], dtype=torch.int32)
    zeros = (lambda t, w, dt: torch.zeros(1, S, KV, t, w, dtype=dt, device="cuda"))
    cross = [zeros(F, 64, torch.uint8), zeros(F, 64, torch.uint8), zeros(F, 4, BF), zeros(F, 4, BF)]
    own = [zeros(T, 64, torch.uint8), zeros(T, 64, torch.uint8), zeros(T, 4, BF), zeros(T, 4, BF)]
    active = torch.tensor(slots, dtype=torch.int32)
    pos = torch.zeros(S, dtype=torch.int32)
    pos[torch.tensor(slots)] = torch.tensor([0, 3, 1], dtype=torch.int32)
    length = torch.zeros(S, dtype=torch.int32)
    length[torch.tensor(slots)] = torch.tensor(frames, dtype=torch.int32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ad, pd, ld = active.cuda(), pos.cuda(), length.cuda()
        ext.dec_scatter_kv_q4(kv.cuda(), slot_of.cuda(), frame_of.cuda(), *cross)
        x = torch.zeros(rows, (H + 2 * KV) * 128, dtype=BF, device="cuda")
        q2 = torch.zeros(rows, H * 128, dtype=BF, device="cuda")
        o1, o2 = torch.zeros_like(q2), torch.zeros_like(q2)
        part = torch.zeros(rows * H * 2 * 130, device="cuda")

        def step():
            ext.dec_attention_q4(True, ad, x, *(t[0] for t in own), pd, scale, 1, None, o1)
            ext.dec_attention_q4(False, ad, q2, *(t[0] for t in cross), ld, scale, 2, part, o2)
            pd.add_(1)

        graph = None
        if captured:
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step()
        mirror = [t[0].cpu() for t in own]
        fixed = [t[0].cpu() for t in cross]
        for i in range(6):
            xs, qs = torch.randn(x.shape, generator=g).to(BF), torch.randn(q2.shape, generator=g).to(BF)
            x.copy_(xs)
            q2.copy_(qs)
            graph.replay() if captured else step()
            side.synchronize()
            n = pos + i
            for o, (is_self, q, c, lens) in ((o1, (True, xs, mirror, n)), (o2, (False, qs, fixed, length))):
                want, bound = attention64(is_self, active, q, *c, lens, scale, H)
                _close(o.cpu(), want, bound)
            for r, s in enumerate(slots):
                c, m = codes64(xs[r, H * 128:].reshape(2, KV, 128))
                mirror[0][s, :, n[s]], mirror[1][s, :, n[s]] = pack(c)
                mirror[2][s, :, n[s]], mirror[3][s, :, n[s]] = m.to(BF)
            for got, want in zip(own, mirror):
                assert torch.equal(got[0].cpu(), want)


def test_one_slot_twice(gpu):
    """Two rows of one slot in a self-attention call: each gets its own result, and of the cache only their position
    changes."""
    active, q, k4, v4, ks, vs, n, H = _case(8, True, 2, 1, 1, 90, [70, 70])
    active[1] = active[0]
    want, bound = attention64(True, active, q, k4, v4, ks, vs, n, 128 ** -0.5, H)
    out, k, *_ = _run(True, active, q, k4, v4, ks, vs, n, H)
    _close(out, want, bound)
    k[int(active[0]), :, 70] = k4[int(active[0]), :, 70]
    assert torch.equal(k, k4)


def test_many_rows(gpu):
    """More rows than a grid's second dimension holds: bit for bit the results of two calls of half the rows."""
    from kernels.cuda_ext import ext

    rows, T = 70001, 3
    g = torch.Generator(device="cuda").manual_seed(2)
    active = torch.randperm(rows, generator=g, device="cuda").to(torch.int32)
    n = (torch.arange(rows, device="cuda") % (T + 1)).to(torch.int32)
    k4, v4 = (torch.randint(0, 256, (rows, 1, T, 64), generator=g, device="cuda").to(torch.uint8) for _ in range(2))
    ks, vs = (torch.rand(rows, 1, T, 4, generator=g, device="cuda").to(BF) for _ in range(2))
    q = torch.randn(rows, 128, generator=g, device="cuda").to(BF)
    out, want = torch.empty_like(q), torch.empty_like(q)
    call = (lambda a, x, o: ext.dec_attention_q4(False, a, x, k4, v4, ks, vs, n, 0.1, 1, None, o))
    call(active, q, out)
    for part in (slice(0, 35000), slice(35000, None)):
        call(active[part], q[part], want[part])
    assert torch.equal(out.view(torch.int16), want.view(torch.int16)) and not out[n[active.long()] == 0].float().any()


def test_refusals_on_the_gpu(gpu):
    """Tensors of another device than the current GPU, no rows, and too short rows."""
    from kernels.cuda_ext import ext

    a = [t.cuda() if torch.is_tensor(t) else t for t in _case(1, False, 2, 1, 1, 4, [1, 2])]
    active, q, k4, v4, ks, vs, n, H = a
    out = torch.empty(2, 128, dtype=BF, device="cuda")
    with pytest.raises(RuntimeError, match="current GPU"):
        ext.dec_attention_q4(False, active, q, k4, v4, ks, vs, n.cpu(), 1.0, 1, None, out)
    with pytest.raises(RuntimeError, match="row stride"):
        ext.dec_attention_q4(False, active, q.new_zeros(2, 129)[:, 1:], k4, v4, ks, vs, n, 1.0, 1, None, out)
    ext.dec_attention_q4(False, active[:0], q[:0], k4, v4, ks, vs, n, 1.0, 1, None, out[:0])
    torch.cuda.synchronize()
