"""What attention over 4-bit caches keeps of small weights and queries, against the definition in 64 bits and a bound that knows
nothing of how the kernel holds its weights and queries."""

from __future__ import annotations

import pytest
import torch

from q4_helpers import BF, attention64, codes64, pack, value64

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _close(out, active, q, k4, v4, ks, vs, n, H, self_attn=False, scale=SCALE):
    """out against the 64-bit form. A score may be off by what fp32 makes of it: 16 roundings of 2^-24 of sum |q k| scale
    and 2^-22 of itself (the hardware's exponential and its argument); weights off by exp(+-d) move an output by at most
    (exp(2 d) - 1) sum p |v|. The sums of n weights and outputs add n / 256 + 64 roundings of 2^-24 of sum p |v|, a weight
    as the kernel holds it may be off by 2^-10 of itself, the result's rounding is 2^-8 of it. Weights that are below
    2^-117 of the largest may be lost: 2^(s - m) ends at 2^-126, fp32's smallest normal number, and m may lie 8 above the
    largest s. For the same reason sums of values below 2^-118 lose bits at fp32's lower end: outputs are summed in steps
    of 2^-7 times a weight's, so a weight times its value's maximum is held in steps of no less than 2^-142, off by
    2^-143, which the division by the sum of weights, no less than 2^-8 over the largest p, makes 2^-135 times that p: for
    each key."""
    want, _ = attention64(self_attn, active, q, k4, v4, ks, vs, n, scale, H)
    rows, KV = q.shape[0], k4.shape[1]
    bound = torch.zeros(rows, H, 128, dtype=torch.float64)
    for r in range(rows):
        s = int(active[r])
        t = int(n[s])
        k, v = value64(k4[s, :, :t], ks[s, :, :t]), value64(v4[s, :, :t], vs[s, :, :t])
        qr = q[r].double()
        if self_attn:
            new = qr[H * 128:(H + 2 * KV) * 128].reshape(2, KV, 1, 128)
            k, v = torch.cat((k, new[0]), 1), torch.cat((v, new[1]), 1)
        if k.shape[1] == 0:
            continue
        qh = qr[:H * 128].reshape(KV, H // KV, 128)
        kt = k.transpose(1, 2).contiguous()
        sc = torch.matmul(qh, kt) * scale
        d = torch.matmul(qh.abs(), kt.abs()) * scale * 16 * 2.0 ** -24 + sc.abs() * 2.0 ** -22
        d = d.amax(-1, keepdim=True) + 2.0 ** -22
        p = torch.softmax(sc, -1)
        spread = torch.matmul(p, v.abs())
        lost = torch.matmul(torch.where(p < 2.0 ** -117 * p.amax(-1, keepdim=True), p, torch.zeros_like(p)), v.abs())
        bound[r] = ((torch.expm1(2 * d) + (k.shape[1] / 256 + 64) * 2.0 ** -24 + 2.0 ** -10) * spread + lost +
                    2.0 ** -135 * k.shape[1] * p.amax(-1, keepdim=True)).reshape(H, 128)
    bound = bound.reshape(rows, -1) * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs() + 2.0 ** -134
    err = (out.cpu().double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {float((err / bound)[bad].max()):.3f} x bound"


def _run(self_attn, active, q, k4, v4, ks, vs, n, H, splits=1, scale=SCALE):
    from kernels.cuda_ext import ext

    out = torch.full((q.shape[0], H * 128), float("nan"), dtype=BF).cuda()
    part = torch.full((q.shape[0] * H * splits * 130,), float("nan")).cuda() if splits > 1 else None
    dev = [t.cuda() for t in (active, q, k4, v4, ks, vs, n)]
    ext.dec_attention_q4(self_attn, *dev, scale, splits, part, out)
    torch.cuda.synchronize()
    return out.cpu()


def _held(x):
    c, m = codes64(x.to(BF))
    return pack(c), m.to(BF)


@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("ratio", [1, 2, 3, 4])
@pytest.mark.parametrize("gap", [4.0, 11.1, 16.0, 30.0, 60.0])
def test_small_weights_beside_a_large_one(gpu, gap, ratio, splits):
    """One key far above the others, whose value is zero in all but one dimension of each group: elsewhere the others'
    weights, exp(-gap) and less, are all there is."""
    print(f"attention_q4 gap={gap} ratio={ratio} splits={splits}", flush=True)
    T = 200
    g = torch.Generator().manual_seed(int(10 * gap))
    k, v = torch.zeros(3, 2, T, 128), torch.randn(3, 2, T, 128, generator=g)
    k[..., 0] = -1.0 - torch.arange(T) / T / 7
    top = torch.tensor([5, 70, T - 1])  # among the first 64 keys, the next, the last
    for s in range(3):
        k[s, :, top[s]], v[s, :, top[s]] = 0.0, 0.0
        v[s, :, top[s], ::32] = 1.0
    (k4, ks), (v4, vs) = _held(k), _held(v)
    q = torch.zeros(3, 2 * ratio, 128)
    q[..., 0] = gap / SCALE * (1 + torch.arange(2 * ratio) / 64)
    a = (torch.arange(3, dtype=torch.int32), q.reshape(3, -1).to(BF), k4, v4, ks, vs,
         torch.full((3,), T, dtype=torch.int32), 2 * ratio)
    _close(_run(False, *a, splits=splits), *a)


@pytest.mark.parametrize("self_attn", [False, True])
@pytest.mark.parametrize("spread", [3.0, 12.0, 40.0])
def test_scores_far_apart(gpu, spread, self_attn):
    """Scores spread over +-2 spread, values with whole dimensions that only some keys have."""
    print(f"attention_q4 spread={spread} self={self_attn}", flush=True)
    g = torch.Generator().manual_seed(int(spread))
    KV, ratio, T, rows = 2, 3, 700, 3
    k, v = torch.randn(rows, KV, T, 128, generator=g), torch.randn(rows, KV, T, 128, generator=g)
    v *= torch.rand(rows, KV, T, 128, generator=g) < 0.01
    (k4, ks), (v4, vs) = _held(k), _held(v)
    H = KV * ratio
    q = spread * torch.randn(rows, (H + (2 * KV if self_attn else 0)) * 128, generator=g)
    if self_attn:
        q[:, H * 128:] /= spread
    a = (torch.arange(rows, dtype=torch.int32), q.to(BF), k4, v4, ks, vs, torch.tensor([699, 64, 300], dtype=torch.int32), H)
    _close(_run(self_attn, *a), *a, self_attn=self_attn)


@pytest.mark.parametrize("ratio,self_attn,splits", [(1, False, 1), (1, True, 4), (2, False, 1), (3, True, 1), (4, False, 4)])
@pytest.mark.parametrize("factor", [2.0 ** 8, 2.0 ** 9, 2.0 ** 16, 2.0 ** 24, 2.0 ** 50, 2.0 ** 120])
def test_one_large_query_channel(gpu, factor, ratio, self_attn, splits):
    """One channel of a query group far larger than the others, and zero in every key: the scores are the others'."""
    print(f"attention_q4 factor={factor} ratio={ratio} self={self_attn} splits={splits}", flush=True)
    g = torch.Generator().manual_seed(ratio)
    KV, T, rows = 2, 2048, 2
    H = KV * ratio
    k, v = torch.randn(rows, KV, T, 128, generator=g), torch.randn(rows, KV, T, 128, generator=g)
    q = 1.5 * torch.randn(rows, H + (2 * KV if self_attn else 0), 128, generator=g)
    for i, d in enumerate((0, 37, 95, 96)):
        k[..., d] = 0
        q[:, H:H + KV, d] = 0
        q[:, i % H, d] = 1.5 * factor * (-1) ** i
        q[:, H - 1, d] = 1.25 * factor
    (k4, ks), (v4, vs) = _held(k), _held(v)
    a = (torch.arange(rows, dtype=torch.int32), q.reshape(rows, -1).to(BF), k4, v4, ks, vs,
         torch.tensor([T - 1, 1000], dtype=torch.int32), H)
    _close(_run(self_attn, *a, splits=splits), *a, self_attn=self_attn)


@pytest.mark.parametrize("ratio", [1, 2, 4])
@pytest.mark.parametrize("low,high", [(-20, 60), (-133, 127), (-60, 0)])
def test_queries_of_all_magnitudes(gpu, low, high, ratio):
    """Query values of every exponent in one group, keys that are zero where the queries are large."""
    print(f"attention_q4 exponents {low} .. {high} ratio={ratio}", flush=True)
    g = torch.Generator().manual_seed(high - low)
    KV, T, rows = 1, 600, 3
    H = KV * ratio
    q = torch.ldexp(1 + torch.rand(rows, 1, 128, generator=g), torch.randint(low, high, (rows, 1, 128), generator=g))
    q = torch.where(torch.rand(rows, H, 128, generator=g) < 0.5, -q, q)
    q[..., ::4] = torch.randn(rows, H, 32, generator=g)
    k, v = 2 * torch.randn(rows, KV, T, 128, generator=g), torch.randn(rows, KV, T, 128, generator=g)
    k = torch.where((q.abs().amax(1) > 4)[:, None, None, :], torch.zeros_like(k), k)
    (k4, ks), (v4, vs) = _held(k), _held(v)
    a = (torch.arange(rows, dtype=torch.int32), q.reshape(rows, -1).to(BF), k4, v4, ks, vs,
         torch.tensor([T, 1, 257], dtype=torch.int32), H)
    _close(_run(False, *a), *a)


@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("ratio", [1, 3])
@pytest.mark.parametrize("largest,lengths", [(torch.finfo(BF).max, [0, 1]), (2.0 ** 126, [0, 1, 2]), (2.0 ** 118, [700, 600, 3]),
                                             (2.0 ** -100, [5, 0, 700]), (2.0 ** -126, [5, 0, 300])])
@pytest.mark.parametrize("self_attn", [False, True])
def test_values_at_the_ends_of_the_range(gpu, self_attn, largest, lengths, ratio, splits):
    """Values whose sum over the keys fp32 holds, up to the type's largest and down to its smallest: finite, and a lone
    value as it is."""
    print(f"attention_q4 largest={largest} self={self_attn} ratio={ratio} splits={splits}", flush=True)
    if largest == torch.finfo(BF).max and self_attn:
        lengths = [0, 0]
    g = torch.Generator().manual_seed(7)
    KV, T, rows = 2, 701, len(lengths)
    H = KV * ratio
    k, v = torch.randn(rows, KV, T, 128, generator=g), largest * (2 * torch.rand(rows, KV, T, 128, generator=g) - 1)
    v[..., ::32] = largest
    q = torch.randn(rows, H + (2 * KV if self_attn else 0), 128, generator=g)
    if self_attn:
        q[:, H + KV:] = largest * (2 * torch.rand(rows, KV, 128, generator=g) - 1)
        q[:, H + KV:, :4] = largest
    (k4, ks), (v4, vs) = _held(k), _held(v)
    a = (torch.arange(rows, dtype=torch.int32), q.reshape(rows, -1).to(BF), k4, v4, ks, vs,
         torch.tensor(lengths, dtype=torch.int32), H)
    out = _run(self_attn, *a, splits=splits)
    _close(out, *a, self_attn=self_attn)
    for r in range(rows):
        if self_attn and lengths[r] == 0:
            new = a[1][r, (H + KV) * 128:].reshape(KV, 1, 128)
            assert torch.equal(out[r].reshape(KV, ratio, 128), new.expand(KV, ratio, 128))


@pytest.mark.parametrize("ratio,splits", [(1, 1), (1, 3), (2, 1), (4, 2)])
@pytest.mark.parametrize("step", [0.02, 0.05, 0.3])
def test_weights_that_fall_over_many_keys(gpu, step, ratio, splits):
    """Scores that fall by `step` from key to key (and from the last key to the first), values that only every ninth key
    has: outputs made of weights of any size beside larger ones, in every pass over the keys."""
    print(f"attention_q4 step={step} ratio={ratio} splits={splits}", flush=True)
    g = torch.Generator().manual_seed(int(100 * step))
    KV, T, rows = 2, 1500, 2
    H = KV * ratio
    k, v = torch.zeros(rows, KV, T, 128), torch.randn(rows, KV, T, 128, generator=g)
    at = torch.arange(T).float()
    for i in range(4):  # a key's place in its four groups' maxima, which bf16 holds to 8 bits each
        k[..., 32 * i] = (at if i < 2 else at.remainder(7)) / T
    k[1] = k[1].flip(1)
    v = torch.where(torch.arange(T)[:, None] % 9 == torch.arange(128)[None, :] % 9, v, torch.zeros_like(v))
    q = torch.zeros(rows, H, 128)
    q[..., ::32] = -step * T / SCALE / 2 * (1 + torch.arange(H)[:, None] / 100)
    (k4, ks), (v4, vs) = _held(k), _held(v)
    a = (torch.arange(rows, dtype=torch.int32), q.reshape(rows, -1).to(BF), k4, v4, ks, vs,
         torch.tensor([T, T - 1], dtype=torch.int32), H)
    _close(_run(False, *a, splits=splits), *a)


@pytest.mark.parametrize("ratio,self_attn", [(1, False), (1, True), (3, False), (4, True)])
@pytest.mark.parametrize("size", [2.0 ** -119, 2.0 ** -90, 2.0 ** -60, 2.0 ** 60, 2.0 ** 90, 2.0 ** 121])
def test_queries_and_keys_of_opposite_magnitudes(gpu, size, ratio, self_attn):
    """Queries as small (or large) as bf16 has them over keys as large (or small): ordinary scores."""
    print(f"attention_q4 size={size} ratio={ratio} self={self_attn}", flush=True)
    g = torch.Generator().manual_seed(13)
    KV, T, rows = 2, 300, 2
    H = KV * ratio
    k, v = torch.randn(rows, KV, T, 128, generator=g) / size, torch.randn(rows, KV, T, 128, generator=g)
    q = torch.randn(rows, H + (2 * KV if self_attn else 0), 128, generator=g)
    q[:, :H] *= size
    q[:, H:H + KV] /= size
    (k4, ks), (v4, vs) = _held(k), _held(v)
    a = (torch.arange(rows, dtype=torch.int32), q.reshape(rows, -1).to(BF), k4, v4, ks, vs,
         torch.tensor([T - 1, 70], dtype=torch.int32), H)
    _close(_run(self_attn, *a), *a, self_attn=self_attn)
