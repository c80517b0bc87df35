"""Plain 64-bit forms of the operators over 4-bit caches and of the rules on logits, and inputs for their tests."""

from __future__ import annotations

import math

import torch

BF = torch.bfloat16


def codes64(x):
    """Codes (..., 128) and maxima (..., 4) of bf16 vectors, from the definition: c = round_half_even(7 x / m)."""
    g = x.double().reshape(*x.shape[:-1], 4, 32)
    m = g.abs().amax(-1)
    c = (7 * g / torch.where(m > 0, m, torch.ones_like(m)).unsqueeze(-1)).round()
    return c.reshape(x.shape), m


def pack(c):
    """Codes (..., 128) as bytes (..., 64): dimension 2j low, 2j + 1 high."""
    n = c.to(torch.int64) % 16
    return (n[..., 0::2] + 16 * n[..., 1::2]).to(torch.uint8)


def value64(codes, maxima):
    n = torch.stack((codes % 16, codes // 16), -1).reshape(*codes.shape[:-1], 128).double()
    c = torch.where(n > 7, n - 16, n)
    return c * (maxima.double() / 7).repeat_interleave(32, -1)


def filled(g, slots, kv, T, std=1.0):
    """Random caches (codes, maxima) on the CPU."""
    c, m = codes64((std * torch.randn(slots, kv, T, 128, generator=g)).to(BF))
    return pack(c), m.to(BF)


def attention64(self_attn, active, q, k4, v4, ks, vs, n, scale, heads):
    """(out, bound): the attention in 64 bits (all on the CPU) and how far a right kernel may be off, elementwise.

    Bound. The kernel holds a query group of 32 in fixed point, its largest magnitude above 16319 steps, so a score is off
    by at most sum_g m_g / 32638 * sum |k| * scale, and by the fp32 roundings of about 16 operations on terms of sum |q k|
    scale (2^-24 each, and 2^-22 for the hardware's exponential with its argument). A weight changed by a factor within
    exp(+-d) changes the output by at most (exp(2 d) - 1) sum p |v|. The weights times the value's maximum m_g are held in
    fixed point too, the largest of 64 keys above 16319 steps: each is off by at most half a step of the largest of all,
    Y / 32638, and by no more than itself (below half a step it becomes 0), which moves the output by that times |c| / 7.
    The sums of n weights and outputs in fp32 add n / 512 + 64 roundings (a lane adds n / 512 products, then they meet) of
    2^-24 of sum p |v|; the result's own rounding is 2^-8 of it. The new token's weight and value are not in fixed
    point."""
    rows, KV = q.shape[0], k4.shape[1]
    S, T = k4.shape[0], k4.shape[2]
    out = torch.zeros(rows, heads, 128, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for r in range(rows):
        s = int(active[r])
        if not 0 <= s < S or int(n[s]) < 0 or (self_attn and int(n[s]) >= T):
            continue
        t = min(int(n[s]), T)
        k, v = value64(k4[s, :, :t], ks[s, :, :t]), value64(v4[s, :, :t], vs[s, :, :t])
        qr = q[r].double()
        if self_attn:
            new = qr[heads * 128:(heads + 2 * KV) * 128].reshape(2, KV, 1, 128)
            k, v = torch.cat((k, new[0]), 1), torch.cat((v, new[1]), 1)
        if k.shape[1] == 0:
            continue
        qh = qr[:heads * 128].reshape(KV, heads // KV, 128)
        sc = torch.matmul(qh, k.transpose(1, 2).contiguous()) * scale  # (KV, ratio, keys)
        p = torch.softmax(sc, -1)
        mg = qh.abs().reshape(*qh.shape[:2], 4, 32).amax(-1).repeat_interleave(32, -1)
        kt = k.abs().transpose(1, 2).contiguous()
        d = (torch.matmul(mg, kt) / 32638 + torch.matmul(qh.abs(), kt) * 16 * 2.0 ** -24 + sc.abs() * 2.0 ** -22) * abs(scale)
        d = d.amax(-1, keepdim=True) + 2.0 ** -22
        spread = torch.matmul(p, v.abs())
        o = torch.matmul(p, v)
        out[r] = o.reshape(heads, 128)
        b = (torch.expm1(2 * d) + (k.shape[1] / 512 + 64) * 2.0 ** -24) * spread
        if t:
            vm = vs[s, :, :t].double()  # (KV, t, 4)
            w = p[..., :t, None] * vm[:, None]  # (KV, ratio, t, 4)
            w = torch.minimum(w.amax(2, keepdim=True) / 32638, w).repeat_interleave(32, -1)
            share = (v[:, :t].abs() / vm.repeat_interleave(32, -1).clamp_min(1e-300))[:, None]  # |c| / 7
            b = b + (w * share).sum(2)
        bound[r] = (b * (1 + 2.0 ** -8) + 2.0 ** -8 * o.abs() + 2.0 ** -134).reshape(heads, 128)
    return out.reshape(rows, -1), bound.reshape(rows, -1)


def logits64(logits, active, pos, tokens=None, first=None, plen=None, pen=None, bias=None, bias_of=None, mask=None,
             classes=None, trans=None, start=None, state=None):
    """(y, slack, state): the rules in 64 bits; slack: what the fp32 roundings of the four operations may add (each
    2^-24 of its result's largest operand). Index values out of range switch rules off."""
    y, state = logits.double(), None if state is None else state.clone()
    slack = torch.zeros_like(y)
    S, V = pos.numel(), logits.shape[1]
    for r in range(logits.shape[0]):
        s = int(active[r])
        if not 0 <= s < S:
            continue
        p, big = int(pos[s]), y[r].abs()
        if pen is not None:
            lo, hi = max(int(first[s]), 0), min(p, tokens.shape[1] - 1)
            for v, c in _counts(tokens[s, lo:hi + 1] if lo <= hi else tokens[s, :0]).items():
                if 0 <= v < V:
                    rep, presence, freq = (float(x) for x in pen[s])
                    l = float(y[r, v])
                    l1 = l / rep if l > 0 else l * rep
                    y[r, v] = l1 - (c * freq + presence)
                    big[v] = max(abs(l), abs(l1), abs(c * freq) + abs(presence), abs(float(y[r, v])))
        if bias is not None and 0 <= int(bias_of[s]) < bias.shape[0]:
            add = bias[int(bias_of[s])].double()
            y[r] += add
            big = torch.maximum(big, torch.maximum(add.abs(), y[r].abs()))
        slack[r] = torch.where(torch.isfinite(big), 4 * 2.0 ** -24 * big, torch.zeros_like(big))
        if mask is None:
            continue
        cur = int(start[s])
        if classes is not None:
            if p >= int(plen[s]):
                cur = int(state[s, (p + 1) % 2])
                t = int(tokens[s, p]) if 0 <= p < tokens.shape[1] else -1
                c = int(classes[t]) if 0 <= t < V else -1
                cur = int(trans[cur, c]) if 0 <= cur < mask.shape[0] and 0 <= c < trans.shape[1] else -1
            state[s, p % 2] = cur
        if 0 <= cur < mask.shape[0]:
            w = mask[cur].long()
            v = torch.arange(V)
            y[r, (w[v // 32] >> (v % 32)) % 2 == 0] = -math.inf
            slack[r, y[r] == -math.inf] = 0
    return y, slack, state


def _counts(t):
    out: dict = {}
    for v in t.tolist():
        out[v] = out.get(v, 0) + 1
    return out


def assert_rounded(got, want, slack):
    """bf16 got is want (64 bits) rounded once, after an error of at most slack: 2^-8 of the value beside it."""
    got, want = got.double().cpu(), want.cpu()
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    tol = slack * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs() + 2.0 ** -134
    bad = ~inf & ~((got - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} beyond tolerance, worst " \
                          f"{float(((got - want).abs() / tol)[bad].max()):.3f}"
