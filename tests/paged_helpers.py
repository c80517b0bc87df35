"""Plain 64-bit forms of the operators over caches in pages and of beam search, and inputs for their tests."""

from __future__ import annotations

import math

import numpy as np
import torch

BF = torch.bfloat16
D = 128


def held_q8(x):
    """Codes (int8) and scales (fp32) of bf16 vectors (..., 128), from the definition: s = max(fp32(m / 127), 2^-126),
    c = round_half_even(fp32(x fp32(1 / s)))."""
    f = x.float().numpy()
    s = np.maximum(np.abs(f).max(-1, keepdims=True) / np.float32(127), np.float32(2.0 ** -126))
    c = np.rint(f * (np.float32(1) / s))
    return torch.from_numpy(c.astype(np.int8)), torch.from_numpy(s[..., 0])


class Paged:
    """A paged cache on the CPU with sequences of given lengths in slots and pages of any order; positions that nothing
    holds are NaN. chunk: new tokens of each sequence; front, back: rows of q and out outside every sequence."""

    def __init__(self, seed, held, chunk, kv, ratio, page, bits, front=0, back=0, pad=0, extra_slots=1, q_std=1.5,
                 v_std=0.5, absent=()):
        g = torch.Generator().manual_seed(seed)
        self.kv, self.ratio, self.P, self.bits = kv, ratio, page, bits
        self.H, self.scale = kv * ratio, D ** -0.5
        seqs, self.chunk = len(held), list(chunk)
        slots = seqs + extra_slots
        self.active = torch.randperm(slots, generator=g)[:seqs].to(torch.int32)
        self.n = torch.full((slots,), -1, dtype=torch.int32)
        self.n[self.active.long()] = torch.tensor(held, dtype=torch.int32)
        need = [(h + c + page - 1) // page for h, c in zip(held, chunk)]
        self.pages = sum(need) + 2
        ids = torch.randperm(self.pages, generator=g).tolist()
        self.table = torch.full((slots, max(max(need), 1) + 1), -1, dtype=torch.int32)
        at = 0
        for s, k in zip(self.active.tolist(), need):
            self.table[s, :k] = torch.tensor(ids[at:at + k], dtype=torch.int32)
            at += k
        shape = (self.pages, kv, page, D)
        mean = 0.7 * torch.randn(kv, 1, D, generator=g)
        x = [(std * (mean + torch.randn(*shape, generator=g))).to(BF) for std in (1.0, v_std)]
        dead = torch.ones(self.pages, page, dtype=torch.bool)
        for s, h in zip(self.active.tolist(), held):
            for t in range(0, h, page):
                dead[self.table[s, t // page], :min(page, h - t)] = False
        dead = dead[:, None, :].expand(self.pages, kv, page)
        self.ks = self.vs = None
        if bits == 16:
            for t in x:
                t[dead] = float("nan")
            self.k, self.v = x
        else:
            (self.k, self.ks), (self.v, self.vs) = held_q8(x[0]), held_q8(x[1])
            self.ks[dead] = float("nan")
            self.vs[dead] = float("nan")
        for s, col in absent:  # pages that a slot lacks
            self.table[int(self.active[s]), col] = [-1, self.pages, 2 ** 31 - 1][(s + col) % 3]
        self.rows = front + sum(chunk) + back
        ends = np.cumsum([front] + list(chunk))
        self.starts = torch.tensor(ends, dtype=torch.int32)
        cols = (self.H + 2 * kv) * D
        q = torch.randn(self.rows, cols + pad, generator=g)
        q[:, :self.H * D] *= q_std
        self.q = q.to(BF)[:, :cols]

    def place(self, slot, t):
        """(page, offset) of a position, or None where there is none."""
        col = t // self.P
        if t < 0 or col >= self.table.shape[1]:
            return None
        page = int(self.table[slot, col])
        return (page, t % self.P) if 0 <= page < self.pages else None

    def held64(self, slot, n):
        """Keys and values (kv, positions that there are, 128) in 64 bits."""
        at = [p for p in (self.place(slot, t) for t in range(n)) if p is not None]
        pages, offs = (torch.tensor([p[i] for p in at], dtype=torch.long) for i in (0, 1))
        out = []
        for x, sc in ((self.k, self.ks), (self.v, self.vs)):
            y = x[pages, :, offs].double()
            out.append((y if sc is None else y * sc[pages, :, offs].double().unsqueeze(-1)).transpose(0, 1))
        return out

    def attention64(self, starts=None, weights_bf16=False):
        """(out, bound, written): the attention in 64 bits, how far a right kernel may be off, and the rows it writes.

        Bound. Products of bf16 numbers (and of int8 codes with them) are exact in fp32; a score's 128 are summed with at
        most one rounding each, 2^-24 of sum |q k|, and scaled with three more; the hardware's exponential is off by 2^-22
        of a weight. Weights changed by factors within exp(+-d) change an output by at most (exp(2 d) - 1) sum p |v|. A
        lane adds one rounding for every four keys, then a few to join; scales of values add one. Weights held in bf16
        (weights_bf16) are off by at most 2^-9 of themselves, and so is their sum if it is made of them. The result's own
        rounding is 2^-8 of it, an error before it included."""
        starts = self.starts if starts is None else starts
        out = torch.zeros(self.rows, self.H, D, dtype=torch.float64)
        bound, written = torch.zeros_like(out), torch.zeros(self.rows, dtype=torch.bool)
        for i, s in enumerate(self.active.tolist()):
            a, b = int(starts[i]), int(starts[i + 1])
            written[a:b] = True
            if not 0 <= s < self.table.shape[0] or int(self.n[s]) < 0 or a == b:
                continue
            n = min(int(self.n[s]), self.table.shape[1] * self.P)
            k, v = self.held64(s, n)
            new = self.q[a:b].double()
            kn, vn = (new[:, (self.H + z * self.kv) * D:(self.H + (z + 1) * self.kv) * D].reshape(b - a, self.kv, D)
                      .transpose(0, 1) for z in (0, 1))
            held = k.shape[1]
            for j in range(b - a):
                kk, vv = torch.cat((k, kn[:, :j + 1]), 1), torch.cat((v, vn[:, :j + 1]), 1)
                qh = new[j, :self.H * D].reshape(self.kv, self.ratio, D)
                kt = kk.transpose(1, 2).contiguous()
                sc = torch.matmul(qh, kt) * self.scale
                p = torch.softmax(sc, -1)
                d = (131 * 2.0 ** -24 * torch.matmul(qh.abs(), kt.abs()) * abs(self.scale)).amax(-1, keepdim=True) + 2.0 ** -21
                o, spread = torch.matmul(p, vv), torch.matmul(p, vv.abs())
                e = (torch.expm1(2 * d) + (held / 4 + 80) * 2.0 ** -24) * spread
                if weights_bf16:
                    e = e + 2 * 2.0 ** -9 * spread
                out[a + j] = o.reshape(self.H, D)
                bound[a + j] = (e * (1 + 2.0 ** -8) + 2.0 ** -8 * o.abs() + 2.0 ** -134).reshape(self.H, D)
        return out.reshape(self.rows, -1), bound.reshape(self.rows, -1), written

    def appended(self, starts=None):
        """(k, v, ks, vs) after the call."""
        starts = self.starts if starts is None else starts
        new = [None if t is None else t.clone() for t in (self.k, self.v, self.ks, self.vs)]
        for i, s in enumerate(self.active.tolist()):
            a, b = int(starts[i]), int(starts[i + 1])
            if not 0 <= s < self.table.shape[0] or int(self.n[s]) < 0:
                continue
            for j in range(b - a):
                at = self.place(s, int(self.n[s]) + j)
                if at is None:
                    continue
                for z in (0, 1):
                    x = self.q[a + j, (self.H + z * self.kv) * D:(self.H + (z + 1) * self.kv) * D].reshape(self.kv, D)
                    if self.bits == 16:
                        new[z][at[0], :, at[1]] = x
                    else:
                        new[z][at[0], :, at[1]], new[2 + z][at[0], :, at[1]] = held_q8(x)
        return new

    def run(self, splits=1, starts="own", out=None, sentinel=7.0):
        """(out, k, v, ks, vs) of the kernel, on the CPU."""
        from kernels.cuda_ext import ext

        dev = lambda t: None if t is None else t.cuda()  # noqa: E731
        q = torch.empty(self.rows, self.q.stride(0), dtype=BF).cuda()[:, :self.q.shape[1]]
        q.copy_(self.q)
        out = torch.full((self.rows, self.H * D), sentinel, dtype=BF).cuda()
        part = torch.full((self.rows * self.H * splits * 130,), float("nan")).cuda() if splits > 1 else None
        starts = self.starts if isinstance(starts, str) else starts
        cache = [dev(t) for t in (self.k, self.v, self.ks, self.vs)]
        args = (dev(self.table), dev(self.n), self.scale, splits, part, out)
        if self.bits == 16:
            ext.dec_attention_paged(dev(self.active), dev(starts), q, *cache[:2], *args)
        else:
            ext.dec_attention_paged_q8(dev(self.active), dev(starts), q, *cache, *args)
        torch.cuda.synchronize()
        return [out.cpu()] + [None if t is None else t.cpu() for t in cache]


def same_bits(a, b):
    """Equal bit by bit (NaN payloads aside)."""
    if a is None:
        return b is None
    if a.dtype.is_floating_point:
        return bool(((a == b) | (a.isnan() & b.isnan())).all())
    return torch.equal(a, b)


def close(got, want, bound):
    err = (got.double() - want).abs()
    bad = ~(err <= bound) & ~(got.isnan() & want.isnan())  # NaN where the definition has NaN
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {float((err / bound)[bad].max()):.3f} x bound"


def select64(logits, groups, score, finished, made, norm, pad, ranks=None):
    """(parent, token, total) by the definition, in 64 bits; logits on the CPU. ranks: a list that gets every group's
    (beams, V) ranks."""
    n, (G, B), V = len(groups), score.shape, logits.shape[1]
    parent, token = torch.zeros(n, B, dtype=torch.int32), torch.zeros(n, B, dtype=torch.int64)
    out = torch.zeros(n, B, dtype=torch.float64)
    for i, g in enumerate(groups.tolist()):
        if not 0 <= g < G:
            parent[i], token[i], out[i] = torch.arange(B), pad, -math.inf
            if ranks is not None:
                ranks.append(None)
            continue
        total = np.full((B, V), -np.inf)
        rank = np.full((B, V), -np.inf)
        for b in range(B):
            if finished[g, b]:
                total[b, pad] = float(score[g, b])
            else:
                l = logits[i * B + b].double()
                l = torch.where(l.isnan(), torch.full_like(l, -math.inf), l).clamp_max(torch.finfo(BF).max)
                m = l.max()
                x = l if m == -math.inf else l - m - torch.log(torch.exp(l - m).sum())
                total[b] = (float(score[g, b]) + x).numpy()
            rank[b] = total[b]
            if norm is not None:
                at = min(max(int(made[g, b]) + (0 if finished[g, b] else 1), 0), len(norm) - 1)
                rank[b] = total[b] * float(norm[at])
        total, rank = np.nan_to_num(total, nan=-np.inf, posinf=np.inf, neginf=-np.inf), \
            np.nan_to_num(rank, nan=-np.inf, posinf=np.inf, neginf=-np.inf)
        if ranks is not None:
            ranks.append(rank)
        best = np.argsort(-rank.reshape(-1), kind="stable")[:B]
        parent[i], token[i] = torch.from_numpy((best // V).astype(np.int32)), torch.from_numpy(best % V)
        out[i] = torch.from_numpy(total.reshape(-1)[best])
    return parent, token, out


def reorder64(groups, parent, n, done, P, table, tokens, states, k, v, ks, vs):
    """The state after the reordering, new tensors (the pages' number limits the table's entries)."""
    B = parent.shape[1]
    old = [None if t is None else t.clone() for t in (table, tokens, states, k, v, ks, vs)]
    new = [None if t is None else t.clone() for t in old]
    for i, g in enumerate(groups.tolist()):
        if not 0 <= g < n.numel() // B or (done is not None and done[g]):
            continue
        length = max(int(n[g * B]), 0)
        for b in range(B):
            a = int(parent[i, b])
            a = a if 0 <= a < B else b
            to, fro = g * B + b, g * B + a
            full = length // P
            if table is not None:
                new[0][to, :full] = old[0][fro, :full]
            if tokens is not None:
                new[1][to, :length] = old[1][fro, :length]
            if states is not None:
                new[2][to] = old[2][fro]
            if k is not None and length % P and full < table.shape[1] and a != b:
                src, dst = int(old[0][fro, full]), int(old[0][to, full])
                if 0 <= src < k.shape[1] and 0 <= dst < k.shape[1]:
                    for z in range(3, 7):
                        if old[z] is not None:
                            new[z][:, dst, :, :length % P] = old[z][:, src, :, :length % P]
    return new
