"""Beam search with continuous batching on gfx950 (no counterpart in the reference, whose decoder is greedy): the layers,
weights and cross-attention caches of kernels.stream_decoder.StreamDecoder, with several hypotheses ("beams") a slot.

  prompt     read in one pass (ext.dec_attention_paged over chunks), one row a token, shared by a slot's beams
  step       one token per beam: ext.dec_attention_paged over the beams' pages, the head, the rules, then
             ext.dec_beam_select (the best continuations of all beams), ext.dec_beam_reorder (each takes over its parent's
             history) and ext.dec_beam_advance (tokens, scores, end flags, the next embeddings); one HIP graph per bucket
  caches     the self-attention's in pages: a beam writes each position into a page of its own and reads its history
             through its row of the table, so that taking over a parent's history moves table entries, not keys

Pages hold one position by default: nothing is ever copied then (with longer pages a step copies what the page in part
filled holds, ext.dec_beam_reorder). The hypotheses of a slot are ranked by the sum of their tokens' log probabilities, by
length_penalty divided by (tokens made) ^ length_penalty; ended ones stay among them. One whose rules leave it no token ends
with the end token at no cost, as a row of StreamDecoder does. A slot is done once its best
hypothesis has ended (without length_penalty: no other can pass it), once all have, or at its token limit.

    dec = BeamDecoder(model, beams=4, slots=16, int8=True)
    dec.fill_cross(hidden, lengths, slots); dec.admit(slots, prompts, lengths); b = dec.set_active(slots)
    dec.step(b)                                      # one graph replay
    dec.tokens(slot)                                 # the best hypothesis; dec.score[slot] all scores, best first
"""

from __future__ import annotations

import types

import torch

from kernels.cuda_ext import ext
from kernels.stream_decoder import Grammar, Rules, StreamDecoder


class BeamDecoder(StreamDecoder):
    """StreamDecoder with `beams` hypotheses (1..16) a slot; buckets count slots. length_penalty: 0 ranks by the sum of
    log probabilities, 1 by their mean. page: positions a page (a power of two up to 256). kv_bits: 16 or 8. A request's
    hypotheses do not depend on the others admitted or stepped with it."""

    def __init__(self, model, slots: int = 32, max_new_tokens: int = 448, max_prompt: int = 16, max_audio_s: float = 36.0,
                 buckets=None, int8: bool = False, frames: int | None = None, capture: bool = True,
                 fused: bool | None = None, chunk: int = 4, kv_bits: int | None = None, penalties: bool = False,
                 bias: torch.Tensor | None = None, grammar: Grammar | None = None, *, beams: int = 4,
                 length_penalty: float = 0.0, page: int = 1):
        if not 1 <= beams <= 16:
            raise ValueError(f"BeamDecoder: 1 to 16 beams (got {beams})")
        if page not in (1, 2, 4, 8, 16, 32, 64, 128, 256):
            raise ValueError(f"BeamDecoder: pages of a power of two up to 256 positions (got {page})")
        if not 0.0 <= length_penalty <= 16.0:
            raise ValueError(f"BeamDecoder: a length penalty of 0 to 16 (got {length_penalty})")
        if kv_bits == 4:
            raise ValueError("BeamDecoder: caches of 16 or 8 bits")
        self.beams, self.page, self.length_penalty = beams, page, float(length_penalty)
        super().__init__(model, slots, max_new_tokens, max_prompt, max_audio_s, buckets, int8, frames, capture, fused,
                         chunk, kv_bits, penalties, bias, grammar)

    # ---- state -----------------------------------------------------------------------------------------------------

    def _self_caches(self) -> None:
        """The pages and the beams' state: row r = slot * beams + beam owns pages r * width .., one for each place of its
        table."""
        S1, B, P, dev = self.slots + 1, self.beams, self.page, self.device
        self.width_pages = (self.seq + P - 1) // P
        if S1 * B * self.width_pages >= 2 ** 31:
            raise ValueError("BeamDecoder: too many slots, beams and positions")
        pages = S1 * B * self.width_pages
        self.self_k, self.self_ks = self._cache(pages, P)
        self.self_v, self.self_vs = self._cache(pages, P)
        self.own_pages = torch.arange(pages, device=dev, dtype=torch.int32).reshape(S1 * B, self.width_pages)
        self.table = self.own_pages.clone()
        i32 = dict(device=dev, dtype=torch.int32)
        self.held = torch.ones(S1 * B, **i32)
        self.score = torch.zeros(S1, B, device=dev)
        self.ended = torch.ones(S1, B, device=dev, dtype=torch.uint8)
        self.made = torch.zeros(S1, B, **i32)
        self.norm = None
        if self.length_penalty:
            lengths = torch.arange(self.max_new_tokens + 2, dtype=torch.float64).clamp_min(1)
            self.norm = lengths.pow(-self.length_penalty).float().to(dev)
        bm = self.buckets[-1]
        self.groups = torch.full((bm,), self.dummy, **i32)
        self.slot_of = torch.full((bm * B,), self.dummy, **i32)  # each row's slot: its cross-attention cache
        self.parent = torch.zeros(bm, B, **i32)
        self.token = torch.zeros(bm, B, device=dev, dtype=torch.long)
        self.total = torch.zeros(bm, B, device=dev)
        self.work = torch.empty(ext.dec_beam_select_work(bm * B, self.head.n, B), device=dev, dtype=torch.uint8)

    def _idle_rows(self) -> torch.Tensor:
        return self._rows(self.groups).reshape(-1)

    # ---- the step --------------------------------------------------------------------------------------------------

    def _paged(self, i: int, act, starts, n, qkv, out):
        """Layer i's self-attention over pages (and the append) of rows qkv."""
        k, v, table, scale = self.self_k[i], self.self_v[i], self.table, self.scale
        if self.kv_bits == 8:
            ks, vs = self.self_ks[i], self.self_vs[i]
            return lambda: ext.dec_attention_paged_q8(act, starts, qkv, k, v, ks, vs, table, n, scale, 1, None, out)
        return lambda: ext.dec_attention_paged(act, starts, qkv, k, v, table, n, scale, 1, None, out)

    def _cross(self, i: int, slot_of, q, out):
        return super()._attention(i, False, slot_of, q, 1, out)

    def _program(self, b: int) -> list:
        rows = b * self.beams
        act, groups, slot_of = self.active[:rows], self.groups[:b], self.slot_of[:rows]
        bufs, logits = self._buffers(rows), self.logits[:rows]
        parent, token, total = self.parent[:b], self.token[:b], self.total[:b]
        layers = range(len(self.blocks))
        select = (self.score, self.ended, None if self.norm is None else self.made, self.norm, self.pad, parent, token,
                  total, self.work, self.eos if 0 <= self.eos < self.head.n else -1)
        reorder = (self.held, self.finished, self.table, self.out, self.gstate, self.self_k, self.self_v, self.self_ks,
                   self.self_vs)
        advance = (self.dummy, self.tok, self.pos, self.held, self.score, self.ended, self.made, self.finished, self.limit,
                   self.out, self.eos, self.norm is not None, *self._embedding(), bufs.x, bufs.hn, self.flags)
        return (self._layers(bufs, [self._paged(i, act, None, self.pos, bufs.qkv, bufs.att) for i in layers],
                             [self._cross(i, slot_of, bufs.q, bufs.att) for i in layers])
                + self._head(bufs, logits) + self._rules(act, logits)
                + [lambda: ext.dec_beam_select(logits, groups, *select),
                   lambda: ext.dec_beam_reorder(groups, parent, *reorder),
                   lambda: ext.dec_beam_advance(groups, parent, token, total, *advance)])

    @property
    def _embeds_ahead(self) -> bool:
        return True

    # ---- host side -------------------------------------------------------------------------------------------------

    def _rows(self, slots: torch.Tensor) -> torch.Tensor:
        """The rows of slots (n) as (n, beams)."""
        return slots.unsqueeze(-1) * self.beams + torch.arange(self.beams, device=slots.device, dtype=slots.dtype)

    def reset(self) -> None:
        super().reset()
        with torch.cuda.stream(self.stream):
            self.ended.fill_(1)
            self.held.fill_(1)
            self.table.copy_(self.own_pages)
            self.groups.fill_(self.dummy)
            self.slot_of.fill_(self.dummy)
            self.active.copy_(self._idle_rows())

    def set_active(self, slots: list[int]) -> int:
        b = self.bucket(max(1, len(slots)))
        host = torch.full((b,), self.dummy, dtype=torch.int32)
        host[:len(slots)] = torch.tensor(slots, dtype=torch.int32)
        rows = self._rows(host)
        host = torch.cat((host, rows.reshape(-1), host.unsqueeze(-1).expand_as(rows).reshape(-1)))
        with torch.cuda.stream(self.stream):
            dev = self._to_device(host)
            n = b * self.beams
            self.groups[:b].copy_(dev[:b])
            self.active[:n].copy_(dev[b:b + n])
            self.slot_of[:n].copy_(dev[b + n:])
        self._embed_stale = True
        return b

    @torch.no_grad()
    def admit(self, slots: list[int], prompts: list[torch.Tensor], frames: list[int],
              max_new: list[int] | None = None, rules: list[Rules | None] | None = None) -> None:
        """Start decoding in the given slots (on the decoder stream): their prompts are read in one pass but for the last
        token, which the first step feeds to every beam. `frames` encoder frames are attended to, at most max_new tokens
        made, each under its rules (None: none), which hold for all of a slot's beams."""
        n, B = len(slots), self.beams
        if n == 0:
            return
        rules = [None] * n if rules is None else list(rules)
        if len(rules) != n:
            raise ValueError(f"StreamDecoder: {len(rules)} rules for {n} slots")
        for r in rules:
            self.check_rules(r)
        forced, nums = self._requests(prompts, frames, max_new)
        plen = nums[:, 0].long()
        out_rows = torch.full((n, self.seq + 1), self.pad, dtype=torch.long)
        out_rows[:, :self.max_prompt] = forced
        last = forced.gather(1, plen[:, None] - 1)
        idx_host = torch.tensor(slots, dtype=torch.long)
        with torch.cuda.stream(self.stream):
            idx, out_d, last_d, nums_d = (self._to_device(t) for t in (idx_host, out_rows, last, nums))
            rows = self._rows(idx).reshape(-1)
            pos = (nums_d[:, :1] - 1).expand(n, B)
            self.out.index_copy_(0, rows, out_d.repeat_interleave(B, 0))
            self.tok.index_copy_(0, rows, last_d.expand(n, B).reshape(-1))
            self.pos.index_copy_(0, rows, pos.reshape(-1))
            self.held.index_copy_(0, rows, pos.reshape(-1))  # of the prompt, until its pages are shared out
            self.plen.index_copy_(0, rows, nums_d[:, :1].expand(n, B).reshape(-1))
            self.limit.index_copy_(0, idx, nums_d[:, 1].contiguous())
            self.cross_len.index_copy_(0, idx, nums_d[:, 2].contiguous())
            start = torch.full((n, B), -float("inf"), device=self.device)
            start[:, 0] = 0.0
            self.score.index_copy_(0, idx, start)
            self.ended.index_fill_(0, idx, 0)
            self.made.index_fill_(0, idx, 0)
            self.table.index_copy_(0, rows, self.own_pages.index_select(0, rows))
            self.finished.index_fill_(0, idx, 0)
            if self.rules_on:
                self._admit_rules(rows, [r or Rules() for r in rules for _ in range(B)], plen.repeat_interleave(B))
            self._read_prompts(idx_host, forced, plen)
            # every beam takes over what the first one read
            groups = idx.to(torch.int32)
            ext.dec_beam_reorder(groups, torch.zeros(n, B, device=self.device, dtype=torch.int32), self.held, None,
                                 self.table, None, None, self.self_k, self.self_v, self.self_ks, self.self_vs)
            self.held.index_copy_(0, rows, (pos + 1).reshape(-1))
        self.flags[idx_host] = 0
        self._embed_stale = True

    def _read_prompts(self, slots: torch.Tensor, forced: torch.Tensor, plen: torch.Tensor) -> None:
        """The layers over all prompts' tokens but the last ones, into the pages of each slot's first beam."""
        chunk = plen - 1
        rows = int(chunk.sum())
        if rows == 0:
            return
        at = torch.repeat_interleave(torch.arange(len(slots)), chunk)
        starts = torch.zeros(len(slots) + 1, dtype=torch.int32)
        starts[1:] = chunk.cumsum(0)
        pos = torch.arange(rows) - starts[:-1].long()[at]
        i32 = torch.cat((torch.arange(rows), pos, slots[at], slots * self.beams, starts)).to(torch.int32)
        i32 = self._to_device(i32)
        tok = self._to_device(forced[at, pos])
        every, pos_d, slot_of, first, starts_d = i32.split([rows, rows, rows, len(slots), len(slots) + 1])
        new = lambda n: torch.empty(rows, n, device=self.device, dtype=self.embed.dtype)  # noqa: E731
        w = self.width
        bufs = types.SimpleNamespace(x=new(w), hn=new(w), att=new(w), qkv=new(3 * w), q=new(w), proj=new(w),
                                     ffn=new(self.blocks[0].fc1.n))
        ext.dec_embed(every, tok, pos_d, *self._embedding(), bufs.x, bufs.hn)
        nothing = torch.zeros_like(self.pos)  # nothing is held yet
        layers = range(len(self.blocks))
        ops = self._layers(bufs, [self._paged(i, first, starts_d, nothing, bufs.qkv, bufs.att) for i in layers],
                           [self._cross(i, slot_of, bufs.q, bufs.att) for i in layers])
        per = len(ops) // len(self.blocks)
        for op in ops[:-(per - 2)]:  # behind the last layer's keys and values nothing is read
            op()

    def tokens(self, slot: int) -> torch.Tensor:
        return self.out[slot * self.beams]

    @staticmethod
    def steps_to_limit(prompt: int, max_new: int) -> int:
        return max_new


__all__ = ["BeamDecoder"]
