"""Greedy decoding with continuous batching on gfx950 (the call surface of the reference's kernels/stream_decoder.py):
the int8-weight (W8A16) layout and 64-row chunked projection calls (prepare_w8 38-48, W8_CONFIGS 30-35, _w8 148-158)
over the skinny HIP GEMMs of csrc/dec_w8.hip, and StreamDecoder (73-276): per-slot state and KV caches, one step =
embedding, 8 x (self-attention over the slot's int8 cache, cross-attention, feed-forward), head and greedy pick, held
as a fixed list of launches over preallocated buffers and captured into one HIP graph per bucket of row counts
(csrc/decoder_ops.hip for the non-GEMM kernels).

    wq = prepare_w8(w_bf16)                          # (uint8 (N, K), fp32 (N))
    y = w8_linear(x, wq, bias, relu=False, ws=ws, counters=counters)
    y = bf16_linear(x, w_bf16, bias)                 # o / cross-q / cross-o (the reference's Triton `linear`)
    dec = StreamDecoder(model, slots=64, int8=True)  # model: transformers CohereAsrForConditionalGeneration
    dec.fill_cross(hidden, lengths, slots); dec.admit(slots, prompts, lengths); b = dec.set_active(slots)
    dec.step(b)                                      # one graph replay
"""

from __future__ import annotations

import contextlib
import dataclasses
import gc
import math
import types

import numpy as np
import torch

from kernels.cuda_ext import DEC_EP_NONE, DEC_EP_RELU, DEC_EP_RESID, ext
from kernels.fast_encoder import RCP127

# (N, K) -> {rows up to: (columns per CTA, K splits)}: the reference's A10 table, accepted for compatibility. The gfx950
# kernel checks these like the reference does and then chooses its own tiling (results never depend on it).
W8_CONFIGS = {
    (1024, 4096): {1: (64, 4), 8: (16, 4), 16: (16, 4), 24: (16, 2), 32: (32, 4), 48: (64, 4), 64: (64, 4)},
    (3072, 1024): {1: (32, 1), 8: (32, 1), 16: (32, 1), 24: (32, 1), 32: (32, 1), 48: (64, 1), 64: (64, 1)},
    (4096, 1024): {1: (32, 1), 8: (32, 1), 16: (32, 1), 24: (64, 1), 32: (64, 1), 48: (64, 1), 64: (64, 1)},
    (16384, 1024): {1: (16, 1), 8: (16, 1), 16: (32, 1), 24: (64, 1), 32: (64, 1), 48: (64, 1), 64: (64, 1)},
}
DEFAULT_CONFIG = (64, 4)

# physical byte j of every 16 along K holds logical K W8_PERM[j] (the reference's layout, stream_decoder.py:38)
W8_PERM = (0, 1, 8, 9, 2, 3, 10, 11, 4, 5, 12, 13, 6, 7, 14, 15)


def prepare_w8(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 (N, K) -> (uint8 (N, K) = int8 + 128 with K permuted within every 16 by W8_PERM, fp32 per-channel
    scales). Quantization: s = max(amax|w|, 1e-12) / 127, q = clamp(round_half_even(w / s), +-127), the scale's
    division by 127 as the reference's GPU execution of it: a multiplication by fp32(1 / 127) (RCP127, see
    kernels.fast_encoder.quantize_rows), on any device."""
    n, k = w.shape
    assert k % 16 == 0
    wf = w.float()
    s = wf.abs().amax(1).clamp_min(1e-12) * RCP127
    q = (torch.round(wf / s[:, None]).clamp(-127, 127) + 128).to(torch.uint8)
    perm = torch.tensor(W8_PERM, device=w.device)
    return q.reshape(n, k // 16, 16).index_select(2, perm).reshape(n, k).contiguous(), s.contiguous()


def unprepare_w8(wq: torch.Tensor) -> torch.Tensor:
    """The int8 (N, K) weights in natural K order of a prepare_w8 layout."""
    n, k = wq.shape
    inv = torch.empty(16, dtype=torch.long, device=wq.device)
    inv[torch.tensor(W8_PERM, device=wq.device)] = torch.arange(16, device=wq.device)
    return (wq.reshape(n, k // 16, 16).index_select(2, inv).reshape(n, k).to(torch.int16) - 128).to(torch.int8)


def w8_config(n: int, k: int, rows: int) -> tuple[int, int]:
    configs = W8_CONFIGS.get((n, k))
    if configs is None:
        return DEFAULT_CONFIG if k % (128 * DEFAULT_CONFIG[1]) == 0 and n % 64 == 0 else (16, 1)
    return configs[next(c for c in sorted(configs) if c >= rows)]


def w8_linear(x: torch.Tensor, wq: tuple[torch.Tensor, torch.Tensor], bias: torch.Tensor | None, relu: bool = False,
              ws: torch.Tensor | None = None, counters: torch.Tensor | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """x @ dequant(wq)^T + bias through dec_w8_linear, 64 rows at a time (the reference's StreamDecoder._w8)."""
    (w, scale), (n, k) = wq, wq[0].shape
    y = out if out is not None else torch.empty(x.shape[0], n, device=x.device, dtype=x.dtype)
    for r in range(0, x.shape[0], 64):
        m = min(64, x.shape[0] - r)
        bn, splits = w8_config(n, k, m)
        if ws is None or counters is None:
            splits = 1
        ext.dec_w8_linear(x[r:r + m], w, scale, bias, y[r:r + m], relu, bn, splits, ws, counters)
    return y


def bf16_linear(x: torch.Tensor, w: torch.Tensor, b: torch.Tensor | None, relu: bool = False,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """x @ w^T + b (relu) with bf16 weights, 64 rows at a time (the reference's `linear`, stream_decoder.py:23-27)."""
    y = out if out is not None else torch.empty(x.shape[0], w.shape[0], device=x.device, dtype=x.dtype)
    for r in range(0, x.shape[0], 64):
        m = min(64, x.shape[0] - r)
        ext.linear_bf16(x[r:r + m], w, b, y[r:r + m], relu)
    return y


# ---- caches in 4 bits -------------------------------------------------------------------------------------------------

def quantize_q4(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 vectors (..., 128) in the 4-bit caches' form, as the kernels write it: codes uint8 (..., 64), byte j dimension
    2j in the low nibble and 2j + 1 in the high one (two's complement), and the maxima m bf16 (..., 4) of the four groups
    of 32 values. A code is round_half_even(7 x / m), -7..7 (0 where m = 0). A group with a NaN or an infinity holds the
    maximum NaN and codes 0."""
    g = x.double().reshape(*x.shape[:-1], 4, 32)
    m = g.abs().amax(-1, keepdim=True)
    ok = torch.isfinite(m) & (m > 0)
    c = torch.where(ok, torch.round(7 * g / torch.where(ok, m, torch.ones_like(m))), torch.zeros_like(g))
    n = (c.to(torch.int32) & 15).reshape(*x.shape[:-1], 64, 2)
    held = torch.where(torch.isfinite(m), m, torch.full_like(m, float("nan"))).squeeze(-1).to(torch.bfloat16)
    return (n[..., 0] | (n[..., 1] << 4)).to(torch.uint8), held


def dequantize_q4(codes: torch.Tensor, maxima: torch.Tensor) -> torch.Tensor:
    """The values c m / 7 (fp32, rounded once) of codes (..., 64) and maxima (..., 4)."""
    n = torch.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], 4, 32).to(torch.float64)
    c = torch.where(n > 7, n - 16, n)
    return (c * maxima.double().unsqueeze(-1) / 7).float().reshape(*codes.shape[:-1], 128)


# ---- rules on the choice of tokens ------------------------------------------------------------------------------------

class Grammar:
    """A deterministic automaton over token classes: classes (V) gives each token's class 0..C-1, transitions (M, C) the
    state that a class leads to from each of M states, -1 where it is not allowed. `mask` has a bit per state and token
    that is allowed (int32 (M, ceil(V / 32)), bit v % 32 of word v / 32)."""

    def __init__(self, classes, transitions):
        c, t = torch.as_tensor(classes).cpu().long(), torch.as_tensor(transitions).cpu().long()
        if c.dim() != 1 or t.dim() != 2 or c.numel() == 0 or t.numel() == 0:
            raise ValueError("Grammar: classes (V) and transitions (M, C)")
        if c.min() < 0 or c.max() >= t.shape[1] or t.min() < -1 or t.max() >= t.shape[0]:
            raise ValueError("Grammar: a class outside the transitions' columns, or a state outside their rows")
        self.classes, self.transitions = c.to(torch.int32), t.to(torch.int32)
        allowed = torch.zeros(t.shape[0], (c.numel() + 31) // 32 * 32, dtype=torch.bool)
        allowed[:, :c.numel()] = (t >= 0)[:, c]
        bits = np.packbits(allowed.numpy(), axis=1, bitorder="little")
        self.mask = torch.from_numpy(bits.view("<i4").astype(np.int32))

    @property
    def states(self) -> int:
        return self.transitions.shape[0]


@dataclasses.dataclass(frozen=True)
class Rules:
    """What one request asks of its tokens (StreamDecoder.admit, Pipeline.submit): penalties for tokens that it has made
    already (repetition divides a positive logit and multiplies a negative one, frequency counts, presence does not;
    with `prompt`, the prompt's tokens too), the row of the decoder's bias table, and the grammar's state behind the
    prompt (-1: none)."""

    repetition: float = 1.0
    presence: float = 0.0
    frequency: float = 0.0
    prompt: bool = False
    bias: int = -1
    start: int = -1


# ---- the decoder and its captured step ------------------------------------------------------------------------------

@contextlib.contextmanager
def _no_collection():
    """No garbage collection in the block: the end of another graph, of anything in a cycle, is an error while one is
    captured (it waits for the GPU), which ends the process."""
    was = gc.isenabled()
    gc.disable()
    try:
        yield
    finally:
        if was:
            gc.enable()



class _Projection:
    """One decoder linear bound to its skinny kernel: int8 weights in prepare_w8's layout through dec_w8_linear, or
    bf16 weights through linear_bf16. A call writes y (rows, N) from x (rows, K), 64 rows per launch."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None, int8: bool):
        self.n, self.k = weight.shape
        self.bias = None if bias is None else bias.contiguous()
        if int8:
            self.weight, self.scale = prepare_w8(weight)
        else:
            self.weight, self.scale = weight.contiguous(), None

    @property
    def nbytes(self) -> int:
        return self.weight.numel() * self.weight.element_size()

    def __call__(self, x: torch.Tensor, y: torch.Tensor, relu: bool = False) -> None:
        for r in range(0, x.shape[0], 64):
            xr, yr = x[r:r + 64], y[r:r + 64]
            if self.scale is None:
                ext.linear_bf16(xr, self.weight, self.bias, yr, relu)
            else:
                bn, _ = w8_config(self.n, self.k, xr.shape[0])
                ext.dec_w8_linear(xr, self.weight, self.scale, self.bias, yr, relu, bn, 1, None, None)

    def fused(self, x: torch.Tensor, y: torch.Tensor, epilogue: int = DEC_EP_NONE, ln=None) -> None:
        """The projection with its neighbouring residual LayerNorm folded in (ext.dec_linear_fused): ln normalises
        x's rows first; DEC_EP_RESID adds the result into y (the residual stream) in place."""
        for r in range(0, x.shape[0], 64):
            ext.dec_linear_fused(x[r:r + 64], self.weight, self.scale, self.bias, y[r:r + 64], epilogue, ln)


class _Block:
    """One decoder layer: its three LayerNorms (weight, bias, eps) and six projections. With int8, the
    self-attention's fused q/k/v and the feed-forward's two linears hold int8 weights; the attention outputs and the
    cross-attention query stay bf16 (the reference's int8 layout, stream_decoder.py:106-113)."""

    def __init__(self, layer, int8: bool):
        sa, ca, mlp = layer.self_attn, layer.encoder_attn, layer.mlp
        self.norms = tuple((m.weight, m.bias, float(m.eps)) for m in
                           (layer.input_layernorm, layer.post_attention_layernorm, layer.final_layernorm))
        self.qkv = _Projection(torch.cat([sa.q_proj.weight, sa.k_proj.weight, sa.v_proj.weight]),
                               torch.cat([sa.q_proj.bias, sa.k_proj.bias, sa.v_proj.bias]), int8)
        self.o = _Projection(sa.o_proj.weight, sa.o_proj.bias, False)
        self.cq = _Projection(ca.q_proj.weight, ca.q_proj.bias, False)
        self.co = _Projection(ca.o_proj.weight, ca.o_proj.bias, False)
        self.fc1 = _Projection(mlp.fc1.weight, mlp.fc1.bias, int8)
        self.fc2 = _Projection(mlp.fc2.weight, mlp.fc2.bias, int8)

    def projections(self):
        return (self.qkv, self.o, self.cq, self.co, self.fc1, self.fc2)


class StreamDecoder:
    """Greedy decoding with continuous batching (reference kernels/stream_decoder.py, same constructor, attributes
    and methods). State lives in `slots` slots plus one dummy slot that padding rows point at; a step feeds one token
    per active row. The step is a fixed list of launches over buffers allocated once (no allocation inside a step),
    built per bucket of row counts and captured into one HIP graph per bucket, so a step is one graph replay whatever
    the rows' positions and audio lengths. The model is a transformers CohereAsrForConditionalGeneration (or anything
    with its decoder attributes); `frames` may be given instead of asking the encoder for its subsampled length.

    kv_bits: 16, 8 or 4 bits a cached value (default: 8 with int8, else 16; 4: quantize_q4's form, 72 bytes a vector of
    128 where 8 bits take 132). penalties, bias (B, vocabulary; held in bf16) and grammar (a Grammar) let requests have
    Rules; any of them puts one launch (ext.dec_logits) between the head and the pick of every step."""

    BUCKETS = (1, 2, 4, 8, 16, 24, 32, 48, 64, 80, 96, 112, 128)
    beams = 1  # rows of a slot

    def __init__(self, model, slots: int = 128, max_new_tokens: int = 448, max_prompt: int = 16,
                 max_audio_s: float = 36.0, buckets=None, int8: bool = False, frames: int | None = None,
                 capture: bool = True, fused: bool | None = None, chunk: int = 4, kv_bits: int | None = None,
                 penalties: bool = False, bias: torch.Tensor | None = None, grammar: Grammar | None = None):
        dec, cfg = model.model.decoder, model.config
        self.model, self.int8 = model, int8
        self.kv_bits = kv_bits if kv_bits is not None else (8 if int8 else 16)
        if self.kv_bits not in (4, 8, 16):
            raise ValueError(f"StreamDecoder: caches of 16, 8 or 4 bits (got {kv_bits})")
        self.buckets = tuple(sorted(b for b in (buckets or self.BUCKETS) if b <= slots))
        if not self.buckets:
            raise ValueError("StreamDecoder: no bucket fits the slots")
        self.h, self.width = cfg.num_attention_heads, cfg.hidden_size
        self.d = getattr(cfg, "head_dim", None) or self.width // self.h
        if self.d != 128:
            raise ValueError("StreamDecoder: the decoder kernels take head size 128")
        self.eos, self.pad, self.scale = cfg.eos_token_id, cfg.pad_token_id, self.d ** -0.5
        self.slots, self.dummy = slots, slots
        self.max_new_tokens, self.max_prompt = max_new_tokens, max_prompt
        self.seq = max_prompt + max_new_tokens + 1  # cache positions per slot
        if frames is None:
            frames = int(model.model.encoder._get_subsampling_output_length(
                torch.tensor([int(max_audio_s * 100) + 1])).item())
        self.frames = frames
        # residual LayerNorms folded into the projections (ext.dec_linear_fused) where its prologue takes the width;
        # fused=False keeps the reference's separate dec_add_ln launches (the same bits)
        can_fuse = 512 <= self.width <= 1024 and self.width % 64 == 0
        if fused and not can_fuse:
            raise ValueError(f"StreamDecoder: fused projections take widths 512-1024 (got {self.width})")
        self.fused = can_fuse if fused is None else bool(fused)

        # weights
        self.embed, self.pos_table = dec.embed_tokens.weight, dec.pos_emb.weight
        self.device = dev = self.embed.device
        self.emb_ln = (dec.embedding_layernorm.weight, dec.embedding_layernorm.bias, float(dec.embedding_layernorm.eps))
        self.final_ln = (dec.norm.weight, dec.norm.bias, float(dec.norm.eps))
        self.blocks = [_Block(layer, int8) for layer in dec.layers]
        self.layers = self.blocks
        self.head = _Projection(model.proj_out.weight, model.proj_out.bias, int8)
        self.proj = (dec.proj.weight.contiguous(), None if dec.proj.bias is None else dec.proj.bias.contiguous())
        kv_w = [w for layer in dec.layers for w in (layer.encoder_attn.k_proj.weight, layer.encoder_attn.v_proj.weight)]
        kv_b = [b for layer in dec.layers for b in (layer.encoder_attn.k_proj.bias, layer.encoder_attn.v_proj.bias)]
        self.cross_w, self.cross_b = torch.cat(kv_w).contiguous(), torch.cat(kv_b).contiguous()

        # caches: (layer, slot, head, position, 128), in 8 bits int8 with one fp32 scale per 128-vector, in 4 bits 64
        # bytes of codes with four bf16 maxima
        S1, S1B = slots + 1, (slots + 1) * self.beams
        self._self_caches()
        self.cross_k, self.cross_ks = self._cache(S1, frames)
        self.cross_v, self.cross_vs = self._cache(S1, frames)

        # slot state (row `slots` is the dummy, never advanced); with beams, what each of a slot's beams has of its own
        # is held for slot * beams + beam
        i32, i64 = dict(device=dev, dtype=torch.int32), dict(device=dev, dtype=torch.long)
        self.tok = torch.full((S1B,), self.pad, **i64)
        self.pos = torch.zeros(S1B, **i32)
        self.plen = torch.ones(S1B, **i32)
        self.limit = torch.zeros(S1, **i32)
        self.cross_len = torch.ones(S1, **i32)
        self.finished = torch.ones(S1, device=dev, dtype=torch.uint8)
        self.forced = torch.full((S1, max_prompt), self.pad, **i64)
        self.out = torch.full((S1B, self.seq + 1), self.pad, **i64)
        self.flags = torch.ones(S1, dtype=torch.uint8).pin_memory()  # `finished`, copied out by every step

        # rules on the choice (kernel arguments of ext.dec_logits; None: absent)
        self.grammar, self.rules_on = grammar, penalties or bias is not None or grammar is not None
        if bias is not None and (bias.dim() != 2 or bias.shape[0] == 0 or bias.shape[1] != self.head.n):
            raise ValueError(f"StreamDecoder: a bias table (rows, {self.head.n})")
        if grammar is not None and grammar.classes.numel() != self.head.n:
            raise ValueError(f"StreamDecoder: a grammar over {self.head.n} tokens (got {grammar.classes.numel()})")
        self.bias = None if bias is None else bias.to(device=dev, dtype=torch.bfloat16).contiguous()
        self.bias_of = None if bias is None else torch.full((S1B,), -1, **i32)
        self.first = self.pen = self.mask = self.classes = self.trans = self.start = self.gstate = None
        if penalties:
            self.first = torch.zeros(S1B, **i32)
            self.pen = torch.tensor([1.0, 0.0, 0.0], device=dev).repeat(S1B, 1)
        if grammar is not None:
            self.mask, self.classes, self.trans = (t.to(dev) for t in (grammar.mask, grammar.classes,
                                                                       grammar.transitions))
            self.start, self.gstate = torch.full((S1B,), -1, **i32), torch.full((S1B, 2), -1, **i32)

        # step buffers, sized for the largest bucket
        bm, bf = self.buckets[-1] * self.beams, dict(device=dev, dtype=self.embed.dtype)
        self.active = self._idle_rows()
        self.x, self.hn, self.att = (torch.zeros(bm, self.width, **bf) for _ in range(3))
        self.qkv_out = torch.zeros(bm, 3 * self.width, **bf)
        self.q_out = torch.zeros(bm, self.width, **bf)
        self.proj_out = torch.zeros(bm, self.width, **bf)
        self.ffn_out = torch.zeros(bm, self.blocks[0].fc1.n, **bf)
        self.logits = torch.zeros(bm, self.head.n, **bf)
        self.part = torch.empty(max(b * self.beams * self.h * self._splits(b) * (self.d + 2) for b in self.buckets),
                                device=dev, dtype=torch.float32)

        self.stream = torch.cuda.Stream(device=dev)
        self._embed_stale, self._embed_rows = True, 0
        self.programs = {b: self._program(b) for b in self.buckets}
        self.graphs: dict[int, torch.cuda.CUDAGraph] = {}
        # `chunk` consecutive steps recorded into one graph per bucket as well (step(bucket, chunk)): a graph boundary
        # costs a few microseconds of idle GPU, which one replay per step pays every step
        self.chunk = max(1, int(chunk))
        self.chunk_graphs: dict[int, torch.cuda.CUDAGraph] = {}
        if capture:
            self._capture()

    def __del__(self):
        # what is still queued on the decoder's stream reads and writes buffers that are about to be freed
        with contextlib.suppress(Exception):
            self.stream.synchronize()

    def _cache(self, slots: int, t: int):
        """A cache of every layer and its scales (None in 16 bits): (layer, slot, head, position, ..), or pages."""
        dims, dev = (len(self.blocks), slots, self.h, t), dict(device=self.device)
        if self.kv_bits == 4:
            return (torch.zeros(*dims, self.d // 2, dtype=torch.uint8, **dev),
                    torch.zeros(*dims, 4, dtype=torch.bfloat16, **dev))
        if self.kv_bits == 8:
            return torch.zeros(*dims, self.d, dtype=torch.int8, **dev), torch.ones(*dims, dtype=torch.float32, **dev)
        return torch.zeros(*dims, self.d, dtype=self.embed.dtype, **dev), None

    def _self_caches(self) -> None:
        self.self_k, self.self_ks = self._cache(self.slots + 1, self.seq)
        self.self_v, self.self_vs = self._cache(self.slots + 1, self.seq)

    def _idle_rows(self) -> torch.Tensor:
        """The active rows of the largest bucket where no slot is active."""
        return torch.full((self.buckets[-1],), self.dummy, device=self.device, dtype=torch.int32)

    @staticmethod
    def _splits(b: int) -> int:
        """Workgroups per (row, head) of the cross-attention: one for every bucket. The reference splits the frames
        over 4 for one or two rows (stream_decoder.py:140-144); a split changes the fp32 combine order, so a piece's
        tokens would then depend on how many rows it shares a step with. One split keeps every row's result
        independent of the batch (at 375 frames a workgroup's 64 key groups cover the frames in one pass anyway)."""
        return 1

    # ---- the step as a list of launches ------------------------------------------------------------------------

    def _attention(self, i: int, self_attn: bool, act, q, splits: int, out):
        if self_attn:
            k, v, ks, vs, n = self.self_k[i], self.self_v[i], self.self_ks, self.self_vs, self.pos
        else:
            k, v, ks, vs, n = self.cross_k[i], self.cross_v[i], self.cross_ks, self.cross_vs, self.cross_len
        scale, part = self.scale, self.part
        if self.kv_bits == 4:
            ks, vs = ks[i], vs[i]
            return lambda: ext.dec_attention_q4(self_attn, act, q, k, v, ks, vs, n, scale, splits, part, out)
        if self.kv_bits == 8:
            ks, vs = ks[i], vs[i]
            return lambda: ext.dec_attention_q8(self_attn, act, q, k, v, ks, vs, n, scale, splits, part, out)
        return lambda: ext.dec_attention(self_attn, act, q, k, v, n, scale, splits, part, out)

    def _program(self, b: int) -> list:
        """The step for the first b active rows (reference stream_decoder.py:176-199): embedding + first LayerNorm,
        per layer self-attention (qkv, attention over the slot's cache, o, residual + LayerNorm), cross-attention (q,
        attention over the slot's frames, o, residual + LayerNorm) and feed-forward (fc1 + ReLU, fc2, residual + the
        next LayerNorm), then the head, the greedy pick and the end flags' copy to the host.

        The launches hold tensors and weights, not the decoder: in a cycle with its program it would live on until a
        garbage collection, which may come while a graph is captured, where its own graphs' end is an error that ends
        the process."""
        act, bufs, logits = self.active[:b], self._buffers(b), self.logits[:b]
        state = (self.dummy, self.tok, self.pos, self.finished, self.forced, self.plen, self.limit, self.out, self.pad,
                 self.eos)
        embedding = self._embedding()
        flags, finished = self.flags, self.finished
        self_attn = [self._attention(i, True, act, bufs.qkv, 1, bufs.att) for i in range(len(self.blocks))]
        cross = [self._attention(i, False, act, bufs.q, self._splits(b), bufs.att) for i in range(len(self.blocks))]
        ops = self._layers(bufs, self_attn, cross) + self._head(bufs, logits) + self._rules(act, logits)
        if self.fused:
            # the pick computes the next step's embedding of its row and writes the end flags to the host itself. The
            # same bits as the unfused step. The step's own embedding comes from the previous step's pick, or from
            # step() when the rows changed.
            return ops + [lambda: ext.dec_pick_embed(logits, act, *state, *embedding, bufs.x, bufs.hn, flags)]
        tok, pos = self.tok, self.pos
        return [lambda: ext.dec_embed(act, tok, pos, *embedding, bufs.x, bufs.hn)] + ops + [
            lambda: ext.dec_pick(logits, act, *state),
            lambda: flags.copy_(finished, non_blocking=True)]

    def _embedding(self) -> tuple:
        """The embedding's tables and LayerNorms, and the first layer's."""
        return (self.embed, self.pos_table, *self.emb_ln, *self.blocks[0].norms[0])

    def _buffers(self, rows: int) -> types.SimpleNamespace:
        """The step buffers of the first `rows` rows."""
        return types.SimpleNamespace(x=self.x[:rows], hn=self.hn[:rows], att=self.att[:rows], qkv=self.qkv_out[:rows],
                                     q=self.q_out[:rows], proj=self.proj_out[:rows], ffn=self.ffn_out[:rows])

    def _layers(self, bufs, self_attn: list, cross: list) -> list:
        """The layers' launches on rows whose embedding and first LayerNorm are in x, hn; self_attn and cross are each
        layer's attention launches (qkv -> att, q -> att)."""
        x, hn, att, qkv, q, proj, ffn = (bufs.x, bufs.hn, bufs.att, bufs.qkv, bufs.q, bufs.proj, bufs.ffn)
        ops = []
        if self.fused:
            # the residual adds ride on o / cross-o / fc2's epilogues and the LayerNorms on the next projection's
            # prologue (8 launches a layer instead of 11)
            for i, blk in enumerate(self.blocks):
                ops += [(lambda blk=blk: blk.qkv.fused(hn, qkv)) if i == 0 else
                        (lambda blk=blk: blk.qkv.fused(x, qkv, ln=blk.norms[0])),
                        self_attn[i],
                        lambda blk=blk: blk.o.fused(att, x, DEC_EP_RESID),
                        lambda blk=blk: blk.cq.fused(x, q, ln=blk.norms[1]),
                        cross[i],
                        lambda blk=blk: blk.co.fused(att, x, DEC_EP_RESID),
                        lambda blk=blk: blk.fc1.fused(x, ffn, DEC_EP_RELU, ln=blk.norms[2]),
                        lambda blk=blk: blk.fc2.fused(ffn, x, DEC_EP_RESID)]
            return ops
        for i, blk in enumerate(self.blocks):
            after_ffn = self.blocks[i + 1].norms[0] if i + 1 < len(self.blocks) else self.final_ln
            ops += [lambda blk=blk: blk.qkv(hn, qkv),
                    self_attn[i],
                    lambda blk=blk: blk.o(att, proj),
                    lambda blk=blk: ext.dec_add_ln(x, proj, *blk.norms[1], hn),
                    lambda blk=blk: blk.cq(hn, q),
                    cross[i],
                    lambda blk=blk: blk.co(att, proj),
                    lambda blk=blk: ext.dec_add_ln(x, proj, *blk.norms[2], hn),
                    lambda blk=blk: blk.fc1(hn, ffn, relu=True),
                    lambda blk=blk: blk.fc2(ffn, proj),
                    lambda ln=after_ffn: ext.dec_add_ln(x, proj, *ln, hn)]
        return ops

    def _head(self, bufs, logits) -> list:
        head, ln = self.head, self.final_ln
        if self.fused:
            return [lambda: head.fused(bufs.x, logits, ln=ln)]
        return [lambda: head(bufs.hn, logits)]

    def _rules(self, act, logits) -> list:
        """The requests' rules on the logits, in place (nothing where the decoder was built without any)."""
        if not self.rules_on:
            return []
        rules = (self.pos, self.out, self.first, self.plen, self.pen, self.bias, self.bias_of, self.mask, self.classes,
                 self.trans, self.start, self.gstate)
        return [lambda: ext.dec_logits(logits, logits, act, *rules)]

    def _embed(self, b: int) -> None:
        """The embedding and first LayerNorm of the bucket's active rows (x, hn), on the current stream."""
        rows = b * self.beams
        ext.dec_embed(self.active[:rows], self.tok, self.pos, *self._embedding(), self.x[:rows], self.hn[:rows])

    @property
    def _embeds_ahead(self) -> bool:
        """Whether a step leaves the next step's embeddings (the program then begins behind them)."""
        return self.fused

    def _run(self, b: int) -> None:
        if self._embeds_ahead:
            self._embed(b)
        for op in self.programs[b]:
            op()

    @torch.no_grad()
    def _capture(self) -> None:
        """One graph per bucket, on the decoder stream; each program runs once eagerly first (every launch
        validated), then is recorded. The state is reset afterwards (the runs advanced the dummy rows only). The runs
        read the slots' state and the weights, which the constructor filled on the current stream: the decoder stream
        waits for those fills (behind other queued work they may be far from done, and a token or an active row read
        before its fill is an arbitrary index)."""
        self.stream.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(self.stream):
            for b in reversed(self.buckets):
                self._run(b)
                self.stream.synchronize()
                g = torch.cuda.CUDAGraph()
                with _no_collection(), torch.cuda.graph(g, stream=self.stream):
                    for op in self.programs[b]:  # the program only: step() adds the embedding when the rows change
                        op()
                self.graphs[b] = g
                if self.chunk > 1:
                    g = torch.cuda.CUDAGraph()
                    with _no_collection(), torch.cuda.graph(g, stream=self.stream):
                        for _ in range(self.chunk):
                            for op in self.programs[b]:
                                op()
                    self.chunk_graphs[b] = g
        self.reset()
        self.stream.synchronize()

    # ---- host side -------------------------------------------------------------------------------------------------

    def reset(self) -> None:
        """Every slot free (on the decoder stream)."""
        self._embed_stale = True
        with torch.cuda.stream(self.stream):
            self.finished.fill_(1)
            self.pos.zero_()
            self.cross_len.fill_(1)
            self.active.fill_(self.dummy)

    def bucket(self, rows: int) -> int:
        """The smallest bucket of at least `rows` rows."""
        for b in self.buckets:
            if b >= rows:
                return b
        raise ValueError(f"StreamDecoder: {rows} rows exceed the largest bucket {self.buckets[-1]}")

    def _to_device(self, host: torch.Tensor) -> torch.Tensor:
        return host.pin_memory().to(self.device, non_blocking=True)

    def fill_cross(self, hidden: torch.Tensor, lengths: list[int], slots: list[int], projected: bool = False) -> None:
        """Cross-attention keys and values of packed encoder frames hidden (sum(lengths), width) into the given slots,
        on the current stream: the decoder's input projection (unless projected), every layer's key and value
        projections in one bf16 GEMM whose epilogue writes the slots' caches (quantized per 128-vector in 8 bits, per 32
        values in 4)."""
        from kernels.cuda_ext import EPI_BIAS

        rows = hidden.shape[0]
        if rows == 0:
            return
        mem = hidden.contiguous()
        if not projected:
            out = torch.empty(rows, self.proj[0].shape[0], device=hidden.device, dtype=hidden.dtype)
            ext.gemm(mem, self.proj[0], self.proj[1], out, EPI_BIAS, None, 1.0, 8)
            mem = out
        where = torch.empty(2, rows, device=hidden.device, dtype=torch.int32)
        ext.piece_rows(slots, lengths, where[0], where[1])
        gemm_kv = ext.gemm_kv_q4 if self.kv_bits == 4 else ext.gemm_kv
        gemm_kv(mem, self.cross_w, self.cross_b, where[0], where[1], self.cross_k, self.cross_v, self.cross_ks,
                self.cross_vs)

    def check_rules(self, rules: Rules | None) -> None:
        """Raise ValueError for rules that this decoder was not built for, or whose numbers no slot can have."""
        if rules is None:
            return
        numbers = (rules.repetition, rules.presence, rules.frequency)
        held = torch.tensor(numbers, dtype=torch.float32).tolist()  # what a slot holds of them
        if not all(math.isfinite(x) for x in held) or held[0] <= 0:
            raise ValueError(f"StreamDecoder: penalties {numbers} (finite in fp32, the repetition penalty above 0)")
        if numbers != (1.0, 0.0, 0.0) and self.pen is None:
            raise ValueError("StreamDecoder: penalties need a decoder built with penalties=True")
        if not -1 <= rules.bias < (0 if self.bias is None else self.bias.shape[0]):
            raise ValueError(f"StreamDecoder: bias row {rules.bias} of a table of "
                             f"{0 if self.bias is None else self.bias.shape[0]}")
        if not -1 <= rules.start < (0 if self.grammar is None else self.grammar.states):
            raise ValueError(f"StreamDecoder: state {rules.start} of a grammar of "
                             f"{0 if self.grammar is None else self.grammar.states}")

    def admit(self, slots: list[int], prompts: list[torch.Tensor], frames: list[int],
              max_new: list[int] | None = None, rules: list[Rules | None] | None = None) -> None:
        """Start decoding in the given slots (on the decoder stream): each slot's prompt is forced by the steps
        themselves, `frames` encoder frames attended to, at most max_new (default max_new_tokens) tokens made, each
        under its rules (None: none)."""
        n = len(slots)
        if n == 0:
            return
        rules = [None] * n if rules is None else list(rules)
        if len(rules) != n:
            raise ValueError(f"StreamDecoder: {len(rules)} rules for {n} slots")
        for r in rules:
            self.check_rules(r)
        forced, nums = self._requests(prompts, frames, max_new)
        out_rows = torch.full((n, self.seq + 1), self.pad, dtype=torch.long)
        out_rows[:, :self.max_prompt] = forced
        with torch.cuda.stream(self.stream):
            idx = self._to_device(torch.tensor(slots, dtype=torch.long))
            forced_d, nums_d, out_d = (self._to_device(t) for t in (forced, nums, out_rows))
            self.forced.index_copy_(0, idx, forced_d)
            self.out.index_copy_(0, idx, out_d)
            self.tok.index_copy_(0, idx, forced_d[:, 0].contiguous())
            self.pos.index_fill_(0, idx, 0)
            self.plen.index_copy_(0, idx, nums_d[:, 0].contiguous())
            self.limit.index_copy_(0, idx, nums_d[:, 1].contiguous())
            self.cross_len.index_copy_(0, idx, nums_d[:, 2].contiguous())
            self.finished.index_fill_(0, idx, 0)
            if self.rules_on:
                self._admit_rules(idx, [r or Rules() for r in rules], nums[:, 0])
        self.flags[torch.tensor(slots, dtype=torch.long)] = 0
        self._embed_stale = True

    def _requests(self, prompts, frames, max_new) -> tuple[torch.Tensor, torch.Tensor]:
        """Host tensors of requests: their prompts (n, max_prompt), padded, and (prompt length, position limit, frames)."""
        n = len(prompts)
        forced = torch.full((n, self.max_prompt), self.pad, dtype=torch.long)
        nums = torch.empty(n, 3, dtype=torch.int32)
        for i, p in enumerate(prompts):
            p = torch.as_tensor(p, dtype=torch.long).flatten()
            if not 1 <= len(p) <= self.max_prompt:
                raise ValueError(f"StreamDecoder: a prompt of {len(p)} tokens (1..{self.max_prompt})")
            if not 1 <= frames[i] <= self.frames:
                raise ValueError(f"StreamDecoder: {frames[i]} encoder frames (1..{self.frames})")
            forced[i, :len(p)] = p
            nums[i] = torch.tensor([len(p), len(p) - 1 + (max_new[i] if max_new else self.max_new_tokens),
                                    frames[i]])
        return forced, nums

    def _admit_rules(self, idx: torch.Tensor, rules: list[Rules], plen: torch.Tensor) -> None:
        """The slots' rules (the grammar's states need none: they follow from the start and the tokens)."""
        def put(t, values, dtype):
            if t is not None:
                t.index_copy_(0, idx, self._to_device(torch.tensor(values, dtype=dtype)))

        put(self.pen, [(r.repetition, r.presence, r.frequency) for r in rules], torch.float32)
        put(self.first, [0 if r.prompt else int(p) for r, p in zip(rules, plen)], torch.int32)
        put(self.bias_of, [r.bias for r in rules], torch.int32)
        put(self.start, [r.start for r in rules], torch.int32)

    def set_active(self, slots: list[int]) -> int:
        """The active rows of the next steps (on the decoder stream), padded with the dummy slot; returns the
        bucket to step."""
        b = self.bucket(max(1, len(slots)))
        host = torch.full((b,), self.dummy, dtype=torch.int32)
        host[:len(slots)] = torch.tensor(slots, dtype=torch.int32)
        with torch.cuda.stream(self.stream):
            self.active[:b].copy_(self._to_device(host))
        self._embed_stale = True
        return b

    def step(self, bucket: int, n: int = 1) -> None:
        """`n` decoding steps of the first `bucket` active rows (graph replays on the decoder stream; n == chunk is
        one replay of the chunk graph). With the fused program the rows' embeddings come from the previous step's
        pick; after admit / set_active / reset, or on a different bucket, they are computed first."""
        with torch.cuda.stream(self.stream):
            if bucket in self.graphs:
                if self._embeds_ahead and (self._embed_stale or bucket != self._embed_rows):
                    self._embed(bucket)
                if n > 1 and n == self.chunk and bucket in self.chunk_graphs:
                    self.chunk_graphs[bucket].replay()
                else:
                    for _ in range(n):
                        self.graphs[bucket].replay()
            else:
                for _ in range(n):
                    self._run(bucket)
            self._embed_stale, self._embed_rows = False, bucket

    def tokens(self, slot: int) -> torch.Tensor:
        """The slot's tokens by position, on the GPU."""
        return self.out[slot]

    @staticmethod
    def steps_to_limit(prompt: int, max_new: int) -> int:
        """The steps from admission to the one that ends a slot by its token limit."""
        return prompt - 1 + max_new

    def weight_bytes(self) -> int:
        """Bytes of projection weights one step reads."""
        return sum(p.nbytes for blk in self.blocks for p in blk.projections()) + self.head.nbytes


__all__ = ["DEFAULT_CONFIG", "Grammar", "Rules", "StreamDecoder", "W8_CONFIGS", "W8_PERM", "bf16_linear",
           "dequantize_q4", "prepare_w8", "quantize_q4", "unprepare_w8", "w8_config", "w8_linear"]
