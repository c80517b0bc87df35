"""StreamDecoder with the cache's bits chosen apart from the weights': bf16 caches under int8 weights, int8 caches under
bf16 weights. The fill, every attention of a step, captured against eager."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import oracle
from helpers import bf16_bits, bf16_float, bf16_ulp
from test_decoder_q4_gpu import _decoder, _start

pytestmark = pytest.mark.gpu
PAIRS = [(True, 16), (False, 8)]


def _close(got_bits, want_bits):
    """The attention kernels' bar over bf16 and int8 caches (their sums are fp32, in another order than the checker's)."""
    got, want = bf16_float(got_bits).astype(np.float64), bf16_float(want_bits).astype(np.float64)
    rms = np.sqrt(np.mean(want ** 2))
    diff = np.abs(got - want)
    assert (diff <= np.maximum(1e-2 * rms, bf16_ulp(want) * 1.0001)).all()
    assert np.sqrt(np.mean(diff ** 2)) <= 2e-3 * rms


@pytest.mark.parametrize("int8,kv_bits", PAIRS)
def test_caches_and_attentions_of_a_step(gpu, int8, kv_bits):
    print(f"kv_bits={kv_bits} int8={int8}", flush=True)
    dec = _decoder(gpu, capture=False, kv_bits=kv_bits, int8=int8)
    assert dec.self_k.dtype == dec.cross_v.dtype == (torch.int8 if kv_bits == 8 else torch.bfloat16)
    assert (dec.cross_ks is None) == (kv_bits == 16)
    slots, b = _start(dec)
    per, seen = 8, 0
    for _ in range(5):
        dec.stream.synchronize()
        with torch.cuda.stream(dec.stream):
            dec._embed(b)
            for i, op in enumerate(dec.programs[b]):
                layer, at = divmod(i, per)
                attend, is_self = layer < len(dec.blocks) and at in (1, 4), at == 1
                if attend:
                    dec.stream.synchronize()
                    caches = [None if t is None else t[layer].cpu() for t in
                              ((dec.self_k, dec.self_v, dec.self_ks, dec.self_vs) if is_self else
                               (dec.cross_k, dec.cross_v, dec.cross_ks, dec.cross_vs))]
                    q, n = (dec.qkv_out if is_self else dec.q_out)[:b].cpu(), (dec.pos if is_self else dec.cross_len).cpu()
                op()
                if not attend:
                    continue
                dec.stream.synchronize()
                rows = slice(0, len(slots))  # the padding row's slot is no one's
                act = dec.active[rows].cpu().numpy()
                if kv_bits == 8:
                    ck, cv, cks, cvs = (t.numpy().copy() for t in caches)
                    kw = dict(k8=ck, v8=cv, ks=cks, vs=cvs)
                else:
                    ck, cv = (bf16_bits(t).copy() for t in caches[:2])
                    kw = dict(k=ck, v=cv)
                want = oracle.dec_attention(is_self, act, bf16_bits(q[rows]), n.numpy(), dec.scale, **kw)
                _close(bf16_bits(dec.att[rows]), want)
                seen += 1
                if is_self:  # what was appended
                    for s in slots:
                        got = [t[layer, s, :, int(n[s])].cpu() for t in (dec.self_k, dec.self_v)]
                        got = [t.numpy() if kv_bits == 8 else bf16_bits(t) for t in got]
                        assert np.array_equal(got[0], ck[s, :, int(n[s])]) and np.array_equal(got[1], cv[s, :, int(n[s])])
    assert seen == 20 and dec.pos[torch.tensor(slots)].tolist() == [5, 5, 5]


@pytest.mark.parametrize("int8,kv_bits", PAIRS)
def test_fill_is_the_scatter_of_the_projections(gpu, int8, kv_bits):
    from kernels.cuda_ext import ext

    print(f"kv_bits={kv_bits} int8={int8}", flush=True)
    dec = _decoder(gpu, capture=False, kv_bits=kv_bits, int8=int8)
    g = torch.Generator().manual_seed(9)
    slots, lengths = [5, 1, 2], [24, 1, 13]
    mem = torch.randn(sum(lengths), dec.width, generator=g).to(torch.bfloat16).to(gpu)
    dec.fill_cross(mem, lengths, slots, projected=True)
    kv = torch.empty(mem.shape[0], dec.cross_w.shape[0], dtype=torch.bfloat16, device=gpu)
    ext.gemm(mem, dec.cross_w, dec.cross_b, kv, 0, None, 1.0, 8)
    where = [torch.tensor(v, dtype=torch.int32, device=gpu) for v in
             ([s for s, n in zip(slots, lengths) for _ in range(n)], [t for n in lengths for t in range(n)])]
    own = [torch.zeros_like(t) for t in (dec.cross_k, dec.cross_v)]
    if kv_bits == 8:
        own += [torch.ones_like(t) for t in (dec.cross_ks, dec.cross_vs)]
        ext.dec_scatter_kv_q8(kv, *where, *own)
    else:
        ext.dec_scatter_kv(kv, *where, *own)
    for got, want in zip((dec.cross_k, dec.cross_v, dec.cross_ks, dec.cross_vs), own):
        assert torch.equal(got, want)


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("int8,kv_bits", PAIRS)
def test_captured_equals_eager(gpu, int8, kv_bits, fused):
    print(f"kv_bits={kv_bits} int8={int8} fused={fused}", flush=True)
    decs = [_decoder(gpu, capture=c, kv_bits=kv_bits, int8=int8, fused=fused) for c in (False, True)]
    for d in decs:
        _, b = _start(d)
        for n in (1, 1, 4, 1, 4):
            d.step(b, n)
        torch.cuda.synchronize()
    for name in ("tok", "pos", "out", "finished", "self_k", "self_v", "self_ks", "self_vs"):
        x, y = (getattr(d, name) for d in decs)
        if x is not None:
            x, y = (x[:, :6], y[:, :6]) if name.startswith("self") else (x[:6], y[:6])  # not the padding rows' slot
            assert torch.equal(x, y), name
