"""Decoders that are dropped: freed at once, and without harm to graphs that are captured then."""

from __future__ import annotations

import gc
import weakref

import pytest
import torch

from decoder_helpers import make_decoder
from paged_helpers import BF

pytestmark = pytest.mark.gpu


def _decoder(kind, model, **kw):
    from kernels.beam_decoder import BeamDecoder
    from kernels.stream_decoder import Grammar, StreamDecoder

    a = dict(slots=4, max_new_tokens=8, max_prompt=4, buckets=(1, 2), int8=True, frames=8, penalties=True,
             grammar=Grammar(torch.arange(512) % 2, torch.tensor([[0, 0]])), bias=torch.zeros(1, 512))
    a.update(kw)
    return BeamDecoder(model, beams=2, **a) if kind == "beam" else StreamDecoder(model, **a)


def _model(gpu):
    return make_decoder(hidden=512, heads=4, layers=2, ffn=512, vocab=512, seed=3, device=gpu, dtype=BF)


@pytest.mark.parametrize("kind", ["greedy", "beam"])
@pytest.mark.parametrize("kw", [dict(), dict(capture=False), dict(capture=False, fused=False), dict(kv_bits=16)])
def test_a_dropped_decoder_is_freed_at_once(gpu, kind, kw):
    """Nothing holds a decoder in a cycle: its buffers and graphs end with its last reference, after what is queued."""
    dec = _decoder(kind, _model(gpu), **kw)
    dec.fill_cross(torch.randn(8, dec.width).to(BF).cuda(), [8], [1], projected=True)
    dec.stream.wait_stream(torch.cuda.current_stream())
    dec.admit([1], [torch.tensor([4, 5])], [8])
    dec.step(dec.set_active([1]), 4)
    alive, flags = weakref.ref(dec), weakref.ref(dec.flags)
    was = gc.isenabled()
    gc.disable()
    try:
        del dec
        assert alive() is None and flags() is None
    finally:
        if was:
            gc.enable()
    torch.cuda.synchronize()


@pytest.mark.parametrize("kind", ["greedy", "beam"])
def test_garbage_with_graphs_while_a_decoder_captures(gpu, kind, monkeypatch):
    """Graphs in cycles that nothing else holds come up while a decoder captures its steps, and so many new objects that a
    collection would be due: none runs until the capture has ended."""
    from kernels import stream_decoder

    class Holder:
        pass

    x = torch.zeros(8, device=gpu)
    held = []
    for _ in range(4):
        h = Holder()
        h.graph, h.me = torch.cuda.CUDAGraph(), h
        with stream_decoder._no_collection(), torch.cuda.graph(h.graph):
            x.add_(1)
        held.append(h)
    del h
    inside, due = [], []
    plain = stream_decoder.StreamDecoder._head

    def head(self, bufs, logits):
        def litter():
            if torch.cuda.is_current_stream_capturing():
                inside.append(gc.isenabled())
                if held:
                    due.append(weakref.ref(held.pop()))
                junk = [[i] for i in range(3000)]
                del junk
        return plain(self, bufs, logits) + [litter]

    monkeypatch.setattr(stream_decoder.StreamDecoder, "_head", head)
    threshold = gc.get_threshold()
    gc.collect()
    gc.set_threshold(50, 2, 2)
    try:
        dec = _decoder(kind, _model(gpu))
    finally:
        gc.set_threshold(*threshold)
    assert len(due) == 4 and inside and not any(inside) and gc.isenabled()
    torch.cuda.synchronize()
    gc.collect()
    assert all(r() is None for r in due)
    dec.step(dec.set_active([]), 4)
    torch.cuda.synchronize()
