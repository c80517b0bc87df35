"""Beams whose logits hold nothing above -inf (a grammar's state without a successor): they end there, as a greedy row
does, with the end token and the score that they have."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from decoder_helpers import make_decoder
from paged_helpers import BF, select64

pytestmark = pytest.mark.gpu
V, EOS = 512, 3


def _ending(logits, groups, score, finished, eos):
    """The logits with the definition's one candidate of a beam that nothing is left for: the end token, at log 1."""
    x = logits.clone()
    B = score.shape[1]
    for i, g in enumerate(groups.tolist()):
        for b in range(B):
            row = x[i * B + b].float()
            if 0 <= g < score.shape[0] and not finished[g, b] and not (row > -math.inf).any():
                x[i * B + b] = -math.inf
                x[i * B + b, eos] = 0.0
    return x


@pytest.mark.parametrize("B", [1, 2, 4, 16])
@pytest.mark.parametrize("n,Vs", [(7, 64), (7, 4096), (70, 40000)])
@pytest.mark.parametrize("eos", [0, 3, "last"])
def test_select_ends_beams_that_have_nothing(gpu, B, n, Vs, eos):
    """All, one or none of a group's beams without a logit above -inf, NaN beside them, ended and new beams too; ranked by
    total and by length. Totals of -inf and of ended beams are equal, the others as test_beam_gpu.py derives."""
    from kernels.cuda_ext import ext

    eos = Vs - 1 if eos == "last" else eos
    g = torch.Generator().manual_seed(B + Vs)
    G = n + 1
    groups = torch.randperm(G, generator=g)[:n].to(torch.int32)
    x = (3 * torch.randn(n, B, Vs, generator=g)).to(BF)
    score = -30 * torch.rand(G, B, generator=g)
    finished = torch.zeros(G, B, dtype=torch.uint8)
    made = torch.randint(0, 40, (G, B), generator=g, dtype=torch.int32)
    x[0] = -math.inf
    x[1, 0] = -math.inf
    x[2, B // 2:] = -math.inf
    x[3] = float("nan")
    x[4, -1, 1:] = -math.inf  # one token left
    x[5] = -math.inf
    finished[groups[5].long(), ::2] = 1
    x[6, 0] = -math.inf  # a request's first step
    score[groups[6].long(), 0], score[groups[6].long(), 1:] = 0.0, -math.inf
    logits = x.reshape(n * B, Vs)
    norm = torch.arange(33).clamp_min(1).double().pow(-0.7).float()
    for use in (False, True):
        dev = [t.cuda() for t in (logits, groups, score, finished)] + ([made.cuda(), norm.cuda()] if use else [None, None])
        parent, token = torch.full((n, B), -7, dtype=torch.int32).cuda(), torch.full((n, B), -7).cuda()
        total = torch.full((n, B), float("nan")).cuda()
        work = torch.empty(ext.dec_beam_select_work(n * B, Vs, B), dtype=torch.uint8).cuda()
        ext.dec_beam_select(*dev, 2, parent, token, total, work, eos)
        want = select64(_ending(logits, groups, score, finished, eos), groups, score, finished, made if use else None,
                        norm if use else None, 2)
        assert torch.equal(parent.cpu(), want[0]) and torch.equal(token.cpu(), want[1])
        inf = torch.isinf(want[2])
        assert torch.equal(total.cpu()[inf].double(), want[2][inf])
        err = (total.cpu().double() - want[2]).abs()[~inf]
        assert (err <= 2.0 ** -24 * want[2].abs()[~inf] * (1 + 2.0 ** -20) + 2.0 ** -32).all()
        # the score itself, to the bit
        for i in (0, 3):
            first = want[0][i, 0]
            assert token[i, 0] == eos and total[i, 0] == score[groups[i].long(), first]


def _model(gpu):
    model = make_decoder(hidden=512, heads=4, layers=2, ffn=512, vocab=V, seed=21, device=gpu, dtype=BF)
    with torch.no_grad():
        model.proj_out.weight.mul_(4)
    return model


def _memory(width, frames, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(frames, width, generator=g).to(BF).cuda()


PROMPTS = [torch.tensor([7, 8, 9]), torch.tensor([11]), torch.tensor([4, 5, 6, 10])]
FRAMES, SLOTS = [24, 9, 1], [4, 0, 2]


def _texts(dec, rules, steps, max_new=None):
    for i in range(3):
        dec.fill_cross(_memory(dec.width, FRAMES[i], i), [FRAMES[i]], [SLOTS[i]], projected=True)
    dec.stream.wait_stream(torch.cuda.current_stream())
    dec.admit(SLOTS, PROMPTS, FRAMES, max_new, rules)
    b = dec.set_active(SLOTS)
    for _ in range(steps):
        dec.step(b)
    torch.cuda.synchronize()
    return [dec.tokens(s).cpu().tolist() for s in SLOTS]


def _margins():
    """A bias row that makes the choice of every class clear: 32 apart, where roundings move logits by less than 1."""
    bias = torch.full((1, V), -64.0)
    for c in range(3):
        bias[0, 30 + c], bias[0, 60 + c] = 32.0, 0.0
    return bias


@pytest.mark.parametrize("capture", [False, True])
def test_one_beam_and_greedy_end_alike(gpu, capture):
    """Requests that end by a mask that leaves nothing, by the end token and by the limit: the same texts from BeamDecoder
    with one beam and from StreamDecoder."""
    from kernels.beam_decoder import BeamDecoder
    from kernels.stream_decoder import Grammar, Rules, StreamDecoder

    model = _model(gpu)
    classes = torch.arange(V) % 3
    classes[EOS] = 3
    # 0 -> 1 -> 2 -> nothing; 3 -> 4 -> the end token alone; 5 for ever
    trans = torch.tensor([[1, -1, -1, -1], [-1, 2, -1, -1], [-1, -1, -1, -1], [4, -1, -1, -1], [-1, -1, -1, 5],
                          [5, 5, 5, -1]])
    a = dict(slots=6, max_new_tokens=20, max_prompt=4, buckets=(4,), int8=True, frames=24, capture=capture, bias=_margins(),
             grammar=Grammar(classes, trans))
    rules = [Rules(start=0, bias=0), Rules(start=3, bias=0), Rules(start=5, bias=0)]
    texts = []
    for dec, steps in ((StreamDecoder(model, **a), 16), (BeamDecoder(model, beams=1, **a), 16)):
        got = _texts(dec, rules, steps, [9, 9, 5])
        texts.append([t[:len(p) + 9] for t, p in zip(got, PROMPTS)])
        assert dec.finished[SLOTS].all()
    for i, (x, y) in enumerate(zip(*texts)):
        p = len(PROMPTS[i])
        n = p + [3, 2, 5][i]  # two tokens and the end, one and the end, five
        assert x[:n] == y[:n], (i, x, y)
        assert i == 2 or x[n - 1] == EOS
        assert x[:p] == PROMPTS[i].tolist()
    assert texts[0][0][3:5] == [30, 31] and texts[0][1][1] == 30


@pytest.mark.parametrize("beams", [1, 3, 8])
@pytest.mark.parametrize("length_penalty", [0.0, 0.7])
def test_dead_ends_keep_their_rank(gpu, beams, length_penalty):
    """A grammar in which one class leads to a state that allows nothing and another goes on: every launch of the
    selection against the definition; hypotheses that can be follow the grammar, and end with the end token where it
    leaves nothing; a request whose beams all get there is done, with its best hypothesis' text and score."""
    from kernels.beam_decoder import BeamDecoder
    from kernels.stream_decoder import Grammar, Rules

    classes = torch.arange(V) % 3
    trans = torch.tensor([[1, 0, -1], [2, -1, -1], [-1, -1, -1]])  # 0: on (class 1), or to 1; 1 -> 2; 2: nothing
    dec = BeamDecoder(_model(gpu), slots=6, max_new_tokens=20, max_prompt=4, buckets=(4,), int8=True, frames=24,
                      capture=False, beams=beams, length_penalty=length_penalty, grammar=Grammar(classes, trans))
    for i in range(3):
        dec.fill_cross(_memory(dec.width, FRAMES[i], i), [FRAMES[i]], [SLOTS[i]], projected=True)
    dec.stream.wait_stream(torch.cuda.current_stream())
    dec.admit(SLOTS, PROMPTS, FRAMES, [7, 7, 7], [Rules(start=0), Rules(start=1), Rules(start=2)])
    b = dec.set_active(SLOTS)
    norm = None if dec.norm is None else dec.norm.cpu()
    with torch.cuda.stream(dec.stream):
        dec._embed(b)
        for _ in range(7):
            for op in dec.programs[b][:-3]:
                op()
            dec.stream.synchronize()
            groups, logits = dec.groups[:3].cpu(), dec.logits[:3 * beams].cpu()
            small = [t.cpu() for t in (dec.score, dec.ended, dec.made, dec.finished)]
            want = select64(_ending(logits, groups, small[0], small[1], EOS), *(groups, *small[:3]), norm, dec.pad)
            for op in dec.programs[b][-3:]:
                op()
            dec.stream.synchronize()
            live = small[3][groups.long()] == 0
            assert torch.equal(dec.parent[:3].cpu()[live], want[0][live])
            assert torch.equal(dec.token[:3].cpu()[live], want[1][live])
    assert dec.finished[SLOTS].all()
    for i, s in enumerate(SLOTS):
        p, real = len(PROMPTS[i]), 0
        for beam in range(beams):
            if not math.isfinite(float(dec.score[s, beam])):
                continue  # no candidate: the grammar allows fewer texts
            real += 1
            text = dec.out[s * beams + beam, p:p + int(dec.made[s, beam])].tolist()
            state = i
            for at, t in enumerate(text):
                if (trans[state] < 0).all():
                    assert t == EOS and at == len(text) - 1
                    break
                state = int(trans[state, t % 3])
                assert state >= 0, (i, beam, text)
        assert real >= 1 and math.isfinite(float(dec.score[s, 0]))
        if i == 1:
            assert dec.out[s * beams, p + 1] == EOS and dec.out[s * beams, p] % 3 == 0
        if i == 2:  # nothing from the start on: the end token at once, at no cost
            assert dec.out[s * beams, p] == EOS and dec.score[s, 0] == 0 and real == 1


@pytest.mark.parametrize("beams", [1, 3])
def test_pipeline_with_a_grammar_that_ends(gpu, beams):
    """The service's texts under a grammar of two tokens and then nothing: prompt, the two, the end token."""
    import bench
    from kernels.pipeline import Pipeline
    from kernels.stream_decoder import Grammar, Rules

    model = bench.random_asr_model(gpu, enc_layers=1, seed=6)
    vocab = model.proj_out.weight.shape[0]
    grammar = Grammar(torch.arange(vocab) % 2, torch.tensor([[1, -1], [-1, 2], [-1, -1]]))
    pipe = Pipeline(model, None, 4, 12, True, True, buckets=(1, 2, 4), beams=beams, grammar=grammar)
    xs = [Pipeline.prepare(x) for x in bench.synthetic_audio([32000, 17600, 9600], seed=10)]
    prompt = torch.tensor([4, 5, 6, 7])
    want = pipe.transcribe([torch.from_numpy(x).to(gpu) for x in xs], prompt, None, Rules(start=0))
    got = pipe.submit(xs, prompt, None, Rules(start=0)).result(timeout=120)
    pipe.close()
    for a, b in zip(got, want):
        assert np.array_equal(a, b) and np.array_equal(a[:4], prompt.numpy())
        assert len(a) == 7 and a[4] % 2 == 0 and a[5] % 2 == 1 and a[6] == pipe.decoder.eos
