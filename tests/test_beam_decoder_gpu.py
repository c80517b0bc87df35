"""BeamDecoder and Pipeline with beams: every launch of a step against its definition on the step's own inputs, captured
against eager, pages of every length, scores against the hypotheses read token by token, the service against the batch
path."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from decoder_helpers import make_decoder
from paged_helpers import BF, D, Paged, close, reorder64, same_bits, select64

pytestmark = pytest.mark.gpu
PROMPTS = [torch.tensor([7, 8, 9]), torch.tensor([11]), torch.tensor([4, 5, 6, 10])]
FRAMES = [24, 9, 1]
SLOTS = [4, 0, 2]


def _decoder(gpu, seed=21, **kw):
    from kernels.beam_decoder import BeamDecoder

    model = make_decoder(hidden=512, heads=4, layers=2, ffn=512, vocab=512, seed=seed, device=gpu, dtype=BF)
    with torch.no_grad():
        model.proj_out.weight.mul_(4)  # choices that differ
    a = dict(slots=6, max_new_tokens=20, max_prompt=4, buckets=(2, 4), int8=True, frames=24, beams=3)
    a.update(kw)
    return BeamDecoder(model, **a)


def _memory(dec, lengths, seed=5):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(sum(lengths), dec.width, generator=g).to(BF).cuda()


def _start(dec, which=(0, 1, 2), max_new=None, rules=None):
    """The requests `which` in their slots; the bucket to step."""
    for i in which:
        dec.fill_cross(_memory(dec, [FRAMES[i]], seed=i), [FRAMES[i]], [SLOTS[i]], projected=True)
    dec.stream.wait_stream(torch.cuda.current_stream())
    slots = [SLOTS[i] for i in which]
    dec.admit(slots, [PROMPTS[i] for i in which], [FRAMES[i] for i in which], max_new, rules)
    return dec.set_active(slots)


def _cpu(*ts):
    return [None if t is None else t.cpu() for t in ts]


def _paged_of(dec, layer, active, starts, n, qkv):
    """A Paged on what a layer's launch is about to read."""
    c = Paged.__new__(Paged)
    c.kv, c.ratio, c.P, c.bits, c.H, c.scale = dec.h, 1, dec.page, dec.kv_bits, dec.h, dec.scale
    c.active, c.n, c.table, c.q = active.cpu(), n.cpu(), dec.table.cpu(), qkv.cpu()
    c.k, c.v, c.ks, c.vs = _cpu(dec.self_k[layer], dec.self_v[layer], *(
        (dec.self_ks[layer], dec.self_vs[layer]) if dec.kv_bits == 8 else (None, None)))
    c.pages, c.rows = c.k.shape[0], c.q.shape[0]
    c.starts = torch.arange(c.rows + 1, dtype=torch.int32) if starts is None else starts.cpu()
    return c


@pytest.mark.parametrize("kv_bits,page,length_penalty,fused", [(16, 1, 0.0, True), (8, 16, 0.7, True), (8, 1, 0.0, False),
                                                               (16, 4, 1.0, False)])
def test_every_launch_of_a_step(gpu, kv_bits, page, length_penalty, fused):
    print(f"beams kv_bits={kv_bits} page={page} fused={fused}", flush=True)
    dec = _decoder(gpu, capture=False, kv_bits=kv_bits, page=page, length_penalty=length_penalty, fused=fused)
    b = _start(dec)
    B, real = dec.beams, 3 * dec.beams  # rows of no padding group
    per = 8 if fused else 11
    dec.stream.synchronize()
    ops = dec.programs[b]
    assert len(ops) == per * 2 + 1 + 3
    for step in range(8):
        with torch.cuda.stream(dec.stream):
            if step == 0:
                dec._embed(b)
            for i, op in enumerate(ops):
                layer, at = divmod(i, per)
                dec.stream.synchronize()
                if layer < 2 and at == 1:
                    c = _paged_of(dec, layer, dec.active[:real], None, dec.pos, dec.qkv_out[:real])
                    want, bound, _ = c.attention64()
                    kept = c.appended()
                if i >= len(ops) - 3:
                    groups = dec.groups[:3].cpu()
                    state = _cpu(dec.table, dec.out, None, dec.self_k, dec.self_v, dec.self_ks, dec.self_vs)
                    small = _cpu(dec.score, dec.ended, dec.made, dec.finished, dec.pos, dec.held)
                op()
                dec.stream.synchronize()
                if layer < 2 and at == 1:
                    close(dec.att[:real].cpu(), want, bound)
                    dummy = dec.own_pages[dec.dummy * B:].reshape(-1).cpu().long()  # of the padding rows
                    mine = torch.ones(c.pages, dtype=torch.bool)
                    mine[dummy] = False
                    for got, w in zip(_cpu(dec.self_k, dec.self_v, dec.self_ks, dec.self_vs), kept):
                        assert w is None or same_bits(got[layer][mine], w[mine])
                elif i == len(ops) - 3:
                    norm = None if dec.norm is None else dec.norm.cpu()
                    want = select64(dec.logits[:real].cpu(), groups, small[0], small[1], small[2], norm, dec.pad)
                    live = small[3][groups.long()] == 0
                    assert torch.equal(dec.parent[:3].cpu()[live], want[0][live])
                    assert torch.equal(dec.token[:3].cpu()[live], want[1][live])
                    assert ((dec.total[:3].cpu() - want[2]).abs()[live] <= 2.0 ** -23 * want[2].abs()[live]).all()
                elif i == len(ops) - 2:
                    assert torch.equal(small[5][:-B][small[3][:-1].repeat_interleave(B) == 0],
                                       (small[4] + 1)[:-B][small[3][:-1].repeat_interleave(B) == 0])
                    want = reorder64(groups, dec.parent[:3].cpu(), small[5], small[3], page, *state)
                    for got, w in zip(_cpu(dec.table, dec.out, None, dec.self_k, dec.self_v, dec.self_ks, dec.self_vs),
                                      want):
                        assert same_bits(got, w)
    assert dec.pos.reshape(-1, B)[SLOTS].tolist() == [[len(p) - 1 + 8] * B for p in PROMPTS]


@pytest.mark.parametrize("kv_bits", [16, 8])
def test_prompts_in_one_pass(gpu, kv_bits):
    """The first beam's pages hold every prompt token's key and value but the last one's, whatever is read beside it, and
    the other beams' tables lead to the same."""
    from kernels.cuda_ext import ext

    held = []
    for which in ((0, 1, 2), (0,), (2,)):
        dec = _decoder(gpu, capture=False, kv_bits=kv_bits, page=2)
        _start(dec, which)
        dec.stream.synchronize()
        for i in which:
            n = len(PROMPTS[i]) - 1
            for beam in range(dec.beams):
                kv = torch.empty(n, 2 * 2 * dec.h * D, dtype=BF, device=gpu)
                slot = torch.full((n,), SLOTS[i] * dec.beams + beam, dtype=torch.int32, device=gpu)
                at = torch.arange(n, dtype=torch.int32, device=gpu)
                if kv_bits == 16:
                    ext.dec_gather_paged(slot, at, dec.table, dec.self_k, dec.self_v, kv)
                else:
                    ext.dec_gather_paged_q8(slot, at, dec.table, dec.self_k, dec.self_v, dec.self_ks, dec.self_vs, kv)
                held.append((i, kv.cpu()))
    for i in range(3):
        same = [kv for j, kv in held if j == i]
        assert len(same) >= 3 and all(torch.equal(kv, same[0]) for kv in same)
        assert i == 1 or (same[0].float().abs().amax(1) > 0).all()


@pytest.mark.parametrize("kv_bits,length_penalty", [(16, 0.0), (8, 0.6)])
def test_captured_equals_eager_and_pages_of_any_length(gpu, kv_bits, length_penalty):
    """Tokens and scores are the same bits captured or not, stepped one by one or in chunks, and for pages of 1, 4 and 64
    positions."""
    runs = []
    for kw in (dict(capture=False), dict(), dict(page=4), dict(page=64), dict(page=4, capture=False)):
        dec = _decoder(gpu, kv_bits=kv_bits, length_penalty=length_penalty, **kw)
        b = _start(dec)
        for n in (1, 4, 1, 4, 4, 4, 4):
            dec.step(b, n)
        torch.cuda.synchronize()
        rows = dec._rows(torch.tensor(SLOTS)).reshape(-1).cuda()
        runs.append(_cpu(dec.out[rows], dec.score[SLOTS], dec.made[SLOTS], dec.ended[SLOTS], dec.pos[rows],
                         dec.finished[SLOTS]) + [dec.flags[SLOTS].clone()])
    for r in runs[1:]:
        for x, y in zip(r, runs[0]):
            assert torch.equal(x, y)
    assert runs[0][5].all() and runs[0][6].all()  # 22 steps: all at their limit of 20 tokens, or ended


def test_requests_do_not_depend_on_each_other(gpu):
    """A request's hypotheses are the same bits alone, beside others, and in a slot used before."""
    dec = _decoder(gpu)
    b = _start(dec)
    dec.step(b, 12)
    torch.cuda.synchronize()
    want = [dec.out[dec._rows(torch.tensor([s])).reshape(-1).cuda()].cpu() for s in SLOTS]
    scores = dec.score[SLOTS].cpu()
    for i in (2, 0, 1):
        b = _start(dec, (i,))
        dec.step(b, 12)
        torch.cuda.synchronize()
        rows = dec._rows(torch.tensor([SLOTS[i]])).reshape(-1).cuda()
        assert torch.equal(dec.out[rows].cpu(), want[i]) and torch.equal(dec.score[SLOTS[i]].cpu(), scores[i])


def test_as_many_requests_as_slots(gpu):
    """The buckets that are there by default hold as many requests as the service's default slots; a request's tokens are
    the same among many."""
    few = _decoder(gpu)
    b = _start(few)
    for _ in range(8):
        few.step(b)
    few.stream.synchronize()
    want = [few.tokens(s).cpu() for s in SLOTS]
    dec = _decoder(gpu, slots=128, buckets=None, capture=False)
    assert dec.bucket(128) == 128
    n = 101
    for i in range(n):
        dec.fill_cross(_memory(dec, [FRAMES[i % 3]], seed=i % 3), [FRAMES[i % 3]], [i], projected=True)
    dec.stream.wait_stream(torch.cuda.current_stream())
    dec.admit(list(range(n)), [PROMPTS[i % 3] for i in range(n)], [FRAMES[i % 3] for i in range(n)])
    b = dec.set_active(list(range(n)))
    assert b == 112
    for _ in range(8):
        dec.step(b)
    dec.stream.synchronize()
    for i in range(n):
        assert torch.equal(dec.tokens(i).cpu(), want[i % 3]), i


def test_scores_are_the_hypotheses_own(gpu):
    """Each hypothesis read token by token by a greedy decoder gives its score: the sum of its tokens' log probabilities.
    The two decoders' logits differ by the order of fp32 sums in the attentions, which moves bf16 roundings behind it: a
    few steps of 2^-8 of the largest logit in each term of a log probability."""
    from kernels.stream_decoder import StreamDecoder

    new = 10
    dec = _decoder(gpu, kv_bits=16, int8=False, beams=4)
    b = _start(dec, max_new=[new] * 3)
    dec.step(b, new)
    torch.cuda.synchronize()
    model = dec.model
    ref = StreamDecoder(model, slots=12, max_new_tokens=4, max_prompt=20, buckets=(12,), int8=False, frames=24,
                        capture=False)
    checked = 0
    for i in range(3):
        p = len(PROMPTS[i])
        hyps = dec.out[dec._rows(torch.tensor([SLOTS[i]])).reshape(-1).cuda()].cpu()
        score, ended, made = (t[SLOTS[i]].cpu() for t in (dec.score, dec.ended, dec.made))
        texts = [h[:p + int(m)] for h, m in zip(hyps, made)]
        ref.reset()
        for j in range(4):
            ref.fill_cross(_memory(ref, [FRAMES[i]], seed=i), [FRAMES[i]], [j], projected=True)
        ref.stream.wait_stream(torch.cuda.current_stream())
        ref.admit([0, 1, 2, 3], texts, [FRAMES[i]] * 4)
        rb = ref.set_active([0, 1, 2, 3])
        sums, worst = torch.zeros(4, dtype=torch.float64), 0.0
        for t in range(p + new - 1):
            ref.step(rb)
            ref.stream.synchronize()
            l = ref.logits[:4].double().cpu()
            worst = max(worst, float(l.abs().max()))
            lp = torch.log_softmax(l, -1)
            for j, text in enumerate(texts):
                if p <= t + 1 < len(text):
                    sums[j] += lp[j, int(text[t + 1])]
        tol = new * 2 * 4 * 2.0 ** -8 * worst
        assert ((sums - score.double()).abs() <= tol).all(), (sums, score, tol)
        assert (score[:-1] >= score[1:]).all()  # best first
        distinct = {tuple(t.tolist()) for t in texts}
        assert len(distinct) == 4
        checked += 1
        # the greedy text is among what the search has seen: the best hypothesis is at least about as likely
        assert float((sums[0] - sums.max())) >= -tol
    assert checked == 3


def test_one_beam_is_greedy(gpu):
    """With one beam every step takes its own logits' first largest entry."""
    dec = _decoder(gpu, capture=False, beams=1)
    b = _start(dec)
    for _ in range(10):
        dec.step(b)
        dec.stream.synchronize()
        live = dec.finished[SLOTS].cpu() == 0
        top = dec.logits[:3].float().argmax(1).cpu()
        tok = dec.tok[SLOTS].cpu()
        assert torch.equal(tok[live], top[live])


def test_rules_hold_for_every_beam(gpu):
    """Grammar, penalties and biases: every hypothesis follows its grammar (its state moves with the beams), repeats no
    token under a prohibitive penalty, and avoids what its bias row forbids."""
    from kernels.stream_decoder import Grammar, Rules

    V = 512
    classes = torch.arange(V) % 3
    trans = torch.tensor([[1, -1, -1], [-1, 2, -1], [-1, -1, 0]])  # classes 0, 1, 2 in turn
    bias = torch.zeros(1, V)
    bias[0, ::2] = -1e4
    for kw in (dict(capture=False), dict()):
        dec = _decoder(gpu, grammar=Grammar(classes, trans), penalties=True, bias=bias, beams=4, **kw)
        rules = [Rules(start=0), Rules(frequency=1e4, bias=0), Rules(start=2, presence=1e4)]
        b = _start(dec, rules=rules, max_new=[9, 9, 9])
        for n in (1, 4, 4):
            dec.step(b, n)
        torch.cuda.synchronize()
        for i, s in enumerate(SLOTS):
            p = len(PROMPTS[i])
            for beam in range(4):
                row, made = s * 4 + beam, int(dec.made[s, beam])
                text = dec.out[row, p:p + made].tolist()
                assert made >= 1
                if i != 1:
                    assert [t % 3 for t in text] == [((0 if i == 0 else 2) + j) % 3 for j in range(made)]
                if i == 1:
                    assert all(t % 2 for t in text)
                if i:
                    assert len(set(text)) == len(text)


def test_refuses(gpu):
    from kernels.stream_decoder import Rules

    for kw in (dict(beams=0), dict(beams=17), dict(page=3), dict(page=512), dict(kv_bits=4), dict(length_penalty=-1.0),
               dict(length_penalty=float("nan"))):
        with pytest.raises(ValueError, match="BeamDecoder"):
            _decoder(gpu, capture=False, **kw)
    dec = _decoder(gpu, capture=False)
    for prompt, frames in ((torch.zeros(0), 3), (torch.zeros(5), 3), (torch.zeros(2), 0), (torch.zeros(2), 25)):
        with pytest.raises(ValueError, match="StreamDecoder"):
            dec.admit([0], [prompt], [frames])
    with pytest.raises(ValueError, match="penalties"):
        dec.admit([0], [torch.ones(2)], [3], rules=[Rules(presence=1.0)])


@pytest.mark.parametrize("length_penalty,page", [(0.0, 1), (1.0, 16)])
def test_pipeline_with_beams(gpu, length_penalty, page):
    """The service and the batch path give the same texts; a beam's text is made of its prompt and ends at the end token
    or its limit."""
    import bench
    from kernels.pipeline import Pipeline

    model = bench.random_asr_model(gpu, enc_layers=1, seed=6)
    pipe = Pipeline(model, None, 4, 12, True, True, buckets=(1, 2, 4), beams=3, length_penalty=length_penalty, page=page)
    xs = [Pipeline.prepare(x) for x in bench.synthetic_audio([32000, 52800, 17600, 9600, 30000], seed=10)]
    prompt = torch.tensor([4, 5, 6, 7])
    want = pipe.transcribe([torch.from_numpy(x).to(gpu) for x in xs], prompt)
    f1, f2 = pipe.submit(xs, prompt), pipe.submit(xs[:2], prompt, [3, 5])
    got, short = f1.result(timeout=120), f2.result(timeout=120)
    pipe.close()
    assert [len(t) for t in short] == [7, 9] or any(t[-1] == pipe.decoder.eos for t in short)
    for a, b in zip(got, want):
        assert np.array_equal(a[:4], prompt.numpy()) and len(a) <= 16
        assert np.array_equal(a, b), (a, b)
    with pytest.raises(ValueError, match="beams above 1"):
        Pipeline(model, None, 4, 12, True, True, length_penalty=1.0)
