"""StreamDecoder and Pipeline over 4-bit caches and under rules: the fill, every attention of a step, the rules on the
logits, captured against eager, and the service against the batch path."""

from __future__ import annotations

import pytest
import torch

from decoder_helpers import make_decoder
from q4_helpers import BF, assert_rounded, attention64, codes64, logits64, pack

pytestmark = pytest.mark.gpu


def _ext():
    from kernels.cuda_ext import ext

    return ext


@pytest.mark.parametrize("rows,L,H", [(1, 1, 1), (70, 2, 3), (400, 3, 8), (1500, 8, 8)])
def test_gemm_kv_q4_equals_gemm_then_scatter(gpu, rows, L, H):
    print(f"gemm_kv_q4 rows={rows} L={L} H={H}", flush=True)
    ext, K, S = _ext(), 1024, 3
    g = torch.Generator().manual_seed(rows)
    a = torch.randn(rows, K, generator=g).to(BF).to(gpu)
    w = (0.03 * torch.randn(L * 2 * H * 128, K, generator=g)).to(BF).to(gpu)
    bias = torch.randn(L * 2 * H * 128, generator=g).to(BF).to(gpu)
    T = rows // 2 + 1
    where = torch.randperm(S * T, generator=g)[:rows]
    slot, frame = (where // T).to(torch.int32), (where % T).to(torch.int32)
    if rows > 3:
        slot[1], slot[2], frame[3], frame[0] = -1, S, T, -2
    slot, frame = slot.to(gpu), frame.to(gpu)
    caches = [[torch.full((L, S, H, T, 64), 0x5a, dtype=torch.uint8, device=gpu) for _ in range(2)] +
              [torch.full((L, S, H, T, 4), -3.0, dtype=BF, device=gpu) for _ in range(2)] for _ in range(2)]
    kv = torch.empty(rows, L * 2 * H * 128, dtype=BF, device=gpu)
    ext.gemm(a, w, bias, kv, 0, None, 1.0, 8)
    ext.dec_scatter_kv_q4(kv, slot, frame, *caches[0])
    ext.gemm_kv_q4(a, w, bias, slot, frame, *caches[1])
    for x, y in zip(*caches):
        assert torch.equal(x, y)
    # and the scatter's bytes are the definition's
    c, m = codes64(kv.cpu().reshape(rows, L, 2, H, 128))
    for i in range(rows - 1, max(-1, rows - 4), -1):
        if 0 <= int(slot[i]) < S and 0 <= int(frame[i]) < T:
            assert torch.equal(caches[1][0][:, slot[i], :, frame[i]].cpu(), pack(c[i, :, 0]))
            assert torch.equal(caches[1][3][:, slot[i], :, frame[i]].cpu(), m[i, :, 1].to(BF))


def _decoder(gpu, seed=21, **kw):
    from kernels.stream_decoder import StreamDecoder

    model = make_decoder(hidden=512, heads=4, layers=2, ffn=512, vocab=512, seed=seed, device=gpu, dtype=BF)
    a = dict(slots=6, max_new_tokens=20, max_prompt=4, buckets=(2, 4), int8=True, frames=24)
    a.update(kw)
    return StreamDecoder(model, **a)


def _start(dec, rules=None):
    g = torch.Generator().manual_seed(3)
    slots, lengths = [4, 0, 3], [24, 5, 11]
    mem = torch.randn(sum(lengths), dec.width, generator=g).to(BF).to(dec.device)
    prompts = [torch.randint(5, 512, (n,), generator=g) for n in (3, 1, 4)]
    dec.fill_cross(mem, lengths, slots)
    torch.cuda.synchronize()
    dec.admit(slots, prompts, lengths, None, rules)
    return slots, dec.set_active(slots)


@pytest.mark.parametrize("int8", [True, False])
def test_attentions_of_a_step(gpu, int8):
    """Every attention of six eager steps against the 64-bit form on the caches as they stand; the caches hold the
    definition's codes of what was appended."""
    dec = _decoder(gpu, capture=False, kv_bits=4, int8=int8)
    slots, b = _start(dec)
    per, bound = 8, None
    for step in range(6):
        dec.stream.synchronize()
        with torch.cuda.stream(dec.stream):
            dec._embed(b)
            for i, op in enumerate(dec.programs[b]):
                layer, at = divmod(i, per)
                is_self = at == 1
                attend = layer < len(dec.blocks) and at in (1, 4)
                if attend:
                    dec.stream.synchronize()
                    caches = [t[layer].cpu() for t in ((dec.self_k, dec.self_v, dec.self_ks, dec.self_vs) if is_self else
                                                       (dec.cross_k, dec.cross_v, dec.cross_ks, dec.cross_vs))]
                    q, n = (dec.qkv_out if is_self else dec.q_out)[:b].cpu(), (dec.pos if is_self else dec.cross_len).cpu()
                op()
                if attend:
                    dec.stream.synchronize()
                    act = dec.active[:b].cpu()
                    want, bound = attention64(is_self, act, q, *caches, n, dec.scale, dec.h)
                    err = (dec.att[:b].cpu().double() - want).abs()
                    assert (err <= bound).all(), (step, layer, is_self, float((err / bound).max()))
                    if is_self:
                        c, m = codes64(q[:, dec.width:].reshape(b, 2, dec.h, 128))
                        for r, s in enumerate(slots):
                            assert torch.equal(dec.self_k[layer, s, :, n[s]].cpu(), pack(c[r, 0]))
                            assert torch.equal(dec.self_vs[layer, s, :, n[s]].cpu(), m[r, 1].to(BF))
    assert bound is not None and dec.pos[torch.tensor(slots)].tolist() == [6, 6, 6]


@pytest.mark.parametrize("fused", [True, False])
def test_captured_equals_eager(gpu, fused):
    """With 4-bit caches and every rule: replays of one step and of chunks against the eager program, bit for bit."""
    from kernels.stream_decoder import Grammar, Rules

    classes = torch.arange(512) % 4
    grammar = Grammar(classes, [[1, 1, -1, 2], [0, -1, 2, 2], [0, 1, 2, -1]])
    bias = torch.randn(2, 512, generator=torch.Generator().manual_seed(5))
    kw = dict(kv_bits=4, fused=fused, penalties=True, bias=bias, grammar=grammar)
    rules = [Rules(repetition=1.3, prompt=True, start=1), Rules(presence=0.4, frequency=0.2, bias=1), None]
    decs = [_decoder(gpu, capture=False, **kw), _decoder(gpu, **kw)]
    for d in decs:
        _, b = _start(d, rules)
        for n in (1, 1, 4, 1, 4, 4):
            d.step(b, n)
        torch.cuda.synchronize()
    for name in ("logits", "tok", "pos", "out", "finished", "self_k", "self_v", "self_ks", "self_vs", "gstate"):
        x, y = (getattr(d, name) for d in decs)
        x, y = (x[:, :6], y[:, :6]) if name.startswith("self") else (x[:6], y[:6])  # not the padding rows' slot
        if name == "logits":
            x, y = x[:3], y[:3]
        assert torch.equal(x, y), name


def test_rules_of_requests(gpu):
    """Each step's logits under the requests' rules against the 64-bit form, the token the pick makes of them, and a slot
    taken over by a request without rules."""
    from kernels.stream_decoder import Grammar, Rules

    classes = torch.arange(512) % 5
    trans = torch.tensor([[1, -1, 0, -1, -1], [-1, 2, -1, 1, -1], [0, 0, -1, -1, 2]])
    dec = _decoder(gpu, capture=False, kv_bits=4, penalties=True, grammar=Grammar(classes, trans),
                   bias=2 * torch.randn(3, 512, generator=torch.Generator().manual_seed(6)))
    rules = [Rules(repetition=1.5, presence=0.3, frequency=0.2, prompt=True, bias=2, start=0), Rules(start=2),
             Rules(repetition=0.5)]
    slots, b = _start(dec, rules)

    def steps(count):
        for _ in range(count):
            with torch.cuda.stream(dec.stream):
                dec._embed(b)
                for op in dec.programs[b][:-2]:
                    op()
                dec.stream.synchronize()
                args = [t.cpu() for t in (dec.logits[:b], dec.active[:b], dec.pos, dec.out, dec.first, dec.plen, dec.pen,
                                          dec.bias, dec.bias_of, dec.mask, dec.classes, dec.trans, dec.start, dec.gstate)]
                want, slack, state = logits64(*args)
                for op in dec.programs[b][-2:]:
                    op()
                dec.stream.synchronize()
            assert_rounded(dec.logits[:b], want, slack)
            assert torch.equal(dec.gstate.cpu(), state)
            for r, s in enumerate(slots):
                if int(args[2][s]) + 1 >= int(dec.plen[s]) and not args[2][s] == dec.pos[s].cpu():
                    assert int(dec.tok[s]) == int(dec.logits[r].float().argmax())

    steps(12)
    made = dec.out.cpu()
    st = 0
    for t in made[4, 3:int(dec.pos[4]) + 1].tolist():  # the first request's tokens are the grammar's
        assert trans[st, classes[t]] >= 0
        st = int(trans[st, classes[t]])
    dec.admit([4], [torch.tensor([7, 8])], [24])
    dec._embed_stale = True
    assert dec.pen[4].tolist() == [1.0, 0.0, 0.0] and int(dec.bias_of[4]) == -1 and int(dec.start[4]) == -1
    steps(3)


def test_rules_refused(gpu):
    from kernels.stream_decoder import Grammar, Rules, StreamDecoder

    plain = _decoder(gpu, capture=False)
    assert plain.kv_bits == 8 and not plain.rules_on
    for r in (Rules(repetition=1.1), Rules(presence=1.0), Rules(bias=0), Rules(start=0)):
        with pytest.raises(ValueError):
            plain.admit([0], [torch.tensor([5])], [3], None, [r])
    with pytest.raises(ValueError):
        plain.admit([0], [torch.tensor([5])], [3], None, [None, None])
    dec = _decoder(gpu, capture=False, penalties=True, bias=torch.zeros(2, 512))
    for r in (Rules(repetition=0.0), Rules(repetition=float("nan")), Rules(presence=float("inf")), Rules(bias=2),
              Rules(bias=-2), Rules(start=0)):
        with pytest.raises(ValueError):
            dec.admit([0], [torch.tensor([5])], [3], None, [r])
    for kw in (dict(kv_bits=5), dict(bias=torch.zeros(2, 511)), dict(bias=torch.zeros(0, 512)),
               dict(grammar=Grammar([0] * 511, [[0]]))):
        with pytest.raises(ValueError):
            StreamDecoder(plain.model, slots=2, buckets=(2,), frames=8, capture=False, **kw)


def test_pipeline_under_rules(gpu):
    """A service over 4-bit caches with rules per request: the tokens of transcribe(), requests of different rules side by
    side, tokens of the grammar only."""
    import bench
    from kernels.pipeline import Pipeline
    from kernels.stream_decoder import Grammar, Rules

    model = bench.random_asr_model(gpu, enc_layers=1, seed=6)
    V = model.proj_out.weight.shape[0]
    grammar = Grammar(torch.arange(V) % 3, [[1, -1, -1], [-1, 0, 1]])
    pipe = Pipeline(model, None, 4, 12, True, True, buckets=(1, 2, 4), kv_bits=4, penalties=True, grammar=grammar)
    assert pipe.decoder.kv_bits == 4 and pipe.decoder.cross_k.dtype == torch.uint8
    lengths = [32000, 52800, 17600]
    xs = [Pipeline.prepare(x) for x in bench.synthetic_audio(lengths, seed=10)]
    gpu_xs = [torch.from_numpy(x).to(gpu) for x in xs]
    prompt = torch.tensor([4, 5, 6, 7])
    bound, free = Rules(repetition=1.2, start=0), None
    want = [pipe.transcribe(gpu_xs, prompt, None, r) for r in (bound, free)]
    with pytest.raises(ValueError):
        pipe.submit(xs, prompt, None, Rules(bias=1))
    futures = [pipe.submit(xs, prompt, None, r) for r in (bound, free)]
    got = [f.result(timeout=60) for f in futures]
    pipe.close()
    for row in want[0]:
        st = 0
        for t in row[4:].tolist():
            nxt = int(grammar.transitions[st, t % 3])
            assert nxt >= 0, (row.tolist(), st)
            st = nxt
    for w, g in zip(want, got):
        for a, b in zip(w, g):
            assert a.tolist() == b.tolist()
    assert any(a.tolist() != b.tolist() for a, b in zip(*want))
