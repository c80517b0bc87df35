"""Single tokens, short and long chunks in one call over pages: a sequence's rows depend on that sequence alone, to the
bit, and are as exact as its own length says; prompts of any length in BeamDecoder with them."""

from __future__ import annotations

import pytest
import torch

from decoder_helpers import make_decoder
from paged_helpers import BF, D, Paged, close, same_bits

pytestmark = pytest.mark.gpu


def _check_each(c, got):
    """Every sequence within its own bound: weights to 2^-17 up to 16 query rows to a key head, in bf16 above."""
    fine, coarse = c.attention64(), c.attention64(weights_bf16=True)
    for i, rows in enumerate(c.chunk):
        a, b = int(c.starts[i]), int(c.starts[i + 1])
        want, bound, _ = coarse if rows * c.ratio > 16 else fine
        close(got[a:b], want[a:b], bound[a:b])
    assert (got[~fine[2]] == 7).all()


def _alone(c, i):
    """A call of sequence i of c alone."""
    x = Paged.__new__(Paged)
    x.__dict__.update(c.__dict__)
    a, b = int(c.starts[i]), int(c.starts[i + 1])
    x.q, x.rows, x.chunk = c.q[a:b].contiguous(), b - a, [b - a]
    x.active, x.starts = c.active[i:i + 1].contiguous(), torch.tensor([0, b - a], dtype=torch.int32)
    return x


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("splits", [1, 2, 3, 8, 16])
@pytest.mark.parametrize("ratio,page,chunk,held", [
    (1, 16, [1, 300, 16, 17, 0, 40, 1, 5], [700, 90, 33, 0, 8, 2000, 0, 15]),
    (3, 4, [5, 1, 6, 70, 1], [64, 1500, 0, 300, 7]),
    (2, 64, [1] * 9 + [500], [100] * 9 + [30]), (1, 1, [1] * 60 + [900], [20] * 60 + [0]),
    (16, 16, [1, 2, 0, 9], [300, 5, 3, 0]), (17, 16, [1, 3, 1], [300, 5, 700])])
def test_a_sequence_alone_and_beside_others(gpu, bits, splits, ratio, page, chunk, held):
    print(f"mixed bits={bits} splits={splits} ratio={ratio} page={page}", flush=True)
    c = Paged(40 + page + ratio, held, chunk, 2, ratio, page, bits, front=2, back=3)
    got = c.run(splits)
    _check_each(c, got[0])
    for a, b in zip(got[1:], c.appended()):
        assert same_bits(a, b)
    for i in {0, 1, 2, len(chunk) // 2, len(chunk) - 1}:
        if chunk[i]:
            alone = _alone(c, i).run(splits)[0]
            assert torch.equal(got[0][int(c.starts[i]):int(c.starts[i + 1])], alone), (i, chunk[i])


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("copies", [3, 40, 90])
def test_many_sequences_of_all_lengths(gpu, bits, copies):
    """Few, and more than one wave's lanes of, sequences; the same sequence in every group of them has the same rows."""
    chunk, held = [3, 1, 0, 33, 18, 1], [40, 7, 5, 0, 130, 64]
    c = Paged(50 + copies, held * copies, chunk * copies, 1, 2, 16, bits, front=1, back=2)
    for splits in (1, 2, 4):
        _check_each(c, c.run(splits)[0])


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("splits", [1, 3, 9])
@pytest.mark.parametrize("ratio,page,chunk", [(1, 16, [2, 15, 16, 9]), (2, 4, [8, 3, 1, 5]), (5, 1, [3, 2]), (8, 64, [2, 1])])
def test_few_rows_hold_weights_to_2_17(gpu, bits, splits, ratio, page, chunk):
    """Chunks of up to 16 query rows to a key head, several tokens among them, absent pages and odd ends, at the tight
    bound."""
    held = [70, 33, 0, 129][:len(chunk)]
    c = Paged(60 + page, held, chunk, 2, ratio, page, bits, front=1, back=1, absent=((0, 1),) if page == 16 else ())
    got = c.run(splits)
    want, bound, written = c.attention64()
    close(got[0][written], want[written], bound[written])
    for a, b in zip(got[1:], c.appended()):
        assert same_bits(a, b)


@pytest.mark.parametrize("starts", [[9, 0, 200], [150, 40, 30], [200, 200, 0], [-5, 7, 1000], [2 ** 31 - 1, 0, -2 ** 31]])
def test_starts_that_do_not_ascend(gpu, starts):
    """Nothing outside the rows that are there is read or written: neighbours of out stay as they were."""
    from kernels.cuda_ext import ext

    c = Paged(70, [30, 20], [100, 100], 2, 3, 16, 16)
    q, guard = c.q.contiguous().cuda(), torch.full((c.rows + 64, c.H * D), 7.0, dtype=BF, device="cuda")
    args = (c.k.cuda(), c.v.cuda(), c.table.cuda(), c.n.cuda(), c.scale)
    for splits in (1, 2, 3):
        part = torch.empty(c.rows * c.H * splits * 130, device="cuda") if splits > 1 else None
        ext.dec_attention_paged(c.active.cuda(), torch.tensor(starts, dtype=torch.int32).cuda(), q, *args, splits, part,
                                guard[32:-32])
        assert (guard[:32] == 7).all() and (guard[-32:] == 7).all()


@pytest.mark.parametrize("kv_bits", [16, 8])
def test_prompts_of_any_length_do_not_depend_on_each_other(gpu, kv_bits):
    """What the pages hold of a prompt, and the hypotheses behind it, are the same bits alone and beside others."""
    from kernels.beam_decoder import BeamDecoder

    model = make_decoder(hidden=512, heads=4, layers=2, ffn=512, vocab=512, seed=23, device=gpu, dtype=BF)
    with torch.no_grad():
        model.proj_out.weight.mul_(4)
    dec = BeamDecoder(model, slots=6, max_new_tokens=8, max_prompt=48, buckets=(2, 6), int8=True, frames=24, beams=3,
                      kv_bits=kv_bits, capture=False)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(4, 500, (n,), generator=g) for n in (41, 3, 18, 48, 17, 2)]
    frames = [24, 9, 1, 7, 24, 3]

    def run(which):
        dec.reset()
        for i in which:
            m = torch.randn(frames[i], dec.width, generator=torch.Generator().manual_seed(i)).to(BF).cuda()
            dec.fill_cross(m, [frames[i]], [i], projected=True)
        dec.stream.wait_stream(torch.cuda.current_stream())
        dec.admit(list(which), [prompts[i] for i in which], [frames[i] for i in which])
        dec.stream.synchronize()
        held = [[x[:, dec.table[i * 3, :len(prompts[i]) - 1].long()].cpu() for x in
                 (dec.self_k, dec.self_v) + ((dec.self_ks, dec.self_vs) if kv_bits == 8 else ())] for i in which]
        dec.step(dec.set_active(list(which)), 6)
        dec.stream.synchronize()
        return {i: h + [dec.out[i * 3:i * 3 + 3].cpu(), dec.score[i].cpu()] for i, h in zip(which, held)}

    together = run((0, 1, 2, 3, 4, 5))
    for which in ((0,), (3,), (2,), (4, 1), (0, 1)):
        for i, got in run(which).items():
            for a, b in zip(got, together[i]):
                assert same_bits(a, b), (which, i)
