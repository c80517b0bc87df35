"""What the entry points over pages and of beam search refuse, on the CPU."""

from __future__ import annotations

import pytest
import torch

from paged_helpers import BF, held_q8

I32, I64, U8 = (dict(dtype=t) for t in (torch.int32, torch.int64, torch.uint8))


def _attention(bits, **change):
    pages = dict(k=torch.zeros(5, 2, 4, 128, dtype=BF), v=torch.zeros(5, 2, 4, 128, dtype=BF))
    if bits == 8:
        pages = dict(k=torch.zeros(5, 2, 4, 128, dtype=torch.int8), v=torch.zeros(5, 2, 4, 128, dtype=torch.int8),
                     ks=torch.zeros(5, 2, 4), vs=torch.zeros(5, 2, 4))
    a = dict(active=torch.zeros(2, **I32), starts=torch.tensor([0, 1, 3], **I32), q=torch.zeros(3, 8 * 128, dtype=BF),
             **pages, table=torch.zeros(3, 6, **I32), n=torch.zeros(3, **I32), scale=1.0, splits=1, part=None,
             out=torch.zeros(3, 4 * 128, dtype=BF))
    a.update(change)
    return a


ATTENTION = [
    dict(q=torch.zeros(3, 7 * 128, dtype=BF)), dict(q=torch.zeros(3, 8 * 128)),
    dict(q=torch.zeros(8 * 128, 3, dtype=BF).t()), dict(q=torch.zeros(4, 8 * 128, dtype=BF)),
    dict(active=torch.zeros(2, **I64)), dict(active=torch.zeros(3, **I32)), dict(starts=None),
    dict(starts=torch.zeros(2, **I32)), dict(starts=torch.zeros(3, **I64)), dict(table=torch.zeros(3, 6, **I64)),
    dict(table=torch.zeros(18, **I32)), dict(table=torch.zeros(3, 0, **I32)), dict(table=torch.zeros(6, 3, **I32).t()),
    dict(n=torch.zeros(2, **I32)), dict(splits=0), dict(splits=65, part=torch.zeros(10 ** 6)), dict(splits=2),
    dict(splits=2, part=torch.zeros(3 * 4 * 2 * 130 - 1)), dict(splits=2, part=torch.zeros(3 * 4 * 2 * 130, dtype=BF)),
    dict(out=torch.zeros(3, 3 * 128, dtype=BF)), dict(out=torch.zeros(3, 500, dtype=BF)),
    dict(out=torch.zeros(2, 4 * 128, dtype=BF)), dict(out=torch.zeros(3, 0, dtype=BF))]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("change", ATTENTION)
def test_attention_refuses(bits, change):
    from kernels.cuda_ext import ext

    fn = ext.dec_attention_paged if bits == 16 else ext.dec_attention_paged_q8
    with pytest.raises(RuntimeError, match="dec_attention_paged"):
        fn(*_attention(bits, **change).values())


@pytest.mark.parametrize("bits,change", [
    (16, dict(k=torch.zeros(5, 2, 4, 128))), (16, dict(k=torch.zeros(5, 2, 4, 64, dtype=BF))),
    (16, dict(v=torch.zeros(5, 2, 8, 128, dtype=BF))), (16, dict(v=torch.zeros(5, 2, 4, 256, dtype=BF)[..., :128])),
    (16, dict(k=torch.zeros(0, 2, 4, 128, dtype=BF), v=torch.zeros(0, 2, 4, 128, dtype=BF))),
    (16, dict(k=torch.zeros(5, 3, 4, 128, dtype=BF), v=torch.zeros(5, 3, 4, 128, dtype=BF))),
    (8, dict(k=torch.zeros(5, 2, 4, 128, dtype=torch.uint8))), (8, dict(ks=torch.zeros(5, 2, 4, 1))),
    (8, dict(vs=torch.zeros(5, 2, 4, dtype=BF))), (8, dict(vs=torch.zeros(5, 4, 2).transpose(1, 2)))])
def test_attention_refuses_pages(bits, change):
    from kernels.cuda_ext import ext

    fn = ext.dec_attention_paged if bits == 16 else ext.dec_attention_paged_q8
    with pytest.raises(RuntimeError, match="dec_attention_paged"):
        fn(*_attention(bits, **change).values())


def test_c_abi_refuses_sizes():
    """Sizes that only the C entry checks (page sizes, row strides, alignment), without a launch."""
    import ctypes

    from kernels.cuda_ext import ext

    lib, buf = ext._lib, torch.zeros(4096)
    p = buf.data_ptr()

    def attention(**kw):
        a = dict(active=p, starts=p, seqs=2, q=p, ldq=1024, rows=3, k=p, v=p, pages=5, P=4, table=p, width=6, n=p, slots=3,
                 heads=4, kv=2, scale=ctypes.c_float(1.0), splits=1, part=None, part_len=0, out=p, stream=None)
        a.update(kw)
        return lib.cohere_dec_attention_paged(*a.values())

    for bad in (dict(P=3), dict(P=512), dict(P=0), dict(ldq=1020), dict(ldq=1000), dict(q=p + 2), dict(k=p + 8),
                dict(out=p + 2), dict(pages=0), dict(width=2 ** 29), dict(heads=5), dict(heads=0), dict(slots=0),
                dict(splits=2, part=p, part_len=3 * 4 * 2 * 130 - 1), dict(rows=-1), dict(starts=None), dict(active=None)):
        assert attention(**bad) == 1, bad
        assert lib.cohere_last_error()
    assert attention(rows=0) == 0 and attention(seqs=0) == 0
    assert lib.cohere_dec_attention_paged_splits(0, 1, 8, 8, 100) == 1
    assert lib.cohere_dec_attention_paged_splits(4, 4, 8, 3, 100) == 1

    def gather(**kw):
        a = dict(slot=p, pos=p, rows=3, table=p, slots=3, width=6, k=p, v=p, L=2, pages=5, kv=2, P=4, out=p, ldkv=1024,
                 stream=None)
        a.update(kw)
        return lib.cohere_dec_gather_paged(*a.values())

    for bad in (dict(P=5), dict(ldkv=1016), dict(ldkv=1028), dict(out=p + 8), dict(k=None), dict(L=0), dict(rows=2 ** 31)):
        assert gather(**bad) == 1, bad
    assert gather(rows=0) == 0

    def select(**kw):
        a = dict(logits=p, ld=64, n=2, beams=4, V=64, groups=p, slots=3, score=p, finished=p, made=None, norm=None,
                 norm_len=0, pad=3, parent=p, token=p, total=p, work=p, work_bytes=8 * (16 + 32), stream=None)
        a.update(kw)
        return lib.cohere_dec_beam_select(*a.values())

    assert lib.cohere_dec_beam_select_work(8, 64, 4) == 8 * (16 + 32)
    for bad in (dict(beams=0), dict(beams=17), dict(V=60), dict(V=0), dict(ld=56), dict(ld=68), dict(pad=-1), dict(pad=64),
                dict(norm=p, made=p, norm_len=0), dict(norm=p, norm_len=4), dict(work_bytes=8 * 48 - 1), dict(work=None),
                dict(work=p + 4), dict(logits=p + 4), dict(n=20000), dict(beams=16, V=8)):
        assert select(**bad) == 1, bad
    assert select(n=0) == 0

    def reorder(**kw):
        a = dict(groups=p, m=2, beams=4, parent=p, n=p, done=None, slots=3, table=p, width=6, tokens=p, OUT=9, states=None,
                 NS=0, k=p, v=p, ks=None, vs=None, L=2, pages=5, kv=2, P=4, bits=16, stream=None)
        a.update(kw)
        return lib.cohere_dec_beam_reorder(*a.values())

    for bad in (dict(beams=17), dict(beams=0), dict(P=3), dict(bits=4), dict(bits=8), dict(table=None), dict(k=None),
                dict(OUT=0), dict(states=p), dict(m=65536), dict(L=2 ** 20, kv=2 ** 10), dict(n=None), dict(k=p + 8)):
        assert reorder(**bad) == 1, bad
    assert reorder(m=0) == 0


def _select(**change):
    a = dict(logits=torch.zeros(8, 64, dtype=BF), groups=torch.zeros(2, **I32), score=torch.zeros(3, 4),
             finished=torch.zeros(3, 4, **U8), made=torch.zeros(3, 4, **I32), norm=torch.ones(5), pad=1,
             parent=torch.zeros(2, 4, **I32), token=torch.zeros(2, 4, **I64), total=torch.zeros(2, 4),
             work=torch.zeros(10 ** 4, **U8))
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    dict(logits=torch.zeros(7, 64, dtype=BF)), dict(logits=torch.zeros(8, 64)), dict(logits=torch.zeros(64, 8, dtype=BF).t()),
    dict(groups=torch.zeros(2, **I64)), dict(score=torch.zeros(3, 17)), dict(score=torch.zeros(3, 4, dtype=torch.float64)),
    dict(score=torch.zeros(0, 4)), dict(score=torch.zeros(4, 3).t()), dict(finished=torch.zeros(3, 4, dtype=torch.bool)),
    dict(finished=torch.zeros(2, 4, **U8)), dict(made=None), dict(made=torch.zeros(3, 4, **I64)),
    dict(norm=torch.ones(5, dtype=torch.float64)), dict(norm=torch.ones(0)), dict(parent=torch.zeros(1, 4, **I32)),
    dict(token=torch.zeros(2, 4, **I32)), dict(total=torch.zeros(2, 5)), dict(work=torch.zeros(100)), dict(pad="x")])
def test_select_refuses(change):
    from kernels.cuda_ext import ext

    with pytest.raises(RuntimeError, match="dec_beam_select"):
        ext.dec_beam_select(*_select(**change).values())


def _reorder(**change):
    a = dict(groups=torch.zeros(2, **I32), parent=torch.zeros(2, 4, **I32), n=torch.zeros(12, **I32),
             done=torch.zeros(3, **U8), table=torch.zeros(12, 6, **I32), tokens=torch.zeros(12, 9, **I64),
             states=torch.zeros(12, 2, **I32), k=torch.zeros(1, 5, 2, 4, 128, dtype=torch.int8),
             v=torch.zeros(1, 5, 2, 4, 128, dtype=torch.int8), ks=torch.zeros(1, 5, 2, 4), vs=torch.zeros(1, 5, 2, 4))
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    dict(parent=torch.zeros(2, 17, **I32)), dict(parent=torch.zeros(3, 4, **I64)), dict(parent=torch.zeros(1, 4, **I32)),
    dict(n=torch.zeros(11, **I32)), dict(n=torch.zeros(12, **I64)), dict(done=torch.zeros(2, **U8)),
    dict(table=torch.zeros(11, 6, **I32)), dict(table=None), dict(tokens=torch.zeros(12, 9, **I32)),
    dict(tokens=torch.zeros(12, 0, **I64)), dict(states=torch.zeros(11, 2, **I32)), dict(v=None), dict(ks=None),
    dict(ks=None, vs=None), dict(k=None, v=None), dict(k=torch.zeros(1, 5, 2, 4, 64, dtype=torch.int8)),
    dict(vs=torch.zeros(1, 5, 2, 3))])
def test_reorder_refuses(change):
    from kernels.cuda_ext import ext

    with pytest.raises(RuntimeError, match="dec_beam_reorder"):
        ext.dec_beam_reorder(*_reorder(**change).values())


def test_advance_refuses():
    from kernels.cuda_ext import ext

    a = dict(groups=torch.zeros(2, **I32), parent=torch.zeros(2, 4, **I32), token=torch.zeros(2, 4, **I64),
             total=torch.zeros(2, 4), dummy=2, tok=torch.zeros(12, **I64), pos=torch.zeros(12, **I32), held=None,
             score=torch.zeros(3, 4), finished=torch.zeros(3, 4, **U8), made=torch.zeros(3, 4, **I32),
             done=torch.zeros(3, **U8), limit=torch.zeros(3, **I32), out=torch.zeros(12, 9, **I64), eos=1, by_length=False,
             emb=torch.zeros(64, 256, dtype=BF), ptab=torch.zeros(9, 256, dtype=BF), w0=torch.zeros(256, dtype=BF),
             b0=torch.zeros(256, dtype=BF), eps0=1e-5, w1=torch.zeros(256, dtype=BF), b1=torch.zeros(256, dtype=BF),
             eps1=1e-5, x=torch.zeros(8, 256, dtype=BF), h=torch.zeros(8, 256, dtype=BF), flags=None)
    for change in (dict(tok=torch.zeros(11, **I64)), dict(pos=torch.zeros(12, **I64)), dict(made=torch.zeros(3, 3, **I32)),
                   dict(done=torch.zeros(2, **U8)), dict(out=torch.zeros(12, 0, **I64)),
                   dict(emb=torch.zeros(64, 128, dtype=BF)), dict(w0=torch.zeros(255, dtype=BF)),
                   dict(x=torch.zeros(7, 256, dtype=BF)), dict(flags=torch.zeros(2, **U8)), dict(held=torch.zeros(11, **I32)), dict(score=torch.zeros(3, 17)),
                   dict()):  # the last one only for its place
        with pytest.raises(RuntimeError, match="dec_beam_advance"):
            ext.dec_beam_advance(*{**a, **change}.values())


def test_no_gpu_tensors_refused():
    from kernels.cuda_ext import ext

    for bits, fn in ((16, ext.dec_attention_paged), (8, ext.dec_attention_paged_q8)):
        with pytest.raises(RuntimeError, match="current GPU"):
            fn(*_attention(bits).values())
    with pytest.raises(RuntimeError, match="current GPU"):
        ext.dec_beam_select(*_select().values())
    with pytest.raises(RuntimeError, match="current GPU"):
        ext.dec_beam_reorder(*_reorder().values())
    with pytest.raises(TypeError):
        ext._lib and __import__("kernels.cuda_ext", fromlist=["_calls"])._calls.dec_beam_select(1, 2)


def test_held_q8_form():
    """The 8-bit form's own test: codes of a vector that reaches 127 exactly, ties to even, tiny vectors."""
    x = torch.zeros(3, 128)
    x[0, :4] = torch.tensor([127.0, -127.0, 0.5, 1.5])
    x[1, 0] = 2.0 ** -133
    c, s = held_q8(x.to(BF))
    assert s[0] == 1 and c[0, :4].tolist() == [127, -127, 0, 2]
    assert s[1] == 2.0 ** -126 and s[2] == 2.0 ** -126 and (c[1:] == 0).all()
