"""The 4-bit form on the host, and what the entry points over 4-bit caches and the rules on logits refuse, on the CPU."""

from __future__ import annotations

import pytest
import torch

from q4_helpers import BF, codes64, pack, value64


def test_quantize_q4_form():
    from kernels.stream_decoder import dequantize_q4, quantize_q4

    x = torch.zeros(2, 128)
    x[0, :4] = torch.tensor([7.0, -7.0, 0.5, 1.5])  # m = 7: codes 7, -7, 0 (half to even), 2
    x[0, 33], x[0, 95] = -14.0, 3.0
    x[1] = torch.linspace(-1, 1, 128)
    codes, m = quantize_q4(x.to(BF))
    assert m[0].tolist() == [7.0, 14.0, 3.0, 0.0]
    assert codes[0, 0] == 0x97 and codes[0, 1] == 0x20 and codes[0, 16] == 0x90 and codes[0, 47] == 0x70
    c, _ = codes64(x.to(BF))
    assert torch.equal(codes, pack(c))
    assert torch.equal(dequantize_q4(codes, m).double(), value64(codes, m).float().double())
    # a value is off by at most half a step
    step = (m.double() / 7).repeat_interleave(32, -1)
    assert ((dequantize_q4(codes, m).double() - x.to(BF).double()).abs() <= step * (0.5 + 1e-6)).all()


def _attention_args(**change):
    a = dict(self_attn=True, active=torch.zeros(2, dtype=torch.int32), q=torch.zeros(2, 8 * 128, dtype=BF),
             k4=torch.zeros(3, 2, 5, 64, dtype=torch.uint8), v4=torch.zeros(3, 2, 5, 64, dtype=torch.uint8),
             ks=torch.zeros(3, 2, 5, 4, dtype=BF), vs=torch.zeros(3, 2, 5, 4, dtype=BF),
             n=torch.zeros(3, dtype=torch.int32), scale=1.0, splits=1, part=None,
             out=torch.zeros(2, 4 * 128, dtype=BF))
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 7 * 128, dtype=BF)), dict(q=torch.zeros(2, 8 * 128)), dict(q=torch.zeros(8 * 128, 2, dtype=BF).t()),
    dict(k4=torch.zeros(3, 2, 5, 64, dtype=torch.int8)), dict(k4=torch.zeros(3, 2, 4, 64, dtype=torch.uint8)),
    dict(v4=torch.zeros(3, 2, 5, 128, dtype=torch.uint8)[..., :64]), dict(ks=torch.zeros(3, 2, 5, 4)),
    dict(vs=torch.zeros(3, 2, 5, 1, dtype=BF)), dict(active=torch.zeros(2, dtype=torch.int64)),
    dict(active=torch.zeros(1, dtype=torch.int32)), dict(n=torch.zeros(2, dtype=torch.int32)), dict(splits=0),
    dict(splits=2), dict(splits=65, part=torch.zeros(10 ** 6)), dict(splits=2, part=torch.zeros(2 * 4 * 2 * 130 - 1)),
    dict(out=torch.zeros(2, 3 * 128, dtype=BF)), dict(out=torch.zeros(2, 500, dtype=BF)),
    dict(out=torch.zeros(1, 4 * 128, dtype=BF)), dict(out=torch.zeros(2, 0, dtype=BF)),
    dict(k4=torch.zeros(3, 2, 0, 64, dtype=torch.uint8), v4=torch.zeros(3, 2, 0, 64, dtype=torch.uint8),
         ks=torch.zeros(3, 2, 0, 4, dtype=BF), vs=torch.zeros(3, 2, 0, 4, dtype=BF))])
def test_attention_refuses(change):
    from kernels.cuda_ext import ext

    with pytest.raises(RuntimeError, match="dec_attention_q4"):
        ext.dec_attention_q4(*_attention_args(**change).values())


def test_no_gpu_tensors_refused():
    from kernels.cuda_ext import ext

    with pytest.raises(RuntimeError, match="current GPU"):
        ext.dec_attention_q4(*_attention_args().values())
    x = torch.zeros(1, 16, dtype=BF)
    with pytest.raises(RuntimeError, match="current GPU"):
        ext.dec_logits(x, x, torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("name", ["dec_scatter_kv_q4", "dec_gather_kv_q4"])
@pytest.mark.parametrize("change", [dict(kv=torch.zeros(2, 511, dtype=BF)), dict(kv=torch.zeros(2, 512)),
                                    dict(slot_of=torch.zeros(1, dtype=torch.int32)),
                                    dict(frame_of=torch.zeros(2, dtype=torch.int64)),
                                    dict(cks=torch.zeros(1, 1, 2, 3, 4)),
                                    dict(cv=torch.zeros(1, 1, 2, 4, 64, dtype=torch.uint8))])
def test_kv_refuses(name, change):
    from kernels.cuda_ext import ext

    a = dict(kv=torch.zeros(2, 512, dtype=BF), slot_of=torch.zeros(2, dtype=torch.int32),
             frame_of=torch.zeros(2, dtype=torch.int32), ck=torch.zeros(1, 1, 2, 3, 64, dtype=torch.uint8),
             cv=torch.zeros(1, 1, 2, 3, 64, dtype=torch.uint8), cks=torch.zeros(1, 1, 2, 3, 4, dtype=BF),
             cvs=torch.zeros(1, 1, 2, 3, 4, dtype=BF))
    a.update(change)
    kv = a.pop("kv")
    with pytest.raises(RuntimeError, match=name):
        getattr(ext, name)(*((kv, *a.values()) if "scatter" in name else (*a.values(), kv)))


I32 = dict(dtype=torch.int32)


@pytest.mark.parametrize("change", [
    dict(logits=torch.zeros(2, 12, dtype=BF), y=torch.zeros(2, 12, dtype=BF)), dict(y=torch.zeros(2, 32, dtype=BF)),
    dict(logits=torch.zeros(2, 40)), dict(active=torch.zeros(1, **I32)), dict(pos=torch.zeros(3, dtype=torch.int64)),
    dict(penalties=torch.zeros(3, 2)), dict(penalties=torch.zeros(3, 3), first=None), dict(tokens=torch.zeros(3, 4, **I32)),
    dict(tokens=torch.zeros(2, 4, dtype=torch.int64)), dict(bias_of=None), dict(bias=torch.zeros(2, 32, dtype=BF)),
    dict(bias=torch.zeros(0, 40, dtype=BF)), dict(start=None), dict(mask=torch.zeros(3, 1, **I32)),
    dict(classes=None), dict(trans=torch.zeros(2, 5, **I32)), dict(trans=torch.zeros(3, 0, **I32)),
    dict(state=torch.zeros(3, 1, **I32)), dict(state=None), dict(plen=None), dict(mask=None),
    dict(classes=torch.zeros(39, **I32))])
def test_logits_refuses(change):
    from kernels.cuda_ext import ext

    a = dict(logits=torch.zeros(2, 40, dtype=BF), y=torch.zeros(2, 40, dtype=BF), active=torch.zeros(2, **I32),
             pos=torch.zeros(3, **I32), tokens=torch.zeros(3, 4, dtype=torch.int64), first=torch.zeros(3, **I32),
             plen=torch.zeros(3, **I32), penalties=torch.zeros(3, 3), bias=torch.zeros(2, 40, dtype=BF),
             bias_of=torch.zeros(3, **I32), mask=torch.zeros(3, 2, **I32), classes=torch.zeros(40, **I32),
             trans=torch.zeros(3, 5, **I32), start=torch.zeros(3, **I32), state=torch.zeros(3, 2, **I32))
    a.update(change)
    with pytest.raises(RuntimeError, match="dec_logits"):
        ext.dec_logits(*a.values())


def test_c_abi_refuses_without_launching():
    from kernels.cuda_ext import _lib as lib

    fake = 1 << 20  # never dereferenced
    def refused(name, *args):
        assert getattr(lib, name)(*args) != 0
        return lib.cohere_last_error().decode()

    ok = [0, fake, 2, fake, 512, fake, fake, fake, fake, fake, 3, 4, 2, 5, 1.0, 1, None, 0, fake, None]
    for at, value in ((1, None), (4, 511), (4, 504), (5, fake + 8), (7, fake + 4), (10, 0), (11, 5), (13, 0), (13, 1 << 25),
                      (15, 0), (15, 65), (15, 2), (18, None)):
        args = list(ok)
        args[at] = value
        assert "dec_attention_q4" in refused("cohere_dec_attention_q4", *args)
    assert lib.cohere_dec_attention_q4_splits(1, 8, 3, 100) == 1
    assert lib.cohere_dec_attention_q4_splits(64, 8, 8, 465) == 1
    assert 1 < lib.cohere_dec_attention_q4_splits(1, 8, 8, 65536) <= 64
    ok = [fake, 512, 2, fake, fake, fake, fake, fake, fake, 1, 3, 2, 5, None]
    for at, value in ((0, None), (1, 504), (1, 513), (2, -1), (5, fake + 2), (7, fake + 2), (9, 0), (12, 0)):
        args = list(ok)
        args[at] = value
        assert "dec_scatter_kv_q4" in refused("cohere_dec_scatter_kv_q4", *args)
    ok = [fake, 40, fake, 40, 2, 40, fake, fake, 3, fake, 4, fake, fake, fake, fake, 2, fake, fake, 3, fake, fake, 5, fake,
          fake, None]
    for at, value in ((0, fake + 2), (1, 39), (3, 44), (4, 70000), (5, 44), (8, 0), (9, None), (10, 0), (16, None),
                      (19, None), (22, None), (23, None)):
        args = list(ok)
        args[at] = value
        assert "dec_logits" in refused("cohere_dec_logits", *args), at


def test_grammar():
    from kernels.stream_decoder import Grammar

    classes = [0, 1, 2] * 13 + [0]
    trans = [[0, -1, 1], [-1, -1, -1]]
    g = Grammar(classes, trans)
    assert g.states == 2 and g.mask.shape == (2, 2) and g.mask.dtype == torch.int32
    for s in range(2):
        for v in range(40):
            assert (int(g.mask[s, v // 32]) >> (v % 32)) & 1 == (trans[s][classes[v]] >= 0)
        assert int(g.mask[s, 1]) & ~0xff == 0
    for c, t in (([], trans), (classes, []), ([3], trans), ([-1], trans), ([0], [[1]]), ([0], [[-2]]), ([[0]], trans)):
        with pytest.raises(ValueError):
            Grammar(c, t)


def test_check_rules():
    from kernels.stream_decoder import Grammar, Rules, StreamDecoder

    dec = object.__new__(StreamDecoder)
    dec.pen = dec.bias = dec.grammar = None
    dec.check_rules(None)
    dec.check_rules(Rules())
    for r in (Rules(frequency=0.1), Rules(bias=0), Rules(start=0), Rules(repetition=-1.0)):
        with pytest.raises(ValueError):
            dec.check_rules(r)
    dec.pen, dec.bias, dec.grammar = torch.zeros(1, 3), torch.zeros(2, 8), Grammar([0] * 8, [[0]])
    dec.check_rules(Rules(1.2, 0.1, -0.1, True, 1, 0))
    for r in (Rules(bias=2), Rules(start=1), Rules(start=-2), Rules(presence=float("nan"))):
        with pytest.raises(ValueError):
            dec.check_rules(r)


@pytest.mark.parametrize("numbers", [dict(repetition=1e-300), dict(repetition=1e300), dict(presence=-1e39),
                                     dict(frequency=3.5e38)])
def test_check_rules_in_fp32(numbers):
    """Penalties that fp32 holds as 0 or infinite."""
    from kernels.stream_decoder import Rules, StreamDecoder

    dec = object.__new__(StreamDecoder)
    dec.pen, dec.bias, dec.grammar = torch.zeros(1, 3), None, None
    dec.check_rules(Rules(1e-40, -3e38, 3e38))
    with pytest.raises(ValueError, match="penalties"):
        dec.check_rules(Rules(**numbers))
