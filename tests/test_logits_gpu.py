"""Rules on a step's logits (penalties for repeated tokens, biases, grammar masks) against the definition in 64 bits."""

from __future__ import annotations

import pytest
import torch

from q4_helpers import BF, assert_rounded, logits64

pytestmark = pytest.mark.gpu


def _rules(seed, rows, V, OUT, B=3, M=5, C=4):
    g = torch.Generator().manual_seed(seed)
    S = rows + 2
    pos = torch.randint(0, OUT, (S,), generator=g).to(torch.int32)
    plen = torch.randint(0, 4, (S,), generator=g).to(torch.int32)
    tokens = torch.randint(0, V, (3, S, OUT), generator=g).amin(0)
    pen = torch.rand(S, 3, generator=g) * torch.tensor([1.0, 2.0, 0.5]) + torch.tensor([0.8, -0.5, -0.1])
    pen[::3] = torch.tensor([1.0, 0.0, 0.0])
    mask = torch.randint(-2 ** 31, 2 ** 31, (M, (V + 31) // 32), generator=g).to(torch.int32)
    mask[0] = 0
    return dict(logits=(4 * torch.randn(rows, V, generator=g)).to(BF),
                active=torch.randperm(S, generator=g)[:rows].to(torch.int32), pos=pos, tokens=tokens,
                first=torch.randint(-2, OUT, (S,), generator=g).to(torch.int32), plen=plen, pen=pen,
                bias=torch.randn(B, V, generator=g).to(BF) if B else None,
                bias_of=torch.randint(-2, B + 1, (S,), generator=g).to(torch.int32) if B else None,
                mask=mask, classes=torch.randint(0, C, (V,), generator=g).to(torch.int32),
                trans=torch.randint(-1, M + 1, (M, C), generator=g).to(torch.int32),
                start=torch.randint(-1, M + 1, (S,), generator=g).to(torch.int32),
                state=torch.randint(-1, M + 1, (S, 2), generator=g).to(torch.int32))


def _run(a, y=None):
    from kernels.cuda_ext import ext

    d = {k: None if v is None else v.cuda() for k, v in a.items()}
    y = torch.full_like(d["logits"], float("nan")) if y is None else d["logits"]
    ext.dec_logits(d["logits"], y, d["active"], d["pos"], d["tokens"], d["first"], d["plen"], d["pen"], d["bias"],
                   d["bias_of"], d["mask"], d["classes"], d["trans"], d["start"], d["state"])
    torch.cuda.synchronize()
    return y.cpu(), None if d["state"] is None else d["state"].cpu()


def _check(a, **kw):
    want, slack, state = logits64(**a)
    y, got_state = _run(a, **kw)
    assert_rounded(y, want, slack)
    if state is not None:
        assert torch.equal(got_state, state)
    return y


@pytest.mark.parametrize("rows,V,OUT", [(1, 8, 1), (3, 40, 2), (5, 2048, 70), (2, 4104, 300), (4, 16384, 466),
                                        (2, 100008, 1200), (61, 69640, 90)])
def test_rules(gpu, rows, V, OUT):
    print(f"dec_logits rows={rows} V={V} OUT={OUT}", flush=True)
    for seed in range(3 if rows < 10 else 1):
        _check(_rules(seed + V, rows, V, OUT))


@pytest.mark.parametrize("off", [("pen",), ("bias", "bias_of"), ("classes", "trans", "state", "plen"),
                                 ("mask", "classes", "trans", "start", "state"),
                                 ("pen", "tokens", "first", "plen", "mask", "classes", "trans", "start", "state"),
                                 ("pen", "tokens", "first", "plen", "bias", "bias_of", "mask", "classes", "trans", "start",
                                  "state")])
def test_rules_absent(gpu, off):
    print(f"dec_logits without {off}", flush=True)
    _check({**_rules(7, 4, 264, 30), **{k: None for k in off}})


def test_in_place(gpu):
    _check(_rules(2, 3, 5000, 50), y="logits")


def test_repeats_and_foreign_tokens(gpu):
    """One token held many times, tokens outside the vocabulary, a history of one, histories that are empty, rows whose slot
    is out of range (copied), a position beyond the tokens."""
    a = _rules(4, 6, 4096 + 64, 3000)
    a["tokens"][:, ::2] = 4097
    a["tokens"][:, 1::4] = torch.tensor([-1, 4160, 2 ** 32 + 5, -2 ** 40]).repeat_interleave(188)[:750]
    s = a["active"].long()
    a["first"][s[0]], a["pos"][s[0]] = 17, 17
    a["first"][s[1]], a["pos"][s[1]] = 18, 17
    a["pos"][s[2]], a["first"][s[2]] = 5000, 0
    a["first"][s[5]], a["pos"][s[5]] = 0, 2999
    a["pen"][:] = torch.tensor([1.3, 0.25, 0.01])
    a["active"][3], a["active"][4] = -1, 8
    _check(a)


def test_more_repeats_than_16_bits(gpu):
    """One token 70000 times, another 65536 times, a third once."""
    a = _rules(3, 1, 4104, 135537)
    a["tokens"][:, :70000], a["tokens"][:, 70000:135536], a["tokens"][:, 135536] = 4100, 7, 9
    a["first"][:], a["pos"][:] = 0, 135536
    a["pen"][:] = torch.tensor([1.1, 0.5, 0.001])
    _check({**a, **{k: None for k in ("bias", "bias_of", "mask", "classes", "trans", "start", "state", "plen")}})


def test_special_logits(gpu):
    """Zeros, infinities and the type's lowest value among penalised, biased and masked tokens; a row left empty."""
    a = _rules(6, 2, 64, 64, B=1, M=2, C=1)
    low = torch.finfo(BF).min
    a["logits"][:, :8] = torch.tensor([0.0, -0.0, float("inf"), float("-inf"), low, -low, 1e-40, -1e-40], dtype=BF)
    a["tokens"][:] = torch.arange(64) % 12
    a["first"][:], a["pos"][:], a["bias_of"][:] = 0, 63, 0
    a["bias"][0, :8] = torch.tensor([0, 0, 1, -1, 0, 0, 0, 0], dtype=BF)
    a["pen"][:] = torch.tensor([2.0, 0.0, 0.0])
    a["start"][:], a["plen"][:] = 1, 100
    a["mask"][1] = torch.tensor([-2, -1])
    # the lowest value doubled is below bf16's range: -inf, as the rounding of the product gives
    want, slack, _ = logits64(**a)
    want[want < -3.39e38] = float("-inf")
    y, _ = _run(a)
    assert_rounded(y, want, slack)
    a["start"][:] = 0
    assert (_run(a)[0] == float("-inf")).all()


@pytest.mark.parametrize("rep", [0.5, 0.75, 1e-39, 2.0 ** -149, 2.0 ** -126, 1e-20, 1e20, 2.0 ** 126, 3e38])
def test_quotients_at_the_ends_of_the_range(gpu, rep):
    """A repetition penalty over the whole range of fp32, logits over bf16's: quotients beyond it are infinite (never
    NaN), those below it zero."""
    print(f"dec_logits rep={rep}", flush=True)
    a = {**_rules(6, 1, 64, 64, B=0), **{k: None for k in ("mask", "classes", "trans", "start", "state", "plen")}}
    big = torch.finfo(BF).max
    a["logits"][0, :16] = torch.tensor([big, 1.0, 2.0 ** -20, 1e-30, 1e-38, 1e-40, 1e30, 3.0, -big, -1.0, -1e-30, -1e-40,
                                        0.0, -0.0, float("inf"), float("-inf")], dtype=BF)
    a["tokens"][:] = torch.arange(64)
    a["first"][:], a["pos"][:] = 0, 63
    a["pen"][:] = torch.tensor([rep, 0.0, 0.0])
    want, slack, _ = logits64(**a)
    # halfway from bf16's largest value to 2^128, and above it: infinite, in fp32 already or by the last rounding
    over = want.abs() >= 2.0 ** 128 - 2.0 ** 119
    want[over] = want[over].sign() * float("inf")
    slack[over] = 0
    assert_rounded(_run(a)[0], want, slack)


def test_nan_stays_where_it_is(gpu):
    a = _rules(6, 1, 64, 8, B=0, M=1)
    a["logits"][0, 5], a["start"][:], a["plen"][:] = float("nan"), 5, 100
    y, _ = _run(a)
    assert y.isnan().sum() == 1 and y[0, 5].isnan()
    a["start"][:] = 0
    assert (_run(a)[0] == float("-inf")).all()


def test_grammar_follows_the_tokens(gpu):
    """Greedy steps under a grammar: rules, then the pick; every token is one that the grammar allows, the states are the
    automaton's, and a state that allows nothing ends the row. Captured, replayed per step, with eager work between."""
    from kernels.cuda_ext import ext

    g = torch.Generator().manual_seed(3)
    V, S, T, eos = 64, 4, 24, 63
    classes = torch.arange(V, dtype=torch.int32) % 3
    trans = torch.tensor([[1, -1, -1], [-1, 2, -1], [0, -1, 3], [-1, -1, -1]], dtype=torch.int32)
    allowed = (trans >= 0)[:, classes.long()]
    mask = torch.zeros(4, 2, dtype=torch.int64)
    for v in range(V):
        mask[:, v // 32] += allowed[:, v].long() << (v % 32)
    mask = torch.where(mask >= 2 ** 31, mask - 2 ** 32, mask).to(torch.int32).cuda()
    i32 = (lambda v: torch.tensor(v, dtype=torch.int32).cuda())
    active, pos, plen, limit = i32([2, 0, 1]), i32([0] * S), i32([1, 2, 3, 1]), i32([20] * S)
    start, state = i32([0, 2, -1, -1]), torch.full((S, 2), -7, dtype=torch.int32).cuda()
    tok, forced = torch.zeros(S, dtype=torch.long).cuda(), torch.full((S, 4), 11, dtype=torch.long).cuda()
    out, fin = torch.zeros(S, T, dtype=torch.long).cuda(), torch.zeros(S, dtype=torch.uint8).cuda()
    logits, y = torch.zeros(3, V, dtype=BF).cuda(), torch.zeros(3, V, dtype=BF).cuda()

    def step():
        ext.dec_logits(logits, y, active, pos, out, None, plen, None, None, None, mask, classes_d, trans_d, start, state)
        ext.dec_pick(y, active, S, tok, pos, fin, forced, plen, limit, out, 0, eos)

    classes_d, trans_d = classes.cuda(), trans.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            step()
        for i in range(12):
            logits.copy_(torch.randn(3, V, generator=g))
            graph.replay()
            side.synchronize()
    out, pos, fin = out.cpu(), pos.cpu(), fin.cpu()
    for s, st in ((0, 0), (1, 2), (2, -1)):
        for at in range(int(plen[s]), int(pos[s]) + 1):
            t = int(out[s, at])
            if st < 0:
                continue
            if not allowed[st].any():
                assert t == eos and at == int(pos[s]) and fin[s]
                break
            assert allowed[st, t], (s, at, st, t)
            st = int(trans[st, classes[t]])
    assert int(pos[2]) == 12 or fin[2]  # free of the grammar


@pytest.mark.parametrize("embed", [False, True])
def test_pick_from_nothing_ends_the_row(gpu, embed):
    """A row of nothing but -inf (or NaN) picks the end token; the others pick as ever."""
    from kernels.cuda_ext import ext

    V, S = 40, 3
    logits = torch.randn(3, V).to(BF)
    logits[0], logits[2] = float("-inf"), float("nan")
    i32 = (lambda v: torch.tensor(v, dtype=torch.int32).cuda())
    tok, pos, fin = torch.zeros(S + 1, dtype=torch.long).cuda(), i32([0] * 4), torch.zeros(S + 1, dtype=torch.uint8).cuda()
    forced, out = torch.zeros(S + 1, 2, dtype=torch.long).cuda(), torch.zeros(S + 1, 9, dtype=torch.long).cuda()
    a = (logits.cuda(), i32([0, 1, 2]), S, tok, pos, fin, forced, i32([1] * 4), i32([8] * 4), out, 0, 7)
    if embed:
        w = torch.ones(64, dtype=BF).cuda()
        x, h = (torch.zeros(3, 64, dtype=BF).cuda() for _ in range(2))
        ext.dec_pick_embed(*a, torch.randn(V, 64).to(BF).cuda(), torch.randn(9, 64).to(BF).cuda(), w, w, 1e-5, w, w, 1e-5,
                           x, h)
    else:
        ext.dec_pick(*a)
    assert out[:3, 1].tolist() == [7, int(logits[1].float().argmax()), 7]
    assert fin[:3].tolist() == [1, int(logits[1].float().argmax() == 7), 1]
