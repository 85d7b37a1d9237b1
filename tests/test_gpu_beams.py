"""Beam search's selection on the GPU against a full sort in 64 bits, and a cache that runs on it."""

import math

import numpy as np
import pytest
import torch

from hackaton_amd import PagedCache, paged_append, paged_attention, select_beams
from tests.test_gpu_paged import banner, ints

pytestmark = pytest.mark.gpu

FP16, BF16, FP32 = torch.float16, torch.bfloat16, torch.float32
INF = math.inf


def reference(logits, scores, beams, count, ended=None, end=None):
    """(scores, rows, tokens) of a stable sort of all continuations, 64 bits, on the GPU."""
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    x = x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True)))
    if ended is not None:
        x = torch.where(ended[:, None], -INF, x)
        x[:, end] = torch.where(ended, 0.0, x[:, end])
    x = x + scores.double()[:, None]
    x = torch.where(torch.isnan(x), -INF, x).reshape(-1, beams * logits.shape[1])
    value, place = torch.sort(x, dim=1, descending=True, stable=True)
    value, place = value[:, :count], place[:, :count]
    first = torch.arange(x.shape[0], device=x.device)[:, None] * beams
    return value, first + place // logits.shape[1], place % logits.shape[1], x


def bound_of(vocab):
    """How far a score may be from the exact one before its last rounding: the sum of a row's exponentials
    in fp32. A lane adds at most 8 * ceil(cells / 4) of them, each addition off by 2^-24 of the sum; a
    term e^-d has an argument off by 3 d 2^-24 and an exponential by 2^-23 of it, and the terms' mean d,
    weighted by themselves, is at most ln(vocab) <= 12.5: 40 * 2^-24. Six more additions join the lanes."""
    return (8 * -(-vocab // 2048) + 48) * 2.0 ** -24


def check(logits, scores, beams, count=None, ended=None, end=None):
    """The selection is the sort's; two continuations of different rows whose scores are closer than twice
    the bound may change places (their difference is the two rows' sums')."""
    n = beams if count is None else count
    got = select_beams(logits, scores, beams, count, ended, end)
    again = select_beams(logits, scores, beams, count, ended, end)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    value, rows, tokens, every = reference(logits, scores, beams, n, ended, end)
    score, parents, picked = got
    assert score.dtype == FP32 and parents.dtype == picked.dtype == torch.int32
    assert score.shape == parents.shape == picked.shape == (logits.shape[0] // beams, n)
    vocab, limit = logits.shape[1], bound_of(logits.shape[1])
    place = (parents.long() % beams) * vocab + picked
    exact = torch.gather(every, 1, place)
    assert torch.equal(parents.long() // beams, torch.arange(score.shape[0], device="cuda")[:, None].expand_as(parents))
    off = (score.double() - exact).abs()
    assert (torch.nan_to_num(off, nan=0.0) <= limit + 2.0 ** -24 * exact.abs().clamp(max=3e38)).all()
    assert torch.equal(torch.isinf(score), torch.isinf(exact))
    same = (parents == rows) & (picked == tokens)
    if not same.all():  # near ties of different rows only
        assert (torch.nan_to_num((exact - value).abs(), nan=0.0)[~same] <= 2 * limit).all()
        order = place.sort(1).values
        assert (order[:, 1:] > order[:, :-1]).all()
    for a in range(n - 1):  # in one row: by logits, ties to the lower token
        one = parents[:, a] == parents[:, a + 1]
        x, y = (logits[parents[:, a + i].long(), picked[:, a + i].long()].double() for i in (0, 1))
        if ended is None:
            lives = torch.isfinite(exact[:, a + 1])
            assert ((x > y) | ((x == y) & (picked[:, a] < picked[:, a + 1])) | ~one | ~lives).all()
    return got


def draw(seed, rows, vocab, dtype, scale=2.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn(rows, vocab, generator=gen, device="cuda") * scale
    scores = -torch.rand(rows, generator=gen, device="cuda") * 3
    return logits.to(dtype), scores


VOCABS = [1, 2, 7, 8, 9, 63, 511, 512, 513, 1023, 4097, 32000]


@pytest.mark.parametrize("dtype", [FP16, BF16, FP32])
@pytest.mark.parametrize("vocab", VOCABS)
def test_sizes(vocab, dtype):
    for groups, beams, count in ((1, 1, 1), (3, 1, 5), (1, 4, 4), (5, 3, 7), (2, 8, 16), (1, 16, 64), (2, 64, 64)):
        banner("beams", vocab, dtype, groups, beams, count)
        check(*draw(vocab + beams, groups * beams, vocab, dtype), beams, min(count, beams * vocab))


@pytest.mark.parametrize("groups,beams,vocab,dtype,count", [
    (1, 4, 150001, BF16, 4), (3, 5, 100003, FP32, 10), (2, 64, 1 << 18, FP16, 64), (600, 4, 3001, FP16, 8),
    (1, 64, 65536, BF16, 64), (2500, 1, 777, FP32, 2), (1, 1, 1 << 18, BF16, 64), (70000, 1, 40, FP16, 1)])
def test_large_and_many(groups, beams, vocab, dtype, count):
    banner("beams", groups, beams, vocab, dtype, count)
    check(*draw(vocab, groups * beams, vocab, dtype), beams, count)


@pytest.mark.parametrize("count", [1, 4, 17, 64])
def test_ties(count):
    """Equal logits everywhere, in runs, and in rows of equal scores: the lowest row and token first."""
    banner("ties", count)
    zeros = torch.zeros(8, 3000, device="cuda")
    score = torch.zeros(8, device="cuda")
    for dtype in (FP16, BF16, FP32):
        got = check(zeros.to(dtype), score, 4, count)
        assert got[2].tolist() == [list(range(count))] * 2 and got[1].tolist() == [[0] * count, [4] * count]
        steps = (torch.arange(3000, device="cuda") // 700 % 3).expand(8, -1).contiguous().to(dtype)
        check(steps, score, 4, count)
        logits, _ = draw(count, 2, 5000, BF16)
        logits = logits.to(dtype).repeat_interleave(4, 0)  # a prompt's first step: its beams are alike
        check(logits, score, 4, count)
        first = torch.tensor([0.0, -INF, -INF, -INF] * 2, device="cuda")
        got = check(logits, first, 4, count)
        assert got[1].tolist() == [[0] * count, [4] * count]


@pytest.mark.parametrize("count", [2, 33, 64])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_where_the_best_ones_lie_together(count, dtype):
    """The best continuations in one cell, in one thread's numbers, in ascending or descending order."""
    banner("together", count, dtype)
    vocab, score = 20000, torch.tensor([-1.0, -0.5, 0.0], device="cuda")
    rise = torch.arange(vocab, device="cuda").float() / 256
    for row in (rise, -rise, (rise * 37) % 13):
        check(row.expand(3, -1).contiguous().to(dtype), score, 3, count)
    for period in (8, 32, 64, 512, 1024, 2048, 4096):
        logits, _ = draw(period, 3, vocab, FP32, 0.5)
        logits[1, period // 2::period] += 8
        check(logits.to(dtype), score, 3, count)
    logits, _ = draw(1, 3, vocab, FP32, 0.5)
    logits[2, 512 * 7:512 * 8] += 20
    check(logits.to(dtype), score, 3, count)


def test_not_finite():
    """-inf logits (tokens that are not allowed), whole rows of them, +inf, not-a-numbers, beams at -inf and
    at not a number: they count as -inf, and are chosen, lowest first, only where nothing else is left."""
    banner("not finite")
    logits, scores = draw(3, 12, 1000, FP32)
    logits[:, 5::7] = -INF
    logits[2], logits[3, 17], logits[4, 999] = -INF, INF, math.nan
    logits[6, :-1] = -INF
    logits[9, :998], logits[9, 999] = -INF, -INF
    scores[7], scores[8] = -INF, math.nan
    check(logits, scores, 12, 64)
    check(logits, scores, 4, 9)
    got = check(logits, scores, 1, 3)
    for row, tokens in ((2, [0, 1, 2]), (3, [0, 1, 2]), (4, [0, 1, 2]), (6, [0, 1, 2]), (7, [0, 1, 2]),
                        (8, [0, 1, 2]), (9, [998, 0, 1])):
        assert got[2][row].tolist() == tokens, row
    assert got[0][9].tolist() == [float(scores[9]), -INF, -INF]  # (the only token left has all the weight)
    check(logits.to(FP16), scores, 3, 20)
    top = torch.full((2, 50), 3e38, device="cuda")
    top[1, 7] = -3e38
    check(top, torch.tensor([0.0, 1.0], device="cuda"), 2, 64)


def test_ended_beams():
    banner("ended")
    logits, scores = draw(4, 40, 3000, BF16)
    ended = torch.zeros(40, dtype=torch.bool, device="cuda")
    ended[[1, 6, 7, 8, 9, 10, 20, 21, 22, 23, 39]] = True
    hidden = logits.clone()
    hidden[ended] = math.nan  # not read
    for end in (0, 2, 2999):
        for beams, count in ((4, 4), (4, 8), (10, 20), (1, 3), (40, 64)):
            a = check(logits, scores, beams, count, ended, end)
            b = select_beams(hidden, scores, beams, count, ended, end)
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    got = check(logits, scores, 4, 5, ended, 2)
    best = scores[20:24].sort(descending=True)
    assert torch.equal(got[0][5, :4], best.values)
    assert torch.equal(got[1][5, :4].long(), 20 + best.indices) and got[2][5, :4].tolist() == [2] * 4
    assert got[0][5, 4] == -INF and (got[1][5, 4], got[2][5, 4]) == (20, 0)
    check(logits, scores, 4, 4, torch.zeros_like(ended), 5)


@pytest.mark.parametrize("dtype", [FP16, FP32])
def test_rows_at_any_address(dtype):
    """Rows that lie apart, begin at any element, and run backwards in memory or across columns (copied)."""
    banner("strides", dtype)
    logits, scores = draw(5, 12, 2049, dtype)
    want = select_beams(logits, scores, 4, 8)
    for shift, width in ((1, 2060), (3, 2053), (7, 4096), (8, 2064)):
        held = torch.full((13 * width,), 50.0, dtype=dtype, device="cuda")
        view = held[shift:shift + 12 * width].view(12, width)[:, :2049]
        view.copy_(logits)
        assert all(torch.equal(a, b) for a, b in zip(select_beams(view, scores, 4, 8), want))
    assert all(torch.equal(a, b) for a, b in zip(select_beams(logits.t().contiguous().t(), scores, 4, 8), want))
    one = logits[:1].expand(4, -1)  # the first step's beams: one row, seen four times
    got = select_beams(one, scores[:4], 4, 8)
    assert all(torch.equal(a, b) for a, b in zip(got, select_beams(one.contiguous(), scores[:4], 4, 8)))
    every = torch.stack((scores, scores), 1)[:, 0]
    assert all(torch.equal(a, b) for a, b in zip(select_beams(logits, every, 4, 8), want))


def test_rows_past_32_bits():
    """Logits whose offsets pass 32 bits."""
    banner("beams past 32 bits")
    rows, width = 20, 1 << 28  # 10.7 GB of bf16
    held = torch.empty(rows, width, dtype=BF16, device="cuda")
    view = held[:, -9001:]
    logits, scores = draw(6, rows, 9001, BF16)
    view.copy_(logits)
    assert all(torch.equal(a, b) for a, b in zip(select_beams(view, scores, 4, 8),
                                                 select_beams(logits, scores, 4, 8)))
    del held, view
    torch.cuda.empty_cache()


def test_captured_and_at_once():
    """Two captured selections replayed over changing inputs, eager work between; several streams."""
    banner("captured beams")
    logits, scores = draw(7, 24, 40000, FP16)
    ended = torch.zeros(24, dtype=torch.bool, device="cuda")
    graphs = []
    for beams, count in ((4, 8), (8, 8)):
        select_beams(logits, scores, beams, count, ended, 3)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = select_beams(logits, scores, beams, count, ended, 3)
        graphs.append((graph, got, beams, count))
    for seed in range(4):
        x, y = draw(10 + seed, 24, 40000, FP16)
        logits.copy_(x)
        scores.copy_(y)
        ended.copy_(torch.arange(24, device="cuda") % 5 == seed)
        for graph, got, beams, count in graphs:
            want = check(x, y, beams, count, ended, 3)
            for _ in range(3):
                graph.replay()
                torch.cuda.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, want))
    streams, results = [torch.cuda.Stream() for _ in range(3)], []
    want = select_beams(logits, scores, 4)
    torch.cuda.synchronize()
    for _ in range(5):
        for stream in streams:
            with torch.cuda.stream(stream):
                results.append(select_beams(logits, scores, 4))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for got in results for a, b in zip(got, want))


def test_refusals():
    logits, scores = draw(8, 12, 100, FP16)
    ended = torch.zeros(12, dtype=torch.bool, device="cuda")
    for bad in ((logits.int(), scores, 4), (logits[0], scores, 4), (logits, scores, 5), (logits, scores, 0),
                (logits, scores[:11], 4), (logits, scores.half(), 4), (logits, scores.cpu(), 4),
                (logits, scores, 4, 0), (logits, scores, 4, -1), (logits, scores, 4, 4, ended),
                (logits, scores, 4, 4, ended[:11], 1), (logits, scores, 4, 4, ended.int(), 1),
                (logits, scores, 4, 4, ended.cpu(), 1)):
        with pytest.raises(ValueError):
            select_beams(*bad)
    for bad in ((logits, scores, 4, 65), (logits, scores, 4, 4, ended, 100), (logits, scores, 4, 4, ended, -1),
                (logits[:, :2], scores, 4, 9), (logits[:, :0], scores, 4)):
        with pytest.raises(RuntimeError):
            select_beams(*bad)
    wide = torch.zeros(65, 10, device="cuda")
    with pytest.raises(RuntimeError, match="beams"):
        select_beams(wide, torch.zeros(65, device="cuda"), 65)
    with pytest.raises(RuntimeError, match="vocab"):
        select_beams(torch.zeros(1, (1 << 18) + 1, device="cuda"), torch.zeros(1, device="cuda"), 1)
    with pytest.raises(RuntimeError, match="no backward"):
        select_beams(logits.float().requires_grad_(), scores, 4)
    with pytest.raises(RuntimeError, match="no backward"):
        select_beams(logits, scores.clone().requires_grad_(), 4)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(logits.float(), torch.ones(12, 100, device="cuda"))
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            select_beams(dual, scores, 4)
    # (what passes 32 bits is refused too, not cut to its low bits)
    with pytest.raises(RuntimeError, match="end_token"):
        select_beams(logits, scores, 4, 4, ended, 1 + (1 << 32))
    with pytest.raises(ValueError, match="count"):
        select_beams(logits, scores, 4, 4 + (1 << 32))
    got = select_beams(logits[:0], scores[:0], 4)
    assert [x.shape for x in got] == [(0, 4)] * 3
    cache = PagedCache(1, 8, 16, 1, 4, 64)
    with pytest.raises(ValueError):
        cache.select(logits, scores, 4)


@pytest.mark.parametrize("dtype", [FP16, torch.float8_e4m3fn])
def test_a_beam_search(dtype):
    """Two prompts of three beams through a cache: its answers are those of a search that keeps every beam's
    rows as a list, attends to them densely and sorts all continuations."""
    banner("a beam search", dtype)
    heads, kv_heads, beams, prompts, vocab, dim = 4, 2, 3, 2, 50, 128
    slots, gen = prompts * beams, torch.Generator().manual_seed(5)
    embed = torch.randn(vocab, (heads + 2 * kv_heads) * dim, generator=gen).to(FP16).cuda()
    out_proj = (torch.randn(heads * dim, vocab, generator=gen) * 0.2).cuda()
    cache = PagedCache(1, 60, 16, kv_heads, slots, 128, dtype)
    cos, sin = torch.ones(1, 128, dim, device="cuda"), torch.zeros(1, 128, dim, device="cuda")

    def logits_of(tokens, q_lengths):
        """Next-token logits of every slot after its new tokens (embeddings as projections)."""
        plan = cache.step(q_lengths, len(tokens), heads)
        qkv = embed[tokens].split([heads * dim, kv_heads * dim, kv_heads * dim], 1)
        keys, values = cache.keys(0), cache.values(0)
        query = paged_append(*qkv, cos, sin, keys, values, plan, FP16)
        attn = paged_attention(query, keys, values, plan, dim ** -0.5).float()
        return attn @ out_proj

    prompt = [torch.randint(0, vocab, (n,), generator=gen).tolist() for n in (20, 33)]
    x = logits_of(torch.tensor(prompt[0] + prompt[1], device="cuda"), [20, 0, 0, 33, 0, 0])
    cache.remap({1: 0, 2: 0, 4: 3, 5: 3})
    logits = torch.cat((x[19].expand(beams, -1), x[52].expand(beams, -1)))
    scores = torch.tensor([0.0, -INF, -INF] * prompts, device="cuda")
    ended = torch.zeros(slots, dtype=torch.bool, device="cuda")
    history = [list(prompt[s // beams]) for s in range(slots)]
    for turn in range(12):
        value, rows, tokens, _ = reference(logits, scores, beams, beams, ended, 7)
        scores, parents, picked = cache.select(logits, scores, beams, ended, 7)
        assert torch.equal(parents.long(), rows.flatten()) and torch.equal(picked.long(), tokens.flatten())
        assert (scores.double() - value.flatten()).abs().max() <= 2.0 ** -18
        history = [history[p] + [t] for p, t in zip(parents.tolist(), picked.tolist())]
        ended = ended[parents.long()] | (picked == 7)
        logits = logits_of(picked.long(), ints([1] * slots))
        assert cache.lengths.tolist() == [len(h) for h in history]
        # the cache holds each beam's own tokens: the same logits as from a cache that is given them at once
        fresh = PagedCache(1, 60, 16, kv_heads, slots, 128, dtype)
        cache, held = fresh, cache
        again = logits_of(torch.tensor(sum(history, []), device="cuda"), [len(h) for h in history])
        cache = held
        last = np.cumsum([len(h) for h in history]) - 1
        assert (again[torch.from_numpy(last).cuda()] - logits).abs().max() <= 0.05
    cache.check()
