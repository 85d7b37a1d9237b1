"""The paged cache at the edges of its sizes: work lists of many and of long sequences, calls that are
refused or cut, and what they leave unchanged."""

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from hackaton_amd import (PagedCache, compact_pages, paged_append, paged_attention, paged_plan,
                          remap_pages)
from hackaton_amd._lib import check, lib
from tests import paged_oracle as orc
from tests.paged_oracle import DIM, SCALE
from tests.test_gpu_paged import BF16, FP16, attend, banner, check_attention, ints

pytestmark = pytest.mark.gpu

FEW, MANY, PAD, NONE = range(4)  # kinds of items


def places_of(plan):
    """Where the counts, the items and the merge records of a plan whose table rows pass 1024 keys lie."""
    n = plan.n_tokens
    counts = -(-(plan.n_seqs + 1) // 4) * 4 + 2 * (-(-n // 4) * 4)
    tiles = min(plan.n_seqs, n) + n * (plan.heads // plan.kv_heads) // 128
    max_items = tiles * plan.kv_heads + 512 + 256 + -(-n // 64)
    return counts, counts + 4, counts + 4 + 12 * max_items


def lists_of(plan):
    """(items (n, 12), merge records (n, 8)) of such a plan."""
    words, (counts, items, merges) = plan.words.cpu().numpy(), places_of(plan)
    n_items, n_merges = words[counts], words[counts + 1]
    assert 0 <= n_items <= (merges - items) // 12 and 0 <= n_merges <= (words.size - merges) // 8
    return (words[items:items + 12 * n_items].reshape(-1, 12),
            words[merges:merges + 8 * n_merges].reshape(-1, 8))


def check_lists(plan, q, kv):
    """Every row of every key/value head: its keys in parts that join without a gap, each part with
    workspace rows of its own, and a merge record wherever there is more than one. Returns how many
    parts the split tiles of both kinds have, by kind."""
    q, kv = np.asarray(q, dtype=np.int64), np.asarray(kv, dtype=np.int64)
    group, hkv = plan.heads // plan.kv_heads, plan.kv_heads
    rows_of, cu = q * group, np.concatenate(([0], np.cumsum(q)))
    items, merges = lists_of(plan)
    items = items.astype(np.int64)
    kind = items[:, 3] >> 16
    pads = items[kind == PAD]
    assert (pads[:, 5] - pads[:, 4]).sum() == plan.n_tokens - cu[-1]
    items = items[(kind == FEW) | (kind == MANY)]
    token0, seq, pos0, head, row, end, key, key_end, part_row = items[:, :9].T
    kind, head = head >> 16, head & 0xffff
    rows = rows_of[seq]
    assert (token0 == cu[seq]).all() and (pos0 == (kv - q)[seq]).all() and (head < hkv).all()
    assert ((kind == FEW) == (rows <= 32)).all()
    assert (row % 128 == 0).all() and (end == np.minimum(row + 128, rows)).all()
    keys = np.maximum(pos0 + (end - 1) // group + 1, 0)
    # parts in order of their keys, tile after tile
    order = np.lexsort((key, row, head, seq))
    tile = np.stack((seq, head, row), 1)[order]
    first = np.concatenate(([True], (tile[1:] != tile[:-1]).any(1)))
    last = np.concatenate((first[1:], [True]))
    tiles = np.where(rows_of == 0, 0, np.where(rows_of <= 32, 1, -(-rows_of // 128)))
    assert first.sum() == tiles.sum() * hkv
    key, key_end, part_row, count = key[order], key_end[order], part_row[order], (end - row)[order]
    assert (key[first] == 0).all() and (key_end[last] == keys[order][last]).all()
    assert (key[1:] == key_end[:-1])[~first[1:]].all() and (key % 64 == 0).all()
    parts = np.diff(np.append(np.flatnonzero(first), first.size))
    split = np.repeat(parts > 1, parts)
    assert ((part_row >= 0) == split).all()
    places = np.sort(np.concatenate([part_row[split][:, None], (part_row + count)[split][:, None]], 1), 0)
    assert (places[1:, 0] >= places[:-1, 1]).all()
    assert not split.any() or places[-1, 1] <= plan.workspace_bytes // (4 * (DIM + 2))
    # the merge records' rows are the split tiles' rows, and read the parts of theirs
    want = {}
    for t in np.flatnonzero(first & split):
        n = int(parts[np.searchsorted(np.flatnonzero(first), t)])
        stride = int(part_row[t + 1] - part_row[t])
        assert (np.diff(part_row[t:t + n]) == stride).all()
        for i in range(int(count[t])):
            s, h, r = (int(x) for x in tile[t])
            want[int(cu[s]), h, r + i] = (int(part_row[t]) + i, stride, n)
    got = {}
    for token, h, r, n, place, stride, n_parts, _ in merges.tolist():
        for i in range(n if n_parts > 1 else 0):
            assert (token, h, r + i) not in got
            got[token, h, r + i] = (place + i, stride, n_parts)
    assert got == want
    of = kind[order][first]
    return parts[of == FEW], parts[of == MANY]


def long_plan(q, kv, heads, kv_heads, page_size=256):
    """The plan of a step whose pages nothing reads."""
    table = torch.zeros(len(q), -(-max(kv) // page_size), dtype=torch.int32, device="cuda")
    plan = paged_plan(table, ints(q), ints(kv), sum(q), heads, kv_heads, page_size)
    torch.cuda.synchronize()
    return plan


@pytest.mark.parametrize("n_seqs,q,kv,heads,kv_heads", [
    (4096, 1, 600064, 12, 2), (4096, 1, 600064, 1, 1), (2049, 1, 1048575, 12, 2),
    (4096, 512, 32768, 12, 2), (4096, 183, 65336, 28, 4)])
def test_lists_of_many_long_sequences(n_seqs, q, kv, heads, kv_heads):
    """Steps whose keys sum to more than 2^31: the shares follow the sum, so the lists have room."""
    banner("many long sequences", n_seqs, q, kv, heads, kv_heads)
    plan = long_plan([q] * n_seqs, [kv] * n_seqs, heads, kv_heads)
    few, many = check_lists(plan, [q] * n_seqs, [kv] * n_seqs)
    assert (few == 1).all() and (many == 1).all()  # (more tiles than parts: nothing to split)


@pytest.mark.parametrize("q,kv,heads,kv_heads", [
    (1 << 20, 1 << 20, 32, 8), (1 << 20, (1 << 20) + 2, 32, 8), (1 << 20, (1 << 20) + 256, 32, 8),
    (1 << 20, 1 << 20, 28, 4), (1 << 19, 1 << 22, 32, 8), (1 << 20, (1 << 30) - 256, 12, 2)])
def test_lists_of_long_prompts(q, kv, heads, kv_heads):
    """Prompts whose share of keys passes 2^31, 2^32 and further: none of their ranges is split."""
    banner("long prompts", q, kv, heads, kv_heads)
    few, many = check_lists(long_plan([q, 1], [kv, 700000], heads, kv_heads), [q, 1], [kv, 700000])
    assert (many == 1).all() and (few > 8).all()


def test_many_forks_of_a_long_prompt():
    """4096 single tokens over 600,064 keys each, all of which are the 256 rows of one page: the weights
    repeat, so every row equals the attention over the page. The bound adds the worst case of the fp32
    sums, a quarter of the keys (one wave's) times half a step of 2^-23, in the sum and the output."""
    banner("many forks of a long prompt")
    n, ps, kv = 4096, 256, 600064
    gen = torch.Generator().manual_seed(0)
    query = torch.randn(n, 1, DIM, generator=gen).to(FP16)
    k, v = (torch.randn(1, 1, ps, DIM, generator=gen).to(FP16) for _ in range(2))
    table = torch.zeros(n, kv // ps, dtype=torch.int32, device="cuda")
    plan = paged_plan(table, ints([1] * n), ints([kv] * n), n, 1, 1, ps)
    out = paged_attention(query.cuda(), k.cuda(), v.cuda(), plan, SCALE).cpu().double()
    weights = torch.softmax(query[:, 0].double() @ k[0, 0].double().T * SCALE, 1)
    want, size = weights @ v[0, 0].double(), weights @ v[0, 0].double().abs()
    bound = orc.attention_bound(want, size, FP16) + 2 * kv / 4 * 2.0 ** -24 * size
    assert float(want.abs().max(1).values.min()) > float(bound.max())  # (an unwritten row would show)
    assert ((out - want).abs() <= bound).all()


@pytest.mark.parametrize("n_seqs", [256, 257, 1024, 1025, 4096])
def test_split_ranges_among_many_sequences(n_seqs):
    """A few long answers and prompts between many short sequences, at the borders of the planning
    threads' shares: both kinds of tiles are split, whatever the number of sequences per thread."""
    rng = np.random.default_rng(n_seqs)
    kv = rng.integers(0, 12, n_seqs)
    q = np.minimum(rng.integers(0, 3, n_seqs), kv)
    for at, new, total in ((0, 1, 9000), (3, 40, 1500), (4, 2, 700), (15, 90, 2500), (16, 1, 1200),
                           (63, 1, 3000), (64, 33, 1030), (255, 5, 4000), (n_seqs - 1, 70, 2000)):
        q[at], kv[at] = new, total
    q, kv = q.tolist(), kv.tolist()
    for heads, kv_heads, dtype in ((2, 1, FP16), (2, 2, BF16)):
        _, plan = check_attention(q, kv, heads, kv_heads, dtype, 16, padding=3)
        few, many = check_lists(plan, q, kv)
        assert (few > 1).any() and (many > 1).any() and (few > 8).any()


def test_merge_records_of_parts_in_one_place_are_skipped():
    """Records whose parts do not lie apart, of any number: they name no parts of a sequence, so their
    rows are left out; the others come out as before."""
    banner("merge records of parts in one place")
    heads, kv_heads, ps, q, kv = 4, 2, 16, [20, 1], [3000, 4000]
    query, k, v, table = (x.cuda() for x in orc.paged_case(14, q, kv, heads, kv_heads, FP16, ps))
    n, group, stride = sum(q), heads // kv_heads, kv_heads * ps * DIM
    plan = paged_plan(table, q, kv, n, heads, kv_heads, ps)
    good = plan.words.cpu()
    records = lists_of(plan)[1]
    ws = torch.zeros(plan.workspace_bytes, dtype=torch.uint8, device="cuda")

    def run():
        out = torch.full((n, heads, DIM), 7.0, dtype=FP16, device="cuda")
        check(lib().va_paged_attention(
            plan._step, query.data_ptr(), k.data_ptr(), v.data_ptr(), stride, stride, k.shape[0], DIM,
            SCALE, 0, out.data_ptr(), ws.data_ptr(), ws.numel(),
            torch.cuda.current_stream().cuda_stream), "va_paged_attention")
        torch.cuda.synchronize()
        return out

    whole = run()
    assert (whole != 7).all()
    for i in (0, len(records) - 1):  # a record of eight rows, one of the single token
        token0, head, row, rows, _, step, parts = records[i, :7].tolist()
        at = places_of(plan)[2] + 8 * i
        assert good[at:at + 7].tolist() == records[i, :7].tolist() and parts > 1 and step >= rows
        skipped = torch.zeros_like(whole, dtype=torch.bool)
        for r in range(row, row + rows):
            skipped[token0 + r // group, head * group + r % group] = True
        for bad, many in ((0, parts), (0, 9), (0, (1 << 31) - 1), (0, (1 << 31) - 64), (rows - 1, parts)):
            words = good.clone()
            words[at + 5], words[at + 6] = bad, many
            plan.words.copy_(words)
            out = run()
            assert torch.equal(out[~skipped], whole[~skipped]) and (out[skipped] == 7).all(), (i, bad, many)
    plan.words.copy_(good)
    assert torch.equal(run(), whole)


def state_of(cache):
    return [x.clone() for x in (cache.table, cache.lengths, cache.refs)]


def same_state(cache, kept):
    return all(torch.equal(a, b) for a, b in zip(kept, (cache.table, cache.lengths, cache.refs)))


def test_a_refused_step_changes_nothing():
    banner("refused steps")
    cache = PagedCache(1, 8, 16, 2, 2, 64)
    cache.step([5, 20], 25, 4)
    kept = state_of(cache)
    for q, n, heads in (([1, 1], 2, 5), (ints([1, 1]), 2, 0), (ints([1, 1]), -1, 4), ([1, 1], 1 << 30, 4),
                        (ints([1, 1]), 1 << 40, 4)):
        with pytest.raises(RuntimeError):
            cache.step(q, n, heads)
        assert same_state(cache, kept)
    wide = PagedCache(1, 8, 16, 2, 5000, 64)
    kept = state_of(wide)
    with pytest.raises(RuntimeError, match="4096"):
        wide.step(ints([1] * 5000), 5000, 4)
    assert same_state(wide, kept)
    assert cache.step([1, 1], 2, 4).positions.tolist() == [5, 20]
    cache.check()


@pytest.mark.parametrize("slots,seed", [(1, 0), (3, 1), (1000, 2), (1025, 3), (4096, 4)])
def test_a_step_of_more_tokens_than_rows_changes_nothing(slots, seed):
    """Device lengths that sum to the rows, to one more and past 32 bits; eagerly and replayed."""
    banner("more tokens than rows", slots)
    rng = np.random.default_rng(seed)
    n = 2 * slots
    cache = PagedCache(1, 5 * slots, 16, 1, slots, 64)
    fits = rng.multinomial(n, np.ones(slots) / slots).clip(max=30)
    fits[int(rng.integers(slots))] += n - fits.sum()
    cache.step(ints(fits.tolist()), n, 1)
    assert cache.lengths.tolist() == fits.tolist()
    cache.check()
    q = ints(fits.tolist())
    cache.remap(None, torch.zeros_like(q))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        plan = cache.step(q, n, 1)
    one_more = fits.copy()
    one_more[-1] += 1
    negative = np.where(np.arange(slots) % 2 == 0, fits, -fits - 1)
    over = (one_more, np.full(slots, (1 << 31) - 1), np.full(slots, n + 1))
    for given in (fits, *over, negative, *over, fits * 0):
        kept, want = state_of(cache), np.maximum(given, 0)
        q.copy_(ints(given.tolist()))
        graph.replay()
        torch.cuda.synchronize()
        if want.sum() <= n:
            assert cache.lengths.tolist() == (kept[1].cpu().numpy() + want).tolist()
            assert plan.sequences.tolist() == np.repeat(np.arange(slots), want).tolist() + \
                [-1] * (n - int(want.sum()))
            cache.check()
            continue
        assert same_state(cache, kept) and set(plan.sequences.tolist()) == {-1}
        eager = cache.step(q, n, 1)
        assert same_state(cache, kept) and set(eager.sequences.tolist()) == {-1}
        lacking = min(int(want.sum()) - n, (1 << 31) - 1)
        with pytest.raises(RuntimeError, match=f"lacked {lacking} rows"):
            cache.check()
        cache.check()


@pytest.mark.parametrize("slots", [1, 1024, 1025, 3000])
def test_a_pool_without_pages(slots):
    """Nothing to hand out: a shortfall and the state as it was, on both sides of the one-work-group
    path; no shortfall where nothing is asked for."""
    banner("a pool without pages", slots)
    pages = torch.zeros(1, 2, 0, 1, 16, DIM, dtype=FP16, device="cuda")
    table = torch.full((slots, 3), -1, dtype=torch.int32, device="cuda")
    lengths, none = torch.zeros_like(table[:, 0]), ints([])
    out = remap_pages(pages, table, lengths, none, None, lengths + 20)
    assert int(out[3]) == 2 * slots
    assert torch.equal(out[0], table) and torch.equal(out[1], lengths) and out[2].numel() == 0
    out = remap_pages(pages, table, lengths, none)
    assert int(out[3]) == 0 and torch.equal(out[0], table) and torch.equal(out[1], lengths)
    assert int(compact_pages(pages, table, lengths, none)[2]) == 0


def test_tensors_that_ask_for_derivatives_are_refused():
    """Every floating tensor of every call: requires_grad while gradients are on, tangents always."""
    banner("derivatives")
    q, kv, heads, kv_heads, ps = [1, 2], [40, 33], 4, 2, 16
    query, k, v, table = (x.cuda() for x in orc.paged_case(1, q, kv, heads, kv_heads, FP16, ps))
    plan = paged_plan(table, q, kv, 3, heads, kv_heads, ps)
    rows = [torch.zeros(3, h * DIM, dtype=FP16, device="cuda") for h in (heads, kv_heads, kv_heads)]
    cos = torch.ones(1, 50, DIM, device="cuda")
    pages = torch.zeros(1, 2, 4, kv_heads, ps, DIM, dtype=FP16, device="cuda")
    state = [ints([[0, 1]]), ints([20]), ints([1, 1, 0, 0])]

    def calls():
        yield lambda *x: paged_attention(*x, plan, SCALE), [query, k, v]
        yield lambda *x: paged_append(*x, plan), [*rows, cos, cos.clone(), k, v]
        yield lambda x: remap_pages(x, *state), [pages]
        yield lambda x: compact_pages(x, *state), [pages]

    for call, tensors in calls():
        for i, x in enumerate(tensors):
            if not (x.dtype == torch.float32):  # (the rotary tables are constants, as in qkv_rotate)
                bad = [t.clone().requires_grad_() if j == i else t for j, t in enumerate(tensors)]
                with pytest.raises(RuntimeError, match="no backward"):
                    call(*bad)
                with torch.no_grad():
                    call(*bad)
            with torch.no_grad(), forward_ad.dual_level():
                bad = [forward_ad.make_dual(t, t) if j == i else t for j, t in enumerate(tensors)]
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*bad)
                call(*tensors)


def test_wide_lengths_past_their_bounds_are_cut():
    """64-bit device lengths follow the rules of the 32-bit ones."""
    banner("64-bit lengths")
    q, kv = [2, 3], [50, 64]
    query, k, v, table = (x.cuda() for x in orc.paged_case(6, q, kv, 12, 2, FP16, 16, width=4))

    def run(q, kv):
        plan = paged_plan(table, q, kv, 5, 12, 2, 16)
        return paged_attention(query, k, v, plan, SCALE), plan.positions

    for wide, narrow in (([2, (1 << 32) + 3], [2, (1 << 31) - 1]), ([2, -(1 << 32) + 3], [2, -5])):
        got, want = (run(torch.tensor(x, device="cuda"), ints(kv)) for x in (wide, narrow))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    got, want = (run(ints(q), torch.tensor([50, x], device="cuda")) for x in ((1 << 32) + 1, 64))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    cache = PagedCache(1, 8, 16, 2, 2, 64)
    kept = state_of(cache)
    cache.step(torch.tensor([1, (1 << 32) + 1], device="cuda"), 2, 4)
    assert same_state(cache, kept)
    with pytest.raises(RuntimeError, match="rows"):
        cache.check()


@pytest.mark.parametrize("q,kv,heads,kv_heads", [
    ([30], [70], 2, 2), ([5, 1], [300, 90], 6, 1),  # single tiles of few rows
    ([300], [300], 2, 2), ([200, 1], [330, 40], 12, 2),  # prompts, whole ranges
    ([200], [2300], 2, 2), ([20], [5000], 1, 1),  # split ranges
    ([320] * 9, [330] * 9, 24, 24)])  # four waves a tile
def test_how_far_values_that_are_not_finite_reach(q, kv, heads, kv_heads):
    """A key of infinities, then a value of them, at one position of the last new rows: what comes before
    a key keeps its bits, what comes more than 63 + ceil(31 / group) positions before a value does, and so
    does every other sequence."""
    banner("values that are not finite", q, kv, heads, kv_heads)
    ps, group, dtype = 16, heads // kv_heads, FP16
    query, k, v, table = orc.paged_case(21, q, kv, heads, kv_heads, dtype, ps)
    want, plan = attend(query, k, v, table, q, kv, ps)
    pos, own = plan.positions.cpu(), plan.sequences.cpu() == 0
    assert torch.isfinite(want).all()
    for back in (1, 2, 40, 64, 130):
        at = kv[0] - back
        if back > q[0]:
            continue
        page, row = int(table[0, at // ps]), at % ps
        for x, reach in ((k.clone(), 0), (v.clone(), 63 + -(-31 // group))):
            x[page, :, row] = float("inf")
            pools = (k, x) if reach else (x, v)
            got, _ = attend(query, *pools, table, q, kv, ps)
            safe = (~own | (pos < at - reach)).cuda()
            assert torch.equal(got[safe], want[safe]), (back, reach)
            if reach:
                assert not torch.isfinite(got[(own & (pos >= at)).cuda()]).any()


def test_a_graph_keeps_the_plan_of_another():
    """A plan made in one capture and read by the calls of a second: the second graph keeps it when the
    first one and the plan object are gone; the calls of the plan's own capture need not."""
    from hackaton_amd import attention as att

    banner("a plan of another graph")
    q, kv = [1, 50, 3], [1400, 90, 65]
    query, k, v, table = (x.cuda() for x in orc.paged_case(12, q, kv, 12, 2, FP16, 16))
    want, plan = attend(query, k, v, table, q, kv, 16)
    q_len, kv_len = ints(q), ints(kv)
    paged_attention(query, k, v, plan, SCALE)
    att.release_captured_plans()
    torch.cuda.synchronize()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        plan = paged_plan(table, q_len, kv_len, sum(q), 12, 2, 16)
        own = paged_attention(query, k, v, plan, SCALE)
    assert not att._CAPTURED_PLANS
    with torch.cuda.graph(second):
        out = paged_attention(query, k, v, plan, SCALE)
    assert att._CAPTURED_PLANS == {plan}
    first.replay()
    second.replay()
    torch.cuda.synchronize()
    assert torch.equal(own.view_as(want), want) and torch.equal(out.view_as(want), want)
    size = plan.words.numel()
    del plan, own, first
    torch.cuda.empty_cache()
    fill = [torch.full((size,), 1 << 20, dtype=torch.int32, device="cuda") for _ in range(8)]
    for _ in range(3):
        out.zero_()
        second.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view_as(want), want)
    del fill, second
    att.release_captured_plans()
