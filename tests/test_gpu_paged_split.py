"""Work lists of steps of prompts and trees alone: ranges of unequal lengths are split at their average and go
longest first, a few long ones are split among twice the places; and the attention over such lists."""

import numpy as np
import pytest
import torch

from hackaton_amd import paged_plan
from tests import paged8_oracle as o8
from tests.test_gpu_paged import banner, check_attention, ints
from tests.test_gpu_paged8 import check_attention as check_attention8
from tests.test_gpu_paged_edges import check_lists, lists_of, long_plan
from tests.test_gpu_tree import check_tree

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16


def lengths(seed, count, lo, hi):
    return np.exp(np.random.default_rng(seed).uniform(np.log(lo), np.log(hi), count)).astype(int).tolist()


STEPS = {  # new tokens, cached tokens, heads, key/value heads
    "trees": ([24] * 64, lengths(1, 64, 64, 8192), 28, 4),
    "ragged chunks": (lengths(2, 16, 64, 2048), lengths(3, 16, 64, 16384), 28, 4),
    "256 sequences": ([40] * 256, lengths(4, 256, 64, 4096), 12, 2),
    "257 sequences": ([40] * 257, lengths(5, 257, 64, 4096), 12, 2),
    "4096 sequences": ([9] * 4096, lengths(6, 4096, 16, 2048), 8, 2),
    "one long among many": ([40] * 100, [64] * 99 + [30000], 12, 2),
    "some without rows": ([0, 40] * 60, lengths(7, 120, 64, 6000), 12, 2),
    "few": (lengths(8, 8, 48, 64), lengths(9, 8, 28000, 32000), 28, 4),
    "one": ([128], [32640], 28, 4),
    "one of many parts": ([40], [60000], 6, 1),
    "three": ([300, 17, 900], [1200, 60000, 9], 12, 2),
    "few with answers": ([64, 64, 1, 1, 1], [30000, 9000, 20000, 500, 3000], 28, 4),
    "many with answers": ([40] * 70 + [1] * 40, lengths(10, 110, 64, 9000), 28, 4),
    "before the cache": ([40] * 90, [-20] * 40 + lengths(11, 50, 64, 5000), 12, 2),
}


@pytest.mark.parametrize("name", STEPS)
def test_lists(name):
    """Every row and key once, in the room that there is; the longest sequences first where nothing but prompt
    tiles, more of them than the card has places, is split."""
    q, past, heads, kv_heads = STEPS[name]
    kv = [n + p for n, p in zip(q, past)]
    banner("lists", name, len(q))
    plan = long_plan(q, kv, heads, kv_heads) if min(past) >= 0 else paged_plan(
        torch.zeros(len(q), 40, dtype=torch.int32, device="cuda"), ints(q), ints(kv), sum(q), heads, kv_heads, 256)
    few, many = check_lists(plan, q, kv)
    # (of 8192 items, those of 16 times the average would be: the parts are at most 512)
    assert (many > 1).any() == (name != "4096 sequences")
    items, _ = lists_of(plan)
    tiles = sum(-(-n * heads // kv_heads // 128) for n in q if n * heads // kv_heads > 32) * kv_heads
    extra = int((many - 1).sum() + (few - 1).sum())
    assert extra <= 768
    if not len(few) and len(items) > 256 and len(q) <= 256:
        # (within 16 items tiles that read the same keys may be put together)
        order = [[kv[s] for s in items[i:i + 16, 1]] for i in range(0, len(items), 16)]
        assert "before" in name or all(min(a) >= max(b) for a, b in zip(order, order[1:]))
    # the longest part is no longer than the average share of the kind's parts, or than the shortest one: twice
    # that where the parts of a range are rounded down to a multiple of 8 / kv_heads (3 to 2, 7 to 4, 15 to 8)
    if not len(few):
        longest = int((items[:, 7] - items[:, 6]).max())
        total = sum(-(-n * heads // kv_heads // 128) * max(x, 0) for n, x in zip(q, kv)) * kv_heads
        assert longest <= 2 * (max(512, total / min(max(tiles, 64), 512)) + 64)


@pytest.mark.parametrize("heads,kv_heads", [(28, 4), (12, 2), (8, 1), (6, 3), (16, 8)])
@pytest.mark.parametrize("count,rows", [(32, 24), (31, 24), (5, 24), (64, 40), (1, 700)])
def test_tiles_that_read_the_same_keys(count, rows, heads, kv_heads):
    """Ranges that are not split: the list holds every tile once, and the two tiles of a sequence and head lie a
    multiple of 8 apart (work-groups go round the 8 XCDs) wherever whole 16 items are there to be ordered."""
    plan = long_plan([rows] * count, [3000 + rows] * count, heads, kv_heads)
    few, many = check_lists(plan, [rows] * count, [3000 + rows] * count)
    items, _ = lists_of(plan)
    two = -(-rows * heads // kv_heads // 128) == 2
    if two and (many == 1).all() and kv_heads in (1, 2, 4, 8):
        at = {}
        for i, (seq, head) in enumerate(zip(items[:, 1], items[:, 3] & 0xffff)):
            at.setdefault((seq, head), []).append(i)
        for places in at.values():
            if max(places) < len(items) // 16 * 16:
                assert (places[1] - places[0]) % 8 == 0


@pytest.mark.parametrize("q,kv,heads,kv_heads", [
    ([1 << 20], [1 << 20], 28, 4), ([1 << 20, 40], [1 << 20, 1 << 20], 32, 8), ([1 << 19] * 2, [1 << 22] * 2, 12, 2),
    ([40] * 600, [1 << 20] * 600, 12, 2)])
def test_lists_of_long_prompts_alone(q, kv, heads, kv_heads):
    banner("long prompts alone", q[:3], kv[:3], heads)
    few, many = check_lists(long_plan(q, kv, heads, kv_heads), q, kv)
    assert not len(few) and (many == 1).all()


@pytest.mark.parametrize("heads,kv_heads,dtype", [(8, 2, FP16), (7, 1, BF16)])
def test_attention_over_sorted_lists(heads, kv_heads, dtype):
    rng = np.random.default_rng(heads)
    q = [40, 9, 0, 33] * 16
    kv = [n + int(np.exp(rng.uniform(3, 7.3))) for n in q]
    check_attention(q, kv, heads, kv_heads, dtype, 16, padding=3)


def test_attention_of_few_long_rows_in_many_parts():
    """More parts than a merge record of 8 rows adds at once, and than it takes."""
    check_attention([40, 5], [2600, 3000], 6, 1, FP16, 16)
    check_attention([8], [9000], 6, 1, BF16, 64)
    rng = np.random.default_rng(5)
    for bits in (16, 8):
        check_tree(bits, [o8.random_tree(rng, 12, 5)], [14012], 4, 1, BF16, 64)


@pytest.mark.parametrize("n_seqs", [256, 257, 1030])
def test_trees_of_many_sequences(n_seqs):
    """Paths within the plan's launch, and in one of their own."""
    rng = np.random.default_rng(n_seqs)
    sizes = rng.integers(0, 3, n_seqs).tolist()
    sizes[3], sizes[n_seqs // 2], sizes[-1] = 60, 256, 257
    trees = [o8.random_tree(rng, n, 9) for n in sizes]
    check_tree(16, trees, [n + int(rng.integers(0, 30)) for n in sizes], 2, 1, FP16, 16, padding=300)


# 240 tiles x heads, and 204: 8 waves a tile, over ranges that are split
WIDE = [([900, 40, 700], [1800, 2100, 700], 16, 16), ([700, 3, 820, 1], [1500, 2300, 830, 1900], 14, 14)]


@pytest.mark.parametrize("q,kv,heads,kv_heads", WIDE)
@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_attention_of_8_waves_over_split_ranges(q, kv, heads, kv_heads, dtype):
    check_attention(q, kv, heads, kv_heads, dtype, 32, padding=3)
    check_attention8(q, kv, heads, kv_heads, dtype, 32, padding=3)


@pytest.mark.parametrize("bits", [8, 16])
def test_trees_of_8_waves_over_split_ranges(bits):
    past, rng = [1500, 300, 20, 900, 0, 64, 1100, 600], np.random.default_rng(3)
    check_tree(bits, [o8.random_tree(rng, 100, 6) for _ in past], [100 + p for p in past], 28, 4, BF16, 16)


@pytest.mark.parametrize("bits", [8, 16])
def test_trees_that_are_more_than_the_places_of_8_waves(bits):
    """37 sequences of two tiles of four heads, in ranges that are split and that are not."""
    for past, count in ((500, 37), (1100, 37)):
        rng = np.random.default_rng(past)
        check_tree(bits, [o8.random_tree(rng, 19, 6) for _ in range(count)], [past + 19 + s for s in range(count)], 28, 4,
                   FP16, 16, width=80)
