"""Steps over short tables: prompt tiles of 32 rows while they are few, of 128 else; the lists of both and the
attention over them, and small steps over tables that are long enough for tiles of 128."""

import numpy as np
import pytest
import torch

from hackaton_amd import paged_plan
from tests import paged8_oracle as o8
from tests.test_gpu_paged import banner, check_attention, ints
from tests.test_gpu_paged8 import check_attention as check8
from tests.test_gpu_paged_edges import FEW, MANY, PAD
from tests.test_gpu_tree import check_tree as check_trees

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16

# new tokens, cached tokens, padding, heads, key/value heads, rows of a tile
STEPS = {
    "four trees": ([16] * 4, [512] * 4, 0, 12, 2, 32),
    "no fewer rows than sequences": ([1] * 6, [300] * 6, 0, 12, 2, 128),
    "one row more": ([2] + [1] * 5, [300] * 6, 0, 12, 2, 32),
    "mixed": ([1, 0, 5, 33, 1, 0, 64, 100, 2, 3, 130, 1], [6, 40, 0, 267, 259, 0, 0, 65, 0, 497, 1, 76], 5, 12, 2, 32),
    "256 items": ([128] * 6 + [63], [10, 70, 0, 600, 64, 65, 3], 0, 8, 8, 32),       # (7 + 831 / 32) * 8
    "a row past 256 items": ([128] * 6 + [63], [10, 70, 0, 600, 64, 65, 3], 1, 8, 8, 128),
    "512 items of long prompts": ([1015, 1000], [9, 0], 0, 8, 8, 32),                # (2 + 2015 / 32) * 8
    "a row past 512 items": ([1015, 1000], [9, 0], 1, 8, 8, 128),
    "tiles of many sequences": ([24] * 30, [300] * 30, 0, 12, 2, 128),               # (30 + 135) * 2, 4.5 a sequence
    "eight tiles a sequence": ([43] * 16, [300] * 16, 0, 12, 2, 32),                 # (16 + 129) * 2
    "rows of padding count": ([2] * 3, [50] * 3, 3000, 12, 2, 128),
    "no sequence has rows": ([0] * 4, [50] * 4, 70, 12, 2, 32),
    "before the cache": ([40, 20], [-20, -30], 0, 12, 2, 32),
    "groups of 40": ([3, 1, 7], [30, 1000, 0], 2, 40, 1, 32),
}


def check_tree(q, past, heads, kv_heads, dtype, bits, **more):
    rng = np.random.default_rng(sum(q))
    check_trees(bits, [o8.random_tree(rng, n, 5) for n in q], [n + p for n, p in zip(q, past)], heads, kv_heads,
                dtype, 16, **more)


@pytest.mark.parametrize("name", STEPS)
def test_lists(name):
    """Every row of every key/value head in one item, of the rows that its step's tiles have, with all of
    its keys."""
    q, past, padding, heads, kv_heads, each = STEPS[name]
    q, past = np.asarray(q), np.asarray(past)
    n, group, width = int(q.sum()) + padding, heads // kv_heads, 64
    banner("lists", name, n)
    plan = paged_plan(torch.zeros(len(q), width, dtype=torch.int32, device="cuda"), ints(q.tolist()),
                      ints((q + past).tolist()), n, heads, kv_heads, 16)
    words = plan.words.cpu().numpy().astype(np.int64)
    counts = -(-(len(q) + 1) // 4) * 4 + 2 * (-(-n // 4) * 4)
    n_items, n_merges = words[counts], words[counts + 1]
    assert n_merges == 0 and n_items <= (words.size - counts - 4) // 12
    items = words[counts + 4:counts + 4 + 12 * n_items].reshape(-1, 12)
    kind = items[:, 3] >> 16
    pads = items[kind == PAD]
    assert (pads[:, 5] - pads[:, 4]).sum() == padding
    items = items[kind != PAD]
    token0, seq, pos0, head, row, end, key, key_end, part_row = items[:, :9].T
    kind, head = head >> 16, head & 0xffff
    rows, cu = (q * group)[seq], np.concatenate(([0], np.cumsum(q)))
    lengths = np.maximum(q + past, 0)
    assert (token0 == cu[seq]).all() and (pos0 == (lengths - q)[seq]).all()
    if each == 32:
        assert (kind == FEW).all()
    else:
        assert ((kind == FEW) == (rows <= 32)).all() and ((kind == FEW) | (kind == MANY)).all()
    assert (row % each == 0).all() and (end == np.minimum(row + each, rows)).all()
    assert (key == 0).all() and (part_row == -1).all()
    assert (key_end == np.maximum(pos0 + (end - 1) // group + 1, 0)).all()
    seen = sorted(zip(seq.tolist(), head.tolist(), row.tolist()))
    assert seen == [(s, h, r) for s in range(len(q)) for h in range(kv_heads) for r in range(0, q[s] * group, each)]


@pytest.mark.parametrize("name", [x for x in STEPS if x not in ("no sequence has rows", "before the cache")])
def test_attention(name):
    q, past, padding, heads, kv_heads, _ = STEPS[name]
    kv = [n + p for n, p in zip(q, past)]
    padding = min(padding, 70) if name != "rows of padding count" else padding
    dtype = BF16 if len(name) % 2 else FP16
    check_attention(q, kv, heads, kv_heads, dtype, 16, padding=padding)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("name", ["four trees", "one row more", "mixed", "256 items", "eight tiles a sequence",
                                  "groups of 40"])
def test_trees(name, bits):
    q, past, padding, heads, kv_heads, _ = STEPS[name]
    check_tree(q, past, heads, kv_heads, BF16 if len(name) % 2 else FP16, bits, padding=padding)


@pytest.mark.parametrize("name", ["mixed", "512 items of long prompts", "eight tiles a sequence", "groups of 40"])
def test_8_bits(name):
    q, past, padding, heads, kv_heads, _ = STEPS[name]
    check8(q, [n + p for n, p in zip(q, past)], heads, kv_heads, BF16 if len(name) % 2 else FP16, 16, padding=padding)


MIXED = ([1, 0, 5, 33, 1, 0, 64, 100, 2, 3, 130, 1], [7, 40, 5, 300, 260, 0, 64, 165, 2, 500, 131, 77])


@pytest.mark.parametrize("heads,kv_heads,dtype", [(12, 2, FP16), (28, 4, BF16), (4, 4, FP16), (16, 2, BF16),
                                                  (3, 1, FP16), (40, 1, BF16)])
def test_small_steps_over_long_tables(heads, kv_heads, dtype):
    """Table rows past 1024 tokens, of which little is used: tiles of 128 rows, ranges that could be split."""
    q, kv = MIXED
    check_attention(q, kv, heads, kv_heads, dtype, 16, padding=5, width=80)
    check8(q, kv, heads, kv_heads, dtype, 16, padding=5, width=80)
    for bits in (8, 16):
        check_tree(q, [k - n for n, k in zip(q, kv)], heads, kv_heads, dtype, bits, padding=5, width=80)


@pytest.mark.parametrize("past", [0, 1, 30, 31, 32, 33, 62, 63, 64, 65, 127, 128, 200])
def test_every_border_of_the_cached_rows(past):
    """Trees and prompts of 40 and 90 tokens behind `past` cached ones, in tiles of 128 rows."""
    for bits in (8, 16):
        check_tree([40, 90], [past, past + 3], 6, 1, FP16, bits, width=80)
    check_attention([40, 90], [past + 40, past + 93], 6, 1, BF16, 16, width=80)
