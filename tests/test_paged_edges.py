"""The paged cache's refusals in an order that changes nothing, without a GPU."""

import pytest

from hackaton_amd import PagedCache
from hackaton_amd._lib import VarlenAttnError


@pytest.mark.parametrize("slots,q_lengths,n_tokens,heads,words", [
    (2, [1, 1], 2, 5, "Hq"), (2, [1, 1], 2, 0, "Hq"), (2, [1, 1], 2, 8192, "Hq"),
    (2, [1, 1], 1 << 30, 4, "n_tokens"), (2, [0, 0], 1 << 40, 4, "n_tokens"),
    (4097, [1] * 4097, 4097, 4, "n_seqs")])
def test_a_step_is_checked_before_the_cache_grows(slots, q_lengths, n_tokens, heads, words):
    """(On host memory any call that would grow the cache raises a ValueError.)"""
    cache = PagedCache(1, 4, 16, 2, slots, 64, device="cpu")
    with pytest.raises(VarlenAttnError, match=words):
        cache.step(q_lengths, n_tokens, heads)
