"""The paged cache's refusals in an order that changes nothing, without a GPU."""

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from hackaton_amd import PagedCache, _lib, paged
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


@pytest.mark.parametrize("at,value,code", [
    (0, None, _lib.VA_EINVAL), (1, None, _lib.VA_EINVAL), (2, -1, _lib.VA_ESHAPE),
    (2, (1 << 20) + 1, _lib.VA_ESHAPE), (3, -1, _lib.VA_ESHAPE), (4, None, _lib.VA_EINVAL),
    (5, None, _lib.VA_EINVAL)])
def test_growth_arguments_are_checked(at, value, code):
    raw = np.zeros(64, dtype=np.int32)
    args = [raw.ctypes.data, raw.ctypes.data, 4, 8, raw.ctypes.data, raw.ctypes.data, None]
    args[at] = value
    assert _lib.lib().va_pages_growth(*args) == code
    args = [raw.ctypes.data, raw.ctypes.data, 4, 8, raw.ctypes.data, raw.ctypes.data, None]
    if at in (0, 1, 4, 5):
        args[at] += 2  # not a word
        assert _lib.lib().va_pages_growth(*args) == _lib.VA_EINVAL
    assert _lib.lib().va_pages_growth(None, None, 0, 8, None, None, None) == 0


def test_tangents_are_refused():
    x = torch.randn(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x)
        for off in (torch.enable_grad, torch.no_grad):  # (no_grad leaves forward mode on)
            with off(), pytest.raises(RuntimeError, match="forward-mode"):
                paged._no_grad(x, dual)
        paged._no_grad(x, forward_ad.unpack_dual(dual).primal)
    paged._no_grad(x)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.int16, torch.uint8])
def test_lengths_of_any_whole_type(dtype):
    """Those that pass 32 bits are cut to the largest; negative ones count as 0 either way."""
    top = torch.iinfo(dtype).max
    given = torch.tensor([0, 7, min(top, (1 << 32) + 5), min(top, 1 << 40), top], dtype=dtype)
    got = paged._lengths("q_lengths", given, 5, given.device)
    assert got.dtype == torch.int32 and got.is_contiguous()
    assert got.tolist() == [min(x, (1 << 31) - 1) for x in given.tolist()]
    strided = torch.stack((given, given), 1)[:, 0]
    assert torch.equal(paged._lengths("q_lengths", strided, 5, given.device), got)
    if dtype == torch.int64:
        low = torch.tensor([-1, -(1 << 32) + 9, -(1 << 63)])
        assert paged._lengths("q_lengths", low, 3, low.device).clamp(min=0).tolist() == [0, 0, 0]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64, torch.complex64, torch.bool])
def test_lengths_of_other_types_are_refused(dtype):
    with pytest.raises(ValueError, match="whole numbers"):
        paged._lengths("q_lengths", torch.zeros(2).to(dtype), 2, torch.device("cpu"))
