"""A cache's layers are those of the memory that its pages are set to when they are asked for."""

import pytest
import torch

from hackaton_amd import PagedCache

E4M3 = torch.float8_e4m3fn


def check(cache):
    for layer in range(cache.pages.shape[0]):
        for which, got in enumerate((cache.keys(layer), cache.values(layer))):
            pairs = [(got, cache.pages)]
            if cache.exponents is not None:
                pairs = [(got.codes, cache.pages), (got.exponents, cache.exponents)]
            for x, held in pairs:
                assert x.is_set_to(held[layer, which]) and x.dtype == held.dtype
                assert x.requires_grad == held.requires_grad


@pytest.mark.parametrize("dtype", [torch.float16, E4M3])
def test_pages_that_are_set_to_other_memory(dtype):
    cache = PagedCache(3, 8, 16, 2, 2, 64, dtype, device="cpu")
    check(cache)
    cache.pages.data = torch.zeros_like(cache.pages)
    check(cache)
    cache.pages.data = cache.pages.data[:, :, :4]  # (the same address, fewer pages)
    check(cache)
    cache.pages.data = torch.zeros(2, 2, 8, 2, 16, 128).to(dtype)  # (fewer layers)
    check(cache)
    with pytest.raises(IndexError):
        cache.keys(2)
    cache.pages.set_(torch.zeros(3, 2, 8, 2, 16, 128).to(dtype))
    check(cache)
    cache.pages = cache.pages.clone()
    check(cache)


def test_pages_that_are_set_to_another_type():
    cache = PagedCache(2, 8, 16, 2, 2, 64, device="cpu")
    check(cache)
    cache.pages.data = cache.pages.data.view(torch.bfloat16)  # (the same address and sizes)
    check(cache)


def test_exponents_that_are_set_to_other_memory():
    cache = PagedCache(2, 8, 16, 2, 2, 64, E4M3, device="cpu")
    check(cache)
    cache.exponents.data = torch.zeros_like(cache.exponents.view(torch.uint8)).view(cache.exponents.dtype)
    check(cache)
    cache.exponents = cache.exponents.clone()
    check(cache)
    cache.pages, cache.exponents = cache.pages.to(torch.float16), None
    check(cache)
    exponents = torch.zeros(cache.pages.shape[:-1], dtype=torch.uint8).view(torch.float8_e8m0fnu)
    cache.exponents = exponents  # (before the pages)
    check(cache)


def test_pages_that_require_gradients_later():
    cache = PagedCache(2, 8, 16, 2, 2, 64, device="cpu")
    check(cache)
    cache.pages.requires_grad_()
    check(cache)
    cache.pages = cache.pages.detach()
    check(cache)
