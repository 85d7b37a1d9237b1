"""Entry points of 8-bit pages, trees and beam selection without a GPU: refusals before any launch, and the
references that the GPU tests compare with."""

import ctypes

import numpy as np
import pytest
import torch

import hackaton_amd
from hackaton_amd import PagedCache, QuantizedPages, _lib, beams, paged, select_beams
from tests import paged8_oracle as o8
from tests import paged_oracle as orc
from tests.test_paged import buffers, step


def test_the_entry_points_are_public():
    for name in ("QuantizedPages", "paged_accept", "select_beams"):
        assert name in hackaton_amd.__all__ and hasattr(hackaton_amd, name)
    assert select_beams is beams.select_beams and paged.TREE_TOKENS == _lib.VA_TREE_TOKENS == 256


def pages(p, **more):
    stride = 2 * 16 * 128
    base = dict(k_pages=p, v_pages=p, k_exps=p, v_exps=p, k_stride=stride, v_stride=stride,
                k_exp_stride=32, v_exp_stride=32, n_pages=4, dtype=_lib.VA_E4M3)
    return _lib.PagedPages(*(dict(base, **more)[k] for k in base))


BAD_PAGES = [(dict(k_pages=None), _lib.VA_EINVAL), (dict(v_exps=None), _lib.VA_EINVAL),
             (dict(k_stride=2 * 16 * 128 + 8), _lib.VA_EINVAL), (dict(v_stride=2 * 16 * 128 - 16), _lib.VA_EINVAL),
             (dict(k_exp_stride=31), _lib.VA_EINVAL), (dict(v_exp_stride=1 << 31), _lib.VA_EINVAL),
             (dict(n_pages=-1), _lib.VA_ESHAPE), (dict(dtype=_lib.VA_F32), _lib.VA_EDTYPE),
             (dict(dtype=_lib.VA_BF16), _lib.VA_EDTYPE), (dict(k_stride=1 << 32), _lib.VA_ESHAPE)]


@pytest.mark.parametrize("more,code", BAD_PAGES)
def test_pages_are_checked(more, code):
    raw, p = buffers()
    L = _lib.lib()
    attend = [step(p), None, p, pages(p, **more), 128, 0.1, _lib.VA_F16, p, p, 1 << 40, None]
    assert L.va_paged_attention_pages(*attend) == code and L.va_last_error()
    append = [step(p), None, p, p, p, p, p, 0, 128, 0, 64, p, pages(p, **more), 128, 0, _lib.VA_F16, None]
    assert L.va_paged_append_pages(*append) == code


@pytest.mark.parametrize("at,value,code", [
    (0, None, _lib.VA_EINVAL), (1, 8, _lib.VA_EINVAL), (2, None, _lib.VA_EINVAL), (3, None, _lib.VA_EINVAL),
    (4, 64, _lib.VA_ESHAPE), (5, 0.0, _lib.VA_EINVAL), (6, _lib.VA_E4M3, _lib.VA_EDTYPE), (7, None, _lib.VA_EINVAL)])
def test_attention_arguments_are_checked(at, value, code):
    raw, p = buffers()
    args = [step(p), None, p, pages(p), 128, 0.1, _lib.VA_F16, p, p, 1 << 40, None]
    args[at] = value if at != 1 else p + 8  # a tree that is not 16-byte aligned
    assert _lib.lib().va_paged_attention_pages(*args) == code


def test_tree_arguments_are_checked():
    raw, p = buffers()
    L, words = _lib.lib(), ctypes.c_int64()
    assert L.va_paged_tree_words(step(p, n_tokens=10), ctypes.byref(words)) == 0
    assert words.value == 10 * 8 + 12
    assert L.va_paged_tree_words(None, ctypes.byref(words)) == _lib.VA_EINVAL
    assert L.va_paged_tree_words(step(p), None) == _lib.VA_EINVAL
    assert L.va_paged_tree_words(step(p, hq=13), ctypes.byref(words)) == _lib.VA_ESHAPE
    need, room = 8 * 8 + 8, 1 << 30
    for args, code in (((step(p), p, p, room, None, p, need, None), _lib.VA_EINVAL),
                       ((step(p), p, p, room, p, None, need, None), _lib.VA_EINVAL),
                       ((step(p), p, p, room, p + 2, p, need, None), _lib.VA_EINVAL),
                       ((step(p), p, p, room, p, p + 4, need, None), _lib.VA_EINVAL),
                       ((step(p), None, p, room, p, p, need, None), _lib.VA_EINVAL),
                       ((step(p), p, p, 8, p, p, need, None), _lib.VA_ECAPACITY),
                       ((step(p), p, p, room, p, p, need - 1, None), _lib.VA_ECAPACITY),
                       ((step(p, page_size=20), p, p, room, p, p, need, None), _lib.VA_ESHAPE),
                       ((step(p, n_tokens=0), None, None, 0, None, None, 0, None), _lib.VA_OK)):
        assert L.va_paged_plan_tree(*args) == code


@pytest.mark.parametrize("at,value,code", [
    (0, None, _lib.VA_EINVAL), (1, "+8", _lib.VA_EINVAL), (2, None, _lib.VA_EINVAL), (3, "+8", _lib.VA_EINVAL),
    (4, -1, _lib.VA_ESHAPE), (5, -1, _lib.VA_ESHAPE), (6, 0, _lib.VA_ESHAPE), (7, 64, _lib.VA_ESHAPE),
    (8, None, _lib.VA_EINVAL), (9, None, _lib.VA_EINVAL), (10, "+2", _lib.VA_EINVAL)])
def test_accept_arguments_are_checked(at, value, code):
    raw, p = buffers()
    args = [step(p), p, p, p, 2, 4, 2, 128, p, p, p, None]
    args[at] = p + int(value) if isinstance(value, str) else value
    assert _lib.lib().va_paged_accept(*args) == code


@pytest.mark.parametrize("name", ["va_pages_remap8", "va_pages_compact8"])
def test_exponents_of_a_pool_are_checked(name):
    raw, p = buffers()
    remap = name == "va_pages_remap8"
    for exps in (None, p + 8):
        args = [p, exps, 2, 4, 2, 16, 128, p, p, p] + ([None, None] if remap else []) + [3, 2]
        args += ([p + 64, p + 128, p + 192, p, p] if remap else [p + 64, p + 192, p, p]) + [1 << 20, None]
        assert getattr(_lib.lib(), name)(*args) == _lib.VA_EINVAL


def beams_args(p):
    return [p, _lib.VA_F16, 100, 3, 4, 100, p, None, 0, 4, p, p, p, p, 1 << 30, None]


@pytest.mark.parametrize("at,value,code", [
    (0, None, _lib.VA_EINVAL), (0, "+1", _lib.VA_EINVAL), (1, 3, _lib.VA_EDTYPE), (1, -1, _lib.VA_EDTYPE),
    (2, 99, _lib.VA_EINVAL), (3, -1, _lib.VA_ESHAPE), (3, 1 << 40, _lib.VA_ESHAPE), (4, 0, _lib.VA_ESHAPE),
    (4, 65, _lib.VA_ESHAPE), (5, 0, _lib.VA_ESHAPE), (5, (1 << 18) + 1, _lib.VA_ESHAPE), (6, None, _lib.VA_EINVAL),
    (9, 0, _lib.VA_ESHAPE), (9, 65, _lib.VA_ESHAPE), (10, None, _lib.VA_EINVAL), (11, "+2", _lib.VA_EINVAL),
    (12, None, _lib.VA_EINVAL), (13, "+8", _lib.VA_EINVAL), (14, 16, _lib.VA_ECAPACITY)])
def test_selection_arguments_are_checked(at, value, code):
    raw, p = buffers()
    args = beams_args(p)
    args[at] = p + int(value) if isinstance(value, str) else value
    assert _lib.lib().va_select_beams(*args) == code


def test_selection_sizes():
    raw, p = buffers()
    L, nbytes = _lib.lib(), ctypes.c_int64()
    assert L.va_select_beams_workspace(3, 4, 100, ctypes.byref(nbytes)) == 0 and nbytes.value > 0
    assert L.va_select_beams_workspace(3, 4, 100, None) == _lib.VA_EINVAL
    assert L.va_select_beams_workspace(1 << 20, 1, 1 << 18, ctypes.byref(nbytes)) == 0
    for bad in ((-1, 4, 100), (3, 65, 100), (3, 4, 0), ((1 << 20) + 1, 1, 5), (1 << 19, 3, 5)):
        assert L.va_select_beams_workspace(*bad, ctypes.byref(nbytes)) == _lib.VA_ESHAPE
    args = beams_args(p)
    args[7], args[8] = p, 100  # an end token that is none
    assert L.va_select_beams(*args) == _lib.VA_EINVAL
    args = beams_args(p)
    args[5], args[2], args[9] = 1, 1, 5  # more than there are continuations
    assert L.va_select_beams(*args) == _lib.VA_ESHAPE
    args = beams_args(None)
    args[3] = 0
    assert L.va_select_beams(*args) == 0


def test_host_memory_is_refused():
    logits, scores = torch.zeros(4, 10), torch.zeros(4)
    with pytest.raises(ValueError, match="GPU"):
        select_beams(logits, scores, 4)
    cache = PagedCache(2, 4, 16, 2, 2, 64, o8.E4M3, device="cpu")
    assert isinstance(cache.keys(1), QuantizedPages) and cache.values(0).codes.shape == (4, 2, 16, 128)
    assert cache.pool.exponents.shape == (2, 2, 4, 2, 16)
    assert PagedCache(1, 4, 16, 2, 2, 64, device="cpu").pool.dtype == torch.float16
    for dtype in (torch.float32, torch.float8_e5m2, torch.int8):
        with pytest.raises(ValueError):
            PagedCache(1, 4, 16, 2, 2, 64, dtype, device="cpu")


@pytest.mark.parametrize("tree,q_lengths,rows", [
    ([-1, 0, 3, -1, 0], [3, 2], 6), ([-1, 0, 2, -1, 0], [3, 2], 6), ([-1, 0, 1, 0, 0], [3, 2], 6),
    ([-1, 0], [3, 2], 6), ([-1] * 7, [3, 2], 6), ([-1] * 257, [257], 257)])
def test_host_trees_are_checked(tree, q_lengths, rows):
    with pytest.raises(ValueError):
        paged._parents(tree, q_lengths, rows, torch.device("cpu"))


def test_host_trees():
    device = torch.device("cpu")
    got = paged._parents([-1, 0, 0, -5, 0], [3, 2], 7, device)
    assert got.tolist() == [-1, 0, 0, -1, 0, -1, -1] and got.dtype == torch.int32
    chain = [j - 1 for j in range(300)]
    assert paged._parents(chain, [300], 300, device).tolist() == chain
    # device lengths: what the tree says cannot be held against them
    assert paged._parents([5, 1 << 40], torch.tensor([2]), 3, device).tolist() == [5, (1 << 31) - 1, -1]
    for bad in (torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int64),
                torch.zeros(6, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError):
            paged._parents(bad, [3], 3, device)


def test_the_quantization_is_what_it_says():
    """The reference against torch's own e4m3 numbers, borders of the exponent, and its error: half a step of
    a number, or of the smallest step of its row."""
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(200, 128, generator=gen) * torch.exp2(torch.randint(-30, 30, (200, 1), generator=gen))
    numbers, exponents = o8.quantize(x)
    codes, exps = o8.bytes_of(numbers, exponents)
    assert torch.equal(codes.double(), numbers) and torch.equal(
        codes.view(torch.uint8), (x / torch.exp2(exponents)[:, None].float()).to(o8.E4M3).view(torch.uint8))
    top = numbers.abs().amax(-1)
    assert (top <= 448).all() and (top >= 224).all()
    held = o8.values(codes, exps)
    assert torch.equal(QuantizedPages(codes, exps).dequantize().double(), held)
    assert ((held - x).abs() <= torch.maximum(2.0 ** -4 * x.abs(), 2.0 ** -10 * torch.exp2(exponents)[:, None])).all()
    edge = torch.tensor([448.0, 448.0001, 224.0, 1e-40, 0.0, 3.4e38])
    assert o8.exponent_of(edge[:, None]).tolist() == [0, 1, -1, -100, -100, 120]
    odd = torch.tensor([[1.0, float("inf"), float("nan"), -2.0]])
    assert torch.equal(torch.isnan(o8.quantize(odd)[0]), torch.tensor([[False, True, True, False]]))


def test_the_references_agree():
    """A chain's attention is the causal one; a tree's is that of every path by itself."""
    rng = np.random.default_rng(0)
    q, kv = [4, 1], [20, 5]
    query, k, v, table = orc.paged_case(1, q, kv, 4, 2, torch.float16, 16)
    exact = [torch.nan_to_num(x.double()) for x in (k, v)]
    want = orc.attention(query, k, v, table, q, kv)
    for a, b in zip(want, o8.attention(query, *exact, table, q, kv)):
        assert torch.equal(a, b)
    tree = o8.random_tree(rng, 4, 2)
    assert tree[0] == -1 and all(p < j for j, p in enumerate(tree))
    got, _ = o8.attention(query, *exact, table, q, kv, [tree, [-1]])
    on = o8.paths(tree)
    for j in range(4):
        path = np.nonzero(on[j])[0].tolist()
        rows = [o8.orc.rows_of(x, table[0], 20)[:, list(range(16)) + [16 + i for i in path]] for x in exact]
        for h in range(4):
            w = torch.softmax(rows[0][h // 2] @ query[j, h].double() * orc.SCALE, 0)
            assert torch.allclose(got[j, h], w @ rows[1][h // 2], atol=1e-12)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float8_e4m3fn])
def test_layers_of_a_cache_are_views_of_its_pages(dtype):
    cache = PagedCache(3, 8, 16, 2, 2, 64, dtype, device="cpu")
    for _ in range(2):
        for layer in (0, 2, -1):
            for which, got in enumerate((cache.keys(layer), cache.values(layer))):
                quantized = dtype == torch.float8_e4m3fn
                pages, want = got.codes if quantized else got, cache.pages[layer, which]
                assert pages.data_ptr() == want.data_ptr() and pages.shape == want.shape
                assert pages.stride() == want.stride()
                if quantized:
                    assert got.exponents.data_ptr() == cache.exponents[layer, which].data_ptr()
                    assert got.exponents.shape == cache.exponents[layer, which].shape
        with pytest.raises(IndexError):
            cache.keys(3)
        cache.pages = torch.zeros_like(cache.pages)  # (others that the program sets are followed)
