"""A paged key/value cache for answering with the model that `packed_attention` trains: the new
tokens of every sequence of a step are appended to pages and attend to them, one token each, a few
drafted ones or a prompt's chunk, all in one call. Hand-written gfx950 kernels through the C ABI; the
reference trains only and has no counterpart.

    paged_plan(page_table, q_lengths, kv_lengths, n_tokens, heads, kv_heads, page_size, tree)
    paged_append(q, k, v, cos, sin, k_pages, v_pages, plan, dtype)
    paged_attention(query, k_pages, v_pages, plan, scale)
    paged_accept(pages, plan, lengths, accepted)
    remap_pages(pages, table, lengths, refs, parents, new_lengths)
    compact_pages(pages, table, lengths, refs)
    PagedCache       a pool, its page tables and the calls above on them
    QuantizedPages   pages in 8 bits, where these calls take pages

Pages hold `page_size` rows (a power of two, 16 to 256) of every key/value head: one layer's keys are
(n_pages, kv_heads, page_size, 128). Row t of a sequence lies in page `page_table[sequence, t //
page_size]`, row `t % page_size`; entries outside the pool name no page. Lengths, tables and counts are
int32 and stay on the GPU: no call reads them back, so a captured step follows them. None of the calls
has a backward or a forward-mode derivative; tensors that ask for one are refused.
"""

import ctypes
import functools
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib, attention
from ._lib import check, lib
from .attention import _DTYPES, HEAD_DIM, _attn_dtype, _rope_strides, _tables
from .beams import select_beams

PAGE_SIZES = (16, 32, 64, 128, 256)
TREE_TOKENS = _lib.VA_TREE_TOKENS  # the most new tokens of a sequence that form a tree


class QuantizedPages(NamedTuple):
    """Pages in 8 bits: `codes` (..., n_pages, kv_heads, page_size, 128) float8_e4m3fn and `exponents`
    (..., n_pages, kv_heads, page_size) float8_e8m0fnu. A row's values are its codes times its power of
    two, the smallest from 2^-100 on that brings the row's largest finite number to 448 or less; numbers
    are rounded once, to nearest even, and what is not finite is held as not a number. A row takes 129
    bytes instead of 256. (`paged_append` writes exponent bytes of 27 to 247. Rows that a program writes itself
    may have 1 to 254: 0 and 255, 2^-127 and not a number to `dequantize`, mean nothing to the attention.)
    One layer's keys or values for `paged_append` and `paged_attention`, the whole
    pool (layers, 2, ...) for the page bookkeeping."""

    codes: torch.Tensor
    exponents: torch.Tensor

    def dequantize(self, dtype=torch.float32):
        """The values, as one tensor of another type."""
        return (self.codes.float() * self.exponents.float()[..., None]).to(dtype)


def _split(pages):
    """(pages or codes, exponents or None)."""
    return pages if isinstance(pages, QuantizedPages) else (pages, None)


def _no_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise RuntimeError("the paged cache has no backward: call it under torch.no_grad() "
                                   "or torch.inference_mode()")
    if forward_ad._current_level >= 0:  # inside forward_ad.dual_level()
        _no_tangent(*tensors)


def _no_tangent(*tensors):
    for t in tensors:
        if forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("the paged cache has no forward-mode derivative: pass the primals "
                               "(torch.autograd.forward_ad.unpack_dual)")


def _one_device(first, *tensors):
    device = first.device
    if not first.is_cuda:
        raise ValueError(f"the paged cache lives on the GPU only: got a tensor on {device}")
    index = device.index
    for t in tensors:
        if t.get_device() != index:  # (-1: not on a GPU)
            raise ValueError(f"tensors on {device} and {t.device}")
    return device


_current_device = torch._C._cuda_getDevice
_current_stream = torch._C._cuda_getCurrentRawStream


def _page_size(page_size):
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
    return int(page_size)


def _int32(name, t, *shape):
    if t.dtype != torch.int32 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor, got {t.dtype}, "
                         f"strides {t.stride()}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")


def _lengths(name, lengths, n_seqs, device):
    """Lengths of every sequence as an int32 device tensor, from one or from a host list."""
    if not isinstance(lengths, torch.Tensor):
        lengths = torch.tensor([int(x) for x in lengths], dtype=torch.int32, device=device)
    dtype = lengths.dtype
    if dtype != torch.int32 and (dtype.is_floating_point or dtype.is_complex or dtype == torch.bool):
        raise ValueError(f"{name} must be whole numbers, got {dtype}")
    if lengths.device != device:
        raise ValueError(f"{name} on {lengths.device}, page_table on {device}")
    if lengths.numel() != n_seqs:
        raise ValueError(f"{lengths.numel()} {name} for {n_seqs} page table rows")
    if dtype != torch.int32:  # (cut to their bounds, not to their low bits)
        lengths = lengths.to(torch.int64).clamp(0, 2 ** 31 - 1).to(torch.int32)
    return lengths if lengths.is_contiguous() else lengths.contiguous()


def _check_host_lengths(q_lengths, kv_lengths, n_tokens, most):
    """Host lists are checked before anything runs; device lengths cannot be without a read."""
    if isinstance(q_lengths, torch.Tensor) and isinstance(kv_lengths, torch.Tensor):
        return
    q_host = None if isinstance(q_lengths, torch.Tensor) else [int(x) for x in q_lengths]
    kv_host = None if isinstance(kv_lengths, torch.Tensor) else [int(x) for x in kv_lengths]
    if q_host is not None:
        if min(q_host, default=0) < 0:
            raise ValueError("q_lengths must not be negative")
        if sum(q_host) > n_tokens:
            raise ValueError(f"q_lengths sum to {sum(q_host)}, the step has {n_tokens} rows")
    if kv_host is not None and (min(kv_host, default=0) < 0 or max(kv_host, default=0) > most):
        raise ValueError(f"kv_lengths must lie in [0, {most}], what a page table row can name")
    if q_host is not None and kv_host is not None:
        if any(q > kv for q, kv in zip(q_host, kv_host)):
            raise ValueError("kv_lengths count the new tokens too: q_lengths may not exceed them")


@functools.lru_cache(maxsize=256)
def _plan_sizes(n_seqs, n_tokens, heads, kv_heads, page_size, width):
    """(int32 words of a plan, workspace bytes of an attention over it)."""
    words, nbytes = ctypes.c_int64(), ctypes.c_int64()
    step = _lib.PagedStep(None, None, n_tokens, n_seqs, width, page_size, heads, kv_heads)
    check(lib().va_paged_plan_words(step, ctypes.byref(words)), "va_paged_plan_words")
    check(lib().va_paged_attention_workspace(step, ctypes.byref(nbytes)),
          "va_paged_attention_workspace")
    return words.value, nbytes.value


class PagedPlan:
    """A step's rows and work list, shared by all of its layers: made by `paged_plan`. It keeps the
    page table and follows its entries as they are when a call runs; the lengths were read when the
    plan was made (a captured plan reads them again in every replay)."""

    __slots__ = ("page_table", "words", "n_tokens", "n_seqs", "heads", "kv_heads", "page_size",
                 "workspace_bytes", "_step", "_page", "_strides", "_stream",
                 "_capture", "_tree", "_paths")  # (_tree: the address of the tree's words, _paths: in `words`)

    def _rows(self, which):
        rows = -(-self.n_tokens // 4) * 4
        at = -(-(self.n_seqs + 1) // 4) * 4 + which * rows
        return self.words[at:at + self.n_tokens]

    @property
    def sequences(self):
        """(n_tokens) int32: the sequence of every row, -1 for padding."""
        return self._rows(0)

    @property
    def positions(self):
        """(n_tokens) int32: the position of every row in its sequence, -1 for padding. With a tree:
        the tokens that come before it, cached ones and those on its path."""
        if self._tree is None:
            return self._rows(1)
        at = self._paths + self.n_tokens * (TREE_TOKENS // 32)
        return self.words[at:at + self.n_tokens]

    @property
    def places(self):
        """(n_tokens) int32: where every row lies in its sequence's pages, -1 for padding: its position,
        but for the tokens of a tree, which lie in the order of the rows."""
        return self._rows(1)

    def _use(self):
        """The current stream, with the plan's memory kept for it: a graph that captures a call over a
        plan made before (by another graph too) reads it in every replay, whatever becomes of the plan
        object (kept until `release_captured_plans()`, as the work lists of `varlen_attention`); another
        stream than the plan's own reads it before it is handed out again."""
        stream = _current_stream(_current_device())
        if torch._C._cuda_isCurrentStreamCapturing():
            if self._capture != attention._capture_id():
                attention._CAPTURED_PLANS.add(self)
        elif stream != self._stream:
            current = torch.cuda.current_stream()
            self.words.record_stream(current)
            self.page_table.record_stream(current)
        return stream


def _parents(tree, q_lengths, n_tokens, device):
    """A step's tree as (n_tokens) int32 on the device, from such a tensor or from a host list."""
    if isinstance(tree, torch.Tensor):
        if tree.device != device:
            raise ValueError(f"tree on {tree.device}, page_table on {device}")
        _int32("tree", tree, n_tokens)
        return tree
    tree = [int(x) for x in tree]
    if len(tree) > n_tokens:
        raise ValueError(f"a tree of {len(tree)} rows, the step has {n_tokens}")
    if not isinstance(q_lengths, torch.Tensor):
        at = 0
        for count in (int(x) for x in q_lengths):
            rows, at = tree[at:at + count], at + count
            if len(rows) < count:
                raise ValueError(f"a tree of {len(tree)} rows for {sum(map(int, q_lengths))} new tokens")
            if any(p >= j for j, p in enumerate(rows)):
                raise ValueError("a token of a tree follows an earlier one of its sequence, or none (-1)")
            if count > TREE_TOKENS and any(p != j - 1 for j, p in enumerate(rows)):
                raise ValueError(f"a tree of {count} tokens: at most {TREE_TOKENS} of a sequence form one")
    out = torch.tensor(tree + [-1] * (n_tokens - len(tree)), dtype=torch.int64)
    return out.clamp(-1, 2 ** 31 - 1).to(device=device, dtype=torch.int32)


@functools.lru_cache(maxsize=256)
def _tree_words(n_seqs, n_tokens, heads, kv_heads, page_size, width):
    words = ctypes.c_int64()
    step = _lib.PagedStep(None, None, n_tokens, n_seqs, width, page_size, heads, kv_heads)
    check(lib().va_paged_tree_words(step, ctypes.byref(words)), "va_paged_tree_words")
    return words.value


def paged_plan(page_table, q_lengths, kv_lengths, n_tokens, heads, kv_heads, page_size, tree=None):
    """The plan of a step: `q_lengths[s]` new tokens of every sequence (packed rows, one sequence
    after the other, `n_tokens` rows in all; rows behind the last sequence are padding) and
    `kv_lengths[s]` cached tokens with the new ones included. Both are host lists or device tensors
    (for a captured step: device tensors); `page_table` is (sequences, pages per sequence) int32 on
    the GPU, at most 4096 sequences. Device lengths are not read back: negative ones count as 0, kv
    lengths end with the table row, new tokens with the rows. One launch.

    `tree`: the new tokens of a sequence form trees instead of following each other: of every row the
    number, among its sequence's new tokens, of the earlier one that it follows, or -1 where it follows the
    cached tokens directly; (n_tokens) int32 on the GPU or a host list. A row then sees the tokens cached
    before the step, those on its path, and itself. At most 256 new tokens of a sequence form a tree; those
    of a longer one follow each other whatever `tree` holds (host lists that say otherwise are refused,
    device ones are not read; there, what names no earlier token counts as -1)."""
    device = _one_device(page_table)
    if device.index != _current_device():  # launches and allocations go to the tensors' device
        with torch.cuda.device(device):
            return paged_plan(page_table, q_lengths, kv_lengths, n_tokens, heads, kv_heads,
                              page_size, tree)
    if page_table.dim() != 2:
        raise ValueError(f"page_table must be (sequences, pages), got {tuple(page_table.shape)}")
    n_seqs, width = page_table.shape
    _int32("page_table", page_table, n_seqs, width)
    page_size, n_tokens = _page_size(page_size), int(n_tokens)
    _check_host_lengths(q_lengths, kv_lengths, n_tokens, width * page_size)
    plan = PagedPlan()
    parents = None if tree is None else _parents(tree, q_lengths, n_tokens, device)
    n_words, plan.workspace_bytes = _plan_sizes(n_seqs, n_tokens, heads, kv_heads, page_size, width)
    q_lengths = _lengths("q_lengths", q_lengths, n_seqs, device)
    kv_lengths = _lengths("kv_lengths", kv_lengths, n_seqs, device)
    plan.page_table, plan.n_tokens, plan.n_seqs = page_table, n_tokens, n_seqs
    plan.heads, plan.kv_heads, plan.page_size = heads, kv_heads, page_size
    plan._page = (kv_heads, page_size, HEAD_DIM)
    plan._strides = (page_size * HEAD_DIM, HEAD_DIM, 1)
    tree_words = 0 if parents is None else _tree_words(n_seqs, n_tokens, heads, kv_heads, page_size, width)
    plan.words = torch.empty(n_words + tree_words, dtype=torch.int32, device=device)
    plan._stream = _current_stream(device.index)
    plan._capture = attention._capture_id() if torch._C._cuda_isCurrentStreamCapturing() else None
    plan._step = _lib.PagedStep(page_table.data_ptr(), plan.words.data_ptr(), n_tokens, n_seqs, width,
                                page_size, heads, kv_heads)
    if parents is None:
        plan._tree = plan._paths = None
        check(lib().va_paged_plan(plan._step, q_lengths.data_ptr(), kv_lengths.data_ptr(), n_words,
                                  plan._stream), "va_paged_plan")
        return plan
    plan._paths, plan._tree = n_words, plan._step.plan + 4 * n_words  # (whole pieces of 16 bytes)
    check(lib().va_paged_plan_tree(plan._step, q_lengths.data_ptr(), kv_lengths.data_ptr(), n_words,
                                   parents.data_ptr(), plan._tree, tree_words, plan._stream),
          "va_paged_plan_tree")
    return plan


def _pages_of(k_pages, v_pages, plan):
    """(elements from one key page to the next, value page, number of pages) of one layer."""
    shape = k_pages.shape
    if v_pages.shape != shape or shape[1:] != plan._page:
        raise ValueError("pages must be (n_pages, %d, %d, %d), got " % plan._page +
                         f"{tuple(shape)} and {tuple(v_pages.shape)}")
    if k_pages.dtype != v_pages.dtype:
        raise ValueError(f"keys in {k_pages.dtype}, values in {v_pages.dtype}")
    k_stride, v_stride = k_pages.stride(), v_pages.stride()
    if k_stride[1:] != plan._strides or v_stride[1:] != plan._strides:
        for stride in (k_stride, v_stride):
            if stride[2:] != plan._strides[1:] or plan.kv_heads != 1:  # (one head: its stride is free)
                raise ValueError(f"every page must be contiguous, got strides {stride}")
    if shape[0] <= 1:  # a pool of one page: its stride is free
        least = plan.kv_heads * plan.page_size * HEAD_DIM
        return max(k_stride[0], least), max(v_stride[0], least), shape[0]
    return k_stride[0], v_stride[0], shape[0]


def _exponents_of(k_pages, v_pages, n_pages, plan):
    """Elements from one page's exponents to the next, of keys and of values."""
    (codes, k), (_, v) = k_pages, v_pages
    if codes.dtype != torch.float8_e4m3fn or k.dtype != torch.float8_e8m0fnu or v.dtype != k.dtype:
        raise ValueError("8-bit pages are float8_e4m3fn codes and float8_e8m0fnu exponents, got "
                         f"{codes.dtype} and {k.dtype}, {v.dtype}")
    if k.device != codes.device or v.device != codes.device:
        raise ValueError(f"tensors on {codes.device}, {k.device} and {v.device}")
    kv_heads, page_size = plan.kv_heads, plan.page_size
    shape = (n_pages, kv_heads, page_size)
    if k.shape != shape or v.shape != shape:
        raise ValueError(f"exponents must be {shape}, got {tuple(k.shape)} and {tuple(v.shape)}")
    k_stride, v_stride = k.stride(), v.stride()
    for stride in (k_stride, v_stride):
        if stride[2] != 1 or (stride[1] != page_size and kv_heads != 1):
            raise ValueError(f"every page's exponents must be contiguous, got strides {stride}")
    if n_pages <= 1:
        least = kv_heads * page_size
        return max(k_stride[0], least), max(v_stride[0], least)
    return k_stride[0], v_stride[0]


def _layer(k_pages, v_pages, plan):
    """va_paged_pages of one layer's keys and values, in 8 bits or in 16."""
    if isinstance(k_pages, QuantizedPages) != isinstance(v_pages, QuantizedPages):
        raise ValueError("keys and values must both be pages in 8 bits, or neither")
    (k, k_exps), (v, v_exps) = _split(k_pages), _split(v_pages)
    k_stride, v_stride, n_pages = _pages_of(k, v, plan)
    if k_exps is None:
        return _lib.PagedPages(k.data_ptr(), v.data_ptr(), None, None, k_stride, v_stride, 0, 0, n_pages,
                               _attn_dtype(k))
    k_exp_stride, v_exp_stride = _exponents_of(k_pages, v_pages, n_pages, plan)
    return _lib.PagedPages(k.data_ptr(), v.data_ptr(), k_exps.data_ptr(), v_exps.data_ptr(), k_stride,
                           v_stride, k_exp_stride, v_exp_stride, n_pages, _lib.VA_E4M3)


def paged_append(q, k, v, cos, sin, k_pages, v_pages, plan, dtype=None):
    """The step's new rows: q (n_tokens, heads * 128), k and v (n_tokens, kv_heads * 128) projections
    in fp16, bf16 or fp32. Returns q rotated, (n_tokens, heads, 128) in the pages' type; k rotated and
    v go into `k_pages` / `v_pages` (n_pages, kv_heads, page_size, 128) at the rows' positions, rotated
    in fp32 and rounded once. cos / sin: (1 or sequences, T, 128) read by position, or (n_tokens, 128)
    read by row. Rows without a place (padding, positions past the tables or in no page) write
    nothing; padding and positions outside the cos / sin table give zeros in q. Pages may be
    `QuantizedPages`: keys, rotated, and values go into them in 8 bits. `dtype` is then q's, fp16 or bf16
    (None: the projections' type, fp16 for fp32 ones)."""
    (keys, k_exps), (values, v_exps) = _split(k_pages), _split(v_pages)
    device = _one_device(q, k, v, cos, sin, keys, values, plan.words)
    if device.index != _current_device():  # launches and allocations go to the tensors' device
        with torch.cuda.device(device):
            return paged_append(q, k, v, cos, sin, k_pages, v_pages, plan, dtype)
    _no_grad(q, k, v, keys, values)
    if forward_ad._current_level >= 0:  # (the tables are constants, as in qkv_rotate)
        _no_tangent(cos, sin)
    n, heads, kv_heads = plan.n_tokens, plan.heads, plan.kv_heads
    if (q.shape != (n, heads * HEAD_DIM) or k.shape != (n, kv_heads * HEAD_DIM)
            or v.shape != k.shape):
        raise ValueError(f"projections must be ({n}, {heads} and {kv_heads} * {HEAD_DIM}), got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if not (q.dtype == k.dtype == v.dtype) or q.dtype not in _DTYPES:
        raise ValueError(f"q, k and v must share a dtype (fp16, bf16 or fp32), got {q.dtype}, "
                         f"{k.dtype}, {v.dtype}")
    plain = plan._tree is None and k_exps is None and v_exps is None  # 16 bits, no tree
    if dtype is None:
        dtype = keys.dtype if k_exps is None else q.dtype if q.dtype != torch.float32 else torch.float16
    elif dtype not in (torch.float16, torch.bfloat16) or (k_exps is None and dtype != keys.dtype):
        raise ValueError(f"queries in {dtype} over pages in {keys.dtype}")
    if plain:
        out_dtype = _attn_dtype(k_pages)
        k_stride, v_stride, n_pages = _pages_of(k_pages, v_pages, plan)
    else:
        out_dtype, layer = _DTYPES[dtype], _layer(k_pages, v_pages, plan)
    by_row = cos.dim() == 2
    if by_row and (tuple(cos.shape) != (n, HEAD_DIM) or sin.shape != cos.shape):
        raise ValueError(f"cos/sin by row must be ({n}, {HEAD_DIM}), got {tuple(cos.shape)}, "
                         f"{tuple(sin.shape)}")
    cos, sin = _tables(cos[None] if by_row else cos, sin[None] if by_row else sin)
    if not by_row and cos.shape[0] not in (1, plan.n_seqs):
        raise ValueError(f"cos/sin for {cos.shape[0]} sequences, the plan has {plan.n_seqs}")
    query = torch.empty(n, heads, HEAD_DIM, dtype=dtype, device=device)
    if n == 0:
        return query
    if cos.shape[1] == 0:
        raise ValueError("cos/sin hold no positions")
    batch, row = (0, 0) if by_row else _rope_strides(cos)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    if not plain:
        check(lib().va_paged_append_pages(
            plan._step, plan._tree, q.data_ptr(), k.data_ptr(), v.data_ptr(), cos.data_ptr(),
            sin.data_ptr(), batch, row, HEAD_DIM if by_row else 0, 0 if by_row else cos.shape[1],
            query.data_ptr(), layer, HEAD_DIM, _DTYPES[q.dtype], out_dtype, plan._use()),
            "va_paged_append_pages")
        return query
    check(lib().va_paged_append(
        plan._step, q.data_ptr(), k.data_ptr(), v.data_ptr(), cos.data_ptr(), sin.data_ptr(), batch,
        row, HEAD_DIM if by_row else 0, 0 if by_row else cos.shape[1], query.data_ptr(),
        k_pages.data_ptr(), v_pages.data_ptr(), k_stride, v_stride, n_pages, HEAD_DIM,
        _DTYPES[q.dtype], out_dtype, plan._use()), "va_paged_append")
    return query


def paged_attention(query, k_pages, v_pages, plan, scale):
    """Every new token attends to its sequence's keys at positions up to its own. query
    (n_tokens, heads, 128) in the pages' type; returns (n_tokens, heads * 128), zeros for padding and
    for rows that see no key. Key/value heads are shared by heads / kv_heads query heads each. What a
    page holds behind its sequence's end never reaches a result. (Keys that a row does not see never reach it,
    whatever they hold. Values that are infinite or not a number do where they lie in a 64-key tile that
    another of the 32 rows computed together sees, rows being pairs of a token and a query head of the
    group: in rows of the same sequence up to 63 + ceil(31 kv_heads / heads) positions before their own;
    with a tree, places before or behind it: rows that do not see each other share tiles.)
    The same step gives the same bits; the same sequence in another step agrees to rounding. Pages may be
    `QuantizedPages`, under queries in fp16 or bf16: their values are multiplied as numbers of that type,
    exactly but for fp16's range: past 65504 they are infinite, below 2^-14 multiples of 2^-24."""
    (keys, k_exps), (values, v_exps) = _split(k_pages), _split(v_pages)
    device = _one_device(query, keys, values, plan.words)
    if device.index != _current_device():  # launches and allocations go to the tensors' device
        with torch.cuda.device(device):
            return paged_attention(query, k_pages, v_pages, plan, scale)
    _no_grad(query, keys, values)
    dtype = _attn_dtype(query)
    if k_exps is None and keys.dtype != query.dtype:
        raise ValueError(f"query in {query.dtype}, pages in {keys.dtype}")
    n, heads = plan.n_tokens, plan.heads
    if query.shape != (n, heads, HEAD_DIM):
        raise ValueError(f"query must be ({n}, {heads}, {HEAD_DIM}), got {tuple(query.shape)}")
    plain = plan._tree is None and k_exps is None and v_exps is None  # 16 bits, no tree
    if plain:
        k_stride, v_stride, n_pages = _pages_of(k_pages, v_pages, plan)
    else:
        layer = _layer(k_pages, v_pages, plan)
    query = query.contiguous()
    out = torch.empty(n, heads * HEAD_DIM, dtype=query.dtype, device=device)
    if n == 0:
        return out
    nbytes = plan.workspace_bytes
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    if not plain:
        check(lib().va_paged_attention_pages(
            plan._step, plan._tree, query.data_ptr(), layer, HEAD_DIM, scale, dtype, out.data_ptr(),
            ws.data_ptr() if nbytes else None, nbytes, plan._use()), "va_paged_attention_pages")
        return out
    check(lib().va_paged_attention(
        plan._step, query.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), k_stride, v_stride,
        n_pages, HEAD_DIM, scale, dtype, out.data_ptr(), ws.data_ptr() if nbytes else None, nbytes,
        plan._use()), "va_paged_attention")
    return out


# ------------------------------------------------------------------------------------------------
# page bookkeeping
# ------------------------------------------------------------------------------------------------
def _pool_of(pages, exponents):
    """(layers * 2, n_pages, kv_heads, page_size) of a whole pool."""
    shape = pages.shape
    if len(shape) != 6 or shape[1] != 2 or shape[5] != HEAD_DIM:
        raise ValueError(f"pages must be (layers, 2, n_pages, kv_heads, page_size, {HEAD_DIM}), got "
                         f"{tuple(shape)}")
    if not pages.is_contiguous():
        raise ValueError(f"pages must be contiguous, got strides {pages.stride()}")
    if exponents is None:
        _attn_dtype(pages)
    elif pages.dtype != torch.float8_e4m3fn or exponents.dtype != torch.float8_e8m0fnu:
        raise ValueError("8-bit pages are float8_e4m3fn codes and float8_e8m0fnu exponents, got "
                         f"{pages.dtype} and {exponents.dtype}")
    elif (exponents.shape != shape[:-1] or not exponents.is_contiguous()
          or exponents.device != pages.device):
        raise ValueError(f"exponents must be {tuple(shape[:-1])}, contiguous, on {pages.device}, got "
                         f"{tuple(exponents.shape)}, strides {exponents.stride()} on {exponents.device}")
    return 2 * shape[0], shape[2], shape[3], _page_size(shape[4])


def _state_of(n_pages, table, lengths, refs, **more):
    """(slots, pages per slot) of a cache's state, every tensor of which is checked; `more` holds one
    number per slot each (or None)."""
    if table.dim() != 2:
        raise ValueError(f"table must be (slots, pages), got {tuple(table.shape)}")
    slots, width = table.shape
    _int32("table", table, slots, width)
    _int32("lengths", lengths, slots)
    _int32("refs", refs, n_pages)
    for name, t in more.items():
        if t is not None:
            _int32(name, t, slots)
    return slots, width


@functools.lru_cache(maxsize=64)
def _scratch_words(slots, n_pages):
    words = ctypes.c_int64()
    check(lib().va_pages_scratch_words(slots, n_pages, ctypes.byref(words)),
          "va_pages_scratch_words")
    return words.value


def remap_pages(pages, table, lengths, refs, parents=None, new_lengths=None):
    """The page tables of the next step. Slot i goes on as slot `parents[i]` (None: every slot as
    itself; outside the table: as nobody), cut to `new_lengths[i]` tokens or grown to them with free
    pages (None: as long as the parent). One call forks, reorders, frees, enters, cuts back and grows
    sequences:

        fork i into j       parents[j] = i
        free j              parents[j] = -1, new_lengths[j] = 0
        enter n tokens      parents[j] = -1, new_lengths[j] = n
        grow or cut         new_lengths[i]

    pages (layers, 2, n_pages, kv_heads, page_size, 128); table (slots, pages per slot), lengths
    (slots) and refs (n_pages: how often each page is held, 0 = free) int32. Returns new (table,
    lengths, refs, shortfall). Slots share full pages; a part-filled last page stays with the lowest
    slot that ends in it if nobody else holds it, and the others get a copy of its filled rows, in
    every layer. Free pages are handed out in ascending order, slot after slot. shortfall (1): 0, or
    how many pages the pool or the table rows lack, in which case nothing changes."""
    codes, exponents = _split(pages)
    device = _one_device(codes, table, lengths, refs,
                         *(t for t in (parents, new_lengths) if t is not None))
    if device.index != _current_device():  # launches and allocations go to the tensors' device
        with torch.cuda.device(device):
            return remap_pages(pages, table, lengths, refs, parents, new_lengths)
    _no_grad(codes)
    outer, n_pages, kv_heads, page_size = _pool_of(codes, exponents)
    slots, width = _state_of(n_pages, table, lengths, refs, parents=parents, new_lengths=new_lengths)
    table_out, lengths_out, refs_out = (torch.empty_like(table), torch.empty_like(lengths),
                                        torch.empty_like(refs))
    shortfall = torch.empty(1, dtype=torch.int32, device=device)
    words = _scratch_words(slots, n_pages)
    scratch = torch.empty(words, dtype=torch.int32, device=device)
    rest = (outer, n_pages, kv_heads, page_size, HEAD_DIM, table.data_ptr(), lengths.data_ptr(),
            refs.data_ptr(), None if parents is None else parents.data_ptr(),
            None if new_lengths is None else new_lengths.data_ptr(), slots, width,
            table_out.data_ptr(), lengths_out.data_ptr(), refs_out.data_ptr(), shortfall.data_ptr(),
            scratch.data_ptr(), words, _current_stream(device.index))
    if exponents is None:
        check(lib().va_pages_remap(codes.data_ptr(), *rest), "va_pages_remap")
    else:
        check(lib().va_pages_remap8(codes.data_ptr(), exponents.data_ptr(), *rest), "va_pages_remap8")
    return table_out, lengths_out, refs_out, shortfall


def compact_pages(pages, table, lengths, refs):
    """The live pages (refs > 0) to the front of the pool: the k-th live page at or past their number
    moves to the k-th free page below it, in every layer. Arguments as for `remap_pages`. Returns
    new (table, refs, live); live (1): how many pages are in use, all of them below that number. Pages
    that the program holds without a table row move too: a row of their own keeps track of them."""
    codes, exponents = _split(pages)
    device = _one_device(codes, table, lengths, refs)
    if device.index != _current_device():  # launches and allocations go to the tensors' device
        with torch.cuda.device(device):
            return compact_pages(pages, table, lengths, refs)
    _no_grad(codes)
    outer, n_pages, kv_heads, page_size = _pool_of(codes, exponents)
    slots, width = _state_of(n_pages, table, lengths, refs)
    table_out, refs_out = torch.empty_like(table), torch.empty_like(refs)
    live = torch.empty(1, dtype=torch.int32, device=device)
    words = _scratch_words(slots, n_pages)
    scratch = torch.empty(words, dtype=torch.int32, device=device)
    rest = (outer, n_pages, kv_heads, page_size, HEAD_DIM, table.data_ptr(), lengths.data_ptr(),
            refs.data_ptr(), slots, width, table_out.data_ptr(), refs_out.data_ptr(), live.data_ptr(),
            scratch.data_ptr(), words, _current_stream(device.index))
    if exponents is None:
        check(lib().va_pages_compact(codes.data_ptr(), *rest), "va_pages_compact")
    else:
        check(lib().va_pages_compact8(codes.data_ptr(), exponents.data_ptr(), *rest),
              "va_pages_compact8")
    return table_out, refs_out, live


def paged_accept(pages, plan, lengths, accepted):
    """The end of a step whose new tokens were drafted: the tokens up to `accepted[s]` on its path stay.
    pages: the whole pool, (layers, 2, n_pages, kv_heads, page_size, 128) or `QuantizedPages`; plan: the
    step's, with its tree (or without: the tokens follow each other); lengths (sequences) int32: the cached
    tokens, the new ones included; accepted (sequences) int32: the number of a new token of the sequence,
    anything else: none stays. The rows that stay move together behind the tokens cached before, in order
    and in every layer; rows behind them hold what they held or what moved over them. Returns the lengths
    (sequences) int32, up to the last row that stays, by the plan's places (which end with the step's rows and
    the table row); sequences without rows in the step keep theirs. Pages past them are given back by
    `remap_pages(pages, table, lengths, refs, None, new_lengths)` over the lengths of before the call.
    The call belongs to its step: before the sequences are forked, reordered or stepped again, since it
    follows the page table as it is and moves rows within pages that no other sequence may hold."""
    codes, exponents = _split(pages)
    device = _one_device(codes, plan.words, lengths, accepted)
    if device.index != _current_device():  # launches and allocations go to the tensors' device
        with torch.cuda.device(device):
            return paged_accept(pages, plan, lengths, accepted)
    _no_grad(codes)
    outer, n_pages, kv_heads, page_size = _pool_of(codes, exponents)
    if (kv_heads, page_size) != (plan.kv_heads, plan.page_size):
        raise ValueError(f"pages of {page_size} rows of {kv_heads} heads, the plan's have "
                         f"{plan.page_size} of {plan.kv_heads}")
    _int32("lengths", lengths, plan.n_seqs)
    _int32("accepted", accepted, plan.n_seqs)
    out = torch.empty_like(lengths)
    check(lib().va_paged_accept(
        plan._step, plan._tree, codes.data_ptr(), None if exponents is None else exponents.data_ptr(),
        outer, n_pages, kv_heads, HEAD_DIM, lengths.data_ptr(), accepted.data_ptr(), out.data_ptr(),
        plan._use()), "va_paged_accept")
    return out


class PagedCache:
    """Keys and values of `layers` layers in one pool of `n_pages` pages, and up to `slots` sequences
    of at most `max_length` tokens (rounded up to whole pages) in it, in fp16, bf16 or, with
    `dtype=torch.float8_e4m3fn`, in 8 bits (`QuantizedPages`). State, all on the GPU: `pages` (8 bits: the
    codes, and `exponents`), `table`, `lengths`, `refs`. Every call updates it in place on the current
    stream, so the calls of one cache belong on one stream or in order across streams, and a captured
    step replays on the state it finds. A call that lacks pages (or a step that lacks rows) changes
    nothing; `check()` reports it."""

    def __init__(self, layers, n_pages, page_size, kv_heads, slots, max_length,
                 dtype=torch.float16, device="cuda"):
        self.page_size = _page_size(page_size)
        width = -(-int(max_length) // self.page_size)
        self.pages = torch.empty(layers, 2, n_pages, kv_heads, page_size, HEAD_DIM, dtype=dtype,
                                 device=device)
        self.exponents = None
        if dtype == torch.float8_e4m3fn:
            self.exponents = torch.empty(self.pages.shape[:-1], dtype=torch.float8_e8m0fnu, device=device)
        else:
            _attn_dtype(self.pages)
        self._held = self._views()
        ints = {"dtype": torch.int32, "device": self.pages.device}
        self.table = torch.full((slots, width), -1, **ints)
        self.lengths = torch.zeros(slots, **ints)
        self.refs = torch.zeros(n_pages, **ints)
        self._lacking = torch.zeros(2, **ints)
        self.shortfall = self._lacking[:1]  # the most pages that a call has lacked since the last check
        self.excess = self._lacking[1:]     # the most rows that a step has lacked

    @property
    def slots(self):
        return self.table.shape[0]

    @property
    def pool(self):
        """All pages, as the page bookkeeping takes them."""
        return self.pages if self.exponents is None else QuantizedPages(self.pages, self.exponents)

    def _views(self):
        """The layers as views, made once (made in every call, two to four of them take as long as its kernel's
        launch): every layer's keys, its values, and what they are views of, with the memory it was set to."""
        def views(which):
            codes = [self.pages[layer, which] for layer in range(self.pages.shape[0])]
            if self.exponents is None:
                return codes
            return [QuantizedPages(x, self.exponents[layer, which]) for layer, x in enumerate(codes)]

        held = [t if t is None else (t, t.detach(), t.dtype) for t in (self.pages, self.exponents)]
        return views(0), views(1), *held

    def _layer(self, layer, which):
        held = self._held
        pages, as_set, dtype = held[2]
        # (the program has set other pages, or the same tensor to other memory, sizes or another type)
        if pages is not self.pages or not pages.is_set_to(as_set) or pages.dtype is not dtype:
            held = self._held = self._views()
        elif held[3] is None:
            if self.exponents is not None:
                held = self._held = self._views()
        else:
            exponents, as_set, dtype = held[3]
            if exponents is not self.exponents or not exponents.is_set_to(as_set) or exponents.dtype is not dtype:
                held = self._held = self._views()
        return held[which][layer]

    def keys(self, layer):
        return self._layer(layer, 0)

    def values(self, layer):
        return self._layer(layer, 1)

    def _slots(self, values, fill):
        """One int32 per slot: a device tensor as it is, or `fill` with a host dict's entries."""
        if values is None or isinstance(values, torch.Tensor):
            return values
        out = list(fill)
        for slot, value in values.items():
            if not 0 <= slot < self.slots:
                raise ValueError(f"slot {slot} of {self.slots}")
            out[slot] = int(value)
        return torch.tensor(out, dtype=torch.int32, device=self.table.device)

    def remap(self, parents=None, new_lengths=None):
        """`remap_pages` on the cache's state. parents: (slots) int32 tensor or a dict {slot: parent}
        (the other slots go on as themselves); new_lengths: (slots) int32 tensor or None."""
        parents = self._slots(parents, range(self.slots))
        table, lengths, refs, shortfall = remap_pages(self.pool, self.table, self.lengths,
                                                      self.refs, parents, new_lengths)
        self.table.copy_(table)
        self.lengths.copy_(lengths)
        self.refs.copy_(refs)
        torch.maximum(self.shortfall, shortfall, out=self.shortfall)

    def fork(self, source, targets):
        """Each slot of `targets` goes on as a copy of slot `source` (what it held is given back)."""
        if not 0 <= source < self.slots:
            raise ValueError(f"slot {source} of {self.slots}")
        self.remap({t: source for t in targets})

    def free(self, slots):
        """The sequences of these slots are given up."""
        self.remap({s: -1 for s in slots})

    def step(self, q_lengths, n_tokens, heads, tree=None):
        """Room for `q_lengths[s]` new tokens of every slot, and the step's plan: `n_tokens` rows in
        all, no fewer than their sum. At most 4096 slots. Where pages are lacking, or device lengths sum
        to more than `n_tokens` (host lists are refused), no slot grows and every row of the plan is
        padding. `tree` as for `paged_plan`; `accept` then keeps a path of it."""
        n_tokens, kv_heads = int(n_tokens), self.pages.shape[3]
        _check_host_lengths(q_lengths, self.lengths, n_tokens, 0)
        # (a step that the plan would refuse is refused before a slot has grown)
        _plan_sizes(self.slots, n_tokens, heads, kv_heads, self.page_size, self.table.shape[1])
        if tree is not None:
            tree = _parents(tree, q_lengths, n_tokens, self.table.device)
        q = _lengths("q_lengths", q_lengths, self.slots, self.table.device)
        before = self.lengths.clone()
        self.remap(None, self._grown(q, n_tokens))
        return paged_plan(self.table, self.lengths - before, self.lengths, n_tokens, heads, kv_heads,
                          self.page_size, tree)

    def accept(self, plan, accepted):
        """Of the last step's new tokens (`plan`: what `step` returned) those up to `accepted[s]` on its
        path stay, `paged_accept`; pages that are not needed any more are given back. accepted: (slots)
        int32 tensor, or a dict {slot: number} (the other slots' new tokens go). Once per step, before
        any other call that changes the slots."""
        accepted = self._slots(accepted, [-1] * self.slots)
        self.remap(None, paged_accept(self.pool, plan, self.lengths, accepted))

    def _grown(self, q_lengths, n_tokens):
        """The slots' lengths with their new tokens, or as they are where those pass the rows."""
        device = self.table.device
        if device.index != _current_device():  # launches and allocations go to the tensors' device
            with torch.cuda.device(device):
                return self._grown(q_lengths, n_tokens)
        out = torch.empty_like(self.lengths)
        check(lib().va_pages_growth(self.lengths.data_ptr(), q_lengths.data_ptr(), self.slots, n_tokens,
                                    out.data_ptr(), self.excess.data_ptr(),
                                    _current_stream(device.index)), "va_pages_growth")
        return out

    def select(self, logits, scores, beams, ended=None, end_token=None):
        """Beam search over the slots, `beams` of them a prompt: `select_beams` on the slots' next-token
        logits (slots, vocab) and scores (slots), and every slot goes on as the one that it continues.
        Returns (scores, parents, tokens), each (slots): the slots' scores, the slots that they were, and
        their next tokens."""
        if logits.dim() != 2 or logits.shape[0] != self.slots:
            raise ValueError(f"logits must be ({self.slots}, vocab), got {tuple(logits.shape)}")
        scores, parents, tokens = (x.view(-1) for x in select_beams(logits, scores, beams, None, ended,
                                                                    end_token))
        self.remap(parents)
        return scores, parents, tokens

    def compact(self):
        """The live pages to the front of the pool; returns their number as a (1) int32 tensor."""
        table, refs, live = compact_pages(self.pool, self.table, self.lengths, self.refs)
        self.table.copy_(table)
        self.refs.copy_(refs)
        return live

    def check(self):
        """Raise if a call since the last check lacked pages or rows (reads the GPU)."""
        pages, rows = self._lacking.tolist()
        if pages or rows:
            self._lacking.zero_()
            what = f"{pages} pages" if pages else f"{rows} rows for a step's new tokens"
            raise RuntimeError(f"the paged cache lacked {what}: that call changed nothing")
