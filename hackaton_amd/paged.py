"""A paged key/value cache for answering with the model that `packed_attention` trains: the new
tokens of every sequence of a step are appended to pages and attend to them, one token each, a few
drafted ones or a prompt's chunk, all in one call. Hand-written gfx950 kernels through the C ABI; the
reference trains only and has no counterpart.

    paged_plan(page_table, q_lengths, kv_lengths, n_tokens, heads, kv_heads, page_size)
    paged_append(q, k, v, cos, sin, k_pages, v_pages, plan)
    paged_attention(query, k_pages, v_pages, plan, scale)
    remap_pages(pages, table, lengths, refs, parents, new_lengths)
    compact_pages(pages, table, lengths, refs)
    PagedCache       a pool, its page tables and the calls above on them

Pages hold `page_size` rows (a power of two, 16 to 256) of every key/value head: one layer's keys are
(n_pages, kv_heads, page_size, 128). Row t of a sequence lies in page `page_table[sequence, t //
page_size]`, row `t % page_size`; entries outside the pool name no page. Lengths, tables and counts are
int32 and stay on the GPU: no call reads them back, so a captured step follows them. None of the calls
has a backward or a forward-mode derivative; tensors that ask for one are refused.
"""

import ctypes
import functools

import torch
from torch.autograd import forward_ad

from . import _lib, attention
from ._lib import check, lib
from .attention import _DTYPES, HEAD_DIM, _attn_dtype, _rope_strides, _tables

PAGE_SIZES = (16, 32, 64, 128, 256)


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
    for t in tensors:
        if t.device != device:
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
                 "_capture")

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
        """(n_tokens) int32: the position of every row in its sequence, -1 for padding."""
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


def paged_plan(page_table, q_lengths, kv_lengths, n_tokens, heads, kv_heads, page_size):
    """The plan of a step: `q_lengths[s]` new tokens of every sequence (packed rows, one sequence
    after the other, `n_tokens` rows in all; rows behind the last sequence are padding) and
    `kv_lengths[s]` cached tokens with the new ones included. Both are host lists or device tensors
    (for a captured step: device tensors); `page_table` is (sequences, pages per sequence) int32 on
    the GPU, at most 4096 sequences. Device lengths are not read back: negative ones count as 0, kv
    lengths end with the table row, new tokens with the rows. One launch."""
    device = _one_device(page_table)
    if device.index != _current_device():  # launches and allocations go to the tensors' device
        with torch.cuda.device(device):
            return paged_plan(page_table, q_lengths, kv_lengths, n_tokens, heads, kv_heads,
                              page_size)
    if page_table.dim() != 2:
        raise ValueError(f"page_table must be (sequences, pages), got {tuple(page_table.shape)}")
    n_seqs, width = page_table.shape
    _int32("page_table", page_table, n_seqs, width)
    page_size, n_tokens = _page_size(page_size), int(n_tokens)
    _check_host_lengths(q_lengths, kv_lengths, n_tokens, width * page_size)
    plan = PagedPlan()
    n_words, plan.workspace_bytes = _plan_sizes(n_seqs, n_tokens, heads, kv_heads, page_size, width)
    q_lengths = _lengths("q_lengths", q_lengths, n_seqs, device)
    kv_lengths = _lengths("kv_lengths", kv_lengths, n_seqs, device)
    plan.page_table, plan.n_tokens, plan.n_seqs = page_table, n_tokens, n_seqs
    plan.heads, plan.kv_heads, plan.page_size = heads, kv_heads, page_size
    plan._page = (kv_heads, page_size, HEAD_DIM)
    plan._strides = (page_size * HEAD_DIM, HEAD_DIM, 1)
    plan.words = torch.empty(n_words, dtype=torch.int32, device=device)
    plan._stream = _current_stream(device.index)
    plan._capture = attention._capture_id() if torch._C._cuda_isCurrentStreamCapturing() else None
    plan._step = _lib.PagedStep(page_table.data_ptr(), plan.words.data_ptr(), n_tokens, n_seqs, width,
                                page_size, heads, kv_heads)
    check(lib().va_paged_plan(plan._step, q_lengths.data_ptr(), kv_lengths.data_ptr(), n_words,
                              plan._stream), "va_paged_plan")
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


def paged_append(q, k, v, cos, sin, k_pages, v_pages, plan):
    """The step's new rows: q (n_tokens, heads * 128), k and v (n_tokens, kv_heads * 128) projections
    in fp16, bf16 or fp32. Returns q rotated, (n_tokens, heads, 128) in the pages' type; k rotated and
    v go into `k_pages` / `v_pages` (n_pages, kv_heads, page_size, 128) at the rows' positions, rotated
    in fp32 and rounded once. cos / sin: (1 or sequences, T, 128) read by position, or (n_tokens, 128)
    read by row. Rows without a place (padding, positions past the tables or in no page) write
    nothing; padding and positions outside the cos / sin table give zeros in q."""
    device = _one_device(q, k, v, cos, sin, k_pages, v_pages, plan.words)
    if device.index != _current_device():  # launches and allocations go to the tensors' device
        with torch.cuda.device(device):
            return paged_append(q, k, v, cos, sin, k_pages, v_pages, plan)
    _no_grad(q, k, v, k_pages, v_pages)
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
    out_dtype = _attn_dtype(k_pages)
    k_stride, v_stride, n_pages = _pages_of(k_pages, v_pages, plan)
    by_row = cos.dim() == 2
    if by_row and (tuple(cos.shape) != (n, HEAD_DIM) or sin.shape != cos.shape):
        raise ValueError(f"cos/sin by row must be ({n}, {HEAD_DIM}), got {tuple(cos.shape)}, "
                         f"{tuple(sin.shape)}")
    cos, sin = _tables(cos[None] if by_row else cos, sin[None] if by_row else sin)
    if not by_row and cos.shape[0] not in (1, plan.n_seqs):
        raise ValueError(f"cos/sin for {cos.shape[0]} sequences, the plan has {plan.n_seqs}")
    query = torch.empty((n, heads, HEAD_DIM), dtype=k_pages.dtype, device=device)
    if n == 0:
        return query
    if cos.shape[1] == 0:
        raise ValueError("cos/sin hold no positions")
    batch, row = (0, 0) if by_row else _rope_strides(cos)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
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
    page holds behind its sequence's end is never read. (Keys that a row does not see never reach it,
    whatever they hold. Values that are infinite or not a number do where they lie in a 64-key tile that
    another of the 32 rows computed together sees, rows being pairs of a token and a query head of the
    group: in rows of the same sequence up to 63 + ceil(31 kv_heads / heads) positions before their own.)
    The same step gives the same bits; the same sequence in another step agrees to rounding."""
    device = _one_device(query, k_pages, v_pages, plan.words)
    if device.index != _current_device():  # launches and allocations go to the tensors' device
        with torch.cuda.device(device):
            return paged_attention(query, k_pages, v_pages, plan, scale)
    _no_grad(query, k_pages, v_pages)
    dtype = _attn_dtype(query)
    if k_pages.dtype != query.dtype:
        raise ValueError(f"query in {query.dtype}, pages in {k_pages.dtype}")
    n, heads = plan.n_tokens, plan.heads
    if query.shape != (n, heads, HEAD_DIM):
        raise ValueError(f"query must be ({n}, {heads}, {HEAD_DIM}), got {tuple(query.shape)}")
    k_stride, v_stride, n_pages = _pages_of(k_pages, v_pages, plan)
    query = query.contiguous()
    out = torch.empty((n, heads * HEAD_DIM), dtype=query.dtype, device=device)
    if n == 0:
        return out
    nbytes = plan.workspace_bytes
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    check(lib().va_paged_attention(
        plan._step, query.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), k_stride, v_stride,
        n_pages, HEAD_DIM, scale, dtype, out.data_ptr(), ws.data_ptr() if nbytes else None, nbytes,
        plan._use()), "va_paged_attention")
    return out


# ------------------------------------------------------------------------------------------------
# page bookkeeping
# ------------------------------------------------------------------------------------------------
def _pool_of(pages):
    shape = pages.shape
    if len(shape) != 6 or shape[1] != 2 or shape[5] != HEAD_DIM:
        raise ValueError(f"pages must be (layers, 2, n_pages, kv_heads, page_size, {HEAD_DIM}), got "
                         f"{tuple(shape)}")
    if not pages.is_contiguous():
        raise ValueError(f"pages must be contiguous, got strides {pages.stride()}")
    _attn_dtype(pages)
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
    device = _one_device(pages, table, lengths, refs,
                         *(t for t in (parents, new_lengths) if t is not None))
    if device.index != _current_device():  # launches and allocations go to the tensors' device
        with torch.cuda.device(device):
            return remap_pages(pages, table, lengths, refs, parents, new_lengths)
    _no_grad(pages)
    outer, n_pages, kv_heads, page_size = _pool_of(pages)
    slots, width = _state_of(n_pages, table, lengths, refs, parents=parents, new_lengths=new_lengths)
    table_out, lengths_out, refs_out = (torch.empty_like(table), torch.empty_like(lengths),
                                        torch.empty_like(refs))
    shortfall = torch.empty(1, dtype=torch.int32, device=device)
    words = _scratch_words(slots, n_pages)
    scratch = torch.empty(words, dtype=torch.int32, device=device)
    check(lib().va_pages_remap(
        pages.data_ptr(), outer, n_pages, kv_heads, page_size, HEAD_DIM, table.data_ptr(),
        lengths.data_ptr(), refs.data_ptr(), None if parents is None else parents.data_ptr(),
        None if new_lengths is None else new_lengths.data_ptr(), slots, width, table_out.data_ptr(),
        lengths_out.data_ptr(), refs_out.data_ptr(), shortfall.data_ptr(), scratch.data_ptr(), words,
        _current_stream(device.index)), "va_pages_remap")
    return table_out, lengths_out, refs_out, shortfall


def compact_pages(pages, table, lengths, refs):
    """The live pages (refs > 0) to the front of the pool: the k-th live page at or past their number
    moves to the k-th free page below it, in every layer. Arguments as for `remap_pages`. Returns
    new (table, refs, live); live (1): how many pages are in use, all of them below that number. Pages
    that the program holds without a table row move too: a row of their own keeps track of them."""
    device = _one_device(pages, table, lengths, refs)
    if device.index != _current_device():  # launches and allocations go to the tensors' device
        with torch.cuda.device(device):
            return compact_pages(pages, table, lengths, refs)
    _no_grad(pages)
    outer, n_pages, kv_heads, page_size = _pool_of(pages)
    slots, width = _state_of(n_pages, table, lengths, refs)
    table_out, refs_out = torch.empty_like(table), torch.empty_like(refs)
    live = torch.empty(1, dtype=torch.int32, device=device)
    words = _scratch_words(slots, n_pages)
    scratch = torch.empty(words, dtype=torch.int32, device=device)
    check(lib().va_pages_compact(
        pages.data_ptr(), outer, n_pages, kv_heads, page_size, HEAD_DIM, table.data_ptr(),
        lengths.data_ptr(), refs.data_ptr(), slots, width, table_out.data_ptr(), refs_out.data_ptr(),
        live.data_ptr(), scratch.data_ptr(), words, _current_stream(device.index)),
        "va_pages_compact")
    return table_out, refs_out, live


class PagedCache:
    """Keys and values of `layers` layers in one pool of `n_pages` pages, and up to `slots` sequences
    of at most `max_length` tokens (rounded up to whole pages) in it. State, all on the GPU: `pages`,
    `table`, `lengths`, `refs`. Every call updates it in place on the current stream, so the calls of one
    cache belong on one stream or in order across streams, and a captured step replays on the state it
    finds. A call that lacks pages (or a step that lacks rows) changes nothing; `check()` reports it."""

    def __init__(self, layers, n_pages, page_size, kv_heads, slots, max_length,
                 dtype=torch.float16, device="cuda"):
        self.page_size = _page_size(page_size)
        width = -(-int(max_length) // self.page_size)
        self.pages = torch.empty(layers, 2, n_pages, kv_heads, page_size, HEAD_DIM, dtype=dtype,
                                 device=device)
        _attn_dtype(self.pages)
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

    def keys(self, layer):
        return self.pages[layer, 0]

    def values(self, layer):
        return self.pages[layer, 1]

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
        table, lengths, refs, shortfall = remap_pages(self.pages, self.table, self.lengths,
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

    def step(self, q_lengths, n_tokens, heads):
        """Room for `q_lengths[s]` new tokens of every slot, and the step's plan: `n_tokens` rows in
        all, no fewer than their sum. At most 4096 slots. Where pages are lacking, or device lengths sum
        to more than `n_tokens` (host lists are refused), no slot grows and every row of the plan is
        padding."""
        n_tokens, kv_heads = int(n_tokens), self.pages.shape[3]
        _check_host_lengths(q_lengths, self.lengths, n_tokens, 0)
        # (a step that the plan would refuse is refused before a slot has grown)
        _plan_sizes(self.slots, n_tokens, heads, kv_heads, self.page_size, self.table.shape[1])
        q = _lengths("q_lengths", q_lengths, self.slots, self.table.device)
        before = self.lengths.clone()
        self.remap(None, self._grown(q, n_tokens))
        return paged_plan(self.table, self.lengths - before, self.lengths, n_tokens, heads, kv_heads,
                          self.page_size)

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

    def compact(self):
        """The live pages to the front of the pool; returns their number as a (1) int32 tensor."""
        table, refs, live = compact_pages(self.pages, self.table, self.lengths, self.refs)
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
