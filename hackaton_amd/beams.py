"""Beam search's selection: the best continuations of every prompt's beams by their next-token logits, by
hand-written gfx950 kernels through the C ABI; the reference trains only and has no counterpart. The rows
that the chosen continuations go on from are the `parents` of `remap_pages` and `PagedCache.remap`;
`PagedCache.select` does both.

    select_beams(logits, scores, beams, count, ended, end_token)
"""

import ctypes
import functools

import torch
from torch.autograd import forward_ad

from ._lib import check, lib
from .attention import _DTYPES

_current_device = torch._C._cuda_getDevice
_current_stream = torch._C._cuda_getCurrentRawStream


@functools.lru_cache(maxsize=64)
def _workspace_bytes(groups, beams, vocab):
    nbytes = ctypes.c_int64()
    check(lib().va_select_beams_workspace(groups, beams, vocab, ctypes.byref(nbytes)),
          "va_select_beams_workspace")
    return nbytes.value


def select_beams(logits, scores, beams, count=None, ended=None, end_token=None):
    """The `count` (1 to 64; None: `beams`) best continuations of every prompt. logits (rows, vocab) in
    fp16, bf16 or fp32, rows next to each other or apart, vocab at most 2^18; rows g * beams to
    (g + 1) * beams - 1 are the beams (at most 64) of prompt g. scores (rows) fp32: the beams' sums of log
    probabilities so far (-inf: a beam that is not used yet). A continuation's score is its beam's plus
    the token's log softmax, formed and compared in 64 bits (the row's exponentials are summed in 32 by
    every wave of a work-group, in 64 over them); what is not a number counts as -inf. Tokens that are not allowed
    are best masked with -inf: beside numbers past some 10^10 the logarithm of the sum loses digits, and a row
    that holds nothing but fp32's or bf16's lowest number scores as its beam, for every token.

    Returns (scores (prompts, count) fp32, parents (prompts, count) int32: the row that each goes on from,
    tokens (prompts, count) int32), the best first, ties to the lowest row and token: the order of a
    stable sort of all continuations, but for those of rows that differ whose scores are within the error of the rows'
    sums (2.1e-5 at most at 32,000 tokens, 1.3e-4 at 2^18, both rows together). ended (rows) bool: beams
    that have ended; their logits are not read, they go on with `end_token` at their score, and at -inf with
    every other token. Nothing is read back, so a captured step follows its inputs. No backward: a choice has none, and the scores' is refused."""
    device = logits.device
    if not logits.is_cuda:
        raise ValueError(f"the selection runs on the GPU only: got a tensor on {device}")
    if device.index != _current_device():  # launches and allocations go to the tensors' device
        with torch.cuda.device(device):
            return select_beams(logits, scores, beams, count, ended, end_token)
    if torch.is_grad_enabled() and (logits.requires_grad or scores.requires_grad):
        raise RuntimeError("the selection has no backward: call it under torch.no_grad() or "
                           "torch.inference_mode()")
    if forward_ad._current_level >= 0:  # inside forward_ad.dual_level()
        for t in (logits, scores):
            if forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("the selection has no forward-mode derivative: pass the primals "
                                   "(torch.autograd.forward_ad.unpack_dual)")
    if logits.dim() != 2 or logits.dtype not in _DTYPES:
        raise ValueError(f"logits must be (rows, vocab) in fp16, bf16 or fp32, got {tuple(logits.shape)} in "
                         f"{logits.dtype}")
    rows, vocab = logits.shape
    beams = int(beams)
    count = beams if count is None else int(count)
    if beams < 1 or rows % beams != 0:
        raise ValueError(f"{rows} rows are no whole number of prompts of {beams} beams")
    if scores.shape != (rows,) or scores.dtype != torch.float32 or scores.device != device:
        raise ValueError(f"scores must be ({rows},) in fp32 on {device}, got {tuple(scores.shape)} in "
                         f"{scores.dtype} on {scores.device}")
    if ended is not None and end_token is None:
        raise ValueError("ended beams go on with an end_token: give both")
    if ended is not None and (ended.shape != (rows,) or ended.dtype != torch.bool or ended.device != device):
        raise ValueError(f"ended must be ({rows},) in bool on {device}, got {tuple(ended.shape)} in "
                         f"{ended.dtype} on {ended.device}")
    groups = rows // beams
    nbytes = _workspace_bytes(groups, beams, vocab)
    if vocab > 1 and logits.stride(1) != 1 or rows > 1 and logits.stride(0) < vocab:
        logits = logits.contiguous()
    scores = scores.contiguous()
    if ended is not None:
        ended = ended.contiguous()
    if not 1 <= count < 1 << 20:
        raise ValueError(f"count must be 1 to 64, got {count}")
    out = torch.empty(groups, count, dtype=torch.float32, device=device)
    parents = torch.empty(groups, count, dtype=torch.int32, device=device)
    tokens = torch.empty_like(parents)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    check(lib().va_select_beams(
        logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0), groups, beams, vocab,
        scores.data_ptr(), None if ended is None else ended.data_ptr(),
        0 if end_token is None else max(-1, min(int(end_token), vocab)), count, out.data_ptr(),
        parents.data_ptr(), tokens.data_ptr(), ws.data_ptr(), nbytes, _current_stream(device.index)),
        "va_select_beams")
    return out, parents, tokens
