"""8-bit pages under fp16 queries whose rows leave fp16's range: so small that their values fall below its normal
numbers (2^-14) or its smallest step (2^-24), where each is multiplied as the fp16 number next to it, or so large
that they pass 65504. And rows of all the exponents that a row may have."""

import pytest
import torch

from hackaton_amd import paged_attention, paged_plan
from tests import paged8_oracle as o8
from tests import paged_oracle as orc
from tests.paged_oracle import DIM, SCALE
from tests.test_gpu_paged import banner
from tests.test_gpu_paged8 import cuda

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16
CASES = [([1, 1], [300, 33], 12, 2), ([50, 1], [200, 64], 12, 2), ([300], [340], 4, 2), ([3], [5000], 7, 1)]


def smaller(pages, values, shift):
    """The same rows times 2^-shift, exactly."""
    codes, exps = pages
    raw = exps.view(torch.uint8)
    raw = torch.where(raw == 255, raw, raw - shift)
    return (codes, raw.view(o8.E8M0)), values * 2.0 ** -shift


@pytest.mark.parametrize("shift", [8, 12, 16, 20, 24, 30])
@pytest.mark.parametrize("q,kv,heads,kv_heads", CASES)
def test_small_values(q, kv, heads, kv_heads, shift):
    """A value's rounding is half a step of fp16's smallest numbers at most, 2^-25, and the weights of a row,
    rounded, add up to less than 1 + 2^-10."""
    banner("small values", q, kv, heads, kv_heads, shift)
    for dtype, more in ((FP16, 2.0 ** -25 * (1 + 2.0 ** -10)), (BF16, 0.0)):
        query, k, v, (k64, v64), table = o8.case8(shift, q, kv, heads, kv_heads, dtype, 16)
        v, v64 = smaller(v, v64, shift)
        plan = paged_plan(table.cuda(), q, kv, sum(q), heads, kv_heads, 16)
        out = paged_attention(query.cuda(), cuda(k), cuda(v), plan, SCALE).cpu().double().view(sum(q), heads, DIM)
        ref, size = o8.attention(query, k64, v64, table, q, kv)
        assert ((out - ref).abs() <= orc.attention_bound(ref, size, dtype) + more).all()


@pytest.mark.parametrize("shift", [8, 12, 16])
@pytest.mark.parametrize("q,kv,heads,kv_heads", CASES[:3])
def test_small_keys(q, kv, heads, kv_heads, shift):
    """Keys of 2^-shift under a scale of 2^shift. A key's rounding of 2^-25 moves a score by the sum of the
    query's sizes times that, and a normalised weight by twice as much of itself."""
    banner("small keys", q, kv, heads, kv_heads, shift)
    query, k, v, (k64, v64), table = o8.case8(shift, q, kv, heads, kv_heads, FP16, 16)
    k, k64 = smaller(k, k64, shift)
    scale = SCALE * 2.0 ** shift
    plan = paged_plan(table.cuda(), q, kv, sum(q), heads, kv_heads, 16)
    out = paged_attention(query.cuda(), cuda(k), cuda(v), plan, scale).cpu().double().view(sum(q), heads, DIM)
    ref, size = o8.attention(query, k64, v64, table, q, kv, scale=scale)
    more = torch.expm1(2 * query.double().abs().sum(-1, keepdim=True) * 2.0 ** -25 * scale)
    assert ((out - ref).abs() <= orc.attention_bound(ref, size, FP16) + more * (size + 2.0 ** -24)).all()


@pytest.mark.parametrize("count", [1, 3, 40])
def test_large_values(count):
    """Values past 65504 are infinite under fp16 queries and numbers under bf16 ones."""
    banner("large values", count)
    q, kv = [count], [40]
    for dtype in (FP16, BF16):
        query, k, v, (k64, v64), table = o8.case8(1, q, kv, 4, 2, dtype, 16)
        numbers, exponents = o8.quantize(torch.full(v64.shape, 65536.0, dtype=torch.float64))
        v, v64 = o8.bytes_of(numbers, exponents), numbers * torch.exp2(exponents)[..., None]
        assert (v64 == 65536).all()
        plan = paged_plan(table.cuda(), q, kv, count, 4, 2, 16)
        out = paged_attention(query.cuda(), cuda(k), cuda(v), plan, SCALE).cpu().double().view(count, 4, DIM)
        ref, size = o8.attention(query, k64, v64, table, q, kv)
        if dtype == FP16:  # (rows before the last one have keys beside them that they do not see: no weight times infinity)
            assert (out[-1] == torch.inf).all() and not torch.isfinite(out).any()
        else:
            assert ((out - ref).abs() <= orc.attention_bound(ref, size, dtype)).all()


@pytest.mark.parametrize("count", [1, 40])
def test_every_exponent(count):
    """Sequences whose values have exponent bytes of 1 to 254, under bf16 queries: numbers of 2^-112 to 2^118 and
    what lies on both sides of them (above bf16's range: infinite; below its normal numbers: zero or as they are)."""
    banner("every exponent", count)
    q, kv = [count] * 254, [count] * 254
    query, k, _, (k64, _), table = o8.case8(2, q, kv, 2, 1, BF16, 64)
    codes = torch.full((*k[0].shape[:-1], DIM), 1.5).to(o8.E4M3)  # (every number of a row 1.5)
    exps = torch.full(k[1].shape, 127, dtype=torch.uint8)
    for s in range(254):
        exps[int(table[s, 0])] = s + 1
    v = (codes, exps.view(o8.E8M0))
    plan = paged_plan(table.cuda(), q, kv, sum(q), 2, 1, 64)
    out = paged_attention(query.cuda(), cuda(k), cuda(v), plan, SCALE).cpu().double().view(254, count, 2, DIM)
    want = 1.5 * torch.exp2(torch.arange(1, 255).double() - 127)
    off = (out / want[:, None, None, None] - 1).abs()
    assert (off[14:244] <= 2.0 ** -8 * 4).all()  # (the weights' rounding, twice, and the result's)
    assert torch.isfinite(out[:14]).all() and (out[:14].abs() <= 2 * want[:14, None, None, None]).all()
