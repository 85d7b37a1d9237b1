"""Plain 64-bit references of 8-bit pages and of trees of new tokens, on the CPU."""

import math

import numpy as np
import torch

from tests import paged_oracle as orc
from tests.paged_oracle import DIM, SCALE

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
LEAST = -100  # exponent of the smallest power of two of a row


def exponent_of(x):
    """The smallest exponent >= -100 whose power brings a row's largest finite number to 448 or less."""
    size = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1).double()
    out = torch.full(size.shape, float(LEAST), dtype=torch.float64)
    for e in range(LEAST, 130):
        out = torch.where(size > 448 * 2.0 ** e, e + 1.0, out)
    return out


def e4m3(x):
    """64-bit numbers of size 448 at most, rounded to e4m3 by its definition: three digits after the
    leading one, exponents from -6 on, to nearest even; not finite: not a number."""
    lead = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(lead - 3)
    return torch.where(torch.isfinite(x), torch.round(x / step) * step, math.nan)


def quantize(x):
    """(numbers, exponents) of rows, 64 bits."""
    e = exponent_of(x)
    return e4m3(x.double() / torch.exp2(e)[..., None]), e


def bytes_of(numbers, exponents):
    """The same as float8_e4m3fn and float8_e8m0fnu (exactly: the numbers are e4m3 ones)."""
    return numbers.float().to(E4M3), (exponents + 127).to(torch.uint8).view(E8M0)


def values(codes, exponents):
    return codes.double() * torch.exp2(exponents.view(torch.uint8).double() - 127)[..., None]


def case8(seed, q_lengths, kv_lengths, heads, kv_heads, dtype, page_size, padding=0, width=None, qk=1.0,
          spread=0):
    """(query, (k codes, k exponents), (v codes, v exponents), (k, v) values in 64 bits, table): rows that no
    sequence uses hold not-a-number codes and exponents. `spread`: rows of sizes 2^-spread to 2^spread."""
    query, k, v, table = orc.paged_case(seed, q_lengths, kv_lengths, heads, kv_heads, torch.float32,
                                        page_size, padding, width=width, qk=qk)
    query = query.to(dtype)
    gen = torch.Generator().manual_seed(seed + 1)
    out = []
    for pool in (k, v):
        stale = torch.isnan(pool).all(-1)
        if spread:
            pool = pool * torch.exp2(torch.randint(-spread, spread + 1, stale.shape, generator=gen))[..., None]
        numbers, exponents = quantize(torch.where(stale[..., None], 0.0, pool))
        codes, exps = bytes_of(numbers, exponents)
        codes.view(torch.uint8)[stale] = 0x7f
        exps.view(torch.uint8)[stale] = 0xff
        out.append((codes, exps))
    return query, *out, [torch.nan_to_num(values(*x)) for x in out], table


def paths(parents):
    """(tokens, tokens): whether the second is on the path of the first, itself included."""
    on = np.zeros((len(parents), len(parents)), dtype=bool)
    for j, p in enumerate(parents):
        if 0 <= p < j:
            on[j] = on[p]
        on[j, j] = True
    return on


def attention(query, k_pool, v_pool, table, q_lengths, kv_lengths, trees=None, scale=SCALE):
    """(out, sum of weight * |value|) (n, heads, DIM) as orc.attention, over (n_pages, kv_heads, page_size,
    DIM) values; trees: per sequence the parents of its new tokens (None: they follow each other)."""
    n, heads, _ = query.shape
    group = heads // k_pool.shape[1]
    out = torch.zeros(n, heads, DIM, dtype=torch.float64)
    size = torch.zeros_like(out)
    at = 0
    for s, (new, kv) in enumerate(zip(q_lengths, kv_lengths)):
        k, v = orc.rows_of(k_pool, table[s], kv), orc.rows_of(v_pool, table[s], kv)
        on = np.tril(np.ones((new, new), dtype=bool)) if trees is None else paths(trees[s])
        for j in range(new):
            seen = np.concatenate((np.ones(max(kv - new, 0), dtype=bool), on[j][max(new - kv, 0):]))
            seen = torch.from_numpy(np.nonzero(seen[:kv])[0])
            if kv - new + j < 0 or not len(seen):
                continue
            for h in range(heads):
                z = k[h // group, seen] @ query[at + j, h].double() * scale
                w = torch.softmax(z, 0)
                out[at + j, h] = w @ v[h // group, seen]
                size[at + j, h] = w @ v[h // group, seen].abs()
        at += new
    return out, size


def random_tree(rng, count, span):
    """Parents of `count` tokens: each one of the last `span` before it, now and then none."""
    return [-1 if j == 0 or rng.random() < 0.08 else int(rng.integers(max(0, j - span), j))
            for j in range(count)]
