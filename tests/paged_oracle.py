"""Plain 64-bit references of the paged cache's operators, on the CPU, page by page and slot by slot."""

import math

import numpy as np
import torch

DIM = 128
SCALE = DIM ** -0.5
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def rows_of(pool, table_row, tokens):
    """(kv_heads, tokens, DIM) in 64 bits; entries outside the pool give zeros."""
    n_pages, kv_heads, ps, _ = pool.shape
    out = torch.zeros(kv_heads, max(tokens, 0), DIM, dtype=torch.float64)
    for t in range(0, tokens, ps):
        page, count = int(table_row[t // ps]), min(ps, tokens - t)
        if 0 <= page < n_pages:
            out[:, t:t + count] = pool[page, :, :count].double()
    return out


def attention(query, k_pool, v_pool, table, q_lengths, kv_lengths, scale=SCALE):
    """(out, sum of weight * |value|) (n, heads, DIM): zeros for padding and rows without a key."""
    n, heads, _ = query.shape
    group = heads // k_pool.shape[1]
    out = torch.zeros(n, heads, DIM, dtype=torch.float64)
    size = torch.zeros_like(out)
    at = 0
    for s, (new, kv) in enumerate(zip(q_lengths, kv_lengths)):
        k, v = rows_of(k_pool, table[s], kv), rows_of(v_pool, table[s], kv)
        for j in range(new):
            pos = kv - new + j
            if pos < 0:
                continue
            for h in range(heads):
                z = k[h // group, :pos + 1] @ query[at + j, h].double() * scale
                w = torch.softmax(z, 0)
                out[at + j, h] = w @ v[h // group, :pos + 1]
                size[at + j, h] = w @ v[h // group, :pos + 1].abs()
        at += new
    return out, size


def attention_bound(out, size, dtype, qk=1.0):
    """How far a 16-bit result may be from `out`, with `size` the weighted sum of |values|: the result's
    rounding, half a step of it; each weight rounded to 16 bits for the product with the values, half a
    step in the numerator and, where the sum is over the rounded weights, in the denominator; the scores'
    sums of 128 products in fp32, off by at most 128 * 2^-24 times the sum of the products' sizes, which
    is about 128 * 0.64 * qk^2 * SCALE = 7.2 qk^2 for normal queries and keys of size qk: 2^-14 qk^2 in a
    score, twice that in a normalised weight. (The fp32 sums over the keys add the root of their count
    times 2^-24, less than 2^-16.)"""
    u = HALF_STEP[dtype]
    return u * out.abs() * (1 + 2 * u) + (2 * u + 2.0 ** -13 * qk ** 2 + 2.0 ** -16) * size + 2.0 ** -24


def rotate(x, cos, sin):
    """(n, heads, DIM) in 64 bits with tables (n, DIM)."""
    half = DIM // 2
    turned = torch.cat((-x[..., half:], x[..., :half]), -1)
    return x * cos[:, None].double() + turned * sin[:, None].double()


def remap(table, lengths, refs, parents, new_lengths, page_size):
    """(table, lengths, refs, shortfall, [(source, target, rows)]) from lists."""
    slots, width, pages = len(table), len(table[0]) if table else 0, len(refs)
    ids = range(slots)
    parents = [i for i in ids] if parents is None else [p if 0 <= p < slots else -1 for p in parents]
    had = [min(max(lengths[p], 0), width * page_size) if p >= 0 else 0 for p in parents]
    wanted = had if new_lengths is None else [max(x, 0) for x in new_lengths]
    kept = [min(h, w) for h, w in zip(had, wanted)]
    rows = [list(table[p][:-(-k // page_size)]) if p >= 0 else [] for p, k in zip(parents, kept)]
    refs_out = list(refs)
    for row, length in zip(table, lengths):
        for page in row[:-(-min(max(length, 0), width * page_size) // page_size)]:
            if 0 <= page < pages:
                refs_out[page] -= 1
    for row, k in zip(rows, kept):
        for page in row[:k // page_size]:
            if 0 <= page < pages:
                refs_out[page] += 1
    tails = {row[-1] for row, k in zip(rows, kept) if k % page_size}
    free = [p for p in range(pages) if refs_out[p] <= 0 and p not in tails]
    need, beyond, copies = 0, 0, []
    for row, k, w in zip(rows, kept, wanted):
        if k % page_size and 0 <= row[-1] < pages:
            if refs_out[row[-1]] > 0:
                target = free[need] if need < len(free) else None
                copies.append((row[-1], target, k % page_size))
                row[-1] = target
                need += 1
            else:
                refs_out[row[-1]] = 1
        for _ in range(-(-w // page_size) - -(-k // page_size)):
            row.append(free[need] if need < len(free) else None)
            need += 1
        beyond += max(0, -(-w // page_size) - width)
    shortfall = max(0, need - len(free)) + beyond
    if shortfall:
        return table, lengths, refs, shortfall, []
    for page in free[:need]:
        refs_out[page] = 1
    return [r + [-1] * (width - len(r)) for r in rows], wanted, refs_out, 0, copies


def compact(table, lengths, refs, page_size):
    """(table, refs, live, [(source, target)]) from lists."""
    live = sum(r > 0 for r in refs)
    holes = [p for p in range(live) if refs[p] <= 0]
    movers = [p for p in range(live, len(refs)) if refs[p] > 0]
    place = {p: p for p in range(live)}
    place.update(zip(movers, holes))
    counts = [0] * len(refs)
    for p, r in enumerate(refs):
        if r > 0:
            counts[place[p]] = r
    width = len(table[0]) if table else 0
    out = []
    for row, n in zip(table, lengths):
        used = row[:-(-n // page_size)]
        out.append([place[p] for p in used] + [-1] * (width - len(used)))
    return out, counts, live, list(zip(movers, holes))


def random_state(rng, slots, width, pages, page_size, pins=0):
    """A consistent (table, lengths, refs): rows share leading full pages with earlier rows, and the
    program holds `pins` pages itself."""
    order, refs = [int(x) for x in rng.permutation(pages)], [0] * pages
    table, lengths = [], []
    for i in range(slots):
        length = int(rng.integers(0, width * page_size + 1)) if rng.random() < 0.85 else 0
        row = []
        if i and rng.random() < 0.5:
            other = int(rng.integers(0, i))
            row = table[other][:min(length, lengths[other]) // page_size]
            row = row[:int(rng.integers(0, len(row) + 1))]
        while len(row) < -(-length // page_size):
            if not order:
                break
            row.append(order.pop())
        length = min(length, len(row) * page_size)
        for p in row:
            refs[p] += 1
        table.append(row)
        lengths.append(length)
    for _ in range(pins):
        refs[int(rng.integers(0, pages))] += 1
    return [r + [-1] * (width - len(r)) for r in table], lengths, refs


def paged_case(seed, q_lengths, kv_lengths, heads, kv_heads, dtype, page_size, padding=0,
               stale=math.nan, width=None, qk=1.0):
    """(query, k_pool, v_pool, table) on the CPU: pages in any order, rows that no sequence uses
    `stale`."""
    gen = torch.Generator().manual_seed(seed)
    counts = [-(-x // page_size) for x in kv_lengths]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=gen).tolist()
    pools = [torch.full((pages, kv_heads, page_size, DIM), stale, dtype=dtype) for _ in range(2)]
    table = np.full((len(counts), width or max(counts + [0]) + 2), -1, dtype=np.int32)
    for s, (c, kv) in enumerate(zip(counts, kv_lengths)):
        for j in range(c):
            table[s, j] = page = order.pop()
            rows = min(page_size, kv - j * page_size)
            for pool, size in zip(pools, (qk, 1.0)):
                pool[page, :, :rows] = (torch.randn(kv_heads, rows, DIM, generator=gen) * size).to(dtype)
    n = sum(q_lengths) + padding
    query = (torch.randn(n, heads, DIM, generator=gen) * qk).to(dtype)
    return query, pools[0], pools[1], torch.from_numpy(table)
