"""A whole model that answers through the patched layers: drafted trees of which a path stays, beams, and a
cache in 8 bits."""

import numpy as np
import pytest
import torch

from hackaton_amd import PagedCache
from tests import paged8_oracle as o8
from tests.test_gpu_beams import reference as best_of
from tests.test_gpu_paged import banner, ints
from tests.test_patch import DIM, HEADS, HIDDEN, KV_HEADS, patched, tiny_model  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu
NO_MASK = {"full_attention": None}


def step_of(model, cache, tokens, q, tree=None):
    """Logits of a step's rows (two more than needed are padding), and its plan."""
    n = sum(q) + 2
    plan = cache.step(ints(q), n, HEADS, None if tree is None else ints(sum(tree, []) + [0, 0]))
    rows = torch.nn.functional.pad(torch.tensor(tokens, device="cuda"), (0, 2))
    out = model(input_ids=rows[None], position_ids=plan.positions.clamp(min=0).long()[None],
                attention_mask=NO_MASK, paged=(cache, plan), use_cache=False).logits[0]
    return out[:sum(q)], plan


def dense(model, tokens):
    return model(input_ids=torch.tensor(tokens, device="cuda")[None], use_cache=False).logits[0]


# (logits of an fp32 model over fp16 pages: two layers, each off by six half steps of fp16 of its size, 3e-3,
# in logits of size up to 2)
LOGITS = 1.2e-2


def test_drafted_trees_of_a_model(patched):  # noqa: F811
    """Every drafted token's logits are those of the dense model over the prompt and the token's path; after
    a path is accepted the slot goes on from it."""
    banner("a model that drafts")
    model, rng = tiny_model("cuda").eval(), np.random.default_rng(3)
    cache = PagedCache(2, 32, 16, KV_HEADS, 3, 128)
    with torch.inference_mode():
        text = [rng.integers(0, 1000, n).tolist() for n in (17, 40, 5)]
        step_of(model, cache, sum(text, []), [len(t) for t in text])
        for q, last in (([7, 20, 1], [5, 12, 0]), ([12, 0, 9], [-1, 3, 8]), ([3, 11, 16], [2, 10, 7])):
            tree = [o8.random_tree(rng, n, 4) for n in q]
            drafts = [rng.integers(0, 1000, n).tolist() for n in q]
            logits, plan = step_of(model, cache, sum(drafts, []), q, tree)
            at = 0
            for s, n in enumerate(q):
                on = o8.paths(tree[s])
                for j in range(n):
                    path = [drafts[s][i] for i in np.nonzero(on[j])[0]]
                    assert int(plan.positions[at + j]) == len(text[s]) + len(path) - 1
                    want = dense(model, text[s] + path)[-1]
                    assert (logits[at + j] - want).abs().max() <= LOGITS, (s, j)
                if 0 <= last[s] < n:
                    text[s] += [drafts[s][i] for i in np.nonzero(on[last[s]])[0]]
                at += n
            cache.accept(plan, ints(last))
            assert cache.lengths.tolist() == [len(t) for t in text]
        cache.check()


@pytest.mark.parametrize("held", [torch.float16, o8.E4M3])
def test_beams_of_a_model(patched, held):  # noqa: F811
    """Two prompts of four beams: each turn takes the best continuations of the logits that it has, and the
    next logits are those of every beam's own tokens."""
    banner("a model with beams", held)
    model, rng = tiny_model("cuda").eval(), np.random.default_rng(4)
    beams, slots = 4, 8
    cache = PagedCache(2, 64, 16, KV_HEADS, slots, 64, held)
    with torch.inference_mode():
        prompts = [rng.integers(0, 1000, n).tolist() for n in (13, 30)]
        logits, _ = step_of(model, cache, sum(prompts, []), [13, 0, 0, 0, 30, 0, 0, 0])
        cache.remap({1: 0, 2: 0, 3: 0, 5: 4, 6: 4, 7: 4})
        logits = torch.cat((logits[12].expand(beams, -1), logits[42].expand(beams, -1)))
        scores = torch.tensor([0.0] + [-torch.inf] * 3, device="cuda").repeat(2)
        text = [list(prompts[s // beams]) for s in range(slots)]
        for _ in range(6):
            value, rows, tokens, _ = best_of(logits, scores, beams, beams)
            scores, parents, picked = cache.select(logits, scores, beams)
            assert torch.equal(parents.long(), rows.flatten()) and torch.equal(picked.long(), tokens.flatten())
            text = [text[p] + [t] for p, t in zip(parents.tolist(), picked.tolist())]
            logits, _ = step_of(model, cache, picked.tolist(), [1] * slots)
            if held == torch.float16:
                for s in range(slots):
                    assert (logits[s] - dense(model, text[s])[-1]).abs().max() <= LOGITS
            assert cache.lengths.tolist() == [len(t) for t in text]
        cache.check()


def test_a_layer_over_8_bit_pages(patched):  # noqa: F811
    """A prompt and then a tree through the patched layers, against attention in 64 bits over the rotated keys
    and values rounded to 8 bits by their definition. The layers' inputs are given, so that what is rounded is
    the same; the rest is six half steps of fp16 of a layer's output, of size up to 1 (a number that falls on
    the other side of a tie by the rotation's own rounding, 2^-3 of a value of 0.5 at a weight of 1/10 and
    through projections of 0.02, counts a tenth of that)."""
    banner("layers over 8-bit pages")
    model, gen = tiny_model("cuda").eval(), torch.Generator().manual_seed(6)
    rng = np.random.default_rng(6)
    layers = [layer.self_attn for layer in model.model.layers]
    cache = PagedCache(2, 16, 16, KV_HEADS, 2, 128, o8.E4M3)
    kept = [[[] for _ in range(2)] for _ in layers]  # per layer and slot: (k, v) rows in 64 bits
    with torch.inference_mode():
        for q, tree in (([21, 50], None), ([16, 9], [o8.random_tree(rng, n, 5) for n in (16, 9)])):
            n = sum(q)
            plan = cache.step(ints(q), n, HEADS, None if tree is None else ints(sum(tree, [])))
            hidden = torch.randn(n, HIDDEN, generator=gen).cuda()
            tables = model.model.rotary_emb(hidden[None], plan.positions.long()[None])
            cos, sin = (x[0].cpu().double() for x in tables)
            for i, layer in enumerate(layers):
                out, _ = layer(hidden, tables, None, paged=(cache, plan))
                size = out.abs().max()
                assert 0.05 < size <= 1

                def rotated(x):
                    x = x.view(n, -1, DIM)
                    half = torch.cat((-x[..., DIM // 2:], x[..., :DIM // 2]), -1)
                    return x * cos[:, None] + half * sin[:, None]

                query = rotated(layer.q_proj(hidden).cpu().double())
                k = o8.quantize(rotated(layer.k_proj(hidden).cpu().double()))
                v = o8.quantize(layer.v_proj(hidden).cpu().double().view(n, -1, DIM))
                k, v = (x * torch.exp2(e)[..., None] for x, e in (k, v))
                attn, at = torch.zeros(n, HEADS, DIM, dtype=torch.float64), 0
                for s, count in enumerate(q):
                    old = kept[i][s]
                    on = np.tril(np.ones((count, count), dtype=bool)) if tree is None else o8.paths(tree[s])
                    for j in range(count):
                        seen = old + [(k[at + m], v[at + m]) for m in np.nonzero(on[j])[0]]
                        ks, vs = (torch.stack([x[w] for x in seen], 1) for w in (0, 1))
                        for h in range(HEADS):
                            w = torch.softmax(ks[h // 2] @ query[at + j, h] * layer.scaling, 0)
                            attn[at + j, h] = w @ vs[h // 2]
                    kept[i][s] = old + [(k[at + m], v[at + m]) for m in range(count)]
                    at += count
                want = attn.view(n, -1) @ layer.o_proj.weight.cpu().double().T
                assert (out.cpu().double() - want).abs().max() <= 6 * 2.0 ** -11
        cache.check()
