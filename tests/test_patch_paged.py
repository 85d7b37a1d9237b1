"""The patched layer's serving calls as a program makes them through the whole model: what the model
does around them, and which ones are refused."""

import pytest
import torch

from hackaton_amd import PagedCache, patches
from tests.test_patch import HEADS, KV_HEADS, patched, tiny_model  # noqa: F401 (a fixture)

NO_MASK = {"full_attention": None}


@pytest.mark.parametrize("n", [1, 300])
def test_a_serving_call_builds_no_mask(patched, monkeypatch, n):  # noqa: F811
    """The documented call: the layers are handed no mask and transformers makes none."""
    from transformers.models.qwen2 import modeling_qwen2

    def never(*args, **kwargs):
        raise AssertionError("a mask is built")

    seen = []
    monkeypatch.setattr(patches, "_paged_forward", lambda layer, hidden, *rest: hidden * 0)
    monkeypatch.setattr(modeling_qwen2, "create_causal_mask", never)
    forward = modeling_qwen2.Qwen2Attention.forward

    def spy(self, hidden_states, position_embeddings, attention_mask, **kwargs):
        seen.append(attention_mask)
        return forward(self, hidden_states, position_embeddings, attention_mask, **kwargs)

    monkeypatch.setattr(modeling_qwen2.Qwen2Attention, "forward", spy)
    model = tiny_model("cpu").eval()
    positions = (torch.arange(n) % max(1, 2 * n // 3))[None]  # two sequences
    with torch.inference_mode():
        out = model(input_ids=torch.zeros(1, n, dtype=torch.long), position_ids=positions,
                    attention_mask=NO_MASK, paged=(None, None), use_cache=False).logits
    assert out.shape == (1, n, 1000) and seen == [None, None]


@pytest.mark.gpu
def test_a_serving_step_reads_nothing_back(patched):  # noqa: F811
    """A step of the whole model with device lengths: no call waits for the GPU, a captured one replays
    on the cache that it finds, and both give what a call without the argument gives, bit by bit."""
    model = tiny_model("cuda").eval()
    caches = [PagedCache(2, 32, 16, KV_HEADS, 2, 128) for _ in range(2)]
    gen = torch.Generator().manual_seed(3)
    tokens = torch.randint(0, 1000, (40,), generator=gen).cuda()
    lengths = torch.tensor([21, 19], dtype=torch.int32, device="cuda")
    one = torch.ones_like(lengths)

    def step(cache, q, rows, **mask):
        plan = cache.step(q, rows.numel(), HEADS)
        return model(input_ids=rows[None], position_ids=plan.positions.clamp(min=0).long()[None],
                     paged=(cache, plan), use_cache=False, **mask).logits[0]

    with torch.inference_mode():
        for cache in caches:
            cache.pages.zero_()
        step(caches[0], lengths, tokens, attention_mask=NO_MASK)  # (the library's first calls may wait)
        caches[0].remap(None, lengths * 0)
        torch.cuda.synchronize()
        torch.cuda.set_sync_debug_mode("error")
        try:
            first = step(caches[0], lengths, tokens, attention_mask=NO_MASK)
        finally:
            torch.cuda.set_sync_debug_mode("default")
        assert torch.equal(first, step(caches[1], lengths, tokens))
        rows = tokens[:2].clone()
        step(caches[0], one, rows, attention_mask=NO_MASK)
        caches[0].remap(None, lengths)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(caches[0], one, rows, attention_mask=NO_MASK)
        for i in range(4):
            rows.copy_(tokens[2 * i:2 * i + 2])
            graph.replay()
            want = step(caches[1], one, rows)
            torch.cuda.synchronize()
            assert torch.equal(got, want) and caches[0].lengths.tolist() == [22 + i, 20 + i]
        for cache in caches:
            cache.check()
