"""The patched layer's serving calls as a program makes them through the whole model: what the model
does around them, and which ones are refused."""

from types import SimpleNamespace

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


@pytest.mark.parametrize("window,width,fits", [(None, 1000, True), (64, 4, True), (64, 5, False),
                                               (63, 4, False), (0, 1, False)])
def test_a_window_shorter_than_the_tables_is_refused(patched, monkeypatch, window, width, fits):  # noqa: F811
    """The paged attention sees every key up to a row's own: a layer with a sliding window that a page
    table row passes would get other answers than transformers' forward."""
    layer = tiny_model("cpu").model.layers[0].self_attn
    layer.sliding_window = window
    monkeypatch.setattr(patches, "paged_append", lambda q, *rest: q)
    monkeypatch.setattr(patches, "paged_attention", lambda query, *rest: query)
    cache = SimpleNamespace(keys=lambda i: None, values=lambda i: None)
    plan = SimpleNamespace(page_table=torch.zeros(2, width, dtype=torch.int32), page_size=16)
    x, tables = torch.zeros(3, HEADS * 128), (torch.ones(3, 128), torch.zeros(3, 128))
    if fits:
        assert layer(x, tables, None, paged=(cache, plan))[0].shape == x.shape
    else:
        with pytest.raises(ValueError, match="window"):
            layer(x, tables, None, paged=(cache, plan))


def test_layers_with_windows_of_a_model_are_refused(patched):  # noqa: F811
    from transformers import Qwen2Config, Qwen2ForCausalLM

    config = Qwen2Config(vocab_size=100, hidden_size=256, intermediate_size=64, num_hidden_layers=2,
                         num_attention_heads=2, num_key_value_heads=1, use_sliding_window=True,
                         sliding_window=32, max_window_layers=0)
    model = Qwen2ForCausalLM(config).eval()
    plan = SimpleNamespace(page_table=torch.zeros(1, 3, dtype=torch.int32), page_size=16)
    masks = {"full_attention": None, "sliding_attention": None}
    with torch.inference_mode(), pytest.raises(ValueError, match="window of 32"):
        model(input_ids=torch.zeros(1, 4, dtype=torch.long), position_ids=torch.arange(4)[None],
              attention_mask=masks, paged=(None, plan), use_cache=False)


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
