"""The installed surface: `hackaton_amd.apply()` and the patched Qwen2Attention.forward
(solution/patches.py:81-113, solution/__init__.py:23-33), checked end to end against transformers'
own forward on a tiny Qwen2 built from Qwen2Config (no download), as solution/test_packed.py:17-76
checks the reference's.

* CPU: apply() installs the patch, a call without `packed` runs transformers' forward unchanged,
  and unpatching restores the class.
* GPU: the packed branch (right padding, lengths given: packed_attention) and the fallback branch
  (lengths None: qkv_rotate padded, SDPA with the caller's mask, pack_rows) against the unpatched
  forward on the padded layout with the causal & real mask, under fp16 autocast like the Soup
  step: outputs within 3e-2 (the reference test's logits tolerance) and every gradient with
  cosine > 0.995 (its gradient check).
"""

import pytest
import torch

import hackaton_amd
from hackaton_amd import patches

HEADS, KV_HEADS, DIM = 4, 2, 128
HIDDEN = HEADS * DIM


def tiny_model(device):
    from transformers import Qwen2Config, Qwen2ForCausalLM

    torch.manual_seed(0)
    config = Qwen2Config(vocab_size=1000, hidden_size=HIDDEN, intermediate_size=1024,
                         num_hidden_layers=2, num_attention_heads=HEADS,
                         num_key_value_heads=KV_HEADS, max_position_embeddings=256)
    return Qwen2ForCausalLM._from_config(config, attn_implementation="sdpa").to(device).train()


@pytest.fixture
def patched():
    hackaton_amd.apply()
    try:
        yield
    finally:
        patches.unpatch_qwen2_attention()


def cosine(a, b):
    return float(torch.nn.functional.cosine_similarity(a.float().flatten(), b.float().flatten(),
                                                       dim=0))


def test_apply_installs_the_patch_and_keeps_unpacked_calls_unchanged():
    from transformers.models.qwen2 import modeling_qwen2

    before = modeling_qwen2.Qwen2Attention.forward
    model = tiny_model("cpu")
    layer = model.model.layers[0].self_attn
    hidden = torch.randn(2, 6, HIDDEN)
    pos = torch.arange(6)[None]
    cos, sin = model.model.rotary_emb(hidden, pos)
    mask = torch.ones(6, 6, dtype=torch.bool).tril()[None, None].expand(2, 1, 6, 6)
    ref, _ = layer(hidden, (cos, sin), mask)
    hackaton_amd.apply()
    try:
        assert modeling_qwen2.Qwen2Attention.forward is not before
        out, _ = layer(hidden, (cos, sin), mask)  # no `packed`: transformers' code path
        assert torch.equal(out, ref)
    finally:
        patches.unpatch_qwen2_attention()
    assert modeling_qwen2.Qwen2Attention.forward is before


def padded_batch(lengths, seq, left, device):
    """(B, T) bool mask of real tokens, right or left padded, and the packed row maps."""
    real = torch.zeros(len(lengths), seq, dtype=torch.bool, device=device)
    for row, length in enumerate(lengths):
        if left:
            real[row, seq - length:] = True
        else:
            real[row, :length] = True
    rows = torch.nonzero(real.reshape(-1), as_tuple=True)[0]
    return real, rows, (rows // seq).to(torch.int32), (rows % seq).to(torch.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("left", [False, True], ids=["right_padded_packed", "left_padded_mask"])
def test_patched_attention_matches_original_forward(left, patched):
    dev = torch.device("cuda")
    print(f"\n[case] patched Qwen2Attention, {'left' if left else 'right'} padding", flush=True)
    model = tiny_model(dev)
    layer = model.model.layers[1].self_attn
    lengths, seq = [40, 25, 33], 40
    real, rows, b_idx, t_idx = padded_batch(lengths, seq, left, dev)
    g = torch.Generator(device=dev).manual_seed(1)
    hidden = torch.randn(len(lengths), seq, HIDDEN, device=dev, generator=g)
    grad = torch.randn(rows.numel(), HIDDEN, device=dev, generator=g)
    cos, sin = model.model.rotary_emb(hidden, torch.arange(seq, device=dev)[None])
    mask = torch.ones(seq, seq, dtype=torch.bool, device=dev).tril()[None, None] & real[:, None,
                                                                                         None]
    params = dict(layer.named_parameters())

    def run(packed):
        layer.zero_grad()
        if packed is None:  # transformers' forward on the padded layout
            x = hidden.clone().requires_grad_()
            with torch.autocast("cuda", dtype=torch.float16):
                out, _ = patches._ORIGINAL["forward"](layer, x, (cos, sin), mask)
            out = out.reshape(-1, HIDDEN)[rows]
        else:
            x = hidden.reshape(-1, HIDDEN)[rows].clone().requires_grad_()
            with torch.autocast("cuda", dtype=torch.float16):
                out, weights = layer(x, (cos, sin), None if not left else mask, packed=packed)
            assert weights is None
        out.float().backward(grad)
        grads = {n: p.grad.clone() for n, p in params.items() if p.grad is not None}
        xg = x.grad.reshape(-1, HIDDEN) if packed is not None else x.grad.reshape(-1, HIDDEN)[rows]
        return out.detach().float(), grads, xg

    ref_out, ref_grads, ref_xg = run(None)
    out, grads, xg = run((b_idx, t_idx, len(lengths), seq, None if left else lengths))
    assert out.shape == ref_out.shape == (rows.numel(), HIDDEN)
    torch.testing.assert_close(out, ref_out, rtol=3e-2, atol=3e-2)
    assert set(grads) == set(ref_grads) and len(grads) >= 4
    for name in ref_grads:
        assert cosine(grads[name], ref_grads[name]) > 0.995, name
    assert cosine(xg, ref_xg) > 0.995


@pytest.mark.gpu
@pytest.mark.parametrize("shape", ["rows", "batch of one"])
def test_paged_branch_answers_like_the_dense_cache(patched, shape):
    """Two prompts of different lengths, then single tokens, through the patched layers with a
    PagedCache, against transformers' own forward over the whole sequences (causal mask, fp32): hidden
    states in fp16 with fp32 accumulation differ by the same 3e-2 as the packed branch's."""
    from hackaton_amd import PagedCache

    torch.manual_seed(1)
    model = tiny_model("cuda").eval().half()
    layers = [layer.self_attn for layer in model.model.layers]
    lengths, extra = [23, 70], 3
    hidden = [torch.randn(n + extra, HIDDEN, device="cuda").half() for n in lengths]
    cache = PagedCache(len(layers), 16, 16, KV_HEADS, 2, 128)
    got = [[[] for _ in hidden] for _ in layers]
    with torch.no_grad():
        done = [0, 0]
        for step in [lengths] + [[1, 1]] * extra:
            plan = cache.step(torch.tensor(step, dtype=torch.int32, device="cuda"), sum(step), HEADS)
            rows = torch.cat([h[d:d + n] for h, d, n in zip(hidden, done, step)])
            tables = model.model.rotary_emb(rows[None].float(), plan.positions.long()[None])
            for i, layer in enumerate(layers):
                given = rows if shape == "rows" else rows[None]
                out, weights = layer(given, tables, None, paged=(cache, plan))
                assert weights is None and out.shape == given.shape
                for s, part in enumerate(out.reshape(-1, HIDDEN).split(step)):
                    got[i][s].append(part)
            done = [d + n for d, n in zip(done, step)]
        cache.check()
        reference = tiny_model("cuda").eval()
        reference.load_state_dict({k: v.float() for k, v in model.state_dict().items()})
        for s, h in enumerate(hidden):
            n = h.shape[0]
            pos = torch.arange(n, device="cuda")[None]
            tables = reference.model.rotary_emb(h[None].float(), pos)
            mask = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()[None, None]
            for i in range(len(layers)):
                ref, _ = reference.model.layers[i].self_attn(h[None].float(), tables, mask)
                out = torch.cat(got[i][s]).float()
                assert float((out - ref[0]).abs().max()) <= 3e-2


@pytest.mark.gpu
def test_the_whole_model_answers_from_pages(patched):
    """Two prompts in one call of the model, one of them in two chunks, then single tokens, against the
    dense forward of each sequence. fp32 model, fp16 pages: a layer's branch is off by at most six half
    steps of fp16 of its size (q and k in scores of size about 1, weights, values, output), 3e-3; two
    layers, logits up to 2: 1.2e-2."""
    from hackaton_amd import PagedCache

    model = tiny_model("cuda").eval()
    gen = torch.Generator().manual_seed(2)
    tokens = [torch.randint(0, 1000, (n,), generator=gen).cuda() for n in (41, 90)]
    cache = PagedCache(2, 16, 16, KV_HEADS, 2, 128)
    got, done = [[], []], [0, 0]
    with torch.inference_mode():
        for step in ([39, 50], [1, 38], [1, 1], [0, 1]):
            plan = cache.step(step, sum(step) + 2, HEADS)  # (two rows of padding)
            rows = torch.cat([t[d:d + n] for t, d, n in zip(tokens, done, step)])
            rows = torch.nn.functional.pad(rows, (0, 2))
            out = model(input_ids=rows[None], position_ids=plan.positions.clamp(min=0).long()[None],
                        paged=(cache, plan), use_cache=False).logits[0]
            for s, part in enumerate(out[:sum(step)].split(step)):
                got[s].append(part)
            done = [d + n for d, n in zip(done, step)]
        cache.check()
        assert done == [41, 90] and cache.lengths.tolist() == done
        for t, parts in zip(tokens, got):
            ref = model(input_ids=t[None], use_cache=False).logits[0]
            assert float((torch.cat(parts) - ref).abs().max()) <= 1.2e-2


def test_a_call_is_either_packed_or_paged(patched):
    layer = tiny_model("cpu").model.layers[0].self_attn
    with pytest.raises(ValueError, match="packed or paged"):
        layer(torch.zeros(1, HIDDEN), (None, None), None, packed=(0,) * 5, paged=(None, None))
