"""The Qwen2 attention patch: transformers' Qwen2Attention.forward with the rotation and the
attention of the packed rows done by the gfx950 kernels (solution/patches.py:81-113).

Calls that carry `packed=(b_idx, t_idx, batch, seq, lengths)` (a padding-free training step, as
built by solution/packed.py:153-176) take the packed path: the q/k/v projections, then
`packed_attention` when the rows are right padded (`lengths` is a list), otherwise the padded
layout with the caller's mask through `qkv_rotate(padded=True)`, SDPA and `pack_rows`. Calls that
carry `paged=(cache, plan)` (a serving step over a `PagedCache`: hidden rows of the step's new
tokens, rotary tables by row) append the rows to the layer's pages and attend to them; they read no
mask, and a model called with `attention_mask={"full_attention": None}` builds none. Every other call
runs the original forward unchanged.
"""

import torch

from .attention import pack_rows, packed_attention, qkv_rotate
from .paged import paged_append, paged_attention

_ORIGINAL = {}


def patch_qwen2_attention():
    from transformers.models.qwen2 import modeling_qwen2

    cls = modeling_qwen2.Qwen2Attention
    if "forward" not in _ORIGINAL:
        _ORIGINAL["forward"] = cls.forward
    original = _ORIGINAL["forward"]

    def forward(self, hidden_states, position_embeddings, attention_mask, past_key_values=None,
                **kwargs):
        packed, paged = kwargs.pop("packed", None), kwargs.pop("paged", None)
        if paged is not None:
            if packed is not None:
                raise ValueError("a call is either packed or paged")
            return _paged_forward(self, hidden_states, position_embeddings, *paged), None
        if packed is None:  # an ordinary call (generation, eval, padded batches): unchanged
            return original(self, hidden_states, position_embeddings, attention_mask,
                            past_key_values, **kwargs)
        b_idx, t_idx, batch, seq, lengths = packed
        cos, sin = position_embeddings
        config = self.config
        q, k, v = (self.q_proj(hidden_states), self.k_proj(hidden_states),
                   self.v_proj(hidden_states))
        if lengths is not None:  # documents are contiguous row blocks: attend on the rows
            attn = packed_attention(q, k, v, cos, sin, b_idx, t_idx, seq,
                                    config.num_attention_heads, config.num_key_value_heads,
                                    lengths, self.scaling)
            return self.o_proj(attn), None
        # lengths unknown (e.g. left padding): rebuild the padded batch, use the caller's mask
        query, key, value = qkv_rotate(q, k, v, cos, sin, b_idx, t_idx, batch, seq,
                                       config.num_attention_heads, config.num_key_value_heads,
                                       True)
        attn = torch.nn.functional.scaled_dot_product_attention(
            query, key, value, attn_mask=attention_mask, dropout_p=0.0, scale=self.scaling)
        return self.o_proj(pack_rows(attn, b_idx, t_idx)), None

    cls.forward = forward


def _paged_forward(layer, hidden_states, position_embeddings, cache, plan):
    """The layer's rows of a serving step, (N, hidden) or (1, N, hidden): projections, append to the
    layer's pages, attention over them, output projection."""
    window, reach = getattr(layer, "sliding_window", None), plan.page_table.shape[1] * plan.page_size
    if window is not None and window < reach:  # a row past the window would see too many keys
        raise ValueError(f"layer {layer.layer_idx} attends to a window of {window} tokens: the paged "
                         f"attention has none, and a page table row holds {reach}")
    rows = hidden_states.reshape(-1, hidden_states.shape[-1])
    cos, sin = (x.reshape(-1, x.shape[-1]) for x in position_embeddings)
    keys, values = cache.keys(layer.layer_idx), cache.values(layer.layer_idx)
    k, v = layer.k_proj(rows), layer.v_proj(rows)
    q = layer.q_proj(rows)
    query = paged_append(q, k, v, cos, sin, keys, values, plan)
    attn = paged_attention(query, keys, values, plan, layer.scaling)
    return layer.o_proj(attn.to(q.dtype)).reshape(hidden_states.shape)


def unpatch_qwen2_attention():
    """Restore transformers' forward (tests)."""
    from transformers.models.qwen2 import modeling_qwen2

    if "forward" in _ORIGINAL:
        modeling_qwen2.Qwen2Attention.forward = _ORIGINAL["forward"]
