"""A dense model to hold a model on the 8-bit cache against (test infrastructure): the library's own masks, and
attention in 64 bits over the keys and values that the codes stand for."""

from __future__ import annotations

import torch
from transformers import AttentionMaskInterface
from transformers.cache_utils import Cache, DynamicLayer
from transformers.masking_utils import eager_mask
from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS

from community_kv_amd import QuantizedKVCache

DENSE = "dense_over_codes"


class _Layer(DynamicLayer):
    """Quantises what it is given with `append` and hands back everything as numbers."""

    def __init__(self, append, rows: int, block: int) -> None:
        super().__init__()
        self.append, self.capacity, self.block, self.store = append, rows, block, None

    def update(self, key_states, value_states, *args, **kwargs):
        if self.store is None:
            self.lazy_initialization(key_states, value_states)
            self.store = QuantizedKVCache.allocate(kv_heads=key_states.shape[1], capacity=self.capacity, block=self.block,
                                                   device=key_states.device)
        self.append(self.store, key_states, value_states)
        rows = self.get_seq_length() + key_states.shape[2]
        self.keys, self.values = (x[:, :, :rows] for x in self.store.dequantize())
        return self.keys, self.values


def dense_cache(append, *, layers: int, rows: int, block: int) -> Cache:
    return Cache(layers=[_Layer(append, rows, block) for _ in range(layers)])


def register(noise: float = 0.0, window: bool = True) -> str:
    """Dense attention under the library's mask; `noise`: every output off by up to that share of the
    largest value; without `window` the sliding layers' mask is lost (a planted mistake)."""
    gen = torch.Generator().manual_seed(7)

    def forward(module, query, key, value, attention_mask, scaling, **kwargs):
        group = query.shape[1] // key.shape[1]
        key, value = (x.double().repeat_interleave(group, 1) for x in (key, value))
        scores = query.double() @ key.transpose(2, 3).contiguous() * scaling
        tokens, rows = scores.shape[2:]
        mask = attention_mask
        if not window:
            at = torch.arange(rows, device=scores.device)
            mask = torch.where(at <= at[rows - tokens:, None], 0.0, -torch.inf)
        out = torch.softmax(scores + mask.double(), -1) @ value
        if noise:
            sign = torch.rand(out.shape, generator=gen, dtype=torch.float64).to(out.device) * 2 - 1
            out = out + noise * value.abs().max() * sign
        return out.transpose(1, 2).contiguous().to(query.dtype), None

    ALL_ATTENTION_FUNCTIONS[DENSE] = forward
    AttentionMaskInterface.register(DENSE, eager_mask)
    return DENSE


def logits(model, cache, pieces) -> list:
    """The model's logits of every call, the pieces one after another."""
    at, got = 0, []
    with torch.no_grad():
        for piece in pieces:
            n = piece.shape[1]
            position = torch.arange(at, at + n, device=piece.device)[None]
            got.append(model(piece, past_key_values=cache, position_ids=position, use_cache=True).logits.double())
            at += n
    return got
