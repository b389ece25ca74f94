"""Hugging Face cache and attention function over the 8-bit KV cache.

No reference counterpart: next to the ``community_kv`` attention function and
its bf16 ``StaticCache`` this pair runs a model on ``QuantizedKVCache``::

    cache = QuantizedCache(num_hidden_layers=model.config.num_hidden_layers, max_cache_len=33_000)
    model.set_attn_implementation(QuantizedCacheAttention(cache).register())
    model.generate(input_ids, past_key_values=cache, ...)

Every new token's key and value are quantised into the layer's cache, and the
queries, of the prompt as of a single token, attend to what the cache holds.
With ``budget`` a layer that holds more than ``budget + slack`` rows after a
call is cut to its ``budget`` most attended rows (the first ``num_sink``
positions and the newest ``recent`` ones among them), so a request of any
length runs in ``max(prompt, budget + slack + 1)`` rows.

One sequence at a time, as the CommunityKV runtime, and without padding (a
padding mask raises); ragged batches call ``quantized_append`` and
``quantized_attention`` with ``counts``.
"""

from __future__ import annotations

import weakref
from typing import Any

import torch
from transformers.cache_utils import Cache, CacheLayerMixin

from community_kv_amd.attention.quantized import QuantizedKVCache, evict, quantized_append, quantized_attention

QUANTIZED_ATTENTION_IMPLEMENTATION = "community_kv_quantized"


class QuantizedCacheLayer(CacheLayerMixin):
    """One decoder layer's 8-bit cache, allocated on the first write.  The row
    count is kept on the host too (every write and eviction is known there), so
    nothing is read back."""

    def __init__(self, max_cache_len: int, *, block: int = 64, budget: int = 0, num_sink: int = 4, recent: int = 64,
                 slack: int = 64) -> None:
        super().__init__()
        if max_cache_len <= 0:
            raise ValueError("max_cache_len must be positive")
        if budget < 0 or slack < 0 or num_sink < 0 or recent < 0:
            raise ValueError("budget, slack, num_sink and recent must be non-negative")
        if budget and (num_sink + recent > budget or budget + slack >= max_cache_len):
            raise ValueError("budget must hold num_sink + recent rows, and max_cache_len more than budget + slack")
        self.max_cache_len = max_cache_len
        self.block, self.budget, self.num_sink, self.recent, self.slack = block, budget, num_sink, recent, slack
        self.store: QuantizedKVCache | None = None
        self.rows = 0  # in the cache
        self.seen = 0  # ever written: the next token's position
        self._latest: Any = None  # the keys written last, to tell a call with another cache's keys

    # -- Hugging Face cache-layer protocol ----------------------------------

    def lazy_initialization(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        if key_states.shape[0] != 1:
            raise ValueError("the 8-bit cache layer holds one sequence")
        self.store = QuantizedKVCache.allocate(kv_heads=key_states.shape[1], capacity=self.max_cache_len,
                                               block=self.block, track_weights=self.budget > 0,
                                               device=key_states.device)
        self.dtype, self.device = key_states.dtype, key_states.device
        self.is_initialized = True

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args: object,
               **kwargs: object) -> tuple[torch.Tensor, torch.Tensor]:
        """Appends the new tokens and returns them (the attention function reads the cache itself)."""
        tokens = key_states.shape[2]
        if self.rows + tokens > self.max_cache_len:
            raise ValueError(f"KV cache capacity exceeded: {self.rows + tokens} > {self.max_cache_len}")
        if self.store is None:
            self.lazy_initialization(key_states, value_states)
        quantized_append(self.store, key_states, value_states)
        self.rows += tokens
        self.seen += tokens
        self._latest = weakref.ref(key_states)
        return key_states, value_states

    def get_mask_sizes(self, query_length: int, *args: object, **kwargs: object) -> tuple[int, int]:
        return self.seen + query_length, 0

    def get_seq_length(self, *args: object, **kwargs: object) -> int:
        return self.seen

    def get_max_length(self) -> int:
        return -1 if self.budget else self.max_cache_len

    def reset(self) -> None:
        if self.store is not None:
            self.store.reset()
        self.rows = self.seen = 0
        self._latest = None

    def crop(self, max_length: int) -> None:
        """Takes back the newest tokens, down to a positive ``max_length``, else ``-max_length`` of them (0: none,
        what assisted generation asks for where every candidate was right; the library passes 0-dim tensors too).
        With a budget the weight that their queries gave to older rows stays, and counts in later evictions."""
        max_length = int(max_length)
        drop = min(self.seen - max_length if max_length > 0 else -max_length, self.seen)
        if drop <= 0:
            return
        if drop > self.rows or (self.budget and self.seen != self.rows):
            raise ValueError("the tokens to take back may have been evicted")
        self.store.rewind(drop)
        self.rows -= drop
        self.seen -= drop

    def reorder_cache(self, beam_idx: torch.LongTensor) -> None:
        raise NotImplementedError("the 8-bit cache holds one sequence: no beam search")

    def offload(self) -> None:
        raise NotImplementedError("the 8-bit cache stays on its GPU")

    prefetch = offload

    # -- attention -----------------------------------------------------------

    def attend(self, query: torch.Tensor, key: torch.Tensor, scaling: float, window: int = 0) -> torch.Tensor:
        """Attention of the queries of the tokens written last, whose keys are
        ``key`` as ``update`` returned them, then the eviction where the layer
        holds more than its budget and slack."""
        if self.store is None or self._latest is None or self._latest() is not key or query.shape[2] != key.shape[2]:
            raise RuntimeError("the tokens of this call were not written into this cache: pass the cache that the "
                               "attention function was registered with as past_key_values")
        out, _ = quantized_attention(query, self.store, softmax_scale=scaling, window=window,
                                     accumulate=self.budget > 0)
        if self.budget and self.rows > self.budget + self.slack:
            evict(self.store, keep=self.budget, num_sink=self.num_sink, recent=self.recent)
            self.rows = self.budget
        return out


class QuantizedCache(Cache):
    """``QuantizedCacheLayer`` per decoder layer."""

    def __init__(self, *, num_hidden_layers: int, max_cache_len: int, block: int = 64, budget: int = 0,
                 num_sink: int = 4, recent: int = 64, slack: int = 64) -> None:
        super().__init__(layers=[QuantizedCacheLayer(max_cache_len, block=block, budget=budget, num_sink=num_sink,
                                                     recent=recent, slack=slack) for _ in range(num_hidden_layers)])

    def layer(self, layer_idx: int) -> QuantizedCacheLayer:
        found = self.layers[layer_idx]
        if isinstance(found, QuantizedCacheLayer):
            return found
        raise TypeError(f"layer {layer_idx} is a {type(found).__name__}, not a QuantizedCacheLayer")


class QuantizedCacheAttention:
    """The attention function of a model whose cache is ``cache``.  One
    function is registered at a time; a model that runs with another cache than
    the one registered last is told so (``RuntimeError``)."""

    IMPL_NAME = QUANTIZED_ATTENTION_IMPLEMENTATION

    def __init__(self, cache: QuantizedCache) -> None:
        self.cache = cache

    def register(self) -> str:
        from transformers import AttentionMaskInterface
        from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS

        ALL_ATTENTION_FUNCTIONS[self.IMPL_NAME] = self.forward
        AttentionMaskInterface.register(self.IMPL_NAME, self.mask)
        return self.IMPL_NAME

    @staticmethod
    def mask(*args: Any, attention_mask: torch.Tensor | None = None, **kwargs: Any) -> None:
        """The model's mask: none, as ``forward`` masks by position.  The library asks for it once a forward call,
        with the padding mask [1, rows] (without a function of this name it drops that mask unseen).  Reading it
        waits for the device; a caller who captures passes no mask."""
        config, local = kwargs.get("config"), kwargs.get("local_size")
        # the library may not skip a causal mask that a model adds to, or of packed sequences; chunks come as a local
        # size, as a sliding window does
        if (not kwargs.get("allow_is_causal_skip", True) or local not in (None, getattr(config, "sliding_window", None)) or
                "chunked_attention" in (getattr(config, "layer_types", None) or ())):
            raise ValueError("attention over the 8-bit cache is causal, with or without a sliding window, and takes no "
                             "other mask")
        if attention_mask is None:
            return
        if attention_mask.is_cuda and torch.cuda.is_current_stream_capturing():
            raise ValueError("a captured call takes no attention_mask: it cannot be looked at for padding")
        if not bool(attention_mask.all()):
            raise ValueError("attention over the 8-bit cache takes no padding: pass the sequence without it")

    def forward(self, module: torch.nn.Module, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                attention_mask: torch.Tensor | None, scaling: float, dropout: float = 0.0,
                **kwargs: Any) -> tuple[torch.Tensor, None]:
        """query [1, Hq, S, 128]; key/value the new tokens, which the cache's
        update has just written.  Returns ([1, S, Hq, 128], None)."""
        if dropout:
            raise ValueError("attention over the 8-bit cache has no dropout")
        if attention_mask is not None or kwargs.get("is_causal") is False:
            raise ValueError("attention over the 8-bit cache is causal and takes no mask")
        for name in ("softcap", "s_aux"):
            if kwargs.get(name) is not None:
                raise ValueError(f"attention over the 8-bit cache does not support {name}")
        layer = self.cache.layer(int(module.layer_idx))
        return layer.attend(query, key, float(scaling), int(kwargs.get("sliding_window") or 0)), None


__all__ = ["QUANTIZED_ATTENTION_IMPLEMENTATION", "QuantizedCache", "QuantizedCacheAttention", "QuantizedCacheLayer"]
