"""A transformers model on the 8-bit cache without a GPU: the oracle stands in for the operators, so that what is
tested is how the cache and the attention function meet the library's generation, masks and cache protocol."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from community_kv_amd import QuantizedCache, QuantizedCacheAttention
from community_kv_amd.attention import quantized_cache
from oracle import quantized as oq
from tests import _dense_codes as dense_codes

LAYERS = 2


def _store(oracle, cache):
    for i, (codes, scales) in enumerate(((cache.key_codes, cache.key_scales), (cache.value_codes, cache.value_scales))):
        codes.view(torch.uint8).copy_(torch.from_numpy(oracle.codes[i]))
        scales.copy_(torch.from_numpy(oracle.scales[i]))
    cache.positions.copy_(torch.from_numpy(oracle.positions))
    cache.cursors.copy_(torch.from_numpy(oracle.cursors))
    if cache.weights is not None:
        cache.weights.copy_(torch.from_numpy(oracle.weights))


@pytest.fixture
def on_cpu(monkeypatch):
    """The operators that the cache calls, as the oracle computes them, without gradients."""

    def append(cache, key, value):
        oracle = oq.Cache.of(cache)
        oracle.append(key.double().numpy(), value.double().numpy())
        _store(oracle, cache)

    def attention(query, cache, *, softmax_scale, window=0, accumulate=False):
        (out, lse, got), _ = oq.Cache.of(cache).attend(query.double().numpy(), scale=softmax_scale, window=window)
        if accumulate:
            cache.weights.add_(torch.from_numpy(got.astype(np.float32)))
        return torch.from_numpy(out).to(query.dtype), torch.from_numpy(lse).float()

    def evict(cache, **kwargs):
        oracle = oq.Cache.of(cache)
        oracle.evict(**kwargs)
        _store(oracle, cache)

    monkeypatch.setattr(quantized_cache, "quantized_append", append)
    monkeypatch.setattr(quantized_cache, "quantized_attention", attention)
    monkeypatch.setattr(quantized_cache, "evict", evict)
    with torch.no_grad():
        yield


def _model(**change):
    from transformers import Qwen3Config, Qwen3ForCausalLM

    cfg = Qwen3Config(**(dict(vocab_size=64, hidden_size=128, intermediate_size=128, num_hidden_layers=LAYERS,
                              num_attention_heads=2, num_key_value_heads=1, head_dim=128, max_position_embeddings=512,
                              tie_word_embeddings=False) | change))
    torch.manual_seed(0)
    return Qwen3ForCausalLM(cfg).eval()


def _on_cache(model, **kwargs):
    cache = QuantizedCache(**(dict(num_hidden_layers=LAYERS, max_cache_len=96, block=16) | kwargs))
    model.set_attn_implementation(QuantizedCacheAttention(cache).register())
    return cache


def _prompt(n, seed=1):
    return torch.randint(0, 64, (1, n), generator=torch.Generator().manual_seed(seed))


# ------------------------------------------------------------------------------------------ tokens taken back

def test_crop_by_nothing_keeps_all(on_cpu):
    """crop(0) takes nothing back, as the library's own cache, and crop(-n) the newest n."""
    from transformers import DynamicCache

    cache, dynamic = _on_cache(_model()), DynamicCache()
    x = torch.randn(1, 1, 20, 128)
    for layer in range(LAYERS):
        cache.update(x, x, layer)
        dynamic.update(x, x, layer)
    for n, left in ((0, 20), (-4, 16), (0, 16)):
        cache.crop(n)
        dynamic.crop(n)
        assert cache.get_seq_length() == dynamic.get_seq_length() == left
        for layer in range(LAYERS):
            assert cache.layer(layer).store.cursors.tolist() == [[left], [left], [0]]


def test_assisted_generation(on_cpu):
    """Prompt-lookup generation takes rejected candidates back after every verification, none where all were right,
    and gives the tokens of plain greedy generation."""
    model = _model()
    prompt = torch.cat([_prompt(6), _prompt(6), _prompt(4)], 1)
    taken = []

    def generate(**kwargs):
        cache = _on_cache(model)
        crop = cache.crop
        cache.crop = lambda n: (taken.append(n), crop(n))
        out = model.generate(prompt, past_key_values=cache, max_new_tokens=24, do_sample=False, **kwargs)
        for layer in range(LAYERS):
            assert cache.layer(layer).rows == cache.layer(layer).seen == out.shape[1] - 1
            assert cache.layer(layer).store.lengths.tolist() == [out.shape[1] - 1]
        return out

    plain = generate()
    assert not taken
    assert torch.equal(generate(prompt_lookup_num_tokens=3), plain)
    assert 0 in taken and min(taken) < 0


def test_crop_counts(on_cpu):
    """Counts come as 0-dim tensors from the library; the host's own counts stay integers, which nothing waits for.
    More than there are empties the cache, as the library's own does, also before anything was written."""
    from transformers import DynamicCache

    cache, dynamic = _on_cache(_model()), DynamicCache()
    cache.crop(-3)
    x = torch.randn(1, 1, 20, 128)
    for layer in range(LAYERS):
        cache.update(x, x, layer)
        dynamic.update(x, x, layer)
    for n in (torch.tensor(-3), torch.tensor(0), np.int64(-1), -100):
        cache.crop(n)
        dynamic.crop(n)
        assert cache.get_seq_length() == dynamic.get_seq_length()
        for layer in range(LAYERS):
            held = cache.layer(layer)
            assert type(held.rows) is int and type(held.seen) is int and held.rows == held.seen
            assert held.store.cursors.tolist() == [[held.rows], [held.rows], [0]]
    assert held.rows == 0


# ------------------------------------------------------------------------------------------ masks

def test_a_mask_of_ones_is_no_padding(on_cpu):
    model = _model()
    prompt, mask = _prompt(12), torch.ones(1, 12, dtype=torch.long)
    want = model(prompt, past_key_values=_on_cache(model)).logits
    assert torch.equal(model(prompt, attention_mask=mask, past_key_values=_on_cache(model)).logits, want)
    model.generate(prompt, attention_mask=mask, past_key_values=_on_cache(model), max_new_tokens=2, do_sample=False)


@pytest.mark.parametrize("padded", [slice(0, 1), slice(0, 5), slice(11, 12), slice(4, 6)])
def test_padding_is_refused(on_cpu, padded):
    """A padded sequence raises from the model's own call, left, right and within, before anything is written."""
    model = _model()
    prompt, mask = _prompt(12), torch.ones(1, 12, dtype=torch.long)
    mask[:, padded] = 0
    for call in (model, lambda *args, **kwargs: model.generate(*args, max_new_tokens=2, do_sample=False, **kwargs)):
        cache = _on_cache(model)
        with pytest.raises(ValueError, match="padding"):
            call(prompt, attention_mask=mask, past_key_values=cache)
        assert cache.get_seq_length() == 0


def test_padding_is_refused_behind_a_prompt(on_cpu):
    model = _model()
    cache = _on_cache(model)
    model(_prompt(12), past_key_values=cache)
    mask = torch.ones(1, 13, dtype=torch.long)
    mask[0, 3] = 0
    with pytest.raises(ValueError, match="padding"):
        model(_prompt(1), attention_mask=mask, past_key_values=cache)
    assert cache.get_seq_length() == 12


def test_a_mask_in_a_captured_call_is_refused(monkeypatch):
    """Whether it masks anything cannot be read while a stream is captured."""
    class Mask:
        is_cuda = True

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    assert QuantizedCacheAttention.mask(attention_mask=None) is None
    with pytest.raises(ValueError, match="captured"):
        QuantizedCacheAttention.mask(attention_mask=Mask())


def test_other_patterns_than_causal_and_sliding_are_refused(on_cpu):
    """Chunks of attention, packed sequences and a model's own additions to the causal mask: the operator has no such
    mask, and would attend past it."""
    from transformers import masking_utils

    model = _model(sliding_window=8, use_sliding_window=True, max_window_layers=1)
    cache = _on_cache(model)
    call = dict(config=model.config, inputs_embeds=torch.zeros(1, 5, 128), attention_mask=None, past_key_values=cache)
    model.config.attention_chunk_size = 4
    assert masking_utils.create_causal_mask(**call) is None
    assert masking_utils.create_sliding_window_causal_mask(**call) is None
    for make, extra in ((masking_utils.create_chunked_causal_mask, {}),
                        (masking_utils.create_causal_mask, dict(or_mask_function=lambda b, h, q, k: k < 3)),
                        (masking_utils.create_sliding_window_causal_mask, dict(and_mask_function=lambda b, h, q, k: k < 3)),
                        (masking_utils.create_causal_mask, dict(past_key_values=None,
                                                                position_ids=torch.tensor([[0, 1, 2, 0, 1]])))):
        with pytest.raises(ValueError, match="causal"):
            make(**(call | extra))
    model.config.attention_chunk_size = model.config.sliding_window
    model.config.layer_types = ["full_attention", "chunked_attention"]
    with pytest.raises(ValueError, match="causal"):
        masking_utils.create_chunked_causal_mask(**call)


# ------------------------------------------------------------------------------------------ the dense model

def test_a_model_on_the_cache_is_the_dense_model(on_cpu):
    """Prompt pieces and single tokens of a model with a full and a sliding layer, against dense attention over what the
    codes stand for.  Both attentions are in 64 bits here and rounded to 32, so an output is off by far less than 2^-16 of
    the largest value; how far so much moves the logits, through codes that flip too, is measured on the dense model.
    The sliding mask lost moves them much further."""
    model = _model(sliding_window=9, use_sliding_window=True, max_window_layers=1)
    assert model.config.layer_types == ["full_attention", "sliding_attention"]
    prompt = _prompt(36)
    pieces = [prompt[:, :17], prompt[:, 17:30]] + [prompt[:, i:i + 1] for i in range(30, 36)]
    got = dense_codes.logits(model, _on_cache(model), pieces)

    def dense(**kwargs):
        model.set_attn_implementation(dense_codes.register(**kwargs))
        cache = dense_codes.dense_cache(quantized_cache.quantized_append, layers=LAYERS, rows=96, block=16)
        return dense_codes.logits(model, cache, pieces)

    want, moved, wrong = dense(), dense(noise=2.0 ** -16), dense(window=False)
    off, tol, far = (max(float((a - b).abs().max()) for a, b in zip(want, other)) for other in (got, moved, wrong))
    assert off <= 2 * tol and far > 100 * tol, (off, tol, far)
