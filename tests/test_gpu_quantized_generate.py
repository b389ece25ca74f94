"""A model run on the 8-bit cache (QuantizedCache + QuantizedCacheAttention): every layer's calls are recorded and
repeated on caches of their own, to the bit, and those calls are what test_gpu_quantized.py checks against the oracle;
the bound on the rows is kept, and an unbounded run stays near the dense model."""

from __future__ import annotations

import pytest
import torch

from community_kv_amd import QuantizedCache, QuantizedCacheAttention, QuantizedKVCache, evict, quantized_append, \
    quantized_attention

pytestmark = pytest.mark.gpu

LAYERS = 2


def _model(device, dtype=torch.bfloat16):
    from transformers import Qwen3Config, Qwen3ForCausalLM

    cfg = Qwen3Config(vocab_size=512, hidden_size=512, intermediate_size=1024, num_hidden_layers=LAYERS,
                      num_attention_heads=8, num_key_value_heads=2, head_dim=128, max_position_embeddings=8192,
                      rope_theta=1e6, tie_word_embeddings=False)
    torch.manual_seed(0)
    with torch.device(device):
        model = Qwen3ForCausalLM(cfg)
    return model.to(dtype).eval()


@pytest.mark.parametrize("budget", [0, 96])
def test_generate_on_the_8_bit_cache(device, budget):
    print(f"generate on the 8-bit cache, budget {budget}", flush=True)
    model = _model(device)
    prompt = torch.randint(0, 512, (1, 150), generator=torch.Generator().manual_seed(1)).to(device)
    new, slack = 40, 8
    cache = QuantizedCache(num_hidden_layers=LAYERS, max_cache_len=256, block=32, budget=budget, num_sink=4, recent=16,
                           slack=slack)
    attention = QuantizedCacheAttention(cache)
    calls = []

    class Recording(QuantizedCacheAttention):
        def forward(self, module, query, key, value, mask, scaling, **kwargs):
            out, none = super().forward(module, query, key, value, mask, scaling, **kwargs)
            calls.append((int(module.layer_idx), query.clone(), key.clone(), value.clone(), scaling, out.clone(),
                          self.cache.layer(int(module.layer_idx)).rows))
            return out, none

    model.set_attn_implementation(Recording(attention.cache).register())
    with torch.no_grad():
        out = model.generate(prompt, past_key_values=cache, max_new_tokens=new, do_sample=False)
    assert out.shape[1] == 150 + new and len(calls) == LAYERS * new
    stores = [QuantizedKVCache.allocate(kv_heads=2, capacity=256, block=32, track_weights=budget > 0, device=device)
              for _ in range(LAYERS)]
    held = [0] * LAYERS
    for layer, query, key, value, scaling, got, rows in calls:
        quantized_append(stores[layer], key, value)
        want, _ = quantized_attention(query, stores[layer], softmax_scale=scaling, accumulate=budget > 0)
        held[layer] += key.shape[2]
        if budget and held[layer] > budget + slack:
            evict(stores[layer], keep=budget, num_sink=4, recent=16)
            held[layer] = budget
        assert torch.equal(got, want) and rows == held[layer]
        assert not budget or rows <= budget + slack
    for layer in range(LAYERS):
        store = cache.layer(layer).store
        store.assert_no_overflow()
        assert store.lengths.tolist() == [held[layer]] == [cache.layer(layer).rows]
        assert cache.layer(layer).get_seq_length() == 150 + new - 1  # the last token is not written
        # the sinks and the newest positions are always there
        live = store.positions[0, :, :held[layer]]
        for position in [0, 1, 2, 3] + list(range(150 + new - 1 - (16 if budget else 60), 150 + new - 1)):
            assert bool((live == position).any(-1).all())


def test_prompt_in_pieces_and_crop(device):
    """The prompt in two forward calls, tokens taken back and written again: the same logits as in one call (rows,
    their order and the block scales are the same; the queries' grouping is not, so up to rounding)."""
    model = _model(device, torch.float32)
    prompt = torch.randint(0, 512, (1, 90), generator=torch.Generator().manual_seed(2)).to(device)
    logits = []
    for pieces in ([90], [50, 40], [70, -10, 30]):
        cache = QuantizedCache(num_hidden_layers=LAYERS, max_cache_len=128, block=16)
        model.set_attn_implementation(QuantizedCacheAttention(cache).register())
        at = 0
        with torch.no_grad():
            for n in pieces:
                if n < 0:
                    cache.crop(at + n)
                    at += n
                    continue
                out = model(prompt[:, at:at + n], past_key_values=cache,
                            position_ids=torch.arange(at, at + n, device=device)[None], use_cache=True)
                at += n
        logits.append(out.logits[:, -1])
    for other in logits[1:]:
        # a query's output does not depend on the others of its call but for the order of 32-bit sums
        assert (other - logits[0]).abs().max() <= 1e-3 * logits[0].abs().max()


def test_another_cache_is_refused(device):
    """Two caches, one registered function: a model run with the other cache, or with none, raises."""
    model = _model(device)
    prompt = torch.randint(0, 512, (1, 20), generator=torch.Generator().manual_seed(3)).to(device)
    caches = [QuantizedCache(num_hidden_layers=LAYERS, max_cache_len=64) for _ in range(2)]
    for cache in caches:
        model.set_attn_implementation(QuantizedCacheAttention(cache).register())
    with torch.no_grad():
        model(prompt, past_key_values=caches[1], use_cache=True)
        with pytest.raises(RuntimeError, match="not written into this cache"):
            model(prompt, past_key_values=caches[0], use_cache=True)
        with pytest.raises(RuntimeError, match="not written into this cache"):
            model(prompt, use_cache=False)


def _windowed_model(device):
    """As _model, in f32, with a sliding layer behind the full one."""
    from transformers import Qwen3ForCausalLM

    cfg = _model("cpu").config
    cfg.use_sliding_window, cfg.sliding_window = True, 33
    cfg.layer_types = ["full_attention", "sliding_attention"]
    torch.manual_seed(0)
    with torch.device(device):
        model = Qwen3ForCausalLM(cfg)
    return model.float().eval()


@pytest.mark.parametrize("sizes", [[90, 61, 1, 1, 5, 1], [200], [1, 1, 1, 140, 1]])
def test_unbounded_run_is_the_dense_model(device, sizes):
    """Prompt pieces, drafts and single tokens of a model with a full and a sliding layer, f32, against the same model
    with the library's masks and attention in 64 bits over the numbers that the codes stand for.

    Queries and keys have norm sqrt(128) (RMS norm, weights of one), so sum|q k| / sqrt(128) <= 11.4, and the oracle's
    bound puts a score within d = 772 * 2^-24 * 11.4 = 5.3e-4, a probability within e^(2 d) - 1 = 1.1e-3 < 2^-9, an
    output within 2^-9 of the largest value.  What so much does to the logits, through codes that flip too, is measured
    on the dense model."""
    from tests import _dense_codes as dense_codes

    model = _windowed_model(device)
    assert [layer.self_attn.sliding_window for layer in model.model.layers] == [None, 33]
    prompt = torch.randint(0, 512, (1, sum(sizes)), generator=torch.Generator().manual_seed(4)).to(device)
    pieces = prompt.split(sizes, 1)
    cache = QuantizedCache(num_hidden_layers=LAYERS, max_cache_len=256, block=32)
    model.set_attn_implementation(QuantizedCacheAttention(cache).register())
    got = dense_codes.logits(model, cache, pieces)

    def dense(noise):
        model.set_attn_implementation(dense_codes.register(noise))
        return dense_codes.logits(model, dense_codes.dense_cache(quantized_append, layers=LAYERS, rows=256, block=32), pieces)

    want, moved = dense(0.0), dense(2.0 ** -9)
    off, tol = (max(float((a - b).abs().max()) for a, b in zip(want, other)) for other in (got, moved))
    assert off <= 2 * tol < 0.2 * max(float(a.abs().max()) for a in want), (off, tol)


def test_assisted_generation_gives_the_greedy_tokens(device):
    """Prompt lookup: rejected candidates are taken back after every verification, none where all were right."""
    model = _model(device, torch.float32)
    some = torch.randint(0, 512, (1, 40), generator=torch.Generator().manual_seed(5))
    prompt = torch.cat([some, some, some[:, :20]], 1).to(device)
    taken, tokens = [], []
    for kwargs in ({}, dict(prompt_lookup_num_tokens=3)):
        cache = QuantizedCache(num_hidden_layers=LAYERS, max_cache_len=256, block=32)
        crop = cache.crop
        cache.crop = lambda n, crop=crop: (taken.append(int(n)), crop(n))
        model.set_attn_implementation(QuantizedCacheAttention(cache).register())
        with torch.no_grad():
            tokens.append(model.generate(prompt, past_key_values=cache, max_new_tokens=60, do_sample=False, **kwargs))
        for layer in range(LAYERS):
            held = cache.layer(layer)
            assert held.rows == held.seen == tokens[-1].shape[1] - 1 and held.store.lengths.tolist() == [held.rows]
    assert torch.equal(tokens[0], tokens[1]) and 0 in taken and min(taken) < 0


def test_padding_is_refused(device):
    model = _model(device)
    prompt = torch.randint(0, 512, (1, 20), generator=torch.Generator().manual_seed(6)).to(device)
    mask = torch.ones_like(prompt)
    for padded in (None, 0, 19):
        cache = QuantizedCache(num_hidden_layers=LAYERS, max_cache_len=64)
        model.set_attn_implementation(QuantizedCacheAttention(cache).register())
        if padded is None:
            model.generate(prompt, attention_mask=mask, past_key_values=cache, max_new_tokens=2, do_sample=False)
            continue
        mask[0, padded] = 0
        with pytest.raises(ValueError, match="padding"):
            model.generate(prompt, attention_mask=mask, past_key_values=cache, max_new_tokens=2, do_sample=False)
        assert cache.get_seq_length() == 0
        mask[0, padded] = 1
