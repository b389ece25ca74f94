"""8-bit KV cache: refusals, layouts and the oracle's own rules, without a GPU."""

from __future__ import annotations

import ctypes
import os

import numpy as np
import pytest
import torch

from community_kv_amd import QuantizedKVCache, evict, quantized_append, quantized_attention
from community_kv_amd import _native as nat
from oracle import quantized as oq


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(nat.LIB_PATH):
        nat.build()
    return nat.lib()


def _cache(**kwargs):
    return QuantizedKVCache.allocate(**dict(dict(batch=2, kv_heads=2, capacity=100, block=32, track_weights=True,
                                                 device="cpu"), **kwargs))


def test_allocate_layout():
    cache = _cache()
    assert cache.capacity == 128 and cache.batch == 2 and cache.kv_heads == 2
    assert cache.key_codes.dtype == torch.float8_e4m3fn and cache.key_codes.shape == (2, 2, 128, 128)
    assert cache.key_scales.shape == cache.value_scales.shape == (2, 2, 4)
    assert cache.positions.shape == cache.weights.shape == (2, 2, 128)
    assert cache.cursors.shape == (3, 2) and cache.lengths.tolist() == [0, 0]
    assert _cache(track_weights=False).weights is None


def test_reset_rewind_overflow_flag():
    cache = _cache()
    cache.cursors.copy_(torch.tensor([[7, 5], [9, 5], [0, 0]], dtype=torch.int32))
    cache.rewind(torch.tensor([2, 0], dtype=torch.int32))
    cache.rewind(1)
    with pytest.raises(ValueError):
        cache.rewind(-1)
    assert cache.cursors.tolist() == [[4, 4], [6, 4], [0, 0]]
    cache.assert_no_overflow()
    cache.cursors[2, 1] = 1
    with pytest.raises(RuntimeError, match="overflow"):
        cache.assert_no_overflow()
    cache.reset()
    assert not cache.cursors.any()


@pytest.mark.parametrize("change,error", [
    (dict(batch=0), ValueError), (dict(kv_heads=0), ValueError), (dict(capacity=0), ValueError),
    (dict(block=48), ValueError), (dict(block=256), ValueError)])
def test_allocate_refuses(change, error):
    with pytest.raises(error):
        _cache(**change)


def _tensors(cache):
    return dict(key_codes=cache.key_codes, value_codes=cache.value_codes, key_scales=cache.key_scales,
                value_scales=cache.value_scales, positions=cache.positions, cursors=cache.cursors, block=cache.block,
                weights=cache.weights)


@pytest.mark.parametrize("name,value,error", [
    ("key_codes", torch.zeros(2, 2, 128, 64), ValueError),
    ("key_codes", torch.zeros(2, 2, 128, 128, dtype=torch.uint8), TypeError),
    ("key_codes", torch.zeros(2, 2, 96, 128, dtype=torch.uint8).view(torch.float8_e4m3fn), ValueError),
    ("value_codes", torch.zeros(2, 2, 128, 128), TypeError),
    ("key_scales", torch.zeros(2, 2, 5), ValueError),
    ("value_scales", torch.zeros(2, 2, 4, dtype=torch.float64), TypeError),
    ("key_scales", torch.full((2, 2, 4), 1.5), ValueError),
    ("value_scales", torch.full((2, 2, 4), float("inf")), ValueError),
    ("value_scales", torch.full((2, 2, 4), -1.0), ValueError),
    ("value_scales", torch.full((2, 2, 4), 2.0 ** -65), ValueError),
    ("positions", torch.zeros(2, 2, 128, dtype=torch.int64), TypeError),
    ("cursors", torch.zeros(2, 2, dtype=torch.int32), ValueError),
    ("weights", torch.zeros(2, 2, 128, 2)[..., 0], ValueError),
    ("block", 24, ValueError)])
def test_from_tensors_refuses(name, value, error):
    good = _tensors(_cache())
    assert QuantizedKVCache.from_tensors(**good).key_codes is good["key_codes"]
    with pytest.raises(error):
        QuantizedKVCache.from_tensors(**(good | {name: value}))


def test_from_tensors_takes_the_whole_range_of_scales():
    good = _tensors(_cache())
    good["key_scales"] = torch.tensor([0.0, 2.0 ** -64, 1.0, 2.0 ** 120]).expand(2, 2, 4).contiguous()
    QuantizedKVCache.from_tensors(**good)


def test_calls_refuse_bad_arguments():
    cache, other = _cache(), _cache()
    x = torch.zeros(2, 2, 3, 128)
    bad = [(TypeError, lambda: quantized_append(cache, x.double(), x.double())),
           (TypeError, lambda: quantized_append(cache, x, x.half())),
           (ValueError, lambda: quantized_append(cache, x[:1], x[:1])),
           (ValueError, lambda: quantized_append(cache, x[:, :1], x[:, :1])),
           (ValueError, lambda: quantized_append(cache, x, x[:, :, :2])),
           (ValueError, lambda: quantized_append(cache, x[..., :64], x[..., :64])),
           (ValueError, lambda: quantized_append(cache, x[0], x[0])),
           (TypeError, lambda: quantized_append(cache, x, x, counts=torch.tensor([1, 2]))),
           (TypeError, lambda: quantized_append(cache, x, x, counts=torch.tensor([1], dtype=torch.int32))),
           (RuntimeError, lambda: quantized_append(cache, x.clone().requires_grad_(), x)),
           (ValueError, lambda: quantized_attention(torch.zeros(2, 3, 1, 128), cache, softmax_scale=1.0)),
           (ValueError, lambda: quantized_attention(torch.zeros(2, 34, 1, 128), cache, softmax_scale=1.0)),
           (ValueError, lambda: quantized_attention(x, cache, softmax_scale=0.0)),
           (ValueError, lambda: quantized_attention(x, cache, softmax_scale=float("nan"))),
           (ValueError, lambda: quantized_attention(x, cache, softmax_scale=float("inf"))),
           (ValueError, lambda: quantized_attention(x, cache, softmax_scale=1.0, window=-1)),
           (ValueError, lambda: quantized_attention(x, _cache(track_weights=False), softmax_scale=1.0, accumulate=True)),
           (RuntimeError, lambda: quantized_attention(x.clone().requires_grad_(), cache, softmax_scale=1.0)),
           (ValueError, lambda: evict(_cache(track_weights=False), keep=4)),
           (ValueError, lambda: evict(cache, keep=0)),
           (ValueError, lambda: evict(cache, keep=8, num_sink=5, recent=4)),
           (ValueError, lambda: evict(cache, keep=8, num_sink=-1)),
           (ValueError, lambda: evict(cache, keep=8, recent=-1)),
           (ValueError, lambda: evict(cache, keep=8, into=cache)),
           (ValueError, lambda: evict(cache, keep=8, into=_cache(block=64))),
           (ValueError, lambda: evict(cache, keep=8, into=_cache(batch=1))),
           (ValueError, lambda: evict(cache, keep=100, into=_cache(capacity=64)))]
    for error, call in bad:
        with pytest.raises(error):
            call()
    # nothing runs on the CPU in the kernels' place
    for call in (lambda: quantized_append(cache, x, x), lambda: quantized_attention(x, cache, softmax_scale=1.0),
                 lambda: evict(cache, keep=8), lambda: evict(cache, keep=8, into=other)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def _struct(**change):
    s = nat.QuantCache(*[0x1000] * 8, 128, 2, 2, 32)
    for name, value in change.items():
        setattr(s, name, value)
    return s


@pytest.mark.parametrize("change", [
    dict(key_codes=None), dict(value_codes=None), dict(key_scales=None), dict(value_scales=None), dict(positions=None),
    dict(cursors=None), dict(counters=None), dict(capacity=0), dict(capacity=100), dict(batch=0), dict(kv_heads=-1),
    dict(block=48), dict(block=0), dict(key_codes=0x1008), dict(batch=40000), dict(capacity=(1 << 30) + 32)])
def test_c_entries_refuse_a_bad_cache(lib, change):
    rows, bad = nat.QuantRows(0x1000, 0, 0, 0), _struct(**change)
    b, r = ctypes.byref(bad), ctypes.byref(rows)
    assert lib.ckv_quant_append(b, r, r, 1, None, nat.CKV_BF16, None) != 0
    assert lib.ckv_quant_attention(b, r, 4, 1, None, nat.CKV_BF16, 1.0, 0, 0, 0x1000, 0x1000, 0x1000, None) != 0
    assert lib.ckv_quant_evict(b, None, 16, 0, 0, 0x1000, None) != 0
    assert lib.ckv_last_error()


def test_c_entries_refuse_bad_arguments(lib):
    good, rows = _struct(), nat.QuantRows(0x1000, 256, 128, 128)
    c, r = ctypes.byref(good), ctypes.byref(rows)

    def append(key=r, value=r, tokens=1, dtype=nat.CKV_BF16):
        return lib.ckv_quant_append(c, key, value, tokens, None, dtype, None)

    def attend(query=r, heads=4, tokens=1, dtype=nat.CKV_BF16, scale=1.0, window=0, accumulate=0, out=0x1000,
               lse=0x1000, workspace=0x1000, cache=c):
        return lib.ckv_quant_attention(cache, query, heads, tokens, None, dtype, scale, window, accumulate, out, lse,
                                       workspace, None)

    odd = ctypes.byref(nat.QuantRows(0x1000, 256, 128, 132))
    off = ctypes.byref(nat.QuantRows(0x1008, 256, 128, 128))
    none = ctypes.byref(nat.QuantRows(None, 256, 128, 128))
    for rc in (append(tokens=0), append(dtype=nat.CKV_E4M3), append(dtype=9), append(key=odd), append(value=off),
               append(value=none), attend(query=odd), attend(query=off), attend(query=none), attend(heads=3),
               attend(heads=0), attend(heads=34), attend(tokens=0), attend(tokens=1 << 24), attend(dtype=7),
               attend(scale=0.0), attend(scale=float("nan")), attend(scale=float("inf")), attend(window=-1),
               attend(out=None), attend(lse=None), attend(workspace=None, accumulate=1), attend(workspace=0x1004, accumulate=1),
               attend(cache=ctypes.byref(_struct(weights=None)), accumulate=1)):
        assert rc in (1, 2)

    def evicting(cache=c, into=None, keep=16, num_sink=0, recent=0, workspace=0x1000):
        return lib.ckv_quant_evict(cache, into, keep, num_sink, recent, workspace, None)

    def to(**change):
        apart = dict(key_codes=0x2000, value_codes=0x2000, cursors=0x2000)
        return ctypes.byref(_struct(**(apart | change)))

    for rc in (evicting(cache=ctypes.byref(_struct(weights=None))), evicting(keep=0), evicting(num_sink=-1),
               evicting(recent=-1), evicting(num_sink=9, recent=8), evicting(workspace=None),
               evicting(workspace=0x1004), evicting(into=c), evicting(into=to(block=64)), evicting(into=to(batch=1)),
               evicting(into=to(kv_heads=1)), evicting(into=to(capacity=32), keep=64),
               evicting(num_sink=2**31 - 1, recent=2**31 - 1)):
        assert rc in (1, 2)
    assert evicting(keep=128) == 0  # no sequence can hold more: nothing to launch


def test_workspace_sizes(lib):
    c = ctypes.byref(_struct())
    assert lib.ckv_quant_evict_workspace_bytes(c, 16) >= 4 * (128 + 16) * 4
    assert lib.ckv_quant_evict_workspace_bytes(c, 0) == lib.ckv_quant_evict_workspace_bytes(None, 4) == 0
    assert lib.ckv_quant_attention_workspace_bytes(c, 3, 1, nat.CKV_BF16, 0) == 0
    assert lib.ckv_quant_attention_workspace_bytes(None, 4, 1, nat.CKV_BF16, 0) == 0
    plain = lib.ckv_quant_attention_workspace_bytes(c, 4, 5, nat.CKV_F32, 0)
    assert lib.ckv_quant_attention_workspace_bytes(c, 4, 5, nat.CKV_F32, 1) >= plain + 2 * 2 * 10 * 8


def test_oracle_block_scale_and_growth():
    assert oq.block_scale(448.0) == 1.0 and oq.block_scale(448.0 * (1 + 2.0 ** -20)) == 2.0
    assert oq.block_scale(0.0) == 2.0 ** -64 and oq.block_scale(3.4e38) == 2.0 ** 120
    cache = oq.Cache.of(_cache(batch=1, kv_heads=1))
    rng = np.random.default_rng(0)
    x = rng.standard_normal((1, 1, 40, 128)) * np.exp(rng.standard_normal((1, 1, 40, 1)))
    for t in range(40):  # token by token: scales grow within a block
        cache.append(x[:, :, t:t + 1], x[:, :, t:t + 1])
    whole = oq.Cache.of(_cache(batch=1, kv_heads=1))
    whole.append(x, x)
    assert np.array_equal(cache.scales[0], whole.scales[0])
    got, want = cache.value(0, 0, 0, np.arange(40)), x[0, 0]
    step = np.maximum(np.abs(want) * 2.0 ** -4, whole.scales[0][0, 0, np.arange(40) // 32][:, None] * 2.0 ** -9)
    assert (np.abs(got - want) <= step).all()  # half a step, and another half among the subnormals


# ------------------------------------------------------------------------------------------ Hugging Face cache

@pytest.mark.parametrize("change", [dict(max_cache_len=0), dict(budget=-1), dict(budget=64, num_sink=10, recent=60),
                                    dict(budget=64, slack=64), dict(slack=-1)])
def test_cache_layer_refuses(change):
    from community_kv_amd.attention import QuantizedCacheLayer

    with pytest.raises(ValueError):
        QuantizedCacheLayer(**(dict(max_cache_len=128, num_sink=4, recent=16) | change))


def test_cache_layer_protocol():
    from community_kv_amd import QuantizedCache

    cache = QuantizedCache(num_hidden_layers=2, max_cache_len=100)
    layer = cache.layer(1)
    assert cache.get_seq_length() == 0 and layer.get_max_length() == 100 and not layer.is_initialized
    x = torch.zeros(1, 2, 101, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="capacity"):
        cache.update(x, x, 1)
    with pytest.raises(ValueError, match="one sequence"):
        cache.update(x.expand(2, 2, 101, 128)[:, :, :3], x.expand(2, 2, 101, 128)[:, :, :3], 1)
    with pytest.raises(RuntimeError, match="GPU only"):
        cache.update(x[:, :, :3], x[:, :, :3], 1)
    assert layer.seen == 0 and layer.rows == 0
    with pytest.raises(RuntimeError, match="not written into this cache"):
        layer.attend(x[:, :, :1], x[:, :, :1], 1.0)
    with pytest.raises(NotImplementedError):
        layer.reorder_cache(torch.zeros(1, dtype=torch.long))
    with pytest.raises(NotImplementedError):
        layer.offload()
    layer.rows, layer.seen = 40, 40
    layer.store.cursors[:2] = 40
    layer.crop(38)
    layer.crop(-3)
    layer.crop(99)
    assert layer.rows == layer.seen == 35 and layer.store.cursors.tolist() == [[35], [35], [0]]
    layer.budget, layer.seen = 30, 60
    with pytest.raises(ValueError, match="evicted"):
        layer.crop(50)
    layer.reset()
    assert layer.seen == 0 and not layer.store.cursors.any()


def test_attention_function_refuses_what_it_does_not_do():
    from community_kv_amd import QuantizedCache, QuantizedCacheAttention

    attention = QuantizedCacheAttention(QuantizedCache(num_hidden_layers=1, max_cache_len=64))
    module = torch.nn.Module()
    module.layer_idx = 0
    x = torch.zeros(1, 2, 1, 128)
    for extra in (dict(dropout=0.1), dict(softcap=30.0), dict(s_aux=torch.zeros(2)), dict(is_causal=False),
                  dict(attention_mask=torch.zeros(1, 1, 1, 1))):
        with pytest.raises(ValueError):
            attention.forward(module, x, x, x, **(dict(attention_mask=None, scaling=1.0) | extra))


@pytest.mark.parametrize("keep,num_sink,recent", [(1000, 10, 500), (200, 4, 126), (129, 64, 65), (2**40, 2**39, 2**39),
                                                  (128, 128, 0), (100, 0, 100)])
@pytest.mark.parametrize("into", [False, True])
def test_evict_to_more_rows_than_there_are(lib, monkeypatch, keep, num_sink, recent, into):
    """`keep` may exceed the capacity, and the protected rows with it: the C entry gets numbers that it takes."""
    from community_kv_amd.attention import quantized

    cache, target = _cache(), _cache() if into else None  # 128 rows
    calls = []
    monkeypatch.setattr(nat, "require_device", lambda *tensors: torch.device("cpu"))
    monkeypatch.setattr(quantized, "_call", lambda device, function, *args: calls.append(args))
    evict(cache, keep=keep, num_sink=num_sink, recent=recent, into=target)
    (_, _, c_keep, c_sink, c_recent, _), = calls
    assert 0 < c_keep <= 128 and 0 <= c_sink and 0 <= c_recent and c_sink + c_recent <= c_keep
    if keep <= 128:
        assert (c_keep, c_sink, c_recent) == (keep, num_sink, recent)
    if not into and c_keep == 128:
        # no sequence can hold more, so nothing is launched and the entry itself may be called
        assert lib.ckv_quant_evict(cache._ref, None, c_keep, c_sink, c_recent, 0x1000, None) == 0


@pytest.mark.parametrize("shared", ["key_codes", "value_codes", "key_scales", "value_scales", "positions", "weights",
                                    "cursors"])
@pytest.mark.parametrize("whole", [False, True])
def test_evict_refuses_a_target_that_shares_memory(lib, shared, whole):
    """Any tensor of the source's among the target's, or one that begins within it."""
    cache, tensors = _cache(), _tensors(_cache())
    if whole:
        tensors[shared] = getattr(cache, shared)
    else:
        good = tensors[shared]
        bytes_ = torch.zeros(2 * good.nbytes, dtype=torch.uint8)

        def part(first):
            return bytes_[first:first + good.nbytes].view(good.dtype).view(good.shape)

        step = max(16, good.nbytes // 32 * 16)
        cache = QuantizedKVCache.from_tensors(**(_tensors(cache) | {shared: part(0)}))
        tensors[shared] = part(min(step, good.nbytes - 8))
    into = QuantizedKVCache.from_tensors(**tensors)
    for a, b in ((cache, into), (into, cache)):
        assert lib.ckv_quant_evict(a._ref, b._ref, 16, 0, 0, 0x1000, None) == 1
        assert b"another cache" in lib.ckv_last_error()


@pytest.mark.parametrize("one,other", [("key_codes", "value_codes"), ("key_scales", "value_scales"),
                                       ("positions", "weights")])
def test_a_cache_over_one_tensor_twice_is_refused(one, other):
    tensors = _tensors(_cache())
    tensors[other] = tensors[one].view(tensors[other].dtype)
    with pytest.raises(ValueError, match="share"):
        QuantizedKVCache.from_tensors(**tensors)
    buffer = torch.zeros(tensors[one].nbytes * 2, dtype=torch.uint8)
    for gap in (0, tensors[one].nbytes // 32 * 16):
        first, second = buffer[:tensors[one].nbytes], buffer[tensors[one].nbytes - gap:2 * tensors[one].nbytes - gap]
        for name, part in ((one, first), (other, second)):
            tensors[name] = part.view(tensors[name].dtype).view(tensors[name].shape)
        if gap:
            with pytest.raises(ValueError, match="share"):
                QuantizedKVCache.from_tensors(**tensors)
        else:
            QuantizedKVCache.from_tensors(**tensors)
