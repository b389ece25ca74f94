"""8-bit KV cache on the GPU against the 64-bit oracle (oracle/quantized.py):
codes, scales, positions and cursors equal, attention and received weights
within the bounds derived there."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from community_kv_amd import QuantizedKVCache, evict, quantized_append, quantized_attention
from oracle import quantized as oq

pytestmark = pytest.mark.gpu

D = 128
SCALE = D ** -0.5
PIECES = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _rows(gen, *shape, dtype=torch.float32, size=1.0):
    x = torch.randn(*shape, D, generator=gen) * torch.exp(0.5 * torch.randn(*shape, 1, generator=gen)) * size
    return x.to(dtype)


def _i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _same(cache, oracle, what=""):
    got = oq.Cache.of(cache)
    for name, a, b in (("positions", got.positions, oracle.positions), ("cursors", got.cursors, oracle.cursors),
                       ("key scales", got.scales[0], oracle.scales[0]),
                       ("value scales", got.scales[1], oracle.scales[1]), ("weights", got.weights, oracle.weights)):
        assert np.array_equal(a, b, equal_nan=a.dtype.kind == "f"), (what, name)
    for name, a, b in (("keys", got.codes[0], oracle.codes[0]), ("values", got.codes[1], oracle.codes[1])):
        # a NaN may carry either sign
        nan_a, nan_b = (a & 0x7F) == 0x7F, (b & 0x7F) == 0x7F
        assert np.array_equal(nan_a, nan_b) and np.array_equal(a[~nan_a], b[~nan_b]), (what, name)


def _append(cache, oracle, key, value, counts=None):
    dev = cache.device
    quantized_append(cache, key.to(dev), value.to(dev), counts=None if counts is None else _i32(counts, dev))
    oracle.append(key.double().numpy(), value.double().numpy(), counts)


def _fill(device, gen, *, batch, heads, capacity, block, lengths, weights=True, mixed=True):
    """A cache with `lengths` rows in use, rows in mixed order, and garbage (NaN codes too) past them."""
    cache = QuantizedKVCache.allocate(batch=batch, kv_heads=heads, capacity=capacity, block=block,
                                      track_weights=weights, device=device)
    for codes in (cache.key_codes, cache.value_codes):
        codes.view(torch.uint8).copy_(torch.randint(0, 256, codes.shape, generator=gen, dtype=torch.uint8))
    most = max(lengths)
    if most:
        quantized_append(cache, _rows(gen, batch, heads, most).to(device), _rows(gen, batch, heads, most).to(device),
                         counts=_i32(lengths, device))
    if mixed:
        for b, n in enumerate(lengths):
            for h in range(heads):
                order = torch.randperm(n, generator=gen).to(device)
                cache.positions[b, h, :n] = cache.positions[b, h, :n][order]
    if weights:
        # few distinct values, so that equal weights occur
        cache.weights.copy_((torch.rand(cache.weights.shape, generator=gen) * 30).round() / 4)
    return cache


# ------------------------------------------------------------------------------------------ append

@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_append_matches_oracle(device, block, dtype):
    """Appends of many sizes behind one another, ragged counts, rows past the length untouched."""
    print(f"append block={block} dtype={dtype}", flush=True)
    gen = torch.Generator().manual_seed(block)
    cache = _fill(device, gen, batch=3, heads=2, capacity=640, block=block, lengths=[0, 5, 130], mixed=False)
    oracle = oq.Cache.of(cache)
    for step, (tokens, counts, size) in enumerate([(1, None, 1.0), (1, None, 30.0), (70, [70, 0, 33], 0.2), (17, None, 1e-3),
                                                   (200, [1, 200, 199], 500.0), (1, [0, 1, 0], 1.0), (3, [-4, 9, 2], 2.0)]):
        key = _rows(gen, 3, 2, tokens, dtype=dtype, size=size)
        value = _rows(gen, 3, 2, tokens, dtype=dtype, size=1 / size if dtype != torch.float16 else size)
        _append(cache, oracle, key, value, counts)
        torch.cuda.synchronize()
        _same(cache, oracle, f"step {step}")


def test_append_token_by_token(device):
    """Single tokens of growing size: the block's earlier codes follow its scale, subnormals included."""
    gen = torch.Generator().manual_seed(3)
    cache = QuantizedKVCache.allocate(batch=1, kv_heads=3, capacity=128, block=64, device=device)
    oracle = oq.Cache.of(cache)
    for t in range(80):
        size = 2.0 ** ((t % 40) / 3 - 6)
        _append(cache, oracle, _rows(gen, 1, 3, 1, size=size), _rows(gen, 1, 3, 1, size=1 / size))
    torch.cuda.synchronize()
    _same(cache, oracle)


def test_append_strides_and_alignment(device):
    """[batch, token, head] memory order, a slice of a wider tensor, broadcast rows, an odd offset, a strided last dim."""
    gen = torch.Generator().manual_seed(4)
    wide = _rows(gen, 2, 9, 6, dtype=torch.bfloat16)  # [B, T, heads]
    flat = torch.randn(2 * 2 * 9 * D + 1, generator=gen).bfloat16()
    views = [wide[:, :, 2:4].transpose(1, 2), wide[:, :1, :2].transpose(1, 2).expand(2, 2, 9, D),
             flat[1:].view(2, 2, 9, D), _rows(gen, 2, 2, 9, dtype=torch.bfloat16).repeat_interleave(2, -1)[..., ::2],
             wide[:, 3:4, 2:4].transpose(1, 2)]
    for i, view in enumerate(views):
        cache = QuantizedKVCache.allocate(batch=2, kv_heads=2, capacity=64, block=32, device=device)
        oracle = oq.Cache.of(cache)
        base = [wide, wide, flat, None, wide][i]
        if base is None:
            dev_view = view.repeat_interleave(2, -1).to(device)[..., ::2]
        else:
            dev_view = base.to(device).as_strided(view.shape, view.stride(), view.storage_offset())
        quantized_append(cache, dev_view, dev_view)
        oracle.append(view.double().numpy(), view.double().numpy())
        torch.cuda.synchronize()
        _same(cache, oracle, f"view {i}")


def test_append_special_values(device):
    """NaN and infinities become NaN in their place and leave the scale alone; zeros, the types' extremes."""
    for dtype, big, tiny in ((torch.float32, 3.4e38, 1e-45), (torch.float16, 65504.0, 6e-8),
                             (torch.bfloat16, 3.38e38, 1e-40)):
        key = torch.zeros(1, 2, 40, D, dtype=dtype)
        key[0, 0, :, ::3] = 1.5
        key[0, 0, 3, 5], key[0, 0, 20, 7], key[0, 0, 20, 8] = float("nan"), float("inf"), -float("inf")
        key[0, 1, 1, 1], key[0, 1, 33, 2], key[0, 1, 35, 2] = big, tiny, -tiny
        value = torch.full((1, 2, 40, D), float("nan"), dtype=dtype)
        value[0, 1, 32:] = 0
        cache = QuantizedKVCache.allocate(kv_heads=2, capacity=64, block=32, device=device)
        oracle = oq.Cache.of(cache)
        _append(cache, oracle, key, value)
        _append(cache, oracle, key[:, :, :7] * 0.5, value[:, :, :7])
        torch.cuda.synchronize()
        _same(cache, oracle, str(dtype))


def test_append_overflow(device):
    """Tokens past the capacity are dropped and flagged; the rest is written."""
    gen = torch.Generator().manual_seed(5)
    cache = _fill(device, gen, batch=3, heads=1, capacity=64, block=32, lengths=[60, 64, 10], mixed=False)
    oracle = oq.Cache.of(cache)
    _append(cache, oracle, _rows(gen, 3, 1, 6), _rows(gen, 3, 1, 6))
    torch.cuda.synchronize()
    _same(cache, oracle)
    assert cache.cursors.tolist() == [[64, 64, 16], [64, 64, 16], [1, 1, 0]]
    with pytest.raises(RuntimeError, match="overflow"):
        cache.assert_no_overflow()
    _append(cache, oracle, _rows(gen, 3, 1, 300), _rows(gen, 3, 1, 300))
    torch.cuda.synchronize()
    _same(cache, oracle)
    quantized_append(cache, torch.zeros(3, 1, 0, D, device=device), torch.zeros(3, 1, 0, D, device=device))
    torch.cuda.synchronize()
    _same(cache, oracle)


# ------------------------------------------------------------------------------------------ attention

def _attend_case(device, gen, cache, *, group, tokens, dtype, counts=None, window=0, accumulate=False, query=None,
                 scale=SCALE, what=""):
    heads = cache.kv_heads
    if query is None:
        query = _rows(gen, cache.batch, heads * group, tokens, dtype=dtype)
    before = cache.weights.clone() if accumulate else None
    out, lse = quantized_attention(query.to(device), cache, softmax_scale=scale, window=window, accumulate=accumulate,
                                   counts=None if counts is None else _i32(counts, device))
    torch.cuda.synchronize()
    oracle = oq.Cache.of(cache)
    want, tol = oracle.attend(query.double().numpy(), scale=scale, counts=counts, window=window,
                              pieces=PIECES[dtype], half_step=HALF_STEP[dtype])
    assert out.dtype == dtype and out.shape == want[0].shape and lse.shape == want[1].shape
    got = out.double().cpu().numpy()
    assert (np.abs(got - want[0]) <= tol[0]).all(), (what, "out", float(np.abs(got - want[0]).max()))
    got = lse.double().cpu().numpy()
    empty = np.isneginf(want[1])
    assert np.array_equal(np.isneginf(got), empty), (what, "empty rows")
    assert (np.abs(got[~empty] - want[1][~empty]) <= tol[1][~empty]).all(), (what, "lse")
    if accumulate:
        got = (cache.weights - before).double().cpu().numpy()
        # the sums went onto weights up to 8 (a rounding of the sum), and the difference is exact or rounded once
        slack = 2 * oq.U * (np.abs(cache.weights.double().cpu().numpy()) + np.abs(before.double().cpu().numpy()))
        assert (np.abs(got - want[2]) <= tol[2] + slack).all(), (what, "weights")
    return out, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("block", [16, 64, 128])
def test_attend_single_token(device, dtype, block):
    """One query a sequence over lengths around every tile edge, an empty sequence among them."""
    gen = torch.Generator().manual_seed(block)
    lengths = [0, 1, 31, 33, 128, 129, 511, 640]
    print(f"attend one token block={block} dtype={dtype}", flush=True)
    cache = _fill(device, gen, batch=8, heads=2, capacity=640, block=block, lengths=lengths)
    for group in (1, 4, 16):
        _attend_case(device, gen, cache, group=group, tokens=1, dtype=dtype, accumulate=True, what=f"group {group}")


@pytest.mark.parametrize("tokens,group,dtype", [(2, 1, torch.float32), (5, 4, torch.bfloat16), (7, 7, torch.float32),
                                                (33, 2, torch.float16), (40, 5, torch.bfloat16)])
@pytest.mark.parametrize("window", [0, 1, 37, 2**31 - 1])
def test_attend_several_tokens(device, tokens, group, dtype, window):
    """Several queries a sequence: masks by position over mixed rows, ragged counts, windows that leave few rows."""
    gen = torch.Generator().manual_seed(tokens)
    print(f"attend tokens={tokens} group={group} dtype={dtype} window={window}", flush=True)
    cache = _fill(device, gen, batch=3, heads=2, capacity=320, block=32, lengths=[tokens, 100 + tokens, 290])
    _attend_case(device, gen, cache, group=group, tokens=tokens, dtype=dtype, window=window, accumulate=True)
    _attend_case(device, gen, cache, group=group, tokens=tokens, dtype=dtype, window=window, accumulate=True,
                 counts=[tokens, 0, (tokens + 1) // 2])


@pytest.mark.parametrize("tokens,group,dtype", [(33, 2, torch.float16), (40, 5, torch.bfloat16), (80, 1, torch.bfloat16),
                                                (30, 7, torch.float32)])
@pytest.mark.parametrize("window", [0, 1, 37, 2**31 - 1])
@pytest.mark.parametrize("accumulate", [False, True])
def test_attend_many_rows_of_a_large_cache(device, tokens, group, dtype, window, accumulate):
    """Short sequences in a large cache, whose capacity alone sends the calls to the many-row kernels."""
    gen = torch.Generator().manual_seed(tokens + 7)
    print(f"attend many rows tokens={tokens} group={group} dtype={dtype} window={window}", flush=True)
    cache = _fill(device, gen, batch=3, heads=2, capacity=24_064, block=32, lengths=[tokens, 100 + tokens, 290])
    for counts in (None, [tokens, 0, (tokens + 1) // 2]):
        _attend_case(device, gen, cache, group=group, tokens=tokens, dtype=dtype, window=window, accumulate=accumulate,
                     counts=counts)


def test_attend_same_rows_in_a_small_and_a_large_cache(device):
    """The kernels that a call goes to depend on the capacity: their results agree within the roundings of both."""
    gen = torch.Generator().manual_seed(40)
    key, value, query = (_rows(gen, 1, heads, 260) for heads in (2, 2, 8))
    seen = []
    for capacity in (320, 65_536):
        cache = QuantizedKVCache.allocate(kv_heads=2, capacity=capacity, block=32, device=device)
        quantized_append(cache, key.to(device), value.to(device))
        seen.append(quantized_attention(query.to(device), cache, softmax_scale=SCALE))
    torch.cuda.synchronize()
    # both are within the oracle's bound (test_attend_several_tokens), here 2^-16 of values up to 5 at the least
    assert (seen[0][0] - seen[1][0]).abs().max() <= 2 * 5 * 2.0 ** -16
    assert (seen[0][1] - seen[1][1]).abs().max() <= 2 * 10 * 2.0 ** -16


@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("tokens,dtype", [(1, torch.bfloat16), (4, torch.float16), (6, torch.float32), (30, torch.bfloat16)])
def test_attend_window_over_long_caches(device, mixed, tokens, dtype):
    """Most steps hold no row in sight and are passed over, in parts of one or several units; also where the window
    begins or ends inside a step, with sequences that are shorter than it, empty or without a query."""
    print(f"attend window mixed={mixed} tokens={tokens} dtype={dtype}", flush=True)
    gen = torch.Generator().manual_seed(tokens + 100)
    lengths = [4000, 2913, 35, 0, 1025]
    cache = _fill(device, gen, batch=5, heads=1, capacity=4000, block=16, lengths=lengths, mixed=mixed)
    counts = [tokens, 0, (tokens + 1) // 2, 0, tokens]
    for window in (1, 33, 96, 1000):
        _attend_case(device, gen, cache, group=4, tokens=tokens, dtype=dtype, window=window, accumulate=True,
                     counts=counts, what=f"window {window}")
    one = _fill(device, gen, batch=1, heads=8, capacity=9008, block=16, lengths=[9001], mixed=mixed)
    _attend_case(device, gen, one, group=2, tokens=tokens, dtype=dtype, window=700, accumulate=True, what="one")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attend_parts_of_many_rows(device, dtype):
    """Prompt rows in several parts, of sequences some of which are one part."""
    gen = torch.Generator().manual_seed(31)
    cache = _fill(device, gen, batch=3, heads=1, capacity=3200, block=64, lengths=[3200, 300, 90])
    for counts in ([80, 80, 80], [80, 33, 0]):
        _attend_case(device, gen, cache, group=1, tokens=80, dtype=dtype, accumulate=True, counts=counts)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attend_long_prompt_rows(device, dtype):
    """A whole prompt's queries at once (many row blocks, the causal diagonal)."""
    gen = torch.Generator().manual_seed(8)
    cache = _fill(device, gen, batch=1, heads=1, capacity=320, block=64, lengths=[300], mixed=False)
    _attend_case(device, gen, cache, group=4, tokens=300, dtype=dtype, accumulate=True)
    _attend_case(device, gen, cache, group=4, tokens=211, dtype=dtype, accumulate=True, window=64)


def test_attend_many_sequences(device):
    """More sequences than lanes of a wave, lengths from none to several parts, one KV head."""
    gen = torch.Generator().manual_seed(15)
    lengths = torch.randint(0, 700, (70,), generator=gen).tolist()
    lengths[0], lengths[64], lengths[69] = 0, 0, 704
    cache = _fill(device, gen, batch=70, heads=1, capacity=704, block=32, lengths=lengths)
    _attend_case(device, gen, cache, group=2, tokens=1, dtype=torch.bfloat16, accumulate=True)
    counts = [min(3, n) for n in lengths]
    _attend_case(device, gen, cache, group=2, tokens=3, dtype=torch.float16, accumulate=True, counts=counts)


@pytest.mark.parametrize("group,tokens,dtype", [(2, 3, torch.bfloat16), (4, 12, torch.bfloat16), (5, 40, torch.bfloat16),
                                                (4, 20, torch.float32)])
@pytest.mark.parametrize("capacity", [320, 65_536])  # few-row kernels, many-row ones
def test_attend_padded_queries_hold_anything(device, group, tokens, dtype, capacity):
    """Queries past a sequence's count, NaN here, touch neither the others' outputs nor the received weights."""
    gen = torch.Generator().manual_seed(16)
    cache = _fill(device, gen, batch=2, heads=2, capacity=capacity, block=64, lengths=[300, 129])
    query = _rows(gen, 2, 2 * group, tokens, dtype=dtype)
    counts = [tokens - 1, tokens // 2]
    weights = cache.weights.clone()
    clean = quantized_attention(query.to(device), cache, softmax_scale=SCALE, counts=_i32(counts, device), accumulate=True)
    clean += (cache.weights.clone(),)
    cache.weights.copy_(weights)
    for b in range(2):
        query[b, :, counts[b]:] = float("nan")
    got = quantized_attention(query.to(device), cache, softmax_scale=SCALE, counts=_i32(counts, device), accumulate=True)
    torch.cuda.synchronize()
    for a, b in zip(clean, got + (cache.weights,)):
        assert torch.equal(a, b) and not b.isnan().any()


def test_attend_window_leaves_rows_empty(device):
    """Rows whose window holds no cached position: zeros and -inf, no NaN, no weight."""
    gen = torch.Generator().manual_seed(9)
    cache = _fill(device, gen, batch=2, heads=2, capacity=128, block=32, lengths=[90, 128], mixed=False)
    cache.cursors[1] += 500  # far ahead of every cached position
    out, lse = _attend_case(device, gen, cache, group=2, tokens=3, dtype=torch.bfloat16, window=100, accumulate=True)
    assert not out.any() and bool((lse == -float("inf")).all())


@pytest.mark.parametrize("group,tokens,dtype", [(2, 4, torch.bfloat16), (16, 20, torch.bfloat16),
                                                (5, 30, torch.float32)])
@pytest.mark.parametrize("capacity", [192, 131_072])
def test_attend_ignores_nan_in_masked_rows(device, group, tokens, dtype, capacity):
    """NaN keys and values at masked positions and past the length change nothing; a NaN value that a query does
    see makes that query's dim NaN, and a NaN key the whole query.  Few query rows, and many."""
    gen = torch.Generator().manual_seed(10)
    cache = _fill(device, gen, batch=1, heads=1, capacity=capacity, block=32, lengths=[100], mixed=False)
    query = _rows(gen, 1, group, tokens, dtype=dtype)
    last = tokens - 2  # queries from here on see position 98
    clean, clean_lse = quantized_attention(query.to(device), cache, softmax_scale=SCALE)
    for codes in (cache.key_codes, cache.value_codes):
        codes.view(torch.uint8)[0, 0, 98:, :] = 0x7F  # positions 98, 99 and what lies past the length
    got, got_lse = quantized_attention(query.to(device), cache, softmax_scale=SCALE)
    torch.cuda.synchronize()
    assert torch.equal(got[:, :last], clean[:, :last]) and torch.equal(got_lse[..., :last], clean_lse[..., :last])
    assert bool(got[:, last:].isnan().all()) and bool(got_lse[..., last:].isnan().all())
    cache = _fill(device, gen, batch=1, heads=1, capacity=capacity, block=32, lengths=[100], mixed=False)
    clean, _ = quantized_attention(query.to(device), cache, softmax_scale=SCALE)
    cache.value_codes.view(torch.uint8)[0, 0, 98, 5] = 0xFF
    cache.value_codes.view(torch.uint8)[0, 0, 7, 77] = 0x7F
    cache.value_codes.view(torch.uint8)[0, 0, 70, 126] = 0x7F
    got, _ = quantized_attention(query.to(device), cache, softmax_scale=SCALE)
    one, _ = quantized_attention(query[:, :, tokens - 1:].to(device), cache, softmax_scale=SCALE)
    torch.cuda.synchronize()
    nan = torch.zeros_like(got, dtype=torch.bool)
    at = torch.arange(100 - tokens, 100, device=device)  # positions of the queries
    for position, dim in ((98, 5), (7, 77), (70, 126)):
        nan[0, at >= position, :, dim] = True
    assert torch.equal(got.isnan(), nan) and torch.equal(got[~nan], clean[~nan])
    assert torch.equal(one.isnan(), nan[:, tokens - 1:])


def test_attend_extreme_scores(device):
    """Scores of hundreds: one row takes all; a rising order moves the running maximum again and again."""
    gen = torch.Generator().manual_seed(11)
    for order in (1, -1):
        cache = QuantizedKVCache.allocate(kv_heads=1, capacity=512, block=16, track_weights=True, device=device)
        ramp = (order * torch.linspace(-40, 40, 500)).reshape(1, 1, 500, 1)
        key = torch.ones(1, 1, 500, D) * ramp
        quantized_append(cache, key.to(device), _rows(gen, 1, 1, 500).to(device))
        query = torch.ones(1, 4, 1, D) * torch.tensor([1.0, -1.0, 0.01, 0.0]).reshape(1, 4, 1, 1)
        _attend_case(device, gen, cache, group=4, tokens=1, dtype=torch.float32, accumulate=True, query=query)


def test_attend_query_strides(device):
    """Queries as views of [batch, token, head] memory and of a fused projection give the contiguous result."""
    gen = torch.Generator().manual_seed(13)
    cache = _fill(device, gen, batch=2, heads=2, capacity=128, block=64, lengths=[100, 77])
    fused = _rows(gen, 2, 3, 12, dtype=torch.bfloat16).to(device)  # [B, T, heads]
    view = fused[:, :, 2:10].transpose(1, 2)
    a = quantized_attention(view, cache, softmax_scale=SCALE)
    b = quantized_attention(view.contiguous(), cache, softmax_scale=SCALE)
    odd = torch.empty(view.numel() + 1, dtype=torch.bfloat16, device=device)[1:].view(view.shape)
    odd.copy_(view)
    c = quantized_attention(odd, cache, softmax_scale=SCALE)
    torch.cuda.synchronize()
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)
    none = quantized_attention(view[:, :, :0], cache, softmax_scale=SCALE)
    assert none[0].shape == (2, 0, 8, D) and none[1].shape == (2, 8, 0)


def test_attend_long_cache_split(device):
    """A long cache over all its parts: the planted rows' values come out, at places beyond 2^31 bytes too."""
    gen = torch.Generator().manual_seed(14)
    batch, heads, capacity = 2, 4, 2_400_000  # 2.46 GB of codes each
    print("attend 2 x 4 heads x 2.4 M rows", flush=True)
    cache = QuantizedKVCache.allocate(batch=batch, kv_heads=heads, capacity=capacity, block=64, device=device)
    n = capacity - 5
    cache.key_scales.fill_(1.0)
    cache.value_scales.fill_(2.0)
    cache.cursors.copy_(_i32([[n, n], [n, n], [0, 0]], device))
    where = torch.randint(0, n, (batch, heads), generator=gen)
    where[1, 3] = n - 1
    query = torch.zeros(batch, heads, 1, D)
    for b in range(batch):
        for h in range(heads):
            code = torch.randint(0, 2, (D,), generator=gen).float() * 2 - 1
            cache.key_codes.view(torch.uint8)[b, h, where[b, h]] = (code * 8).to(torch.float8_e4m3fn).view(torch.uint8).to(device)
            cache.value_codes.view(torch.uint8)[b, h, where[b, h]] = (code * 3).to(torch.float8_e4m3fn).view(torch.uint8).to(device)
            query[b, h, 0] = code
    out, lse = quantized_attention(query.to(device), cache, softmax_scale=SCALE)
    torch.cuda.synchronize()
    # scores: 1024 / sqrt(128) = 90.51 for the planted row, 0 for the others, whose share is below 2.4e6 e^-90
    assert torch.equal(out[:, 0].cpu(), query[:, :, 0] * 6)
    assert (lse.cpu() - 1024 * SCALE).abs().max() <= 90.51 * 8 * 2.0 ** -24


# ------------------------------------------------------------------------------------------ eviction

@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("keep,num_sink,recent", [(100, 4, 20), (1, 0, 0), (128, 0, 128), (64, 64, 0), (200, 0, 0),
                                                  (383, 10, 30), (384, 1, 1)])
def test_evict_matches_oracle(device, block, into, keep, num_sink, recent):
    print(f"evict block={block} into={into} keep={keep} sink={num_sink} recent={recent}", flush=True)
    gen = torch.Generator().manual_seed(keep + block)
    lengths = [384, 50, 201, 100, 0]
    cache = _fill(device, gen, batch=5, heads=2, capacity=384, block=block, lengths=lengths)
    target = _fill(device, gen, batch=5, heads=2, capacity=384, block=block, lengths=[3, 0, 9, 1, 2]) if into else None
    oracle, to = oq.Cache.of(cache), oq.Cache.of(target) if into else None
    evict(cache, keep=keep, num_sink=num_sink, recent=recent, into=target)
    torch.cuda.synchronize()
    oracle.evict(keep=keep, num_sink=num_sink, recent=recent, into=to)
    _same(cache, oracle, "cache")
    if into:
        _same(target, to, "into")


def test_evict_orders_special_weights(device):
    """NaN above infinity above numbers above negatives; zeros of either sign alike; ties to the lower row."""
    gen = torch.Generator().manual_seed(20)
    cache = _fill(device, gen, batch=1, heads=1, capacity=64, block=16, lengths=[64])
    special = torch.tensor([0.0, -0.0, 1.0, float("inf"), -float("inf"), float("nan"), -3.0, 1e-45, -1e-45, 1.0])
    for keep in (1, 7, 8, 20, 30, 45, 63):
        cache.cursors.copy_(_i32([[64], [64], [0]], device))
        cache.weights.copy_(special[torch.randint(0, 10, (64,), generator=gen)].reshape(1, 1, 64))
        oracle = oq.Cache.of(cache)
        evict(cache, keep=keep)
        torch.cuda.synchronize()
        oracle.evict(keep=keep)
        _same(cache, oracle, f"keep {keep}")


@pytest.mark.parametrize("keep,num_sink,recent", [(5000, 10, 64), (1, 0, 0), (4096, 0, 4096), (12_287, 3, 5),
                                                  (8193, 100, 0)])
@pytest.mark.parametrize("capacity", [12_288, 20_480])  # one workgroup, several
def test_evict_long_with_ties(device, keep, num_sink, recent, capacity):
    """Long sequences: special weights, many ties, lengths at and around the chunks."""
    gen = torch.Generator().manual_seed(keep)
    lengths = [12_288, 4096, 9001, 4097]
    cache = _fill(device, gen, batch=4, heads=2, capacity=capacity, block=64, lengths=lengths)
    special = torch.tensor([0.0, -0.0, 1.0, 1.0, float("inf"), -float("inf"), float("nan"), -3.0, 1e-45, 7.25])
    pick = torch.randint(0, 10, cache.weights.shape, generator=gen)
    cache.weights.copy_(torch.where(torch.rand(cache.weights.shape, generator=gen) < 0.7, special[pick],
                                    torch.rand(cache.weights.shape, generator=gen) ** 8))
    oracle = oq.Cache.of(cache)
    evict(cache, keep=keep, num_sink=num_sink, recent=recent)
    torch.cuda.synchronize()
    oracle.evict(keep=keep, num_sink=num_sink, recent=recent)
    _same(cache, oracle)


@pytest.mark.parametrize("capacity,block", [(2048, 32), (2064, 16), (8192, 64), (8208, 16), (16_384, 128), (16_400, 16),
                                            (20_480, 64)])
@pytest.mark.parametrize("share", [0.0, 0.5, 1.0])
def test_evict_at_each_capacity(device, capacity, block, share):
    """Both sides of every capacity where the selection's form changes, full and nearly full sequences."""
    print(f"evict capacity={capacity} block={block} share={share}", flush=True)
    gen = torch.Generator().manual_seed(capacity)
    keep = max(1, min(capacity - 1, int(capacity * share)))
    cache = _fill(device, gen, batch=3, heads=1, capacity=capacity, block=block, lengths=[capacity, capacity - 1, 1500])
    weights = torch.rand(cache.weights.shape, generator=gen)
    cache.weights.copy_(torch.where(weights < 0.4, 0.25, weights))
    oracle = oq.Cache.of(cache)
    evict(cache, keep=keep, num_sink=min(2, keep // 2), recent=min(9, keep // 2))
    torch.cuda.synchronize()
    oracle.evict(keep=keep, num_sink=min(2, keep // 2), recent=min(9, keep // 2))
    _same(cache, oracle)


def test_evict_moves_between_scales(device):
    """Rows of very different size meet in one block; NaN codes move as they are."""
    gen = torch.Generator().manual_seed(21)
    cache = QuantizedKVCache.allocate(kv_heads=2, capacity=256, block=32, track_weights=True, device=device)
    size = torch.exp2(torch.randint(-12, 12, (1, 2, 250, 1), generator=gen).float())
    key = _rows(gen, 1, 2, 250) * size
    key[0, 0, 200, 3] = float("nan")
    quantized_append(cache, key.to(device), (key * 3).to(device))
    cache.weights.copy_(torch.rand(1, 2, 256, generator=gen))
    cache.weights[0, 0, 200] = 9
    for keep in (130, 70, 33):
        oracle = oq.Cache.of(cache)
        evict(cache, keep=keep, num_sink=2, recent=5)
        torch.cuda.synchronize()
        oracle.evict(keep=keep, num_sink=2, recent=5)
        _same(cache, oracle, f"keep {keep}")


@pytest.mark.parametrize("n,keep", [(70_001, 4096), (131_072, 100_000), (3000, 2999)])
def test_evict_long(device, n, keep):
    """Long sequences: the kept set against a stable sort, every kept row's content where its position says."""
    gen = torch.Generator(device=device).manual_seed(n)
    cache = QuantizedKVCache.allocate(kv_heads=2, capacity=n, block=64, track_weights=True, device=device)
    n_rows = torch.arange(n, device=device, dtype=torch.int32)
    cache.positions[..., :n] = n_rows
    cache.cursors.copy_(_i32([[n], [n], [0]], device))
    cache.weights.copy_((torch.rand(cache.weights.shape, generator=gen, device=device) ** 4 * 1000).round())
    cache.key_scales.fill_(0.5)
    cache.value_scales.fill_(4.0)
    tag = cache.key_codes.view(torch.uint8)
    tag[..., :n, 0], tag[..., :n, 1], tag[..., :n, 2] = n_rows % 97, n_rows // 97 % 97, n_rows // 9409 % 97
    cache.value_codes.view(torch.uint8).copy_(tag)
    weights = cache.weights.clone()
    evict(cache, keep=keep, num_sink=3, recent=50)
    torch.cuda.synchronize()
    assert cache.lengths.tolist() == [keep]
    for h in range(2):
        rank = weights[0, h, :n].clone()
        rank[:3] = float("inf")
        rank[n - 50:] = float("inf")
        kept = torch.sort(rank, descending=True, stable=True).indices[:keep].sort().values
        got = cache.positions[0, h, :keep].long()
        assert torch.equal(got.sort().values, kept)
        stay = got == torch.arange(keep, device=device)
        moved = got[~stay]
        assert bool((moved >= keep).all()) and bool((moved.diff() > 0).all())
        assert torch.equal(cache.weights[0, h, :keep], weights[0, h][got])
        for codes in (cache.key_codes, cache.value_codes):
            c = codes.view(torch.uint8)[0, h, :keep].int()
            assert torch.equal(c[:, 0], (got % 97).int()) and torch.equal(c[:, 1], (got // 97 % 97).int())
            assert torch.equal(c[:, 2], (got // 9409 % 97).int())


# ------------------------------------------------------------------------------------------ together

def _request(device, gen, prompt, dtype=torch.bfloat16):
    key, value, query = (_rows(gen, 2, heads, prompt + 40, dtype=dtype).to(device) for heads in (2, 2, 8))
    return key, value, query


@pytest.mark.parametrize("graph", [False, True])
def test_bounded_request(device, graph):
    """A request within a fixed number of rows: the prompt appended in pieces and attended with its weights summed,
    cut to its budget, then decode steps with an eviction every eighth, against the oracle after every step.  With
    `graph` append and attention of a step are one replayed HIP graph, and the eviction another."""
    gen = torch.Generator().manual_seed(30)
    prompt, budget, sinks, recent = 150, 96, 4, 24
    key, value, query = _request(device, gen, prompt)
    cache = QuantizedKVCache.allocate(batch=2, kv_heads=2, capacity=192, block=32, track_weights=True, device=device)
    oracle = oq.Cache.of(cache)

    def host(t):
        return t.double().cpu().numpy()

    def check(out, lse, q, k, v, counts=None):
        oracle.append(host(k), host(v), counts)
        want, tol = oracle.attend(host(q), scale=SCALE, counts=counts)
        torch.cuda.synchronize()
        assert (np.abs(host(out) - want[0]) <= tol[0]).all()
        live = ~np.isneginf(want[1])
        assert (np.abs(host(lse) - want[1])[live] <= tol[1][live]).all()
        got = oq.Cache.of(cache)
        assert (np.abs(got.weights - (oracle.weights + want[2]))[:, :, :got.cursors[0].max()] <=
                (tol[2] + 4 * oq.U * (oracle.weights + want[2]))[:, :, :got.cursors[0].max()]).all()
        oracle.weights = got.weights  # eviction goes by the kernel's own sums
        _same(cache, oracle)

    at = 0
    for piece, counts in ((100, [100, 61]), (50, [50, 50])):
        rows = slice(at, at + piece)
        k, v, q = key[:, :, rows], value[:, :, rows], query[:, :, rows]
        quantized_append(cache, k, v, counts=_i32(counts, device))
        out, lse = quantized_attention(q, cache, softmax_scale=SCALE, counts=_i32(counts, device), accumulate=True)
        check(out, lse, q, k, v, counts)
        at += piece

    def trim():
        evict(cache, keep=budget, num_sink=sinks, recent=recent)

    def trim_check():
        oracle.evict(keep=budget, num_sink=sinks, recent=recent)
        torch.cuda.synchronize()
        _same(cache, oracle)

    trim()
    trim_check()
    static = [torch.empty_like(t[:, :, :1]) for t in (key, value, query)]
    result = {}

    def step():
        quantized_append(cache, static[0], static[1])
        result["out"], result["lse"] = quantized_attention(static[2], cache, softmax_scale=SCALE, accumulate=True)

    steps = trims = None
    if graph:
        saved = [t.clone() for t in (cache.key_codes.view(torch.uint8), cache.value_codes.view(torch.uint8),
                                     cache.key_scales, cache.value_scales, cache.positions, cache.weights,
                                     cache.cursors)]
        steps, trims = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(steps):
            step()
        with torch.cuda.graph(trims):
            trim()
        for t, s in zip((cache.key_codes.view(torch.uint8), cache.value_codes.view(torch.uint8), cache.key_scales,
                         cache.value_scales, cache.positions, cache.weights, cache.cursors), saved):
            assert torch.equal(t, s)  # a capture runs nothing
    for i in range(20):
        for t, source in zip(static, (key, value, query)):
            t.copy_(source[:, :, prompt + i:prompt + i + 1])
        steps.replay() if graph else step()
        check(result["out"], result["lse"], static[2], static[0], static[1])
        if i % 8 == 7:
            trims.replay() if graph else trim()
            trim_check()
    cache.assert_no_overflow()


def test_draft_tokens_taken_back(device):
    """Rejected draft tokens are rewound and the next ones written over them."""
    gen = torch.Generator().manual_seed(31)
    cache = _fill(device, gen, batch=2, heads=2, capacity=128, block=64, lengths=[50, 62], mixed=False)
    oracle = oq.Cache.of(cache)
    _append(cache, oracle, _rows(gen, 2, 2, 5), _rows(gen, 2, 2, 5))
    back = np.array([3, 5], dtype=np.int32)
    cache.rewind(torch.from_numpy(back).to(device))
    oracle.cursors[:2] -= back
    _append(cache, oracle, _rows(gen, 2, 2, 4), _rows(gen, 2, 2, 4))
    torch.cuda.synchronize()
    _same(cache, oracle)
    _attend_case(device, gen, cache, group=2, tokens=4, dtype=torch.bfloat16)


def test_calls_on_a_side_stream(device):
    """Calls follow the current stream: a chain on a side stream, waited for by an event, equals the default one's."""
    gen = torch.Generator().manual_seed(32)
    key, value, query = _request(device, gen, 60)
    caches = [QuantizedKVCache.allocate(batch=2, kv_heads=2, capacity=128, block=32, track_weights=True, device=device)
              for _ in range(2)]
    side = torch.cuda.Stream(device)
    results = []
    for cache, stream in zip(caches, (torch.cuda.current_stream(device), side)):
        stream.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(stream):
            quantized_append(cache, key, value)
            quantized_attention(query, cache, softmax_scale=SCALE, accumulate=True)
            evict(cache, keep=64, num_sink=2, recent=8)
            results.append(quantized_attention(query[:, :, :1], cache, softmax_scale=SCALE))
    torch.cuda.synchronize()
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    _same(caches[0], oq.Cache.of(caches[1]))


def test_same_call_twice_is_bit_equal(device):
    """No atomics on results: the same calls on equal caches give equal bits."""
    gen = torch.Generator().manual_seed(33)
    key, value, query = _request(device, gen, 400)
    seen = []
    for _ in range(2):
        cache = QuantizedKVCache.allocate(batch=2, kv_heads=2, capacity=512, block=64, track_weights=True, device=device)
        quantized_append(cache, key, value)
        out, lse = quantized_attention(query, cache, softmax_scale=SCALE, accumulate=True)
        evict(cache, keep=200, num_sink=1, recent=1)
        one, _ = quantized_attention(query[:, :, -1:], cache, softmax_scale=SCALE, accumulate=True)
        seen.append((out, lse, one, cache.weights.clone(), cache.positions.clone(), cache.key_codes.view(torch.uint8).clone()))
    torch.cuda.synchronize()
    for a, b in zip(*seen):
        assert torch.equal(a, b)


@pytest.mark.parametrize("tokens,window,capacity,dtype", [(1, 200, 4096, torch.bfloat16), (9, 0, 20_480, torch.float16),
                                                          (40, 300, 12_288, torch.float32),
                                                          (130, 0, 2048, torch.bfloat16)])
def test_replays_equal_eager_calls(device, tokens, window, capacity, dtype):
    """Every form of the kernels captured: an append, attention with received weights and an eviction, replayed with
    eager work of other caches between, against the same calls made eagerly; two graphs of one cache in turn."""
    print(f"replay tokens={tokens} window={window} capacity={capacity}", flush=True)
    gen = torch.Generator().manual_seed(capacity)
    full = capacity - tokens - 3
    caches = [_fill(device, torch.Generator().manual_seed(capacity), batch=2, heads=2, capacity=capacity, block=64,
                    lengths=[full, full - 500]) for _ in range(2)]
    key, value, query = (_rows(gen, 2, heads, tokens, dtype=dtype).to(device) for heads in (2, 2, 8))
    other = _fill(device, gen, batch=1, heads=2, capacity=320, block=32, lengths=[300])

    def step(cache):
        quantized_append(cache, key, value)
        out, lse = quantized_attention(query, cache, softmax_scale=SCALE, window=window, accumulate=True)
        evict(cache, keep=full - 700, num_sink=2, recent=tokens + 5)
        return out, lse

    def drawn():
        for x in (key, value, query):
            x.copy_(_rows(gen, *x.shape[:3], dtype=dtype))

    warm = torch.cuda.Stream(device)
    warm.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(warm):
        step(caches[0])
    torch.cuda.current_stream(device).wait_stream(warm)
    step(caches[1])
    graphs, results = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            results.append(step(caches[0]))
    for i in range(6):
        drawn()
        graphs[i % 2].replay()
        quantized_attention(query[:1, :, :1], other, softmax_scale=SCALE, accumulate=True)
        want = step(caches[1])
        torch.cuda.synchronize()
        for got, eager in zip(results[i % 2], want):
            assert torch.equal(got, eager), i
        _same(caches[0], oq.Cache.of(caches[1]), f"replay {i}")


@pytest.mark.parametrize("group,tokens,dtype", [(4, 40, torch.bfloat16), (2, 50, torch.float16), (4, 30, torch.float32),
                                                (2, 3, torch.bfloat16), (8, 15, torch.bfloat16)])
@pytest.mark.parametrize("window", [0, 17])
@pytest.mark.parametrize("capacity", [320, 65_536])  # few-row kernels, many-row ones
@pytest.mark.parametrize("mixed", [False, True])
def test_nan_reaches_the_weights_of_the_rows_seen_alone(device, group, tokens, dtype, window, capacity, mixed):
    """A NaN query, or a NaN key among the rows that a query sees, makes the received weights of the rows which that
    query sees NaN, and no others: those are as they are without it, to the bit."""
    print(f"nan weights group={group} tokens={tokens} dtype={dtype} window={window} capacity={capacity}", flush=True)
    gen = torch.Generator().manual_seed(51)
    n = 300
    cache = _fill(device, gen, batch=1, heads=2, capacity=capacity, block=32, lengths=[n], mixed=mixed)
    query = _rows(gen, 1, 2 * group, tokens, dtype=dtype)
    weights, at = cache.weights.clone(), torch.arange(n - tokens, n, device=device)
    position = cache.positions[0, :, :n]

    def received(q):
        cache.weights.copy_(weights)
        quantized_attention(q.to(device), cache, softmax_scale=SCALE, window=window, accumulate=True)
        torch.cuda.synchronize()
        return cache.weights[0, :, :n].clone()

    def seen_by(t):  # rows that query t sees, by head
        return (position <= at[t]) & ((position > at[t] - window) if window else True)

    clean = received(query)
    assert not clean.isnan().any()
    bad = tokens // 2
    for value in (float("nan"), float("inf")):
        broken = query.clone()
        broken[0, group - 1, bad] = value  # a query head of KV head 0
        got = received(broken)
        want = seen_by(bad)
        want[1] = False
        assert torch.equal(got.isnan(), want) and torch.equal(got[~want], clean[~want]), value
    # a NaN key: every query that sees it gives NaN to all that it sees
    row = int((position[1] == n - tokens // 2 - 1).nonzero()[0])
    cache.key_codes.view(torch.uint8)[0, 1, row, 3] = 0x7F
    got = received(query)
    want = torch.zeros_like(position, dtype=torch.bool)
    for t in range(tokens):
        if bool(seen_by(t)[1, row]):
            want[1] |= seen_by(t)[1]
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1].isnan(), want[1])
    assert torch.equal(got[1][~want[1]], clean[1][~want[1]])


@pytest.mark.parametrize("group,tokens", [(4, 1), (2, 3), (8, 15), (4, 40)])
@pytest.mark.parametrize("window", [0, 90])
@pytest.mark.parametrize("capacity", [320, 65_536])
@pytest.mark.parametrize("lengths", [[300], [300, 300]])
def test_an_infinite_query_makes_all_that_it_sees_nan(device, group, tokens, window, capacity, lengths):
    """One infinite element: scores are infinities of both signs, the softmax is NaN, and every row that the query sees
    gets NaN, those of minus infinity too."""
    print(f"infinite query group={group} tokens={tokens} window={window} capacity={capacity}", flush=True)
    gen = torch.Generator().manual_seed(52)
    n, batch = 300, len(lengths)
    cache = _fill(device, gen, batch=batch, heads=1, capacity=capacity, block=32, lengths=lengths)
    query = _rows(gen, batch, group, tokens, dtype=torch.bfloat16)
    weights, at = cache.weights.clone(), n - tokens + tokens // 2
    quantized_attention(query.to(device), cache, softmax_scale=SCALE, window=window, accumulate=True)
    clean = cache.weights.clone()
    cache.weights.copy_(weights)
    query[0, group - 1, tokens // 2, 7] = -float("inf")
    out, lse = quantized_attention(query.to(device), cache, softmax_scale=SCALE, window=window, accumulate=True)
    torch.cuda.synchronize()
    position = cache.positions[0, 0, :n]
    want = torch.zeros_like(cache.weights, dtype=torch.bool)
    want[0, 0, :n] = (position <= at) & ((position > at - window) if window else True)
    assert torch.equal(cache.weights.isnan(), want) and torch.equal(cache.weights[~want], clean[~want])
    nan = torch.zeros_like(lse, dtype=torch.bool)
    nan[0, group - 1, tokens // 2] = True
    assert torch.equal(lse.isnan(), nan) and torch.equal(out.isnan(), nan.transpose(1, 2)[..., None].expand(out.shape))


@pytest.mark.parametrize("keep,num_sink,recent", [(1000, 10, 500), (200, 4, 126), (2**40, 2**39, 2**39)])
@pytest.mark.parametrize("into", [False, True])
def test_evict_to_more_rows_than_there_are(device, keep, num_sink, recent, into):
    """In place nothing happens; another cache gets a copy."""
    gen = torch.Generator().manual_seed(53)
    cache = _fill(device, gen, batch=2, heads=2, capacity=128, block=32, lengths=[128, 70])
    target = _fill(device, gen, batch=2, heads=2, capacity=160, block=32, lengths=[3, 0]) if into else None
    oracle, to = oq.Cache.of(cache), oq.Cache.of(target) if into else None
    evict(cache, keep=keep, num_sink=num_sink, recent=recent, into=target)
    torch.cuda.synchronize()
    _same(cache, oracle, "cache")
    if into:
        oracle.evict(keep=keep, into=to)
        _same(target, to, "into")


@pytest.mark.parametrize("tracked", [False, True])
def test_evict_into_the_other_half_of_one_storage(device, tracked):
    """Two caches that lie behind one another in the same tensors share no memory; a target that keeps no weights gets
    none."""
    gen = torch.Generator().manual_seed(54)
    both = _fill(device, gen, batch=2, heads=2, capacity=128, block=32, lengths=[128, 128])
    cursors = [_i32([[n], [n], [0]], device) for n in (128, 0)]
    halves = [QuantizedKVCache.from_tensors(
        key_codes=both.key_codes[b:b + 1], value_codes=both.value_codes[b:b + 1], key_scales=both.key_scales[b:b + 1],
        value_scales=both.value_scales[b:b + 1], positions=both.positions[b:b + 1], cursors=cursors[b], block=32,
        weights=both.weights[b:b + 1] if b == 0 or tracked else None) for b in range(2)]
    left = both.weights[1].clone()
    oracle, to = oq.Cache.of(halves[0]), oq.Cache.of(halves[1])
    evict(halves[0], keep=50, num_sink=2, recent=9, into=halves[1])
    torch.cuda.synchronize()
    oracle.evict(keep=50, num_sink=2, recent=9, into=to)
    if not tracked:
        to.weights[:] = 0
        assert torch.equal(both.weights[1], left)
    _same(halves[0], oracle, "cache")
    _same(halves[1], to, "into")
