"""Performance cases of the 8-bit key/value cache: writing into it, attention over it, eviction from it.

A layer's cache holds E4M3 codes ``[batch, kv_heads, capacity, 128]`` with one scale for each block of tokens and head,
the position of every row, and the attention weight that every row has received.  A serving program appends each
step's keys and values, attends to the cache with the step's queries and, where the cache is bounded, evicts rows:

* ``append`` - ``quantized_append``: new tokens quantised into the cache, block scales kept
* ``attend`` - ``quantized_attention``: attention of the newest tokens over the whole cache, with the rows' received
  weight summed where the program evicts
* ``evict``  - ``evict``: the cache reduced to its most attended rows, written into another cache (so that every pass
  finds the same source)

Everything is made from the seed with plain torch operations on the GPU.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
D = 128
SCALE = D ** -0.5
CODE = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # A server's step over eight requests: one token each, into caches of odd lengths.
        dict(name="append_step_b8", kind="append", batch=8, kv_heads=8, tokens=1, ctx_min=1001, ctx_max=8191, mix=1,
             block=64, dtype="bf16", ragged=False, layout="heads"),
        # A long prompt written in one call into an empty cache, keys as the projection leaves them ([token, head]).
        dict(name="append_prompt_32k", kind="append", batch=1, kv_heads=8, tokens=32768, ctx_min=0, ctx_max=0, mix=2,
             block=64, dtype="bf16", ragged=False, layout="tokens"),
        # Prompt pieces of uneven lengths appended to started sequences, 32-bit inputs, small blocks.
        dict(name="append_ragged_f32", kind="append", batch=5, kv_heads=2, tokens=777, ctx_min=0, ctx_max=1900, mix=3,
             block=32, dtype="f32", ragged=True, layout="tokens"),
        # A short chat turn of a small model: latency is all there is.
        dict(name="attend_chat_300", kind="attend", batch=1, q_heads=8, kv_heads=2, tokens=1, ctx_min=300, ctx_max=300,
             mix=4, block=64, dtype="bf16", ragged=False, window=0, accumulate=False),
        # A server's decode step over eight requests of uneven lengths (16k to 128k).
        dict(name="attend_step_b8_131k", kind="attend", batch=8, q_heads=32, kv_heads=8, tokens=1, ctx_min=16384,
             ctx_max=131072, mix=5, block=64, dtype="bf16", ragged=False, window=0, accumulate=False),
        # One long document, fp16 model, wide blocks.
        dict(name="attend_131k_f16", kind="attend", batch=1, q_heads=32, kv_heads=8, tokens=1, ctx_min=131071,
             ctx_max=131071, mix=6, block=128, dtype="f16", ragged=False, window=0, accumulate=False),
        # Draft tokens of speculative decoding checked in one call, 32-bit, group of seven, a sliding window.
        dict(name="attend_draft_f32", kind="attend", batch=4, q_heads=28, kv_heads=4, tokens=6, ctx_min=900,
             ctx_max=5003, mix=7, block=32, dtype="f32", ragged=True, window=2048, accumulate=False),
        # A piece of a long prompt (chunked prefill) over what is cached so far.
        dict(name="attend_chunk_2k_of_32k", kind="attend", batch=1, q_heads=32, kv_heads=8, tokens=2048, ctx_min=32768,
             ctx_max=32768, mix=8, block=64, dtype="bf16", ragged=False, window=0, accumulate=False),
        # A whole prompt at once, every row's received weight summed: what eviction after the prompt goes by.
        dict(name="attend_prompt_4k_weights", kind="attend", batch=1, q_heads=32, kv_heads=8, tokens=4095, ctx_min=4095,
             ctx_max=4095, mix=9, block=64, dtype="bf16", ragged=False, window=0, accumulate=True),
        # A decode step of a bounded cache: attention and the weights' sums.
        dict(name="attend_step_b8_weights", kind="attend", batch=8, q_heads=32, kv_heads=8, tokens=1, ctx_min=8192,
             ctx_max=16384, mix=10, block=64, dtype="bf16", ragged=False, window=0, accumulate=True),
        # A small bounded cache that ran full.
        dict(name="evict_1500_to_1024", kind="evict", batch=2, kv_heads=2, ctx_min=1200, ctx_max=1500, mix=11, keep=1024,
             num_sink=10, recent=128, block=64),
        # Two long prompts compressed to a decode budget.
        dict(name="evict_131k_to_16k", kind="evict", batch=2, kv_heads=8, ctx_min=120001, ctx_max=131072, mix=12,
             keep=16384, num_sink=10, recent=1024, block=64),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "evict"])
    block = rng.choice([16, 32, 64, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    mix = rng.randrange(1 << 20)
    if kind == "append":
        batch, kv_heads = rng.choice([(1, 8), (1, 1), (3, 4), (8, 8), (16, 2)])
        tokens = _log_int(rng, 1, 32768 * 8 // (batch * kv_heads) // (2 if dtype == "f32" else 1))
        low = rng.choice([0, _log_int(rng, 1, 4000)])
        return dict(kind=kind, batch=batch, kv_heads=kv_heads, tokens=tokens, ctx_min=low,
                    ctx_max=low + rng.randint(0, 3000), mix=mix, block=block, dtype=dtype, ragged=rng.random() < 0.5,
                    layout=rng.choice(["heads", "tokens"]))
    if kind == "evict":
        batch, kv_heads = rng.choice([(1, 8), (2, 4), (4, 2), (8, 1), (2, 8)])
        high = _log_int(rng, 200, 131072)
        keep = rng.randint(64, max(64, min(16384, high // 2)))
        recent = rng.randint(0, keep // 2)
        return dict(kind=kind, batch=batch, kv_heads=kv_heads, ctx_min=max(1, high // 2), ctx_max=high, mix=mix,
                    keep=keep, num_sink=min(rng.choice([0, 4, 10]), keep - recent), recent=recent, block=block)
    q_heads, kv_heads = rng.choice([(8, 2), (32, 8), (32, 8), (28, 4), (16, 1), (8, 8), (64, 8)])
    batch = rng.choice([1, 1, 2, 5, 8])
    tokens = rng.choice([1, 1, 1, rng.randint(2, 9), _log_int(rng, 10, 2048 // batch)])
    most = 800000 // batch if tokens == 1 else 32768 if tokens < 10 else 32768 * 2048 * 32 // (4 * q_heads * batch * tokens)
    high = max(tokens, _log_int(rng, 100, min(131072, max(200, most))))
    return dict(kind=kind, batch=batch, q_heads=q_heads, kv_heads=kv_heads, tokens=tokens,
                ctx_min=max(tokens, high // rng.choice([1, 2, 8])), ctx_max=high, mix=mix, block=block, dtype=dtype,
                ragged=rng.random() < 0.3, window=rng.choice([0, 0, 0, rng.randint(1, 4096)]),
                accumulate=rng.random() < 0.4)


# ------------------------------------------------------------------------------------------ inputs

def _lengths(case):
    """Rows in use of each sequence before an append, with the new tokens for attention and eviction."""
    rng = random.Random(case["mix"])
    sizes = [rng.randint(case["ctx_min"], case["ctx_max"]) for _ in range(case["batch"])]
    sizes[0] = case["ctx_max"]
    return sizes


def _counts(case):
    """New tokens of each sequence, or None where every sequence has all of them."""
    if not case.get("ragged"):
        return None
    rng = random.Random(case["mix"] + 1)
    return [case["tokens"]] + [rng.randint(0, case["tokens"]) for _ in range(case["batch"] - 1)]


def _capacity(case):
    rows = max(_lengths(case)) + (case["tokens"] if case["kind"] == "append" else 0)
    return -(-max(rows, 1) // case["block"]) * case["block"]


def _exponent(amax):
    """Exponent of the smallest power of two s with amax <= 448 s (448 = 0.875 * 2^9), at least -64."""
    mantissa, exponent = torch.frexp(amax)
    return torch.where(amax > 0, exponent - torch.where(mantissa <= 0.875, 9, 8), -64).clamp_min(-64)


def _scale(amax):
    return torch.exp2(_exponent(amax).float())


def _rows(gen, batch, heads, tokens, drift):
    """Keys or values as models have them: a few strong channels, and tokens of uneven size."""
    channels = 1 + 6 * torch.rand(1, heads, 1, D, generator=gen, device=DEVICE) ** 8
    size = torch.exp(0.3 * torch.randn(batch, heads, tokens, 1, generator=gen, device=DEVICE))
    return (torch.randn(batch, heads, tokens, D, generator=gen, device=DEVICE) * size + drift) * channels


def _quantised(x, block):
    b, h, rows, _ = x.shape
    scale = _scale(x.abs().reshape(b, h, rows // block, block * D).amax(-1))
    return (x / scale.repeat_interleave(block, 2)[..., None]).to(CODE), scale


def _cache_tensors(case, gen, lengths, new, weights):
    """A cache as earlier calls left it: older rows in any order (an eviction moves rows), the newest ones last."""
    b, h, block, cap = case["batch"], case["kv_heads"], case["block"], _capacity(case)
    key_codes, key_scales = _quantised(_rows(gen, b, h, cap, 0.3), block)
    value_codes, value_scales = _quantised(_rows(gen, b, h, cap, 0.0), block)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
    fresh = torch.tensor(new, dtype=torch.int32, device=DEVICE)
    seen = n + n // 4
    row = torch.arange(cap, device=DEVICE, dtype=torch.int32).expand(b, h, cap)
    old = (n - fresh)[:, None, None]
    # older rows: distinct positions below the newest tokens', about a fifth of the positions gone
    mixed = torch.where(row < old, torch.rand(b, h, cap, generator=gen, device=DEVICE), 2.0).argsort(-1)
    skip = torch.where(mixed < (seen - n)[:, None, None], mixed, mixed + (seen - n)[:, None, None]).int()
    positions = torch.where(row < old, skip, row + (seen - n)[:, None, None]).int().contiguous()
    cursors = torch.stack([n, seen, torch.zeros_like(n)])
    tensors = dict(key_codes=key_codes, value_codes=value_codes, key_scales=key_scales, value_scales=value_scales,
                   positions=positions, cursors=cursors)
    if weights:
        share = torch.rand(b, h, cap, generator=gen, device=DEVICE) ** 6
        tensors["weights"] = (share * 40).half().float()  # rounded, so that equal weights occur
    return tensors


def _handle(tensors, block):
    """The program's cache object over these tensors; the plain form takes the tensors themselves."""
    if not own:
        return tensors
    from community_kv_amd import QuantizedKVCache

    return QuantizedKVCache.from_tensors(block=block, **tensors)


def _given(tensor, layout):
    """[batch, head, token, dim] values in memory order [batch, token, head, dim] where the layout says so."""
    return tensor.transpose(1, 2).contiguous().transpose(1, 2) if layout == "tokens" else tensor


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    lengths = _lengths(case)
    counts = _counts(case)
    tokens = case.get("tokens", 0)
    new = [0] * case["batch"] if case["kind"] != "attend" else [tokens] * case["batch"] if counts is None else counts
    tensors = _cache_tensors(case, gen, lengths, new, case["kind"] == "evict" or bool(case.get("accumulate")))
    state = dict(case=case, tensors=tensors, rows=max(lengths),
                 counts=None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEVICE))
    dtype = TYPES[case.get("dtype", "f32")]
    if case["kind"] == "append":
        state["cursors"] = tensors["cursors"].clone()
        for name, drift in (("key", 0.3), ("value", 0.0)):
            state[name] = _given(_rows(gen, case["batch"], case["kv_heads"], tokens, drift).to(dtype), case["layout"])
    elif case["kind"] == "attend":
        # queries near some of the cached keys, so that a few rows take much of the weight
        b, hq, h = case["batch"], case["q_heads"], case["kv_heads"]
        pick = (torch.rand(b, h, hq // h * tokens, generator=gen, device=DEVICE) * min(lengths)).long()
        near = tensors["key_codes"].view(torch.uint8).gather(2, pick[..., None].expand(-1, -1, -1, D)).view(CODE).float()
        near = near / near.square().mean(-1, keepdim=True).sqrt().clamp_min(1e-6)
        query = torch.randn(b, hq, tokens, D, generator=gen, device=DEVICE) + 0.5 * near.reshape(b, hq, tokens, D)
        state["query"] = query.to(dtype)
    else:
        keep = -(-case["keep"] // case["block"]) * case["block"]
        small = {name: t[:, :, :keep // (case["block"] if name.endswith("scales") else 1)].clone()
                 for name, t in tensors.items() if name != "cursors"}
        state["into_tensors"] = _padded(small, keep, case["block"]) | dict(cursors=tensors["cursors"].clone())
        state["into"] = _handle(state["into_tensors"], case["block"])
    state["cache"] = _handle(tensors, case["block"])
    return state


def _padded(small, keep, block):
    """Tensors of a cache of `keep` rows, where the source has fewer."""
    sizes = {name: keep // block if name.endswith("scales") else keep for name in small}
    return {name: t if t.shape[2] == sizes[name] else
            torch.cat([t, t.new_zeros(*t.shape[:2], sizes[name] - t.shape[2], *t.shape[3:])], 2).contiguous()
            if t.dtype != CODE else
            torch.cat([t.view(torch.uint8), torch.zeros(*t.shape[:2], sizes[name] - t.shape[2], D, dtype=torch.uint8,
                                                        device=DEVICE)], 2).view(CODE)
            for name, t in small.items()}


# ------------------------------------------------------------------------------------------ plain forms

def _plain_write(codes, scales, x, block, row, valid, start):
    """Quantises x [B,H,T,D] into rows `row` [B,T] (where valid), scales growing; `start` [B] rows were there."""
    b, h, tokens, _ = x.shape
    cap = codes.shape[2]
    x = x.float()
    finite = torch.where(torch.isfinite(x), x, 0).abs().amax(-1)
    inside = torch.where(valid, row, 0)
    blk = (inside // block)[:, None].expand(b, h, tokens)
    amax = torch.zeros_like(scales).scatter_reduce(2, blk, torch.where(valid[:, None], finite, 0), "amax")
    hit = torch.zeros_like(scales).scatter_reduce(2, blk, valid[:, None].expand(b, h, tokens).float(), "amax") > 0
    first = torch.arange(cap // block, device=DEVICE) * block
    before = torch.where((first < start[:, None])[:, None], scales, 0)
    grown = torch.where(hit, torch.maximum(before, _scale(amax)), scales)
    # earlier rows of the block that the first new token falls into
    here = (start.clamp_max(cap - 1) // block).long()
    batch = torch.arange(b, device=DEVICE)
    ratio = torch.where(first[here][:, None] < start[:, None], before[batch, :, here] / grown[batch, :, here], 1)
    old_rows = first[here][:, None] + torch.arange(block, device=DEVICE)
    old = codes.view(torch.uint8)[batch[:, None], :, old_rows]
    finer = (old.view(CODE).float() * ratio[:, None, :, None]).to(CODE).view(torch.uint8)
    codes.view(torch.uint8)[batch[:, None], :, old_rows] = torch.where((old_rows < start[:, None])[..., None, None], finer, old)
    code = (x / grown.gather(2, blk)[..., None]).to(CODE).view(torch.uint8)
    at, token = valid.nonzero(as_tuple=True)
    codes.view(torch.uint8)[at, :, row[at, token]] = code[at, :, token]
    scales.copy_(grown)


def _plain_append(state):
    c, block = state["cache"], state["case"]["block"]
    key, value = state["key"], state["value"]
    tokens, cap = key.shape[2], c["key_codes"].shape[2]
    start, seen = c["cursors"][0].long(), c["cursors"][1].long()
    t = torch.arange(tokens, device=DEVICE)
    count = torch.full_like(start, tokens) if state["counts"] is None else state["counts"].long()
    row = start[:, None] + t
    valid = (t < count[:, None]) & (row < cap)
    _plain_write(c["key_codes"], c["key_scales"], key, block, row, valid, start)
    _plain_write(c["value_codes"], c["value_scales"], value, block, row, valid, start)
    at, token = valid.nonzero(as_tuple=True)
    c["positions"][at, :, row[at, token]] = (seen[at] + token)[:, None].int()
    taken = valid.sum(1).int()
    c["cursors"][0] += taken
    c["cursors"][1] += taken
    c["cursors"][2] |= (start + count > cap).int()


def _values(codes, scales, rows, block):
    return codes[:, :, :rows].float() * scales.repeat_interleave(block, 2)[:, :, :rows, None]


def _plain_attend(state):
    c, case, rows = state["cache"], state["case"], state["rows"]
    b, hq, tokens, _ = state["query"].shape
    h = case["kv_heads"]
    length, seen = c["cursors"][0], c["cursors"][1]
    count = torch.full_like(seen, tokens) if state["counts"] is None else state["counts"]
    t = torch.arange(tokens, device=DEVICE)
    at = (seen - count)[:, None] + t                                             # [B, T] positions of the queries
    position = c["positions"][:, :, :rows]
    live = torch.arange(rows, device=DEVICE) < length[:, None]
    mask = (live[:, None, None] & (t < count[:, None])[:, None, :, None] & (position[:, :, None] <= at[:, None, :, None]))
    if case["window"]:
        mask &= position[:, :, None] > (at - case["window"])[:, None, :, None]
    mask = mask[:, :, None]                                                      # [B, H, 1, T, rows]
    key = _values(c["key_codes"], c["key_scales"], rows, case["block"])
    value = _values(c["value_codes"], c["value_scales"], rows, case["block"])
    query = state["query"].float().reshape(b, h, hq // h * tokens, D)
    score = (query @ key.transpose(-1, -2)).reshape(b, h, hq // h, tokens, rows) * SCALE
    score = score.masked_fill_(~mask, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0, top)
    share = (score - top).exp_()
    total = share.sum(-1, keepdim=True)
    lse = torch.where(total > 0, top + total.log(), -math.inf).reshape(b, hq, tokens)
    share = share.div_(torch.where(total > 0, total, 1))
    out = (share.reshape(b, h, hq // h * tokens, rows) @ value).reshape(b, hq, tokens, D)
    out = out.transpose(1, 2).to(state["query"].dtype)
    if not case["accumulate"]:
        return dict(out=out, lse=lse)
    c["weights"][:, :, :rows] += share.sum((2, 3))
    return dict(out=out, lse=lse, weights=c["weights"])


def _plain_evict(state):
    c, to, case = state["cache"], state["into"], state["case"]
    block, keep, cap = case["block"], case["keep"], c["key_codes"].shape[2]
    b, h = case["batch"], case["kv_heads"]
    n, seen = c["cursors"][0][:, None, None], c["cursors"][1][:, None, None]
    row = torch.arange(cap, device=DEVICE)
    held = (c["positions"] < case["num_sink"]) | (c["positions"] >= seen - case["recent"])
    rank = torch.where(row < n, torch.where(held, math.inf, c["weights"]), -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.zeros(b, h, cap, dtype=torch.bool, device=DEVICE).scatter_(2, order, True) & (row < n)
    size = min(keep, cap)
    hole = ~kept[..., :size] & (n > keep)
    mover = kept & (row >= keep)
    movers = torch.argsort((~mover).byte(), dim=-1, stable=True)[..., :size]                 # moving rows first, ascending
    source = torch.where(hole, movers.gather(2, (hole.int().cumsum(-1) - 1).clamp_min(0).long()), row[:size])
    live = (row[:size] < n).expand(b, h, size)
    pad = -size % block
    blocks = (size + pad) // block
    for name in ("key", "value"):  # the two halves of the cache
        scales = c[name + "_scales"]
        code = c[name + "_codes"].view(torch.uint8).gather(2, source[..., None].expand(-1, -1, -1, D)).view(CODE).float()
        value = code * scales.gather(2, source // block)[..., None]
        need = torch.where(hole, torch.where(torch.isfinite(value), value, 0).abs().amax(-1), 0)
        need = torch.nn.functional.pad(need, (0, pad)).reshape(b, h, blocks, block).amax(-1)
        any_hole = torch.nn.functional.pad(hole, (0, pad)).reshape(b, h, blocks, block).any(-1)
        used = torch.nn.functional.pad(live, (0, pad)).reshape(b, h, blocks, block).any(-1)
        grown = torch.where(any_hole, torch.maximum(scales[..., :blocks], _scale(need)), scales[..., :blocks])
        fresh = (value / grown.repeat_interleave(block, 2)[:, :, :size, None]).to(CODE).view(torch.uint8)
        target = to[name + "_codes"].view(torch.uint8)[:, :, :size]
        target.copy_(torch.where(live[..., None], fresh, target))
        to[name + "_scales"][..., :blocks] = torch.where(used, grown, to[name + "_scales"][..., :blocks])
    for name in ("positions", "weights"):
        to[name][..., :size] = torch.where(live, c[name].gather(2, source), to[name][..., :size])
    to["cursors"][0] = c["cursors"][0].clamp_max(keep)
    to["cursors"][1:] = c["cursors"][1:]


# ------------------------------------------------------------------------------------------ one pass

NAMES = ("key_codes", "value_codes", "key_scales", "value_scales", "positions", "cursors")


def run(state):
    case, tensors = state["case"], state["tensors"]
    if case["kind"] == "append":
        tensors["cursors"].copy_(state["cursors"])  # every pass appends behind the same rows
        if own:
            from community_kv_amd import quantized_append

            quantized_append(state["cache"], state["key"], state["value"], counts=state["counts"])
        else:
            _plain_append(state)
        return {name: tensors[name] for name in NAMES}
    if case["kind"] == "attend":
        if case["accumulate"]:
            tensors["weights"].zero_()
        if not own:
            return _plain_attend(state)
        from community_kv_amd import quantized_attention

        out, lse = quantized_attention(state["query"], state["cache"], softmax_scale=SCALE, counts=state["counts"],
                                       window=case["window"], accumulate=case["accumulate"])
        return dict(out=out, lse=lse, weights=tensors["weights"]) if case["accumulate"] else dict(out=out, lse=lse)
    if own:
        from community_kv_amd import evict

        evict(state["cache"], keep=case["keep"], num_sink=case["num_sink"], recent=case["recent"], into=state["into"])
    else:
        _plain_evict(state)
    return {name: state["into_tensors"][name] for name in NAMES + ("weights",)}


# ------------------------------------------------------------------------------------------ what a pass needs

def work(case):
    lengths, h = _lengths(case), case["kv_heads"]
    if case["kind"] == "append":
        new = sum(_counts(case) or [case["tokens"]] * case["batch"])
        wide = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
        return dict(bytes=new * h * (2 * D * (wide + 1) + 8 / case["block"] + 4), flops=new * h * 2 * D * 2)
    if case["kind"] == "evict":
        moved = sum(min(n, case["keep"]) for n in lengths)
        return dict(bytes=sum(lengths) * h * 8 + moved * h * 2 * (2 * D + 8 / case["block"] + 8), flops=sum(lengths) * h)
    counts = _counts(case) or [case["tokens"]] * case["batch"]
    pairs = touched = 0
    for n, count in zip(lengths, counts):
        window = case["window"] or n + n // 4
        old = n - count
        pairs += sum(min(old + t + 1, window) for t in range(count))
        touched += min(n, window + count) if count else 0
    wide = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    byte = touched * h * (2 * D + 8 / case["block"]) + sum(counts) * case["q_heads"] * (2 * D * wide + 4)
    if case["tokens"] > 1 or case["window"]:
        byte += sum(lengths) * h * 4
    if case["accumulate"]:
        byte += touched * h * 8
    return dict(bytes=byte, flops=pairs * case["q_heads"] * (4 * D))


# ------------------------------------------------------------------------------------------ definitions in 64 bits

def _rounded(y):
    """The E4M3 value nearest to y (ties to even): 3 bits behind the leading one, no exponent below -6."""
    a = y.abs()
    e = torch.floor(torch.log2(a.clamp_min(2.0 ** -20)))
    e = e + (a >= torch.exp2(e + 1)).double() - (a < torch.exp2(e)).double()
    step = torch.exp2(e.clamp_min(-6) - 3)
    return torch.round(y / step) * step


def _power(amax):
    """2^e, the smallest with amax <= 448 * 2^e and e >= -64."""
    e = torch.ceil(torch.log2(amax.clamp_min(1e-300) / 448))
    e = e + (amax > 448 * torch.exp2(e)).double()
    e = e - (amax <= 448 * torch.exp2(e - 1)).double()
    return torch.exp2(e.clamp_min(-64))


def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)  # the inputs alone
    finally:
        own = was
    return {"append": _exact_append, "attend": _exact_attend, "evict": _exact_evict}[case["kind"]](state, case)


def _exact_append(state, case):
    c, block, cap = state["tensors"], case["block"], _capacity(case)
    counts = _counts(case) or [case["tokens"]] * case["batch"]
    result = dict(positions=None, cursors=None)
    for name in ("key", "value"):
        codes, scales = c[name + "_codes"].double(), c[name + "_scales"].double()
        for b, (start, count) in enumerate(zip(_lengths(case), counts)):
            count = min(count, cap - start)
            if not count:
                continue
            first, last = start // block, (start + count - 1) // block + 1
            old = scales[b, :, first].clone() if start % block else torch.zeros_like(scales[b, :, first])
            rows = torch.zeros(case["kv_heads"], (last - first) * block, D, dtype=torch.float64, device=DEVICE)
            lead = start - first * block
            rows[:, lead:lead + count] = state[name][b, :, :count].double()
            s = _power(rows.reshape(case["kv_heads"], last - first, -1).abs().amax(-1))
            s[:, 0] = torch.maximum(s[:, 0], old)
            codes[b, :, first * block:start] = _rounded(codes[b, :, first * block:start] * (old / s[:, 0])[:, None, None])
            wide = s.repeat_interleave(block, 1)[:, lead:lead + count, None]
            codes[b, :, start:start + count] = _rounded(state[name][b, :, :count].double() / wide)
            scales[b, :, first:last] = s
        result[name + "_codes"], result[name + "_scales"] = codes, scales
    return {name: result[name] for name in NAMES}


def _exact_attend(state, case):
    c, block = state["tensors"], case["block"]
    b, hq, tokens, _ = state["query"].shape
    group = hq // case["kv_heads"]
    counts = _counts(case) or [tokens] * b
    out = torch.zeros(b, tokens, hq, D, dtype=torch.float64, device=DEVICE)
    lse = torch.full((b, hq, tokens), -math.inf, dtype=torch.float64, device=DEVICE)
    weights = torch.zeros(b, case["kv_heads"], _capacity(case), dtype=torch.float64, device=DEVICE)
    seen = c["cursors"][1].tolist()
    for i, (n, count) in enumerate(zip(_lengths(case), counts)):
        at = seen[i] - count + torch.arange(count, device=DEVICE)
        for head in range(case["kv_heads"]):
            scale = [c[x][i, head].double().repeat_interleave(block)[:n, None] for x in ("key_scales", "value_scales")]
            key, value = c["key_codes"][i, head, :n].double() * scale[0], c["value_codes"][i, head, :n].double() * scale[1]
            position = c["positions"][i, head, :n]
            seeing = position <= at[:, None]
            if case["window"]:
                seeing &= position > at[:, None] - case["window"]
            for g in range(head * group, head * group + group):
                if not count:
                    continue
                s = torch.where(seeing, (state["query"][i, g, :count].double() @ key.t()) * SCALE, -math.inf)
                z = torch.logsumexp(s, -1)
                p = torch.where(seeing, (s - torch.where(z == -math.inf, 0, z)[:, None]).exp(), 0)
                out[i, :count, g], lse[i, g, :count] = p @ value, z
                weights[i, head, :n] += p.sum(0)
    return dict(out=out, lse=lse, weights=weights) if case["accumulate"] else dict(out=out, lse=lse)


def _exact_evict(state, case):
    c, block, keep = state["tensors"], case["block"], case["keep"]
    to = {name: t.double() if name != "cursors" else None for name, t in state["into_tensors"].items()}
    to["positions"] = None
    seen = c["cursors"][1].tolist()
    for b, n in enumerate(_lengths(case)):
        for h in range(case["kv_heads"]):
            position, weight = c["positions"][b, h, :n].tolist(), c["weights"][b, h, :n].tolist()
            held = [p < case["num_sink"] or p >= seen[b] - case["recent"] for p in position]
            best = sorted(range(n), key=lambda r: (not held[r], -weight[r], r))[:keep]
            source = [r if r < min(n, keep) else None for r in range(min(n, keep))]
            kept = set(best)
            movers = sorted(r for r in best if r >= keep)
            holes = [r for r in range(min(n, keep)) if r not in kept]
            for r, m in zip(holes, movers):
                source[r] = m
            at = torch.tensor(source, device=DEVICE, dtype=torch.long)
            moved = torch.zeros(len(source), dtype=torch.bool, device=DEVICE)
            moved[torch.tensor(holes, device=DEVICE, dtype=torch.long)] = True
            to["weights"][b, h, :len(source)] = c["weights"][b, h].double()[at]
            for name in ("key", "value"):
                s = c[name + "_scales"][b, h].double()
                value = c[name + "_codes"][b, h].double()[at] * s[at // block][:, None]
                size = value.abs().amax(-1)
                blocks = -(-len(source) // block)
                need = torch.zeros(blocks * block, dtype=torch.float64, device=DEVICE)
                need[:len(source)] = torch.where(moved, size, -1.0)
                need[len(source):] = -1.0
                top = need.reshape(blocks, block).amax(-1)
                grown = torch.where(top >= 0, torch.maximum(s[:blocks], _power(top.clamp_min(0))), s[:blocks])
                to[name + "_scales"][b, h, :blocks] = grown
                to[name + "_codes"][b, h, :len(source)] = _rounded(value / grown.repeat_interleave(block)[:len(source), None])
    return {name: to[name] for name in NAMES + ("weights",)}
