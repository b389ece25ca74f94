"""Paged KV cache, drafted trees and their attention on the GPU against the 64-bit oracle (oracle/paged.py): plans, moved
rows and lengths equal, rotated rows within a rounding, attention within the bounds derived there."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from community_kv_amd import DraftTree, PagedKVCache, RotaryTable, paged_append, paged_attention, paged_commit
from oracle import paged as op

pytestmark = pytest.mark.gpu

D = 128
SCALE = D ** -0.5
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}


def _rand(gen, *shape, dtype=F32, size=1.0):
    x = torch.randn(*shape, D, generator=gen) * torch.exp(0.5 * torch.randn(*shape, 1, generator=gen)) * size
    return x.to(dtype)


def _i32(values, device):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device=device)


def _host(t):
    return t.detach().cpu().double().numpy()


LARGE = 262_144  # rows a sequence's table may name: which kernel takes a call goes by that, the host knows no lengths


def _cache(device, gen, *, lengths, heads=2, page=16, room=64, dtype=BF16, layers=1, spare=2, capacity=0):
    """A cache with `lengths` committed rows in pages of any order, random rows everywhere, and `room` rows more;
    `capacity`: so many rows' entries in the page table, most of them without a page."""
    need = [-(-(n + room) // page) for n in lengths]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=gen).tolist()
    table = torch.full((len(lengths), max(max(need), capacity // page)), -1, dtype=torch.int32)
    at = 0
    for b, pages in enumerate(need):
        table[b, :pages] = torch.tensor(order[at:at + pages], dtype=torch.int32)
        at += pages
    pages = [_rand(gen, layers, pool, heads, page, dtype=dtype).to(device) for _ in range(2)]
    return PagedKVCache(key_pages=pages[0], value_pages=pages[1], page_table=table.to(device), lengths=_i32(lengths, device))


def _parents(gen, batch, tokens, shape):
    """Parents of drafted trees, None for a chain, with a few that are no earlier token."""
    if shape == "chain":
        return None
    p = torch.zeros(batch, tokens, dtype=torch.int64)
    for t in range(tokens):
        back = torch.randint(1, 4 if shape == "deep" else max(t, 1) + 2, (batch,), generator=gen)
        p[:, t] = (t - back).clamp_min(-1)
    odd = torch.rand(batch, tokens, generator=gen)
    p = torch.where(odd < 0.03, torch.randint(tokens, 2 * tokens + 9, (batch, tokens), generator=gen), p)
    return torch.where(odd > 0.97, -7, p).int()


# ------------------------------------------------------------------------------------------ plans

@pytest.mark.parametrize("tokens", [1, 2, 63, 64, 65, 200, 511, 512])
@pytest.mark.parametrize("shape", ["deep", "wide", "line"])
def test_plan_matches_oracle(device, tokens, shape):
    print(f"plan tokens={tokens} shape={shape}", flush=True)
    gen = torch.Generator().manual_seed(tokens)
    if shape == "line":
        parents = torch.arange(-1, tokens - 1, dtype=torch.int32).expand(3, tokens).contiguous()
    else:
        parents = _parents(gen, 3, tokens, shape)
    for counts in (None, [tokens // 2, -3, tokens + 9]):
        tree = DraftTree.from_parents(parents.to(device), counts=None if counts is None else _i32(counts, device))
        torch.cuda.synchronize()
        depths, masks = op.plan(parents.numpy(), counts)
        assert np.array_equal(tree.depths.cpu().numpy(), depths) and np.array_equal(tree.masks.cpu().numpy(), masks)


def test_plan_takes_strided_parents(device):
    gen = torch.Generator().manual_seed(1)
    parents = _parents(gen, 4, 30, "wide")
    a = DraftTree.from_parents(parents.to(device))
    b = DraftTree.from_parents(parents.t().contiguous().to(device).t())
    torch.cuda.synchronize()
    assert torch.equal(a.depths, b.depths) and torch.equal(a.masks, b.masks)


# ------------------------------------------------------------------------------------------ append

def _append_case(device, gen, cache, *, tokens, query_heads=0, dtype=BF16, rotary=0, interleaved=False, shape="chain",
                 counts=None, layer=0, layout="heads"):
    heads, batch = cache.kv_heads, cache.batch
    oracle = op.Paged.of(cache)
    before = (cache.key_pages.clone(), cache.value_pages.clone())
    key, value, query = (_rand(gen, batch, n, tokens, dtype=dtype) for n in (heads, heads, query_heads))
    if layout == "tokens":
        key, value, query = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (key, value, query))
    parents = _parents(gen, batch, tokens, shape)
    count_t = None if counts is None else _i32(counts, device)
    tree = None if parents is None else DraftTree.from_parents(parents.to(device), counts=count_t)
    table = None
    if rotary:
        table = RotaryTable.from_frequencies((1e4 ** -(torch.arange(rotary // 2, dtype=torch.float64) / (rotary // 2))).to(device),
                                             cache.capacity + 3, interleaved=interleaved)
    got = paged_append(cache, key.to(device), value.to(device), layer=layer, query=query.to(device) if query_heads else None,
                       rotary=table, tree=tree, counts=count_t if tree is None else None)
    torch.cuda.synchronize()
    angles = None if table is None else (_host(table.cosines), _host(table.sines))
    turned, written = oracle.append(layer, _host(key), _host(value), _host(query) if query_heads else None, angles, interleaved,
                                    None if parents is None else parents.numpy(), counts)
    half = HALF_STEP[cache.dtype]
    # two rounded products, or one and a fused sum: 2 u of |x| + |y| each; then half a step of the type, and of its subnormals
    size = np.sqrt(2.0) * max(np.abs(_host(key)).max(), np.abs(_host(query)).max() if query_heads else 0.0)

    def near(a, b):
        return (np.abs(a - b) <= half * np.abs(b) + 4 * op.U * (1 + half) * size + 2.0 ** -25).all()

    assert near(_host(cache.key_pages)[layer][written], oracle.keys[layer][written])
    assert (np.abs(_host(cache.value_pages) - oracle.values)[layer][written] <=
            half * np.abs(oracle.values[layer][written]) + 2.0 ** -25).all()
    if not rotary and dtype == cache.dtype:
        assert np.array_equal(_host(cache.key_pages), oracle.keys) and np.array_equal(_host(cache.value_pages), oracle.values)
    for now, then in zip((cache.key_pages, cache.value_pages), before):  # everything else is as it was
        same = (now == then).cpu().numpy()
        same[layer][written] = True
        assert same.all()
    assert np.array_equal(cache.overflow.cpu().numpy(), oracle.overflow)
    assert np.array_equal(cache.lengths.cpu().numpy(), oracle.lengths)
    if query_heads:
        assert got.shape == (batch, query_heads, tokens, D) and got.dtype == cache.dtype and near(_host(got), turned)
        dead = np.zeros((batch, tokens), bool) if counts is None else np.arange(tokens) >= np.array(counts)[:, None]
        assert not _host(got).transpose(0, 2, 1, 3)[dead].any()
    else:
        assert got is None


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype,store", [(BF16, BF16), (F16, F16), (F32, BF16), (F32, F16), (BF16, F16), (F16, BF16)])
def test_append_matches_oracle(device, page, dtype, store):
    print(f"append page={page} dtype={dtype} store={store}", flush=True)
    gen = torch.Generator().manual_seed(page)
    cache = _cache(device, gen, lengths=[0, 5, 130], heads=3, page=page, room=200, dtype=store, layers=2)
    for tokens, kwargs in ((1, {}), (1, dict(rotary=128, query_heads=6)), (70, dict(counts=[70, 0, 33], rotary=64, query_heads=3)),
                           (17, dict(rotary=16, interleaved=True, shape="deep", layer=1, layout="tokens", query_heads=9)),
                           (200, dict(rotary=96, counts=[1, 200, 199], layer=1)), (9, dict(counts=[-4, 99, 2])),
                           (33, dict(rotary=128, interleaved=True, shape="wide", counts=[33, 0, 20], query_heads=3))):
        _append_case(device, gen, cache, tokens=tokens, dtype=dtype, **kwargs)


def test_append_many_tokens_and_heads(device):
    """A wave a token (long prompts), rows that do not fill the last round of eight, one KV head."""
    gen = torch.Generator().manual_seed(2)
    _append_case(device, gen, _cache(device, gen, lengths=[3], heads=1, page=64, room=9000), tokens=8999, rotary=128, query_heads=3)
    _append_case(device, gen, _cache(device, gen, lengths=[7, 0], heads=5, page=32, room=600), tokens=600, rotary=32, query_heads=5,
                 counts=[599, 311], layout="tokens")


def test_append_past_the_capacity_and_without_pages(device):
    """Tokens without a row are dropped and flagged, for their sequence alone; queries are turned all the same."""
    gen = torch.Generator().manual_seed(3)
    cache = _cache(device, gen, lengths=[30, 40, 10], page=16, room=16)
    cache.page_table[1, 3] = -1
    cache.page_table[2, 0] = cache.pages  # one past the pool; rows 10 .. 15 of sequence 2
    capacity = cache.capacity
    assert capacity == 64
    _append_case(device, gen, cache, tokens=34, rotary=64, query_heads=4, counts=[34, 8, 3])
    assert cache.overflow.tolist() == [1, 0, 1]  # sequence 0 has pages for rows 0 .. 47
    _append_case(device, gen, cache, tokens=35, rotary=64, query_heads=4, counts=[34, 9, 0], shape="wide")
    assert cache.overflow.tolist() == [1, 1, 1]
    with pytest.raises(RuntimeError, match="overflow"):
        cache.assert_no_overflow()
    cache.overflow.zero_()
    cache.lengths.copy_(_i32([capacity, -5, 1 << 30], device))  # a full one, and cursors out of range
    _append_case(device, gen, cache, tokens=2, counts=[1, 2, 2])
    assert cache.overflow.tolist() == [1, 0, 1]


def test_append_strides(device):
    """Views of a fused projection, broadcast values and addresses that are not 16-byte aligned give the contiguous result."""
    gen = torch.Generator().manual_seed(4)
    fused = _rand(gen, 2, 7, 12, dtype=BF16).to(device)  # [B, T, heads]
    key, value, query = (fused[:, :, a:b].transpose(1, 2) for a, b in ((0, 2), (2, 4), (4, 12)))
    odd = torch.empty(key.numel() + 1, dtype=BF16, device=device)[1:].view(key.shape)
    odd.copy_(key)
    results = []
    for k, v, q in ((key, value, query), (key.contiguous(), value.contiguous(), query.contiguous()), (odd, value, query)):
        g = torch.Generator().manual_seed(5)
        cache = _cache(device, g, lengths=[20, 3])
        table = RotaryTable.from_frequencies(torch.rand(32, generator=g).double().to(device), cache.capacity)
        results.append((paged_append(cache, k, v, query=q, rotary=table), cache.key_pages, cache.value_pages))
    wide = value[:, :1].expand(-1, 2, -1, -1)
    caches = [_cache(device, torch.Generator().manual_seed(5), lengths=[20, 3]) for _ in range(2)]
    paged_append(caches[0], wide, wide)
    paged_append(caches[1], wide.contiguous(), wide.contiguous())
    none = _cache(device, torch.Generator().manual_seed(5), lengths=[20, 3])
    assert paged_append(none, key[:, :, :0], value[:, :, :0]) is None
    torch.cuda.synchronize()
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
    assert torch.equal(caches[0].key_pages, caches[1].key_pages) and torch.equal(caches[0].value_pages, caches[1].value_pages)


def test_append_keeps_special_values(device):
    """Infinities and NaN stay in their dims (the rotation spreads them to the partner)."""
    gen = torch.Generator().manual_seed(6)
    cache = _cache(device, gen, lengths=[0], heads=1, room=16)
    x = _rand(gen, 1, 1, 3, dtype=F32)
    x[0, 0, 1, 5], x[0, 0, 2, 127] = float("inf"), float("nan")
    paged_append(cache, x.to(device), x.to(device))
    torch.cuda.synchronize()
    rows = cache.key_pages[0, cache.page_table[0, 0], 0, :3].cpu()
    assert torch.equal(rows.isnan(), x[0, 0].isnan()) and torch.equal(rows.isinf(), x[0, 0].isinf())


# ------------------------------------------------------------------------------------------ attention

def _attend_case(device, gen, cache, *, group, tokens, shape="chain", counts=None, window=0, query=None, layer=0, scale=SCALE):
    batch, heads, dtype = cache.batch, cache.kv_heads, cache.dtype
    if query is None:
        query = _rand(gen, batch, heads * group, tokens, dtype=dtype)
    parents = _parents(gen, batch, tokens, shape)
    count_t = None if counts is None else _i32(counts, device)
    tree = None if parents is None else DraftTree.from_parents(parents.to(device), counts=count_t)
    out, lse = paged_attention(query.to(device), cache, layer=layer, softmax_scale=scale, tree=tree,
                               counts=count_t if tree is None else None, window=window)
    torch.cuda.synchronize()
    assert out.shape == (batch, tokens, heads * group, D) and out.dtype == dtype and lse.shape == (batch, heads * group, tokens)
    want, tol = op.Paged.of(cache).attend(layer, _host(query), scale=scale, parents=None if parents is None else parents.numpy(),
                                          counts=counts, window=window, half_step=HALF_STEP[dtype])
    got_out, got_lse = _host(out), _host(lse)
    live = ~np.isneginf(want[1])
    assert np.array_equal(np.isneginf(got_lse), ~live)
    assert (np.abs(got_lse[live] - want[1][live]) <= tol[1][live]).all()
    worst = np.abs(got_out - want[0]) - tol[0]
    assert (worst <= 0).all(), float(worst.max())
    assert not got_out[~live.transpose(0, 2, 1)].any()
    return out, lse


FORMS = [  # heads, group, tokens: all forms of the kernels
    (2, 1, 1), (2, 4, 1), (1, 16, 1), (3, 7, 2), (2, 4, 8), (2, 2, 15), (1, 16, 3), (2, 7, 9), (1, 1, 100), (2, 4, 31),
    (1, 16, 16), (2, 3, 50), (1, 8, 65), (1, 4, 90)]


@pytest.mark.parametrize("heads,group,tokens", FORMS)
@pytest.mark.parametrize("dtype,page,capacity", [(BF16, 16, 0), (F16, 64, 0), (F16, 16, LARGE), (BF16, 128, LARGE)])
def test_attend_matches_oracle(device, heads, group, tokens, dtype, page, capacity):
    """Ragged lengths (none, one row, page and tile ends), chains and trees, counts from none to all, windows."""
    gen = torch.Generator().manual_seed(heads * group + tokens)
    cache = _cache(device, gen, lengths=[0, 1, 63, 64, 200, 391], heads=heads, page=page, room=tokens, dtype=dtype, capacity=capacity)
    counts = [tokens, 0, max(tokens - 1, 0), tokens + 3, tokens // 2, -1]
    for shape, count, window in (("chain", None, 0), ("chain", counts, 0), ("chain", None, 1), ("chain", None, 70), ("wide", None, 0),
                                 ("deep", counts, 0), ("deep", None, 5), ("wide", counts, 129)):
        print(f"attend {heads} x {group} x {tokens} {dtype} page={page} capacity={capacity} {shape} counts={count is not None} window={window}", flush=True)
        _attend_case(device, gen, cache, group=group, tokens=tokens, shape=shape, counts=count, window=window)


@pytest.mark.parametrize("heads,group,tokens,lengths,page", [
    (2, 4, 1, [3000, 17, 2049], 128), (1, 2, 12, [2500], 256), (2, 4, 16, [1800, 900], 32), (1, 4, 30, [2600, 0], 64),
    (1, 4, 70, [2300, 640], 16)])
@pytest.mark.parametrize("shape,window", [("chain", 0), ("deep", 0), ("chain", 700), ("wide", 300)])
@pytest.mark.parametrize("capacity", [0, LARGE])
def test_attend_long_caches_in_parts(device, heads, group, tokens, lengths, page, shape, window, capacity):
    print(f"attend parts {heads} x {group} x {tokens} over {lengths} page={page} {shape} window={window}", flush=True)
    gen = torch.Generator().manual_seed(sum(lengths))
    cache = _cache(device, gen, lengths=lengths, heads=heads, page=page, room=tokens, capacity=capacity)
    _attend_case(device, gen, cache, group=group, tokens=tokens, shape=shape, window=window)


@pytest.mark.parametrize("group,tokens,shape", [(4, 300, "deep"), (1, 512, "wide"), (2, 512, "deep"), (3, 511, "chain")])
@pytest.mark.parametrize("capacity", [0, LARGE])
def test_attend_large_trees(device, group, tokens, shape, capacity):
    """Masks of many words whose draft starts inside a tile."""
    print(f"attend large {group} x {tokens} {shape}", flush=True)
    gen = torch.Generator().manual_seed(tokens + group)
    cache = _cache(device, gen, lengths=[77, 128], heads=1, page=32, room=tokens, dtype=F16, capacity=capacity)
    _attend_case(device, gen, cache, group=group, tokens=tokens, shape=shape, counts=[tokens, tokens - 70])


def test_attend_one_layer_of_several(device):
    gen = torch.Generator().manual_seed(7)
    cache = _cache(device, gen, lengths=[100, 33], layers=3, room=40)
    for layer in (0, 2):
        _attend_case(device, gen, cache, group=2, tokens=1, layer=layer)
        _attend_case(device, gen, cache, group=4, tokens=40, shape="wide", layer=layer)


def test_attend_many_sequences(device):
    """As many sequences as fill the chip without parts, and more than a wave counts at once."""
    gen = torch.Generator().manual_seed(8)
    lengths = [int(x) for x in torch.randint(0, 90, (130,), generator=gen)]
    cache = _cache(device, gen, lengths=lengths, heads=4, room=2)
    _attend_case(device, gen, cache, group=2, tokens=2)
    lengths = [int(x) for x in torch.randint(0, 1500, (70,), generator=gen)]
    cache = _cache(device, gen, lengths=lengths, heads=1, page=64, room=1)
    _attend_case(device, gen, cache, group=1, tokens=1)


@pytest.mark.parametrize("batch,group,tokens,shape,long", [(70, 1, 1, "chain", 5000), (40, 3, 9, "deep", 3000), (18, 2, 65, "wide", 2500)])
def test_attend_one_long_sequence_among_many(device, batch, group, tokens, shape, long):
    """Whole sequences fill the chip, and the long one is cut all the same: some parts are joined, some are not."""
    print(f"attend one long of {batch} {group} x {tokens}", flush=True)
    gen = torch.Generator().manual_seed(batch)
    lengths = [int(x) for x in torch.randint(0, 60, (batch,), generator=gen)]
    lengths[batch // 3] = long
    cache = _cache(device, gen, lengths=lengths, heads=8, room=tokens, capacity=8192)
    _attend_case(device, gen, cache, group=group, tokens=tokens, shape=shape)


@pytest.mark.parametrize("group,tokens,capacity", [(2, 3, 0), (4, 16, LARGE), (4, 70, LARGE)])
@pytest.mark.parametrize("scale", [1e-30, 1e-10])
def test_attend_smallest_scales(device, group, tokens, capacity, scale):
    gen = torch.Generator().manual_seed(tokens)
    cache = _cache(device, gen, lengths=[700, 5, 1500], room=tokens, page=64, capacity=capacity)
    _attend_case(device, gen, cache, group=group, tokens=tokens, scale=scale)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attend_extreme_scores(device, dtype):
    """Scores of hundreds: one row takes all; a rising order moves the running maximum again and again."""
    gen = torch.Generator().manual_seed(9)
    for order in (1, -1):
        for group, tokens, capacity in ((4, 1, 0), (8, 40, 0), (8, 10, LARGE), (8, 40, LARGE)):
            cache = _cache(device, gen, lengths=[500], heads=1, room=tokens, dtype=dtype, capacity=capacity)
            ramp = order * torch.linspace(-40, 40, 500 + tokens)
            for r in range(500 + tokens):
                cache.key_pages[0, cache.page_table[0, r // 16], 0, r % 16] = ramp[r].to(device, dtype)
            query = torch.ones(1, group, tokens, D, dtype=dtype) * torch.linspace(-1, 1, group).reshape(1, group, 1, 1).to(dtype)
            _attend_case(device, gen, cache, group=group, tokens=tokens, query=query)


@pytest.mark.parametrize("group", [2, 16])
def test_attend_fp16_keeps_small_probabilities(device, group):
    """A row with most of the weight and thousands of others with 2^-18 of its: together they count."""
    n = 12_000
    gen = torch.Generator().manual_seed(10)
    for tokens in (1, 20):
        cache = _cache(device, gen, lengths=[n], heads=1, page=256, room=tokens, dtype=F16, capacity=LARGE)
        cache.key_pages.zero_()
        cache.value_pages.fill_(1.0)
        query = torch.zeros(1, group, tokens, D, dtype=F16)
        query[..., 0] = 1.0
        big = torch.zeros(D)
        big[0] = 18 * np.log(2.0) / SCALE  # in fp16: a score of 18 ln 2 within 2^-11 of it
        cache.key_pages[0, cache.page_table[0, 0], 0, 7] = big.to(device, F16)
        cache.value_pages[0, cache.page_table[0, 0], 0, 7] = 0.0
        out, _ = _attend_case(device, gen, cache, group=group, tokens=tokens, query=query)
        weight = np.exp(float(big.half()[0]) * SCALE)
        for t in range(tokens):
            rest = n + t  # rows of value one that token t sees
            # the numbers above are the same for all of them, so a rounding of one is a rounding of their sum: 2^-11, and one more
            assert abs(float(out[0, t, 0, 0]) * (weight + rest) / rest - 1) < 2 * 2.0 ** -11 + 2.0 ** -13 + 2.0 ** -24 * weight / rest * 4


@pytest.mark.parametrize("group,tokens,capacity", [(2, 1, 0), (2, 6, 0), (4, 8, 0), (4, 30, 0), (4, 16, LARGE), (4, 30, LARGE),
                                                   (8, 40, LARGE)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attend_special_values_reach_only_who_sees_them(device, group, tokens, capacity, dtype):
    """Infinities and NaN in rows of other branches, before a window, past the length, in spare pages: no change; a
    value that is not finite and seen appears in its dim alone, a NaN key makes the query NaN."""
    print(f"special {group} x {tokens} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(group * tokens)
    nan, inf = float("nan"), float("inf")

    def rows(cache, which):
        pages = cache.key_pages if which == "key" else cache.value_pages

        def put(r, value, dim=slice(None)):
            pages[0, cache.page_table[0, r // 16], 0, r % 16, dim] = value
        return put

    for shape, window in (("chain", 0), ("chain", 30), ("wide", 0), ("deep", 30)):
        cache = _cache(device, gen, lengths=[100], heads=1, room=tokens, dtype=dtype, capacity=capacity)
        parents = _parents(gen, 1, tokens, shape)
        tree = None if parents is None else DraftTree.from_parents(parents.to(device))
        query = _rand(gen, 1, group, tokens, dtype=dtype).to(device)

        def call():
            out, lse = paged_attention(query, cache, softmax_scale=SCALE, tree=tree, window=window)
            torch.cuda.synchronize()
            return out[0].cpu(), lse[0].cpu()

        oracle = op.Paged.of(cache)
        depths, kin = oracle._steps(tokens, None if parents is None else parents.numpy(), None, 0)
        seen = np.zeros((tokens, 100 + tokens), bool)
        for t in range(tokens):
            seen[t, oracle.sees(0, t, depths, kin, window)] = True
        seen = torch.from_numpy(seen)
        clean, clean_lse = call()
        pool = torch.ones(cache.pages, 16, dtype=torch.bool)
        for r in range(100 + tokens):
            pool[int(cache.page_table[0, r // 16]), r % 16] = False
        for pages in (cache.key_pages, cache.value_pages):  # whatever no row uses
            pages[0, :, 0][pool.to(device)] = nan
        key, value = rows(cache, "key"), rows(cache, "value")
        hidden = [r for r in range(100 + tokens) if not seen[:, r].any()]
        for r in hidden:
            key(r, nan)
            value(r, inf)
        got, got_lse = call()
        assert torch.equal(got, clean) and torch.equal(got_lse, clean_lse)
        # rows that some see: the last one, and one before the draft
        value(99 + tokens, nan, 5)
        value(99, inf, 77)
        value(98, -inf, 126)
        got, got_lse = call()
        assert torch.equal(got_lse, clean_lse)
        for t in range(tokens):
            expect = clean[t].clone()
            if seen[t, 99 + tokens]:
                expect[:, 5] = nan
            if seen[t, 99]:
                expect[:, 77] = inf
            if seen[t, 98]:
                expect[:, 126] = -inf
            assert torch.equal(got[t].isnan(), expect.isnan()), (shape, window, t)
            ok = ~expect.isnan()
            assert torch.equal(got[t][ok], expect[ok]), (shape, window, t)
        key(99 + tokens, nan, 3)
        got, got_lse = call()
        for t in range(tokens):
            if seen[t, 99 + tokens]:
                assert bool(got[t].isnan().all()) and bool(got_lse[:, t].isnan().all())
            else:
                assert torch.equal(got_lse[:, t], clean_lse[:, t]) and not bool(got[t].isnan().any())


@pytest.mark.parametrize("group,tokens,capacity", [(2, 1, 0), (2, 12, 0), (4, 16, 0), (4, 16, LARGE), (4, 32, LARGE), (4, 70, LARGE)])
def test_attend_passes_over_missing_pages(device, group, tokens, capacity):
    """Rows whose page number is none are not attended, whatever the number is; a draft without pages sees the rest."""
    print(f"missing pages {group} x {tokens}", flush=True)
    gen = torch.Generator().manual_seed(group + tokens)
    cache = _cache(device, gen, lengths=[150, 70, 40], heads=2, room=tokens, capacity=capacity)
    cache.page_table[0, 3], cache.page_table[0, 7] = -1, cache.pages
    cache.page_table[1, 0], cache.page_table[1, 2] = -2**31, 2**31 - 1
    cache.page_table[2] = -1
    for shape, window in (("chain", 0), ("wide", 0), ("chain", 60)):
        _attend_case(device, gen, cache, group=group, tokens=tokens, shape=shape, window=window)


def test_attend_past_the_capacity(device):
    """Tokens without a row see those that have one; cursors out of range are taken as the nearest."""
    gen = torch.Generator().manual_seed(11)
    cache = _cache(device, gen, lengths=[60, 64, 30], room=0, page=16)
    assert cache.capacity == 64
    for group, tokens in ((2, 8), (8, 20)):
        cache.lengths.copy_(_i32([60, 64, 30], device))
        _attend_case(device, gen, cache, group=group, tokens=tokens, counts=[tokens, 3, tokens])
        cache.lengths.copy_(_i32([1 << 30, -9, -2**31], device))
        cache.page_table[:] = cache.page_table[:1].clone()
        _attend_case(device, gen, cache, group=group, tokens=tokens)


def test_attend_shared_pages(device):
    """Two sequences over the pages of one prompt, with drafts of their own."""
    gen = torch.Generator().manual_seed(12)
    for capacity in (0, LARGE):
        cache = _cache(device, gen, lengths=[64, 64], room=20, capacity=capacity)
        cache.page_table[1, :4] = cache.page_table[0, :4]
        _attend_case(device, gen, cache, group=4, tokens=20, shape="wide")
        _attend_case(device, gen, cache, group=4, tokens=1)


def test_attend_strides(device):
    gen = torch.Generator().manual_seed(13)
    for tokens, capacity in ((3, 0), (40, LARGE)):
        cache = _cache(device, gen, lengths=[100, 77], capacity=capacity)
        fused = _rand(gen, 2, tokens, 12, dtype=BF16).to(device)
        view = fused[:, :, 2:10].transpose(1, 2)
        odd = torch.empty(view.numel() + 1, dtype=BF16, device=device)[1:].view(view.shape)
        odd.copy_(view)
        a, b, c = (paged_attention(q, cache, softmax_scale=SCALE) for q in (view, view.contiguous(), odd))
        torch.cuda.synchronize()
        for x, y, z in zip(a, b, c):
            assert torch.equal(x, y) and torch.equal(x, z)
    none = paged_attention(view[:, :, :0], cache, softmax_scale=SCALE)
    assert none[0].shape == (2, 0, 8, D) and none[1].shape == (2, 8, 0)


def test_places_beyond_32_bits(device):
    """Layers and pages whose bytes and elements are beyond 2^32: written, attended and committed where they belong."""
    print("pages beyond 2^32 elements", flush=True)
    gen = torch.Generator().manual_seed(14)
    pages = 140_000  # 2 layers of 2.3 G elements each, keys and values
    cache = PagedKVCache.allocate(layers=2, batch=1, kv_heads=2, capacity=pages * 64, page_size=64, device=device)
    n = pages * 64 - 40
    cache.lengths.fill_(n)
    x = [_rand(gen, 1, 2, 8, dtype=BF16).to(device) for _ in range(2)]
    for layer in range(2):
        paged_append(cache, x[0] + layer, x[1] - layer, layer=layer)
    query = (20 * x[0][:, :, 5:6] / x[0][:, :, 5:6].float().norm(dim=-1, keepdim=True)).to(BF16)
    paged_commit(cache, 2, path=_i32([[3, 5]], device))
    cache.lengths.fill_(n + 2)
    torch.cuda.synchronize()
    for layer in range(2):
        for j, p in enumerate((3, 5)):
            page, at = (n + j) // 64, (n + j) % 64
            assert torch.equal(cache.key_pages[layer, page, :, at], (x[0] + layer)[0, :, p])
            assert torch.equal(cache.value_pages[layer, page, :, at], (x[1] - layer)[0, :, p])
    # all other rows are zeros: a score of 0 each
    cache.lengths.fill_(n + 1)
    out, lse = paged_attention(query, cache, layer=1, softmax_scale=1.0)
    many, _ = paged_attention(query.expand(-1, -1, 40, -1), cache, layer=1, softmax_scale=1.0, counts=_i32([1], device))
    torch.cuda.synchronize()
    page = n // 64
    s = torch.stack([query[0, :, 0].double() @ torch.zeros(D, device=device).double()] * 1, 0)[0]
    key, value = (t[1, page, :, n % 64:n % 64 + 2].double() for t in (cache.key_pages, cache.value_pages))
    score = (key @ query[0, :, 0].double()[..., None])[..., 0]
    z = torch.logsumexp(torch.cat([score, torch.full((2, 1), float(np.log(float(n))), device=device).double()], 1), 1)
    want = ((score - z[:, None]).exp()[..., None] * value).sum(1)
    # 9 M terms of one size: their sum in 32 bits is off by some of 2^-24 a term of a lane's share, far below 2^-8
    assert (lse[0, :, 0].double() - z).abs().max() < 2.0 ** -8 and s.abs().max() == 0
    assert ((out[0, 0].double() - want).abs() <= 2.0 ** -6 * value.abs().sum(1)).all()
    assert ((many[0, 0].double() - want).abs() <= 2.0 ** -6 * value.abs().sum(1)).all() and not many[0, 1:].any()


# ------------------------------------------------------------------------------------------ commit

@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("layers,heads", [(1, 1), (3, 2), (2, 5)])
def test_commit_matches_oracle(device, page, layers, heads):
    """Paths of every kind: none, whole, gaps, entries that do not ascend, come twice, are negative or past the table."""
    gen = torch.Generator().manual_seed(page + layers)
    paths = [[0, 1, 2, 3], [2, 5, 9, 30], [4, 4, 5, 6], [3, 2, 8, 9], [-1, 0, 1, 2], [1, 2, 3, 5000], [0, 2, 3, 5], [7, 8, 9, 10]]
    for dtype in (BF16, F16):
        for counts in ([4] * 8, [0, 1, 4, 3, 4, 4, 2, 9], [-2, 4, 1, 4, 0, 3, 4, 4], 3):
            cache = _cache(device, gen, lengths=[0, 5, 16, 31, 90, 7, 64, 100], heads=heads, page=page, room=40, dtype=dtype, layers=layers)
            oracle = op.Paged.of(cache)
            paged_commit(cache, counts if isinstance(counts, int) else _i32(counts, device), path=_i32(paths, device))
            torch.cuda.synchronize()
            oracle.commit(counts, paths)
            assert np.array_equal(_host(cache.key_pages), oracle.keys) and np.array_equal(_host(cache.value_pages), oracle.values)
            assert np.array_equal(cache.lengths.cpu().numpy(), oracle.lengths)


@pytest.mark.parametrize("entries", [1, 16, 17, 64, 65, 300, 512])
def test_commit_long_paths(device, entries):
    """Rows that move into places that later entries' rows left, over several rounds and pages."""
    gen = torch.Generator().manual_seed(entries)
    cache = _cache(device, gen, lengths=[11, 40], heads=2, page=32, room=700, layers=2)
    paths = torch.stack([torch.randperm(700, generator=gen)[:entries].sort().values for _ in range(2)])
    paths[1, entries // 2:] = torch.arange(entries // 2, entries) + int(paths[1, max(entries // 2 - 1, 0)]) + 1
    paths = paths.clamp_max(10_000)
    oracle = op.Paged.of(cache)
    paged_commit(cache, _i32([entries, entries], device), path=paths.int().to(device))
    torch.cuda.synchronize()
    oracle.commit([entries, entries], paths.numpy())
    assert np.array_equal(_host(cache.key_pages), oracle.keys) and np.array_equal(_host(cache.value_pages), oracle.values)
    assert np.array_equal(cache.lengths.cpu().numpy(), oracle.lengths)


def test_commit_without_a_path_and_without_pages(device):
    gen = torch.Generator().manual_seed(15)
    cache = _cache(device, gen, lengths=[10, 20, 60], room=4)
    before = cache.key_pages.clone()
    for counts in (1, 0, [3, 0, 2], [-4, 2**31 - 1, 1], 2**40):
        oracle = op.Paged.of(cache)
        paged_commit(cache, counts if isinstance(counts, int) else _i32(counts, device))
        torch.cuda.synchronize()
        oracle.commit(counts)
        assert np.array_equal(cache.lengths.cpu().numpy(), oracle.lengths)
    assert cache.lengths.tolist() == [cache.capacity] * 3 and torch.equal(cache.key_pages, before)
    cache = _cache(device, gen, lengths=[10, 20, 28], room=36)
    cache.page_table[0, 1], cache.page_table[1, 1], cache.page_table[2, 3] = -1, cache.pages + 5, -3
    oracle = op.Paged.of(cache)
    path = [[1, 8, 20], [2, 13, 14], [3, 9, 25]]
    paged_commit(cache, 3, path=_i32(path, device))
    torch.cuda.synchronize()
    oracle.commit(3, path)
    assert np.array_equal(_host(cache.key_pages), oracle.keys) and np.array_equal(cache.lengths.cpu().numpy(), oracle.lengths)


# ------------------------------------------------------------------------------------------ together

def _run(device, dtype, *, graph, seed=20, steps=6, drafts=11):
    """A batch's requests as a server decodes them: prompts in two ragged pieces, then steps of drafted trees of which a
    path is kept, and single tokens.  Checks every output; returns what was computed."""
    gen = torch.Generator().manual_seed(seed)
    layers, batch, heads, group = 2, 2, 2, 4
    cache = PagedKVCache.allocate(layers=layers, batch=batch, kv_heads=heads, capacity=256, page_size=16, pages=40, dtype=dtype, device=device)
    order = torch.randperm(40, generator=gen)
    cache.page_table[0, :16], cache.page_table[1, :16] = order[:16].int().to(device), order[16:32].int().to(device)
    rotary = RotaryTable.from_frequencies((1e4 ** -(torch.arange(32) / 32)).double().to(device), cache.capacity)
    angles = (_host(rotary.cosines), _host(rotary.sines))
    oracle = op.Paged.of(cache)
    results = []

    def drawn(tokens):
        return [[_rand(gen, batch, n, tokens, dtype=dtype) for n in (heads, heads, heads * group)] for _ in range(layers)]

    def step(rows, parents=None, counts=None):
        tree = None if parents is None else DraftTree.from_parents(parents, counts=counts)
        given = []
        for layer in range(layers):
            key, value, query = rows[layer]
            query = paged_append(cache, key, value, layer=layer, query=query, rotary=rotary, tree=tree,
                                 counts=counts if tree is None else None)
            given.append((query, *paged_attention(query, cache, layer=layer, softmax_scale=SCALE, tree=tree,
                                                  counts=counts if tree is None else None)))
        return given

    def check(rows, given, parents=None, counts=None):
        torch.cuda.synchronize()
        host_counts = None if counts is None else counts.cpu().numpy()
        host_parents = None if parents is None else parents.cpu().numpy()
        for layer, (query, out, lse) in enumerate(given):
            turned, written = oracle.append(layer, *(_host(x) for x in rows[layer]), angles, False, host_parents, host_counts)
            half = HALF_STEP[dtype]
            size = 8 * op.U * max(np.abs(_host(x)).max() for x in rows[layer]) + 2.0 ** -25
            assert (np.abs(_host(query) - turned) <= half * np.abs(turned) + size).all()
            now = _host(cache.key_pages)[layer]
            assert (np.abs(now - oracle.keys[layer])[written] <= (half * np.abs(oracle.keys[layer]) + size)[written]).all()
            oracle.keys[layer] = now  # attention goes by the rounded keys
            assert np.array_equal(_host(cache.value_pages)[layer], oracle.values[layer])
            want, tol = oracle.attend(layer, _host(query), scale=SCALE, parents=host_parents, counts=host_counts, half_step=half)
            live = ~np.isneginf(want[1])
            assert (np.abs(_host(out) - want[0]) <= tol[0]).all()
            assert np.array_equal(~np.isneginf(_host(lse)), live)
            assert (np.abs(_host(lse)[live] - want[1][live]) <= tol[1][live]).all()
            results.append((query.clone(), out.clone(), lse.clone()))

    def commit(counts, path=None):
        oracle.commit(counts.cpu().numpy(), None if path is None else path.cpu().numpy())
        torch.cuda.synchronize()
        assert np.array_equal(cache.lengths.cpu().numpy(), oracle.lengths)
        assert np.array_equal(_host(cache.key_pages), oracle.keys) and np.array_equal(_host(cache.value_pages), oracle.values)

    for counts in ([37, 20], [5, 18]):
        rows, counts = drawn(37), _i32(counts, device)
        rows = [[x.to(device) for x in layer] for layer in rows]
        check(rows, step(rows, counts=counts), counts=counts)
        paged_commit(cache, counts)
        commit(counts)
    static = [[x.to(device) for x in layer] for layer in drawn(drafts)]
    single = [[x.to(device) for x in layer] for layer in drawn(1)]
    parents = torch.zeros(batch, drafts, dtype=torch.int32, device=device)
    counts, accepted = (torch.zeros(batch, dtype=torch.int32, device=device) for _ in range(2))
    path = torch.zeros(batch, drafts, dtype=torch.int32, device=device)
    ones = torch.ones(batch, dtype=torch.int32, device=device)
    given = {}
    calls = {"draft": lambda: given.update(draft=step(static, parents, counts)),
             "commit": lambda: paged_commit(cache, accepted, path=path),
             "token": lambda: (given.update(token=step(single)), paged_commit(cache, 1))}
    if graph:
        graphs = {}
        before = [t.clone() for t in (cache.key_pages, cache.value_pages, cache.lengths)]
        for name, call in calls.items():
            graphs[name] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graphs[name]):
                call()
        for t, s in zip((cache.key_pages, cache.value_pages, cache.lengths), before):
            assert torch.equal(t, s)  # a capture runs nothing
        calls = {name: g.replay for name, g in graphs.items()}
    for _ in range(steps):
        for to, source in zip(static + single, drawn(drafts) + drawn(1)):
            for t, s in zip(to, source):
                t.copy_(s)
        tree = _parents(gen, batch, drafts, "wide")
        parents.copy_(tree)
        counts.copy_(torch.randint(1, drafts + 1, (batch,), generator=gen))
        calls["draft"]()
        check(static, given["draft"], parents, counts)
        host_counts = counts.tolist()
        for b in range(batch):  # the branch of some drafted token
            _, kin = op.tree_of(tree[b].numpy(), host_counts[b])
            kept = kin[int(torch.randint(0, host_counts[b], (1,), generator=gen))]
            path[b, :len(kept)] = _i32(kept, device)
            accepted[b] = len(kept)
        calls["commit"]()
        commit(accepted, path)
        torch.ones(1000, device=device).sum().item()  # the program's own work between
        calls["token"]()
        lengths = cache.lengths.clone()
        cache.lengths.sub_(1)
        check(single, given["token"])
        cache.lengths.copy_(lengths)
        commit(ones)
    cache.assert_no_overflow()
    return results, cache


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_speculative_run(device, dtype):
    """Eager and captured, checked step by step and equal to the bit."""
    eager, a = _run(device, dtype, graph=False)
    replayed, b = _run(device, dtype, graph=True)
    for x, y in zip(eager, replayed):
        assert all(torch.equal(p, q) for p, q in zip(x, y))
    assert torch.equal(a.key_pages, b.key_pages) and torch.equal(a.value_pages, b.value_pages) and torch.equal(a.lengths, b.lengths)


@pytest.mark.parametrize("group,tokens,lengths,window,capacity", [
    (4, 1, [4000, 300], 0, 0), (2, 16, [2000, 100], 0, 0), (4, 16, [900, 3000], 100, 0), (4, 16, [900, 3000], 0, LARGE),
    (4, 32, [2500, 700], 0, LARGE), (4, 64, [1500, 2100], 500, LARGE), (4, 100, [90, 3000], 0, LARGE)])
def test_replays_equal_eager_calls(device, group, tokens, lengths, window, capacity):
    """Every form of the kernels captured, two graphs of one cache in turn with eager work between, lengths and tables that
    change between replays."""
    print(f"replay {group} x {tokens} over {lengths}", flush=True)
    gen = torch.Generator().manual_seed(tokens)
    cache = _cache(device, gen, lengths=lengths, page=32, room=tokens + 8, capacity=capacity)
    query = _rand(gen, 2, 2 * group, tokens, dtype=BF16).to(device)
    parents = _parents(gen, 2, tokens, "wide").to(device)

    def whole():
        return paged_attention(query, cache, softmax_scale=SCALE, tree=DraftTree.from_parents(parents), window=window)

    def one():
        return paged_attention(query[:, :, :1], cache, softmax_scale=SCALE)

    graphs, results = [], []
    for call in (whole, one):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            results.append(call())
    for turn in range(4):
        for graph, got, call in zip(graphs, results, (whole, one)):
            query.copy_(_rand(gen, 2, 2 * group, tokens, dtype=BF16))
            cache.lengths.sub_(_i32([11 * turn, 5], device))
            cache.page_table[0, :2] = cache.page_table[0, :2].flip(0).clone()
            graph.replay()
            want = call()
            torch.cuda.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_calls_on_a_side_stream(device):
    """Calls follow the current stream: a chain on a side stream, waited for by an event, equals the default one's."""
    results = []
    side = torch.cuda.Stream(device)
    for stream in (torch.cuda.current_stream(device), side):
        gen = torch.Generator().manual_seed(21)
        cache = _cache(device, gen, lengths=[500, 90], layers=2)
        key, value, query = (_rand(gen, 2, n, 30, dtype=BF16).to(device) for n in (2, 2, 8))
        parents = _parents(gen, 2, 30, "wide").to(device)
        table = RotaryTable.from_frequencies(torch.rand(64, generator=gen).double().to(device), cache.capacity)
        path = _i32([[1, 4, 9], [0, 2, 3]], device)
        stream.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(stream):
            tree = DraftTree.from_parents(parents)
            turned = paged_append(cache, key, value, layer=1, query=query, rotary=table, tree=tree)
            out, lse = paged_attention(turned, cache, layer=1, softmax_scale=SCALE, tree=tree)
            paged_commit(cache, 3, path=path)
            results.append((turned, out, lse, *paged_attention(turned[:, :, :1], cache, layer=1, softmax_scale=SCALE),
                            cache.key_pages, cache.lengths))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_same_call_twice_is_bit_equal(device):
    """No atomics on results: the same calls give equal bits."""
    gen = torch.Generator().manual_seed(22)
    for group, tokens, capacity in ((4, 1, 0), (4, 8, 0), (4, 16, 0), (4, 32, LARGE), (4, 70, LARGE)):
        cache = _cache(device, gen, lengths=[3000, 40, 900], page=64, room=70, capacity=capacity)
        query = _rand(gen, 3, 2 * group, tokens, dtype=BF16).to(device)
        a, b = (paged_attention(query, cache, softmax_scale=SCALE) for _ in range(2))
        torch.cuda.synchronize()
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_results_do_not_depend_on_the_batch(device):
    """Dead queries (counts) with NaN change nothing for the others."""
    gen = torch.Generator().manual_seed(23)
    for group, tokens, capacity in ((4, 3, 0), (4, 8, 0), (4, 16, LARGE), (4, 64, LARGE)):
        cache = _cache(device, gen, lengths=[300, 40], room=70, capacity=capacity)
        counts = [tokens - 1, 1]
        query = _rand(gen, 2, 2 * group, tokens, dtype=BF16)
        clean = paged_attention(query.to(device), cache, softmax_scale=SCALE, counts=_i32(counts, device))
        for b in range(2):
            query[b, :, counts[b]:] = float("nan")
        got = paged_attention(query.to(device), cache, softmax_scale=SCALE, counts=_i32(counts, device))
        torch.cuda.synchronize()
        assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1]) and not got[0].isnan().any()
