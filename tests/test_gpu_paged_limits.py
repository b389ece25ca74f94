"""Paged KV cache on the GPU at the limits of its arguments: the largest scores, trees that the caller makes, counts that
change, commits through the C entry, workspaces of mixed batches, far places."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from community_kv_amd import DraftTree, PagedKVCache, RotaryTable, paged_append, paged_attention
from community_kv_amd import _native as nat
from oracle import paged as op
from tests.test_gpu_paged import BF16, D, F16, HALF_STEP, LARGE, SCALE, _cache, _host, _i32, _parents

pytestmark = pytest.mark.gpu

FORMS = [(2, 3, 0), (4, 6, 0), (4, 16, 0), (4, 32, LARGE), (4, 70, LARGE), (8, 40, LARGE)]  # group, tokens, capacity


# ------------------------------------------------------------------------------------------ scores

def _whole_numbers(device, gen, *, group, tokens, capacity, dtype, size):
    """Keys and queries of whole numbers times `size`, a power of two: every product q . k is exact in 32 bits."""
    cache = _cache(device, gen, lengths=[700, 5, 1500], room=tokens, page=64, capacity=capacity, dtype=dtype)
    cache.key_pages.copy_(torch.randint(-2, 3, cache.key_pages.shape, generator=gen) * size)
    query = torch.randint(-2, 3, (3, 2 * group, tokens, D), generator=gen).to(dtype) * size
    return cache, query


def _best_rows(cache, query, scale):
    """Outputs and log-sums where neighbouring scores are far apart: the mean of the values of the best rows, and the
    best score plus the log of their number.  A probability is 1 for the best rows and 0 for the others, so what is
    rounded is the sum of the values in 32 bits (some of 2^-24 a row), the division, and the result to its type."""
    state = op.Paged.of(cache)
    batch, hq, tokens, _ = query.shape
    group = hq // cache.kv_heads
    q = _host(query)
    out, size, lse = np.zeros((batch, tokens, hq, D)), np.zeros((batch, tokens, hq, D)), np.zeros((batch, hq, tokens))
    for b in range(batch):
        places = np.array([state.place(b, r) for r in range(int(state.lengths[b]) + tokens)])
        for h in range(hq):
            k, v = (t[0, places[:, 0], h // group, places[:, 1]] for t in (state.keys, state.values))
            for t in range(tokens):
                s = k[:int(state.lengths[b]) + t + 1] @ q[b, h, t]
                best = np.flatnonzero(s == s.max())
                out[b, t, h], size[b, t, h] = v[best].mean(0), np.abs(v[best]).mean(0)
                lse[b, h, t] = s.max() * scale + np.log(len(best))
    return out, size, lse


def _check_best_rows(cache, query, scale):
    out, lse = paged_attention(query.to(cache.device), cache, softmax_scale=scale)
    torch.cuda.synchronize()
    want, size, want_lse = _best_rows(cache, query, scale)
    got, got_lse = _host(out), _host(lse)
    off = np.abs(got - want) - (HALF_STEP[cache.dtype] * np.abs(want) + 2.0 ** -25 + 32 * op.U * size)
    assert (off <= 0).all(), float(np.nanmax(off))
    with np.errstate(over="ignore"):
        beyond = ~np.isfinite(want_lse.astype(np.float32))
    assert np.array_equal(got_lse[beyond], np.sign(want_lse[beyond]) * np.inf)
    # the scale, its log2 e, the product, the sum and ln 2 are rounded to 32 bits: 2^-24 each
    assert (np.abs(got_lse - want_lse)[~beyond] <= (8 * op.U * (np.abs(want_lse) + 8))[~beyond]).all()


@pytest.mark.parametrize("group,tokens,capacity", FORMS)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("scale", [1e3, 1e6, 1e10, 1e30])
def test_attend_largest_scales(device, group, tokens, capacity, dtype, scale):
    """Scores up to the scale times 500, at least the scale apart: the best rows take all, none are lost."""
    print(f"largest scales {group} x {tokens} capacity={capacity} {dtype} {scale}", flush=True)
    gen = torch.Generator().manual_seed(tokens)
    _check_best_rows(*_whole_numbers(device, gen, group=group, tokens=tokens, capacity=capacity, dtype=dtype, size=1.0), scale)


@pytest.mark.parametrize("group,tokens,capacity", FORMS)
@pytest.mark.parametrize("dtype,size,scale", [(BF16, 2.0 ** 20, SCALE), (F16, 2.0 ** 13, SCALE), (BF16, 2.0 ** 50, 1e30)])
def test_attend_largest_products(device, group, tokens, capacity, dtype, size, scale):
    """Large keys and queries under an ordinary scale; products whose scores are beyond 32 bits though they are not:
    their order decides all the same."""
    print(f"largest products {group} x {tokens} capacity={capacity} {dtype} {size} {scale}", flush=True)
    gen = torch.Generator().manual_seed(tokens)
    _check_best_rows(*_whole_numbers(device, gen, group=group, tokens=tokens, capacity=capacity, dtype=dtype, size=size), scale)


@pytest.mark.parametrize("group,tokens,capacity", FORMS)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attend_far_scores_beside_ordinary_ones(device, group, tokens, capacity, dtype):
    """One query head of far larger scores leaves the others' results as they are, to the bit."""
    print(f"far scores {group} x {tokens} capacity={capacity} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(tokens)
    cache, query = _whole_numbers(device, gen, group=group, tokens=tokens, capacity=capacity, dtype=dtype, size=1.0)
    a = paged_attention(query.to(device), cache, softmax_scale=SCALE)
    query[:, 1] *= 2.0 ** 13
    b = paged_attention(query.to(device), cache, softmax_scale=SCALE)
    torch.cuda.synchronize()
    rest = [h for h in range(query.shape[1]) if h != 1]
    assert torch.equal(a[0][:, :, rest], b[0][:, :, rest]) and torch.equal(a[1][:, rest], b[1][:, rest])
    want, size, _ = _best_rows(cache, query, SCALE)
    off = np.abs(_host(b[0]) - want)[:, :, 1] - (HALF_STEP[dtype] * np.abs(want) + 2.0 ** -25 + 32 * op.U * size)[:, :, 1]
    assert (off <= 0).all()


# ------------------------------------------------------------------------------------------ trees that the caller makes

class _Given(op.Paged):
    """The oracle over given (depths, kin) of every sequence in the place of parents."""

    @staticmethod
    def _steps(tokens, trees, counts, b):
        count = tokens if counts is None else min(max(int(counts[b]), 0), tokens)
        depths, kin = trees[b]
        return [min(max(d, 0), 2 ** 30 - 1) for d in depths[:count]], [[j for j in k if j < count] for k in kin[:count]]


def _given_tree(gen, device, batch, tokens, order, counts=None):
    """Depths and masks in orders that no plan makes."""
    trees = []
    for _ in range(batch):
        if order == "backwards":  # a chain whose last token comes first
            depths = list(range(tokens - 1, -1, -1))
            kin = [list(range(t, tokens)) for t in range(tokens)]
        else:
            most = {"near": 2, "far": 3 * tokens + 40, "limits": 1}[order]
            depths = torch.randint(0, most, (tokens,), generator=gen).tolist()
            if order == "limits":
                depths = [(-5, 0, 2 ** 31 - 1, 2 ** 30 - 1, -2 ** 31)[t % 5] for t in range(tokens)]
            kin = [sorted(torch.randperm(tokens, generator=gen)[:int(torch.randint(0, tokens + 1, (1,), generator=gen))].tolist())
                   for _ in range(tokens)]
            kin = [sorted(set(k) | {t}) if t % 3 else k for t, k in enumerate(kin)]  # some do not see themselves
        trees.append((depths, kin))
    masks = np.zeros((batch, tokens, -(-tokens // 64)), np.uint64)
    for b, (_, kin) in enumerate(trees):
        for t, k in enumerate(kin):
            for j in k:
                masks[b, t, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    tree = DraftTree(_i32([d for d, _ in trees], device), torch.from_numpy(masks.view(np.int64)).to(device),
                     None if counts is None else _i32(counts, device))
    return tree, trees


@pytest.mark.parametrize("group,tokens,capacity", [(2, 2, 0), (1, 9, 0), (4, 7, 0), (4, 9, LARGE), (4, 40, LARGE), (2, 130, LARGE),
                                                   (1, 200, 0)])
@pytest.mark.parametrize("order", ["backwards", "near", "far", "limits"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attend_given_trees(device, group, tokens, capacity, order, dtype):
    """A window goes by positions, a draft row's by its depth: trees listed from their ends, depths beyond the tokens'
    number, equal ones, negative ones and ones near 2^31."""
    gen = torch.Generator().manual_seed(tokens)
    cache = _cache(device, gen, lengths=[300, 0, 65], room=tokens, page=32, dtype=dtype, capacity=capacity)
    query = torch.randn(3, 2 * group, tokens, D, generator=gen).to(dtype)
    for counts, window in ((None, 0), (None, 1), (None, 2), ([tokens, 2, tokens - 1], 6), (None, tokens + 20), (None, 3 * tokens + 90)):
        print(f"given tree {order} {group} x {tokens} capacity={capacity} window={window} counts={counts}", flush=True)
        tree, trees = _given_tree(gen, device, 3, tokens, order, counts)
        out, lse = paged_attention(query.to(device), cache, softmax_scale=SCALE, tree=tree, window=window)
        torch.cuda.synchronize()
        want, tol = _Given.of(cache).attend(0, _host(query), scale=SCALE, parents=trees, counts=counts, window=window,
                                            half_step=HALF_STEP[dtype])
        live = ~np.isneginf(want[1])
        assert np.array_equal(~np.isneginf(_host(lse)), live)
        assert (np.abs(_host(lse)[live] - want[1][live]) <= tol[1][live]).all()
        assert (np.abs(_host(out) - want[0]) <= tol[0]).all()


@pytest.mark.parametrize("group,tokens,capacity", [(4, 7, 0), (4, 40, LARGE), (8, 40, LARGE)])
def test_given_trees_keep_special_values_out(device, group, tokens, capacity):
    """Values that are not finite in committed rows before every query's window, where depths are far beyond the tokens'
    number: not seen, so no trace of them."""
    gen = torch.Generator().manual_seed(31)
    cache = _cache(device, gen, lengths=[300], heads=1, room=tokens, page=16, capacity=capacity)
    query = torch.randn(1, group, tokens, D, generator=gen).to(device, BF16)
    masks = torch.full((1, tokens, 1), (1 << tokens) - 1, dtype=torch.int64, device=device)
    tree = DraftTree(torch.full((1, tokens), 250, dtype=torch.int32, device=device), masks)
    window = 300  # positions 251 to 550: rows up to 250 are out of it
    clean = paged_attention(query, cache, softmax_scale=SCALE, tree=tree, window=window)
    for r in range(251):
        cache.value_pages[0, cache.page_table[0, r // 16], 0, r % 16] = float("nan")
        cache.key_pages[0, cache.page_table[0, r // 16], 0, r % 16] = float("inf")
    got = paged_attention(query, cache, softmax_scale=SCALE, tree=tree, window=window)
    torch.cuda.synchronize()
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])


@pytest.mark.parametrize("order", ["backwards", "near", "far", "limits"])
def test_append_given_trees(device, order):
    """Keys and queries turn by their depth, whatever it is; past the table's end by its last position."""
    gen = torch.Generator().manual_seed(32)
    batch, heads, tokens = 2, 2, 19
    cache = _cache(device, gen, lengths=[60, 3], room=tokens + 120)
    table = RotaryTable.from_frequencies((1e4 ** -(torch.arange(32) / 32)).double().to(device), cache.capacity)
    key, value, query = (torch.randn(batch, n, tokens, D, generator=gen) for n in (heads, heads, 4))
    tree, trees = _given_tree(gen, device, batch, tokens, order)
    oracle = _Given.of(cache)
    got = paged_append(cache, key.to(device), value.to(device), query=query.to(device), rotary=table, tree=tree)
    torch.cuda.synchronize()
    turned, written = oracle.append(0, _host(key), _host(value), _host(query), (_host(table.cosines), _host(table.sines)), False, trees)
    size = 2.0 ** -8 * np.abs(turned) + 8 * op.U * float(query.abs().max()) + 2.0 ** -25
    assert (np.abs(_host(got) - turned) <= size).all()
    off = np.abs(_host(cache.key_pages) - oracle.keys)[0]
    assert (off <= 2.0 ** -8 * np.abs(oracle.keys[0]) + 8 * op.U * float(key.abs().max()) + 2.0 ** -25)[written].all()


def test_a_tree_keeps_its_counts(device):
    """Parents and counts that are used again before the last layer leave the tree as it was planned."""
    gen = torch.Generator().manual_seed(33)
    tokens, given = 9, [9, 0, 4, 30, -2]
    cache = _cache(device, gen, lengths=[40, 7, 90, 20, 3], room=tokens)
    parents = _parents(gen, 5, tokens, "wide").to(device)
    query = torch.randn(5, 4, tokens, D, generator=gen).to(device, BF16)
    for counts in (_i32(given, device), _i32([x for x in given for _ in range(2)], device)[::2]):
        tree = DraftTree.from_parents(parents, counts=counts)
        before = paged_attention(query, cache, softmax_scale=SCALE, tree=tree)
        counts.fill_(2)
        parents_before = parents.clone()
        parents.zero_()
        after = paged_attention(query, cache, softmax_scale=SCALE, tree=tree)
        pages = cache.key_pages.clone()
        paged_append(cache, query[:, :2], query[:, 2:], tree=tree)
        torch.cuda.synchronize()
        assert tree.counts.tolist() == [9, 0, 4, 9, 0]
        assert torch.equal(before[0], after[0]) and torch.equal(before[1], after[1])
        changed = (cache.key_pages != pages).any(-1).sum().item()
        assert changed == 2 * sum(tree.counts.tolist())  # rows of both heads
        parents.copy_(parents_before)
        cache.key_pages.copy_(pages)
    assert DraftTree.from_parents(parents).counts is None


# ------------------------------------------------------------------------------------------ commits through the C entry

@pytest.mark.parametrize("counts", [None, [1, 3, 0], [9, -1, 4]])
@pytest.mark.parametrize("tokens", [0, 2, 4, 2 ** 31 - 1])
@pytest.mark.parametrize("with_path", [False, True])
def test_commit_c_entry_counts(device, counts, tokens, with_path):
    """`tokens` of every sequence where counts is null, with a path too (whose padding ascends); counts alone otherwise."""
    gen = torch.Generator().manual_seed(34)
    cache = _cache(device, gen, lengths=[10, 0, 33], room=20, layers=2)
    path = [[0, 2, 5, 7], [1, 2, 3, 9], [3, 4, 5, 6]] if with_path else None
    oracle = op.Paged.of(cache)
    path_t, counts_t = (None if x is None else _i32(x, device) for x in (path, counts))
    rc = nat.lib().ckv_paged_commit(cache._ref, tokens, None if counts is None else counts_t.data_ptr(),
                                    path_t.data_ptr() if with_path else None, 4 if with_path else 0,
                                    torch.cuda.current_stream(device).cuda_stream)
    torch.cuda.synchronize()
    assert rc == 0
    oracle.commit([tokens] * 3 if counts is None else counts, path)
    assert np.array_equal(cache.lengths.cpu().numpy(), oracle.lengths)
    assert np.array_equal(_host(cache.key_pages), oracle.keys) and np.array_equal(_host(cache.value_pages), oracle.values)


# ------------------------------------------------------------------------------------------ workspaces

@pytest.mark.parametrize("batch,heads,group,tokens,long", [(70, 4, 1, 1, [5]), (70, 4, 1, 1, [0, 33, 64, 69]), (40, 8, 3, 9, [1, 39]),
                                                           (18, 8, 2, 65, [17]), (18, 8, 2, 65, [0, 9]), (18, 2, 4, 130, [3, 4, 5, 6, 7]),
                                                           (3, 2, 4, 70, [0, 1, 2]), (3, 2, 1, 1, [0, 2])])
def test_workspace_of_mixed_batches(device, batch, heads, group, tokens, long):
    """Sequences that are cut among ones that are not: results as the oracle's, nothing behind the workspace written."""
    print(f"mixed batch {batch} {heads} x {group} x {tokens} long={long}", flush=True)
    gen = torch.Generator().manual_seed(batch + tokens)
    lengths = [int(x) for x in torch.randint(0, 60, (batch,), generator=gen)]
    for i, b in enumerate(long):
        lengths[b] = 3000 - 700 * i
    cache = _cache(device, gen, lengths=lengths, heads=heads, room=tokens, page=32, capacity=8192)
    query = torch.randn(batch, heads * group, tokens, D, generator=gen).to(BF16)
    on = query.to(device)
    size = nat.lib().ckv_paged_attention_workspace_bytes(cache._ref, heads * group, tokens, 0)
    assert size > 0
    out = torch.empty(batch, tokens, heads * group, D, dtype=BF16, device=device)
    lse = torch.empty(batch, heads * group, tokens, device=device)
    workspace = torch.full((size + 65536,), 0x5A, dtype=torch.uint8, device=device)
    args = nat.PAGED_ATTENTION_ARGS.pack(on.data_ptr(), *on.stride()[:3], 0, 0, out.data_ptr(), lse.data_ptr(), workspace.data_ptr(),
                                         0, heads * group, tokens, 0, SCALE, 0)
    assert nat.lib().ckv_paged_attention(cache._ref, args, torch.cuda.current_stream(device).cuda_stream) == 0
    torch.cuda.synchronize()
    assert bool((workspace[size:] == 0x5A).all())
    want, tol = op.Paged.of(cache).attend(0, _host(query), scale=SCALE)
    assert (np.abs(_host(lse) - want[1]) <= tol[1]).all() and (np.abs(_host(out) - want[0]) <= tol[0]).all()


# ------------------------------------------------------------------------------------------ far places

@pytest.mark.parametrize("dtype", [BF16, F16])
def test_far_rows_weigh_what_they_should(device, dtype):
    """Nine million rows of key 0 in pages up to beyond 2^32 elements weigh 1 each; a few keys far apart, and the step's own
    token, weigh e^16 each, about as much as all of the others together: each part of the sum shows in the result.

    A lane adds at most 2^15 terms of a part, each with half a step of a sum below 2: 2^-24.  So its share, and with it the
    sum, is off by at most 2^-9 of itself, and twice that where a probability next to a larger one is rounded too."""
    print(f"far rows {dtype}", flush=True)
    gen = torch.Generator().manual_seed(35)
    pages, heads = 140_000, 2  # 2.3 G elements a layer
    cache = PagedKVCache.allocate(layers=2, batch=1, kv_heads=heads, capacity=pages * 64, page_size=64, dtype=dtype, device=device)
    cache.page_table.copy_(cache.page_table.flip(1).clone())
    n = pages * 64 - 3
    cache.lengths.fill_(n)
    far = [0, 77, 64 * 9_000 + 5, 64 * 70_000, 64 * 130_001 + 63, n - 1]  # pages 139,999 to 0
    assert ((2 * pages - 1) * heads * 64 * D) > 2 ** 32
    value = torch.randn(heads, len(far) + 1, D, generator=gen).to(dtype)
    key = torch.zeros(heads, 1, D, dtype=dtype)
    key[..., 0] = 16.0
    for layer in range(2):
        for i, r in enumerate(far):
            page, at = int(cache.page_table[0, r // 64]), r % 64
            cache.key_pages[layer, page, :, at, 0] = 16.0 if layer else -3.0  # the other layer's rows are others
            cache.value_pages[layer, page, :, at] = value[:, i].to(device)
    paged_append(cache, key[None].to(device), value[None, :, -1:].to(device), layer=1)
    query = torch.zeros(1, heads, 40, D, dtype=dtype, device=device)
    query[..., 0] = 1.0
    rows = n - len(far)
    z = rows + (len(far) + 1) * np.exp(16.0)
    want = np.exp(16.0) / z * _host(value).sum(1)
    size = np.exp(16.0) / z * np.abs(_host(value)).sum(1)
    for tokens in (1, 40):  # few query rows, many
        out, lse = paged_attention(query[:, :, :tokens], cache, layer=1, softmax_scale=1.0, counts=_i32([1], device))
        torch.cuda.synchronize()
        assert (np.abs(_host(lse)[0, :, 0] - np.log(z)) <= 2.0 ** -8).all()
        assert (np.abs(_host(out)[0, 0] - want) <= (2.0 ** -8 + 2 * HALF_STEP[dtype]) * size + 2.0 ** -25).all()
        assert not out[0, 1:].any() and bool(lse[0, :, 1:].isneginf().all())
