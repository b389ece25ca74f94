"""Paged KV cache and drafted trees: refusals, layouts and the oracle's own rules, without a GPU."""

from __future__ import annotations

import ctypes
import os

import numpy as np
import pytest
import torch

from community_kv_amd import DraftTree, PagedKVCache, RotaryTable, paged_append, paged_attention, paged_commit
from community_kv_amd import _native as nat
from oracle import paged as op

BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(nat.LIB_PATH):
        nat.build()
    return nat.lib()


def _cache(**kwargs):
    return PagedKVCache.allocate(**dict(dict(layers=2, batch=2, kv_heads=2, capacity=100, page_size=32, device="cpu"), **kwargs))


def _tensors(cache):
    return dict(key_pages=cache.key_pages, value_pages=cache.value_pages, page_table=cache.page_table, lengths=cache.lengths)


def _table(positions=128, half=64):
    return RotaryTable(torch.ones(positions, half), torch.zeros(positions, half))


def _tree(batch=2, tokens=3):
    return DraftTree(torch.zeros(batch, tokens, dtype=torch.int32), torch.zeros(batch, tokens, -(-tokens // 64), dtype=torch.int64))


def test_allocate_layout():
    cache = _cache()
    assert (cache.layers, cache.batch, cache.kv_heads, cache.page_size, cache.capacity) == (2, 2, 2, 32, 128)
    assert cache.pages == 8 and cache.key_pages.shape == (2, 8, 2, 32, 128) and cache.dtype == BF16
    assert cache.page_table.tolist() == [[0, 1, 2, 3], [4, 5, 6, 7]] and cache.lengths.tolist() == [0, 0]
    pool = _cache(pages=5, dtype=F16)
    assert pool.pages == 5 and pool.dtype == F16 and bool((pool.page_table == -1).all())
    cache.assert_no_overflow()
    cache.overflow[1] = 1
    with pytest.raises(RuntimeError, match="overflow"):
        cache.assert_no_overflow()


@pytest.mark.parametrize("change", [dict(layers=0), dict(batch=0), dict(kv_heads=0), dict(capacity=0), dict(pages=0),
                                    dict(page_size=8), dict(page_size=48), dict(page_size=512)])
def test_allocate_refuses(change):
    with pytest.raises(ValueError):
        _cache(**change)


@pytest.mark.parametrize("name,value,error", [
    ("key_pages", torch.zeros(2, 8, 2, 32, 64, dtype=BF16), ValueError),
    ("key_pages", torch.zeros(8, 2, 32, 128, dtype=BF16), ValueError),
    ("key_pages", torch.zeros(2, 8, 2, 32, 128), TypeError),
    ("key_pages", torch.zeros(2, 0, 2, 32, 128, dtype=BF16), ValueError),
    ("key_pages", torch.zeros(2, 8, 2, 24, 128, dtype=BF16), ValueError),
    ("value_pages", torch.zeros(2, 8, 2, 32, 128, dtype=F16), TypeError),
    ("value_pages", torch.zeros(2, 7, 2, 32, 128, dtype=BF16), ValueError),
    ("value_pages", torch.zeros(2, 8, 32, 2, 128, dtype=BF16).transpose(2, 3), ValueError),
    ("value_pages", torch.zeros(2 * 8 * 2 * 32 * 128 + 1, dtype=BF16)[1:].view(2, 8, 2, 32, 128), ValueError),
    ("page_table", torch.zeros(2, 4, dtype=torch.int64), TypeError),
    ("page_table", torch.zeros(8, dtype=torch.int32), ValueError),
    ("page_table", torch.zeros(2, 0, dtype=torch.int32), ValueError),
    ("page_table", torch.zeros(4, 2, dtype=torch.int32).t(), ValueError),
    ("lengths", torch.zeros(3, dtype=torch.int32), ValueError),
    ("lengths", torch.zeros(2), TypeError),
    ("lengths", torch.zeros(4, dtype=torch.int32)[::2], ValueError)])
def test_cache_refuses(name, value, error):
    good = _tensors(_cache())
    PagedKVCache(**good)
    with pytest.raises(error):
        PagedKVCache(**(good | {name: value}))


def test_cache_refuses_shared_memory_and_too_many_rows():
    good = _tensors(_cache())
    with pytest.raises(ValueError, match="share"):
        PagedKVCache(**(good | dict(value_pages=good["key_pages"])))
    both = torch.zeros(6, dtype=torch.int32)
    with pytest.raises(ValueError, match="share"):
        PagedKVCache(**(good | dict(page_table=both[:4].view(2, 2), lengths=both[2:4])))
    table = torch.zeros(1, (1 << 25) + 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="rows"):
        PagedKVCache(**(good | dict(page_table=table, lengths=torch.zeros(1, dtype=torch.int32))))
    with pytest.raises(ValueError, match="65535"):
        PagedKVCache(**(good | dict(page_table=torch.zeros(32768, 1, dtype=torch.int32),
                                    lengths=torch.zeros(32768, dtype=torch.int32))))


def test_rotary_table():
    table = RotaryTable.from_frequencies(10000.0 ** -(torch.arange(32) / 32), 50, interleaved=True, scale=1.5)
    assert table.positions == 50 and table.cosines.shape == (50, 32) and table.interleaved
    want = 49 * 10000.0 ** -(np.float32(np.arange(32) / 32)).astype(np.float64)
    assert np.abs(table.sines[49].double().numpy() - 1.5 * np.sin(want)).max() < 49 * 2.0 ** -23
    far = RotaryTable.from_frequencies(torch.full((8,), 0.75), 1 << 21)
    at = (1 << 21) - 1  # an angle of a million and a half, whose 32-bit product would be off by up to 0.06
    assert abs(float(far.cosines[at, 0]) - np.cos(0.75 * at)) < 2.0 ** -23


@pytest.mark.parametrize("cosines,sines,error", [
    (torch.zeros(0, 8), torch.zeros(0, 8), ValueError), (torch.zeros(9), torch.zeros(9), ValueError),
    (torch.zeros(9, 12), torch.zeros(9, 12), ValueError), (torch.zeros(9, 72), torch.zeros(9, 72), ValueError),
    (torch.zeros(9, 8), torch.zeros(9, 16), ValueError), (torch.zeros(9, 8), torch.zeros(9, 8).double(), TypeError),
    (torch.zeros(9, 8), torch.zeros(8, 9).t(), ValueError)])
def test_rotary_table_refuses(cosines, sines, error):
    with pytest.raises(error):
        RotaryTable(cosines, sines)


def test_rotary_frequencies_refuse():
    for args in ((torch.zeros(2, 8), 4), (torch.zeros(8), 0)):
        with pytest.raises(ValueError):
            RotaryTable.from_frequencies(*args)


def test_tree_refuses():
    good = torch.zeros(2, 3, dtype=torch.int32)
    for parents, kwargs, error in (
            (good.long(), {}, TypeError), (good[0], {}, ValueError), (good[:, :0], {}, ValueError),
            (torch.zeros(1, 513, dtype=torch.int32), {}, ValueError), (good, dict(counts=torch.zeros(2)), TypeError),
            (good, dict(counts=torch.zeros(3, dtype=torch.int32)), TypeError), (good, {}, RuntimeError)):
        with pytest.raises(error):
            DraftTree.from_parents(parents, **kwargs)
    masks = torch.zeros(2, 3, 1, dtype=torch.int64)
    assert DraftTree(good, masks).tokens == 3
    for depths, mask, counts, error in ((good.long(), masks, None, TypeError), (good[0], masks, None, ValueError),
                                        (good, masks[:, :, :0], None, ValueError), (good, masks.int(), None, TypeError),
                                        (good, masks, torch.zeros(2), TypeError), (good.t(), masks, None, ValueError),
                                        (torch.zeros(1, 513, dtype=torch.int32), torch.zeros(1, 513, 9, dtype=torch.int64),
                                         None, ValueError)):
        with pytest.raises(error):
            DraftTree(depths, mask, counts)


def test_append_refuses():
    cache, x = _cache(), torch.zeros(2, 2, 3, 128)
    q = torch.zeros(2, 4, 3, 128)
    for error, call in (
            (TypeError, lambda: paged_append(cache, x.double(), x.double())),
            (TypeError, lambda: paged_append(cache, x, x.half())),
            (ValueError, lambda: paged_append(cache, x[:1], x[:1])),
            (ValueError, lambda: paged_append(cache, x[:, :1], x[:, :1])),
            (ValueError, lambda: paged_append(cache, x, x[:, :, :2])),
            (ValueError, lambda: paged_append(cache, x[..., :64], x[..., :64])),
            (ValueError, lambda: paged_append(cache, x[0], x[0])),
            (ValueError, lambda: paged_append(cache, x, x, layer=2)),
            (ValueError, lambda: paged_append(cache, x, x, layer=-1)),
            (RuntimeError, lambda: paged_append(cache, x.clone().requires_grad_(), x)),
            (RuntimeError, lambda: paged_append(cache, x, x.clone().requires_grad_())),
            (TypeError, lambda: paged_append(cache, x, x, counts=torch.tensor([1, 2]))),
            (TypeError, lambda: paged_append(cache, x, x, counts=torch.tensor([1], dtype=torch.int32))),
            (ValueError, lambda: paged_append(cache, x, x, query=q)),
            (TypeError, lambda: paged_append(cache, x, x, query=q.half(), rotary=_table())),
            (ValueError, lambda: paged_append(cache, x, x, query=q[:, :, :2], rotary=_table())),
            (ValueError, lambda: paged_append(cache, x, x, query=q[:, :0], rotary=_table())),
            (ValueError, lambda: paged_append(cache, x, x, rotary=_table(127))),
            (ValueError, lambda: paged_append(cache, x, x, tree=_tree(2, 4))),
            (ValueError, lambda: paged_append(cache, x, x, tree=_tree(1, 3))),
            (ValueError, lambda: paged_append(cache, x, x, tree=_tree(), counts=torch.zeros(2, dtype=torch.int32))),
            (RuntimeError, lambda: paged_append(cache, x, x, query=q, rotary=_table()))):  # on the CPU
        with pytest.raises(error):
            call()


def test_attention_refuses():
    cache, q = _cache(), torch.zeros(2, 4, 3, 128, dtype=BF16)
    for error, call in (
            (TypeError, lambda: paged_attention(q.half(), cache, softmax_scale=1.0)),
            (TypeError, lambda: paged_attention(q.float(), cache, softmax_scale=1.0)),
            (ValueError, lambda: paged_attention(q[:, :3], cache, softmax_scale=1.0)),
            (ValueError, lambda: paged_attention(q[:, :0], cache, softmax_scale=1.0)),
            (ValueError, lambda: paged_attention(torch.zeros(2, 34, 1, 128, dtype=BF16), cache, softmax_scale=1.0)),
            (ValueError, lambda: paged_attention(q[:1], cache, softmax_scale=1.0)),
            (ValueError, lambda: paged_attention(q[..., :64], cache, softmax_scale=1.0)),
            (ValueError, lambda: paged_attention(q, cache, softmax_scale=1.0, layer=2)),
            (ValueError, lambda: paged_attention(q, cache, softmax_scale=0.0)),
            (ValueError, lambda: paged_attention(q, cache, softmax_scale=1e-38)),
            (ValueError, lambda: paged_attention(q, cache, softmax_scale=float("nan"))),
            (ValueError, lambda: paged_attention(q, cache, softmax_scale=float("inf"))),
            (ValueError, lambda: paged_attention(q, cache, softmax_scale=1.0, window=-1)),
            (ValueError, lambda: paged_attention(q, cache, softmax_scale=1.0, tree=_tree(2, 2))),
            (ValueError, lambda: paged_attention(q, cache, softmax_scale=1.0, tree=_tree(), counts=torch.zeros(2, dtype=torch.int32))),
            (TypeError, lambda: paged_attention(q, cache, softmax_scale=1.0, counts=torch.zeros(2))),
            (RuntimeError, lambda: paged_attention(q.clone().requires_grad_(), cache, softmax_scale=1.0)),
            (RuntimeError, lambda: paged_attention(q, cache, softmax_scale=1.0))):  # on the CPU
        with pytest.raises(error):
            call()


def test_commit_refuses():
    cache = _cache()
    path = torch.zeros(2, 3, dtype=torch.int32)
    for error, call in (
            (ValueError, lambda: paged_commit(cache, -1)),
            (TypeError, lambda: paged_commit(cache, torch.zeros(2))),
            (TypeError, lambda: paged_commit(cache, torch.zeros(3, dtype=torch.int32))),
            (TypeError, lambda: paged_commit(cache, 1, path=path.long())),
            (TypeError, lambda: paged_commit(cache, 1, path=path[:1])),
            (TypeError, lambda: paged_commit(cache, 1, path=path[0])),
            (ValueError, lambda: paged_commit(cache, 1, path=path[:, :0])),
            (ValueError, lambda: paged_commit(cache, 1, path=torch.zeros(2, 513, dtype=torch.int32))),
            (RuntimeError, lambda: paged_commit(cache, 1, path=path)),  # on the CPU
            (RuntimeError, lambda: paged_commit(cache, 1))):
        with pytest.raises(error):
            call()
    paged_commit(cache, 0, path=path)  # nothing to take over


def _c_cache(lib, **change):
    c = nat.PagedCache(0x1000, 0x2000, 0x3000, 0x4000, 0x5000, 0x6000, 2, 8, 2, 32, 4, 2, nat.CKV_BF16, 0)
    for name, value in change.items():
        setattr(c, name, value)
    return ctypes.byref(c)


def _rows(address=0x1000, stride=128):
    return (address, stride, stride, stride)


def _append_args(**change):
    args = dict(key=_rows(), value=_rows(), query=_rows(0), counts=0, depths=0, rotary=0, out=0, layer=0, tokens=1, heads=0,
                dtype=nat.CKV_BF16) | change
    return nat.PAGED_APPEND_ARGS.pack(*args.pop("key"), *args.pop("value"), *args.pop("query"), *args.values())


def _attention_args(**change):
    args = dict(query=_rows(), counts=0, tree=0, out=0x1000, lse=0x1000, workspace=0x1000, layer=0, heads=4, tokens=3, window=0,
                scale=1.0, reserved=0) | change
    return nat.PAGED_ATTENTION_ARGS.pack(*args.pop("query"), *args.values())


@pytest.mark.parametrize("change,rc", [
    (dict(key_pages=None), 1), (dict(value_pages=0x2008), 1), (dict(page_table=None), 1), (dict(lengths=None), 1),
    (dict(overflow=None), 1), (dict(counters=None), 1), (dict(layers=0), 1), (dict(pages=0), 1), (dict(kv_heads=-1), 1), (dict(page_size=24), 1),
    (dict(page_size=8), 1), (dict(page_size=512), 1), (dict(table_pages=0), 1), (dict(batch=0), 1), (dict(dtype=nat.CKV_F32), 1),
    (dict(table_pages=(1 << 25) + 1), 2), (dict(batch=32768), 2), (dict(kv_heads=32768), 2),
    (dict(batch=300, kv_heads=300), 2), (dict(batch=16384, table_pages=1 << 25), 2)])
def test_c_entries_refuse_bad_caches(lib, change, rc):
    c = _c_cache(lib, **change)
    for got in (lib.ckv_paged_append(c, _append_args(), None), lib.ckv_paged_attention(c, _attention_args(), None),
                lib.ckv_paged_commit(c, 1, None, None, 0, None)):
        assert got == rc, lib.ckv_last_error()
    assert lib.ckv_paged_attention_workspace_bytes(c, 2, 1, 0) == 0


def test_c_entries_refuse_bad_arguments(lib):
    c = _c_cache(lib)
    tables = []

    def rotary(**change):
        t = nat.Rotary(0x1000, 0x1000, 128, 64, 0, 0)
        for name, value in change.items():
            setattr(t, name, value)
        tables.append(t)
        return ctypes.addressof(t)

    for change in (dict(layer=2), dict(layer=-1), dict(key=_rows(0)), dict(key=_rows(0x1008)), dict(value=_rows(0)),
                   dict(value=_rows(0x1000, 4)), dict(dtype=2), dict(tokens=0), dict(query=_rows()),
                   dict(query=_rows(), heads=4, out=0x1000), dict(query=_rows(), heads=4, rotary=rotary()),
                   dict(query=_rows(), heads=4, rotary=rotary(), out=0x1008),
                   dict(query=_rows(), heads=0, rotary=rotary(), out=0x1000),
                   dict(query=_rows(0x1002), heads=4, rotary=rotary(), out=0x1000),
                   dict(rotary=rotary(cosines=None)), dict(rotary=rotary(sines=0x1004)), dict(rotary=rotary(dim=0)),
                   dict(rotary=rotary(dim=24)), dict(rotary=rotary(dim=144)), dict(rotary=rotary(positions=127))):
        assert lib.ckv_paged_append(c, _append_args(**change), None) == 1, change
    assert lib.ckv_paged_append(c, None, None) == 1 and lib.ckv_paged_attention(c, None, None) == 1
    half, whole = nat.TreeMasks(0x1000, None), nat.TreeMasks(0x1000, 0x1000)
    for change, rc in ((dict(layer=2), 1), (dict(query=_rows(0)), 1), (dict(query=_rows(0x1008)), 1), (dict(heads=3), 1),
                       (dict(heads=0), 1), (dict(heads=34), 2), (dict(tokens=0), 1), (dict(window=-1), 1), (dict(scale=0.0), 1),
                       (dict(scale=float("nan")), 1), (dict(scale=2e30), 1), (dict(scale=1e-31), 1), (dict(out=0), 1), (dict(out=0x1008), 1),
                       (dict(lse=0), 1), (dict(tree=ctypes.addressof(half)), 1), (dict(tokens=(1 << 20) + 1), 2),
                       (dict(tokens=513, tree=ctypes.addressof(whole)), 2)):
        assert lib.ckv_paged_attention(c, _attention_args(**change), None) == rc, change
    large = _c_cache(lib, table_pages=1 << 16)
    for workspace in (0, 0x1008):  # several parts a sequence
        assert lib.ckv_paged_attention_workspace_bytes(large, 4, 1, 0) > 0
        assert lib.ckv_paged_attention(large, _attention_args(tokens=1, workspace=workspace), None) == 1
    for args in ((0, None, None, 1, 0x1000, 0x1000, None), (0x1000, None, 0, 1, 0x1000, 0x1000, None),
                 (0x1000, None, 1, 0, 0x1000, 0x1000, None), (0x1000, None, 1, 1, None, 0x1000, None),
                 (0x1000, None, 1, 1, 0x1000, None, None)):
        args = args if args[0] else (None,) + (None, 1) + args[3:]
        assert lib.ckv_draft_tree_plan(*args) == 1, args
    assert lib.ckv_draft_tree_plan(0x1000, None, 1, 513, 0x1000, 0x1000, None) == 2
    assert lib.ckv_paged_commit(c, -1, None, None, 0, None) == 1
    assert lib.ckv_paged_commit(c, 1, None, 0x1000, 0, None) == 1
    assert lib.ckv_paged_commit(c, 1, None, 0x1000, 513, None) == 2


def test_workspace_is_the_call_s_own_size(lib):
    c = _c_cache(lib, table_pages=1 << 12)
    for heads, tokens, window in ((3, 1, 0), (0, 1, 0), (4, 0, 0), (4, 1, -1), (4, (1 << 20) + 1, 0)):
        assert lib.ckv_paged_attention_workspace_bytes(c, heads, tokens, window) == 0
    one = lib.ckv_paged_attention_workspace_bytes(c, 4, 1, 0)
    # at least the outputs of two parts a sequence, head and (padded) query row
    assert one >= 2 * 2 * 2 * 16 * 128 * 4
    assert lib.ckv_paged_attention_workspace_bytes(c, 4, 1, 100) <= one


# ------------------------------------------------------------------------------------------ the oracle

def test_oracle_plan_by_hand():
    depths, masks = op.plan(np.array([[-1, 0, 0, 1, 9, 4]], np.int32))
    assert depths.tolist() == [[0, 1, 1, 2, 0, 1]]
    assert masks[0, :, 0].tolist() == [0b1, 0b11, 0b101, 0b1011, 0b10000, 0b110000]
    depths, masks = op.plan(np.array([list(range(-1, 69))], np.int32), [66])
    assert depths[0, 65] == 65 and masks[0, 65].tolist() == [-1, 3] and not masks[0, 66:].any()


def test_oracle_run_equals_attention_of_the_kept_tokens():
    """A prompt, a tree and its accepted path against the softmax of the kept tokens in one piece."""
    rng = np.random.default_rng(0)
    table = np.array([[2, 0, 3, 1]], np.int32)
    cache = op.Paged(np.zeros((1, 4, 1, 4, 128)), np.zeros((1, 4, 1, 4, 128)), table, np.zeros(1, np.int32))
    key, value, query = rng.standard_normal((3, 1, 1, 9, 128))
    cache.append(0, key[:, :, :5], value[:, :, :5])
    cache.commit(5)
    parents = np.array([[-1, -1, 0, 1]], np.int32)
    angles = np.arange(16)[:, None] * np.ones(8)
    turned, _ = cache.append(0, key[:, :, 5:], value[:, :, 5:], query[:, :, 5:], (np.cos(angles * 0), np.sin(angles * 0)),
                             parents=parents)
    assert np.array_equal(turned, query[:, :, 5:])
    (out, _), _ = cache.attend(0, turned, scale=0.3, parents=parents)
    cache.commit([2], [[1, 3]])
    kept = [0, 1, 2, 3, 4, 6, 8]
    assert cache.lengths[0] == 7
    k, v = key[0, 0, kept], value[0, 0, kept]
    s = k @ query[0, 0, 8] * 0.3
    p = np.exp(s - s.max())
    assert np.abs(out[0, 3, 0] - p @ v / p.sum()).max() < 1e-12
    again = np.stack([cache.keys[0, table[0, r // 4], 0, r % 4] for r in range(7)])
    assert np.array_equal(again, k)
