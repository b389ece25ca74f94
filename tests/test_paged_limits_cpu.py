"""Paged KV cache without a GPU: workspace sizes, refusals of gradients."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from community_kv_amd import PagedKVCache, RotaryTable, paged_append, paged_attention
from tests.test_paged_cpu import _c_cache, _cache, _table, _tensors, lib  # noqa: F401 (a fixture)


@pytest.mark.parametrize("batch,heads,query_heads,tokens,pages", [(64, 8, 32, 512, 64), (64, 8, 32, 512, 128), (64, 8, 32, 1, 2048),
                                                                  (24, 8, 32, 64, 256), (200, 1, 1, 1, 128)])
def test_workspace_holds_the_parts_of_cut_sequences_alone(lib, batch, heads, query_heads, tokens, pages):  # noqa: F811
    """Parts are cut for 512 workgroups (one token) or 256, or a batch that fills the chip gets batch / 2 more than
    sequences at most, none over 32 units of 128 rows or fewer.  Each of the parts above the sequences cuts one more of them at
    most, so twice as many have 32-bit outputs and two sums a query row."""
    c = _c_cache(lib, batch=batch, kv_heads=heads, table_pages=pages, page_size=64)
    rows = (tokens * (query_heads // heads) + 15) // 16 * 16
    blocks = -(-rows // 256) if rows > 32 else 1
    want = (512 if rows == 16 else 256) // (heads * blocks)
    if want >= (2 * batch if rows > 32 else batch + 1):  # the kernel of many query rows is cut later
        parts = want
    else:
        parts = batch + (min(want, batch // 2) if pages * 64 > 32 * 128 else 0)
    slots = min(parts, 2 * (parts - batch))
    size = lib.ckv_paged_attention_workspace_bytes(c, query_heads, tokens, 0)
    assert (size > 0) == (slots > 0) and size <= slots * heads * rows * (128 + 2) * 4 + 8 * batch + 64


def test_tangents_are_refused():
    """Forward-mode derivatives would be lost: every tensor that goes into the result is looked at; others pass."""
    cache, x, q = _cache(dtype=torch.float16), torch.zeros(2, 2, 3, 128, dtype=torch.float16), torch.zeros(2, 4, 3, 128, dtype=torch.float16)
    with forward_ad.dual_level():
        x_dual, q_dual = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, q))
        table = _table()
        dual_table = RotaryTable(forward_ad.make_dual(table.cosines, table.sines), table.sines)
        dual_pages = PagedKVCache(**(_tensors(cache) | dict(value_pages=forward_ad.make_dual(cache.value_pages,
                                                                                            torch.ones_like(cache.value_pages)))))
        for call in (lambda: paged_append(cache, x_dual, x), lambda: paged_append(cache, x, x_dual),
                     lambda: paged_append(cache, x, x, query=q_dual, rotary=table),
                     lambda: paged_append(cache, x, x, query=q, rotary=dual_table), lambda: paged_append(dual_pages, x, x),
                     lambda: paged_attention(q_dual, cache, softmax_scale=1.0),
                     lambda: paged_attention(q, dual_pages, softmax_scale=1.0)):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
                call()
        for call in (lambda: paged_append(cache, x, x, query=q, rotary=table), lambda: paged_attention(q, cache, softmax_scale=1.0)):
            with pytest.raises(RuntimeError, match="GPU"):
                call()


@pytest.mark.parametrize("name", ["key_pages", "value_pages"])
def test_pages_that_require_a_gradient_are_refused(name):
    """They are written in place, past autograd; under no_grad nobody asks for one."""
    good = _tensors(_cache())
    good[name] = torch.zeros_like(good[name]).requires_grad_()
    with pytest.raises(RuntimeError, match="gradient"):
        PagedKVCache(**good)
    with torch.no_grad():
        PagedKVCache(**good)


def test_rotation_tables_that_require_a_gradient_are_refused():
    angles = torch.rand(128, 64)
    for cosines, sines in ((angles.clone().requires_grad_(), angles), (angles, angles.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="gradient"):
            RotaryTable(cosines, sines)
        with torch.no_grad():
            RotaryTable(cosines, sines)
    frequencies = torch.rand(16).requires_grad_()
    with pytest.raises(RuntimeError, match="gradient"):
        RotaryTable.from_frequencies(frequencies, 10)
    with torch.no_grad():
        assert RotaryTable.from_frequencies(frequencies, 10).positions == 10
