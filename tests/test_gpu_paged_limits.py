"""Paged KV cache on the GPU at the limits of its arguments: the largest scores, trees that the caller makes, counts that
change, commits through the C entry, workspaces of mixed batches, far places."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from community_kv_amd import paged_attention
from oracle import paged as op
from tests.test_gpu_paged import BF16, D, F16, HALF_STEP, LARGE, SCALE, _cache, _host

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
