"""Performance cases of the paged key/value cache and of drafted tokens over it.

A cache keeps the keys and values of all layers in pages ``[layers, pages, kv_heads, page_size, 128]``; a page table
names the pages of every sequence, and ``lengths`` its committed rows.  A serving program writes the tokens of a step
behind those rows, with the position rotation applied on the way, attends to the cache with the step's queries, and
commits the tokens that it keeps.  The tokens of a step are a prompt (or a piece of one), a single token, or a tree of
drafted tokens, of which one path is kept:

* ``tree``   - ``DraftTree.from_parents``: depths and ancestor masks of drafted tokens from their parents
* ``append`` - ``paged_append``: keys rotated and written into pages with their values, queries rotated
* ``attend`` - ``paged_attention``: attention of the step's tokens over the committed rows and their own ancestors
* ``commit`` - ``paged_commit``: the accepted path's rows moved behind the committed ones, in all layers

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
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
WIDE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # Eight requests' draft trees of one speculative step.
        dict(name="tree_b8_64", kind="tree", batch=8, tokens=64, mix=1, shape="wide", ragged=False),
        # Many requests with wide and deep trees of uneven sizes.
        dict(name="tree_b64_500", kind="tree", batch=64, tokens=500, mix=2, shape="deep", ragged=True),
        # A server's step over eight requests: one token each, at odd lengths, queries rotated with the keys.
        dict(name="append_step_b8", kind="append", batch=8, q_heads=32, kv_heads=8, tokens=1, ctx_min=1001,
             ctx_max=8191, mix=3, page=64, dtype="bf16", store="bf16", shape="chain", ragged=False, layout="heads",
             rotary=128, interleaved=False),
        # A long prompt written in one call into an empty cache, rows as the projections leave them ([token, head]).
        dict(name="append_prompt_32k", kind="append", batch=1, q_heads=32, kv_heads=8, tokens=32768, ctx_min=0,
             ctx_max=0, mix=4, page=64, dtype="bf16", store="bf16", shape="chain", ragged=False, layout="tokens",
             rotary=128, interleaved=False),
        # Draft trees of uneven sizes, 32-bit inputs into an fp16 cache of small pages, half of the dims rotated in pairs.
        dict(name="append_draft_f32", kind="append", batch=5, q_heads=28, kv_heads=4, tokens=61, ctx_min=100,
             ctx_max=1900, mix=5, page=16, dtype="f32", store="f16", shape="wide", ragged=True, layout="tokens",
             rotary=64, interleaved=True),
        # A short chat turn of a small model: latency is all there is.
        dict(name="attend_chat_300", kind="attend", batch=1, q_heads=8, kv_heads=2, tokens=1, ctx_min=300, ctx_max=300,
             mix=6, page=16, dtype="f16", shape="chain", ragged=False, window=0),
        # A server's decode step over eight requests of uneven lengths (16k to 128k).
        dict(name="attend_step_b8_131k", kind="attend", batch=8, q_heads=32, kv_heads=8, tokens=1, ctx_min=16384,
             ctx_max=131071, mix=7, page=64, dtype="bf16", shape="chain", ragged=False, window=0),
        # Eight requests' draft trees of 64 tokens checked in one call.
        dict(name="attend_tree_b8_64", kind="attend", batch=8, q_heads=32, kv_heads=8, tokens=64, ctx_min=4096,
             ctx_max=16384, mix=8, page=64, dtype="bf16", shape="wide", ragged=False, window=0),
        # Small ragged trees, fp16, group of seven, a sliding window, small pages.
        dict(name="attend_draft_window", kind="attend", batch=4, q_heads=28, kv_heads=4, tokens=13, ctx_min=900,
             ctx_max=5003, mix=9, page=16, dtype="f16", shape="deep", ragged=True, window=2048),
        # A piece of a long prompt (chunked prefill) behind what is cached so far.
        dict(name="attend_chunk_2k_of_32k", kind="attend", batch=1, q_heads=32, kv_heads=8, tokens=2048, ctx_min=30720,
             ctx_max=30720, mix=10, page=128, dtype="bf16", shape="chain", ragged=False, window=0),
        # One request's accepted tokens, a small model.
        dict(name="commit_4_layers", kind="commit", layers=4, batch=1, kv_heads=2, tokens=16, most=4, ctx_min=300,
             ctx_max=300, mix=11, page=16, store="f16"),
        # Eight requests' accepted paths out of trees of 64 tokens, in the 36 layers of a model.
        dict(name="commit_b8_36_layers", kind="commit", layers=36, batch=8, kv_heads=8, tokens=64, most=7, ctx_min=100,
             ctx_max=400, mix=12, page=64, store="bf16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["tree", "append", "append", "attend", "attend", "attend", "attend", "commit"])
    mix = rng.randrange(1 << 20)
    page = rng.choice([16, 32, 64, 64, 128])
    shape = rng.choice(["chain", "wide", "deep"])
    if kind == "tree":
        return dict(kind=kind, batch=_log_int(rng, 1, 64), tokens=_log_int(rng, 2, 500), mix=mix,
                    shape=rng.choice(["wide", "deep"]), ragged=rng.random() < 0.5)
    if kind == "commit":
        batch, tokens = rng.choice([1, 2, 5, 8]), _log_int(rng, 4, 200)
        low = rng.randint(0, 200)
        return dict(kind=kind, layers=rng.choice([1, 4, 17, 36]), batch=batch, kv_heads=rng.choice([1, 2, 4, 8]),
                    tokens=tokens, most=rng.randint(1, max(1, tokens // 3)), ctx_min=low,
                    ctx_max=low + rng.randint(0, 200), mix=mix, page=page, store=rng.choice(["bf16", "f16"]))
    q_heads, kv_heads = rng.choice([(8, 2), (32, 8), (32, 8), (28, 4), (16, 1), (8, 8), (64, 8)])
    if kind == "append":
        batch = rng.choice([1, 1, 3, 8, 16])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        most = 32768 * 48 // ((q_heads + 2 * kv_heads) * batch) // (2 if dtype == "f32" else 1)
        tokens = _log_int(rng, 1, most) if shape == "chain" else _log_int(rng, 2, min(500, most))
        low = rng.choice([0, _log_int(rng, 1, 4000)])
        return dict(kind=kind, batch=batch, q_heads=q_heads, kv_heads=kv_heads, tokens=tokens, ctx_min=low,
                    ctx_max=low + rng.randint(0, 3000), mix=mix, page=page, dtype=dtype,
                    store=dtype if dtype != "f32" else rng.choice(["bf16", "f16"]), shape=shape,
                    ragged=rng.random() < 0.5, layout=rng.choice(["heads", "tokens"]),
                    rotary=rng.choice([32, 64, 96, 128, 128]), interleaved=rng.random() < 0.3)
    batch = rng.choice([1, 1, 2, 5, 8])
    tokens = rng.choice([1, 1, rng.randint(2, 16), _log_int(rng, 10, 200), _log_int(rng, 10, 2048 // batch)])
    if tokens == 1:
        shape = "chain"
    elif shape != "chain":
        tokens = min(tokens, 500)
    most = 560000 // batch if tokens == 1 else 30720 * 2048 * 32 // (q_heads * batch * tokens)
    high = _log_int(rng, 100, min(131071 if tokens == 1 else 30720, max(200, most)))
    return dict(kind=kind, batch=batch, q_heads=q_heads, kv_heads=kv_heads, tokens=tokens,
                ctx_min=high // rng.choice([1, 2, 8]), ctx_max=high, mix=mix, page=page,
                dtype=rng.choice(["bf16", "bf16", "f16"]), shape=shape, ragged=rng.random() < 0.3,
                window=rng.choice([0, 0, 0, rng.randint(1, 4096)]))


# ------------------------------------------------------------------------------------------ inputs

def _lengths(case):
    """Committed rows of each sequence."""
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


def _parents(case):
    """Parents of every sequence's drafted tokens (-1: a child of the last committed token), or None for a chain."""
    if case["shape"] == "chain":
        return None
    rng = random.Random(case["mix"] + 2)
    trees = []
    for _ in range(case["batch"]):
        if case["shape"] == "wide":  # every token has the same number of children, level by level
            children = rng.randint(2, 8)
            trees.append([i // children - 1 for i in range(case["tokens"])])
        else:  # long branches that part now and then
            trees.append([rng.choice([i - 1, i - 1, i - 1, rng.randint(max(-1, i - 6), i - 1)])
                          for i in range(case["tokens"])])
    return trees


def _path(case):
    """Accepted tokens of each sequence: some first ones of the draft, then ones far enough behind that a pass leaves
    the rows that the next one reads as they are."""
    rng = random.Random(case["mix"] + 3)
    paths = []
    for _ in range(case["batch"]):
        size = rng.randint(1, case["most"])
        first = rng.randint(0, size) if rng.random() < 0.5 else 0
        later = range(size, case["tokens"])
        rest = sorted(rng.sample(later, min(size - first, len(later))))
        paths.append(list(range(first)) + rest)
    return paths


def _depths(parents):
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _table(case):
    """A page table [batch, pages a sequence] over a pool in any order, -1 where a sequence has no page, and the pool's size."""
    rng = random.Random(case["mix"] + 4)
    need = [-(-(n + case["tokens"]) // case["page"]) for n in _lengths(case)]
    pool = sum(need) + 3
    order = list(range(pool))
    rng.shuffle(order)
    table, at = [], 0
    for pages in need:
        table.append(order[at:at + pages] + [-1] * (max(need) - pages))
        at += pages
    return table, pool


def _values(gen, *shape, drift=0.0):
    """Keys or values as models have them: a few strong channels, and tokens of uneven size; heads in front of tokens."""
    channels = 1 + 6 * torch.rand(shape[-2], 1, D, generator=gen, device=DEVICE) ** 8
    size = torch.exp(0.3 * torch.randn(*shape, 1, generator=gen, device=DEVICE))
    x = torch.randn(*shape, D, generator=gen, device=DEVICE).mul_(size)
    return x.add_(drift).mul_(channels)


def _given(tensor, layout):
    """[batch, head, token, dim] values in memory order [batch, token, head, dim] where the layout says so."""
    return tensor.transpose(1, 2).contiguous().transpose(1, 2) if layout == "tokens" else tensor


def _tree(parents, counts):
    """The program's plan of a step's trees; the plain form keeps its tensors."""
    if own:
        from community_kv_amd import DraftTree

        return DraftTree.from_parents(parents, counts=counts)
    depths, masks = _plain_tree(parents, counts)
    return dict(depths=depths, masks=masks, counts=counts)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    state = dict(case=case)
    counts = _counts(case)
    state["counts"] = None if counts is None else _i32(counts)
    if case["kind"] == "tree":
        order = torch.rand(case["tokens"], generator=gen, device=DEVICE)  # other trees of the same shape for another seed
        parents = _i32(_parents(case))
        drop = (order < 0.02).expand_as(parents)
        state["parents"] = torch.where(drop, -1, parents).contiguous()
        return state
    table, pool = _table(case)
    lengths = _lengths(case)
    store = TYPES[case.get("store", case.get("dtype"))]
    heads = case["kv_heads"]

    def pages(drift):
        made = [_values(gen, pool, case["page"], heads, drift=drift).transpose(1, 2).to(store).contiguous()
                for _ in range(case.get("layers", 1))]
        return torch.stack(made)

    state["key_pages"], state["value_pages"] = pages(0.3), pages(0.0)
    state["page_table"], state["lengths"] = _i32(table), _i32(lengths)
    if own:
        from community_kv_amd import PagedKVCache

        state["cache"] = PagedKVCache(key_pages=state["key_pages"], value_pages=state["value_pages"],
                                      page_table=state["page_table"], lengths=state["lengths"])
    if case["kind"] == "commit":
        paths = _path(case)
        state["start"] = state["lengths"].clone()
        state["path"] = _i32([p + [0] * (case["most"] - len(p)) for p in paths])
        state["accepted"] = _i32([len(p) for p in paths])
        return state
    parents = _parents(case)
    state["tree"] = None if parents is None else _tree(_i32(parents), state["counts"])
    b, hq, tokens = case["batch"], case["q_heads"], case["tokens"]
    dtype = TYPES[case["dtype"]]
    if case["kind"] == "append":
        for name, count, drift in (("key", heads, 0.3), ("value", heads, 0.0), ("query", hq, 0.0)):
            state[name] = _given(_values(gen, b, tokens, count, drift=drift).transpose(1, 2).to(dtype), case["layout"])
            if case["layout"] == "heads":
                state[name] = state[name].contiguous()
        half = case["rotary"] // 2
        rows = len(table[0]) * case["page"]
        step = torch.arange(half, device=DEVICE, dtype=torch.float64) / half
        angle = torch.arange(rows, device=DEVICE, dtype=torch.float64)[:, None] * 1e6 ** -step
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
        if own:
            from community_kv_amd import RotaryTable

            state["rotary"] = RotaryTable(state["cos"], state["sin"], interleaved=case["interleaved"])
        return state
    # queries near some of the cached keys, so that a few rows take much of the weight
    group = hq // heads
    row = (torch.rand(b, heads, group * tokens, generator=gen, device=DEVICE) *
           (state["lengths"].clamp_min(1))[:, None, None]).long()
    batch = torch.arange(b, device=DEVICE)[:, None, None]
    page = state["page_table"][batch, row // case["page"]].long()
    head = torch.arange(heads, device=DEVICE)[:, None]
    near = state["key_pages"][0][page, head, row % case["page"]].float()
    near = near / near.square().mean(-1, keepdim=True).sqrt().clamp_min(1e-6)
    query = torch.randn(b, hq, tokens, D, generator=gen, device=DEVICE) + 0.5 * near.reshape(b, hq, tokens, D)
    state["query"] = query.to(dtype)
    return state


# ------------------------------------------------------------------------------------------ plain forms

def _plain_tree(parents, counts):
    """Depths [B, T] int32 and ancestor masks [B, T, ceil(T / 64)] int64: bit j % 64 of word j / 64 of token t is set
    where j is t or one of its ancestors; zeros for tokens past the counts."""
    b, tokens = parents.shape
    at = torch.arange(tokens, device=DEVICE)
    good = (parents >= 0) & (parents < at)
    jump = torch.where(good, parents, tokens).long()  # `tokens`: none
    jump = torch.cat([jump, jump.new_full((b, 1), tokens)], 1)
    seen = torch.eye(tokens + 1, dtype=torch.bool, device=DEVICE)[:, :tokens].expand(b, -1, -1)
    reach = 1
    while reach < tokens:  # ancestors up to twice as far each time
        seen = seen | seen.gather(1, jump[..., None].expand(-1, -1, tokens))
        jump = jump.gather(1, jump)
        reach *= 2
    seen = seen[:, :tokens]
    if counts is not None:
        seen = seen & (at < counts[:, None])[..., None]
    words = -(-tokens // 64)
    bits = torch.nn.functional.pad(seen, (0, words * 64 - tokens)).reshape(b, tokens, words, 64)
    masks = (bits.long() << torch.arange(64, device=DEVICE)).sum(-1)
    return (seen.sum(-1) - 1).clamp_min(0).int(), masks


def _plain_rotate(x, position, state):
    """The first `rotary` dims of x [B, H, T, D] turned by their position's angles, in pairs (i, i + rotary / 2) or (2 i, 2 i + 1)."""
    case = state["case"]
    half = case["rotary"] // 2
    cos, sin = state["cos"][position][:, None], state["sin"][position][:, None]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if case["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _plain_append(state):
    case, page = state["case"], state["case"]["page"]
    b, tokens = case["batch"], case["tokens"]
    t = torch.arange(tokens, device=DEVICE)
    start = state["lengths"].long()
    valid = torch.ones(b, tokens, dtype=torch.bool, device=DEVICE) if state["counts"] is None else t < state["counts"][:, None]
    depth = t.expand(b, tokens) if state["tree"] is None else state["tree"]["depths"].long()
    position = torch.where(valid, start[:, None] + depth, 0)
    row = start[:, None] + t
    at, token = valid.nonzero(as_tuple=True)
    where = state["page_table"][at, row[at, token] // page].long()
    offset = row[at, token] % page
    key = _plain_rotate(state["key"].float(), position, state)
    for name, x in (("key_pages", key), ("value_pages", state["value"].float())):
        state[name][0][where, :, offset] = x[at, :, token].to(state[name].dtype)
    query = _plain_rotate(state["query"].float(), position, state)
    query = torch.where(valid[:, None, :, None], query, 0)
    return query.to(state["key_pages"].dtype)


def _seeing(state, rows):
    """[B, T, rows]: which rows each of the step's tokens sees."""
    case = state["case"]
    tokens = case["tokens"]
    start = state["lengths"].long()[:, None]
    t = torch.arange(tokens, device=DEVICE)
    row = torch.arange(rows, device=DEVICE)
    count = tokens if state["counts"] is None else state["counts"][:, None]
    if state["tree"] is None:
        depth = t.expand(case["batch"], tokens)
        mask = row <= (start + t)[..., None]
    else:
        depth, masks = state["tree"]["depths"].long(), state["tree"]["masks"]
        drafted = (row - start)[:, None, :]                                       # [B, 1, rows]
        inside = (drafted >= 0) & (drafted < tokens)
        j = torch.where(inside, drafted, 0).expand(-1, tokens, -1)
        mask = (drafted < 0) | (inside & ((masks.gather(2, j // 64) >> (j % 64)) & 1).bool())
    if case["window"]:
        if state["tree"] is None:
            at = row.expand(case["batch"], rows)
        else:
            drafted = (row - start).clamp(0, tokens - 1)
            at = torch.where(row < start, row, start + depth.gather(1, drafted))
        mask = mask & (at[:, None] > (start + depth - case["window"])[..., None])
    return mask & (t < count).expand(case["batch"], tokens)[..., None]


def _plain_attend(state):
    case = state["case"]
    b, hq, tokens, _ = state["query"].shape
    h, page = case["kv_heads"], case["page"]
    rows = state["page_table"].shape[1] * page
    table = state["page_table"].long().clamp_min(0)
    mask = _seeing(state, rows)[:, None, None]
    key, value = (state[name][0][table].transpose(1, 2).reshape(b, h, rows, D).float()
                  for name in ("key_pages", "value_pages"))
    query = state["query"].float().reshape(b, h, hq // h * tokens, D)
    score = (query @ key.transpose(-1, -2)).reshape(b, h, hq // h, tokens, rows).mul_(SCALE)
    score = score.masked_fill_(~mask, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0, top)
    share = score.sub_(top).exp_()
    total = share.sum(-1, keepdim=True)
    lse = torch.where(total > 0, top + total.log(), -math.inf).reshape(b, hq, tokens)
    share = share.div_(torch.where(total > 0, total, 1))
    out = (share.reshape(b, h, hq // h * tokens, rows) @ value).reshape(b, hq, tokens, D)
    return dict(out=out.transpose(1, 2).to(state["query"].dtype), lse=lse)


def _plain_commit(state):
    case, page = state["case"], state["case"]["page"]
    start, path, accepted = state["lengths"].long()[:, None], state["path"].long(), state["accepted"].long()
    j = torch.arange(path.shape[1], device=DEVICE)
    at, place = (j < accepted[:, None]).nonzero(as_tuple=True)
    source, to = (start + path)[at, place], (start + j)[at, place]
    from_page, to_page = (state["page_table"][at, r // page].long() for r in (source, to))
    for name in ("key_pages", "value_pages"):
        pages = state[name]
        pages[:, to_page, :, to % page] = pages[:, from_page, :, source % page]
    state["lengths"] += state["accepted"]


# ------------------------------------------------------------------------------------------ one pass

def run(state):
    case = state["case"]
    if case["kind"] == "tree":
        tree = _tree(state["parents"], state["counts"])
        return dict(depths=tree.depths, masks=tree.masks) if own else dict(depths=tree["depths"], masks=tree["masks"])
    if case["kind"] == "append":
        if own:
            from community_kv_amd import paged_append

            query = paged_append(state["cache"], state["key"], state["value"], query=state["query"],
                                 rotary=state["rotary"], tree=state["tree"],
                                 counts=state["counts"] if state["tree"] is None else None)
        else:
            query = _plain_append(state)
        return dict(query=query, key_pages=state["key_pages"], value_pages=state["value_pages"])
    if case["kind"] == "attend":
        if not own:
            return _plain_attend(state)
        from community_kv_amd import paged_attention

        out, lse = paged_attention(state["query"], state["cache"], softmax_scale=SCALE, tree=state["tree"],
                                   counts=state["counts"] if state["tree"] is None else None, window=case["window"])
        return dict(out=out, lse=lse)
    state["lengths"].copy_(state["start"])  # every pass commits behind the same rows
    if own:
        from community_kv_amd import paged_commit

        paged_commit(state["cache"], state["accepted"], path=state["path"])
    else:
        _plain_commit(state)
    return dict(key_pages=state["key_pages"], value_pages=state["value_pages"], lengths=state["lengths"])


# ------------------------------------------------------------------------------------------ what a pass needs

def work(case):
    counts = _counts(case) or [case["tokens"]] * case["batch"]
    if case["kind"] == "tree":
        tokens = case["batch"] * case["tokens"]
        return dict(bytes=tokens * (8 + 8 * -(-case["tokens"] // 64)), flops=sum(counts))
    heads = case["kv_heads"]
    if case["kind"] == "commit":
        moved = sum(sum(p != j for j, p in enumerate(path)) for path in _path(case))
        return dict(bytes=moved * case["layers"] * heads * 2 * 2 * D * 2 + case["batch"] * 8, flops=case["batch"])
    wide = WIDE[case["dtype"]]
    if case["kind"] == "append":
        new = sum(counts)
        return dict(bytes=new * ((2 * heads + case["q_heads"]) * D * (wide + 2) + case["rotary"] * 4),
                    flops=new * (heads + case["q_heads"]) * case["rotary"] * 3)
    parents = _parents(case)
    pairs = touched = 0
    for b, (n, count) in enumerate(zip(_lengths(case), counts)):
        depths = list(range(count)) if parents is None else _depths(parents[b])[:count]
        window = case["window"] or n + count
        pairs += sum(min(n + d + 1, window) for d in depths)
        touched += min(n + count, window + count) if count else 0
    return dict(bytes=touched * heads * 2 * D * wide + sum(counts) * case["q_heads"] * (2 * D * wide + 4),
                flops=pairs * case["q_heads"] * 4 * D)


# ------------------------------------------------------------------------------------------ definitions in 64 bits

def exact(case, seed):
    global own
    if case["kind"] == "tree":
        return None  # whole numbers
    was, own = own, False
    try:
        state = prepare(case, seed)  # the inputs alone
    finally:
        own = was
    return {"append": _exact_append, "attend": _exact_attend, "commit": _exact_commit}[case["kind"]](state, case)


def _place(state, case, b, row):
    """Page and offset of rows of sequence b."""
    return state["page_table"][b][row // case["page"]].long(), row % case["page"]


def _exact_append(state, case):
    counts = _counts(case) or [case["tokens"]] * case["batch"]
    parents = _parents(case)
    half = case["rotary"] // 2
    cos, sin = state["cos"].double(), state["sin"].double()
    first = torch.arange(half, device=DEVICE) * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else half)
    result = {name: state[name].double() for name in ("key_pages", "value_pages")}
    result["query"] = torch.zeros(state["query"].shape, dtype=torch.float64, device=DEVICE)
    for b, (n, count) in enumerate(zip(_lengths(case), counts)):
        depths = list(range(count)) if parents is None else _depths(parents[b])[:count]
        at = n + torch.tensor(depths, dtype=torch.long, device=DEVICE)
        page, offset = _place(state, case, b, n + torch.arange(count, device=DEVICE))
        for name in ("query", "key"):
            x = state[name][b, :, :count].double()
            turned = x.clone()
            turned[..., first] = x[..., first] * cos[at] - x[..., second] * sin[at]
            turned[..., second] = x[..., first] * sin[at] + x[..., second] * cos[at]
            if name == "query":
                result["query"][b, :, :count] = turned
            else:
                result["key_pages"][0, page, :, offset] = turned.transpose(0, 1)
        result["value_pages"][0, page, :, offset] = state["value"][b, :, :count].double().transpose(0, 1)
    return {name: result[name] for name in ("query", "key_pages", "value_pages")}


def _exact_attend(state, case):
    b, hq, tokens, _ = state["query"].shape
    group = hq // case["kv_heads"]
    counts = _counts(case) or [tokens] * b
    parents = _parents(case)
    out = torch.zeros(b, tokens, hq, D, dtype=torch.float64, device=DEVICE)
    lse = torch.full((b, hq, tokens), -math.inf, dtype=torch.float64, device=DEVICE)
    for i, (n, count) in enumerate(zip(_lengths(case), counts)):
        if not count:
            continue
        kin = torch.ones(count, count, dtype=torch.bool).tril()
        depths = list(range(count)) if parents is None else _depths(parents[i])[:count]
        for t in range(count if parents is not None else 0):
            kin[t] = kin[parents[i][t]] if parents[i][t] >= 0 else False
            kin[t, t] = True
        depth = torch.tensor(depths, device=DEVICE)
        position = torch.cat([torch.arange(n, device=DEVICE), n + depth])
        seeing = torch.cat([torch.ones(count, n, dtype=torch.bool, device=DEVICE), kin.to(DEVICE)], 1)
        if case["window"]:
            seeing &= position > (n + depth - case["window"])[:, None]
        page, offset = _place(state, case, i, torch.arange(n + count, device=DEVICE))
        for head in range(case["kv_heads"]):
            key = state["key_pages"][0, page, head, offset].double()
            value = state["value_pages"][0, page, head, offset].double()
            for g in range(head * group, head * group + group):
                s = torch.where(seeing, (state["query"][i, g, :count].double() @ key.t()) * SCALE, -math.inf)
                z = torch.logsumexp(s, -1)
                out[i, :count, g], lse[i, g, :count] = (s - z[:, None]).exp() @ value, z
    return dict(out=out, lse=lse)


def _exact_commit(state, case):
    result = {name: state[name].double() for name in ("key_pages", "value_pages")}
    for b, (n, path) in enumerate(zip(_lengths(case), _path(case))):
        for j, p in enumerate(path):
            (from_page, from_at), (to_page, to_at) = (_place(state, case, b, torch.tensor(n + x, device=DEVICE)) for x in (p, j))
            for pages in result.values():
                pages[:, to_page, :, to_at] = pages[:, from_page, :, from_at]
    return dict(result, lengths=None)
