"""Paged KV cache of a batch, with position rotation, and trees of drafted tokens over it.

No reference counterpart (its cache holds one sequence at fixed addresses): this
is the cache of a server whose requests come and go, and of speculative
decoding, where a step's tokens are a tree of drafts of which one path is kept.
The kernels are ``ckv_draft_tree_plan_counts``, ``ckv_paged_append``,
``ckv_paged_attention`` and ``ckv_paged_commit``.

A step writes its tokens behind every sequence's committed rows and attends to
both; then ``paged_commit`` takes over the tokens that are kept, in all layers
at once::

    tree = DraftTree.from_parents(parents)                 # [batch, tokens]; none: a prompt, a piece of one, one token
    for layer in range(cache.layers):
        query = paged_append(cache, key, value, layer=layer, query=query, rotary=rotary, tree=tree)
        out, _ = paged_attention(query, cache, layer=layer, softmax_scale=scale, tree=tree)
        ...
    paged_commit(cache, accepted, path=path)               # or paged_commit(cache, tokens)

A step that is not committed is overwritten by the next.  Lengths and the page
table live on the device, so a captured step runs on what they hold when it is
replayed.  Calls on one cache are ordered by the stream they are made on; calls
on the same cache from two streams at once need an event between them.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass, field

import torch
from torch.autograd import forward_ad

from community_kv_amd import _native as nat
from community_kv_amd.attention.quantized import _rows

HEAD_DIM = nat.HEAD_DIM
PAGE_SIZES = (16, 32, 64, 128, 256)
MAX_DRAFT = nat.MAX_DRAFT
MAX_CAPACITY = 1 << 30
_STORES = {torch.bfloat16: nat.CKV_BF16, torch.float16: nat.CKV_F16}
_DTYPES = _STORES | {torch.float32: nat.CKV_F32}


def _expect(name: str, tensor: torch.Tensor, dtype: torch.dtype, shape: tuple[int, ...], device: torch.device) -> None:
    if tensor.dtype != dtype:
        raise TypeError(f"{name} must use {dtype}, not {tensor.dtype}")
    if tensor.shape != torch.Size(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(tensor.shape)}")
    if not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if tensor.device != device:
        raise ValueError(f"{name} must be on {device}")
    if tensor.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient; the paged cache has no backward pass (use torch.no_grad())")


@dataclass(frozen=True, eq=False)
class PagedKVCache:
    """All layers' keys and values in pages.  Row ``r`` of sequence ``b`` lies in
    page ``page_table[b, r // page_size]``, the same in every layer; a number
    outside the pool (-1) is no page.  The tensors keep their addresses for
    life, so captured graphs may hold them; their owner hands out pages by
    writing ``page_table`` (on the stream of the calls).  Sequences may share
    pages of committed rows (a common prompt), as long as none writes there."""

    key_pages: torch.Tensor    # [layers, pages, kv_heads, page_size, 128] bfloat16 or float16
    value_pages: torch.Tensor  # same
    page_table: torch.Tensor   # [batch, pages a sequence] int32
    lengths: torch.Tensor      # [batch] int32: committed rows
    overflow: torch.Tensor = field(init=False)  # [batch] int32: 1 where tokens found no row
    _counters: torch.Tensor = field(init=False, repr=False)
    # made once: a call costs microseconds
    _struct: nat.PagedCache = field(init=False, repr=False)
    _ref: object = field(init=False, repr=False)  # the struct by reference
    _facts: tuple = field(init=False, repr=False)  # layers, batch, kv_heads, capacity, device number
    _sizes: dict = field(init=False, repr=False)  # workspace bytes by call shape

    def __post_init__(self) -> None:
        pages = self.key_pages
        if pages.ndim != 5 or pages.shape[-1] != HEAD_DIM or 0 in pages.shape:
            raise ValueError(f"pages must be a non-empty [layers, pages, KV heads, page size, {HEAD_DIM}] tensor")
        if pages.dtype not in _STORES:
            raise TypeError(f"pages must use bfloat16 or float16, not {pages.dtype}")
        if pages.shape[3] not in PAGE_SIZES:
            raise ValueError(f"the page size must be one of {PAGE_SIZES}, not {pages.shape[3]}")
        if self.page_table.ndim != 2 or 0 in self.page_table.shape:
            raise ValueError("page_table must be a non-empty [batch, pages a sequence] tensor")
        batch, table_pages = self.page_table.shape
        layers, count, heads, size, _ = pages.shape
        expected = [("key_pages", pages, pages.dtype, pages.shape), ("value_pages", self.value_pages, pages.dtype, pages.shape),
                    ("page_table", self.page_table, torch.int32, (batch, table_pages)),
                    ("lengths", self.lengths, torch.int32, (batch,))]
        for name, tensor, dtype, shape in expected:
            _expect(name, tensor, dtype, shape, pages.device)
        if table_pages * size > MAX_CAPACITY:
            raise ValueError(f"a sequence may have at most {MAX_CAPACITY} rows, not {table_pages * size}")
        if batch * heads > 65535 or batch > 32767 or heads > 32767:
            raise ValueError("batch and KV heads may be at most 32767 each and 65535 together")
        if any(t.data_ptr() % 16 for t in (pages, self.value_pages)):
            raise ValueError("pages must be 16-byte aligned")
        spans = sorted((tensor.data_ptr(), tensor.data_ptr() + tensor.nbytes) for _, tensor, _, _ in expected)
        if any(start < end for (_, end), (start, _) in zip(spans, spans[1:])):
            raise ValueError("the tensors of a cache must not share memory")
        overflow, counters = (torch.zeros(batch * each, dtype=torch.int32, device=pages.device)
                              for each in (1, nat.QUANT_COUNTERS))
        struct = nat.PagedCache(pages.data_ptr(), self.value_pages.data_ptr(), self.page_table.data_ptr(),
                                self.lengths.data_ptr(), overflow.data_ptr(), counters.data_ptr(), layers, count, heads, size,
                                table_pages, batch, _STORES[pages.dtype], 0)
        facts = (layers, batch, heads, table_pages * size, pages.get_device())
        for name, value in (("overflow", overflow), ("_counters", counters), ("_struct", struct), ("_ref", ctypes.byref(struct)), ("_facts", facts),
                            ("_sizes", {})):
            object.__setattr__(self, name, value)

    @classmethod
    def allocate(cls, *, layers: int, batch: int, kv_heads: int, capacity: int, page_size: int = 64,
                 pages: int | None = None, dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str) -> "PagedKVCache":
        """An empty cache whose sequences may have up to ``capacity`` rows each
        (rounded up to whole pages).  Without ``pages`` every sequence has pages
        of its own for all of them; with it the pool has that many and the table
        names none yet."""
        if min(layers, batch, kv_heads, capacity) <= 0 or (pages is not None and pages <= 0):
            raise ValueError("layers, batch, kv_heads, capacity and pages must be positive")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"the page size must be one of {PAGE_SIZES}, not {page_size}")
        each = -(-capacity // page_size)
        shape = (layers, batch * each if pages is None else pages, kv_heads, page_size, HEAD_DIM)
        table = (torch.arange(batch * each, dtype=torch.int32, device=device).reshape(batch, each) if pages is None else
                 torch.full((batch, each), -1, dtype=torch.int32, device=device))
        return cls(key_pages=torch.zeros(shape, dtype=dtype, device=device),
                   value_pages=torch.zeros(shape, dtype=dtype, device=device), page_table=table,
                   lengths=torch.zeros(batch, dtype=torch.int32, device=device))

    @property
    def layers(self) -> int:
        return self.key_pages.shape[0]

    @property
    def pages(self) -> int:
        return self.key_pages.shape[1]

    @property
    def kv_heads(self) -> int:
        return self.key_pages.shape[2]

    @property
    def page_size(self) -> int:
        return self.key_pages.shape[3]

    @property
    def batch(self) -> int:
        return self.page_table.shape[0]

    @property
    def capacity(self) -> int:
        """Rows that a sequence's table can name."""
        return self.page_table.shape[1] * self.page_size

    @property
    def dtype(self) -> torch.dtype:
        return self.key_pages.dtype

    @property
    def device(self) -> torch.device:
        return self.key_pages.device

    def assert_no_overflow(self) -> None:
        """Raises if tokens found no row (reads the device)."""
        if bool(self.overflow.any()):
            raise RuntimeError(f"paged KV cache overflow: capacity {self.capacity}, flags {self.overflow.tolist()}")


@dataclass(frozen=True, eq=False)
class RotaryTable:
    """Cosines and sines [positions, dims / 2] float32 of every position's angles.
    The first ``dims`` dimensions of a row turn in pairs (i, i + dims / 2), or
    (2 i, 2 i + 1) where ``interleaved``; the others stay."""

    cosines: torch.Tensor
    sines: torch.Tensor
    interleaved: bool = False
    _struct: nat.Rotary = field(init=False, repr=False)
    _facts: tuple = field(init=False, repr=False)  # the struct's address, positions, device number

    def __post_init__(self) -> None:
        if self.cosines.ndim != 2 or self.cosines.shape[0] == 0:
            raise ValueError("cosines must be a non-empty [positions, dims / 2] tensor")
        positions, half = self.cosines.shape
        if half % 8 or not 8 <= half <= HEAD_DIM // 2:
            raise ValueError(f"the rotated dims must be a multiple of 16 up to {HEAD_DIM}, not {2 * half}")
        if positions > 2**31 - 1:
            raise ValueError("too many positions")
        for name, tensor in (("cosines", self.cosines), ("sines", self.sines)):
            _expect(name, tensor, torch.float32, (positions, half), self.cosines.device)
            if tensor.data_ptr() % 16:
                raise ValueError(f"{name} must be 16-byte aligned")
        struct = nat.Rotary(self.cosines.data_ptr(), self.sines.data_ptr(), positions, 2 * half, int(self.interleaved), 0)
        object.__setattr__(self, "_struct", struct)
        object.__setattr__(self, "_facts", (ctypes.addressof(struct), positions, self.cosines.get_device()))

    @classmethod
    def from_frequencies(cls, frequencies: torch.Tensor, positions: int, *, interleaved: bool = False,
                         scale: float = 1.0) -> "RotaryTable":
        """The table of ``positions`` positions from a model's angles a position
        [dims / 2]: angles in 64 bits, so far positions keep theirs; ``scale``
        multiplies cosines and sines (models with stretched contexts)."""
        if frequencies.ndim != 1 or positions <= 0:
            raise ValueError("frequencies must be a vector and positions positive")
        at = torch.arange(positions, dtype=torch.float64, device=frequencies.device)
        angles = at[:, None] * frequencies.double()
        return cls((angles.cos() * scale).float(), (angles.sin() * scale).float(), interleaved)

    @property
    def positions(self) -> int:
        return self.cosines.shape[0]


class DraftTree:
    """The drafted tokens of a step, made once and used by every layer.  Token
    ``t`` stands ``depths[b, t]`` positions behind the first drafted ones, and
    bit ``j % 64`` of ``masks[b, t, j // 64]`` is set where ``j`` is ``t`` or one
    of its ancestors.  A caller's own depths and masks may be any: tokens in any
    order, depths from 0 on (negative ones count as 0, ones from 2**30 on as
    2**30 - 1), any set of drafted tokens to attend.

    ``depths`` [batch, tokens] int32, ``masks`` [batch, tokens, ceil(tokens / 64)]
    int64, ``counts`` [batch] int32 (tokens of each sequence) or None: a caller's
    own are kept by reference and stay as they are until the last layer's call;
    those of ``from_parents`` are the tree's."""

    __slots__ = ("depths", "masks", "counts", "_struct", "_facts")

    def __init__(self, depths: torch.Tensor, masks: torch.Tensor, counts: torch.Tensor | None = None) -> None:
        if depths.ndim != 2 or 0 in depths.shape:
            raise ValueError("depths must be a non-empty [batch, tokens] tensor")
        batch, tokens = depths.shape
        if tokens > MAX_DRAFT:
            raise ValueError(f"a tree may have at most {MAX_DRAFT} tokens, not {tokens}")
        _expect("depths", depths, torch.int32, (batch, tokens), depths.device)
        _expect("masks", masks, torch.int64, (batch, tokens, -(-tokens // 64)), depths.device)
        if counts is not None:
            _expect("counts", counts, torch.int32, (batch,), depths.device)
        self._hold(depths, masks, counts, batch, tokens, depths.get_device())

    def _hold(self, depths, masks, counts, batch, tokens, device) -> None:
        self.depths, self.masks, self.counts = depths, masks, counts
        at = depths.data_ptr()
        self._struct = nat.TreeMasks(at, masks.data_ptr())
        # batch, tokens, device number, addresses of the struct, the depths and the counts
        self._facts = (batch, tokens, device, ctypes.addressof(self._struct), at, 0 if counts is None else counts.data_ptr())

    @classmethod
    def from_parents(cls, parents: torch.Tensor, *, counts: torch.Tensor | None = None) -> "DraftTree":
        """``parents`` [batch, tokens] int32 names each token's parent, an earlier
        token of the draft; any other value (-1) makes it a child of the last
        committed token.  ``counts`` (int32, clamped to [0, tokens]): the first
        tokens of each sequence that are there.  Neither is needed afterwards."""
        if parents.dtype != torch.int32:
            raise TypeError(f"parents must use int32, not {parents.dtype}")
        shape = parents.shape
        if len(shape) != 2 or 0 in shape:
            raise ValueError("parents must be a non-empty [batch, tokens] tensor")
        batch, tokens = shape
        if tokens > MAX_DRAFT:
            raise ValueError(f"a tree may have at most {MAX_DRAFT} tokens, not {tokens}")
        device = parents.get_device()
        counts_at = kept_at = 0
        kept = None
        if counts is not None:
            counts = _counts_vector(counts, batch, device)
            counts_at = counts.data_ptr()
        if device < 0:
            raise RuntimeError(_NEED_GPU)
        if counts is not None:
            kept = counts.new_empty(batch)
            kept_at = kept.data_ptr()
        parents = parents.contiguous()
        depths = parents.new_empty((batch, tokens))
        masks = parents.new_empty((batch, tokens, (tokens + 63) // 64), dtype=torch.int64)
        tree = cls.__new__(cls)
        tree._hold(depths, masks, kept, batch, tokens, device)
        _launch(device, nat.lib().ckv_draft_tree_plan_counts, parents.data_ptr(), counts_at, batch, tokens, depths.data_ptr(),
                masks.data_ptr(), kept_at)
        return tree

    @property
    def batch(self) -> int:
        return self.depths.shape[0]

    @property
    def tokens(self) -> int:
        return self.depths.shape[1]


_NEED_GPU = "the paged cache runs on the GPU only (got a CPU tensor)"


def _launch(device: int, function, *args) -> None:
    """Calls a C entry on the current stream of device number ``device``."""
    if device == torch._C._cuda_getDevice():
        rc = function(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = function(*args, torch._C._cuda_getCurrentRawStream(device))
    if rc:
        nat.check(rc)


def _counts_vector(counts: torch.Tensor, batch: int, device: int) -> torch.Tensor:
    if counts.dtype != torch.int32 or counts.shape != (batch,):
        raise TypeError(f"counts must be an int32 vector of one entry a sequence ({batch})")
    if counts.get_device() != device:
        raise ValueError("all tensors must share one device")
    return counts.contiguous()


def _refuse_tangents(**tensors: torch.Tensor | None) -> None:
    """Inside a forward_ad level (its number is negative outside, which a call looks at first)."""
    for name, tensor in tensors.items():
        if tensor is not None and forward_ad.unpack_dual(tensor).tangent is not None:
            raise RuntimeError(f"{name} carries a tangent; the paged cache has no forward-mode derivative")


def _check_step(cache: PagedKVCache, layer: int, name: str, tensor: torch.Tensor) -> torch.Size:
    shape = tensor.shape
    layers, batch, _, _, device = cache._facts
    if len(shape) != 4 or shape[0] != batch or shape[3] != HEAD_DIM:
        raise ValueError(f"{name} must have shape [{batch}, heads, tokens, {HEAD_DIM}], not {tuple(shape)}")
    if not 0 <= layer < layers:
        raise ValueError(f"layer {layer} of a cache of {layers}")
    if tensor.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient; the paged cache has no backward pass (use torch.no_grad())")
    if tensor.get_device() != device:
        raise ValueError("all tensors must share one device")
    return shape


def _step_counts(cache: PagedKVCache, tokens: int, tree: DraftTree | None,
                 counts: torch.Tensor | None) -> tuple[int, torch.Tensor | None]:
    """Address of a step's counts (0: all tokens), and the tensor that holds them."""
    _, batch, _, _, device = cache._facts
    if tree is not None:
        if counts is not None:
            raise ValueError("a tree has its own counts")
        facts = tree._facts
        if facts[0] != batch or facts[1] != tokens:
            raise ValueError(f"the tree holds {facts[:2]} tokens, the call {(batch, tokens)}")
        if facts[2] != device:
            raise ValueError("all tensors must share one device")
        return facts[5], tree.counts
    if counts is None:
        return 0, None
    counts = _counts_vector(counts, batch, device)
    return counts.data_ptr(), counts


def _view(tensor: torch.Tensor) -> tuple[tuple[int, int, int, int], torch.Tensor]:
    """Address and strides of [batch, heads, tokens, 128], and the tensor that they are of (a copy where they do not
    suit 16-byte loads)."""
    b, h, t, d = tensor.stride()
    at = tensor.data_ptr()
    if d == 1 and not ((b | h | t) * tensor.element_size() | at) & 15:
        return (at, b, h, t), tensor
    rows, tensor = _rows(tensor)
    return (rows.data, rows.batch_stride, rows.head_stride, rows.token_stride), tensor


_NO_ROWS = (0, 0, 0, 0)


def paged_append(cache: PagedKVCache, key: torch.Tensor, value: torch.Tensor, *, layer: int = 0,
                 query: torch.Tensor | None = None, rotary: RotaryTable | None = None, tree: DraftTree | None = None,
                 counts: torch.Tensor | None = None) -> torch.Tensor | None:
    """Writes a step's ``key``/``value`` [batch, kv_heads, tokens, 128] (bf16, fp16
    or f32, any strides) into layer ``layer``, behind the committed rows: the first
    ``counts[b]`` tokens (int32 on the device, clamped to [0, tokens]; a tree brings
    its own) or all of them.  With ``rotary`` keys are turned by their position on
    the way: the committed length plus the token's place, or its depth in ``tree``.

    ``query`` [batch, query heads, tokens, 128] in the keys' dtype is turned
    likewise and returned in the cache's dtype, as [batch, query heads, tokens, 128]
    over memory [batch, tokens, query heads, 128]; zeros past the counts.

    Tokens whose row is past the capacity or has no page are dropped and raise the
    overflow flag (``assert_no_overflow``)."""
    layers, batch, heads, capacity, device = cache._facts
    if forward_ad._current_level >= 0:
        _refuse_tangents(key=key, value=value, query=query, key_pages=cache.key_pages, value_pages=cache.value_pages,
                         cosines=None if rotary is None else rotary.cosines, sines=None if rotary is None else rotary.sines)
    shape, kind = key.shape, key.dtype
    dtype = _DTYPES.get(kind)
    if (dtype is None or value.dtype != kind or value.shape != shape or len(shape) != 4 or shape[1] != heads or
            value.requires_grad or value.get_device() != device):
        _check_step(cache, layer, "value", value)
        if dtype is None:
            raise TypeError(f"key must use bfloat16, float16 or float32, not {key.dtype}")
        if len(shape) != 4 or shape[1] != heads or value.shape != shape:
            raise ValueError(f"key and value must both have {heads} heads and the same tokens")
        if value.dtype != kind:
            raise TypeError("key and value must share a dtype")
    _check_step(cache, layer, "key", key)
    tokens = shape[2]
    rotary_at = query_heads = turned_at = 0
    query_view = _NO_ROWS
    if rotary is not None:
        rotary_at, positions, table_device = rotary._facts
        if positions < capacity:
            raise ValueError(f"the rotation table holds {positions} positions, the cache {capacity} rows")
        if table_device != device:
            raise ValueError("all tensors must share one device")
    if query is not None:
        if rotary is None:
            raise ValueError("queries are only turned: query needs rotary")
        _, query_heads, query_tokens, _ = _check_step(cache, layer, "query", query)
        if query.dtype != key.dtype:
            raise TypeError("query and key must share a dtype")
        if query_heads == 0 or query_tokens != tokens:
            raise ValueError(f"query must have heads and the keys' {tokens} tokens")
    counts_at, counts = _step_counts(cache, tokens, tree, counts)
    if device < 0:
        raise RuntimeError(_NEED_GPU)
    turned = None
    if query is not None:
        row = query_heads * HEAD_DIM
        turned = cache.key_pages.new_empty_strided((batch, query_heads, tokens, HEAD_DIM), (tokens * row, HEAD_DIM, row, 1))
        turned_at = turned.data_ptr()
        query_view, query = _view(query)
    if tokens:
        key_view, key = _view(key)
        value_view, value = _view(value)
        args = nat.PAGED_APPEND_ARGS.pack(*key_view, *value_view, *query_view, counts_at, 0 if tree is None else tree._facts[4],
                                          rotary_at, turned_at, layer, tokens, query_heads, dtype)
        _launch(device, nat.lib().ckv_paged_append, cache._ref, args)
    return turned


def paged_attention(query: torch.Tensor, cache: PagedKVCache, *, softmax_scale: float, layer: int = 0,
                    tree: DraftTree | None = None, counts: torch.Tensor | None = None,
                    window: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of a step's tokens, already written, over layer ``layer``.

    ``query`` [batch, query heads, tokens, 128] (the cache's dtype, any strides) are
    the queries of the tokens behind the committed rows, of the first ``counts[b]`` or
    of all.  A query attends the committed rows and the step's tokens up to its own,
    or with ``tree`` its own and its ancestors; with ``window`` > 0 only those at the
    last ``window`` positions, its own among them.

    Returns (output [batch, tokens, query heads, 128] in the queries' dtype, lse
    [batch, query heads, tokens] float32, natural log); a query past the counts gives
    zeros and -inf.  What a query does not see does not reach it, infinities and NaN
    included; an infinite value that it sees makes its output infinite or NaN.  Scores
    may be as large as products of finite queries and keys in 32 bits are, times the
    scale; an lse beyond 32 bits is infinite."""
    _, batch, kv_heads, _, device = cache._facts
    if forward_ad._current_level >= 0:
        _refuse_tangents(query=query, key_pages=cache.key_pages, value_pages=cache.value_pages)
    _, heads, tokens, _ = _check_step(cache, layer, "query", query)
    if query.dtype != cache.key_pages.dtype:
        raise TypeError(f"query must use the cache's {cache.dtype}, not {query.dtype}")
    if heads % kv_heads or not 1 <= heads // kv_heads <= nat.MAX_GROUP:
        raise ValueError(f"query heads must be 1 to {nat.MAX_GROUP} times the {kv_heads} KV heads, not {heads}")
    if not 1e-30 <= softmax_scale <= 1e30:
        raise ValueError("softmax_scale must be between 1e-30 and 1e30")
    if window < 0:
        raise ValueError("window must be non-negative")
    counts_at, counts = _step_counts(cache, tokens, tree, counts)
    if device < 0:
        raise RuntimeError(_NEED_GPU)
    out = query.new_empty((batch, tokens, heads, HEAD_DIM))
    lse = query.new_empty((batch, heads, tokens), dtype=torch.float32)
    if tokens == 0:
        return out, lse
    lib = nat.lib()
    window = min(window, 2**31 - 1)
    call = (heads, tokens, window)
    size = cache._sizes.get(call)
    if size is None:
        if len(cache._sizes) >= 1024:
            cache._sizes.clear()
        size = cache._sizes[call] = lib.ckv_paged_attention_workspace_bytes(cache._ref, heads, tokens, window)
    workspace = query.new_empty(size, dtype=torch.uint8) if size else None
    view, query = _view(query)
    args = nat.PAGED_ATTENTION_ARGS.pack(*view, counts_at, 0 if tree is None else tree._facts[3], out.data_ptr(),
                                         lse.data_ptr(), workspace.data_ptr() if size else 0, layer, heads, tokens, window,
                                         softmax_scale, 0)
    _launch(device, lib.ckv_paged_attention, cache._ref, args)
    return out, lse


def paged_commit(cache: PagedKVCache, counts: int | torch.Tensor, *, path: torch.Tensor | None = None) -> None:
    """Takes over a step's tokens in all layers.  Without ``path`` the first
    ``counts`` of every sequence (a number, or int32 [batch] on the device):
    ``lengths`` grows by them, up to the capacity.  With ``path`` (int32 [batch, n],
    n <= 512) the tokens ``path[b, :counts[b]]``, in ascending order, as a branch of a
    tree has them: their rows move together behind the committed ones.  A path ends
    at the first entry that does not ascend or lies past the capacity."""
    _, batch, _, _, device = cache._facts
    amount = counts_at = path_at = entries = 0
    if isinstance(counts, torch.Tensor):
        counts = _counts_vector(counts, batch, device)
        counts_at = counts.data_ptr()
        amount = 2**31 - 1
    else:
        if counts < 0:
            raise ValueError("counts must be non-negative")
        amount, counts = min(counts, 2**31 - 1), None
    if path is not None:
        shape = path.shape
        if path.dtype != torch.int32 or len(shape) != 2 or shape[0] != batch:
            raise TypeError(f"path must be an int32 tensor [{batch}, entries]")
        if not 1 <= shape[1] <= MAX_DRAFT:
            raise ValueError(f"a path may have 1 to {MAX_DRAFT} entries, not {shape[1]}")
        if path.get_device() != device:
            raise ValueError("all tensors must share one device")
        if counts is None:
            path = path[:, :amount]
        path = path.contiguous()
        path_at, entries = path.data_ptr(), path.shape[1]
        if entries == 0:
            return
    if device < 0:
        raise RuntimeError(_NEED_GPU)
    _launch(device, nat.lib().ckv_paged_commit, cache._ref, amount, counts_at, path_at, entries)


__all__ = ["DraftTree", "PagedKVCache", "RotaryTable", "paged_append", "paged_attention", "paged_commit"]
