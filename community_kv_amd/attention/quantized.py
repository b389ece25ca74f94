"""8-bit KV cache: block-scaled E4M3 storage, attention over it, eviction from it.

No reference counterpart (its cache is bf16): this is the cache for contexts
that should take half the memory and half the bytes a decode step, and, with
``evict``, for requests that run within a fixed number of rows.  The kernels
are ``ckv_quant_append``, ``ckv_quant_attention`` and ``ckv_quant_evict``.

A cache holds one layer's rows of ``batch`` sequences.  It is a set of
(position, key, value) rows per KV head: masks go by position, never by the
place of a row, because an eviction moves rows.  Write cursors live on the
device, so a captured step appends where its last replay stopped.  Calls on
one cache are ordered by the stream they are made on; calls on the same cache
from two streams at once need an event between them.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass, field

import torch

from community_kv_amd import _native as nat

HEAD_DIM = nat.HEAD_DIM
BLOCKS = (16, 32, 64, 128)
_DTYPES = {torch.bfloat16: nat.CKV_BF16, torch.float16: nat.CKV_F16, torch.float32: nat.CKV_F32}


@dataclass(frozen=True, eq=False)
class QuantizedKVCache:
    """One layer's 8-bit cache.  The tensors keep their addresses for life, so
    captured graphs may hold them; ``allocate`` makes an empty cache,
    ``from_tensors`` takes existing tensors without copying them.

    A row's key is ``key_codes * key_scales`` of its block, and so its value.
    ``cursors`` rows: rows in use, tokens ever appended, and the overflow flag
    (1 where tokens did not fit)."""

    key_codes: torch.Tensor     # [batch, kv_heads, capacity, 128] float8_e4m3fn
    value_codes: torch.Tensor   # same
    key_scales: torch.Tensor    # [batch, kv_heads, capacity / block] float32
    value_scales: torch.Tensor  # same
    positions: torch.Tensor     # [batch, kv_heads, capacity] int32
    cursors: torch.Tensor       # [3, batch] int32
    block: int = 64
    weights: torch.Tensor | None = None  # [batch, kv_heads, capacity] float32: attention received
    _counters: torch.Tensor = field(init=False, repr=False)
    _struct: nat.QuantCache = field(init=False, repr=False)
    _ref: object = field(init=False, repr=False)  # the struct by reference, made once: a call costs microseconds
    _sizes: dict = field(init=False, repr=False)  # workspace bytes by call shape

    def __post_init__(self) -> None:
        codes = self.key_codes
        if self.block not in BLOCKS:
            raise ValueError(f"block must be one of {BLOCKS}")
        if codes.ndim != 4 or codes.shape[-1] != HEAD_DIM or 0 in codes.shape or codes.shape[2] % self.block:
            raise ValueError(f"codes must be a non-empty [batch, KV heads, capacity, {HEAD_DIM}] tensor with capacity "
                             f"a multiple of block ({self.block})")
        batch, heads, capacity, _ = codes.shape
        expected = [("key_codes", codes, torch.float8_e4m3fn, codes.shape),
                    ("value_codes", self.value_codes, torch.float8_e4m3fn, codes.shape),
                    ("key_scales", self.key_scales, torch.float32, (batch, heads, capacity // self.block)),
                    ("value_scales", self.value_scales, torch.float32, (batch, heads, capacity // self.block)),
                    ("positions", self.positions, torch.int32, (batch, heads, capacity)),
                    ("cursors", self.cursors, torch.int32, (3, batch))]
        if self.weights is not None:
            expected.append(("weights", self.weights, torch.float32, (batch, heads, capacity)))
        for name, tensor, dtype, shape in expected:
            if tensor.dtype != dtype:
                raise TypeError(f"{name} must use {dtype}, not {tensor.dtype}")
            if tensor.shape != torch.Size(shape):
                raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(tensor.shape)}")
            if not tensor.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
            if tensor.device != codes.device:
                raise ValueError("all tensors of a cache must share one device")
        if any(t.data_ptr() % 16 for t in (codes, self.value_codes, self.positions, self.weights) if t is not None):
            raise ValueError("codes, positions and weights must be 16-byte aligned")
        spans = sorted((tensor.data_ptr(), tensor.data_ptr() + tensor.nbytes) for _, tensor, _, _ in expected)
        if any(start < end for (_, end), (start, _) in zip(spans, spans[1:])):
            raise ValueError("the tensors of a cache must not share memory")
        counters = torch.zeros(batch * nat.QUANT_COUNTERS, dtype=torch.int32, device=codes.device)
        struct = nat.QuantCache(
            codes.data_ptr(), self.value_codes.data_ptr(), self.key_scales.data_ptr(), self.value_scales.data_ptr(),
            self.positions.data_ptr(), nat.ptr(self.weights), self.cursors.data_ptr(), counters.data_ptr(), capacity,
            batch, heads, self.block)
        for name, value in (("_counters", counters), ("_struct", struct), ("_ref", ctypes.byref(struct)), ("_sizes", {})):
            object.__setattr__(self, name, value)

    @classmethod
    def allocate(cls, *, batch: int = 1, kv_heads: int, capacity: int, block: int = 64, track_weights: bool = False,
                 device: torch.device | str) -> "QuantizedKVCache":
        """An empty cache of ``capacity`` rows a sequence (rounded up to whole
        blocks); ``track_weights`` keeps the sums that ``evict`` goes by."""
        if batch <= 0 or kv_heads <= 0 or capacity <= 0:
            raise ValueError("batch, kv_heads and capacity must be positive")
        if block not in BLOCKS:
            raise ValueError(f"block must be one of {BLOCKS}")
        capacity = -(-capacity // block) * block
        rows = (batch, kv_heads, capacity)

        def zeros(shape, dtype):
            return torch.zeros(shape, dtype=dtype, device=device)

        return cls(key_codes=zeros((*rows, HEAD_DIM), torch.uint8).view(torch.float8_e4m3fn),
                   value_codes=zeros((*rows, HEAD_DIM), torch.uint8).view(torch.float8_e4m3fn),
                   key_scales=zeros((batch, kv_heads, capacity // block), torch.float32),
                   value_scales=zeros((batch, kv_heads, capacity // block), torch.float32),
                   positions=zeros(rows, torch.int32), cursors=zeros((3, batch), torch.int32), block=block,
                   weights=zeros(rows, torch.float32) if track_weights else None)

    @classmethod
    def from_tensors(cls, *, key_codes: torch.Tensor, value_codes: torch.Tensor, key_scales: torch.Tensor,
                     value_scales: torch.Tensor, positions: torch.Tensor, cursors: torch.Tensor, block: int = 64,
                     weights: torch.Tensor | None = None) -> "QuantizedKVCache":
        """A cache over tensors that the caller has (an imported or restored
        cache).  Scales must be powers of two in [2^-64, 2^120], or 0 where no
        row is in use (checked, which reads the device); the rows in use must
        have distinct positions in [0, seen) (not checked)."""
        for name, scales in (("key_scales", key_scales), ("value_scales", value_scales)):
            mantissa, exponent = torch.frexp(scales)
            good = (mantissa == 0.5) & (exponent >= -63) & (exponent <= 121)
            if not bool((good | (scales == 0)).all()):
                raise ValueError(f"{name} must be powers of two in [2^-64, 2^120], or 0")
        return cls(key_codes=key_codes, value_codes=value_codes, key_scales=key_scales, value_scales=value_scales,
                   positions=positions, cursors=cursors, block=block, weights=weights)

    @property
    def batch(self) -> int:
        return self.key_codes.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.key_codes.shape[1]

    @property
    def capacity(self) -> int:
        return self.key_codes.shape[2]

    @property
    def device(self) -> torch.device:
        return self.key_codes.device

    @property
    def lengths(self) -> torch.Tensor:
        """Rows in use of every sequence (device int32)."""
        return self.cursors[0]

    def reset(self) -> None:
        """Empties the cache (its memory is kept, and need not be cleared)."""
        self.cursors.zero_()

    def rewind(self, counts: int | torch.Tensor) -> None:
        """Takes back the newest ``counts`` tokens of every sequence (rejected
        draft tokens): at most those appended since the last eviction.  Block
        scales stay as they have grown, and other rows keep the weight that the
        tokens' queries gave them (attend to drafts without ``accumulate`` where
        it must not count)."""
        if isinstance(counts, int) and counts < 0:
            raise ValueError("counts must be non-negative")
        self.cursors[:2].sub_(counts)

    def dequantize(self) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values [batch, kv_heads, capacity, 128] in float32, with
        whatever the rows past the lengths hold."""
        return tuple(codes.float() * scales.repeat_interleave(self.block, 2)[..., None]
                     for codes, scales in ((self.key_codes, self.key_scales), (self.value_codes, self.value_scales)))

    def assert_no_overflow(self) -> None:
        """Raises if an append found no room (reads the device)."""
        if bool(self.cursors[2].any()):
            raise RuntimeError(f"8-bit KV cache overflow: capacity {self.capacity}, flags {self.cursors[2].tolist()}")


def _rows(tensor: torch.Tensor) -> tuple[nat.QuantRows, torch.Tensor]:
    """The C view of [batch, heads, tokens, 128] and the tensor it points to
    (a copy where the strides or the address do not suit 16-byte loads)."""
    unit = 4 if tensor.dtype is torch.float32 else 8
    b, h, t, d = tensor.stride()
    address = tensor.data_ptr()
    if d != 1 or address % 16 or (b | h | t) % unit:
        b, h, t = (0 if size == 1 else stride for size, stride in zip(tensor.shape, (b, h, t)))
        if d != 1 or address % 16 or (b | h | t) % unit:
            tensor = tensor.contiguous() if d != 1 or address % 16 == 0 else tensor.clone(
                memory_format=torch.contiguous_format)
            if tensor.data_ptr() % 16:
                tensor = tensor.clone()
            b, h, t, d = tensor.stride()
            address = tensor.data_ptr()
    return nat.QuantRows(address, b, h, t), tensor


def _check_rows(cache: QuantizedKVCache, name: str, tensor: torch.Tensor) -> None:
    shape = tensor.shape
    if len(shape) != 4 or shape[0] != cache._struct.batch or shape[3] != HEAD_DIM:
        raise ValueError(f"{name} must have shape [{cache.batch}, heads, tokens, {HEAD_DIM}], not {tuple(shape)}")
    if tensor.dtype not in _DTYPES:
        raise TypeError(f"{name} must use bfloat16, float16 or float32, not {tensor.dtype}")
    if tensor.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient; the 8-bit cache has no backward pass (use torch.no_grad())")


def _check_counts(cache: QuantizedKVCache, counts: torch.Tensor | None) -> torch.Tensor | None:
    if counts is None:
        return None
    if counts.dtype != torch.int32 or counts.shape != (cache.batch,):
        raise TypeError(f"counts must be an int32 vector of one entry a sequence ({cache.batch})")
    return counts.contiguous()


def _call(device: torch.device, function, *args) -> None:
    """Calls a C entry on the current stream of ``device``."""
    if device.index == torch.cuda.current_device():
        rc = function(*args, nat.stream_handle(device))
    else:
        with torch.cuda.device(device):
            rc = function(*args, nat.stream_handle(device))
    if rc:
        nat.check(rc)


def quantized_append(cache: QuantizedKVCache, key: torch.Tensor, value: torch.Tensor, *,
                     counts: torch.Tensor | None = None) -> None:
    """Quantises ``key``/``value`` [batch, kv_heads, tokens, 128] (bf16, fp16 or
    f32, any strides) behind every sequence's rows: the first ``counts[b]``
    tokens (int32 on the device, clamped to [0, tokens]) or all of them.

    Tokens past the capacity are dropped and raise the overflow flag
    (``assert_no_overflow``).  A value that is not finite is stored as NaN."""
    _check_rows(cache, "key", key)
    _check_rows(cache, "value", value)
    if key.shape[1] != cache._struct.kv_heads or value.shape != key.shape:
        raise ValueError(f"key and value must both have {cache.kv_heads} heads and the same tokens")
    if value.dtype != key.dtype:
        raise TypeError("key and value must share a dtype")
    counts = _check_counts(cache, counts)
    device = nat.require_device(cache.key_codes, key, value, *(() if counts is None else (counts,)))
    tokens = key.shape[2]
    if tokens == 0:
        return
    key_rows, key = _rows(key)
    value_rows, value = _rows(value)
    _call(device, nat.lib().ckv_quant_append, cache._ref, ctypes.byref(key_rows),
          ctypes.byref(value_rows), tokens, nat.ptr(counts), _DTYPES[key.dtype])


def quantized_attention(query: torch.Tensor, cache: QuantizedKVCache, *, softmax_scale: float,
                        counts: torch.Tensor | None = None, window: int = 0,
                        accumulate: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of the newest tokens, already appended, over the cache.

    ``query`` [batch, query heads, tokens, 128] (bf16, fp16 or f32, any
    strides) are the queries of the last ``tokens`` tokens, or of the last
    ``counts[b]`` in the first ``counts[b]`` places.  A query attends the rows
    at positions up to its own and, with ``window`` > 0, of the last
    ``window`` positions (its own among them).  ``accumulate`` adds the
    probability that each row received, summed over the queries and the heads
    of its group, to ``cache.weights``; a query whose softmax is NaN gives NaN
    to the rows that it attends.

    Returns (output [batch, tokens, query heads, 128] in the queries' dtype,
    lse [batch, query heads, tokens] float32, natural log); a query that
    attends nothing gives zeros and -inf."""
    _check_rows(cache, "query", query)
    if query.shape[1] % cache.kv_heads or not 1 <= query.shape[1] // cache.kv_heads <= nat.MAX_GROUP:
        raise ValueError(f"query heads must be 1 to {nat.MAX_GROUP} times the {cache.kv_heads} KV heads, "
                         f"not {query.shape[1]}")
    if not 0.0 < softmax_scale <= 1e30:
        raise ValueError("softmax_scale must be positive and finite")
    if window < 0:
        raise ValueError("window must be non-negative")
    if accumulate and cache.weights is None:
        raise ValueError("accumulate needs a cache that tracks weights")
    counts = _check_counts(cache, counts)
    device = nat.require_device(cache.key_codes, query, *(() if counts is None else (counts,)))
    batch, heads, tokens, _ = query.shape
    out = torch.empty((batch, tokens, heads, HEAD_DIM), dtype=query.dtype, device=device)
    lse = torch.empty((batch, heads, tokens), dtype=torch.float32, device=device)
    if tokens == 0:
        return out, lse
    lib = nat.lib()
    dtype = _DTYPES[query.dtype]
    call = (heads, tokens, dtype, accumulate)
    size = cache._sizes.get(call)
    if size is None:
        size = cache._sizes[call] = lib.ckv_quant_attention_workspace_bytes(cache._ref, heads, tokens, dtype, accumulate)
    workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    rows, query = _rows(query)
    _call(device, lib.ckv_quant_attention, cache._ref, ctypes.byref(rows), heads, tokens, nat.ptr(counts), dtype,
          softmax_scale, min(window, 2**31 - 1), accumulate, out.data_ptr(), lse.data_ptr(), nat.ptr(workspace))
    return out, lse


def evict(cache: QuantizedKVCache, *, keep: int, num_sink: int = 0, recent: int = 0,
          into: QuantizedKVCache | None = None) -> None:
    """Reduces every sequence of more than ``keep`` rows to ``keep`` rows a KV
    head: the first ``num_sink`` positions and the newest ``recent`` ones that
    are still there, then the rows that received the most attention
    (``cache.weights``), equal ones by the lower row.

    Rows that stay keep their place; each freed row below ``keep`` takes a kept
    row from above, so the order of the rows changes but not the set (masks go
    by position).  A moved row is written by the append's scale rule: exact
    unless its value is an E4M3 subnormal of the new block.  In place by
    default (the addresses stay, so a step may be captured around it);
    ``into``: the rows and cursors go to another cache of the same batch, heads
    and block that shares no memory with this one, which stays as it is; the
    weights go along if the other cache tracks them.  Evict between steps: after
    a call's attention, before the next append."""
    if cache.weights is None:
        raise ValueError("evict needs a cache that tracks weights")
    if keep <= 0 or num_sink < 0 or recent < 0 or num_sink + recent > keep:
        raise ValueError("keep must be positive and hold num_sink + recent rows")
    if into is not None:
        if into is cache or into.key_codes.data_ptr() == cache.key_codes.data_ptr():
            raise ValueError("into must be another cache")
        if (into.batch, into.kv_heads, into.block) != (cache.batch, cache.kv_heads, cache.block):
            raise ValueError("into must have the cache's batch, heads and block")
        if into.capacity < min(keep, cache.capacity):
            raise ValueError(f"into holds {into.capacity} rows, keep needs {min(keep, cache.capacity)}")
    device = nat.require_device(cache.key_codes, *(() if into is None else (into.key_codes,)))
    keep = min(keep, cache.capacity)  # a lower one holds the protected rows; at the capacity no row is chosen
    num_sink = min(num_sink, keep)
    recent = min(recent, keep - num_sink)
    lib = nat.lib()
    size = lib.ckv_quant_evict_workspace_bytes(cache._ref, keep)
    workspace = torch.empty(size, dtype=torch.uint8, device=device)
    _call(device, lib.ckv_quant_evict, cache._ref, None if into is None else into._ref, keep, num_sink, recent,
          workspace.data_ptr())


__all__ = ["QuantizedKVCache", "evict", "quantized_append", "quantized_attention"]
