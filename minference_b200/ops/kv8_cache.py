"""The 8-bit key/value cache of one layer and the operators over it: store, load, attention, eviction.

What the sparse prefill leaves behind is the K and V of a long prompt, and every decoding step reads all of it.  Here
it is held in 8 bits (e4m3 or int8) with one fp32 scale for each block of 64 tokens of a head; the tokens behind the
last complete block stay in bf16 until their block fills.  The attention weights that decoding gives each token can be
summed up on the way, and ``kv8_evict`` keeps the tokens that hold most of them.

Sequences of a batch may hold different numbers of tokens.  Lengths and positions are Python integers (checked here)
or int32 tensors ``[B]`` on the device, which keeps a decoding step free of synchronisation and fit for a CUDA graph; a
value that does not fit is then reported in ``cache.status`` (``cache.check()`` raises for it) and clipped.
The reference has no counterpart (its quantised cache is a 2-bit one of another package).
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from .. import _cabi

BLOCK = 64          # tokens that share a scale
HEAD_DIM = 128
_FORMATS = {torch.float8_e4m3fn: _cabi.KV8_E4M3, torch.int8: _cabi.KV8_INT8}


_I64x3 = ctypes.c_int64 * 3


@functools.lru_cache(maxsize=1024)
def _scratch_bytes(batch: int, hq: int, heads: int, n_q: int, max_length: int, with_weights: bool) -> int:
    return _cabi.lib().minf_kv8_attention_scratch_bytes(batch, hq, heads, n_q, max_length, with_weights)


@functools.lru_cache(maxsize=None)
def _like(device, dtype):
    """An empty tensor to make others like: the cheapest way to allocate."""
    return torch.empty(0, dtype=dtype, device=device)


# the current stream's handle without a Stream object around it, where torch offers that (2 us less a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _launch(entry: str, cache, *args) -> None:
    """Call a C entry point with the current stream of the cache's device appended.  The device is switched only where it
    is not the current one: a decoding step is a few microseconds of work."""
    index = cache.device.index
    fn = getattr(_cabi.lib(), entry)
    if torch.cuda.current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _cabi.check(rc)


def _fail(msg: str):
    raise _cabi.MInferB200Error(msg)


class KV8Cache:
    """Tensors of one layer's cache: ``k, v [B, Hkv, capacity, 128]`` codes (``torch.float8_e4m3fn`` or ``torch.int8``),
    ``k_scale, v_scale [B, Hkv, capacity / 64]`` fp32, ``k_tail, v_tail [B, Hkv, 64, 128]`` bf16 (token t of the last,
    incomplete block in row ``t % 64``), all contiguous on one CUDA device.  The number of tokens held is the caller's
    (it is an argument of every call), so one cache serves captured graphs whose lengths change between replays.

    Tokens are dropped from the end by going on with a smaller number of them: a multiple of 64, or one that ends in the block
    that was incomplete, whose tokens the tail holds.  To go back from n to m tokens inside a complete block, put its values into
    the tail first: ``cache.k_tail[:], cache.v_tail[:] = kv8_load(cache, n, first=m // 64 * 64, count=64)`` (rounded by their 8
    bits then)."""

    def __init__(self, k, v, k_scale, v_scale, k_tail, v_tail):
        _cabi.require_cuda(k, v, k_scale, v_scale, k_tail, v_tail)
        _cabi.lib()
        if k.dtype not in _FORMATS or v.dtype != k.dtype:
            _fail(f"cache codes must both be float8_e4m3fn or int8 (got {k.dtype}, {v.dtype})")
        if k.dim() != 4 or k.shape[3] != HEAD_DIM or k.shape[2] % BLOCK or k.shape[2] == 0:
            _fail(f"cache codes must be [B, Hkv, capacity, {HEAD_DIM}] with a capacity that is a multiple of {BLOCK} (got {tuple(k.shape)})")
        b, h, cap, d = k.shape
        for t, shape, dtype in ((v, k.shape, k.dtype), (k_scale, (b, h, cap // BLOCK), torch.float32), (v_scale, (b, h, cap // BLOCK), torch.float32),
                                (k_tail, (b, h, BLOCK, d), torch.bfloat16), (v_tail, (b, h, BLOCK, d), torch.bfloat16)):
            if t.shape != torch.Size(shape) or t.dtype != dtype:
                _fail(f"cache tensor {tuple(t.shape)} {t.dtype} where {tuple(shape)} {dtype} was expected")
        for t in (k, v, k_scale, v_scale, k_tail, v_tail):
            if not t.is_contiguous() or t.data_ptr() % 16:
                _fail("cache tensors must be contiguous and 16-byte aligned")
            if t.device != k.device:
                _fail("cache tensors must be on one device")
        self._set(k, v, k_scale, v_scale, k_tail, v_tail, _cabi.new_status(k.device))

    def _set(self, k, v, k_scale, v_scale, k_tail, v_tail, status):
        self._tensors = (k, v, k_scale, v_scale, k_tail, v_tail)
        self.batch, self.kv_heads, self.capacity, _ = k.shape
        self.dtype, self.device, self.status = k.dtype, k.device, status
        self._desc = _cabi.Kv8Desc(*[t.data_ptr() for t in self._tensors], status.data_ptr(), self.batch, self.kv_heads, self.capacity, _FORMATS[k.dtype])
        self._ref = ctypes.byref(self._desc)

    def _sibling(self, capacity: int):
        """An empty cache like this one; it reports into this one's status.  Its tensors are views of one allocation, made when
        somebody asks for them."""
        b, h, cap = self.batch, self.kv_heads, (capacity + BLOCK - 1) // BLOCK * BLOCK
        codes, scales, tails = b * h * cap * HEAD_DIM, (b * h * cap // BLOCK * 4 + 15) // 16 * 16, b * h * BLOCK * HEAD_DIM * 2
        new = KV8Cache.__new__(KV8Cache)
        new.batch, new.kv_heads, new.capacity, new.dtype, new.device, new.status = b, h, cap, self.dtype, self.device, self.status
        new._tensors = None
        new._storage = self.status.new_empty((2 * (codes + scales + tails)) // 4)
        at = new._storage.data_ptr()
        new._places = (0, codes, 2 * codes, 2 * codes + scales, 2 * (codes + scales), 2 * (codes + scales) + tails)
        new._desc = _cabi.Kv8Desc(*[at + x for x in new._places], self.status.data_ptr(), b, h, cap, _FORMATS[self.dtype])
        new._ref = ctypes.byref(new._desc)
        return new

    def _views(self):
        if self._tensors is None:
            b, h, cap, raw = self.batch, self.kv_heads, self.capacity, self._storage.view(torch.uint8)
            shapes = [((b, h, cap, HEAD_DIM), self.dtype)] * 2 + [((b, h, cap // BLOCK), torch.float32)] * 2 + [((b, h, BLOCK, HEAD_DIM), torch.bfloat16)] * 2
            self._tensors = tuple(raw[at: at + math.prod(shape) * dtype.itemsize].view(dtype).view(shape)
                                  for at, (shape, dtype) in zip(self._places, shapes))
        return self._tensors

    k = property(lambda self: self._views()[0])
    v = property(lambda self: self._views()[1])
    k_scale = property(lambda self: self._views()[2])
    v_scale = property(lambda self: self._views()[3])
    k_tail = property(lambda self: self._views()[4])
    v_tail = property(lambda self: self._views()[5])

    @classmethod
    def empty(cls, batch: int, kv_heads: int, capacity: int, dtype=torch.float8_e4m3fn, device="cuda"):
        """A cache with room for ``capacity`` tokens (rounded up to whole blocks)."""
        if batch < 1 or kv_heads < 1 or capacity < 1:
            _fail(f"bad cache sizes: batch {batch}, kv_heads {kv_heads}, capacity {capacity}")
        cap = (capacity + BLOCK - 1) // BLOCK * BLOCK
        codes = lambda: torch.empty((batch, kv_heads, cap, HEAD_DIM), dtype=dtype, device=device)
        scale = lambda: torch.empty((batch, kv_heads, cap // BLOCK), dtype=torch.float32, device=device)
        tail = lambda: torch.empty((batch, kv_heads, BLOCK, HEAD_DIM), dtype=torch.bfloat16, device=device)
        return cls(codes(), codes(), scale(), scale(), tail(), tail())

    def check(self) -> None:
        """Synchronising check that every length and position so far fitted; clears what it reports."""
        bits = int(self.status[_cabi.ST_ERROR])
        if bits:
            self.status.zero_()
            _fail(f"8-bit cache: device reported error bits {bits:#x} (16 = a length or position outside the cache of "
                  f"{self.capacity} tokens, or outside max_length; 1 = an abandoned wait)")

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self._views())


def _per_sequence(cache: KV8Cache, x, what: str, low: int, high: int):
    """(device pointer or None, host value, tensor to keep alive) of an int or an int32 tensor ``[B]``."""
    if isinstance(x, torch.Tensor):
        if x.dtype != torch.int32 or x.shape != (cache.batch,) or x.device != cache.device or not x.is_contiguous():
            _fail(f"{what} must be an int or a contiguous int32 tensor [{cache.batch}] on {cache.device} (got {x.dtype} {tuple(x.shape)} on {x.device})")
        return x.data_ptr(), 0
    x = int(x)
    if not low <= x <= high:
        _fail(f"{what} {x} is outside [{low}, {high}]")
    return None, x


def _rows(t: torch.Tensor, what: str, cache: KV8Cache):
    shape = t.shape
    if len(shape) != 4 or shape[0] != cache.batch or shape[3] != HEAD_DIM or t.dtype != torch.bfloat16 or t.device != cache.device:
        _fail(f"{what} must be bf16 [{cache.batch}, heads, tokens, {HEAD_DIM}] on {cache.device} (got {t.dtype} {tuple(t.shape)} on {t.device})")
    s0, s1, s2, s3 = t.stride()
    if s3 != 1 or (s0 | s1 | s2) & 7 or t.data_ptr() & 15:
        t = t.clone(memory_format=torch.contiguous_format)      # (contiguous() leaves a contiguous tensor at an odd address where it is)
    return t


@functools.lru_cache(maxsize=4096)
def _c_strides(*strides):
    return _I64x3(*strides[:3])


def _strides(t: torch.Tensor):
    """The first three strides for a C entry point (the array of equal ones is made once: it is only read)."""
    return _c_strides(*t.stride())


def kv8_store(cache: KV8Cache, key: torch.Tensor, value: torch.Tensor, start, counts=None) -> None:
    """Append tokens ``key, value [B, Hkv, n, 128]`` (bf16) behind the ``start`` tokens each sequence holds (an int or an
    int32 tensor ``[B]``; ``KV8Cache`` says how to drop tokens before); of a padded batch only the first ``counts[b]`` of the
    n.  One token and whole prompts take the same call.  A block that fills is quantised from its 64 tokens' bf16 values.  Only
    the touched blocks are written."""
    key, value = _rows(key, "key", cache), _rows(value, "value", cache)
    _, h, n, _ = shape = key.shape
    if h != cache.kv_heads or shape != value.shape:
        _fail(f"key and value must be [{cache.batch}, {cache.kv_heads}, n, {HEAD_DIM}] both (got {tuple(shape)}, {tuple(value.shape)})")
    dev_counts = None
    if counts is not None:
        if not isinstance(counts, torch.Tensor):
            _fail("counts must be an int32 tensor")
        dev_counts, _ = _per_sequence(cache, counts, "counts", 0, n)
    dev_start, start = _per_sequence(cache, start, "start", 0, cache.capacity - (n if counts is None else 0))
    _launch("minf_kv8_store", cache, cache._ref, key.data_ptr(), value.data_ptr(), _strides(key), _strides(value), n, dev_start, start, dev_counts)


def kv8_load(cache: KV8Cache, lengths, first=0, count: int | None = None):
    """Values of tokens ``first .. first + count`` (``count=None``, for an int ``first``: to the end of the capacity) as
    ``(k, v)``, bf16 ``[B, Hkv, count, 128]``; zeros outside ``[0, length)``.  ``lengths`` and ``first``: int or int32 tensor ``[B]``."""
    dev_n, n = _per_sequence(cache, lengths, "lengths", 0, cache.capacity)
    if count is None:
        if isinstance(first, torch.Tensor):
            _fail("count must be given where first is a tensor")
        count = cache.capacity - int(first)
    dev_first, first = _per_sequence(cache, first, "first", -(1 << 30), 1 << 30)
    if count < 0:
        _fail(f"count {count} must not be negative")
    shape = (cache.batch, cache.kv_heads, count, HEAD_DIM)
    like = _like(cache.device, torch.bfloat16)
    k, v = like.new_empty(shape), like.new_empty(shape)
    _launch("minf_kv8_load", cache, cache._ref, dev_n, n, dev_first, first, count, k.data_ptr(), v.data_ptr())
    return k, v


def _weights_arg(t, what: str, cache: KV8Cache, max_length: int):
    if t.dtype != torch.float32 or t.dim() != 3 or t.shape[:2] != (cache.batch, cache.kv_heads) or t.shape[2] < max_length or t.device != cache.device:
        _fail(f"{what} must be fp32 [{cache.batch}, {cache.kv_heads}, >= {max_length}] on {cache.device} (got {t.dtype} {tuple(t.shape)} on {t.device})")
    if t.stride(2) != 1 and t.shape[2] > 1:
        _fail(f"{what} must be contiguous along its tokens")


def _extent(t: torch.Tensor):
    """First and last byte address of a tensor's elements."""
    return t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _check_written(weights: torch.Tensor, add_to: torch.Tensor | None, tokens: int) -> None:
    """No element of ``weights`` may be written twice (the first ``tokens`` of every head are), or be read as ``add_to`` of
    another token."""
    (b, h, _), (sb, sh, _) = weights.shape, weights.stride()
    if not ((h == 1 or sh >= tokens) and (b == 1 or sb >= (h - 1) * sh + tokens)):      # (as a contiguous tensor has them)
        starts = sorted(i * sb + j * sh for i in range(b) for j in range(h))
        if any(y - x < tokens for x, y in zip(starts, starts[1:])):
            _fail("weights must not be an expanded or overlapping view: its elements are written")
    if add_to is not None and add_to is not weights:
        a, b = _extent(weights), _extent(add_to)
        if a[0] < b[1] and b[0] < a[1] and (a[0] != b[0] or weights.stride() != add_to.stride()):
            _fail("add_to overlaps weights without being the same view")


def _max_length(cache: KV8Cache, lengths, max_length):
    if max_length is None:
        return cache.capacity if isinstance(lengths, torch.Tensor) else int(lengths)
    if not 0 <= max_length <= cache.capacity:
        _fail(f"max_length {max_length} is outside [0, {cache.capacity}]")
    return int(max_length)


class _ForwardOnly(torch.autograd.Function):
    """The attention of queries that require a gradient: there is no backward pass, so one that would need it is an error."""

    @staticmethod
    def forward(ctx, *args):
        return kv8_attention(*args)

    @staticmethod
    def backward(ctx, *grads):
        _fail("kv8_attention is forward only: no gradient can pass through it")


def kv8_attention(query: torch.Tensor, cache: KV8Cache, lengths, max_length: int | None = None, sm_scale: float | None = None,
                  weights: torch.Tensor | None = None, add_to: torch.Tensor | None = None, return_lse: bool = False):
    """Attention of the last S tokens of every sequence, ``query [B, H, S, 128]`` (bf16, H a multiple of the cache's
    heads), over the cache that already holds them: query i of a sequence of n tokens sees its first ``n - S + 1 + i``.
    Returns ``[B, H, S, 128]`` bf16 (in memory in the query's order of dimensions) and, with ``return_lse``, the base-2 log-sum-exp of the scaled logits, fp32
    ``[B, H, S]``.  A row that sees nothing gives zeros and -inf.

    ``lengths``: int or int32 tensor ``[B]``, the new tokens included; ``max_length``: an upper bound of them known on the
    host (the capacity if not given), by which the work is split and scratch memory sized.
    ``weights [B, Hkv, >= max_length]`` fp32 receives the attention weight of each token -- the probabilities summed over
    the head's queries -- plus ``add_to`` (``add_to=weights`` sums up in place); entries behind a sequence's length are
    left as they were.  It takes scratch memory of 4 bytes for every query row and token.
    Forward only: a backward pass through it raises.  One to 24 rows per cache head (H / Hkv * S) and more take different
    kernels; both are within the roundings of P to 16 bits of the exact result.
    """
    if query.requires_grad and torch.is_grad_enabled():
        return _ForwardOnly.apply(query, cache, lengths, max_length, sm_scale, weights, add_to, return_lse)
    query = _rows(query, "query", cache)
    b, hq, s, d = query.shape
    if s < 1 or hq % cache.kv_heads:
        _fail(f"query must be [B, H, S >= 1, {HEAD_DIM}] with H a multiple of {cache.kv_heads} (got {tuple(query.shape)})")
    longest = _max_length(cache, lengths, max_length)
    dev_n, n = _per_sequence(cache, lengths, "lengths", 0, longest)
    if weights is not None:
        _weights_arg(weights, "weights", cache, longest)
    if add_to is not None:
        if weights is None:
            _fail("add_to without weights")
        _weights_arg(add_to, "add_to", cache, longest)
    if weights is not None:
        _check_written(weights, add_to, longest)
    out = torch.empty_like(query)           # in the query's order of dimensions: what a projection behind it wants
    lse = _like(cache.device, torch.float32).new_empty((b, hq, s)) if return_lse else None
    nbytes = _scratch_bytes(b, hq, cache.kv_heads, s, longest, weights is not None)
    scratch = cache.status.new_empty(nbytes // 4) if nbytes else None       # (in words of four bytes)
    _launch("minf_kv8_attention", cache,
            cache._ref, query.data_ptr(), _strides(query), out.data_ptr(), _strides(out), hq, s, dev_n, n, longest,
            d ** -0.5 if sm_scale is None else float(sm_scale), lse.data_ptr() if return_lse else None,
            weights.data_ptr() if weights is not None else None, _strides(weights) if weights is not None else None,
            add_to.data_ptr() if add_to is not None else None, _strides(add_to) if add_to is not None else None,
            scratch.data_ptr() if nbytes else None)
    return (out, lse) if return_lse else out


def kv8_evict(cache: KV8Cache, lengths, weights: torch.Tensor, budget: int, recent: int, sink: int = 0,
              max_length: int | None = None, out: KV8Cache | None = None):
    """Keep ``budget`` tokens of every head: the first ``sink``, the last ``recent`` and those with the largest ``weights
    [B, Hkv, >= max_length]`` (fp32, as ``kv8_attention`` sums them up) of the others; equal weights: the earlier token, NaN
    is the largest.
    Sequences of ``budget`` tokens or fewer are copied.

    Writes into ``out`` (another cache of the same type, batch and heads; a new one with room for ``budget`` tokens, which
    reports into this cache's status, if not given) and returns ``(out, lengths int32 [B], weights fp32 [B, Hkv, out.capacity] -- zeros behind the last --, kept int32
    [B, Hkv, budget] -- old positions, ascending, -1 behind the last)``.  Keys keep the rotary phase they were stored
    with: the caller goes on counting positions from the full sequence."""
    budget, recent, sink = int(budget), int(recent), int(sink)
    if budget < 1 or recent < 0 or sink < 0 or recent + sink > budget:
        _fail(f"budget {budget} must hold the {sink} first and {recent} last tokens")
    longest = _max_length(cache, lengths, max_length)
    dev_n, n = _per_sequence(cache, lengths, "lengths", 0, longest)
    _weights_arg(weights, "weights", cache, longest)
    if out is None:
        out = cache._sibling(budget)
    elif out is cache or (out.batch, out.kv_heads, out.dtype, out.device) != (cache.batch, cache.kv_heads, cache.dtype, cache.device) or out.capacity < budget:
        _fail("out must be another cache of the same batch, heads, type and device with room for the budget")
    kept = cache.status.new_empty((cache.batch, cache.kv_heads, budget))
    weights_out = _like(cache.device, torch.float32).new_empty((cache.batch, cache.kv_heads, out.capacity))
    lengths_out = cache.status.new_empty((cache.batch,))
    _launch("minf_kv8_evict", cache, cache._ref, out._ref, dev_n, n, longest, weights.data_ptr(), _strides(weights), budget, recent, sink,
            kept.data_ptr(), weights_out.data_ptr(), lengths_out.data_ptr())
    return out, lengths_out, weights_out, kept
