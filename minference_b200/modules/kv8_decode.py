"""One attention layer's keys and values between the sparse prefill and the decoding steps after it.

``KV8Layer`` holds them in an 8-bit cache (``ops/kv8_cache.py``), attends over it for new tokens and, where a budget is
set, sums the attention weights and cuts the cache down by them; the prompt's weights are the estimator's column sums (the
softmax of its last 64 queries), the same numbers the vertical lines are selected by; a model with another logit scale than
1/sqrt(128) takes its own last queries' weights over the cache instead.  ``KV8HFCache`` is the same as a
``past_key_values`` object for a Hugging Face model patched with ``MInference``.  The role of the reference's kv_type
caches (minference/modules/kvcompression.py's SnapKV and its decoding forward); the methods are this repository's own.
"""
from __future__ import annotations

import functools

import torch

from .. import _cabi
from ..ops.kv8_cache import BLOCK, KV8Cache, kv8_attention, kv8_evict, kv8_store
from .minference_forward import last_q, vertical_slash_estimate


def prompt_weights(query: torch.Tensor, key: torch.Tensor) -> torch.Tensor:
    """Attention weight of every prompt token, ``[B, Hkv, N]`` fp32: the probabilities of the last 64 queries summed over
    them and over each key head's query heads (the estimator's vertical scores)."""
    b, h, n, _ = query.shape
    *_, vertical, _ = vertical_slash_estimate(query, key, 30, 50, return_scores=True)
    hkv = key.shape[1]
    return vertical.view(b, hkv, h // hkv, n).sum(2)


class KV8Layer:
    """Tokens of one layer, the same number for every sequence of the batch.

    ``dtype``: ``torch.float8_e4m3fn`` or ``torch.int8``.  ``budget``: tokens kept per head when the cache is cut down
    (None: never); ``sink`` first and ``recent`` last tokens are always kept (``recent=None``: a quarter of the budget).
    The cache is cut down after the prompt, and again whenever ``slack`` more tokens than the budget have come in.
    ``seen`` counts all tokens (the next one's position), ``held`` those in the cache; ``cache.check()`` raises for what the
    device reported since the layer was last reset.  ``taken`` is False between the ``update`` of a ``KV8HFCache`` and the
    attention function that takes its tokens."""

    def __init__(self, dtype=torch.float8_e4m3fn, budget: int | None = None, recent: int | None = None, sink: int = 4, slack: int = 256,
                 capacity: int = 0):
        if dtype not in (torch.float8_e4m3fn, torch.int8):
            raise _cabi.MInferB200Error(f"cache codes must be float8_e4m3fn or int8 (got {dtype})")
        if budget is not None:
            recent = budget // 4 if recent is None else recent
            if budget < 1 or recent < 0 or sink < 0 or recent + sink > budget or slack < 1:
                raise _cabi.MInferB200Error(f"budget {budget} must hold the {sink} first and {recent} last tokens, slack {slack} be positive")
        self.dtype, self.budget, self.recent, self.sink, self.slack, self.capacity = dtype, budget, recent, sink, slack, capacity
        self.reset()

    def reset(self) -> None:
        self.cache: KV8Cache | None = None
        self.sums: torch.Tensor | None = None
        self.held = self.seen = 0
        self.taken = True

    def _room(self, key: torch.Tensor) -> None:
        b, h, n, _ = key.shape
        need = self.held + n
        if self.cache is not None and need <= self.cache.capacity:
            return
        # the prompt and what decoding adds to it; doubled when that runs out
        cap = max(self.capacity, need + 512 if self.cache is None else 2 * need)
        new = KV8Cache.empty(b, h, cap, self.dtype, key.device) if self.cache is None else self.cache._sibling(cap)
        sums = torch.zeros((b, h, new.capacity), dtype=torch.float32, device=key.device) if self.budget is not None else None
        if self.cache is not None and self.held:
            self._copy(new)
            if sums is not None:
                sums[..., : self.held] = self.sums[..., : self.held]
        self.cache, self.sums = new, sums

    def _copy(self, new: KV8Cache) -> None:
        old, blocks = self.cache, self.held // BLOCK
        for name in ("k", "v"):
            getattr(new, name)[:, :, : blocks * BLOCK] = getattr(old, name)[:, :, : blocks * BLOCK]
            getattr(new, name + "_scale")[..., :blocks] = getattr(old, name + "_scale")[..., :blocks]
            getattr(new, name + "_tail").copy_(getattr(old, name + "_tail"))

    def append(self, key: torch.Tensor, value: torch.Tensor) -> None:
        """Store new tokens ``[B, Hkv, n, 128]`` behind those held."""
        if self.cache is not None and (key.shape[0], key.shape[1]) != (self.cache.batch, self.cache.kv_heads):
            raise _cabi.MInferB200Error(f"the layer holds {self.cache.batch} sequences of {self.cache.kv_heads} heads (got {tuple(key.shape)})")
        self._room(key)
        kv8_store(self.cache, key, value, self.held)
        self.held += key.shape[2]
        self.seen += key.shape[2]

    def attend(self, query: torch.Tensor, sm_scale: float | None = None) -> torch.Tensor:
        """Attention of the last tokens appended, ``query [B, H, S, 128]``; their weights are added up where a budget is
        set, and the cache cut down once it is ``slack`` tokens over it.  Of more than 64 new tokens the last 64 count, as of a
        prompt: a long follow-up does not outweigh all that came before, nor need 4 bytes for each of its rows and tokens held."""
        if self.cache is None:
            raise _cabi.MInferB200Error("the layer holds no tokens")
        weights = {} if self.budget is None else {"weights": self.sums, "add_to": self.sums}
        if not weights or query.shape[2] <= last_q:
            out = kv8_attention(query, self.cache, self.held, sm_scale=sm_scale, **weights)
        else:
            out = kv8_attention(query, self.cache, self.held, sm_scale=sm_scale)
            kv8_attention(query[:, :, -last_q:], self.cache, self.held, sm_scale=sm_scale, **weights)
        if self.budget is not None and self.held >= self.budget + self.slack:
            self.evict()
        return out

    def after_prompt(self, query: torch.Tensor, key: torch.Tensor, sm_scale: float | None = None) -> None:
        """Cut the prompt down to the budget by its own weights (``query`` and ``key`` as its attention saw them)."""
        if self.budget is None:
            return
        plain = query.shape[-1] ** -0.5
        if sm_scale is None or abs(float(sm_scale) - plain) <= 1e-6 * plain:
            self.sums[..., : self.held] = prompt_weights(query, key)
        else:
            # the estimator knows no other scale: the same queries' weights over the cache, one query head of each cache head
            # at a time, because a call needs 4 bytes for every row and token
            last, hkv = query[:, :, -last_q:], self.cache.kv_heads
            for g in range(query.shape[1] // hkv):
                kv8_attention(last.unflatten(1, (hkv, -1))[:, :, g], self.cache, self.held, sm_scale=sm_scale, weights=self.sums,
                              add_to=self.sums if g else None)
        if self.held > self.budget:
            self.evict()

    def evict(self) -> None:
        """Cut the cache down to the budget."""
        if self.budget is None or self.cache is None:
            raise _cabi.MInferB200Error("the layer has no budget" if self.budget is None else "the layer holds no tokens")
        out = self.cache._sibling(self.budget + self.slack + 1)
        self.cache, _, self.sums, _ = kv8_evict(self.cache, self.held, self.sums, self.budget, recent=self.recent, sink=self.sink, out=out)
        self.held = min(self.held, self.budget)


@functools.lru_cache(maxsize=1)
def _hf_base():
    from transformers.cache_utils import Cache, CacheLayerMixin

    class Layer(CacheLayerMixin):
        """A layer of ``KV8HFCache``.  ``update`` returns the new tokens only, marked with the layer that holds the others:
        the patched attention function attends over the 8-bit cache.  A function that does not know the mark would attend
        over the new tokens alone, so the next ``update`` of any layer (``last``, shared by the cache's layers, is the one before
        it) looks whether they were taken: in the same pass of the model if it has two layers or more."""
        is_sliding = False

        def __init__(self, make, last):
            super().__init__()
            self.kv, self.last = make(), last
            self.is_initialized = True

        def lazy_initialization(self, key_states, value_states):
            pass

        def update(self, key_states, value_states, *args, **kwargs):
            if key_states.shape[0] != 1:
                raise _cabi.MInferB200Error("the 8-bit cache of a Hugging Face model takes one sequence, like the sparse prefill")
            if self.last and not self.last[0].taken:
                raise _cabi.MInferB200Error("no attention function took the tokens that were last put into the 8-bit cache: the model is not "
                                            "patched with MInference, or makes other tensors of the keys before its attention")
            self.kv.append(key_states, value_states)
            self.kv.taken, self.last[:] = False, [self.kv]
            key_states = key_states.view(key_states.shape)      # a tensor object of its own to carry the mark
            key_states.minf_kv8 = self.kv
            return key_states, value_states

        def get_seq_length(self):
            return self.kv.seen

        def get_mask_sizes(self, query_length):
            return self.kv.seen + query_length, 0

        def get_max_cache_shape(self):
            return -1

        def reset(self):
            self.kv.reset()

        def _refuse(self, *args, **kwargs):
            raise _cabi.MInferB200Error("the 8-bit cache cannot be cropped, reordered, offloaded or resized in its batch")

        offload = prefetch = reorder_cache = crop = batch_repeat_interleave = batch_select_indices = _refuse

    class KV8HFCache(Cache):
        def __init__(self, **options):
            last = []
            super().__init__(layer_class_to_replicate=lambda: Layer(lambda: KV8Layer(**options), last))

    return KV8HFCache


def KV8HFCache(dtype=torch.float8_e4m3fn, budget: int | None = None, recent: int | None = None, sink: int = 4, slack: int = 256, capacity: int = 0):
    """``past_key_values`` for a model patched with ``MInference(...)(model)``: keys and values in 8 bits, options as in
    ``KV8Layer``.  One sequence; ``model(ids, past_key_values=KV8HFCache(...))`` or ``model.generate(...)``.  A model that is not
    patched is refused."""
    KV8Layer(dtype, budget, recent, sink, slack, capacity)       # the options' own checks, now rather than at the first token
    return _hf_base()(dtype=dtype, budget=budget, recent=recent, sink=sink, slack=slack, capacity=capacity)
