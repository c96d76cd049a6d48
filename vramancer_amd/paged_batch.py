"""Batched decode of Hugging Face models over the paged KV cache: the decode
step of VRAMancer's continuous batcher (core/continuous_batcher.py:693-816)
with the paged kernel in place of pad-and-concat.

The reference coalesces the decode requests into one forward by
concatenating their per-request Hugging Face caches, padding the shorter ones
to the longest with zeros (left padding) and masking the padding (:711-756,
:818-891), so every step copies every request's whole cache; the model then
places every request's new token at the padded length.  Here the requests' K/V stay
in the pages of a ``PagedKVCacheManager``, and ``PagedBatchCache`` is the
Hugging Face ``Cache`` of an ordered batch of request ids:

* the update of layer 0 starts a step: the manager appends one token to every
  request (``append_tokens``: a page id and slot each, a page allocated where
  the last one is full);
* each layer's update writes its new K/V rows into those slots with one
  ``vrm_kv_write`` launch (``write_kv_batch``) and tags the key it returns
  with the batch and the layer;
* the attention function registered as ``"vramancer_paged"``
  (``enable_paged_attention``) sees the tag and runs the paged decode of that
  layer over the batch's block table, which the manager builds on the device
  once per step.  Each request attends exactly its own tokens: no padding, no
  mask, no copy of the cache.

``decode_step`` runs one step of a batch, each request at its own position
(its token count, as a request decoded alone by ``_forward_single`` is), and
returns the last-position logits; ``prefill`` runs a
request's prompt through the model with an ordinary cache and stores the
result in its pages (``from_hf_cache``), as the reference batcher does after
its prefill (:594-597).

Only decode steps (one new token per request) go through a
``PagedBatchCache``; its multi-token update raises.  ``PagedChunkCache`` is its
form for several tokens per request: the update writes them into their pages
and the attention function attends them there
(``PagedKVCacheManager.append_chunk`` and what takes its batch).  ``chunk_step``
runs one such step, ``prefill_chunked`` a prompt in chunks, which needs neither
a second copy of the cache nor scores of the whole prompt.

``sample_step`` is a decode step up to its tokens, drawn on the GPU
(``sampling.sample_tokens``); ``speculative_step`` runs drafted tokens through
the model, verifies them (``sampling.verify_drafts``) and takes those that are
refused out of the pages again.

Calls of the attention function on any other cache attend with PyTorch's SDPA,
causal and unmasked (prefill one request at a time, as the reference does).
"""
from __future__ import annotations

import math
from typing import Any, Optional, Sequence, Tuple

import numpy as np
import torch
from transformers.cache_utils import Cache, CacheLayerMixin

from .paged_attention import ChunkBatch, PagedKVCacheManager

__all__ = ["PagedBatchCache", "PagedBatchLayer", "PagedChunkCache", "PagedChunkLayer", "decode_step", "chunk_step",
           "sample_step", "speculative_step", "prefill", "prefill_chunked", "paged_attention_forward",
           "enable_paged_attention", "ATTENTION_NAME"]

ATTENTION_NAME = "vramancer_paged"


class PagedBatchLayer(CacheLayerMixin):
    """One layer of a ``PagedBatchCache``: writes the step's K/V rows into
    the manager's pages and returns the new states, tagged."""

    is_sliding = False

    def __init__(self, cache: "PagedBatchCache", layer_idx: int):
        super().__init__()
        self.cache = cache
        self.layer_idx = layer_idx

    def lazy_initialization(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        self.dtype, self.device = key_states.dtype, key_states.device
        self.is_initialized = True

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args, **kwargs
               ) -> Tuple[torch.Tensor, torch.Tensor]:
        if not self.is_initialized:
            self.lazy_initialization(key_states, value_states)
        B, _, q, _ = key_states.shape
        if q != 1:
            raise RuntimeError(f"PagedBatchCache takes decode steps of one token per request (got {q}); "
                               "prefill with an ordinary cache and PagedKVCacheManager.from_hf_cache")
        if B != len(self.cache.request_ids):
            raise RuntimeError(f"batch of {B} rows for {len(self.cache.request_ids)} request ids")
        if self.layer_idx == 0:
            self.cache._begin_step()
        page_ids, slots = self.cache._step_slots()
        self.cache.manager.write_kv_batch(self.layer_idx, page_ids, slots, key_states[:, :, 0],
                                          value_states[:, :, 0])
        key_states._vrm_paged_batch = (self.cache, self.layer_idx)
        return key_states, value_states

    def get_seq_length(self) -> int:
        return self.cache.get_seq_length()

    def get_max_length(self) -> int:
        return -1

    def get_max_cache_shape(self) -> int:
        return -1

    def get_mask_sizes(self, query_length) -> Tuple[int, int]:
        q = query_length if isinstance(query_length, int) else query_length.shape[0]
        return self.get_seq_length() + q, 0


class PagedBatchCache(Cache):
    """Hugging Face cache of a batch of requests held by a
    ``PagedKVCacheManager``; batch row i is ``request_ids[i]``.  The cache
    keeps no tensors of its own and can be kept across steps while the batch
    stays the same."""

    def __init__(self, manager: PagedKVCacheManager, request_ids: Sequence[str]):
        if manager.gpu_pool is None:
            raise RuntimeError("PagedBatchCache needs a manager with a GPU pool")
        known = manager.request_ids()
        missing = [rid for rid in request_ids if rid not in known]
        if missing:
            raise KeyError(f"unknown request ids {missing}")
        self.manager = manager
        self.request_ids = list(request_ids)
        self._slots: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
        self._undo: Optional[list] = None  # of the running step, where it is taken back if it fails
        super().__init__(layers=[PagedBatchLayer(self, i) for i in range(manager.config.num_layers)])

    def token_counts(self) -> np.ndarray:
        """Each request's token count (the position of its next token)."""
        return self.manager.token_counts(self.request_ids)

    def _begin_step(self) -> None:
        self._slots = self.manager._append_tokens(self.request_ids, True, self._undo)

    def _watch_step(self) -> None:
        """The next step is one that ``_undo_step`` takes back."""
        self._undo = []

    def _undo_step(self) -> bool:
        """Takes the tokens of a step that failed back; False where a request
        has changed in the meantime, whose tokens stay then."""
        undo, self._undo = self._undo, None
        try:
            for step in undo or []:
                self.manager._take_back(step, self._slots and self._slots[0])
        except RuntimeError:
            return False
        return True

    def _step_slots(self) -> Tuple[torch.Tensor, torch.Tensor]:
        if self._slots is None:
            raise RuntimeError("a decode step starts with the update of layer 0")
        return self._slots

    def get_seq_length(self, layer_idx: int = 0) -> int:
        counts = self.token_counts()
        return int(counts.max()) if counts.size else 0

    def get_max_cache_shape(self, layer_idx: int = 0) -> int:
        return -1

    def attend(self, query: torch.Tensor, layer_idx: int, scale: float) -> torch.Tensor:
        """Paged decode of one layer: query [B, H, 1, D] -> [B, 1, H, D] in
        the query's dtype, the layout attention functions return."""
        out = self.manager.compute_attention_decode(query[:, :, 0].contiguous(), self.request_ids, layer_idx, scale)
        if out is None:
            raise RuntimeError("paged decode over a batch with no pages")
        return out.to(query.dtype).unsqueeze(1)


class PagedChunkLayer(PagedBatchLayer):
    """One layer of a ``PagedChunkCache``: writes the step's K/V rows, as many
    per request as the step has tokens, into the manager's pages."""

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args, **kwargs
               ) -> Tuple[torch.Tensor, torch.Tensor]:
        if not self.is_initialized:
            self.lazy_initialization(key_states, value_states)
        B, _, q, _ = key_states.shape
        if B != len(self.cache.request_ids):
            raise RuntimeError(f"batch of {B} rows for {len(self.cache.request_ids)} request ids")
        if self.layer_idx == 0:
            self.cache._begin_chunk(q)
        chunk = self.cache._step_chunk(q)
        self.cache.manager.write_chunk(self.layer_idx, chunk, key_states.transpose(1, 2).flatten(0, 1),
                                       value_states.transpose(1, 2).flatten(0, 1))
        key_states._vrm_paged_batch = (self.cache, self.layer_idx)
        return key_states, value_states


class PagedChunkCache(PagedBatchCache):
    """``PagedBatchCache`` for steps of several new tokens per request, the
    same number for every request of the batch."""

    def __init__(self, manager: PagedKVCacheManager, request_ids: Sequence[str]):
        super().__init__(manager, request_ids)
        self._chunk: Optional[ChunkBatch] = None
        self.layers = [PagedChunkLayer(self, i) for i in range(manager.config.num_layers)]

    def _begin_chunk(self, q: int) -> None:
        self._chunk = self.manager.append_chunk(self.request_ids, [q] * len(self.request_ids))

    def _watch_step(self) -> None:
        self._chunk = None  # (the step before is no concern of the next one)

    def _undo_step(self) -> bool:
        chunk, self._chunk = self._chunk, None
        try:
            if chunk is not None:
                self.manager._take_back(chunk)
        except RuntimeError:
            return False
        return True

    def _step_chunk(self, q: int) -> ChunkBatch:
        if self._chunk is None or any(n != q for n in self._chunk.counts):
            raise RuntimeError("a step starts with the update of layer 0, and every layer has its tokens")
        return self._chunk

    def attend(self, query: torch.Tensor, layer_idx: int, scale: float) -> torch.Tensor:
        """Attention of one layer over the pages: query [B, H, q, D] ->
        [B, q, H, D] in the query's dtype."""
        B, H, q, D = query.shape
        chunk = self._step_chunk(q)
        out = self.manager.compute_attention_chunk(query.transpose(1, 2).flatten(0, 1), chunk, layer_idx, scale)
        return out.view(B, q, H, D)


def paged_attention_forward(module, query, key, value, attention_mask, dropout: float = 0.0,
                            scaling: Optional[float] = None, **kwargs):
    """Attention function for ``attn_implementation="vramancer_paged"``.

    Keys returned by a ``PagedBatchCache`` are attended by the paged decode
    over the batch's pages; any other call attends with SDPA."""
    from transformers.integrations.sdpa_attention import sdpa_attention_forward

    tag = getattr(key, "_vrm_paged_batch", None)
    if scaling is None:
        scaling = 1.0 / math.sqrt(query.shape[-1])
    if tag is None:
        return sdpa_attention_forward(module, query, key, value, attention_mask, dropout=dropout, scaling=scaling,
                                      **kwargs)
    if dropout or kwargs.get("softcap") is not None or kwargs.get("sliding_window") is not None:
        raise NotImplementedError("paged decode supports neither dropout, softcap nor sliding windows")
    cache, layer_idx = tag
    return cache.attend(query, layer_idx, float(scaling)), None


def enable_paged_attention(model) -> None:
    """Registers ``paged_attention_forward`` and selects it for ``model``."""
    from transformers import AttentionInterface

    AttentionInterface.register(ATTENTION_NAME, paged_attention_forward)
    model.set_attn_implementation(ATTENTION_NAME)


def decode_step(model, manager: PagedKVCacheManager, request_ids: Sequence[str], input_ids: torch.Tensor,
                cache: Optional[PagedBatchCache] = None) -> torch.Tensor:
    """One batched decode step (core/continuous_batcher.py:693-770): token
    ``input_ids[i]`` of request ``request_ids[i]`` at position = that
    request's token count; one forward over the batch.  Returns the logits
    [B, vocab].  The model must use ``enable_paged_attention``; pass the
    ``cache`` of the previous step to reuse it."""
    if cache is None or cache.request_ids != list(request_ids):
        cache = PagedBatchCache(manager, request_ids)
    ids = input_ids.reshape(len(request_ids), 1)
    pos = torch.from_numpy(cache.token_counts()).to(ids.device).reshape(-1, 1)
    out = model(ids, position_ids=pos, past_key_values=cache, use_cache=True)
    logits = out.logits if hasattr(out, "logits") else out[0]
    return logits[:, -1]


def prefill(model, manager: PagedKVCacheManager, request_id: str, input_ids: torch.Tensor) -> torch.Tensor:
    """Runs a request's prompt [1, S] through the model with an ordinary
    cache and stores its K/V in the request's pages (``from_hf_cache``).
    Returns the last-position logits [1, vocab]."""
    out = model(input_ids.reshape(1, -1), use_cache=True)
    manager.from_hf_cache(request_id, out.past_key_values)
    return out.logits[:, -1]


def chunk_step(model, manager: PagedKVCacheManager, request_ids: Sequence[str], input_ids: torch.Tensor,
               cache: Optional[PagedChunkCache] = None) -> torch.Tensor:
    """One forward over q new tokens ``input_ids`` [B, q] of each request, at
    the positions after those it has (a prompt's chunk, drafted tokens to
    verify).  Returns the logits [B, q, vocab].  The model must use
    ``enable_paged_attention``; pass the ``cache`` of the previous step to
    reuse it.  A forward that raises leaves the requests as they were."""
    if not isinstance(cache, PagedChunkCache) or cache.manager is not manager or cache.request_ids != list(request_ids):
        cache = PagedChunkCache(manager, request_ids)
    ids = input_ids.reshape(len(request_ids), -1)
    pos = torch.from_numpy(cache.token_counts()).to(ids.device).reshape(-1, 1)
    pos = pos + torch.arange(ids.shape[1], device=ids.device)
    cache._watch_step()
    try:
        out = model(ids, position_ids=pos, past_key_values=cache, use_cache=True)
    except BaseException:
        cache._undo_step()
        raise
    return out.logits if hasattr(out, "logits") else out[0]


def sample_step(model, manager: PagedKVCacheManager, request_ids: Sequence[str], input_ids: torch.Tensor,
                uniforms: torch.Tensor, temperature: Any = None, top_k: Any = None, top_p: Any = None,
                probs: Any = None, cache: Optional[PagedBatchCache] = None) -> torch.Tensor:
    """``decode_step`` and a token for each request, int64 [B], drawn from its
    logits with ``uniforms`` [B] (``sampling.sample_tokens``).  A step that
    raises leaves the requests as they were.

    A row of logits without a token gives -1.  Such a request is the caller's to
    end; where its -1 is an input again, the model gets token 0 for it."""
    from .sampling import sample_tokens

    if cache is None or cache.manager is not manager or cache.request_ids != list(request_ids):
        cache = PagedBatchCache(manager, request_ids)
    cache._watch_step()
    try:
        logits = decode_step(model, manager, request_ids, input_ids.clamp(min=0), cache)
        tokens = sample_tokens(logits, uniforms, temperature=temperature, top_k=top_k, top_p=top_p, probs=probs)
    except BaseException:
        cache._undo_step()
        raise
    cache._undo = None
    return tokens


def speculative_step(model, manager: PagedKVCacheManager, request_ids: Sequence[str], input_ids: torch.Tensor,
                     drafts: torch.Tensor, accept_uniforms: torch.Tensor, draw_uniforms: torch.Tensor,
                     draft_probs: Any = None, temperature: Any = None, top_k: Any = None, top_p: Any = None,
                     cache: Optional[PagedChunkCache] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One forward over each request's pending token ``input_ids`` [B] and its
    ``drafts`` [B, K], the drafts verified against the model's distributions:
    (tokens [B, K + 1], accepted [B]) of ``sampling.verify_drafts``.

    Afterwards a request has its pending token and the accepted drafts in its
    pages; the token after them, ``tokens[b, accepted[b]]``, is its next
    pending one (-1 where a row of logits has no token: such a request is the
    caller's to end, and the model gets token 0 for a pending -1).  Reads
    ``accepted`` back, since the pages are the host's.  A step that raises leaves
    the requests as they were."""
    from .sampling import verify_drafts

    B = len(request_ids)
    if drafts.dim() != 2 or drafts.shape[0] != B:
        raise RuntimeError(f"drafts must be [{B}, K], got shape {tuple(drafts.shape)}")
    if not isinstance(cache, PagedChunkCache) or cache.manager is not manager or cache.request_ids != list(request_ids):
        cache = PagedChunkCache(manager, request_ids)
    # (a draft outside the vocabulary ends the list: the model gets some token there)
    vocab = model.get_input_embeddings().weight.shape[0]
    known = drafts.clamp(0, vocab - 1).to(input_ids.dtype)
    logits = chunk_step(model, manager, request_ids, torch.cat([input_ids.reshape(B, 1).clamp(min=0), known], 1),
                        cache)
    try:
        tokens, accepted = verify_drafts(logits, drafts, accept_uniforms, draw_uniforms, draft_probs=draft_probs,
                                         temperature=temperature, top_k=top_k, top_p=top_p)
        kept = [1 + n for n in accepted.tolist()]
    except BaseException:
        cache._undo_step()
        raise
    chunk, cache._chunk = cache._chunk, None
    manager.keep_chunk(chunk, kept)
    return tokens, accepted


def prefill_chunked(model, manager: PagedKVCacheManager, request_id: str, input_ids: torch.Tensor,
                    chunk_size: int = 2048) -> torch.Tensor:
    """Runs a request's prompt [1, S] through the model ``chunk_size`` tokens
    at a time, straight into its pages, after the tokens that it has already
    (a prefix, an earlier turn).  Returns the last-position logits [1, vocab].

    Unlike ``prefill`` it keeps no second copy of the cache.  Where a chunk
    fails (no page left, a model that raises) the request is left as it was
    before the first one."""
    if chunk_size < 1:
        raise RuntimeError(f"chunk_size must be positive, got {chunk_size}")
    ids = input_ids.reshape(1, -1)
    if ids.shape[1] == 0:
        raise RuntimeError("an empty prompt has no logits")
    new = request_id not in manager.request_ids()
    manager.allocate(request_id)
    cache = PagedChunkCache(manager, [request_id])
    done = []
    try:
        for start in range(0, ids.shape[1], chunk_size):
            logits = chunk_step(model, manager, [request_id], ids[:, start:start + chunk_size], cache)
            done.append(cache._chunk)
    except BaseException:
        for chunk in reversed(done):
            cache._chunk = chunk
            if not cache._undo_step():
                break
        else:
            if new:
                manager.free(request_id)
        raise
    return logits[:, -1]
