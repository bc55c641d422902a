"""The sparse method ``accumulated_weight``: a request keeps at most ``budget`` cached tokens (and a page and a step's
portion more for as long as the step lasts); per layer and kv head the last ``recent`` and those of the others that have
gathered the most attention weight.

Every attention adds the softmax weights its rows give to the cached keys (``HipKernels.attention_weights``) to a float
per key, kept in pages beside the cache.  When a step leaves a request a page or more above its budget, its tokens are
moved to fresh pages layer by layer (``HipKernels.evict_tokens``), each layer and kv head keeping its own, and the old
pages return to the pool.  Keys have been rotated by their positions in the sequence before they were cached, so a kept
token goes on as it is; the cache's length and the next token's position part ways (``CacheManager.row_dropped``).
Preempted requests start from nothing, weights included, as their cache does.
"""
from __future__ import annotations

import numpy as np
import torch

from ..config.method_registry import MethodRuntime


class AccumulatedWeightMethod(MethodRuntime):
    name = "accumulated_weight"
    wants_attention = True
    kernel_libraries = ("attention_weights", "evict")

    def __init__(self, budget: int = 0, recent: int = 0, portion: int = 0):
        """``budget`` tokens kept, ``recent`` of them the last ones; ``portion``: the largest number of tokens a
        step adds to a request (``configure`` takes all three from the runtime configuration)."""
        self.budget, self.recent, self.portion = int(budget), int(recent), int(portion)
        self.cache = None
        self.weights: dict[int, torch.Tensor] = {}      # cache position -> float32 [pages, kv_heads, page_size]
        self.evictions = 0                              # how often a request's tokens were cut
        self._kept = None

    def configure(self, config) -> None:
        self.budget, self.recent = config.eviction_budget, config.eviction_recent
        self.portion = min(config.engine_prefill_chunk_size, config.max_num_batched_tokens)

    def bind(self, cache) -> None:
        super().bind(cache)
        if not 1 <= self.budget or not 0 <= self.recent <= self.budget:
            raise ValueError(f"accumulated_weight: a budget of {self.budget} tokens with the last {self.recent}")
        for group in cache.groups:
            if group.window is not None:
                raise ValueError("accumulated_weight: a layer with an attention window gives its tokens back by itself")
            if group.request.head_dim % 8:
                raise ValueError(f"accumulated_weight takes head sizes in steps of 8, got {group.request.head_dim}")
            for position, layer in group.layers.items():
                self.weights[position] = torch.zeros(layer.shape[0], layer.shape[2], layer.shape[3], dtype=torch.float32,
                                                     device=layer.device)

    def bytes_per_token(self, request) -> int:
        return 4 * request.kv_heads

    def _limit(self) -> int:
        """The cached length at which a step's end cuts a request."""
        return self.budget + max((g.page_size for g in self.cache.groups), default=1)

    def reserved_pages(self) -> dict[int, int]:
        # one request's fresh pages: then every cut can be made, one after the other, as each gives its old pages back
        if self._limit() > self.cache.max_model_len:
            return {}
        return {g.index: -(-self.budget // g.page_size) for g in self.cache.groups}

    def reserved_tokens(self, page: int, longest: int) -> int:
        return self.budget + page - 1 if self.budget + page <= longest else 0

    def tokens_taken(self, length: int, new_tokens: int) -> int:
        # less than the limit between two steps, and what one step adds
        return max(min(new_tokens, max(1, self.portion)), min(new_tokens, self._limit() - 1 + max(1, self.portion) - length))

    def attended(self, position: int, fb, q, cache, meta, lse, scale: float, window: int) -> None:
        weights = self.weights[position]
        fb.kernels.attention_weights(q, cache, meta, lse, weights, scale, window, previous=weights)

    def finish_step(self, fb) -> None:
        over = [int(row) for row in fb.item_rows_host if self.cache.row_len[row] >= self._limit()]
        while over:
            room = min(g.pool.free_count // -(-self.budget // g.page_size) for g in self.cache.groups)
            if room < 1:
                return          # the next step tries again
            self._evict(fb, over[:room])
            over = over[room:]

    def _evict(self, fb, rows: list[int]) -> None:
        cache, keep = self.cache, self.budget
        lengths = cache.row_len[rows].astype(np.int32)
        longest = int(lengths.max())
        tables = cache.begin_eviction(rows, keep)
        try:
            on_device = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(fb.device)
            lengths_there = on_device(lengths)
            for group in cache.groups:
                old = on_device(group.table[rows, :-(-longest // group.page_size)])
                new = on_device(tables[group.index])
                kept = fb.buffer("evict.kept", (len(rows), group.request.kv_heads, keep), torch.int32)
                for position, layer in group.layers.items():
                    fb.kernels.evict_tokens(layer, self.weights[position], old, lengths_there, new, keep, self.recent, kept,
                                            longest=longest)
        except Exception:      # the old pages are as they were
            cache.abort_eviction(rows, tables)
            raise
        cache.finish_eviction(rows, keep, tables)
        self.evictions += len(rows)
