"""Embeddings of texts that grow.

The reference's worker runs every text from its first token (``core/gpu_worker.py:216-222``).
``IncrementalEmbedder`` keeps what a text has computed, its keys and values in an 8-bit paged cache,
so that only the tokens added since go through the model: a conversation's next turn, a stream's
next words, or many queries after one instruction (``fork``).  Each call returns the L2-normalised
last-token states, as ``GPUWorker.embed`` does.

A text may be given a budget: when its cache grows past it, the tokens with the smallest accumulated
attention weight are dropped, for each layer and kv head by itself; the most recent ones stay.
Positions go on counting from the text's first token.

Every layer has its own cache and all layers use the same pages, so one block table serves a step.
Runs of at most 16 new tokens in all take the matrix-vector kernels; longer ones the GEMMs.
"""
from __future__ import annotations

import numpy as np
import torch

from .. import _C
from ..layers.kv_cache import CacheStep, KV8Cache


class _Text:
    """A text's pages, its cached tokens and the position of its next token."""

    def __init__(self) -> None:
        self.pages: list[int] = []
        self.cached = 0
        self.position = 0


class IncrementalEmbedder:

    def __init__(self, model, num_pages: int, page_size: int = 64, dtype: torch.dtype = torch.int8,
                 budget: int | None = None, recent: int | None = None, observe: int = 16) -> None:
        """``model``: a ``Qwen3ForCausalLM`` / ``Qwen2ForCausalLM`` on its device (e.g.
        ``GPUWorker.model``).  ``num_pages`` pages of ``page_size`` tokens are shared by all texts.
        ``budget``: cached tokens a text is cut down to once it has a quarter more, ``recent`` of
        them (default: a quarter) the last ones; of a new text, or of more tokens than that added
        to one, the last ``observe`` give the attention weights."""
        self.model = model.model
        layers = self.model.layers
        self.device = self.model.embed_tokens.weight.device
        self.page_size = page_size
        if budget is not None and budget <= 0:
            raise ValueError("the budget is a number of tokens")
        self.budget = budget
        self.recent = (budget // 4 if recent is None else recent) if budget is not None else 0
        if budget is not None and not 0 <= self.recent <= budget:
            raise ValueError("recent is at most the budget")
        self.observe = observe
        self.caches = [KV8Cache(num_pages, page_size, layer.self_attn.num_kv_heads, dtype, self.device,
                                track_weights=budget is not None) for layer in layers]
        self._free = list(range(num_pages - 1, -1, -1))
        self._texts: dict[int, _Text] = {}
        self._next = 0

    # ------------------------------------------------------------------ pages
    def _pages_for(self, tokens: int) -> int:
        return -(-tokens // self.page_size)

    def _need(self, n: int) -> None:
        if n > len(self._free):
            raise _C.MesError(f"the cache has {len(self._free)} free pages of {self.page_size} tokens, {n} are needed")

    def _take(self, n: int) -> list[int]:
        self._need(n)
        return [self._free.pop() for _ in range(n)]

    def _over(self, tokens: int) -> bool:
        return self.budget is not None and tokens > self.budget + self.budget // 4

    def _int32(self, values) -> torch.Tensor:
        return torch.as_tensor(np.asarray(values, dtype=np.int32)).to(self.device, non_blocking=True)

    def _table(self, pages: list[list[int]]) -> torch.Tensor:
        table = np.zeros((len(pages), max(len(p) for p in pages)), dtype=np.int32)
        for row, p in zip(table, pages):
            row[:len(p)] = p
        return self._int32(table)

    # ------------------------------------------------------------------ calls
    @torch.no_grad()
    def add(self, texts) -> tuple[list[int], torch.Tensor]:
        """Start a text for each non-empty list of token ids; returns ``(handles, fp32 [B, H]
        embeddings on the device)``."""
        texts = [np.asarray(t, dtype=np.int64).reshape(-1) for t in texts]
        if any(len(t) == 0 for t in texts):
            raise _C.MesError("a text has at least one token")
        new = []
        for _ in texts:
            self._texts[self._next] = _Text()
            new.append(self._next)
            self._next += 1
        try:
            return new, self._run(new, texts, first=True)
        except Exception:
            self.drop(new)
            raise

    @torch.no_grad()
    def extend(self, handles, texts) -> torch.Tensor:
        """Append a non-empty list of token ids to each of the texts; fp32 ``[B, H]`` embeddings."""
        texts = [np.asarray(t, dtype=np.int64).reshape(-1) for t in texts]
        if len(texts) != len(handles) or len(set(handles)) != len(handles):
            raise _C.MesError("one list of tokens for each of different texts")
        if any(len(t) == 0 for t in texts):
            raise _C.MesError("at least one token is added to a text")
        return self._run(handles, texts, first=False)

    @torch.no_grad()
    def fork(self, handle: int, count: int) -> list[int]:
        """``count`` new texts that begin with what ``handle`` has cached (copied, since the pages
        of a text are written as it grows)."""
        text, out = self._texts[handle], []
        pages = self._take(len(text.pages) * count)
        src = torch.as_tensor(text.pages, device=self.device).repeat(count)
        dst = torch.as_tensor(pages, device=self.device)
        for cache in self.caches:
            codes = cache.codes.view(torch.int8)
            codes[dst] = codes[src]
            cache.scales[dst] = cache.scales[src]
            if cache.sums is not None:
                cache.sums[dst] = cache.sums[src]
        for i in range(count):
            t = _Text()
            t.pages = pages[i * len(text.pages):(i + 1) * len(text.pages)]
            t.cached, t.position = text.cached, text.position
            self._texts[self._next] = t
            out.append(self._next)
            self._next += 1
        return out

    def drop(self, handles) -> None:
        """Forget texts and free their pages."""
        for h in handles:
            self._free.extend(self._texts.pop(h).pages)

    def cached_tokens(self, handle: int) -> int:
        return self._texts[handle].cached

    # ------------------------------------------------------------------ a step
    def _run(self, handles, tokens, first: bool) -> torch.Tensor:
        texts = [self._texts[h] for h in handles]
        if not texts:
            return torch.empty(0, self.model.norm.hidden_size, dtype=torch.float32, device=self.device)
        counts = [len(t) for t in tokens]
        need = [self._pages_for(t.cached + n) - len(t.pages) for t, n in zip(texts, counts)]
        # Those that eviction copies to are there before anything runs, so that a text is extended whole or not at all.
        self._need(sum(need) + sum(self._pages_for(self.budget) for t, n in zip(texts, counts) if self._over(t.cached + n)))
        pages = self._take(sum(need))
        for t, n in zip(texts, need):
            t.pages += [pages.pop() for _ in range(n)]
        ids = torch.as_tensor(np.concatenate(tokens)).to(self.device, non_blocking=True)
        positions = torch.as_tensor(np.concatenate(
            [np.arange(t.position, t.position + n, dtype=np.int64) for t, n in zip(texts, counts)])).to(self.device, non_blocking=True)
        ends = np.cumsum(counts)
        rows = torch.as_tensor(ends - 1).to(self.device, non_blocking=True)
        table = self._table([t.pages for t in texts])
        lens = self._int32([t.cached + n for t, n in zip(texts, counts)])
        step = CacheStep(table, self._int32([0, *ends]), lens, max(counts))
        seen = None
        observe = self.observe if first else max(self.observe, 1)
        if self.budget is not None and observe > 0 and (first or max(counts) > observe):
            last = [min(n, observe) for n in counts]
            seen = (torch.as_tensor(np.concatenate([np.arange(e - m, e) for e, m in zip(ends, last)])).to(self.device),
                    CacheStep(table, self._int32([0, *np.cumsum(last)]), lens, max(last)))
        hidden = self.model.step(ids, positions, rows, self.caches, step, first, seen)
        for t, n in zip(texts, counts):
            t.cached += n
            t.position += n
        out = _C.last_token_l2(hidden, torch.arange(len(texts), device=self.device))
        self._evict([t for t in texts if self._over(t.cached)])
        return out

    def _evict(self, texts) -> None:
        if not texts:
            return
        per = self._pages_for(self.budget)
        step = CacheStep(self._table([t.pages for t in texts]), self._int32([0] * (len(texts) + 1)),
                         self._int32([t.cached for t in texts]), 0)
        taken = self._take(per * len(texts))
        pages = [taken[i * per:(i + 1) * per] for i in range(len(texts))]
        new_table = self._table(pages)
        for cache in self.caches:
            cache.evict(step, new_table, self.budget, self.recent)
        for t, p in zip(texts, pages):
            self._free.extend(t.pages)
            t.pages, t.cached = p, self.budget
