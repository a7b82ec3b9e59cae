"""Embeddings of texts that grow.

The reference's worker runs every text from its first token (``core/gpu_worker.py:216-222``).
``IncrementalEmbedder`` keeps what a text has computed, its keys and values in an 8-bit paged cache,
so that only the tokens added since go through the model: a conversation's next turn, a stream's
next words, or many queries after one instruction (``fork``).  Each call returns the L2-normalised
last-token states, as ``GPUWorker.embed`` does.

A text may be given a budget: when its cache grows past it, the tokens with the smallest accumulated
attention weight are dropped, for each layer and kv head by itself; the most recent ones stay.
Positions go on counting from the text's first token, so a text ends with the model's rotary table: a call that
would pass it raises ``MesError`` and changes nothing.

Every layer has its own cache and all layers use the same pages, so one block table serves a step.
Runs of at most 16 new tokens in all take the matrix-vector kernels, as CUDA graphs once their sizes come
back; longer ones the GEMMs.  Calls are made on one stream at a time.
"""
from __future__ import annotations

import collections
import dataclasses
import os
import warnings

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


class _Step:
    """What a step reads, on the device: int64 ``[2 T + B]`` ids, positions and each text's last row, int32
    ``[B width + 2 B + 1]`` block table, offsets and lengths."""

    def __init__(self, device, B: int, T: int, width: int, max_new: int, longs, ints) -> None:
        self.longs, self.ints = (torch.as_tensor(x).to(device) for x in (longs, ints))
        self.ids, self.positions, self.rows = self.longs.split([T, T, B])
        table, cu_new, lens = self.ints.split([B * width, B + 1, B])
        self.cache_step = CacheStep(table.view(B, width), cu_new, lens, max_new)
        self.texts = torch.arange(B, device=device)


class _StepGraph:
    """A captured step of ``B`` texts with ``T`` new tokens in all."""

    def __init__(self, embedder: "IncrementalEmbedder", B: int, T: int, width: int, max_new: int) -> None:
        self.step = _Step(embedder.device, B, T, width, max_new, np.zeros(2 * T + B, np.int64),
                          np.zeros(B * width + 2 * B + 1, np.int32))
        if embedder._pool is None:
            embedder._pool = torch.cuda.graph_pool_handle()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, pool=embedder._pool):
            self.out = embedder._forward(self.step, False)

    def replay(self, longs, ints) -> torch.Tensor:
        self.step.longs.copy_(torch.as_tensor(longs))
        self.step.ints.copy_(torch.as_tensor(ints))
        self.graph.replay()
        return self.out.clone()


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
        self.use_cuda_graphs = self.device.type == "cuda" and os.environ.get("MES_CUDA_GRAPHS", "1") != "0"
        self.max_graphs = 32
        self._positions = layers[0].self_attn.rotary_emb.cos_sin_cache.shape[0] if len(layers) else None
        self._tp_size = layers[0].self_attn.o_proj.tp_size if len(layers) else 1
        self._graphs: collections.OrderedDict[tuple, _StepGraph | None] = collections.OrderedDict()
        self._pool = None

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
        if count < 0:
            raise _C.MesError(f"a text is forked into some others, not {count}")
        if count == 0:
            return out
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
        end = max(t.position + n for t, n in zip(texts, counts))
        if self._positions is not None and end > self._positions:
            raise _C.MesError(f"the model has {self._positions} positions, a text would have {end} tokens")
        parts = self._parts(texts, counts, first)
        # The pages that new tokens need, and those that eviction copies to, are there before anything runs.
        need = [max(self._pages_for(t.cached + n) - len(t.pages), 0) for t, n in zip(texts, counts)]
        self._need(sum(need) + sum(self._pages_for(self.budget) for t, n in zip(texts, counts) if self._over(t.cached + n)))
        out = [self._run_part(texts[a:b], tokens[a:b], counts[a:b], need[a:b], first) for a, b in parts]
        return out[0] if len(out) == 1 else torch.cat(out)

    def _parts(self, texts, counts, first: bool) -> list[tuple[int, int]]:
        """The texts cut into ranges that the cache attention takes in one call."""
        if not len(self.model.layers) or first and (self.budget is None or self.observe <= 0):
            return [(0, len(texts))]
        attn, parts, a, new, tokens = self.model.layers[0].self_attn, [], 0, 0, 0
        for i, (t, n) in enumerate(zip(texts, counts)):
            n, c = min(n, self.observe) if first else n, max(self._pages_for(t.cached + n), len(t.pages)) * self.page_size
            if i > a and not _C.kv8_attention_fits(i + 1 - a, max(new, n), attn.num_heads, attn.num_kv_heads, max(tokens, c)):
                parts.append((a, i))
                a, new, tokens = i, 0, 0
            new, tokens = max(new, n), max(tokens, c)
            if i == a and not _C.kv8_attention_fits(1, new, attn.num_heads, attn.num_kv_heads, tokens):
                raise _C.MesError(f"{n} new tokens of a text of {t.cached + n} are more than one call takes")
        return parts + [(a, len(texts))]

    def _run_part(self, texts, tokens, counts, need, first: bool) -> torch.Tensor:
        pages = self._take(sum(need))
        for t, n in zip(texts, need):
            t.pages += [pages.pop() for _ in range(n)]
        positions = [np.arange(t.position, t.position + n) for t, n in zip(texts, counts)]
        lens = [t.cached + n for t, n in zip(texts, counts)]
        observe = self.observe if first else max(self.observe, 1)
        seen = self.budget is not None and observe > 0 and (first or max(counts) > observe)
        graph, width = None, max(len(t.pages) for t in texts)
        if self.use_cuda_graphs and not first and not seen and sum(counts) <= _C.GEMV_MAX_ROWS and self._tp_size == 1:
            width = max(8, 1 << (width - 1).bit_length())
            graph = self._graph_for((len(texts), sum(counts), width, max(counts)))
        longs, ints = self._pack(tokens, positions, counts, [t.pages for t in texts], width, lens)
        if graph is not None:
            out = graph.replay(longs, ints)
        else:
            step = _Step(self.device, len(texts), sum(counts), width, max(counts), longs, ints)
            observed = None
            if seen:
                last = [min(n, observe) for n in counts]
                rows = np.concatenate([np.arange(e - m, e) for e, m in zip(np.cumsum(counts), last)])
                observed = (torch.as_tensor(rows).to(self.device), dataclasses.replace(
                    step.cache_step, cu_new=self._int32([0, *np.cumsum(last)]), max_new=max(last)))
            out = self._forward(step, first, observed)
        for t, n in zip(texts, counts):
            t.cached += n
            t.position += n
        self._evict([t for t in texts if self._over(t.cached)])
        return out

    def _pack(self, tokens, positions, counts, pages, width: int, lens):
        """What a step reads, as two host arrays (see :class:`_Step`)."""
        ends = np.cumsum(counts)
        table = np.zeros((len(pages), width), dtype=np.int32)
        for row, p in zip(table, pages):
            row[:len(p)] = p
        return (np.concatenate([*tokens, *positions, ends - 1]).astype(np.int64, copy=False),
                np.concatenate([table.reshape(-1), [0], ends, lens]).astype(np.int32, copy=False))

    def _forward(self, step: "_Step", first: bool, observed: tuple | None = None) -> torch.Tensor:
        hidden = self.model.step(step.ids, step.positions, step.rows, self.caches, step.cache_step, first, observed)
        return _C.last_token_l2(hidden, step.texts)

    # A token step is some ten launches a layer of a few microseconds each, less than the host needs for
    # them, so a step of sizes that come back is captured the second time (the first, run eagerly,
    # sets the kernels up; a step cannot be run twice, since it adds to the weights).
    def _graph_for(self, key: tuple):
        graph = self._graphs.get(key)
        if graph is None and key not in self._graphs:
            self._graphs[key] = None
            while len(self._graphs) > self.max_graphs:
                self._graphs.popitem(last=False)
            return None
        self._graphs.move_to_end(key)
        if graph is None:
            try:
                graph = self._graphs[key] = _StepGraph(self, *key)
            except Exception as exc:
                warnings.warn(f"CUDA-graph capture of a token step failed ({exc!r}); steps run eagerly", RuntimeWarning,
                              stacklevel=3)
                self.use_cuda_graphs = False
        return graph

    def release_graphs(self) -> None:
        """Drop every captured step."""
        self._graphs.clear()

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
