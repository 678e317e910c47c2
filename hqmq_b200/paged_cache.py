"""Sequences of any lengths in a paged compressed cache: pages are handed out, steps are laid out, layers follow.

The counterpart of ``PackedKVCache`` for a serving program (the reference's cache holds one batch of equal lengths:
src/model_utils.py:22-32): sequences come and go, every forward pass brings some of them a prompt chunk or a token, and a sequence can
be cut down to the tokens that attention looks at.  Pages are numbered once for all layers; every layer has a pool of its own."""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import _lib
from .packed import PackedKV
from .paged import PagedBatch, PagedKV, paged_attention, paged_attention_mass, paged_evict, paged_store


class PagedKVCache:
    """``quantizer``: an ``HQMQ`` or its outlier-aware wrapper, as for ``PackedKVCache``; every ``update`` takes its own Med3x median
    per head over the tokens of all sequences in it.  ``sliding_window``: {layer: window}.  ``outlier_capacity``: share of a page's
    chunks that its side buffer holds (``check()``).

        a, b = cache.add(2)
        cache.begin([a, b], [700, 55])                       # two prompts
        for layer: cache.update(K, V, layer); O = cache.attend(Q, layer)           # (755, heads, d)
        cache.begin([a, b], [1, 1])                          # a token each
    """

    def __init__(self, quantizer, n_pages: int, page_tokens: int = 64, sliding_window: Optional[Dict[int, int]] = None,
                 outlier_capacity: float = 0.125):
        self.quantizer, self.n_pages, self.page_tokens = quantizer, int(n_pages), int(page_tokens)
        self.sliding_window = dict(sliding_window or {})
        self.outlier_capacity = float(outlier_capacity)
        self._free: List[int] = list(range(self.n_pages - 1, -1, -1))
        self._table: Dict[int, List[int]] = {}
        self._len: Dict[int, int] = {}
        self._next = 0
        self._pools: Dict[int, PagedKV] = {}
        self._mass: Dict[int, torch.Tensor] = {}
        self._step: Optional[Tuple[List[int], List[int]]] = None
        self._updated: set = set()               # layers whose new tokens of the step are stored
        self._batches: dict = {}

    @property
    def _inner(self):
        return getattr(self.quantizer, "inner", self.quantizer)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        """Tokens that a sequence holds."""
        return self._len[seq]

    def pool(self, layer_idx: int) -> PagedKV:
        return self._pools[layer_idx]

    def mass(self, layer_idx: int) -> torch.Tensor:
        """Weights of a layer's tokens, see ``weigh``."""
        return self._mass[layer_idx]

    def add(self, n: int = 1) -> List[int]:
        """New, empty sequences."""
        ids = list(range(self._next, self._next + n))
        self._next += n
        for i in ids:
            self._table[i], self._len[i] = [], 0
        return ids

    def drop(self, seqs: Sequence[int]) -> None:
        """Sequences that are done; their pages are free again."""
        self._known(seqs)
        for i in seqs:
            self._free.extend(reversed(self._table.pop(i)))
            del self._len[i]
        self._step, self._batches = None, {}

    def _known(self, seqs):
        for i in seqs:
            if i not in self._table:
                raise KeyError(f"no sequence {i}")
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is named twice")

    def _next_pages(self, n: int) -> List[int]:
        """The next free pages, without weights; they stay free until ``_hand_out``, so that what raises in between leaves all as it was."""
        if n > len(self._free):
            raise _lib.HqmqError(f"hqmq_b200: {n} pages wanted, {len(self._free)} of {self.n_pages} free")
        pages = self._free[len(self._free) - n:][::-1]
        if pages:
            for mass in self._mass.values():     # (a page's earlier tokens leave no weight)
                mass[torch.tensor(pages, device=mass.device)] = 0.0
        return pages

    def _hand_out(self, n: int) -> None:
        del self._free[len(self._free) - n:]

    def begin(self, seqs: Sequence[int], new_tokens: Sequence[int]) -> None:
        """The next forward pass: every one of ``seqs`` gets so many new tokens.  ``update`` and ``attend`` of all layers follow."""
        seqs, new = [int(i) for i in seqs], [int(n) for n in new_tokens]
        self._known(seqs)
        if len(seqs) != len(new) or not seqs or min(new) < 0:
            raise ValueError(f"{len(seqs)} sequences and {len(new)} counts of new tokens")
        more = [-(-(self._len[i] + n) // self.page_tokens) - len(self._table[i]) for i, n in zip(seqs, new)]
        pages = self._next_pages(sum(more))
        self._hand_out(sum(more))
        for i, n, m in zip(seqs, new, more):
            self._table[i] += pages[:m]
            pages = pages[m:]
            self._len[i] += n
        self._step, self._batches, self._updated = (seqs, new), {}, set()

    def batch(self, layer_idx: int, n_heads: Optional[int] = None) -> PagedBatch:
        """The step's batch for a layer (made once for all layers of a window whose pools are alike: a device, KV heads and a head dim)."""
        if self._step is None:
            raise _lib.HqmqError("hqmq_b200: begin() a step first")
        pool = self._pools[layer_idx]
        key = (n_heads, self.sliding_window.get(layer_idx) if n_heads else None, *self._shape(pool))
        if key not in self._batches:
            seqs, new = self._step
            self._batches[key] = PagedBatch(pool, [self._table[i] for i in seqs], [self._len[i] for i in seqs], new,
                                            n_heads=key[0], window=key[1])
        return self._batches[key]

    @staticmethod
    def _shape(pool: PagedKV):
        return pool.device, pool.H_kv, pool.d_head

    def _new_pool(self, k: torch.Tensor) -> PagedKV:
        q, outl = self._inner, hasattr(self.quantizer, "median_mult")
        cap = max(16, int(self.outlier_capacity * self.page_tokens * (k.shape[-1] // 4))) if outl else None
        return PagedKV(self.n_pages, q.n_heads, k.shape[-1], q.secondary_size, q.radius_bits, k.device, page_tokens=self.page_tokens,
                       dtype=k.dtype, outliers_K=outl, outliers_V=outl, out_cap=cap)

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int) -> PagedKV:
        """The step's new tokens of one layer, (total_new, H_kv, d), sequence after sequence: encoded, and stored in their pages."""
        if self._step is None:
            raise _lib.HqmqError("hqmq_b200: begin() a step first")
        total = sum(self._step[1])
        if key_states.shape != value_states.shape or key_states.dim() != 3 or key_states.shape[0] != total:
            raise ValueError(f"keys and values are ({total}, H_kv, d), got {tuple(key_states.shape)} and {tuple(value_states.shape)}")
        _lib.require_cuda(key_states, "PagedKVCache.update")
        pool = self._pools.get(layer_idx)
        if pool is None:
            pool = self._pools[layer_idx] = self._new_pool(key_states)
        if total == 0:
            return pool
        outl = pool.K.with_outliers
        pair = tuple(self._inner.new_cache(1, total, pool.d_head, pool.device, scale_dtype=pool.dtype, with_outliers=outl,
                                           out_dtype=pool.dtype, place=False) for _ in range(2))
        PackedKV.place(pool.device, *pair)
        k, v = (x.transpose(0, 1).unsqueeze(0) for x in (key_states, value_states))
        self.quantizer.encode_pair(k, v, layer_idx, *pair)
        paged_store(pool, *pair, self.batch(layer_idx))
        self._updated.add(layer_idx)
        return pool

    def attend(self, query_states: torch.Tensor, layer_idx: int, softmax_scale: Optional[float] = None,
               softcap: Optional[float] = None, sinks: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of the step's new tokens, (total_new, H_q, d), over their sequences (``update`` first), see ``paged_attention``."""
        tk, tv = (self._inner.tables(layer_idx, kv, query_states.device) for kv in (0, 1))
        return paged_attention(query_states, self._pools[layer_idx], self.batch(layer_idx, query_states.shape[1]), tk["table16"], tv["table16"],
                               softmax_scale=softmax_scale, softcap=softcap, sinks=sinks, out=out)

    def weigh(self, query_states: torch.Tensor, layer_idx: int, decay: float = 1.0, softmax_scale: Optional[float] = None,
              softcap: Optional[float] = None, sinks: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Add the attention weights that the step's queries give to the layer's tokens, times ``decay`` what they had (see
        ``paged_attention_mass``); ``evict`` goes by them."""
        pool = self._pools[layer_idx]
        if layer_idx not in self._mass:
            self._mass[layer_idx] = pool.new_mass()
        mass = self._mass[layer_idx]
        return paged_attention_mass(query_states, pool, self.batch(layer_idx, query_states.shape[1]),
                                    self._inner.tables(layer_idx, 0, query_states.device)["table16"], softmax_scale=softmax_scale,
                                    softcap=softcap, sinks=sinks, prior=mass, decay=decay, out=mass)

    def evict(self, seqs: Sequence[int], keep: int, first: int = 4, last: int = 16) -> Dict[int, torch.Tensor]:
        """Cut sequences of more than ``keep`` tokens down to it, in every layer by the layer's own weights (all layers have some: see
        ``weigh``).  Returns {layer: positions that stayed}, see ``paged_evict``; ends the step.  What stays is numbered anew: a layer's
        sliding window counts tokens that are held."""
        self._known(seqs)
        if first < 0 or last < 0:
            raise ValueError(f"first={first}, last={last}: counts of tokens")
        if keep < first + last:
            raise ValueError(f"keep={keep}: at least the {first} first and {last} last tokens stay")
        missing = [layer for layer in self._pools if layer not in self._mass]
        if missing:
            raise _lib.HqmqError(f"hqmq_b200: no weights of layers {missing} (weigh() first)")
        cut = [int(i) for i in seqs if self._len[i] > keep]
        per = -(-keep // self.page_tokens)
        if not cut or not self._pools:
            self._step, self._batches = None, {}
            return {}
        pages = self._next_pages(per * len(cut))  # (the tokens move to free pages: until all have, raising leaves everything as it was)
        tables = [pages[per * k:per * (k + 1)] for k in range(len(cut))]
        moves: dict = {}                         # old and new batch by what a batch is bound to
        for pool in self._pools.values():
            if self._shape(pool) not in moves:
                moves[self._shape(pool)] = (PagedBatch(pool, [self._table[i] for i in cut], [self._len[i] for i in cut]),
                                            PagedBatch(pool, tables, [keep] * len(cut)))
        kept = {layer: paged_evict(pool, *moves[self._shape(pool)], self._mass[layer], first=first, last=last)
                for layer, pool in self._pools.items()}
        self._hand_out(len(pages))
        self._step, self._batches = None, {}
        for i, table in zip(cut, tables):
            self._free.extend(reversed(self._table[i]))
            self._table[i], self._len[i] = table, keep
        return kept

    def check(self) -> None:
        """Synchronise and raise if the side buffer of a page that is held overflowed, or an update gave up on a bounded wait of the encoder
        (its tokens have a scale of NaN).  Of a step under way, a layer's new tokens count from its ``update`` on."""
        for layer, pool in self._pools.items():
            late = dict(zip(*self._step)) if self._step and layer not in self._updated else {}
            lens = {i: self._len[i] - late.get(i, 0) for i in self._table}
            held = [(p, min(self.page_tokens, lens[i] - k * self.page_tokens)) for i, t in self._table.items()
                    for k, p in enumerate(t[:-(-lens[i] // self.page_tokens)])]
            if not held:
                continue
            try:
                pool.check([p for p, _ in held])
            except _lib.HqmqError as e:
                raise _lib.HqmqError(f"{e} (layer {layer}: raise outlier_capacity)") from None
            pages, tokens = torch.tensor(held, device=pool.device).unbind(1)
            live = torch.arange(self.page_tokens, device=pool.device) < tokens.view(-1, 1, 1)      # (rows behind them are of another life)
            if any(bool((x.pages("rs")[pages].isnan() & live).any()) for x in (pool.K, pool.V)):
                raise _lib.HqmqError(f"hqmq_b200: an update of layer {layer} gave up on a bounded wait")
