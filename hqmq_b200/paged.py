"""A paged compressed cache: a pool of pages, batches of ragged sequences over it, and the operators on them.

The reference serves one batch of equal lengths at a time (its cache: src/model_utils.py:22-32; its kernel takes one
(B, H, T) tuple: src/quantizers/hqmq_attention.py:425-518).  Here the tokens of a sequence live in pages of a pool, so that
sequences of any lengths share a batch, grow a page at a time, and are cut down to a budget:

    pool  = PagedKV(n_pages, n_kv_heads, d_head, S, radius_bits, "cuda")            # one layer's keys and values
    batch = PagedBatch(pool, tables, kv_lens, q_lens, n_heads=32)                    # a step's tables, lengths and plan
    paged_store(pool, K_encoded, V_encoded, batch)                                   # encoded new tokens go to their pages
    O     = paged_attention(Q, pool, batch, table_K, table_V, softcap=30.0, sinks=s)  # (total_q, H_q, d)
    mass  = paged_attention_mass(Q, pool, batch, table_K, prior=mass, decay=0.9)      # weight that every token received
    kept  = paged_evict(pool, batch, smaller_batch, mass)                            # the heaviest tokens move to fewer pages

All arithmetic runs in the kernels of csrc/paged_*; CPU tensors raise.
"""
from __future__ import annotations

import ctypes as C
from threading import get_ident
from typing import Optional, Sequence

import numpy as np
import torch

from . import _lib
from .packed import PackedKV


class PagePlanes(PackedKV):
    """One tensor's planes of a pool: a ``PackedKV`` whose batch entries are pages."""

    def pages(self, name: str) -> torch.Tensor:
        """A plane as a tensor with one row per page: ``codes`` (pages, H, tokens, row bytes), ``rs`` and ``flags`` (pages, H,
        tokens), ``out_off`` (pages, H, tokens / 16 + 1), ``out_vals`` (pages, H, out_cap, 4), ``out_count`` (pages, H)."""
        t = getattr(self, name)
        if t is None:
            raise _lib.HqmqError(f"hqmq_b200: these pages have no plane {name!r} (no outliers)")
        views = self.__dict__.setdefault("_views", {})
        if name not in views or views[name][0] is not t:
            views[name] = (t, self._as_pages(t, name))
        return views[name][1]

    def __getstate__(self):
        return {k: v for k, v in super().__getstate__().items() if k != "_views"}

    def _as_pages(self, t, name):
        rows = self.B * self.H * self.T_cap
        if name == "codes":
            return t[:rows * self.row_bytes].view(self.B, self.H, self.T_cap, self.row_bytes)
        if name in ("rs", "flags"):
            return t[:rows].view(self.B, self.H, self.T_cap)
        if name == "out_vals":
            return t[:self.B * self.H * self.out_cap * 4].view(self.B, self.H, self.out_cap, 4)
        if name == "out_off":
            return t.view(self.B, self.H, -1)
        if name == "out_count":
            return t.view(self.B, self.H)
        raise ValueError(f"no plane {name!r}")

    def planes(self) -> dict:
        """All planes by name, see ``pages``."""
        names = ("codes", "rs") + (("flags", "out_off", "out_vals", "out_count") if self.with_outliers else ())
        return {name: self.pages(name) for name in names}


class PagedKV:
    """The pages of one layer's keys and values.  ``page_tokens``: a power of two, 64 to 1024.  ``dtype`` (fp16 or bf16): type of
    the scales and of the flagged chunks' values.  ``out_cap``: flagged chunks a page can hold per head, one number or (K's, V's);
    by default an eighth of its chunks; ``check()`` tells whether it was exceeded."""

    def __init__(self, n_pages: int, n_kv_heads: int, d_head: int, S: int, radius_bits: int, device, page_tokens: int = 64,
                 dtype: torch.dtype = torch.bfloat16, outliers_K: bool = False, outliers_V: bool = False, out_cap=None):
        if page_tokens < _lib.T_ALIGN or page_tokens & (page_tokens - 1) or page_tokens > 1024:
            raise ValueError(f"page_tokens={page_tokens}: a power of two from {_lib.T_ALIGN} to 1024")
        if d_head not in (64, 128):
            raise ValueError(f"d_head={d_head}: a paged cache has heads of 64 or 128")
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"hqmq_b200: a paged cache keeps fp16 or bf16 scales and outliers, not {dtype}")
        if n_pages < 1:
            raise ValueError("a pool has at least one page")
        self.n_pages, self.page_tokens, self.H_kv, self.d_head, self.dtype = n_pages, page_tokens, n_kv_heads, d_head, dtype
        self.S, self.radius_bits = S, radius_bits
        caps = out_cap if isinstance(out_cap, (tuple, list)) else (out_cap, out_cap)
        self.K, self.V = (PagePlanes(n_pages, n_kv_heads, page_tokens, d_head // 4, S, radius_bits, device, scale_dtype=dtype,
                                     with_outliers=outl, out_dtype=dtype, place=False,
                                     out_cap=(page_tokens * (d_head // 4) // 8 if cap is None else cap) if outl else None)
                          for outl, cap in ((outliers_K, caps[0]), (outliers_V, caps[1])))
        PackedKV.place(torch.device(device), self.K, self.V)
        self.device = self.K.device
        self.K.T = self.V.T = page_tokens
        # what the arguments of a call depend on, besides addresses
        self.kind = (n_pages, page_tokens, n_kv_heads, d_head, S, radius_bits, dtype, self.device, bool(outliers_K), bool(outliers_V),
                     self.K.out_cap, self.V.out_cap)

    def new_mass(self) -> torch.Tensor:
        """Zeroed weights, one per token, page and KV head (see ``paged_attention_mass``)."""
        return torch.zeros(self.n_pages, self.H_kv, self.page_tokens, dtype=torch.float32, device=self.device)

    def check(self, pages: Optional[Sequence[int]] = None) -> None:
        """Synchronise and raise if a page's side buffer was too small for the outliers it was given (rows and flags are complete
        then, but values beyond the capacity were dropped and read as 0).  ``pages``: those that hold tokens (None: all)."""
        at = None if pages is None else torch.tensor(list(pages), dtype=torch.int64, device=self.device)
        for name, pk in (("K", self.K), ("V", self.V)):
            if pk.with_outliers and (at is None or at.numel()):
                most = int((pk.out_count if at is None else pk.pages("out_count")[at]).max())
                if most > pk.out_cap:
                    raise _lib.HqmqError(f"hqmq_b200: the outliers of a page of {name} overflowed ({most} > {pk.out_cap} chunks); raise out_cap")


def _int_array(x, what: str) -> np.ndarray:
    if isinstance(x, torch.Tensor):
        if x.is_cuda:
            raise TypeError(f"hqmq_b200: {what} are host values (a plan is made on the host)")
        x = x.numpy()
    a = np.asarray(x)
    if a.size and a.dtype.kind not in "iu":
        raise TypeError(f"hqmq_b200: {what} are integers")
    if a.size and (int(a.min()) < -(1 << 31) or int(a.max()) >= 1 << 31):
        raise ValueError(f"{what} out of range")
    return np.array(a, dtype=np.int32, order="C")     # (a copy: the caller's array may count on)


class PagedBatch:
    """Sequences over a pool: their tables of pages, their lengths, and the plan of the calls over them.

    ``tables``: per sequence its pages in order (lists, or one integer array with a row per sequence; entries behind the last
    page are not read).  ``kv_lens``: tokens of every sequence, new ones included.  ``q_lens``: its new tokens, the last ones (by default one
    each with ``n_heads`` given, else none).  ``n_heads``: query heads; without it the batch serves ``paged_store`` and
    ``paged_evict`` only.  ``window``: a query sees the last ``window`` positions up to its own.

    A batch serves every layer of a step.  It is copied to the device on the stream that is current when it is made; a call on
    another stream has to be ordered behind that by the caller, like any tensor's.  With ``reserve_pages`` (at least the pages its tables will ever
    hold) ``renew`` gives a batch of single tokens or a few drafted ones other lengths and tables in place, and calls that a CUDA graph has captured follow."""

    def __init__(self, pool: PagedKV, tables, kv_lens, q_lens=None, n_heads: Optional[int] = None, window: Optional[int] = None,
                 reserve_pages: int = 0):
        if pool.device.type == "cuda" and _lib.capturing(torch.cuda.current_stream(pool.device).cuda_stream):
            raise _lib.HqmqError("hqmq_b200: a PagedBatch is made outside of a graph's capture (renew() updates it in place)")
        if n_heads is not None and (n_heads < 1 or n_heads % pool.H_kv):
            raise ValueError(f"n_heads={n_heads} must be a positive multiple of the pool's {pool.H_kv} KV heads")
        if window is not None and window < 1:
            raise ValueError("window is at least 1 (None: no window)")
        if not 0 <= reserve_pages <= 1 << 24:
            raise ValueError(f"reserve_pages={reserve_pages}: from 0 to {1 << 24}")
        self.n_pages, self.page_tokens, self.H_kv, self.d_head, self.device = pool.n_pages, pool.page_tokens, pool.H_kv, pool.d_head, pool.device
        self.n_heads, self.window = n_heads, window
        p = self.plan = _lib.PagedPlan()
        p.struct_size = C.sizeof(_lib.PagedPlan)
        p.n_pages, p.page_tokens, p.H_q, p.H_kv, p.d, p.window = pool.n_pages, pool.page_tokens, n_heads or 0, pool.H_kv, pool.d_head, min(window or 0, 1 << 30)
        p.tab_room = int(reserve_pages)
        host, kv, q, pages = self._lay_out(p, tables, kv_lens, q_lens)
        self._take(kv, q, pages)
        self.data = host.to(self.device, non_blocking=True) if self.device.type == "cuda" else host

    def _lay_out(self, p, tables, kv_lens, q_lens):
        kv = _int_array(kv_lens, "kv_lens")
        n = len(kv)
        if n < 1 or kv.ndim != 1:
            raise ValueError("a batch has at least one sequence")
        if q_lens is None:
            q = np.full(n, 1 if p.H_q else 0, dtype=np.int32)
        else:
            q = _int_array(q_lens, "q_lens")
        if q.shape != kv.shape or len(tables) != n:
            raise ValueError(f"{n} kv_lens, {len(q)} q_lens and {len(tables)} tables")
        if (kv < 0).any() or (q < 0).any() or (q > kv).any():
            raise ValueError("lengths: 0 <= q_len <= kv_len of every sequence (its new tokens are part of it)")
        need = -(-kv.astype(np.int64) // self.page_tokens)
        wide = max(1, int(need.max()))
        if isinstance(tables, (list, tuple)) and not (n and isinstance(tables[0], (torch.Tensor, np.ndarray))):
            table = np.zeros((n, wide), dtype=np.int32)
            for i, row in enumerate(tables):
                if len(row) < need[i]:
                    raise ValueError(f"sequence {i}: {len(row)} pages for {kv[i]} tokens")
                if need[i]:
                    table[i, :need[i]] = _int_array(list(row[:need[i]]), "tables")
        else:
            table = _int_array(np.stack([np.asarray(t) for t in tables]) if isinstance(tables, (list, tuple)) else tables, "tables")
            if table.ndim != 2 or (need > table.shape[1]).any():
                raise ValueError(f"tables of shape {table.shape} for up to {wide} pages a sequence")
        pages = table[:, :wide][np.arange(wide) < need[:, None]] if table.shape[1] >= 1 else np.zeros(0, dtype=np.int32)
        if pages.size and (int(pages.min()) < 0 or int(pages.max()) >= self.n_pages):
            raise ValueError(f"tables name pages outside of 0 .. {self.n_pages - 1}")
        p.n_seqs = n
        L = _lib.lib()
        _lib.check(L.hqmq_paged_plan_size(C.byref(p), kv.ctypes.data, q.ctypes.data), "hqmq_paged_plan_size")
        host = torch.empty(p.words, dtype=torch.int32, pin_memory=self.device.type == "cuda")
        _lib.check(L.hqmq_paged_plan_fill(C.byref(p), kv.ctypes.data, q.ctypes.data, table.ctypes.data, table.shape[1] if table.size else 0, host.data_ptr()),
                   "hqmq_paged_plan_fill")
        return host, kv, q, (table, need, pages)

    def _keep(self, key, call):
        if len(self._calls) >= 64:
            self._calls.clear()
        self._calls[key] = call
        return call

    def _take(self, kv, q, pages):
        self._calls: dict = {}                   # argument structs of repeated calls
        self.kv_lens, self.q_lens = kv, q
        self.total_q, self.longest, self.shortest = int(q.sum()), int(kv.max()), int(kv.min())
        self._table, self._need, flat = pages
        self.pages = frozenset(flat.tolist())
        self._unshared = len(self.pages) == flat.size
        self._stored = None                      # whether the pages that new tokens go to belong to one sequence each

    def renew(self, tables, kv_lens) -> None:
        """Other lengths and tables for the same new tokens, in place (see ``reserve_pages``), on the current stream."""
        if not self.plan.tab_room:
            raise _lib.HqmqError("hqmq_b200: renew() needs a batch made with reserve_pages")
        if _lib.capturing(torch.cuda.current_stream(self.device).cuda_stream):
            raise _lib.HqmqError("hqmq_b200: renew() is a call between replays, not part of a graph")
        if len(kv_lens) != len(self.kv_lens):
            raise ValueError(f"{len(kv_lens)} kv_lens for a batch of {len(self.kv_lens)} sequences")
        p = _lib.PagedPlan.from_buffer_copy(self.plan)
        p.renew = 1
        host, kv, q, pages = self._lay_out(p, tables, kv_lens, self.q_lens)
        p.renew = 0
        with _lib.device_guard(self.device):
            self.data.copy_(host, non_blocking=True)
        self.plan = p
        self._take(kv, q, pages)

    def stores_alone(self) -> bool:
        """Whether every page that a new token goes to belongs to one sequence of the batch, once."""
        if self._stored is None:
            self._stored = self._unshared or self._written_alone()
        return self._stored

    def _written_alone(self) -> bool:
        uses: dict = {}
        for row, n in zip(self._table, self._need):
            for page in row[:n].tolist():
                uses[page] = uses.get(page, 0) + 1
        for row, n, kv, q in zip(self._table, self._need, self.kv_lens, self.q_lens):
            if q and any(uses[page] > 1 for page in row[(kv - q) // self.page_tokens:n].tolist()):
                return False
        return True


def _belongs(pool: PagedKV, batch: PagedBatch, what: str):
    _lib.require_cuda(pool.K.rs, what)
    _lib.check_device(pool.device)
    if (batch.n_pages, batch.page_tokens, batch.H_kv, batch.d_head, batch.device) != (pool.n_pages, pool.page_tokens, pool.H_kv, pool.d_head, pool.device):
        raise ValueError(f"{what}: the batch was made for another pool's geometry or device")


def _codebook(t: torch.Tensor, pool: PagedKV, what: str) -> None:
    if t.shape != (pool.H_kv, 24 * pool.S, 4) or t.dtype != torch.float16 or t.device != pool.device:
        raise ValueError(f"{what}: an fp16 table of shape {(pool.H_kv, 24 * pool.S, 4)} on {pool.device} "
                         f"(got {t.dtype} {tuple(t.shape)} on {t.device})")


def _attn_args(Q, pool, batch, table_K, softmax_scale, softcap, sinks, what):
    """Checks, and the argument struct of a call without its addresses."""
    _lib.require_cuda(Q, what)
    _belongs(pool, batch, what)
    if batch.n_heads is None:
        raise ValueError(f"{what}: the batch was made without n_heads")
    if Q.dim() != 3 or Q.shape != (batch.total_q, batch.n_heads, pool.d_head):
        raise ValueError(f"{what}: Q is (total_q, H_q, d) = {(batch.total_q, batch.n_heads, pool.d_head)}, got {tuple(Q.shape)}")
    if Q.device != pool.device:
        raise ValueError(f"{what}: Q on {Q.device}, the pool on {pool.device}")
    if Q.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f"{what}: Q is fp32, fp16 or bf16, not {Q.dtype}")
    if softcap is not None and not 1e-3 <= softcap <= 1e4:
        raise ValueError(f"softcap={softcap}: a number from 0.001 to 10000 (None: no cap)")
    if softmax_scale is not None and not 0.0 < softmax_scale < float("inf"):
        raise ValueError(f"softmax_scale={softmax_scale}: a positive number (None: 1 / sqrt(d_head))")
    if sinks is not None and (sinks.shape != (batch.n_heads,) or sinks.device != pool.device):
        raise ValueError(f"{what}: sinks are one number per query head on {pool.device}")
    _codebook(table_K, pool, what)
    a = _lib.PagedAttnArgs()
    a.struct_size = C.sizeof(_lib.PagedAttnArgs)
    a.q_dtype = _lib.dtype_enum(Q.dtype)
    a.q_stride[0], a.q_stride[1] = Q.stride(0), Q.stride(1)
    a.r_qmax = pool.K.qmax
    a.softmax_scale = pool.d_head ** -0.5 if softmax_scale is None else float(softmax_scale)
    a.softcap = 0.0 if softcap is None else float(softcap)
    return a


def _sized(a, pool, batch, size_fn, fn, Q, tables, sinks, what):
    """The workspace of a call with these arguments (addresses as they are: some are checked)."""
    a.K, a.V, a.plan, a.plan_data = pool.K.c_struct(), pool.V.c_struct(), batch.plan, batch.data.data_ptr()
    a.Q, a.table_K = Q.data_ptr(), tables[0].data_ptr()
    if len(tables) > 1:
        a.table_V = tables[1].data_ptr()
    with _lib.device_guard(pool.device):
        nbytes = size_fn(C.byref(a))
        if not nbytes:                           # the arguments are refused: the call says why
            _lib.check(fn(C.byref(a), None, 0, _lib.stream_ptr()), what)
    return nbytes


def paged_attention(Q: torch.Tensor, pool: PagedKV, batch: PagedBatch, table_K: torch.Tensor, table_V: torch.Tensor,
                    softmax_scale: Optional[float] = None, softcap: Optional[float] = None, sinks: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the batch's new tokens over their sequences' pages: (total_q, H_q, d), the queries of sequence after
    sequence.  Query i of a sequence stands at its position kv_len - q_len + i and sees the keys up to there (with the batch's window,
    the last ones).  ``softcap``: scores become softcap * tanh(score / softcap).  ``sinks`` (H_q): a logit per head that takes part in the
    softmax and has no value.  ``table_K`` / ``table_V``: the quantizer's fp16 tables, as in ``fused_attention_packed``.

    Operands are 16-bit as in the framework's other attention calls: queries (every row relative to a power of two of its own), decoded keys and
    values and the softmax weights have 11 bits, whatever the types of Q and ``out``; products are summed in fp32.

    Sequences with few rows (new tokens times heads per KV head up to 32) are read in place; the pages of prompt chunks are decoded
    once per call into operand tiles for the tensor cores, half a gigabyte at a time."""
    if Q.stride(-1) != 1:
        Q = Q.contiguous()
    if sinks is not None:
        sinks = sinks.to(torch.float32).contiguous()
    table_K, table_V = table_K.contiguous(), table_V.contiguous()
    O = torch.empty(Q.shape, dtype=Q.dtype, device=Q.device) if out is None else out
    # (a batch serves call after call, layer after layer: the struct of a call that differs in addresses only is kept with it, per thread)
    key = ("attn", get_ident(), pool.kind, Q.shape, Q.stride(), Q.dtype, Q.device, O.shape, O.stride(), O.dtype, O.device, table_K.shape,
           table_K.dtype, table_K.device, table_V.shape, table_V.dtype, table_V.device, softmax_scale, softcap,
           None if sinks is None else (sinks.shape, sinks.device))
    L = _lib.lib()
    hit = batch._calls.get(key)
    if hit is None:
        a = _attn_args(Q, pool, batch, table_K, softmax_scale, softcap, sinks, "paged_attention")
        _codebook(table_V, pool, "paged_attention")
        if O.shape != Q.shape or O.device != Q.device:
            raise ValueError(f"paged_attention: out is {tuple(Q.shape)} on {Q.device}")
        if batch.total_q == 0:
            return O
        if O.stride(-1) != 1:
            raise _lib.HqmqError("hqmq_b200: the output tensor needs unit stride on the last dim")
        a.o_dtype, a.O = _lib.dtype_enum(O.dtype), O.data_ptr()
        a.o_stride[0], a.o_stride[1] = O.stride(0), O.stride(1)
        nbytes = _sized(a, pool, batch, L.hqmq_paged_attn_workspace_bytes, L.hqmq_paged_attn, Q, (table_K, table_V), sinks, "hqmq_paged_attn")
        hit = batch._keep(key, (a, C.byref(a), nbytes))
    a, ref, nbytes = hit
    a.K, a.V = pool.K.c_struct(), pool.V.c_struct()
    a.Q, a.O, a.table_K, a.table_V = Q.data_ptr(), O.data_ptr(), table_K.data_ptr(), table_V.data_ptr()
    a.sinks = None if sinks is None else sinks.data_ptr()
    with _lib.device_guard(pool.device):
        ws = torch.empty(nbytes, dtype=torch.uint8, device=pool.device)
        rc = L.hqmq_paged_attn(ref, ws.data_ptr(), nbytes, _lib.stream_ptr())
        if rc:
            _lib.check(rc, "hqmq_paged_attn")
    return O


def _check_mass(t: torch.Tensor, pool: PagedKV, what: str):
    if t.shape != (pool.n_pages, pool.H_kv, pool.page_tokens) or t.dtype != torch.float32 or t.device != pool.device or not t.is_contiguous() or t.data_ptr() & 15:
        raise ValueError(f"{what}: weights are contiguous fp32 {(pool.n_pages, pool.H_kv, pool.page_tokens)} on {pool.device}, "
                         f"as PagedKV.new_mass gives them")


def paged_attention_mass(Q: torch.Tensor, pool: PagedKV, batch: PagedBatch, table_K: torch.Tensor,
                         softmax_scale: Optional[float] = None, softcap: Optional[float] = None, sinks: Optional[torch.Tensor] = None,
                         prior: Optional[torch.Tensor] = None, decay: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The softmax weight that every token of the batch's sequences receives from ``paged_attention``'s queries, summed over the
    queries that see it and over the query heads of its KV head, on top of ``decay * prior``: fp32 (pages, H_kv, page tokens), a
    new zeroed tensor or ``out`` (which may be ``prior``).  Only the batch's tokens are written.  Products are kept to 22 bits and sums
    in fp32, so weights may be compared and accumulated over many steps.  Q is fp16 or bf16; the scores of all queries are held
    in the workspace, so this is for decode steps and for the last tokens of a prompt."""
    if Q.stride(-1) != 1:
        Q = Q.contiguous()
    if sinks is not None:
        sinks = sinks.to(torch.float32).contiguous()
    table_K = table_K.contiguous()
    for t, what in ((prior, "prior"), (out, "out")):
        if t is not None:
            _check_mass(t, pool, f"paged_attention_mass: {what}")
    key = ("mass", get_ident(), pool.kind, Q.shape, Q.stride(), Q.dtype, Q.device, table_K.shape, table_K.dtype, table_K.device, softmax_scale,
           softcap, decay, None if sinks is None else (sinks.shape, sinks.device))
    L = _lib.lib()
    hit = batch._calls.get(key)
    if hit is None:
        a = _attn_args(Q, pool, batch, table_K, softmax_scale, softcap, sinks, "paged_attention_mass")
        if Q.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"paged_attention_mass: Q is fp16 or bf16, not {Q.dtype}")
        if batch.plan.no_mass:
            raise ValueError("paged_attention_mass: the scores of all of the batch's queries have no room; weigh a prompt's last tokens in a batch of their own")
        if not abs(decay) <= torch.finfo(torch.float32).max:
            raise ValueError(f"decay={decay}: a number that fp32 holds")
        a.decay, a.mass = float(decay), pool.K.c_struct().rs         # (any address: it is set below)
        nbytes = _sized(a, pool, batch, L.hqmq_paged_mass_workspace_bytes, L.hqmq_paged_mass, Q, (table_K,), sinks, "hqmq_paged_mass")
        hit = batch._keep(key, (a, C.byref(a), nbytes))
    if batch._unshared is False:
        raise ValueError("paged_attention_mass: a page of the batch belongs to two sequences, whose weights would be one")
    if out is None:
        out = pool.new_mass()
    a, ref, nbytes = hit
    a.K, a.V = pool.K.c_struct(), pool.V.c_struct()
    a.Q, a.table_K, a.mass = Q.data_ptr(), table_K.data_ptr(), out.data_ptr()
    a.prior = None if prior is None else prior.data_ptr()
    a.sinks = None if sinks is None else sinks.data_ptr()
    with _lib.device_guard(pool.device):
        ws = torch.empty(nbytes, dtype=torch.uint8, device=pool.device)
        rc = L.hqmq_paged_mass(ref, ws.data_ptr(), nbytes, _lib.stream_ptr())
        if rc:
            _lib.check(rc, "hqmq_paged_mass")
    return out


def paged_store(pool: PagedKV, K: PackedKV, V: PackedKV, batch: PagedBatch) -> None:
    """Encoded keys and values (``HQMQ.encode`` of (1, H_kv, total_q, d), tokens in the order of the batch's queries) become the last
    ``q_len`` tokens of their sequences.  What the pages held from the first of them on is gone: a sequence whose drafted tokens were
    rejected goes on with a batch of its shorter length, and storing a step twice stores it once (weights that its tokens had, see
    ``paged_attention_mass``, are the caller's to reset).  Pages that are written belong to one sequence."""
    _belongs(pool, batch, "paged_store")
    for name, src, dst in (("K", K, pool.K), ("V", V, pool.V)):
        if src.B != 1 or src.T < batch.total_q or (src.H, src.n_chunks, src.S, src.radius_bits) != (dst.H, dst.n_chunks, dst.S, dst.radius_bits):
            raise ValueError(f"paged_store: {name} holds {src.B} x {src.T} tokens of {src.H} heads, {4 * src.n_chunks} values, s{src.S}_r{src.radius_bits}; "
                             f"the batch has {batch.total_q} new ones of {dst.H}, {4 * dst.n_chunks}, s{dst.S}_r{dst.radius_bits}")
        if src.device != pool.device:
            raise ValueError(f"paged_store: {name} on {src.device}, the pool on {pool.device}")
        if src.scale_dtype != dst.scale_dtype or (src.with_outliers and (not dst.with_outliers or src.out_dtype != dst.out_dtype)):
            raise ValueError(f"paged_store: {name} has scales or outliers of a type that the pool does not keep")
    if not batch.stores_alone():
        raise ValueError("paged_store: a page that new tokens go to belongs to two sequences")
    a = _lib.PagedStoreArgs()
    a.struct_size = C.sizeof(_lib.PagedStoreArgs)
    a.src_K, a.src_V, a.K, a.V = K.c_struct(), V.c_struct(), pool.K.c_struct(), pool.V.c_struct()
    a.plan, a.plan_data = batch.plan, batch.data.data_ptr()
    with _lib.device_guard(pool.device):
        _lib.check(_lib.lib().hqmq_paged_store(C.byref(a), _lib.stream_ptr()), "hqmq_paged_store")


def paged_evict(pool: PagedKV, batch: PagedBatch, target: PagedBatch, mass: torch.Tensor, first: int = 4, last: int = 16,
                out_mass: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Cut every sequence of ``batch`` down to the length it has in ``target``, a batch of the same sequences over other pages of
    the pool: per KV head the last ``last`` tokens stay, the first ``first`` ones and, of the others, those with the largest
    ``mass`` (of equal ones the earlier; what is no number counts as the smallest).  The tokens that stay move, in order, to target's pages, their
    weights with them into ``out_mass`` (by default ``mass`` itself).  Returns the positions that were kept: int32 (sequences,
    H_kv, longest target), -1 behind a sequence's last."""
    _belongs(pool, batch, "paged_evict")
    _belongs(pool, target, "paged_evict")
    if len(batch.kv_lens) != len(target.kv_lens):
        raise ValueError(f"paged_evict: {len(batch.kv_lens)} sequences, and {len(target.kv_lens)} in the target")
    if first < 0 or last < 0:
        raise ValueError("paged_evict: first and last are counts")
    gone = batch.kv_lens - target.kv_lens
    if gone.min() < 0:
        more = gone < 0
        raise ValueError(f"paged_evict: sequence {int(more.argmax())} would grow from {int(batch.kv_lens[more][0])} to {int(target.kv_lens[more][0])} tokens")
    if target.shortest < first + last and ((gone > 0) & (target.kv_lens < first + last)).any():
        short = (gone > 0) & (target.kv_lens < first + last)
        raise ValueError(f"paged_evict: sequence {int(short.argmax())} keeps {int(target.kv_lens[short][0])} tokens, fewer than the {first} first and {last} last")
    if not target._unshared or not target.pages.isdisjoint(batch.pages):
        raise ValueError("paged_evict: target's pages belong to one sequence each and are none of the batch's")
    _check_mass(mass, pool, "paged_evict: mass")
    if out_mass is None:
        out_mass = mass
    _check_mass(out_mass, pool, "paged_evict: out_mass")
    n = len(batch.kv_lens)
    kept = torch.empty(n, pool.H_kv, target.longest, dtype=torch.int32, device=pool.device)
    if target.longest == 0:
        return kept
    key = ("evict", get_ident(), pool.kind, first, last, target.longest)
    hit = batch._calls.get(key)
    if hit is None:
        a = _lib.PagedEvictArgs()
        a.struct_size = C.sizeof(_lib.PagedEvictArgs)
        a.first, a.last, a.kept_stride = int(first), int(last), target.longest
        a.longest, a.most_kept = batch.longest, target.longest
        a.src = batch.plan
        hit = batch._keep(key, (a, C.byref(a)))
    a, ref = hit
    a.K, a.V, a.dst = pool.K.c_struct(), pool.V.c_struct(), target.plan
    a.mass, a.new_mass, a.kept = mass.data_ptr(), out_mass.data_ptr(), kept.data_ptr()
    a.src_data, a.dst_data = batch.data.data_ptr(), target.data.data_ptr()
    with _lib.device_guard(pool.device):
        rc = _lib.lib().hqmq_paged_evict(ref, _lib.stream_ptr())
        if rc:
            _lib.check(rc, "hqmq_paged_evict")
    return kept
