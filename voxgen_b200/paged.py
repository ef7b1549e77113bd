"""A paged KV cache for requests that come, grow and finish, over the ``vg_k_paged_*`` entry points.

K and V rows lie in pages of one pool. A :class:`PageTable` says on the device which pages each
sequence holds; one :meth:`PageTable.step` a token of the loop drops what finished or was rejected,
takes pages for the new tokens and gives their slot map. A :class:`PagedCache` holds the rows of one
or many layers over the same table::

    table = PageTable(seqs=64, pages=4096, page_rows=64, seq_pages=512)
    cache = PagedCache(table, kv_heads=2, head_dim=128, layers=28, summaries=True)
    step = table.step(counts, tokens, keep=keep)     # new rows of each sequence, packed in their order
    cache.append(step, k, v, layer=i)                # [tokens, 2, 128], any strides with contiguous channels
    out = cache.attention(q, sequences=step.sequences, positions=step.positions, layer=i)
    # long contexts: only the pages whose summaries allow the largest scores
    chosen = cache.select(q, budget=64, sinks=1, recent=2, sequences=step.sequences, positions=step.positions, layer=i)
    out = cache.attention(q, sequences=step.sequences, positions=step.positions, chosen=chosen, layer=i)

The calls run on the current CUDA stream (or ``stream``) and do not wait for the host; which sequences
a step refused is in ``table.status`` on the device. A table and its caches are used by one stream at a
time; a program that changes streams orders them itself, as for any tensor. The calls can be captured
in CUDA graphs; table and cache have to outlive them (:meth:`PagedCache.reserve`). Errors raise
:class:`~voxgen_b200.api.VoxGenError`.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Union

import torch

from . import api
from .api import VoxGenError
from .kv4 import DTYPES, _capturing, _check, _current_stream, _invalid, _on_its_device

STATUS_FULL, STATUS_NO_PAGES, STATUS_BAD_COUNT, STATUS_TIMEOUT, STATUS_NONFINITE = 1, 2, 4, 8, 16


def _device_of(device, given) -> torch.device:
    if device is None:
        device = given.device if given is not None else torch.device("cuda")
    device = torch.device(device)
    if device.type != "cuda":
        raise _invalid("a paged cache lives on a CUDA device")
    return torch.device("cuda", torch.cuda.current_device()) if device.index is None else device


def _expect(x: torch.Tensor, dtype, shape, device, what: str) -> torch.Tensor:
    if x.dtype != dtype or tuple(x.shape) != tuple(shape) or x.device != device or not x.is_contiguous():
        raise _invalid(f"{what}: expected contiguous {dtype} {list(shape)} on {device}, got {x.dtype} {list(x.shape)} "
                       f"on {x.device}")
    return x


def _ints(x: Optional[torch.Tensor], shape, device, what: str) -> Optional[int]:
    """Device address of an int32 tensor of a shape."""
    return None if x is None else _expect(x, torch.int32, shape, device, what).data_ptr()


def _sizes(**sizes) -> None:
    for name, x in sizes.items():
        if not 0 <= x < 1 << 32:
            raise _invalid(f"{name}: {x} is not a size")


class Step:
    """What a step leaves for the calls after it (int32 on the device): ``starts`` [seqs + 1], the first token of each
    sequence and the number of all; ``slots`` (page * page_rows + row), ``positions`` and ``sequences`` of each token, -1
    for those past the last and those of a refused sequence; ``runs`` [n, 4], the new rows page by page."""

    _NAMES = ("starts", "slots", "positions", "sequences", "runs")

    def __init__(self, table: "PageTable", tokens: int):
        self.table, self.tokens = table, tokens
        total, offsets, self._views = table._layout(tokens)[:3]
        self._buffer = torch.empty(total, dtype=torch.int32, device=table.device)
        self._parts, self._age = [None] * 5, None
        at = self._buffer.data_ptr()
        self.desc = api.PagedStepDesc(*[at + 4 * o for o in offsets], tokens)
        self._ref = C.byref(self.desc)

    @classmethod
    def of(cls, table: "PageTable", starts: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor,
           sequences: torch.Tensor, runs: torch.Tensor) -> "Step":
        """A step from arrays in hand, such as copies of an earlier one's (each starts on 16 bytes). That they are those of the
        table's last step is up to the caller."""
        step = cls.__new__(cls)
        step.table, step.tokens, step._age = table, slots.numel(), None
        tokens = step.tokens
        shapes = (table.seqs + 1,), (tokens,), (tokens,), (tokens,), (table._layout(tokens)[3], 4)
        step._parts = [_expect(x, torch.int32, shape, table.device, what) for x, shape, what in
                       zip((starts, slots, positions, sequences, runs), shapes, cls._NAMES)]
        # an array of no tokens has no address; the entry points want one that is not null, and do not read it
        step.desc = api.PagedStepDesc(*[x.data_ptr() or 64 for x in step._parts], tokens)
        step._ref = C.byref(step.desc)
        return step

    def _part(self, i: int) -> torch.Tensor:
        x = self._parts[i]
        if x is None:
            x = self._parts[i] = self._buffer.as_strided(*self._views[i])
        return x

    starts = property(lambda self: self._part(0))
    slots = property(lambda self: self._part(1))
    positions = property(lambda self: self._part(2))
    sequences = property(lambda self: self._part(3))
    runs = property(lambda self: self._part(4))


class PageTable:
    """Which of a pool's ``pages`` pages of ``page_rows`` rows each of ``seqs`` sequences holds, ``seq_pages`` at most.

    ``table`` int32 [seqs, seq_pages], ``rows`` and ``status`` int32 [seqs], ``free`` int32 [pages] (a stack of free pages)
    and ``pool`` int32 [2] are on the device; they may be given instead of allocated. ``pool`` holds the stack's height, and
    STATUS_TIMEOUT once a wait inside an attention ran out, STATUS_NONFINITE once an append met a NaN or a value past the
    cache's largest. ``status`` is that of the last step: STATUS_FULL, STATUS_NO_PAGES or
    STATUS_BAD_COUNT for a sequence that it refused, else 0."""

    def __init__(self, seqs: int, pages: int, page_rows: int, seq_pages: int, *, device=None,
                 table: Optional[torch.Tensor] = None, rows: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None, free: Optional[torch.Tensor] = None,
                 pool: Optional[torch.Tensor] = None):
        _sizes(seqs=seqs, pages=pages, page_rows=page_rows, seq_pages=seq_pages)
        probe = api.PagedTableDesc(*[64] * 5, seqs, seq_pages, pages, page_rows)   # sizes before memory
        _check(api.lib().vg_k_paged_runs(C.byref(probe), 1, C.byref(C.c_uint32())),
               f"a table of {seqs} sequences of {seq_pages} pages, {pages} pages of {page_rows} rows")
        self.device = device = _device_of(device, table)
        self._index = device.index
        self.seqs, self.pages, self.page_rows, self.seq_pages = seqs, pages, page_rows, seq_pages

        def ints(x, shape, what, make):
            return make() if x is None else _expect(x, torch.int32, shape, device, what)

        on = dict(dtype=torch.int32, device=device)
        self.table = ints(table, (seqs, seq_pages), "table", lambda: torch.full((seqs, seq_pages), -1, **on))
        self.rows = ints(rows, (seqs,), "rows", lambda: torch.zeros(seqs, **on))
        self.status = ints(status, (seqs,), "status", lambda: torch.zeros(seqs, **on))
        self.free = ints(free, (pages,), "free", lambda: torch.arange(pages, **on))
        self.pool = ints(pool, (2,), "pool", lambda: torch.tensor([pages, 0], **on))
        self.desc = api.PagedTableDesc(*[x.data_ptr() for x in (self.table, self.rows, self.status, self.free, self.pool)],
                                       seqs, seq_pages, pages, page_rows)
        self._ref = C.byref(self.desc)
        self._layouts = {}
        self._age = 0            # steps taken by calls (and resets); those of a graph's replays are not known here
        self._lib = api.lib()

    def _layout(self, tokens: int):
        """Of a step's arrays: the sum of their sizes, where each starts, (size, strides, start) of each, and the runs."""
        found = self._layouts.get(tokens)
        if found is None:
            _sizes(tokens=tokens)
            n = C.c_uint32()
            _check(self._lib.vg_k_paged_runs(self._ref, tokens, C.byref(n)), f"a step of {tokens} tokens")
            offsets, total = [], 0
            for x in (self.seqs + 1, tokens, tokens, tokens, 4 * n.value):
                offsets.append(total)
                total += x + -x % 4      # each starts on 16 bytes
            views = [((x,), (1,), at) for x, at in zip((self.seqs + 1, tokens, tokens, tokens), offsets)]
            views.append(((n.value, 4), (4, 1), offsets[4]))
            if len(self._layouts) > 256:
                self._layouts.clear()
            found = self._layouts[tokens] = total, offsets, views, n.value
        return found

    @_on_its_device
    def step(self, counts: torch.Tensor, tokens: int, *, keep: Optional[torch.Tensor] = None,
             into: Optional[Step] = None) -> Step:
        """Cuts each sequence to its first ``keep[s]`` rows (default, or below 0: all), gives back the pages that it then
        does not need, and makes room for ``counts[s]`` new rows; both int32 [seqs]. The new tokens are packed in the order
        of sequences into ``tokens`` places (at least their number). A sequence that does not fit keeps its rows, its tokens
        have no slot, and ``status`` says why. ``into``: an earlier step of as many tokens to write over."""
        if into is None:
            into = Step(self, tokens)
        elif into.table is not self or into.tokens != tokens:
            raise _invalid(f"into: another table's step, or one of {into.tokens} tokens for one of {tokens}")
        rc = self._lib.vg_k_paged_step(self._ref, _ints(counts, (self.seqs,), self.device, "counts"),
                                       _ints(keep, (self.seqs,), self.device, "keep"), into._ref, _current_stream(self._index))
        if rc:
            raise VoxGenError(rc, f"a step of {tokens} tokens")
        if _capturing():
            into._age = None
        else:
            into._age = self._age = self._age + 1
        return into

    def reset(self) -> None:
        """Empties every sequence: all pages are free again."""
        if not _capturing():
            self._age += 1
        self.table.fill_(-1)
        self.rows.zero_()
        self.status.zero_()
        torch.arange(self.pages, dtype=torch.int32, device=self.device, out=self.free)
        self.pool[0].fill_(self.pages)
        self.pool[1].zero_()


class PagedCache:
    """K and V rows of ``layers`` layers in the pages of a table, ``dtype`` float16 or bfloat16.

    ``data`` [layers, pages, kv_heads, 2 (K, V), page_rows, head_dim] may be given instead of allocated, with one layer
    without the first dimension; so may ``summaries`` [layers, pages, kv_heads, 2, head_dim] of the same type: per channel
    the smallest and the largest K of the rows that a page held at its last append, which :meth:`select` needs (True
    allocates them). A step that cuts a page's rows and adds none to it leaves its summary as it was: still a bound for the
    rows that are left, though perhaps a loose one, until the page's next append."""

    def __init__(self, table: PageTable, kv_heads: int, head_dim: int, *, dtype: torch.dtype = torch.float16,
                 layers: int = 1, data: Optional[torch.Tensor] = None,
                 summaries: Union[bool, torch.Tensor, None] = False):
        nbytes = cache_bytes(table.pages, table.page_rows, kv_heads, head_dim)
        if dtype not in (torch.float16, torch.bfloat16):
            raise VoxGenError(-4, f"a cache of {dtype} is not supported")
        if layers < 1:
            raise _invalid(f"{layers} layers")
        self.table, self.device, self._index = table, table.device, table._index
        self.kv_heads, self.head_dim, self.dtype, self.layers = kv_heads, head_dim, dtype, layers
        shape = layers, table.pages, kv_heads, 2, table.page_rows, head_dim

        def pool(x, shape, what):
            if not isinstance(x, torch.Tensor):
                return torch.zeros(shape, dtype=dtype, device=self.device)
            if x.dim() == len(shape) - 1 and layers == 1:
                x = x.unsqueeze(0)
            return _expect(x, dtype, shape, self.device, what)

        self.data = pool(data, shape, "data")
        keeps = isinstance(summaries, torch.Tensor) or bool(summaries)
        self.summaries = pool(summaries, (*shape[:4], head_dim), "summaries") if keeps else None
        self._descs = [api.PagedCacheDesc(C.pointer(table.desc), self.data.data_ptr() + i * nbytes[0],
                                          self.summaries.data_ptr() + i * nbytes[1] if keeps else None,
                                          DTYPES[dtype], kv_heads, head_dim) for i in range(layers)]
        self._refs = [C.byref(d) for d in self._descs]
        self._scale = 1.0 / math.sqrt(head_dim)
        self._need = {}
        self._workspace = None
        self._captured = False   # whether a CUDA graph holds the workspace's address
        self._kept = []          # workspaces outgrown since, which graphs still write to
        self._lib = api.lib()

    # -- rows -------------------------------------------------------------------------------
    def k(self, layer: int = 0) -> torch.Tensor:
        """A layer's K rows [pages, kv_heads, page_rows, head_dim] (a view)."""
        return self.data[layer, :, :, 0]

    def v(self, layer: int = 0) -> torch.Tensor:
        """A layer's V rows, likewise."""
        return self.data[layer, :, :, 1]

    def _layer(self, layer: int):
        if not 0 <= layer < self.layers:
            raise _invalid(f"layer {layer} of {self.layers}")
        return self._refs[layer]

    def _rows_of(self, x: torch.Tensor, heads: int, what: str) -> int:
        """The type of rows [n, heads, head_dim]."""
        shape = x.shape
        if len(shape) != 3 or shape[1] != heads or shape[2] != self.head_dim or x.device != self.device:
            raise _invalid(f"{what}: expected [n, {heads}, {self.head_dim}] on {self.device}, got {list(shape)} on {x.device}")
        dtype = DTYPES.get(x.dtype)
        if dtype is None:
            raise VoxGenError(-4, f"{what}: {x.dtype} is not supported")
        return dtype

    @staticmethod
    def _strides(x: torch.Tensor):
        """Element strides {row, head} for the C ABI; None when contiguous."""
        if x.is_contiguous():
            return None
        if x.stride(2) != 1:
            raise _invalid("channels must be contiguous")
        return (C.c_int64 * 2)(*x.stride()[:2])

    @_on_its_device
    def append(self, step: Step, k: torch.Tensor, v: torch.Tensor, *, layer: int = 0) -> None:
        """Stores the K and V rows [tokens, kv_heads, head_dim] of the table's last step (an older one is refused: its pages
        may be another sequence's by now); rows of tokens without a slot are passed over. Values are rounded to the cache's
        type; those past its largest finite number are held as that one, and ``table.pool[1]`` then has STATUS_NONFINITE, as
        for NaN."""
        ref = self._layer(layer)
        dtype = self._rows_of(k, self.kv_heads, "k")
        if step.table is not self.table:
            raise _invalid("the step is another table's")
        if step._age is not None and step._age != self.table._age:
            raise _invalid("the step is not the table's last one")
        if v.shape != k.shape or v.dtype is not k.dtype or v.device != self.device or k.shape[0] != step.tokens:
            raise _invalid(f"k and v must agree in shape, type and device, and have the step's {step.tokens} rows")
        rc = self._lib.vg_k_paged_append(ref, step._ref, k.data_ptr(), v.data_ptr(), dtype, self._strides(k),
                                         self._strides(v), _current_stream(self._index))
        if rc:
            raise VoxGenError(rc, f"append of {step.tokens} rows")

    # -- attention --------------------------------------------------------------------------
    def _queries(self, q: torch.Tensor, sequences, positions):
        if q.dim() != 3:
            raise _invalid("q: expected [queries, heads, head_dim]")
        n, heads, _ = q.shape
        return (n, heads, self._rows_of(q, heads, "q"),
                None if sequences is None else _ints(sequences, (n,), self.device, "sequences"),
                None if positions is None else _ints(positions, (n,), self.device, "positions"))

    @_on_its_device
    def select(self, q: torch.Tensor, budget: int, *, sinks: int = 0, recent: int = 1,
               sequences: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
               layer: int = 0) -> torch.Tensor:
        """The ``budget`` pages that each query [queries, heads, head_dim] is to attend, int32 [queries, kv_heads, budget]
        in ascending order, -1 past a query's pages: its first ``sinks`` and last ``recent`` ones and those whose summaries
        allow the largest scores, summed over the heads that share a KV head. ``sequences`` and ``positions`` as for
        :meth:`attention`."""
        ref = self._layer(layer)
        n, heads, dtype, sequences, positions = self._queries(q, sequences, positions)
        if self.summaries is None:
            raise _invalid("this cache keeps no summaries")
        _sizes(budget=budget, sinks=sinks, recent=recent)
        chosen = torch.empty((n, self.kv_heads, budget), dtype=torch.int32, device=self.device)
        if n == 0:
            return chosen
        rc = self._lib.vg_k_paged_select(ref, q.data_ptr(), dtype, n, heads, self._strides(q), sequences, positions, budget,
                                         sinks, recent, chosen.data_ptr(), _current_stream(self._index))
        if rc:
            raise VoxGenError(rc, f"selection of {budget} pages ({sinks} sinks, {recent} recent) for {n} queries of {heads} "
                              f"heads on {self.kv_heads} KV heads, {self.table.seqs} sequences of {self.table.seq_pages} pages")
        return chosen

    def _work(self, queries: int, heads: int, budget: int) -> torch.Tensor:
        """A zeroed workspace, large enough for the call; while a graph is being captured the cache's own does not grow,
        and such a call has one of its own, zeroed by every replay (as for the 4-bit cache)."""
        need = self._need.get((queries, heads, budget))
        if need is None:
            n = C.c_uint64()
            _check(self._lib.vg_k_paged_attention_bytes(self._refs[0], queries, heads, budget, C.byref(n)),
                   f"attention of {queries} queries of {heads} heads over {self.kv_heads} KV heads")
            if len(self._need) > 1024:
                self._need.clear()
            need = self._need[queries, heads, budget] = n.value
        ws, capturing = self._workspace, _capturing()
        if ws is None or ws.numel() < need:
            fresh = torch.zeros(need, dtype=torch.uint8, device=self.device)
            if capturing:
                return fresh
            if ws is not None:
                ws.record_stream(torch.cuda.current_stream(self._index))
                if self._captured:
                    self._kept.append(ws)
            self._workspace, self._captured = fresh, False
            return fresh
        self._captured |= capturing
        return ws

    @_on_its_device
    def reserve(self, queries: int, heads: int, budget: int = 0) -> None:
        """Makes the workspace large enough for :meth:`attention` of up to ``queries`` queries of ``heads`` heads (with lists of
        up to ``budget`` pages, if not 0), before a CUDA graph of such calls is captured: without it each of the graph's
        replays zero-fills a workspace of its own."""
        if _capturing():
            raise _invalid("reserve: the workspace does not grow while a graph is being captured")
        if not (0 < heads < 1 << 32 and 0 < queries < 1 << 32 and 0 <= budget < 1 << 32):
            raise _invalid(f"reserve: {queries} queries, {heads} heads, {budget} pages")
        while queries:     # fewer queries may need more: very many are not cut into pieces, which the workspace is for
            self._work(queries, heads, budget)
            queries //= 2

    @_on_its_device
    def attention(self, q: torch.Tensor, *, sequences: Optional[torch.Tensor] = None,
                  positions: Optional[torch.Tensor] = None, chosen: Optional[torch.Tensor] = None,
                  scale: Optional[float] = None, out: Optional[torch.Tensor] = None, layer: int = 0) -> torch.Tensor:
        """Attention of single tokens' queries [queries, heads, head_dim].

        Query i is of sequence ``sequences[i]`` (default: i) and attends its rows 0 .. ``positions[i]`` (default: all that
        are held); a position of -1 sees no row and gives zeros. ``chosen`` int32 [queries, kv_heads, n] restricts it to
        rows of these pages of the sequence. ``scale`` is 1/sqrt(head_dim) by default. ``out`` does not overlap ``q``."""
        ref = self._layer(layer)
        n, heads, dtype, sequences, positions = self._queries(q, sequences, positions)
        strides = self._strides(q)
        if out is None:
            out = torch.empty_like(q) if strides is None else torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != self.device or not out.is_contiguous():
            raise _invalid("out must be contiguous and like q")
        budget, pages = 0, None
        if chosen is not None:
            budget = chosen.shape[-1] if chosen.dim() == 3 else 0
            pages = _ints(chosen, (n, self.kv_heads, max(budget, 1)), self.device, "chosen")
        if n == 0:
            return out
        ws = self._work(n, heads, budget)
        rc = self._lib.vg_k_paged_attention(
            ref, q.data_ptr(), dtype, n, heads, strides, sequences, positions, pages, budget,
            self._scale if scale is None else scale, out.data_ptr(), ws.data_ptr(), ws.numel(), _current_stream(self._index))
        if rc:
            raise VoxGenError(rc, f"attention of {n} queries of {heads} heads on {self.kv_heads} KV heads, {self.table.seqs} "
                              "sequences")
        return out


def cache_bytes(pages: int, page_rows: int, kv_heads: int, head_dim: int):
    """Device bytes of one layer's rows and of its summaries. Needs no GPU."""
    _sizes(pages=pages, page_rows=page_rows, kv_heads=kv_heads, head_dim=head_dim)
    data, summaries = C.c_uint64(), C.c_uint64()
    _check(api.lib().vg_k_paged_bytes(pages, page_rows, kv_heads, head_dim, C.byref(data), C.byref(summaries)),
           f"a paged cache of {pages} pages of {page_rows} rows, {kv_heads} KV heads of {head_dim}")
    return data.value, summaries.value
