"""Sessions on a KV cache held in 4 bits, over the ``vg_k_kv4_*`` entry points.

:class:`Kv4Cache` holds the rows of one or many sequences (streams, or the layers of a session)
on the device, 4.5 bits a value. The calls of a serving loop take and return torch tensors on the
cache's device, run on the current CUDA stream (or ``stream``), and do not wait for the host:
how many rows a sequence holds lives in ``cache.state`` on the device::

    cache = Kv4Cache(seqs=16, kv_heads=2, head_dim=128, capacity=4096, track=True)
    cache.append(k, v)                  # [16, new, 2, 128], any strides with contiguous channels
    out = cache.attention(q)            # [16, new, 16, 128], causal within the new tokens
    accepted, token = verify_draft(drafted, draft_probs, target_probs, u_accept, u_sample)
    cache.append(k, v, at=rows)         # overwrites what was appended past rows[s]
    cache.evict(budget=2048, recent=256, sinks=4)

A cache is used by one stream at a time; a program that changes streams orders them itself, as for
any tensor. The calls can be captured in CUDA graphs; the cache has to outlive them
(:meth:`Kv4Cache.reserve`). Errors raise :class:`~voxgen_b200.api.VoxGenError`; what only the device can know (an
append past the capacity, a NaN or a value past 7168 among the rows) is in ``cache.status()``.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
from typing import Optional, Tuple

import torch

from . import api
from .api import VoxGenError

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
STATUS_FULL, STATUS_BAD_ROW, STATUS_NONFINITE, STATUS_TIMEOUT = 1, 2, 4, 8


def _check(rc: int, what: str) -> None:
    if rc:
        raise VoxGenError(rc, what)


def _invalid(what: str) -> VoxGenError:
    return VoxGenError(-1, what)


# The current stream's address without building a Stream object, which takes as long as a small kernel.
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", None) or torch.cuda.is_current_stream_capturing


def _on(device, stream):
    """A context in which ``device`` is current, and ``stream`` (an address or a torch stream) when one is given."""
    if stream is None:
        return torch.cuda.device(device)
    if isinstance(stream, int):   # torch takes address 0 for a request of a stream from its pool
        stream = torch.cuda.ExternalStream(stream, device=device) if stream else torch.cuda.default_stream(device)
    return torch.cuda.stream(stream)


def _on_its_device(call):
    """Runs a method with the cache's device as the current one, on ``stream`` when one is given: what it allocates
    then belongs to that stream too."""
    def run(self, *args, stream=None, **kwargs):
        if stream is None and _current_device() == self._index:
            return call(self, *args, **kwargs)
        with _on(self.device, stream):
            return call(self, *args, **kwargs)
    return functools.wraps(call)(run)


def _ints(x: Optional[torch.Tensor], n: int, device, what: str) -> Optional[int]:
    """Device address of an int32 tensor with one value per sequence."""
    if x is None:
        return None
    if x.dtype != torch.int32 or x.shape != (n,) or x.device != device or not x.is_contiguous():
        raise _invalid(f"{what} must be {n} contiguous int32 values on {device}")
    return x.data_ptr()


def _strides(x: torch.Tensor):
    """Element strides of [seqs, tokens, heads, head_dim] for the C ABI; None when contiguous."""
    if x.is_contiguous():
        return None
    if x.shape[3] > 1 and x.stride(3) != 1:
        raise _invalid("channels must be contiguous")
    return (C.c_int64 * 3)(*x.stride()[:3])


class Kv4Cache:
    """K and V rows of ``seqs`` sequences in 4 bits, ``capacity`` rows each.

    ``track`` keeps the attention that each row draws and the position it holds, which
    :meth:`evict` needs. ``data``, ``state``, ``weights`` and ``positions`` may be given instead
    of allocated: uint8 of :func:`cache_bytes` bytes, int32 ``[seqs, 4]`` (rows held, next
    position, status bits, 0), fp32 and int32 ``[seqs, kv_heads, capacity]``.
    """

    def __init__(self, seqs: int, kv_heads: int, head_dim: int, capacity: int, *, track: bool = False, device=None,
                 data: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                 weights: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None):
        nbytes = cache_bytes(seqs, kv_heads, head_dim, capacity)
        if device is None:
            device = data.device if data is not None else torch.device("cuda", torch.cuda.current_device())
        self.device = device = torch.device(device)
        if device.type != "cuda":
            raise _invalid("a 4-bit cache lives on a CUDA device")
        if device.index is None:
            self.device = device = torch.device("cuda", torch.cuda.current_device())
        rows = (seqs, kv_heads, capacity)
        if data is None:
            data = torch.empty(nbytes, dtype=torch.uint8, device=device)
        if state is None:
            state = torch.zeros(seqs, 4, dtype=torch.int32, device=device)
        if track and weights is None:
            weights = torch.zeros(rows, dtype=torch.float32, device=device)
        if track and positions is None:
            positions = torch.zeros(rows, dtype=torch.int32, device=device)
        for x, dtype, shape, what in ((data, torch.uint8, None, "data"), (state, torch.int32, (seqs, 4), "state"),
                                      (weights, torch.float32, rows, "weights"),
                                      (positions, torch.int32, rows, "positions")):
            if x is None:
                continue
            if x.dtype != dtype or x.device != device or not x.is_contiguous() or (shape and tuple(x.shape) != shape) \
                    or (shape is None and x.numel() < nbytes):
                raise _invalid(f"{what}: expected contiguous {dtype} of {shape or nbytes} on {device}")
        self.seqs, self.kv_heads, self.head_dim, self.capacity = seqs, kv_heads, head_dim, capacity
        self._index = device.index
        self._scale = 1.0 / math.sqrt(head_dim)
        self.data, self.state, self.weights, self.positions = data, state, weights, positions
        address = [None if x is None else x.data_ptr() for x in (data, state, weights, positions)]
        self.desc = api.Kv4CacheDesc(*address, seqs, kv_heads, head_dim, capacity)
        self._ref = C.byref(self.desc)
        self._need = {}
        self._workspace = None
        self._captured = False   # whether a CUDA graph holds the workspace's address
        self._kept = []          # workspaces outgrown since, which graphs still write to
        self._lib = api.lib()

    # -- rows -------------------------------------------------------------------------------
    def rows(self) -> torch.Tensor:
        """Rows held by each sequence (a view of the device state)."""
        return self.state[:, 0]

    def status(self) -> list:
        """Status bits of each sequence (STATUS_FULL, STATUS_BAD_ROW, STATUS_NONFINITE,
        STATUS_TIMEOUT). Waits for the device."""
        return self.state[:, 2].tolist()

    def reset(self) -> None:
        """Empties every sequence and clears its status."""
        self.state.zero_()

    def _rows_of(self, x: torch.Tensor, heads: int, what: str) -> int:
        shape = x.shape
        if len(shape) != 4 or shape[0] != self.seqs or shape[2] != heads or shape[3] != self.head_dim \
                or x.device != self.device:
            raise _invalid(f"{what}: expected [{self.seqs}, tokens, {heads}, {self.head_dim}] on {self.device}, "
                           f"got {list(shape)} on {x.device}")
        dtype = DTYPES.get(x.dtype)
        if dtype is None:
            raise VoxGenError(-4, f"{what}: {x.dtype} is not supported")
        return dtype

    @_on_its_device
    def append(self, k: torch.Tensor, v: torch.Tensor, *, at: Optional[torch.Tensor] = None,
               counts: Optional[torch.Tensor] = None) -> None:
        """Stores new K and V rows ``[seqs, tokens, kv_heads, head_dim]`` from row ``at[s]`` on (default: after
        the rows held); ``counts[s]`` says how many of them a sequence has (default: all)."""
        dtype = self._rows_of(k, self.kv_heads, "k")
        if v.shape != k.shape or v.dtype is not k.dtype or v.device != self.device:
            raise _invalid("k and v must agree in shape, type and device")
        tokens = k.shape[1]
        rc = self._lib.vg_k_kv4_append(
            self._ref, k.data_ptr(), v.data_ptr(), dtype, tokens, _strides(k), _strides(v),
            _ints(at, self.seqs, self.device, "at"), _ints(counts, self.seqs, self.device, "counts"),
            _current_stream(self._index))
        if rc:
            raise VoxGenError(rc, f"append of {tokens} rows to a cache of {self.capacity}")

    @_on_its_device
    def read(self, tokens: int, *, first: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float16
             ) -> Tuple[torch.Tensor, torch.Tensor]:
        """Values of rows ``first[s] .. first[s] + tokens - 1`` (default: from row 0), K and V; rows that are not
        held read as 0."""
        if dtype not in DTYPES:
            raise VoxGenError(-4, f"{dtype} is not supported")
        k, v = self.data.new_empty((2, self.seqs, tokens, self.kv_heads, self.head_dim), dtype=dtype).unbind()
        rc = self._lib.vg_k_kv4_read(self._ref, _ints(first, self.seqs, self.device, "first"), tokens, DTYPES[dtype],
                                     k.data_ptr(), v.data_ptr(), _current_stream(self._index))
        if rc:
            raise VoxGenError(rc, f"read of {tokens} rows")
        return k, v

    # -- attention --------------------------------------------------------------------------
    def _work(self, heads: int, tokens: int) -> torch.Tensor:
        """A zeroed workspace, large enough for the call. While a graph is being captured the cache's own does not grow:
        its zero-fill would run with the replay only, after calls that need it. Such a call has one of its own, zeroed
        by every replay."""
        need = self._need.get((heads, tokens))
        if need is None:
            n = C.c_uint64()
            _check(self._lib.vg_k_kv4_attention_bytes(self._ref, heads, tokens, C.byref(n)),
                   f"attention of {heads} heads over {self.kv_heads} KV heads, {tokens} tokens")
            need = self._need[heads, tokens] = n.value
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
    def reserve(self, heads: int, tokens: int) -> None:
        """Makes the workspace large enough for :meth:`attention` of ``tokens`` tokens and ``heads`` heads, before a
        CUDA graph of such calls is captured: without it each of the graph's replays zero-fills a workspace of its own."""
        if _capturing():
            raise _invalid("reserve: the workspace does not grow while a graph is being captured")
        if not (0 < heads < 1 << 32 and 0 < tokens < 1 << 32):
            raise _invalid(f"reserve: {heads} heads, {tokens} tokens")
        self._work(heads, tokens)

    @_on_its_device
    def attention(self, q: torch.Tensor, *, counts: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                  track: Optional[bool] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of the last ``tokens`` rows' queries ``[seqs, tokens, heads, head_dim]``, causal within them.

        Adds the attention that each row draws to ``weights`` when the cache tracks it (``track=False`` leaves
        them). ``scale`` is 1/sqrt(head_dim) by default. ``out`` may be ``q`` itself where nothing is tracked."""
        if q.dim() != 4:
            raise _invalid("q: expected [seqs, tokens, heads, head_dim]")
        _, tokens, heads, _ = q.shape
        dtype = self._rows_of(q, heads, "q")
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != self.device or not out.is_contiguous():
            raise _invalid("out must be contiguous and like q")
        if track is None:
            track = self.weights is not None
        elif track and self.weights is None:
            raise _invalid("this cache does not track attention")
        if track and out.data_ptr() == q.data_ptr():
            raise _invalid("out cannot be q in a call that tracks attention")
        ws = self._work(heads, tokens)
        rc = self._lib.vg_k_kv4_attention(
            self._ref, q.data_ptr(), dtype, heads, tokens, _strides(q),
            _ints(counts, self.seqs, self.device, "counts"), self._scale if scale is None else scale, track,
            out.data_ptr(), ws.data_ptr(), ws.numel(), _current_stream(self._index))
        if rc:
            raise VoxGenError(rc, f"attention of {tokens} tokens, {heads} heads")
        return out

    # -- eviction ---------------------------------------------------------------------------
    @_on_its_device
    def evict(self, budget: int, recent: int = 0, sinks: int = 0, *, into: Optional["Kv4Cache"] = None) -> None:
        """Cuts sequences that hold more than ``budget`` rows to it: the last ``recent`` and first ``sinks``
        positions stay, and the rest that drew the most attention. Rows then are not in the order of their positions:
        drop rejected rows (``append`` with ``at``) before this call, not after it. ``into``: a cache over the same ``data``
        whose state, weights and positions receive the result instead."""
        rc = self._lib.vg_k_kv4_evict(self._ref, budget, recent, sinks, None if into is None else into._ref,
                                      _current_stream(self._index))
        if rc:
            raise VoxGenError(rc, f"eviction to {budget} rows ({recent} recent, {sinks} sinks) of a cache of "
                              f"{self.capacity}" + ("" if self.weights is not None else " that does not track attention"))


def cache_bytes(seqs: int, kv_heads: int, head_dim: int, capacity: int) -> int:
    """Device bytes of a cache's rows. Needs no GPU."""
    n = C.c_uint64()
    for x in (seqs, kv_heads, head_dim, capacity):
        if not 0 <= x < 1 << 32:
            raise _invalid(f"{x} is not a size")
    _check(api.lib().vg_k_kv4_bytes(seqs, kv_heads, head_dim, capacity, C.byref(n)),
           f"a 4-bit cache of {seqs} sequences, {kv_heads} KV heads of {head_dim}, {capacity} rows")
    return n.value


def verify_draft(tokens: torch.Tensor, draft: torch.Tensor, target: torch.Tensor, u_accept: torch.Tensor,
                 u_sample: torch.Tensor, *, counts: Optional[torch.Tensor] = None,
                 stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Accepts drafted tokens and draws the token after them, from given random numbers in [0, 1).

    ``tokens`` int32 ``[seqs, drafted]``, ``draft`` ``[seqs, drafted, vocab]`` and ``target``
    ``[seqs, drafted + 1, vocab]`` fp32 probabilities, ``u_accept`` ``[seqs, drafted]``, ``u_sample``
    ``[seqs]``. Returns int32 ``accepted`` and ``next``, one of each per sequence."""
    if tokens.dim() != 2 or draft.dim() != 3:
        raise _invalid("verify_draft: expected tokens [seqs, drafted] and draft [seqs, drafted, vocab]")
    seqs, drafted = tokens.shape
    vocab = draft.shape[2]
    device = tokens.device
    for x, dtype, shape, what in ((tokens, torch.int32, (seqs, drafted), "tokens"),
                                  (draft, torch.float32, (seqs, drafted, vocab), "draft"),
                                  (target, torch.float32, (seqs, drafted + 1, vocab), "target"),
                                  (u_accept, torch.float32, (seqs, drafted), "u_accept"),
                                  (u_sample, torch.float32, (seqs,), "u_sample")):
        if x.dtype != dtype or x.shape != shape or x.device != device or not x.is_contiguous():
            raise _invalid(f"verify_draft: {what} must be contiguous {dtype} {list(shape)} on {device}")
    if device.type != "cuda":
        raise _invalid("verify_draft runs on a CUDA device")
    if stream is not None or _current_device() != device.index:
        with _on(device, stream):
            return verify_draft(tokens, draft, target, u_accept, u_sample, counts=counts)
    accepted, token = tokens.new_empty((2, seqs)).unbind()
    rc = api.lib().vg_k_verify_draft(
        tokens.data_ptr(), draft.data_ptr(), target.data_ptr(), u_accept.data_ptr(), u_sample.data_ptr(),
        _ints(counts, seqs, device, "counts"), seqs, drafted, vocab, accepted.data_ptr(), token.data_ptr(),
        _current_stream(device.index))
    if rc:
        raise VoxGenError(rc, f"verification of {drafted} tokens of a vocabulary of {vocab}")
    return accepted, token
