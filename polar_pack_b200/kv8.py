"""The 8-bit KV cache and the operators that work on it.

A :class:`KV8Cache` holds one layer's keys and values of ``batch`` sequences
as uint8 codes with one float32 scale for each block of 64 positions and head:
``value = (code - 128) * scale``.  The block of a sequence's last token is kept
in FP16 (the tail) until it is complete, so the cache never depends on how its
tokens were split into calls.  At a head dimension of 128 a token takes 256
bytes per kv head instead of the 512 of an FP16 cache.

* :func:`kv8_append` writes tokens (prompts or single ones),
* :func:`kv8_attention` attends from a prompt's tokens, causally,
* :func:`kv8_decode` appends one token per sequence and attends, in one call,
  and can accumulate each position's attention weight,
* :func:`kv8_evict` keeps the positions with the largest accumulated weight,
* :func:`kv8_restore` gives the stored values back in FP16.

Lengths, positions and counts are int32 CUDA tensors with one entry per
sequence; the caller advances them, so a captured CUDA graph of a step can be
replayed.  Queries, keys and values are FP16 with contiguous rows; other
strides are free (views whose rows are not 16-byte aligned are copied first).
``cache.status`` is a device int that becomes 5 when a sequence would pass the
cache's capacity or its rotation tables; such a sequence is left unwritten and
its outputs are zero.

Lengths grow: the first token of a block takes the place of the block before it
in the tail, so after it no call may go back to a length up to that block's end.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

BLOCK = 64


class KV8Cache:
    """One layer's cache over the caller's tensors (nothing is copied).

    ``k_codes`` / ``v_codes`` uint8 ``[batch, kv_heads, capacity, head_dim]``,
    ``k_scales`` / ``v_scales`` float32 ``[batch, kv_heads, capacity / 64]``,
    ``k_tail`` / ``v_tail`` FP16 ``[batch, kv_heads, 64, head_dim]``; capacity
    a multiple of 64, head_dim 64 or 128.
    """

    def __init__(self, k_codes, v_codes, k_scales, v_scales, k_tail, v_tail, status: torch.Tensor | None = None):
        if k_codes.dim() != 4:
            raise ValueError("codes must be [batch, kv_heads, capacity, head_dim]")
        b, h, cap, hd = k_codes.shape
        want = ((k_codes, (b, h, cap, hd), torch.uint8), (v_codes, (b, h, cap, hd), torch.uint8),
                (k_scales, (b, h, cap // BLOCK), torch.float32), (v_scales, (b, h, cap // BLOCK), torch.float32),
                (k_tail, (b, h, BLOCK, hd), torch.float16), (v_tail, (b, h, BLOCK, hd), torch.float16))
        if cap % BLOCK or cap == 0 or hd not in (64, 128):
            raise ValueError(f"capacity must be a multiple of {BLOCK} and head_dim 64 or 128")
        for t, shape, dtype in want:
            if tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous():
                raise ValueError(f"cache tensors must be contiguous; expected {shape} {dtype}, "
                                 f"got {tuple(t.shape)} {t.dtype}")
        self.device = _lib.require_cuda(*(t for t, _, _ in want), status)
        if status is not None and (status.dtype is not torch.int32 or status.numel() < 1):
            raise ValueError("status must be an int32 tensor")
        self.k_codes, self.v_codes, self.k_scales, self.v_scales = k_codes, v_codes, k_scales, v_scales
        self.k_tail, self.v_tail = k_tail, v_tail
        self.batch, self.kv_heads, self.capacity, self.head_dim = b, h, cap, hd
        self.status = status if status is not None else torch.zeros(1, dtype=torch.int32, device=self.device)
        pair = ctypes.c_void_p * 2
        self.desc = _lib.Kv8CacheDesc(pair(k_codes.data_ptr(), v_codes.data_ptr()),
                                      pair(k_scales.data_ptr(), v_scales.data_ptr()),
                                      pair(k_tail.data_ptr(), v_tail.data_ptr()), b, h, cap, hd)
        self.ref = ctypes.byref(self.desc)
        self.index = self.device.index
        self.status_ptr = self.status.data_ptr()
        self._ws: dict = {}

    @classmethod
    def empty(cls, batch: int, kv_heads: int, capacity: int, head_dim: int, device,
              status: torch.Tensor | None = None) -> "KV8Cache":
        """A cache for ``capacity`` positions (rounded up to whole blocks)."""
        cap = -(-max(capacity, 1) // BLOCK) * BLOCK
        new = lambda *s, t: torch.zeros(*s, dtype=t, device=device)
        codes = [new(batch, kv_heads, cap, head_dim, t=torch.uint8) for _ in "kv"]
        scales = [new(batch, kv_heads, cap // BLOCK, t=torch.float32) for _ in "kv"]
        tails = [new(batch, kv_heads, BLOCK, head_dim, t=torch.float16) for _ in "kv"]
        return cls(*codes, *scales, *tails, status=status)

    def new_weights(self) -> torch.Tensor:
        """Zeroed attention weights for :func:`kv8_decode` to accumulate (what the queries of
        :func:`kv8_attention` look at is not added)."""
        return torch.zeros(self.batch, self.kv_heads, self.capacity, dtype=torch.float32, device=self.device)

    def new_workspace(self, n: int, q_heads: int, weights: bool = False) -> torch.Tensor:
        """Scratch for attention calls of ``n`` query tokens and ``q_heads`` heads on this cache's
        shape (other sizes may need more, and refuse it then)."""
        return torch.zeros(self.workspace_bytes(n, q_heads, weights), dtype=torch.uint8, device=self.device)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k_codes, self.v_codes, self.k_scales, self.v_scales,
                                                          self.k_tail, self.v_tail))

    def workspace_bytes(self, n: int, q_heads: int, weights: bool) -> int:
        key = (n, q_heads, weights)
        nb = self._ws.get(key)
        if nb is None:
            size = _lib._size_t()
            _lib.check(_lib.load().pp_kv8_attention_workspace_bytes(self.ref, n, q_heads, int(weights),
                                                                    ctypes.byref(size)))
            nb = self._ws[key] = size.value
        return nb


_strides: dict = {}
_scratch: dict = {}
_scratch_kept: list = []


def _workspace(cache: KV8Cache, n: int, q_heads: int, weights: bool, given) -> tuple:
    """Zero-filled scratch (address, bytes, tensor) of the attention calls; the
    kernels leave its counters at zero.  Without a given one there is one per
    (device, stream), and an outgrown buffer is kept, since launched work may
    still use it.  A call in a capture gets its own, whose fill is part of the
    graph: the graph may be replayed on any stream."""
    nbytes = cache.workspace_bytes(n, q_heads, weights)
    if given is not None:
        if (given.dtype is not torch.uint8 or given.get_device() != cache.index or not given.is_contiguous()
                or given.data_ptr() & 255 or given.numel() < nbytes):
            raise ValueError(f"workspace must be a contiguous 256-byte aligned uint8 tensor of at least {nbytes} "
                             f"bytes on {cache.device}")
        return given.data_ptr(), given.numel(), given
    if torch.cuda.is_current_stream_capturing():
        new = torch.empty(nbytes, dtype=torch.uint8, device=cache.device)
        new[:4096].zero_()  # the counters
        return new.data_ptr(), nbytes, new
    key = (cache.index, _lib.stream_handle(cache.device))
    buf = _scratch.get(key)
    if buf is None or buf[1] < nbytes:
        new = torch.zeros(max(nbytes, 1 << 20) * 5 // 4, dtype=torch.uint8, device=cache.device)
        if buf is not None:
            _scratch_kept.append(buf)
        buf = _scratch[key] = (new.data_ptr(), new.numel(), new)
    return buf


def _c_strides(*s: int):
    """Row strides of a checked tensor for the C call.  Only a dimension of one
    can have a stride there that is no multiple of 8 (_rows, _output): it
    addresses nothing."""
    a = _strides.get(s)
    if a is None:
        if len(_strides) >= 1024:
            _strides.clear()
        a = _strides[s] = (ctypes.c_int64 * len(s))(*(0 if x & 7 else x for x in s))
    return a


def _odd_rows(t: torch.Tensor) -> bool:
    """Rows that the kernels cannot read: strided, or not 16-byte aligned."""
    st = t.stride()
    return st[-1] != 1 or t.data_ptr() & 15 != 0 or any(s & 7 and n > 1 for s, n in zip(st[:-1], t.shape))


def _rows(t: torch.Tensor, name: str, shape: tuple, cache: KV8Cache) -> torch.Tensor:
    """FP16 rows as the kernels read them: contiguous and 16-byte aligned."""
    if t.dtype is not torch.float16 or t.shape != shape or t.get_device() != cache.index:
        raise ValueError(f"{name} must be FP16 {list(shape)} on {cache.device}, "
                         f"got {t.dtype} {list(t.shape)} on {t.device}")
    if (t.data_ptr() & 15 or not t.is_contiguous()) and _odd_rows(t):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _ints(t, name: str, cache: KV8Cache):
    if t is None:
        return None
    if t.dtype is not torch.int32 or t.get_device() != cache.index or t.shape != (cache.batch,) or \
            not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor [{cache.batch}] on {cache.device}")
    return t.data_ptr()


def _rope(rope, cache: KV8Cache):
    """``(cos, sin, pos)`` -> the four C arguments (all empty without rotation)."""
    if rope is None:
        return None, None, None, 0
    cos, sin, pos = rope
    for t in (cos, sin):
        if (t.dtype != torch.float16 or t.device != cache.device or t.dim() != 2 or t.shape[1] != cache.head_dim
                or t.shape != cos.shape or not t.is_contiguous()):
            raise ValueError(f"rotation tables must be contiguous FP16 [positions, {cache.head_dim}]")
    return cos.data_ptr(), sin.data_ptr(), _ints(pos, "rotation positions", cache), cos.shape[0]


def _weights(w, name: str, cache: KV8Cache):
    if w is None:
        return None
    if (w.dtype is not torch.float32 or w.get_device() != cache.index or not w.is_contiguous()
            or w.shape != (cache.batch, cache.kv_heads, cache.capacity)):
        raise ValueError(f"{name} must be contiguous float32 [{cache.batch}, {cache.kv_heads}, {cache.capacity}] "
                         f"on {cache.device}")
    return w.data_ptr()


def _output(out, q, cache: KV8Cache):
    """The output for queries q: given, or new (with q's layout if that is whole)."""
    if out is None:
        if q.is_contiguous():
            return torch.empty_like(q)
        return torch.empty(q.shape, dtype=torch.float16, device=cache.device)
    if (out.dtype is not torch.float16 or out.get_device() != cache.index or out.shape != q.shape
            or _odd_rows(out)):
        raise ValueError(f"out must be FP16 {list(q.shape)} on {cache.device} with 16-byte aligned contiguous rows")
    return out


def _call(cache: KV8Cache, fn: str, *args) -> None:
    """The C call on the current stream of the cache's device."""
    f = getattr(_lib.load(), fn)
    if torch.cuda.current_device() != cache.index:
        with torch.cuda.device(cache.device):
            rc = f(cache.ref, *args, cache.status_ptr, _lib.stream_handle(cache.device))
    else:
        rc = f(cache.ref, *args, cache.status_ptr, _lib.stream_handle(cache.device))
    if rc:
        _lib.check(rc)


def kv8_append(cache: KV8Cache, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor,
               counts: torch.Tensor | None = None, rope=None) -> None:
    """Append rows ``i < counts[b]`` (default: all) of ``k``, ``v``
    ``[batch, n, kv_heads, head_dim]`` at positions ``pos[b] + i``.

    ``pos[b]`` is the number of tokens sequence b holds; a negative one marks an
    unused sequence.  ``rope = (cos, sin, positions)`` rotates the keys.
    """
    shape = (cache.batch, k.shape[1] if k.dim() == 4 else 0, cache.kv_heads, cache.head_dim)
    k, v = _rows(k, "k", shape, cache), _rows(v, "v", shape, cache)
    _call(cache, "pp_kv8_append", k.data_ptr(), _c_strides(*k.stride()[:3]), v.data_ptr(),
          _c_strides(*v.stride()[:3]), shape[1], _ints(pos, "pos", cache), _ints(counts, "counts", cache),
          *_rope(rope, cache))


def kv8_restore(cache: KV8Cache, lens: torch.Tensor, start: torch.Tensor | None = None,
                count: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Stored keys and values ``[batch, count, kv_heads, head_dim]`` (FP16) of
    positions ``start[b] + i`` (default: the whole capacity from 0), zeros
    outside the sequence's ``lens[b]`` tokens."""
    n = cache.capacity if count is None else int(count)
    if n < 0:
        raise ValueError("count must not be negative")
    k = torch.empty(cache.batch, n, cache.kv_heads, cache.head_dim, dtype=torch.float16, device=cache.device)
    v = torch.empty_like(k)
    _call(cache, "pp_kv8_restore", _ints(lens, "lens", cache), _ints(start, "start", cache), n, k.data_ptr(),
          v.data_ptr())
    return k, v


def kv8_attention(q: torch.Tensor, cache: KV8Cache, lens: torch.Tensor, counts: torch.Tensor | None = None,
                  scale: float | None = None, rope=None, out: torch.Tensor | None = None,
                  workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of the last ``counts[b]`` (default: n) of each sequence's
    ``lens[b]`` tokens: ``q`` ``[batch, n, q_heads, head_dim]`` -> the same shape.

    Rows ``i >= counts[b]`` and rows that attend nothing are zero.  ``scale``
    defaults to ``1 / sqrt(head_dim)``; ``rope = (cos, sin, positions)``
    rotates the queries.  ``q_heads`` is a multiple of ``kv_heads``, at most 16
    to each.  ``workspace`` (:meth:`KV8Cache.new_workspace`) may be given for
    calls that run in order; otherwise one is kept per stream.
    """
    if q.dim() != 4:
        raise ValueError("q must be [batch, tokens, q_heads, head_dim]")
    n, nq = q.shape[1], q.shape[2]
    shape = (cache.batch, n, nq, cache.head_dim)
    q = _rows(q, "q", shape, cache)
    out = _output(out, q, cache)
    ws = _workspace(cache, n, nq, False, workspace)
    _call(cache, "pp_kv8_attention", q.data_ptr(), _c_strides(*q.stride()[:3]), n, nq, _ints(lens, "lens", cache),
          _ints(counts, "counts", cache), 1 / math.sqrt(cache.head_dim) if scale is None else scale, out.data_ptr(),
          _c_strides(*out.stride()[:3]), *_rope(rope, cache), ws[0], ws[1])
    return out


def kv8_decode(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: KV8Cache, pos: torch.Tensor,
               weights: torch.Tensor | None = None, scale: float | None = None, rope=None,
               out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """One token per sequence: append ``k``, ``v`` ``[batch, kv_heads, head_dim]``
    at ``pos[b]`` and attend with ``q`` ``[batch, q_heads, head_dim]`` to positions
    ``0 .. pos[b]``.

    ``weights`` (:meth:`KV8Cache.new_weights`), if given, has each position's
    softmax weights added, summed over the query heads of the kv head.  A
    negative position marks an unused sequence (zero output).  ``rope`` rotates
    queries and keys; ``workspace`` as in :func:`kv8_attention`.
    """
    if q.dim() != 3:
        raise ValueError("q must be [batch, q_heads, head_dim]")
    b, nq, hd = cache.batch, q.shape[1], cache.head_dim
    q = _rows(q, "q", (b, nq, hd), cache)
    k, v = _rows(k, "k", (b, cache.kv_heads, hd), cache), _rows(v, "v", (b, cache.kv_heads, hd), cache)
    out = _output(out, q, cache)
    ws = _workspace(cache, 1, nq, weights is not None, workspace)
    _call(cache, "pp_kv8_decode", q.data_ptr(), _c_strides(*q.stride()[:2]), nq, k.data_ptr(),
          _c_strides(*k.stride()[:2]), v.data_ptr(), _c_strides(*v.stride()[:2]), _ints(pos, "pos", cache),
          1 / math.sqrt(hd) if scale is None else scale, _weights(weights, "weights", cache), out.data_ptr(),
          _c_strides(*out.stride()[:2]), *_rope(rope, cache), ws[0], ws[1])
    return out


def kv8_evict(cache: KV8Cache, into: KV8Cache, lens: torch.Tensor, weights: torch.Tensor, keep: int, sinks: int = 4,
              recent: int = 64, into_weights: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Move at most ``keep`` tokens of every sequence and kv head into another
    cache: the first ``sinks``, the last ``recent`` and those with the largest
    accumulated ``weights`` (equal ones by the lower position), in order.

    ``into_weights`` receives the kept tokens' weights (zero past them).
    Returns ``(new_lens, kept)``: the new lengths and the old positions
    ``[batch, kv_heads, keep]`` (-1 past the new length), int32.
    """
    if (into.batch, into.kv_heads, into.head_dim) != (cache.batch, cache.kv_heads, cache.head_dim) or \
            into.device != cache.device:
        raise ValueError("the caches differ in sequences, kv heads, head_dim or device")
    if into_weights is None:
        into_weights = into.new_weights()
    dev = cache.device
    new_lens = torch.empty(cache.batch, dtype=torch.int32, device=dev)
    kept = torch.empty(cache.batch, cache.kv_heads, max(int(keep), 0), dtype=torch.int32, device=dev)
    w = _weights(weights, "weights", cache)
    if w is None:
        raise ValueError("weights are required")
    _call(cache, "pp_kv8_evict", into.ref, _ints(lens, "lens", cache), w,
          _weights(into_weights, "into_weights", into), new_lens.data_ptr(), kept.data_ptr(), int(keep), int(sinks),
          int(recent))
    return new_lens, kept
