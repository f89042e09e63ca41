"""Rotary position embedding, dense or on the way into the paged cache.

The reference's model code rotates queries and keys (engine/model.py:174-181)
before it writes the keys (184-187) and attends. Here:

* ``rotary_embed``  -- a chunk's queries and keys, dense (before
  ``prefill_attention``, or for a caller that writes by itself);
* ``rotary_append`` -- ``PagedKVCache.write_block_device`` of a chunk whose keys
  are rotated on the way, the queries in the same launch.

Queries, keys and values may be views of one fused projection's output: any
strides, as long as the elements of a head row are contiguous.

``Rotary`` holds the frequencies. Angles are formed in 64 bits on the device, so
there is no table and no largest position. Positions are given apart from the
pool's: they differ where a sequence continues a shared prefix (pool position
plus the prefix's length) and for the tokens of an image, which have one
position per axis (time, height, width).
"""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _hip
from ._hip import call, ptr
from .kv import PagedKVCache, WritePlan

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_Strides = ctypes.c_int64 * 12


class Rotary:
    """The rotary frequencies of a model's heads, on the device.

    Frequency ``i < rotary_dim / 2`` is ``base ** (-2 i / rotary_dim)``, or
    ``inv_freq[i]`` (scaled variants). It turns the elements ``(i, i +
    rotary_dim / 2)`` of a head row, or ``(2 i, 2 i + 1)`` with
    ``interleaved``; ``rotary_dim`` (default: the whole row) leaves the rest of
    the row as it is. ``factor`` scales the rotated elements. With several
    position axes, ``sections`` gives the number of consecutive frequencies of
    each, or ``axis_of`` the axis of every frequency. The caller keeps this object as
    long as a captured graph that used it may replay.
    """

    def __init__(self, head_dim: int, device: torch.device, base: float = 10000.0,
                 rotary_dim: Optional[int] = None, interleaved: bool = False,
                 inv_freq: Optional[Sequence[float]] = None, sections: Optional[Sequence[int]] = None,
                 axis_of: Optional[Sequence[int]] = None, factor: float = 1.0) -> None:
        self.head_dim = int(head_dim)
        self.rotary_dim = self.head_dim if rotary_dim is None else int(rotary_dim)
        if self.head_dim < 1 or not 0 <= self.rotary_dim <= self.head_dim or self.rotary_dim % 2:
            raise ValueError("rotary_dim must be even and within the head")
        n = self.rotary_dim // 2
        if inv_freq is None:
            if not base > 0:
                raise ValueError("base must be > 0")
            inv_freq = [float(base) ** (-2.0 * i / self.rotary_dim) for i in range(n)]
        inv_freq = [float(x) for x in inv_freq]
        if len(inv_freq) != n:
            raise ValueError("inv_freq must have rotary_dim / 2 = {} entries".format(n))
        if sections is not None:
            if axis_of is not None:
                raise ValueError("give sections or axis_of, not both")
            axis_of = [a for a, w in enumerate(sections) for _ in range(int(w))]
            self.axes = len(sections)
        else:
            axis_of = [0] * n if axis_of is None else [int(a) for a in axis_of]
            self.axes = max(axis_of, default=0) + 1
        if len(axis_of) != n or any(a < 0 for a in axis_of):
            raise ValueError("every one of the rotary_dim / 2 = {} frequencies needs its axis".format(n))
        self.device = _hip.require_gpu(device)
        self.interleaved = int(bool(interleaved))
        self.factor = float(factor)
        self.inv_freq = torch.tensor(inv_freq, dtype=torch.float64, device=self.device)
        self.axis_of = torch.tensor(axis_of, dtype=torch.int32, device=self.device)
        # argument shapes, strides and types that passed the checks, with the launch's
        # share of them: a serving loop repeats a few, and the checks cost as much
        # host time as the launch
        self._passed: dict = {}
        self._made_on = _hip.stream_of(self.device)

    @property
    def inv_freq(self) -> torch.Tensor:
        """The frequencies, ``rotary_dim / 2`` float64 on the device; may be replaced by others."""
        return self._inv_freq

    @inv_freq.setter
    def inv_freq(self, t: torch.Tensor) -> None:
        self._inv_freq = self._readable(t, torch.float64)

    @property
    def axis_of(self) -> torch.Tensor:
        """The position axis of every frequency, int32 on the device; may be replaced by others."""
        return self._axis_of

    @axis_of.setter
    def axis_of(self, t: torch.Tensor) -> None:
        self._axis_of = self._readable(t, torch.int32)

    def _readable(self, t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
        n = self.rotary_dim // 2
        if not isinstance(t, torch.Tensor) or t.dtype is not dtype or tuple(t.shape) != (n,) or \
                t.device != self.device or not t.is_contiguous():
            raise ValueError("the kernels read {} contiguous {} on {}".format(n, dtype, self.device))
        self._made_on = None  # a caller's tensor may be of any stream
        return t

    def _stream(self) -> int:
        """The current stream, for a launch that reads the frequencies."""
        return _hip.kept_for(_hip.stream_of(self.device), self._made_on, self._inv_freq, self._axis_of)

    def _args(self) -> tuple:
        """The launch arguments of the frequencies, asked anew in every call: a copy of this
        object has tensors of its own, and a caller may replace them."""
        return self._inv_freq.data_ptr(), self._axis_of.data_ptr(), self.axes, self.factor

    def _positions(self, positions: torch.Tensor, B: int, C: int) -> torch.Tensor:
        """int32 ``(axes, B, C)``; ``(B, C)`` stands for every axis."""
        if not isinstance(positions, torch.Tensor) or positions.is_floating_point() or positions.is_complex():
            raise ValueError("positions must be an integer tensor")
        if positions.device != self.device:
            raise ValueError("positions must live on {}".format(self.device))
        if positions.dtype is torch.int32 and positions.shape == (self.axes, B, C) and positions.is_contiguous():
            return positions
        if positions.dim() == 2 and self.axes > 1:
            positions = positions.expand(self.axes, -1, -1)
        want = (B, C) if positions.dim() == 2 else (self.axes, B, C)
        if tuple(positions.shape) != want:
            raise ValueError("positions must be ({}, {}) or ({}, {}, {})".format(B, C, self.axes, B, C))
        return positions.to(torch.int32).contiguous()


def _span(t: torch.Tensor) -> Tuple[int, int]:
    """First and one-past-last byte that a view with non-negative strides reaches."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two views share no memory: ranges apart, or the heads of one token
    row of a common buffer (equal batch and token strides, heads side by side)."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a1 <= b0 or b1 <= a0:
        return True
    if a0 > b0:
        a, b, a0, b0 = b, a, b0, a0
    row = [s for n, s in zip(a.shape[:2], a.stride()[:2]) if n > 1]
    if [s for n, s in zip(b.shape[:2], b.stride()[:2]) if n > 1] != row or a.dtype != b.dtype:
        return False
    extent = lambda t: ((t.shape[2] - 1) * t.stride(2) + t.shape[3]) * t.element_size()  # noqa: E731
    return a0 + extent(a) <= b0 and b0 - a0 + extent(b) <= min(row, default=0) * a.element_size()


def _one_place(t: torch.Tensor) -> bool:
    """Whether every element of a view has a place of its own."""
    reach = 1
    for s, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if s < reach:
            return False
        reach = s * (n - 1) + reach
    return True


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with contiguous head rows (a copy only where they are not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check_out(out: torch.Tensor, x: torch.Tensor, others: Sequence[torch.Tensor], dtype: torch.dtype) -> None:
    if tuple(out.shape) != tuple(x.shape) or out.dtype != dtype or out.device != x.device or \
            (out.stride(-1) != 1 and out.shape[-1] > 1):
        raise ValueError("an output must be like its input, with contiguous head rows")
    same = out.data_ptr() == x.data_ptr() and out.stride() == x.stride() and out.dtype == x.dtype
    if not _one_place(out) or not all(_apart(out, t) for t in ((*others,) if same else (x, *others))):
        raise ValueError("an output must be its own input or overlap no input, and have a place for every element")


def _strides(*tensors: Optional[torch.Tensor]) -> ctypes.Array:
    out = []
    for t in tensors:
        out.extend((0, 0, 0) if t is None else t.stride()[:3])
    return _Strides(*out)


def _remember(rotary: Rotary, key, value):
    if len(rotary._passed) >= 256:
        rotary._passed.clear()
    rotary._passed[key] = value
    return value


def _like(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)


def rotary_embed(query: torch.Tensor, key: Optional[torch.Tensor], rotary: Rotary, positions: torch.Tensor,
                 query_out: Optional[torch.Tensor] = None, key_out: Optional[torch.Tensor] = None,
                 key_dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(query, key)`` rotated, in one launch.

    ``query`` (B, C, Hq, d) and ``key`` (B, C, Hkv, d, or None) in float32,
    bfloat16 or float16; ``positions`` an integer device tensor (B, C), or
    (axes, B, C) for a ``Rotary`` of several axes. An output given by the caller
    is the input itself (in place) or overlaps no input. ``key_dtype``
    float32 keeps the rotated keys unrounded.
    """
    plain = query_out is None and key_out is None and key is not None
    sig = (query.shape, query.stride(), query.dtype, query.device, key.shape, key.stride(), key.dtype, key.device,
           key_dtype) if plain else None
    done = rotary._passed.get(sig) if plain else None
    if done is None:
        done = _check_embed(query, key, rotary, query_out, key_out, key_dtype)
        if plain and done[0]:
            _remember(rotary, sig, done)
    rows, B, C, hq, hkv, d, code, key_code, key_dtype, strides = done
    pos = rotary._positions(positions, B, C)
    if not rows:  # a copy where head rows are not contiguous
        query, key = _rows(query), None if key is None else _rows(key)
    if query_out is None:
        query_out = _like(query, query.dtype)
    if key is not None and key_out is None:
        key_out = _like(key, key_dtype)
    if B == 0 or C == 0:
        return query_out, key_out
    if strides is None:
        strides = _strides(query_out, query, key_out, key)
    call("spv_rotary", query_out.data_ptr(), query.data_ptr(), ptr(key_out), ptr(key), code, key_code, strides,
         pos.data_ptr(), *rotary._args(), B, C, hq, hkv, d, rotary.rotary_dim, rotary.interleaved,
         rotary._stream())
    return query_out, key_out


def _dense(shape) -> Tuple[int, int, int]:
    return shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3]


def _check_embed(query, key, rotary, query_out, key_out, key_dtype):
    if query.dim() != 4 or query.dtype not in _FLOATS:
        raise ValueError("query must be (B, C, heads, d) in float32, bfloat16 or float16")
    B, C, hq, d = (int(n) for n in query.shape)
    if d != rotary.head_dim:
        raise ValueError("the rows have {} elements, the rotary frequencies are for {}".format(d, rotary.head_dim))
    if key is not None and (key.dim() != 4 or tuple(key.shape[:2]) != (B, C) or key.shape[3] != d
                            or key.dtype != query.dtype):
        raise ValueError("key must be ({}, {}, heads, {}) in the query's dtype".format(B, C, d))
    for t in (query, key):
        if t is not None and t.device != rotary.device:
            raise ValueError("query and key must live on {}".format(rotary.device))
    if key_dtype is None:
        key_dtype = query.dtype
    if key_dtype not in (query.dtype, torch.float32):
        raise ValueError("key_dtype must be the query's dtype or float32")
    if query_out is not None:
        _check_out(query_out, query, () if key is None else (key,), query.dtype)
    if key_out is not None:
        if key is None:
            raise ValueError("key_out without a key")
        _check_out(key_out, key, (query,), key_dtype)
        if query_out is not None and not _apart(query_out, key_out):
            raise ValueError("the outputs overlap")
    rows = _rows(query) is query and (key is None or _rows(key) is key)
    strides = None
    if rows and query_out is None and key_out is None and key is not None:
        strides = _Strides(*_dense(query.shape), *query.stride()[:3], *_dense(key.shape), *key.stride()[:3])
    return (rows, B, C, hq, 0 if key is None else int(key.shape[2]), d, _hip.dtype_code(query.dtype),
            _hip.dtype_code(key_dtype), key_dtype, strides)


def rotary_append(query: Optional[torch.Tensor], k_new: torch.Tensor, v_new: torch.Tensor, kv: PagedKVCache,
                  layer: int, seq_ids: Union[Sequence[int], torch.Tensor],
                  start_positions: Union[Sequence[int], torch.Tensor], rotary: Rotary,
                  positions: Optional[torch.Tensor] = None, alloc: bool = True, plan: Optional[WritePlan] = None,
                  query_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Write a chunk's rotated keys and its values into the cache; returns the rotated queries.

    ``kv.write_block_device(layer, seq_ids, start_positions, rotated k_new,
    v_new, alloc, plan)`` with the same rules of allocation, exhaustion and
    write plans, and ``query`` (B, C, Hq, d, or None) rotated in the same launch.
    ``k_new`` / ``v_new`` (B, C, Hkv, d) and ``query`` share the pool's dtype
    (an fp8 pool: one of float32, bfloat16, float16; the rotated keys are
    quantised unrounded). fp8 pools, and pools of 2^31 token rows or more, are
    written in a launch behind the rotation's and ignore ``plan``.
    ``positions``: as in ``rotary_embed``; None takes the pool positions
    ``start_positions[b] + j``. No host synchronisation with device tensors of
    distinct, added ``seq_ids``. A later layer's call of a round passes
    ``alloc=False`` and the first one's ``plan``.
    """
    plain = query is not None and query_out is None
    sig = (kv._dt, kv.num_kv_heads, kv.head_dim, kv.device, query.shape, query.stride(), query.dtype, query.device,
           k_new.shape, k_new.stride(), k_new.dtype, k_new.device, v_new.shape, v_new.stride(), v_new.dtype,
           v_new.device) if plain else None
    done = rotary._passed.get(sig) if plain else None
    if done is None:
        done = _check_append(query, k_new, v_new, kv, rotary, query_out)
        if plain and done[0]:
            _remember(rotary, sig, done)
    rows_ok, B, C, hq, strides = done
    layer = int(layer)
    if not 0 <= layer < kv.num_layers:
        raise IndexError("layer {} out of range".format(layer))
    if positions is not None:
        pos = rotary._positions(positions, B, C)
    elif rotary.axes > 1:
        raise ValueError("a Rotary of several axes needs positions")
    else:
        pos = None
    if _hip.ids_ready(seq_ids, B, kv.device) and _hip.ids_ready(start_positions, B, kv.device):
        sid_t, start_t = seq_ids, start_positions
    else:
        sid_t, start_t = _append_ids(kv, seq_ids, start_positions, B, C)
    q, k, v = query, k_new, v_new
    if not rows_ok:
        q, k, v = None if q is None else _rows(q), _rows(k), _rows(v)
    if q is not None and query_out is None:
        query_out = _like(q, q.dtype)
    if B == 0 or C == 0:
        return query_out
    a = kv.allocator
    if kv.fp8 or a.capacity * kv.block_size >= 2 ** 31:
        if pos is None:
            pos = start_t.view(B, 1) + torch.arange(C, dtype=torch.int32, device=kv.device)
        _append_apart(q, k, v, kv, layer, sid_t, start_t, rotary, pos, alloc, query_out)
        return query_out
    rows, follow = None, 0
    if plan is not None:
        if alloc:
            plan._reserve(B, C, kv.device)
            rows = plan.rows
        elif plan.ready:
            plan._check(a.epoch, B, C, sid_t, start_t)
            rows, follow = plan.rows, 1
    call("spv_kv_rotary_append", ptr(query_out), ptr(q), k.data_ptr(), v.data_ptr(), kv._dt,
         _strides(query_out, q, k, v) if strides is None else strides, *kv._addresses(), sid_t.data_ptr(),
         start_t.data_ptr(), ptr(pos), *rotary._args(), B, C, hq, kv.num_kv_heads, kv.head_dim, rotary.rotary_dim,
         rotary.interleaved, layer, a.capacity, kv.block_size, bool(alloc), follow, ptr(rows),
         rotary._stream())
    if not follow:
        if rows is not None:
            plan._record(a.epoch, sid_t, start_t)
        kv._stale = True
        a._stale = True
    return query_out


def _check_append(query, k_new, v_new, kv, rotary, query_out):
    if k_new.dim() != 4:
        raise ValueError("k/v must have shape (B, chunk, {}, {})".format(kv.num_kv_heads, kv.head_dim))
    B, C = int(k_new.shape[0]), int(k_new.shape[1])
    d = kv.head_dim
    shape = (B, C, kv.num_kv_heads, d)
    if tuple(k_new.shape) != shape or tuple(v_new.shape) != shape:
        raise ValueError("k/v must have shape {}".format(shape))
    if rotary.head_dim != d or rotary.device != kv.device:
        raise ValueError("the rotary frequencies are for heads of {} on {}".format(rotary.head_dim, rotary.device))
    dtype = k_new.dtype if kv.fp8 else kv.dtype
    if dtype not in _FLOATS:
        raise ValueError("keys must be float32, bfloat16 or float16")
    tensors = (k_new, v_new) if query is None else (k_new, v_new, query)
    for t in tensors:
        if t.dtype != dtype:
            raise ValueError("query, keys and values must be {}".format(dtype))
        if t.device != kv.device:
            raise ValueError("query, keys and values must live on {}".format(kv.device))
    if query is not None and (query.dim() != 4 or tuple(query.shape[:2]) != (B, C) or query.shape[3] != d):
        raise ValueError("query must be ({}, {}, heads, {})".format(B, C, d))
    if query_out is not None:
        if query is None:
            raise ValueError("query_out without a query")
        _check_out(query_out, query, (k_new, v_new), dtype)
    rows = all(_rows(t) is t for t in tensors)
    strides = None
    if rows and query is not None and query_out is None:
        strides = _Strides(*_dense(query.shape), *query.stride()[:3], *k_new.stride()[:3], *v_new.stride()[:3])
    return rows, B, C, 0 if query is None else int(query.shape[2]), strides


def _append_ids(kv, seq_ids, start_positions, B, C):
    """Sequence ids and start positions on the device; lists are checked as in ``write_block``."""
    given = [not isinstance(t, torch.Tensor) for t in (seq_ids, start_positions)]
    if any(given):
        kv._refresh()
        if given[0]:
            seq_ids = [kv._check_sid(s) for s in seq_ids]
            if len(set(seq_ids)) != len(seq_ids):
                raise ValueError("a batched write needs distinct sequence ids")
        if given[1]:
            start_positions = [int(s) for s in start_positions]
            if any(s < 0 for s in start_positions):
                raise ValueError("start positions must be >= 0")
            if start_positions:
                kv._grow_width(-(-(max(start_positions) + C) // kv.block_size))
    sid_t, start_t = _hip.i32s(kv.device, seq_ids, start_positions)
    if sid_t.numel() != B or start_t.numel() != B:
        raise ValueError("one seq_id and start position per batch row")
    return sid_t, start_t


def _append_apart(q, k, v, kv, layer, sid_t, start_t, rotary, pos, alloc, query_out) -> None:
    """The rotated keys by themselves, then the append of both: an fp8 pool's, which quantises
    (from float32, so that a key is rounded once), and that of a pool of 2^31 token rows or
    more (the one launch counts rows in 32 bits)."""
    dtype = torch.float32 if kv.fp8 else k.dtype
    turned = torch.empty(k.shape, dtype=dtype, device=k.device)
    call("spv_rotary", ptr(query_out), ptr(q), ptr(turned), ptr(k), _hip.dtype_code(k.dtype), _hip.dtype_code(dtype),
         _strides(query_out, q, turned, k), ptr(pos), *rotary._args(), k.shape[0], k.shape[1],
         0 if q is None else int(q.shape[2]), kv.num_kv_heads, kv.head_dim, rotary.rotary_dim,
         rotary.interleaved, rotary._stream())
    kv.write_block_device(layer, sid_t, start_t, turned, v.to(dtype), alloc=alloc)
