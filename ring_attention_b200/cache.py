"""Decoding: a key/value cache held in 4 bits, attention that reads it, eviction by attention weight.

The host side of the `ra_cache4_*` calls (include/ring_attention_b200.h has the formulas).  A program
prefills with `ring_self_attention`, appends the keys and values, and answers token by token:

    cache = KVCache4(batch, kv_heads, capacity, head_dim)
    cache.append(k, v)                                        # [b, t, kv_heads, d]
    out = cache_attention(q, cache, weights_out=cache.weights)  # [b, lq, heads, d]
    cache.evict(keep, recent=256)

Lengths live on the device: no call here synchronises, and all of them can be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch

from . import _lib
from ._lib import RaCache4, RaScoreMod, RaTensor, check, lib
from .ring import ScoreMod, _blhd, _dtype_code, _i32, _need_cuda

_GROUP, _ALIGN = 64, 64


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _view(t: torch.Tensor):
    """[b, l, h, d] tensor -> reference to a ra_tensor_t."""
    sb, sl, sh, _ = t.stride()
    return C.byref(RaTensor(t.data_ptr(), sb, sl, sh))


class _On:
    """Makes `device` the current one inside the `with` block; yields its current stream."""

    def __init__(self, device: torch.device):
        # (torch.cuda.current_device and current_stream without their checks: a tensor of the device is at hand)
        self.guard = None if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)
        self.index = device.index

    def __enter__(self) -> int:
        if self.guard is not None:
            self.guard.__enter__()
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


class KVCache4:
    """Keys and values of `batch` sequences in 4 bits a channel, up to `capacity` rows (tokens) each.

    `capacity` is rounded up to a multiple of 64; `head_dim` is 64, 128 or 256.  A row is 16 levels for every
    64 channels between limits of its own (0.5 bytes a channel and 4 bytes a group).  On the device, for the
    caller to read: `lengths` [b] rows held, `seen` [b] position after the last one, `positions` and `weights`
    [b, kv_heads, capacity].  Rows may lie in any order (eviction fills gaps); each carries its position."""

    def __init__(self, batch: int, kv_heads: int, capacity: int, head_dim: int, device=None):
        if head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
        if min(batch, kv_heads, capacity) < 1:
            raise ValueError("batch, kv_heads and capacity must be at least 1")
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise _lib.RingAttentionError("ring_attention_b200 needs CUDA tensors (there is no CPU path)")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        capacity = (capacity + _ALIGN - 1) // _ALIGN * _ALIGN
        rows, d = (batch, kv_heads, capacity), head_dim
        self.batch, self.kv_heads, self.capacity, self.head_dim, self.device = batch, kv_heads, capacity, head_dim, device

        def new(shape, dtype):
            return torch.zeros(shape, dtype=dtype, device=device)

        self.k_codes, self.v_codes = new(rows + (d // 2,), torch.uint8), new(rows + (d // 2,), torch.uint8)
        self.k_limits = new(rows + (d // _GROUP, 2), torch.bfloat16)
        self.v_limits = new(rows + (d // _GROUP, 2), torch.bfloat16)
        self.positions, self.weights = new(rows, torch.int32), new(rows, torch.float32)
        self.lengths, self.seen = new((batch,), torch.int32), new((batch,), torch.int32)
        self._struct = RaCache4(batch, kv_heads, capacity, d, *(t.data_ptr() for t in (
            self.k_codes, self.v_codes, self.k_limits, self.v_limits, self.positions, self.weights, self.lengths, self.seen)))
        self._ref = C.byref(self._struct)
        self._workspace = {}  # bytes of an attention call, by (heads, lq, type)

    def _here(self, what: str, t: torch.Tensor):
        if t.device != self.device:
            _need_cuda(t)
            raise _lib.RingAttentionError(f"{what} is on {t.device}, the cache on {self.device}")

    def _per_sequence(self, what: str, t: Optional[torch.Tensor], shape) -> Optional[torch.Tensor]:
        if t is None:
            return None
        self._here(what, t)
        if t.shape != shape:
            raise ValueError(f"{what} has shape {tuple(t.shape)}, expected {shape}")
        if t.dtype == torch.int32:
            return t if t.is_contiguous() else t.contiguous()
        if t.dtype != torch.int64:
            raise TypeError(f"{what} must be int32 or int64, got {t.dtype}")
        return _i32(t)

    def reset(self) -> None:
        """Empties the cache."""
        self.lengths.zero_()
        self.seen.zero_()

    def append(self, k: torch.Tensor, v: torch.Tensor, counts: Optional[torch.Tensor] = None,
               start: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None) -> None:
        """Adds the rows k, v [b, t, kv_heads, d] (float32 or bfloat16).

        `counts` [b]: only the first counts[i] rows of sequence i (a padded batch).  `start` [b]: from slot
        start[i] on instead of behind the last row, dropping what lies behind the new rows (rejected drafts).
        `positions` [b, t]: default is to go on where the sequence stands, with `start` at the position of the first
        row dropped, or behind the row before it where that is later (branches of drafts repeat positions).  Rows beyond the capacity are
        dropped and set bit 17 of `device_status()`.  There is no backward pass: the cache holds rounded copies."""
        shape = (self.batch, k.shape[1] if k.dim() == 4 else -1, self.kv_heads, self.head_dim)
        if k.shape != shape or v.shape != shape:
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be [{self.batch}, t, {self.kv_heads}, {self.head_dim}]")
        if k.dtype != v.dtype:
            raise TypeError(f"k and v must have one type, got {k.dtype} and {v.dtype}")
        self._here("k", k)
        self._here("v", v)
        t = shape[1]
        if t > self.capacity:
            raise ValueError(f"{t} rows do not fit a capacity of {self.capacity}")
        if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad):
            raise _lib.RingAttentionError("KVCache4.append has no backward pass: call it under torch.no_grad() or detach k and v")
        counts = self._per_sequence("counts", counts, (self.batch,))
        start = self._per_sequence("start", start, (self.batch,))
        positions = self._per_sequence("positions", positions, (self.batch, t))
        dtype = _dtype_code(k)
        if t == 0:
            if start is None:
                return
            # nothing comes in the dropped rows' place: a row for each sequence of which none counts
            k = v = k.new_zeros((self.batch, 1, self.kv_heads, self.head_dim))
            t, positions, counts = 1, None, torch.zeros_like(start)
        k, v = _blhd(k), _blhd(v)
        with _On(self.device) as stream:
            check(lib.ra_cache4_append(self._ref, _view(k), _view(v), dtype, t, _ptr(counts),
                                       _ptr(start), _ptr(positions), stream))

    def read(self, count: int, start: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16):
        """The values (k, v) [b, count, kv_heads, d] of the slots start[i] (default 0) and on; zeros where there is no row."""
        if count < 1:
            raise ValueError(f"count must be at least 1, got {count}")
        start = self._per_sequence("start", start, (self.batch,))
        k = torch.empty((self.batch, count, self.kv_heads, self.head_dim), dtype=dtype, device=self.device)
        code = _dtype_code(k)
        v = torch.empty_like(k)
        with _On(self.device) as stream:
            check(lib.ra_cache4_read(self._ref, _view(k), _view(v), code, count, _ptr(start), stream))
        return k, v

    def evict(self, keep: int, recent: int = 0, out: Optional["KVCache4"] = None) -> "KVCache4":
        """Leaves each sequence and head at most `keep` rows: the last `recent` positions, then the largest
        accumulated `weights` (the lowest slot first among equals).  In place, or into another cache `out`
        (same batch, heads and head_dim, room for `keep` rows), which is returned."""
        if not 1 <= keep <= self.capacity:
            raise ValueError(f"keep must be between 1 and the capacity {self.capacity}, got {keep}")
        if not 0 <= recent <= keep:
            raise ValueError(f"recent must be between 0 and keep, got {recent}")
        to = self if out is None else out
        if (to.batch, to.kv_heads, to.head_dim) != (self.batch, self.kv_heads, self.head_dim) or to.capacity < keep:
            raise ValueError("out must have the cache's batch, kv_heads and head_dim and room for `keep` rows")
        self._here("out", to.lengths)
        with _On(self.device) as stream:
            nbytes = lib.ra_cache4_evict_workspace(self._ref, keep)
            check(min(nbytes, 0))
            ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            check(lib.ra_cache4_evict(self._ref, keep, recent, to._ref, _ptr(ws), nbytes, stream))
        return to


def cache_attention(
    q: torch.Tensor,
    cache: KVCache4,
    q_positions: Optional[torch.Tensor] = None,
    bias_fn: Optional[ScoreMod] = None,
    sm_scale: Optional[float] = None,
    return_lse: bool = False,
    weights_out: Optional[torch.Tensor] = None,
):
    """Attention of q [b, lq, heads, d] (float32 or bfloat16) over the rows of `cache`; the result has q's shape and type.

    `heads` is a multiple of the cache's kv_heads: head i reads key/value head i // (heads // kv_heads).
    `bias_fn`: None (every row is visible) or a `ScoreMod` (causal, window, ALiBi) over the rows' positions and
    `q_positions` [b, lq]; by default the queries are the last lq tokens given to the cache.  A query that sees
    no row gets NaN and a log-sum-exp of -inf.  `return_lse`: also L [b, heads, lq] in float32, with which parts
    of a cache held apart (the shards of a ring, say) can be joined: L = log sum exp(L_i), out = sum exp(L_i - L) out_i
    over the parts with L_i > -inf; the others' out_i is NaN and is left out (a weight of 0 would not hide it).
    `weights_out` float32 [b, kv_heads, capacity]: receives `cache.weights` plus the probabilities of every row summed
    over the queries and heads that read it; `cache.weights` itself accumulates in place.  The probabilities are those of
    this call, over this cache: for a part held apart they add up to 1 over the part, not over the whole.
    There is no backward pass: the cache holds rounded copies."""
    if not isinstance(cache, KVCache4):
        raise TypeError("cache_attention reads a KVCache4")
    if bias_fn is not None and not isinstance(bias_fn, ScoreMod):
        raise ValueError("cache_attention takes a ScoreMod bias_fn (or None)")
    cache._here("q", q)
    if q.dim() != 4 or q.shape[0] != cache.batch or q.shape[3] != cache.head_dim or q.shape[2] % cache.kv_heads or not q.shape[2]:
        raise ValueError(f"q {tuple(q.shape)} must be [{cache.batch}, lq, a multiple of {cache.kv_heads}, {cache.head_dim}]")
    if q.requires_grad and torch.is_grad_enabled():
        raise _lib.RingAttentionError("cache_attention has no backward pass: call it under torch.no_grad()")
    dtype = _dtype_code(q)
    b, lq, h, d = q.shape
    q_positions = cache._per_sequence("q_positions", q_positions, (b, lq))
    if weights_out is not None:
        cache._here("weights_out", weights_out)
        if weights_out.shape != cache.weights.shape or weights_out.dtype != torch.float32 or not weights_out.is_contiguous():
            raise ValueError(f"weights_out must be a contiguous float32 tensor of shape {tuple(cache.weights.shape)}")
    mod = slopes = None
    if bias_fn is not None:
        mod = RaScoreMod()
        mod.kinds = bias_fn.kinds({}, {}) & ~_lib.RA_MOD_STRICT_NAN  # that one is about gradients
        mod.window = bias_fn.window
        if q_positions is not None:
            mod.q_pos = q_positions.data_ptr()
        if bias_fn.alibi_slopes is not None:
            slopes = bias_fn.alibi_slopes.to(torch.float32).contiguous()
            cache._here("alibi_slopes", slopes)
            if slopes.numel() != h:
                raise ValueError(f"alibi_slopes has {slopes.numel()} entries for {h} heads")
            mod.alibi_slopes = slopes.data_ptr()
    q = _blhd(q)
    out = q.new_empty((b, lq, h, d))
    lse = q.new_empty((b, h, lq), dtype=torch.float32) if return_lse else None
    if lq:
        scale = 1 / math.sqrt(d) if sm_scale is None else float(sm_scale)
        with _On(cache.device) as stream:
            nbytes = cache._workspace.get((h, lq, dtype))
            if nbytes is None:
                nbytes = lib.ra_cache4_attention_workspace(cache._ref, h, lq, dtype)
                check(min(nbytes, 0))
                cache._workspace[h, lq, dtype] = nbytes
            ws = q.new_empty(nbytes, dtype=torch.uint8)
            check(lib.ra_cache4_attention(cache._ref, _view(q), _view(out), _ptr(lse), h, lq, dtype,
                                          scale, C.byref(mod) if mod is not None else None, _ptr(weights_out), _ptr(ws), nbytes,
                                          stream))
    elif weights_out is not None and weights_out.data_ptr() != cache.weights.data_ptr():
        # (no query, no probability; slots behind the last row are left as they are, as in any call)
        live = torch.arange(cache.capacity, device=cache.device) < cache.lengths[:, None, None]
        weights_out.copy_(torch.where(live, cache.weights, weights_out))
    return (out, lse) if return_lse else out
