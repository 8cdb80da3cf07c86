"""Context keys and values kept in eight bits, and attention that reads them so.

Next to the functional operators of ``triton_kernels``: those take the context as [H,Nc,Dh] tensors of the queries'
type; here it is written once into a ``ContextCache`` (half of a bf16 context's memory, a quarter of an fp32 one's),
grows in place, and is attended to as a whole or, on long contexts, in the blocks that matter to a query:

    cache = quantize_context(k_ctx, v_ctx, capacity=4096)      # [H,Nc,Dh] shared, or [G,H,Nc,Dh]: one context per stream
    append_context(cache, k_new, v_new)                        # more rows, in place
    out, lse = context_cache_attention(q, cache)               # q [B,H,Lq,Dh]: as triton_context_attention
    blocks = select_context_blocks(q, cache, 16)               # [B,H,Lq,16]
    out, lse = block_context_attention(q, cache, blocks)
    out = merge_attention_outputs(out, lse, *pytorch_buffer_attention(q, k_buf, v_buf))   # with private buffers

Rows are kept in blocks of ``CONTEXT_BLOCK`` with a scale per (group, head, block) for the keys and one for the
values: ``scale = largest magnitude / 127``, ``code = whole number nearest to x / scale`` (ties to even).  Rows that join
a block may raise its scale; the older ones are then rounded again.  A block that took in a value that is not finite
has NaN for its scale: what attends it becomes NaN.

Types: float32 or bfloat16 for queries, keys and values; head sizes 16, 32 and 64.  float32 queries get float32
accuracy (products with the codes are exact to 22 bits), bfloat16 ones the accuracy of their type.  No gradients.
Calls on one cache belong on one stream, or in an order that the caller sees to.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from .. import _lib

CONTEXT_BLOCK = 64
_MOST_ROWS = 1 << 30          # of a cache; also of a call
_MOST_LISTED = 1 << 30        # blocks of a query
_MOST_INT = (1 << 31) - 1
_Strides = C.c_int64 * 3
Lengths = Union[Tensor, Sequence[int]]


class ContextCache:
    """The tensors of an 8-bit context (``quantize_context`` makes one; these four may also be kept and put
    together again):

      codes   uint8 [G,H,blocks,2,64*Dh]: keys [64,Dh], then values transposed, [Dh,64] (their row order: ``VALUE_ROWS``);
              a code c stands for (c - 128) * scale
      scales  float32 [G,H,blocks,2]: of the keys, of the values
      bounds  float16 [G,H,blocks,2,Dh]: smallest and largest key code (less 128) of each channel over a block's rows
      lens    int32 [G]: rows in use.  Kernels read it on the device

    They are worked on in place, where they are now: another tensor put in a field's place is not seen.
    ``length``: a bound of ``lens`` known to the host (default: the capacity).  A captured ``append_context`` counts once
    in it, however often it is replayed; appending and reading outside a capture then look ``lens`` up.  Attention picks its
    kernel and how it splits the rows by ``length``: the same rows with another ``length`` may differ in the last bits."""

    __slots__ = ("codes", "scales", "bounds", "lens", "length", "n_groups", "n_heads", "head_dim", "capacity", "captured", "_c", "_ref")

    def __init__(self, codes: Tensor, scales: Tensor, bounds: Tensor, lens: Tensor, length: Optional[int] = None):
        shape = codes.shape
        if len(shape) != 5 or shape[3] != 2 or codes.dtype is not torch.uint8:
            raise ValueError("ContextCache: codes must be uint8 [G,H,blocks,2,64*Dh]")
        G, H, blocks, _, size = shape
        Dh = size // CONTEXT_BLOCK
        if Dh not in (16, 32, 64) or size % CONTEXT_BLOCK:
            raise ValueError(f"ContextCache: head size {size / CONTEXT_BLOCK:g} not supported (16, 32, 64)")
        if G < 1 or H < 1 or blocks < 1:
            raise ValueError(f"ContextCache: empty cache {tuple(shape)}")
        if scales.shape != (G, H, blocks, 2) or scales.dtype is not torch.float32:
            raise ValueError("ContextCache: scales must be float32 [G,H,blocks,2]")
        if bounds.shape != (G, H, blocks, 2, Dh) or bounds.dtype is not torch.float16:
            raise ValueError("ContextCache: bounds must be float16 [G,H,blocks,2,Dh]")
        if lens.shape != (G,) or lens.dtype is not torch.int32:
            raise ValueError("ContextCache: lens must be int32 [G]")
        if not (codes.is_contiguous() and scales.is_contiguous() and bounds.is_contiguous() and lens.is_contiguous()):
            raise ValueError("ContextCache: tensors must be contiguous")
        if not scales.get_device() == bounds.get_device() == lens.get_device() == codes.get_device():
            raise ValueError("ContextCache: all tensors must live on one device")
        if length is not None and length < 0:
            raise ValueError(f"ContextCache: a length of {length}")
        self._set(codes, scales, bounds, lens, blocks * CONTEXT_BLOCK if length is None else length)

    def _set(self, codes: Tensor, scales: Tensor, bounds: Tensor, lens: Tensor, length: int) -> "ContextCache":
        G, H, blocks, _, size = codes.shape
        Dh = size // CONTEXT_BLOCK
        self.codes, self.scales, self.bounds, self.lens = codes, scales, bounds, lens
        self.n_groups, self.n_heads, self.head_dim, self.capacity = G, H, Dh, blocks * CONTEXT_BLOCK
        self.length = min(int(length), self.capacity)
        self.captured = False      # a graph may have moved lens since `length` was set
        self._c = _lib.Cache(G, H, Dh, blocks, codes.data_ptr(), scales.data_ptr(), bounds.data_ptr(), lens.data_ptr())
        self._ref = C.byref(self._c)
        return self

    @property
    def device(self) -> torch.device:
        return self.codes.device


# row of a block at each place of a value channel
VALUE_ROWS = tuple(16 * s + 8 * h + 2 * t + e for t in range(4) for s in range(4) for h in range(2) for e in range(2))


class _Launch:
    """The library and the current stream of the device with number ``device``, which is the current device inside (a
    launch goes to the current one)."""

    __slots__ = ("device", "outer")

    def __init__(self, device: int):
        self.device = device

    def __enter__(self):
        lib = _lib.lib()
        if self.device < 0:
            raise ValueError("context cache: tensors must live on a CUDA device")
        self.outer = None
        if _current_device() != self.device:
            self.outer = torch.cuda.device(self.device)
            self.outer.__enter__()
        return lib, _raw_stream(self.device)

    def __exit__(self, *exc):
        if self.outer is not None:
            self.outer.__exit__(*exc)
        return False


def _current_device() -> int:
    return torch._C._cuda_getDevice()      # torch.cuda.current_device() without its check that CUDA is up


def _raw_stream(device: int) -> int:
    return torch._C._cuda_getCurrentRawStream(device)   # the address alone, no Stream object


def _strided(t: Tensor):
    """``t`` with neighbouring elements in its last axis, its address and its other strides (None: contiguous)."""
    if t.is_contiguous():
        return t, t.data_ptr(), None
    strides = t.stride()
    if strides[-1] != 1:
        t = t.contiguous()
        return t, t.data_ptr(), None
    return t, t.data_ptr(), _Strides(*strides[:3])


def _lengths(x: Optional[Lengths], G: int, device: torch.device, what: str) -> Optional[Tensor]:
    """Row counts as an int32 [G] tensor on ``device``."""
    if x is None:
        return None
    if not isinstance(x, Tensor):
        x = torch.tensor(list(x))
    if x.dtype.is_floating_point or x.dtype.is_complex or x.dtype in (torch.bool, torch.uint64):
        raise ValueError(f"{what} must be whole numbers")
    if x.shape != (G,):
        raise ValueError(f"{what} must have one entry per context: ({G},), not {tuple(x.shape)}")
    if x.dtype in (torch.int64, torch.uint32):
        x = x.to(torch.int64).clamp(-1, _MOST_INT)           # what does not fit 32 bits stays out of range
    if x.dtype is not torch.int32 or x.device != device or not x.is_contiguous():
        x = x.to(device=device, dtype=torch.int32).contiguous()
    return x


def _rows_of(k: Tensor, v: Tensor, what: str) -> Tuple[Tensor, Tensor, int]:
    """Keys and values as [G,H,N,Dh], and the code of their type."""
    if k.dim() == 3:
        k, v = k.unsqueeze(0), v.unsqueeze(0)
    if k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"{what}: keys {tuple(k.shape)} and values {tuple(v.shape)} must both be [H,N,Dh] or [G,H,N,Dh]")
    if k.shape[2] > _MOST_ROWS:
        raise ValueError(f"{what}: {k.shape[2]} rows at once")
    if v.dtype is not k.dtype:
        raise ValueError(f"{what}: keys are {k.dtype}, values {v.dtype}")
    code = _lib.dtype_code(k.dtype)
    if v.get_device() != k.get_device():
        raise ValueError(f"{what}: keys and values must live on one device")
    return k, v, code


def _write(lib, stream, cache: ContextCache, code: int, k: Tensor, v: Tensor, start, counts, fresh: int) -> None:
    k, k_at, k_strides = _strided(k)
    v, v_at, v_strides = _strided(v)
    _lib.check(lib.artab_cache_write(code, k_at, k_strides, v_at, v_strides, k.shape[2], _address(start), _address(counts),
                                     fresh, cache._ref, stream))


def _address(t: Optional[Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def quantize_context(k_ctx: Tensor, v_ctx: Tensor, lens: Optional[Lengths] = None,
                     capacity: Optional[int] = None) -> ContextCache:
    """A cache of the context rows k_ctx / v_ctx, [H,Nc,Dh] (shared by all streams) or [G,H,Nc,Dh] (one context per
    stream).  ``lens`` [G]: rows in use of each (default: all Nc; the others are not read).  ``capacity``: rows that
    there is room for (rounded up to whole blocks; default Nc)."""
    k, v, code = _rows_of(k_ctx, v_ctx, "quantize_context")
    G, H, N, Dh = k.shape
    if Dh not in (16, 32, 64):
        raise ValueError(f"quantize_context: head_dim {Dh} not supported (16, 32, 64)")
    capacity = N if capacity is None else int(capacity)
    if not max(N, 1) <= capacity <= _MOST_ROWS or G < 1 or H < 1:
        raise ValueError(f"quantize_context: no room for {N} rows of {G} x {H} heads in a capacity of {capacity}")
    counts = _lengths(lens, G, k.device, "lens")
    blocks = (capacity + CONTEXT_BLOCK - 1) // CONTEXT_BLOCK
    with _Launch(k.get_device()) as (lib, stream):
        new = k.new_zeros if N == 0 else k.new_empty      # without rows nothing is launched
        cache = ContextCache.__new__(ContextCache)._set(
            k.new_empty((G, H, blocks, 2, CONTEXT_BLOCK * Dh), dtype=torch.uint8), new((G, H, blocks, 2), dtype=torch.float32),
            new((G, H, blocks, 2, Dh), dtype=torch.float16), new((G,), dtype=torch.int32), N)
        if N:
            _write(lib, stream, cache, code, k, v, None, counts, 1)
    return cache


def _look_up(cache: ContextCache) -> None:
    cache.length = min(max(int(cache.lens.max()), 0), cache.capacity)


def append_context(cache: ContextCache, k_new: Tensor, v_new: Tensor, counts: Optional[Lengths] = None,
                   start: Optional[Lengths] = None) -> None:
    """Put rows k_new / v_new [G,H,n,Dh] ([H,n,Dh] for a shared context) behind those in use, in place.

    ``counts`` [G]: how many of the n rows each context takes (default: all).  ``start`` [G]: where they begin
    (default: ``cache.lens``); what was at or behind it is dropped, which takes rows back that did not stand.  ``lens``
    becomes start + counts.  ``start`` is at most ``lens``, and rows beyond the capacity are left out; without
    ``start`` they raise before anything is written."""
    k, v, code = _rows_of(k_new, v_new, "append_context")
    G, H, n, Dh = k.shape
    if (G, H, Dh) != (cache.n_groups, cache.n_heads, cache.head_dim):
        raise ValueError(f"append_context: rows {tuple(k.shape)} do not fit a cache of {cache.n_groups} contexts, "
                         f"{cache.n_heads} heads of size {cache.head_dim}")
    if k.get_device() != cache.codes.get_device():
        raise ValueError("append_context: rows must live on the device of the cache")
    counts = _lengths(counts, G, k.device, "counts")
    start = _lengths(start, G, k.device, "start")
    if n == 0 and start is None:
        return
    with _Launch(k.get_device()) as (lib, stream):
        capturing = torch.cuda.is_current_stream_capturing()
        if cache.captured and not capturing:
            _look_up(cache)
        if start is None and cache.length + n > cache.capacity:
            # the bound that the host keeps may be too high: contexts that took fewer rows, a cache put together from tensors
            if capturing:
                raise ValueError("append_context: the cache may be full, and its lengths cannot be looked up during capture")
            room = cache.lens if counts is None else cache.lens + counts.clamp(0, n)
            _look_up(cache)
            if int(room.max()) + (n if counts is None else 0) > cache.capacity:
                raise ValueError("append_context: context cache exceeded; increase its capacity")
        if n == 0:
            k = v = cache.scales.new_empty(G, H, 1, Dh)      # nothing is read from it: start alone takes effect
            counts = torch.zeros(G, dtype=torch.int32, device=k.device)
        _write(lib, stream, cache, code, k, v, start, counts, 0)
        cache.length = min(cache.length + n, cache.capacity)
        cache.captured = cache.captured or capturing


def read_context(cache: ContextCache, start: Optional[Lengths] = None, n: Optional[int] = None,
                 dtype: torch.dtype = torch.float32) -> Tuple[Tensor, Tensor]:
    """The rows that the cache stands for: k, v [G,H,n,Dh], from row ``start`` [G] on (default 0; ``n``: default
    ``cache.length``).  Rows that are not in use are zero."""
    code = _lib.dtype_code(dtype)
    G, H, Dh = cache.n_groups, cache.n_heads, cache.head_dim
    if n is None:
        if cache.captured:
            with _Launch(cache.codes.get_device()):
                if not torch.cuda.is_current_stream_capturing():
                    _look_up(cache)
        n = cache.length
    n = int(n)
    if not 0 <= n <= _MOST_ROWS:
        raise ValueError(f"read_context: {n} rows")
    start = _lengths(start, G, cache.device, "start")
    k = cache.scales.new_empty((G, H, n, Dh), dtype=dtype)
    v = torch.empty_like(k)
    if n:
        with _Launch(k.get_device()) as (lib, stream):
            _lib.check(lib.artab_cache_read(code, cache._ref, _address(start), n, k.data_ptr(), v.data_ptr(), stream))
    return k, v


def _queries(q: Tensor, cache: ContextCache, what: str):
    """Sizes [B,H,Lq,Dh], type and device of queries that fit the cache."""
    shape = q.shape
    if len(shape) != 4 or shape[1] != cache.n_heads or shape[3] != cache.head_dim:
        raise ValueError(f"{what}: queries {tuple(shape)} do not fit a cache of {cache.n_heads} heads of size "
                         f"{cache.head_dim}")
    if cache.n_groups != 1 and cache.n_groups != shape[0]:
        raise ValueError(f"{what}: {cache.n_groups} contexts for {shape[0]} streams (one, or one each)")
    code, device = _lib.dtype_code(q.dtype), q.get_device()
    if device != cache.codes.get_device():
        raise ValueError(f"{what}: queries must live on the device of the cache")
    return shape, code, device


def context_cache_attention(q: Tensor, cache: ContextCache, scale: Optional[float] = None) -> Tuple[Tensor, Tensor]:
    """Attention of q [B,H,Lq,Dh] over every row in use of its context: out [B,H,Lq,Dh] (q dtype), lse [B,H,Lq] fp32
    (natural log), as ``triton_context_attention``.  A context without rows gives 0 and -inf."""
    (B, H, Lq, Dh), code, device = _queries(q, cache, "context_cache_attention")
    out, lse = torch.empty_like(q, memory_format=torch.contiguous_format), q.new_empty((B, H, Lq), dtype=torch.float32)
    if B and Lq:
        q, at, strides = _strided(q)
        with _Launch(device) as (lib, stream):
            _lib.check(lib.artab_cache_attention(code, at, strides, B, Lq, cache._ref, cache.length,
                                                 Dh ** -0.5 if scale is None else float(scale), out.data_ptr(),
                                                 lse.data_ptr(), stream))
    return out, lse


def select_context_blocks(q: Tensor, cache: ContextCache, n_blocks: int) -> Tensor:
    """For every query of q [B,H,Lq,Dh] the ``n_blocks`` blocks of its context with the largest upper bound of a score:
    int32 [B,H,Lq,n_blocks] in ascending order, -1 behind the last where a context has fewer.

    The bound of a block is sum_d max(q_d lo_d, q_d hi_d) over the extreme keys of its channels, with the query rounded
    to whole numbers (largest magnitude 127): whole-number arithmetic, so the choice is reproducible to the bit; equal
    bounds go to the lower index.  A query that is not finite gets the first blocks, a block whose scale is NaN ranks before
    all others.  Capacities of up to 221184 rows, whatever is in use of them."""
    (B, H, Lq, _), code, device = _queries(q, cache, "select_context_blocks")
    n = int(n_blocks)
    if not 1 <= n <= _MOST_LISTED:
        raise ValueError(f"select_context_blocks: {n} blocks")
    index = q.new_empty((B, H, Lq, n), dtype=torch.int32)
    if B and Lq:
        q, at, strides = _strided(q)
        with _Launch(device) as (lib, stream):
            _lib.check(lib.artab_cache_select(code, at, strides, B, Lq, cache._ref, cache.length, n, index.data_ptr(),
                                              stream))
    return index


def block_context_attention(q: Tensor, cache: ContextCache, blocks: Tensor,
                            scale: Optional[float] = None) -> Tuple[Tensor, Tensor]:
    """``context_cache_attention`` over the rows of the listed blocks only: blocks int32 [B,H,Lq,S], as
    ``select_context_blocks`` gives them (at most 2^30 a query).  An index that is no block in use counts for nothing, one listed twice counts
    twice, a query whose list holds no block gets 0 and -inf."""
    (B, H, Lq, Dh), code, device = _queries(q, cache, "block_context_attention")
    shape = blocks.shape
    if len(shape) != 4 or shape[:3] != (B, H, Lq) or blocks.dtype is not torch.int32:
        raise ValueError(f"block_context_attention: blocks must be int32 [{B},{H},{Lq},S]")
    if shape[3] > _MOST_LISTED:
        raise ValueError(f"block_context_attention: {shape[3]} blocks a query")
    if blocks.get_device() != device:
        raise ValueError("block_context_attention: blocks must live on the device of the queries")
    out, lse = torch.empty_like(q, memory_format=torch.contiguous_format), q.new_empty((B, H, Lq), dtype=torch.float32)
    if shape[3] == 0:
        return out.zero_(), lse.fill_(float("-inf"))
    if B and Lq:
        blocks = blocks.contiguous()
        q, at, strides = _strided(q)
        with _Launch(device) as (lib, stream):
            need = lib.artab_cache_block_workspace(cache._ref, B, Lq, shape[3])
            ws = q.new_empty(need, dtype=torch.uint8) if need else None
            _lib.check(lib.artab_cache_block_attention(code, at, strides, B, Lq, cache._ref, blocks.data_ptr(), shape[3],
                                                       Dh ** -0.5 if scale is None else float(scale), out.data_ptr(),
                                                       lse.data_ptr(), _address(ws), need, stream))
    return out, lse
