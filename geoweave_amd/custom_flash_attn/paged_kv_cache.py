"""Writing a paged key-value cache and reading it back on gfx950: 16-bit rows, or 4-bit ones in a quarter of the memory.

``paged_flash_attn`` attends over a cache that holds the new tokens already. Here they are put there, in one launch
that turns k and q by their positions on the way (``rotary``), and whole sequences come back as packed rows, as
``packed_flash_attn`` takes them where a step has many new tokens.

* ``paged_kv_append_func(k, v, k_cache, v_cache, block_table, cache_seqlens, q=None, positions=None, axis_dims=None,
  bases=100.0, cu_seqlens=None) -> turned q | None``
* ``paged_kv_read_func(k_cache, v_cache, block_table, cu_seqlens, tokens, dtype=None) -> (k, v)``
* ``FP4Cache(codes, scales)``, ``fp4_paged_cache(pages, page_size, heads, head_dim)``: a cache in 4 bits.

A 16-bit cache is a tensor ``[pages, page_size, Hk, D]``, bf16 or fp16, D 64 or 128, any strides with 16-byte
aligned rows. An :class:`FP4Cache` holds uint8 ``codes [pages, page_size, Hk, D / 2]`` (e2m1: 0, 1/2, 1, 3/2, 2, 3, 4, 6
and a sign, two to a byte, the even dim in the low half) and uint8 ``scales [pages, page_size, Hk, D / 32]``, the biased
exponent of the power of two that 32 dims share (255: not a number): 4.25 bits a value. The power brings the
largest of the 32 to (3.5, 7] units, so a value is off by at most one unit and normal rows by 0.112 of their
rms. Nothing is divided or fitted: the same row always gets the same codes.

Key j of sequence b is slot ``j % page_size`` of page ``block_table[b, j // page_size]``, as in ``paged_flash_attn``.
Tables, lengths and bounds are int32 on the GPU and read by the kernels only: no call waits for the GPU, and a captured
graph follows them. These functions have no gradients; caches are written in place.
"""
from __future__ import annotations

import functools
import math
from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch

from .. import _lib
from ..rotary import MAX_AXES, _POS_CODES, _axis_args
from .sparse_index_flash_attn import NATIVE_HEAD_DIMS

__all__ = ["FP4Cache", "fp4_paged_cache", "paged_kv_append_func", "paged_kv_read_func"]

MAX_KEYS = 0x7FFFF000


class FP4Cache(NamedTuple):
    """A paged cache of keys or values in 4 bits (see the module docstring)."""

    codes: torch.Tensor
    scales: torch.Tensor


Cache = Union[torch.Tensor, FP4Cache]


def fp4_paged_cache(pages: int, page_size: int, heads: int, head_dim: int, device=None) -> FP4Cache:
    """Zeros. A head's slots of a page lie one behind the other in memory, so that attention, which takes a head at a
    time, reads whole lines."""
    if head_dim not in NATIVE_HEAD_DIMS:
        raise ValueError(f"head dims {NATIVE_HEAD_DIMS} are supported in a paged cache, got {head_dim}")
    if min(pages, page_size, heads) < 0:
        raise ValueError("sizes must not be negative")
    return FP4Cache(*(torch.zeros(pages, heads, page_size, head_dim // n, dtype=torch.uint8, device=device).transpose(1, 2)
                      for n in (2, 32)))


def _layout(x: torch.Tensor, align: int):
    """(address, strides of the first three dims) of x [.., .., .., row], None where its rows are not contiguous and aligned to
    ``align`` bytes."""
    s0, s1, s2, s3 = x.stride()
    at, units = x.data_ptr(), align // x.element_size() - 1
    if s3 != 1 or (s0 | s1 | s2) & units or at & (align - 1):
        if x.numel() == 0:
            return None, _lib.strides3(0, 0, 0)
        s0, s1, s2 = _lib.row_strides(x)  # dims of one entry have any strides
        if s3 != 1 and x.shape[3] != 1 or (s0 | s1 | s2) & units or at & (align - 1):
            return None
    return at, _lib.strides3(s0, s1, s2)


def cache_args(k_cache: Cache, v_cache: Cache):
    """(format, rows, heads, head dim, the C entries' k and v arguments) of a checked pair of caches; ``rows``: the
    tensor of k's rows."""
    fp4 = isinstance(k_cache, FP4Cache)
    if fp4 != isinstance(v_cache, FP4Cache):
        raise TypeError("k_cache and v_cache must both be 16-bit tensors or both FP4Cache")
    k, v = (k_cache[0], v_cache[0]) if fp4 else (k_cache, v_cache)
    if not (isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor)):
        raise TypeError("a cache is a tensor or an FP4Cache")
    shape = k.shape
    if len(shape) != 4 or v.shape != shape:
        raise ValueError(f"caches must be [pages, page_size, Hk, D], got {tuple(shape)} and {tuple(v.shape)}")
    pages, page, hk, d = shape
    if fp4:
        d *= 2
    if d not in NATIVE_HEAD_DIMS:
        raise ValueError(f"head dims {NATIVE_HEAD_DIMS} are supported over a paged cache, got {d}")
    if page < 1 or hk < 1:
        raise ValueError("pages must have at least one slot, and slots a head")
    # Copying a cache to align it would cost more than the call: the caller lays it out.
    kl, vl = _layout(k, 16), _layout(v, 16)
    if kl is None or vl is None:
        raise ValueError("caches need a unit last stride and 16-byte aligned rows")
    device = k.device
    if not fp4:
        if k.dtype != v.dtype:
            raise TypeError("All tensors must have the same type")
        if k.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError("Only support fp16 and bf16")
        if v.device != device:
            raise ValueError("k_cache and v_cache must be tensors of one GPU")
        return _lib.GW_CACHE_16BIT, k, hk, d, (*kl, None, None, *vl, None, None)
    ks, vs = k_cache[1], v_cache[1]
    if any(t.dtype != torch.uint8 for t in (k, ks, v, vs)):
        raise TypeError("codes and scales of an FP4Cache must be uint8")
    if ks.shape != (pages, page, hk, d // 32) or vs.shape != ks.shape:
        raise ValueError(f"scales {tuple(ks.shape)} and {tuple(vs.shape)} of codes {tuple(shape)} must have a byte for 32 dims")
    ksl, vsl = _layout(ks, d // 32), _layout(vs, d // 32)
    if ksl is None or vsl is None:
        raise ValueError(f"scales need a unit last stride and rows aligned to their {d // 32} bytes")
    if not device == ks.device == v.device == vs.device:
        raise ValueError("codes and scales of k and v must be tensors of one GPU")
    return _lib.GW_CACHE_FP4, k, hk, d, (*kl, *ksl, *vl, *vsl)


def _check_table(rows, block_table, *more):
    """block_table with unit column stride, checked together with the lists of lengths and bounds."""
    device = rows.device
    if not rows.is_cuda:
        raise ValueError("the caches, block_table, lengths and bounds must be tensors of one GPU")
    for t in (block_table, *more):
        if t.dtype != torch.int32:
            raise TypeError("block_table, lengths and bounds must be int32")
        if t.device != device:
            raise ValueError("the caches, block_table, lengths and bounds must be tensors of one GPU")
    if block_table.shape[1] * rows.shape[1] > MAX_KEYS:
        raise ValueError(f"keys of a sequence must not exceed {MAX_KEYS}")
    return block_table if block_table.stride(1) == 1 or block_table.shape[1] == 1 else block_table.contiguous()


def _token_rows(x: torch.Tensor, packed: bool):
    """(x with 16-byte aligned rows, its {sequence, token, head} strides)."""
    st = x.stride()
    if st[-1] != 1 or any(s & 7 for s in st[:-1]) or x.data_ptr() & 15:
        st = _lib.row_strides(x)  # dims of one entry have any strides
        if x.stride(-1) != 1 or any(s & 7 for s in st) or x.data_ptr() & 15:
            x = x.clone(memory_format=torch.contiguous_format)
            st = x.stride()
    if x.dim() == 4:
        return x, _lib.strides3(st[0], st[1], st[2])
    return x, _lib.strides3(0, st[0], st[1]) if packed else _lib.strides3(st[0], 0, st[1])


@functools.lru_cache(maxsize=256)
def _axes(axis_dims: Tuple[int, ...], bases: Union[float, Tuple[float, ...]], d: int):
    """The C entry's axes, checked."""
    if not 1 <= len(axis_dims) <= MAX_AXES:
        raise ValueError(f"1 to {MAX_AXES} axes, got {len(axis_dims)}")
    if any(int(n) != n or n < 0 or n % 2 for n in axis_dims) or sum(axis_dims) > d:
        raise ValueError(f"axis dims {axis_dims} must be even and fit the head dim {d}")
    if isinstance(bases, (int, float)):
        bases = (bases,) * len(axis_dims)
    bases = tuple(float(b) for b in bases)
    if len(bases) != len(axis_dims) or any(not (b > 0 and math.isfinite(b)) for b in bases):
        raise ValueError(f"one positive finite base per axis is needed, got {bases}")
    return _axis_args(tuple(int(n) for n in axis_dims), bases)


def paged_kv_append_func(k: torch.Tensor, v: torch.Tensor, k_cache: Cache, v_cache: Cache, block_table: torch.Tensor,
                         cache_seqlens: torch.Tensor, q: Optional[torch.Tensor] = None,
                         positions: Optional[torch.Tensor] = None, axis_dims: Optional[Sequence[int]] = None,
                         bases: Union[float, Sequence[float]] = 100.0,
                         cu_seqlens: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes new tokens' k and v into the caches, in place, and returns q turned (None without q).

    k, v: ``[B, N, Hk, D]`` (N new tokens of each sequence), ``[B, Hk, D]`` (one), or packed ``[T, Hk, D]`` with
    ``cu_seqlens`` (int32 ``[B + 1]``, non-decreasing: sequence b has the tokens ``[cu[b], cu[b + 1])``), bf16 or fp16, for a
    16-bit cache of the same type; q alike with any number of heads. All may be column blocks of one projection.
    ``cache_seqlens`` int32 ``[B]``: keys of each sequence with the new tokens counted: new token i of n becomes key
    ``cache_seqlens - n + i``.

    ``positions`` (``k.shape[:-2] + (A,)``, int32, int64 or float32) and ``axis_dims`` (of A axes) turn k and q as
    ``rotary_axes_func`` does, with ``bases``; without them nothing is turned. The result is rounded once,
    to the tokens' type or to 4 bits; 32 dims with an inf or NaN are kept as NaN in 4 bits, bf16 values above 3.5 * 2^126 as inf.

    A token whose key has no slot (below 0, behind the table, in a page outside the pool) and a token of no
    sequence is written nowhere; its q is turned all the same. Two new tokens that come to one slot (pages that
    sequences share) leave unspecified contents there. The caches must not overlap each other, q, k or v."""
    fmt, rows, hk, d, args = cache_args(k_cache, v_cache)
    packed = cu_seqlens is not None
    shape, dtype, dev = k.shape, k.dtype, rows.device
    nd = len(shape)
    if nd != 3 and (packed or nd != 4) or v.shape != shape or shape[-2] != hk or shape[-1] != d:
        raise ValueError(f"k {tuple(shape)} and v {tuple(v.shape)} must be "
                         f"{'[T, Hk, D]' if packed else '[B, Hk, D] or [B, N, Hk, D]'} of the caches' Hk = {hk}, D = {d}")
    if dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("Only support fp16 and bf16")
    if v.dtype != dtype or (q is not None and q.dtype != dtype) or (fmt == _lib.GW_CACHE_16BIT and rows.dtype != dtype):
        raise TypeError("All tensors must have the same type")
    if q is not None and (q.dim() != nd or q.shape[:-2] != shape[:-2] or q.shape[-1] != d):
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(shape)} differ in more than their heads")
    if (positions is None) != (axis_dims is None):
        raise ValueError("positions and axis_dims go together")
    n = cache_seqlens.shape[0] if cache_seqlens.dim() == 1 else -1
    if block_table.dim() != 2 or block_table.shape[0] != n:
        raise ValueError(f"block_table {tuple(block_table.shape)} and cache_seqlens {tuple(cache_seqlens.shape)} must be "
                         "[sequences, W] and [sequences]")
    if packed:
        if cu_seqlens.shape != (n + 1,):
            raise ValueError(f"cu_seqlens {tuple(cu_seqlens.shape)} does not go with cache_seqlens of {n} sequences")
        block_table = _check_table(rows, block_table, cache_seqlens, cu_seqlens)
        tokens, count = shape[0], shape[0]
        cu_seqlens = cu_seqlens.contiguous()
    else:
        if shape[0] != n:
            raise ValueError(f"k {tuple(shape)} does not go with cache_seqlens of {n} sequences")
        block_table = _check_table(rows, block_table, cache_seqlens)
        count = 1 if nd == 3 else shape[1]
        tokens = n * count
    if k.device != dev or v.device != dev or (q is not None and q.device != dev):
        raise ValueError("q, k, v and the caches must be tensors of one GPU")
    hq = 0 if q is None else q.shape[-2]
    if tokens * (hq + 2 * hk) > MAX_KEYS:
        raise ValueError(f"tokens x heads must not exceed {MAX_KEYS}")
    axes, pos = (0, None, None), (0, None, None)
    if positions is not None:
        axes = _axes(tuple(axis_dims), bases if isinstance(bases, (int, float)) else tuple(bases), d)
        if positions.dtype not in _POS_CODES:
            raise TypeError(f"positions must be int32, int64 or float32, not {positions.dtype}")
        if positions.shape != (*shape[:-2], axes[0]):
            raise ValueError(f"positions {tuple(positions.shape)} must be {(*shape[:-2], axes[0])}")
        if positions.device != dev:
            raise ValueError("positions must lie on the caches' GPU")
        st = positions.stride()
        pos = (_POS_CODES[positions.dtype], positions.data_ptr(),
               _lib.strides3(*st) if nd == 4 else _lib.strides3(0, *st) if packed else _lib.strides3(st[0], 0, st[1]))
    turned = None if q is None else _lib.empty_rows(q)
    if tokens == 0:
        return turned
    k, k_strides = _token_rows(k, packed)
    v, v_strides = _token_rows(v, packed)
    q_args = (None, None, None, 0)
    if q is not None:
        q, q_strides = _token_rows(q, packed)
        q_args = (q.data_ptr(), q_strides, turned.data_ptr(), hq)
    cache_seqlens = cache_seqlens.contiguous()
    with _lib.on_device(dev):
        rc = _lib.load().gw_paged_kv_append(
            _lib.dtype_code(dtype), *q_args, k.data_ptr(), k_strides, v.data_ptr(), v_strides, hk, d, fmt, *args,
            block_table.data_ptr(), block_table.stride(0), cache_seqlens.data_ptr(), _lib.ptr(cu_seqlens), n, count, rows.shape[0],
            rows.shape[1], block_table.shape[1], *pos, *axes, _lib.stream_handle(dev))
    _lib.check(rc, "gw_paged_kv_append")
    return turned


def paged_kv_read_func(k_cache: Cache, v_cache: Cache, block_table: torch.Tensor, cu_seqlens: torch.Tensor, tokens: int,
                       dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v), contiguous ``[tokens, Hk, D]``: row ``cu_seqlens[b] + j`` holds key j of sequence b, for
    ``cu_seqlens[b + 1] - cu_seqlens[b]`` keys (int32 ``[B + 1]``, non-decreasing). ``dtype``: bf16 (the default) or fp16 for an
    :class:`FP4Cache`, whose values bf16 holds exactly and fp16 where its range allows; a 16-bit cache's own type.
    Rows of no sequence, and of keys without a slot, are zeros: leave the latter, which paged attention shows to nobody, out of
    the bounds."""
    fmt, rows, hk, d, args = cache_args(k_cache, v_cache)
    if dtype is None:
        dtype = torch.bfloat16 if fmt == _lib.GW_CACHE_FP4 else rows.dtype
    if dtype not in (torch.float16, torch.bfloat16) or (fmt == _lib.GW_CACHE_16BIT and dtype != rows.dtype):
        raise TypeError(f"{dtype}: an FP4Cache is read as bf16 or fp16, a 16-bit cache as its own type")
    if block_table.dim() != 2 or cu_seqlens.dim() != 1 or cu_seqlens.shape[0] != block_table.shape[0] + 1:
        raise ValueError(f"block_table {tuple(block_table.shape)} and cu_seqlens {tuple(cu_seqlens.shape)} must be "
                         "[sequences, W] and [sequences + 1]")
    tokens = int(tokens)
    if tokens < 0 or tokens * 2 * hk > MAX_KEYS:
        raise ValueError(f"tokens x heads must lie in [0, {MAX_KEYS}], got {tokens} x {2 * hk}")
    block_table = _check_table(rows, block_table, cu_seqlens)
    dev = rows.device
    k, v = (torch.empty((tokens, hk, d), dtype=dtype, device=dev) for _ in range(2))
    if tokens == 0:
        return k, v
    cu_seqlens = cu_seqlens.contiguous()
    with _lib.on_device(dev):
        rc = _lib.load().gw_paged_kv_read(
            _lib.dtype_code(dtype), fmt, *args, block_table.data_ptr(), block_table.stride(0), cu_seqlens.data_ptr(),
            block_table.shape[0], tokens, hk, d, rows.shape[0], rows.shape[1], block_table.shape[1], k.data_ptr(), v.data_ptr(),
            _lib.stream_handle(dev))
    _lib.check(rc, "gw_paged_kv_read")
    return k, v
