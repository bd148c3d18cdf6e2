"""Attention of one new token, or a few, over a paged key-value cache on gfx950.

``packed_flash_attn`` over a whole batch of tokens has this as its form for single tokens: the keys and
values of the tokens seen so far stay in a pool of pages, each sequence's block table names its
pages, and a step's new tokens (one, or a new view's special tokens) attend to them. The keys are
split over workgroups by the lengths on the device and the parts joined.

``paged_flash_attn_inference_func(q, k_cache, v_cache, block_table, cache_seqlens, causal=True,
softmax_scale=None, return_lse=False) -> (o, lse | None)``

q: ``[B, Hq, D]`` (one new token per sequence) or ``[B, N, Hq, D]``; k_cache/v_cache: ``[pages, page_size,
Hk, D]``, Hq a multiple of Hk, bf16 or fp16, D 64 or 128 (a cache is not padded per call), any page
size; block_table: int32 ``[B, W]``; cache_seqlens: int32 ``[B]``, the keys of each sequence, those of
the new tokens included (the caller has written them, as ``paged_kv_append_func`` does). Key j of sequence b is slot
``j % page_size`` of page
``block_table[b, j // page_size]``; the keys of a page number outside ``[0, pages)`` are seen by nobody, as
``kv_positions`` outside ``[0, S)`` are in sparse_index_flash_attn. Causal order (the default): new token i of
N sees the keys below ``cache_seqlens - N + 1 + i``. A token that sees no key gets o = 0, lse = -inf.
Table and lengths are read by the kernels only.

The caches may also be a pair of ``paged_kv_cache.FP4Cache``: the same attention over the values that 4 bits hold, at a
quarter of the bytes. They enter the products exactly, and the weights keep 16 bits. 32 values kept as not a number
are NaN, and values of 2^128 and above inf, in the rows that see them.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _lib
from .packed_flash_attn import _check_heads, _check_scale
from .paged_kv_cache import MAX_KEYS, Cache, FP4Cache, cache_args
from .sparse_index_flash_attn import NATIVE_HEAD_DIMS

__all__ = ["paged_flash_attn_inference_func"]


def _check_fp4(q, k_cache, v_cache, block_table, cache_seqlens, softmax_scale):
    """(scale, the C entry's k and v arguments), checked."""
    if q.dim() not in (3, 4):
        raise ValueError(f"q must be [B, Hq, D] or [B, N, Hq, D], got {tuple(q.shape)}")
    _, rows, hk, d, args = cache_args(k_cache, v_cache)
    if q.shape[-1] != d:
        raise ValueError(f"q's head dim {q.shape[-1]} is not the caches' {d}")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("Only support fp16 and bf16")
    if q.shape[-2] < 1 or q.shape[-2] % hk:
        raise ValueError(f"{q.shape[-2]} query heads are not a multiple of {hk} key heads")
    _check_lists(q, rows, block_table, cache_seqlens)
    return _check_scale(softmax_scale, d), args


def _check_lists(q, k_cache, block_table, cache_seqlens):
    if block_table.dtype != torch.int32 or cache_seqlens.dtype != torch.int32:
        raise TypeError("block_table and cache_seqlens must be int32")
    if block_table.dim() != 2 or block_table.shape[0] != q.shape[0] or tuple(cache_seqlens.shape) != (q.shape[0],):
        raise ValueError(f"block_table {tuple(block_table.shape)} and cache_seqlens {tuple(cache_seqlens.shape)} must be "
                         f"[{q.shape[0]}, W] and [{q.shape[0]}]")
    if block_table.shape[1] * k_cache.shape[1] > MAX_KEYS or q.numel() // q.shape[-1] > MAX_KEYS:
        raise ValueError(f"keys of a sequence, and new tokens x heads, must not exceed {MAX_KEYS}")
    device = q.device
    if not (q.is_cuda and k_cache.device == block_table.device == cache_seqlens.device == device):
        raise ValueError("q, the caches, block_table and cache_seqlens must be tensors of one GPU")


def _check_inputs(q, k_cache, v_cache, block_table, cache_seqlens, softmax_scale):
    """(scale, strides of k_cache, of v_cache), checked."""
    if q.dim() not in (3, 4):
        raise ValueError(f"q must be [B, Hq, D] or [B, N, Hq, D], got {tuple(q.shape)}")
    if k_cache.dim() != 4:
        raise ValueError(f"caches must be [pages, page_size, Hk, D], got {tuple(k_cache.shape)}")
    _check_heads(q, k_cache, v_cache)
    d = q.shape[-1]
    if d not in NATIVE_HEAD_DIMS:
        raise ValueError(f"head dims {NATIVE_HEAD_DIMS} are supported over a paged cache, got {d}")
    if k_cache.shape[1] < 1:
        raise ValueError("pages must have at least one slot")
    scale = _check_scale(softmax_scale, d)
    _check_lists(q, k_cache, block_table, cache_seqlens)
    if v_cache.device != q.device:
        raise ValueError("q, the caches, block_table and cache_seqlens must be tensors of one GPU")
    strides = []
    for c in (k_cache, v_cache):
        # Copying a cache to align it would cost more than the call: the caller lays it out.
        page, slot, head = _lib.row_strides(c)
        if c.numel() and (c.stride(3) != 1 or (page | slot | head) & 7 or c.data_ptr() % 16):
            raise ValueError("caches need a unit last stride and 16-byte aligned rows")
        strides.append(_lib.strides3(page, slot, head))
    return scale, *strides


def paged_flash_attn_inference_func(q: torch.Tensor, k_cache: Cache, v_cache: Cache,
                                    block_table: torch.Tensor, cache_seqlens: torch.Tensor, causal: bool = True,
                                    softmax_scale: Optional[float] = None, return_lse: bool = False,
                                    ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(o in q's shape and dtype, lse fp32 ``q.shape[:-1]`` where asked for); see the module docstring."""
    fp4 = isinstance(k_cache, FP4Cache) or isinstance(v_cache, FP4Cache)
    if fp4:
        scale, args = _check_fp4(q, k_cache, v_cache, block_table, cache_seqlens, softmax_scale)
        pages, page, hk, _ = k_cache.codes.shape
    else:
        scale, k_strides, v_strides = _check_inputs(q, k_cache, v_cache, block_table, cache_seqlens, softmax_scale)
        args = (k_cache.data_ptr(), k_strides, v_cache.data_ptr(), v_strides)
        pages, page, hk, _ = k_cache.shape
    new = _lib.row_strides(q)
    if q.stride(-1) != 1 or any(s & 7 for s in new) or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)  # a contiguous tensor may start anywhere
        new = _lib.row_strides(q)
    if block_table.stride(-1) != 1:
        block_table = block_table.contiguous()
    cache_seqlens = cache_seqlens.contiguous()
    dev = q.device
    o = _lib.empty_rows(q)
    lse = torch.empty(q.shape[:-1], device=dev, dtype=torch.float32) if return_lse else None
    if q.dim() == 4:
        b, n, hq, d = q.shape
        q_strides, o_strides = _lib.strides3(*new), _lib.strides3(n * hq * d, hq * d, d)
    else:
        (b, hq, d), n = q.shape, 1
        q_strides, o_strides = _lib.strides3(new[0], 0, new[1]), _lib.strides3(hq * d, 0, d)
    if b == 0 or n == 0:
        return o, lse
    lib = _lib.load()
    size, fwd = ((lib.gw_paged_attn_fp4_fwd_workspace_size, lib.gw_paged_attn_fp4_fwd) if fp4 else
                 (lib.gw_paged_attn_fwd_workspace_size, lib.gw_paged_attn_fwd))
    nbytes = int(size(b, n, hq, hk, d))
    ws = torch.empty(nbytes, device=dev, dtype=torch.uint8) if nbytes else None
    with _lib.on_device(dev):
        rc = fwd(_lib.dtype_code(q.dtype), q.data_ptr(), q_strides, *args, block_table.data_ptr(), block_table.stride(0),
                 cache_seqlens.data_ptr(), o.data_ptr(), o_strides, _lib.ptr(lse), b, n, hq, hk, d, pages, page,
                 block_table.shape[1], int(causal), scale, _lib.ptr(ws), nbytes, _lib.stream_handle(dev))
    _lib.check(rc, "gw_paged_attn_fp4_fwd" if fp4 else "gw_paged_attn_fwd")
    return o, lse
