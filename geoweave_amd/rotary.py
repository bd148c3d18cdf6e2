"""Rotary positions with several axes (time or view, row, column, ...) on gfx950.

The layer glue turns 64-wide heads by two axes (``RotaryPositionEmbedding2D``,
``easyvolcap/official_vggt/layers/rope.py:62-188``) inside its LayerNorm pass. Here any number of
axes from one to eight shares the head dim, each with its own block of dims and base, as video
(view, row, column) and finer grids need; with two axes of half the head dim each and positions
(row, column) the rotation is the glue's. Forward and backward run in ``gw_rotary_axes``; q and k
of a layer are turned in one launch that forms each angle once.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Sequence, Tuple, Union

import torch

from . import _lib

__all__ = ["rotary_axes_func", "rotary_axes_qk_func", "view_grid_positions"]

MAX_AXES = 8
MAX_HEAD_DIM = 256
_POS_CODES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}


def view_grid_positions(views: int, grid_h: int, grid_w: int, n_special: int = 5, device=None,
                        first_view: int = 0) -> torch.Tensor:
    """int32 ``[views * (n_special + grid_h * grid_w), 3]`` positions (view, row, column): a view's
    special tokens at (view, 0, 0), its patches at (view, row + 1, column + 1), row-major (the row and
    column of ``dsa_layer.grid_positions``)."""
    if min(views, grid_h, grid_w, n_special) < 0:
        raise ValueError("sizes must not be negative")
    ys = torch.arange(grid_h, device=device, dtype=torch.int32).repeat_interleave(grid_w) + 1
    xs = torch.arange(grid_w, device=device, dtype=torch.int32).repeat(grid_h) + 1
    zeros = torch.zeros(n_special, device=device, dtype=torch.int32)
    row, col = torch.cat([zeros, ys]), torch.cat([zeros, xs])
    view = torch.arange(first_view, first_view + views, device=device, dtype=torch.int32)
    return torch.stack([view.repeat_interleave(row.numel()), row.repeat(views), col.repeat(views)], dim=-1)


@functools.lru_cache(maxsize=256)
def _axis_args(axis_dims: Tuple[int, ...], bases: Tuple[float, ...]):
    n = len(axis_dims)
    return n, (ctypes.c_int32 * n)(*axis_dims), (ctypes.c_double * n)(*bases)


def _strides(x: torch.Tensor):
    """{batch, token, head or axis} strides; a tensor without a batch has one of one."""
    st = x.stride()
    return _lib.strides3(0, *st[-3:-1]) if x.dim() == 3 else _lib.strides3(*st[:3])


def _check(q, k, positions, axis_dims, bases):
    """Checked (axis_dims, bases)."""
    if q.dim() not in (3, 4):
        raise ValueError(f"expected [T, H, D] or [B, T, H, D], got {tuple(q.shape)}")
    if q.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"unsupported dtype {q.dtype}; the rotary kernel takes bfloat16, float16 or float32")
    if k is not None:
        if k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]:
            raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in more than their heads")
        if k.dtype != q.dtype:
            raise TypeError("q and k must have the same type")
    axis_dims = [int(n) for n in axis_dims]
    d = q.shape[-1]
    if not 1 <= len(axis_dims) <= MAX_AXES:
        raise ValueError(f"1 to {MAX_AXES} axes, got {len(axis_dims)}")
    if any(n < 0 or n % 2 for n in axis_dims) or sum(axis_dims) > d or (d - sum(axis_dims)) % 2:
        raise ValueError(f"axis dims {axis_dims} must be even and fit the head dim {d} with an even rest")
    if d < 1 or d > MAX_HEAD_DIM:
        raise ValueError(f"head dims from 1 to {MAX_HEAD_DIM} are supported, got {d}")
    if isinstance(bases, (int, float)):
        bases = [bases] * len(axis_dims)
    bases = [float(b) for b in bases]
    if len(bases) != len(axis_dims) or any(not (b > 0 and math.isfinite(b)) for b in bases):
        raise ValueError(f"one positive finite base per axis is needed, got {bases}")
    if positions.dtype not in _POS_CODES:
        raise TypeError(f"positions must be int32, int64 or float32, not {positions.dtype}")
    shape = tuple(positions.shape)
    want = tuple(q.shape[:-2]) + (len(axis_dims),)
    if shape != want and shape != want[-2:]:
        raise ValueError(f"positions {shape} must be {want}" + (f" or {want[-2:]}" if len(want) == 3 else ""))
    if not (q.is_cuda and positions.device == q.device and (k is None or k.device == q.device)):
        raise ValueError("q, k and positions must be tensors of one GPU")
    return tuple(axis_dims), tuple(bases)


def _rotate(xs, positions, axis_dims, bases, inverse: bool):
    """Turned copies (contiguous) of one or two tensors."""
    xs = [x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous() for x in xs]
    ys = [_lib.empty_rows(x) for x in xs]
    B = xs[0].shape[0] if xs[0].dim() == 4 else 1
    T, D = xs[0].shape[-3], xs[0].shape[-1]
    if B == 0 or T == 0 or all(x.shape[-2] == 0 for x in xs):
        return ys
    args = []
    for x, y in zip(xs, ys):
        h = x.shape[-2]
        args += [x.data_ptr(), _strides(x), y.data_ptr(), _lib.strides3(T * h * D, h * D, D), h]
    if len(xs) == 1:
        args += [None, None, None, None, 0]
    pos_strides = _lib.strides3(*positions.stride()) if positions.dim() == 3 else _lib.strides3(0, *positions.stride())
    dev = xs[0].device
    code = _lib.dtype_code(xs[0].dtype, allow_fp32=True)
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.gw_rotary_axes(code, *args, _POS_CODES[positions.dtype], positions.data_ptr(), pos_strides, B, T, D,
                                *_axis_args(axis_dims, bases), int(inverse), _lib.stream_handle(dev))
    _lib.check(rc, "gw_rotary_axes")
    return ys


class RotaryAxesFunc(torch.autograd.Function):
    """``(positions, axis_dims, bases, *tensors) -> turned tensors``; the gradient is turned back."""

    @staticmethod
    def forward(ctx, positions, axis_dims, bases, *xs):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)
        ctx.axis_dims, ctx.bases = axis_dims, bases
        return tuple(_rotate(xs, positions, axis_dims, bases, False))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        (positions,) = ctx.saved_tensors
        given = [g for g in grads if g is not None]
        turned = iter(_rotate(given, positions, ctx.axis_dims, ctx.bases, True)) if given else iter(())
        return (None, None, None) + tuple(None if g is None else next(turned) for g in grads)


def rotary_axes_func(x: torch.Tensor, positions: torch.Tensor, axis_dims: Sequence[int],
                     bases: Union[float, Sequence[float]] = 100.0) -> torch.Tensor:
    """``x`` (``[T, H, D]`` or ``[B, T, H, D]``, bf16, fp16 or fp32) turned by ``positions``
    (``[T, A]`` or ``[B, T, A]``; int32, int64 or float32): axis ``a`` turns dims ``i`` and ``i + d/2``
    of its block of ``d = axis_dims[a]`` dims by ``positions[..., a] * bases[a] ** (-2 i / d)``. The
    blocks lie one behind the other; dims behind the last are copied. The result is contiguous.
    Differentiable in ``x`` (positions get no gradient)."""
    axis_dims, bases = _check(x, None, positions, axis_dims, bases)
    return RotaryAxesFunc.apply(positions, axis_dims, bases, x)[0]


def rotary_axes_qk_func(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, axis_dims: Sequence[int],
                        bases: Union[float, Sequence[float]] = 100.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`rotary_axes_func` of a layer's q and k (their numbers of heads may differ) in one launch;
    either may be a column block of a fused projection."""
    axis_dims, bases = _check(q, k, positions, axis_dims, bases)
    return RotaryAxesFunc.apply(positions, axis_dims, bases, q, k)
