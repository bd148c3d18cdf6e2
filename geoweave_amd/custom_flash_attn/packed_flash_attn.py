"""Attention over packed sequences of different lengths on gfx950: bidirectional or causal, grouped
heads, forward and backward.

The tokens of all sequences lie one behind the other and ``cu_seqlens`` bounds them, so scenes of
different numbers of views, and views of different grids, share one call without padding: global
attention is the call with a scene per sequence, frame attention (``easyvolcap/official_vggt/
layers/attention.py:38-98`` over ``[B * S, P]``) the call with a view per sequence.

* ``packed_flash_attn_func(q, k, v, cu_seqlens_q, cu_seqlens_k=None, causal=False,
  softmax_scale=None) -> o`` with autograd;
* ``packed_flash_attn_inference_func(..., return_lse=False) -> (o, lse | None)``.

q: ``[Tq, Hq, D]``, k/v: ``[Tk, Hk, D]`` with Hq a multiple of Hk (query head h reads key head
``h // (Hq // Hk)``), bf16 or fp16, any D <= 128 (the kernels are built for 64 and 128; other D run on
inputs zero-padded to the next of those). ``cu_seqlens_*``: int32 ``[n + 1]`` on the GPU, starting at 0,
non-decreasing; sequence i has the query tokens ``[cu_q[i], cu_q[i + 1])`` and the keys ``[cu_k[i],
cu_k[i + 1])``. Causal order counts from the end: query i of Lq sees key j of Lk when
``j <= i + Lk - Lq``. A query that sees no key gets o = 0 and lse = -inf and passes no gradient on; tokens
behind the last bound get zeros as well. The bounds are read by the kernels only: no call waits
for the GPU, and a captured graph may be replayed with other bounds of as many sequences.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from .. import _lib
from .sparse_index_flash_attn import NATIVE_HEAD_DIMS, _pad_head_dim, _padded_head_dim

__all__ = ["packed_flash_attn_func", "packed_flash_attn_inference_func", "PackedFlashAttnFunc"]

# The kernels' 32-bit load offsets bound a token stride (64 rows of a tile).
MAX_ROW_STRIDE = 1 << 24
MAX_TOKEN_HEADS = 0x7FFFF000


def _check_heads(q, k, v):
    """The checks of q, k, v that the packed and the paged call share (heads in dim -2)."""
    d = q.shape[-1]
    if k.shape != v.shape or k.shape[-1] != d:
        raise ValueError(f"k/v shapes {tuple(k.shape)}/{tuple(v.shape)} do not match each other and the head dim {d}")
    if not 1 <= d <= 128:
        raise ValueError(f"head dimensions from 1 to 128 are supported, got {d}")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError("All tensors must have the same type")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("Only support fp16 and bf16")
    hq, hk = q.shape[-2], k.shape[-2]
    if hk < 1 or hq < 1 or hq % hk:
        raise ValueError(f"{hq} query heads are not a multiple of {hk} key heads")


def _check_scale(softmax_scale: Optional[float], d: int) -> float:
    scale = 1.0 / math.sqrt(d) if softmax_scale is None else float(softmax_scale)
    # The kernels hold scale * log2(e) in fp32.
    if not 1e-30 <= scale <= 1e30:
        raise ValueError(f"softmax_scale must lie in [1e-30, 1e30], got {softmax_scale}")
    return scale


def _check_inputs(q, k, v, cu_q, cu_k, softmax_scale):
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"q {tuple(q.shape)} and k/v {tuple(k.shape)} must be [tokens, heads, head dim]")
    _check_heads(q, k, v)
    if cu_k is None:
        cu_k = cu_q
        if k.shape[0] != q.shape[0]:
            raise ValueError("cu_seqlens_k is needed where q and k have different numbers of tokens")
    for cu in (cu_q, cu_k):
        if cu.dtype != torch.int32:
            raise TypeError("cu_seqlens must be int32")
        if cu.dim() != 1 or cu.numel() < 1:
            raise ValueError(f"cu_seqlens must be [sequences + 1], got {tuple(cu.shape)}")
    if cu_q.numel() != cu_k.numel():
        raise ValueError(f"cu_seqlens of {cu_q.numel() - 1} and {cu_k.numel() - 1} sequences")
    if max(q.shape[0], k.shape[0]) * q.shape[1] > MAX_TOKEN_HEADS:
        raise ValueError(f"tokens x query heads must not exceed {MAX_TOKEN_HEADS}")
    scale = _check_scale(softmax_scale, q.shape[-1])
    if not (q.is_cuda and all(t.device == q.device for t in (k, v, cu_q, cu_k))):
        raise ValueError("q, k, v and cu_seqlens must be tensors of one GPU")
    return cu_q.contiguous(), cu_k.contiguous(), scale


def _rows(x: torch.Tensor):
    """(x, (its address, its strides)) with 16-byte rows, and a token stride within the kernels' offsets; of a copy
    where they are not (clone: a contiguous tensor may start anywhere)."""
    st, sh = _lib.row_strides(x)
    if x.stride(2) != 1 or (st | sh) & 7 or st >= MAX_ROW_STRIDE or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        st, sh = _lib.row_strides(x)
    return x, (x.data_ptr(), _lib.strides2(st, sh))


def _forward(q, k, v, cu_q, cu_k, causal: bool, scale: float, want_lse: bool, want_rest: bool = False):
    """(o, lse | None, what o's rounding left | None) for a native head dim."""
    tq, hq, d = q.shape
    o = _lib.empty_rows(q)
    lse = torch.empty((tq, hq), device=q.device, dtype=torch.float32) if want_lse else None
    rest = _lib.empty_rows(q) if want_rest else None
    if tq == 0:
        return o, lse, rest
    (q, qr), (k, kr), (v, vr) = _rows(q), _rows(k), _rows(v)
    lib = _lib.load()
    sizes = (cu_q.numel() - 1, tq, k.shape[0], hq, k.shape[1], d)
    nbytes = int(lib.gw_packed_attn_fwd_workspace_size(*sizes))
    ws = torch.empty(nbytes, device=q.device, dtype=torch.uint8) if nbytes else None
    with _lib.on_device(q.device):
        rc = lib.gw_packed_attn_fwd(_lib.dtype_code(q.dtype), *qr, *kr, *vr, cu_q.data_ptr(), cu_k.data_ptr(),
                                    o.data_ptr(), _lib.strides2(hq * d, d), _lib.ptr(rest), _lib.ptr(lse), *sizes,
                                    int(causal), scale, _lib.ptr(ws), nbytes, _lib.stream_handle(q.device))
    _lib.check(rc, "gw_packed_attn_fwd")
    return o, lse, rest


def _backward(do, q, k, v, cu_q, cu_k, o, rest, lse, causal: bool, scale: float):
    dq, dk, dv = _lib.empty_rows(q), _lib.empty_rows(k), _lib.empty_rows(v)
    (tq, hq, d), (tk, hk, _) = q.shape, k.shape
    if tq == 0 and tk == 0:
        return dq, dk, dv
    (q, qr), (k, kr), (v, vr), (o, orow), (do, dor) = _rows(q), _rows(k), _rows(v), _rows(o), _rows(do)
    n, q_out, k_out = cu_q.numel() - 1, _lib.strides2(hq * d, d), _lib.strides2(hk * d, d)
    lib = _lib.load()
    nbytes = int(lib.gw_packed_attn_bwd_workspace_size(n, tq, tk, hq, hk, d))
    ws = torch.empty(max(nbytes, 16), device=q.device, dtype=torch.uint8)
    with _lib.on_device(q.device):
        rc = lib.gw_packed_attn_bwd(_lib.dtype_code(q.dtype), *qr, *kr, *vr, cu_q.data_ptr(), cu_k.data_ptr(), *orow,
                                    rest.data_ptr(), *dor, lse.data_ptr(), dq.data_ptr(), q_out, dk.data_ptr(), k_out,
                                    dv.data_ptr(), k_out, n, tq, tk, hq, hk, d, int(causal), scale, ws.data_ptr(), nbytes,
                                    _lib.stream_handle(q.device))
    _lib.check(rc, "gw_packed_attn_bwd")
    return dq, dk, dv


class PackedFlashAttnFunc(torch.autograd.Function):
    """``(q, k, v, cu_q, cu_k, causal, scale) -> o`` on checked arguments."""

    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, causal, scale):
        d = q.shape[-1]
        dp = d if d in NATIVE_HEAD_DIMS else _padded_head_dim(d)
        qp, kp, vp = (q, k, v) if dp == d else (_pad_head_dim(x, dp) for x in (q, k, v))
        o, lse, rest = _forward(qp, kp, vp, cu_q, cu_k, causal, scale, True, True)
        if dp != d:
            o = o[..., :d].contiguous()
        ctx.save_for_backward(q, k, v, cu_q, cu_k, o, rest, lse)
        ctx.causal, ctx.scale = causal, scale
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        q, k, v, cu_q, cu_k, o, rest, lse = ctx.saved_tensors
        d = q.shape[-1]
        dp = d if d in NATIVE_HEAD_DIMS else _padded_head_dim(d)
        args = [do, q, k, v] if dp == d else [_pad_head_dim(x, dp) for x in (do, q, k, v)]
        op = o if dp == d else _pad_head_dim(o, dp)
        grads = _backward(*args, cu_q, cu_k, op, rest, lse, ctx.causal, ctx.scale)
        if dp != d:
            grads = [g[..., :d].contiguous() for g in grads]
        return (*grads, None, None, None, None)


def packed_flash_attn_func(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                           cu_seqlens_k: Optional[torch.Tensor] = None, causal: bool = False,
                           softmax_scale: Optional[float] = None) -> torch.Tensor:
    """Attention of each packed sequence (see the module docstring): o, contiguous, in q's shape and
    dtype. Differentiable in q, k and v; the gradients are the same bits for the same inputs."""
    cu_q, cu_k, scale = _check_inputs(q, k, v, cu_seqlens_q, cu_seqlens_k, softmax_scale)
    return PackedFlashAttnFunc.apply(q, k, v, cu_q, cu_k, bool(causal), scale)


def packed_flash_attn_inference_func(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                                     cu_seqlens_k: Optional[torch.Tensor] = None, causal: bool = False,
                                     softmax_scale: Optional[float] = None, return_lse: bool = False,
                                     ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(o, lse): :func:`packed_flash_attn_func` without autograd; lse (natural log, fp32
    ``[Tq, Hq]``) only where asked for, else None."""
    cu_q, cu_k, scale = _check_inputs(q, k, v, cu_seqlens_q, cu_seqlens_k, softmax_scale)
    d = q.shape[-1]
    if d in NATIVE_HEAD_DIMS:
        return _forward(q, k, v, cu_q, cu_k, bool(causal), scale, return_lse)[:2]
    dp = _padded_head_dim(d)
    o, lse, _ = _forward(_pad_head_dim(q, dp), _pad_head_dim(k, dp), _pad_head_dim(v, dp), cu_q, cu_k, bool(causal),
                         scale, return_lse)
    return o[..., :d].contiguous(), lse
