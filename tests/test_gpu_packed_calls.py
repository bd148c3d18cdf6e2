"""Calls that the documentation allows beside the usual ones: a whole view's tokens over a paged cache, rotation in
place through the C entry, gradients of some inputs only and twice, calls on two streams at once, more key heads than
parts, bounds and tables that are views."""
import ctypes

import pytest
import torch

from geoweave_amd import _lib
from geoweave_amd.custom_flash_attn.packed_flash_attn import packed_flash_attn_func, packed_flash_attn_inference_func
from geoweave_amd.custom_flash_attn.paged_flash_attn import paged_flash_attn_inference_func
from geoweave_amd.rotary import rotary_axes_func
from oracle.packed_attention import packed_attention, paged_attention
from test_gpu_packed_attention import check, make
from test_gpu_paged_attention import check as check_paged
from test_gpu_paged_attention import make as make_paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,hk", [(64, 2, 2), (128, 4, 1)])
@pytest.mark.parametrize("new,lens,causal", [(200, [200, 1500, 333], True), (1374, [4122], True), (600, [700, 599, 0], True),
                                             (257, [900], False)])
def test_many_new_tokens_over_a_cache(gpu_device, dtype, d, hq, hk, new, lens, causal):
    args = make_paged(lens, new, hq, hk, d, 32, dtype, 40)
    o, lse = paged_flash_attn_inference_func(*(t.to(gpu_device) for t in args), causal=causal, return_lse=True)
    check_paged(o, lse, paged_attention(*args, causal=causal), dtype, d)


@pytest.mark.parametrize("dims", [(16, 24, 24), (18, 14, 20), (64,)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rotation_over_its_input(gpu_device, dims, dtype):
    """gw_rotary_axes with y = x and the same strides."""
    dev, t, h, d = gpu_device, 333, 5, 64
    x = torch.randn(t, h, d, device=dev, dtype=dtype)
    pos = torch.randint(0, 50, (t, len(dims)), device=dev, dtype=torch.int32)
    want = rotary_axes_func(x, pos, dims, 100.0)
    lib, strides = _lib.load(), _lib.strides3(0, h * d, d)
    rc = lib.gw_rotary_axes(_lib.dtype_code(dtype, allow_fp32=True), x.data_ptr(), strides, x.data_ptr(), strides, h, None, None,
                            None, None, 0, 0, pos.data_ptr(), _lib.strides3(0, len(dims), 1), 1, t, d, len(dims),
                            (ctypes.c_int32 * len(dims))(*dims), (ctypes.c_double * len(dims))(*[100.0] * len(dims)), 0,
                            _lib.stream_handle(dev))
    _lib.check(rc, "gw_rotary_axes")
    torch.cuda.synchronize(dev)
    assert torch.equal(x, want)


@pytest.mark.parametrize("d", [64, 128])
def test_gradients_of_some_inputs_and_twice(gpu_device, d):
    args = make([130, 70], None, 4, 2, d, torch.bfloat16, 41)
    q, k, v, do = (t.to(gpu_device) for t in args[:4])
    cu = torch.tensor(args[4], dtype=torch.int32, device=gpu_device)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    o = packed_flash_attn_func(*leaves, cu, None, True)
    want = torch.autograd.grad(o, leaves, do, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(o, leaves, do)))
    for i in range(3):
        some = [x.clone().requires_grad_(j == i) for j, x in enumerate((q, k, v))]
        (got,) = torch.autograd.grad(packed_flash_attn_func(*some, cu, None, True), [some[i]], do)
        assert torch.equal(got, want[i])
    with torch.no_grad():
        assert torch.equal(packed_flash_attn_func(q, k, v, cu, None, True), o)
    # one tensor in three places: the gradients add
    x = k.clone().requires_grad_()
    (got,) = torch.autograd.grad(packed_flash_attn_func(x, x, x, cu), [x], do[:, :2])
    three = [k.clone().requires_grad_() for _ in range(3)]
    parts = torch.autograd.grad(packed_flash_attn_func(*three, cu), three, do[:, :2])
    total = sum(p.double() for p in parts)
    # the sum of three rounded terms, rounded once or twice more on the way
    assert ((got.double() - total).abs() <= 2 * 2.0 ** -8 * sum(p.double().abs() for p in parts)).all()


def test_two_streams_at_once(gpu_device):
    dev = gpu_device
    calls = []
    for seed, (lens_q, lens_k) in enumerate([([2, 3], [9000, 4000]), ([1500, 300], [1500, 300])]):
        args = make(lens_q, lens_k, 4, 2, 64, torch.float16, seed)
        q, k, v, do = (t.to(dev) for t in args[:4])
        cu_q, cu_k = (torch.tensor(c, dtype=torch.int32, device=dev) for c in args[4:])

        def call(q=q, k=k, v=v, do=do, cu_q=cu_q, cu_k=cu_k):
            leaves = [x.detach().requires_grad_() for x in (q, k, v)]
            o = packed_flash_attn_func(*leaves, cu_q, cu_k, True)
            return (o.detach(), *torch.autograd.grad(o, leaves, do))

        calls.append(call)
    want = [call() for call in calls]
    torch.cuda.synchronize(dev)
    streams = [torch.cuda.Stream(dev) for _ in calls]
    got = [[], []]
    for _ in range(5):
        for i, (s, call) in enumerate(zip(streams, calls)):
            with torch.cuda.stream(s):
                got[i].append(call())
    torch.cuda.synchronize(dev)
    for outs, ref in zip(got, want):
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, ref))


def test_more_key_heads_than_parts(gpu_device):
    """1,100 key heads: one part per head is aimed at."""
    args = make([2, 1], [700, 600], 1100, 1100, 64, torch.bfloat16, 42)
    q, k, v = (t.to(gpu_device) for t in args[:3])
    cu = [torch.tensor(c, dtype=torch.int32, device=gpu_device) for c in args[4:]]
    o, _ = packed_flash_attn_inference_func(q, k, v, *cu)
    pick = [0, 1, 550, 1099]
    ref = packed_attention(*(t[:, pick] for t in args[:3]), *args[4:], False)
    check(o[:, pick], ref, "o", torch.bfloat16, 64)


def test_bounds_lengths_and_tables_that_are_views(gpu_device):
    dev = gpu_device
    q, k, v, table, lens = (t.to(dev) for t in make_paged([300, 77], 2, 4, 2, 64, 16, torch.bfloat16, 43))
    want, _ = paged_flash_attn_inference_func(q, k, v, table, lens)
    wide = torch.zeros(2, 2 * table.shape[1] + 3, dtype=torch.int32, device=dev)
    wide[:, 3::2] = table
    many = torch.zeros(4, dtype=torch.int32, device=dev)
    many[1::2] = lens
    got, _ = paged_flash_attn_inference_func(q, k, v, wide[:, 3::2], many[1::2])
    assert torch.equal(want, got)
    args = make([40, 33], None, 4, 2, 64, torch.bfloat16, 44)
    q, k, v = (t.to(dev) for t in args[:3])
    cu = torch.tensor(args[4], dtype=torch.int32, device=dev)
    spread = torch.zeros(9, dtype=torch.int32, device=dev)
    spread[::3][:3] = cu
    want, _ = packed_flash_attn_inference_func(q, k, v, cu)
    got, _ = packed_flash_attn_inference_func(q, k, v, spread[::3][:3])
    assert torch.equal(want, got)
