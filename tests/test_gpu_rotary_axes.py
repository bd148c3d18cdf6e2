"""Rotary positions with several axes (gw_rotary_axes) against the 64-bit oracle.

A turned element x1 cos - x2 sin is two fp32 products and one fp32 sum of a cosine and a sine
rounded to fp32: off by at most 4 2^-24 (|x1| + |x2|), and rounded once more to the output's type (half a
step, and for fp16 at least half of its fixed step of 2^-24)."""
import pytest
import torch

from geoweave_amd import dsa_layer
from geoweave_amd.rotary import rotary_axes_func, rotary_axes_qk_func, view_grid_positions
from oracle.packed_attention import rotary_axes

pytestmark = pytest.mark.gpu


def check(got, x, pos, dims, bases, sign=1.0):
    x, pos = x.cpu(), pos.cpu()
    ref = rotary_axes(x, pos, dims, bases, sign)
    size = rotary_axes(x.abs(), torch.zeros_like(pos), dims, bases)
    at = 0
    mag = size.clone()
    for n in dims:  # |x1| + |x2| of every pair
        half = n // 2
        both = size[..., at:at + half] + size[..., at + half:at + n]
        mag[..., at:at + half], mag[..., at + half:at + n] = both, both
        at += n
    lim = torch.finfo(x.dtype).eps / 2 * 1.01 * ref.abs() + 4 * 2.0 ** -24 * mag + (2.0 ** -25 if x.dtype == torch.float16 else 0)
    err = (got.double().cpu() - ref).abs()
    assert (err <= lim).all(), float((err / lim.clamp_min(1e-300)).max())
    assert torch.equal(got.cpu()[..., at:], x[..., at:])


CASES = [
    (1, 1, 1, 64, (64,), 40),
    (77, 3, 2, 64, (16, 24, 24), 40),
    (301, 16, 4, 128, (32, 48, 48), 100000),
    (50, 5, 5, 80, (18, 14, 20, 20), 1000000),
    (33, 2, 2, 96, (10, 22), 500),
    (9, 2, 1, 256, (128, 128), 64),
    (1500, 7, 1, 34, (2, 4, 6, 0, 8), 3000000),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("pos_dtype", [torch.int32, torch.int64, torch.float32])
@pytest.mark.parametrize("t,h,hk,d,dims,far", CASES)
def test_values_and_gradients(gpu_device, dtype, pos_dtype, t, h, hk, d, dims, far):
    g = torch.Generator().manual_seed(t)
    q, k = torch.randn(t, h, d, generator=g).to(dtype), torch.randn(t, hk, d, generator=g).to(dtype)
    dq, dk = torch.randn(t, h, d, generator=g).to(dtype), torch.randn(t, hk, d, generator=g).to(dtype)
    pos = torch.randint(-far, far, (t, len(dims)), generator=g).to(pos_dtype)
    bases = [10000.0, 100.0, 50.0, 7.5, 1e6][:len(dims)]
    a, b = q.to(gpu_device).requires_grad_(), k.to(gpu_device).requires_grad_()
    yq, yk = rotary_axes_qk_func(a, b, pos.to(gpu_device), dims, bases)
    check(yq.detach(), q, pos, dims, bases)
    check(yk.detach(), k, pos, dims, bases)
    gq, gk = torch.autograd.grad([yq, yk], [a, b], [dq.to(gpu_device), dk.to(gpu_device)])
    check(gq, dq, pos, dims, bases, -1.0)
    check(gk, dk, pos, dims, bases, -1.0)
    assert torch.equal(rotary_axes_func(a, pos.to(gpu_device), dims, bases), yq)


def test_two_axes_are_the_layer_glue_rotation(gpu_device):
    """Half the head per axis, base 100 and (row, column): the rotation of dsa_glue_forward."""
    dev, h = gpu_device, 4
    pos = dsa_layer.grid_positions(2, 9, 7, device=dev).reshape(1, -1, 2)
    n = pos.shape[1]
    layout = dsa_layer.GlueLayout(h, 64, 0, 64)
    y = torch.randn(1, n, layout.ldy, device=dev, dtype=torch.bfloat16)
    q, k, _, _, _, _ = dsa_layer.dsa_glue_forward(y, layout, pos=pos, rope_base=100.0, rope_len=16)
    yq, yk = rotary_axes_qk_func(y[..., :h * 64].view(1, n, h, 64), y[..., h * 64:2 * h * 64].view(1, n, h, 64), pos,
                                 (32, 32), 100.0)
    # The glue's angles are fp32 (a position of at most 15 keeps them to 2^-20, an element of at most 6
    # to 2^-16). Each side then rounds once, by half a step (2^-8 of its value) at most, so two values
    # next to a border lie a whole step (2^-7) apart.
    for a, b in ((q, yq), (k, yk)):
        assert ((a.float() - b.float()).abs() <= 2 * 1.01 * 2.0 ** -8 * a.float().abs() + 2.0 ** -16).all()


def test_views_positions(gpu_device):
    pos = view_grid_positions(3, 4, 5, device=gpu_device, first_view=2)
    assert pos.shape == (3 * 25, 3)
    two = dsa_layer.grid_positions(3, 4, 5, device=gpu_device).reshape(-1, 2)
    assert torch.equal(pos[:, 1:], two)
    assert pos[:, 0].tolist() == [2] * 25 + [3] * 25 + [4] * 25


def test_batches_strides_and_shared_positions(gpu_device):
    dev, b, t, h, d = gpu_device, 3, 41, 4, 64
    dims, bases = (16, 24, 24), [100.0] * 3
    y = torch.randn(b, t, 3 * h * d + 2, device=dev, dtype=torch.bfloat16)
    q, k = y[..., :h * d].view(b, t, h, d), y[..., h * d + 2:2 * h * d + 2].view(b, t, h, d)
    pos = torch.randint(0, 40, (b, t, 3), device=dev)
    yq, yk = rotary_axes_qk_func(q, k, pos, dims, bases)
    check(yq, q, pos, dims, bases)
    check(yk, k, pos, dims, bases)
    shared = rotary_axes_func(q, pos[1], dims, bases)
    assert torch.equal(shared[1], yq[1])
    odd = torch.randn(t, d + 1, h, device=dev, dtype=torch.float16).transpose(1, 2)[..., 1:]  # last stride not 1
    check(rotary_axes_func(odd, pos[0], dims, bases), odd, pos[0], dims, bases)
    cols = torch.randint(0, 40, (3, t), device=dev).t()  # positions axis-major in memory
    check(rotary_axes_func(q[0], cols, dims, bases), q[0], cols, dims, bases)
    # one head broadcast: the gradient is summed over the heads
    one = torch.randn(t, 1, d, device=dev, dtype=torch.float32).requires_grad_()
    out = rotary_axes_func(one.expand(t, h, d), pos[0], dims, bases)
    (grad,) = torch.autograd.grad(out, one, torch.ones_like(out))
    want = rotary_axes(torch.ones(t, 1, d), pos[0].cpu(), dims, bases, -1.0) * h
    assert (grad.double().cpu() - want).abs().max() < 1e-5


def test_empty_and_one_gradient_only(gpu_device):
    dev = gpu_device
    e = torch.empty(0, 4, 64, device=dev, dtype=torch.bfloat16)
    assert rotary_axes_func(e, torch.empty(0, 1, device=dev, dtype=torch.int32), [64]).shape == e.shape
    q = torch.randn(5, 2, 64, device=dev).requires_grad_()
    k = torch.randn(5, 1, 64, device=dev).requires_grad_()
    pos = torch.arange(5, device=dev)[:, None]
    yq, yk = rotary_axes_qk_func(q, k, pos, [64], 100.0)
    (gk,) = torch.autograd.grad(yk.sum(), [k])
    check(gk, torch.ones(5, 1, 64), pos, [64], [100.0], -1.0)


def test_replays_follow_the_positions(gpu_device):
    dev = gpu_device
    q = torch.randn(64, 4, 64, device=dev, dtype=torch.bfloat16)
    pos = torch.zeros(64, 2, device=dev, dtype=torch.int32)
    rotary_axes_func(q, pos, (32, 32))
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rotary_axes_func(q, pos, (32, 32))
    for i in range(3):
        pos.copy_(torch.randint(0, 50, pos.shape, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize(dev)
        assert torch.equal(y, rotary_axes_func(q, pos, (32, 32)))
    # position 0 leaves every bit
    pos.zero_()
    assert torch.equal(rotary_axes_func(q, pos, (32, 32)), q)
