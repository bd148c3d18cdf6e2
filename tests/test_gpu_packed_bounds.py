"""The backward on bounds that are out of order or outside the tensors: values are unspecified, and nothing else is
touched (the arithmetic of every index is checked in test_packed_bounds_model). Afterwards an ordinary call gives its
bits, and a graph captured with ordinary bounds comes back to them."""
import pytest
import torch

from geoweave_amd.custom_flash_attn.packed_flash_attn import packed_flash_attn_func

pytestmark = pytest.mark.gpu

WILD = [[0, 150, 50, 200], [-7, 90, 1 << 30, 5], [300, 300, 300, 300], [200, 100, 50, 0], [-(1 << 31), 0, (1 << 31) - 1, 7]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,hk", [(64, 2, 2), (64, 6, 1), (128, 4, 2)])
@pytest.mark.parametrize("causal", [False, True])
def test_backward_of_bounds_out_of_order(gpu_device, dtype, d, hq, hk, causal):
    dev, t = gpu_device, 200
    g = torch.Generator().manual_seed(d)
    q, do = (torch.randn(t, hq, d, generator=g).to(dev, dtype) for _ in range(2))
    k, v = (torch.randn(t, hk, d, generator=g).to(dev, dtype) for _ in range(2))
    cu_q = torch.tensor([0, 10, 128, 200], dtype=torch.int32, device=dev)
    cu_k = cu_q.clone()

    def call():
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        o = packed_flash_attn_func(*leaves, cu_q, cu_k, causal)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    want = call()
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = call()
    inputs = [x.clone() for x in (q, k, v, do)]
    for a in WILD:
        for b in ([0, 10, 128, 200], a, a[::-1]):
            cu_q.copy_(torch.tensor(a, dtype=torch.int32))
            cu_k.copy_(torch.tensor(b, dtype=torch.int32))
            for x, like in zip(call(), (q, q, k, v)):
                assert x.shape == like.shape
            graph.replay()
            torch.cuda.synchronize(dev)
    assert all(torch.equal(x, y) for x, y in zip(inputs, (q, k, v, do)))
    for cu in (cu_q, cu_k):
        cu.copy_(torch.tensor([0, 10, 128, 200], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize(dev)
    assert all(torch.equal(x, y) for x, y in zip(want, captured))
    assert all(torch.equal(x, y) for x, y in zip(want, call()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_backward_of_many_sequences_out_of_order(gpu_device, dtype):
    """More tiles than the lists have room for, and cut loops."""
    dev, t, n = gpu_device, 3000, 400
    g = torch.Generator().manual_seed(3)
    q, k, v, do = (torch.randn(t, 4, 64, generator=g).to(dev, dtype) for _ in range(4))
    for cu in (torch.randint(0, t, (n + 1,), generator=g), torch.tensor([0, t] * (n // 2) + [0])):
        cu = cu.to(dev, torch.int32)
        for causal in (False, True):
            leaves = [x.detach().requires_grad_() for x in (q, k, v)]
            grads = torch.autograd.grad(packed_flash_attn_func(*leaves, cu, None, causal), leaves, do)
            torch.cuda.synchronize(dev)
            assert all(x.shape == y.shape for x, y in zip(grads, leaves))
