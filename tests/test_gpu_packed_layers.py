"""The packed operators as the framework's layers use them: dense layers on packed batches, scenes of
different numbers of views through the aggregator, and a training step of projection, norm, rotary
positions with three axes and packed attention."""
import pytest
import torch
import torch.nn.functional as F

from geoweave_amd import aggregator as agg
from geoweave_amd.rotary import view_grid_positions
from oracle.packed_attention import rotary_axes

pytestmark = pytest.mark.gpu


def _model(indexer_layers, reuse=None, topk=32, **kw):
    torch.manual_seed(0)
    m = agg.Aggregator(dim=256, depth=4, num_heads=4, indexer_layers=indexer_layers, reuse_topk_groups=reuse,
                       topk=topk, patch_depth=2, img_size=70, **kw)
    with torch.no_grad():
        for name, p in m.named_parameters():
            if p.dim() >= 2:
                p.normal_(0.0, p.shape[-1] ** -0.5 if p.dim() == 2 else 0.02)
            elif name.endswith("gamma"):
                p.fill_(0.5)
            elif "norm" in name and name.endswith("weight"):
                p.normal_(1.0, 0.1)
            elif "w_proj" in name:
                p.fill_(1.0)
            else:
                p.normal_(0.0, 0.02)
    return m.cuda().to(torch.bfloat16)


def _close(got, want):
    """Two bf16 runs of the same layers that round at different places (other attention kernels, library
    products of other row counts). A run rounds about 14 times per block (norms, projections, rotation,
    weights, o, MLP, scales, sums) over 4 frame, 4 global and 2 patch blocks, each time by 2^-8 / sqrt(3) of
    the 2-norm of what it rounds, which is at most the residual's; independent errors of two runs then
    add to sqrt(2 * 140) * 2^-8 / sqrt(3) = 3.8e-2 of the 2-norm at most (single elements are off by more).
    Attending across a scene's bound changes the outputs by their own size."""
    assert torch.isfinite(got).all()
    assert float((got.float() - want.float()).norm() / want.float().norm()) <= 4e-2


def test_scenes_of_different_numbers_of_views(gpu_device):
    """Dense layers only: each scene's rows are those of a forward on it alone."""
    m = _model("")
    views = [3, 1, 4]
    images = torch.rand(sum(views), 3, 70, 70, generator=torch.Generator().manual_seed(2)).to(gpu_device)
    outs, start = m.forward_scenes(images, views)
    assert start == 5 and len(outs) == 4
    at = 0
    for n in views:
        want, _ = m(images[at:at + n][None])
        for a, b in zip(outs, want):
            _close(a[at:at + n], b[0])
        at += n


def test_scenes_with_sparse_layers_that_select_every_key(gpu_device):
    """Sparse layers take the scenes one by one, one of them reusing another's selection."""
    m = _model("1-3", reuse="1:2", topk=1000)
    views = [2, 3]
    images = torch.rand(sum(views), 3, 70, 70, generator=torch.Generator().manual_seed(3)).to(gpu_device)
    outs, _ = m.forward_scenes(images, views)
    at = 0
    for n in views:
        want, _ = m(images[at:at + n][None])
        for a, b in zip(outs, want):
            _close(a[at:at + n], b[0])
        at += n


def test_scene_refusals(gpu_device):
    m = _model("1-3")
    images = torch.rand(4, 3, 70, 70).to(gpu_device)
    for views in ([3], [2, 3], [4, 0], []):
        with pytest.raises(ValueError, match="views"):
            m.forward_scenes(images, views)
    with pytest.raises(NotImplementedError, match="one scene"):
        m.global_blocks[1](torch.zeros(1, 30, 256, device=gpu_device, dtype=torch.bfloat16),
                           cu_seqlens=torch.tensor([0, 30], dtype=torch.int32, device=gpu_device))


@pytest.mark.parametrize("qk_norm,rope", [(True, 100.0), (False, None)])
def test_dense_layer_on_a_packed_batch(gpu_device, qk_norm, rope):
    torch.manual_seed(1)
    layer = agg.DenseAttention(256, 4, qk_norm, rope).cuda().to(torch.bfloat16)
    lens = [70, 1, 200, 33]
    cu = torch.tensor([0, 70, 71, 271, 304], dtype=torch.int32, device=gpu_device)
    x = torch.randn(1, 304, 256, device=gpu_device, dtype=torch.bfloat16)
    pos = torch.randint(0, 15, (1, 304, 2), device=gpu_device, dtype=torch.int32)
    with torch.no_grad():
        got = layer(x, pos, 16, cu_seqlens=cu)
        at = 0
        for n in lens:
            want = layer(x[:, at:at + n].contiguous(), pos[:, at:at + n].contiguous(), 16)
            _close(got[:, at:at + n], want)
            at += n
        with pytest.raises(ValueError, match="packed batch"):
            layer(x.view(2, 152, 256), None, cu_seqlens=cu)


def _reference_layer(layer, x, pos, bounds, dims, base, causal):
    """forward_train in 64 bits on the CPU, with torch's autograd."""
    p = {n: t.detach().double().cpu().requires_grad_() for n, t in layer.named_parameters()}
    x = x.detach().double().cpu().requires_grad_()
    h, d, t = layer.num_heads, layer.head_dim, x.shape[0]
    q, k, v = F.linear(x, p["qkv.weight"], p["qkv.bias"]).view(t, 3, h, d).unbind(1)
    q = F.layer_norm(q, (d,), p["q_norm.weight"], p["q_norm.bias"])
    k = F.layer_norm(k, (d,), p["k_norm.weight"], p["k_norm.bias"])

    def turn(y):
        parts, at = [], 0
        for a, n in enumerate(dims):
            i = torch.arange(n // 2, dtype=torch.float64)
            angle = pos[:, a].double().cpu()[:, None] * base ** (-2 * i / n)
            c, s = angle.cos()[:, None], angle.sin()[:, None]
            y1, y2 = y[..., at:at + n // 2], y[..., at + n // 2:at + n]
            parts += [y1 * c - y2 * s, y2 * c + y1 * s]
            at += n
        return torch.cat(parts + [y[..., at:]], -1)

    q, k = turn(q), turn(k)
    assert torch.allclose(turn(v.detach()), rotary_axes(v.detach(), pos.cpu(), dims, [base] * len(dims)))
    outs = []
    for a, b in zip(bounds[:-1], bounds[1:]):
        s = torch.einsum("ihd,jhd->hij", q[a:b], k[a:b]) * d ** -0.5
        if causal:
            s = s.masked_fill(~torch.ones(b - a, b - a, dtype=torch.bool).tril(), float("-inf"))
        outs.append(torch.einsum("hij,jhd->ihd", s.softmax(-1), v[a:b]))
    o = torch.cat(outs).reshape(t, -1)
    return F.linear(o, p["proj.weight"], p["proj.bias"]), x, p


@pytest.mark.parametrize("causal", [False, True])
def test_training_step_of_projection_norm_rotation_and_attention(gpu_device, causal):
    """The step as a whole against 64 bits. About fourteen stages round to bf16 on the way to a gradient
    (projection, norm, rotation, weights, o, output, and their backward), each by at most 2^-8 of a value, on
    average 2^-8 / sqrt(3), and add like independent errors: 14 ** 0.5 * 2^-8 / 3 ** 0.5 = 8e-3 of the
    2-norm; norms and softmax enlarge an error a few times at most: 3e-2 for gradients, half for the
    output."""
    torch.manual_seed(2)
    layer = agg.DenseAttention(256, 4, True, 100.0).cuda()
    with torch.no_grad():
        for n, p in layer.named_parameters():
            p.normal_(0.0, 256 ** -0.5) if p.dim() == 2 else (p.normal_(1.0, 0.1) if "norm.weight" in n else p.normal_(0, 0.02))
    layer = layer.to(torch.bfloat16)
    pos = torch.cat([view_grid_positions(n, 4, 5, device=gpu_device) for n in (2, 1, 3)])
    bounds = [0, 50, 75, 150]
    cu = torch.tensor(bounds, dtype=torch.int32, device=gpu_device)
    dims = (16, 24, 24)
    x = torch.randn(150, 256, device=gpu_device, dtype=torch.bfloat16).requires_grad_()
    w = torch.randn(150, 256, device=gpu_device, dtype=torch.bfloat16)
    out = layer.forward_train(x, pos, cu, axis_dims=dims, causal=causal)
    names, params = zip(*layer.named_parameters())
    grads = dict(zip(("x",) + names, torch.autograd.grad(out, [x, *params], w)))
    ref, rx, rp = _reference_layer(layer, x, pos, bounds, dims, 100.0, causal)
    want = dict(zip(("x",) + tuple(rp), torch.autograd.grad(ref, [rx, *rp.values()], w.double().cpu())))
    rel = lambda a, b: float((a.double().cpu() - b).norm() / b.norm())  # noqa: E731
    assert rel(out.detach(), ref.detach()) <= 1.5e-2
    for n, g in grads.items():
        assert rel(g, want[n]) <= 3e-2, n


def test_one_sequence_is_the_default(gpu_device):
    torch.manual_seed(3)
    layer = agg.DenseAttention(128, 2, False, 100.0).cuda().to(torch.bfloat16)
    x = torch.randn(40, 128, device=gpu_device, dtype=torch.bfloat16)
    pos = torch.randint(0, 9, (40, 2), device=gpu_device)
    cu = torch.tensor([0, 40], dtype=torch.int32, device=gpu_device)
    assert torch.equal(layer.forward_train(x, pos), layer.forward_train(x, pos, cu))
