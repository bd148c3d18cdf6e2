"""Packed attention (gw_packed_attn_fwd / gw_packed_attn_bwd) against the 64-bit oracle.

Tolerances, with u = eps / 2 of the 16-bit type (half a step): the weights P (relative to the row's
sum, which adds them unrounded) and dS are rounded once before their products and every output
once; sums are fp32, delta comes from the unrounded o. Hence, per element and with the oracle's sums of
magnitudes, |o error| <= u (|o| + P|V|), |dv error| <= u (|dv| + P^T|dO|), |dq error| <= u (|dq| + scale
P(|dP| + |o||dO|) |K|), dk the same with Q. A score's fp32 sum of D products is off
by at most D 2^-24 of its terms' magnitudes, which changes a weight by that relative amount (twice, with the
lse); the fp32 sums over keys and the exp2 add less than 2^-18 of the magnitudes."""
import math

import pytest
import torch

from geoweave_amd.custom_flash_attn.packed_flash_attn import packed_flash_attn_func, packed_flash_attn_inference_func
from oracle.packed_attention import packed_attention

pytestmark = pytest.mark.gpu

LENS = {
    "one": ([1], [1]),
    "odd": ([1, 0, 5, 64, 65, 127, 128, 129, 300], None),
    "two sides": ([5, 0, 3, 130, 1, 70], [0, 7, 64, 130, 700, 33]),
    "tiles": ([256, 513, 31], None),
    "few rows": ([3, 1, 40, 0, 2, 17], [2000, 777, 1500, 600, 33, 1300]),
    "few rows only": ([2], [2700]),
    "keys split": ([140, 150], [5000, 1201]),
    "queries split": ([2500, 1700, 0], [40, 90, 3]),
}


def _cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def make(lens_q, lens_k, hq, hk, d, dtype, seed=0, gain=1.5):
    g = torch.Generator().manual_seed(seed)
    cu_q, cu_k = _cu(lens_q), _cu(lens_k if lens_k is not None else lens_q)
    q = (torch.randn(cu_q[-1], hq, d, generator=g) * gain).to(dtype)
    k, v = (torch.randn(cu_k[-1], hk, d, generator=g).to(dtype) for _ in range(2))
    do = torch.randn(cu_q[-1], hq, d, generator=g).to(dtype)
    return q, k, v, do, cu_q, cu_k


def bound(ref, name, dtype, d, times):
    u = torch.finfo(dtype).eps / 2
    s = 2 * d * 2.0 ** -24 * float(ref["s_mag"].max()) + 2.0 ** -18
    # the smallest normal step of fp16, below which P and dS are rounded to a fixed one
    floor = 2.0 ** -20 if dtype == torch.float16 else 2.0 ** -60
    return (u * 1.01) * ref[name].abs() + (times * u + 4 * s) * ref[name + "_mag"] + floor


def check(got, ref, name, dtype, d, times=1):
    err = (got.double().cpu() - ref[name]).abs()
    lim = bound(ref, name, dtype, d, times)
    assert torch.isfinite(got).all(), name
    worst = (err / lim).max() if err.numel() else torch.zeros(())
    assert worst <= 1.0, f"{name}: {float(worst):.2f} of the bound, largest error {float(err.max()):.3g}"


def part(ref, name, rows):
    """The oracle's ``name`` of some rows."""
    return {"s_mag": ref["s_mag"], name: ref[name][rows], name + "_mag": ref[name + "_mag"][rows]}


def check_lse(lse, ref):
    a, b = lse.double().cpu(), ref["lse"]
    assert torch.equal(a == -math.inf, b == -math.inf)
    on = b != -math.inf
    assert ((a - b)[on].abs() <= 2.0 ** -17 * (1 + ref["s_mag"][on])).all()


def step(args, dev, causal, scale=None):
    q, k, v, do, cu_q, cu_k = args
    q, k, v = (t.to(dev).requires_grad_() for t in (q, k, v))
    cq, ck = (torch.tensor(c, dtype=torch.int32, device=dev) for c in (cu_q, cu_k))
    o = packed_flash_attn_func(q, k, v, cq, ck, causal, scale)
    return (o.detach(), *torch.autograd.grad(o, [q, k, v], do.to(dev)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,hk", [(64, 2, 2), (64, 6, 2), (128, 4, 1), (80, 3, 3), (17, 2, 1)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens", list(LENS))
def test_forward_and_gradients(gpu_device, dtype, d, hq, hk, causal, lens):
    args = make(*LENS[lens], hq, hk, d, dtype)
    ref = packed_attention(*args[:3], args[4], args[5], causal, do=args[3])
    o, dq, dk, dv = step(args, gpu_device, causal)
    q, k, v = (t.to(gpu_device) for t in args[:3])
    cq, ck = (torch.tensor(c, dtype=torch.int32, device=gpu_device) for c in args[4:])
    o2, lse = packed_flash_attn_inference_func(q, k, v, cq, ck, causal=causal, return_lse=True)
    assert torch.equal(o, o2)
    check(o, ref, "o", dtype, d)
    check_lse(lse, ref)
    check(dv, ref, "dv", dtype, d)
    check(dq, ref, "dq", dtype, d)
    check(dk, ref, "dk", dtype, d)
    again = step(args, gpu_device, causal)
    assert all(torch.equal(a, b) for a, b in zip((o, dq, dk, dv), again)), "the same inputs give the same bits"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_one_long_sequence_among_short_ones(gpu_device, dtype, d, causal):
    """The long one's loops are cut into parts, the others' are not."""
    args = make([3, 1500, 40, 0, 17, 1], None, 6, 1, d, dtype, seed=4)
    q, k, v, do, cu_q, cu_k = args
    got = step(args, gpu_device, causal)
    ref = packed_attention(q, k, v, cu_q, cu_k, causal, do=do)
    for name, x in zip(("o", "dq", "dk", "dv"), got):
        check(x, ref, name, dtype, d)
    assert all(torch.equal(a, b) for a, b in zip(got, step(args, gpu_device, causal))), "the same bits again"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_long_rows_with_rising_scores(gpu_device, dtype):
    """Scores that grow along the keys move the running reference many times."""
    args = list(make([40, 7], [2100, 3], 2, 1, 64, dtype, 3))
    ramp = torch.linspace(0.1, 6.0, 2103)[:, None, None]
    args[1] = (args[1].float() * ramp).to(dtype)
    ref = packed_attention(*args[:3], args[4], args[5], False, do=args[3])
    o, dq, dk, dv = step(args, gpu_device, False)
    check(o, ref, "o", dtype, 64)
    check(dv, ref, "dv", dtype, 64)
    check(dq, ref, "dq", dtype, 64)
    check(dk, ref, "dk", dtype, 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
def test_rows_that_see_one_key_pass_no_gradient_to_scores(gpu_device, dtype, causal):
    args = make([3, 1, 200, 1], [1, 1, 200, 700], 4, 2, 64, dtype, 10)
    _, dq, dk, _ = step(args, gpu_device, causal)
    rows = [0, 1, 2, 3] + ([4] if causal else [])
    assert (dq[rows] == 0).all() and (dk[:2] == 0).all()
    assert (dq[204] != 0).any() and (dk[5] != 0).any()


def test_small_gradients_in_fp16(gpu_device):
    """Gradients of a mean over many tokens: dO of 2^-12, weights of 2^-11."""
    args = list(make([33, 900], [2000, 900], 2, 2, 64, torch.float16, 4, gain=0.3))
    args[3] = (args[3].float() * 2.0 ** -12).to(torch.float16)
    ref = packed_attention(*args[:3], args[4], args[5], False, do=args[3])
    o, dq, dk, dv = step(args, gpu_device, False)
    for name, got, times in (("dv", dv, 1), ("dq", dq, 1), ("dk", dk, 1)):
        u = 2.0 ** -11
        # outputs below fp16's normal range are rounded to its fixed step of 2^-24
        lim = u * 1.01 * ref[name].abs() + (times * u + 2.0 ** -16) * ref[name + "_mag"] + 2.0 ** -25
        assert ((got.double().cpu() - ref[name]).abs() <= lim).all(), name


@pytest.mark.parametrize("causal", [False, True])
def test_tokens_behind_the_last_bound_and_between(gpu_device, causal):
    """Tokens of no sequence hold inf and NaN: zeros come out for them, and nothing of them anywhere."""
    q, k, v, do, cu_q, cu_k = make([70, 33, 20], [45, 60, 90], 2, 2, 64, torch.bfloat16, 5)
    ref = packed_attention(q, k, v, cu_q[:3], cu_k[:3], causal, do=do)
    for t, end in ((q, 103), (do, 103), (k, 105), (v, 105)):
        t[end:] = math.nan
    k[110:], v[108:] = math.inf, -math.inf
    args = (q, k, v, do, cu_q[:3], cu_k[:3])
    o, dq, dk, dv = step(args, gpu_device, causal)
    for name, got, times in (("o", o, 1), ("dq", dq, 1)):
        assert (got[103:] == 0).all()
        check(got[:103], part(ref, name, slice(103)), name, torch.bfloat16, 64, times)
    for name, got, times in (("dk", dk, 1), ("dv", dv, 1)):
        assert (got[105:] == 0).all()
        check(got[:105], part(ref, name, slice(105)), name, torch.bfloat16, 64, times)


def test_a_sequence_with_nan_leaves_the_others_alone(gpu_device):
    args = make([65, 40, 130], None, 4, 2, 64, torch.float16, 6)
    clean = step(args, gpu_device, False)
    for t in args[:4]:
        t[70:75] = math.nan
    out = step(args, gpu_device, False)
    for a, b in zip(clean, out):
        assert torch.equal(a[:65], b[:65]) and torch.equal(a[105:], b[105:])
        assert b[65:105].isnan().any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,hk", [(64, 2, 2), (128, 4, 2)])
@pytest.mark.parametrize("lens_q,lens_k", [([300, 77], None), ([9, 3], [1500, 800]), ([200], [3300])])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_a_causal_row_does_not_see(gpu_device, dtype, d, hq, hk, lens_q, lens_k, value):
    """inf and NaN in later values change no bit of the rows before them, and reach those behind; in a
    query's q and dO they change no bit of the gradients of the keys that it does not see."""
    args = make(lens_q, lens_k, hq, hk, d, dtype, 11)
    ref = packed_attention(*args[:3], args[4], args[5], True, do=args[3])
    clean = step(args, gpu_device, True)
    n_q, n_k = lens_q[0], (lens_k or lens_q)[0]
    shift = n_k - n_q
    for cut in (1, n_q // 2, n_q - 1):  # the first query that sees what is planted
        q, k, v, do, cu_q, cu_k = (t.clone() if torch.is_tensor(t) else t for t in args)
        v[cut + shift, 0, 5] = value
        out = step((q, k, v, do, cu_q, cu_k), gpu_device, True)
        for a, b in zip(clean[:2], out[:2]):
            assert torch.equal(a[:cut], b[:cut]) and torch.equal(a[n_q:], b[n_q:])
        assert not torch.isfinite(out[0][cut:n_q, 0, 5]).any()
        if value == value:
            assert (out[0][cut:n_q, 0, 5] == value).all()
        # A key: the rows of a block raise their running reference together, so rows beside one that sees
        # the key are rounded otherwise, within the bounds.
        k[cut + shift] = value
        out = step((q, k, v, do, cu_q, cu_k), gpu_device, True)
        for name, got, times in (("o", out[0], 1), ("dq", out[1], 1)):
            check(got[:cut], part(ref, name, slice(cut)), name, dtype, d, times)
            check(got[n_q:], part(ref, name, slice(n_q, None)), name, dtype, d, times)
        q, k, v, do, cu_q, cu_k = (t.clone() if torch.is_tensor(t) else t for t in args)
        do[cut - 1, :, 3] = value
        out = step((q, k, v, do, cu_q, cu_k), gpu_device, True)
        for a, b in zip(clean, out):
            if a.shape[0] == cu_k[-1] and a.shape[1] == hk:
                assert torch.equal(a[cut + shift:], b[cut + shift:])
        assert not torch.isfinite(out[3][:cut + shift, :, 3]).any()
        q[cut - 1] = value
        out = step((q, k, v, do, cu_q, cu_k), gpu_device, True)
        for name, got, times in (("dk", out[2], 1), ("dv", out[3], 1)):
            check(got[cut + shift:], part(ref, name, slice(cut + shift, None)), name, dtype, d, times)


def test_strides_layouts_and_broadcast_heads(gpu_device):
    dev, t, h, d = gpu_device, 333, 4, 64
    cu = torch.tensor([0, 100, 101, 333], dtype=torch.int32, device=dev)
    y = torch.randn(t, 3 * h * d + 8, device=dev, dtype=torch.bfloat16)
    q, k, v = (y[:, i * h * d:(i + 1) * h * d].view(t, h, d) for i in range(3))
    want, _ = packed_flash_attn_inference_func(q.contiguous(), k.contiguous(), v.contiguous(), cu, causal=True)
    got, _ = packed_flash_attn_inference_func(q, k, v, cu, causal=True)
    assert torch.equal(want, got)
    qh = q.transpose(0, 1).contiguous().transpose(0, 1)  # [H, T, D] in memory
    got, _ = packed_flash_attn_inference_func(qh, k, v, cu, causal=True)
    assert torch.equal(want, got)
    odd = torch.randn(t, h, d + 1, device=dev, dtype=torch.bfloat16)[..., 1:]  # rows that are not 16-byte aligned
    want, _ = packed_flash_attn_inference_func(odd.contiguous(), k, v, cu)
    got, _ = packed_flash_attn_inference_func(odd, k, v, cu)
    assert torch.equal(want, got)
    # one key head for all: as Hk = 1 and as a broadcast view, whose gradient is summed over the heads
    k1 = k[:, :1].detach().contiguous().requires_grad_()
    do = torch.randn(t, h, d, device=dev, dtype=torch.bfloat16)
    o1 = packed_flash_attn_func(q.detach(), k1, k1, cu)
    o2 = packed_flash_attn_func(q.detach(), k1.expand(t, h, d), k1.expand(t, h, d), cu)
    assert torch.equal(o1, o2)
    (g1,), (g2,) = torch.autograd.grad(o1, [k1], do), torch.autograd.grad(o2, [k1], do)
    torch.testing.assert_close(g1.float(), g2.float(), atol=0.1, rtol=0.05)  # sums of four rounded terms each


def test_broadcast_tokens(gpu_device):
    """Tensors whose tokens are one row of memory, forward and backward."""
    dev, t = gpu_device, 150
    cu = torch.tensor([0, 70, 150], dtype=torch.int32, device=dev)
    base = [torch.randn(1, 2, 64, device=dev, dtype=torch.bfloat16) for _ in range(4)]
    full = [torch.randn(t, 2, 64, device=dev, dtype=torch.bfloat16) for _ in range(4)]
    for i in range(4):  # q, k, v or dO broadcast
        wide = [x.expand(t, 2, 64) if j == i else full[j] for j, x in enumerate(base)]
        outs = []
        for args in (wide, [x.contiguous() for x in wide]):
            leaves = [x.detach().requires_grad_() for x in args[:3]]
            o = packed_flash_attn_func(*leaves, cu, None, True)
            outs.append((o, *torch.autograd.grad(o, leaves, args[3])))
        assert all(torch.equal(a, b) for a, b in zip(*outs)), i


def test_single_tokens_and_tensors_that_start_anywhere(gpu_device):
    """Dims of one entry keep whatever stride they had, and a contiguous tensor may start at any element."""
    dev = gpu_device
    cu = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    y = torch.randn(128, device=dev, dtype=torch.bfloat16)
    one = y.as_strided((1, 2, 64), (5, 64, 1))
    assert one.stride(0) % 8 and one.is_contiguous()
    o, _ = packed_flash_attn_inference_func(one, one, one, cu)
    assert torch.equal(o, one)
    flat = torch.randn(3 + 40 * 2 * 64, device=dev, dtype=torch.bfloat16)
    off = flat[3:].view(40, 2, 64)
    cu = torch.tensor([0, 11, 40], dtype=torch.int32, device=dev)
    want, _ = packed_flash_attn_inference_func(off.clone(), off.clone(), off.clone(), cu, causal=True)
    got, _ = packed_flash_attn_inference_func(off, off, off, cu, causal=True)
    assert torch.equal(want, got)
    leaf = off.detach().requires_grad_()
    out = packed_flash_attn_func(leaf, leaf, leaf, cu)
    (g1,) = torch.autograd.grad(out.sum(), leaf)  # a gradient without strides
    leaf2 = off.clone().requires_grad_()
    (g2,) = torch.autograd.grad(packed_flash_attn_func(leaf2, leaf2, leaf2, cu).sum(), leaf2)
    assert torch.equal(g1, g2)


def test_no_sequences_and_no_tokens(gpu_device):
    dev = gpu_device
    for tq, tk, bounds in ((5, 1000, [0]), (300, 7, [0]), (40, 900, [0, 0, 0]), (0, 9, [0, 0]), (6, 0, [0, 0])):
        q = torch.full((tq, 2, 64), float("nan"), device=dev, dtype=torch.bfloat16).requires_grad_()
        k = torch.full((tk, 1, 64), float("nan"), device=dev, dtype=torch.bfloat16).requires_grad_()
        cu = torch.tensor(bounds, dtype=torch.int32, device=dev)
        o = packed_flash_attn_func(q, k, k, cu, cu)
        assert o.shape == q.shape and (o == 0).all()
        _, lse = packed_flash_attn_inference_func(q, k, k, cu, cu, return_lse=True)
        assert (lse == -math.inf).all()
        gq, gk = torch.autograd.grad(o, [q, k], torch.ones_like(o))
        assert (gq == 0).all() and (gk == 0).all()


def test_offsets_past_32_bits(gpu_device):
    """Key rows 2^20 elements apart: the last lie more than 2^32 bytes behind the first."""
    dev, n, d = gpu_device, 2600, 64
    room = torch.empty((n - 1) * (1 << 20) + 2 * d, device=dev, dtype=torch.bfloat16)
    far = room.as_strided((n, 2, d), (1 << 20, d, 1))
    near = torch.randn(n, 2, d, device=dev, dtype=torch.bfloat16)
    far.copy_(near)
    q = torch.randn(50, 2, d, device=dev, dtype=torch.bfloat16)
    cq, ck = (torch.tensor([0, 20, m], dtype=torch.int32, device=dev) for m in (50, n))
    want, _ = packed_flash_attn_inference_func(q, near, near, cq, ck)
    got, _ = packed_flash_attn_inference_func(q, far, far, cq, ck)
    assert torch.equal(want, got)
    outs = []
    for k in (near, far):
        k = k.detach().requires_grad_()
        outs.append(torch.autograd.grad(packed_flash_attn_func(q, k, k, cq, ck), [k], q)[0])
    assert torch.equal(*outs)


def test_graph_replays_with_other_bounds_and_on_a_side_stream(gpu_device):
    dev, t = gpu_device, 400
    q, k, v, do = (torch.randn(t, 4, 64, device=dev, dtype=torch.float16) for _ in range(4))
    cu = torch.tensor([0, 10, 300, 400], dtype=torch.int32, device=dev)

    def both():
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        o = packed_flash_attn_func(*leaves, cu, None, True)
        return (o, *torch.autograd.grad(o, leaves, do))

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        eager_side = [x.clone() for x in both()]
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize(dev)
    assert all(torch.equal(a, b) for a, b in zip(eager_side, both()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = both()
    for bounds in ([0, 10, 300, 400], [0, 0, 1, 400], [0, 128, 256, 384], [0, 400, 400, 400]):
        cu.copy_(torch.tensor(bounds, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize(dev)
        got = [x.clone() for x in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, both())), bounds
        q.copy_(torch.randn_like(q))


def test_many_sequences(gpu_device):
    """More sequences than one round of the search holds, most of them empty or one token."""
    dev, n = gpu_device, 5000
    lens = torch.randint(0, 3, (n,), generator=torch.Generator().manual_seed(7))
    lens[4000] = 700
    cu = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)]).to(torch.int32)
    t = int(cu[-1])
    q, k, v, do = (torch.randn(t, 1, 64).bfloat16() for _ in range(4))
    ref = packed_attention(q, k, v, cu, cu, True, do=do)
    o, dq, dk, dv = step((q, k, v, do, cu.tolist(), cu.tolist()), dev, True)
    check(o, ref, "o", torch.bfloat16, 64)
    check(dv, ref, "dv", torch.bfloat16, 64)
    check(dq, ref, "dq", torch.bfloat16, 64)
    check(dk, ref, "dk", torch.bfloat16, 64)


def test_bounds_that_are_not_in_order_stay_in_the_tensors(gpu_device):
    dev = gpu_device
    q, k, v = (torch.randn(200, 2, 64, device=dev, dtype=torch.bfloat16) for _ in range(3))
    for bounds in ([0, 150, 50, 200], [-7, 90, 1 << 30, 5], [300, 300, 300, 300]):
        cu = torch.tensor(bounds, dtype=torch.int32, device=dev)
        o, _ = packed_flash_attn_inference_func(q, k, v, cu)
        torch.cuda.synchronize(dev)
        assert o.shape == q.shape


def test_bounds_out_of_order_over_few_rows(gpu_device):
    """Bounds that run back name more tiles of few rows than the call has workgroups: every access stays in the
    workspace."""
    dev, t, n, h = gpu_device, 400, 900, 16
    back = torch.tensor([0] + [17 * (i % 21) for i in range(n - 1)] + [t], dtype=torch.int32, device=dev)
    q = torch.randn(t, h, 64, device=dev, dtype=torch.bfloat16)
    k, v = (torch.randn(n * 512 + 600, 1, 64, device=dev, dtype=torch.bfloat16) for _ in range(2))
    cu_k = torch.arange(n + 1, dtype=torch.int32, device=dev) * 512
    cu_k[-1] += 600
    heads = [x.expand(-1, h, -1) for x in (k, v)]
    for _ in range(2):
        o, lse = packed_flash_attn_inference_func(q, *heads, back, cu_k, return_lse=True)
        torch.cuda.synchronize(dev)
        assert o.shape == q.shape and lse.shape == (t, h)
    # in order again: the values of an ordinary call
    ordered = torch.arange(n + 1, device=dev).clamp(max=t).to(torch.int32)
    o, _ = packed_flash_attn_inference_func(q, *heads, ordered, cu_k)
    for i in (0, h - 1):
        ref = packed_attention(q[:, i:i + 1].cpu(), k.cpu(), v.cpu(), ordered.cpu(), cu_k.cpu(), False)
        check(o[:, i:i + 1], ref, "o", torch.bfloat16, 64)


def test_gradients_against_differences(gpu_device):
    """The directional derivative of sum(o w) by central differences of the 64-bit oracle."""
    args = make([20, 45], [33, 45], 4, 2, 64, torch.bfloat16, 8)
    _, dq, dk, dv = step(args, gpu_device, True)
    g = torch.Generator().manual_seed(9)
    q, k, v, do, cu_q, cu_k = args
    f = lambda a, b, c: float((packed_attention(a, b, c, cu_q, cu_k, True)["o"] * do.double()).sum())  # noqa: E731
    for i, grad in enumerate((dq, dk, dv)):
        base = [q.double(), k.double(), v.double()]
        r = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + 1e-5 * r, base[i] - 1e-5 * r
        want = (f(*up) - f(*down)) / 2e-5
        got = float((grad.double().cpu() * r).sum())
        # each of the n terms is off by about 2^-8 of its size, with signs that do not agree
        assert abs(got - want) <= 4 * 2.0 ** -8 * float((grad.double().cpu() * r).norm()) + 1e-3
