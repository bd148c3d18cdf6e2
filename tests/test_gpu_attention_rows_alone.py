"""A row's o, lse and dq depend, bit by bit, on its query and on what it sees alone: not on later keys, nor on the
queries of other tokens and other heads that share its tile; a key's dk and dv on the queries that see it."""
import pytest
import torch

from geoweave_amd.custom_flash_attn.packed_flash_attn import packed_flash_attn_inference_func
from geoweave_amd.custom_flash_attn.paged_flash_attn import paged_flash_attn_inference_func
from test_gpu_packed_attention import make, step
from test_gpu_paged_attention import make as make_paged

pytestmark = pytest.mark.gpu

HEADS = [(64, 4, 2), (128, 4, 1)]


def call(args, dev, causal):
    cu = [torch.tensor(c, dtype=torch.int32, device=dev) for c in args[4:]]
    return packed_flash_attn_inference_func(*(t.to(dev) for t in args[:3]), *cu, causal=causal, return_lse=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,hk", HEADS)
@pytest.mark.parametrize("lens_q,lens_k", [([700, 33], None), ([2, 5], [3000, 600]), ([150], [6000])])
@pytest.mark.parametrize("gain", [1.5, 12.0])
def test_later_keys(gpu_device, dtype, d, hq, hk, lens_q, lens_k, gain):
    args = list(make(lens_q, lens_k, hq, hk, d, dtype, 30, gain))
    n_q, n_k = args[4][1], args[5][1]
    want = call(args, gpu_device, True)
    changed = False
    for cut in sorted({1, n_q // 2, n_q - 1}):  # the first row that sees the change
        k, v = args[1].clone(), args[2].clone()
        k[cut + n_k - n_q:n_k] *= 5
        v[cut + n_k - n_q:n_k] += 3
        got = call((args[0], k, v, *args[3:]), gpu_device, True)
        for a, b in zip(want, got):
            assert torch.equal(a[:cut], b[:cut]) and torch.equal(a[n_q:], b[n_q:])
            changed |= not torch.equal(a[cut:n_q], b[cut:n_q])
    assert changed or gain > 2  # sharp rows may give the changed keys no weight


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,hk", HEADS)
@pytest.mark.parametrize("lens_q,lens_k", [([700, 33], None), ([2, 5], [3000, 600]), ([150], [6000])])
@pytest.mark.parametrize("causal", [False, True])
def test_other_queries_of_the_tile(gpu_device, dtype, d, hq, hk, lens_q, lens_k, causal):
    args = list(make(lens_q, lens_k, hq, hk, d, dtype, 31))
    want = call(args, gpu_device, causal)
    q = args[0].clone()
    q[:, 1::2] *= 9  # every second head
    q[1::3] *= 4     # every third token
    same = torch.ones(q.shape[:2], dtype=torch.bool)
    same[:, 1::2], same[1::3] = False, False
    got = call((q, *args[1:]), gpu_device, causal)
    for a, b in zip(want, got):
        assert torch.equal(a[same], b[same]) and not torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,hk", HEADS)
def test_new_tokens_over_a_cache(gpu_device, dtype, d, hq, hk):
    q, k, v, table, lens = make_paged([900, 40], 6, hq, hk, d, 16, dtype, 32)
    call = lambda q, k: paged_flash_attn_inference_func(  # noqa: E731
        *(t.to(gpu_device) for t in (q, k, v, table, lens)), return_lse=True)
    want = call(q, k)
    far = k.clone()
    for j in range(897, 900):  # seen by the last three new tokens
        far[table[0, j // 16], j % 16] *= 20
    for a, b in zip(want, call(q, far)):
        assert torch.equal(a[0, :3], b[0, :3]) and torch.equal(a[1], b[1]) and not torch.equal(a[0], b[0])
    loud = q.clone()
    loud[:, 1::2] *= 9
    for a, b in zip(want, call(loud, k)):
        assert torch.equal(a[:, ::2], b[:, ::2]) and not torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,hk", HEADS)
@pytest.mark.parametrize("lens_q,lens_k", [([700, 33], None), ([150], [6000]), ([5], [900])])
def test_gradients(gpu_device, dtype, d, hq, hk, lens_q, lens_k):
    args = make(lens_q, lens_k, hq, hk, d, dtype, 33)
    n_q, n_k = args[4][1], args[5][1]
    shift, cut = n_k - n_q, n_q // 2
    _, dq, dk, dv = step(args, gpu_device, True)
    q, k, v, do, cu_q, cu_k = (t.clone() if torch.is_tensor(t) else t for t in args)
    k[cut + shift:n_k] *= 5
    v[cut + shift:n_k] += 3
    _, dq2, _, _ = step((q, k, v, do, cu_q, cu_k), gpu_device, True)
    assert torch.equal(dq[:cut], dq2[:cut]) and torch.equal(dq[n_q:], dq2[n_q:]) and not torch.equal(dq, dq2)
    q, k, v, do, cu_q, cu_k = (t.clone() if torch.is_tensor(t) else t for t in args)
    q[:cut] *= 4
    do[:cut] -= 2
    _, _, dk2, dv2 = step((q, k, v, do, cu_q, cu_k), gpu_device, True)
    first = cut + shift  # the first key that none of those queries sees
    for a, b in ((dk, dk2), (dv, dv2)):
        assert torch.equal(a[first:], b[first:]) and not torch.equal(a, b)
