"""Gradients beside outliers: a row with a large dO and a key with a large value leave the gradients of what does
not see them as exact as before (the bounds of test_gpu_packed_attention), bit by bit the same, and those of what
does see them within the bounds."""
import math

import pytest
import torch

from oracle.packed_attention import packed_attention
from test_gpu_packed_attention import check, make, step

pytestmark = pytest.mark.gpu


def check_in_range(got, ref, name, dtype, d):
    """:func:`check`; an element beyond the type's range (one of the oracle's dk is 66,182) is inf."""
    got, big = got.double().cpu(), ref[name].abs() > torch.finfo(dtype).max
    assert torch.equal(got[big], ref[name][big].sign() * math.inf)
    check(torch.where(big, ref[name], got), ref, name, dtype, d)


HEADS = [(64, 2, 2), (64, 4, 1), (128, 2, 1), (40, 2, 2)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,hk", HEADS)
@pytest.mark.parametrize("ratio", [2.0 ** 12, 2.0 ** 15, 2.0 ** 20])
def test_a_large_gradient_and_a_large_value(gpu_device, dtype, d, hq, hk, ratio):
    """Row 10 of 1,024 in causal order has dO ``ratio`` times the others', key 5 values of 64 times the others'."""
    args = make([1024, 70], None, hq, hk, d, dtype, seed=1)
    q, k, v, do, cu_q, cu_k = args
    do.mul_(2048.0 / ratio)
    do[10] *= ratio
    v[5] *= 64
    ref = packed_attention(q, k, v, cu_q, cu_k, True, do=do)
    for name, got in zip(("o", "dq", "dk", "dv"), step(args, gpu_device, True)):
        check_in_range(got, ref, name, dtype, d)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,hk", HEADS)
def test_small_values_before_a_large_one(gpu_device, dtype, d, hq, hk):
    """The last key's value is 2^25 times the others'; the one row that sees it has dO = 0."""
    args = make([1000], None, hq, hk, d, dtype, seed=2)
    q, k, v, do, cu_q, cu_k = args
    v.mul_(2.0 ** -10)
    v[-1] = 32768.0
    do.mul_(256.0)
    do[-1] = 0
    ref = packed_attention(q, k, v, cu_q, cu_k, True, do=do)
    for name, got in zip(("o", "dq", "dk", "dv"), step(args, gpu_device, True)):
        check(got, ref, name, dtype, d)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,hk", HEADS)
@pytest.mark.parametrize("lens_q,lens_k", [([1024, 70], None), ([300], [2100]), ([700], [400])])
def test_what_does_not_see_an_outlier_keeps_its_bits(gpu_device, dtype, d, hq, hk, lens_q, lens_k):
    args = make(lens_q, lens_k, hq, hk, d, dtype, seed=3)
    clean = step(args, gpu_device, True)
    n_q, n_k = lens_q[0], (lens_k or lens_q)[0]
    cut = n_q - 1 - n_q // 5  # the first row that sees the key
    q, k, v, do, cu_q, cu_k = (t.clone() if torch.is_tensor(t) else t for t in args)
    v[cut + n_k - n_q] *= 1000
    out = step((q, k, v, do, cu_q, cu_k), gpu_device, True)
    assert torch.equal(clean[1][:cut], out[1][:cut]) and torch.equal(clean[1][n_q:], out[1][n_q:])
    assert not torch.equal(clean[1][cut:n_q], out[1][cut:n_q])
    row = n_q // 3 if n_q <= n_k else n_q - n_k + n_k // 3
    v = args[2]
    do[row] *= 1000
    out = step((q, k, v, do, cu_q, cu_k), gpu_device, True)
    first = row + n_k - n_q + 1  # the first key that the row does not see
    for i in (2, 3):
        assert torch.equal(clean[i][first:], out[i][first:])
        assert not torch.equal(clean[i][:first], out[i][:first])


@pytest.mark.parametrize("d,hq,hk", [(64, 2, 2), (128, 2, 1)])
@pytest.mark.parametrize("causal", [False, True])
def test_gradients_that_grow_along_the_sequence(gpu_device, d, hq, hk, causal):
    """dO and values that rise by 2^24 and fall again: the powers of two of dS follow."""
    args = make([900, 130], None, hq, hk, d, torch.float16, seed=4)
    q, k, v, do, cu_q, cu_k = args
    x = torch.linspace(-12, 12, 450)
    ramp = torch.cat([x, x.flip(0), torch.zeros(130)])[:, None, None]
    do.copy_((do.float() * 2 ** ramp).half())
    v.copy_((v.float() * 2 ** (ramp / 3)).half())
    ref = packed_attention(q, k, v, cu_q, cu_k, causal, do=do)
    for name, got in zip(("o", "dq", "dk", "dv"), step(args, gpu_device, causal)):
        check(got, ref, name, torch.float16, d)
