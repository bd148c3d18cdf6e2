"""Gradients where a key or a query holds -inf in one dim and the scores with it are -inf: its weights are 0, and
0 * inf in that dim is NaN wherever the two see each other, as in the definition, and nowhere else, whichever tile
they meet in. Everything else is held to the bounds of test_gpu_packed_attention."""
import math

import pytest
import torch

from oracle.packed_attention import packed_attention
from test_gpu_packed_attention import check, make, step

pytestmark = pytest.mark.gpu

DIM = 5
CASES = [([300, 77], None), ([70], [150]), ([200], [3300]), ([333, 64], [90, 640])]


def check_but(got, ref, name, dtype, d, nan):
    """:func:`check` outside the places ``nan`` of DIM, which are NaN."""
    got = got.double().cpu()
    assert got[..., DIM][nan].isnan().all(), f"{name}: finite where 0 * inf is seen"
    want, mag = ref[name].clone(), ref[name + "_mag"].clone()
    got[..., DIM][nan] = 0
    want[..., DIM][nan] = 0
    mag[..., DIM][nan] = 0
    check(got, {"s_mag": ref["s_mag"], name: want, name + "_mag": mag}, name, dtype, d)


def positive(args):
    """The inputs with q and k positive in DIM."""
    q, k, v, do, cu_q, cu_k = args
    q[..., DIM], k[..., DIM] = q[..., DIM].abs() + 0.5, k[..., DIM].abs() + 0.5
    return q, k, v, do, cu_q, cu_k


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,hk", [(64, 2, 2), (128, 4, 2)])
@pytest.mark.parametrize("lens_q,lens_k", CASES)
@pytest.mark.parametrize("causal", [False, True])
def test_a_key_that_scores_minus_infinity(gpu_device, dtype, d, hq, hk, lens_q, lens_k, causal):
    q, k, v, do, cu_q, cu_k = positive(make(lens_q, lens_k, hq, hk, d, dtype, 20))
    n_q, n_k = cu_q[1], cu_k[1]
    s_mag = packed_attention(q, k, v, cu_q, cu_k, causal)["s_mag"]
    for j in (n_k // 2, n_k - 1):
        kj = k.clone()
        kj[j, :, DIM] = -math.inf
        far = k.double()
        far[j, :, DIM] = -1e30  # a weight of 0 without the inf
        ref = packed_attention(q, far, v, cu_q, cu_k, causal, do=do)
        ref["s_mag"] = s_mag
        o, dq, dk, dv = step((q, kj, v, do, cu_q, cu_k), gpu_device, causal)
        check(o, ref, "o", dtype, d)
        rows = torch.arange(cu_q[-1])
        sees = (rows < n_q) & (rows + n_k - n_q >= j if causal else True)
        check_but(dq, ref, "dq", dtype, d, sees)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,hk", [(64, 2, 2), (128, 4, 2)])
@pytest.mark.parametrize("lens_q,lens_k", CASES)
@pytest.mark.parametrize("causal", [False, True])
def test_a_query_that_scores_minus_infinity(gpu_device, dtype, d, hq, hk, lens_q, lens_k, causal):
    q, k, v, do, cu_q, cu_k = positive(make(lens_q, lens_k, hq, hk, d, dtype, 21))
    n_q, n_k = cu_q[1], cu_k[1]
    for i in (n_q // 2, n_q - 1):
        qi, none = q.clone(), do.clone()
        qi[i, :, DIM] = -math.inf
        none[i] = 0  # a row of weights 0 adds nothing
        ref = packed_attention(q, k, v, cu_q, cu_k, causal, do=none)
        o, dq, dk, dv = step((qi, k, v, do, cu_q, cu_k), gpu_device, causal)
        assert (o[i] == 0).all() and (dq[i] == 0).all()
        check(dv, ref, "dv", dtype, d)
        keys = torch.arange(cu_k[-1])
        seen = (keys < n_k) & (keys <= i + n_k - n_q if causal else True)
        check_but(dk, ref, "dk", dtype, d, seen)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,hk", [(64, 2, 2), (128, 4, 2), (64, 1, 1)])
@pytest.mark.parametrize("lens_q,lens_k", CASES + [([65], [65]), ([129, 3], [1, 700]), ([1], [64])])
@pytest.mark.parametrize("causal", [False, True])
def test_gradients_of_a_key_that_scores_minus_infinity(gpu_device, dtype, d, hq, hk, lens_q, lens_k, causal):
    """Its weights are 0, so its dk and dv are 0; queries behind the sequence's end, which a tile holds as zeros, are
    no queries (0 times its inf would be NaN)."""
    q, k, v, do, cu_q, cu_k = positive(make(lens_q, lens_k, hq, hk, d, dtype, 22))
    n_k = cu_k[1]
    s_mag = packed_attention(q, k, v, cu_q, cu_k, causal)["s_mag"]
    for j in {n_k // 2, n_k - 1}:
        kj, far = k.clone(), k.double()
        kj[j, :, DIM], far[j, :, DIM] = -math.inf, -1e30
        ref = packed_attention(q, far, v, cu_q, cu_k, causal, do=do)
        ref["s_mag"] = s_mag
        _, _, dk, dv = step((q, kj, v, do, cu_q, cu_k), gpu_device, causal)
        if n_k > 1:
            assert (dk[j] == 0).all() and (dv[j] == 0).all()
            check(dv, ref, "dv", dtype, d)
            check(dk, ref, "dk", dtype, d)
