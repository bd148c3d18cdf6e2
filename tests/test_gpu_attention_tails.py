"""fp16 attention whose first key outweighs every other by 2^16 to 2^25 and holds a value of 0 (a sink): the
output is made of the long tail alone. Against the 64-bit oracle, within the bounds of test_gpu_packed_attention
(half a step of the 16-bit type per weight and output, floor 2^-20)."""
import math

import pytest
import torch

from geoweave_amd.custom_flash_attn.packed_flash_attn import packed_flash_attn_inference_func
from geoweave_amd.custom_flash_attn.paged_flash_attn import paged_flash_attn_inference_func
from oracle.packed_attention import packed_attention, paged_attention
from test_gpu_packed_attention import check, check_lse, step

pytestmark = pytest.mark.gpu


def sink(lens_q, lens_k, h, d, octaves, dtype=torch.float16):
    """q, k, v, do, cu_q, cu_k: the first key of every sequence scores ``octaves`` above the others (which lie
    within half an octave of 0) and has v = 0, the others v near 1."""
    g = torch.Generator().manual_seed(d)
    cu_q, cu_k = ([sum(n[:i]) for i in range(len(n) + 1)] for n in (lens_q, lens_k))
    q = 1 + 0.01 * torch.randn(cu_q[-1], h, d, generator=g)
    k = 0.02 * torch.randn(cu_k[-1], h, d, generator=g)
    v = 1 + 0.1 * torch.randn(cu_k[-1], h, d, generator=g)
    k[cu_k[:-1]] = octaves * math.log(2) / math.sqrt(d)  # d elements of it, times d ** -0.5
    v[cu_k[:-1]] = 0
    do = torch.randn(cu_q[-1], h, d, generator=g)
    return (*(t.to(dtype) for t in (q, k, v, do)), cu_q, cu_k)


# Tile kernel, split keys, few rows, and several sequences of both kinds.
SHAPES = {"tiles": ([600], [9000]), "split": ([140], [20000]), "few rows": ([2], [43968]),
          "mixed": ([3, 200, 40], [9000, 4000, 6000])}


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("octaves", [16.3, 22.7, 25.1])
def test_packed_tail(gpu_device, d, shape, octaves):
    args = sink(*SHAPES[shape], 2, d, octaves)
    ref = packed_attention(*args[:3], *args[4:], False, do=args[3])
    cu = [torch.tensor(c, dtype=torch.int32, device=gpu_device) for c in args[4:]]
    o, lse = packed_flash_attn_inference_func(*(t.to(gpu_device) for t in args[:3]), *cu, return_lse=True)
    check(o, ref, "o", torch.float16, d)
    check_lse(lse, ref)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("octaves", [22.7, 25.1])
def test_packed_tail_gradients(gpu_device, d, octaves):
    """P is formed again from the lse, delta from o: they have to agree on the tail."""
    args = sink([600, 30], [9000, 5000], 2, d, octaves)
    ref = packed_attention(*args[:3], *args[4:], False, do=args[3])
    for name, got in zip(("o", "dq", "dk", "dv"), step(args, gpu_device, False)):
        check(got, ref, name, torch.float16, d)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("octaves", [16.3, 22.7, 25.1])
def test_paged_tail(gpu_device, d, octaves):
    lens, page, new = [20000, 9000], 16, 3
    q, k, v, _, _, cu_k = sink([new, new], lens, 2, d, octaves)
    table = torch.full((2, 1250), -1, dtype=torch.int32)
    pages, at = [], 0
    for b, n in enumerate(lens):
        for j in range(0, n, page):
            table[b, j // page] = at
            rows = slice(cu_k[b] + j, cu_k[b] + min(j + page, n))
            blank = torch.zeros(2, page, 2, d, dtype=torch.float16)
            blank[0, :rows.stop - rows.start], blank[1, :rows.stop - rows.start] = k[rows], v[rows]
            pages.append(blank)
            at += 1
    kc, vc = torch.stack(pages, 1)
    args = (q.view(2, new, 2, d), kc, vc, table, torch.tensor(lens, dtype=torch.int32))
    o, lse = paged_flash_attn_inference_func(*(t.to(gpu_device) for t in args), return_lse=True)
    want, want_lse, mag, s_mag = paged_attention(*args)
    check(o, {"s_mag": s_mag, "o": want, "o_mag": mag}, "o", torch.float16, d)
    check_lse(lse, {"s_mag": s_mag, "lse": want_lse})
