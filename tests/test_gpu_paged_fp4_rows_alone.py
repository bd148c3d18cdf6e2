"""Attention over 4 bits: for given lengths, the bits of a row's o and lse depend on its query and on what it sees, and not on
what later keys and unused slots hold, whatever their powers of two are."""
import pytest
import torch

from test_gpu_paged_attention_fp4 import make, run

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
# Beside the usual powers: outside fp16's normal numbers on either side, the least, the largest, not a number.
SCALES = [126, 100, 150, 0, 254, 255]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,hq,hk,page", [(64, 2, 2, 16), (64, 4, 1, 100), (128, 8, 1, 64), (128, 3, 3, 7)])
@pytest.mark.parametrize("n", [40, 1500])
@pytest.mark.parametrize("scale", SCALES)
def test_later_keys(gpu_device, dtype, d, hq, hk, page, n, scale):
    new = 20
    args = make([n, 33], new, hq, hk, d, page, dtype, 90)
    _, k, v, table, _ = args
    want, changed = run(args, gpu_device), False
    g = torch.Generator().manual_seed(91)
    for cut in (1, 9, 19):  # the first new token that sees the change
        kept = [t.clone() for t in (*k, *v)]
        for j in range(n - new + cut, n):
            at = int(table[0, j // page]), j % page
            for c in (k, v):
                c[0][at] = torch.randint(0, 256, c[0][at].shape, generator=g).to(torch.uint8)
                c[1][at] = scale
        got = run(args, gpu_device)
        for t, old in zip((*k, *v), kept):
            t.copy_(old)
        for a, b in zip(want, got):
            assert torch.equal(a[0, :cut], b[0, :cut]) and torch.equal(a[1], b[1])
            changed |= not torch.equal(a, b)
    assert changed  # (a single one of 1,500 keys may weigh less than a rounding)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,hq,hk,page", [(64, 2, 2, 16), (64, 8, 1, 100), (128, 8, 1, 64), (128, 3, 3, 7)])
@pytest.mark.parametrize("scale", SCALES)
def test_unused_slots(gpu_device, dtype, d, hq, hk, page, scale):
    args = make([1, 37, 600, 0, 129], 1, hq, hk, d, page, dtype, 92)
    _, k, v, table, lens = args
    want = run(args, gpu_device)
    used = torch.zeros(k[0].shape[:2], dtype=torch.bool)
    for b, n in enumerate(lens.tolist()):
        for j in range(n):
            used[table[b, j // page], j % page] = True
    for c in (k, v):
        c[0][~used], c[1][~used] = 0x5E, scale
    for a, b in zip(want, run(args, gpu_device)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("d,hq,hk,new,lens", [(64, 16, 16, 1, [5496]), (128, 16, 2, 8, [5000, 60000, 31000]),
                                              (64, 16, 4, 5, [20000, 1, 700, 9000])])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_the_same_call_again(gpu_device, dtype, d, hq, hk, new, lens):
    """Units that end one row tile and begin another, joined in a fixed order: the same bits every time."""
    args = make(lens, new, hq, hk, d, 64, dtype, 93)
    want = run(args, gpu_device)
    for _ in range(8):
        for a, b in zip(want, run(args, gpu_device)):
            assert torch.equal(a, b)
