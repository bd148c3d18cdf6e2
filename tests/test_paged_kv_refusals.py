"""CPU checks of what the paged caches' entry points refuse, in Python and at the C ABI, before anything touches a GPU,
and of the sizes that the host plans with."""
import ctypes
import math

import pytest
import torch

from geoweave_amd import _lib
from geoweave_amd import aggregator as agg
from geoweave_amd.custom_flash_attn.paged_flash_attn import paged_flash_attn_inference_func
from geoweave_amd.custom_flash_attn.paged_kv_cache import (FP4Cache, fp4_paged_cache, paged_kv_append_func,
                                                           paged_kv_read_func)

BF, HF = torch.bfloat16, torch.float16


def cache16(pages=3, page=16, hk=2, d=64, dtype=BF):
    return torch.zeros(pages, page, hk, d, dtype=dtype)


def cache4(pages=3, page=16, hk=2, d=64):
    return fp4_paged_cache(pages, page, hk, d)


def base(fp4=False, b=2, n=1, hk=2, d=64, dtype=BF):
    x = torch.zeros(b, n, hk, d, dtype=dtype)
    c = cache4(hk=hk, d=d) if fp4 else cache16(hk=hk, d=d, dtype=dtype)
    return dict(k=x, v=x, k_cache=c, v_cache=c, block_table=torch.zeros(b, 2, dtype=torch.int32),
                cache_seqlens=torch.zeros(b, dtype=torch.int32))


INT2, POS = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 1, 2, dtype=torch.int32)
X = torch.zeros(2, 1, 2, 64, dtype=BF)

APPEND = [
    ({}, ValueError, "one GPU"),
    (dict(v=X.half()), TypeError, "same type"),
    (dict(q=X.half()), TypeError, "same type"),
    (dict(k=X.half(), v=X.half()), TypeError, "same type"),
    (dict(k=X.float(), v=X.float()), TypeError, "fp16 and bf16"),
    (dict(v=X[:, :, :1]), ValueError, "must be"),
    (dict(k=X[:, :, :1], v=X[:, :, :1]), ValueError, "caches' Hk"),
    (dict(k=X[..., :32], v=X[..., :32]), ValueError, "caches' Hk"),
    (dict(k=X[None], v=X[None]), ValueError, "caches' Hk"),
    (dict(k=X[:1], v=X[:1]), ValueError, "does not go"),
    (dict(q=X[:1]), ValueError, "differ"),
    (dict(q=X[:, 0]), ValueError, "differ"),
    (dict(q=torch.zeros(2, 1, 2, 128, dtype=BF)), ValueError, "differ"),
    (dict(k_cache=cache4()), TypeError, "both"),
    (dict(v_cache=cache4()), TypeError, "both"),
    (dict(k_cache=tuple(cache4()), v_cache=tuple(cache4())), TypeError, "a cache is"),
    (dict(v_cache=cache16(page=8)), ValueError, "caches must be"),
    (dict(k_cache=cache16()[0], v_cache=cache16()[0]), ValueError, "caches must be"),
    (dict(v_cache=cache16(dtype=HF)), TypeError, "same type"),
    (dict(k_cache=cache16(dtype=torch.float32), v_cache=cache16(dtype=torch.float32)), TypeError, "fp16 and bf16"),
    (dict(k_cache=cache16(d=96), v_cache=cache16(d=96)), ValueError, "head dims"),
    (dict(k_cache=cache16(page=0), v_cache=cache16(page=0)), ValueError, "slot"),
    (dict(k_cache=cache16(d=128)[..., ::2]), ValueError, "aligned"),
    (dict(k_cache=torch.zeros(3, 16, 2, 68, dtype=BF)[..., :64]), ValueError, "aligned"),
    (dict(k_cache=torch.zeros(3 * 16 * 128 + 4, dtype=BF)[4:].view(3, 16, 2, 64)), ValueError, "aligned"),
    (dict(block_table=torch.zeros(2, 2)), TypeError, "int32"),
    (dict(block_table=INT2), ValueError, "block_table"),
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int32)), ValueError, "block_table"),
    (dict(cache_seqlens=INT2.long()), TypeError, "int32"),
    (dict(cache_seqlens=INT2[None]), ValueError, "cache_seqlens"),
    (dict(block_table=torch.zeros(2, 1, dtype=torch.int32).expand(2, 1 << 27)), ValueError, "must not exceed"),
    (dict(positions=POS), ValueError, "go together"),
    (dict(axis_dims=(32, 32)), ValueError, "go together"),
    (dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), ValueError, "must be"),
    (dict(k=X[:, 0], v=X[:, 0], cu_seqlens=INT2), ValueError, "cu_seqlens"),
    (dict(k=X[:, 0], v=X[:, 0], cu_seqlens=torch.zeros(3)), TypeError, "int32"),
]


class _OnGpu(torch.Tensor):
    """Says that it lies on a GPU: what is checked behind that question is reached without one."""

    is_cuda = property(lambda self: True)


@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(case):
    over, error, match = APPEND[case]
    args = base()
    args.update(over)
    if match in ("int32", "must not exceed"):
        args["k_cache"] = args["k_cache"].as_subclass(_OnGpu)
    with pytest.raises(error, match=match):
        paged_kv_append_func(**args)


AXES = [
    (dict(positions=POS, axis_dims=()), ValueError, "axes"),
    (dict(positions=POS, axis_dims=(2,) * 9), ValueError, "axes"),
    (dict(positions=POS, axis_dims=(32, 31)), ValueError, "even"),
    (dict(positions=POS, axis_dims=(32, 34)), ValueError, "even"),
    (dict(positions=POS, axis_dims=(-2, 34)), ValueError, "even"),
    (dict(positions=POS, axis_dims=(32, 32), bases=0.0), ValueError, "base"),
    (dict(positions=POS, axis_dims=(32, 32), bases=(1.0,)), ValueError, "base"),
    (dict(positions=POS, axis_dims=(32, 32), bases=(1.0, math.inf)), ValueError, "base"),
    (dict(positions=POS.double(), axis_dims=(32, 32)), TypeError, "positions"),
    (dict(positions=POS, axis_dims=(64,)), ValueError, "positions"),
    (dict(positions=POS[:, 0], axis_dims=(32, 32)), ValueError, "positions"),
]


@pytest.mark.parametrize("case", range(len(AXES)))
def test_append_axes(case):
    over, error, match = AXES[case]
    args = base()
    args.update(over)
    args["k_cache"] = args["k_cache"].as_subclass(_OnGpu)
    with pytest.raises(error, match=match):
        paged_kv_append_func(**args)


def _codes(c, **kw):
    return FP4Cache(kw.get("codes", c.codes), kw.get("scales", c.scales))


FP4 = [
    (lambda c: _codes(c, codes=c.codes.to(torch.int16)), TypeError, "uint8"),
    (lambda c: _codes(c, scales=c.scales.float()), TypeError, "uint8"),
    (lambda c: _codes(c, scales=c.scales[..., :1]), ValueError, "32 dims"),
    (lambda c: _codes(c, scales=c.scales[:2]), ValueError, "32 dims"),
    (lambda c: _codes(c, scales=torch.zeros(3, 16, 2, 3, dtype=torch.uint8)[..., :2]), ValueError, "scales need"),
    (lambda c: _codes(c, codes=torch.zeros(3, 16, 2, 40, dtype=torch.uint8)[..., :32]), ValueError, "aligned"),
    (lambda c: _codes(c, codes=torch.zeros(3, 16, 2, 48, dtype=torch.uint8)), ValueError, "head dims"),
    (lambda c: _codes(c, codes=c.codes[:, 0]), ValueError, "caches must be"),
]


@pytest.mark.parametrize("which", ["append", "read", "attend"])
@pytest.mark.parametrize("case", range(len(FP4)))
def test_fp4_caches(case, which):
    make, error, match = FP4[case]
    c = make(cache4())
    table, lens = torch.zeros(2, 2, dtype=torch.int32), INT2
    with pytest.raises(error, match=match):
        if which == "append":
            paged_kv_append_func(X, X, c, c, table, lens)
        elif which == "read":
            paged_kv_read_func(c, c, table, torch.zeros(3, dtype=torch.int32), 4)
        else:
            paged_flash_attn_inference_func(X, c, c, table, lens)


def test_fp4_attention():
    c, table = cache4(), torch.zeros(2, 2, dtype=torch.int32)
    for q, kw, error, match in ((X, {}, ValueError, "one GPU"), (X.float(), {}, TypeError, "fp16 and bf16"),
                                (torch.zeros(2, 1, 3, 64, dtype=BF), {}, ValueError, "multiple"),
                                (torch.zeros(2, 1, 0, 64, dtype=BF), {}, ValueError, "multiple"),
                                (torch.zeros(2, 1, 2, 128, dtype=BF), {}, ValueError, "head dim"),
                                (X[0, 0], {}, ValueError, r"\[B, Hq, D\]")):
        with pytest.raises(error, match=match):
            paged_flash_attn_inference_func(q, c, c, table, INT2, **kw)
    with pytest.raises(TypeError, match="both"):
        paged_flash_attn_inference_func(X, c, cache16(), table, INT2)
    with pytest.raises(TypeError, match="both"):
        paged_flash_attn_inference_func(X, cache16(), c, table, INT2)
    with pytest.raises(TypeError, match="int32"):
        paged_flash_attn_inference_func(X, c, c, table.long(), INT2)
    with pytest.raises(ValueError, match="block_table"):
        paged_flash_attn_inference_func(X, c, c, table[:1], INT2)
    q = X.as_subclass(_OnGpu)
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="softmax_scale"):
            paged_flash_attn_inference_func(q, c, c, table, INT2, softmax_scale=scale)


def test_read():
    c, table, cu = cache16(), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for args, kw, error, match in (((c, c, table, cu, 4), {}, ValueError, "one GPU"), ((c, c, table, cu, -1), {}, ValueError, "tokens"),
                                   ((c, c, table, cu, 1 << 30), {}, ValueError, "tokens"),
                                   ((c, c, table, cu[:2], 4), {}, ValueError, "cu_seqlens"),
                                   ((c, c, cu, cu, 4), {}, ValueError, "block_table"),
                                   ((c, c, table, cu, 4), dict(dtype=HF), TypeError, "own type"),
                                   ((cache4(), cache4(), table, cu, 4), dict(dtype=torch.float32), TypeError, "bf16 or fp16")):
        with pytest.raises(error, match=match):
            paged_kv_read_func(*args, **kw)


def test_cache_maker():
    c = fp4_paged_cache(3, 16, 2, 128)
    assert c.codes.shape == (3, 16, 2, 64) and c.scales.shape == (3, 16, 2, 4)
    assert c.codes.stride() == (2 * 16 * 64, 64, 16 * 64, 1) and c.scales.stride() == (2 * 16 * 4, 4, 16 * 4, 1)
    for args in ((3, 16, 2, 96), (-1, 16, 2, 64), (3, -1, 2, 64)):
        with pytest.raises(ValueError):
            fp4_paged_cache(*args)


# --- the C ABI: the addresses are never read, every call ends before a launch -----------------

S = _lib.strides3(1024, 1024, 64)


def append(**over):
    lib = _lib.load()
    a = dict(dtype=0, q=256, qs=S, qo=256, hq=2, k=256, ks=S, v=256, vs=S, hk=2, d=64, fmt=0, kc=256, kcs=S, ksc=None, kscs=None, vc=256,
             vcs=S, vsc=None, vscs=None, table=256, width=4, lens=256, cu=None, n=2, count=3, pages=4, page=16, pt=0, pos=256, ps=S,
             axes=(32, 32), bases=(100.0, 100.0))
    a.update(over)
    dims, bases = (ctypes.c_int32 * max(len(a["axes"]), 1))(*a["axes"]), (ctypes.c_double * max(len(a["axes"]), 1))(*a["bases"])
    rc = lib.gw_paged_kv_append(a["dtype"], a["q"], a["qs"], a["qo"], a["hq"], a["k"], a["ks"], a["v"], a["vs"], a["hk"], a["d"],
                                a["fmt"], a["kc"], a["kcs"], a["ksc"], a["kscs"], a["vc"], a["vcs"], a["vsc"], a["vscs"], a["table"],
                                a["width"], a["lens"], a["cu"], a["n"], a["count"], a["pages"], a["page"], a["width"], a["pt"], a["pos"],
                                a["ps"], len(a["axes"]), dims, bases, None)
    return rc, lib.gw_last_error().decode()


SC = _lib.strides3(64, 4, 2)


@pytest.mark.parametrize("over,code,word", [
    (dict(dtype=2), 1, "dtype"), (dict(d=96), 2, "head dim"), (dict(hk=0), 1, "key heads"), (dict(hq=-1), 1, "negative"),
    (dict(n=-1), 1, "negative"), (dict(count=-1), 1, "negative"), (dict(pages=-1), 1, "negative"), (dict(width=-1), 1, "negative"),
    (dict(page=0), 1, "page size"), (dict(page=1 << 31), 1, "page size"), (dict(fmt=2), 1, "format"), (dict(k=None), 1, "missing"),
    (dict(v=None), 1, "missing"), (dict(q=None), 1, "missing"), (dict(qo=None), 1, "missing"), (dict(lens=None), 1, "missing"),
    (dict(pos=None), 1, "missing"), (dict(table=None), 1, "missing"), (dict(kc=None), 1, "missing"), (dict(vc=None), 1, "missing"),
    (dict(k=264), 1, "aligned"), (dict(ks=_lib.strides3(1024, 1020, 64)), 1, "aligned"), (dict(kc=264), 1, "aligned"),
    (dict(vcs=_lib.strides3(1024, 4, 64)), 1, "aligned"), (dict(qo=264), 1, "aligned"),
    (dict(pt=3), 1, "position type"), (dict(axes=(32, 33)), 1, "even"), (dict(axes=(64, 2)), 1, "exceed"),
    (dict(axes=(2 ** 30, 2 ** 30)), 1, "exceed"), (dict(axes=(2,) * 9, bases=(1.0,) * 9), 1, "axes"), (dict(bases=(1.0, -1.0)), 1, "base"),
    (dict(fmt=1), 1, "scales are missing"), (dict(fmt=1, ksc=256, kscs=SC), 1, "scales are missing"),
    (dict(fmt=1, ksc=257, kscs=SC, vsc=256, vscs=SC), 1, "scales need"),
    (dict(fmt=1, ksc=256, kscs=SC, vsc=256, vscs=_lib.strides3(64, 3, 2)), 1, "scales need"),
    (dict(n=1 << 20, count=1 << 12), 2, "sequences"), (dict(n=1 << 20, count=1 << 10), 2, "2^31"), (dict(width=1 << 28), 2, "2^31"),
    (dict(cu=256, n=1 << 30, count=4), 2, "2^31"), (dict(hk=1 << 19), 2, "2^20"),
    (dict(cu=256, count=1 << 28, hk=1, hq=0, n=1), 2, "2^32 threads"),
])
def test_append_abi(over, code, word):
    rc, msg = append(**over)
    assert rc == code and word in msg, (rc, msg)


def test_empty_appends_are_no_ops():
    assert append(n=0)[0] == 0 and append(count=0)[0] == 0 and append(cu=256, count=0)[0] == 0
    assert append(n=0, k=None, v=None, q=None, lens=None, table=None, kc=None)[0] == 0


def read(**over):
    lib = _lib.load()
    a = dict(dtype=0, fmt=0, kc=256, kcs=S, ksc=None, kscs=None, vc=256, vcs=S, vsc=None, vscs=None, table=256, cu=256, n=2, tokens=10, hk=2,
             d=64, pages=4, page=16, width=4, ko=256, vo=256)
    a.update(over)
    rc = lib.gw_paged_kv_read(a["dtype"], a["fmt"], a["kc"], a["kcs"], a["ksc"], a["kscs"], a["vc"], a["vcs"], a["vsc"], a["vscs"],
                              a["table"], a["width"], a["cu"], a["n"], a["tokens"], a["hk"], a["d"], a["pages"], a["page"], a["width"],
                              a["ko"], a["vo"], None)
    return rc, lib.gw_last_error().decode()


@pytest.mark.parametrize("over,code,word", [
    (dict(dtype=2), 1, "dtype"), (dict(fmt=3), 1, "format"), (dict(d=32), 2, "head dim"), (dict(hk=0), 1, "key heads"),
    (dict(tokens=-1), 1, "negative"), (dict(ko=None), 1, "missing"), (dict(cu=None), 1, "missing"), (dict(vo=264), 1, "aligned"),
    (dict(kc=None), 1, "missing"), (dict(vc=258), 1, "aligned"), (dict(fmt=1), 1, "scales are missing"),
    (dict(tokens=1 << 30), 2, "2^31"), (dict(table=None), 1, "missing"), (dict(tokens=1 << 28, hk=1), 2, "2^32 threads"),
])
def test_read_abi(over, code, word):
    rc, msg = read(**over)
    assert rc == code and word in msg, (rc, msg)
    assert read(tokens=0, ko=None, vo=None, kc=None)[0] == 0


def attend(**over):
    lib = _lib.load()
    a = dict(dtype=0, q=256, qs=S, k=256, ks=S, ksc=256, kscs=SC, v=256, vs=S, vsc=256, vscs=SC, table=256, lens=256, o=256, os=S, b=2, n=1,
             hq=4, hk=2, d=64, pages=4, page=16, width=4, scale=0.125, ws=None, nbytes=0)
    a.update(over)
    rc = lib.gw_paged_attn_fp4_fwd(a["dtype"], a["q"], a["qs"], a["k"], a["ks"], a["ksc"], a["kscs"], a["v"], a["vs"], a["vsc"],
                                   a["vscs"], a["table"], a["width"], a["lens"], a["o"], a["os"], None, a["b"], a["n"], a["hq"],
                                   a["hk"], a["d"], a["pages"], a["page"], a["width"], 1, a["scale"], a["ws"], a["nbytes"], None)
    return rc, lib.gw_last_error().decode()


@pytest.mark.parametrize("over,code,word", [
    (dict(dtype=3), 1, "dtype"), (dict(d=80), 2, "head dim"), (dict(page=0), 1, "page size"), (dict(hq=3), 1, "multiple"),
    (dict(scale=-1.0), 1, "scale"), (dict(scale=math.nan), 1, "scale"), (dict(q=None), 1, "missing"), (dict(k=None), 1, "cache"),
    (dict(ksc=None), 1, "cache"), (dict(kscs=None), 1, "missing"), (dict(table=None), 1, "table"), (dict(k=258), 1, "aligned"),
    (dict(ks=_lib.strides3(1024, 24, 64)), 1, "aligned"), (dict(qs=_lib.strides3(1024, 1024, 60)), 1, "aligned"),
    (dict(vsc=257), 1, "scales need"), (dict(vscs=_lib.strides3(64, 3, 2)), 1, "scales need"), (dict(pages=-1), 1, "negative"),
    (dict(ks=_lib.strides3(-1024, 16, 64)), 1, "negative"), (dict(vscs=_lib.strides3(64, 4, -2)), 1, "negative"), (dict(width=1 << 28), 2, "2^31"), (dict(b=1 << 30), 2, "2^31"),
    (dict(ks=_lib.strides3(1 << 36, 16, 64)), 2, "2^36"), (dict(), 1, "workspace"), (dict(ws=264, nbytes=1 << 30), 1, "workspace"),
    (dict(ws=256, nbytes=100), 1, "workspace"), (dict(b=1 << 23, ws=256, nbytes=1 << 60), 2, "2^32 threads"),
])
def test_attend_abi(over, code, word):
    rc, msg = attend(**over)
    assert rc == code and word in msg, (rc, msg)
    assert attend(b=0, q=None, o=None)[0] == 0


def test_workspaces_are_bounded_by_the_sizes():
    size = _lib.load().gw_paged_attn_fp4_fwd_workspace_size
    for b, n, hq, hk, d in ((1, 1, 1, 1, 64), (64, 1, 32, 8, 128), (1000, 8, 8, 1, 128), (1, 1374, 16, 16, 64), (3, 1, 1100, 1100, 64)):
        assert 0 < size(b, n, hq, hk, d) <= 1 << 26, (b, n, hq, hk, d)
    assert size(8192, 1, 32, 8, 128) == 0  # no split
    assert size(0, 1, 1, 1, 64) == 0 and size(1, 1 << 40, 1, 1, 64) == 0


@pytest.mark.parametrize("lengths", [[20], [20, 20, 20], [20, -1], [33, 20]])
@pytest.mark.parametrize("fp4", [False, True])
def test_lengths_of_a_layer(fp4, lengths):
    """What the host says of the lengths is checked against the table's slots before anything is written."""
    m = agg.DenseAttention(128, 2, False, None).to(BF)
    c = cache4() if fp4 else cache16()
    with pytest.raises(ValueError, match="slots$|lengths of 2 sequences"):
        m.forward_cached(torch.zeros(2, 1, 128, dtype=BF), c, c, torch.zeros(2, 2, dtype=torch.int32), INT2, lengths=lengths)
