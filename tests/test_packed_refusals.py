"""CPU checks of what the packed, paged and rotary entry points refuse, in Python and at the C ABI, before
anything touches a GPU, and of the sizes that the host plans with."""
import ctypes
import math

import pytest
import torch

from geoweave_amd import _lib
from geoweave_amd.custom_flash_attn.packed_flash_attn import packed_flash_attn_func, packed_flash_attn_inference_func
from geoweave_amd.custom_flash_attn.paged_flash_attn import paged_flash_attn_inference_func
from geoweave_amd.rotary import rotary_axes_func, rotary_axes_qk_func, view_grid_positions

BF = torch.bfloat16


def _qkv(tq=8, tk=8, hq=4, hk=2, d=64, dtype=BF):
    return torch.zeros(tq, hq, d, dtype=dtype), torch.zeros(tk, hk, d, dtype=dtype), torch.zeros(tk, hk, d, dtype=dtype)


CU = torch.tensor([0, 8], dtype=torch.int32)

PACKED = [
    (lambda: (*_qkv(), CU), {}, ValueError, "one GPU"),
    (lambda: (*_qkv(dtype=torch.float32), CU), {}, TypeError, "fp16 and bf16"),
    (lambda: (*_qkv()[:2], _qkv()[2].half(), CU), {}, TypeError, "same type"),
    (lambda: (*_qkv(hq=5), CU), {}, ValueError, "multiple"),
    (lambda: (*_qkv(d=136), CU), {}, ValueError, "head dim"),
    (lambda: (*_qkv(d=0), CU), {}, ValueError, "head dim"),
    (lambda: (_qkv()[0], _qkv(d=32)[1], _qkv(d=32)[2], CU), {}, ValueError, "do not match"),
    (lambda: (*_qkv()[:2], _qkv(tk=9)[2], CU), {}, ValueError, "do not match"),
    (lambda: (_qkv()[0][None], *_qkv()[1:], CU), {}, ValueError, "tokens, heads"),
    (lambda: (*_qkv(), CU.long()), {}, TypeError, "int32"),
    (lambda: (*_qkv(), CU[None]), {}, ValueError, "sequences"),
    (lambda: (*_qkv(), CU[:0]), {}, ValueError, "sequences"),
    (lambda: (*_qkv(tk=9), CU), {}, ValueError, "different numbers"),
    (lambda: (*_qkv(), CU, torch.zeros(3, dtype=torch.int32)), {}, ValueError, "sequences"),
    (lambda: (*_qkv(), CU), {"softmax_scale": 0.0}, ValueError, "softmax_scale"),
    (lambda: (*_qkv(), CU), {"softmax_scale": -0.1}, ValueError, "softmax_scale"),
    (lambda: (*_qkv(), CU), {"softmax_scale": math.nan}, ValueError, "softmax_scale"),
    (lambda: (*_qkv(), CU), {"softmax_scale": math.inf}, ValueError, "softmax_scale"),
]


@pytest.mark.parametrize("case", range(len(PACKED)))
@pytest.mark.parametrize("fn", [packed_flash_attn_func, packed_flash_attn_inference_func])
def test_packed(case, fn):
    args, kw, error, match = PACKED[case]
    with pytest.raises(error, match=match):
        fn(*args(), **kw)


def test_packed_too_many_tokens():
    q = torch.zeros(1, 1, 64, dtype=BF).expand(1 << 28, 16, 64)
    with pytest.raises(ValueError, match="tokens x query heads"):
        packed_flash_attn_inference_func(q, q[:, :1], q[:, :1], torch.tensor([0, 1 << 28], dtype=torch.int32))


def _paged(b=2, n=1, hq=4, hk=2, d=64, pages=3, page=16, dtype=BF):
    c = torch.zeros(pages, page, hk, d, dtype=dtype)
    return (torch.zeros(b, n, hq, d, dtype=dtype), c, c.clone(), torch.zeros(b, 2, dtype=torch.int32),
            torch.zeros(b, dtype=torch.int32))


def _with(args, i, x):
    return tuple(x if j == i else a for j, a in enumerate(args))


PAGED = [
    (lambda: _paged(), ValueError, "one GPU"),
    (lambda: _paged(dtype=torch.float32), TypeError, "fp16 and bf16"),
    (lambda: _paged(d=32), ValueError, "head dims"),
    (lambda: _paged(d=96), ValueError, "head dims"),
    (lambda: _paged(hq=3), ValueError, "multiple"),
    (lambda: _paged(page=0), ValueError, "slot"),
    (lambda: _with(_paged(), 0, torch.zeros(2, 64, dtype=BF)), ValueError, r"\[B, Hq, D\]"),
    (lambda: _with(_paged(), 1, torch.zeros(3, 2, 64, dtype=BF)), ValueError, "caches must be"),
    (lambda: _with(_paged(), 2, torch.zeros(4, 16, 2, 64, dtype=BF)), ValueError, "do not match"),
    (lambda: _with(_paged(), 3, torch.zeros(2, 2, dtype=torch.int64)), TypeError, "int32"),
    (lambda: _with(_paged(), 3, torch.zeros(3, 2, dtype=torch.int32)), ValueError, "block_table"),
    (lambda: _with(_paged(), 4, torch.zeros(2, dtype=torch.int64)), TypeError, "int32"),
    (lambda: _with(_paged(), 4, torch.zeros(2, 1, dtype=torch.int32)), ValueError, "cache_seqlens"),
    (lambda: _with(_paged(), 3, torch.zeros(2, 1, dtype=torch.int32).expand(2, 1 << 27)), ValueError, "must not exceed"),
]


@pytest.mark.parametrize("case", range(len(PAGED)))
def test_paged(case):
    args, error, match = PAGED[case]
    with pytest.raises(error, match=match):
        paged_flash_attn_inference_func(*args())


X, POS = torch.zeros(6, 2, 64), torch.zeros(6, 2, dtype=torch.int32)

ROTARY = [
    (lambda: (X, POS, [32, 32]), ValueError, "one GPU"),
    (lambda: (X.double(), POS, [32, 32]), TypeError, "dtype"),
    (lambda: (X[0], POS, [32, 32]), ValueError, "expected"),
    (lambda: (X, POS, [32, 31]), ValueError, "even"),
    (lambda: (X, POS, [32, 34]), ValueError, "even"),
    (lambda: (X, POS, [-2, 34]), ValueError, "even"),
    (lambda: (X[..., :63], POS, [32, 30]), ValueError, "even"),
    (lambda: (X, POS, []), ValueError, "axes"),
    (lambda: (X, torch.zeros(6, 9, dtype=torch.int32), [2] * 9), ValueError, "axes"),
    (lambda: (X, POS, [32]), ValueError, "positions"),
    (lambda: (X, POS[:5], [32, 32]), ValueError, "positions"),
    (lambda: (X, POS.double(), [32, 32]), TypeError, "positions"),
    (lambda: (X, POS, [32, 32], [100.0]), ValueError, "base"),
    (lambda: (X, POS, [32, 32], 0.0), ValueError, "base"),
    (lambda: (X, POS, [32, 32], [100.0, math.inf]), ValueError, "base"),
    (lambda: (torch.zeros(6, 2, 258), POS, [32, 32]), ValueError, "head dim"),
]


@pytest.mark.parametrize("case", range(len(ROTARY)))
def test_rotary(case):
    args, error, match = ROTARY[case]
    with pytest.raises(error, match=match):
        rotary_axes_func(*args())


def test_rotary_pair():
    with pytest.raises(ValueError, match="differ"):
        rotary_axes_qk_func(X, torch.zeros(7, 2, 64), POS, [32, 32])
    with pytest.raises(ValueError, match="differ"):
        rotary_axes_qk_func(X, torch.zeros(6, 2, 32), POS, [32, 32])
    with pytest.raises(TypeError, match="same type"):
        rotary_axes_qk_func(X, X.bfloat16(), POS, [32, 32])


def test_view_positions_on_the_cpu():
    p = view_grid_positions(2, 1, 2, n_special=1)
    assert p.tolist() == [[0, 0, 0], [0, 1, 1], [0, 1, 2], [1, 0, 0], [1, 1, 1], [1, 1, 2]]
    with pytest.raises(ValueError, match="negative"):
        view_grid_positions(-1, 2, 2)


# --- the C ABI: the addresses are never read, every call ends before a launch -----------------


def _fwd(**over):
    lib, s = _lib.load(), _lib.strides2(256, 64)
    a = dict(dtype=0, q=256, qs=s, k=256, ks=s, v=256, vs=s, cu=256, o=256, os=s, rest=None, lse=None, n=1, tq=8, tk=8, hq=4, hk=4,
             d=64, causal=0, scale=0.125, ws=None, nbytes=0)
    a.update(over)
    rc = lib.gw_packed_attn_fwd(a["dtype"], a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["cu"], a["cu"], a["o"],
                                a["os"], a["rest"], a["lse"], a["n"], a["tq"], a["tk"], a["hq"], a["hk"], a["d"], a["causal"],
                                a["scale"], a["ws"], a["nbytes"], None)
    return rc, lib.gw_last_error().decode()


@pytest.mark.parametrize("over,code,word", [
    (dict(dtype=2), 1, "dtype"), (dict(d=96), 2, "head dim"), (dict(hq=5), 1, "multiple"), (dict(hk=0), 1, "multiple"),
    (dict(tq=-1), 1, "negative"), (dict(scale=0.0), 1, "scale"), (dict(scale=math.inf), 1, "scale"),
    (dict(scale=math.nan), 1, "scale"), (dict(q=None), 1, "missing"), (dict(k=None), 1, "missing"),
    (dict(cu=None), 1, "missing"), (dict(q=264), 1, "aligned"), (dict(ks=_lib.strides2(260, 64)), 1, "aligned"),
    (dict(vs=_lib.strides2(1 << 24, 64)), 1, "aligned"), (dict(tq=1 << 30, tk=1 << 30), 2, "2\\^31"),
    (dict(n=1 << 30), 2, "sequences"), (dict(n=1, tk=1 << 20, hq=4), 1, "workspace"),
])
def test_packed_forward_abi(over, code, word):
    rc, msg = _fwd(**over)
    assert rc == code, msg
    with pytest.raises(RuntimeError, match=word):
        _lib.check(rc, "gw_packed_attn_fwd")


def test_empty_calls_are_no_ops():
    assert _fwd(tq=0)[0] == 0
    lib, s3 = _lib.load(), _lib.strides3(256, 256, 64)
    assert lib.gw_paged_attn_fwd(0, None, s3, None, s3, None, s3, None, 0, None, None, s3, None, 0, 1, 4, 4, 64, 0, 16, 0,
                                 1, 0.125, None, 0, None) == 0
    dims, bases = (ctypes.c_int32 * 1)(64), (ctypes.c_double * 1)(100.0)
    assert lib.gw_rotary_axes(0, None, None, None, None, 0, None, None, None, None, 0, 0, None, None, 1, 5, 64, 1, dims,
                              bases, 0, None) == 0


def test_paged_abi():
    lib, s = _lib.load(), _lib.strides3(1024, 256, 64)

    def call(dtype=0, q=256, k=256, ks=s, table=256, b=2, n=1, hq=4, hk=2, d=64, pages=4, page=16, width=2, scale=0.125,
             ws=None, nbytes=0):
        rc = lib.gw_paged_attn_fwd(dtype, q, s, k, ks, k, ks, table, width, 256, 256, s, None, b, n, hq, hk, d, pages, page,
                                   width, 1, scale, ws, nbytes, None)
        return rc, lib.gw_last_error().decode()

    for kw, code, word in ((dict(dtype=3), 1, "dtype"), (dict(d=80), 2, "head dim"), (dict(page=0), 1, "page size"),
                           (dict(hq=3), 1, "multiple"), (dict(scale=-1.0), 1, "scale"), (dict(q=None), 1, "missing"),
                           (dict(k=None), 1, "cache"), (dict(table=None), 1, "table"), (dict(k=258), 1, "aligned"),
                           (dict(ks=_lib.strides3(1024, 257, 64)), 1, "aligned"), (dict(pages=-1), 1, "negative"),
                           (dict(width=1 << 28), 2, "2^31"), (dict(b=1 << 30), 2, "2^31"), (dict(), 1, "workspace"),
                           (dict(ws=264, nbytes=1 << 30), 1, "workspace")):
        rc, msg = call(**kw)
        assert rc == code and word in msg, (kw, rc, msg)


def test_rotary_abi():
    lib, s = _lib.load(), _lib.strides3(0, 128, 64)

    def call(dtype=0, x=256, h=2, d=64, axes=(32, 32), bases=(100.0, 100.0), pos=256, pos_type=0, b=1, strides=s):
        rc = lib.gw_rotary_axes(dtype, x, strides, 256, s, h, None, None, None, None, 0, pos_type, pos, s, b, 4, d, len(axes),
                                (ctypes.c_int32 * max(len(axes), 1))(*axes), (ctypes.c_double * max(len(axes), 1))(*bases), 0,
                                None)
        return rc, lib.gw_last_error().decode()

    for kw, code, word in ((dict(dtype=5), 1, "dtype"), (dict(d=300), 2, "head dim"), (dict(d=0), 1, "head dim"),
                           (dict(axes=(32, 33)), 1, "even"), (dict(axes=(-2, 32)), 1, "even"), (dict(axes=(64, 2)), 1, "exceed"),
                           (dict(axes=(2 ** 30, 2 ** 30)), 1, "exceed"), (dict(d=63, axes=(32, 30)), 1, "even"),
                           (dict(axes=(), bases=()), 1, "axes"), (dict(axes=(2,) * 9, bases=(1.0,) * 9), 1, "axes"),
                           (dict(bases=(100.0, -1.0)), 1, "base"), (dict(bases=(math.nan, 1.0)), 1, "base"),
                           (dict(pos=None), 1, "positions"), (dict(pos_type=3), 1, "position type"),
                           (dict(x=None), 1, "missing"), (dict(x=257), 1, "aligned"), (dict(b=70000), 2, "65535")):
        rc, msg = call(**kw)
        assert rc == code and word in msg, (kw, rc, msg)


def test_backward_abi():
    lib, s = _lib.load(), _lib.strides2(256, 64)
    need = lib.gw_packed_attn_bwd_workspace_size(1, 8, 8, 4, 4, 64)
    assert need >= 8 * 4 * 8

    def call(ws=256, nbytes=need, d=64, do=256, lse=256, rest=256):
        rc = lib.gw_packed_attn_bwd(0, 256, s, 256, s, 256, s, 256, 256, 256, s, rest, do, s, lse, 256, s, 256, s, 256, s, 1, 8, 8, 4,
                                    4, d, 0, 0.125, ws, nbytes, None)
        return rc, lib.gw_last_error().decode()

    for kw, code, word in ((dict(nbytes=need - 1), 1, "workspace"), (dict(ws=None), 1, "workspace"),
                           (dict(ws=264), 1, "workspace"), (dict(d=32), 2, "head dim"), (dict(do=None), 1, "missing"),
                           (dict(lse=None), 1, "missing"), (dict(do=260), 1, "aligned"), (dict(rest=None), 1, "missing"),
                           (dict(rest=8), 1, "aligned")):
        rc, msg = call(**kw)
        assert rc == code and word in msg, (kw, rc, msg)


def test_workspaces_are_bounded_by_the_sizes():
    """The parts of split keys stay below a few hundred MB however the sizes lie."""
    lib = _lib.load()
    for n, tq, tk in ((1, 1, 1 << 24), (1, 40, 1 << 24), (1, 1374, 1 << 20), (8, 40, 200000), (1000, 1000, 1 << 24),
                      (1, 1 << 22, 1 << 22), (64, 64 * 100, 1 << 22)):
        for hq, hk, d in ((16, 16, 64), (32, 1, 128)):
            fwd = lib.gw_packed_attn_fwd_workspace_size(n, tq, tk, hq, hk, d)
            assert fwd <= 1 << 29, (n, tq, tk, hq, hk, d, fwd)
    assert lib.gw_paged_attn_fwd_workspace_size(64, 1, 32, 8, 128) <= 1 << 26
    assert lib.gw_paged_attn_fwd_workspace_size(8192, 1, 32, 8, 128) == 0  # no split


def test_backward_workspaces_are_bounded_by_the_sizes():
    """Beside 8 bytes per (token, head) and per (sequence, key head), the parts stay below 512 MiB a pass."""
    lib = _lib.load()
    for n, tq, tk in ((1, 1, 1 << 24), (1, 40, 1 << 24), (1, 1374, 1 << 20), (8, 200000, 40), (1, 1 << 22, 1 << 22),
                      (200, 30000, 30000), (1, 8000, 8000)):
        for hq, hk, d in ((16, 16, 64), (32, 1, 128), (2, 1, 64)):
            got = lib.gw_packed_attn_bwd_workspace_size(n, tq, tk, hq, hk, d)
            assert got <= 8 * tq * hq + 8 * (n + 2) * hk + (1 << 30) + (1 << 17), (n, tq, tk, hq, hk, d, got)
