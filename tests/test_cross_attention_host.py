"""Cross attention: the C entries' refusals and workspace sizes (no GPU)."""

import ctypes

import pytest

from slimdit import _native

D = ctypes.c_void_p(16)


def view(ptr=16, b=0, s=0, h=0):
    return _native.View(ptr, b, s, h)


def call(dtype=_native.BF16, b=2, sq=4, sk=8, h=2, hk=2, d=64, q=None, k=None, out=None, mask=None, mask_type=0,
         lengths=None, bits=32, scale=0.125, ws=D, size=1 << 20):
    good = view(b=4096, s=512, h=64)
    return _native.load().slim_cross_attn(q or good, k or good, good, out or good, dtype, b, sq, sk, h, hk, d, mask,
                                          mask_type, 0, 1, lengths, bits, scale, ws, size, None)


@pytest.mark.parametrize("kwargs,code", [
    (dict(dtype=_native.F32), _native.SLIM_ERR_DTYPE),
    (dict(mask=D, mask_type=4), _native.SLIM_ERR_DTYPE),
    (dict(lengths=D, bits=16), _native.SLIM_ERR_DTYPE),
    (dict(d=136), _native.SLIM_ERR_SHAPE), (dict(d=60), _native.SLIM_ERR_SHAPE), (dict(d=0), _native.SLIM_ERR_SHAPE),
    (dict(h=3, hk=2), _native.SLIM_ERR_SHAPE), (dict(h=258, hk=2), _native.SLIM_ERR_SHAPE),
    (dict(h=0), _native.SLIM_ERR_SHAPE), (dict(sk=-1), _native.SLIM_ERR_SHAPE),
    (dict(sq=1 << 31), _native.SLIM_ERR_SHAPE), (dict(b=1 << 16), _native.SLIM_ERR_SHAPE),
    (dict(scale=0.0), _native.SLIM_ERR_SHAPE), (dict(scale=float("nan")), _native.SLIM_ERR_SHAPE),
    (dict(scale=float("inf")), _native.SLIM_ERR_SHAPE), (dict(scale=3e38), _native.SLIM_ERR_SHAPE),
    (dict(q=view(0)), _native.SLIM_ERR_NULL), (dict(k=view(0)), _native.SLIM_ERR_NULL),
    (dict(q=view(18)), _native.SLIM_ERR_ALIGN), (dict(k=view(s=65)), _native.SLIM_ERR_ALIGN),
    (dict(out=view(h=4)), _native.SLIM_ERR_ALIGN),
    (dict(mask=D, size=0), _native.SLIM_ERR_SHAPE), (dict(mask=D, ws=None), _native.SLIM_ERR_NULL),
    (dict(sq=0, q=view(0)), _native.SLIM_OK), (dict(b=0), _native.SLIM_OK),
])
def test_the_c_entry_refuses_before_any_device_work(kwargs, code):
    assert call(**kwargs) == code


def test_workspace_sizes():
    lib = _native.load()
    n = ctypes.c_uint64(0)
    assert lib.slim_cross_attn_workspace_bytes(2, 300, 77, 4, 4, 64, 1, ctypes.byref(n)) == _native.SLIM_OK
    assert n.value >= 2 * 128 * 4 + 2 * 4
    assert lib.slim_cross_attn_workspace_bytes(2, 300, 77, 4, 4, 64, 1, None) == _native.SLIM_ERR_NULL
    assert lib.slim_cross_attn_workspace_bytes(2, 300, 77, 4, 3, 64, 1, ctypes.byref(n)) == _native.SLIM_ERR_SHAPE


def layout(*shape):
    pieces, tiles = ctypes.c_int(-1), ctypes.c_int(-1)
    rc = _native.load().slim_cross_attn_layout(*shape, ctypes.byref(pieces), ctypes.byref(tiles))
    return rc, pieces.value, tiles.value


def test_layouts():
    assert layout(1, 4096, 4096, 40, 40, 128) == (_native.SLIM_OK, 0, 32)   # enough pairs of row tiles
    assert layout(1, 1, 200, 8, 8, 64) == (_native.SLIM_OK, 1, 2)           # too few keys to cut
    rc, pieces, tiles = layout(1, 1, 131071, 32, 8, 128)
    assert rc == _native.SLIM_OK and 1 < pieces <= 128 and (pieces - 1) * tiles < 1024 <= pieces * tiles
    assert layout(2, 300, 77, 4, 3, 64)[0] == _native.SLIM_ERR_SHAPE
    assert _native.load().slim_cross_attn_layout(1, 1, 1, 1, 1, 64, None, None) == _native.SLIM_ERR_NULL
    # one row tile a key head: never paired, however many there are
    assert layout(74, 1, 2048, 32, 8, 128)[1:] == layout(75, 1, 2048, 32, 8, 128)[1:] == (1, 16)
    assert layout(4000, 100, 300, 8, 8, 64)[1:] == (1, 3)
    # many rows: joining pieces of their keys costs more than it saves, few rows: it does not
    assert layout(2, 200, 4000, 24, 24, 64)[1] == 1 and layout(2, 7, 4000, 24, 24, 64)[1] > 1
