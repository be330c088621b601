"""Rotary positions: the frequency tables, the checks of arguments and the C entry's refusals (no GPU)."""

import ctypes
import math

import numpy as np
import pytest
import torch

from slimdit import _native, ops, rope


def test_the_checkpoint_table_is_the_plain_table_of_its_length():
    f, m = rope.rope_frequencies(32)
    assert f.dtype == np.float32 and m == 1.0
    # both evaluate 10000^(-k/16); the checkpoint's in float32 throughout
    assert np.allclose(f, rope.rope_inv_freq(), rtol=4 * 2.0**-23)


@pytest.mark.parametrize("rot", [2, 20, 64, 128])
def test_scalings_change_what_they_say(rot):
    f, _ = rope.rope_frequencies(rot, theta=50000.0)
    assert f[0] == 1.0 and f.shape == (rot // 2,)
    lin, m = rope.rope_frequencies(rot, theta=50000.0, scaling="linear", factor=4.0)
    assert np.allclose(lin, f / 4) and m == 1.0
    ntk, _ = rope.rope_frequencies(rot, theta=50000.0, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0
    if rot > 2:
        assert np.isclose(ntk[-1], f[-1] / 4, rtol=1e-6)
    yarn, m = rope.rope_frequencies(rot, theta=50000.0, scaling="yarn", factor=4.0, original_length=4096)
    parts, one = rope.rope_frequencies(rot, theta=50000.0, scaling="parts", factor=4.0, original_length=4096)
    assert np.array_equal(yarn, parts) and one == 1.0 and math.isclose(m, 0.1 * math.log(4) + 1)
    turns = 4096 * f.astype(np.float64) / (2 * math.pi)
    assert np.allclose(yarn[turns >= 32], f[turns >= 32]) and np.allclose(yarn[turns <= 1], f[turns <= 1] / 4)
    assert np.all((yarn <= f * (1 + 1e-6)) & (yarn >= f / 4 * (1 - 1e-6)))


@pytest.mark.parametrize("kwargs", [dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=8, scaling="cubic"),
                                    dict(rot_dim=8, scaling="yarn", factor=2.0), dict(rot_dim=8, factor=0.5),
                                    dict(rot_dim=8, theta=0.0),
                                    dict(rot_dim=8, scaling="parts", original_length=10, slow=4, fast=4)])
def test_frequencies_refuse(kwargs):
    with pytest.raises(ValueError):
        rope.rope_frequencies(**kwargs)


def test_shared_memory_is_recognised():
    buf = torch.zeros(2, 6, 3 * 4 * 8)
    q = buf[..., :32].unflatten(-1, (4, 8))
    k = buf[..., 32:64].unflatten(-1, (4, 8))
    assert not ops._share(q, k) and not ops._share(k, q)
    assert ops._share(q, q) and ops._share(q, buf[..., 24:56].unflatten(-1, (4, 8)))
    assert not ops._share(q[:, :1], k[:, :1])              # one token of two sequences
    assert not ops._share(q[:1, :1], k[:1, :1])            # one token
    assert ops._share(q[:, :1], q[:, :1])
    apart = torch.zeros(2, 2, 4, 6, 8)
    assert not ops._share(apart[0].transpose(1, 2), apart[1].transpose(1, 2))
    assert ops._share(apart[0].transpose(1, 2), apart[0].transpose(1, 2))
    # the last rows of k wrap into the next row's q
    assert ops._share(q, buf.view(-1)[80:80 + 2 * 5 * 96].view(2, 5, 96)[..., :32].unflatten(-1, (4, 8)))
    assert ops._spans_overlap(torch.zeros(1, 1, 4, 8).expand(1, 3, 4, 8))
    assert not ops._spans_overlap(q) and not ops._spans_overlap(apart[0].transpose(1, 2))
    assert ops._spans_overlap(torch.zeros(64).as_strided((1, 4, 2, 8), (64, 8, 4, 1)))


def test_the_c_entry_refuses_before_any_device_work():
    lib = _native.load()
    v = _native.View(16, 0, 0, 0)
    d = ctypes.c_void_p(16)

    def call(dtype=1, batch=1, seq=4, heads=2, heads_k=0, dim=64, rot=64, layout=0, bits=64, sections=None, axes=1,
             q=v, k=None, pos=d):
        sec = None if sections is None else (ctypes.c_int * len(sections))(*sections)
        return lib.slim_rotary(q, q, heads, k, k, heads_k, dtype, batch, seq, dim, rot, layout, pos, bits, 0, 1, 0, d,
                               sec, axes, 1.0, 0, None)

    assert call(dtype=7) == _native.SLIM_ERR_DTYPE
    assert call(layout=2) == _native.SLIM_ERR_DTYPE
    assert call(bits=16) == _native.SLIM_ERR_DTYPE
    assert call(rot=66) == _native.SLIM_ERR_SHAPE
    assert call(rot=7) == _native.SLIM_ERR_SHAPE
    assert call(rot=0) == _native.SLIM_ERR_SHAPE
    assert call(dim=4096) == _native.SLIM_ERR_SHAPE
    assert call(heads=0) == _native.SLIM_ERR_SHAPE
    assert call(seq=-1) == _native.SLIM_ERR_SHAPE
    assert call(batch=1 << 20, seq=1 << 20) == _native.SLIM_ERR_SHAPE
    assert call(axes=3) == _native.SLIM_ERR_SHAPE                       # sections missing
    assert call(axes=3, sections=(16, 16, 1)) == _native.SLIM_ERR_SHAPE  # 33 of 32 pairs
    assert call(axes=3, sections=(16, 8, 4)) == _native.SLIM_ERR_SHAPE
    assert call(axes=9, sections=(4,) * 9) == _native.SLIM_ERR_SHAPE
    assert call(q=None) == _native.SLIM_ERR_NULL
    assert call(heads_k=1) == _native.SLIM_ERR_NULL
    assert call(pos=None) == _native.SLIM_ERR_NULL
    assert call(seq=0) == _native.SLIM_OK
    assert call(batch=0, q=None) == _native.SLIM_OK


def test_tensors_that_expect_a_derivative_are_refused():
    from torch.autograd import forward_ad

    x = torch.zeros(3)
    ops._no_grad(x, None, 1.0)
    with pytest.raises(ValueError, match="backward"):
        ops._no_grad(None, x.clone().requires_grad_())
    with torch.no_grad():
        ops._no_grad(x.clone().requires_grad_())
        with forward_ad.dual_level():   # which no_grad does not close
            dual = forward_ad.make_dual(x, torch.ones(3))
            ops._no_grad(x, dual.detach())
            with pytest.raises(ValueError, match="forward"):
                ops._no_grad(x, dual)
    with pytest.raises(ValueError, match="forward"):
        torch.func.jvp(lambda t: (ops._no_grad(t), t)[1], (x,), (x,))
