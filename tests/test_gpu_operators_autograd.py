"""Rotary positions and cross attention beside autograd: they record nothing, so tensors that expect a derivative are
refused and those written in place are marked as changed."""

import pytest
import torch
from torch.autograd import forward_ad

from slimdit import attention, ops

pytestmark = pytest.mark.gpu


@pytest.fixture
def qkv(cuda):
    g = torch.Generator(device="cuda").manual_seed(1)
    return tuple(torch.randn(1, 6, 2, 64, device=cuda, generator=g).to(torch.bfloat16) for _ in range(3))


def test_learned_frequencies_and_scales_are_refused(cuda, qkv):
    q, k, v = qkv
    pos, freq = torch.arange(6, device=cuda), torch.rand(32, device=cuda)
    learned = freq.clone().requires_grad_()
    with pytest.raises(ValueError, match="backward"):
        ops.rotary(q, k, pos, learned)
    with torch.no_grad():
        assert torch.equal(ops.rotary(q, None, pos, learned), ops.rotary(q, None, pos, freq))
    with pytest.raises(ValueError, match="backward"):
        attention.cross_attention(q, k, v, scale=torch.tensor(0.1, requires_grad=True))


@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_forward_mode_duals_are_refused(cuda, qkv, which):
    pos, freq = torch.arange(6, device=cuda), torch.rand(32, device=cuda)
    with torch.no_grad(), forward_ad.dual_level():
        args = [*qkv, torch.zeros(1, 6, device=cuda)]
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(ValueError, match="forward"):
            attention.cross_attention(*args)
        turned = [args[0], args[1], pos, freq]
        if which >= 2:
            turned[3] = forward_ad.make_dual(freq, torch.ones_like(freq))
        for inplace in (False, True):
            before = qkv[0].clone()
            with pytest.raises(ValueError, match="forward"):
                ops.rotary(*turned, inplace=inplace)
            assert torch.equal(qkv[0], before)


def test_a_rotation_in_place_is_seen_by_autograd(cuda, qkv):
    q, k, _ = qkv
    pos, freq = torch.arange(6, device=cuda), torch.rand(32, device=cuda)
    w = torch.ones(64, device=cuda, dtype=q.dtype, requires_grad=True)
    versions = q._version, k._version
    with torch.no_grad():
        ops.rotary(q, k, pos, freq)
    assert (q._version, k._version) == versions
    loss = (w * q).sum()                    # saves q
    ops.rotary(q, k, pos, freq, inplace=True)
    assert q._version > versions[0] and k._version > versions[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    loss = (w * k).sum()
    ops.rotary(k[0], None, pos, freq, inplace=True)   # a view of it, without a batch
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        made = torch.ones(1, 6, 2, 64, device=cuda)
        want = ops.rotary(made, None, pos, freq)
        assert ops.rotary(made, None, pos, freq, inplace=True) is made and torch.equal(made, want)
