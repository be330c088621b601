"""GPU parity of cross attention's layouts (csrc/cross_attn.cu) where a row's maximum grows along the keys,
so that the weights are taken again and the sums and the output rescaled inside a CTA.

The tolerance is the one of test_gpu_cross_attention.py, per output element. The values shrink as the
weights grow, so that a tile's share of the result stays within what the tolerance tells apart.
"""

import ctypes
import math

import pytest
import torch

from slimdit import _native, attention
from test_gpu_cross_attention import check, inputs

pytestmark = pytest.mark.gpu


def rising(cuda, dtype, b, sq, sk, h, hk, d):
    """Logits that rise by 6 (2^8.7), by 3, not at all or fall by 6 from one 128-key tile to the next,
    neighbouring rows differently; values that shrink by 2^-8 (fp16: 2^-2) a tile."""
    q, k, v = inputs(cuda, dtype, b, sq, sk, h, hk, d, peak=1.0)
    tile = (torch.arange(sk, device=cuda) // 128).float()
    slope = torch.tensor([1.0, 0.5, 0.0, -1.0], device=cuda) * d**0.5
    row = torch.arange(sq, device=cuda)[:, None] + torch.arange(h, device=cuda)
    q[..., 0] = slope[row % 4].to(q.dtype)
    k[..., 0] = (6 * tile)[:, None].to(k.dtype)
    v = (v.float() * torch.exp2(tile * (-8 if dtype == "bf16" else -2))[:, None, None]).to(v.dtype)
    return q, k, v


def layout(b, sq, sk, h, hk, d):
    """(pieces of a row tile's keys, 0 for pairs of row tiles; most key tiles of one)"""
    pieces, tiles = ctypes.c_int(), ctypes.c_int()
    _native.check(_native.load().slim_cross_attn_layout(b, sq, sk, h, hk, d, pieces, tiles))
    return pieces.value, tiles.value


def run(cuda, dtype, kind, b, sq, sk, h, hk, d):
    q, k, v = rising(cuda, dtype, b, sq, sk, h, hk, d)
    bias = mask = None
    if kind != "none":  # whole tiles without keys in front, holes, and one key alone in the last sequence
        g = torch.Generator(device="cuda").manual_seed(11)
        keep = torch.rand(b, sk, device=cuda, generator=g) < 0.8
        keep[:, :300] = False
        keep[:, -1] = True
        if b > 1:
            keep[-1, :-1] = False
        bias = torch.where(keep, 0.0, -math.inf)
        mask = keep
        if kind == "additive":
            bias = mask = bias + torch.randn(b, sk, device=cuda, generator=g)
        k[~keep], v[~keep] = math.nan, math.nan
    check(attention.cross_attention(q, k, v, key_mask=mask), q, k, v, bias)


NARROW = [(1, 130, 640, 2, 2, 64), (1, 130, 640, 2, 2, 128), (2, 50, 600, 6, 2, 128), (1, 1, 700, 8, 8, 64),
          (301, 1, 600, 2, 2, 64), (75, 3, 390, 16, 8, 128)]   # more row tiles than four an SM, one a key head
PIECES = [(1, 130, 2560, 20, 20, 128), (2, 40, 2500, 30, 10, 64)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("kind", ["none", "bool", "additive"])
@pytest.mark.parametrize("shape", NARROW + PIECES)
def test_a_maximum_that_grows_within_a_row_tile(cuda, shape, kind, dtype):
    pieces, tiles = layout(*shape)
    assert tiles >= 3 and (pieces == 1 if shape in NARROW else pieces > 1), "the shape no longer gives this layout"
    run(cuda, dtype, kind, *shape)


# pairs of row tiles, and (9 of them) a single one at the end
WIDE = [(2, 1000, 1000, 40, 40, 64), (2, 1100, 640, 40, 40, 128), (1, 1300, 700, 48, 24, 72)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("kind", ["none", "bool", "additive"])
@pytest.mark.parametrize("shape", WIDE)
def test_a_maximum_that_grows_within_a_pair_of_row_tiles(cuda, shape, kind, dtype):
    assert layout(*shape)[0] == 0 and layout(*shape)[1] >= 5, "the shape no longer gives this layout"
    run(cuda, dtype, kind, *shape)


@pytest.mark.parametrize("shape", [NARROW[0], PIECES[0], WIDE[1]])
@pytest.mark.parametrize("at", [0, 77, -1])
@pytest.mark.parametrize("kind", ["none", "additive"])
def test_a_long_tail_behind_one_key_that_takes_nearly_all(cuda, shape, at, kind):
    """One key about 2^25 times as heavy as each of the others, its value 0: what is left is the tail's. Logits
    without rounding (one element of q and k, scale 1). The largest weight of a row is held as 2^7 or more, so a
    tiny weight is off by half a step of fp16, 2^-25, over 2^7 of the largest; the other roundings as in
    test_gpu_cross_attention.py."""
    b, sq, sk, h, hk, d = shape
    _, _, v = inputs(cuda, "f16", *shape)
    q, k = torch.zeros(b, sq, h, d, device=cuda).half(), torch.zeros(b, sk, hk, d, device=cuda).half()
    q[..., 0] = (1 - 0.03 * (torch.arange(sq, device=cuda) % 4))[:, None].half()
    k[:, at, :, 0] = 17.5
    v[:, at] = 0
    bias = torch.linspace(-1, 0, sk, device=cuda)[None].expand(b, sk) if kind == "additive" else None
    got = attention.cross_attention(q, k, v, key_mask=bias, scale=1.0).double()
    logit = torch.einsum("bqhd,bkhd->bhqk", q[..., :1].double(), k[..., :1].double().repeat_interleave(h // hk, 2))
    if bias is not None:
        logit = logit + bias.double()[:, None, None]
    w = torch.softmax(logit, -1)
    z = v.double().repeat_interleave(h // hk, 2).permute(0, 2, 1, 3)
    want, mass = ((w @ x).transpose(1, 2) for x in (z, z.abs()))
    eps, half_step = 2.0**-11, 2.0**-25
    tol = (eps * 1.01 + 2 * 20 * 2.0**-21 + 2.0**-20) * mass + eps * 1.01 * want.abs() + half_step \
        + 2.0**-32 * z.abs().sum(2)[:, None]
    err = (got - want).abs()
    assert torch.all(err <= tol), f"worst {float((err / tol).max()):.3f} of the tolerance"
    assert float((tol / mass).median()) < 0.1   # the tolerance does tell the tail from nothing


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", [NARROW[0], PIECES[0], WIDE[1]])
def test_logits_whose_own_steps_exceed_one_give_an_average_still(cuda, shape, dtype):
    """Logits of 10^7 and more, which 32 bits hold to a whole number at best: every result is an average of values
    all the same, within the roundings of its weights and of itself."""
    q, k, v = inputs(cuda, dtype, *shape)
    q, k = (q.float() * 500).to(q.dtype), (k.float() * 1000).to(k.dtype)
    out = attention.cross_attention(q, k, v, scale=1.0).double()
    most = v.double().abs().amax(1).repeat_interleave(shape[3] // shape[4], 1)[:, None] * (1 + 2 * torch.finfo(q.dtype).eps)
    assert bool((out.abs() <= most).all())
    # a far larger score than any other takes all
    k[:, 5] = k[:, 5].abs() + 20000
    out = attention.cross_attention(q.abs(), k, v, scale=1.0)
    assert torch.equal(out, v[:, 5:6].repeat_interleave(shape[3] // shape[4], 2).expand_as(out))
