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
