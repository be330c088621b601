"""The rotation in place on the packed qkv buffer and the packed attention after it, as a block of the DiT runs them."""

import pytest
import torch

from slimdit import attention, ops, rope

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seq,heads", [(1, 1), (333, 3), (1024, 2)])
@pytest.mark.parametrize("sections", [None, (16, 16, 16)])
def test_the_packed_buffer_is_rotated_in_place_and_attended(cuda, seq, heads, sections):
    g = torch.Generator(device="cuda").manual_seed(seq)
    width = heads * 128
    rows = torch.randn(seq, 3 * width, device=cuda, generator=g).to(torch.bfloat16)
    freq, magnitude = rope.rope_frequencies(96 if sections is None else 32, scaling="yarn", factor=2.0, original_length=512)
    freq = torch.from_numpy(freq).to(cuda).repeat(1 if sections is None else 3)
    token = torch.arange(seq, device=cuda)
    pos = token if sections is None else torch.stack([token // 64, token // 8 % 8, token % 8], -1)

    def views(buf):
        return tuple(buf[:, i * width:(i + 1) * width].unflatten(-1, (heads, 128)) for i in range(3))

    q, k, v = views(rows)
    qr, kr = ops.rotary(q, k, pos, freq, sections=sections, magnitude=magnitude)
    apart = torch.cat([t.flatten(1) for t in (qr, kr, v)], -1)
    ops.rotary(q, k, pos, freq, sections=sections, magnitude=magnitude, inplace=True)
    assert torch.equal(rows, apart)
    out = attention.attention_packed(rows, heads)
    assert out.shape == (seq, width) and torch.isfinite(out).all()
    assert torch.equal(out, attention.attention_packed(apart, heads))
    # the rotation turns q and k alike: one constant position for all leaves every product, but for magnitude^2
    same = torch.full_like(pos, 1234)
    again = torch.cat([t.flatten(1) for t in (*ops.rotary(*views(apart)[:2], same, freq, sections=sections), v)], -1)
    a, b = (attention.cross_attention(*views(x)) for x in (apart, again))
    # q and k are rounded once more, by half a step of 2^-8 each: a logit moves by 2 * 2^-8 of |q| |k| / sqrt(128)
    # at most, a weight by twice that in the exponent; the weights and the results are rounded apart, 4 * 2^-8
    x, y, z = (t.double().transpose(0, 1) for t in views(apart))
    moved = 2.02 * 2.0**-8 * 128**-0.5 * x.norm(dim=-1, keepdim=True) * y.norm(dim=-1).amax(-1)[:, None, None]
    w = torch.softmax(x @ y.transpose(1, 2) * 128**-0.5, -1)
    tol = (((2 * moved).exp() - 1 + 4 * 2.0**-8) * (w @ z.abs())).transpose(0, 1)
    assert bool(((a - b).abs().double() <= tol).all())
