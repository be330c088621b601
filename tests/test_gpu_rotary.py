"""GPU parity of the rotary positions (slimdit.ops.rotary, csrc/rotary.cu) against the definition in
64 bits on the same inputs.

Tolerance. The definition's value is m (x cos a - y sin a). The kernel's cos and sin (times m) are
each within 2^-22 (1.5 ulp of sincospi below 1, the fraction of a turn rounded to fp32: 2^-25 of a
turn = 2^-22.3 radians, the product with m) of magnitude m, the three fp32 roundings add 2^-23 of
|x| + |y|: together 2^-21 m (|x| + |y|). The definition's own angle is rounded to 2^-53 of itself,
which far positions feel: |a| 2^-53 m (|x| + |y|) more. The rounding to the element type is half a step of the
result, eps/2 |result|, or half the smallest step for results near zero (fp16 subnormals).
"""

import numpy as np
import pytest
import torch

from slimdit import _native, ops, rope

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def definition(x, pos, freq, layout, sections, magnitude, inverse):
    """float64 result and the tolerance before the last rounding, on the CPU. x [B, S, H, D], pos [B, S, A]."""
    x, freq = x.double().cpu(), freq.double().cpu()
    n = freq.numel()
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    a = pos.cpu().double()[..., axis] * freq
    a = (-a if inverse else a)[:, :, None]
    i, j = (torch.arange(n), torch.arange(n) + n) if layout == "half" else (2 * torch.arange(n), 2 * torch.arange(n) + 1)
    u, v = x[..., i], x[..., j]
    y, size = x.clone(), torch.zeros_like(x)
    y[..., i] = magnitude * (u * a.cos() - v * a.sin())
    y[..., j] = magnitude * (u * a.sin() + v * a.cos())
    size[..., i] = size[..., j] = magnitude * (u.abs() + v.abs()) * (2.0**-21 + a.abs() * 2.0**-53)
    return y, size


def check(got, want, size):
    eps = torch.finfo(got.dtype).eps / 2
    floor = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    tol = want.abs() * eps * 1.001 + size + floor
    err = (got.cpu().double() - want).abs()
    assert torch.all(err <= tol), f"worst {float((err / tol).max()):.2f} of the tolerance"


def positions3(pos, b, s):
    p = pos if pos.dim() == 3 else pos.reshape(-1, s)[..., None] if pos.dim() == 2 else pos.reshape(1, s, -1)
    return p.expand(b, s, p.shape[-1])


def run(cuda, dtype, b, s, h, hk, d, rot, layout="half", sections=None, start=0, magnitude=1.0, inverse=False,
        inplace=False, pos32=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(b, s, h, d, device=cuda, generator=g).to(DT[dtype])
    k = torch.randn(b, s, hk, d, device=cuda, generator=g).to(DT[dtype]) if hk else None
    freq = torch.from_numpy(rope.rope_frequencies(rot)[0]).to(cuda)
    axes = 1 if sections is None else len(sections)
    pos = start + torch.randint(0, 5000, (b, s, axes), device=cuda, generator=g)
    arg = pos[..., 0] if sections is None else pos
    if pos32:
        arg = arg.to(torch.int32)
    q0, k0 = q.clone(), None if k is None else k.clone()
    out = ops.rotary(q, k, arg, freq, layout=layout, sections=sections, magnitude=magnitude, inverse=inverse,
                     inplace=inplace)
    for got, x, orig in zip((out,) if k is None else out, (q, k), (q0, k0)):
        want, size = definition(orig, pos, freq, layout, sections or (rot // 2,), magnitude, inverse)
        check(got, want, size)
        assert got.is_contiguous() and (got.data_ptr() == x.data_ptr()) == inplace
        if not inplace:
            assert torch.equal(x, orig)
    assert _native.device_error() == 0


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d,rot", [(128, 128), (64, 32), (80, 20), (6, 6), (66, 2), (96, 72), (256, 250), (2048, 2048),
                                   (1026, 1026)])
def test_heads_and_parts_of_all_widths(cuda, dtype, layout, d, rot):
    run(cuda, dtype, 2, 5, 3, 2, d, rot, layout=layout)


@pytest.mark.parametrize("b,s,h,hk", [(1, 1, 1, 0), (8, 1, 32, 8), (3, 1021, 5, 1), (1, 4099, 56, 56), (2, 17, 130, 0)])
@pytest.mark.parametrize("inplace", [False, True])
def test_batches_lengths_and_head_counts(cuda, b, s, h, hk, inplace):
    run(cuda, "bf16", b, s, h, hk, 128, 96, inplace=inplace)


@pytest.mark.parametrize("start", [-70000, 1 << 20, 2_000_000_000])
def test_far_and_negative_positions_keep_their_angle(cuda, start):
    run(cuda, "f32", 1, 64, 2, 0, 64, 64, start=start, magnitude=1.2, pos32=True)
    run(cuda, "f32", 1, 64, 2, 1, 64, 64, start=start * 8, layout="interleaved", inverse=True)


@pytest.mark.parametrize("sections", [(16, 16, 16), (0, 30, 18), (48,), (6,) * 8])
def test_several_position_axes(cuda, sections):
    run(cuda, "bf16", 2, 33, 4, 4, 128, 96, sections=sections)


def test_shared_and_broadcast_positions(cuda):
    q = torch.randn(3, 20, 2, 64, device=cuda)
    freq = torch.from_numpy(rope.rope_frequencies(64)[0]).to(cuda)
    pos = torch.randint(0, 900, (20,), device=cuda)
    want = ops.rotary(q, None, pos.expand(3, 20).contiguous(), freq)
    assert torch.equal(ops.rotary(q, None, pos, freq), want)
    assert torch.equal(ops.rotary(q, None, pos[None], freq), want)
    assert torch.equal(ops.rotary(q, None, pos.expand(3, 20), freq), want)
    wide = torch.stack([pos, pos + 1, pos], -1)            # strided positions
    assert torch.equal(ops.rotary(q, None, wide[:, 2], freq), want)
    assert torch.equal(ops.rotary(q[0], None, pos, freq), want[0])


def test_views_of_a_packed_buffer_and_other_strides(cuda):
    b, s, h, d = 2, 37, 4, 64
    freq = torch.from_numpy(rope.rope_frequencies(48)[0]).to(cuda)
    pos = torch.arange(s, device=cuda)
    for pitch in (3 * h * d, 3 * h * d + 8, 3 * h * d + 1):     # 16-byte rows, and rows that are not
        rows = torch.randn(b, s, pitch, device=cuda).to(torch.bfloat16)
        q = rows[..., :h * d].unflatten(-1, (h, d))
        k = rows[..., h * d:2 * h * d].unflatten(-1, (h, d))
        rest = rows[..., 2 * h * d:].clone()
        want = ops.rotary(q.contiguous(), k.contiguous(), pos, freq)
        got = ops.rotary(q, k, pos, freq)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        out = ops.rotary(q, k, pos, freq, inplace=True)
        assert out[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])
        assert torch.equal(rows[..., 2 * h * d:], rest)         # v and the pitch stay as they were
    x = torch.randn(b, h, s, d, device=cuda)                    # heads before tokens
    want = ops.rotary(x.transpose(1, 2).contiguous(), None, pos, freq)
    assert torch.equal(ops.rotary(x.transpose(1, 2), None, pos, freq), want)
    shared = torch.randn(1, s, 1, d, device=cuda).expand(b, s, h, d)
    assert torch.equal(ops.rotary(shared, None, pos, freq), ops.rotary(shared.contiguous(), None, pos, freq))
    odd = torch.randn(s * h * d + 1, device=cuda)[1:].view(s, h, d)  # 4-byte aligned base
    assert torch.equal(ops.rotary(odd, None, pos, freq), ops.rotary(odd.clone(), None, pos, freq))
    back = torch.randn(s, h, 2 * d, device=cuda)[..., ::2]      # elements apart: copied
    assert torch.equal(ops.rotary(back, None, pos, freq), ops.rotary(back.contiguous(), None, pos, freq))
    part = torch.randn(s, h, 96, device=cuda)                   # the last 48 of 96 elements, in place
    keep = part[..., :48].clone()
    want = ops.rotary(part[..., 48:].contiguous(), None, pos, freq)
    ops.rotary(part[..., 48:], None, pos, freq, inplace=True)
    assert torch.equal(part[..., 48:], want) and torch.equal(part[..., :48], keep)


def test_the_inverse_undoes_and_transposes(cuda):
    freq, m = rope.rope_frequencies(64, scaling="yarn", factor=8.0, original_length=1024)
    freq = torch.from_numpy(freq).to(cuda)
    pos = torch.randint(0, 100000, (2, 50), device=cuda)
    x, y = torch.randn(2, 2, 50, 3, 80, device=cuda)
    rx = ops.rotary(x, None, pos, freq, magnitude=m)
    back = ops.rotary(rx, None, pos, freq, magnitude=1 / m, inverse=True)
    assert torch.all((back - x).abs() <= 2.0**-18 * (1 + x.abs().amax(-1, keepdim=True)))
    # <R x, y> = <x, R^T y>: the gradient of the rotation is the rotation back
    ry = ops.rotary(y, None, pos, freq, magnitude=m, inverse=True)
    a, b = (rx.double() * y.double()).sum(), (x.double() * ry.double()).sum()
    assert abs(float(a - b)) <= 2.0**-19 * float((rx.abs().double() * y.abs().double()).sum())


def test_non_finite_values_stay_in_their_pair(cuda):
    x = torch.randn(1, 4, 2, 64, device=cuda)
    x[0, 1, 0, 3] = float("nan")
    x[0, 2, 1, 40] = float("inf")
    freq = torch.from_numpy(rope.rope_frequencies(64)[0]).to(cuda)
    y = ops.rotary(x, None, torch.arange(1, 5, device=cuda), freq)
    bad = (~torch.isfinite(y)).nonzero().tolist()
    assert bad == [[0, 1, 0, 3], [0, 1, 0, 35], [0, 2, 1, 8], [0, 2, 1, 40]]


def test_another_stream_and_a_captured_call(cuda):
    x = torch.randn(2, 300, 8, 128, device=cuda).to(torch.bfloat16)
    freq = torch.from_numpy(rope.rope_frequencies(128)[0]).to(cuda)
    pos = torch.arange(300, device=cuda)
    want = ops.rotary(x, None, pos, freq)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.rotary(x, None, pos, freq)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.rotary(x, None, pos, freq)
    pos += 7
    x.neg_()
    graph.replay()
    assert torch.equal(out, ops.rotary(x, None, pos, freq)) and not torch.equal(out, want)


def test_empty_inputs(cuda):
    freq = torch.from_numpy(rope.rope_frequencies(64)[0]).to(cuda)
    for b, s in ((0, 4), (2, 0)):
        q, k = ops.rotary(torch.empty(b, s, 3, 64, device=cuda), torch.empty(b, s, 1, 64, device=cuda),
                          torch.empty(b, s, dtype=torch.int64, device=cuda), freq)
        assert q.shape == (b, s, 3, 64) and k.shape == (b, s, 1, 64)


def test_refusals(cuda):
    freq = torch.from_numpy(rope.rope_frequencies(64)[0]).to(cuda)
    q = torch.zeros(2, 4, 2, 64, device=cuda)
    pos = torch.arange(4, device=cuda)
    for bad, error in [
        (lambda: ops.rotary(q.cpu(), None, pos, freq), TypeError),
        (lambda: ops.rotary(q.long(), None, pos, freq), TypeError),
        (lambda: ops.rotary(q[0, 0], None, pos, freq), ValueError),
        (lambda: ops.rotary(q, None, pos.float(), freq), TypeError),
        (lambda: ops.rotary(q, None, pos[:3], freq), ValueError),
        (lambda: ops.rotary(q, None, pos.cpu(), freq), ValueError),
        (lambda: ops.rotary(q, None, pos, freq, layout="whole"), ValueError),
        (lambda: ops.rotary(q, None, pos, freq, sections=(16, 16)), ValueError),
        (lambda: ops.rotary(q, None, torch.zeros(4, 2, device=cuda, dtype=torch.int64), freq, sections=(16, 8)), ValueError),
        (lambda: ops.rotary(q[..., :32], None, pos, freq), ValueError),
        (lambda: ops.rotary(q, q[:, :3], pos, freq), ValueError),
        (lambda: ops.rotary(q, q.half(), pos, freq), ValueError),
        (lambda: ops.rotary(q, q, pos, freq, inplace=True), ValueError),
        (lambda: ops.rotary(q[:, :, :1].expand(2, 4, 2, 64), None, pos, freq, inplace=True), ValueError),
        (lambda: ops.rotary(torch.zeros(4, 2, 128, device=cuda)[..., ::2], None, pos, freq, inplace=True), ValueError),
        (lambda: ops.rotary(q.clone().requires_grad_(), None, pos, freq), ValueError),
    ]:
        with pytest.raises(error):
            bad()
    with torch.no_grad():
        ops.rotary(q.clone().requires_grad_(), None, pos, freq)


def test_against_differences(cuda):
    """The derivative along a direction equals the rotation of the direction (the operator is linear)."""
    freq = torch.from_numpy(rope.rope_frequencies(32)[0]).to(cuda)
    pos = torch.arange(9, device=cuda) * 1000
    x, dx = torch.randn(2, 9, 2, 40, device=cuda)
    step = 2.0**-6
    diff = (ops.rotary(x + step * dx, None, pos, freq).double() - ops.rotary(x, None, pos, freq).double()) / step
    # rounding of x + step dx and of the two results: 2^-23 of values below 8 each, over the step
    assert torch.all((diff - ops.rotary(dx, None, pos, freq).double()).abs() <= 4 * 8 * 2.0**-23 / step)
    assert np.isfinite(diff.cpu().numpy()).all()
