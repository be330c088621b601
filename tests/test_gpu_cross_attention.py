"""GPU parity of cross attention (slimdit.attention.cross_attention, csrc/cross_attn.cu) against the
definition in 64 bits on the same inputs.

Tolerance, per output element, with weights w (sum 1), A = sum w |v| and o = sum w v:
* a logit is off by at most d = 2^-20 scale sum|q k| (fp32 accumulation in the tensor core) plus
  2^-21 of the largest logit and bias (fp32 scaling, bias and exponent argument); a weight is then off
  by d relative in numerator and sum: 2 d A (d << 1), with 2^-20 A for exponential, sum and division;
* weights are rounded to the type of v for the second product: eps/2 A, and half the type's smallest
  step for tiny ones, absolute against the largest weight 1: step/2 * sum|v| / l with l >= 1 the sum of
  weights relative to the largest;
* the result is rounded once: eps/2 |o|, half the smallest step near zero.
"""

import math

import pytest
import torch

from slimdit import _native, attention, ops, rope

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def definition(q, k, v, bias, scale):
    """(o, tolerance) in float64; q [B, Sq, H, D], bias [B, Skv] with -inf for excluded keys."""
    dt = q.dtype
    eps, tiny = torch.finfo(dt).eps / 2, torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2
    b, sq, h, d = q.shape
    g = h // k.shape[2]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o) + tiny
    for i in range(b):
        use = (bias[i] > -math.inf).nonzero().flatten()
        if use.numel() == 0:
            continue
        add = bias[i, use].double()
        add = add - add.max()
        for j in range(h):
            x, y, z = q[i, :, j].double(), k[i, use, j // g].double(), v[i, use, j // g].double()
            s = scale * x @ y.T
            size = scale * (x.abs() @ y.abs().T).amax(-1, keepdim=True)
            logit = s + add
            top = logit.amax(-1, keepdim=True)
            e = (logit - top).exp()
            l = e.sum(-1, keepdim=True)
            near = torch.where(logit > top - 200, logit.abs() + add.abs(), 0.0).amax(-1, keepdim=True)
            delta = 2.0**-20 * size + 2.0**-21 * near
            o[i, :, j] = e @ z / l
            mass = e @ z.abs() / l
            tol[i, :, j] += (eps * 1.01 + 2 * delta + 2.0**-20) * mass + eps * 1.01 * o[i, :, j].abs() \
                + tiny * z.abs().sum(0) / l
    return o, tol


def check(got, q, k, v, bias=None, scale=None):
    if bias is None:
        bias = torch.zeros(k.shape[:2], device=q.device)
    want, tol = definition(q, k, v, bias, q.shape[-1] ** -0.5 if scale is None else scale)
    assert got.shape == q.shape and got.dtype == q.dtype and got.is_contiguous()
    err = (got.double() - want).abs()
    assert torch.all(err <= tol), f"worst {float((err / tol).max()):.3f} of the tolerance at " \
        f"{torch.unravel_index((err / tol).argmax(), err.shape)}"
    assert _native.device_error() == 0
    return want


def inputs(cuda, dtype, b, sq, sk, h, hk, d, seed=0, peak=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed + 7919 * sq + 104729 * sk + d)
    q = (torch.randn(b, sq, h, d, device=cuda, generator=g) * peak).to(DT[dtype])
    k = torch.randn(b, sk, hk, d, device=cuda, generator=g).to(DT[dtype])
    v = torch.randn(b, sk, hk, d, device=cuda, generator=g).to(DT[dtype])
    return q, k, v


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("sk", [1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 640, 1003])
@pytest.mark.parametrize("sq", [1, 16, 130])
def test_key_lengths(cuda, dtype, sq, sk):
    q, k, v = inputs(cuda, dtype, 1, sq, sk, 2, 2, 128)
    check(attention.cross_attention(q, k, v), q, k, v)


@pytest.mark.parametrize("d", [8, 16, 40, 64, 72, 80, 96, 120, 128])
@pytest.mark.parametrize("sq,sk", [(1, 300), (3, 40), (200, 333)])
def test_head_sizes(cuda, d, sq, sk):
    q, k, v = inputs(cuda, "bf16", 2, sq, sk, 3, 3, d)
    check(attention.cross_attention(q, k, v), q, k, v)


@pytest.mark.parametrize("sq", [1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 385, 511, 513, 1000])
@pytest.mark.parametrize("d", [64, 128])
def test_query_lengths(cuda, sq, d):
    q, k, v = inputs(cuda, "bf16", 1, sq, 200, 2, 1, d)
    check(attention.cross_attention(q, k, v), q, k, v)


@pytest.mark.parametrize("h,hk", [(1, 1), (8, 1), (6, 2), (7, 1), (32, 8), (56, 56), (128, 1), (65, 1), (200, 2)])
@pytest.mark.parametrize("sq", [1, 5, 150])
def test_grouped_heads(cuda, h, hk, sq):
    q, k, v = inputs(cuda, "f16", 2, sq, 190, h, hk, 64)
    check(attention.cross_attention(q, k, v), q, k, v)


@pytest.mark.parametrize("sq,sk,h,hk,b,d", [(1, 20011, 8, 2, 1, 128), (1, 131071, 4, 1, 1, 128), (4, 9000, 16, 16, 1, 64),
                                            (1, 1500, 16, 16, 4, 64), (17, 40000, 1, 1, 1, 128), (2, 5000, 3, 3, 2, 72)])
def test_few_queries_over_many_keys(cuda, sq, sk, h, hk, b, d):
    q, k, v = inputs(cuda, "bf16", b, sq, sk, h, hk, d)
    check(attention.cross_attention(q, k, v), q, k, v)


@pytest.mark.parametrize("b,sq,sk,h,d", [(1, 4099, 512, 8, 128), (2, 1024, 2048, 4, 64), (1, 2500, 77, 24, 128)])
def test_many_queries(cuda, b, sq, sk, h, d):
    q, k, v = inputs(cuda, "bf16", b, sq, sk, h, h, d)
    check(attention.cross_attention(q, k, v), q, k, v)


SHAPES = [(1, 300, 4, 2, 64), (130, 300, 2, 2, 128), (300, 130, 3, 1, 72), (1, 4000, 2, 1, 128)]


@pytest.mark.parametrize("sq,sk,h,hk,d", SHAPES)
@pytest.mark.parametrize("wide", [False, True])
def test_lengths(cuda, sq, sk, h, hk, d, wide):
    lens = [0, 1, sk // 2, sk - 1, sk, sk + 50, -3, 128]
    q, k, v = inputs(cuda, "bf16", len(lens), sq, sk, h, hk, d)
    lengths = torch.tensor(lens, device=cuda, dtype=torch.int64 if wide else torch.int32)
    keep = torch.arange(sk, device=cuda) < lengths[:, None]
    for bad in (math.nan, math.inf, 1e4):   # whatever stands behind the last key
        k[~keep], v[~keep] = bad, bad
        want = check(attention.cross_attention(q, k, v, kv_lengths=lengths), q, k, v,
                     torch.where(keep, 0.0, -math.inf))
        assert torch.all(want[0] == 0) and torch.all(want[6] == 0)


@pytest.mark.parametrize("sq,sk,h,hk,d", SHAPES)
@pytest.mark.parametrize("kind", ["bool", "f32", "bf16", "f16"])
def test_masks(cuda, sq, sk, h, hk, d, kind):
    b = 6
    q, k, v = inputs(cuda, "f16", b, sq, sk, h, hk, d)
    g = torch.Generator(device="cuda").manual_seed(5)
    keep = torch.rand(b, sk, device=cuda, generator=g) < 0.6
    keep[0] = False                       # nothing left
    keep[1, :-1], keep[1, -1] = False, True   # the last key alone
    keep[2] = True
    keep[3, : sk // 2] = False            # whole tiles in front
    keep[4, sk // 2:] = False             # and behind
    if kind == "bool":
        mask = keep
        bias = torch.where(keep, 0.0, -math.inf)
    else:
        dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[kind]
        mask = torch.where(keep, torch.randn(b, sk, device=cuda, generator=g) * 3, -math.inf).to(dt)
        bias = mask.float()
    k[~keep], v[~keep] = math.nan, math.nan
    out = attention.cross_attention(q, k, v, key_mask=mask)
    check(out, q, k, v, bias)
    assert torch.all(out[0] == 0)
    assert torch.equal(attention.cross_attention(q, k, v, key_mask=mask[:, None, None]), out)
    wide = torch.stack([mask, mask], -1)[..., 0]   # strided
    assert torch.equal(attention.cross_attention(q, k, v, key_mask=wide), out)


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sq", [1, 140])
def test_lowest_values_mask_and_a_row_of_them_is_no_mask(cuda, kind, sq):
    q, k, v = inputs(cuda, "bf16", 2, sq, 300, 2, 2, 64)
    mask = torch.zeros(2, 300, device=cuda, dtype=kind)
    mask[0, 100:] = torch.finfo(kind).min
    mask[1] = torch.finfo(kind).min       # every key alike: the softmax of the scores alone
    out = attention.cross_attention(q, k, v, key_mask=mask)
    bias = torch.zeros(2, 300, device=cuda)
    bias[0, 100:] = -math.inf
    check(out, q, k, v, bias)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sq", [100, 300])   # one row tile, and pairs of them with a single one at the end
@pytest.mark.parametrize("kind", ["none", "lengths", "bool", "additive"])
def test_many_items_of_all_lengths_on_one_sm(cuda, kind, sq, d):
    """More (sequence, head, rows) pieces than SMs, so that a CTA goes from one to the next: sequences
    without keys, of one key, of whole tiles and of several."""
    lens = [0, 640, 1, 128, 513, 0, 300, 77]
    b, h, sk = len(lens), 40, 640
    q, k, v = inputs(cuda, "bf16", b, sq, sk, h, h, d)
    lengths = torch.tensor(lens, device=cuda)
    keep = torch.arange(sk, device=cuda) < lengths[:, None]
    bias = torch.where(keep, 0.0, -math.inf)
    args = {}
    if kind == "none":
        bias = None
    elif kind == "lengths":
        args["kv_lengths"] = lengths
    elif kind == "bool":
        args["key_mask"] = keep
    else:
        bias = torch.where(keep, torch.randn(b, sk, device=cuda), -math.inf)
        args["key_mask"] = bias
    if bias is not None:
        k[~keep], v[~keep] = math.nan, math.nan
    out = attention.cross_attention(q, k, v, **args)
    check(out, q, k, v, bias)
    for _ in range(3):
        assert torch.equal(attention.cross_attention(q, k, v, **args), out)


@pytest.mark.parametrize("sq", [1, 300])
def test_offsets_past_32_bits(cuda, sq):
    """Rows more than 2^31 elements apart (a long cache of which a part is read)."""
    buf = torch.empty((1 << 31) + (1 << 22), device=cuda, dtype=torch.bfloat16)
    far = torch.as_strided(buf, (2, 500, 2, 64), (1 << 31, 128, 64, 1))
    q, k, v = inputs(cuda, "bf16", 2, sq, 500, 2, 2, 64)
    far.copy_(k)
    want = attention.cross_attention(q, k, v)
    assert torch.equal(attention.cross_attention(q, far, v), want)
    far.copy_(v)
    assert torch.equal(attention.cross_attention(q, k, far), want)
    out = ops.rotary(far, None, torch.arange(500, device=cuda), torch.ones(32, device=cuda))
    assert torch.equal(out, ops.rotary(v, None, torch.arange(500, device=cuda), torch.ones(32, device=cuda)))
    ops.rotary(far, None, torch.arange(500, device=cuda), torch.ones(32, device=cuda), inplace=True)
    assert torch.equal(far, out)


def test_masks_and_lengths_together_and_shared_masks(cuda):
    q, k, v = inputs(cuda, "bf16", 3, 20, 260, 4, 2, 64)
    mask = torch.rand(260, device=cuda) < 0.5
    lengths = torch.tensor([260, 100, 0], device=cuda)
    keep = mask & (torch.arange(260, device=cuda) < lengths[:, None])
    check(attention.cross_attention(q, k, v, key_mask=mask, kv_lengths=lengths), q, k, v, torch.where(keep, 0.0, -math.inf))
    both = attention.cross_attention(q, k, v, key_mask=mask)
    assert torch.equal(attention.cross_attention(q, k, v, key_mask=mask[None]), both)
    assert torch.equal(attention.cross_attention(q, k, v, key_mask=mask.expand(3, 260)), both)


@pytest.mark.parametrize("sq", [1, 3, 150])
def test_strides(cuda, sq):
    b, sk, h, d = 2, 270, 4, 64
    q, k, v = inputs(cuda, "bf16", b, sq, sk, h, h, d)
    want = attention.cross_attention(q, k, v)
    check(want, q, k, v)

    def heads_first(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    assert torch.equal(attention.cross_attention(heads_first(q), heads_first(k), heads_first(v)), want)
    kv = torch.cat([k, v], -1)             # k and v in one buffer
    assert torch.equal(attention.cross_attention(q, kv[..., :d], kv[..., d:]), want)
    check(attention.cross_attention(q[0], k[0], v[0])[None], q[:1], k[:1], v[:1])   # no batch dimension
    odd = torch.empty(b * sk * h * d + 1, device=cuda, dtype=q.dtype)[1:].view(b, sk, h, d).copy_(k)  # 2-byte aligned
    assert torch.equal(attention.cross_attention(q, odd, v), want)
    apart = torch.stack([q, q], -1)[..., 0]
    assert torch.equal(attention.cross_attention(apart, k, v), want)
    part = torch.zeros(b, sq, h + 1, 72, device=cuda, dtype=q.dtype)
    part[:, :, 1:, :d] = q
    assert torch.equal(attention.cross_attention(part[:, :, 1:, :d], k, v), want)
    pitch = torch.zeros(b, sk, h, 68, device=cuda, dtype=q.dtype)   # rows of 136 bytes: copied
    pitch[..., :d] = v
    assert torch.equal(attention.cross_attention(q, k, pitch[..., :d]), want)
    # states shared by the batch, one head shared by all
    want = attention.cross_attention(q, k[:1].expand(b, -1, -1, -1).contiguous(), v[:1].expand(b, -1, -1, -1).contiguous())
    assert torch.equal(attention.cross_attention(q, k[:1].expand(b, -1, -1, -1), v[:1].expand(b, -1, -1, -1)), want)
    want = attention.cross_attention(q, k[:, :, :1].expand(-1, -1, h, -1).contiguous(), v[:, :, :1].expand(-1, -1, h, -1).contiguous())
    assert torch.equal(attention.cross_attention(q, k[:, :, :1].expand(-1, -1, h, -1), v[:, :, :1].expand(-1, -1, h, -1)), want)
    same = q[:, :1].expand(b, sq, h, d)
    assert torch.equal(attention.cross_attention(same, k, v), attention.cross_attention(same.contiguous(), k, v))
    key = k[:, :1].expand(b, sk, h, d)     # one key repeated
    assert torch.equal(attention.cross_attention(q, key, v), attention.cross_attention(q, key.contiguous(), v))


@pytest.mark.parametrize("sq", [1, 200])
def test_growing_and_far_apart_scores(cuda, sq):
    """Maxima that grow along the keys, logits in the hundreds, equal logits."""
    q, k, v = inputs(cuda, "bf16", 1, sq, 1000, 2, 2, 64)
    ramp = torch.linspace(0.1, 12, 1000, device=cuda)[None, :, None, None]
    big = (q[:, :1].float().mean((1,), keepdim=True) * 0 + k.float() * ramp).to(q.dtype)
    check(attention.cross_attention(q, big, v), q, big, v)
    check(attention.cross_attention(q, big, v, scale=1.0), q, big, v, scale=1.0)
    check(attention.cross_attention(q, big.flip(1), v), q, big.flip(1), v)
    check(attention.cross_attention(torch.zeros_like(q), k, v), torch.zeros_like(q), k, v)
    check(attention.cross_attention(q, k, v, scale=1e-3), q, k, v, scale=1e-3)


def test_the_mean_and_a_single_key(cuda):
    q, k, v = inputs(cuda, "bf16", 1, 257, 1, 3, 3, 128)
    assert torch.equal(attention.cross_attention(q, k, v), v.expand_as(q))
    q, k, v = inputs(cuda, "f16", 2, 9, 500, 2, 2, 64)
    ones = torch.ones_like(v)
    # the weights and the result are each rounded once: two half steps
    assert torch.all((attention.cross_attention(q, k, ones) - 1).abs() <= torch.finfo(q.dtype).eps)


def test_a_non_finite_value_reaches_only_its_head(cuda):
    q, k, v = inputs(cuda, "bf16", 1, 140, 300, 4, 2, 64)
    v[0, 7, 1, 3] = math.nan
    out = attention.cross_attention(q, k, v)
    assert torch.isfinite(out[:, :, :2]).all() and torch.isnan(out[:, :, 2:, 3]).all()
    q[0, 5, 0, 0] = math.nan
    out = attention.cross_attention(q, k, v)
    assert torch.isnan(out[0, 5, 0]).all() and torch.isfinite(out[0, :5, 0]).all() and torch.isfinite(out[0, 6:, 0]).all()


def test_empty_inputs(cuda):
    q, k, v = inputs(cuda, "bf16", 2, 5, 8, 2, 2, 64)
    assert torch.equal(attention.cross_attention(q, k[:, :0], v[:, :0]), torch.zeros_like(q))
    mask = torch.zeros(2, 0, device=cuda, dtype=torch.bool)
    assert torch.equal(attention.cross_attention(q, k[:, :0], v[:, :0], key_mask=mask), torch.zeros_like(q))
    assert attention.cross_attention(q[:, :0], k, v).shape == (2, 0, 2, 64)
    assert attention.cross_attention(q[:0], k[:0], v[:0]).shape == (0, 5, 2, 64)


@pytest.mark.parametrize("sq,sk", [(1, 5000), (300, 200)])
def test_streams_graphs_and_repeats(cuda, sq, sk):
    q, k, v = inputs(cuda, "bf16", 2, sq, sk, 4, 4, 128)
    lengths = torch.tensor([sk, sk // 3], device=cuda)
    want = attention.cross_attention(q, k, v, kv_lengths=lengths)
    for _ in range(5):
        assert torch.equal(attention.cross_attention(q, k, v, kv_lengths=lengths), want)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:                       # several calls at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(attention.cross_attention(q, k, v, kv_lengths=lengths))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs, got = [], []
    for _ in range(2):                      # two captured calls with their own workspaces
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(attention.cross_attention(q, k, v, kv_lengths=lengths))
        graphs.append(g)
    lengths.copy_(torch.tensor([sk // 2, sk], device=cuda))   # a replay reads the lengths of its time
    q.neg_()
    for s, g in zip(streams, graphs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    now = attention.cross_attention(q, k, v, kv_lengths=lengths)
    assert all(torch.equal(o, now) for o in got) and not torch.equal(now, want)


def test_refusals(cuda):
    q, k, v = inputs(cuda, "bf16", 2, 5, 8, 4, 2, 64)
    lengths = torch.tensor([3, 4], device=cuda)
    for bad, error in [
        (lambda: attention.cross_attention(q.cpu(), k, v), TypeError),
        (lambda: attention.cross_attention(q.float(), k.float(), v.float()), TypeError),
        (lambda: attention.cross_attention(q, k.half(), v), ValueError),
        (lambda: attention.cross_attention(q[0], k, v), ValueError),
        (lambda: attention.cross_attention(q, k[:, :7], v), ValueError),
        (lambda: attention.cross_attention(q, k[:1], v[:1]), ValueError),
        (lambda: attention.cross_attention(q[:, :, :3], k, v), ValueError),
        (lambda: attention.cross_attention(q[..., :60], k[..., :60], v[..., :60]), ValueError),
        (lambda: attention.cross_attention(q[..., :32], k, v), ValueError),
        (lambda: attention.cross_attention(q, k, v, key_mask=torch.ones(2, 7, device=cuda, dtype=torch.bool)), ValueError),
        (lambda: attention.cross_attention(q, k, v, key_mask=torch.ones(2, 1, 5, 8, device=cuda, dtype=torch.bool)), ValueError),
        (lambda: attention.cross_attention(q, k, v, key_mask=torch.ones(2, 8, device=cuda, dtype=torch.int64)), TypeError),
        (lambda: attention.cross_attention(q, k, v, key_mask=torch.ones(2, 8, dtype=torch.bool)), ValueError),
        (lambda: attention.cross_attention(q, k, v, key_mask=[True] * 8), TypeError),
        (lambda: attention.cross_attention(q, k, v, kv_lengths=[8, 8]), TypeError),
        (lambda: attention.cross_attention(q, k, v, kv_lengths=lengths.float()), TypeError),
        (lambda: attention.cross_attention(q, k, v, kv_lengths=lengths[:1]), ValueError),
        (lambda: attention.cross_attention(q, k, v, kv_lengths=lengths.cpu()), ValueError),
        (lambda: attention.cross_attention(q, k, v, scale=-1.0), ValueError),
        (lambda: attention.cross_attention(q, k, v, scale=math.nan), ValueError),
        (lambda: attention.cross_attention(q.clone().requires_grad_(), k, v), ValueError),
    ]:
        with pytest.raises(error):
            bad()
    big = torch.zeros(1, 2, 1, 136, device=cuda, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="head dim"):
        attention.cross_attention(big, big, big)
    many = torch.zeros(1, 2, 129, 64, device=cuda, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="group"):
        attention.cross_attention(many, many[:, :, :1], many[:, :, :1])


def test_rotated_queries_attend_between_two_linears(cuda):
    """The path of a block: INT8 projections, rotary positions on q and k, cross attention, output
    projection; the attention checked on the operands it got."""
    from slimdit.ops import int8_linear, rotate_quant

    g = torch.Generator(device="cuda").manual_seed(3)
    b, sq, sk, h, d = 2, 150, 77, 4, 64
    width = h * d
    x = torch.randn(b, sq, width, device=cuda, generator=g).to(torch.bfloat16)
    states = torch.randn(b, sk, width, device=cuda, generator=g).to(torch.bfloat16)
    wq, wkv, wo = (rotate_quant(torch.randn(n, width, device=cuda, generator=g).to(torch.bfloat16) * width**-0.5)
                   for n in (width, 2 * width, width))
    q = int8_linear(x, *wq).unflatten(-1, (h, d))
    kv = int8_linear(states, *wkv)
    k, v = (t.unflatten(-1, (h, d)) for t in kv.split(width, -1))
    freq, m = rope.rope_frequencies(32, scaling="yarn", factor=2.0, original_length=64)
    freq = torch.from_numpy(freq).to(cuda)
    qr = ops.rotary(q, None, torch.arange(sq, device=cuda), freq, magnitude=m)
    plain_k = k.clone()
    kr = ops.rotary(k, None, torch.arange(sk, device=cuda), freq, magnitude=m, inplace=True)
    assert torch.equal(kr, ops.rotary(plain_k, None, torch.arange(sk, device=cuda), freq, magnitude=m))
    lengths = torch.tensor([77, 30], device=cuda)
    o = attention.cross_attention(qr, kr, v, kv_lengths=lengths)
    check(o, qr, kr, v, torch.where(torch.arange(sk, device=cuda) < lengths[:, None], 0.0, -math.inf))
    y = int8_linear(o.flatten(-2), *wo)
    assert y.shape == (b, sq, width) and torch.isfinite(y).all()
