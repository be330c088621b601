"""Rotary positions and cross attention: the workloads they are measured on.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits, rounded
once at the end) or, with ``own`` set, through the framework's entry points
``slimdit.ops.rotary`` and ``slimdit.attention.cross_attention``. ``exact`` is the operator's
definition in 64 bits.
"""

import math
import sys

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------- cases
def _rotary(name, batch, seq, heads, kv_heads, dim, rot, layout="half", dtype="bf16", axes=1, packed=False,
            start=0, factor=1.0, inverse=False):
    return {"name": name, "op": "rotary", "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "rot": rot, "layout": layout, "dtype": dtype, "axes": axes, "packed": packed,
            "start": start, "factor": factor, "inverse": inverse}


def _cross(name, batch, q_len, kv_len, heads, kv_heads, dim, dtype="bf16", mask="none", filled=1.0):
    return {"name": name, "op": "cross", "batch": batch, "q_len": q_len, "kv_len": kv_len, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "mask": mask, "filled": filled}


def listed():
    return [
        # one new token of eight sequences, q and k of a grouped-query layer: latency
        _rotary("rotary_step", 8, 1, 32, 8, 128, 128, start=100000),
        # the packed qkv buffer of the 56-head DiT at its benchmark length, three position axes
        # of 16 frequencies each (96 of 128 elements rotate)
        _rotary("rotary_video", 1, 30026, 56, 56, 128, 96, axes=3, packed=True),
        # interleaved pairs in half of the head, a prompt batch of odd length
        _rotary("rotary_partial", 2, 4099, 24, 24, 128, 64, layout="interleaved", dtype="f16"),
        # far positions with frequencies and magnitude scaled for an eight times longer context
        _rotary("rotary_far_f32", 1, 65537, 8, 2, 64, 64, dtype="f32", start=900000, factor=8.0),
        # an odd part of an odd head, rotated back (keys taken to other positions)
        _rotary("rotary_odd_back", 3, 1021, 5, 0, 80, 20, inverse=True),
        # one decoder token of four sequences over an encoder's 1500 states: latency
        _cross("cross_step", 4, 1, 1500, 16, 16, 64, mask="lengths", filled=0.8),
        # one token over a long document, grouped heads: every byte of k and v once
        _cross("cross_step_long", 1, 1, 131071, 32, 8, 128),
        # video tokens of the 56-head DiT attending to a padded prompt
        _cross("cross_video_text", 1, 30026, 512, 56, 56, 128, mask="lengths", filled=0.9),
        # image tokens and a short prompt with a boolean padding mask, two guidance branches
        _cross("cross_image_text", 2, 4096, 77, 10, 10, 64, dtype="f16", mask="bool", filled=0.5),
        # odd lengths and head size, grouped heads, additive mask of the type's lowest value
        _cross("cross_odd", 3, 333, 1003, 9, 3, 72, mask="additive", filled=0.7),
        # long queries over long states: bound by the two products
        _cross("cross_long", 1, 16384, 16111, 24, 24, 128),
    ]


def _spread(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    if rng.random() < 0.5:
        dim = rng.choice([64, 80, 96, 128])
        heads = rng.randint(1, 56)
        axes = rng.choice([1, 1, 3])
        rot = rng.choice([r for r in (12, 24, 48, 60, 72, 96, 120) if r <= dim] if axes == 3
                         else [20, 32, 54, 64, dim])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        batch = rng.randint(1, 4)
        widest = 2 * 30026 * 56 * 128 // (2 if dtype == "f32" else 1)
        packed = rng.random() < 0.3
        kv_heads = heads if packed else rng.choice([0, heads, rng.randint(1, heads)])
        seq = _spread(rng, 1, max(1, min(100000, widest // (batch * (heads + kv_heads) * dim))))
        return _rotary(None, batch, seq, heads, kv_heads, dim, rot, layout=rng.choice(["half", "interleaved"]),
                       dtype=dtype, axes=axes, packed=packed, start=rng.choice([0, 17, 40000, 900000]),
                       factor=rng.choice([1.0, 4.0, 8.0]), inverse=rng.random() < 0.25) | {"name": ""}
    dim = rng.choice([40, 64, 64, 72, 96, 128, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 8, 10, 16, 24])
    group = rng.choice([1, 1, 2, 3, 4, 8])
    batch = rng.randint(1, 4)
    q_len = rng.choice([1, 1, 2, 7, _spread(rng, 16, 30026), _spread(rng, 16, 30026), _spread(rng, 16, 30026)])
    rows = batch * kv_heads * group * q_len
    most = min(131071, 16384 * 16111 * 24 // rows, 2 ** 28 // (batch * kv_heads * dim))
    kv_len = _spread(rng, 1, max(1, most))
    if rows * dim > 30026 * 56 * 128:
        batch = 1
    return _cross("", batch, q_len, kv_len, kv_heads * group, kv_heads, dim,
                  dtype=rng.choice(["bf16", "bf16", "f16"]),
                  mask=rng.choice(["none", "lengths", "bool", "additive"]),
                  filled=rng.choice([0.1, 0.4, 0.7, 1.0]))


# ---------------------------------------------------------------- inputs
def _lengths(case):
    """Keys in use per sequence: the share ``filled`` on average, none for one in five of a mask's
    sequences past the second (an empty prompt)."""
    if case["mask"] == "none":
        return [case["kv_len"]] * case["batch"]
    out = []
    for b in range(case["batch"]):
        part = min(1.0, case["filled"] * (1.0 + 0.15 * ((b % 3) - 1))) if case["batch"] > 1 else case["filled"]
        out.append(0 if b % 5 == 2 and case["mask"] != "additive" else max(1, int(case["kv_len"] * part)))
    return out


def _frequencies(case):
    """Per-pair frequencies 10000^(-j/n), each axis with its own n = pairs / axes; a factor above 1
    divides the slow ones by it (those that turn less than once in 8192 positions), blends up to
    32 turns, and raises the magnitude to 0.1 ln(factor) + 1."""
    n = case["rot"] // 2 // case["axes"]
    f = 10000.0 ** (-np.arange(n, dtype=np.float64) / n)
    if case["factor"] > 1.0:
        keep = np.clip((8192 * f / (2 * math.pi) - 1.0) / 31.0, 0.0, 1.0)
        f = f * keep + f / case["factor"] * (1.0 - keep)
    magnitude = 0.1 * math.log(case["factor"]) + 1.0
    return np.tile(f, case["axes"]).astype(np.float32), magnitude


def _positions(case, generator):
    """Consecutive positions from ``start`` plus a random offset, one row per sequence; with three
    axes the (frame, row, column) of each token of a video."""
    b, s = case["batch"], case["seq"]
    first = case["start"] + torch.randint(0, 1000, (b, 1), generator=generator)
    if case["axes"] == 1:
        return (first + torch.arange(s)).to(torch.int64)
    width = max(1, int(round((s / 2) ** 0.4)))
    token = torch.arange(s)
    grid = torch.stack([token // (width * width), token // width % width, token % width], -1)
    return (first[..., None] + grid).to(torch.int64)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.empty(shape, dtype=dt, device=DEVICE).normal_(generator=gen)

    state = {"case": case}
    if case["op"] == "rotary":
        b, s, h, hk, d = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
        if case["packed"]:  # q and k as they stand in the rows [q heads | k heads | v heads]
            rows = normal(b, s, 3 * h * d)
            state["q"] = rows[..., :h * d].unflatten(-1, (h, d))
            state["k"] = rows[..., h * d:2 * h * d].unflatten(-1, (h, d))
        else:
            state["q"] = normal(b, s, h, d)
            state["k"] = normal(b, s, hk, d) if hk else None
        freq, state["magnitude"] = _frequencies(case)
        state["freq"] = torch.from_numpy(freq).to(DEVICE)
        state["positions"] = _positions(case, host).to(DEVICE)
        state["sections"] = None if case["axes"] == 1 else (case["rot"] // 2 // case["axes"],) * case["axes"]
        return state
    b, sq, sk, h, hk, d = (case[n] for n in ("batch", "q_len", "kv_len", "heads", "kv_heads", "dim"))
    state["q"] = normal(b, sq, h, d).mul_(1.5)
    state["k"] = normal(b, sk, hk, d)
    state["v"] = normal(b, sk, hk, d)
    state["key_mask"] = state["kv_lengths"] = None
    if case["mask"] != "none":
        lengths = torch.tensor(_lengths(case), dtype=torch.int32, device=DEVICE)
        keep = torch.arange(sk, device=DEVICE) < lengths[:, None]
        if case["mask"] == "lengths":
            state["kv_lengths"] = lengths
        elif case["mask"] == "bool":  # padding, and a few holes inside the prompt
            hole = torch.rand((b, sk), device=DEVICE, generator=gen) < 0.03
            state["key_mask"] = keep & ~hole
        else:  # 0 and the type's lowest value, with a bias on some keys
            bias = torch.empty((b, sk), device=DEVICE).normal_(generator=gen).to(dt)
            state["key_mask"] = torch.where(keep, bias, torch.finfo(dt).min)
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    return (_own if own else _plain)(state)


def _own(state):
    package = "viggle-animate-workflow_b200"
    if package not in sys.path:
        sys.path.insert(1, package)
    from slimdit import attention, ops

    case = state["case"]
    if case["op"] == "rotary":
        return ops.rotary(state["q"], state["k"], state["positions"], state["freq"], layout=case["layout"],
                          sections=state["sections"], magnitude=state["magnitude"], inverse=case["inverse"])
    return attention.cross_attention(state["q"], state["k"], state["v"], key_mask=state["key_mask"],
                                     kv_lengths=state["kv_lengths"])


def _plain(state):
    case = state["case"]
    if case["op"] == "rotary":
        cos, sin = _angles(state)
        q = _rotate_plain(state["q"], cos, sin, state)
        return q if state["k"] is None else (q, _rotate_plain(state["k"], cos, sin, state))
    return _attend_plain(state)


def _angles(state):
    """cos and sin of position x frequency, the angle in 64 bits (a far position times a frequency
    loses whole turns' fractions in 32)."""
    pos, freq = state["positions"].double(), state["freq"].double()
    if state["sections"] is None:
        angle = pos[..., None] * freq
    else:
        axis = torch.repeat_interleave(torch.arange(len(state["sections"])), torch.tensor(state["sections"]))
        angle = pos[..., axis.to(pos.device)] * freq
    if state["case"]["inverse"]:
        angle = -angle
    m = state["magnitude"]
    return (angle.cos() * m).float()[:, :, None], (angle.sin() * m).float()[:, :, None]


def _rotate_plain(x, cos, sin, state):
    rot = state["case"]["rot"]
    y = x.float()
    if state["case"]["layout"] == "half":
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, y[..., rot:]], -1).to(x.dtype)


def _attend_plain(state):
    q, k, v = state["q"], state["k"], state["v"]
    b, sq, h, d = q.shape
    sk, hk = k.shape[1:3]
    g = h // hk
    bias = torch.zeros((b, sk), device=q.device)
    if state["kv_lengths"] is not None:
        bias = bias.masked_fill(torch.arange(sk, device=q.device) >= state["kv_lengths"][:, None], -math.inf)
    elif state["key_mask"] is not None:
        m = state["key_mask"]
        bias = bias.masked_fill(~m, -math.inf) if m.dtype == torch.bool else m.float()
    out = torch.empty_like(q)
    rows = max(1, min(sq, 2 ** 28 // (h * sk)))  # score tiles of a GB
    for i in range(b):
        kt = k[i].float().permute(1, 2, 0)
        w = torch.where(bias[i, :, None, None] == -math.inf, 0.0, v[i].float()).transpose(0, 1)
        for r in range(0, sq, rows):
            x = q[i, r:r + rows].float().unflatten(1, (hk, g)).permute(1, 0, 2, 3)
            s = (x.reshape(hk, -1, d) @ kt) * d ** -0.5
            s = torch.where(bias[i] == -math.inf, -math.inf, s + bias[i])
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            total = p.sum(-1, keepdim=True)
            y = (p @ w) / torch.where(total == 0, 1.0, total)
            out[i, r:r + rows] = y.reshape(x.shape).permute(1, 0, 2, 3).reshape(-1, h, d).to(out.dtype)
    return out


# ---------------------------------------------------------------- what a pass has to do
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rotary":
        elements = case["batch"] * case["seq"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        pairs = case["batch"] * case["seq"] * (case["heads"] + case["kv_heads"]) * case["rot"] // 2
        return {"bytes": 2 * size * elements + 8 * case["batch"] * case["seq"] * case["axes"] + 2 * case["rot"],
                "flops": 6 * pairs}
    keys = sum(_lengths(case)) if case["mask"] != "additive" else case["batch"] * case["kv_len"]
    queries = case["batch"] * case["q_len"] * case["heads"] * case["dim"]
    mask_bytes = {"none": 0, "lengths": 4, "bool": case["kv_len"], "additive": size * case["kv_len"]}[case["mask"]]
    return {"bytes": size * 2 * (queries + keys * case["kv_heads"] * case["dim"]) + mask_bytes * case["batch"],
            "flops": 4 * keys * case["q_len"] * case["heads"] * case["dim"]}


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        # each pair as a complex number, multiplied by magnitude * exp(i position frequency)
        sections = state["sections"] or (case["rot"] // 2,)
        pos = state["positions"].double().reshape(case["batch"], case["seq"], case["axes"])
        parts = torch.split(state["freq"].double(), list(sections))
        phase = torch.cat([pos[..., a:a + 1] * f for a, f in enumerate(parts)], -1)
        turn = torch.polar(torch.full_like(phase, state["magnitude"]), -phase if case["inverse"] else phase)
        turn = turn.unsqueeze(2)

        def rotated(x):
            y = x.double()
            n = case["rot"] // 2
            if case["layout"] == "half":
                z = torch.complex(y[..., :n].contiguous(), y[..., n:2 * n].contiguous()) * turn
                y[..., :n], y[..., n:2 * n] = z.real, z.imag
            else:
                z = torch.view_as_complex(y[..., :2 * n].unflatten(-1, (n, 2)).contiguous()) * turn
                y[..., :2 * n] = torch.view_as_real(z).flatten(-2)
            return y

        q = rotated(state["q"])
        return q if state["k"] is None else (q, rotated(state["k"]))
    if work(case)["flops"] > 8e12:  # minutes in 64 bits
        return None
    q, k, v = state["q"], state["k"], state["v"]
    share = case["heads"] // case["kv_heads"]
    result = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for i in range(case["batch"]):
        used = torch.ones(case["kv_len"], dtype=torch.bool, device=q.device)
        extra = torch.zeros(case["kv_len"], dtype=torch.float64, device=q.device)
        if state["kv_lengths"] is not None:
            used[int(state["kv_lengths"][i]):] = False
        if state["key_mask"] is not None and state["key_mask"].dtype == torch.bool:
            used = state["key_mask"][i]
        elif state["key_mask"] is not None:
            extra = state["key_mask"][i].double()
        index = used.nonzero().flatten()
        if index.numel() == 0:
            continue
        step = max(1, 2 ** 27 // index.numel())
        for h in range(case["heads"]):
            keys = k[i, index, h // share].double()
            values = v[i, index, h // share].double()
            for r in range(0, case["q_len"], step):
                logits = torch.einsum("rd,kd->rk", q[i, r:r + step, h].double(), keys) / math.sqrt(case["dim"])
                result[i, r:r + step, h] = torch.softmax(logits + extra[index], -1) @ values
    return result
