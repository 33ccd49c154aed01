"""Timing cases of a decoder layer's operators around the paged attention: ``w4.linear`` and ``w4.gated`` (products with
4-bit weights and group scales, the second with the activation and the product of a gated feed-forward) and
``rotary.Rotary`` (rotary positions with one to four axes, and the inverse rotation, which is its gradient).

A weight is ``(code - zero) * scale``: codes 0 .. 15 ``[N, K]``, one scale (16 bits) and one zero (8 where there are none) for
each row and each ``group`` consecutive k.

``run`` is one pass through one of the operators: in elementary torch operations, or with ``own`` through the package's entry
points.
"""

import math
import os
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _package():
    pkg = os.path.join(os.getcwd(), "minicpm-o-4.5-single-gpu-engine_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from b200t2w import rotary, w4

    return w4, rotary


# ---- cases ----------------------------------------------------------------------------------------------------------


def listed():
    return [
        # one stream's token through a small projection: latency
        dict(name="linear 1x1024x1024", op="linear", rows=1, k=1024, n=1024, group=64, zeros=False, bias=True,
             residual=False, dtype="bf16"),
        # one stream's token, an output projection onto the residual stream
        dict(name="linear 1x4096x4096", op="linear", rows=1, k=4096, n=4096, group=128, zeros=False, bias=False,
             residual=True, dtype="fp16"),
        # a few streams' tokens through the second half of a feed-forward, a width that is no power of two
        dict(name="linear 7x11008x4096", op="linear", rows=7, k=11008, n=4096, group=128, zeros=True, bias=False,
             residual=True, dtype="bf16"),
        # 64 streams' tokens through the fused q | k | v projection with grouped heads
        dict(name="linear 64x4096x6144", op="linear", rows=64, k=4096, n=6144, group=128, zeros=True, bias=True,
             residual=False, dtype="bf16"),
        # 40 streams' logits over the 6561 speech tokens
        dict(name="linear 40x1024x6561", op="linear", rows=40, k=1024, n=6561, group=32, zeros=False, bias=False,
             residual=False, dtype="fp16"),
        # prompts of several requests at once
        dict(name="linear 2000x4096x4096", op="linear", rows=2000, k=4096, n=4096, group=64, zeros=False, bias=False,
             residual=True, dtype="bf16"),
        # one stream's token through the first half of a feed-forward
        dict(name="gated 1x4096x11008", op="gated", rows=1, k=4096, f=11008, group=128, zeros=False, act="silu",
             dtype="bf16"),
        # 50 streams, a smaller decoder
        dict(name="gated 50x2048x5632", op="gated", rows=50, k=2048, f=5632, group=64, zeros=True, act="gelu_tanh",
             dtype="fp16"),
        # prompts of several requests at once: the most work
        dict(name="gated 3000x4096x11008", op="gated", rows=3000, k=4096, f=11008, group=128, zeros=False, act="silu",
             dtype="bf16"),
        # 64 streams' tokens: queries and keys out of the fused q | k | v rows, one axis, far along
        dict(name="rotary 64x(32+8)x128", op="rotary", rows=64, q_heads=32, kv_heads=8, head_dim=128, rotary_dim=128,
             sections="64", pairs="half", far=200000, base=1000000.0, inverse=False, dtype="bf16"),
        # the backward rotation of an image tower's rows: height and width, heads of 80, neighbours paired
        dict(name="rotary 4900x(16+16)x80", op="rotary", rows=4900, q_heads=16, kv_heads=16, head_dim=80, rotary_dim=80,
             sections="20,20", pairs="adjacent", far=70, base=10000.0, inverse=True, dtype="fp16"),
        # prompts with images among the text: time, height and width
        dict(name="rotary 30000x(28+4)x128", op="rotary", rows=30000, q_heads=28, kv_heads=4, head_dim=128, rotary_dim=128,
             sections="16,24,24", pairs="half", far=30000, base=1000000.0, inverse=False, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "gated", "gated", "rotary"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "rotary":
        hd = rng.choice([64, 80, 96, 128])
        rot = rng.choice([hd, hd, hd // 2 // 16 * 16])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4, 5])
        axes, left, sections = rng.randint(1, 4), rot // 2, []
        for a in range(axes - 1):
            sections.append(rng.randint(0, left))
            left -= sections[-1]
        return dict(op=op, rows=_log(rng, 1, 30000 * 4096 // ((heads + kv) * hd)), q_heads=heads, kv_heads=kv, head_dim=hd,
                    rotary_dim=rot, sections=",".join(map(str, sections + [left])), pairs=rng.choice(["half", "half", "adjacent"]),
                    far=_log(rng, 50, 1000000), base=rng.choice([10000.0, 500000.0]), inverse=rng.random() < 0.3, dtype=dtype)
    group = rng.choice([32, 64, 128, 128])
    k = group * (_log(rng, 512, 12288) // group)
    n = _log(rng, 200, 12288)
    # no more products than the largest listed case of the operator
    top = (2000 * 4096 * 4096 if op == "linear" else 3000 * 4096 * 11008) // (k * n)
    rows = _log(rng, 1, max(1, min(4096, top)))
    if op == "linear":
        return dict(op=op, rows=rows, k=k, n=n, group=group, zeros=rng.random() < 0.5, bias=rng.random() < 0.5,
                    residual=rng.random() < 0.5, dtype=dtype)
    return dict(op=op, rows=rows, k=k, f=n, group=group, zeros=rng.random() < 0.5, act=rng.choice(["silu", "gelu_tanh"]),
                dtype=dtype)


# ---- inputs ---------------------------------------------------------------------------------------------------------


def _weights(n, k, case, gen):
    """Rows of a projection in 4 bits: codes as rounding normal weights gives them, scales that differ by row and group."""
    g, dt = case["group"], TYPES[case["dtype"]]
    top = 2.5 + torch.rand(n, k // g, device="cuda", generator=gen)  # a group's largest weight, in standard deviations
    spread = torch.exp(0.3 * torch.randn(n, k // g, device="cuda", generator=gen)) * k ** -0.5
    scales = (spread * top / 7).to(dt)
    zeros = None
    if case["zeros"]:
        zeros = torch.randint(5, 11, (n, k // g), device="cuda", generator=gen, dtype=torch.uint8)
    codes = torch.empty(n, k, device="cuda", dtype=torch.uint8)
    step = max(1, (1 << 25) // k)
    for i in range(0, n, step):
        j = min(n, i + step)
        w = torch.randn(j - i, k // g, g, device="cuda", generator=gen) * (7 / top[i:j])[:, :, None]
        w += 8.0 if zeros is None else zeros[i:j, :, None].float()
        codes[i:j] = w.round().clamp(0, 15).view(j - i, k).to(torch.uint8)
    return codes, scales, zeros


def _sections(case):
    """How many pairs turn by each axis."""
    return [int(s) for s in case["sections"].split(",")]


def _inv_freq(case):
    d = case["rotary_dim"]
    return torch.tensor([case["base"] ** (-2 * i / d) for i in range(d // 2)], dtype=torch.float64, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, rows = TYPES[case["dtype"]], case["rows"]

    def normal(*size):
        return torch.randn(*size, device="cuda", generator=gen)

    if case["op"] == "rotary":
        heads, kv, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
        qkv = normal(rows, heads + 2 * kv, hd).to(dt)
        axes = len(_sections(case))
        st = dict(case=case, q=qkv[:, :heads], k=qkv[:, heads:heads + kv],
                  positions=torch.randint(0, case["far"], (axes, rows), device="cuda", generator=gen, dtype=torch.int32))
        if own:
            st["rotary"] = _package()[1].Rotary(hd, _sections(case), base=case["base"], rotary_dim=case["rotary_dim"],
                                                pairs=case["pairs"])
        else:
            st["inv_freq"] = _inv_freq(case)
            st["axis"] = torch.repeat_interleave(torch.arange(axes, device="cuda"),
                                                 torch.tensor(_sections(case), device="cuda"))
        return st
    st = dict(case=case, x=normal(rows, case["k"]).to(dt))
    if case["op"] == "linear":
        st["w"] = _weights(case["n"], case["k"], case, gen)
        st["bias"] = normal(case["n"]).to(dt) if case["bias"] else None
        st["residual"] = normal(rows, case["n"]).to(dt) if case["residual"] else None
    else:
        st["w"], st["up"] = _weights(case["f"], case["k"], case, gen), _weights(case["f"], case["k"], case, gen)
    if own:  # a layer's weights are laid out once, when they are loaded
        w4 = _package()[0]
        st["w"] = w4.pack(*st["w"]) if case["op"] == "linear" else w4.pack_gated(st["w"], st.pop("up"))
    return st


# ---- one pass -------------------------------------------------------------------------------------------------------


def run(st):
    return {"linear": _run_linear, "gated": _run_gated, "rotary": _run_rotary}[st["case"]["op"]](st)


def _dense(w, group):
    codes, scales, zeros = w
    c = codes.float().view(codes.shape[0], -1, group)
    z = 8.0 if zeros is None else zeros.float()[:, :, None]
    return ((c - z) * scales.float()[:, :, None]).view(codes.shape)


def _run_linear(st):
    if own:
        return _package()[0].linear(st["x"], st["w"], bias=st["bias"], residual=st["residual"])
    y = torch.matmul(st["x"].float(), _dense(st["w"], st["case"]["group"]).T)
    if st["bias"] is not None:
        y = y + st["bias"].float()
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return y.to(st["x"].dtype)


def _run_gated(st):
    act = st["case"]["act"]
    if own:
        return _package()[0].gated(st["x"], st["w"], act=act)
    x, group = st["x"].float(), st["case"]["group"]
    g = torch.matmul(x, _dense(st["w"], group).T)
    if act == "silu":
        a = g / (1 + torch.exp(-g))
    else:
        a = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))
    return (a * torch.matmul(x, _dense(st["up"], group).T)).to(st["x"].dtype)


def _run_rotary(st):
    c = st["case"]
    if own:
        q, k = st["rotary"](st["q"], st["k"], st["positions"], inverse=c["inverse"])
        return dict(q=q, k=k)
    # angles of far positions in 64 bits
    angle = (st["positions"][st["axis"]].double() * st["inv_freq"][:, None]).T  # [rows, pairs]
    if c["inverse"]:
        angle = -angle
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    d = c["rotary_dim"]

    def turned(x):
        y = x.float()
        a, b = (y[..., :d // 2], y[..., d // 2:d]) if c["pairs"] == "half" else (y[..., :d:2], y[..., 1:d:2])
        u, v = a * cos - b * sin, b * cos + a * sin
        r = torch.cat([u, v], -1) if c["pairs"] == "half" else torch.stack([u, v], -1).flatten(-2)
        return torch.cat([r, y[..., d:]], -1).to(x.dtype)

    return dict(q=turned(st["q"]), k=turned(st["k"]))


# ---- what a pass cannot do without ----------------------------------------------------------------------------------


def work(case):
    rows = case["rows"]
    if case["op"] == "rotary":
        values = rows * (case["q_heads"] + case["kv_heads"])
        return {"bytes": 4 * values * case["head_dim"] + 4 * rows * len(_sections(case)),
                "flops": 3 * values * case["rotary_dim"]}
    k, out = case["k"], case["n"] if case["op"] == "linear" else case["f"]
    n = out if case["op"] == "linear" else 2 * out  # rows of the weights
    per_group = 2.5 if case["zeros"] else 2.0  # a 16-bit scale, a 4-bit zero
    extra = (2 * out if case.get("bias") else 0) + (2 * rows * out if case.get("residual") else 0)
    return {"bytes": int(n * k / 2 + n * (k // case["group"]) * per_group) + 2 * rows * k + 2 * rows * out + extra,
            "flops": 2 * rows * n * k}


# ---- 64 bits --------------------------------------------------------------------------------------------------------


def _exact_product(x, w, group):
    """x W^T group by group: sums of whole codes first, then each group's zero and scale."""
    codes, scales, zeros = w
    y = torch.zeros(x.shape[0], codes.shape[0], device="cuda", dtype=torch.float64)
    x = x.double()
    block = 2048 // group  # groups at a time, so that a block of weights is one product
    for i in range(0, scales.shape[1], block):
        j = min(scales.shape[1], i + block)
        c = codes[:, i * group:j * group].double().view(-1, j - i, group)
        c = c - (8 if zeros is None else zeros[:, i:j].double().unsqueeze(2))
        y += x[:, i * group:j * group] @ (c * scales[:, i:j].double().unsqueeze(2)).reshape(codes.shape[0], -1).T
    return y


def exact(case, seed):
    global own
    kept, own = own, False  # the inputs as they are before a user lays them out
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    if case["op"] == "linear":
        y = _exact_product(st["x"], st["w"], case["group"])
        for extra in (st["bias"], st["residual"]):
            if extra is not None:
                y += extra.double()
        return y
    if case["op"] == "gated":
        g = _exact_product(st["x"], st["w"], case["group"])
        u = _exact_product(st["x"], st["up"], case["group"])
        s = 1.0 if case["act"] == "silu" else 2 * math.sqrt(2 / math.pi) * (1 + 0.044715 * g * g)
        return g * torch.sigmoid(g * s) * u  # (1 + tanh(t)) / 2 = sigmoid(2 t)
    d, out = case["rotary_dim"], {}
    first, angles = 0, []
    for axis, size in enumerate(_sections(case)):
        i = torch.arange(first, first + size, device="cuda", dtype=torch.float64)
        inv = torch.exp(-2 * i / d * math.log(case["base"]))
        angles.append(st["positions"][axis].double()[:, None] * inv)
        first += size
    turn = torch.polar(torch.ones((), device="cuda", dtype=torch.float64),
                       torch.cat(angles, 1) * (-1 if case["inverse"] else 1))[:, None]
    for name in ("q", "k"):
        x = st[name].double()
        y = x.clone()
        if case["pairs"] == "half":
            z = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:d].contiguous()) * turn
            y[..., :d // 2], y[..., d // 2:d] = z.real, z.imag
        else:
            z = torch.complex(x[..., :d:2].contiguous(), x[..., 1:d:2].contiguous()) * turn
            y[..., :d:2], y[..., 1:d:2] = z.real, z.imag
        out[name] = y
    return out
