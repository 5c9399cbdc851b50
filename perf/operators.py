"""What the device operators of katago_amd.ops compute, in elementary torch operations, and cases to measure them on.

Three operators that surround the attention of a transformer trunk when its projections run in 8 bits:

  norm     h = x + residual; y = h / rms(h) * weight on the rows that the mask keeps, 0 elsewhere; y itself and / or y in e4m3 with one
           fp32 scale a row ("row") or one power-of-two scale for each 32 channels ("mx"); or the 8-bit form of x alone ("norm": False)
  linear   y = (codes * scales) (weight codes * weight scales)^T + bias, the product of two such 8-bit matrices
  rotary   pairs of q's and k's channels turned by position * frequency: neighbours or halves, part of the head, one or two axes,
           frequencies of their own for each key head, a magnitude, and the inverse turn (its transpose)

`own` False: the plain form. `own` True: the calls a user makes.
"""
import math

import torch

own = False

E4M3_MAX = 448.0
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BOARD = 361  # cells of a 19x19 buffer


def listed():
    return [
        # one token between two layers of a served model: latency
        dict(name="norm one row", op="norm", rows=1, channels=4096, type="bf16", residual=True, masked=False, norm=True, wants="row"),
        # one 19x19 position, 384 channels (the widest trunk of the 18-block nets), between attention and FFN
        dict(name="norm one board", op="norm", rows=361, channels=384, type="fp16", residual=True, masked=True, norm=True, wants="row"),
        # the benchmark's batch of 256 positions
        dict(name="norm 256 boards", op="norm", rows=92416, channels=384, type="fp16", residual=True, masked=True, norm=True, wants="row"),
        # a long prompt's chunk of a wide model, block scales and the 16-bit result beside them
        dict(name="norm wide mx", op="norm", rows=8190, channels=4096, type="bf16", residual=True, masked=False, norm=True, wants="mx+y"),
        # an activation (an attention's or a gated unit's output) brought to 8 bits before its product
        dict(name="quantize", op="norm", rows=16383, channels=1536, type="bf16", residual=False, masked=False, norm=False, wants="row"),
        # one token through a square projection: the weights' bytes
        dict(name="linear one row", op="linear", rows=1, k=4096, n=4096, scales="row", out="bf16", bias=False),
        # one position's q, k and v
        dict(name="linear one board", op="linear", rows=361, k=384, n=1152, scales="row", out="fp16", bias=True),
        # the benchmark's batch through the same projection
        dict(name="linear 256 boards", op="linear", rows=92416, k=384, n=1152, scales="row", out="fp16", bias=True),
        # a chunk of a wide model up into its gated unit, block scales
        dict(name="linear wide mx", op="linear", rows=8190, k=4096, n=11008, scales="mx", out="bf16", bias=False),
        # eight sequences' next tokens, far into their contexts
        dict(name="rotary next tokens", op="rotary", batch=8, seq=1, heads=32, kv_heads=8, head_dim=128, rotary_dim=128, layout="half",
             type="bf16", axes=1, learned=False, far=1000000, inverse=False),
        # 256 boards: neighbouring channels, x and y axes, frequencies learned for each key head
        dict(name="rotary 256 boards", op="rotary", batch=256, seq=361, heads=12, kv_heads=6, head_dim=32, rotary_dim=32, layout="interleaved",
             type="fp16", axes=2, learned=True, far=0, inverse=False),
        # four long sequences, three quarters of each head turned
        dict(name="rotary long", op="rotary", batch=4, seq=8191, heads=32, kv_heads=8, head_dim=128, rotary_dim=96, layout="half",
             type="bf16", axes=1, learned=False, far=100000, inverse=False),
    ]


def _log(rng, low, high):
    return int(min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "linear", "rotary"])
    if op == "norm":
        wants = rng.choice(["y", "row", "mx", "row+y", "mx+y"])
        norm = rng.random() < 0.8
        if not norm:
            wants = rng.choice(["row", "mx"])
        channels = _log(rng, 16, 8192)
        if "mx" in wants:
            channels = max(32, channels // 32 * 32)
        elif rng.random() < 0.6:
            channels = max(8, channels // 8 * 8)
        rows = _log(rng, 1, min(100000, 33000000 // channels))
        return dict(op=op, rows=rows, channels=channels, type=rng.choice(["fp16", "bf16", "bf16", "fp32"]), residual=norm and rng.random() < 0.6,
                    masked=norm and rng.random() < 0.4, norm=norm, wants=wants)
    if op == "linear":
        scales = rng.choice(["row", "mx"])
        k = _log(rng, 64, 11008) // 32 * 32 + (16 if scales == "row" and rng.random() < 0.3 else 0)
        n = _log(rng, 32, 11008)
        if rng.random() < 0.7:
            n = max(32, n // 16 * 16)
        most = min(92416, int(360e9 / (k * n)), int(180e6 / n))
        return dict(op=op, rows=_log(rng, 1, most), k=k, n=n, scales=scales, out=rng.choice(["fp16", "bf16", "bf16", "fp32"]),
                    bias=rng.random() < 0.5)
    head_dim = rng.choice([8, 16, 32, 48, 64, 80, 96, 128, 128, 192, 256])
    rotary_dim = head_dim if rng.random() < 0.6 else max(2, int(head_dim * rng.uniform(0.25, 1.0)) // 2 * 2)
    kv_heads = rng.choice([1, 2, 3, 4, 6, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    axes = rng.choice([1, 1, 2])
    if axes == 2:  # boards
        batch, seq = _log(rng, 1, max(1, min(256, 80000000 // (BOARD * (heads + kv_heads) * head_dim)))), BOARD
    else:
        tokens = _log(rng, 1, min(60000, 80000000 // ((heads + kv_heads) * head_dim)))
        batch = min(tokens, _log(rng, 1, 64))
        seq = max(1, tokens // batch)
    return dict(op=op, batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, head_dim=head_dim, rotary_dim=rotary_dim,
                layout=rng.choice(["half", "interleaved"]), type=rng.choice(["fp16", "bf16", "bf16", "fp32"]), axes=axes,
                learned=rng.random() < 0.3, far=0 if axes == 2 else _log(rng, 1, 1000000), inverse=rng.random() < 0.2)


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _activations(g, rows, channels, dtype):
    """A trunk's activations: channels of different spread, a few of them large."""
    spread = torch.exp(0.5 * torch.randn(channels, device="cuda", generator=g))
    spread = spread * (1 + 15 * (torch.rand(channels, device="cuda", generator=g) < 0.01))
    return (torch.randn(rows, channels, device="cuda", generator=g) * spread).to(dtype)


def _row_scales(v):
    """Scales and codes of each row of v (fp32 or fp64): amax / 448, 1 where the row is all zero."""
    amax = v.abs().amax(dim=1)
    scale = torch.where(amax > 0, (amax / E4M3_MAX).clamp_min(2.0 ** -126), torch.ones_like(amax))
    return (v / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX), scale


def _mx_scales(v):
    """Exponents and codes of each 32 channels of v: the smallest power of two that brings them to at most 448, 1 where all are zero."""
    b = v.view(v.shape[0], -1, 32)
    amax = b.abs().amax(dim=2)
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [1/2, 1); 448 = 7/8 2^9
    e = torch.where(amax > 0, (e - 9 + (m > 0.875).to(e.dtype)).clamp(-127, 127), torch.zeros_like(e))
    # in two steps: 2^127 and 2^-127 are not both normal numbers
    half = torch.div(e, 2, rounding_mode="floor")
    b = torch.ldexp(torch.ldexp(b, -half[..., None].to(b.dtype)), (half - e)[..., None].to(b.dtype))
    return b.reshape(v.shape).clamp(-E4M3_MAX, E4M3_MAX), e


def _eight(v, scales):
    """(codes, scales) of v in e4m3, as the operators lay them out: scales fp32 [rows] or e8m0 [rows][channels / 32]."""
    if scales == "row":
        c, s = _row_scales(v)
        return c.to(torch.float8_e4m3fn), s.float()
    c, e = _mx_scales(v)
    return c.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _of_eight(codes, scales, dtype):
    if scales.dim() == 1:
        return codes.to(dtype) * scales.to(dtype)[:, None]
    return (codes.to(dtype).view(codes.shape[0], -1, 32) * scales.to(dtype)[..., None]).view(codes.shape)


def _frequencies(case, g):
    """fp64 [heads that have their own][axes][pairs]"""
    pairs = case["rotary_dim"] // 2
    own_heads = case["kv_heads"] if case["learned"] else 1
    if case["learned"]:
        return torch.rand(own_heads, case["axes"], pairs, device="cuda", generator=g, dtype=torch.float64) * 1.4 - 0.7
    f = 10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)
    if case["axes"] == 1:
        return f.view(1, 1, pairs)
    x_axis = (torch.arange(pairs, device="cuda") >= pairs // 2).double()  # the first half of the pairs turns with y, the others with x
    return torch.stack([f * x_axis, f * (1 - x_axis)]).view(1, 2, pairs)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = dict(case)
    if case["op"] == "norm":
        dtype = TYPES[case["type"]]
        s["x"] = _activations(g, case["rows"], case["channels"], dtype)
        s["r"] = _activations(g, case["rows"], case["channels"], dtype) if case["residual"] else None
        s["w"] = 1 + 0.3 * torch.randn(case["channels"], device="cuda", generator=g) if case["norm"] else None
        s["mask"] = None
        if case["masked"]:  # boards of 9, 13 and 19 points a side in 19x19 buffers
            r = torch.arange(case["rows"], device="cuda")
            sizes = torch.tensor([19, 13, 9, 19], device="cuda")
            side = sizes[torch.randint(0, 4, (case["rows"] // BOARD + 1,), device="cuda", generator=g)][r // BOARD]
            s["mask"] = ((r % BOARD // 19 < side) & (r % 19 < side)).float()
    elif case["op"] == "linear":
        s["a"], s["as"] = _eight(_activations(g, case["rows"], case["k"], torch.float32), case["scales"])
        w = torch.randn(case["n"], case["k"], device="cuda", generator=g) / math.sqrt(case["k"])
        s["w"], s["ws"] = _eight(w, case["scales"])
        s["bias"] = 0.1 * torch.randn(case["n"], device="cuda", generator=g) if case["bias"] else None
    else:
        dtype = TYPES[case["type"]]
        shape = (case["batch"], case["seq"])
        s["q"] = torch.randn(*shape, case["heads"], case["head_dim"], device="cuda", generator=g).to(dtype)
        s["k"] = torch.randn(*shape, case["kv_heads"], case["head_dim"], device="cuda", generator=g).to(dtype)
        s["f"] = _frequencies(case, g)
        if case["axes"] == 2:  # every board's cells, x and y
            c = torch.arange(case["seq"], device="cuda")
            s["pos"] = torch.stack([c % 19, c // 19], dim=1).int()
        else:  # each sequence from a place of its own
            start = torch.randint(0, case["far"] + 1, (case["batch"], 1), device="cuda", generator=g)
            s["pos"] = start + torch.arange(case["seq"], device="cuda")
        s["magnitude"] = 1.0 if case["axes"] == 2 else 1.0 + 0.1 * (seed % 3)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------

def _norm_plain(s):
    dtype = s["x"].dtype
    out = {}
    h = s["x"].float()
    if s["r"] is not None:
        out["sum"] = (h + s["r"].float()).to(dtype)
        h = out["sum"].float()
    if s["norm"]:
        y = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + 1e-6) * s["w"]
        if s["mask"] is not None:
            y = torch.where(s["mask"][:, None] != 0, y, torch.zeros_like(y))
    else:
        y = h
    if "y" in s["wants"]:
        out["y"] = y.to(dtype)
    if s["wants"] != "y":
        out["codes"], out["scales"] = _eight(y, s["wants"].split("+")[0])
    return out


def _rotary_plain(x, s):
    f, pairs = s["f"], s["rotary_dim"] // 2
    p = s["pos"].double().view(-1 if s["axes"] == 2 else s["batch"], s["seq"], s["axes"])
    if s["axes"] == 2:
        p = p[:1]
    angle = (p[:, :, None, :, None] * f).sum(dim=3)  # [batch or 1][seq][heads of f][pairs], fp64: far positions
    if s["inverse"]:
        angle = -angle
    c, n = (angle.cos() * s["magnitude"]).float(), (angle.sin() * s["magnitude"]).float()
    if f.shape[0] > 1:  # query head h turns as the key head it reads
        c, n = (t.repeat_interleave(x.shape[2] // f.shape[0], dim=2) for t in (c, n))
    v = x.float()
    if s["layout"] == "half":
        a, b = v[..., :pairs], v[..., pairs:2 * pairs]
        turned = torch.cat([a * c - b * n, a * n + b * c], dim=-1)
    else:
        a, b = v[..., 0:2 * pairs:2], v[..., 1:2 * pairs:2]
        turned = torch.stack([a * c - b * n, a * n + b * c], dim=-1).flatten(-2)
    return torch.cat([turned, v[..., 2 * pairs:]], dim=-1).to(x.dtype)


def run(state):
    s = state
    if own:
        from katago_amd import ops

        if s["op"] == "norm":
            scales = None if s["wants"] == "y" else s["wants"].split("+")[0]
            if not s["norm"]:
                codes, sc = ops.quantize(s["x"], scales)
                return {"codes": codes, "scales": sc}
            r = ops.rms_norm(s["x"], s["w"], 1e-6, residual=s["r"], mask=s["mask"], scales=scales, want_y="y" in s["wants"])
            return {k: v for k, v in (("sum", r.sum), ("y", r.y), ("codes", r.codes), ("scales", r.scales)) if v is not None}
        if s["op"] == "linear":
            return ops.linear8(s["a"], s["as"], s["w"], s["ws"], s["bias"], out_dtype=TYPES[s["out"]])
        return ops.rotary(s["q"], s["k"], s["pos"], s["f"], layout=s["layout"], magnitude=s["magnitude"], inverse=s["inverse"])
    if s["op"] == "norm":
        return _norm_plain(s)
    if s["op"] == "linear":
        y = _of_eight(s["a"], s["as"], torch.float32) @ _of_eight(s["w"], s["ws"], torch.float32).t()
        if s["bias"] is not None:
            y = y + s["bias"]
        return y.to(TYPES[s["out"]])
    return _rotary_plain(s["q"], s), _rotary_plain(s["k"], s)


# ---- what a pass cannot do without, and its results in 64 bits -----------------------------------------------------

def work(case):
    size = {"fp16": 2, "bf16": 2, "fp32": 4}
    if case["op"] == "norm":
        n, e = case["rows"] * case["channels"], size[case["type"]]
        b = n * e * (3 if case["residual"] else 1) + (n * e if "y" in case["wants"] else 0)
        if case["wants"] != "y":
            b += n + (4 * case["rows"] if "row" in case["wants"] else n // 32)
        return {"bytes": b + (4 * case["channels"] if case["norm"] else 0) + (4 * case["rows"] if case["masked"] else 0), "flops": 5 * n}
    if case["op"] == "linear":
        b = case["k"] * (case["rows"] + case["n"]) + case["rows"] * case["n"] * size[case["out"]]
        b += 4 * (case["rows"] + case["n"]) if case["scales"] == "row" else case["k"] // 32 * (case["rows"] + case["n"])
        return {"bytes": b + (4 * case["n"] if case["bias"] else 0), "flops": 2 * case["rows"] * case["n"] * case["k"]}
    tokens, heads = case["batch"] * case["seq"], case["heads"] + case["kv_heads"]
    positions = 8 * case["seq"] if case["axes"] == 2 else 8 * tokens
    return {"bytes": 2 * tokens * heads * case["head_dim"] * size[case["type"]] + positions, "flops": 3 * tokens * heads * case["rotary_dim"]}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        out = {}
        v = s["x"].double()
        if s["r"] is not None:
            v = (v + s["r"].double()).to(s["x"].dtype)
            out["sum"], v = v.double(), v.double()
        if case["norm"]:
            v = v / ((v * v).sum(1) / case["channels"] + 1e-6).sqrt()[:, None] * s["w"].double()
            if s["mask"] is not None:
                v[s["mask"] == 0] = 0.0
        if "y" in case["wants"]:
            out["y"] = v
        if "row" in case["wants"]:
            top = v.abs().max(1).values
            out["scales"] = torch.where(top == 0, 1.0, top / 448)
            out["codes"] = (v / out["scales"][:, None]).to(torch.float8_e4m3fn).double()
        elif "mx" in case["wants"]:
            blocks = v.reshape(case["rows"], -1, 32)
            top = blocks.abs().max(2).values
            e = torch.ceil(torch.log2(torch.where(top == 0, 448.0, top) / 448)).clamp(-127, 127)
            out["scales"] = torch.exp2(e)
            out["codes"] = (blocks / out["scales"][..., None]).to(torch.float8_e4m3fn).double().reshape(v.shape)
        return out
    if case["op"] == "linear":
        def values(codes, scales):
            each = scales.double()[:, None] if scales.dim() == 1 else scales.double().repeat_interleave(32, dim=1)
            return codes.double() * each
        y = values(s["a"], s["as"]).mm(values(s["w"], s["ws"]).t())
        return y if s["bias"] is None else y + s["bias"].double()
    pairs, pos = case["rotary_dim"] // 2, s["pos"].double()
    if case["axes"] == 2:
        angle = torch.einsum("sa,hap->shp", pos, s["f"]).unsqueeze(0)
    else:
        angle = torch.einsum("bs,hp->bshp", pos, s["f"][:, 0])
    turn = torch.polar(torch.full_like(angle, s["magnitude"]), -angle if case["inverse"] else angle)

    def turned(x):
        x = x.double()
        u = turn if turn.shape[2] == 1 else turn[:, :, torch.arange(x.shape[2], device=x.device) // (x.shape[2] // turn.shape[2])]
        where = torch.arange(2 * pairs, device=x.device).view((2, pairs) if case["layout"] == "half" else (pairs, 2))
        re, im = (where[0], where[1]) if case["layout"] == "half" else (where[:, 0], where[:, 1])
        z = torch.complex(x[..., re], x[..., im]) * u
        y = x.clone()
        y[..., re], y[..., im] = z.real, z.imag
        return y

    return turned(s["q"]), turned(s["k"])
