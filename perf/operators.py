"""Workloads of the operators between the quantised layers of a transformer block: 4-bit linear layers, RMSNorm
with the residual's addition (16-bit or int8 output), rotary positions.

Sizes are those of the texture UNet (channels 320 / 640 / 1280, 64-wide heads, 77 text tokens of width 1024), of the
image encoder (257 tokens, 1536 / 6144 wide), and generic ones: single tokens, a 32768-token prompt, widths of 4096
and 8192.  ``own`` selects the package's operators; without it the same results come from elementary torch
operations in 32 bits (64 for angles), rounded once at the end.
"""
import importlib
import math

import torch

PKG = "hunyuan3d-tools_b200"
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}

own = False


def _mod(name):
    return importlib.import_module(PKG + "." + name)


def _w4(name, m, k, n, group, zeros=False, epilogue="linear", bias=True, dtype="bf16"):
    return {"name": name, "kind": "w4", "m": m, "k": k, "n": n, "group": group, "zeros": zeros, "epilogue": epilogue,
            "bias": bias, "dtype": dtype}


def _norm(name, rows, width, out, residual, dtype="bf16"):
    return {"name": name, "kind": "norm", "rows": rows, "width": width, "out": out, "residual": residual, "dtype": dtype}


def _rot(name, batch, tokens, heads, kv_heads, dim, rot, interleaved, axes=1, stacked=False, scaling="none", start=0,
         inverse=False, dtype="bf16"):
    return {"name": name, "kind": "rotary", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "rot": rot, "interleaved": interleaved, "axes": axes, "stacked": stacked, "scaling": scaling,
            "start": start, "inverse": inverse, "dtype": dtype}


def listed():
    return [
        # Time-embedding projection of a ResNet block, one row per sample: the smallest layer of a denoise step.
        _w4("w4_time_proj_12x1280x640", 12, 1280, 640, 64),
        # One decode token through the widest generic layer: the weight stream is all there is.
        _w4("w4_token_1x8192x8192", 1, 8192, 8192, 128, bias=False, dtype="fp16"),
        # A few sequences decoding together through a gated up-projection; groups with zero points.
        _w4("w4_geglu_7x1280x10240", 7, 1280, 10240, 32, zeros=True, epilogue="geglu"),
        # Image encoder's first MLP layer: the 257 tokens of one image.
        _w4("w4_encoder_fc1_257x1536x6144", 257, 1536, 6144, 128, epilogue="gelu", dtype="fp16"),
        # Cross-attention keys and values stacked: 12 samples x 77 text tokens, no bias.
        _w4("w4_cross_kv_924x1024x2560", 924, 1024, 2560, 64, bias=False),
        # The norm of one decode token: latency.
        _norm("norm_add_1x4096", 1, 4096, "half", True),
        # Residual stream of the middle resolution into int8 codes for the stacked q / k / v projection.
        _norm("norm_add_int8_12288x640", 12288, 640, "int8", True),
        # The image encoder's tokens of 15 images into int8 codes, no residual.
        _norm("norm_int8_3855x1536", 3855, 1536, "int8", False, dtype="fp16"),
        # A long prompt at the widest generic model, 16-bit output.
        _norm("norm_add_8192x8192", 8192, 8192, "half", True),
        # Eight sequences, one decode token each, far into their context; shared key heads.
        _rot("rotary_token_8x1x32x8x128", 8, 1, 32, 8, 128, 128, False, scaling="by_parts", start=100000),
        # Multiview attention of the middle resolution: q and k inside a stacked projection, positions (view, row,
        # column), pairs interleaved.
        _rot("rotary_views_2x6144x10x64", 2, 6144, 10, 10, 64, 64, True, axes=3, stacked=True),
        # A long prompt with shared key heads, half of each head rotated, context stretched four times.
        _rot("rotary_prompt_1x32768x32x8x128", 1, 32768, 32, 8, 128, 64, False, scaling="linear", dtype="fp16"),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi, max(lo, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choices(["w4", "norm", "rotary"], weights=[5, 4, 3])[0]
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "w4":
        while True:
            m, k, n = _log(rng, 1, 1024), _log(rng, 128, 8192, 64), _log(rng, 64, 16384, 16)
            group = rng.choice([g for g in (32, 64, 128) if k % g == 0])
            epilogue = rng.choice(["linear", "linear", "gelu", "geglu"])
            if epilogue == "geglu":
                n -= n % 32
            if k * n <= 8192 * 8192 and m * k * n <= 257 * 1536 * 6144 and m * (k + n) <= 924 * (1024 + 2560):
                return {"kind": kind, "m": m, "k": k, "n": n, "group": group, "zeros": rng.random() < 0.4,
                        "epilogue": epilogue, "bias": rng.random() < 0.6, "dtype": dtype}
    if kind == "norm":
        while True:
            rows, width = _log(rng, 1, 65536), _log(rng, 64, 16384, 8)
            if rows * width <= 8192 * 8192:
                return {"kind": kind, "rows": rows, "width": width, "out": rng.choice(["half", "int8"]),
                        "residual": rng.random() < 0.7, "dtype": dtype}
    while True:
        batch, tokens = _log(rng, 1, 16), _log(rng, 1, 65536)
        kv, dim = rng.choice([1, 2, 4, 5, 8, 10, 20]), rng.choice([32, 40, 64, 80, 96, 128, 256])
        heads = kv * rng.choice([1, 1, 4, 6])
        if batch * tokens * (heads + kv) * dim <= 32768 * 40 * 128:
            axes = rng.choice([1, 1, 2, 3])
            rot = dim if axes == 3 or rng.random() < 0.6 else dim // 2
            return {"kind": kind, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv, "dim": dim, "rot": rot,
                    "interleaved": rng.random() < 0.5, "axes": axes, "stacked": rng.random() < 0.4,
                    "scaling": rng.choice(["none", "linear", "ntk", "by_parts"]),
                    "start": rng.choice([0, 0, 1000, 500000]), "inverse": rng.random() < 0.2, "dtype": dtype}


# ---------------------------------------------------------------------------------------
# what a program has in hand before the call
# ---------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _activation(g, shape, dtype):
    """N(0,1) with 0.1 % of the entries at +-20, as the linear layers' inputs."""
    x = torch.randn(shape, generator=g, device=DEV)
    u = torch.rand(shape, generator=g, device=DEV)
    x = torch.where(u < 0.0005, 20.0, torch.where(u > 0.9995, -20.0, x))
    return x.to(dtype)


def _axis_dims(case):
    """Rotated dimensions of each axis: even, as equal as they can be."""
    pairs, a = case["rot"] // 2, case["axes"]
    return [2 * (pairs // a + (1 if i < pairs % a else 0)) for i in range(a)]


_SCALING = {"none": None, "linear": {"kind": "linear", "factor": 4.0}, "ntk": {"kind": "ntk", "factor": 4.0},
            "by_parts": {"kind": "by_parts", "factor": 8.0, "original_length": 8192, "slow": 1.0, "fast": 4.0}}


def _positions(case):
    b, n, a, start = case["batch"], case["tokens"], case["axes"], case["start"]
    if a == 1:      # each sequence at a place of its own
        return start + torch.arange(b, device=DEV)[:, None] * 37 + torch.arange(n, device=DEV)
    side = max(1, math.isqrt(max(1, n // 6)))
    i = torch.arange(n, device=DEV)
    grid = [i // (side * side), i // side % side, i % side][3 - a:]
    return torch.stack(grid, dim=-1) + start


def _frequencies(case):
    """Angle per unit of position of each rotated pair, in 64 bits, and the axis it belongs to."""
    out, axis, how = [], [], _SCALING[case["scaling"]]
    for a, d in enumerate(_axis_dims(case)):
        base = 10000.0
        if how and how["kind"] == "ntk" and d > 2:
            base *= how["factor"] ** (d / (d - 2))
        w = base ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
        if how and how["kind"] == "linear":
            w = w / how["factor"]
        elif how and how["kind"] == "by_parts":
            turns = how["original_length"] * w / (2 * math.pi)
            ramp = ((turns - how["slow"]) / (how["fast"] - how["slow"])).clamp(0, 1)
            w = w * ramp + w / how["factor"] * (1 - ramp)
        out.append(w)
        axis += [a] * (d // 2)
    return torch.cat(out).to(DEV), torch.tensor(axis, device=DEV)


def prepare(case, seed):
    g = _gen(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    state = {"kind": kind, "case": case, "dtype": dtype}
    if kind == "w4":
        m, k, n, group = case["m"], case["k"], case["n"], case["group"]
        w = (torch.randn(n, k // group, group, generator=g, device=DEV) * 0.02)
        if case["zeros"]:
            lo, hi = w.amin(-1, keepdim=True), w.amax(-1, keepdim=True)
            scale = ((hi - lo) / 15).to(dtype)
            zero = (-lo / scale.float()).round().clamp(0, 15)
        else:
            scale = (w.abs().amax(-1, keepdim=True) / 7).to(dtype)
            zero = torch.full_like(scale, 8.0, dtype=torch.float32)
        codes = ((w / scale.float()).round() + zero).clamp(0, 15).to(torch.uint8).view(n, k)
        del w
        state.update(x=_activation(g, (m, k), dtype), codes=codes, scale=scale.squeeze(-1),
                     zero=zero.squeeze(-1).to(torch.uint8) if case["zeros"] else None,
                     bias=(torch.randn(n, generator=g, device=DEV) * 0.01).to(dtype) if case["bias"] else None)
        if own:     # the layer, its codes laid out once as a program keeps them
            layer = _mod("quantize_utils").Int4Linear.from_codes(codes, state["scale"], state["zero"], state["bias"])
            if case["epilogue"] == "geglu":
                layer.interleave_geglu_rows()
            else:
                layer.epilogue = case["epilogue"]
            state["layer"] = layer
        return state
    if kind == "norm":
        rows, width = case["rows"], case["width"]
        state.update(x=_activation(g, (rows, width), dtype),
                     add=torch.randn(rows, width, generator=g, device=DEV).to(dtype) if case["residual"] else None,
                     weight=(1.0 + 0.1 * torch.randn(width, generator=g, device=DEV)).to(dtype), eps=1e-6)
        if own:
            norm = torch.nn.RMSNorm(width, eps=1e-6, device=DEV, dtype=dtype).requires_grad_(False)
            norm.weight.copy_(state["weight"])
            qu = _mod("quantize_utils")
            state["norm"] = qu.Int8RMSNorm(norm) if case["out"] == "int8" else qu.AddRMSNorm(norm)
        return state
    b, n, h, hk, d = case["batch"], case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    if case["stacked"]:
        qkv = torch.randn(b, n, (h + 2 * hk) * d, generator=g, device=DEV).to(dtype)
        q, k = qkv[..., :h * d].view(b, n, h, d), qkv[..., h * d:(h + hk) * d].view(b, n, hk, d)
    else:
        q = torch.randn(b, n, h, d, generator=g, device=DEV).to(dtype)
        k = torch.randn(b, n, hk, d, generator=g, device=DEV).to(dtype)
    w, axis = _frequencies(case)
    state.update(q=q, k=k, positions=_positions(case), w=w, axis=axis)
    if own:
        state["rotary"] = _mod("rotary").RotaryPositions(
            d, rotary_dim=case["rot"], base=10000.0, interleaved=case["interleaved"], axes=_axis_dims(case),
            scaling=_SCALING[case["scaling"]])
    return state


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def _plain_gelu(v):
    return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))


def _plain_w4(s):
    case, group = s["case"], s["case"]["group"]
    n, k = s["codes"].shape
    c = s["codes"].view(n, k // group, group).float()
    z = 8.0 if s["zero"] is None else s["zero"].float()[..., None]
    w = ((c - z) * s["scale"].float()[..., None]).view(n, k)
    y = s["x"].float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if case["epilogue"] == "gelu":
        y = _plain_gelu(y)
    elif case["epilogue"] == "geglu":
        y = y[:, :n // 2] * _plain_gelu(y[:, n // 2:])
    return y.to(s["dtype"])


def _plain_norm(s):
    x, dtype = s["x"], s["dtype"]
    total = None
    if s["add"] is not None:
        total = x = (x.float() + s["add"].float()).to(dtype)
    f = x.float()
    y = (f * torch.rsqrt((f * f).mean(-1, keepdim=True) + s["eps"]) * s["weight"].float()).to(dtype)
    if s["case"]["out"] == "int8":
        f = y.float()
        scale = f.abs().amax(-1, keepdim=True).clamp(min=1e-8) / 127.0
        y = ((f / scale).round().clamp(-128, 127) * scale).to(dtype)
    return y if total is None else (total, y)


def _plain_rotary(s):
    case, dtype = s["case"], s["dtype"]
    p = s["positions"] if case["axes"] > 1 else s["positions"][..., None]
    angle = p.double()[..., s["axis"]] * s["w"]
    cos, sin = angle.cos().float()[..., None, :], angle.sin().float()[..., None, :]
    if case["inverse"]:
        sin = -sin
    rot, half = case["rot"], case["rot"] // 2

    def turn(t):
        f = t[..., :rot].float()
        if case["interleaved"]:
            u, v = f[..., 0::2], f[..., 1::2]
            r = torch.stack([u * cos - v * sin, v * cos + u * sin], dim=-1).flatten(-2)
        else:
            u, v = f[..., :half], f[..., half:]
            r = torch.cat([u * cos - v * sin, v * cos + u * sin], dim=-1)
        return torch.cat([r.to(dtype), t[..., rot:]], dim=-1)

    return turn(s["q"]), turn(s["k"])


@torch.no_grad()
def run(state):
    kind = state["kind"]
    if own:
        if kind == "w4":
            return state["layer"](state["x"])
        if kind == "norm":
            if state["case"]["out"] == "int8":     # the codes as the values they stand for
                if state["add"] is None:
                    return state["norm"](state["x"]).dequantize()
                total, y = state["norm"](state["x"], state["add"])
                return total, y.dequantize()
            return state["norm"](state["x"]) if state["add"] is None else state["norm"](state["x"], state["add"])
        return state["rotary"](state["q"], state["k"], state["positions"], inverse=state["case"]["inverse"])
    return {"w4": _plain_w4, "norm": _plain_norm, "rotary": _plain_rotary}[kind](state)


# ---------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "w4":
        m, k, n = case["m"], case["k"], case["n"]
        n_out = n // 2 if case["epilogue"] == "geglu" else n
        groups = n * (k // case["group"])
        return {"bytes": n * k / 2 + groups * (3 if case["zeros"] else 2) + 2 * m * (k + n_out) + (2 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    if kind == "norm":
        e = case["rows"] * case["width"]
        read = 4 * e if case["residual"] else 2 * e
        write = (2 * e if case["residual"] else 0) + (e + 4 * case["rows"] if case["out"] == "int8" else 2 * e)
        return {"bytes": read + write + 2 * case["width"], "flops": 5 * e}
    tokens = case["batch"] * case["tokens"]
    e = tokens * (case["heads"] + case["kv_heads"]) * case["dim"]
    positions = 8 * (tokens if case["axes"] == 1 else case["tokens"] * case["axes"])
    return {"bytes": 4 * e + positions, "flops": 3 * e}


# ---------------------------------------------------------------------------------------
# the operators' definitions in 64 bits
# ---------------------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "w4":
        g = case["group"]
        w = s["codes"].double() - (8.0 if s["zero"] is None else s["zero"].double().repeat_interleave(g, dim=1))
        w *= s["scale"].double().repeat_interleave(g, dim=1)
        y = torch.nn.functional.linear(s["x"].double(), w, None if s["bias"] is None else s["bias"].double())
        if case["epilogue"] == "linear":
            return y
        value, gate = (1.0, y) if case["epilogue"] == "gelu" else y.tensor_split(2, dim=1)
        return value * gate * torch.special.ndtr(gate)
    if case["kind"] == "norm":
        t = s["x"].double()
        if s["add"] is not None:
            t = (t + s["add"].double()).to(s["dtype"]).double()       # the stream is kept in its own type
        y = t / (t.square().sum(-1, keepdim=True) / case["width"] + s["eps"]).sqrt() * s["weight"].double()
        if case["out"] == "int8":
            y = y.to(s["dtype"]).double()                             # what is quantised is the stored norm
            step = y.abs().amax(-1, keepdim=True).clamp(min=1e-8) / 127
            y = (y / step).round() * step
        return y if s["add"] is None else (t, y)
    # a pair is a complex number that is multiplied by exp(i angle)
    pairs, how = case["rot"] // 2, case["scaling"]
    p = s["positions"].double()
    angle, first = [], 0
    for a, dims in enumerate(_axis_dims(case)):
        along = p if case["axes"] == 1 else p[..., a]
        for i in range(dims // 2):
            f = math.exp(-math.log(10000.0) * 2 * i / dims)
            if how == "linear":
                f /= 4.0
            elif how == "ntk" and dims > 2:
                f *= 4.0 ** (-2 * i / (dims - 2))
            elif how == "by_parts":
                keep = min(1.0, max(0.0, (8192 * f / (2 * math.pi) - 1.0) / 3.0))
                f = f * keep + f / 8.0 * (1.0 - keep)
            angle.append(along * (-f if case["inverse"] else f))
    factor = torch.polar(torch.ones(1, dtype=torch.float64, device=DEV), torch.stack(angle, dim=-1))[..., None, :]

    def turned(t):
        t = t.double()
        head = t[..., :2 * pairs]
        z = head.unflatten(-1, (pairs, 2)) if case["interleaved"] else head.unflatten(-1, (2, pairs)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * factor)
        z = z if case["interleaved"] else z.transpose(-1, -2)
        return torch.cat([z.flatten(-2), t[..., 2 * pairs:]], dim=-1)

    return turned(s["q"]), turned(s["k"])
