"""Operators of transformer blocks in this library, as measurable cases: the microscaled FP4 linear, the norms before and after a block
fused with its gate and residual, and the rotary embedding over several position axes.

A case is a dict of plain values; "kind" picks the operator, the rest are sizes and options:

  fp4_linear   quantize of x [m, k] and product with a quantized weight [n, k]     m, n, k, fmt, gelu, residual, dtype
  norm         residual + gate * post-norm, then the next block's pre-norm         batch, seq, dim, post, pre, mod, out, dtype
  rope         rotary embedding of q and k, angles from positions on several axes  batch, seq, q_heads, k_heads, head_dim, axes, style, norm,
                                                                                   start, dtype
  norm_linear  the norm with its result in FP4, then the linear that takes it      m, n, k, fmt, dtype

Where `own` is false run() computes the plain form with elementary torch operations in 32 bits; where it is true it makes the calls that a
user of this library makes.  exact() restates the definitions in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
GROUP = {"nvfp4": 16, "mxfp4": 32}
EPS = 1e-6
THETA = 10000.0


def listed():
    return [
        # The modulation linear of a block: one conditioning vector against 28 million weights.  Launches, latency, the weight stream.
        {"name": "fp4_one_row", "kind": "fp4_linear", "m": 1, "n": 9216, "k": 3072, "fmt": "nvfp4", "gelu": False, "residual": False,
         "dtype": "bf16"},
        # Key/value projection of the text in cross attention: 2 x 77 tokens, a small matrix.
        {"name": "fp4_text", "kind": "fp4_linear", "m": 154, "n": 1280, "k": 2048, "fmt": "mxfp4", "gelu": False, "residual": False,
         "dtype": "fp16"},
        # Feed-forward output linear over an odd number of tokens, deep K, with its residual.
        {"name": "fp4_ragged", "kind": "fp4_linear", "m": 1317, "n": 3072, "k": 12288, "fmt": "mxfp4", "gelu": False, "residual": True,
         "dtype": "fp16"},
        # The MLP projection of a block over the tokens of a 1024 x 1024 image: the largest case.
        {"name": "fp4_mlp", "kind": "fp4_linear", "m": 4608, "n": 12288, "k": 3072, "fmt": "nvfp4", "gelu": True, "residual": False,
         "dtype": "bf16"},
        # One token of each of two sequences: nothing but latency.
        {"name": "norm_one_token", "kind": "norm", "batch": 2, "seq": 1, "dim": 3072, "post": "rms", "pre": "rms", "mod": True,
         "out": "h", "dtype": "bf16"},
        # A block of the image stream at 1024 x 1024 with both norms and the modulation: a pure memory pass.
        {"name": "norm_image", "kind": "norm", "batch": 1, "seq": 4608, "dim": 3072, "post": "rms", "pre": "layer", "mod": True,
         "out": "h", "dtype": "bf16"},
        # Two images of odd size, no modulation, the result in e4m3 for an FP8 linear.
        {"name": "norm_ragged_e4m3", "kind": "norm", "batch": 2, "seq": 1155, "dim": 1280, "post": "layer", "pre": "layer", "mod": False,
         "out": "e4m3", "dtype": "fp16"},
        # A single new token of three sequences, far along its axes, fewer key heads than query heads, part of the head rotated.
        {"name": "rope_one_token", "kind": "rope", "batch": 3, "seq": 1, "q_heads": 24, "k_heads": 8, "head_dim": 128, "axes": "16,24,24",
         "style": "halves", "norm": False, "start": 1000003, "dtype": "fp16"},
        # q and k of an image block out of the packed projection: three axes, interleaved pairs, QK norm.
        {"name": "rope_image", "kind": "rope", "batch": 1, "seq": 4608, "q_heads": 24, "k_heads": 24, "head_dim": 128, "axes": "16,56,56",
         "style": "interleaved", "norm": True, "start": 0, "dtype": "bf16"},
        # A video clip of 21 latent frames of 30 x 52 patches: time, height and width.
        {"name": "rope_video", "kind": "rope", "batch": 1, "seq": 32760, "q_heads": 12, "k_heads": 12, "head_dim": 128, "axes": "44,42,42",
         "style": "halves", "norm": False, "start": 0, "dtype": "bf16"},
        # The end of one block and the start of the next: norm, FP4 activations written by it, the QKV projection.
        {"name": "norm_fp4_qkv", "kind": "norm_linear", "m": 1155, "n": 9216, "k": 3072, "fmt": "nvfp4", "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case of the same ranges; costs no more than the largest listed one."""
    kind = rng.choice(["fp4_linear", "fp4_linear", "norm", "rope", "norm_linear"])
    dtype = rng.choice(["bf16", "fp16"])
    fmt = rng.choice(["nvfp4", "mxfp4"])
    if kind == "fp4_linear":
        while True:
            m, n, k = _log(rng, 1, 4608), _log(rng, 64, 18432), 32 * _log(rng, 2, 480)
            n = n if rng.random() < 0.3 else (n + 7) // 8 * 8
            if m * n * k <= 4608 * 12288 * 3072:
                break
        return {"kind": kind, "m": m, "n": n, "k": k, "fmt": fmt, "gelu": rng.random() < 0.4, "residual": rng.random() < 0.4, "dtype": dtype}
    if kind == "norm":
        batch, dim = rng.choice([1, 1, 2, 3]), 8 * _log(rng, 8, 1024)
        seq = _log(rng, 1, max(1, min(4608, 4608 * 3072 // dim)) // batch)
        return {"kind": kind, "batch": batch, "seq": seq, "dim": dim, "post": rng.choice(["none", "rms", "layer"]),
                "pre": rng.choice(["rms", "layer"]), "mod": rng.random() < 0.6, "out": rng.choice(["h", "h", "e4m3"]), "dtype": dtype}
    if kind == "rope":
        batch, q_heads = rng.choice([1, 1, 2, 3]), rng.choice([1, 8, 12, 16, 20, 24, 32, 40])
        head_dim = rng.choice([64, 64, 72, 80, 96, 128, 128, 256])
        axes = rng.choice([1, 2, 3])
        pairs = head_dim // 2 if rng.random() < 0.7 else head_dim // 4
        cut = [pairs // axes] * axes
        cut[0] += pairs - sum(cut)
        seq = _log(rng, 1, max(2, min(32760, 4608 * 48 * 128 // (2 * q_heads * head_dim * batch))))
        return {"kind": kind, "batch": batch, "seq": seq, "q_heads": q_heads, "k_heads": q_heads // rng.choice([1, 1, 4]) or 1,
                "head_dim": head_dim, "axes": ",".join(str(2 * c) for c in cut), "style": rng.choice(["interleaved", "halves"]),
                "norm": rng.random() < 0.5, "start": rng.choice([0, 0, 4000, 1000003]), "dtype": dtype}
    return {"kind": kind, "m": _log(rng, 1, 4608), "n": 8 * _log(rng, 16, 1152), "k": 32 * _log(rng, 8, 96), "fmt": fmt, "dtype": dtype}


# ----------------------------------------------------------------------------- inputs
def _randn(g, shape, std, dtype):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _activations(g, rows, dim, dtype):
    """N(0, 1) with some channels several times as large, as the streams of a transformer have them."""
    x = torch.randn(rows, dim, generator=g, device="cuda")
    x *= 1 + 5 * (torch.rand(dim, generator=g, device="cuda") < 0.02).float()
    return x.to(dtype)


def _positions(case):
    """[batch * seq, axes] int64: a grid of frames, rows and columns in row-major order (one axis: the index), each sequence from its
    own start."""
    axes = len(case["axes"].split(","))
    seq = case["seq"]
    i = torch.arange(seq, device="cuda")
    side = max(1, math.isqrt(seq // (21 if axes == 3 and seq > 441 else 1)))
    cols = [i % side, i // side % side if axes == 3 else i // side, i // (side * side)]
    pos = i[:, None] if axes == 1 else torch.stack(cols[:axes][::-1], dim=-1)
    first = case["start"] + 17 * torch.arange(case["batch"], device="cuda")
    return (first[:, None, None] + pos[None]).reshape(case["batch"] * seq, axes).contiguous()


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 12345)
    kind, T = case["kind"], DTYPES[case["dtype"]]
    s = {"case": case}
    if kind in ("fp4_linear", "norm_linear"):
        m, n, k = case["m"], case["n"], case["k"]
        s["w"] = _randn(g, (n, k), 0.02, T)
        s["bias"] = _randn(g, (n,), 0.02, T)
        # calibrated static scale of the activations: a power of two that keeps their expected maximum within what a block can hold, 6 x 448
        s["x_scale"] = torch.full((1,), 2.0 ** -6, dtype=torch.float32, device="cuda") if case["fmt"] == "nvfp4" else None
        if kind == "fp4_linear":
            s["x"] = _activations(g, m, k, T)
            s["residual"] = _randn(g, (m, n), 1.0, T) if case["residual"] else None
    if kind in ("norm", "norm_linear"):
        batch, seq, dim = (case["batch"], case["seq"], case["dim"]) if kind == "norm" else (1, case["m"], case["k"])
        s["y"] = _activations(g, batch * seq, dim, T).reshape(batch, seq, dim)
        s["stream"] = _activations(g, batch * seq, dim, T).reshape(batch, seq, dim)
        s["post_weight"] = (1 + _randn(g, (dim,), 0.2, torch.float32)).to(T) if case.get("post", "rms") != "none" else None
        s["pre_weight"] = (1 + _randn(g, (dim,), 0.2, torch.float32)).to(T)
        # gate, scale and shift as a modulation linear leaves them: thirds of one row per batch entry
        mod = _randn(g, (batch, 3 * dim), 0.3, T) if case.get("mod", True) else None
        s["gate"], s["scale"], s["shift"] = (None, None, None) if mod is None else mod.chunk(3, dim=-1)
        s["f8_scale"] = torch.full((1,), 0.03, dtype=torch.float32, device="cuda")
    if kind == "rope":
        rows, hq, hk, d = case["batch"] * case["seq"], case["q_heads"], case["k_heads"], case["head_dim"]
        # q and k heads side by side with the v heads behind them, as the projection writes them
        qkv = torch.randn(rows, (hq + 2 * hk) * d, generator=g, device="cuda").to(T)
        s["q"] = qkv[:, :hq * d].view(case["batch"], case["seq"], hq, d)
        s["k"] = qkv[:, hq * d:(hq + hk) * d].view(case["batch"], case["seq"], hk, d)
        s["pos"] = _positions(case).reshape(case["batch"], case["seq"], -1)
        s["q_norm"] = (1 + _randn(g, (d,), 0.2, torch.float32)).to(T) if case["norm"] else None
        s["k_norm"] = (1 + _randn(g, (d,), 0.2, torch.float32)).to(T) if case["norm"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind in ("fp4_linear", "norm_linear"):
        # the weight is quantized once, when a model is loaded: the plain form keeps the values, the library its layer
        if own:
            from lyradiff_b200 import layers
            s["layer"] = layers.Fp4Linear(s["w"], s["bias"], s["x_scale"], gelu=case.get("gelu", False), fmt=case["fmt"])
        else:
            s["w_scale"], s["w_values"] = _plain_weight(s["w"], case["fmt"])
    if kind == "rope" and own:
        from lyradiff_b200 import rope
        s["plan"] = rope.AxisRope([int(a) for a in case["axes"].split(",")], theta=THETA, interleaved=case["style"] == "interleaved",
                                  device="cuda")
    return s


# ----------------------------------------------------------------------------- the plain forms
def _plain_e2m1(t):
    """Nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with the sign of t, ties to the even code, saturating."""
    a = t.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign((torch.round(a / step) * step).clamp_max(6.0), t)


def _plain_power(e):
    """2^e for whole e from -127 to 127, by its bits: exact, which pow need not be."""
    return torch.where(e < -126, 2.0 ** -127, ((e.clamp_min(-126) + 127) << 23).int().view(torch.float32))


def _plain_e4m3(a):
    """Nearest e4m3 number of non-negative a, ties to even, saturating at 448."""
    e = torch.frexp(a)[1] - 1
    step = _plain_power(e.clamp_min(-6) - 3)
    return (torch.round(a / step) * step).clamp_max(448.0)


def _plain_fp4(x, fmt, scale):
    """x [rows, k] fp32 -> the values that its FP4 form stands for, without the tensor scale."""
    b = x.reshape(x.shape[0], -1, GROUP[fmt])
    a = b.abs().amax(dim=-1, keepdim=True)
    if fmt == "mxfp4":
        e = (torch.frexp(a)[1] - 3).clamp_min(-127)     # floor(log2 a) - 2
        s = _plain_power(e)
        return (_plain_e2m1(b / s) * s).reshape(x.shape)
    s = _plain_e4m3(a / (scale * 6.0))
    t = s * scale
    q = _plain_e2m1(torch.where(t > 0, b / torch.where(t > 0, t, 1.0), 0.0))
    return (q * s).reshape(x.shape)


def _plain_weight(w, fmt):
    """The weight's own tensor scale, the least power of two with which its maximum is within 6 x 448, and the values of its FP4 form,
    scale included."""
    w = w.float()
    scale = None
    if fmt == "nvfp4":
        m, e = torch.frexp(w.abs().amax().reshape(1) / torch.full((1,), 2688.0, device=w.device))
        scale = _plain_power(torch.where(m == 0.5, e - 1, e))
    values = _plain_fp4(w, fmt, scale)
    return scale, values if scale is None else values * scale


def _plain_gelu(v):
    return 0.5 * v * (1 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))


def _plain_linear(s, x):
    case = s["case"]
    v = _plain_fp4(x, case["fmt"], s["x_scale"])
    y = v @ s["w_values"].t()
    if s["x_scale"] is not None:
        y = y * s["x_scale"]
    if s.get("residual") is not None:
        y = y + s["residual"].float()
    y = y + s["bias"].float()
    return (_plain_gelu(y) if case.get("gelu") else y).to(s["w"].dtype)


def _plain_normed(v, kind):
    if kind == "layer":
        v = v - v.mean(dim=-1, keepdim=True)
    return v * torch.rsqrt((v * v).mean(dim=-1, keepdim=True) + EPS) if kind != "none" else v


def _plain_norm(s, post, pre):
    u = _plain_normed(s["y"].float(), post)
    if s["post_weight"] is not None:
        u = u * s["post_weight"].float()
    if s["gate"] is not None:
        u = u * s["gate"].float()[:, None]
    v = s["stream"].float() + u
    h = _plain_normed(v, pre) * s["pre_weight"].float()
    if s["scale"] is not None:
        h = h * (1 + s["scale"].float()[:, None]) + s["shift"].float()[:, None]
    return v.to(s["y"].dtype), h.to(s["y"].dtype)


def _plain_rotate(x, cos, sin, weight, case):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * weight.float()
    rd = 2 * cos.shape[-1]
    r, rest = x[..., :rd], x[..., rd:]
    if case["style"] == "interleaved":
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = r[..., :rd // 2], r[..., rd // 2:]
        r = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([r, rest], dim=-1)


def _plain_rope(s):
    case = s["case"]
    parts = []
    for a, dim in enumerate(int(v) for v in case["axes"].split(",")):
        # angles of far positions need 64 bits
        freq = THETA ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
        parts.append(s["pos"][..., a:a + 1].double() * freq)
    ang = torch.cat(parts, dim=-1)[:, :, None]
    cos, sin = torch.cos(ang).float(), torch.sin(ang).float()
    return (_plain_rotate(s["q"], cos, sin, s["q_norm"], case).to(s["q"].dtype),
            _plain_rotate(s["k"], cos, sin, s["k_norm"], case).to(s["k"].dtype))


# ----------------------------------------------------------------------------- one pass
def run(state):
    s, case = state, state["case"]
    kind = case["kind"]
    if own:
        return _own(s, case, kind)
    if kind == "fp4_linear":
        return _plain_linear(s, s["x"].float())
    if kind == "norm":
        x, h = _plain_norm(s, case["post"], case["pre"])
        if case["out"] == "e4m3":
            h = (h.float() * (1.0 / s["f8_scale"])).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        return x, h
    if kind == "norm_linear":
        x, h = _plain_norm(s, "rms", "layer")
        return x, _plain_linear(s, h[0].float())
    return _plain_rope(s)


def _own(s, case, kind):
    from lyradiff_b200 import ops
    if kind == "fp4_linear":
        return s["layer"].forward(s["x"], residual=s["residual"])
    if kind == "norm":
        mods = {"gate": s["gate"], "scale": s["scale"], "shift": s["shift"], "post_weight": s["post_weight"],
                "pre_weight": s["pre_weight"], "post": case["post"], "pre": case["pre"], "eps": EPS}
        if case["out"] == "e4m3":
            q = torch.empty(s["y"].shape, dtype=torch.uint8, device="cuda")
            x, _ = ops.gated_residual_norm(s["y"], s["stream"], qf8=q, f8_scale=s["f8_scale"], **mods)
            return x, q.view(torch.float8_e4m3fn)
        return ops.gated_residual_norm(s["y"], s["stream"], **mods)
    if kind == "norm_linear":
        q = s["layer"].empty_input(case["m"])
        x, _ = ops.gated_residual_norm(s["y"], s["stream"], gate=s["gate"], scale=s["scale"], shift=s["shift"],
                                       post_weight=s["post_weight"], pre_weight=s["pre_weight"], post="rms", pre="layer", eps=EPS, q4=q)
        return x, s["layer"].forward_quantized(q, s["w"].dtype)
    return ops.rope_axes(s["plan"], s["pos"], s["q"], s["k"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind in ("fp4_linear", "norm_linear"):
        m, n, k = case["m"], case["n"], case["k"]
        weight = n * k // 2 + n * k // GROUP[case["fmt"]]
        if kind == "fp4_linear":
            move = 2 * m * k + weight + 2 * n + 2 * m * n * (2 if case["residual"] else 1)
        else:
            move = 3 * 2 * m * k + 2 * 5 * k + weight + 2 * n + 2 * m * n
        return {"bytes": move, "flops": 2 * m * n * k}
    if kind == "norm":
        rows, dim = case["batch"] * case["seq"], case["dim"]
        move = rows * dim * (6 + (1 if case["out"] == "e4m3" else 2)) + 2 * dim * ((case["post"] != "none") + 1)
        return {"bytes": move + (6 * case["batch"] * dim if case["mod"] else 0), "flops": 14 * rows * dim}
    rows = case["batch"] * case["seq"]
    elems = rows * (case["q_heads"] + case["k_heads"]) * case["head_dim"]
    return {"bytes": 4 * elems + 8 * rows * len(case["axes"].split(",")), "flops": (7 if case["norm"] else 3) * elems}


# ----------------------------------------------------------------------------- the definitions in 64 bits
def _exact_e2m1(t):
    a = t.abs()
    index = torch.zeros(a.shape, dtype=torch.int64, device=a.device)
    for border, up in ((0.25, 0), (0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1), (5.0, 0)):   # a tie goes to the even code
        index += (a >= border) if up else (a > border)
    return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=a.device)[index] * torch.sign(t)


def _exact_power(e):
    return (((e.long() + 1023) << 52)).view(torch.float64)


def _exact_e4m3(a):
    code = torch.arange(127, dtype=torch.int64, device=a.device)
    e, f = code >> 3, (code & 7).double()
    value = torch.where(e == 0, f / 512, (1 + f / 8) * _exact_power(e - 7))
    border = (value[1:] + value[:-1]) / 2
    low = torch.searchsorted(border, a.contiguous())              # borders below a
    tie = (low < 126) & (border[low.clamp_max(125)] == a) & (low % 2 == 1)
    return value[low + tie]


def _exact_fp4(x, fmt, scale):
    b = x.unflatten(-1, (-1, GROUP[fmt]))
    a = b.abs().amax(dim=-1, keepdim=True)
    if fmt == "mxfp4":
        t = _exact_power(torch.frexp(a.clamp_min(2.0 ** -125)).exponent - 3)      # a is at least 2^(exponent - 1)
    else:
        t = _exact_e4m3(a / (6 * scale)) * scale
    return torch.where(t > 0, _exact_e2m1(b / t.clamp_min(1e-300)) * t, 0.0).flatten(-2)


def _exact_linear(s, x):
    case = s["case"]
    w = s["w"].double()
    w_scale = None
    if case["fmt"] == "nvfp4":
        power = torch.frexp(w.abs().max() / 2688)
        w_scale = _exact_power(power.exponent - (power.mantissa == 0.5).int())
    x_scale = s["x_scale"].double() if case["fmt"] == "nvfp4" else None
    y = torch.matmul(_exact_fp4(x, case["fmt"], x_scale), _exact_fp4(w, case["fmt"], w_scale).mT) + s["bias"].double()
    if s.get("residual") is not None:
        y += s["residual"].double()
    if case.get("gelu"):
        y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y


def _exact_norm(s, post, pre):
    def normed(v, kind):
        if kind == "rms":
            return v / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)
        return (v - v.mean(-1, keepdim=True)) / torch.sqrt(v.var(-1, unbiased=False, keepdim=True) + EPS) if kind == "layer" else v

    f = {key: None if s[key] is None else s[key].double() for key in ("y", "stream", "post_weight", "pre_weight", "gate", "scale", "shift")}
    u = normed(f["y"], post) * (1 if f["post_weight"] is None else f["post_weight"])
    v = f["stream"] + u * (1 if f["gate"] is None else f["gate"].unsqueeze(1))
    h = normed(v, pre) * f["pre_weight"]
    return v, h if f["scale"] is None else h * (1 + f["scale"].unsqueeze(1)) + f["shift"].unsqueeze(1)


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "fp4_linear":
        return _exact_linear(s, s["x"].double())
    if kind == "norm":
        v, h = _exact_norm(s, case["post"], case["pre"])
        return v, (h / s["f8_scale"].double()).clamp(-448, 448) if case["out"] == "e4m3" else h
    if kind == "norm_linear":
        v, h = _exact_norm(s, "rms", "layer")
        # the quantizer takes the 16-bit result of the norm: that rounding is part of the definition
        return v, _exact_linear(s, h[0].to(DTYPES[case["dtype"]]).double())
    dims = [int(a) for a in case["axes"].split(",")]
    turn = torch.cat([s["pos"][..., a, None].double() / torch.pow(torch.tensor(THETA, dtype=torch.float64, device="cuda"),
                                                                 torch.arange(dims[a] // 2, device="cuda").double() * 2 / dims[a])
                      for a in range(len(dims))], dim=-1).unsqueeze(2)
    z = torch.polar(torch.ones_like(turn), turn)
    out = []
    for x, w in ((s["q"].double(), s["q_norm"]), (s["k"].double(), s["k_norm"])):
        if w is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()
        p = z.shape[-1]
        first, second = (x[..., 0:2 * p:2], x[..., 1:2 * p:2]) if case["style"] == "interleaved" else (x[..., :p], x[..., p:2 * p])
        y = torch.complex(first, second) * z
        x = x.clone()
        if case["style"] == "interleaved":
            x[..., 0:2 * p:2], x[..., 1:2 * p:2] = y.real, y.imag
        else:
            x[..., :p], x[..., p:2 * p] = y.real, y.imag
        out.append(x)
    return tuple(out)
