"""Measured cases of the 8-bit linear path: block-scaled quantization, the product of two
block-scaled matrices, the norms around a block with its gate and residual, and rotary positions.

`run` computes each case in elementary torch operations, or (with `own` true) through the
library's entry points.  Sizes are the trunk's (width 1024, MLP 4736, 5184 tokens an image,
16 heads of 64), the encoder's and decoder's (width 256, 33 prompt tokens, 201 queries), and
generic odd ones.
"""

import math

import torch

own = False

BLOCK = 128            # columns of a scale group; rows of a weight block
E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
LARGEST = 82944        # tokens of 16 images


# ------------------------------------------------------------------ cases ---

def listed():
    return [
        # the 33 prompt tokens of the encoder's width on their way into an 8-bit product
        {"name": "quantize prompt", "op": "quantize", "rows": 33, "cols": 256, "type": "bf16", "block_rows": 1, "pad": 0},
        # a float32 MLP weight, once per load, in 128 x 128 blocks
        {"name": "quantize weight", "op": "quantize", "rows": 4736, "cols": 1024, "type": "f32", "block_rows": 128,
         "pad": 0},
        # the MLP's hidden activations of 16 images
        {"name": "quantize 16 images", "op": "quantize", "rows": LARGEST, "cols": 4736, "type": "f16", "block_rows": 1,
         "pad": 0},
        # one token through an MLP weight: all latency and weight bytes
        {"name": "product 1 token", "op": "product", "m": 1, "n": 4736, "k": 1024, "act": "none", "out": "bf16",
         "bias": True, "pad": 0},
        # the decoder's 201 queries, sizes that divide nothing, float32 out
        {"name": "product 201 ragged", "op": "product", "m": 201, "n": 2053, "k": 1000, "act": "none", "out": "f32",
         "bias": True, "pad": 3},
        # fc1 of one image: GELU and the 8-bit operand of fc2 in the epilogue
        {"name": "product image fc1", "op": "product", "m": 5184, "n": 4736, "k": 1024, "act": "gelu", "out": "e4m3",
         "bias": True, "pad": 0},
        # fc2 of 16 images
        {"name": "product 16 images fc2", "op": "product", "m": LARGEST, "n": 1024, "k": 4736, "act": "none",
         "out": "f16", "bias": True, "pad": 0},
        # one token between two blocks
        {"name": "norm 1 token", "op": "norm", "rows": 1, "dim": 1024, "type": "bf16", "resid": "f32", "layer": False,
         "post": True, "gate": "none", "gate_rows": 1, "channel": True, "out": "bf16", "pad": 0},
        # the decoder's queries with an odd width and a gate row of their own
        {"name": "norm 201 ragged", "op": "norm", "rows": 201, "dim": 1001, "type": "f16", "resid": "f16", "layer": True,
         "post": True, "gate": "tanh", "gate_rows": 1, "channel": False, "out": "f16", "pad": 5},
        # 16 images: a gate row per image, layer scale, float32 residual, the next product's 8-bit operand
        {"name": "norm 16 images", "op": "norm", "rows": LARGEST, "dim": 1024, "type": "f16", "resid": "f32",
         "layer": True, "post": True, "gate": "plain", "gate_rows": 5184, "channel": True, "out": "e4m3", "pad": 0},
        # one new token for each of 8 sequences, far into a scaled context
        {"name": "rotary 8 tokens", "op": "rotary", "tokens": 8, "q_heads": 16, "k_heads": 4, "dim": 64, "rot": 64,
         "type": "bf16", "interleaved": False, "inverse": False, "scaling": "parts", "factor": 8.0, "far": 1000000,
         "pad": 0},
        # a long prompt: three quarters of each head turned, padded rows left alone
        {"name": "rotary 65536 tokens", "op": "rotary", "tokens": 65536, "q_heads": 16, "k_heads": 4, "dim": 128,
         "rot": 96, "type": "f16", "interleaved": True, "inverse": False, "scaling": "ntk", "factor": 4.0, "far": 65536,
         "pad": 0},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(("quantize", "product", "product", "norm", "rotary"))
    pad = rng.choice((0, 0, 1, 8, 16))
    if op == "quantize":
        cols = _spread(rng, 1, 8192)
        return {"op": op, "rows": _spread(rng, 1, min(LARGEST, LARGEST * 4736 // cols)), "cols": cols,
                "type": rng.choice(tuple(TYPES)), "block_rows": rng.choice((1, 128)), "pad": pad}
    if op == "product":
        n, k = _spread(rng, 1, 8192), _spread(rng, 1, 8192)
        m = _spread(rng, 1, max(1, min(LARGEST, LARGEST * 4736 // n, LARGEST * 4736 // k, LARGEST * 1024 * 4736 // (n * k))))
        out = rng.choice(("f32", "f16", "bf16", "e4m3"))
        return {"op": op, "m": m, "n": n, "k": k, "act": rng.choice(("none", "none", "gelu")), "out": out,
                "bias": rng.random() < 0.5, "pad": pad}
    if op == "norm":
        dim = _spread(rng, 1, 16384)
        kind, rows = rng.choice(tuple(TYPES)), _spread(rng, 1, min(LARGEST, LARGEST * 512 // dim))
        return {"op": op, "rows": rows, "dim": dim, "type": kind, "resid": rng.choice(("f32", kind)),
                "layer": rng.random() < 0.5, "post": rng.random() < 0.7,
                "gate": rng.choice(("none", "plain", "sigmoid", "tanh")), "gate_rows": rng.choice((1, 7, 5184)),
                "channel": rng.random() < 0.5, "out": rng.choice((kind, "e4m3")), "pad": pad}
    dim = rng.choice((32, 64, 80, 96, 128, 256, 2 * rng.randint(1, 128)))
    q_heads = _spread(rng, 1, 64)
    k_heads = rng.choice((0, 1, 4, q_heads))
    tokens = _spread(rng, 1, min(65536, 65536 * 20 * 64 // ((q_heads + k_heads) * dim)))
    return {"op": op, "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
            "rot": rng.choice((dim, dim, 2 * rng.randint(1, dim // 2))), "type": rng.choice(tuple(TYPES)),
            "interleaved": rng.random() < 0.5, "inverse": rng.random() < 0.25,
            "scaling": rng.choice(("none", "linear", "ntk", "parts")), "factor": rng.choice((2.0, 8.0, 40.0)),
            "far": _spread(rng, 1, 10000000), "pad": pad}


# ------------------------------------------------------------ input making ---

def _up(n, m):
    return -(-n // m) * m


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _rows(values, dtype, pad):
    """The values as rows of a wider buffer, `pad` elements behind each row."""
    wide = torch.zeros(values.shape[0], values.shape[1] + pad, device="cuda", dtype=dtype)
    wide[:, :values.shape[1]] = values
    return wide


def _coded(g, rows, cols, block_rows):
    """A matrix as an 8-bit product finds it: e4m3 values in rows of a multiple of 16 bytes, scales [groups][blocks]."""
    codes = (_normal(g, rows, cols) * 100).clamp_(-E4M3_MAX, E4M3_MAX)
    wide = torch.zeros(rows, _up(cols, 16), device="cuda", dtype=torch.float8_e4m3fn)
    wide[:, :cols] = codes.to(torch.float8_e4m3fn)
    scale = torch.exp(_normal(g, _up(cols, BLOCK) // BLOCK, _up(rows, block_rows) // block_rows) * 0.5)
    return wide, scale


def _eight(rows, cols):
    return (torch.zeros(rows, _up(cols, 16), device="cuda", dtype=torch.float8_e4m3fn),
            torch.zeros(_up(cols, BLOCK) // BLOCK, rows, device="cuda"))


def _frequencies(rot, scaling, factor, original=8192.0, base=10000.0, fast=32.0, slow=1.0):
    """Radians a position of each pair, and the magnitude, of rotary positions scaled for a context
    `factor` times the original one: not at all, linearly, by the base, or by parts (full turns within the
    original context decide between the unscaled and the linear frequency)."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    if scaling == "ntk" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2 * i / rot)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "parts":
        kept = ((original * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        return f * kept + f / factor * (1 - kept), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "quantize":
        rows, cols = case["rows"], case["cols"]
        x = _normal(g, rows, cols)
        x *= torch.exp(_normal(g, rows, 1))                      # tokens of different size
        x[:, :: 61] *= 20                                        # and a few large channels
        x[rows // 2, : cols // 2] = 0
        s["x"] = _rows(x, TYPES[case["type"]], case["pad"])
        s["q"] = torch.zeros(rows, _up(cols, 16), device="cuda", dtype=torch.float8_e4m3fn)
        s["scale"] = torch.zeros(_up(cols, BLOCK) // BLOCK, _up(rows, case["block_rows"]) // case["block_rows"],
                                 device="cuda")
    elif case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        s["x"], s["x_scale"] = _coded(g, m, k, 1)
        s["w"], s["w_scale"] = _coded(g, n, k, BLOCK)
        s["w_scale"] *= 1e-4 / math.sqrt(k)                      # outputs near 1
        s["bias_row"] = _normal(g, n) * 0.1 if case["bias"] else None
        if case["out"] == "e4m3":
            s["y"], s["y_scale"] = _eight(m, n)
        else:
            s["y"] = torch.zeros(m, n + case["pad"], device="cuda", dtype=TYPES[case["out"]])
    elif case["op"] == "norm":
        rows, dim, kind, pad = case["rows"], case["dim"], TYPES[case["type"]], case["pad"]
        x = _normal(g, rows, dim) * 2
        x[:, :: 97] *= 10
        s["x"] = _rows(x, TYPES[case["resid"]], pad)
        s["y"] = _rows(_normal(g, rows, dim) + 0.1, kind, pad)
        s["y"][rows // 2] = 0                                    # a block that answers nothing
        gates = _up(rows, case["gate_rows"]) // case["gate_rows"]
        s["gate_row"] = None if case["gate"] == "none" else _rows(_normal(g, gates, dim), kind, pad)
        s["channel_row"] = torch.exp(_normal(g, dim) * 0.3) * 0.1 if case["channel"] else None
        for at in ("post", "pre"):
            s[at + "_weight"] = 1 + 0.1 * _normal(g, dim)
            s[at + "_bias"] = 0.1 * _normal(g, dim) if case["layer"] else None
        s["x_out"] = torch.zeros_like(s["x"])
        if case["out"] == "e4m3":
            s["u"], s["u_scale"] = _eight(rows, dim)
        else:
            s["u"] = torch.zeros(rows, dim + pad, device="cuda", dtype=kind)
    else:
        tokens, dim, pad = case["tokens"], case["dim"], case["pad"]
        heads = case["q_heads"] + case["k_heads"]
        # q and k lie side by side in a token's row, as a projection leaves them
        s["qk"] = _rows(_normal(g, tokens, heads * dim), TYPES[case["type"]], pad)
        s["q_out"] = torch.zeros(tokens, case["q_heads"], dim, device="cuda", dtype=TYPES[case["type"]])
        s["k_out"] = torch.zeros(tokens, case["k_heads"], dim, device="cuda", dtype=TYPES[case["type"]])
        start = torch.randint(0, case["far"], (1,), generator=g, device="cuda")
        s["positions"] = torch.arange(tokens, device="cuda") % 8192 + start
        s["positions"][tokens - tokens // 16:] = -1              # rows behind the last sequence
        f, s["magnitude"] = _frequencies(case["rot"], case["scaling"], case["factor"])
        s["frequencies"] = f.cuda()
    return s


# ------------------------------------------------------------- plain forms ---

def _quantize(v, block_rows):
    """(e4m3 values, scales [groups][row blocks]) of float32 rows."""
    rows, cols = v.shape
    up = torch.nn.functional.pad(v, (0, _up(cols, BLOCK) - cols, 0, _up(rows, block_rows) - rows))
    b = up.view(up.shape[0] // block_rows, block_rows, up.shape[1] // BLOCK, BLOCK)
    a = b.abs().amax((1, 3)).clamp(min=AMAX_FLOOR)
    q = (b * (E4M3_MAX / a)[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(up.shape)[:rows, :cols], (a / E4M3_MAX).t().contiguous()


def _spans(scale, rows, cols, block_rows):
    """Scales [groups][row blocks] as one factor for each value."""
    full = scale.t().repeat_interleave(block_rows, 0)[:rows]
    return full.repeat_interleave(BLOCK, 1)[:, :cols]


def _norm(v, weight, bias, layer, eps=1e-5):
    if layer:
        v = v - v.mean(1, keepdim=True)
    v = v * torch.rsqrt(v.square().mean(1, keepdim=True) + eps) * weight
    return v if bias is None else v + bias


def _plain_product(s):
    m, n, k = s["m"], s["n"], s["k"]
    x = s["x"][:, :k].float() * _spans(s["x_scale"], m, k, 1)
    w = s["w"][:, :k].float() * _spans(s["w_scale"], n, k, BLOCK)
    y = x @ w.t()
    if s["bias_row"] is not None:
        y += s["bias_row"]
    if s["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y / math.sqrt(2.0)))
    if s["out"] == "e4m3":
        q, scale = _quantize(y, 1)
        return {"y": q, "y_scale": scale}
    return {"y": y.to(s["y"].dtype)}


def _plain_norm(s):
    rows, dim = s["rows"], s["dim"]
    h = s["y"][:, :dim].float()
    if s["post"]:
        h = _norm(h, s["post_weight"], s["post_bias"], s["layer"])
    if s["gate_row"] is not None:
        gate = s["gate_row"][:, :dim].float()
        gate = torch.sigmoid(gate) if s["gate"] == "sigmoid" else torch.tanh(gate) if s["gate"] == "tanh" else gate
        h = h * gate[torch.arange(rows, device="cuda") // s["gate_rows"]]
    if s["channel_row"] is not None:
        h = h * s["channel_row"]
    x = s["x"][:, :dim].float() + h
    u = _norm(x, s["pre_weight"], s["pre_bias"], s["layer"])
    out = {"x": x.to(s["x"].dtype)}
    if s["out"] == "e4m3":
        out["u"], out["u_scale"] = _quantize(u, 1)
    else:
        out["u"] = u.to(s["u"].dtype)
    return out


def _turned(x, cos, sin, rot, interleaved):
    """Heads [tokens][heads][dim] with the pairs of their first `rot` columns turned; cos and sin [tokens][1][rot / 2]."""
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., : rot // 2], x[..., rot // 2: rot])
    turned = (a * cos - b * sin, a * sin + b * cos)
    turned = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_rotary(s):
    positions, dim = s["positions"], s["dim"]
    angle = positions.double()[:, None, None] * s["frequencies"] * (-1 if s["inverse"] else 1)
    cos, sin = (torch.cos(angle) * s["magnitude"]).float(), (torch.sin(angle) * s["magnitude"]).float()
    x = s["qk"][:, : (s["q_heads"] + s["k_heads"]) * dim].view(s["tokens"], -1, dim).float()
    y = _turned(x, cos, sin, s["rot"], s["interleaved"]).to(s["qk"].dtype)
    there = (positions >= 0)[:, None, None]
    return {"q": torch.where(there, y[:, : s["q_heads"]], s["q_out"]),
            "k": torch.where(there, y[:, s["q_heads"]:], s["k_out"])}


def _plain(s):
    if s["op"] == "quantize":
        q, scale = _quantize(s["x"][:, : s["cols"]].float(), s["block_rows"])
        return {"q": q, "scale": scale}
    return {"product": _plain_product, "norm": _plain_norm, "rotary": _plain_rotary}[s["op"]](s)


# ------------------------------------------------------- the library's calls ---

def _matrix(s3t, t, scale=None):
    return s3t.Matrix(t.data_ptr(), t.stride(0), scale.data_ptr() if scale is not None else None,
                      scale.stride(0) if scale is not None else 0)


def _own(s):
    import sam3cpp_b200 as s3t
    kinds = {"f32": s3t.TYPE_F32, "f16": s3t.TYPE_F16, "bf16": s3t.TYPE_BF16, "e4m3": s3t.TYPE_E4M3}
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    stream = torch.cuda.current_stream().cuda_stream
    if s["op"] == "quantize":
        s3t.quantize_fp8(0, kinds[s["type"]], s["x"].data_ptr(), s["rows"], s["cols"], s["x"].stride(0), s["block_rows"],
                         _matrix(s3t, s["q"], s["scale"]), stream)
        return {"q": s["q"][:, : s["cols"]], "scale": s["scale"]}
    if s["op"] == "product":
        eight = s["out"] == "e4m3"
        s3t.gemm_fp8(0, _matrix(s3t, s["x"], s["x_scale"]), _matrix(s3t, s["w"], s["w_scale"]), ptr(s["bias_row"]),
                     s["m"], s["n"], s["k"], int(s["act"] == "gelu"), kinds[s["out"]],
                     _matrix(s3t, s["y"], s["y_scale"] if eight else None), stream)
        y = s["y"][:, : s["n"]]
        return {"y": y, "y_scale": s["y_scale"]} if eight else {"y": y}
    if s["op"] == "norm":
        eight, gate = s["out"] == "e4m3", s["gate_row"]
        flags = ((s3t.NORM_LAYER if s["layer"] else 0) | (s3t.NORM_POST if s["post"] else 0)
                 | {"sigmoid": s3t.NORM_GATE_SIGMOID, "tanh": s3t.NORM_GATE_TANH}.get(s["gate"], 0))
        s3t.norm_residual(0, s3t.NormArgs(
            rows=s["rows"], dim=s["dim"], type=kinds[s["type"]], resid_type=kinds[s["resid"]], u_type=kinds[s["out"]],
            flags=flags, eps=1e-5, resid_scale=1.0, branch_scale=1.0, y=s["y"].data_ptr(), y_stride=s["y"].stride(0),
            post_weight=ptr(s["post_weight"]) if s["post"] else None, post_bias=ptr(s["post_bias"]) if s["post"] else None,
            gate=ptr(gate), gate_stride=0 if gate is None else gate.stride(0), gate_rows=s["gate_rows"],
            channel_scale=ptr(s["channel_row"]), x=s["x"].data_ptr(), x_stride=s["x"].stride(0),
            x_out=s["x_out"].data_ptr(), x_out_stride=s["x_out"].stride(0), pre_weight=ptr(s["pre_weight"]),
            pre_bias=ptr(s["pre_bias"]), u=_matrix(s3t, s["u"], s["u_scale"] if eight else None)), stream)
        out = {"x": s["x_out"][:, : s["dim"]], "u": s["u"][:, : s["dim"]]}
        return out | {"u_scale": s["u_scale"]} if eight else out
    qk, dim, size = s["qk"], s["dim"], s["qk"].element_size()

    def view(first, heads, out):
        return s3t.RotaryView(qk.data_ptr() + first * dim * size, out.data_ptr(), heads, qk.stride(0), dim, heads * dim, dim)

    s3t.rotary(0, s["frequencies"].data_ptr(), s["rot"], s["magnitude"], s["positions"].data_ptr(), s["tokens"],
               kinds[s["type"]], dim, view(0, s["q_heads"], s["q_out"]),
               view(s["q_heads"], s["k_heads"], s["k_out"]) if s["k_heads"] else None,
               (s3t.ROTARY_INTERLEAVED if s["interleaved"] else 0) | (s3t.ROTARY_INVERSE if s["inverse"] else 0), stream)
    return {"q": s["q_out"], "k": s["k_out"]}


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ------------------------------------------------------------- definitions ---

def _blocked(v, block_rows):
    """Rows as [row blocks][rows][groups][columns], zeros behind the last row and column."""
    rows, cols = v.shape
    wide = v.new_zeros(_up(rows, block_rows), _up(cols, BLOCK))
    wide[:rows, :cols] = v
    return wide.reshape(-1, block_rows, wide.shape[1] // BLOCK, BLOCK)


def _exact_codes(v, block_rows):
    """What the 8-bit values and the scales stand for before their rounding, in 64 bits."""
    b = _blocked(v, block_rows)
    scale = torch.maximum(b.amax((1, 3)), -b.amin((1, 3))).clamp(min=AMAX_FLOOR) / E4M3_MAX
    b /= scale[:, None, :, None]
    return b.reshape(b.shape[0] * block_rows, -1)[: v.shape[0], : v.shape[1]], scale.t()


def _exact_values(codes, scale, cols, block_rows):
    b = _blocked(codes[:, :cols].double(), block_rows)
    b *= scale.t().double()[:, None, :, None]
    return b.reshape(b.shape[0] * block_rows, -1)[: codes.shape[0], :cols]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        v, scale = _exact_codes(s["x"][:, : case["cols"]].double(), case["block_rows"])
        return {"q": v, "scale": scale}
    if case["op"] == "product":
        y = torch.einsum("mk,nk->mn", _exact_values(s["x"], s["x_scale"], case["k"], 1),
                         _exact_values(s["w"], s["w_scale"], case["k"], BLOCK))
        if case["bias"]:
            y += s["bias_row"].double()
        if case["act"] == "gelu":
            y *= 0.5 * torch.special.erfc(y * -math.sqrt(0.5))
        if case["out"] != "e4m3":
            return {"y": y}
        y, scale = _exact_codes(y, 1)
        return {"y": y, "y_scale": scale}
    if case["op"] == "norm":
        dim = case["dim"]

        def normed(v, at):
            mean = v.sum(1, keepdim=True) / dim if case["layer"] else 0.0
            var = ((v - mean) ** 2).sum(1, keepdim=True) / dim
            v = (v - mean) / torch.sqrt(var + 1e-5) * s[at + "_weight"].double()
            return v + s[at + "_bias"].double() if case["layer"] else v

        h = s["y"][:, :dim].double()
        if case["post"]:
            h = normed(h, "post")
        if case["gate"] != "none":
            gate = s["gate_row"][:, :dim].double()
            gate = {"plain": lambda t: t, "sigmoid": lambda t: 1 / (1 + torch.exp(-t)), "tanh": torch.tanh}[case["gate"]](gate)
            h *= gate.repeat_interleave(case["gate_rows"], 0)[: case["rows"]]
        if case["channel"]:
            h *= s["channel_row"].double()
        h += s["x"][:, :dim].double()
        u = normed(h, "pre")
        if case["out"] != "e4m3":
            return {"x": h, "u": u}
        u, scale = _exact_codes(u, 1)
        return {"x": h, "u": u, "u_scale": scale}
    dim, rot, n = case["dim"], case["rot"], case["q_heads"] + case["k_heads"]
    x = s["qk"][:, : n * dim].double().view(case["tokens"], n, dim)
    even = torch.arange(0, rot, 2, device="cuda") if case["interleaved"] else torch.arange(rot // 2, device="cuda")
    odd = even + (1 if case["interleaved"] else rot // 2)
    turn = torch.polar(torch.full((), s["magnitude"], device="cuda", dtype=torch.float64),
                       s["positions"].double()[:, None] * s["frequencies"])[:, None]
    z = torch.complex(x[..., even], x[..., odd]) * (turn.conj() if case["inverse"] else turn)
    x[..., even], x[..., odd] = z.real, z.imag
    x[s["positions"] < 0] = 0
    return {"q": x[:, : case["q_heads"]], "k": x[:, case["q_heads"]:]}


def work(case):
    """Bytes and operations that a pass cannot do without."""
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (BYTES[case["type"]] + 1) + 4 * n // (BLOCK * case["block_rows"]), "flops": 2 * n}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        scales = 4 * (_up(k, BLOCK) // BLOCK) * (m + _up(n, BLOCK) // BLOCK)
        return {"bytes": m * k + n * k + scales + m * n * BYTES[case["out"]] + (4 * n if case["bias"] else 0)
                + (4 * m * _up(n, BLOCK) // BLOCK if case["out"] == "e4m3" else 0), "flops": 2 * m * n * k}
    if case["op"] == "norm":
        n = case["rows"] * case["dim"]
        gates = 0 if case["gate"] == "none" else _up(case["rows"], case["gate_rows"]) // case["gate_rows"]
        return {"bytes": n * (BYTES[case["type"]] + 2 * BYTES[case["resid"]] + BYTES[case["out"]])
                + gates * case["dim"] * BYTES[case["type"]] + 20 * case["dim"], "flops": 16 * n}
    n = case["tokens"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
    return {"bytes": 2 * n * BYTES[case["type"]] + 8 * case["tokens"], "flops": 3 * n}
