"""Frozen weights in microscaled 4-bit floating point and the gated feed-forward block over them, as cases that can be timed and compared.

A case is a dict of plain values.  `kind` names the operator:

    pack        a tensor put into 4 bits (E2M1 codes, one power-of-two scale per 32 neighbouring values of a row) and brought back
    forward     activations times a frozen weight of that kind
    gradient    the same projection's input gradient
    product     activations put into 4 bits, times the weight: both operands of the matrix cores have 4 bits
    gated       silu(gate projection) * up projection of a feed-forward block
    gated_back  that block's backward pass: gradients of both projections, and of the input

`weight` is "mx" for 4 bits, "same" for a weight stored in the activations' own type.  Activations are N(0, 1), gradients N(0, 1e-3), weights
N(0, 0.02)."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 32
LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def listed():
    return [
        # an activation of odd width in the default type
        {"name": "pack-999", "kind": "pack", "dtype": "f32", "m": 999, "k": 1403},
        # a whole weight, as it is put away once: the up projection of an 8B feed-forward block
        {"name": "pack-14336", "kind": "pack", "dtype": "bf16", "m": 14336, "k": 4096},
        # the smallest call: one request decodes through that projection
        {"name": "forward-1", "kind": "forward", "dtype": "bf16", "m": 1, "n": 14336, "k": 4096},
        # a decode step of 24 requests through the down projection, fp16
        {"name": "forward-24", "kind": "forward", "dtype": "f16", "m": 24, "n": 4096, "k": 14336},
        # a training step's 4096 tokens through the up projection of a 7B feed-forward block
        {"name": "forward-4096", "kind": "forward", "dtype": "bf16", "m": 4096, "n": 11008, "k": 4096},
        # a small ragged batch in the default type, odd sizes
        {"name": "gradient-333", "kind": "gradient", "dtype": "f32", "m": 333, "n": 2048, "k": 1403},
        # the input gradient of that block's down projection
        {"name": "gradient-4096", "kind": "gradient", "dtype": "bf16", "m": 4096, "n": 4096, "k": 11008},
        # 32 requests, activations in 4 bits too
        {"name": "product-32", "kind": "product", "dtype": "bf16", "m": 32, "n": 14336, "k": 4096},
        # a long prompt, activations in 4 bits too
        {"name": "product-4096", "kind": "product", "dtype": "bf16", "m": 4096, "n": 14336, "k": 4096},
        # eight requests decode through a feed-forward block
        {"name": "gated-8", "kind": "gated", "dtype": "bf16", "m": 8, "n": 14336, "k": 4096, "weight": "mx", "keep": False},
        # a training step's forward of a block stored in bf16, gate and up kept
        {"name": "gated-2048", "kind": "gated", "dtype": "bf16", "m": 2048, "n": 11008, "k": 4096, "weight": "same", "keep": True},
        # the training step's backward, weights in 4 bits
        {"name": "gated-back-2048", "kind": "gated_back", "dtype": "bf16", "m": 2048, "n": 11008, "k": 4096, "weight": "mx"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Mostly multiples of 64, one in four any number."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.25 else max(lo, n // 64 * 64)


def draw(rng):
    kind = rng.choice(["pack", "forward", "forward", "gradient", "product", "gated", "gated", "gated_back"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    case = {"kind": kind, "dtype": dtype, "m": _log_int(rng, 1, 2048), "k": _width(rng, 256, 4096)}
    if kind == "pack":
        return {**case, "m": _log_int(rng, 1, 8192)}
    case["n"] = _width(rng, 256, 8192)
    if kind in ("gated", "gated_back"):
        case["weight"] = "same" if dtype != "f32" and rng.random() < 0.4 else "mx"
    return {**case, "keep": rng.random() < 0.5} if kind == "gated" else case


# ------------------------------------------------------------------------------------------------ what a program holds
def _normal(gen, shape, std, dtype):
    return torch.empty(shape, device="cuda").normal_(0, std, generator=gen).to(dtype)


def _tables():
    """The values of the sixteen codes, of the scales' bytes (the last one is a NaN), and the scales' inverses."""
    at = torch.tensor(LEVELS, dtype=torch.float32)
    codes = torch.cat([at, -at]).cuda()
    scales = torch.tensor([2.0 ** (i - 127) for i in range(255)] + [math.nan], dtype=torch.float32).cuda()
    return {"codes": codes, "scales": scales, "inverse": 1 / scales}


def _in_blocks(x):
    """x [m, k] as [m, blocks, BLOCK], zeros behind the last column."""
    return torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK)).reshape(x.shape[0], -1, BLOCK)


def _pack(x, tables):
    """codes uint8 [m, 16 blocks] (two of them a byte) and scales uint8 [m, blocks] of finite values."""
    v = _in_blocks(x.float())
    peak = v.abs().amax(-1)
    scales = (torch.frexp(peak).exponent - 3 + 127).clamp(0, 254)          # peak = mantissa in [1/2, 1) times 2^exponent
    scales = torch.where(peak == 0, torch.zeros_like(scales), scales).to(torch.uint8)
    v = v * tables["inverse"][scales.long()][..., None]
    a = v.abs()
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
    code = code + 8 * (v < 0)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8).reshape(x.shape[0], -1), scales


def _unpack(codes, scales, tables):
    """fp32 [m, 32 blocks]"""
    pair = torch.stack([codes & 15, codes >> 4], -1).reshape(*scales.shape, BLOCK)
    return (tables["codes"][pair.int()] * tables["scales"][scales.int()][..., None]).reshape(scales.shape[0], -1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype, m, k = case["kind"], DTYPES[case["dtype"]], case["m"], case["k"]
    s = {"kind": kind, "dtype": dtype, "tables": _tables(), "k": k}
    if kind == "pack":
        return {**s, "x": _normal(gen, (m, k), 1, dtype)}
    n = case["n"]

    def weight():
        w = _normal(gen, (n, k), 0.02, dtype)
        return w if case.get("weight") == "same" else _pack(w, s["tables"])

    if kind == "gated":
        return {**s, "x": _normal(gen, (m, k), 1, dtype), "gate": weight(), "up": weight(), "keep": case["keep"]}
    if kind == "gated_back":
        return {**s, "grad": _normal(gen, (m, n), 1e-3, dtype), "g": _normal(gen, (m, n), 1, dtype), "u": _normal(gen, (m, n), 1, dtype),
                "gate": weight(), "up": weight()}
    return {**s, "x": _normal(gen, (m, n), 1e-3, dtype) if kind == "gradient" else _normal(gen, (m, k), 1, dtype), "w": weight()}


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _own(s)
    return {"pack": _there_and_back, "forward": _forward, "gradient": _gradient, "product": _product, "gated": _gated, "gated_back": _gated_back}[s["kind"]](s)


def _frozen(w, k):
    from caif_amd import torch_ops as T
    if isinstance(w, tuple):
        return T.FrozenWeight(w[0], T.W_MXFP4, w[1], w[0].shape[0], k, 1, BLOCK)
    return T.FrozenWeight(w, T.W_F16 if w.dtype == torch.float16 else T.W_BF16, None, w.shape[0], k)


def _own(s):
    from caif_amd import torch_ops as T
    kind, k = s["kind"], s["k"]
    if kind == "pack":
        return T.mxfp4_dequantize(*T.mxfp4_quantize(s["x"]), k, s["dtype"])
    code = T.CODE_OF[s["dtype"]]
    if kind == "forward":
        return T.qlinear_forward(s["x"], _frozen(s["w"], k), code, code)
    if kind == "gradient":
        return T.qlinear_backward_input(s["x"], _frozen(s["w"], k), code, code)
    if kind == "product":
        return T.mxfp4_matmul(*T.mxfp4_quantize(s["x"]), *s["w"], code)
    gate, up = _frozen(s["gate"], k), _frozen(s["up"], k)
    if kind == "gated":
        return T.gated_forward(s["x"], gate, up, keep=s["keep"])
    return T.gated_backward(s["grad"], s["g"], s["u"], gate, up)


def _values(w, s):
    """A weight in fp32, [n, k]."""
    return _unpack(*w, s["tables"])[:, :s["k"]] if isinstance(w, tuple) else w.float()


def _there_and_back(s):
    return _unpack(*_pack(s["x"], s["tables"]), s["tables"])[:, :s["k"]].to(s["dtype"])


def _forward(s):
    return (s["x"].float() @ _values(s["w"], s).T).to(s["dtype"])


def _gradient(s):
    return (s["x"].float() @ _values(s["w"], s)).to(s["dtype"])


def _product(s):
    return (_unpack(*_pack(s["x"], s["tables"]), s["tables"]) @ _unpack(*s["w"], s["tables"]).T).to(s["dtype"])


def _gated(s):
    x = s["x"].float()
    g, u = x @ _values(s["gate"], s).T, x @ _values(s["up"], s).T
    hidden = (g / (1 + torch.exp(-g)) * u).to(s["dtype"])
    return (hidden, g.to(s["dtype"]), u.to(s["dtype"])) if s["keep"] else hidden


def _gated_back(s):
    g, u, d = s["g"].float(), s["u"].float(), s["grad"].float()
    at = 1 / (1 + torch.exp(-g))
    dg, du = d * u * (at * (1 + g * (1 - at))), d * (g * at)
    return (dg @ _values(s["gate"], s) + du @ _values(s["up"], s)).to(s["dtype"]), dg.to(s["dtype"]), du.to(s["dtype"])


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _decoded(w, k):
    """A weight in 64 bits, from the bits of its codes: sign, two of exponent, one of mantissa."""
    if not isinstance(w, tuple):
        return w.double()
    codes, scales = w
    out = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.float64, device="cuda")
    for half in (0, 1):
        c = ((codes >> (4 * half)) & 15).double()
        sign = torch.where(c >= 8, -1.0, 1.0)
        c = c - 8 * (c >= 8)
        e, m = torch.floor(c / 2), c % 2
        out[:, half::2] = sign * torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2(e - 1))
    out *= torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, dim=1)
    return out[:, :k]


def _kept(x):
    """What a tensor [m, k] of finite values is after 4 bits: the nearest level, the one with an even mantissa in the middle between two."""
    out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    for c in range(0, x.shape[1], BLOCK):
        v = x[:, c:c + BLOCK].double()
        peak = v.abs().max(dim=1, keepdim=True).values
        scale = torch.exp2(torch.clamp(torch.floor(torch.log2(peak.clamp(min=2.0 ** -140))) - 2, min=-127))
        a = v.abs() / scale
        nearest, off = torch.zeros_like(a), a.clone()
        for i in range(1, 8):
            d = (a - LEVELS[i]).abs()
            better = (d < off) | ((d == off) & (i % 2 == 0))
            nearest = torch.where(better, LEVELS[i], nearest)
            off = torch.where(better, d, off)
        out[:, c:c + BLOCK] = torch.sign(v) * nearest * scale
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind, k = s["kind"], s["k"]
    if kind == "pack":
        return _kept(s["x"])
    if kind == "forward":
        return s["x"].double() @ _decoded(s["w"], k).T
    if kind == "gradient":
        return s["x"].double() @ _decoded(s["w"], k)
    if kind == "product":
        return _kept(s["x"]) @ _decoded(s["w"], k).T
    if kind == "gated":
        g, u = s["x"].double() @ _decoded(s["gate"], k).T, s["x"].double() @ _decoded(s["up"], k).T
        hidden = g * torch.sigmoid(g) * u
        return (hidden, g, u) if s["keep"] else hidden
    g, u, d = s["g"].double(), s["u"].double(), s["grad"].double()
    sg = torch.sigmoid(g)
    dg, du = d * u * (sg + g * sg * (1 - sg)), d * g * sg
    return dg @ _decoded(s["gate"], k) + du @ _decoded(s["up"], k), dg, du


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind, m, k, e = case["kind"], case["m"], case["k"], 4 if case["dtype"] == "f32" else 2
    if kind == "pack":                    # in, codes and scales out and in again, out
        return {"bytes": 2 * m * k * e + 2 * m * 17 * -(-k // BLOCK), "flops": 4.0 * m * k}
    n = case["n"]
    weight = n * k * e if case.get("weight") == "same" else n * 17 * -(-k // BLOCK)
    if kind == "gated":
        return {"bytes": 2 * weight + m * k * e + m * n * e * (3 if case["keep"] else 1), "flops": 4.0 * m * n * k}
    if kind == "gated_back":              # gradient, gate, up in; three gradients out
        return {"bytes": 2 * weight + 5 * m * n * e + m * k * e, "flops": 4.0 * m * n * k}
    return {"bytes": weight + m * (k + n) * e, "flops": 2.0 * m * n * k}
