"""Microscaled 4-bit floating point and the gated feed-forward block in 64 bits, from their definitions."""
import torch

LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
BLOCK = 32


def blocks_of(cols):
    return -(-cols // BLOCK)


def quantize(x):
    """(codes uint8 [rows, 16 * blocks], scales uint8 [rows, blocks]) of x [rows, cols] on the CPU, value by value of the definition."""
    rows, cols = x.shape
    v = torch.zeros(rows, blocks_of(cols) * BLOCK, dtype=torch.float64)
    v[:, :cols] = x.double()
    v = v.reshape(rows, -1, BLOCK)
    finite = torch.isfinite(v).all(-1)
    v = torch.where(finite[..., None], v, torch.zeros_like(v))
    peak = v.abs().amax(-1)
    exponent = torch.floor(torch.log2(peak.clamp(min=2.0 ** -200)))
    # log2 in 64 bits is a rounded value: the exponent is the one with 2^e <= peak < 2^(e + 1)
    exponent = torch.where(torch.exp2(exponent) > peak, exponent - 1, exponent)
    exponent = torch.where(torch.exp2(exponent + 1) <= peak, exponent + 1, exponent)
    s = torch.where(peak > 0, (exponent - 2).clamp(-127, 127), torch.full_like(peak, -127.0))
    a = v.abs() * torch.exp2(-s)[..., None]
    code = torch.zeros_like(a)
    for i in range(7):
        middle = (LEVELS[i] + LEVELS[i + 1]) / 2
        up = (a > middle) if i % 2 == 0 else (a >= middle)          # a tie goes to the even mantissa: codes 0, 2, 4, 6
        code = torch.where(up, torch.full_like(code, float(i + 1)), code)
    code = code + 8 * torch.signbit(v)
    code = torch.where(finite[..., None], code, torch.zeros_like(code)).to(torch.uint8)
    scales = torch.where(finite, s + 127, torch.full_like(s, 255.0)).to(torch.uint8)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).reshape(rows, -1).contiguous(), scales


def decode(codes, scales, cols):
    """fp64 [rows, cols]"""
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(*scales.shape, BLOCK).long()
    levels = torch.tensor(LEVELS + [-v for v in LEVELS], dtype=torch.float64, device=codes.device)
    scale = torch.exp2(scales.double() - 127)
    scale = torch.where(scales == 255, torch.full_like(scale, float("nan")), scale)
    return (levels[c] * scale[..., None]).reshape(scales.shape[0], -1)[:, :cols]


def random_weight(gen, n, k, low=118, high=124, device="cpu"):
    """Random codes, zeros behind the last column, and scales around 2^-6."""
    codes = torch.randint(0, 256, (n, 16 * blocks_of(k)), dtype=torch.uint8, generator=gen)
    tail = torch.zeros(n, 32 * blocks_of(k), dtype=torch.uint8)
    tail[:, :k] = 15
    codes &= tail[:, 0::2] | (tail[:, 1::2] << 4)
    return codes.to(device), torch.randint(low, high + 1, (n, blocks_of(k)), dtype=torch.uint8, generator=gen).to(device)


def bound(exact, magnitude, length, dtype, pieces=1):
    """How far a product of `length` terms may be off, rounded once to `dtype`.  magnitude: the same sum of absolute values.  A term passes
    through at most 32 additions inside an instruction, one per instruction (length / 32 of them for each piece of an operand) and 16 where
    the waves' sums meet, each off by at most 2^-23 of what it adds up to; the result is rounded to half a step."""
    steps = pieces * (length / 32 + 1) + 48
    top = torch.finfo(dtype)
    return steps * 2.0 ** -23 * magnitude + top.eps / 2 * exact.abs() + top.smallest_normal * top.eps


def silu(g):
    return g * torch.sigmoid(g)


def gating_backward(d, g, u):
    """(grad_gate, grad_up)"""
    s = torch.sigmoid(g)
    return d * u * s * (1 + g * (1 - s)), d * g * s
