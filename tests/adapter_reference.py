"""The adapter branch and its gradients in 64 bits, and how far results in a smaller type may be from them.

Every quantity comes with its magnitude, the same formula over absolute values.  A sum of n terms in fp32 is off by the rounding of its
partial sums, each at most 2^-24 of the magnitude and of random sign: their sum's standard deviation is below sqrt(n / 3) 2^-24, six of
them below 4 sqrt(n) 2^-24 times the magnitude.  Where a 16-bit tensor type meets an fp32 factor on the matrix cores, the factor may be
two pieces of 8 bits each: off by 2^-17 of itself, twice (hidden and gradient rows) 2^-16.  The result is rounded once, by at most half a
step of its type; below the normal range of fp16 by half of 2^-24."""
import math

import torch

GROUP = 128
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}


def sums(*lengths):
    return sum(4 * math.sqrt(n) for n in lengths) * 2.0 ** -24


def pieces(dtype):
    return 0.0 if dtype == torch.float32 else 2.0 ** -16


def check(got, want, magnitude, dtype, slack, what):
    """|got - want| within half a step of dtype (fp32 results: of fp32) and `slack` of the magnitude, elementwise; NaN where want is."""
    got, want = got.double().cpu(), want.cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bound = HALF_STEP[dtype] * want.abs() * (1 + 2.0 ** -8) + slack * magnitude.cpu() + SMALLEST[dtype]
    far = ~((got - want).abs() <= bound) & ~(want.isnan() & got.isnan()) & ~((got == want) & want.isinf())
    if far.any():
        at = tuple(int(v) for v in far.nonzero()[0])
        raise AssertionError(f"{what}: {int(far.sum())} of {far.numel()} outside, first at {at}: {got[at]} for {want[at]}, bound {bound[at]}")


def unpacked(codes, scales):
    """What a checkpoint stands for, in 64 bits."""
    return codes.double() * scales.double().repeat_interleave(GROUP, dim=-1)[..., :codes.shape[-1]]


def forward(x, ids, a, b, scaling, base):
    """(y, its magnitude, hidden, its magnitude); all in 64 bits on the CPU."""
    x, a, b, scaling = (t.double().cpu() for t in (x, a, b, scaling))
    m, n, r = x.shape[0], b.shape[1], a.shape[1]
    y = torch.zeros(m, n, dtype=torch.float64) if base is None else base.double().cpu().clone()
    mag, hidden, hmag = y.abs(), torch.zeros(m, r, dtype=torch.float64), torch.zeros(m, r, dtype=torch.float64)
    for l in range(a.shape[0]):
        rows = (ids.cpu() == l).nonzero()[:, 0]
        hidden[rows] = x[rows] @ a[l].T
        hmag[rows] = x[rows].abs() @ a[l].abs().T
        y[rows] += scaling[l] * (hidden[rows] @ b[l].T)
        mag[rows] += scaling[l].abs() * (hmag[rows] @ b[l].abs().T)
    return y, mag, hidden, hmag


def backward(dy, x, hidden, ids, a, b, scaling, base):
    """{name: (value, magnitude)} of dx, grad_a and grad_b; x in 64 bits."""
    dy, x, hidden, a, b, scaling = (t.double().cpu() for t in (dy, x, hidden, a, b, scaling))
    dx = torch.zeros_like(x) if base is None else base.double().cpu().clone()
    dmag, ga, gb = dx.abs(), torch.zeros_like(a), torch.zeros_like(b)
    gamag, gbmag = torch.zeros_like(a), torch.zeros_like(b)
    for l in range(a.shape[0]):
        rows = (ids.cpu() == l).nonzero()[:, 0]
        g, gmag = scaling[l] * (dy[rows] @ b[l]), scaling[l].abs() * (dy[rows].abs() @ b[l].abs())
        dx[rows] += g @ a[l]
        dmag[rows] += gmag @ a[l].abs()
        ga[l], gamag[l] = g.T @ x[rows], gmag.T @ x[rows].abs()
        gb[l] = scaling[l] * (dy[rows].T @ hidden[rows])
        gbmag[l] = scaling[l].abs() * (dy[rows].abs().T @ hidden[rows].abs())
    return {"dx": (dx, dmag), "grad_a": (ga, gamag), "grad_b": (gb, gbmag)}
