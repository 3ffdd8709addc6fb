"""Offsets beyond 32 bits: weights, activations and results of more than 2^32 values.  A few rows and columns against 64 bits."""
import pytest
import torch

from caif_amd import torch_ops as T
import mxfp4_reference as R

pytestmark = pytest.mark.gpu


def fill(shape, dtype=torch.bfloat16, seed=0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(seed))


def codes_of(n, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (n, 16 * R.blocks_of(k)), dtype=torch.uint8, device="cuda", generator=g)
    if k % 32:
        codes.view(n, -1)[:, 16 * (k // 32) + (k % 32 + 1) // 2:] = 0
        if k % 2:
            codes[:, 16 * (k // 32) + k % 32 // 2] &= 15
    return codes, torch.randint(118, 125, (n, R.blocks_of(k)), dtype=torch.uint8, device="cuda", generator=g)


def check(got, want, size, length, dtype, pieces=1):
    off = (got.double() - want).abs()
    assert bool((off <= R.bound(want, size, length, dtype, pieces)).all())


@pytest.mark.parametrize("M", [1, 40, 100])
def test_weight(M):
    """270001 x 16390: 4.4e9 values, of which some rows at both ends are compared, and some columns of the gradient."""
    N, K = 270001, 16390
    codes, scales = codes_of(N, K, 1)
    w = T.FrozenWeight(codes, T.W_MXFP4, scales, N, K, 1, 32)
    x = fill((M, K), seed=2)
    rows = torch.cat([torch.arange(0, 40), torch.arange(N // 2, N // 2 + 40), torch.arange(N - 70, N)]).cuda()
    part = R.decode(codes[rows], scales[rows], K)
    y = T.qlinear_forward(x, w, T.BF16)
    check(y[:, rows], x.double() @ part.T, x.double().abs() @ part.abs().T, K, torch.float32)
    # both operands in 4 bits
    xc, xs = T.mxfp4_quantize(x)
    p = R.decode(xc, xs, K)
    check(T.mxfp4_matmul(xc, xs, codes, scales)[:, rows], p @ part.T, p.abs() @ part.abs().T, K, torch.float32)
    dy = fill((M, N), seed=3)
    dx = T.qlinear_backward_input(dy, w, T.BF16)
    first, last = slice(0, 2), slice(R.blocks_of(K) - 2, R.blocks_of(K))
    for blocks in (first, last):
        lo, hi = 32 * blocks.start, min(K, 32 * blocks.stop)
        m = R.decode(codes[:, 16 * blocks.start:16 * blocks.stop].contiguous(), scales[:, blocks].contiguous(), hi - lo)
        check(dx[:, lo:hi], dy.double() @ m, dy.double().abs() @ m.abs(), N, torch.float32)


def test_activations_and_results():
    """1100001 rows of 4100 values: 4.5e9 of them go in, and come out of the gradient and the gated backward."""
    M, N, K = 1100001, 40, 4100
    codes, scales = codes_of(N, K, 4)
    w, exact = T.FrozenWeight(codes, T.W_MXFP4, scales, N, K, 1, 32), R.decode(codes, scales, K)
    x = fill((M, K), seed=5)
    rows = torch.cat([torch.arange(0, 70), torch.arange(M // 2, M // 2 + 70), torch.arange(M - 140, M)]).cuda()
    y = T.qlinear_forward(x, w, T.BF16)
    p = x[rows].double()
    check(y[rows], p @ exact.T, p.abs() @ exact.abs().T, K, torch.float32)
    hidden, gate, up = T.gated_forward(x, w, w, keep=True)
    want = p @ exact.T
    check(gate[rows], want, p.abs() @ exact.abs().T, K, torch.bfloat16)
    assert torch.equal(gate, up)
    back, at = T.mxfp4_quantize(x)
    values = T.mxfp4_dequantize(back, at, K, torch.bfloat16)
    assert torch.equal(values[rows].double(), R.decode(back[rows], at[rows], K))
    few = x[rows].cpu()
    codes_want, scales_want = R.quantize(few)
    assert torch.equal(back[rows].cpu(), codes_want) and torch.equal(at[rows].cpu(), scales_want)
    del values, back, x
    dx, da, db = T.gated_backward(hidden, gate, up, w, w)
    p, q = da[rows].double(), db[rows].double()
    check(dx[rows], p @ exact + q @ exact, p.abs() @ exact.abs() + q.abs() @ exact.abs(), 2 * N, torch.bfloat16)
    dx = T.qlinear_backward_input(hidden, w, T.BF16, T.BF16)
    p = hidden[rows].double()
    check(dx[rows], p @ exact, p.abs() @ exact.abs(), N, torch.bfloat16)


def test_gating_of_more_than_4_billion_values():
    M, N, K = 300001, 14400, 32
    codes, scales = codes_of(N, K, 6)
    w, exact = T.FrozenWeight(codes, T.W_MXFP4, scales, N, K, 1, 32), R.decode(codes, scales, K)
    x = fill((M, K), seed=7)
    hidden, gate, up = T.gated_forward(x, w, w, keep=True)
    rows = torch.cat([torch.arange(0, 70), torch.arange(M - 140, M)]).cuda()
    p = x[rows].double()
    check(gate[rows], p @ exact.T, p.abs() @ exact.abs().T, K, torch.bfloat16)
    _, da, db = T.gated_backward(hidden, gate, up, w, w, need_dx=False)
    d, g, u = (t[rows].double() for t in (hidden, gate, up))
    want_a, want_b = R.gating_backward(d, g, u)
    top = torch.finfo(torch.bfloat16)
    spread = (d * u).abs() * torch.sigmoid(g) * (1 + g.abs())
    assert bool(((da[rows].double() - want_a).abs() <= 12 * 2.0 ** -24 * spread + top.eps / 2 * want_a.abs() + top.smallest_normal * top.eps).all())
    assert bool(((db[rows].double() - want_b).abs() <= (8 * 2.0 ** -24 + top.eps / 2) * want_b.abs() + top.smallest_normal * top.eps).all())
