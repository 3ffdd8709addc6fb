"""Activations below the smallest normal number against large scales: nothing on the way takes them for zeros, and the pieces of fp32 ones keep
what bf16 has numbers for."""
import pytest
import torch

from caif_amd import torch_ops as T
import mxfp4_reference as R

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 40, 1403), (4, 130, 520), (9, 100, 776), (40, 130, 328), (100, 264, 520), (700, 1100, 512), (1100, 333, 1000)])
def test_products(M, N, K, dtype, backward):
    g = torch.Generator().manual_seed(M + N + K)
    codes, s = R.random_weight(g, N, K, low=220, high=226, device="cuda")
    w, exact = T.FrozenWeight(codes, T.W_MXFP4, s, N, K, 1, 32), R.decode(codes, s, K)
    dt = DTYPES[dtype]
    # 2^-149 to 2^-127, all of them below 2^-126, in bf16 from 2^-133 on
    low = -149 if dtype == "f32" else -133
    steps = torch.randint(1, 2 ** (-126 - low), (M, N if backward else K), generator=g).double()
    x = (steps * 2.0 ** low * (1 - 2 * torch.randint(0, 2, steps.shape, generator=g).double())).to(dt).cuda()
    assert float(x.abs().max()) < 2.0 ** -126 and float(x.abs().min()) > 0
    m = exact if backward else exact.T
    y = (T.qlinear_backward_input if backward else T.qlinear_forward)(x, w, T.CODE_OF[dt], T.F32)
    want, size = x.double() @ m, x.double().abs() @ m.abs()
    most = R.bound(want, size, x.shape[1], torch.float32, 3 if dtype == "f32" else 1)
    if dtype == "f32":
        # bf16's numbers below 2^-126 are 2^-133 apart, so three pieces of an activation, each cut off, leave less than that of it
        most = most + 2.0 ** -133 * m.abs().sum(0)
    off = (y.double() - want).abs()
    assert bool((off <= most).all()), f"{float((off / most).max())} times the bound"
