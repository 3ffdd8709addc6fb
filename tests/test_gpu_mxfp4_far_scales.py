"""Scales beyond those that quantising gives, in the products with a frozen weight."""
import pytest
import torch

from caif_amd import torch_ops as T
import mxfp4_reference as R

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("M", [1, 4, 20, 100, 700])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("backward", [False, True])
def test_values_beyond_fp32(M, dtype, backward):
    """Scale bytes 253 and 254, which quantising never gives, make codes that are beyond fp32: a result with one of them is no finite number, in fp32
    an infinity or a NaN, and every other result is as it is without them."""
    g = gen(M)
    N, K = 70, 200
    codes, s = R.random_weight(g, N, K, low=100, high=110)
    clean = T.FrozenWeight(codes.cuda(), T.W_MXFP4, s.cuda(), N, K, 1, 32)
    codes, s = codes.clone(), s.clone()
    codes[7, 16:32], s[7, 1] = 0x77, 254           # row 7, columns 32 to 63: 6 times 2^127
    codes[40, 0:16], s[40, 0] = 0xEE, 253          # row 40, columns 0 to 31: -4 times 2^126
    far = T.FrozenWeight(codes.cuda(), T.W_MXFP4, s.cuda(), N, K, 1, 32)
    dt = DTYPES[dtype]
    x = (1 + torch.rand(M, N if backward else K, generator=g)).to(dt).cuda()
    call = T.qlinear_backward_input if backward else T.qlinear_forward
    y, want = call(x, far, T.CODE_OF[dt], T.F32), call(x, clean, T.CODE_OF[dt], T.F32)
    touched = torch.zeros(K if backward else N, dtype=torch.bool)
    touched[slice(0, 64) if backward else [7, 40]] = True
    assert not bool(y[:, touched].isfinite().any())
    assert torch.equal(y[:, ~touched], want[:, ~touched])
    if dtype != "f32":           # infinities of their signs
        up, down = (y[:, 32:64], y[:, :32]) if backward else (y[:, 7], y[:, 40])
        assert bool((up == float("inf")).all()) and bool((down == float("-inf")).all())
