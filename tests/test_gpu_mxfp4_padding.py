"""Codes that fill up a weight's last block, in the products with a frozen weight."""
import pytest
import torch

from caif_amd import torch_ops as T
import mxfp4_reference as R

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def fill_behind(codes, k, value):
    """codes uint8 [n, 16 * blocks] with every code from column k on set to `value`"""
    pair = torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)
    pair[:, k:] = value
    return (pair[:, 0::2] | (pair[:, 1::2] << 4)).contiguous()


# rows that end in every dword of a block, less than 16 blocks and more, a block of the row's last unit of 512 values and one before it
@pytest.mark.parametrize("K", [1, 7, 8, 9, 17, 31, 40, 300, 511, 520, 545, 1000, 1403, 2047])
@pytest.mark.parametrize("M", [1, 4, 9, 30, 50, 100])
def test_codes_behind_the_last_column_count_for_nothing(M, K):
    """Also where their values are beyond fp16: zero activations against infinities would be NaN."""
    g = gen(M + K)
    N = 70
    codes, s = R.random_weight(g, N, K, low=127, high=127)
    # the last block's scale takes every code from 1 on beyond fp16, so the codes inside the row are kept below: zeros
    inside = codes.clone()
    if K % 32:
        inside[:, 16 * (K // 32):] = 0
        s[:, -1] = 127 + 18
    full = fill_behind(inside, K, 7)
    for dtype in ("f16", "bf16"):
        dt = DTYPES[dtype]
        x = torch.randn(M, K, generator=g).to(dt)
        exact = R.decode(inside, s, K)
        for kind in (x.cuda(), x.float().cuda()):           # read where they are, and laid out beforehand
            y = T.qlinear_forward(kind, T.FrozenWeight(full.cuda(), T.W_MXFP4, s.cuda(), N, K, 1, 32), T.CODE_OF[dt], T.F32)
            want = x.double() @ exact.T
            assert bool(((y.double().cpu() - want).abs() <= R.bound(want, x.double().abs() @ exact.abs().T, K, torch.float32)).all())
        w = T.FrozenWeight(full.cuda(), T.W_MXFP4, s.cuda(), N, K, 1, 32)
        _, gate, up = T.gated_forward(x.cuda(), w, w, keep=True)
        assert bool(gate.isfinite().all()) and torch.equal(gate, up)
