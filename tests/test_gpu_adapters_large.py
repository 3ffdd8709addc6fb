"""The adapters' calls at sizes where an index of 32 bits would not do, results and gradients, and with more adapters than the backward takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from caif_amd import torch_ops as T                                             # noqa: E402
import adapter_reference as R                                                   # noqa: E402
from test_gpu_adapters import BF16, normal                                      # noqa: E402


@pytest.mark.parametrize("m,r", [(40, 1), (3000, 1), (40, 32)])
def test_a_million_adapters(m, r):
    """Factors of more than 2^32 elements (rank 32: fewer adapters), rows of the first and last adapters among others; row by row and in tiles."""
    k, n, adapters = 4096, 64, 2 ** 20 // r + 3
    gen = torch.Generator(device="cuda").manual_seed(m)
    x, base = normal(gen, (m, k), 1, BF16), normal(gen, (m, n), 1, BF16)
    a = torch.empty(adapters, r, k, device="cuda", dtype=BF16).normal_(0, 0.05, generator=gen)
    b = torch.empty(adapters, n, r, device="cuda", dtype=BF16).normal_(0, 0.3, generator=gen)
    scaling = torch.rand(adapters, device="cuda", generator=gen) + 0.5
    few = torch.cat([torch.tensor([0, adapters - 1, adapters - 2], device="cuda"), torch.randint(0, adapters, (20,), device="cuda", generator=gen)])
    of = torch.randint(0, len(few) + 1, (m,), device="cuda", generator=gen)
    ids = torch.cat([few, torch.tensor([adapters], device="cuda")])[of].to(torch.int32)
    y, hidden = T.adapters_forward(x, ids, a, b, scaling, base=base, keep_hidden=True)
    want, mag, h, hmag = R.forward(x, of, a[few], b[few], scaling[few], base)
    R.check(hidden, h, hmag, torch.float32, R.sums(k), "hidden")
    R.check(y, want, mag, BF16, R.sums(k, r) + R.pieces(BF16), "y")
