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


@pytest.mark.parametrize("n,k", [(33000, 64), (64, 33000)])
@pytest.mark.parametrize("packed", [False, True])
def test_gradients_of_more_than_32_bits(n, k, packed):
    """A gradient or an input of 2.2e9 elements and more than sixty slots of one adapter: dx of the first and the last rows, the factors' gradients
    at both ends of either axis, against sums in 64 bits over all rows."""
    m, r = 66000, 8
    gen = torch.Generator(device="cuda").manual_seed(n)
    x, dy = (torch.empty(m, c, device="cuda", dtype=BF16).normal_(0, s, generator=gen) for c, s in ((k, 1), (n, 1e-2)))
    ids = torch.randint(0, 20, (m,), device="cuda", generator=gen)
    ids = torch.where(ids < 18, 0, ids - 17).to(torch.int32)                    # most the first, some the second, some none (2)
    a, b = normal(gen, (2, r, k), 0.1, BF16), normal(gen, (2, n, r), 0.1, BF16)
    scaling, hidden = torch.tensor([1.5, -0.5], device="cuda"), normal(gen, (m, r), 1, torch.float32)
    base = torch.empty(m, k, device="cuda", dtype=BF16).normal_(0, 1e-2, generator=gen)
    kept = T.checkpoint_pack(x) if packed else x
    dx, grad_a, grad_b = T.adapters_backward(dy, kept, hidden, ids, a, b, scaling, base=base)
    g, gmag = torch.zeros(m, r, dtype=torch.float64, device="cuda"), torch.zeros(m, r, dtype=torch.float64, device="cuda")
    for lo in range(0, m, 2000):
        d = dy[lo:lo + 2000].double()
        for l in range(2):
            mine = (ids[lo:lo + 2000] == l)[:, None]
            g[lo:lo + 2000] += torch.where(mine, scaling[l].double() * (d @ b[l].double()), 0.0)
            gmag[lo:lo + 2000] += torch.where(mine, scaling[l].abs().double() * (d.abs() @ b[l].abs().double()), 0.0)
    ends = lambda c: torch.cat([torch.arange(min(c, 130)), torch.arange(max(c - 130, 0), c)]).cuda()         # noqa: E731
    for rows in (slice(0, 100), slice(m - 100, m)):
        of = ids[rows].long().clamp(max=1)
        want = base[rows].double() + (g[rows, None] @ a[of].double())[:, 0]
        mag = base[rows].double().abs() + (gmag[rows, None] @ a[of].double().abs())[:, 0]
        R.check(dx[rows], want, mag, BF16, R.sums(n, r) + R.pieces(BF16), "dx")
    cols = ends(k)
    value = (kept[0][:, cols].double() * kept[1][:, cols // 128].double() if packed else x[:, cols].double()).cpu()
    at, dcols = ends(n), dy[:, ends(n)].double().cpu()
    for l in range(2):
        rows = (ids == l).nonzero()[:, 0].cpu()
        gl, ml, vl = g.cpu()[rows], gmag.cpu()[rows], value[rows]
        R.check(grad_a[l][:, cols], gl.T @ vl, ml.T @ vl.abs(), BF16, R.sums(n, m) + R.pieces(BF16), "grad_a")
        s, dl, hl = float(scaling[l]), dcols[rows], hidden.double().cpu()[rows]
        R.check(grad_b[l][at], s * (dl.T @ hl), abs(s) * (dl.abs().T @ hl.abs()), BF16, R.sums(m) + R.pieces(BF16), "grad_b")
