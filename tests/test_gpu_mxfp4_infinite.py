"""Infinities and NaN of activations, gradients and projections give what the formulas give, in the results that they belong to and nowhere else."""
import pytest
import torch

from caif_amd import torch_ops as T
import mxfp4_reference as R

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
INF, NAN = float("inf"), float("nan")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def weight(g, n, k):
    codes, s = R.random_weight(g, n, k, device="cuda")
    return T.FrozenWeight(codes, T.W_MXFP4, s, n, k, 1, 32), R.decode(codes, s, k)


def plant(g, t, count=6):
    """Infinities of either sign and NaN at some places of `count` rows, one of them twice in a row with either sign, the last column among them"""
    rows, cols = t.shape
    for i, m in enumerate(torch.randperm(rows, generator=g)[:count].tolist()):
        t[m, int(torch.randint(0, cols, (1,), generator=g)) if i else cols - 1] = (INF, -INF, NAN)[i % 3]
        if i == 4:
            t[m, 0], t[m, cols // 2] = INF, -INF
    return t


def same_kind(got, want):
    """Infinities and NaN where 64 bits have them, of the same sign; finite results elsewhere"""
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    at = want.isinf()
    assert torch.equal(got[at].double(), want[at])


def product(a, b):
    """a b^T in 64 bits with every product of an infinity and a zero a NaN, whatever the library does with those"""
    clean = torch.where(a.isfinite(), a, torch.zeros_like(a))
    out = clean @ b.T
    for m in torch.nonzero(~a.isfinite().all(1)).flatten().tolist():
        out[m] = (a[m][None, :] * b).sum(1)
    return out


SHAPES = [(7, 100, 1403), (40, 130, 328), (100, 300, 776), (700, 1100, 520), (1100, 333, 2003)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear(M, N, K, dtype):
    g = gen(M + N + K)
    w, exact = weight(g, N, K)
    dt = DTYPES[dtype]
    code = T.CODE_OF[dt]
    for call, length, m in ((T.qlinear_forward, K, exact), (T.qlinear_backward_input, N, exact.T)):
        x = plant(g, torch.randn(M, length, generator=g)).to(dt).cuda()
        same_kind(call(x, w, code, T.F32), product(x.double(), m))


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated(M, N, K, dtype):
    g = gen(M + N + K + 1)
    (wg, eg), (wu, eu) = weight(g, N, K), weight(g, N, K)
    dt = DTYPES[dtype]
    x = plant(g, torch.randn(M, K, generator=g)).to(dt).cuda()
    hidden, gate, up = T.gated_forward(x, wg, wu, keep=True)
    a, b = product(x.double(), eg), product(x.double(), eu)
    same_kind(gate, a)
    same_kind(up, b)
    same_kind(hidden, R.silu(a) * b)
    d, gate, up = (plant(g, torch.randn(M, N, generator=g)).to(dt).cuda() for _ in range(3))
    dx, da, db = T.gated_backward(d, gate, up, wg, wu)
    want_a, want_b = R.gating_backward(d.double(), gate.double(), up.double())
    same_kind(da, want_a)
    same_kind(db, want_b)
    same_kind(dx, product(torch.cat([da, db], 1).double(), torch.cat([eg, eu]).T))
