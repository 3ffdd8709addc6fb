"""Adapters' calls large enough for the waves of 256 columns (8192 waves of 64 or more along either axis; fp32 above rank 64 stays with 64): rows and
columns that end inside a tile, the last tile whole and not, every rank's kernel, every type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from caif_amd import torch_ops as T                                             # noqa: E402
import adapter_reference as R                                                   # noqa: E402
from test_gpu_adapters import BF16, F16, F32, problem                           # noqa: E402

SIZES = [(2064, 4160, 4160, 8, 3, "runs"), (2064, 4160, 4160, 24, 3, "mixed"), (2064, 4160, 4352, 64, 2, "runs"), (2064, 4352, 4160, 128, 2, "mixed"),
         (2050, 4163, 4165, 24, 3, "runs"), (2050, 4163, 4165, 100, 2, "mixed"), (4200, 2240, 2112, 16, 5, "mixed"), (2064, 4096, 4352, 17, 2, "none")]


@pytest.mark.parametrize("m,k,n,r,adapters,order", SIZES)
def test_sizes_are_wide(m, k, n, r, adapters, order):
    assert min(-(-m // 16) * -(-c // 64) for c in (k, n)) >= 8192


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,k,n,r,adapters,order", SIZES)
def test_forward(m, k, n, r, adapters, order, dtype):
    p, more = problem(m, k, n, r, adapters, dtype, order)
    y, hidden = T.adapters_forward(**p, base=more["base"], keep_hidden=True)
    want, mag, h, hmag = R.forward(**p, base=more["base"])
    R.check(hidden, h, hmag, F32, R.sums(k), "hidden")
    R.check(y, want, mag, dtype, R.sums(k, r) + R.pieces(dtype), "y")
    alone = T.adapters_forward(**p)
    R.check(alone, *R.forward(**p, base=None)[:2], dtype, R.sums(k, r) + R.pieces(dtype), "y without base")
    assert T.adapters_forward(**p, base=more["base"], out=more["base"]) is not None and torch.equal(more["base"], y)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("m,k,n,r,adapters,order", SIZES)
def test_backward(m, k, n, r, adapters, order, packed, dtype):
    p, more = problem(m, k, n, r, adapters, dtype, order)
    x = p.pop("x")
    kept = T.checkpoint_pack(x) if packed else x
    value = R.unpacked(*(t.cpu() for t in kept)) if packed else x
    dx, ga, gb = T.adapters_backward(more["dy"], kept, more["hidden"], **p, base=more["dbase"])
    want = R.backward(more["dy"], value, more["hidden"], **p, base=more["dbase"])
    R.check(dx, *want["dx"], dtype, R.sums(n, r) + R.pieces(dtype), "dx")
    R.check(ga, *want["grad_a"], dtype, R.sums(n, m) + R.pieces(dtype), "grad_a")
    R.check(gb, *want["grad_b"], dtype, R.sums(m) + R.pieces(dtype), "grad_b")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("r", [64, 128])
@pytest.mark.parametrize("m,order", [(300, "mixed"), (607, "runs")])
def test_few_rows_in_many_slices(m, order, r, dtype):
    """Fewer waves than that, whose rows would be read in eight slices for every 64 columns."""
    p, more = problem(m, 4100, 9000, r, 3, dtype, order)
    y, hidden = T.adapters_forward(**p, base=more["base"], keep_hidden=True)
    want, mag, h, hmag = R.forward(**p, base=more["base"])
    R.check(hidden, h, hmag, F32, R.sums(4100), "hidden")
    R.check(y, want, mag, dtype, R.sums(4100, r) + R.pieces(dtype), "y")
    p, more = problem(m, 9000, 4100, r, 3, dtype, order)
    x = p.pop("x")
    got = T.adapters_backward(more["dy"], x, more["hidden"], **p, base=more["dbase"])
    want = R.backward(more["dy"], x, more["hidden"], **p, base=more["dbase"])
    for name, g, slack in zip(("dx", "grad_a", "grad_b"), got, (R.sums(4100, r), R.sums(4100, m), R.sums(m))):
        R.check(g, *want[name], dtype, slack + R.pieces(dtype), name)
