"""Infinities in the adapters' operands: results are what the formulas give in 64 bits, an infinity where those give one.  Signs are chosen so that
they do: a factor's values have the sign of their place on the long axis, so that all ranks of a row with an infinity have one sign."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from caif_amd import torch_ops as T                                             # noqa: E402
import adapter_reference as R                                                   # noqa: E402
from test_gpu_adapters import BF16, F16, F32, problem                           # noqa: E402

INF = float("inf")
# decode rows, tiles that are whole and others, ranks that are whole octets but no whole step, both widths of the long axis's waves
SIZES = [(3, 264, 200, 24, 4), (64, 256, 320, 8, 2), (64, 320, 256, 24, 2), (80, 128, 192, 40, 3), (200, 333, 77, 16, 3), (50, 72, 130, 100, 2),
         (300, 264, 136, 64, 2), (2064, 4160, 4160, 16, 2), (2064, 4160, 4160, 24, 2), (600, 64, 128, 8, 2),
         (600, 128, 256, 24, 2), (600, 192, 320, 40, 3), (600, 65, 129, 72, 2), (2064, 4096, 4352, 24, 2)]


def signed(m, k, n, r, adapters, dtype):
    p, more = problem(m, k, n, r, adapters, dtype, "mixed")
    sign = lambda length: (torch.arange(length, device="cuda") * 7 % 3 - 0.5).sign().to(dtype)      # noqa: E731
    p["a"] = (p["a"].abs() + 2.0 ** -6) * sign(k)
    p["b"] = (p["b"].abs() + 2.0 ** -6) * sign(n)[:, None]
    rows = ((p["ids"] >= 0) & (p["ids"] < adapters)).nonzero()[:, 0]
    return p, more, int(rows[len(rows) // 2])


def forward(p, more, k, r, dtype, what):
    y, hidden = T.adapters_forward(**p, base=more["base"], keep_hidden=True)
    want, mag, h, hmag = R.forward(**p, base=more["base"])
    R.check(hidden, h, hmag, F32, R.sums(k), what + ": hidden")
    R.check(y, want, mag, dtype, R.sums(k, r) + R.pieces(dtype), what + ": y")
    assert torch.equal(T.adapters_forward(**p, base=more["base"], out=more["base"].clone()).isnan(), y.isnan())
    into = more["base"].clone()
    T.adapters_forward(**{**p}, base=into, out=into)
    assert torch.equal(into.nan_to_num(0.0), y.nan_to_num(0.0)), what
    return want


def backward(p, more, x, value, m, n, r, dtype, what):
    rest = {key: p[key] for key in ("ids", "a", "b", "scaling")}
    dx, ga, gb = T.adapters_backward(more["dy"], x, more["hidden"], **rest, base=more["dbase"])
    want = R.backward(more["dy"], value, more["hidden"], **rest, base=more["dbase"])
    R.check(dx, *want["dx"], dtype, R.sums(n, r) + R.pieces(dtype), what + ": dx")
    R.check(ga, *want["grad_a"], dtype, R.sums(n, m) + R.pieces(dtype), what + ": grad_a")
    R.check(gb, *want["grad_b"], dtype, R.sums(m) + R.pieces(dtype), what + ": grad_b")
    return want


def copies(p, more):
    return {k: v.clone() for k, v in p.items()}, {k: v.clone() for k, v in more.items()}


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,k,n,r,adapters", SIZES)
def test_forward(m, k, n, r, adapters, dtype):
    p, more, row = signed(m, k, n, r, adapters, dtype)
    l = int(p["ids"][row])
    q, o = copies(p, more)
    q["x"][row, k // 2] = -INF
    assert forward(q, o, k, r, dtype, "x")[row].isinf().all()
    for j in (0, r - 1):                               # the last values of a factor's row are also what fills a step
        q, o = copies(p, more)
        q["a"][l, j, k - 1] = INF
        assert forward(q, o, k, r, dtype, "a")[row].isinf().all()
        q, o = copies(p, more)
        q["b"][l, n - 1, j] = -INF
        want = forward(q, o, k, r, dtype, "b")
        assert want[row, n - 1].isinf() and want[row, :n - 1].isfinite().all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("m,k,n,r,adapters", SIZES)
def test_backward(m, k, n, r, adapters, packed, dtype):
    p, more, row = signed(m, k, n, r, adapters, dtype)
    l = int(p["ids"][row])
    for t, off in ((p["x"], 2.0 ** -6), (more["dy"], 2.0 ** -10), (more["hidden"], 2.0 ** -6)):      # no products of an infinity and zero
        t += torch.where(t < 0, -off, off).to(t.dtype)

    def kept(q):
        x = T.checkpoint_pack(q["x"]) if packed else q["x"]
        return x, R.unpacked(*(t.cpu() for t in x)) if packed else x

    q, o = copies(p, more)
    o["dy"][row, n // 2] = INF
    want = backward(q, o, *kept(q), m, n, r, dtype, "dy")
    assert want["dx"][0][row].isinf().all() and want["grad_b"][0][l, n // 2].isinf().all() and want["grad_b"][0][l, 0].isfinite().all()
    assert packed or want["grad_a"][0][l].isinf().all()
    q, o = copies(p, more)
    o["hidden"][row, r - 1] = -INF
    want = backward(q, o, *kept(q), m, n, r, dtype, "hidden")
    assert want["grad_b"][0][l, :, r - 1].isinf().all()
    for j in (0, r - 1):
        q, o = copies(p, more)
        q["a"][l, j, k - 1] = INF
        want = backward(q, o, *kept(q), m, n, r, dtype, "a")
        assert want["dx"][0][row, k - 1].isinf() and want["dx"][0][row, :k - 1].isfinite().all()
        q, o = copies(p, more)
        q["b"][l, 0, j] = -INF
        want = backward(q, o, *kept(q), m, n, r, dtype, "b")
        assert want["dx"][0][row].isinf().all()
    if not packed:
        q, o = copies(p, more)
        q["x"][row, 0] = INF
        want = backward(q, o, *kept(q), m, n, r, dtype, "x")
        assert want["grad_a"][0][l, :, 0].isinf().all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_fp32_values_beyond_bf16(dtype):
    """Hidden values between the largest bf16 and the largest fp32 number."""
    p, more, row = signed(130, 264, 200, 24, 3, dtype)
    l = int(p["ids"][row])
    more["hidden"][row, 3] = 3.4e38
    want = backward(p, more, p["x"], p["x"], 130, 200, 24, dtype, "hidden")
    assert want["grad_b"][0][l, :, 3].isfinite().all()
