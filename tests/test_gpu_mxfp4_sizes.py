"""Microscaled 4-bit products and the gated block at sizes that take the forms of large weights: several column tiles of a workgroup, many steps of a
tile, shared reductions, tiles of 256 rows.  Against the definition in 64 bits, on the device."""
import pytest
import torch

from caif_amd import capi, torch_ops as T
import mxfp4_reference as R

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def mx_weight(g, n, k, **scales):
    codes, s = R.random_weight(g, n, k, device="cuda", **scales)
    return T.FrozenWeight(codes, T.W_MXFP4, s, n, k, 1, 32), R.decode(codes, s, k)


def weight(g, kind, dtype, n, k):
    if kind == "mx":
        return mx_weight(g, n, k)
    w = (0.05 * torch.randn(n, k, generator=g)).to(dtype).cuda()
    return T.FrozenWeight(w, T.W_F16 if dtype == torch.float16 else T.W_BF16, None, n, k), w.double()


def normal(g, rows, cols, dtype):
    return torch.randn(rows, cols, generator=g).to(dtype).cuda()


def check(got, want, most):
    off = (got.double() - want).abs()
    assert bool((off <= most).all()), f"{float((off / most).max())} times the bound"


def within(got, a, b, pieces=1):
    """got against a b^T in 64 bits"""
    want = a @ b.T
    check(got, want, R.bound(want, a.abs() @ b.abs().T, a.shape[1], got.dtype, pieces))


def pieces_of(dtype):
    return 3 if dtype == "f32" else 1


# ------------------------------------------------------------------ few rows: the columns of a weight are cut into about 256 parts
# N = 14336 and 14339 give a workgroup 56 and 57 columns, four column tiles; 6001 two; a reduction of 14337 beside 4096 columns is shared by several workgroups
FEW = [(1, 14336, 1056), (4, 14339, 1403), (3, 14336, 330), (9, 14336, 1403), (16, 14339, 300), (24, 14336, 2048), (24, 14339, 1185), (50, 14336, 1056),
       (64, 14339, 471), (100, 14336, 776), (2, 6001, 1403), (30, 6001, 520), (1, 4096, 8200), (24, 4096, 14337), (12, 4090, 16384),
       (50, 4096, 14336)]


@pytest.mark.parametrize("M,N,K", FEW)
@pytest.mark.parametrize("dtype", DTYPES)
def test_few_rows(M, N, K, dtype):
    g = gen(M + N + K)
    w, exact = mx_weight(g, N, K)
    dt = DTYPES[dtype]
    code = T.CODE_OF[dt]
    x = normal(g, M, K, dt)
    y = T.qlinear_forward(x, w, code, code)
    within(y, x.double(), exact, pieces_of(dtype))
    add = normal(g, M, N, dt)
    assert torch.equal(T.qlinear_forward(x, w, code, code, addend=add), (y.float() + add.float()).to(dt))
    # activations of another type are laid out beforehand
    other = DTYPES["bf16" if dtype == "f32" else "f32"]
    x = normal(g, M, K, other)
    # (bf16 activations with fp32 products are multiplied as they are)
    within(T.qlinear_forward(x, w, code, T.F32), x.to(dt).double(), exact)


@pytest.mark.parametrize("M,N,K", FEW)
@pytest.mark.parametrize("kind,dtype", [("mx", "bf16"), ("mx", "f16"), ("mx", "f32"), ("same", "bf16"), ("same", "f16")])
def test_few_rows_gated(M, N, K, kind, dtype):
    g = gen(M + N + K + 1)
    dt = DTYPES[dtype]
    (wg, eg), (wu, eu) = weight(g, kind, dt, N, K), weight(g, kind, dt, N, K)
    x = normal(g, M, K, dt)
    hidden, gate, up = T.gated_forward(x, wg, wu, keep=True)
    gated(hidden, gate, up, x, eg, eu, pieces_of(dtype))
    assert torch.equal(T.gated_forward(x, wg, wu), hidden)


def gated(hidden, gate, up, x, eg, eu, pieces):
    """The three results of a gated forward against 64 bits, bounds as for smaller sizes: silu's slope is at most 1.1, its exponential, inverse and
    three products are within 8 roundings of 32 bits."""
    x, dt, K = x.double(), hidden.dtype, x.shape[1]
    a, b, sa, sb = x @ eg.T, x @ eu.T, x.abs() @ eg.abs().T, x.abs() @ eu.abs().T
    check(gate, a, R.bound(a, sa, K, dt, pieces))
    check(up, b, R.bound(b, sb, K, dt, pieces))
    part = (pieces * (K / 32 + 1) + 48) * 2.0 ** -23
    da, db, top = part * sa, part * sb, torch.finfo(dt)
    want = R.silu(a) * b
    check(hidden, want, 1.1 * da * (b.abs() + db) + R.silu(a).abs() * db + (8 * 2.0 ** -24 + top.eps / 2) * want.abs() + top.smallest_normal * top.eps)


@pytest.mark.parametrize("M,N,K", FEW)
def test_few_rows_in_four_bits(M, N, K):
    g = gen(M + N + K + 2)
    w, exact = mx_weight(g, N, K)
    a, sa = R.random_weight(g, M, K, device="cuda", low=110, high=130)
    within(T.mxfp4_matmul(a, sa, w.wq, w.scales, T.F32), R.decode(a, sa, K), exact)


@pytest.mark.parametrize("M", [1, 4, 20, 50])
@pytest.mark.parametrize("K", [513, 544, 799, 991, 4096 + 96, 8192 + 1])
def test_ends_of_rows_in_16_bits(M, K):
    """Products of one piece keep the bound of one piece."""
    g = gen(M + K)
    w, exact = mx_weight(g, 70, K)
    for dtype in (torch.bfloat16, torch.float16):
        x = normal(g, M, K, dtype)
        within(T.qlinear_forward(x, w, T.CODE_OF[dtype], T.F32), x.double(), exact)


# ------------------------------------------------------------------ input gradients from the stored weights: several steps of a wave, in and without parts
@pytest.mark.parametrize("M,N,K", [(1, 14336, 520), (16, 14336, 1403), (32, 8200, 4096), (100, 4096, 4096), (333, 2048, 1403), (500, 5003, 2000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient(M, N, K, dtype):
    g = gen(M + N + K + 3)
    w, exact = mx_weight(g, N, K)
    dt = DTYPES[dtype]
    code = T.CODE_OF[dt]
    dy = normal(g, M, N, dt)
    within(T.qlinear_backward_input(dy, w, code, code), dy.double(), exact.T, pieces_of(dtype))
    other = DTYPES["bf16" if dtype == "f32" else "f32"]
    dy = normal(g, M, N, other)
    within(T.qlinear_backward_input(dy, w, code, T.F32), dy.to(dt).double(), exact.T)


# ------------------------------------------------------------------ dense products: tiles of every size, several operand pairs, rows of any width
# gated: tiles of 256 x 256 (1030 x 4100, 2048 x 11008, 2041 x 11001), 128 x 256 (2048 x 5501) and 128 x 128
DENSE = [(1030, 4100, 1088), (2048, 11008, 520), (2041, 11001, 1003), (2048, 5501, 600), (330, 4100, 1088), (333, 2003, 1403), (1500, 6000, 1088)]


@pytest.mark.parametrize("M,N,K", DENSE)
@pytest.mark.parametrize("kind,dtype", [("mx", "bf16"), ("mx", "f16"), ("mx", "f32"), ("same", "bf16"), ("same", "f16")])
def test_dense_gated(M, N, K, kind, dtype):
    g = gen(M + N + K + 4)
    dt, pieces = DTYPES[dtype], pieces_of(dtype)
    (wg, eg), (wu, eu) = weight(g, kind, dt, N, K), weight(g, kind, dt, N, K)
    x, d = normal(g, M, K, dt), normal(g, M, N, dt)
    hidden, gate, up = T.gated_forward(x, wg, wu, keep=True)
    gated(hidden, gate, up, x, eg, eu, pieces)
    assert torch.equal(T.gated_forward(x, wg, wu), hidden)
    dx, da, db = T.gated_backward(d, gate, up, wg, wu)
    # the product takes the gradients as they are returned
    p, q = da.double(), db.double()
    want = p @ eg + q @ eu
    check(dx, want, R.bound(want, p.abs() @ eg.abs() + q.abs() @ eu.abs(), 2 * N, dt, pieces))


@pytest.mark.parametrize("M,N,K", DENSE + [(512, 4096, 8192), (2048, 11001, 1088)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_dense(M, N, K, dtype):
    g = gen(M + N + K + 5)
    w, exact = mx_weight(g, N, K)
    dt, pieces = DTYPES[dtype], pieces_of(dtype)
    code = T.CODE_OF[dt]
    x, dy = normal(g, M, K, dt), normal(g, M, N, dt)
    within(T.qlinear_forward(x, w, code, code), x.double(), exact, pieces)
    within(T.qlinear_backward_input(dy, w, code, code), dy.double(), exact.T, pieces)


# ------------------------------------------------------------------ both operands in 4 bits, in tiles
def ordered(M, N, K):
    """What the scales of both operands take in the tiles' order: 1 KB for 64 rows and 16 blocks."""
    groups = -(-K // 512)
    return (-(-M // 64) + -(-N // 64)) * groups * 1024


@pytest.mark.parametrize("parts,M,N,K", [
    (1, 512, 4096, 4096), (1, 500, 4099, 1257), (1, 512, 4096, 1280), (1, 1279, 2555, 4100),                # tiles of 128 x 128: 16, 5, 5 and 17 steps
    (4, 256, 4096, 14336), (4, 250, 4090, 14300), (2, 1000, 2040, 14300),                                  # their steps shared by workgroups
    (1, 1100, 8000, 1280), (1, 1100, 8001, 1500),                                                          # tiles of 256 x 256: 5 and 6 steps
    (1, 1530, 10999, 1257), (1, 2048, 4096, 1300)])                                                        # their last round halved
def test_tiles(parts, M, N, K):
    need = capi.lib().caifx_mxfp4_matmul_workspace_bytes(M, N, K)
    assert need == ordered(M, N, K) + (parts * M * N * 4 if parts > 1 else 0), "another kernel takes this size"
    g = gen(M + N + K + 6)
    a, sa = R.random_weight(g, M, K, device="cuda")
    b, sb = R.random_weight(g, N, K, device="cuda", low=110, high=130)
    p, q = R.decode(a, sa, K), R.decode(b, sb, K)
    for code in (T.F32, T.BF16, T.F16):
        within(T.mxfp4_matmul(a, sa, b, sb, code), p, q)
    # a block that is a NaN: its row and its column, and nothing else
    row, column, block = M - 3, N // 2, K // 32 - 1
    sa[row, block], sb[column, 1] = 255, 255
    y = T.mxfp4_matmul(a, sa, b, sb, T.F32)
    nan = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    nan[row], nan[:, column] = True, True
    assert torch.equal(y.isnan(), nan)
    want = p @ q.T
    check(y[~nan], want[~nan], R.bound(want, p.abs() @ q.abs().T, K, torch.float32)[~nan])


# ------------------------------------------------------------------ the ends of the grids
def test_more_row_tiles_than_a_launch_has():
    """A launch takes 65535 tiles of 64 rows; the rows behind them go in another one."""
    M, N, K = 65535 * 64 + 75, 9, 250
    g = gen(7)
    w, exact = mx_weight(g, N, K)
    L = capi.lib()
    x = torch.empty(M, K, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(7))
    y = torch.empty(M, N, dtype=torch.float32, device="cuda")
    # without room for dense copies (256 elements a row and the weight's) the product stays on the kernels of few rows
    need = L.caifx_qlinear_partials_workspace_bytes(M, N, K, T.BF16, T.BF16, T.W_MXFP4, 0)
    assert need < L.caifx_qlinear_workspace_bytes(M, N, K, T.BF16, T.BF16, T.W_MXFP4, 0)
    T.qlinear_forward(x, w, T.BF16, T.F32, out=y, workspace=torch.empty(need, dtype=torch.uint8, device="cuda"))
    within(y, x.double(), exact)
    codes, scales = T.mxfp4_quantize(x)
    y = T.mxfp4_matmul(codes, scales, w.wq, w.scales)
    within(y, R.decode(codes, scales, K), exact)


@pytest.mark.parametrize("kind,M,K", [("same", 2, 8), ("mx", 1030, 40)])
def test_gradient_of_nearly_4_million_weight_rows(kind, M, K):
    """The last rows below 2^22: the transposed copy's rows are 2^22 long."""
    N = 2 ** 22 - 1
    g = torch.Generator(device="cuda").manual_seed(8)
    if kind == "mx":
        codes = torch.randint(0, 256, (N, 32), dtype=torch.uint8, device="cuda", generator=g)
        codes[:, 20:] = 0
        s = torch.randint(118, 125, (N, 2), dtype=torch.uint8, device="cuda", generator=g)
        w, exact = T.FrozenWeight(codes, T.W_MXFP4, s, N, K, 1, 32), R.decode(codes, s, K)
        dy = torch.empty(M, N, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
        dx = T.qlinear_backward_input(dy, w, T.BF16)
        want, size = torch.zeros(M, K, dtype=torch.float64, device="cuda"), torch.zeros(M, K, dtype=torch.float64, device="cuda")
        for n in range(0, N, 2 ** 17):
            part = dy[:, n:n + 2 ** 17].double()
            want += part @ exact[n:n + 2 ** 17]
            size += part.abs() @ exact[n:n + 2 ** 17].abs()
        check(dx, want, R.bound(want, size, N, torch.float32))
        return
    stored = [torch.empty(N, K, dtype=torch.bfloat16, device="cuda").normal_(generator=g) for _ in range(2)]
    d, gate, up = (torch.empty(M, N, dtype=torch.bfloat16, device="cuda").normal_(generator=g) for _ in range(3))
    dx, da, db = T.gated_backward(d, gate, up, *(T.FrozenWeight(w, T.W_BF16, None, N, K) for w in stored))
    p, q = da.double(), db.double()
    eg, eu = (w.double() for w in stored)
    want = p @ eg + q @ eu
    check(dx, want, R.bound(want, p.abs() @ eg.abs() + q.abs() @ eu.abs(), 2 * N, torch.bfloat16))
