"""Microscaled 4-bit floating point on the GPU: codes and scales value for value, products against the definition in 64 bits."""
import pytest
import torch

from caif_amd import capi, torch_ops as T
import mxfp4_reference as R

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def weight(g, n, k, **scales):
    codes, s = R.random_weight(g, n, k, **scales)
    return T.FrozenWeight(codes.cuda(), T.W_MXFP4, s.cuda(), n, k, 1, 32), R.decode(codes, s, k)


def within(got, exact, magnitude, length, pieces=1):
    off, most = (got.double().cpu() - exact).abs(), R.bound(exact, magnitude, length, got.dtype, pieces)
    ok = bool((off <= most).all())
    assert ok, f"{float((off / most).max())} times the bound"


# ------------------------------------------------------------------ codes and scales
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (5, 32), (2, 33), (7, 64), (64, 1403), (333, 256), (4097, 40)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize(rows, cols, dtype):
    g = gen(rows * cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-12, 12, (rows, 1), generator=g).float())).to(DTYPES[dtype])
    codes, scales = T.mxfp4_quantize(x.cuda())
    want_codes, want_scales = R.quantize(x)
    assert torch.equal(scales.cpu(), want_scales) and torch.equal(codes.cpu(), want_codes)
    back = T.mxfp4_dequantize(codes, scales, cols, DTYPES[dtype])
    assert torch.equal(back.double().cpu(), R.decode(want_codes, want_scales, cols).to(DTYPES[dtype]).double())


def test_quantize_special():
    tiny, most = 2.0 ** -149, torch.finfo(torch.float32).max
    rows = [[0.0] * 40, [-0.0] * 40, [tiny] * 40, [2.0 ** -126, -tiny] * 20, [2.0 ** -125, 2.0 ** -127] * 20, [most, -most, 1.0, 2.0 ** 120] * 10,
            [float("inf")] + [1.0] * 39, [1.0] * 39 + [float("-inf")], [1.0] * 20 + [float("nan")] + [1.0] * 19]
    # every border between two codes, one step below and above it
    ties = []
    for t in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0):
        v = torch.tensor(t)
        ties += [float(v), float(torch.nextafter(v, torch.tensor(9.0))), -float(torch.nextafter(v, torch.tensor(0.0)))]
    rows.append((ties + [6.0] * 40)[:31] + [6.0] + [7.99] * 8)
    x = torch.tensor(rows)
    codes, scales = T.mxfp4_quantize(x.cuda())
    want_codes, want_scales = R.quantize(x)
    assert torch.equal(scales.cpu(), want_scales) and torch.equal(codes.cpu(), want_codes)
    for dtype in DTYPES.values():
        got, want = T.mxfp4_dequantize(codes, scales, 40, dtype).cpu(), R.decode(want_codes, want_scales, 40).float().to(dtype)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


def test_dequantize_every_pair():
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1).reshape(256, 16, 16).cuda()
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 16).cuda()
    for dtype in DTYPES.values():
        got = T.mxfp4_dequantize(codes.reshape(256, 256), scales, 512, dtype).cpu()
        want = R.decode(codes.reshape(256, 256).cpu(), scales.cpu(), 512).float().to(dtype)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


def test_shapes_and_addresses():
    x = torch.randn(2, 3, 40, generator=gen(1)).to(torch.bfloat16).cuda()
    codes, scales = T.mxfp4_quantize(x)
    assert codes.shape == (2, 3, 32) and scales.shape == (2, 3, 2)
    assert T.mxfp4_dequantize(codes, scales, 40, torch.float32).shape == (2, 3, 40)
    odd = torch.empty(6 * 40 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(6, 40)
    odd.copy_(x.view(6, 40))
    assert torch.equal(T.mxfp4_quantize(odd)[0], codes.view(6, 32))
    for shape in ((0, 40), (4, 0)):
        c, s = T.mxfp4_quantize(torch.empty(shape, device="cuda"))
        assert c.numel() == 0 and s.numel() == 0 and T.mxfp4_dequantize(c, s, shape[1], torch.float16).shape == shape


# ------------------------------------------------------------------ products with a frozen weight
SHAPES = [(1, 1, 1), (1, 7, 33), (1, 1024, 256), (2, 16, 64), (3, 100, 1403), (15, 65, 300), (16, 64, 512), (17, 129, 320), (32, 200, 96), (33, 48, 2000),
          (64, 130, 256), (65, 257, 4096), (100, 1000, 136), (128, 256, 1024), (130, 72, 2304), (300, 520, 776), (513, 264, 1001)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_forward(M, N, K, dtype):
    g = gen(M + N + K)
    w, exact = weight(g, N, K)
    x = torch.randn(M, K, generator=g).to(DTYPES[dtype])
    code = T.CODE_OF[x.dtype]
    want, size = x.double() @ exact.T, x.double().abs() @ exact.abs().T
    y = T.qlinear_forward(x.cuda(), w, code, code)
    within(y, want, size, K, 3 if dtype == "f32" else 1)
    addend = torch.randn(M, N, generator=g).to(x.dtype)
    both = T.qlinear_forward(x.cuda(), w, code, code, addend=addend.cuda())
    assert torch.equal(both, (y.float() + addend.cuda().float()).to(y.dtype))


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient(M, N, K, dtype):
    g = gen(M + N + K + 1)
    w, exact = weight(g, N, K)
    dy = torch.randn(M, N, generator=g).to(DTYPES[dtype])
    code = T.CODE_OF[dy.dtype]
    dx = T.qlinear_backward_input(dy.cuda(), w, code, code)
    within(dx, dy.double() @ exact, dy.double().abs() @ exact.abs(), N, 3 if dtype == "f32" else 1)
    addend = torch.randn(M, K, generator=g).to(dy.dtype)
    both = T.qlinear_backward_input(dy.cuda(), w, code, code, addend=addend.cuda())
    assert torch.equal(both, (dx.float() + addend.cuda().float()).to(dx.dtype))


@pytest.mark.parametrize("K", [512, 513, 544, 577, 608, 640, 700, 799, 832, 991, 1024, 1056, 4096 + 32, 4096 + 96, 4096 + 256, 4096 + 416, 8192 + 1])
@pytest.mark.parametrize("M", [1, 9, 20, 50])
def test_ends_of_rows(M, K):
    """Rows that end anywhere in the kernels' units of 512 values, and in their blocks."""
    g = gen(M * K)
    N = 70
    w, exact = weight(g, N, K)
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.randn(M, K, generator=g).to(dtype)
        within(T.qlinear_forward(x.cuda(), w, T.CODE_OF[dtype], T.CODE_OF[dtype]), x.double() @ exact.T, x.double().abs() @ exact.abs().T, K, 3)
    a, sa = R.random_weight(g, M, K)
    p = R.decode(a, sa, K)
    within(T.mxfp4_matmul(a.cuda(), sa.cuda(), w.wq, w.scales), p @ exact.T, p.abs() @ exact.abs().T, K)


@pytest.mark.parametrize("M,N,K", [(300, 1101, 512), (700, 999, 130), (1100, 640, 1000), (2100, 333, 257), (3000, 1024, 64)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows(M, N, K, dtype):
    """Calls that run on dense operands, some into rows that are no whole pieces of 16 bytes, with an addend."""
    g = gen(M + N + K)
    w, exact = weight(g, N, K)
    dt = DTYPES[dtype]
    code, pieces = T.CODE_OF[dt], 3 if dtype == "f32" else 1
    x, dy, add = (torch.randn(M, n, generator=g).to(dt) for n in (K, N, N))
    y = T.qlinear_forward(x.cuda(), w, code, code)
    within(y, x.double() @ exact.T, x.double().abs() @ exact.abs().T, K, pieces)
    assert torch.equal(T.qlinear_forward(x.cuda(), w, code, code, addend=add.cuda()), (y.float() + add.cuda().float()).to(dt))
    dx = T.qlinear_backward_input(dy.cuda(), w, code, code)
    within(dx, dy.double() @ exact, dy.double().abs() @ exact.abs(), N, pieces)
    a = T.mxfp4_quantize(x.cuda())
    p = R.decode(*R.quantize(x), K)
    within(T.mxfp4_matmul(*a, w.wq, w.scales, code), p @ exact.T, p.abs() @ exact.abs().T, K)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("xd,cd,yd", [("f32", "bf16", "f32"), ("f32", "f16", "f16"), ("bf16", "f32", "f32"), ("f16", "bf16", "f32"), ("bf16", "bf16", "f16")])
@pytest.mark.parametrize("M", [5, 70])
def test_types(M, xd, cd, yd, backward):
    """Activations are rounded to the compute type, whatever theirs is."""
    g = gen(M)
    N, K = 136, 328
    w, exact = weight(g, N, K)
    x = torch.randn(M, N if backward else K, generator=g).to(DTYPES[xd])
    used = x.to(DTYPES[cd]).double()
    y = (T.qlinear_backward_input if backward else T.qlinear_forward)(x.cuda(), w, T.CODE_OF[DTYPES[cd]], T.CODE_OF[DTYPES[yd]])
    m = exact if backward else exact.T
    within(y, used @ m, used.abs() @ m.abs(), x.shape[1], 3 if cd == "f32" else 1)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 40])
def test_without_workspace(M, dtype, backward):
    g = gen(5)
    N, K = 100, 200
    w, exact = weight(g, N, K)
    x = torch.randn(M, N if backward else K, generator=g).to(DTYPES[dtype])
    y = torch.empty(M, K if backward else N, dtype=x.dtype, device="cuda")
    none = torch.empty(0, dtype=torch.uint8, device="cuda")
    call = T.qlinear_backward_input if backward else T.qlinear_forward
    assert call(x.cuda(), w, T.CODE_OF[x.dtype], T.CODE_OF[x.dtype], out=y, workspace=none) is y
    m = exact if backward else exact.T
    # the shape-agnostic kernels add one product at a time: in the backward every product passes through all later additions
    off, size = (y.double().cpu() - x.double() @ m).abs(), x.double().abs() @ m.abs()
    assert bool((off <= x.shape[1] * 2.0 ** -23 * size + R.bound(x.double() @ m, size, 32, x.dtype)).all())


def test_scales_over_the_whole_range():
    """Blocks from the smallest scale to the largest that quantising gives: in bf16 every value is exact, also below the normal numbers."""
    g = gen(9)
    N, K = 48, 32 * 253
    codes, _ = R.random_weight(g, N, K)
    scales = torch.arange(253, dtype=torch.uint8).repeat(N, 1)
    w = T.FrozenWeight(codes.cuda(), T.W_MXFP4, scales.cuda(), N, K, 1, 32)
    exact = R.decode(codes, scales, K)
    for block in (0, 1, 2, 60, 126, 200, 252):
        x = torch.zeros(1, K, dtype=torch.float64)
        x[0, 32 * block:32 * block + 32] = torch.randint(-8, 9, (32,), generator=g).double() * 2.0 ** (110 - block if block < 200 else -10)
        for dtype in ("bf16", "f32"):
            y = T.qlinear_forward(x.to(DTYPES[dtype]).cuda(), w, T.CODE_OF[DTYPES[dtype]])
            within(y, x @ exact.T, x.abs() @ exact.abs().T, K, 3)


def test_not_a_number_stays_in_its_rows():
    g = gen(11)
    M, N, K = 20, 40, 100
    w, exact = weight(g, N, K)
    w.scales[7, 1] = 255
    x = torch.randn(M, K, generator=g).to(torch.bfloat16).cuda()
    x[3, 50], x[5, 2], x[6, 99] = float("nan"), float("inf"), float("-inf")
    for dtype in (torch.bfloat16, torch.float32):
        y = T.qlinear_forward(x.to(dtype), w, T.CODE_OF[dtype], T.CODE_OF[dtype])
        plain = x.double().cpu() @ T.mxfp4_dequantize(w.wq, w.scales, K, torch.float32).double().cpu().T
        assert torch.equal(y.cpu().isnan(), plain.isnan()) and torch.equal(y.cpu().isinf(), plain.isinf())
        dx = T.qlinear_backward_input(torch.ones(2, N, dtype=dtype, device="cuda"), w, T.CODE_OF[dtype])
        assert torch.equal(dx.isnan().any(0).cpu(), (torch.arange(K) >= 32) & (torch.arange(K) < 64))


def test_what_is_behind_the_last_column():
    """Codes that fill up the last block count for nothing in the products with a frozen weight, whatever they are."""
    g = gen(12)
    N, K = 33, 40
    w, exact = weight(g, N, K)
    codes = w.wq.view(N, 32)
    codes[:, 20:] = 0x77
    for M in (4, 50):
        x = torch.randn(M, K, generator=g).to(torch.bfloat16)
        within(T.qlinear_forward(x.cuda(), w, T.BF16), x.double() @ exact.T, x.double().abs() @ exact.abs().T, K)
        dy = torch.randn(M, N, generator=g).to(torch.bfloat16)
        within(T.qlinear_backward_input(dy.cuda(), w, T.BF16), dy.double() @ exact, dy.double().abs() @ exact.abs(), N)


# ------------------------------------------------------------------ both operands in 4 bits
@pytest.mark.parametrize("M,N,K", SHAPES + [(1, 14336, 128), (256, 256, 256), (260, 300, 4096), (700, 1100, 544)])
@pytest.mark.parametrize("yd", DTYPES)
def test_matmul(M, N, K, yd):
    g = gen(M * 3 + N + K)
    a, sa = R.random_weight(g, M, K)
    b, sb = R.random_weight(g, N, K, low=110, high=130)
    y = T.mxfp4_matmul(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), T.CODE_OF[DTYPES[yd]])
    p, q = R.decode(a, sa, K), R.decode(b, sb, K)
    within(y, p @ q.T, p.abs() @ q.abs().T, K)


def test_matmul_special():
    g = gen(21)
    M, N, K = 40, 70, 300
    a, sa = R.random_weight(g, M, K)
    b, sb = R.random_weight(g, N, K)
    sa[3, 2], sb[9, 0] = 255, 255
    y = T.mxfp4_matmul(a.cuda(), sa.cuda(), b.cuda(), sb.cuda()).cpu()
    nan = torch.zeros(M, N, dtype=torch.bool)
    nan[3], nan[:, 9] = True, True
    assert torch.equal(y.isnan(), nan)
    # products whose factors' scales are far apart meet near one
    for low, high in ((0, 3), (20, 40), (250, 252)):
        a, sa = R.random_weight(g, M, K, low=low, high=high)
        b, sb = R.random_weight(g, N, K, low=252 - high, high=252 - low)
        p, q = R.decode(a, sa, K), R.decode(b, sb, K)
        within(T.mxfp4_matmul(a.cuda(), sa.cuda(), b.cuda(), sb.cuda()), p @ q.T, p.abs() @ q.abs().T, K)
    out = torch.full((M + 1, N), 7.0, device="cuda")
    assert T.mxfp4_matmul(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), out=out[:M]).data_ptr() == out.data_ptr() and bool((out[M] == 7).all())


def test_activations_and_weight_in_four_bits():
    """As a program uses them: a weight put away once, activations of each call."""
    g = gen(22)
    M, N, K = 70, 260, 1000
    x, w = torch.randn(M, K, generator=g).to(torch.bfloat16), (0.02 * torch.randn(N, K, generator=g)).to(torch.bfloat16)
    wc, ws = T.mxfp4_quantize(w.cuda())
    xc, xs = T.mxfp4_quantize(x.cuda())
    p, q = R.decode(*R.quantize(x), K), R.decode(*R.quantize(w), K)
    within(T.mxfp4_matmul(xc, xs, wc, ws, T.BF16), p @ q.T, p.abs() @ q.abs().T, K)
    # and the frozen weight with the activations' own values is nearer
    y = T.qlinear_forward(x.cuda(), T.FrozenWeight(wc, T.W_MXFP4, ws, N, K, 1, 32), T.BF16, T.BF16)
    exact = x.double() @ q.T
    within(y, exact, x.double().abs() @ q.abs().T, K)
    assert float((p @ q.T - exact).norm() / exact.norm()) > 0.05


# ------------------------------------------------------------------ streams, graphs, bytes beside the result
@pytest.mark.parametrize("M", [1, 40, 520])
def test_other_stream_and_graph(M):
    g = gen(30 + M)
    N, K = 264, 512
    w, exact = weight(g, N, K)
    x = torch.randn(M, K, generator=g).to(torch.bfloat16).cuda()
    dy = torch.randn(M, N, generator=g).to(torch.bfloat16).cuda()

    def step():
        codes = T.mxfp4_quantize(x)
        return T.qlinear_forward(x, w, T.BF16, T.BF16), T.qlinear_backward_input(dy, w, T.BF16, T.BF16), T.mxfp4_matmul(*codes, w.wq, w.scales, T.BF16)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for turn in range(3):
        x.copy_(torch.randn(M, K, generator=g).to(torch.bfloat16))
        dy.copy_(torch.randn(M, N, generator=g).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(kept, step()):
            assert torch.equal(p, q)


@pytest.mark.parametrize("M,N,K", [(1, 30, 70), (20, 33, 100), (40, 130, 328), (300, 520, 776)])
def test_nothing_beside_the_result(M, N, K):
    g = gen(40)
    w, _ = weight(g, N, K)
    L = capi.lib()
    s = torch.cuda.current_stream().cuda_stream
    for backward, columns in ((0, N), (1, K)):
        x = torch.randn(M, N if backward else K, generator=g).to(torch.bfloat16).cuda()
        need = L.caifx_qlinear_workspace_bytes(M, N, K, T.BF16, T.BF16, T.W_MXFP4, backward)
        ws = torch.full((need + 64,), 201, dtype=torch.uint8, device="cuda")
        out = torch.full((M * columns + 64,), 3.0, dtype=torch.bfloat16, device="cuda")
        fn = L.caifx_qlinear_backward_input if backward else L.caifx_qlinear_forward
        assert fn(M, N, K, x.data_ptr(), T.BF16, T.BF16, w.wq.data_ptr(), T.W_MXFP4, w.scales.data_ptr(), 1, 32, out[32:].data_ptr(), T.BF16, ws.data_ptr(), need, s) == 0
        torch.cuda.synchronize()
        assert bool((ws[need:] == 201).all()) and bool((out[:32] == 3).all()) and bool((out[32 + M * columns:] == 3).all())
        call = T.qlinear_backward_input if backward else T.qlinear_forward
        assert torch.equal(out[32:32 + M * columns].view(M, columns), call(x, w, T.BF16, T.BF16))


def test_static_form():
    """caifx_qlinear_forward_static has the bits of the call with a workspace of its size."""
    g = gen(50)
    L = capi.lib()
    s = torch.cuda.current_stream().cuda_stream
    N, K = 96, 320
    w, _ = weight(g, N, K)
    for M in (1, 20, 100):
        x = torch.randn(M, K, generator=g).to(torch.bfloat16).cuda()
        y = torch.empty(M, N, device="cuda")
        need = L.caifx_qlinear_partials_workspace_bytes(M, N, K, T.BF16, T.BF16, T.W_MXFP4, 0)
        assert L.caifx_qlinear_forward_static(M, N, K, x.data_ptr(), T.BF16, T.BF16, w.wq.data_ptr(), T.W_MXFP4, w.scales.data_ptr(), 1, 32, y.data_ptr(), T.F32, s) == 0
        want = T.qlinear_forward(x, w, T.BF16, workspace=torch.empty(need, dtype=torch.uint8, device="cuda"))
        assert torch.equal(y, want)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(3, 48, 512), (20, 512, 16384), (32, 1024, 8192), (100, 264, 8192), (300, 512, 2048)])
def test_activations_at_any_address(M, N, K, dtype, backward):
    """Activations that no 16-byte access takes, in the workspace of the query: nothing behind it is written."""
    g = gen(60)
    L = capi.lib()
    s = torch.cuda.current_stream().cuda_stream
    w, exact = weight(g, N, K)
    t = DTYPES[dtype]
    c = T.CODE_OF[t]
    length, C = (N, K) if backward else (K, N)
    x = torch.randn(M, length, generator=g).to(t).cuda()
    apart = torch.empty(M * length + 1, dtype=t, device="cuda")
    apart[1:] = x.view(-1)
    need = L.caifx_qlinear_workspace_bytes(M, N, K, c, c, T.W_MXFP4, int(backward))
    fn = L.caifx_qlinear_backward_input if backward else L.caifx_qlinear_forward
    m = exact if backward else exact.T
    want, size = x.double().cpu() @ m, x.double().cpu().abs() @ m.abs()
    for a in (x, apart[1:]):
        ws = torch.full((need + (1 << 20),), 201, dtype=torch.uint8, device="cuda")
        y = torch.empty(M, C, dtype=t, device="cuda")
        assert fn(M, N, K, a.data_ptr(), c, c, w.wq.data_ptr(), T.W_MXFP4, w.scales.data_ptr(), 1, 32, y.data_ptr(), c, ws.data_ptr(), need, s) == 0
        assert bool((ws[need:] == 201).all())
        within(y, want, size, length, 3 if dtype == "f32" else 1)


@pytest.mark.parametrize("N", [1, 33, 60])
@pytest.mark.parametrize("M", [3, 40, 600])
def test_gradient_of_weights_beyond_fp16(M, N):
    """A last row beyond fp16 is infinite in that compute type; what is read in place of the rows behind it counts for nothing."""
    g = gen(70 + N)
    K = 100
    codes, s = R.random_weight(g, N, K)
    s[N - 1, 1] = 127 + 20
    exact = R.decode(codes, s, K)
    w = T.FrozenWeight(codes.cuda(), T.W_MXFP4, s.cuda(), N, K, 1, 32)
    x = torch.randn(M, N, generator=g).half()
    y = T.qlinear_backward_input(x.cuda(), w, T.F16, T.F32).cpu()
    used = exact.half().double()
    want = x.double() @ used
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.isinf(), want.isinf()) and bool((y[want.isinf()] == want[want.isinf()]).all())
    ok = want.isfinite().all(dim=0)
    assert bool((~ok).any())
    within(y[:, ok].contiguous(), want[:, ok], x.double().abs() @ used[:, ok].abs(), N)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 4, 5, 30])
@pytest.mark.parametrize("length", [1, 7, 8, 9, 15, 31, 129, 130, 135, 257, 511, 513, 1027])
def test_rows_of_any_length(length, M, dtype):
    """Rows of activations are read eight elements at a time, also where they end in between: what lies beside them counts for nothing."""
    g = gen(90 + length)
    t = DTYPES[dtype]
    c = T.CODE_OF[t]
    other = 40
    x = torch.randn(M, length, generator=g).to(t)
    beside = torch.full((M * length + 40,), float("nan"), dtype=t, device="cuda")
    beside[9:9 + M * length] = x.view(-1).cuda()
    x, used = x.double(), beside[9:9 + M * length].view(M, length)
    for backward in (False, True):
        w, exact = weight(g, *((length, other) if backward else (other, length)))
        m = exact if backward else exact.T
        y = (T.qlinear_backward_input if backward else T.qlinear_forward)(used, w, c, c)
        within(y, x @ m, x.abs() @ m.abs(), length, 3 if dtype == "f32" else 1)
    if dtype == "f32":
        return
    # the gated block over two stored weights: rows of either length are copied where eight elements do not fill them
    kind = T.W_F16 if dtype == "f16" else T.W_BF16
    a, b = (torch.randn(other, length, generator=g).to(t) for _ in range(2))
    _, gate, up = T.gated_forward(used, *(T.FrozenWeight(v.cuda(), kind, None, other, length) for v in (a, b)), keep=True)
    for got, v in ((gate, a.double()), (up, b.double())):
        within(got, x @ v.T, x.abs() @ v.abs().T, length)


# ------------------------------------------------------------------ steps of a tile shared by workgroups, a last round of half tiles
def on_device(codes, scales, cols):
    """fp64 on the device, where the large products of the tests below are fast enough"""
    return R.decode(codes.cuda(), scales.cuda(), cols)


@pytest.mark.parametrize("yd", DTYPES)
@pytest.mark.parametrize("M,N,K", [(256, 512, 8192), (200, 300, 8100), (130, 1000, 4128), (1500, 11000, 96), (1530, 10999, 257)])
def test_matmul_tiles(M, N, K, yd):
    g = gen(M + N + K)
    a, sa = R.random_weight(g, M, K)
    b, sb = R.random_weight(g, N, K, low=110, high=130)
    y = T.mxfp4_matmul(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), T.CODE_OF[DTYPES[yd]])
    p, q = on_device(a, sa, K), on_device(b, sb, K)
    within(y, (p @ q.T).cpu(), (p.abs() @ q.abs().T).cpu(), K)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1100, 4096, 264), (1030, 2000, 70), (1025, 4100, 131)])
def test_gradient_in_parts(M, N, K, dtype):
    g = gen(M + N + K)
    codes, s = R.random_weight(g, N, K)
    w, exact = T.FrozenWeight(codes.cuda(), T.W_MXFP4, s.cuda(), N, K, 1, 32), on_device(codes, s, K)
    dt = DTYPES[dtype]
    code = T.CODE_OF[dt]
    dy = torch.randn(M, N, generator=g).to(dt).cuda()
    dx = T.qlinear_backward_input(dy, w, code, code)
    within(dx, (dy.double() @ exact).cpu(), (dy.double().abs() @ exact.abs()).cpu(), N, 3 if dtype == "f32" else 1)
    add = torch.randn(M, K, generator=g).to(dt).cuda()
    assert torch.equal(T.qlinear_backward_input(dy, w, code, code, addend=add), (dx.float() + add.float()).to(dt))
    assert torch.equal(T.qlinear_backward_input(dy, w, code, code), dx)


def test_calls_on_two_streams():
    """Calls that run at the same time, over the same weight, on two streams keep their results; so do two graphs replayed in turn."""
    g = gen(120)
    N, K = 1030, 520
    w, _ = weight(g, N, K)
    cases = [(M, dt) for M in (1, 30, 200, 1100) for dt in (torch.bfloat16, torch.float32)]
    x = [torch.randn(M, K, generator=g).to(dt).cuda() for M, dt in cases]
    d = [torch.randn(M, N, generator=g).to(dt).cuda() for M, dt in cases]
    a = T.mxfp4_quantize(x[6])

    def step(i):
        c = T.CODE_OF[x[i].dtype]
        return T.qlinear_forward(x[i], w, c, c), T.qlinear_backward_input(d[i], w, c, c), T.gated_forward(x[i], w, w), T.mxfp4_matmul(*a, w.wq, w.scales)
    want = [step(i) for i in range(len(cases))]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for i in range(len(cases)):
            with torch.cuda.stream(streams[i % 2]):
                got.append((i, step(i)))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for i, results in got for p, q in zip(results, want[i]))
    graphs = []
    for i in (2, 5, 6):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, i, step(i)))
    for _ in range(3):
        for graph, i, results in graphs:
            for r in results:
                r.zero_()
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for _, i, results in graphs for p, q in zip(results, want[i]))
