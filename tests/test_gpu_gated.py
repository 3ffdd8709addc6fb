"""The gated feed-forward block on the GPU against its formulas in 64 bits, and against differences."""
import pytest
import torch

from caif_amd import capi, torch_ops as T
import mxfp4_reference as R

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KINDS = [("mx", "bf16"), ("mx", "f16"), ("mx", "f32"), ("same", "bf16"), ("same", "f16")]
SHAPES = [(1, 1, 1), (1, 700, 256), (2, 33, 70), (8, 64, 512), (16, 100, 136), (17, 257, 320), (32, 96, 1001), (33, 72, 256), (65, 130, 2048), (130, 264, 328),
          (257, 300, 776), (520, 136, 1000), (700, 333, 512), (1100, 640, 257), (3, 48, 544), (12, 40, 1185)]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def weight(g, kind, dtype, n, k):
    if kind == "mx":
        codes, s = R.random_weight(g, n, k)
        return T.FrozenWeight(codes.cuda(), T.W_MXFP4, s.cuda(), n, k, 1, 32), R.decode(codes, s, k)
    w = (0.05 * torch.randn(n, k, generator=g)).to(dtype)
    return T.FrozenWeight(w.cuda(), T.W_F16 if dtype == torch.float16 else T.W_BF16, None, n, k), w.double()


def check(got, want, most):
    off = (got.double().cpu() - want).abs()
    ok = bool((off <= most).all())
    assert ok, f"{float((off / most).max())} times the bound"


def sums(length, pieces):
    return (pieces * (length / 32 + 1) + 48) * 2.0 ** -23


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("kind,dtype", KINDS)
def test_forward(M, N, K, kind, dtype):
    g = gen(M + N + K)
    dt, pieces = DTYPES[dtype], 3 if dtype == "f32" else 1
    (wg, eg), (wu, eu) = weight(g, kind, dt, N, K), weight(g, kind, dt, N, K)
    x = torch.randn(M, K, generator=g).to(dt)
    hidden, gate, up = T.gated_forward(x.cuda(), wg, wu, keep=True)
    a, b = x.double() @ eg.T, x.double() @ eu.T
    sa, sb = x.double().abs() @ eg.abs().T, x.double().abs() @ eu.abs().T
    check(gate, a, R.bound(a, sa, K, dt, pieces))
    check(up, b, R.bound(b, sb, K, dt, pieces))
    # silu's slope is at most 1.1; its exponential, inverse and three products are within 8 roundings of 32 bits
    da, db = sums(K, pieces) * sa, sums(K, pieces) * sb
    want = R.silu(a) * b
    top = torch.finfo(dt)
    check(hidden, want, 1.1 * da * (b.abs() + db) + R.silu(a).abs() * db + (8 * 2.0 ** -24 + top.eps / 2) * want.abs() + top.smallest_normal * top.eps)
    assert torch.equal(T.gated_forward(x.cuda(), wg, wu), hidden)


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("kind,dtype", KINDS)
def test_backward(M, N, K, kind, dtype):
    g = gen(M + N + K + 7)
    dt, pieces = DTYPES[dtype], 3 if dtype == "f32" else 1
    (wg, eg), (wu, eu) = weight(g, kind, dt, N, K), weight(g, kind, dt, N, K)
    d, a, b = (torch.randn(M, N, generator=g).to(dt) for _ in range(3))
    dx, da, db = T.gated_backward(d.cuda(), a.cuda(), b.cuda(), wg, wu)
    want_a, want_b = R.gating_backward(d.double(), a.double(), b.double())
    top = torch.finfo(dt)
    # s (1 + g (1 - s)) passes through zero near g = -1.28: 1 + g (1 - s) is off by some roundings of 1 + |g| there
    spread = (d.double() * b.double()).abs() * torch.sigmoid(a.double()) * (1 + a.double().abs())
    check(da, want_a, 12 * 2.0 ** -24 * spread + top.eps / 2 * want_a.abs() + top.smallest_normal * top.eps)
    check(db, want_b, (8 * 2.0 ** -24 + top.eps / 2) * want_b.abs() + top.smallest_normal * top.eps)
    # the product takes the gradients as they are returned
    p, q = da.double().cpu(), db.double().cpu()
    want = p @ eg + q @ eu
    check(dx, want, R.bound(want, p.abs() @ eg.abs() + q.abs() @ eu.abs(), 2 * N, dt, pieces))
    none, ga, gb = T.gated_backward(d.cuda(), a.cuda(), b.cuda(), wg, wu, need_dx=False)
    assert none is None and torch.equal(ga, da) and torch.equal(gb, db)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_infinite_weights_stay_in_their_columns(dtype):
    """An infinity in a stored weight's last row, and one in its last column, reach only what their products reach."""
    g = gen(2)
    dt = DTYPES[dtype]
    for M, N, K in ((3, 33, 40), (20, 41, 100), (100, 70, 130), (300, 70, 264)):
        w = (0.05 * torch.randn(N, K, generator=g)).to(dt)
        w[N - 1, 2], w[4, K - 1] = float("inf"), float("-inf")
        fw = T.FrozenWeight(w.cuda(), T.W_F16 if dt == torch.float16 else T.W_BF16, None, N, K)
        d, a, b = (1 + torch.rand(M, N, generator=g).to(dt) for _ in range(3))
        dx, da, db = T.gated_backward(d.cuda(), a.cuda(), b.cuda(), fw, fw)
        want = (da.double().cpu() + db.double().cpu()) @ w.double()
        assert torch.equal(dx.isfinite().cpu(), want.isfinite()) and torch.equal(dx.isnan().cpu(), want.isnan())
        x = 1 + torch.rand(M, K, generator=g).to(dt)
        _, gate, up = T.gated_forward(x.cuda(), fw, fw, keep=True)
        want = x.double() @ w.double().T
        assert torch.equal(gate.isinf().cpu(), want.isinf()) and torch.equal(up.isnan().cpu(), want.isnan())


def test_against_differences():
    g = gen(3)
    M, N, K = 3, 40, 33
    (wg, eg), (wu, eu) = weight(g, "mx", torch.float32, N, K), weight(g, "mx", torch.float32, N, K)
    x, c = torch.randn(M, K, generator=g), torch.randn(M, N, generator=g)
    _, gate, up = T.gated_forward(x.cuda(), wg, wu, keep=True)
    dx, _, _ = T.gated_backward(c.cuda(), gate, up, wg, wu)

    def loss(v):
        return float((c.double() * R.silu(v @ eg.T) * (v @ eu.T)).sum())
    h = 2.0 ** -13
    for m in range(M):
        for k in range(0, K, 4):
            e = torch.zeros(M, K, dtype=torch.float64)
            e[m, k] = h
            slope = (loss(x.double() + e) - loss(x.double() - e)) / (2 * h)
            # the third derivative adds some h^2, the kernels' fp32 sums some 2^-20 of the terms
            assert abs(slope - float(dx[m, k])) <= 1e-4 * max(1.0, abs(slope))


def test_far_gates_and_infinities():
    """Gates far from zero keep finite gradients; an infinity or NaN of one row stays there."""
    g = gen(4)
    M, N, K = 40, 64, 96
    (wg, _), (wu, _) = weight(g, "mx", torch.bfloat16, N, K), weight(g, "mx", torch.bfloat16, N, K)
    gate = torch.full((M, N), -95.0)
    gate[1], gate[2], gate[3] = 95.0, -1e30, 1e30
    up, d = torch.full((M, N), 2.0), torch.full((M, N), 2.0 ** 100)
    for dtype in (torch.float32, torch.bfloat16):
        _, da, db = T.gated_backward(d.to(dtype).cuda(), gate.to(dtype).cuda(), up.to(dtype).cuda(), wg, wu)
        want_a, want_b = R.gating_backward(d.double(), gate.to(dtype).double(), up.double())
        top = torch.finfo(dtype)
        for got, want in ((da, want_a), (db, want_b)):
            finite = want.abs() < 1e38
            assert bool(((got.double().cpu() - want).abs() <= (top.eps + 2.0 ** -18) * want.abs() + 2.0 ** -40)[finite].all())
    x = torch.randn(M, K, generator=g).to(torch.bfloat16).cuda()
    clean = T.gated_forward(x, wg, wu)
    x[5, 3], x[7, 9] = float("nan"), float("inf")
    y = T.gated_forward(x, wg, wu)
    rows = [m for m in range(M) if m not in (5, 7)]
    assert torch.equal(y[rows], clean[rows]) and bool(y[5].isnan().all()) and not bool(y[7].isfinite().all())


@pytest.mark.parametrize("kind", ["mx", "same"])
@pytest.mark.parametrize("M", [3, 50, 520])
def test_stream_and_graph(M, kind):
    g = gen(60 + M)
    N, K = 264, 512
    (wg, _), (wu, _) = weight(g, kind, torch.bfloat16, N, K), weight(g, kind, torch.bfloat16, N, K)
    x = torch.randn(M, K, generator=g).to(torch.bfloat16).cuda()
    d = torch.randn(M, N, generator=g).to(torch.bfloat16).cuda()

    def step():
        hidden, gate, up = T.gated_forward(x, wg, wu, keep=True)
        return (hidden, *T.gated_backward(d, gate, up, wg, wu))
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
        d.copy_(torch.randn(M, N, generator=g).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(kept, step()))


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("M,N,K", [(3, 50, 72), (40, 33, 70), (300, 264, 512)])
def test_odd_addresses_and_bytes_beside(M, N, K, kind, dtype):
    """Activations and results at any address of their type; nothing written beside the results and the workspace."""
    g = gen(70 + M)
    dt = DTYPES[dtype]
    (wg, _), (wu, _) = weight(g, kind, dt, N, K), weight(g, kind, dt, N, K)
    L, s = capi.lib(), torch.cuda.current_stream().cuda_stream
    code = T.CODE_OF[dt]

    def odd(rows, cols, values=None):
        t = torch.full((rows * cols + 34,), 3.0, dtype=dt, device="cuda")
        if values is not None:
            t[1:1 + rows * cols] = values.reshape(-1)
        return t
    x, d = torch.randn(M, K, generator=g).to(dt).cuda(), torch.randn(M, N, generator=g).to(dt).cuda()
    hidden, gate, up = T.gated_forward(x, wg, wu, keep=True)
    dx, da, db = T.gated_backward(d, gate, up, wg, wu)

    def at(t):
        return t[1:].data_ptr()

    def scales(w):
        return w.scales.data_ptr() if kind == "mx" else None

    def room(backward):
        need = L.caifx_gated_workspace_bytes(M, N, K, wg.w_kind, code, backward)
        return need, torch.full((need + 64,), 201, dtype=torch.uint8, device="cuda")
    xs, outs = odd(M, K, x), [odd(M, N) for _ in range(3)]
    need, ws = room(0)
    assert L.caifx_gated_forward(M, N, K, at(xs), wg.wq.data_ptr(), scales(wg), wu.wq.data_ptr(), scales(wu), wg.w_kind, *(at(o) for o in outs), code, ws.data_ptr(), need, s) == 0
    ins, back = [odd(M, N, t) for t in (d, gate, up)], [odd(M, N), odd(M, N), odd(M, K)]
    need2, ws2 = room(1)
    assert L.caifx_gated_backward(M, N, K, *(at(t) for t in ins), wg.wq.data_ptr(), scales(wg), wu.wq.data_ptr(), scales(wu), wg.w_kind, *(at(o) for o in back), code,
                                  ws2.data_ptr(), need2, s) == 0
    torch.cuda.synchronize()
    assert bool((ws[need:] == 201).all()) and bool((ws2[need2:] == 201).all())
    top = torch.finfo(dt)
    for got, want in zip(outs + back, (hidden, gate, up, da, db, dx)):
        n = want.numel()
        assert bool((got[:1] == 3).all()) and bool((got[1 + n:] == 3).all())
        # (another kernel may take it there: the sums in another order)
        off = (got[1:1 + n].float() - want.reshape(-1).float()).abs()
        assert bool((off <= 2 * top.eps * want.reshape(-1).float().abs() + 2.0 ** -12 * want.float().abs().max()).all())


def test_empty():
    w = T.FrozenWeight(torch.zeros(8, 48, dtype=torch.uint8, device="cuda"), T.W_MXFP4, torch.zeros(8, 3, dtype=torch.uint8, device="cuda"), 8, 70, 1, 32)
    none = torch.empty(0, 70, dtype=torch.bfloat16, device="cuda")
    assert T.gated_forward(none, w, w).shape == (0, 8) and T.qlinear_forward(none, w, T.BF16).shape == (0, 8)
    grad = torch.empty(0, 8, dtype=torch.bfloat16, device="cuda")
    assert T.gated_backward(grad, grad, grad, w, w)[0].shape == (0, 70)


def test_a_block_as_it_is_trained():
    """A frozen block in 4 bits: forward with kept projections, down projection, loss gradient back through both, against 64 bits."""
    g = gen(80)
    M, dim, wide = 96, 256, 520
    dt = torch.bfloat16
    (wg, eg), (wu, eu), (wd, ed) = (weight(g, "mx", dt, n, k) for n, k in ((wide, dim), (wide, dim), (dim, wide)))
    x, c = torch.randn(M, dim, generator=g).to(dt), torch.randn(M, dim, generator=g).to(dt)
    hidden, gate, up = T.gated_forward(x.cuda(), wg, wu, keep=True)
    y = T.qlinear_forward(hidden, wd, T.BF16, T.BF16)
    dh = T.qlinear_backward_input(c.cuda(), wd, T.BF16, T.BF16)
    dx, da, db = T.gated_backward(dh, gate, up, wg, wu)
    v = x.double().requires_grad_()
    h = R.silu(v @ eg.T) * (v @ eu.T)
    out = h @ ed.T
    out.backward(c.double())
    # five roundings to 8 bits on the way, each at most 2^-9 of its tensor's 2-norm in the mean of many values
    for got, want in ((y, out.detach()), (dx, v.grad)):
        assert float((got.double().cpu() - want).norm() / want.norm()) < 5 * 2.0 ** -8
