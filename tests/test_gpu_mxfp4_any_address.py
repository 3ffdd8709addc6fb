"""Large products with activations at any address of their type: the same kernels, and so the same bits, as at a multiple of 16 bytes."""
import pytest
import torch

from caif_amd import capi, torch_ops as T
import mxfp4_reference as R

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SHAPES = [(700, 1024, 512), (1100, 640, 1000), (1030, 2003, 1403)]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def odd(t, by=1):
    """The same values at an address `by` elements past a multiple of 256 bytes."""
    room = torch.empty(t.numel() + by, dtype=t.dtype, device=t.device)
    room[by:] = t.reshape(-1)
    return room[by:].view(t.shape)


def weight(g, n, k):
    codes, s = R.random_weight(g, n, k, device="cuda")
    return T.FrozenWeight(codes, T.W_MXFP4, s, n, k, 1, 32)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("xd,cd", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f16", "f32"), ("bf16", "f32")])
def test_linear(M, N, K, xd, cd, backward):
    g = gen(M + N + K)
    w = weight(g, N, K)
    x = torch.randn(M, N if backward else K, generator=g).to(DTYPES[xd]).cuda()
    call = T.qlinear_backward_input if backward else T.qlinear_forward
    code = T.CODE_OF[DTYPES[cd]]
    want = call(x, w, code, T.F32)
    for by in (1, 3):
        assert torch.equal(call(odd(x, by), w, code, T.F32), want)


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("kind,dtype", [("mx", "bf16"), ("mx", "f32"), ("same", "f16")])
def test_gated(M, N, K, kind, dtype):
    g = gen(M + N + K + 1)
    dt = DTYPES[dtype]
    if kind == "mx":
        wg, wu = weight(g, N, K), weight(g, N, K)
    else:
        wg, wu = (T.FrozenWeight((0.05 * torch.randn(N, K, generator=g)).to(dt).cuda(), T.W_F16, None, N, K) for _ in range(2))
    x = torch.randn(M, K, generator=g).to(dt).cuda()
    want = T.gated_forward(x, wg, wu, keep=True)
    assert all(torch.equal(p, q) for p, q in zip(T.gated_forward(odd(x), wg, wu, keep=True), want))
    # the gradients are the caller's buffers: either of them may begin anywhere
    L, s = capi.lib(), torch.cuda.current_stream().cuda_stream
    code = T.CODE_OF[dt]
    d = torch.randn(M, N, generator=g).to(dt).cuda()
    want = T.gated_backward(d, want[1], want[2], wg, wu)
    gate, up = T.gated_forward(x, wg, wu, keep=True)[1:]
    need = L.caifx_gated_workspace_bytes(M, N, K, wg.w_kind, code, 1)

    def scales(w):
        return w.scales.data_ptr() if kind == "mx" else None
    for at in ((0, 1), (1, 0), (3, 1)):
        grads = [odd(torch.zeros(M, N, dtype=dt, device="cuda"), by) for by in at]
        dx = torch.empty(M, K, dtype=dt, device="cuda")
        ws = torch.full((need + 64,), 201, dtype=torch.uint8, device="cuda")
        assert L.caifx_gated_backward(M, N, K, d.data_ptr(), gate.data_ptr(), up.data_ptr(), wg.wq.data_ptr(), scales(wg), wu.wq.data_ptr(), scales(wu), wg.w_kind,
                                      grads[0].data_ptr(), grads[1].data_ptr(), dx.data_ptr(), code, ws.data_ptr(), need, s) == 0
        torch.cuda.synchronize()
        assert bool((ws[need:] == 201).all())
        assert all(torch.equal(p, q) for p, q in zip((dx, *grads), want))
