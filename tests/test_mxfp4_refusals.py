"""What the 4-bit and gated calls refuse: through the C ABI by status, through the torch calls by exception.  Nothing is launched, so this runs
without a GPU."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from caif_amd import capi, torch_ops as T

OK, INVALID, UNSUPPORTED, SMALL, MISALIGNED = 0, 1, 2, 3, 5
AT = 1 << 20          # an address that is never used
ELSE = 1 << 21
BIG = 1 << 40


def pack(name="caifx_mxfp4_quantize", **over):
    v = dict(first=AT, second=AT + 4096, third=AT + 8192, rows=4, cols=70, dtype=T.BF16)
    v.update(over)
    return getattr(capi.lib(), name)(*v.values(), None)


def matmul(**over):
    v = dict(M=4, N=8, K=70, a=AT, sa=AT, b=AT, sb=AT, y=ELSE, dtype=T.BF16, ws=AT, bytes=BIG)
    v.update(over)
    return capi.lib().caifx_mxfp4_matmul(*v.values(), None)


def forward(**over):
    v = dict(M=4, N=8, K=70, x=AT, wg=AT, sg=AT, wu=AT, su=AT, kind=T.W_MXFP4, hidden=ELSE, gate=ELSE + 4096, up=ELSE + 8192, dtype=T.BF16, ws=AT, bytes=BIG)
    v.update(over)
    return capi.lib().caifx_gated_forward(*v.values(), None)


def backward(**over):
    v = dict(M=4, N=8, K=70, d=AT, gate=AT, up=AT, wg=AT, sg=AT, wu=AT, su=AT, kind=T.W_MXFP4, gg=ELSE, gu=ELSE + 4096, dx=ELSE + 8192, dtype=T.BF16,
             ws=AT, bytes=BIG)
    v.update(over)
    return capi.lib().caifx_gated_backward(*v.values(), None)


@pytest.mark.parametrize("name", ["caifx_mxfp4_quantize", "caifx_mxfp4_dequantize"])
def test_packing(name):
    def call(**over):
        return pack(name, **over)
    assert call(rows=0) == OK and call(cols=0) == OK and call(rows=0, first=None) == OK
    assert call(rows=-1) == INVALID and call(cols=-1) == INVALID and call(dtype=3) == INVALID and call(dtype=-1) == INVALID
    assert all(call(**{k: None}) == INVALID for k in ("first", "second", "third"))
    plain, codes = ("first", "second") if "dequantize" not in name else ("third", "first")
    assert call(**{plain: AT + 1}) == MISALIGNED and call(**{plain: AT + 2}, dtype=T.F32) == MISALIGNED and call(**{codes: AT + 8}) == MISALIGNED
    assert call(rows=2 ** 30) == UNSUPPORTED and call(rows=1, cols=2 ** 50) == UNSUPPORTED and call(rows=2 ** 20, cols=2 ** 20) == UNSUPPORTED
    assert call(rows=2 ** 62, cols=2 ** 62) == UNSUPPORTED


@pytest.mark.parametrize("call", [matmul, forward, backward])
@pytest.mark.parametrize("over,status", [
    (dict(M=-1), INVALID), (dict(N=-1), INVALID), (dict(K=0), INVALID), (dict(K=-3), INVALID), (dict(dtype=3), INVALID), (dict(dtype=-1), INVALID),
    (dict(M=2 ** 31), UNSUPPORTED), (dict(N=2 ** 31), UNSUPPORTED), (dict(K=2 ** 31), UNSUPPORTED), (dict(ws=AT + 1), MISALIGNED), (dict(M=0), OK)])
def test_sizes(call, over, status):
    assert call(**over) == status


def test_matmul():
    assert all(matmul(**{k: None}) == INVALID for k in ("a", "sa", "b", "sb", "y"))
    assert matmul(a=AT + 8) == MISALIGNED and matmul(b=AT + 4) == MISALIGNED and matmul(y=ELSE + 1) == MISALIGNED and matmul(N=0) == OK
    need = capi.lib().caifx_mxfp4_matmul_workspace_bytes(4, 8, 70)
    if need:
        assert matmul(ws=None, bytes=need) == SMALL and matmul(bytes=need - 1) == SMALL
    assert capi.lib().caifx_mxfp4_matmul_workspace_bytes(0, 8, 70) == 0 and capi.lib().caifx_mxfp4_matmul_workspace_bytes(4, 8, -1) == 0


def test_gated_forward():
    assert all(forward(**{k: None}) == INVALID for k in ("x", "wg", "wu", "hidden", "sg", "su", "gate", "up"))
    assert all(forward(**{k: AT + 1}) == MISALIGNED for k in ("x", "hidden", "gate", "up"))
    assert forward(wg=AT + 8) == MISALIGNED and forward(wu=AT + 2) == MISALIGNED and forward(x=AT + 2, dtype=T.F32) == MISALIGNED
    assert forward(hidden=AT) == INVALID and forward(gate=ELSE) == INVALID and forward(up=ELSE + 4096) == INVALID
    need = capi.lib().caifx_gated_workspace_bytes(40, 8, 70, T.W_MXFP4, T.F32, 0)
    assert need > 0 and forward(M=40, dtype=T.F32, ws=None, bytes=need) == SMALL and forward(M=40, dtype=T.F32, bytes=need - 1) == SMALL


def test_gated_backward():
    assert all(backward(**{k: None}) == INVALID for k in ("d", "gate", "up", "wg", "wu", "sg", "su", "gg", "gu"))
    assert all(backward(**{k: AT + 1}) == MISALIGNED for k in ("d", "gate", "up", "gg", "gu", "dx"))
    assert backward(wg=AT + 8) == MISALIGNED and backward(gg=AT) == INVALID and backward(gu=ELSE) == INVALID and backward(dx=ELSE) == INVALID
    need = capi.lib().caifx_gated_workspace_bytes(4, 300, 70, T.W_MXFP4, T.BF16, 1)
    assert need > 0 and backward(N=300, ws=None, bytes=need) == SMALL and backward(N=300, bytes=need - 1) == SMALL


@pytest.mark.parametrize("kind,dtype,status", [
    (T.W_INT8, T.BF16, UNSUPPORTED), (T.W_INT4_GROUP, T.F16, UNSUPPORTED), (T.W_F32, T.F32, UNSUPPORTED), (T.W_F16, T.BF16, UNSUPPORTED),
    (T.W_BF16, T.F16, UNSUPPORTED), (T.W_BF16, T.F32, UNSUPPORTED), (5, T.BF16, INVALID), (7, T.BF16, INVALID), (-1, T.BF16, INVALID)])
def test_gated_kinds(kind, dtype, status):
    assert forward(kind=kind, dtype=dtype) == status and backward(kind=kind, dtype=dtype) == status
    assert capi.lib().caifx_gated_workspace_bytes(4, 8, 70, kind, dtype, 0) == 0


def test_linear_calls():
    L = capi.lib()

    def linear(name="caifx_qlinear_forward", wq=AT, scales=AT, addend=None):
        more = [addend] if "add" in name else []
        return getattr(L, name)(4, 8, 70, AT, T.BF16, T.BF16, wq, T.W_MXFP4, scales, 1, 32, ELSE, T.BF16, *more, None, 0, None)
    for name in ("caifx_qlinear_forward", "caifx_qlinear_backward_input"):
        assert linear(name, scales=None) == INVALID and linear(name, wq=None) == INVALID and linear(name, wq=AT + 8) == MISALIGNED
        assert linear(name + "_add", addend=None) == INVALID
    at = [2, AT, 4, 8, 70, AT, T.BF16, T.BF16, AT, T.W_MXFP4, AT, 1, 32, ELSE, T.BF16]
    assert L.caifx_qlinear_grouped_forward(*at, None, 0, None) == UNSUPPORTED and L.caifx_qlinear_grouped_backward_input(*at, None, 0, None) == UNSUPPORTED
    assert L.caifx_qlinear_grouped_fresh(0, *at, None, None, 0, None) == UNSUPPORTED
    assert L.caifx_qlinear_grouped_forward_swiglu(*at[:13], AT, ELSE, ELSE + 4096, T.BF16, None) == UNSUPPORTED


def test_torch_calls():
    cpu = torch.zeros(4, 64)
    with pytest.raises(RuntimeError, match="host backend"):
        T.mxfp4_quantize(cpu)
    with pytest.raises(KeyError):
        T.mxfp4_dequantize(cpu, cpu, 64, torch.int8)
    with FakeTensorMode():
        def u8(*shape):
            return torch.empty(shape, dtype=torch.uint8, device="cuda")

        def b16(*shape):
            return torch.empty(shape, dtype=torch.bfloat16, device="cuda")

        def weight(n=8, k=70, **over):
            v = dict(wq=u8(n, 16 * -(-k // 32)), scales=u8(n, -(-k // 32)))
            v.update(over)
            return T.FrozenWeight(v["wq"], T.W_MXFP4, v["scales"], n, k, 1, 32)
        with pytest.raises(RuntimeError, match="contiguous"):
            T.mxfp4_quantize(b16(64, 4).T)
        with pytest.raises(KeyError):
            T.mxfp4_quantize(u8(4, 64))
        with pytest.raises(ValueError):
            T.mxfp4_quantize(b16())
        for codes, scales, cols in ((u8(4, 32), u8(4, 2), 65), (u8(4, 32), u8(4, 2), 32), (u8(4, 32), u8(4, 3), 64), (b16(4, 32), u8(4, 2), 64), (u8(8, 16), u8(4, 2), 64)):
            with pytest.raises(ValueError):
                T.mxfp4_dequantize(codes, scales, cols, torch.float32)
        with pytest.raises(ValueError, match="one length"):
            T.mxfp4_matmul(u8(4, 32), u8(4, 2), u8(8, 48), u8(8, 3))
        with pytest.raises(ValueError, match="M x N"):
            T.mxfp4_matmul(u8(4, 32), u8(4, 2), u8(8, 32), u8(8, 2), T.BF16, out=b16(4, 9))
        for w in (weight(wq=u8(8, 47)), weight(scales=u8(8, 2)), weight(wq=b16(8, 48))):
            for call in (lambda: T.qlinear_forward(b16(4, 70), w, T.BF16), lambda: T.qlinear_backward_input(b16(4, 8), w, T.BF16),
                         lambda: T.gated_forward(b16(4, 70), w, w), lambda: T.gated_backward(b16(4, 8), b16(4, 8), b16(4, 8), w, w)):
                with pytest.raises(ValueError, match="W_MXFP4"):
                    call()
        w = weight()
        with pytest.raises(ValueError, match="multiple"):
            T.qlinear_forward(b16(4, 69), w, T.BF16)
        with pytest.raises(ValueError, match="addend"):
            T.qlinear_forward(b16(4, 70), w, T.BF16, T.BF16, addend=b16(4, 9))
        with pytest.raises(ValueError, match="addend"):
            T.qlinear_forward(b16(4, 70), w, T.BF16, T.F32, out=b16(4, 8))
        with pytest.raises(ValueError, match="row of activations"):
            T.gated_forward(b16(4, 71), w, w)
        with pytest.raises(ValueError, match="one shape"):
            T.gated_forward(b16(4, 70), w, weight(n=9))
        with pytest.raises(ValueError, match="gate and up"):
            T.gated_backward(b16(4, 8), b16(4, 7), b16(4, 8), w, w)
        with pytest.raises(ValueError, match="N x K"):
            T.gated_forward(b16(4, 70), T.FrozenWeight(b16(8, 69), T.W_BF16, None, 8, 70), T.FrozenWeight(b16(8, 70), T.W_BF16, None, 8, 70))
