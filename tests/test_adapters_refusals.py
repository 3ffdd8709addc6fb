"""What the adapter and checkpoint calls refuse: through the C ABI by status, through the torch calls by exception.  Nothing is launched, so
this runs without a GPU."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from caif_amd import capi, torch_ops as T

OK, INVALID, UNSUPPORTED, SMALL, MISALIGNED = 0, 1, 2, 3, 5
AT = 1 << 20          # an address that is never used


def forward(**over):
    v = dict(M=4, N=8, K=16, rank=4, L=2, x=AT, ids=AT, a=AT, b=AT, scaling=AT, base=AT, y=AT, hidden=AT, dtype=T.BF16, ws=AT, bytes=1 << 20)
    v.update(over)
    return capi.lib().caifx_adapters_forward(*v.values(), None)


def backward(**over):
    v = dict(M=4, N=8, K=16, rank=4, L=2, dy=AT, x=AT, x_scales=None, hidden=AT, ids=AT, a=AT, b=AT, scaling=AT, base=AT, dx=AT, ga=AT, gb=AT,
             dtype=T.BF16, ws=AT, bytes=1 << 20)
    v.update(over)
    return capi.lib().caifx_adapters_backward(*v.values(), None)


@pytest.mark.parametrize("call", [forward, backward])
@pytest.mark.parametrize("over,status", [
    (dict(M=-1), INVALID), (dict(N=0), INVALID), (dict(K=0), INVALID), (dict(K=-5), INVALID), (dict(rank=0), INVALID), (dict(rank=-1), INVALID),
    (dict(L=0), INVALID), (dict(dtype=3), INVALID), (dict(dtype=-1), INVALID), (dict(rank=129), UNSUPPORTED), (dict(M=2 ** 30 + 1), UNSUPPORTED),
    (dict(N=2 ** 40), UNSUPPORTED), (dict(K=2 ** 31), UNSUPPORTED), (dict(x=None), INVALID), (dict(ids=None), INVALID), (dict(a=None), INVALID),
    (dict(b=None), INVALID), (dict(scaling=None), INVALID), (dict(x=AT + 1), MISALIGNED), (dict(ids=AT + 2), MISALIGNED), (dict(a=AT + 1), MISALIGNED),
    (dict(b=AT + 1), MISALIGNED), (dict(base=AT + 1), MISALIGNED), (dict(scaling=AT + 2), MISALIGNED), (dict(hidden=AT + 2), MISALIGNED),
    (dict(x=AT + 2, dtype=T.F32), MISALIGNED), (dict(ws=AT + 1), MISALIGNED), (dict(M=5000, ws=None), SMALL),
    (dict(M=5000, bytes=15), SMALL)])
def test_adapter_calls(call, over, status):
    assert call(**over) == status


def test_adapter_calls_by_direction():
    assert forward(y=None) == INVALID and forward(y=AT + 1) == MISALIGNED and forward(M=0) == OK
    assert backward(dy=None) == INVALID and backward(hidden=None) == INVALID
    assert all(backward(**{k: AT + 1}) == MISALIGNED for k in ("dy", "dx", "ga", "gb", "x_scales"))
    assert backward(dx=None, ga=None, gb=None) == OK and backward(M=0, ga=None, gb=None) == OK
    assert capi.lib().caifx_adapters_workspace_bytes(4, 8, 16, 0, 2, T.BF16, 0) == 0
    assert capi.lib().caifx_adapters_workspace_bytes(4, 8, 16, 200, 2, T.BF16, 1) == 0


def test_checkpoint_calls():
    L = capi.lib()
    for name, pointers, scales in (("caifx_checkpoint_pack", 3, (2,)), ("caifx_checkpoint_unpack", 3, (1,)), ("caifx_silu_multiply_checkpoint", 7, (4, 6)),
                                   ("caifx_swiglu_backward_checkpoint", 7, (1, 3))):
        def call(ptrs=None, rows=4, cols=200, dtype=T.BF16):
            ptrs = list(ptrs or [AT] * pointers)
            return getattr(L, name)(*ptrs, *([None] if "swiglu" in name else []), rows, cols, dtype, None)
        assert call(rows=0) == OK and call(cols=0) == OK
        assert call(rows=-1) == INVALID and call(cols=-1) == INVALID and call(dtype=7) == INVALID
        assert call(rows=2 ** 30, cols=2 ** 30) == UNSUPPORTED and call(rows=2 ** 31) == UNSUPPORTED and call(rows=1, cols=2 ** 40) == UNSUPPORTED
        for i in range(pointers):
            assert call([AT if j != i else None for j in range(pointers)]) == INVALID
        for i in scales:
            assert call([AT if j != i else AT + 2 for j in range(pointers)]) == MISALIGNED


@pytest.fixture
def fakes():
    with FakeTensorMode():
        yield lambda *s, dtype=torch.bfloat16: torch.empty(s, device="cuda", dtype=dtype)


def arguments(f):
    i32, f32 = torch.int32, torch.float32
    fwd = dict(x=f(4, 16), ids=f(4, dtype=i32), a=f(2, 3, 16), b=f(2, 8, 3), scaling=f(2, dtype=f32))
    bwd = dict(dy=f(4, 8), x=f(4, 16), hidden=f(4, 3, dtype=f32), **{k: fwd[k] for k in ("ids", "a", "b", "scaling")})
    return fwd, bwd


def test_shapes_and_types_are_checked(fakes):
    f = fakes
    fwd, bwd = arguments(f)
    i64, f32, i8 = torch.int64, torch.float32, torch.int8
    for over in (dict(x=f(4, 17)), dict(x=f(4, 16, dtype=f32)), dict(ids=f(5, dtype=torch.int32)), dict(ids=f(4, dtype=i64)), dict(a=f(3, 3, 16)),
                 dict(a=f(2, 4, 16)), dict(a=f(2, 48)), dict(b=f(2, 8, 4)), dict(b=f(2, 0, 3)), dict(scaling=f(3, dtype=f32)), dict(scaling=f(2)),
                 dict(base=f(4, 9)), dict(base=f(4, 8, dtype=f32)), dict(out=f(3, 8))):
        with pytest.raises(ValueError):
            T.adapters_forward(**{**fwd, **over})
    for over in (dict(dy=f(4, 9)), dict(x=f(4, 15)), dict(x=f(4, 16, dtype=i8)), dict(x=(f(4, 16), f(4, 1, dtype=f32))),
                 dict(x=(f(4, 16, dtype=i8), f(4, 2, dtype=f32))), dict(hidden=f(4, 4, dtype=f32)), dict(hidden=f(4, 3)), dict(base=f(4, 8))):
        with pytest.raises(ValueError):
            T.adapters_backward(**{**bwd, **over})
    with pytest.raises(KeyError):
        T.adapters_forward(**{**fwd, "x": f(4, 16, dtype=i64)})
    with pytest.raises(RuntimeError):
        T.adapters_forward(**{**fwd, "x": f(16, 4).T})
    for call in (lambda: T.checkpoint_unpack(f(4, 16), f(4, 1, dtype=f32), f32), lambda: T.checkpoint_unpack(f(4, 16, dtype=i8), f(4, 2, dtype=f32), f32),
                 lambda: T.checkpoint_unpack(f(4, 16, dtype=i8), f(4, 1), f32), lambda: T.silu_multiply_checkpoint(f(4, 16), f(16, 4)),
                 lambda: T.silu_multiply_checkpoint(f(4, 16), f(4, 16, dtype=f32)), lambda: T.checkpoint_pack(f()),
                 lambda: T.swiglu_backward_checkpoint((f(4, 16, dtype=i8), f(4, 1, dtype=f32)), (f(4, 16), f(4, 1, dtype=f32)), f(4, 16)),
                 lambda: T.swiglu_backward_checkpoint((f(4, 16, dtype=i8), f(4, 1, dtype=f32)), (f(16, 4, dtype=i8), f(4, 1, dtype=f32)), f(4, 16))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(KeyError):
        T.checkpoint_unpack(f(4, 16, dtype=i8), f(4, 1, dtype=f32), i64)
    with pytest.raises(KeyError):
        T.checkpoint_pack(f(4, 16, dtype=i8))


def test_host_tensors_and_tensors_without_memory_are_an_error(fakes):
    f = fakes
    fwd, bwd = arguments(f)
    host = torch.empty(4, 16, dtype=torch.bfloat16)
    for call in (lambda: T.adapters_forward(**fwd), lambda: T.adapters_backward(**bwd), lambda: T.checkpoint_pack(f(4, 16)),
                 lambda: T.silu_multiply_checkpoint(f(4, 16), f(4, 16)), lambda: T.adapters_forward(**{**fwd, "x": host}), lambda: T.checkpoint_pack(host)):
        with pytest.raises(RuntimeError):
            call()
