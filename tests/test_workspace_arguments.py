"""A workspace tensor that the kernels cannot write is refused before anything is launched, so this runs without a GPU."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from caif_amd import torch_ops as T


def weight(kind, n=8, k=128):
    def u8(*shape):
        return torch.empty(shape, dtype=torch.uint8, device="cuda")
    if kind == T.W_MXFP4:
        return T.FrozenWeight(u8(n, k // 2), kind, u8(n, k // 32), n, k, 1, 32)
    if kind == T.W_INT4_GROUP:
        return T.FrozenWeight(u8(n * k // 2), kind, torch.empty(n * k // 128, dtype=torch.float16, device="cuda"), n, k, 1, 128)
    return T.FrozenWeight(torch.empty(n * k, dtype=torch.int8, device="cuda"), kind, torch.empty(n, device="cuda"), n, k, n)


@pytest.mark.parametrize("kind", [T.W_MXFP4, T.W_INT4_GROUP, T.W_INT8])
@pytest.mark.parametrize("backward", [False, True])
def test_host_memory_and_gaps(kind, backward):
    with FakeTensorMode():
        w, x = weight(kind), torch.empty(4, 8 if backward else 128, dtype=torch.bfloat16, device="cuda")
        call = T.qlinear_backward_input if backward else T.qlinear_forward
        for workspace in (torch.empty(1 << 16, dtype=torch.uint8), torch.empty(1, dtype=torch.uint8, device="cuda").expand(1 << 16)):
            with pytest.raises(ValueError, match="workspace"):
                call(x, w, T.BF16, workspace=workspace)
        with pytest.raises(ValueError, match="workspace"):
            call(x, w, T.BF16, workspace=torch.empty(1 << 16, dtype=torch.uint8, device="cuda:1"))


@pytest.mark.parametrize("backward", [False, True])
def test_expert_segments(backward):
    with FakeTensorMode():
        class Experts:
            weights = [weight(T.W_INT8), weight(T.W_INT8)]
            N, K, w_kind, scale_period, group_size = 8, 128, T.W_INT8, 8, 128
            wq_ptrs = torch.empty(2, dtype=torch.int64, device="cuda")
            scales_ptrs = torch.empty(2, dtype=torch.int64, device="cuda")
        x = torch.empty(4, 8 if backward else 128, dtype=torch.bfloat16, device="cuda")
        offsets = torch.empty(3, dtype=torch.int32, device="cuda")
        call = T.qlinear_grouped_backward_input if backward else T.qlinear_grouped_forward
        for workspace in (torch.empty(1 << 16, dtype=torch.uint8), torch.empty(1, dtype=torch.uint8, device="cuda").expand(1 << 16)):
            with pytest.raises(ValueError, match="workspace"):
                call(x, offsets, Experts, T.BF16, workspace=workspace)
