"""The gating's backward from checkpoints where 1 + exp(-gate) is beyond 2^126, an inverse below the normal numbers: the gradients are still normal
numbers.  exp(gate) itself is there with a step of 2^-149, at most 2^-19.8 / 2 of it down to a gate of -89.5; with the exponential's own two steps and
the products' roundings the results are within 2^-20 of themselves (silu' has no cancellation below -2)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from caif_amd import torch_ops as T                                             # noqa: E402
import adapter_reference as R                                                   # noqa: E402


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [128, 200])
def test_gates_far_below_zero(cols, dtype):
    gen = torch.Generator(device="cuda").manual_seed(cols)
    rows, groups = 300, -(-cols // 128)
    scales = (torch.linspace(80, 89.5, rows, device="cuda") / 127)[:, None].expand(rows, groups).contiguous()
    gate = torch.full((rows, cols), -127, dtype=torch.int8, device="cuda"), scales
    up = T.checkpoint_pack(torch.rand(rows, cols, device="cuda", generator=gen) + 1)
    grad = (torch.rand(rows, cols, device="cuda", generator=gen) + 1).to(dtype)
    grad_gate, grad_up, hidden = T.swiglu_backward_checkpoint(gate, up, grad, with_hidden=True)
    g, u = (R.unpacked(*(t.cpu() for t in ck)).float().double() for ck in (gate, up))
    d, s = grad.double().cpu(), torch.sigmoid(g)
    for name, got, want in (("grad_up", grad_up, d * g * s), ("grad_gate", grad_gate, d * u * s * (1 + g * (1 - s))), ("hidden", hidden, g * s * u)):
        assert (want.abs() > 2.0 ** -125).all()
        R.check(got, want, want.abs(), dtype, 2.0 ** -20, name)
