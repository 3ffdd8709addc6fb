"""How many adapters each direction takes: the backward has workgroups for every adapter's gradients, the forward none.  Nothing is launched
(the workspace is too small), so this runs without a GPU."""
import pytest

from caif_amd import capi, torch_ops as T
from test_adapters_refusals import SMALL, UNSUPPORTED, backward, forward

MANY = 2 ** 20


@pytest.mark.parametrize("sizes", [dict(N=1024, K=64), dict(N=64, K=1024)])
def test_only_the_backward_is_limited_by_the_number_of_adapters(sizes):
    case = dict(M=5000, L=MANY, bytes=15, dtype=T.BF16, **sizes)
    assert forward(**case) == SMALL and backward(**case) == UNSUPPORTED
    shape = (5000, case["N"], case["K"], 4, MANY, T.BF16)
    assert capi.lib().caifx_adapters_workspace_bytes(*shape, 0) > 0 and capi.lib().caifx_adapters_workspace_bytes(*shape, 1) == 0


@pytest.mark.parametrize("M", [1, 5000, 2 ** 20, 2 ** 23])
@pytest.mark.parametrize("C", [1, 128, 129, 1024])
def test_what_the_backward_always_takes(M, C):
    most = (2 ** 22 - 2 ** 18) // -(-C // 128)
    for sizes in (dict(N=C, K=1), dict(N=1, K=C)):
        assert backward(M=M, L=most, bytes=15, **sizes) == SMALL
        assert backward(M=M, L=2 ** 22 // -(-C // 128) + 1, bytes=15, **sizes) == UNSUPPORTED
