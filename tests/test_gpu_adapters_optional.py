"""Results of the adapters' backward that a caller leaves out, with every operand null that the others do not need."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from caif_amd import capi, torch_ops as T                                       # noqa: E402
from test_gpu_adapters import BF16, F16, F32, problem                           # noqa: E402


def backward(p, more, adapters, x, want, null):
    """caifx_adapters_backward for the results named in `want`; operands that `null` says true for are null."""
    (m, k), n, r, dtype = p["x"].shape, p["b"].shape[1], p["a"].shape[1], p["x"].dtype
    shape = {"dx": (m, k), "ga": (adapters, r, k), "gb": (adapters, n, r)}
    out = {name: torch.full(s, float("nan"), dtype=dtype, device="cuda") if name in want else None for name, s in shape.items()}
    codes, scales = x if isinstance(x, tuple) else (x, None)
    d = {"x": codes, "scales": scales, "hidden": more["hidden"], "a": p["a"], "b": p["b"], "base": more["dbase"]}
    at = {name: None if t is None or null.get(name) else t.data_ptr() for name, t in {**d, **out}.items()}
    code = T.CODE_OF[dtype]
    need = capi.lib().caifx_adapters_workspace_bytes(m, n, k, r, adapters, code, 1)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    capi.call("caifx_adapters_backward", m, n, k, r, adapters, more["dy"].data_ptr(), at["x"], at["scales"], at["hidden"], p["ids"].data_ptr(), at["a"],
              at["b"], p["scaling"].data_ptr(), at["base"], at["dx"], at["ga"], at["gb"], code, ws.data_ptr(), need,
              torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("m,k,n,r,adapters,order", [(30, 264, 392, 16, 3, "runs"), (700, 264, 392, 64, 3, "mixed"), (33, 70, 40, 128, 2100, "mixed")])
def test_every_choice_of_results(m, k, n, r, adapters, order, packed, dtype):
    """grad_b needs neither factor and no x, grad_a no a and no hidden, dx neither x nor hidden; all have the bits they have together."""
    p, more = problem(m, k, n, r, adapters, dtype, order)
    x = T.checkpoint_pack(p["x"]) if packed else p["x"]
    every = backward(p, more, adapters, x, ("dx", "ga", "gb"), {})
    for want in (("gb",), ("ga",), ("dx",), ("dx", "ga"), ("dx", "gb"), ("ga", "gb")):
        null = {"x": "ga" not in want, "scales": "ga" not in want, "hidden": "gb" not in want, "a": "dx" not in want, "b": want == ("gb",),
                "base": "dx" not in want}
        got = backward(p, more, adapters, x, want, null)
        for name in want:
            assert torch.equal(got[name], every[name]), (want, name)


def test_no_rows_need_no_operands():
    p, more = problem(0, 24, 40, 8, 3, BF16, "one")
    got = backward(p, more, 3, p["x"], ("gb",), dict.fromkeys(("x", "hidden", "a", "b", "base"), True))
    assert not got["gb"].any()


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("m", [30, 700])
def test_the_torch_call_leaves_out_what_is_not_needed(m, packed):
    p, more = problem(m, 264, 392, 16, 3, BF16, "runs")
    x = T.checkpoint_pack(p["x"]) if packed else p["x"]
    rest = {key: p[key] for key in ("ids", "a", "b", "scaling")}
    every = T.adapters_backward(more["dy"], x, more["hidden"], **rest, base=more["dbase"])
    for need in range(8):
        dx, a, b = (bool(need >> k & 1) for k in range(3))
        got = T.adapters_backward(more["dy"], x if a else None, more["hidden"] if b else None, **rest, base=more["dbase"], need_dx=dx, need_a=a, need_b=b)
        for wanted, g, e in zip((dx, a, b), got, every):
            assert torch.equal(g, e) if wanted else g is None
    into = more["dbase"].clone()
    got = T.adapters_backward(more["dy"], x, more["hidden"], **rest, base=into, out=into)
    assert got[0].data_ptr() == into.data_ptr() and all(torch.equal(g, e) for g, e in zip(got, every))
    fresh = torch.empty_like(into)
    assert torch.equal(T.adapters_backward(more["dy"], x, more["hidden"], **rest, base=more["dbase"], out=fresh)[0], every[0])


def test_results_that_share_memory_with_inputs_are_refused():
    p, more = problem(20, 64, 64, 8, 2, BF16, "mixed")
    x = p["x"]
    rest = {key: p[key] for key in ("ids", "a", "b", "scaling")}
    room = torch.zeros(21, 64, dtype=BF16, device="cuda")
    for bad in (dict(out=x), dict(base=room[:20], out=room[1:])):
        with pytest.raises(ValueError):
            T.adapters_forward(x, **rest, **bad)
    for bad in (dict(out=more["dy"]), dict(out=x), dict(base=room[1:], out=room[:20]), dict(out=more["dbase"], need_dx=False)):
        with pytest.raises(ValueError):
            T.adapters_backward(more["dy"], x, more["hidden"], **rest, **bad)
    with pytest.raises(TypeError):
        T.adapters_backward(more["dy"], None, more["hidden"], **rest)
    with pytest.raises(TypeError):
        T.adapters_backward(more["dy"], x, None, **rest)
    assert T.adapters_backward(more["dy"], x, more["hidden"], **rest, out=x, need_a=False)[0].data_ptr() == x.data_ptr()
