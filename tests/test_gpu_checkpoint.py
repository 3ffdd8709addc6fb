"""Activation checkpoints in 8 bits: codes, scales and values bit for bit against the definition, the gating's backward from them
against 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from caif_amd import capi, torch_ops as T                                       # noqa: E402
import adapter_reference as R                                                   # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
GROUP = 128
# one value, parts of a lane, of a group and of a workgroup, rows of whole groups, widths around them, many rows
SIZES = [(1, 1), (1, 7), (3, 8), (2, 127), (2, 128), (5, 129), (77, 1407), (100, 1403), (16, 2048), (33, 4100), (1000, 130), (3000, 5), (64, 11008)]


def definition(x):
    """codes and scales by the definition, fp32 operations of numpy one by one."""
    v = x.float().cpu().numpy()
    rows, cols = v.shape
    groups = -(-cols // GROUP)
    wide = np.zeros((rows, groups * GROUP), np.float32)
    wide[:, :cols] = v
    wide = wide.reshape(rows, groups, GROUP)
    with np.errstate(all="ignore"):
        scale = (np.abs(wide).max(-1) * (np.float32(1) / np.float32(127))).astype(np.float32)
        scale[scale == 0] = 1
        odd = ~np.isfinite(wide).all(-1)
        codes = np.clip(np.rint((wide / scale[..., None]).astype(np.float32)), -127, 127)
    scale[odd] = np.nan
    codes[odd] = 0
    return codes.reshape(rows, -1)[:, :cols].astype(np.int8), scale


def special(rows, cols, dtype, seed):
    """Normal values, and rows that go wrong easily: zeros, quotients that are ties, the smallest and largest numbers, infinities, NaN."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.empty(rows, cols, device="cuda").normal_(generator=gen)
    x = x * torch.exp2(torch.randint(-8, 9, (rows, 1), device="cuda", generator=gen).float())
    info = torch.finfo(dtype)
    ties = (torch.arange(cols, device="cuda") % 255 - 127).float() / 2
    ties[::GROUP] = 127
    rows_of = {1: torch.zeros(cols, device="cuda"), 2: ties, 3: -ties * 2.0 ** -9, 4: torch.full((cols,), info.max, device="cuda"),
               5: torch.full((cols,), info.tiny, device="cuda") * (torch.arange(cols, device="cuda") % 5).float()}
    if dtype != F16:
        rows_of[6] = torch.full((cols,), 2.0 ** -130, device="cuda") * (torch.arange(cols, device="cuda") % 7).float()
    for i, row in rows_of.items():
        x[i::11] = row
    x = x.to(dtype)
    if rows > 7:
        x[7::11, cols // 2] = float("inf")
        x[8::11, cols - 1] = float("nan")
        x[9::11, 0] = float("-inf")
    return x


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_pack_and_unpack(rows, cols, dtype):
    x = special(rows, cols, dtype, rows + cols)
    codes, scales = T.checkpoint_pack(x)
    want, want_scales = definition(x)
    assert np.array_equal(scales.cpu().numpy(), want_scales, equal_nan=True)
    assert np.array_equal(codes.cpu().numpy(), want)
    for out in (F32, F16, BF16):
        with np.errstate(all="ignore"):
            value = want.astype(np.float32) * np.repeat(want_scales, GROUP, axis=1)[:, :cols]
        got = T.checkpoint_unpack(codes, scales, out)
        assert got.dtype == out and got.shape == x.shape
        assert torch.equal(got.cpu().isnan(), torch.from_numpy(value).isnan())
        assert torch.equal(got.cpu().nan_to_num(0.0), torch.from_numpy(value).to(out).nan_to_num(0.0))


def test_every_quotient_near_a_tie():
    """Groups whose maximum makes many quotients ties or next to ties."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    top = torch.rand(4096, 1, device="cuda", generator=gen) + 0.5
    k = torch.randint(-127, 127, (4096, GROUP), device="cuda", generator=gen).float() + 0.5
    x = (k * top / 127)
    x = torch.nextafter(x, x + torch.randint(-1, 2, x.shape, device="cuda", generator=gen).float())
    x[:, 0] = top[:, 0]
    codes, scales = T.checkpoint_pack(x)
    want, want_scales = definition(x)
    assert np.array_equal(scales.cpu().numpy(), want_scales) and np.array_equal(codes.cpu().numpy(), want)


def test_every_pair_of_a_maximum_and_a_value_in_16_bits():
    """The quotient of two numbers of 11 bits, scaled by powers of two: all of them, the value up to 2^9 times smaller than the maximum
    (below that its code is zero)."""
    top = torch.arange(1024, 2048, device="cuda")
    value = torch.arange(1024, 2048, device="cuda")
    for shift in range(10):
        v = (value.float() * 2.0 ** -shift).expand(1024, -1)
        keep = torch.where(v <= top[:, None].float(), v, torch.zeros((), device="cuda"))
        x = torch.cat([top.float()[:, None].expand(-1, 8).reshape(1024, 8, 1), keep.reshape(1024, 8, 128)[:, :, :127]], 2).reshape(8192, 128)
        last = torch.cat([top.float()[:, None], keep.reshape(1024, 8, 128)[:, :, 127], torch.zeros(1024, 119, device="cuda")], 1)
        x = torch.cat([x, last]).to(F16)
        assert torch.equal(x.float().amax(1)[:8192:8], top.float())
        codes, scales = T.checkpoint_pack(x)
        want, want_scales = definition(x)
        assert np.array_equal(scales.cpu().numpy(), want_scales) and np.array_equal(codes.cpu().numpy(), want)


def test_more_dimensions_and_no_elements():
    x = torch.randn(3, 5, 200, device="cuda")
    codes, scales = T.checkpoint_pack(x)
    assert codes.shape == (3, 5, 200) and scales.shape == (3, 5, 2)
    flat = T.checkpoint_pack(x.reshape(15, 200))
    assert torch.equal(codes.reshape(15, 200), flat[0]) and torch.equal(scales.reshape(15, 2), flat[1])
    codes, scales = T.checkpoint_pack(torch.empty(0, 200, device="cuda"))
    assert codes.shape == (0, 200) and scales.shape == (0, 2) and T.checkpoint_unpack(codes, scales, F32).shape == (0, 200)
    codes, scales = T.checkpoint_pack(torch.empty(4, 0, device="cuda"))
    assert codes.shape == (4, 0) and scales.shape == (4, 0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_gating_keeps_its_bits_and_packs_its_inputs(rows, cols, dtype):
    gate, up = special(rows, cols, dtype, 1), special(rows, cols, dtype, 2)
    hidden, gate_ck, up_ck = T.silu_multiply_checkpoint(gate, up)
    plain = T.silu_multiply(gate, up)
    assert torch.equal(hidden.isnan(), plain.isnan()) and torch.equal(hidden.nan_to_num(0.0), plain.nan_to_num(0.0))
    for t, got in ((gate, gate_ck), (up, up_ck)):
        codes, scales = T.checkpoint_pack(t)
        assert torch.equal(got[0], codes) and torch.equal(got[1].nan_to_num(-1.0), scales.nan_to_num(-1.0))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_gating_backward(rows, cols, dtype):
    """s = 1 / (1 + exp(-g)) is off by some 2^-22 (an exponential within two steps, two roundings), the results' factors by a few
    roundings more: 2^-20 of d u for grad_gate, whose factor silu' is at most 1.1 and may cancel, of d silu and of u silu for the others."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    gate, up = (torch.empty(rows, cols, device="cuda").normal_(0, 3, generator=gen).to(dtype) for _ in range(2))
    gate[0, 0] = -80.0
    gate[-1, -1] = 200.0
    grad = torch.empty(rows, cols, device="cuda").normal_(0, 0.1, generator=gen).to(dtype)
    _, gate_ck, up_ck = T.silu_multiply_checkpoint(gate, up)
    grad_gate, grad_up, hidden = T.swiglu_backward_checkpoint(gate_ck, up_ck, grad, with_hidden=True)
    g, u = (R.unpacked(*(t.cpu() for t in ck)).float().double() for ck in (gate_ck, up_ck))     # code * scale is one fp32 rounding
    d = grad.double().cpu()
    s = torch.sigmoid(g)
    R.check(grad_up, d * g * s, (d * g * s).abs(), dtype, 2.0 ** -20, "grad_up")
    R.check(grad_gate, d * u * (s + g * s * (1 - s)), (d * u).abs(), dtype, 2.0 ** -20, "grad_gate")
    R.check(hidden, g * s * u, (g * s * u).abs(), dtype, 2.0 ** -20, "hidden")
    without = T.swiglu_backward_checkpoint(gate_ck, up_ck, grad)
    assert len(without) == 2 and torch.equal(without[0], grad_gate) and torch.equal(without[1], grad_up)


def test_an_overflow_shows_in_the_gradients_of_its_group():
    gate, up = torch.randn(4, 300, device="cuda"), torch.randn(4, 300, device="cuda")
    gate[1, 130] = float("inf")
    up[3, 299] = float("nan")
    _, gate_ck, up_ck = T.silu_multiply_checkpoint(gate, up)
    grad_gate, grad_up = T.swiglu_backward_checkpoint(gate_ck, up_ck, torch.ones(4, 300, device="cuda"))
    bad = torch.zeros(4, 300, dtype=torch.bool, device="cuda")
    bad[1, 128:256] = True
    assert torch.equal(grad_up.isnan(), bad)
    bad[3, 256:] = True
    assert torch.equal(grad_gate.isnan(), bad)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols", [(3, 200), (5, 131), (40, 1407)])
def test_any_alignment_and_nothing_around_the_results_is_touched(rows, cols, dtype):
    gen = torch.Generator(device="cuda").manual_seed(9)
    n, groups, code, stream = rows * cols, rows * -(-cols // GROUP), T.CODE_OF[dtype], torch.cuda.current_stream().cuda_stream

    def place(count, dt, value=None):
        room = torch.full((count + 18,), 7, dtype=dt, device="cuda")
        if value is not None:
            room[9:9 + count] = value.reshape(-1)
        return room, room[9:9 + count]

    gate, up, grad = (torch.empty(rows, cols, device="cuda").normal_(generator=gen).to(dtype) for _ in range(3))
    want = T.silu_multiply_checkpoint(gate, up)
    wants = [want[0], *want[1], *want[2]]
    ins = [place(n, dtype, t)[1] for t in (gate, up, grad)]
    outs = [place(c, dt) for c, dt in ((n, dtype), (n, torch.int8), (groups, F32), (n, torch.int8), (groups, F32))]
    capi.call("caifx_silu_multiply_checkpoint", ins[0].data_ptr(), ins[1].data_ptr(), *(o[1].data_ptr() for o in outs), rows, cols, code, stream)
    alone = [place(n, torch.int8), place(groups, F32)]
    capi.call("caifx_checkpoint_pack", ins[0].data_ptr(), alone[0][1].data_ptr(), alone[1][1].data_ptr(), rows, cols, code, stream)
    back = [place(n, dtype) for _ in range(3)]
    capi.call("caifx_swiglu_backward_checkpoint", *(o[1].data_ptr() for o in outs[1:]), ins[2].data_ptr(), *(o[1].data_ptr() for o in back), rows, cols,
              code, stream)
    out = place(n, dtype)
    capi.call("caifx_checkpoint_unpack", alone[0][1].data_ptr(), alone[1][1].data_ptr(), out[1].data_ptr(), rows, cols, code, stream)
    torch.cuda.synchronize()
    wants += [*want[1], *T.swiglu_backward_checkpoint(want[1], want[2], grad, with_hidden=True), T.checkpoint_unpack(*want[1], dtype)]
    for (room, got), v in zip(outs + alone + back + [out], wants):
        assert torch.equal(got.reshape(v.shape), v)
        assert bool((room[:9] == 7).all()) and bool((room[-9:] == 7).all())


def test_offsets_past_32_bits():
    rows, cols = 70000, 32000
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.empty(rows, cols, device="cuda", dtype=BF16).normal_(generator=gen)
    codes, scales = T.checkpoint_pack(x)
    for at in (slice(0, 10), slice(rows - 10, rows)):
        want, want_scales = definition(x[at])
        assert np.array_equal(codes[at].cpu().numpy(), want) and np.array_equal(scales[at].cpu().numpy(), want_scales)
    y = T.checkpoint_unpack(codes, scales, BF16)
    assert torch.equal(y[-10:], T.checkpoint_unpack(codes[-10:].contiguous(), scales[-10:].contiguous(), BF16))
