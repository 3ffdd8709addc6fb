"""Low-rank adapters of many requests (caifx_adapters_forward, caifx_adapters_backward) against the formulas in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from caif_amd import capi, torch_ops as T                                       # noqa: E402
import adapter_reference as R                                                   # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NOT_AN_ADAPTER = (-1, -7, 2 ** 31 - 1, -2 ** 31)


def make_ids(gen, m, adapters, order):
    """`order`: one (all rows the first), none, mixed (any order, some without), runs (neighbours belong together, some without), last
    (all rows the last adapter)."""
    if order in ("one", "none", "last"):
        return torch.full((m,), {"one": 0, "none": -1, "last": adapters - 1}[order], dtype=torch.int32, device="cuda")
    ids = torch.randint(0, adapters, (m,), device="cuda", generator=gen, dtype=torch.int32)
    odd = torch.tensor(NOT_AN_ADAPTER + (adapters,), device="cuda", dtype=torch.int32)
    none = odd[torch.randint(0, len(odd), (m,), device="cuda", generator=gen)]
    ids = torch.where(torch.rand(m, device="cuda", generator=gen) < 0.2, none, ids)
    return ids if order == "mixed" else ids[torch.arange(m, device="cuda") // 21]


def normal(gen, shape, std, dtype):
    return torch.empty(shape, device="cuda").normal_(0, std, generator=gen).to(dtype)


def problem(m, k, n, r, adapters, dtype, order, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(1000 * m + seed)
    p = {"x": normal(gen, (m, k), 1, dtype), "ids": make_ids(gen, m, adapters, order), "a": normal(gen, (adapters, r, k), 0.05, dtype),
         "b": normal(gen, (adapters, n, r), 0.3, dtype), "scaling": torch.rand(adapters, device="cuda", generator=gen) * 3 - 1}
    more = {"base": normal(gen, (m, n), 1, dtype), "dy": normal(gen, (m, n), 1e-2, dtype), "dbase": normal(gen, (m, k), 1e-2, dtype),
            "hidden": normal(gen, (m, r), 1, F32)}
    return p, more


# one row and few, tiles that end inside, ranks that are no multiple of a tile, lengths from one to long, odd ones among them
SIZES = [(1, 1, 1, 1, 1, "one"), (1, 4096, 4096, 16, 4, "last"), (1, 64, 130, 128, 2, "one"), (2, 7, 3, 3, 2, "mixed"), (5, 513, 257, 8, 3, "mixed"),
         (16, 4096, 64, 16, 16, "mixed"), (17, 100, 1408, 17, 5, "mixed"), (32, 2048, 1000, 16, 64, "mixed"), (33, 1403, 96, 64, 2, "runs"),
         (64, 128, 2049, 32, 1, "one"), (65, 520, 72, 100, 3, "runs"), (100, 4100, 40, 24, 7, "mixed"), (129, 9, 640, 4, 9, "runs"),
         (257, 256, 512, 48, 2, "runs"), (300, 40, 24, 128, 3, "mixed"), (70, 333, 77, 16, 4, "none"), (1030, 264, 136, 16, 3, "runs"),
         (2100, 96, 200, 8, 2, "mixed")]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,k,n,r,adapters,order", SIZES)
def test_forward(m, k, n, r, adapters, order, dtype):
    p, more = problem(m, k, n, r, adapters, dtype, order)
    y, hidden = T.adapters_forward(**p, base=more["base"], keep_hidden=True)
    want, mag, h, hmag = R.forward(**p, base=more["base"])
    R.check(hidden, h, hmag, F32, R.sums(k), "hidden")
    R.check(y, want, mag, dtype, R.sums(k, r) + R.pieces(dtype), "y")
    alone = T.adapters_forward(**p)
    want, mag = R.forward(**p, base=None)[:2]
    R.check(alone, want, mag, dtype, R.sums(k, r) + R.pieces(dtype), "y without base")
    # without hidden, and into base itself: the same bits
    assert torch.equal(T.adapters_forward(**p, base=more["base"]), y)
    assert T.adapters_forward(**p, base=more["base"], out=more["base"]) is not None and torch.equal(more["base"], y)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("m,k,n,r,adapters,order", SIZES)
def test_backward(m, k, n, r, adapters, order, packed, dtype):
    p, more = problem(m, k, n, r, adapters, dtype, order)
    x = p.pop("x")
    kept = T.checkpoint_pack(x) if packed else x
    value = R.unpacked(*(t.cpu() for t in kept)) if packed else x
    for base in (more["dbase"], None):
        dx, ga, gb = T.adapters_backward(more["dy"], kept, more["hidden"], **p, base=base)
        want = R.backward(more["dy"], value, more["hidden"], **p, base=base)
        R.check(dx, *want["dx"], dtype, R.sums(n, r) + R.pieces(dtype), "dx")
        R.check(ga, *want["grad_a"], dtype, R.sums(n, m) + R.pieces(dtype), "grad_a")
        R.check(gb, *want["grad_b"], dtype, R.sums(m) + R.pieces(dtype), "grad_b")
    none, ga2, gb2 = T.adapters_backward(more["dy"], kept, more["hidden"], **p, need_dx=False)
    assert none is None and torch.equal(ga2, ga) and torch.equal(gb2, gb)


def test_rows_without_an_adapter_keep_their_base():
    p, more = problem(100, 264, 200, 16, 3, BF16, "mixed")
    more["base"][::7] = float("nan")
    y = T.adapters_forward(**p, base=more["base"])
    none = (p["ids"] < 0) | (p["ids"] >= 3)
    assert none.any() and torch.equal(y[none].view(torch.int16), more["base"][none].view(torch.int16))
    x = p.pop("x")
    dx = T.adapters_backward(more["dy"], x, more["hidden"], **p, base=more["dbase"])[0]
    assert torch.equal(dx[none].view(torch.int16), more["dbase"][none].view(torch.int16))


@pytest.mark.parametrize("m,order", [(3, "mixed"), (40, "mixed"), (200, "runs"), (200, "mixed")])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_infinities_and_nan_stay_where_they_belong(m, order, dtype):
    """A NaN in one row reaches that row alone, one in an adapter the rows of that adapter alone, one in a row without adapter nothing."""
    p, more = problem(m, 264, 200, 24, 4, dtype, order)
    clean_y, clean_h = T.adapters_forward(**p, base=more["base"], keep_hidden=True)
    x = p["x"]
    clean = T.adapters_backward(more["dy"], x, more["hidden"], **{k: p[k] for k in ("ids", "a", "b", "scaling")}, base=more["dbase"])
    valid = (p["ids"] >= 0) & (p["ids"] < 4)
    bad = int(valid.nonzero()[0])
    sick = int(p["ids"][bad])
    for spoil in ("row", "adapter", "none"):
        q = {k: v.clone() for k, v in p.items()}
        n = {k: v.clone() for k, v in more.items()}
        touched = torch.zeros(m, dtype=torch.bool, device="cuda")
        if spoil == "row":
            touched[bad] = True
            q["x"][bad] = float("nan")
            n["dy"][bad] = float("inf")
        elif spoil == "adapter":
            touched = p["ids"] == sick
            q["a"][sick] = float("nan")
            q["b"][sick] = float("inf")
        else:
            for t in (q["x"], n["dy"], n["hidden"]):
                t[~valid] = float("nan")
        y, h = T.adapters_forward(**q, base=n["base"], keep_hidden=True)
        assert torch.equal(y[~touched], clean_y[~touched]) and torch.equal(h[~touched], clean_h[~touched])
        xx = q.pop("x")
        dx, ga, gb = T.adapters_backward(n["dy"], xx, n["hidden"], **q, base=n["dbase"])
        assert torch.equal(dx[~touched], clean[0][~touched])
        others = [l for l in range(4) if l != sick or spoil == "none"]
        assert torch.equal(ga[others], clean[1][others]) and torch.equal(gb[others], clean[2][others])
        if spoil == "row":
            assert not y[bad].isfinite().any() and not dx[bad].isfinite().any()
            assert not ga[sick].isfinite().any() and not gb[sick].isfinite().any()
        if spoil == "adapter":
            assert not y[touched].isfinite().any() and not dx[touched].isfinite().any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,k,n,r", [(3, 264, 200, 16), (50, 1001, 515, 24), (200, 96, 333, 16)])
def test_any_alignment_and_nothing_around_the_results_is_touched(m, k, n, r, dtype):
    """Tensors that begin one element behind a 16-byte boundary, results inside memory that holds a mark."""
    p, more = problem(m, k, n, r, 3, dtype, "mixed")
    want_y, want_h = T.adapters_forward(**p, base=more["base"], keep_hidden=True)
    x = p["x"]
    rest = {key: p[key] for key in ("ids", "a", "b", "scaling")}
    want = T.adapters_backward(more["dy"], x, more["hidden"], **rest, base=more["dbase"])

    def shifted(t):
        room = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        room[1:] = t.reshape(-1)
        return room[1:].reshape(t.shape)

    def marked(count, dt):
        room = torch.full((count + 18,), 7.0, dtype=dt, device="cuda")
        return room, room[9:9 + count]

    def untouched(room, count):
        return bool((room[:9] == 7).all()) and bool((room[9 + count:] == 7).all())

    s = {key: shifted(v) for key, v in {**p, **more}.items()}
    rooms = {name: marked(count, dt) for name, count, dt in (("y", m * n, dtype), ("h", m * r, F32), ("dx", m * k, dtype), ("ga", 3 * r * k, dtype),
                                                             ("gb", 3 * n * r, dtype))}
    ptr = {name: v[1].data_ptr() for name, v in rooms.items()}
    code, stream = T.CODE_OF[dtype], torch.cuda.current_stream().cuda_stream
    lib = capi.lib()
    for back in (0, 1):
        need = lib.caifx_adapters_workspace_bytes(m, n, k, r, 3, code, back)
        room, ws = marked((need + 3) // 4, F32)
        d = {key: v.data_ptr() for key, v in s.items()}
        if back:
            capi.call("caifx_adapters_backward", m, n, k, r, 3, d["dy"], d["x"], None, d["hidden"], d["ids"], d["a"], d["b"], d["scaling"], d["dbase"],
                      ptr["dx"], ptr["ga"], ptr["gb"], code, ws.data_ptr(), need, stream)
        else:
            capi.call("caifx_adapters_forward", m, n, k, r, 3, d["x"], d["ids"], d["a"], d["b"], d["scaling"], d["base"], ptr["y"], ptr["h"], code,
                      ws.data_ptr(), need, stream)
        torch.cuda.synchronize()
        assert untouched(room, (need + 3) // 4)
    for name, v in zip(("y", "h", "dx", "ga", "gb"), (want_y, want_h, *want)):
        room, got = rooms[name]
        assert torch.equal(got.reshape(v.shape), v), name
        assert untouched(room, v.numel()), name


def test_results_repeat_bit_for_bit():
    p, more = problem(700, 1408, 2048, 16, 3, BF16, "runs")
    x = p.pop("x")
    first = T.adapters_backward(more["dy"], x, more["hidden"], **p, base=more["dbase"])
    for _ in range(5):
        again = T.adapters_backward(more["dy"], x, more["hidden"], **p, base=more["dbase"])
        assert all(torch.equal(u, v) for u, v in zip(first, again))


@pytest.mark.parametrize("m", [40, 300])
def test_gradients_are_the_differences_of_the_forward(m):
    """The branch is linear in x, in a and in b: the difference of its results at t + d and t - d is twice its derivative along d, without
    a remainder.  In fp32; the differences' own rounding is that of two results, 2^-24 of their magnitude and the sums' for each."""
    p, more = problem(m, 256, 192, 16, 3, F32, "mixed", seed=1)
    y, hidden = T.adapters_forward(**p, keep_hidden=True)
    rest = {key: p[key] for key in ("ids", "a", "b", "scaling")}
    grads = dict(zip(("x", "a", "b"), T.adapters_backward(more["dy"], p["x"], hidden, **rest)))
    gen = torch.Generator(device="cuda").manual_seed(5)
    for name in ("x", "a", "b"):
        d = torch.empty_like(p[name]).normal_(0, float(p[name].std()), generator=gen)
        up, down = (T.adapters_forward(**{**p, name: p[name] + s * d}).double() for s in (1, -1))
        along = ((up - down) / 2 * more["dy"].double()).sum()
        # every product in the sum is off by its magnitude's share, signs at random: added up in squares, times six
        mag = sum(R.forward(**{**p, name: p[name] + s * d}, base=None)[1] for s in (1, -1)).cuda()
        off = 6 * (mag * more["dy"].abs().double() * (R.sums(256, 16) + 2.0 ** -24)).square().sum().sqrt()
        got = (grads[name].double() * d.double()).sum()
        assert abs(got - along) <= off + 2.0 ** -20 * abs(along), (name, float(got), float(along), float(off))


def test_no_rows_and_adapters_without_rows():
    p, more = problem(0, 24, 40, 8, 3, BF16, "one")
    assert T.adapters_forward(**p).shape == (0, 40)
    x = p.pop("x")
    dx, ga, gb = T.adapters_backward(more["dy"], x, more["hidden"], **p)
    assert dx.shape == (0, 24) and not ga.any() and not gb.any()
    p, more = problem(50, 24, 40, 8, 6, BF16, "one")
    x = p.pop("x")
    ga, gb = T.adapters_backward(more["dy"], x, more["hidden"], **p)[1:]
    assert ga[0].any() and gb[0].any() and not ga[1:].any() and not gb[1:].any()


@pytest.mark.parametrize("m,k,n,r,adapters,order", [(1, 512, 512, 16, 2, "one"), (24, 2048, 1408, 16, 8, "mixed"), (600, 512, 1024, 32, 2, "runs")])
def test_captured_and_replayed(m, k, n, r, adapters, order):
    """A forward and its backward captured once and replayed with new inputs, eager work on the same shapes between the replays."""
    p, more = problem(m, k, n, r, adapters, BF16, order)

    def step(q, n):
        y, hidden = T.adapters_forward(**q, base=n["base"], keep_hidden=True)
        rest = {key: q[key] for key in ("ids", "a", "b", "scaling")}
        return (y, hidden, *T.adapters_backward(n["dy"], T.checkpoint_pack(q["x"]), hidden, **rest, base=n["dbase"]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(p, more)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(p, more)
    for seed in (3, 4, 5):
        q, o = problem(m, k, n, r, adapters, BF16, order, seed)
        want = step(q, o)
        for mine, new in ((p, q), (more, o)):
            for key in mine:
                mine[key].copy_(new[key])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(got, want))


def test_another_stream():
    p, more = problem(300, 512, 640, 16, 3, BF16, "runs")
    want = T.adapters_forward(**p, base=more["base"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [T.adapters_forward(**p, base=more["base"]) for _ in range(4)]
    side.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_offsets_past_32_bits():
    """Results and gradients of more than 2^31 elements: the first and the last rows, the rest by its rows' equality."""
    m, n, r = 66000, 33000, 8
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = normal(gen, (m, 64), 1, BF16)
    x[-100:] = x[:100]
    ids = torch.zeros(m, dtype=torch.int32, device="cuda")
    a, b = normal(gen, (1, r, 64), 0.1, BF16), normal(gen, (1, n, r), 0.1, BF16)
    scaling = torch.ones(1, device="cuda")
    y = T.adapters_forward(x, ids, a, b, scaling)
    want, mag = R.forward(x[:100], ids[:100], a, b, scaling, None)[:2]
    R.check(y[:100], want, mag, BF16, R.sums(64, r) + R.pieces(BF16), "first rows")
    assert torch.equal(y[-100:], y[:100])
    dy = y
    hidden = torch.ones(m, r, device="cuda")
    dx = T.adapters_backward(dy, x, hidden, ids, a, b, scaling)[0]
    want = R.backward(dy[:100], x[:100], hidden[:100], ids[:100], a, b, scaling, None)
    R.check(dx[:100], *want["dx"], BF16, R.sums(n, r) + R.pieces(BF16), "first gradient rows")
    assert torch.equal(dx[-100:], dx[:100])


@pytest.mark.parametrize("tokens", [1, 24, 500])
def test_a_block_with_adapters_and_checkpoints(orc, tokens):
    """A gated feed-forward block over a frozen int4 base, an adapter on each projection, as a step runs it: the forward keeps 8-bit
    checkpoints, the backward works from them.  Against the same calls made one by one on the values that the checkpoints stand for."""
    import numpy as np
    from gpu_helpers import make_weight
    rng = np.random.default_rng(tokens)
    dim, wide, r, count = 256, 512, 16, 3
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    base = [make_weight(orc, rng, wide, dim, "int4")[1], make_weight(orc, rng, wide, dim, "int4")[1], make_weight(orc, rng, dim, wide, "int4")[1]]
    shape = [(wide, dim), (wide, dim), (dim, wide)]
    fac = [(normal(gen, (count, r, k), 0.05, BF16), normal(gen, (count, n, r), 0.05, BF16)) for n, k in shape]
    scaling = torch.tensor([2.0, 0.5, 1.0], device="cuda")
    ids = make_ids(gen, tokens, count, "mixed")
    x, dy = normal(gen, (tokens, dim), 1, BF16), normal(gen, (tokens, dim), 1e-2, BF16)

    def project(v, i):
        y = T.qlinear_forward(v, base[i], T.BF16, T.BF16)
        return T.adapters_forward(v, ids, *fac[i], scaling, base=y, keep_hidden=True, out=y)

    def back(d, v, hidden, i):
        return T.adapters_backward(d, v, hidden, ids, *fac[i], scaling, base=T.qlinear_backward_input(d, base[i], T.BF16, T.BF16))

    (gate, hg), (up, hu), kept = project(x, 0), project(x, 1), T.checkpoint_pack(x)
    hidden, gate_ck, up_ck = T.silu_multiply_checkpoint(gate, up)
    y, hd = project(hidden, 2)
    assert torch.equal(hidden, T.silu_multiply(gate, up))
    grad_gate, grad_up, again = T.swiglu_backward_checkpoint(gate_ck, up_ck, dy.new_zeros(tokens, wide), with_hidden=True)
    assert not grad_gate.any() and not grad_up.any()
    d_hidden, ga, gb = back(dy, again, hd, 2)
    grad_gate, grad_up = T.swiglu_backward_checkpoint(gate_ck, up_ck, d_hidden)
    one, two = back(grad_gate, kept, hg, 0), back(grad_up, kept, hu, 1)
    for d, h, i, got in ((grad_gate, hg, 0, one), (grad_up, hu, 1, two)):
        value = R.unpacked(*(t.cpu() for t in kept))
        want = R.backward(d, value, h, ids, *fac[i], scaling, T.qlinear_backward_input(d, base[i], T.BF16, T.BF16))
        for name, g in zip(("dx", "grad_a", "grad_b"), got):
            R.check(g, *want[name], BF16, R.sums(wide, max(tokens, r)) + R.pieces(BF16), name)
    want = R.backward(dy, again, hd, ids, *fac[2], scaling, T.qlinear_backward_input(dy, base[2], T.BF16, T.BF16))
    for name, g in zip(("dx", "grad_a", "grad_b"), (d_hidden, ga, gb)):
        R.check(g, *want[name], BF16, R.sums(dim, max(tokens, r)) + R.pieces(BF16), name)
    want, mag = R.forward(hidden, ids, *fac[2], scaling, T.qlinear_forward(hidden, base[2], T.BF16, T.BF16))[:2]
    R.check(y, want, mag, BF16, R.sums(wide, r) + R.pieces(BF16), "y")


def call_backward(p, more, adapters, dx, ga, gb, base):
    """caifx_adapters_backward with any of its results, null for None."""
    at = lambda t: None if t is None else t.data_ptr()                                                    # noqa: E731
    (m, k), n, r = p["x"].shape, p["b"].shape[1], p["a"].shape[1]
    code = T.CODE_OF[p["x"].dtype]
    need = capi.lib().caifx_adapters_workspace_bytes(m, n, k, r, adapters, code, 1)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    capi.call("caifx_adapters_backward", m, n, k, r, adapters, at(more["dy"]), at(p["x"]) if ga is not None else None, None,
              at(more["hidden"]) if gb is not None else None, at(p["ids"]), at(p["a"]) if dx is not None else None, at(p["b"]), at(p["scaling"]),
              at(base), at(dx), at(ga), at(gb), code, at(ws), need, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()


@pytest.mark.parametrize("m", [30, 700])
def test_each_result_alone_and_dx_into_its_base(m):
    p, more = problem(m, 264, 392, 16, 3, BF16, "runs")
    want = T.adapters_backward(more["dy"], p["x"], more["hidden"], **{key: p[key] for key in ("ids", "a", "b", "scaling")}, base=more["dbase"])
    for i in range(3):
        out = [None, None, None]
        out[i] = torch.full_like(want[i], float("nan"))
        call_backward(p, more, 3, *out, more["dbase"])
        assert torch.equal(out[i], want[i])
    into = more["dbase"].clone()
    call_backward(p, more, 3, into, None, None, into)
    assert torch.equal(into, want[0])


@pytest.mark.parametrize("adapters", [700, 5000])
def test_more_adapters_than_rows(adapters):
    """Counters of the sorting workgroup for fewer waves than it has, and beyond its local memory."""
    p, more = problem(300, 72, 40, 8, adapters, BF16, "mixed")
    y, hidden = T.adapters_forward(**p, base=more["base"], keep_hidden=True)
    want, mag = R.forward(**p, base=more["base"])[:2]
    R.check(y, want, mag, BF16, R.sums(72, 8) + R.pieces(BF16), "y")
    x = p.pop("x")
    got = T.adapters_backward(more["dy"], x, more["hidden"], **p, base=more["dbase"])
    want = R.backward(more["dy"], x, more["hidden"], **p, base=more["dbase"])
    for name, g in zip(("dx", "grad_a", "grad_b"), got):
        R.check(g, *want[name], BF16, R.sums(40, 300) + R.pieces(BF16), name)


def test_one_adapter_of_many_rows_in_any_order():
    """Several runs of one adapter's rows, the rows of the others between them, through every kernel of the large calls."""
    p, more = problem(4500, 520, 4100, 16, 2, BF16, "mixed")
    y = T.adapters_forward(**p, base=more["base"])
    want, mag = R.forward(**p, base=more["base"])[:2]
    R.check(y, want, mag, BF16, R.sums(520, 16) + R.pieces(BF16), "y")
    x = p.pop("x")
    got = T.adapters_backward(more["dy"], x, more["hidden"], **p, base=more["dbase"])
    want = R.backward(more["dy"], x, more["hidden"], **p, base=more["dbase"])
    for name, g in zip(("dx", "grad_a", "grad_b"), got):
        R.check(g, *want[name], BF16, R.sums(4100, 4500) + R.pieces(BF16), name)
