"""Adapter fine-tuning and serving beside a frozen projection, as cases that can be timed and compared.

A case is a dict of plain values.  `kind` names the operator:

    forward     the low-rank branches of many requests added to the result of the projection that they share
    backward    the branch's gradients: of the input (added to the projection's own), of both factors
    checkpoint  an activation put away in 8 bits, and brought back
    gate        the gating of a feed-forward block with its inputs put away in 8 bits, and its backward pass from them

`ids` gives every row its adapter, -1 none.  `run` is the mean number of neighbouring rows that belong together: 1 in a decode step, a
prompt's or a training sequence's length otherwise.  Activations are N(0, 1), gradients N(0, 1e-3), factors N(0, 0.02)."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GROUP = 128


def listed():
    return [
        # the smallest call: one request decodes through one square projection; four adapters are loaded
        {"name": "forward-1", "kind": "forward", "dtype": "bf16", "m": 1, "k": 4096, "n": 4096, "rank": 16, "adapters": 4, "run": 1, "keep": False},
        # a decode step of 32 requests over 64 adapters, the up projection of an 8B feed-forward block
        {"name": "forward-32", "kind": "forward", "dtype": "bf16", "m": 32, "k": 4096, "n": 14336, "rank": 16, "adapters": 64, "run": 1, "keep": False},
        # several prompts of uneven length in one batch, fp16, a rank that is no multiple of 16
        {"name": "forward-999", "kind": "forward", "dtype": "f16", "m": 999, "k": 4096, "n": 4096, "rank": 24, "adapters": 6, "run": 150, "keep": False},
        # a training step's forward, 4096 tokens through the up projection of a 7B feed-forward block
        {"name": "forward-4096", "kind": "forward", "dtype": "bf16", "m": 4096, "k": 4096, "n": 11008, "rank": 16, "adapters": 1, "run": 4096, "keep": True},
        # a small ragged batch in the default type, odd sizes, three adapters trained at once
        {"name": "backward-333", "kind": "backward", "dtype": "f32", "m": 333, "k": 1403, "n": 2048, "rank": 8, "adapters": 3, "run": 60, "packed": False},
        # the training step above, backward
        {"name": "backward-4096", "kind": "backward", "dtype": "bf16", "m": 4096, "k": 4096, "n": 11008, "rank": 16, "adapters": 1, "run": 4096, "packed": False},
        # four adapters of rank 64 trained side by side, the input kept as an 8-bit checkpoint
        {"name": "backward-packed", "kind": "backward", "dtype": "bf16", "m": 4096, "k": 4096, "n": 11008, "rank": 64, "adapters": 4, "run": 512, "packed": True},
        # a small activation with a width that is no multiple of the group
        {"name": "checkpoint-100", "kind": "checkpoint", "dtype": "f16", "m": 100, "n": 1403},
        # the input of a feed-forward block over 16384 tokens
        {"name": "checkpoint-16384", "kind": "checkpoint", "dtype": "bf16", "m": 16384, "n": 4096},
        # the gating of one small expert's rows, odd width
        {"name": "gate-77", "kind": "gate", "dtype": "f16", "m": 77, "n": 1407},
        # the gating of a dense 7B block, 4096 tokens
        {"name": "gate-4096", "kind": "gate", "dtype": "bf16", "m": 4096, "n": 11008},
        # the gating of all experts' rows, 4096 tokens with six experts each
        {"name": "gate-24576", "kind": "gate", "dtype": "bf16", "m": 24576, "n": 1408},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Mostly multiples of 64, one in four any number."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.25 else max(lo, n // 64 * 64)


def draw(rng):
    kind = rng.choice(["forward", "forward", "forward", "backward", "backward", "checkpoint", "gate"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("checkpoint", "gate"):
        return {"kind": kind, "dtype": dtype, "m": _log_int(rng, 1, 8192), "n": _width(rng, 256, 4096)}
    case = {"kind": kind, "dtype": dtype, "k": _width(rng, 512, 4096), "n": _width(rng, 512, 8192), "rank": rng.choice([4, 8, 16, 16, 24, 32, 64])}
    if kind == "forward" and rng.random() < 0.5:      # a decode step
        return {**case, "m": _log_int(rng, 1, 128), "adapters": _log_int(rng, 1, 64), "run": 1, "keep": False}
    m = _log_int(rng, 64, 4096)
    case.update(m=m, adapters=_log_int(rng, 1, 8), run=_log_int(rng, 16, m))
    return {**case, **({"keep": rng.random() < 0.5} if kind == "forward" else {"packed": rng.random() < 0.5})}


# ------------------------------------------------------------------------------------------------ what a program holds
def _normal(gen, shape, std, dtype):
    return torch.empty(shape, device="cuda").normal_(0, std, generator=gen).to(dtype)


def _ids(gen, case):
    """An adapter for each run of rows, one run in eight without; runs end at random rows."""
    m, runs = case["m"], -(-case["m"] // case["run"])
    where = torch.arange(m, device="cuda")
    if case["run"] > 1:
        ends = torch.randint(0, m, (runs - 1,), device="cuda", generator=gen).sort().values
        where = torch.bucketize(where, ends, right=True)
    of_run = torch.randint(0, case["adapters"], (runs,), device="cuda", generator=gen)
    none = torch.rand(runs, device="cuda", generator=gen) < (0.125 if runs > 1 else 0)
    return torch.where(none, -1, of_run)[where].to(torch.int32)


def _in_groups(x):
    """x [m, n] as [m, groups, GROUP], zeros behind the last column."""
    m, n = x.shape
    return torch.nn.functional.pad(x, (0, -n % GROUP)).reshape(m, -1, GROUP)


def _pack(x):
    """codes int8 [m, n] and scales fp32 [m, groups] of finite values."""
    v = _in_groups(x.float())
    scales = v.abs().amax(-1) / 127
    scales = torch.where(scales == 0, torch.ones_like(scales), scales)
    codes = (v / scales[..., None]).round().clamp(-127, 127)
    return codes.reshape(x.shape[0], -1)[:, :x.shape[1]].to(torch.int8).contiguous(), scales


def _unpack(codes, scales):
    m, n = codes.shape
    return (_in_groups(codes.float()) * scales[..., None]).reshape(m, -1)[:, :n]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype, m, n = case["kind"], DTYPES[case["dtype"]], case["m"], case["n"]
    s = {"kind": kind, "dtype": dtype}
    if kind == "checkpoint":
        return {**s, "x": _normal(gen, (m, n), 1, dtype)}
    if kind == "gate":
        return {**s, "gate": _normal(gen, (m, n), 1, dtype), "up": _normal(gen, (m, n), 1, dtype), "grad": _normal(gen, (m, n), 1e-3, dtype)}
    k, r, count = case["k"], case["rank"], case["adapters"]
    x = _normal(gen, (m, k), 1, dtype)
    s.update(ids=_ids(gen, case), a=_normal(gen, (count, r, k), 0.02, dtype), b=_normal(gen, (count, n, r), 0.02, dtype),
             scaling=torch.rand(count, device="cuda", generator=gen) + 1)
    if kind == "forward":
        return {**s, "x": x, "base": _normal(gen, (m, n), 1, dtype), "keep": case["keep"]}
    rows = torch.where((s["ids"] >= 0)[:, None], _normal(gen, (m, r), 1, torch.float32), torch.zeros((), device="cuda"))
    return {**s, "x": _pack(x) if case["packed"] else x, "dy": _normal(gen, (m, n), 1e-3, dtype), "hidden": rows,
            "base": _normal(gen, (m, k), 1e-3, dtype)}


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _own(s)
    return {"forward": _forward, "backward": _backward, "checkpoint": _checkpoint, "gate": _gate}[s["kind"]](s)


def _own(s):
    from caif_amd import torch_ops as T
    if s["kind"] == "forward":
        return T.adapters_forward(s["x"], s["ids"], s["a"], s["b"], s["scaling"], base=s["base"], keep_hidden=s["keep"])
    if s["kind"] == "backward":
        return T.adapters_backward(s["dy"], s["x"], s["hidden"], s["ids"], s["a"], s["b"], s["scaling"], base=s["base"])
    if s["kind"] == "checkpoint":
        return T.checkpoint_unpack(*T.checkpoint_pack(s["x"]), s["dtype"])
    hidden, gate, up = T.silu_multiply_checkpoint(s["gate"], s["up"])
    return hidden, *T.swiglu_backward_checkpoint(gate, up, s["grad"])


def _spread(rows, ids, count):
    """rows [m, r] as [m, count * r]: each row in its adapter's columns, zeros elsewhere."""
    at = ids[:, None] == torch.arange(count, device="cuda", dtype=torch.int32)
    return torch.where(at[:, :, None], rows[:, None, :], torch.zeros((), device="cuda")).reshape(rows.shape[0], -1)


def _forward(s):
    count, r, k = s["a"].shape
    x, a, b = s["x"].float(), s["a"].float(), s["b"].float()
    every = (x @ a.reshape(count * r, k).T).reshape(-1, count, r)
    at = s["ids"][:, None] == torch.arange(count, device="cuda", dtype=torch.int32)
    mine = torch.where(at[:, :, None], every, torch.zeros((), device="cuda"))
    scaled = (mine * s["scaling"][:, None]).reshape(-1, count * r)
    y = (s["base"].float() + scaled @ b.transpose(1, 2).reshape(count * r, -1)).to(s["dtype"])
    return (y, mine.sum(1)) if s["keep"] else y


def _backward(s):
    count, r, k = s["a"].shape
    dy, a, b = s["dy"].float(), s["a"].float().reshape(count * r, k), s["b"].float()
    n = dy.shape[1]
    x = _unpack(*s["x"]) if isinstance(s["x"], tuple) else s["x"].float()
    every = (dy @ b.transpose(1, 2).reshape(count * r, n).T).reshape(-1, count, r)
    at = s["ids"][:, None] == torch.arange(count, device="cuda", dtype=torch.int32)
    g = (torch.where(at[:, :, None], every, torch.zeros((), device="cuda")) * s["scaling"][:, None]).reshape(-1, count * r)
    h = _spread(s["hidden"], s["ids"], count) * s["scaling"].repeat_interleave(r)
    dx = (s["base"].float() + g @ a).to(s["dtype"])
    grad_a = (g.T @ x).reshape(count, r, k).to(s["dtype"])
    grad_b = (dy.T @ h).reshape(n, count, r).transpose(0, 1).contiguous().to(s["dtype"])
    return dx, grad_a, grad_b


def _checkpoint(s):
    return _unpack(*_pack(s["x"])).to(s["dtype"])


def _gate(s):
    g, u, grad = s["gate"].float(), s["up"].float(), s["grad"].float()
    hidden = (g / (1 + torch.exp(-g)) * u).to(s["dtype"])
    g, u = _unpack(*_pack(s["gate"])), _unpack(*_pack(s["up"]))
    at = 1 / (1 + torch.exp(-g))
    return hidden, (grad * u * (at * (1 + g * (1 - at)))).to(s["dtype"]), (grad * (g * at)).to(s["dtype"])


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _kept(x):
    """What an activation [m, n] is after 8 bits: group by group, the scale and the quotient rounded to 32 bits as the definition says."""
    out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    for c in range(0, x.shape[1], GROUP):
        v = x[:, c:c + GROUP].double()
        scale = (v.abs().max(dim=1, keepdim=True).values / 127).float().double()
        scale[scale == 0] = 1
        out[:, c:c + GROUP] = torch.clamp(torch.round((v / scale).float().double()), -127, 127) * scale
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "checkpoint":
        return _kept(s["x"])
    if s["kind"] == "gate":
        g, u, d = s["gate"].double(), s["up"].double(), s["grad"].double()
        hidden = g * torch.sigmoid(g) * u
        g, u = _kept(s["gate"]), _kept(s["up"])
        sg = torch.sigmoid(g)
        return hidden, d * u * (sg + g * sg * (1 - sg)), d * g * sg
    a, b = s["a"].double(), s["b"].double()
    out = s["base"].double()
    if s["kind"] == "forward":
        hidden = torch.zeros(s["x"].shape[0], a.shape[1], dtype=torch.float64, device="cuda")
        for l in range(a.shape[0]):
            rows = (s["ids"] == l).nonzero()[:, 0]
            hidden[rows] = s["x"][rows].double() @ a[l].T
            out[rows] += float(s["scaling"][l]) * (hidden[rows] @ b[l].T)
        return (out, hidden) if s["keep"] else out
    grad_a, grad_b = torch.zeros_like(a), torch.zeros_like(b)
    for l in range(a.shape[0]):
        rows = (s["ids"] == l).nonzero()[:, 0]
        dy, scale = s["dy"][rows].double(), float(s["scaling"][l])
        if isinstance(s["x"], tuple):
            codes, scales = s["x"]
            x = codes[rows].double() * scales[rows].double().repeat_interleave(GROUP, dim=1)[:, :codes.shape[1]]
        else:
            x = s["x"][rows].double()
        g = scale * (dy @ b[l])
        out[rows] += g @ a[l]
        grad_a[l] = g.T @ x
        grad_b[l] = scale * (dy.T @ s["hidden"][rows].double())
    return out, grad_a, grad_b


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    m, n, e = case["m"], case["n"], 4 if case["dtype"] == "f32" else 2
    kept = m * n + 4 * m * -(-n // GROUP)
    if case["kind"] == "checkpoint":      # in, codes and scales out and in again, out
        return {"bytes": 2 * m * n * e + 2 * kept, "flops": 3.0 * m * n}
    if case["kind"] == "gate":            # gate, up, gradient in; hidden and both gradients out; both checkpoints out and in again
        return {"bytes": 6 * m * n * e + 4 * kept, "flops": 25.0 * m * n}
    k, r, count = case["k"], case["rank"], case["adapters"]
    runs = -(-m // case["run"])
    used = count * (1 - (1 - 1 / count) ** runs)
    factors = used * r * (k + n) * e
    if case["kind"] == "forward":
        return {"bytes": m * (k + 2 * n) * e + 4 * m + factors + (4 * m * r if case["keep"] else 0), "flops": 2.0 * m * r * (k + n)}
    x = m * k + 4 * m * -(-k // GROUP) if case["packed"] else m * k * e
    return {"bytes": m * (n + 2 * k) * e + x + 4 * m * (r + 1) + factors + count * r * (k + n) * e, "flops": 4.0 * m * r * (k + n)}
