"""Timed cases of the 8-bit floating point operators (`crane_b200.fp8`): rows to e4m3 codes with a scale for every 128 columns -- plain, behind
a root-mean-square norm with the residual's addition, behind a gated unit -- and the matrix product of such codes with weights that have a scale for
every block of 128 x 128.

Widths are those of the dense configurations in `crane_b200.synth` (2048 / 6144, 4096 / 12288) and odd ones.
"""
import math

import torch

own = False                      # False: elementary torch operations in 32 bits; True: the framework's kernels

G = 128                          # columns that share a scale
TOP = 448.0                      # largest e4m3 value
TINY = 2.0 ** -100               # largest magnitudes below this count as this
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "": 0}
F8 = torch.float8_e4m3fn


# ------------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one token's q, k and v projections: latency
        {"name": "linear_token", "op": "linear", "m": 1, "n": 4096, "k": 2048, "dtype": "f32", "add": False},
        # a server's decode round: gate and up projections for 33 sequences, bound by the weights' bytes
        {"name": "linear_batch", "op": "linear", "m": 33, "n": 24576, "k": 4096, "dtype": "bf16", "add": False},
        # the next turn of a conversation: a short message through the down projection, added to the residual stream
        {"name": "linear_turn", "op": "linear", "m": 77, "n": 4096, "k": 12288, "dtype": "f32", "add": True},
        # widths that end inside a block of 128 and inside 16 bytes
        {"name": "linear_odd", "op": "linear", "m": 130, "n": 1001, "k": 1037, "dtype": "f16", "add": False},
        # an ordinary prompt
        {"name": "linear_prompt", "op": "linear", "m": 1111, "n": 12288, "k": 2048, "dtype": "bf16", "add": False},
        # a long prompt, or several together, at the widest configuration
        {"name": "linear_long", "op": "linear", "m": 8192, "n": 24576, "k": 4096, "dtype": "bf16", "add": False},
        # the norm ahead of a token's projections, the residual stream in f32
        {"name": "norm_token", "op": "rms_norm", "m": 1, "k": 4096, "dtype": "f32", "residual": "f32"},
        # the same of a long prompt with everything in bf16
        {"name": "norm_long", "op": "rms_norm", "m": 8192, "k": 4096, "dtype": "bf16", "residual": "bf16"},
        # the gated unit of a decode round, and of a long prompt
        {"name": "gate_batch", "op": "silu_mul", "m": 33, "k": 12288, "dtype": "f32"},
        {"name": "gate_long", "op": "silu_mul", "m": 8192, "k": 12288, "dtype": "bf16"},
        # attention outputs ahead of the o projection: odd rows at a width that is no multiple of 128, and a long prompt's
        {"name": "rows_odd", "op": "quantize", "m": 77, "k": 1044, "dtype": "f16"},
        {"name": "rows_long", "op": "quantize", "m": 8191, "k": 4096, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "linear", "rms_norm", "silu_mul", "quantize"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    if op == "linear":
        case = {"op": op, "m": _log(rng, 1, 8192), "n": _log(rng, 16, 24576), "k": _log(rng, 64, 12288), "dtype": dtype, "add": rng.random() < 0.3}
        while case["m"] * case["n"] * case["k"] > 8192 * 24576 * 4096 or case["m"] * case["n"] * BYTES[dtype] > 8192 * 24576 * 2:
            case["m"] = max(1, case["m"] // 2)
        return case
    case = {"op": op, "m": _log(rng, 1, 8192), "k": _log(rng, 64, 12288), "dtype": dtype}
    if op == "rms_norm":
        case["residual"] = rng.choice(("", "f32", dtype))
    return case


def _blocks(n):
    return (n + G - 1) // G


def _codes(rows, cols, like, device="cuda"):
    """Room for [rows, cols] codes whose rows start on 16 bytes."""
    return torch.empty((rows, (cols + 15) // 16 * 16), dtype=like, device=device)[:, :cols]


def _scales(rows, cols, device="cuda"):
    """Room for a scale per row and 128 columns: those of a block lie side by side, 16 bytes the unit."""
    return torch.empty((_blocks(cols), (rows + 3) // 4 * 4), dtype=torch.float32, device=device)[:, :rows].t()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 1000003 + case["m"] * 7919 + case["k"] * 31 + case.get("n", 0))
    m, k, dt = case["m"], case["k"], DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    s = dict(case)
    if case["op"] == "linear":
        n = case["n"]
        # activations have a few columns that are much larger than the rest
        loud = 1 + 15 * (torch.rand(k, generator=gen, device="cuda") < 0.01)
        q, sc = _quantize(normal(m, k) * loud)
        s["x"], s["xs"] = _codes(m, k, F8), _scales(m, k)
        s["x"].copy_(q), s["xs"].copy_(sc)
        w = normal(n, k) / math.sqrt(k)
        pad = torch.zeros((_blocks(n) * G, _blocks(k) * G), device="cuda")
        pad[:n, :k] = w
        top = pad.view(_blocks(n), G, _blocks(k), G).abs().amax((1, 3))
        s["ws"] = top / TOP
        s["w"] = _codes(n, k, F8)
        s["w"].copy_((w / s["ws"].repeat_interleave(G, 0)[:n].repeat_interleave(G, 1)[:, :k]).clamp(-TOP, TOP).to(F8))
        s["add"] = normal(m, n).to(dt) if case["add"] else None
        s["out"] = torch.empty((m, n), dtype=dt, device="cuda")
        return s
    s["out"] = (_codes(m, k, F8), _scales(m, k))
    if case["op"] == "silu_mul":
        s["x"] = normal(m, 2 * k).mul_(1.5).to(dt)
        return s
    s["x"] = (normal(m, k) * (1 + 15 * (torch.rand(k, generator=gen, device="cuda") < 0.01))).to(dt)
    if case["op"] == "rms_norm":
        s["w"], s["eps"] = 1 + 0.2 * normal(k), 1e-6
        s["res"] = normal(m, k).mul_(3).to(DTYPES[case["residual"]]) if case["residual"] else None
        s["res_out"] = torch.empty_like(s["res"]) if case["residual"] else None
    return s


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _quantize(y):
    m, k = y.shape
    pad = torch.nn.functional.pad(y, (0, _blocks(k) * G - k)).view(m, _blocks(k), G)
    top = pad.abs().amax(2).clamp_min(TINY)
    codes = (pad * (TOP / top)[:, :, None]).clamp(-TOP, TOP).to(F8).view(m, _blocks(k) * G)[:, :k]
    return codes, top / TOP


def _plain(s):
    x = s["x"]
    if s["op"] == "linear":
        m, k = x.shape
        a = x.float() * s["xs"].repeat_interleave(G, 1)[:, :k]
        b = s["w"].float() * s["ws"].repeat_interleave(G, 0)[:s["n"]].repeat_interleave(G, 1)[:, :k]
        y = a @ b.t()
        return (y + s["add"].float() if s["add"] is not None else y).to(s["out"].dtype)
    if s["op"] == "quantize":
        return _quantize(x.float())
    if s["op"] == "silu_mul":
        g, u = x[:, :s["k"]].float(), x[:, s["k"]:].float()
        return _quantize(g / (1 + torch.exp(-g)) * u)
    if s["res"] is not None:
        res = (x.float() + s["res"].float()).to(s["res"].dtype)
        h = res.float()
    else:
        res, h = None, x.float()
    codes, scales = _quantize(h * torch.rsqrt((h * h).mean(1, keepdim=True) + s["eps"]) * s["w"])
    return codes, scales, res


def run(s):
    if not own:
        return _plain(s)
    from crane_b200 import fp8
    if s["op"] == "linear":
        return fp8.linear(s["x"], s["xs"], s["w"], s["ws"], add=s["add"], out=s["out"])
    if s["op"] == "quantize":
        return fp8.quantize(s["x"], out=s["out"])
    if s["op"] == "silu_mul":
        return fp8.silu_mul(s["x"], out=s["out"])
    codes, scales = fp8.rms_norm(s["x"], s["w"], s["eps"], residual=s["res"], residual_out=s["res_out"], out=s["out"])
    return codes, scales, s["res_out"]


def work(case):
    m, k, e = case["m"], case["k"], BYTES[case["dtype"]]
    rows = m * k + 4 * m * _blocks(k)                      # codes and scales
    if case["op"] == "linear":
        n = case["n"]
        return {"bytes": rows + n * k + 4 * _blocks(n) * _blocks(k) + m * n * e * (2 if case["add"] else 1), "flops": 2 * m * n * k}
    if case["op"] == "silu_mul":
        return {"bytes": rows + 2 * m * k * e, "flops": 8 * m * k}
    if case["op"] == "quantize":
        return {"bytes": rows + m * k * e, "flops": 3 * m * k}
    return {"bytes": rows + m * k * (e + 2 * BYTES[case["residual"]]) + 4 * k, "flops": 9 * m * k}


# --------------------------------------------------------------------------------------------------------- in 64 bits, from the definition
def _e4m3(v):
    """The nearest e4m3 value, ties to the even one: steps of 2^(e - 3) between 2^e and 2^(e + 1), of 2^-9 below 2^-6."""
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v.abs().clamp_min(2.0 ** -6))[1] - 4)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def _groups(y):
    codes, scales = torch.empty_like(y), []
    for b in range(0, y.shape[1], G):
        top = y[:, b:b + G].abs().amax(1).clamp_min(TINY)
        codes[:, b:b + G] = _e4m3(y[:, b:b + G] / top[:, None] * TOP)
        scales.append(top / TOP)
    return codes, torch.stack(scales, 1)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "linear":
        y = s["add"].double() if case["add"] else torch.zeros((case["m"], case["n"]), dtype=torch.float64, device="cuda")
        for b in range(_blocks(case["k"])):
            at = slice(b * G, (b + 1) * G)
            scale = s["ws"][:, b].double().repeat_interleave(G)[:case["n"]]
            y.addmm_(x[:, at] * s["xs"][:, b:b + 1].double(), (s["w"][:, at].double() * scale[:, None]).t())
        return y
    if case["op"] == "quantize":
        return _groups(x)
    if case["op"] == "silu_mul":
        g, u = x.split(case["k"], 1)
        return _groups(g * torch.sigmoid(g) * u)
    res = None
    if case["residual"]:                                    # the sum is kept in the residual's type
        res = (x + s["res"].double()).to(s["res"].dtype)
        x = res.double()
    codes, scales = _groups(x / torch.sqrt(x.square().mean(1, keepdim=True) + s["eps"]) * s["w"].double())
    return codes, scales, res.double() if res is not None else None
