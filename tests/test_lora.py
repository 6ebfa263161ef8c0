"""Low-rank adapters of many requests (crane_b200.lora, crane_b200_lora_linear of the C ABI).  Refusals on the CPU, results on the GPU (-m gpu) against the formula in 64 bits.

Tolerance per output, fixed ahead of the first run; t = A x, S = |scale| |B| (|A| |x|), all in absolute values:
  t        16-bit types: products exact, K of them summed in f32 in any order: (K / 8 + 48) 2^-23 of |A| |x| (sums of 16 products, then up to 8 warps and 8 CTAs);
           f32 rows: tf32 parts of both, 3 2^-22 of each product more
  t parts  two of the weights' type: bf16 2^-17, f16 2^-22 (of the row's largest: elements below 2^-28 of it to 2^-39), tf32 2^-22; f32 weights' own parts 2^-22
  out      rank products summed in f32, (rank / 8 + 16) 2^-23; the addition, 2^-24 of the result; half a step of its type."""
import math

import pytest
import torch

import crane_b200
from crane_b200 import CraneB200Error

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
PAIRS = [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")]


def lib():
    import __graft_entry__
    __graft_entry__.build()
    return crane_b200.load_library()


P = 1 << 20            # an address that is never used: every call below is refused by its numbers


@pytest.mark.parametrize("change, said", [
    ({"dtype": 3}, "type 3"), ({"w_dtype": 9}, "type 9"), ({"dtype": 1}, "their own type"), ({"rank": 0}, "rank = 0"), ({"rank": 129}, "rank = 129"), ({"k": 0}, "k = 0"),
    ({"adapters": 0}, "adapters"), ({"m": 1 << 40}, "m ="), ({"n": 1 << 33}, "n ="), ({"x": None}, "x is NULL"), ({"a": None}, "a is NULL"), ({"b": P + 2}, "b is not aligned"),
    ({"which": None}, "which"), ({"which": P + 1}, "which"), ({"scales": P + 2}, "scales"), ({"out": None}, "out"), ({"ldx": 7}, "7 apart"), ({"ldo": 5}, "5 apart"),
    ({"ldadd": 5}, "add"), ({"add": 4 * P, "out": 4 * P, "ldadd": 300}, "add is out"), ({"out": P}, "x is out")])
def test_calls_are_refused_by_their_numbers(change, said):
    a = {"device": 0, "x": P, "ldx": 64, "dtype": 0, "a": P, "b": P, "w_dtype": 0, "adapters": 3, "rank": 8, "which": P, "scales": None, "add": 2 * P, "ldadd": 200, "out": 3 * P, "ldo": 200,
         "m": 4, "n": 200, "k": 64, "stream": None}
    a.update(change)
    assert lib().crane_b200_lora_linear(*a.values()) in (crane_b200.INVALID_ARG, crane_b200.UNSUPPORTED)
    assert said in crane_b200.load_library().crane_b200_device_last_error().decode()


def test_tensors_are_refused():
    from crane_b200 import lora
    x = torch.zeros((2, 8))
    with pytest.raises(CraneB200Error, match="CUDA"):
        lora.linear(x, x[None], x[None], torch.zeros(2, dtype=torch.int32))


# ------------------------------------------------------------------------------------------------------------------ results
def gen_of(*key):
    import zlib
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def reference(x, a, b, which, scales, add):
    m, n, k, rank = x.shape[0], b.shape[1], x.shape[1], a.shape[1]
    y = torch.zeros((m, n), dtype=torch.float64, device="cuda") if add is None else add.double()
    off = torch.zeros_like(y)
    for w in set(which.tolist()):
        if not 0 <= w < a.shape[0]:
            continue
        at = which == w
        s = 1.0 if scales is None else float(scales[w])
        aw, bw, xs = a[w].double(), b[w].double(), x[at].double()
        t, size = xs @ aw.t(), xs.abs() @ aw.abs().t()
        y[at] += s * (t @ bw.t())
        dt = (k / 8 + 48) * 2.0 ** -23 * size + (3 * 2.0 ** -22 * size if x.dtype == torch.float32 else 0)
        part = 2.0 ** -17 if b.dtype == torch.bfloat16 and x.dtype != torch.float32 else 2.0 ** -21
        dt = dt + part * t.abs() + 2.0 ** -39 * t.abs().amax(1, keepdim=True)
        off[at] = abs(s) * ((dt @ bw.abs().t()) + (rank / 8 + 16) * 2.0 ** -23 * ((t.abs() + dt) @ bw.abs().t()))
    return y, off


def check(got, ref):
    y, off = ref
    half = torch.finfo(got.dtype).eps / 2
    lim = off + 2.0 ** -24 * y.abs() + half * (y.abs() + off) + (2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -149)
    top = torch.finfo(got.dtype).max
    edge = top + top * half / (2 - 2 * half)                            # half a step above the largest value: from there on the nearest is infinity (f16: 65 504 and 65 520)
    over = torch.isinf(got) & (torch.sign(got.double()) == torch.sign(y)) & (y.abs() + off >= edge)
    err = torch.where(over, 0.0, (got.double() - y).abs())
    assert bool((err <= lim).all()), (int((err > lim).sum()), float((err / lim).max()))


def problem(g, dt, wt, m, n, k, rank, adapters, order):
    x = (torch.randn((m, k), generator=g, device="cuda") * torch.exp(2 * torch.randn((m, 1), generator=g, device="cuda"))).to(TYPES[dt])
    a = (torch.randn((adapters, rank, k), generator=g, device="cuda") / math.sqrt(k)).to(TYPES[wt])
    b = torch.randn((adapters, n, rank), generator=g, device="cuda").to(TYPES[wt])
    scales = torch.randn(adapters, generator=g, device="cuda")
    which = torch.randint(-1, adapters + 1, (m,), generator=g, device="cuda").to(torch.int32)
    if order == "runs":
        which = which.sort().values
    elif order == "one":
        which.fill_(adapters - 1)
    elif order == "none":
        which.fill_(-2 ** 31)
    add = torch.randn((m, n), generator=g, device="cuda").to(TYPES[dt])
    return x, a, b, which, scales, add


SIZES = [  # rows, n, k, rank, adapters, order
    (1, 8, 8, 8, 1, "one"), (1, 1, 1, 1, 1, "one"), (1, 4096, 2048, 16, 3, "one"), (5, 33, 77, 3, 4, "any"), (33, 1000, 520, 16, 9, "any"), (64, 264, 1024, 64, 2, "any"),
    (65, 96, 64, 17, 5, "any"), (256, 512, 256, 128, 3, "any"), (257, 512, 256, 128, 3, "any"), (257, 136, 328, 8, 40, "any"), (300, 1001, 1037, 40, 4, "runs"), (513, 2048, 1536, 32, 5, "runs"),
    (20, 72, 64, 8, 2, "none"), (400, 72, 64, 8, 2, "none"), (1000, 24, 40, 100, 1, "one"), (2500, 640, 128, 64, 6, "runs"),
    (384, 512, 256, 128, 3, "any"), (385, 512, 256, 128, 3, "any"), (390, 136, 328, 8, 40, "any"), (450, 1001, 1037, 40, 4, "runs"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt, wt", PAIRS)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "-".join(map(str, s)))
def test_adapters(size, dt, wt):
    from crane_b200 import lora
    m, n, k, rank, adapters, order = size
    x, a, b, which, scales, add = problem(gen_of(size, dt, wt), dt, wt, *size)
    ref = reference(x, a, b, which, scales, add)
    check(lora.linear(x, a, b, which, scales=scales, add=add), ref)
    y = add.clone()
    assert lora.linear(x, a, b, which, scales=scales, add=y, out=y) is y
    check(y, ref)
    check(lora.linear(x, a, b, which), reference(x, a, b, which, None, None))


@pytest.mark.gpu
@pytest.mark.parametrize("dt, wt", PAIRS)
def test_rows_on_any_boundary(dt, wt):
    """Rows at any distance, off 16 bytes too; columns beside the result's stay."""
    from crane_b200 import lora
    g = gen_of("strides", dt, wt)
    for m in (9, 300):
        x, a, b, which, scales, add = problem(g, dt, wt, m, 64, 96, 8, 3, "runs")
        for off in (1, 8):
            wide, room, base = (torch.full((m, w + 24), 3.0, dtype=TYPES[dt], device="cuda") for w in (96, 64, 64))
            wide[:, off:off + 96], base[:, off:off + 64] = x, add
            out = room[:, off:off + 64]
            lora.linear(wide[:, off:off + 96], a, b, which, scales=scales, add=base[:, off:off + 64], out=out)
            check(out, reference(x, a, b, which, scales, add))
            assert (room[:, :off] == 3).all() and (room[:, off + 64:] == 3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [7, 300])
def test_infinities_and_nan_stay_in_their_rows(m):
    from crane_b200 import lora
    for dt, wt in PAIRS:
        x, a, b, which, scales, add = problem(gen_of("inf", dt, wt, m), dt, wt, m, 40, 64, 8, 2, "one")
        which[0], which[m - 1] = -1, 0
        a[0, 0, 0] = math.nan                                           # of an adapter that the last row alone uses
        x[0], x[1, 3], x[2, 5] = math.nan, math.nan, math.inf
        y = lora.linear(x, a, b, which, scales=scales, add=add)
        assert torch.equal(y[0], add[0]) and torch.isnan(y[1]).all() and not torch.isfinite(y[2]).any() and torch.isnan(y[m - 1]).all()
        check(y[3:m - 1], tuple(t[3:m - 1] for t in reference(x, a, b, which, scales, add)))


TILES = [(2048, 72, 40, 24, 3, "any"), (2100, 1000, 520, 64, 40, "runs"), (3001, 520, 2048, 40, 5, "runs"), (2048, 8, 8, 32, 1, "one"), (4100, 136, 1096, 56, 30, "any"),
         (2177, 4096, 1024, 32, 7, "runs"), (2100, 72, 64, 32, 2, "none"), (6000, 640, 256, 24, 300, "runs")]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("size", TILES, ids=lambda s: "-".join(map(str, s)))
def test_adapters_of_prompts(size, dt):
    from crane_b200 import lora
    x, a, b, which, scales, add = problem(gen_of("tiles", size, dt), dt, dt, *size)
    ref = reference(x, a, b, which, scales, add)
    y = lora.linear(x, a, b, which, scales=scales, add=add)
    check(y, ref)
    check(lora.linear(x, a, b, which), reference(x, a, b, which, None, None))
    m, n, k = size[:3]                                                  # rows further apart, columns beside the result's stay, in place, other rows not finite
    wide, room = torch.full((m, k + 16), math.nan, dtype=TYPES[dt], device="cuda"), torch.full((m, n + 24), 3.0, dtype=TYPES[dt], device="cuda")
    wide[:, 8:8 + k], room[:, 16:16 + n] = x, add
    out = room[:, 16:16 + n]
    bad = [5, m // 2, m - 1]
    wide[bad[0]], wide[bad[1], 9], wide[bad[2], 10] = math.nan, math.inf, -math.inf
    lora.linear(wide[:, 8:8 + k], a, b, which, scales=scales, add=out, out=out)
    rest = torch.ones(m, dtype=torch.bool, device="cuda")
    rest[bad] = False
    assert torch.equal(out[rest], y[rest]) and (room[:, :16] == 3).all() and (room[:, 16 + n:] == 3).all()
    for i in bad:
        assert torch.equal(out[i], add[i]) if not 0 <= int(which[i]) < a.shape[0] else not torch.isfinite(out[i]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt, wt", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("size", [(390, 72, 64, 8, 300), (640, 136, 96, 32, 64), (2048, 136, 72, 24, 200), (2500, 264, 64, 64, 1), (3000, 72, 128, 40, 127), (5000, 72, 64, 64, 500)],
                         ids=lambda s: "-".join(map(str, s)))
def test_adapters_in_any_order_are_dealt_out_to_the_clusters_of_a_tile(size, dt, wt):
    """Up to as many adapters as a tile has rows, more and fewer than it has clusters, rows without one among them: every row once, the same bits as by itself among its own."""
    from crane_b200 import lora
    m, n, k, rank, adapters = size
    x, a, b, which, scales, add = problem(gen_of("dealt", size, dt), dt, wt, m, n, k, rank, adapters, "any")
    y = add.clone()
    lora.linear(x, a, b, which, scales=scales, add=y, out=y)
    check(y, reference(x, a, b, which, scales, add))
    assert torch.equal(lora.linear(x, a, b, which, scales=scales, add=add), y)
    some = int(which[m // 2])
    alone = torch.where(which == some, which, -1)                       # the others have none now
    z = lora.linear(x, a, b, alone, scales=scales, add=add)
    assert torch.equal(z[which == some], y[which == some]) and torch.equal(z[which != some], add[which != some])


@pytest.mark.gpu
def test_prompts_repeat_in_graphs_and_on_streams():
    from crane_b200 import lora
    x, a, b, which, scales, add = problem(gen_of("tiles repeat"), "bf16", "bf16", 2300, 1032, 1024, 64, 5, "runs")
    one = lora.linear(x, a, b, which, scales=scales, add=add)
    outs = []
    for st in [torch.cuda.Stream() for _ in range(3)] * 3:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            outs.append(lora.linear(x, a, b, which, scales=scales, add=add))
    torch.cuda.synchronize()
    assert all(torch.equal(one, o) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = lora.linear(x, a, b, which, scales=scales, add=add)
    for i in range(3):
        which.copy_(which.flip(0) if i else which[torch.randperm(2300, generator=gen_of("order"), device="cuda")])
        graph.replay()
        check(y, reference(x, a, b, which, scales, add))


@pytest.mark.gpu
def test_results_repeat_and_calls_share_nothing():
    from crane_b200 import lora
    x, a, b, which, scales, add = problem(gen_of("repeat"), "bf16", "bf16", 100, 520, 1024, 16, 5, "any")
    one = lora.linear(x, a, b, which, scales=scales, add=add)
    outs = []
    for st in [torch.cuda.Stream() for _ in range(3)] * 3:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            outs.append(lora.linear(x, a, b, which, scales=scales, add=add))
    torch.cuda.synchronize()
    assert all(torch.equal(one, o) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = lora.linear(x, a, b, which, scales=scales, add=add)
    for _ in range(3):
        which.copy_(which.flip(0) if _ else which.roll(7))
        graph.replay()
        check(y, reference(x, a, b, which, scales, add))


@pytest.mark.gpu
def test_beside_a_shared_projection():
    """What a round runs: an 8-bit linear for all rows, each request's adapter on top, in a graph."""
    from crane_b200 import fp8, lora
    g = gen_of("beside")
    x, a, b, which, scales, _ = problem(g, "bf16", "bf16", 33, 384, 256, 16, 4, "any")
    w = fp8.rows(384, 256)[0]
    w.copy_((torch.randn((384, 256), generator=g, device="cuda") * 50).clamp(-448, 448).to(fp8.CODES))
    ws = torch.rand((3, 2), generator=g, device="cuda") * 1e-3
    codes, cs = fp8.quantize(x)
    shared = fp8.linear(codes, cs, w, ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        codes, cs = fp8.quantize(x)
        y = fp8.linear(codes, cs, w, ws)
        lora.linear(x, a, b, which, scales=scales, add=y, out=y)
    graph.replay()
    check(y, reference(x, a, b, which, scales, shared))
