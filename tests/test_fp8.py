"""Linears in 8-bit floating point (crane_b200.fp8, crane_b200_fp8_* of the C ABI): rows to e4m3 codes, codes x codes^T.  Refusals on the CPU, numbers on the GPU (-m gpu).

References are the formulas in 64 bits.  Tolerances, fixed ahead of the first run:
  plain codes and scales   the same f32 operations in torch on the CPU, bit for bit (two IEEE divisions, a product, a rounding to nearest even)
  scales behind a norm or a gated unit   relative 2^-17: f32 sums of squares in trees (width 2^15: (8 + 15) 2^-24), rsqrtf, expf and a division of 2 ulp each, a few products, 448
  codes behind them        a code stands within half an e4m3 step of the quotient, the quotient being 2^-17 of itself off; the steps are 2^-3 of a binade's lower end, 2^-9 below 2^-6
  linears                  block sums of 128 exact products added in f32 in any order, each addition off by at most 2^-23 of the running sum's bound, then one product and one
                           addition for each of the KB blocks: (128 + KB + 4) 2^-23 of A = sum |x| |w|; then the result's own rounding, eps / 2 of its value (f16: and half of its
                           least step, 2^-25), behind the addition of `add` in f32, 2^-24 of the sum"""
import ctypes as C
import math
import zlib

import numpy as np
import pytest
import torch

import crane_b200
from crane_b200 import CraneB200Error

F8 = torch.float8_e4m3fn
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TINY = 2.0 ** -100


def blocks(n):
    return (n + 127) // 128


# -------------------------------------------------------------------------------------------------------------- refusals, without a GPU
def lib():
    import __graft_entry__
    __graft_entry__.build()
    return crane_b200.load_library()


def why():
    return (crane_b200.load_library().crane_b200_fp8_last_error() or b"").decode()


P = 1 << 20            # an address that is never used: every call below is refused by its numbers


@pytest.mark.parametrize("change, said", [
    ({"dtype": 3}, "type 3"), ({"k": 0}, "k = 0"), ({"m": 1 << 40}, "m ="), ({"x": None}, "x is NULL"), ({"ldx": 99}, "99 apart"), ({"x": P + 1}, "not aligned"),
    ({"codes": None}, "NULL"), ({"scales": None}, "NULL"), ({"codes": P + 8}, "16-byte"), ({"ld": 120}, "16-byte"), ({"ld": 96}, "16-byte"), ({"lds": 3}, "scales 3 apart"),
    ({"scales": P + 2}, "scales")])
def test_rows_are_refused_by_their_numbers(change, said):
    a = {"device": 0, "x": P, "dtype": 0, "ldx": 100, "m": 4, "k": 100, "codes": P, "ld": 112, "scales": P, "lds": 4, "stream": None}
    a.update(change)
    assert lib().crane_b200_fp8_quantize(*a.values()) == crane_b200.INVALID_ARG and said in why()
    a["ldx"] *= 2
    assert lib().crane_b200_fp8_silu_mul(*a.values()) == crane_b200.INVALID_ARG and why()


@pytest.mark.parametrize("change, said", [
    ({"eps": -1.0}, "eps"), ({"eps": math.nan}, "eps"), ({"residual_out": None}, "come together"), ({"residual": None}, "come together"), ({"res_dtype": 7}, "residual"),
    ({"w": None}, "weight"), ({"w_dtype": -1}, "weight"), ({"ldr": 64}, "residual"), ({"ld": 100}, "16-byte")])
def test_norms_are_refused_by_their_numbers(change, said):
    a = {"device": 0, "x": P, "dtype": 1, "ldx": 100, "residual": P, "residual_out": P, "res_dtype": 0, "ldr": 100, "w": P, "w_dtype": 0, "eps": 1e-6, "m": 4, "k": 100,
         "codes": P, "ld": 112, "scales": P, "lds": 4, "stream": None}
    a.update(change)
    assert lib().crane_b200_fp8_rms_norm(*a.values()) == crane_b200.INVALID_ARG and said in why()


@pytest.mark.parametrize("change, said", [
    ({"x": None}, "x:"), ({"ldx": 100}, "x:"), ({"w": P + 4}, "w:"), ({"ldw": 96}, "w:"), ({"ws": None}, "w:"), ({"ldws": 1}, "w:"), ({"lds": 2}, "x:"), ({"k": 0}, "k = 0"),
    ({"n": 1 << 33}, "n ="), ({"out": None}, "out"), ({"ldo": 7}, "out"), ({"dtype": 9}, "out"), ({"ldadd": 1}, "add"), ({"add": P + 2}, "add")])
def test_linears_are_refused_by_their_numbers(change, said):
    a = {"device": 0, "x": P, "ldx": 144, "xs": P, "lds": 4, "w": P, "ldw": 144, "ws": P, "ldws": 2, "m": 4, "n": 8, "k": 130, "add": P, "ldadd": 8, "out": P, "dtype": 0, "ldo": 8,
         "stream": None}
    a.update(change)
    assert lib().crane_b200_fp8_linear(*a.values()) == crane_b200.INVALID_ARG and said in why()


def test_nothing_to_do_is_no_error_and_no_gpu_is():
    l = lib()
    assert l.crane_b200_fp8_quantize(0, None, 0, 0, 0, 5, None, 0, None, 0, None) == crane_b200.OK
    assert l.crane_b200_fp8_linear(0, None, 0, None, 0, None, 0, None, 0, 0, 4, 4, None, 0, None, 0, 0, None) == crane_b200.OK
    if not torch.cuda.is_available():
        assert l.crane_b200_fp8_quantize(0, P, 0, 100, 4, 100, P, 112, P, 4, None) == crane_b200.CUDA_ERROR and why()
        assert l.crane_b200_fp8_status(0, None) == crane_b200.CUDA_ERROR


def test_tensors_are_refused_without_a_gpu():
    from crane_b200 import fp8
    for call in (lambda: fp8.quantize(torch.zeros(2, 4)), lambda: fp8.silu_mul(np.zeros((2, 4))), lambda: fp8.rms_norm(torch.zeros(4), torch.zeros(4)),
                 lambda: fp8.linear(torch.zeros(2, 4).to(F8), None, None, None)):
        with pytest.raises(CraneB200Error) as e:
            call()
        assert e.value.code == crane_b200.INVALID_ARG


# ------------------------------------------------------------------------------------------------------------------ references
def plain_codes(y):
    """The formula in f32 on the CPU (numpy: IEEE divisions)."""
    y = y.float().cpu().numpy()
    m, k = y.shape
    pad = np.zeros((m, blocks(k) * 128), np.float32)
    pad[:, :k] = y
    a = np.maximum(np.abs(pad).reshape(m, -1, 128).max(2), np.float32(TINY))
    inv = np.float32(448) / a
    t = (pad.reshape(m, -1, 128) * inv[:, :, None]).reshape(m, -1)[:, :k]
    return torch.from_numpy(np.clip(t, -448, 448)).to(F8), torch.from_numpy(a / np.float32(448))


def step_of(t):
    return torch.ldexp(torch.ones_like(t), torch.frexp(t.abs().clamp_min(2.0 ** -6))[1] - 4)


def check_rows(got, y, k):
    """Codes and scales against the rows y in 64 bits."""
    codes, scales = got[0].double().cpu(), got[1].double().cpu()
    y = y.double().cpu()
    m = y.shape[0]
    pad = torch.nn.functional.pad(y, (0, blocks(k) * 128 - k)).view(m, -1, 128)
    a = pad.abs().amax(2).clamp_min(TINY)
    assert ((scales - a / 448).abs() <= 2.0 ** -17 * a / 448).all()
    t = (pad / a[:, :, None] * 448).view(m, -1)[:, :k]
    slack = 2.0 ** -16 * t.abs()                       # the row's values and the block's largest, 2^-17 each
    assert ((codes - t).abs() <= step_of(t.abs() + slack) / 2 + slack).all()


def rows_of(gen, m, k, dt, loud=True):
    x = torch.randn((m, k), generator=gen, device="cuda")
    if loud:
        x *= 1 + 15 * (torch.rand(k, generator=gen, device="cuda") < 0.02)
    return x.to(dt)


def gen_of(*seed):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(seed).encode()))


def strided(x, extra=0, off=0):
    """x's values in rows that lie `extra` elements further apart, `off` elements behind an allocation's start."""
    m, k = x.shape
    wide = torch.empty(m * (k + extra) + off, dtype=x.dtype, device=x.device)
    v = wide[off:].view(m, k + extra)[:, :k]
    v.copy_(x)
    return v


def e4m3(x):
    return x.clamp(-448, 448).to(F8)


def weights(gen, n, k):
    from crane_b200 import fp8
    w = fp8.rows(n, k)[0]
    w.copy_(e4m3(torch.randn((n, k), generator=gen, device="cuda") * 60))
    return w, torch.rand((blocks(n), blocks(k)), generator=gen, device="cuda") * 1e-3 + 1e-4


def linear_ref(x, xs, w, ws, add=None):
    """(result, bound of the f32 sums' error) in 64 bits."""
    m, k = x.shape
    n = w.shape[0]
    a = x.double() * xs.double().repeat_interleave(128, 1)[:, :k]
    b = w.double() * ws.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    y, size = a @ b.t(), a.abs() @ b.abs().t()
    off = (128 + blocks(k) + 4) * 2.0 ** -23 * size
    if add is not None:
        y = y + add.double()
        off = off + 2.0 ** -24 * y.abs()
    return y, off


def check_linear(out, ref):
    y, off = ref
    half = torch.finfo(out.dtype).eps / 2
    assert out.shape == y.shape
    bad = (out.double() - y).abs() > off + half * (y.abs() + off) + (2.0 ** -25 if out.dtype == torch.float16 else 0)
    assert not bad.any(), (int(bad.sum()), float(((out.double() - y).abs() / (off + 1e-300)).max()))


# ------------------------------------------------------------------------------------------------------------------------ rows
@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m, k", [(1, 1), (1, 7), (3, 8), (2, 127), (5, 128), (1, 129), (17, 136), (33, 1044), (7, 4096), (300, 1037), (2, 20000)])
def test_plain_rows(m, k, dt):
    from crane_b200 import fp8
    gen = gen_of("rows", m, k, dt)
    x = rows_of(gen, m, k, TYPES[dt])
    ref = plain_codes(x)
    for v in (x, strided(x, 3, 1), strided(x, 16, 0), x.repeat_interleave(2, 0)[::2]):
        out = fp8.rows(m, k)
        base = out[0].view(torch.uint8).as_strided((m, (k + 15) // 16 * 16), ((k + 15) // 16 * 16, 1))
        room = out[1].t().as_strided((blocks(k), (m + 3) // 4 * 4), ((m + 3) // 4 * 4, 1))
        base.fill_(77), room.fill_(-5)
        got = fp8.quantize(v, out=out)
        assert torch.equal(got[0].view(torch.uint8).cpu(), ref[0].view(torch.uint8)) and torch.equal(got[1].cpu(), ref[1])
        assert (base[:, k:] == 77).all()                                   # bytes behind the last column stay
        assert (room[:, m:] == -5).all()


@pytest.mark.gpu
def test_rows_of_extreme_values():
    """Empty blocks, subnormal ones, the types' largest values, infinities and NaN."""
    from crane_b200 import fp8
    x = torch.zeros((8, 256), device="cuda")
    x[1] = 1e-40
    x[2] = torch.finfo(torch.float32).max
    x[3, 5], x[3, 200] = 1e-30, -3e38
    x[4] = torch.linspace(-1, 1, 256, device="cuda") * 2.0 ** -100
    x[5, :128] = 448.0
    ref = plain_codes(x)
    got = fp8.quantize(x)
    assert torch.equal(got[0].view(torch.uint8).cpu(), ref[0].view(torch.uint8)) and torch.equal(got[1].cpu(), ref[1])
    assert (got[0][0].float() == 0).all() and torch.isfinite(got[1]).all()
    x[6, 3], x[6, 130], x[7, 0] = math.nan, -math.inf, math.inf
    codes, scales = fp8.quantize(x)
    back = codes.float() * scales.repeat_interleave(128, 1)
    assert torch.isnan(back[6, 3]) and (back[6, :3] == 0).all() and (back[6, 4:128] == 0).all()        # a NaN is its own
    assert torch.isinf(scales[6, 1]) and torch.isnan(back[6, 128:]).all() and torch.isnan(back[7, :128]).all() and (back[7, 128:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m, k", [(1, 1), (2, 4), (3, 128), (9, 129), (33, 1536), (5, 1036), (4, 12288)])
def test_gated_rows(m, k, dt):
    from crane_b200 import fp8
    gen = gen_of("gated", m, k, dt)
    x = rows_of(gen, m, 2 * k, TYPES[dt]) * 2
    g, u = x.double().split(k, 1)
    y = g / (1 + torch.exp(-g)) * u
    one = fp8.silu_mul(x)
    check_rows(one, y, k)
    two = fp8.silu_mul(strided(x, 5, 3))
    assert torch.equal(one[0].view(torch.uint8), two[0].view(torch.uint8)) and torch.equal(one[1], two[1])


@pytest.mark.gpu
def test_gates_of_extreme_values():
    """SiLU far out: -x e^x for large negative gates goes to zero, never to NaN."""
    from crane_b200 import fp8
    g = torch.tensor([-1e4, -200, -104, -88, -50, 0, 50, 88, 1e4, 3e38, -3e38, 1], device="cuda").repeat(11)[:128]
    u = torch.full((128,), 0.5, device="cuda")
    got = fp8.silu_mul(torch.cat([g, u])[None])
    check_rows(got, torch.where(g < -100, 0.0, g.double() * torch.sigmoid(g.double()))[None] * 0.5, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("res", ["", "same", "f32", "f16"])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m, k", [(1, 1), (3, 20), (9, 128), (8, 250), (5, 256), (17, 257), (6, 1037), (2, 2048), (33, 4096), (3, 8192), (2, 8200), (3, 16384), (2, 16400), (1, 20001)])
def test_norms(m, k, dt, res):
    from crane_b200 import fp8
    gen = gen_of("norm", m, k, dt, res)
    x = rows_of(gen, m, k, TYPES[dt])
    w = (1 + 0.2 * torch.randn(k, generator=gen, device="cuda")).to(TYPES[{"f32": "f32", "bf16": "bf16", "f16": "f32"}[dt]])
    h, r, kw = x, None, {}
    if res:
        rt = TYPES[dt if res == "same" else res]
        r = (3 * torch.randn((m, k), generator=gen, device="cuda")).to(rt)
        h = (x.double() + r.double()).to(rt) if rt != torch.float32 else x.float() + r     # (the sum of two such values is exact in 64 bits)
        keep, store = r.clone(), strided(r, 4, 0)
        kw = {"residual": strided(r, 4, 0), "residual_out": store}
    y = h.double() / torch.sqrt(h.double().square().mean(1, keepdim=True) + 1e-5) * w.double()
    got = fp8.rms_norm(x, w, 1e-5, **kw)
    check_rows(got, y, k)
    if res:
        assert torch.equal(store, h) and torch.equal(kw["residual"], keep)
        again = fp8.rms_norm(strided(x, 1, 1), w, 1e-5, residual=r)                        # in place, rows on odd boundaries
        assert torch.equal(r, h)
    else:
        again = fp8.rms_norm(strided(x, 1, 1), w, 1e-5)
    assert torch.equal(got[0].view(torch.uint8), again[0].view(torch.uint8)) and torch.equal(got[1], again[1])


@pytest.mark.gpu
def test_norm_of_zeros_and_infinities():
    from crane_b200 import fp8
    x = torch.zeros((3, 300), device="cuda")
    x[1, 7], x[2, 299] = math.inf, math.nan
    codes, scales = fp8.rms_norm(x, torch.ones(300, device="cuda"), 1e-6)
    back = codes.float() * scales.repeat_interleave(128, 1)[:, :300]
    assert (back[0] == 0).all() and torch.isnan(back[2]).all() and torch.isnan(back[1, 7])


@pytest.mark.gpu
@pytest.mark.parametrize("k", [1, 7, 8, 130, 519, 2049, 4099, 9001, 17001])
@pytest.mark.parametrize("dt", TYPES)
def test_rows_on_every_boundary(dt, k):
    """Rows from every offset inside 16 bytes, NaN between and around them: the bits of rows that lie together, and nothing between them is written."""
    from crane_b200 import fp8
    gen, t = gen_of("boundary", k, dt), TYPES[dt]
    x, gated, r = (rows_of(gen, 5, n, t) for n in (k, 2 * k, k))
    w = 1 + 0.2 * torch.randn(k, generator=gen, device="cuda")

    def among(v, off):
        wide = torch.full((5 * (v.shape[1] + 3) + off + 8,), math.nan, dtype=t, device="cuda")
        at = wide[off:off + 5 * (v.shape[1] + 3)].view(5, -1)[:, :v.shape[1]]
        at.copy_(v)
        return at, wide
    alike = lambda a, b: torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])  # noqa: E731
    plain, unit, sums = fp8.quantize(x), fp8.silu_mul(gated), (x.float() + r.float()).to(t)
    alone, normed = fp8.rms_norm(x, w, 1e-5), fp8.rms_norm(x, w, 1e-5, residual=r.clone())
    for off in range(8):
        xo, (ro, room) = among(x, off)[0], among(r, 7 - off)
        assert alike(fp8.quantize(xo), plain) and alike(fp8.silu_mul(among(gated, off)[0]), unit) and alike(fp8.rms_norm(xo, w, 1e-5), alone)
        assert alike(fp8.rms_norm(xo, w, 1e-5, residual=ro), normed)
        assert torch.equal(ro, sums) and int(torch.isnan(room).sum()) == room.numel() - 5 * k


@pytest.mark.gpu
@pytest.mark.parametrize("k", [300, 512, 9001, 9216, 17000])
def test_norm_whose_rows_times_weights_pass_f32(k):
    """x w lies outside of f32 where (x / rms) w does not: powers of two throughout, so y is 2^100 times the signs and every code the type's largest value."""
    from crane_b200 import fp8
    g = torch.Generator().manual_seed(k)
    signs = (torch.randint(0, 2, (3, k), generator=g) * 2 - 1).float()
    x = (signs * torch.tensor([2.0 ** 50, 2.0 ** 40, 2.0 ** -30])[:, None]).cuda()
    codes, scales = fp8.rms_norm(x, torch.full((k,), 2.0 ** 100, device="cuda"), 0.0)
    assert torch.equal(codes.float().cpu(), signs * 448)
    assert ((scales.cpu() * 448 / 2.0 ** 100 - 1).abs() < 2.0 ** -20).all()            # (a rsqrt of 2 ulp, a product and a quotient; the row's sum of equal squares is exact to k 2^-24 / k)


# --------------------------------------------------------------------------------------------------------------------- linears
SHAPES = [(1, 1, 1), (1, 128, 128), (1, 4096, 2048), (2, 130, 16), (3, 200, 256), (8, 1000, 1037), (15, 129, 4096), (16, 256, 1024), (17, 384, 2048), (31, 1001, 129), (32, 512, 640),
          (33, 24576, 256), (48, 127, 12288), (63, 640, 384), (64, 2048, 1040), (65, 640, 512), (77, 4096, 1536), (127, 300, 300), (128, 128, 4096), (129, 256, 128), (130, 1001, 1037),
          (200, 513, 2048), (255, 1024, 1024), (257, 129, 12288), (300, 4100, 520), (513, 1280, 640), (1111, 1280, 2048), (2048, 2048, 256), (2100, 4224, 400)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m, n, k", SHAPES)
def test_linears(m, n, k, dt):
    from crane_b200 import fp8
    gen = gen_of("linear", m, n, k, dt)
    x, xs = fp8.quantize(rows_of(gen, m, k, torch.float32))
    w, ws = weights(gen, n, k)
    ref = linear_ref(x, xs, w, ws)
    one = fp8.linear(x, xs, w, ws, dtype=TYPES[dt])
    check_linear(one, ref)
    assert torch.equal(one, fp8.linear(x, xs, w, ws, dtype=TYPES[dt]))                     # the order of the sums is fixed
    # results behind odd strides, an addend of its own, and in place
    add = torch.randn((m, n), generator=gen, device="cuda").to(TYPES[dt])
    wide = torch.full((m + 1, n + 3), 99.0, device="cuda").to(TYPES[dt])
    out = fp8.linear(x, xs, w, ws, add=strided(add, 1, 1), out=wide[:m, 1:n + 1])
    check_linear(out, linear_ref(x, xs, w, ws, add))
    assert (wide[m] == 99).all() and (wide[:, 0] == 99).all() and (wide[:, n + 1:] == 99).all()
    assert torch.equal(fp8.linear(x, xs, w, ws, add=add, out=add), out)
    fp8.status()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 20, 100, 600])
def test_linear_of_wide_strides_and_codes_of_every_value(m):
    """Codes at odd row distances (multiples of 16), all finite code values, block scales far apart, columns behind the last that hold NaN."""
    from crane_b200 import fp8
    gen = gen_of("codes", m)
    n, k = 333, 300
    bits = torch.randint(0, 254, (m + n, k + 52), generator=gen, device="cuda")
    bits = (bits + (bits >= 127)).to(torch.uint8)                                          # all but 127 and 255, the NaNs
    bits[:, k:] = 127
    x, w = bits[:m, :k].view(F8), bits[m:, :k].view(F8)
    xs = torch.exp2(torch.randint(-20, 20, (3, m + 5), generator=gen, device="cuda").float())[:, :m].t()
    ws = torch.exp2(torch.randint(-20, 20, (3, 9), generator=gen, device="cuda").float())[:, :3]
    check_linear(fp8.linear(x, xs, w, ws, dtype=torch.float32), linear_ref(x, xs, w, ws))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m, n, k", [(1, 100, 256), (60, 1001, 256), (100, 77, 640), (129, 260, 128), (700, 1001, 256), (1300, 2085, 384), (4900, 4200, 128)])
def test_linear_leaves_what_lies_around_its_rows(m, n, k, dt):
    """Results in rows on 16-byte boundaries that are wider than the result, on every route: columns behind the last and the rows around stay as they are."""
    from crane_b200 import fp8
    gen = gen_of("around", m, n, k, dt)
    x, xs = fp8.quantize(rows_of(gen, m, k, torch.float32))
    w, ws = weights(gen, n, k)
    wide = torch.full((m + 2, (n + 15) // 8 * 8), 99.0, device="cuda", dtype=TYPES[dt])
    out = fp8.linear(x, xs, w, ws, out=wide[1:m + 1, :n])
    check_linear(out, linear_ref(x, xs, w, ws))
    assert (wide[0] == 99).all() and (wide[m + 1] == 99).all() and (wide[:, n:] == 99).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m, n, k", [(60, 1001, 256), (129, 260, 128), (700, 1001, 256), (1300, 2085, 384), (2600, 4198, 130), (4900, 4200, 128)])
def test_linear_of_added_rows_on_every_boundary(m, n, k, dt):
    """An addend in rows on 16-byte boundaries, ragged at their ends, in place and apart, gives the bits of one on odd boundaries; nothing around the rows is written."""
    from crane_b200 import fp8
    gen = gen_of("added", m, n, k, dt)
    x, xs = fp8.quantize(rows_of(gen, m, k, torch.float32))
    w, ws = weights(gen, n, k)
    add = (3 * torch.randn((m, n), generator=gen, device="cuda")).to(TYPES[dt])
    want = fp8.linear(x, xs, w, ws, add=strided(add, 1, 1), out=strided(add, 2 + n % 2, 1))
    check_linear(want, linear_ref(x, xs, w, ws, add))
    wide = torch.full((m + 2, (n + 15) // 8 * 8), 99.0, device="cuda", dtype=TYPES[dt])
    rows = wide[1:m + 1, :n]
    rows.copy_(add)
    assert torch.equal(fp8.linear(x, xs, w, ws, add=rows, out=torch.empty_like(wide)[:m, :n]), want)
    assert torch.equal(fp8.linear(x, xs, w, ws, add=rows, out=rows), want)
    assert (wide[0] == 99).all() and (wide[m + 1] == 99).all() and (wide[:, n:] == 99).all()
    fp8.status()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40, 100, 700])
def test_linear_keeps_nan_and_infinity_in_their_rows(m):
    from crane_b200 import fp8
    gen = gen_of("nan", m)
    n, k = 260, 256
    h = rows_of(gen, m, k, torch.float32)
    w, ws = weights(gen, n, k)
    good = fp8.linear(*fp8.quantize(h), w, ws, dtype=torch.float32)
    h[m // 2, 3] = math.nan
    if m > 1:
        h[0, 200] = math.inf
    got = fp8.linear(*fp8.quantize(h), w, ws, dtype=torch.float32)
    rows = torch.ones(m, dtype=torch.bool, device="cuda")
    rows[m // 2] = rows[0] = False
    assert torch.isnan(got[m // 2]).all() and (m == 1 or torch.isnan(got[0]).all()) and torch.equal(got[rows], good[rows])
    w.view(torch.uint8)[5, 7] = 127
    got = fp8.linear(*fp8.quantize(rows_of(gen, m, k, torch.float32)), w, ws, dtype=torch.float32)
    assert torch.isnan(got[:, 5]).all() and torch.isfinite(got[:, :5]).all() and torch.isfinite(got[:, 6:]).all()


# ------------------------------------------------------------------------------------------------------- together, streams and graphs
def layer(x, stream, p):
    """One pre-norm feed-forward sublayer and the rows of an attention output through a square linear, as a program runs them."""
    from crane_b200 import fp8
    c = fp8.rms_norm(x, p["norm"], 1e-6, residual=stream)
    gu = fp8.linear(*c, *p["gu"])
    stream = fp8.linear(*fp8.silu_mul(gu), *p["down"], add=stream, out=stream)
    return fp8.linear(*fp8.quantize(stream), *p["o"], dtype=torch.float32)


def layer_params(gen, h, i):
    return {"norm": 1 + 0.1 * torch.randn(h, generator=gen, device="cuda"), "gu": weights(gen, 2 * i, h), "down": weights(gen, h, i), "o": weights(gen, h, h)}


def layer_ref(x, stream, p):
    """The same in 64 bits, each kernel on what the one ahead of it gave: every step is checked, none of the errors piles up."""
    from crane_b200 import fp8
    s0 = stream.clone()
    c = fp8.rms_norm(x, p["norm"], 1e-6, residual=stream)
    h = x.float() + s0
    assert torch.equal(stream, h)
    check_rows(c, h.double() / torch.sqrt(h.double().square().mean(1, keepdim=True) + 1e-6) * p["norm"].double(), h.shape[1])
    gu = fp8.linear(*c, *p["gu"])
    check_linear(gu, linear_ref(*c, *p["gu"]))
    c = fp8.silu_mul(gu)
    g, u = gu.double().chunk(2, 1)
    check_rows(c, g * torch.sigmoid(g) * u, g.shape[1])
    s1 = fp8.linear(*c, *p["down"], add=stream)  if stream.dtype == torch.bfloat16 else fp8.linear(*c, *p["down"], add=stream, dtype=torch.float32)
    check_linear(s1, linear_ref(*c, *p["down"], stream))
    c = fp8.quantize(s1)
    out = fp8.linear(*c, *p["o"], dtype=torch.float32)
    check_linear(out, linear_ref(*c, *p["o"]))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 7, 50, 333])
def test_a_layer_of_them(m):
    gen = gen_of("layer", m)
    p = layer_params(gen, 512, 1280)
    x, s = rows_of(gen, m, 512, torch.bfloat16), rows_of(gen, m, 512, torch.float32)
    ref = layer_ref(x, s.clone(), p)
    got = layer(x, s, p)
    assert torch.equal(got, ref)                           # (the same kernels back to back, where one may start before the one ahead has ended)


@pytest.mark.gpu
def test_streams_threads_and_graphs():
    """The same layer captured and replayed on new inputs, twice into graphs that run at the same time, and on streams of several threads: every result is the plain run's."""
    import threading
    gen = gen_of("graphs")
    p = layer_params(gen, 512, 768)
    ins = [(rows_of(gen, 40, 512, torch.bfloat16), rows_of(gen, 40, 512, torch.float32)) for _ in range(6)]
    want = [layer(x, s.clone(), p) for x, s in ins]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        side = torch.cuda.Stream()
        bx, bs = torch.empty_like(ins[0][0]), torch.empty_like(ins[0][1])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = layer(bx, bs, p)
        graphs.append((g, side, bx, bs, out))
    for i in range(0, 6, 2):
        torch.cuda.synchronize()
        for j, (g, side, bx, bs, out) in enumerate(graphs):
            with torch.cuda.stream(side):
                bx.copy_(ins[i + j][0]), bs.copy_(ins[i + j][1])
                g.replay()
        torch.cuda.synchronize()
        for j in range(2):
            assert torch.equal(graphs[j][4], want[i + j])
    got, errors = [None] * 6, []

    def work(t):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(t, 6, 3):
                    for _ in range(5):
                        got[i] = layer(ins[i][0], ins[i][1].clone(), p)
                torch.cuda.current_stream().synchronize()
        except Exception as e:                            # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(t,)) for t in range(3)]
    [t.start() for t in threads], [t.join() for t in threads]
    assert not errors and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_many_rows_of_few_columns():
    """More tiles of rows than a grid's second dimension has room for, offsets past 2^31, and the largest sizes that are taken."""
    from crane_b200 import fp8
    gen = gen_of("many")
    m, n, k = 4_300_000, 3, 16
    x, xs = fp8.quantize(rows_of(gen, m, k, torch.bfloat16, loud=False))
    w, ws = weights(gen, n, k)
    check_linear(fp8.linear(x, xs, w, ws), linear_ref(x, xs, w, ws))
    # rows that lie far apart: the last ones' offsets pass 2^31 elements
    far = torch.zeros(3 * 2 ** 30 + 4096, dtype=torch.bfloat16, device="cuda").as_strided((4, 256), (2 ** 30, 1))
    far.copy_(rows_of(gen, 4, 256, torch.bfloat16))
    near = far.clone()
    for a, b in zip(fp8.quantize(far), fp8.quantize(near)):
        assert torch.equal(a.view(torch.uint8) if a.dtype == F8 else a, b.view(torch.uint8) if b.dtype == F8 else b)
    weight = torch.ones(256, device="cuda")
    for a, b in zip(fp8.rms_norm(near, weight, residual=far, residual_out=far), fp8.rms_norm(near, weight, residual=near.clone())):
        assert torch.equal(a.view(torch.uint8) if a.dtype == F8 else a, b.view(torch.uint8) if b.dtype == F8 else b)
    c, s = fp8.quantize(near)
    w, ws = weights(gen, 130, 256)
    out = far.as_strided((4, 130), (2 ** 30, 1))
    fp8.linear(c, s, w, ws, out=out)
    assert torch.equal(out, fp8.linear(c, s, w, ws))
    del far, out


FIRST_IN_A_CAPTURE = """
import sys, torch
sys.path[:0] = [{root!r}, {tests!r}]
import test_fp8 as t
from crane_b200 import fp8
gen = t.gen_of("first")
p = t.layer_params(gen, 512, 768)
rows = {{m: (t.rows_of(gen, m, 512, torch.bfloat16), t.rows_of(gen, m, 512, torch.float32)) for m in (1, 40, 300)}}
keep = {{m: s.clone() for m, (x, s) in rows.items()}}
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = {{m: t.layer(x, s, p) for m, (x, s) in rows.items()}}
for m, (x, s) in rows.items():
    s.copy_(keep[m])
g.replay()
torch.cuda.synchronize()
for m, (x, s) in rows.items():
    assert torch.equal(out[m], t.layer(x, keep[m].clone(), p)), m
fp8.status()
print("fine")
"""


@pytest.mark.gpu
def test_first_calls_of_a_process_inside_a_capture():
    """The first use of every kernel, and of the stream, happens while torch captures in its strict mode."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", FIRST_IN_A_CAPTURE.format(root=os.path.dirname(here), tests=here)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
def test_tensors_are_refused():
    from crane_b200 import fp8
    x = torch.zeros((4, 256), device="cuda")
    c, s = fp8.quantize(x)
    w, ws = weights(gen_of("refused"), 130, 256)
    for call in (lambda: fp8.quantize(x.double()), lambda: fp8.quantize(x.t()), lambda: fp8.quantize(x[0]), lambda: fp8.quantize(x[:1].expand(4, 256)),
                 lambda: fp8.quantize(x, out=(c, s.contiguous())), lambda: fp8.quantize(x, out=(c[:3], s)), lambda: fp8.quantize(x, out=(c.cpu(), s)), lambda: fp8.silu_mul(x[:, :255]),
                 lambda: fp8.rms_norm(x, torch.ones(255, device="cuda")), lambda: fp8.rms_norm(x, torch.ones(256)), lambda: fp8.rms_norm(x, torch.ones(256, device="cuda"), residual_out=x),
                 lambda: fp8.rms_norm(x, torch.ones(256, device="cuda"), residual=x[:2]), lambda: fp8.rms_norm(x, torch.ones(256, device="cuda"), -1.0),
                 lambda: fp8.linear(c, s, w[:, :128], ws), lambda: fp8.linear(c, s, w, ws[:1]), lambda: fp8.linear(c, s[:, :1], w, ws), lambda: fp8.linear(c.view(torch.uint8), s, w, ws),
                 lambda: fp8.linear(c, s, w, ws, out=torch.empty((4, 131), device="cuda")), lambda: fp8.linear(c, s, w, ws, add=torch.empty((4, 130), device="cuda")),
                 lambda: fp8.linear(c, s, w, ws, dtype=torch.float64), lambda: fp8.linear(c.as_strided((4, 255), (256, 1), 1), s, w[:, :255], ws)):
        with pytest.raises(CraneB200Error) as e:
            call()
        assert e.value.code == crane_b200.INVALID_ARG and str(e.value)
    assert fp8.quantize(x[:0])[0].shape == (0, 256) and fp8.linear(c[:0], s[:0], w, ws).shape == (0, 130)
    l = crane_b200.load_library()
    assert l.crane_b200_fp8_quantize(99, x.data_ptr(), 0, 256, 4, 256, c.data_ptr(), 256, s.data_ptr(), 4, None) == crane_b200.CUDA_ERROR
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_a_wait_that_ran_out_is_reported():
    from crane_b200 import fp8
    l = crane_b200.load_library()
    l.crane_b200_debug_expire_wait.argtypes = [C.c_void_p]
    fp8.status()
    assert l.crane_b200_debug_expire_wait(None) == crane_b200.OK
    with pytest.raises(CraneB200Error, match="ran out"):
        fp8.status()
    fp8.status()
