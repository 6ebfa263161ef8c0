"""Linears in 8-bit floating point where they were wrong once: stores of ragged tiles that follow one another, waits that run out in a replayed graph,
infinite gates and far negative ones.  References and tolerances are test_fp8.py's where nothing else is said."""
import ctypes as C
import math
import os
import subprocess

import pytest
import torch

import crane_b200
from crane_b200 import CraneB200Error
from test_fp8 import TYPES, check_linear, gen_of, linear_ref, rows_of, weights

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_pieces_never_meet_a_store_that_reads(tmp_path):
    """The walk of the tiles and the halves of the patch that results leave through, on the host."""
    exe = str(tmp_path / "test_fp8_tiles")
    subprocess.run(["g++", "-std=c++17", "-O1", os.path.join(ROOT, "tests", "cpp", "test_fp8_tiles.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "fp8_tiles: ok" in r.stdout, r.stdout


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k, dt", [(8192, 4160, 128, "bf16"), (8192, 576, 128, "bf16"), (8192, 4128, 128, "bf16"), (8192, 4128, 128, "f32"), (4096, 4160, 256, "f16"),
                                         (4459, 11616, 104, "f32"), (8192, 24608, 64, "f32")])
def test_ragged_tiles_that_follow_one_another(m, n, k, dt):
    """Tiles with an odd number of pieces, the pair's next tile right behind them: the bits of the route that stores by rows, every time."""
    from crane_b200 import fp8
    gen = gen_of("ragged", m, n, k, dt)
    x, xs = fp8.quantize(rows_of(gen, m, k, torch.bfloat16))
    w, ws = weights(gen, n, k)
    odd = torch.empty((m, n + 1), dtype=TYPES[dt], device="cuda")[:, :n]          # rows on no 16-byte boundaries
    fp8.linear(x, xs, w, ws, out=odd)
    check_linear(odd, linear_ref(x, xs, w, ws))
    for _ in range(20):
        out = torch.full((m, n), 99.0, dtype=TYPES[dt], device="cuda")
        fp8.linear(x, xs, w, ws, out=out)
        assert torch.equal(out, odd)
    fp8.status()


def test_every_stream_hears_of_a_wait_once(tmp_path):
    """What crane_b200_fp8_status looks at, on the host."""
    exe = str(tmp_path / "test_fp8_waits")
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include"),
                    os.path.join(ROOT, "tests", "cpp", "test_fp8_waits.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "fp8_waits: ok" in r.stdout, r.stdout


@pytest.mark.gpu
def test_a_wait_that_ran_out_in_a_replayed_graph_is_reported():
    """Captured on one stream, replayed on another, as torch does it: both streams are told, once; a stream of its own that replays it again is told, too."""
    from crane_b200 import fp8
    expire = crane_b200.load_library().crane_b200_debug_expire_fp8_wait
    expire.argtypes = [C.c_int, C.c_void_p]
    gen = gen_of("replayed")
    x, xs = fp8.quantize(rows_of(gen, 5, 256, torch.float32))
    w, ws = weights(gen, 256, 256)
    fp8.linear(x, xs, w, ws)
    g, side, third = torch.cuda.CUDAGraph(), torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        out = fp8.linear(x, xs, w, ws)
        assert expire(torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream) == crane_b200.OK
    def told(stream):
        with torch.cuda.stream(stream):
            try:
                fp8.status()
            except CraneB200Error as e:
                assert e.code == crane_b200.CUDA_ERROR and "ran out" in str(e)
                return True
            return False
    here = torch.cuda.current_stream()
    for s in (here, side, third):
        told(s)
    assert not told(here) and not told(side) and not told(third)
    for on in (here, third, side):
        with torch.cuda.stream(on):
            g.replay()
        assert told(on) and not told(on)
        for s in (here, side, third):
            assert told(s) == (s != on)
            assert not told(s)
    assert torch.equal(out, fp8.linear(x, xs, w, ws))


@pytest.mark.gpu
@pytest.mark.parametrize("k", [128, 300])
@pytest.mark.parametrize("dt", TYPES)
def test_infinite_and_nan_gates(dt, k):
    """An infinite SiLU(g) u makes its block's scale infinite and the block NaN in use; a NaN (that of g = -inf, -inf / inf, and of inf x 0 among them) is its own."""
    from crane_b200 import fp8
    inf, nan = math.inf, math.nan
    gate, up = torch.ones((8, k), device="cuda"), torch.ones((8, k), device="cuda")
    gate[0, 3], gate[1, 3], gate[2, 3], gate[3, 3] = inf, -inf, nan, inf
    up[3, 3] = 0
    up[4, 3], up[5, 3] = inf, nan
    gate[6, 3], up[6, 3] = inf, -2
    y = gate.double() / (1 + torch.exp(-gate.double())) * up.double()
    codes, scales = fp8.silu_mul(torch.cat([gate, up], 1).to(TYPES[dt]))
    back = codes.double() * scales.double().repeat_interleave(128, 1)[:, :k]
    others = [i for i in range(k) if i != 3]
    for r in range(8):
        if torch.isinf(y[r, 3]):
            assert r in (0, 4, 6) and torch.isinf(scales[r, 0]) and torch.isnan(back[r, :128]).all() and torch.isfinite(back[r, 128:]).all()
        else:
            assert torch.isnan(back[r, 3]) == torch.isnan(y[r, 3]) == (r in (1, 2, 3, 5))
            assert (codes[r, others].float() == 448).all() and torch.isfinite(scales[r]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("lo, hi", [(-8, 8), (8, 89), (-80, -8), (-87.3, -80), (-88.7, -87.3), (-1000, -88.8)])
def test_gated_units_to_their_last_bits(lo, hi):
    """One value a block, so that the block's scale is that value / 448 in f32.  In units of 2^-24: the exponential 4 (2^-22 of itself), its argument 1.4 where it is small (ln 2 x 2^-23),
    its correction 1, 1 + z 1, the reciprocal 2 (an ulp), its quarter 4 where that is no normal number (half of 2^-149 of 2^-128), two products 2, the scale's quotient 1: 16.4; 18 are allowed.
    Below -88.73 the exponential is infinite in f32 and the unit zero."""
    from crane_b200 import fp8
    gen = gen_of("units", lo, hi)
    n = 1 << 18
    g = torch.rand(n, generator=gen, device="cuda") * (hi - lo) + lo
    u = torch.exp2(3 * torch.rand(n, generator=gen, device="cuda")) * 2.0 ** (100 if lo < -80 else 60 if lo < -8 else 0)
    x = torch.zeros((n, 256), device="cuda")
    x[:, 0], x[:, 128] = g, u
    scales = fp8.silu_mul(x)[1][:, 0].double()
    y = (g.double() / (1 + torch.exp(-g.double())) * u.double()).abs()
    if hi < -88.73:
        y.zero_()
    want = y.clamp_min(2.0 ** -100) / 448
    assert ((scales - want).abs() <= 18 * 2.0 ** -24 * want).all(), float(((scales - want) / want).abs().max()) * 2 ** 24


@pytest.mark.gpu
def test_rows_of_the_largest_width():
    """2^30 columns of gates and as many ups on an odd boundary: the bits of the same row on a 16-byte boundary."""
    from crane_b200 import fp8
    k = 2 ** 30
    wide = torch.empty(2 * k + 8, dtype=torch.bfloat16, device="cuda")
    part = rows_of(gen_of("widest"), 1, 2 ** 20, torch.bfloat16)[0]
    for i in range(0, 2 * k, 2 ** 20):
        wide[i:i + 2 ** 20] = part.roll(i >> 20)
    even = fp8.silu_mul(wide[None, :2 * k])
    wide[1:2 * k + 1] = wide[:2 * k].clone()
    odd = fp8.silu_mul(wide[None, 1:2 * k + 1])
    assert torch.equal(even[0].view(torch.uint8), odd[0].view(torch.uint8)) and torch.equal(even[1], odd[1])
