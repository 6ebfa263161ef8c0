"""Linears in 8-bit floating point where they were wrong once: stores of ragged tiles that follow one another, waits that run out in a replayed graph.
References and tolerances are test_fp8.py's."""
import ctypes as C
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
