"""The 8-bit paged cache (crane_b200.kv8, crane_b200_kv8_* of the C ABI): rows into pages, attention over them.  Refusals and what kernels make of bad numbers on the CPU, results on the GPU
(-m gpu) against the formulas in 64 bits.

Codes and scales are held bit for bit: a scale is a power of two, so every quotient is exact and a code its rounding to nearest even.

Tolerance of attention, per output and fixed ahead of the first run; G = sum of w |v| (weights of the exact softmax), T positions, D columns:
  scores   products of f16 parts are exact, their f32 sums off by at most (D + 8) 2^-23 of A = max sum |q k| scale log2 e; f32 queries are two f16 parts, 2^-22 more; the exponent is rounded
           once more, 2^-23 of the distance to the maximum, and the factor scale log2 e of 16-bit rows, 2^-24: all within (D + 16) 2^-23 (A + 2), in units of log2
           bf16 queries of 128 columns in sequences of more than 64 rows of a kv head are two e4m3 parts: the largest element is taken to [2^7, 2^8), a part's steps are 2^-9 there at
           least, so each element is off by 2^-10 2^-7 of the largest at most: 2^-17 max |q| sum |k| scale log2 e more
  weights  ln 2 times that, in the numerator and in the denominator, and 2^-22 of the exponential in each; the numerator's are rounded to f16, 2^-11 (f32: two parts, 2^-22);
           weights below 2^-28 of the largest to 2^-39 of it, T in all
  sums     T / 16 additions of 16 products each, off by 2^-22 of the running sum, and as many joins as there are warps and CTAs: (T / 16 + 64) 2^-22
  result   half a step of its type."""
import ctypes as C
import math
import os
import subprocess

import pytest
import torch

import crane_b200
from crane_b200 import CraneB200Error

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F8 = torch.float8_e4m3fn
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def lib():
    import __graft_entry__
    __graft_entry__.build()
    return crane_b200.load_library()


def why():
    return (crane_b200.load_library().crane_b200_device_last_error() or b"").decode()


# -------------------------------------------------------------------------------------------------------------- without a GPU
P = 1 << 20            # an address that is never used: every call below is refused by its numbers


def test_numbers_of_device_memory_stay_in_range(tmp_path):
    """Lengths, starts and tables of any value, on the CPU: the kernels' own index functions, every row in one place and every step of the attention dealt out and joined once."""
    exe = str(tmp_path / "test_kv8_units")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", os.path.join(ROOT, "tests", "cpp", "test_kv8_units.cpp"), "-o", exe], check=True)
    assert subprocess.run([exe], capture_output=True, text=True, check=True).stdout == "ok\n"


CACHE = {"k_codes": P, "v_codes": P, "scales": P, "pages": 8, "kv_heads": 2, "page": 64, "dim": 128, "table": P, "ldt": 4, "width": 4, "lens": P, "starts": P, "seqs": 2, "rows": 3}
BAD_CACHE = [({"k_codes": None}, "NULL"), ({"scales": None}, "NULL"), ({"v_codes": P + 8}, "16-byte"), ({"scales": P + 4}, "8-byte"), ({"pages": 0}, "pages"), ({"pages": 1 << 40}, "pages"),
             ({"pages": 1 << 25}, "pages"), ({"kv_heads": 0}, "kv_heads"), ({"page": 48}, "page = 48"), ({"dim": 96}, "dim = 96"), ({"table": None}, "table"), ({"table": P + 2}, "table"),
             ({"ldt": 3}, "apart"), ({"width": 0}, "width"), ({"lens": None}, "lens"), ({"starts": None}, "starts"), ({"rows": 1 << 33}, "rows"), ({"seqs": 1 << 33}, "seqs"), ({"seqs": 1 << 25}, "seqs")]


@pytest.mark.parametrize("change, said", BAD_CACHE + [({"dtype": 3}, "type 3"), ({"k": None}, "k is NULL"), ({"v": P + 1}, "not aligned"), ({"ldk": 100}, "100 apart"), ({"ldvh": 5}, "heads of 128")])
def test_rows_are_refused_by_their_numbers(change, said):
    a = {"device": 0, "k": P, "ldk": 256, "ldkh": 128, "v": P, "ldv": 256, "ldvh": 128, "dtype": 1, **CACHE, "stream": None}
    a.update(change)
    assert lib().crane_b200_kv8_append(*a.values()) in (crane_b200.INVALID_ARG, crane_b200.UNSUPPORTED) and said in why()


@pytest.mark.parametrize("change, said", BAD_CACHE + [({"dtype": -1}, "type -1"), ({"q": None}, "q is NULL"), ({"out": None}, "out is NULL"), ({"heads": 3}, "3 heads"), ({"heads": 0}, "0 heads"),
                                                      ({"scale": math.nan}, "scale"), ({"scale": math.inf}, "scale"), ({"ldo": 5}, "5 apart"), ({"ldqh": 4}, "heads of 128"),
                                                      ({"max_rows": 1 << 33}, "max_rows")])
def test_attention_is_refused_by_its_numbers(change, said):
    a = {"device": 0, "q": P, "ldq": 512, "ldqh": 128, "out": P, "ldo": 512, "ldoh": 128, "dtype": 1, "heads": 4, "scale": 0.1, **CACHE, "max_rows": 0, "work": P, "bytes": 1 << 30,
         "stream": None}
    a.update(change)
    assert lib().crane_b200_kv8_attention(*a.values()) in (crane_b200.INVALID_ARG, crane_b200.UNSUPPORTED) and said in why()


def test_sizes_of_workspaces_are_refused():
    n = C.c_size_t()
    for heads, kv, dim, p in ((3, 2, 128, n), (4, 0, 128, n), (4, 2, 100, n)):
        assert lib().crane_b200_kv8_attention_bytes(0, 1, heads, kv, dim, 1, 1, 0, C.byref(p)) in (crane_b200.INVALID_ARG, crane_b200.UNSUPPORTED)
    assert lib().crane_b200_kv8_attention_bytes(0, 1, 4, 2, 128, 1, 1, 0, None) == crane_b200.INVALID_ARG


def test_numbers_of_heads_that_pass_32_bits_are_refused():
    n = C.c_size_t()
    assert lib().crane_b200_kv8_attention_bytes(0, 1, 65535 * 65534, 65534, 128, 1, 1, 0, C.byref(n)) == crane_b200.INVALID_ARG and "heads over 65534" in why()


def test_tensors_are_refused():
    from crane_b200 import kv8
    c = kv8.pages(4, 2, 64, 16, device="cpu")
    x = torch.zeros((3, 2, 64))
    i = torch.zeros((1, 4), dtype=torch.int32)
    with pytest.raises(CraneB200Error, match="CUDA"):
        kv8.append(x, x, c, i, i[0, :1], i[0, :2])
    with pytest.raises(CraneB200Error, match="cache"):
        kv8.attention(x, (x, x), i, i[0, :1], i[0, :2])


def repeating_tables(device):
    """Tables whose rows repeat or overlap: one row for all sequences, windows of one list."""
    i = torch.arange(20, dtype=torch.int32, device=device)
    return [i[:5].expand(4, -1), i.as_strided((4, 5), (2, 1)), i.as_strided((4, 5), (4, 1)), i[3:4].expand(4, 1)]


@pytest.mark.parametrize("which", range(4))
def test_tables_whose_rows_repeat_or_overlap_are_refused(which):
    """They are passed on as they lie: the distance of their rows is less than their width, and no distance that they do not have is made up, which would lead behind the storage."""
    from crane_b200 import kv8
    table, i = repeating_tables("cpu")[which], torch.zeros(5, dtype=torch.int32)
    s = dict(zip(("table", "ldt", "width", "lens", "starts", "seqs"), kv8._seqs(table, i[:4], i, -1)))
    assert s["ldt"] == table.stride(0) and s["width"] == table.shape[1] and s["seqs"] == 4
    cache = {**CACHE, "ldt": s["ldt"], "width": s["width"], "seqs": s["seqs"]}
    a = {"device": 0, "k": P, "ldk": 256, "ldkh": 128, "v": P, "ldv": 256, "ldvh": 128, "dtype": 1, **cache, "stream": None}
    assert lib().crane_b200_kv8_append(*a.values()) == crane_b200.INVALID_ARG and "apart" in why()
    a = {"device": 0, "q": P, "ldq": 512, "ldqh": 128, "out": P, "ldo": 512, "ldoh": 128, "dtype": 1, "heads": 4, "scale": 0.1, **cache, "max_rows": 0, "work": P, "bytes": 1 << 30, "stream": None}
    assert lib().crane_b200_kv8_attention(*a.values()) == crane_b200.INVALID_ARG and "apart" in why()


def test_a_single_row_of_pages_may_lie_at_any_distance():
    from crane_b200 import kv8
    i = torch.zeros(20, dtype=torch.int32)
    for table in (i.as_strided((1, 5), (0, 1)), i.as_strided((1, 5), (2, 1)), i[:5].view(1, 5), i.view(4, 5)[2:3]):
        t, ldt, width, *_, seqs = kv8._seqs(table, i[:1], i[:2], -1)
        assert t == table.data_ptr() and ldt >= width == 5 and seqs == 1


# ------------------------------------------------------------------------------------------------------------------ references
def gen_of(*key):
    import zlib
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def e4m3(v):
    """The nearest e4m3 value, ties to the even one, largest 448; NaN and infinities: NaN."""
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v.abs().clamp_min(2.0 ** -6).clamp_max(1e6))[1] - 4)
    return torch.where(torch.isfinite(v), (torch.round(v / step) * step).clamp(-448, 448), math.nan)


def scale_of(rows):
    finite = torch.where(torch.isfinite(rows), rows, 0.0)
    top = max(float(finite.abs().max()), 2.0 ** -100)
    e = math.floor(math.log2(top)) - 10
    while top > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def plain_append(cache, k, v, table, lens, starts):
    """The rule on f64 copies (k values of codes, v values of codes, scales)."""
    page = cache[0].shape[2]
    for b in range(len(lens)):
        n = starts[b + 1] - starts[b]
        first = lens[b] - n
        for blk in range(max(first, 0) // page, (lens[b] + page - 1) // page):
            lo, hi = max(first, 0, blk * page), min(lens[b], blk * page + page)
            if blk >= len(table[b]) or not 0 <= table[b][blk] < cache[0].shape[0] or lo >= hi:
                continue
            p, kept = table[b][blk], lo - blk * page
            for i, x in enumerate((k, v)):
                for h in range(x.shape[1]):
                    rows = x[starts[b] + lo - first:starts[b] + hi - first, h].double()
                    s = scale_of(rows)
                    if kept:
                        old = float(cache[2][p, h, i])
                        s = max(s, old)
                        if s != old:
                            cache[i][p, h, :kept] = e4m3(cache[i][p, h, :kept] * old / s)
                    cache[i][p, h, kept:kept + hi - lo] = e4m3(rows / s)
                    cache[2][p, h, i] = s


def same(a, b):
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def run_append(cache, k, v, table, lens, starts):
    from crane_b200 import kv8
    ref = [c.double().clone() for c in cache]
    plain_append(ref, k, v, table, lens, starts)
    kv8.append(k, v, cache, ints(table), ints(lens), ints(starts))
    for got, want in zip(cache, ref):
        assert same(got.double(), want)


# ------------------------------------------------------------------------------------------------------------------ rows into pages
@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("dim, page, heads", [(64, 16, 3), (128, 64, 2), (256, 32, 1), (128, 128, 1)])
def test_rows_come_in_one_by_one_and_in_portions(dim, page, heads, dt):
    from crane_b200 import kv8
    g = gen_of("append", dim, page, heads, dt)
    cache = kv8.pages(9, heads, dim, page)
    for c in cache[:2]:
        c.view(torch.uint8).fill_(0x55)
    table = [[3, 0, 8, -1], [5, 7, 900, 2], [1, 6, -7, 4]]
    lens = [0, 0, 0]
    for new in ([1, 0, 3], [page - 1, page + 1, 2], [1, page, 0], [2, 1, 1], [page + 3, 0, 2 * page], [0, 0, 0], [1, 1, 1]):
        starts = [0]
        for b, n in enumerate(new):
            starts.append(starts[-1] + n)
            lens[b] += n
        x = torch.randn((max(starts[-1], 1), 2 * heads + 1, dim), generator=g, device="cuda") * torch.exp(2 * torch.randn((max(starts[-1], 1), 1, 1), generator=g, device="cuda"))
        x = x.to(TYPES[dt])[:starts[-1]]
        run_append(cache, x[:, :heads], x[:, heads:2 * heads], table, list(lens), starts)
    lens = [page + 2, page + 2, 2]                                     # drafts that did not hold: positions are written again
    x = torch.randn((6, heads, dim), generator=g, device="cuda").to(TYPES[dt]) * 0.01
    run_append(cache, x, x, table, lens, [0, 2, 4, 6])


@pytest.mark.gpu
def test_rows_of_extreme_values_and_bad_numbers():
    from crane_b200 import kv8
    cache = kv8.pages(6, 1, 64, 16)
    top = torch.finfo(torch.float32).max
    x = torch.zeros((20, 1, 64), device="cuda")
    x[1], x[2], x[3, 0, 5], x[4, 0, 7], x[5, 0, 1], x[6, 0, 0], x[7, 0, 0] = 1e-40, 2.0 ** -101, math.nan, math.inf, -math.inf, 448.0, 448.0 * (1 + 2.0 ** -20)
    for i in range(8):
        run_append(cache, x[i:i + 1], x[i:i + 1] * -2, [[4, 2]], [i + 1], [0, 1])
    x[9] = top
    run_append(cache, x[8:], -x[8:], [[4, 2]], [20], [0, 12])
    # rows ahead of position 0, behind the table, on pages that do not exist, of no sequence: not stored, and nothing else moves
    y = torch.randn((40, 1, 64), generator=gen_of("bad"), device="cuda")
    run_append(cache, y, y, [[0, -1], [9, 1]], [3, 40], [0, 7, 30])
    kv8.append(y[:0], y[:0], cache, ints([[0, 1]]), ints([5]), ints([0, 0]))
    before = [c.clone() for c in cache]
    kv8.append(y, y, cache, ints([[0, 1]]), ints([-5]), ints([-3, 1 << 30]))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, cache))


@pytest.mark.gpu
def test_rows_on_any_boundary():
    """Rows and heads at any distance, off 16 bytes too, columns side by side."""
    from crane_b200 import kv8
    g = gen_of("strides")
    for dt in TYPES.values():
        x = torch.randn(60000, generator=g, device="cuda").to(dt)
        for ld, ldh, off in ((300, 130, 1), (128, 64, 0), (64, 700, 3), (1000, 192, 8)):
            k, v = x.as_strided((9, 2, 64), (ld, ldh, 1), off), x.as_strided((9, 2, 64), (ldh + ld, ldh, 1), off + 5)
            run_append(kv8.pages(4, 2, 64, 16), k, v, [[2, 1]], [20], [0, 9])


# ------------------------------------------------------------------------------------------------------------------ attention
def attend_ref(q, cache, table, lens, starts, scale):
    """(result, tolerance) in 64 bits; rows of no sequence: NaN."""
    page, hk = cache[0].shape[2], cache[0].shape[1]
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    group, d, exact32 = q.shape[1] // hk, q.shape[2], q.dtype == torch.float32
    for b in range(len(lens)):
        n, t = starts[b + 1] - starts[b], min(lens[b], len(table[b]) * page)
        if n == 0:
            continue
        pages = [p if 0 <= p < cache[0].shape[0] else -1 for p in table[b]]
        there = torch.tensor([pages[i // page] >= 0 for i in range(t)], device="cuda", dtype=torch.bool)
        idx = torch.tensor([max(p, 0) for p in pages], device="cuda")
        seen = (torch.arange(t, device="cuda") <= lens[b] - n + torch.arange(n, device="cuda")[:, None]) & there
        for h in range(q.shape[1]):
            kh = h // group
            k, v = ((cache[i][idx, kh].double() * cache[2][idx, kh, i].double()[:, None, None]).reshape(-1, d)[:t] for i in range(2))
            x = q[starts[b]:starts[b + 1], h].double()
            # (NaN of masked places must not count: products over visible ones only)
            s = torch.where(seen, (x @ torch.nan_to_num(k).t()) * scale, -math.inf)
            bad_k = torch.isnan(k).any(1)
            w = torch.exp(s - s.amax(1, keepdim=True).clamp_min(-1e300))
            w = torch.where(seen, w, 0.0)
            w = w / w.sum(1, keepdim=True).clamp_min(1e-300)
            o = w @ torch.nan_to_num(v)
            o = torch.where((seen.double() @ torch.isnan(v).double()) > 0, math.nan, o)
            o = torch.where((seen & bad_k).any(1, keepdim=True), math.nan, o)
            out[starts[b]:starts[b + 1], h] = o
            size = w @ torch.nan_to_num(v).abs()
            a = torch.where(seen, (x.abs() @ torch.nan_to_num(k).abs().t()) * abs(scale) * 1.4427, 0.0).amax(1, keepdim=True) if t else x[:, :1] * 0
            parts = 0.0
            if q.dtype == torch.bfloat16 and d == 128 and n * group > 64 and t:
                parts = 2.0 ** -17 * x.abs().amax(1, keepdim=True) * torch.nan_to_num(k).abs().sum(1).amax() * abs(scale) * 1.4427
            off = 2 * (0.6932 * ((d + 16) * 2.0 ** -23 * (a + 2) + parts) + 2.0 ** -22) + (2.0 ** -22 if exact32 else 2.0 ** -11) + (t / 16 + 64) * 2.0 ** -22
            tiny = t * 2.0 ** -39 * torch.nan_to_num(v).abs().amax() if t else 0.0
            tol[starts[b]:starts[b + 1], h] = off * size + tiny
    return out, tol


def check(got, ref, exact=False):
    out, tol = ref
    assert same(torch.isnan(got).double(), torch.isnan(out).double()), "NaN in other places"
    ok = ~torch.isnan(out)
    half = torch.finfo(got.dtype).eps / 2
    err = (got.double() - out).abs()[ok]
    lim = (tol + half * (out.abs() + tol) + (2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -149))[ok]
    assert bool((err <= lim).all()), (int((err > lim).sum()), float((err / lim).max()))


def filled(g, pages, heads, dim, page, loud=True):
    """A cache of random codes with scales that differ by page."""
    from crane_b200 import kv8
    c = kv8.pages(pages, heads, dim, page)
    for i in range(2):
        c[i].copy_((torch.randn(c[i].shape, generator=g, device="cuda") * 120).clamp(-448, 448).to(F8))
    c[2].copy_(torch.exp2(torch.randint(-9, -5 if loud else -8, c[2].shape, generator=g, device="cuda").float()))
    return c


def problem(g, dt, heads, kv, dim, page, lens, new, extra=0, loud=True):
    need = [(max(t, 1) + page - 1) // page for t in lens]
    c = filled(g, sum(need) + 2, kv, dim, page, loud)
    order = torch.randperm(sum(need) + 2, generator=g, device="cuda").tolist()
    table = []
    for n in need:
        table.append([order.pop() for _ in range(n)] + [-1 - n] * (max(need) - n))
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = torch.randn((starts[-1] + extra, heads, dim), generator=g, device="cuda").to(TYPES[dt])
    return q, c, table, lens, starts


def run_attention(p, scale=None, **kw):
    from crane_b200 import kv8
    q, c, table, lens, starts = p
    return kv8.attention(q, c, ints(table), ints(lens), ints(starts), scale=scale, **kw)


SIZES = [  # heads, kv heads, dim, page, lens, new rows
    (1, 1, 64, 16, [1], [1]),
    (4, 2, 128, 64, [1, 2, 63, 64, 65, 0, 129], [1, 1, 1, 1, 1, 0, 1]),
    (8, 2, 256, 16, [300, 17, 16, 15], [5, 1, 9, 15]),
    (32, 8, 128, 64, [700, 3, 1500], [1, 1, 1]),
    (7, 1, 64, 32, [100, 33, 250], [3, 33, 1]),
    (6, 3, 128, 128, [400, 130, 127], [70, 1, 127]),
    (16, 8, 128, 64, [333, 5, 2000], [333, 5, 40]),
    (4, 4, 64, 64, [1000], [200]),
    (8, 1, 256, 64, [260, 513], [100, 3]),
    (12, 1, 128, 16, [97, 31], [2, 31]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "-".join(map(str, s[:4])))
def test_attention(size, dt):
    heads, kv, dim, page, lens, new = size
    g = gen_of("attend", size, dt)
    p = problem(g, dt, heads, kv, dim, page, lens, new, extra=2)
    out = torch.full(p[0].shape, 7.0, dtype=TYPES[dt], device="cuda")
    run_attention(p, out=out)
    ref = attend_ref(*p, dim ** -0.5)
    n = p[4][-1]
    check(out[:n], (ref[0][:n], ref[1][:n]))
    assert (out[n:] == 7).all()                                       # rows behind the last sequence
    for hint in (max(new), 1):                                        # (a hint that is too small only takes longer)
        check(run_attention(p, max_rows=hint)[:n], (ref[0][:n], ref[1][:n]))


@pytest.mark.gpu
def test_attention_of_many_sequences():
    """More sequences than a block has threads, most of them with nothing new."""
    g = gen_of("many")
    lens = [int(x) for x in torch.randint(0, 150, (301,), generator=g, device="cuda")]
    new = [min(t, 1 if i % 3 else i % 5) for i, t in enumerate(lens)]
    p = problem(g, "bf16", 4, 2, 64, 16, lens, new)
    check(run_attention(p), attend_ref(*p, 0.125))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows", [3, 150])
def test_rows_that_see_nothing_missing_pages_and_nan(rows, dt):
    """Positions below 0, pages outside the cache, lengths beyond the table; NaN in codes that some rows do not see, in codes behind the last position, in scales of pages that nobody has."""
    g = gen_of("nothing", rows, dt)
    q, c, table, lens, starts = problem(g, dt, 4, 2, 128, 16, [rows, rows + 40, 60, 20], [rows + 2, rows, 1, 1])
    table[1][1], table[2][0] = 10 ** 6, -5
    lens[2] = 16 * len(table[2]) + 9
    last = [table[0][(lens[0] - 1) // 16], (lens[0] - 1) % 16]
    for i in range(2):
        bits = c[i].view(torch.uint8)
        bits[last[0], :, last[1] + 1:] = 0x7f                           # behind the last position
        bits[table[1][(rows + 38) // 16], 1, (rows + 38) % 16, 5] = 0xff      # seen by the last two rows of sequence 1 alone
        bits[table[3][1], :, 4:] = 0xff
    used = {p for t in table for p in t}
    c[2][[p for p in range(c[2].shape[0]) if p not in used]] = math.nan
    p = (q, c, table, lens, starts)
    ref = attend_ref(*p, 0.1)
    got = run_attention(p, scale=0.1)
    check(got, ref)
    assert (got[:2] == 0).all() and torch.isnan(got[2 + rows + 2:]).sum() > 0


@pytest.mark.gpu
def test_queries_of_extreme_values():
    g = gen_of("extreme")
    for dt, big, small in (("f32", 1e30, 1e-30), ("bf16", 1e30, 1e-30), ("f16", 6e4, 1e-6)):
        q, c, table, lens, starts = problem(g, dt, 2, 1, 64, 16, [50], [6], loud=False)
        q[0], q[1], q[2], q[3, 0, 3], q[4, 1, 9] = 0, q[1] * small, q[2] * big, math.nan, math.inf
        ref = attend_ref(q.nan_to_num(0, 0, 0), c, table, lens, starts, 0.125)
        ref[0][3, 0], ref[0][4, 1] = math.nan, math.nan                 # a row's NaN or infinity is its own
        got = run_attention((q, c, table, lens, starts), scale=0.125)
        keep = [0, 1, 3, 4, 5]
        check(got[keep], (ref[0][keep], ref[1][keep]))
        fine = torch.isfinite(q[2]).all(1, keepdim=True)                # (f16 has infinities among these)
        assert torch.equal(torch.isfinite(got[2]), fine.expand_as(got[2]))      # (scores of 1e30: one position takes all, which one is a matter of the last bit)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
def test_queries_with_a_column_far_larger_than_the_rest(dt):
    """... that the keys have little of: the small elements decide."""
    for loud in (30.0, 1000.0):
        q, c, table, lens, starts = problem(gen_of("loud", dt, loud), dt, 8, 2, 128, 64, [200, 90], [150, 2], loud=False)
        q[:, :, 17] *= loud
        c[0][:, :, :, 17] = (c[0][:, :, :, 17].float() / loud).to(F8)
        p = (q, c, table, lens, starts)
        check(run_attention(p, scale=0.3), attend_ref(*p, 0.3))


@pytest.mark.gpu
def test_values_of_very_different_pages():
    """Value scales from 2^-100 to 2^100: the largest weighted value decides what is kept."""
    g = gen_of("scales")
    for dt in TYPES:
        q, c, table, lens, starts = problem(g, dt, 4, 2, 64, 16, [120, 64], [2, 64], loud=False)
        for s in ((2.0 ** 60, 2.0 ** -60), (2.0 ** 15, 2.0 ** -12), (1.0, 2.0 ** -100)):
            c[2][:, :, 1] = torch.where(torch.rand(c[2].shape[:2], generator=g, device="cuda") < 0.5, *s)
            if dt == "f16":
                c[2][:, :, 1].clamp_(max=16.0)
            p = (q, c, table, lens, starts)
            out, tol = attend_ref(*p, 0.125)
            # weights are kept relative to the largest weight times scale: 2^-39 of the largest value of all
            check(run_attention(p, scale=0.125), (out, tol))


@pytest.mark.gpu
def test_attention_over_strided_rows_and_into_them():
    g = gen_of("attend strides")
    for dt in TYPES:
        q, c, table, lens, starts = problem(g, dt, 4, 2, 64, 32, [70, 9], [5, 9])
        ref = attend_ref(q, c, table, lens, starts, 0.2)
        wide = torch.zeros((14, 3, 4, 67), dtype=TYPES[dt], device="cuda")
        wide[:, 1, :, 3:] = q
        out = torch.full((14, 4, 3, 65), 5.0, dtype=TYPES[dt], device="cuda")
        run_attention((wide[:, 1, :, 3:], c, table, lens, starts), scale=0.2, out=out[:, :, 2, 1:])
        check(out[:, :, 2, 1:], ref)
        assert (out[:, :, :2] == 5).all() and (out[:, :, 2, 0] == 5).all()
        heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
        check(run_attention((heads_first, c, table, lens, starts), scale=0.2), ref)


@pytest.mark.gpu
def test_results_repeat_and_calls_share_nothing():
    """The same bits every time, on two streams at once, and in a graph that is replayed with other lengths."""
    from crane_b200 import kv8
    g = gen_of("repeat")
    q, c, table, lens, starts = problem(g, "bf16", 16, 8, 128, 64, [900, 1500, 64], [1, 1, 1])
    t, l, s = ints(table), ints(lens), ints(starts)
    one = kv8.attention(q, c, t, l, s)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for st in streams * 4:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            outs.append(kv8.attention(q, c, t, l, s))
    torch.cuda.synchronize()
    assert all(torch.equal(one, o) for o in outs)
    k = torch.randn((3, 8, 128), generator=g, device="cuda").bfloat16()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv8.append(k, k, c, t, l, s)
        out = kv8.attention(q, c, t, l, s)
    for lens in ([5, 1500, 64], [896, 3, 1], [1, 1, 1]):
        l.copy_(ints(lens))
        graph.replay()
        check(out, attend_ref(q, c, table, lens, starts, 128 ** -0.5))


@pytest.mark.gpu
def test_a_sequence_grows():
    """Rows appended as portions, then one by one, attended over at each step, against attention over the rounded rows themselves."""
    from crane_b200 import kv8
    g = gen_of("grows")
    cache = kv8.pages(12, 2, 128, 16)
    table, lens = [[7, 2, 9, 4], [1, 11, 0, 3]], [0, 0]
    for new in ([20, 3], [1, 1], [1, 1], [13, 30], [2, 5]):
        starts = [0, new[0], sum(new)]
        lens = [lens[0] + new[0], lens[1] + new[1]]
        qkv = torch.randn((sum(new), 4 + 2 + 2, 128), generator=g, device="cuda").bfloat16()
        run_append(cache, qkv[:, 4:6], qkv[:, 6:], table, lens, starts)
        p = (qkv[:, :4], cache, table, lens, starts)
        check(run_attention(p), attend_ref(*p, 128 ** -0.5))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("scale", [0.0, -0.4, 2.5])
def test_scales_of_any_sign(scale, dim):
    """Zero weighs all positions alike; a negative one turns the order round."""
    for dt in TYPES:
        for new in ([1, 2, 1], [100, 5, 70]):
            p = problem(gen_of("sign", dt, scale, dim, new), dt, 8, 2, dim, 64, [150, 90, 200], new, loud=False)
            check(run_attention(p, scale=scale), attend_ref(*p, scale))


@pytest.mark.gpu
def test_a_cache_whose_codes_pass_32_bits():
    """The highest pages of 4.6 GB of codes against the same pages of a small cache, rows and results, the results over the queries too."""
    from crane_b200 import kv8
    big, few = kv8.pages(70000, 8, 128, 64), kv8.pages(6, 8, 128, 64)
    assert big[0].numel() > 1 << 32
    pages = [69999, 3, 68000, 66001, 69998, 5]
    lens, starts = ints([150, 140]), ints([0, 150, 290])
    x = torch.randn((290, 32, 128), generator=gen_of("wide"), device="cuda").bfloat16()
    for cache, table in ((big, pages), (few, list(range(6)))):
        kv8.append(x[:, 16:24], x[:, 24:], cache, ints(table).reshape(2, 3), lens, starts)
    for a, b in zip(big, few):
        assert torch.equal(a.view(torch.uint8)[pages], b.view(torch.uint8))
    for q, s in ((x[:, :16].clone(), starts), (x[:2, :16].clone(), ints([0, 1, 2]))):
        want = kv8.attention(q, few, ints(list(range(6))).reshape(2, 3), lens, s)
        assert torch.equal(kv8.attention(q, big, ints(pages).reshape(2, 3), lens, s, out=q), want)


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(4))
def test_calls_with_tables_whose_rows_repeat_or_overlap_are_refused(which):
    from crane_b200 import kv8
    cache, x = kv8.pages(20, 2, 64, 16), torch.ones((4, 2, 64), device="cuda")
    table, lens, starts = repeating_tables("cuda")[which], ints([3] * 4), ints([0, 1, 2, 3, 4])
    with pytest.raises(CraneB200Error, match="apart"):
        kv8.append(x, x, cache, table, lens, starts)
    with pytest.raises(CraneB200Error, match="apart"):
        kv8.attention(x, cache, table, lens, starts)
    assert all(int(c.view(torch.uint8).count_nonzero()) == 0 for c in cache[:2])
    out = kv8.attention(x, cache, table.contiguous(), lens, starts)     # the same pages for each, in rows of their own
    assert (out == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("dim, page", [(64, 16), (128, 64), (128, 16), (256, 32)])
@pytest.mark.parametrize("new", [1, 4, 9, 90])
def test_a_nan_among_the_values_reaches_every_row_that_sees_it(new, dim, page, dt):
    """At the newest position, the ones ahead of it, the first, in the middle, beside missing pages; sequences of odd and even numbers of tiles.  Each has one, in a column and head of its own."""
    lens, at = [], []
    for t in (new, new + 1, 64, 65, 100, 130, 200, 500):
        if t >= new:
            for pos in {t - 1, t - 2, t - new - 1, t - new, t // 2, 31, 0}:
                if 0 <= pos < t:
                    lens.append(t)
                    at.append(pos)
    lens = lens + lens
    q, c, table, lens, starts = problem(gen_of("seen", new, dim, page, dt), dt, 4, 2, dim, page, lens, [new] * len(lens))
    for b, pos in enumerate(at + at):
        c[1].view(torch.uint8)[table[b][pos // page], b & 1, pos % page, (37 * b) % dim] = 0x7f if b & 2 else 0xff
        if b >= len(at):                                                # the pages on either side of it are not there
            for i in (pos // page - 1, pos // page + 1):
                if 0 <= i < len(table[b]):
                    table[b][i] = -1
    p = (q, c, table, lens, starts)
    ref = attend_ref(*p, dim ** -0.5)
    assert torch.isnan(ref[0]).any(2).any(1).sum() >= len(lens)
    for hint in (0, new):
        check(run_attention(p, max_rows=hint), ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("dim, page", [(64, 32), (128, 16), (256, 16)])
def test_no_nan_of_a_long_history_is_lost(dim, page, dt):
    """However the steps are dealt out: page i of every sequence has one in column i alone."""
    new = [1, 3, 1, 70]
    q, c, table, lens, starts = p = problem(gen_of("history", dim, page, dt), dt, 2, 1, dim, page, [5000, 1777, 900, 2500], new)
    for row, n, t in zip(table, new, lens):
        for i in range(min(dim, (t - n) // page)):
            c[1].view(torch.uint8)[row[i], 0, (7 * i) % page, i] = 0x7f
    ref = attend_ref(*p, dim ** -0.5)
    check(run_attention(p), ref)
    check(run_attention((q[:5], c, table[:3], lens[:3], starts[:4]), max_rows=3), (ref[0][:5], ref[1][:5]))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
def test_an_infinity_among_the_new_rows_is_seen(dt):
    """Rows into the cache make a NaN of it; the rows that see the position get it, in its column."""
    from crane_b200 import kv8
    cache = kv8.pages(6, 1, 128, 64)
    table, lens, starts = ints([[3, 1], [0, 5]]), ints([70, 65]), ints([0, 70, 135])
    x = torch.randn((135, 1, 128), generator=gen_of("new inf", dt), device="cuda").to(TYPES[dt])
    kv8.append(x, x, cache, table, lens, starts)
    for n, col in ((71, 5), (72, 9)):
        y = torch.ones((2, 1, 128), dtype=TYPES[dt], device="cuda")
        v = y.clone()
        v[0, 0, col], v[1, 0, col + 1] = math.inf, math.nan
        lens.copy_(ints([n, n - 5]))
        kv8.append(y, v, cache, table, lens, ints([0, 1, 2]))
        out = kv8.attention(y, cache, table, lens, ints([0, 1, 2]))
        want = torch.zeros((2, 128), dtype=torch.bool, device="cuda")
        for first in range(5, col + 1, 4):
            want[0, first], want[1, first + 1] = True, True
        assert torch.equal(torch.isnan(out[:, 0]), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_results_may_take_the_place_of_the_queries(dim, dt):
    """Units that one CTA has and units that several share, few rows and many beside one another."""
    for new in ([1, 1, 3, 1], [1, 300, 5, 40], [700, 1, 1, 90]):
        q, c, table, lens, starts = problem(gen_of("in place", dim, dt, new), dt, 8, 2, dim, 64, [3000, 1400, 70, 900], new)
        want = run_attention((q, c, table, lens, starts))
        x = q.clone()
        assert run_attention((x, c, table, lens, starts), out=x) is x and torch.equal(x, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_nan_and_infinities_of_queries_and_keys_among_many_rows(dim, dt):
    """A query's is its row's, even beside rows that see nothing; a key's reaches the rows that see it, in every column."""
    q, c, table, lens, starts = problem(gen_of("many rows", dim, dt), dt, 4, 2, dim, 64, [600, 150, 3000, 40], [200, 150, 90, 70], loud=False)
    clean = q.clone()
    q[3, 0, 3], q[70, 1, 9], q[199, 2, 0], q[201, 3, dim - 1], q[399, 0, 5], q[440, 1, 1], q[445, 3, 2] = (math.nan, math.inf, -math.inf, math.nan, math.inf, math.nan, math.inf)
    for b, pos, h in ((0, 450, 0), (1, 149, 1), (2, 2950, 0), (2, 2999, 1)):
        c[0].view(torch.uint8)[table[b][pos // 64], h, pos % 64, 7] = 0x7f
    out, tol = attend_ref(clean, c, table, lens, starts, dim ** -0.5)
    for i in range(440):
        for h in range(4):
            if not torch.isfinite(q[i, h]).all():
                out[i, h] = math.nan
    got = run_attention((q, c, table, lens, starts))
    check(got, (out, tol))
    assert (got[440:470] == 0).all() and torch.isnan(got[399, 0]).all()         # rows ahead of position 0, whatever they hold
