"""Verification of drafted tokens (crane_b200.draft, crane_b200_draft_verify of the C ABI).  Refusals on the CPU, results on the GPU (-m gpu) against the rule in 64 bits: counts and tokens are
whole numbers and have to be equal.

Probabilities are f32 sums of 2^-22 exponentials, joined in 64 bits: 2^-20 of themselves off at most.  A draft whose u q lies that near to p, or a race whose two largest keys do, could go
either way; none of the inputs below is one (`decided` looks, in 64 bits, for a margin of 2^-16)."""
import ctypes as C
import math

import pytest
import torch

import crane_b200
from crane_b200 import CraneB200Error

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MARGIN = 2.0 ** -16


def lib():
    import __graft_entry__
    __graft_entry__.build()
    return crane_b200.load_library()


P = 1 << 20            # an address that is never used: every call below is refused by its numbers


@pytest.mark.parametrize("change, said", [
    ({"dtype": 3}, "type 3"), ({"vocab": 0}, "vocab = 0"), ({"vocab": 1 << 31}, "vocab"), ({"seqs": 1 << 31}, "seqs"), ({"drafts": 1 << 31}, "drafts"), ({"drafts": 1 << 27}, "2^27"), ({"logits": None}, "logits is NULL"),
    ({"ld": 9}, "9 apart"), ({"draft_logits": P + 1}, "draft_logits is not aligned"), ({"ldd": 9}, "draft_logits"), ({"tokens": None}, "tokens"), ({"starts": None}, "starts"),
    ({"starts": P + 2}, "starts"), ({"temperatures": P + 2}, "temperatures"), ({"uniforms": None}, "uniforms"), ({"noise": None}, "noise"), ({"ldn": 3}, "noise"),
    ({"accepted": None}, "accepted"), ({"next": P + 2}, "next")])
def test_calls_are_refused_by_their_numbers(change, said):
    a = {"device": 0, "logits": P, "ld": 100, "draft_logits": P, "ldd": 100, "dtype": 0, "vocab": 100, "tokens": P, "starts": P, "seqs": 2, "drafts": 3, "temperatures": P, "uniforms": P,
         "noise": P, "ldn": 100, "accepted": P, "next": P, "work": P, "bytes": 1 << 30, "stream": None}
    a.update(change)
    assert lib().crane_b200_draft_verify(*a.values()) == crane_b200.INVALID_ARG and said in crane_b200.load_library().crane_b200_device_last_error().decode()
    n = C.c_size_t()
    assert lib().crane_b200_draft_verify_bytes(0, 0, 1, 1, 1, C.byref(n)) == crane_b200.INVALID_ARG and lib().crane_b200_draft_verify_bytes(0, 9, 1, 1, 1, None) == crane_b200.INVALID_ARG


def test_tensors_are_refused():
    from crane_b200 import draft
    with pytest.raises(CraneB200Error, match="CUDA"):
        draft.verify(torch.zeros((2, 8)), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(1), torch.zeros((1, 8)))


# ------------------------------------------------------------------------------------------------------------------ results
def gen_of(*key):
    import zlib
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def softmax(x, t):
    """NaN counts as -inf; where the largest is +inf those share; all -inf: zeros."""
    x = torch.where(torch.isnan(x), -math.inf, x.double())
    top = x.max()
    if top == -math.inf:
        return torch.zeros_like(x)
    e = (x == top).double() if top == math.inf else torch.exp((x - top) / t)
    return e / e.sum()


def rule(logits, tokens, starts, uniforms, noise, q_logits, temps):
    accepted, following, decided = [], [], True
    v = logits.shape[1]
    for b in range(len(starts) - 1):
        s, n, t = starts[b], starts[b + 1] - starts[b], temps[b]
        j = 0
        while True:
            row = torch.where(torch.isnan(logits[s + b + j]), torch.tensor(-math.inf, device="cuda", dtype=logits.dtype), logits[s + b + j])
            first = int(torch.nonzero(row == row.max())[0]) if row.max() > -math.inf else -1
            p = softmax(row, t) if t > 0 else None
            if j == n:
                break
            d = int(tokens[s + j])
            if not 0 <= d < v:
                break
            if t <= 0:
                if d != first:
                    break
            else:
                q = 1.0 if q_logits is None else float(softmax(q_logits[s + j], t)[d])
                uq, pd = float(uniforms[s + j]) * q, float(p[d])
                if uq == pd == 0 or not uq < pd:
                    decided = decided and (uq - pd > MARGIN * pd or uq == pd == 0)
                    break
                decided = decided and pd - uq > MARGIN * pd
            j += 1
        accepted.append(j)
        if t <= 0 or first < 0:
            following.append(first)
            continue
        w = p
        if j < n:
            if q_logits is None:
                w = p.clone()
                if 0 <= int(tokens[s + j]) < v:
                    w[int(tokens[s + j])] = 0
            else:
                w = (p - softmax(q_logits[s + j], t)).clamp_min(0)
            if not (w > 0).any():
                w = p
        key = w / -torch.log(noise[b].double().clamp(2.0 ** -126, 1 - 2.0 ** -24))
        top = torch.topk(key, min(2, v)).values
        decided = decided and (v == 1 or float(top[1]) < float(top[0]) * (1 - MARGIN))
        following.append(int(key.argmax()))
    return accepted, following, decided


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def problem(g, dt, counts, v, near=1.0, temps=None):
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    total, seqs = starts[-1], len(counts)
    logits = torch.randn((total + seqs, v), generator=g, device="cuda") * 3
    at = [i + b for b in range(seqs) for i in range(starts[b], starts[b + 1])]
    q = (logits[at] + near * torch.randn((total, v), generator=g, device="cuda")).to(TYPES[dt])
    logits = logits.to(TYPES[dt])
    temps = temps or [0.0 if b % 4 == 3 else 0.5 + 0.25 * (b % 5) for b in range(seqs)]
    seq = [b for b in range(seqs) for _ in range(counts[b])]
    u = torch.rand((total, v), generator=g, device="cuda").clamp(1e-7, 0.999)
    tokens = [int((q[i].float() / temps[seq[i]] - torch.log(-torch.log(u[i]))).argmax()) if temps[seq[i]] > 0 else int(q[i].argmax()) for i in range(total)]
    return (logits, tokens, starts, torch.rand(total, generator=g, device="cuda"), torch.rand((seqs, v), generator=g, device="cuda").clamp(1e-7, 0.999), q, temps)


def run(p, with_q=True, **kw):
    from crane_b200 import draft
    logits, tokens, starts, uniforms, noise, q, temps = p
    a, f = draft.verify(logits, ints(tokens).reshape(-1), ints(starts), uniforms, noise, draft_logits=q if with_q else None,
                        temperatures=None if temps is None else torch.tensor(temps, dtype=torch.float32, device="cuda"), **kw)
    return a.tolist(), f.tolist()


def check(p, with_q=True):
    logits, tokens, starts, uniforms, noise, q, temps = p
    t32 = [1.0] * (len(starts) - 1) if temps is None else torch.tensor(temps, dtype=torch.float32).tolist()
    accepted, following, decided = rule(logits, tokens, starts, uniforms, noise, q if with_q else None, t32)
    assert decided, "the inputs leave a choice"
    assert run(p, with_q) == (accepted, following)
    return accepted


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("counts, v", [([0], 1), ([0], 7), ([1], 2), ([3], 5), ([4], 1000), ([2, 0, 5, 1, 7, 3], 513), ([7] * 9, 100), ([0, 0, 3], 32000), ([4], 151936), ([1, 2], 248320),
                                       ([40], 1001), ([3, 1] * 40, 64), ([5, 0, 2], 4099)])
def test_drafts(counts, v, dt):
    p = problem(gen_of("drafts", counts, v, dt), dt, counts, v)
    check(p)
    check(p, with_q=False)
    check(p[:6] + (None,))


@pytest.mark.gpu
def test_some_hold_and_some_do_not():
    p = problem(gen_of("some"), "f32", [6] * 30, 300, near=0.3)
    counts = check(p)
    assert len(set(counts)) >= 5 and 6 in counts


@pytest.mark.gpu
@pytest.mark.parametrize("with_q", [True, False])
def test_masked_rows_infinities_and_nan(with_q):
    """-inf where a mask took tokens away, NaN, +inf, rows of nothing, drafts outside the vocabulary, the types' lowest value as a mask."""
    for dt in TYPES:
        logits, tokens, starts, uniforms, noise, q, temps = problem(gen_of("masked", dt), dt, [2, 2, 2, 2, 2, 1, 1, 2], 200, temps=[1.0, 0.7, 1.0, 0.0, 1.0, 2.0, 0.0, 1.0])
        logits[:, 50:150], q[:, 50:150] = -math.inf, -math.inf
        low = torch.finfo(TYPES[dt]).min
        logits[0:3, :50] = low
        tokens[1] = 60                                                  # p and q are 0
        logits[3], q[2] = -math.inf, -math.inf                          # nothing there
        logits[6, 3:9], q[4, 5:7] = math.inf, math.inf
        logits[9, 7], tokens[6] = math.nan, 7
        logits[12:14, :40] = math.nan
        tokens[8], tokens[9] = 200, -1
        logits[15:17] = -math.inf                                       # the sixth sequence's, nothing there
        logits[18, 180:] = low
        p = (logits, tokens, starts, uniforms, noise, q, temps)
        accepted, following, _ = rule(logits, tokens, starts, uniforms, noise, q if with_q else None, [1.0, 0.7, 1.0, 0.0, 1.0, 2.0, 0.0, 1.0])
        got = run(p, with_q)
        assert got == (accepted, following) and got[1][5] == -1


@pytest.mark.gpu
def test_equal_rows_ties_and_borders():
    """Draft and target alike: all hold, whatever u below 1; equal keys and equal maxima: the lowest index; u of 0 and of 1; noise of 0 and of 1."""
    for dt in TYPES:
        logits, tokens, starts, uniforms, noise, q, _ = problem(gen_of("equal", dt), dt, [3, 3, 2], 128, temps=[1.0, 1.0, 0.0])
        for i, r in zip(range(8), (0, 1, 2, 4, 5, 6, 8, 9)):
            q[i] = logits[r]
        uniforms[:3], uniforms[3:6] = 0.0, 0.9375
        logits[8:] = 0
        tokens[6:] = [0, 1]
        logits[3] = 0.0
        noise[0] = 0.5
        noise[1, 5], noise[1, 9] = 0.0, 1.0
        accepted, following = run((logits, tokens, starts, uniforms, noise, q, [1.0, 1.0, 0.0]))
        assert accepted == [3, 3, 1] and following[0] == 0 and following[1] == 9 and following[2] == 0


@pytest.mark.gpu
def test_extreme_temperatures():
    for t in (1e-30, 1e-3, 1e6, 1e38):
        logits, tokens, starts, uniforms, noise, q, _ = problem(gen_of("hot", t), "f32", [2, 0], 300, temps=[1.0, 1.0])
        q[:] = logits[:2]
        p = (logits, [int(logits[0].argmax()), int(logits[1].argmax())], starts, uniforms * 0.5, noise, q, [t, t])
        accepted, following = run(p)
        assert accepted == [2, 0] and all(0 <= f < 300 for f in following)
        if t < 1:
            assert following == [int(logits[2].argmax()), int(logits[3].argmax())]


@pytest.mark.gpu
def test_infinite_and_negative_temperatures():
    """Infinite: all tokens above -inf alike, so the noise alone decides; below zero: greedy."""
    for dt in TYPES:
        logits, _, starts, uniforms, noise, q, _ = problem(gen_of("all", dt), dt, [2, 2], 300, temps=[1.0, 1.0])
        logits[:, 200:], q[:, 200:] = -math.inf, -math.inf
        first = [int(logits[i].argmax()) for i in range(6)]
        accepted, following = run((logits, [3, 250, first[3], first[4]], starts, uniforms * 0.5, noise, q, [math.inf, -1.0]))
        assert accepted == [1, 2] and following[0] == int(noise[0, :200].argmax()) and following[1] == first[5]


@pytest.mark.gpu
def test_rows_on_any_boundary():
    for dt in TYPES:
        p = problem(gen_of("rows", dt), dt, [2, 1, 3], 1001)
        want = run(p)
        for off, wide in ((1, 1003), (3, 1007), (8, 1024)):
            x, q = (torch.full((t.shape[0], wide + 8), 50.0, dtype=t.dtype, device="cuda") for t in (p[0], p[5]))
            x[:, off:off + 1001], q[:, off + 2:off + 1003] = p[0], p[5]
            noise = torch.zeros((3, wide + 1), device="cuda")
            noise[:, 1:1002] = p[4]
            assert run((x[:, off:off + 1001], p[1], p[2], p[3], noise[:, 1:1002], q[:, off + 2:off + 1003], p[6])) == want


@pytest.mark.gpu
def test_starts_of_any_value_reach_nothing_outside():
    from crane_b200 import draft
    p = problem(gen_of("starts"), "f32", [2, 1, 3], 200)
    for starts in ([-5, 2 ** 30, 3, -2 ** 31], [6, 6, 6, 6], [3, 2, 1, 0]):
        a, f = run((p[0], p[1], starts) + p[3:])
        assert all(0 <= x <= 6 for x in a) and all(-1 <= x < 200 for x in f)


@pytest.mark.gpu
def test_results_repeat_and_calls_share_nothing():
    from crane_b200 import draft
    logits, tokens, starts, uniforms, noise, q, temps = p = problem(gen_of("repeat"), "bf16", [3, 1, 4], 5000)
    want = run(p)
    t, s, h = ints(tokens), ints(starts), torch.tensor(temps, device="cuda")
    outs = []
    for st in [torch.cuda.Stream() for _ in range(3)] * 3:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            outs.append(draft.verify(logits, t, s, uniforms, noise, draft_logits=q, temperatures=h))
    torch.cuda.synchronize()
    assert all((a.tolist(), f.tolist()) == want for a, f in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, f = draft.verify(logits, t, s, uniforms, noise, draft_logits=q, temperatures=h)
    graph.replay()
    assert (a.tolist(), f.tolist()) == want
    uniforms.zero_()
    graph.replay()
    assert a.tolist() == rule(logits, tokens, starts, uniforms, noise, q, torch.tensor(temps).tolist())[0]


@pytest.mark.gpu
def test_tokens_come_out_as_the_target_draws_them():
    """Two drafted tokens over a small vocabulary, 20 000 times: the first token out is distributed as p.  Each count is a binomial one: five standard deviations."""
    g = gen_of("distribution")
    n, v = 20000, 6
    x, y = torch.randn(v, generator=g, device="cuda"), torch.randn(v, generator=g, device="cuda")
    q = softmax(y, 1.0)
    tokens = torch.multinomial(q.float(), 2 * n, replacement=True, generator=g).to(torch.int32)
    from crane_b200 import draft
    a, f = draft.verify(x.repeat(3 * n, 1), tokens, torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device="cuda"), torch.rand(2 * n, generator=g, device="cuda"),
                        torch.rand((n, v), generator=g, device="cuda").clamp(1e-7, 1 - 1e-7), draft_logits=y.repeat(2 * n, 1))
    first = torch.where(a > 0, tokens[::2], f)
    p = softmax(x, 1.0)
    count = torch.bincount(first.long(), minlength=v).double()
    assert bool(((count - n * p).abs() <= 5 * torch.sqrt(n * p * (1 - p)) + 1).all())


# ------------------------------------------------------------------------------------------------------------------ borders: sums that matter are those of 64 bits
# Sums of 64-bit terms are off by 2^-40 at most (terms 2^-51, up to 2^28 of them in any order); f32 uniforms near a border are chosen farther from it than that.
@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("v", [1, 2, 127, 1001, 4099, 32003, 151937])
def test_equal_rows_hold_whatever_u_below_one_and_wherever_they_lie(v, dt):
    """Draft rows are the target's at every other boundary: u q < p for the largest u below 1; not for u = 1.  Behind a refused one p - q is zero everywhere: the race is over p."""
    from crane_b200 import draft
    g = gen_of("equal rows", v, dt)
    n, seqs = 8, 4
    x = (torch.randn((n * seqs + seqs, v), generator=g, device="cuda") * 3).to(TYPES[dt])
    at = [i + i // n for i in range(n * seqs)]
    wide = torch.zeros((n * seqs, v + 9), dtype=TYPES[dt], device="cuda")
    starts = ints([i * n for i in range(seqs + 1)])
    tokens = torch.randint(0, v, (n * seqs,), generator=g, device="cuda").to(torch.int32)
    noise = torch.rand((seqs, v), generator=g, device="cuda").clamp(1e-7, 0.999)
    temps = [1.0, 0.7, 0.3, 3.0]
    for off in range(8):
        q = wide[:, off:off + v]
        q.copy_(x[at])
        u = torch.full((n * seqs,), 1 - 2.0 ** -24, device="cuda")
        a, f = draft.verify(x, tokens, starts, u, noise, draft_logits=q, temperatures=torch.tensor(temps, device="cuda"))
        p = [softmax(x[b * (n + 1) + n], float(torch.tensor(temps[b]))) for b in range(seqs)]
        alive = [int(j) for j in a]
        for b in range(seqs):                                           # (a token so unlikely that its probability is 0 is not accepted)
            none = [j for j in range(n) if float(softmax(x[b * (n + 1) + j], float(torch.tensor(temps[b])))[int(tokens[b * n + j])]) == 0]
            assert alive[b] == (none[0] if none else n)
            if not none:
                assert int(f[b]) == int((p[b] / -torch.log(noise[b].double())).argmax())
        u[3::n] = 1.0
        a, f = draft.verify(x, tokens, starts, u, noise, draft_logits=q, temperatures=torch.tensor(temps, device="cuda"))
        for b in range(seqs):
            assert int(a[b]) <= 3
            if int(a[b]) == 3:
                assert int(f[b]) == int((softmax(x[b * (n + 1) + 3], float(torch.tensor(temps[b]))) / -torch.log(noise[b].double())).argmax())


@pytest.mark.gpu
@pytest.mark.parametrize("with_q", [True, False])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("v", [5, 1001, 32000, 151937])
def test_uniforms_next_to_the_border(v, dt, with_q):
    """u is the f32 number just below p / q, or at most two steps above it: 2^-24 of itself away from the border where the sums are of 2^-20."""
    g = gen_of("border", v, dt)
    for t in (1.0, 0.6, 2.0):
        logits, tokens, starts, uniforms, noise, q, temps = problem(g, dt, [5] * 12, v, near=1.0, temps=[t] * 12)
        t32 = float(torch.tensor(t))
        seq = [i // 5 for i in range(60)]
        for i in range(60):
            p, y = softmax(logits[i + seq[i]], t32), softmax(q[i], t32) if with_q else None
            ratio = (p / y) if with_q else p
            ok = torch.nonzero((ratio < 0.9) & (ratio > 1e-30))[:, 0]
            if not len(ok):
                uniforms[i] = 0.0
                continue
            tokens[i] = int(ok[int(torch.randint(0, len(ok), (1,), generator=g, device="cuda"))])
            border = float(ratio[tokens[i]])
            u = torch.tensor(border, dtype=torch.float32)
            below = u if float(u) < border * (1 - 2.0 ** -40) else torch.nextafter(u, torch.tensor(0.0))
            if float(below) >= border * (1 - 2.0 ** -40):
                below = torch.nextafter(below, torch.tensor(0.0))
            above = u if float(u) > border * (1 + 2.0 ** -40) else torch.nextafter(u, torch.tensor(1.0))
            uniforms[i] = above if i % 5 == 4 and seq[i] % 2 or i % 5 == seq[i] % 5 and seq[i] % 3 == 0 else below
        accepted, following, _ = rule(logits, tokens, starts, uniforms, noise, q if with_q else None, [t32] * 12)
        assert run((logits, tokens, starts, uniforms, noise, q, temps), with_q) == (accepted, following)
        assert len(set(accepted)) > 1


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
def test_races_between_keys_next_to_one_another(dt):
    """p - q is a small part of p, a hundredth at one place, a thousandth at another, so that sums of 2^-20 would turn the order of their keys round: those are next to one another in 64 bits."""
    from crane_b200 import draft
    for v in (300, 5003, 151937):
        g = gen_of("race", v, dt)
        seqs = 16
        logits = torch.randn((2 * seqs, v), generator=g, device="cuda")
        q = (logits[0::2] + 0.01 * torch.randn((seqs, v), generator=g, device="cuda")).to(TYPES[dt])
        logits = logits.to(TYPES[dt])
        noise = torch.full((seqs, v), 1e-30, device="cuda")             # (a clock of 69 everywhere else)
        want = []
        for b in range(seqs):
            size = softmax(logits[2 * b], 1.0)
            w = (size - softmax(q[b], 1.0)).clamp_min(0)
            i, j = int(w.argmax()), int((w * (w < 0.1 * w.max()) * (w < 0.002 * size)).argmax())
            assert w[j] > 0 and float(w[j]) * 69 / 0.01 > 4 * float(w[i])
            noise[b, j] = 0.99
            key = float(w[j]) / -math.log(float(noise[b, j]))
            u = torch.tensor(math.exp(-float(w[i]) / key), dtype=torch.float32)      # i's key beside j's: the f32 number of the wanted side that is nearest
            for _ in range(4):
                over = float(w[i]) / -math.log(float(u)) / key - 1
                if over > 2.0 ** -36 if b % 2 else over < -2.0 ** -36:
                    break
                u = torch.nextafter(u, torch.tensor(1.0 if b % 2 else 0.0))
            noise[b, i] = u
            keys = w / -torch.log(noise[b].double().clamp(2.0 ** -126, 1 - 2.0 ** -24))
            want.append(int(keys.argmax()))
            top = torch.topk(keys, 2)
            assert set(top.indices.tolist()) == {i, j} and float(top.values[1]) < float(top.values[0]) * (1 - 2.0 ** -36)
        tokens = torch.tensor([int((softmax(q[b], 1.0) - softmax(logits[2 * b], 1.0)).argmax()) for b in range(seqs)], dtype=torch.int32, device="cuda")
        a, f = draft.verify(logits, tokens, ints(list(range(seqs + 1))), torch.ones(seqs, device="cuda"), noise, draft_logits=q)
        assert a.tolist() == [0] * seqs and f.tolist() == want


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
def test_many_drafts_next_to_the_border_in_a_replayed_graph(dt):
    """More drafts than a block has warps or keeps sums of, every one too close to call by f32 sums; sequences of few beside them; the refused ones change between replays."""
    from crane_b200 import draft
    g = gen_of("many border", dt)
    counts, v = [70, 3, 0, 40], 777
    starts = [0, 70, 73, 73, 113]
    x = (torch.randn((117, v), generator=g, device="cuda") * 2).to(TYPES[dt])
    at = [i + b for b in range(4) for i in range(starts[b], starts[b + 1])]
    wide = torch.zeros((113, v + 3), dtype=TYPES[dt], device="cuda")
    q = wide[:, 1:v + 1].copy_(x[at])
    tokens = [int(t) for t in torch.randint(0, v, (113,), generator=g, device="cuda")]
    noise = torch.rand((4, v), generator=g, device="cuda").clamp(1e-7, 0.999)
    u = torch.full((113,), 1 - 2.0 ** -24, device="cuda")
    t, s = ints(tokens), ints(starts)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, f = draft.verify(x, t, s, u, noise, draft_logits=q)
    for refused in ([], [50, 112], [0, 71, 73], [69, 72, 107]):
        u.fill_(1 - 2.0 ** -24)
        u[refused] = 1.0
        graph.replay()
        want = [min([i - starts[b] for i in refused if starts[b] <= i < starts[b + 1]], default=counts[b]) for b in range(4)]
        assert a.tolist() == want
        for b in range(4):                                              # p - q is zero everywhere: the race is over p
            assert int(f[b]) == int((softmax(x[starts[b] + b + want[b]], 1.0) / -torch.log(noise[b].double())).argmax())
