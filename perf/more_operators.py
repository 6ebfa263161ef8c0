"""Timed cases of what a batch server runs between its linears on tensors it keeps on the device: a paged key/value cache in 8 bits with a scale for every page
and head (`crane_b200.kv8`: rows into the cache, attention over it), low-rank adapters of many requests beside a shared projection (`crane_b200.lora`), and the
verification of drafted tokens from given random numbers (`crane_b200.draft`).

Head counts, widths and vocabularies are those of the dense and hybrid configurations in `crane_b200.synth`, and odd ones.
"""
import math
import random

import torch

own = False                      # False: elementary torch operations in 32 bits (64 where noted); True: the framework's kernels

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
F8 = torch.float8_e4m3fn
TOP = 448.0                      # largest e4m3 value
TINY = 2.0 ** -100               # largest magnitudes of a page below this count as this


# ------------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a decode round of a server: each of 64 sequences stores the keys and values of one token
        {"name": "append_round", "op": "append", "mix": "token", "seqs": 64, "rows": 1, "longest": 500, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # four long prompts come in together
        {"name": "append_prompt", "op": "append", "mix": "prompt", "seqs": 4, "rows": 2048, "longest": 4096, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # one user's next token over a conversation of middling length: latency
        {"name": "attend_token", "op": "attend", "mix": "token", "seqs": 1, "rows": 1, "longest": 1573, "heads": 16, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # a decode round: 64 sequences of very different lengths, bound by the cache's bytes
        {"name": "attend_round", "op": "attend", "mix": "token", "seqs": 64, "rows": 1, "longest": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # drafted tokens of 16 sequences at the hybrid configuration's wide heads, small pages
        {"name": "attend_drafts", "op": "attend", "mix": "drafts", "seqs": 16, "rows": 5, "longest": 16000, "heads": 8, "kv_heads": 2, "dim": 256, "page": 16, "dtype": "f16"},
        # portions of prompts beside decoded tokens, in the engine's own f32
        {"name": "attend_step", "op": "attend", "mix": "step", "seqs": 23, "rows": 333, "longest": 3001, "heads": 16, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "f32"},
        # the next portion of two long prompts: bound by the products
        {"name": "attend_prompt", "op": "attend", "mix": "prompt", "seqs": 2, "rows": 4096, "longest": 12288, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # one token's adapter beside its q, k and v projections: latency
        {"name": "lora_token", "op": "lora", "m": 1, "k": 2048, "n": 4096, "rank": 16, "adapters": 8, "runs": 1, "dtype": "bf16"},
        # a decode round: 33 requests of some twenty tenants beside the gate and up projections, f32 activations
        {"name": "lora_round", "op": "lora", "m": 33, "k": 4096, "n": 24576, "rank": 16, "adapters": 64, "runs": 20, "dtype": "f32"},
        # several tenants' long prompts beside the gate and up projections
        {"name": "lora_prompt", "op": "lora", "m": 8192, "k": 4096, "n": 24576, "rank": 64, "adapters": 16, "runs": 5, "dtype": "bf16"},
        # one user's four drafted tokens
        {"name": "verify_one", "op": "verify", "seqs": 1, "drafts": 4, "vocab": 151936, "greedy": 0.0, "dtype": "f32"},
        # a round of 64 sequences with up to seven drafted tokens each, one in eight of them greedy
        {"name": "verify_round", "op": "verify", "seqs": 64, "drafts": 7, "vocab": 151936, "greedy": 0.125, "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "lora", "lora", "verify"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    if op in ("append", "attend"):
        heads, kv_heads, dim = rng.choice(((16, 8, 128), (32, 8, 128), (8, 2, 256), (4, 2, 64), (6, 3, 128), (7, 1, 64)))
        mix = rng.choice(("token", "drafts", "prompt", "step"))
        case = {"op": op, "mix": mix, "seqs": _log(rng, 1, 64), "rows": 1, "longest": _log(rng, 8, 500 if op == "append" else 12288), "heads": heads, "kv_heads": kv_heads,
                "dim": dim, "page": rng.choice((16, 32, 64, 128)), "dtype": dtype}
        if mix == "drafts":
            case["rows"] = rng.randint(2, 9)
        elif mix != "token":
            case["seqs"] = _log(rng, 1, 8 if mix == "prompt" else 23)
            case["rows"] = _log(rng, 10, 2048)
            while op == "attend" and case["seqs"] * case["rows"] * case["longest"] * heads > 2 * 4096 * 12288 * 32:
                case["rows"] = (case["rows"] + 1) // 2
        case["longest"] = max(case["longest"], case["rows"])
        return case
    if op == "lora":
        case = {"op": op, "m": _log(rng, 1, 8192), "k": _log(rng, 64, 12288), "n": _log(rng, 16, 24576), "rank": _log(rng, 1, 128), "adapters": _log(rng, 1, 64), "dtype": dtype}
        case["runs"] = _log(rng, 1, min(64, case["m"]))
        while case["m"] * (case["n"] + case["k"]) * BYTES[dtype] > 8192 * 28672 * 2:
            case["m"] = max(1, case["m"] // 2)
        return case
    case = {"op": op, "seqs": _log(rng, 1, 64), "drafts": rng.randint(0, 7), "vocab": rng.choice((151936, 248320, _log(rng, 100, 150000))), "greedy": rng.choice((0.0, 0.25, 1.0)),
            "dtype": dtype}
    while case["seqs"] * (case["drafts"] + 1) * case["vocab"] > 64 * 8 * 151936:
        case["seqs"] //= 2
    return case


def _ragged(case):
    """New rows and lengths (new rows among them) of a case's sequences."""
    r = random.Random("/".join(str(case[k]) for k in ("mix", "seqs", "rows", "longest")))
    new, lens = [], []
    for b in range(case["seqs"]):
        n = case["rows"]
        if case["mix"] == "drafts":
            n = r.randint(1, n)
        elif case["mix"] == "prompt":
            n = r.randint(n - n // 10, n)
        elif case["mix"] == "step":              # the first sequence and a quarter of the rest bring portions
            n = n if b == 0 else r.randint(1, n) if r.random() < 0.25 else 1
        new.append(n)
        lens.append(case["longest"] if b == 0 else r.randint(n, case["longest"]))
    return new, lens


def _starts(new):
    s = [0]
    for n in new:
        s.append(s[-1] + n)
    return s


def _drafts(case):
    """Drafted tokens of a case's sequences."""
    r = random.Random("%d/%d" % (case["seqs"], case["drafts"]))
    return [case["drafts"] if b == 0 else r.randint(0, case["drafts"]) for b in range(case["seqs"])]


def _adapters(case):
    """Which adapter each row of a case goes through (-1: none), in runs of one request each."""
    r = random.Random("%d/%d/%d" % (case["m"], case["adapters"], case["runs"]))
    cuts = [0] + sorted(r.sample(range(1, case["m"]), min(case["runs"], case["m"]) - 1)) + [case["m"]]
    which = []
    for i, (a, b) in enumerate(zip(cuts, cuts[1:])):
        which += [-1 if i and r.random() < 0.1 else r.randrange(case["adapters"])] * (b - a)
    return which


# ---------------------------------------------------------------------------------------------------------------- what a program has in hand
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 1000003 + sum(v * (31 + 7 * i) for i, v in enumerate(case.values()) if type(v) is int))
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    s = dict(case)
    dt = DTYPES[case["dtype"]]
    if case["op"] in ("append", "attend"):
        new, lens = _ragged(case)
        h, d, p = case["kv_heads"], case["dim"], case["page"]
        need = [(n + p - 1) // p for n in lens]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((case["seqs"], max(need)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        # keys have a few columns that are much larger than the rest, and so has the first token of a sequence
        loud = 1 + 7 * (torch.rand((h, 1, d), generator=gen, device="cuda") < 0.02)
        s["k_codes"], s["v_codes"] = (torch.empty((pages, h, p, d), dtype=F8, device="cuda") for _ in range(2))
        s["scales"] = torch.empty((pages, h, 2), device="cuda")
        first = table[:, 0].long()
        for lo in range(0, pages, 512):
            hi = min(pages, lo + 512)
            for i, codes in enumerate((s["k_codes"], s["v_codes"])):
                y = normal(hi - lo, h, p, d) * (loud if i == 0 else 1)
                here = first[(first >= lo) & (first < hi)] - lo
                y[here, :, 0] *= 4 if i == 0 else 0.1
                scale = _scale(y.abs().amax((2, 3)))
                codes[lo:hi] = (y / scale[:, :, None, None]).to(F8)
                s["scales"][lo:hi, :, i] = scale
        rows = sum(new)
        s["table"], s["lens"], s["starts"] = table, ints(lens), ints(_starts(new))
        s["new"], s["lens_host"] = new, lens
        if case["op"] == "append":               # keys and values as the q, k and v projections leave them, side by side
            kv = (normal(rows, 2 * h, d) * torch.cat((loud.view(h, d), torch.ones_like(loud.view(h, d))))).to(dt)
            s["k"], s["v"] = kv[:, :h], kv[:, h:]
        else:
            s["q"] = normal(rows, case["heads"], d).to(dt)
            s["out"] = torch.zeros((rows, case["heads"], d), dtype=dt, device="cuda")
            s["scale"] = 1 / math.sqrt(d)
            s["max_rows"] = max(new)
        s["cache"] = s["k_codes"], s["v_codes"], s["scales"]
        return s
    if case["op"] == "lora":
        m, k, n, r = case["m"], case["k"], case["n"], case["rank"]
        s["x"] = (normal(m, k) * (1 + 15 * (torch.rand(k, generator=gen, device="cuda") < 0.01))).to(dt)
        s["a"] = (normal(case["adapters"], r, k) / math.sqrt(k)).to(dt)
        s["b"] = (normal(case["adapters"], n, r) * (0.3 / math.sqrt(r))).to(dt)
        s["scales"] = 0.5 + 1.5 * torch.rand(case["adapters"], generator=gen, device="cuda")
        s["which_host"] = _adapters(case)
        s["which"] = ints(s["which_host"])
        s["add"] = normal(m, n).to(dt)
        s["out"] = torch.empty((m, n), dtype=dt, device="cuda")
        return s
    drafts, v = _drafts(case), case["vocab"]
    total = sum(drafts)
    rows = total + case["seqs"]
    starts = _starts(drafts)
    logits = normal(rows, v).mul_(3.0)
    # a draft model says nearly what the target says, and drafts are drawn from what it says
    target_rows = ints([i + b for b in range(case["seqs"]) for i in range(starts[b], starts[b + 1])]).long()
    s["draft_logits"] = torch.empty((total, v), dtype=dt, device="cuda")
    s["tokens"] = torch.empty(total, dtype=torch.int32, device="cuda")
    temps = [0.6 + 0.1 * (b % 8) if b >= case["greedy"] * case["seqs"] else 0.0 for b in range(case["seqs"])]
    for i in range(total):
        b = next(j for j in range(case["seqs"]) if starts[j + 1] > i)
        y = (logits[target_rows[i]] + normal(v)).to(dt)
        s["draft_logits"][i] = y
        u = torch.rand(v, generator=gen, device="cuda").clamp_(1e-7, 0.999)
        s["tokens"][i] = (y if temps[b] == 0 else y.float() / temps[b] - torch.log(-torch.log(u))).argmax().to(torch.int32)
    s["logits"] = logits.to(dt)
    s["starts"], s["starts_host"] = ints(starts), starts
    s["temperatures"], s["temps_host"] = torch.tensor(temps, device="cuda"), temps
    s["uniforms"] = torch.rand(total, generator=gen, device="cuda")
    s["noise"] = torch.rand((case["seqs"], v), generator=gen, device="cuda").clamp_(1e-7, 0.999)
    return s


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _scale(top):
    """The smallest power of two whose 448-fold holds the magnitudes."""
    m, e = torch.frexp(top.clamp_min(TINY))              # top = m 2^e, m in [0.5, 1); 448 = 0.875 x 2^9
    return torch.ldexp(torch.ones_like(top), e - 9 + (m > 0.875))


def _append(s):
    """Rows into their pages: a page that is begun takes the new rows' scale, one that is continued the larger of its own and theirs."""
    p, count = s["page"], s["starts"].diff()
    seq = torch.repeat_interleave(torch.arange(s["seqs"], device="cuda"), count, output_size=s["k"].shape[0])
    pos = (s["lens"] - s["starts"][1:])[seq] + torch.arange(seq.shape[0], device="cuda")
    first = s["lens"] - count                            # where each sequence's new rows begin
    begun = s["table"].gather(1, (first // p)[:, None].long())[:, 0].long()
    _append_half(s["k"].float(), s["k_codes"], s["scales"][:, :, 0], s["table"][seq, pos // p].long(), pos % p, begun, first % p)
    _append_half(s["v"].float(), s["v_codes"], s["scales"][:, :, 1], s["table"][seq, pos // p].long(), pos % p, begun, first % p)
    return s["cache"]


def _append_half(x, codes, scales, page, offset, begun, kept):
    top = torch.zeros_like(scales).scatter_reduce_(0, page[:, None].expand(-1, scales.shape[1]), x.abs().amax(2), "amax")
    new = _scale(top[begun])
    new = torch.where(kept[:, None] > 0, torch.maximum(new, scales[begun]), new)
    old = codes[begun].float() * (scales[begun] / new)[:, :, None, None]
    mine = torch.arange(codes.shape[2], device="cuda") < kept[:, None]
    bits = codes.view(torch.uint8)
    bits[begun] = torch.where(mine[:, None, :, None], old.to(F8).view(torch.uint8), bits[begun])
    scales[page] = _scale(top[page])
    scales[begun] = new
    bits[page, :, offset] = (x / scales[page][:, :, None]).to(F8).view(torch.uint8)


def _attend(s):
    h, d, p, length = s["kv_heads"], s["dim"], s["page"], s["longest"]
    g, count = s["heads"] // h, s["starts"].diff()
    slot = torch.arange(max(s["new"]), device="cuda")
    real = slot < count[:, None]                         # sequences side by side, as many rows each as the one with the most
    row = (s["starts"][:-1, None] + slot).clamp_max(s["q"].shape[0] - 1).long()
    hidden = torch.arange(length, device="cuda") > (s["lens"] - count)[:, None, None] + slot[:, None]
    at = torch.arange(length, device="cuda")
    page, offset = s["table"][:, at // p].clamp_min(0).long(), at % p
    for head in range(h):                                # (all heads' scores at once would not fit)
        k, v = (codes.view(torch.uint8)[page, head, offset].view(F8).float() * s["scales"][page, head, i][:, :, None] for i, codes in enumerate(s["cache"][:2]))
        v.masked_fill_((at >= s["lens"][:, None])[:, :, None], 0)
        q = s["q"][row, head * g:head * g + g].float().flatten(1, 2)
        score = (q @ k.transpose(1, 2)).mul_(s["scale"]).view(s["seqs"], -1, g, length)
        score.masked_fill_(hidden[:, :, None], -math.inf)
        w = score.sub_(score.amax(3, keepdim=True)).exp_()
        o = (w.view(s["seqs"], -1, length) @ v).view(s["seqs"], -1, g, d) / w.sum(3, keepdim=True)
        s["out"][:, head * g:head * g + g] = o[real].to(s["out"].dtype)
    return s["out"]


def _lora(s):
    out = s["add"].float().clone()
    which, i = s["which_host"], 0
    while i < len(which):
        j = i + 1
        while j < len(which) and which[j] == which[i]:
            j += 1
        w = which[i]
        if w >= 0:
            out[i:j] += s["scales"][w] * ((s["x"][i:j].float() @ s["a"][w].float().t()) @ s["b"][w].float().t())
        i = j
    s["out"].copy_(out)
    return s["out"]


def _verify(s):
    """Probabilities in 64 bits: a token beside the border of two would otherwise be another one."""
    seqs, v = s["noise"].shape
    count, starts = s["starts"].diff().long(), s["starts"].long()
    total = s["tokens"].shape[0]
    seq = torch.repeat_interleave(torch.arange(seqs, device="cuda"), count, output_size=total)
    target = torch.arange(total, device="cuda") + seq    # the logits row that a drafted token is held against; a sequence has one more behind its drafts
    rows_of = torch.repeat_interleave(torch.arange(seqs, device="cuda"), count + 1, output_size=total + seqs)
    t = torch.where(s["temperatures"] > 0, s["temperatures"], 1.0).double()
    greedy = s["temperatures"] <= 0
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    at = torch.arange(v, device="cuda")
    best = torch.where(x == top, at, v).amin(1)
    p = torch.exp((x - top) / t[rows_of][:, None])
    p /= p.sum(1, keepdim=True)
    p = torch.where(greedy[rows_of][:, None], (at == best[:, None]).double(), p)
    y = s["draft_logits"].double()
    q = torch.exp((y - y.amax(1, keepdim=True)) / t[seq][:, None])
    q /= q.sum(1, keepdim=True)
    q.masked_fill_(greedy[seq][:, None], 0)
    d = s["tokens"].long()[:, None]
    refused = s["uniforms"].double() * q.gather(1, d)[:, 0] >= p[target].gather(1, d)[:, 0]
    place = torch.where(refused, torch.arange(total, device="cuda") - starts[seq], v)
    accepted = count.scatter_reduce(0, seq, place, "amin")
    left = p[starts[:-1] + torch.arange(seqs, device="cuda") + accepted]
    behind = torch.cat((q, q.new_zeros((1, v))))[torch.where(accepted < count, starts[:-1] + accepted, total)]
    rest = (left - behind).clamp_min(0)
    race = torch.where(rest.sum(1, keepdim=True) > 0, rest, left) / -torch.log(s["noise"].double())
    following = torch.where(race == race.amax(1, keepdim=True), at, v).amin(1)
    return accepted.int(), following.int()


def run(s):
    op = s["op"]
    if not own:
        return {"append": _append, "attend": _attend, "lora": _lora, "verify": _verify}[op](s)
    if op == "append":
        from crane_b200 import kv8
        kv8.append(s["k"], s["v"], s["cache"], s["table"], s["lens"], s["starts"])
        return s["k_codes"], s["v_codes"], s["scales"]
    if op == "attend":
        from crane_b200 import kv8
        return kv8.attention(s["q"], s["cache"], s["table"], s["lens"], s["starts"], scale=s["scale"], max_rows=s["max_rows"], out=s["out"])
    if op == "lora":
        from crane_b200 import lora
        return lora.linear(s["x"], s["a"], s["b"], s["which"], scales=s["scales"], add=s["add"], out=s["out"])
    from crane_b200 import draft
    return draft.verify(s["logits"], s["tokens"], s["starts"], s["uniforms"], s["noise"], draft_logits=s["draft_logits"], temperatures=s["temperatures"])


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "append":
        new, _ = _ragged(case)
        values = 2 * sum(new) * case["kv_heads"] * case["dim"]
        pages = sum((n + case["page"] - 1) // case["page"] for n in new)
        return {"bytes": values * (e + 1) + 8 * pages * case["kv_heads"], "flops": 2 * values}
    if case["op"] == "attend":
        new, lens = _ragged(case)
        seen = sum(n * t - n * (n - 1) // 2 for n, t in zip(new, lens))
        pages = sum((t + case["page"] - 1) // case["page"] for t in lens)
        return {"bytes": 2 * sum(lens) * case["kv_heads"] * case["dim"] + 8 * pages * case["kv_heads"] + 2 * sum(new) * case["heads"] * case["dim"] * e,
                "flops": 4 * seen * case["heads"] * case["dim"]}
    if case["op"] == "lora":
        which = _adapters(case)
        rows, used = sum(w >= 0 for w in which), len(set(w for w in which if w >= 0))
        m, k, n, r = case["m"], case["k"], case["n"], case["rank"]
        return {"bytes": e * (rows * k + used * r * (k + n) + 2 * m * n) + 4 * m, "flops": 2 * rows * r * (k + n)}
    drafts, temps = _drafts(case), case["greedy"]
    drawn = [n for b, n in enumerate(drafts) if b >= temps * case["seqs"]]
    rows = sum(drafts) + len(drafts) + sum(drawn)
    return {"bytes": case["vocab"] * (e * rows + 4 * len(drawn)) + 8 * sum(drafts), "flops": 4 * case["vocab"] * rows}


# --------------------------------------------------------------------------------------------------------- in 64 bits, from the definition
def _e4m3(v):
    """The nearest e4m3 value, ties to the even one: steps of 2^(e - 3) between 2^e and 2^(e + 1), of 2^-9 below 2^-6."""
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v.abs().clamp_min(2.0 ** -6))[1] - 4)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def _exact_append(s):
    p, out = s["page"], []
    scales = s["scales"].double().clone()
    for i, (x, codes) in enumerate(((s["k"], s["k_codes"]), (s["v"], s["v_codes"]))):
        pool = codes.double()
        starts = _starts(s["new"])
        for b, length in enumerate(s["lens_host"]):
            n = s["new"][b]
            for block in range((length - n) // p, (length - 1) // p + 1):
                lo, hi = max(block * p, length - n), min(block * p + p, length)
                rows = x[starts[b] + lo - (length - n):starts[b] + hi - (length - n)].double()
                page = int(s["table"][b, block])
                for head in range(s["kv_heads"]):
                    top = max(float(rows[:, head].abs().max()), TINY)
                    e = math.ceil(math.log2(top / TOP) - 1e-9)
                    while top > TOP * 2.0 ** e:
                        e += 1
                    while top <= TOP * 2.0 ** (e - 1):
                        e -= 1
                    if lo % p:
                        was = float(scales[page, head, i])
                        e = max(e, round(math.log2(was)))
                        pool[page, head, :lo % p] = _e4m3(pool[page, head, :lo % p] * was / 2.0 ** e)
                    pool[page, head, lo % p:lo % p + hi - lo] = _e4m3(rows[:, head] / 2.0 ** e)
                    scales[page, head, i] = 2.0 ** e
        out.append(pool)
    return out[0], out[1], scales


def _exact_attend(s):
    h, g, p = s["kv_heads"], s["heads"] // s["kv_heads"], s["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    starts = _starts(s["new"])
    for b, length in enumerate(s["lens_host"]):
        n = s["new"][b]
        pages = s["table"][b, :(length + p - 1) // p].long()
        for head in range(h):
            k = (s["k_codes"][pages, head].double() * s["scales"][pages, head, 0].double()[:, None, None]).flatten(0, 1)[:length]
            v = (s["v_codes"][pages, head].double() * s["scales"][pages, head, 1].double()[:, None, None]).flatten(0, 1)[:length]
            for i in range(head * g, head * g + g):
                score = s["q"][starts[b]:starts[b + 1], i].double() @ k.t() * s["scale"]
                score += torch.full_like(score, -math.inf).triu_(length - n + 1)
                out[starts[b]:starts[b + 1], i] = torch.softmax(score, 1) @ v
    return out


def _exact_verify(s):
    accepted, following = [], []
    for b, t in enumerate(s["temps_host"]):
        lo, n = s["starts_host"][b], s["starts_host"][b + 1] - s["starts_host"][b]
        t = float(s["temperatures"][b])
        count = 0
        while True:
            x = s["logits"][lo + b + count].double()
            p = torch.softmax(x / t, 0) if t > 0 else (torch.arange(x.shape[0], device="cuda") == torch.nonzero(x == x.max())[0]).double()
            if count == n:
                break
            q = torch.softmax(s["draft_logits"][lo + count].double() / t, 0) if t > 0 else None
            d = int(s["tokens"][lo + count])
            if t > 0:
                if not float(s["uniforms"][lo + count]) * float(q[d]) < float(p[d]):
                    p = (p - q).clamp_min(0) if bool((p > q).any()) else p
                    break
            elif float(p[d]) == 0:
                break
            count += 1
        key = p / -torch.log(s["noise"][b].double()) if t > 0 else p
        accepted.append(count)
        following.append(int(torch.nonzero(key == key.max())[0]))
    return torch.tensor(accepted, dtype=torch.int32, device="cuda"), torch.tensor(following, dtype=torch.int32, device="cuda")


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["op"] == "verify":
        return _exact_verify(s)
    y = s["add"].double()
    which = s["which"].long()
    for w in sorted(set(s["which_host"]) - {-1}):
        at = torch.nonzero(which == w)[:, 0]
        t = s["x"][at].double() @ s["a"][w].double().t()
        y[at] += t @ s["b"][w].double().t() * s["scales"][w].double()
    return y
