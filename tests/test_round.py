"""A batch server's round on device memory, as one graph that is replayed: every request's rows through a shared 8-bit projection and its own adapter, keys and values into the 8-bit cache,
attention over it, drafted tokens held against the result.  Each stage is checked on the inputs that it had, with that operator's own reference and tolerance; a round that follows takes back
the positions of drafts that did not hold."""
import math

import pytest
import torch

import test_draft
import test_kv8
import test_lora


@pytest.mark.gpu
def test_rounds_of_drafted_tokens():
    from crane_b200 import draft, fp8, kv8, lora
    g = torch.Generator(device="cuda").manual_seed(5)
    seqs, heads, kv, dim, hidden, vocab, page, adapters = 5, 8, 2, 64, 256, 331, 16, 3
    width = (heads + 2 * kv) * dim
    drafts = [3, 0, 2, 1, 3]
    starts = [0]
    for n in drafts:
        starts.append(starts[-1] + n)
    rows_at = [s + b for b, s in enumerate(starts)]                       # a row more than drafts for each sequence: the token ahead of them
    total, rows = starts[-1], starts[-1] + seqs
    lens = [0] * seqs
    order = torch.randperm(30, generator=g, device="cuda").tolist()
    table = [[order.pop() for _ in range(6)] for _ in range(seqs)]
    cache = kv8.pages(30, kv, dim, page)
    w = fp8.rows(width, hidden)[0]
    w.copy_((torch.randn((width, hidden), generator=g, device="cuda") * 60).clamp(-448, 448).to(fp8.CODES))
    ws = torch.rand((math.ceil(width / 128), 2), generator=g, device="cuda") * 1e-3
    a = (torch.randn((adapters, 8, hidden), generator=g, device="cuda") / 16).bfloat16()
    b = torch.randn((adapters, width, 8), generator=g, device="cuda").bfloat16()
    head = torch.randn((vocab, heads * dim), generator=g, device="cuda").bfloat16()
    x = torch.empty((rows, hidden), device="cuda", dtype=torch.bfloat16)
    which, t, l = torch.empty(rows, dtype=torch.int32, device="cuda"), test_kv8.ints(table), test_kv8.ints(lens)
    row_starts, draft_starts = test_kv8.ints(rows_at), test_kv8.ints(starts)
    tokens, u, noise = torch.zeros(total, dtype=torch.int32, device="cuda"), torch.rand(total, device="cuda"), torch.rand((seqs, vocab), device="cuda")
    q_logits = torch.zeros((total, vocab), device="cuda")
    temps = torch.tensor([1.0, 0.7, 0.0, 2.0, 1.0], device="cuda")

    def round_():
        codes, scales = fp8.quantize(x)
        shared = fp8.linear(codes, scales, w, ws)
        qkv = lora.linear(x, a, b, which, add=shared).view(rows, heads + 2 * kv, dim)
        kv8.append(qkv[:, heads:heads + kv], qkv[:, heads + kv:], cache, t, l, row_starts)
        out = kv8.attention(qkv[:, :heads], cache, t, l, row_starts, max_rows=4)
        logits = (out.view(rows, -1) @ head.t()).float() * 0.2
        return shared, qkv, out, logits, draft.verify(logits, tokens, draft_starts, u, noise, draft_logits=q_logits, temperatures=temps)

    def refill():
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        which.copy_(torch.randint(-1, adapters, (rows,), generator=g, device="cuda"))
        tokens.copy_(torch.randint(0, vocab, (total,), generator=g, device="cuda"))
        q_logits.copy_(torch.randn(q_logits.shape, generator=g, device="cuda"))
        u.copy_(torch.rand(total, generator=g, device="cuda") * 0.3)
        noise.copy_(torch.rand(noise.shape, generator=g, device="cuda").clamp(1e-6, 0.999))

    refill()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        round_()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        shared, qkv, out, logits, (accepted, following) = round_()
    for c, v in zip(cache, (0, 0, 1)):
        c.copy_(torch.full_like(c.float(), v).to(c.dtype))
    held = set()
    for _ in range(6):
        refill()
        lens = [n + d + 1 for n, d in zip(lens, drafts)]
        l.copy_(test_kv8.ints(lens))
        before = [c.double().clone() for c in cache]
        graph.replay()
        test_lora.check(qkv.view(rows, width), test_lora.reference(x, a, b, which, None, shared))
        test_kv8.plain_append(before, qkv[:, heads:heads + kv], qkv[:, heads + kv:], table, lens, rows_at)
        assert all(test_kv8.same(c.double(), want) for c, want in zip(cache, before))
        test_kv8.check(out, test_kv8.attend_ref(qkv[:, :heads], cache, table, lens, rows_at, dim ** -0.5))
        want = test_draft.rule(logits, tokens.tolist(), starts, u, noise, q_logits, temps.tolist())
        assert want[2] and (accepted.tolist(), following.tolist()) == want[:2]
        held.update(accepted.tolist())
        lens = [n - d + k for n, d, k in zip(lens, drafts, accepted.tolist())]      # positions of drafts that did not hold are written again
    assert len(held) > 1
