"""Verification of drafted tokens against the target model's probabilities, on CUDA tensors:

    accepted, following = draft.verify(logits, tokens, starts, uniforms, noise, draft_logits=draft_logits, temperatures=temperatures)

The target's tokens come out distributed as if it had drawn them itself.  Random numbers are inputs, as everywhere in this package.  Calls run on the tensors' device and its current
stream, wait for nothing, keep nothing and may be captured into graphs.
"""
from __future__ import annotations

import ctypes as C

import torch

from .fp8 import _F32, _failed, _matrix, _raw_stream, _refuse, _rows_in
from .kv8 import _entry, _ints


def _floats(what: str, t, dev: int, n: int):
    if not isinstance(t, torch.Tensor) or t.dtype is not _F32 or t.shape != (n,) or t.get_device() != dev or (n > 1 and t.stride(0) != 1):
        _refuse(f"{what}: {n} contiguous f32 values on cuda:{dev} are wanted")
    return t.data_ptr()


def verify(logits, tokens, starts, uniforms, noise, *, draft_logits=None, temperatures=None, out=None):
    """(accepted, following), int32 [sequences] each: how many of a sequence's drafts hold, and the token behind those.

    Sequence b has the drafts tokens[starts[b]:starts[b + 1]] (int32, starts [sequences + 1] int32 from 0) and the rows starts[b] + b to starts[b + 1] + b of logits
    [drafts + sequences, vocabulary] (f32, bf16 or f16): one ahead of each draft, one behind the last.  p and q: softmax of a row / temperature, the target's and the draft model's
    (draft_logits [drafts, vocabulary] of the same type; None: the drafts were certain).  Draft j holds while uniforms[j] * q(draft) < p(draft); behind it follows the first argmax of
    w / -log(noise[b]), w = max(p - q, 0) at the first that does not hold, or p behind the last.  temperatures [sequences] f32 (None: 1), 0: greedy.  noise
    [sequences, vocabulary] f32 between 0 and 1.  -1 follows a row without a logit above -inf."""
    dev, rows, vocab, ld, dtype = _rows_in("logits", logits)
    if not isinstance(tokens, torch.Tensor) or tokens.dim() != 1:
        _refuse("tokens: a 1-D tensor is wanted")
    total = tokens.shape[0]
    seqs = rows - total
    if seqs < 0:
        _refuse(f"logits: {rows} rows for {total} drafts and a row more for each sequence")
    tp, sp = _ints("tokens", tokens, dev, (total,)), _ints("starts", starts, dev, (seqs + 1,))
    up = _floats("uniforms", uniforms, dev, total)
    ldn = _matrix("noise", noise, (_F32,), logits.device, (seqs, vocab))
    ldq = 0 if draft_logits is None else _matrix("draft_logits", draft_logits, (logits.dtype,), logits.device, (total, vocab))
    temps = None if temperatures is None else _floats("temperatures", temperatures, dev, seqs)
    if out is None:
        out = torch.empty((2, seqs), dtype=torch.int32, device=logits.device).unbind(0)
    accepted, following = out
    ap, fp = _ints("out[0]", accepted, dev, (seqs,)), _ints("out[1]", following, dev, (seqs,))
    need = C.c_size_t()
    rc = _entry("draft_verify_bytes")(dev, vocab, seqs, total, draft_logits is not None, C.byref(need))
    if rc:
        _failed(rc)
    work = torch.empty(need.value, dtype=torch.uint8, device=logits.device)
    rc = _entry("draft_verify")(dev, logits.data_ptr(), ld, None if draft_logits is None else draft_logits.data_ptr(), ldq, dtype, vocab, tp, sp, seqs, total, temps, up,
                                noise.data_ptr(), ldn, ap, fp, work.data_ptr(), need.value, _raw_stream(dev))
    if rc:
        _failed(rc)
    return accepted, following
