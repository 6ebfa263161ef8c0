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


_I32 = torch.int32
_sizes = {}                # bytes of workspaces by what they depend on


def _floats(what: str, t, dev: int, n: int):
    if not isinstance(t, torch.Tensor) or t.dtype is not _F32 or t.shape != (n,) or t.get_device() != dev or (n > 1 and t.stride(0) != 1):
        _refuse(f"{what}: {n} contiguous f32 values on cuda:{dev} are wanted")
    return t.data_ptr()


def verify(logits, tokens, starts, uniforms, noise, *, draft_logits=None, temperatures=None, out=None):
    """(accepted, following), int32 [sequences] each: how many of a sequence's drafts hold, and the token behind those.

    Sequence b has the drafts tokens[starts[b]:starts[b + 1]] (int32, starts [sequences + 1] int32 from 0) and the rows starts[b] + b to starts[b + 1] + b of logits
    [drafts + sequences, vocabulary] (f32, bf16 or f16): one ahead of each draft, one behind the last.  p and q: softmax of a row / temperature, the target's and the draft model's
    (draft_logits [drafts, vocabulary] of the same type; None: the drafts were certain).  Draft j holds while uniforms[j] * q(draft) < p(draft); behind it follows the first argmax of
    w / -log(noise[b]), w = max(p - q, 0) at the first that does not hold, or p behind the last.  temperatures [sequences] f32 (None: 1), 0 or less: greedy.  noise
    [sequences, vocabulary] f32 between 0 and 1.  -1 follows a row without a logit above -inf."""
    dev, rows, vocab, ld, dtype = _rows_in("logits", logits)
    if not isinstance(tokens, torch.Tensor) or tokens.dim() != 1:
        _refuse("tokens: a 1-D tensor is wanted")
    total = tokens.shape[0]
    seqs = rows - total
    if seqs < 0:
        _refuse(f"logits: {rows} rows for {total} drafts and a row more for each sequence")
    if out is None:
        out = torch.empty((2, seqs), dtype=_I32, device=logits.device).unbind(0)
    accepted, following = out
    q, temps = draft_logits, temperatures
    try:
        ldn, step = noise.stride()
        ldq, qstep = (0, 1) if q is None else q.stride()
        good = (step == qstep == 1 and tokens.dtype is _I32 and starts.dtype is _I32 and accepted.dtype is _I32 and following.dtype is _I32 and uniforms.dtype is _F32 and noise.dtype is _F32
                and starts.shape == (seqs + 1,) and uniforms.shape == (total,) and noise.shape == (seqs, vocab) and accepted.shape == (seqs,) and following.shape == (seqs,)
                and dev == tokens.get_device() == starts.get_device() == uniforms.get_device() == noise.get_device() == accepted.get_device() == following.get_device()
                and (q is None or (q.dtype is logits.dtype and q.shape == (total, vocab) and q.get_device() == dev and ldq >= vocab)) and ldn >= vocab
                and (temps is None or (temps.dtype is _F32 and temps.shape == (seqs,) and temps.get_device() == dev and temps.is_contiguous()))
                and tokens.is_contiguous() and starts.is_contiguous() and uniforms.is_contiguous() and accepted.is_contiguous() and following.is_contiguous())
    except (AttributeError, ValueError):
        good = False
    if not good:                                        # one by one, to name what is wrong or find a rarer layout good
        _ints("tokens", tokens, dev, (total,)), _ints("starts", starts, dev, (seqs + 1,)), _ints("out[0]", accepted, dev, (seqs,)), _ints("out[1]", following, dev, (seqs,))
        _floats("uniforms", uniforms, dev, total)
        ldn = _matrix("noise", noise, (_F32,), logits.device, (seqs, vocab))
        ldq = 0 if q is None else _matrix("draft_logits", q, (logits.dtype,), logits.device, (total, vocab))
        if temps is not None:
            _floats("temperatures", temps, dev, seqs)
    key = (dev, vocab, seqs, total, q is not None)
    need = _sizes.get(key)
    if need is None:
        n = C.c_size_t()
        rc = _entry("draft_verify_bytes")(*key, C.byref(n))
        if rc:
            _failed(rc)
        if len(_sizes) >= 4096:
            _sizes.clear()
        need = _sizes[key] = n.value
    work = torch.empty(need, dtype=torch.uint8, device=logits.device)
    rc = _entry("draft_verify")(dev, logits.data_ptr(), ld, None if q is None else q.data_ptr(), ldq, dtype, vocab, tokens.data_ptr(), starts.data_ptr(), seqs, total,
                                None if temps is None else temps.data_ptr(), uniforms.data_ptr(), noise.data_ptr(), ldn, accepted.data_ptr(), following.data_ptr(), work.data_ptr(), need,
                                _raw_stream(dev))
    if rc:
        _failed(rc)
    return accepted, following
