"""A paged key/value cache in 8 bits on CUDA tensors: e4m3 codes with a scale for every page and head, and attention over it.

    cache = kv8.pages(4096, kv_heads=8, dim=128)                      # (k codes, v codes, scales); any page may be any sequence's
    kv8.append(k, v, cache, table, lens, starts)                      # the new rows of all sequences into their pages
    out = kv8.attention(q, cache, table, lens, starts)                # each new row over what its sequence holds, itself included

`table` [sequences, pages] int32 has the pages of each sequence (the rest: any number outside the cache), `lens` [sequences] int32 the positions it holds, new rows included, and
`starts` [sequences + 1] int32 where each sequence's new rows begin: a decoded token, drafted ones, or portions of prompts, side by side.  These three are read on the device only.
Calls run on the tensors' device and its current stream, wait for nothing, keep nothing and may be captured into graphs.  Sequences may share pages that none of them writes.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import load_library
from .fp8 import _DTYPES, _failed, _raw_stream, _refuse, CODES

_F32, _I32 = torch.float32, torch.int32
_fn = {}


def _entry(name: str):
    fn = _fn.get(name)
    if fn is None:
        fn = _fn[name] = getattr(load_library(), "crane_b200_" + name)
    return fn


def pages(n: int, kv_heads: int, dim: int, page: int = 64, device="cuda"):
    """An empty cache of n pages of `page` positions: (k codes, v codes) [n, kv_heads, page, dim] and scales [n, kv_heads, 2]."""
    k, v = (torch.zeros((n, kv_heads, page, dim), dtype=CODES, device=device) for _ in range(2))
    return k, v, torch.ones((n, kv_heads, 2), dtype=_F32, device=device)


def _cache(cache):
    """(pointers, sizes, device index) of a cache."""
    try:
        k, v, scales = cache
        dev = k.get_device()
        n, h, p, d = k.shape
        if (k.dtype is CODES and v.dtype is CODES and scales.dtype is _F32 and v.shape == k.shape and scales.shape == (n, h, 2) and dev >= 0 and dev == v.get_device()
                and dev == scales.get_device() and k.is_contiguous() and v.is_contiguous() and scales.is_contiguous()):
            return (k.data_ptr(), v.data_ptr(), scales.data_ptr(), n, h, p, d), dev
    except (AttributeError, TypeError, ValueError):
        pass
    _refuse("cache: contiguous CUDA tensors (k codes, v codes [pages, kv_heads, page, dim], scales [pages, kv_heads, 2] f32), as pages() gives them, are wanted")


def _ints(what: str, t, dev: int, shape):
    if not isinstance(t, torch.Tensor) or t.dtype is not _I32 or t.get_device() != dev or t.dim() != len(shape) or any(s is not None and a != s for a, s in zip(t.shape, shape)):
        _refuse(f"{what}: int32 of shape {tuple('any' if s is None else s for s in shape)} on cuda:{dev} is wanted")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        _refuse(f"{what}: its last dimension is not contiguous")
    return t.data_ptr()


def _seqs(table, lens, starts, dev: int):
    t = _ints("table", table, dev, (None, None))
    seqs, width = table.shape
    return (t, table.stride(0) if seqs > 1 else width, width, _ints("lens", lens, dev, (seqs,)), _ints("starts", starts, dev, (seqs + 1,)), seqs)


def _rows(what: str, x, dev: int, rows, heads, dim: int, dtype=None):
    """(address, row distance, head distance) of [rows, heads, dim] with contiguous columns."""
    if (not isinstance(x, torch.Tensor) or x.dim() != 3 or x.dtype not in _DTYPES or (dtype is not None and x.dtype is not dtype) or x.get_device() != dev or x.shape[2] != dim
            or (rows is not None and x.shape[0] != rows) or (heads is not None and x.shape[1] != heads)):
        _refuse(f"{what}: [{'rows' if rows is None else rows}, {'heads' if heads is None else heads}, {dim}] of {dtype or 'f32, bf16 or f16'} on cuda:{dev} is wanted")
    ld, ldh, step = x.stride()
    if step != 1:
        _refuse(f"{what}: its columns are not contiguous")
    return x.data_ptr(), ld, ldh if x.shape[1] > 1 else dim


def append(k, v, cache, table, lens, starts):
    """Rows k and v [rows, kv_heads, dim] (f32, bf16 or f16; any row and head distance) into the pages of their sequences."""
    c, dev = _cache(cache)
    kp, ldk, ldkh = _rows("k", k, dev, None, c[4], c[6])
    vp, ldv, ldvh = _rows("v", v, dev, k.shape[0], c[4], c[6], k.dtype)
    t, ldt, width, l, s, seqs = _seqs(table, lens, starts, dev)
    rc = _entry("kv8_append")(dev, kp, ldk, ldkh, vp, ldv, ldvh, _DTYPES[k.dtype], *c, t, ldt, width, l, s, seqs, k.shape[0], _raw_stream(dev))
    if rc:
        _failed(rc)
    return cache


def attention(q, cache, table, lens, starts, *, scale: float = None, max_rows: int = 0, out=None):
    """q [rows, heads, dim] (f32, bf16 or f16) over the cache -> out of q's shape and type.  `scale`: None is dim ** -0.5.  `max_rows`: the most rows that any sequence brings, 0 if
    not known: decode rounds run faster when it is.  Rows of no sequence are left as they are (in a result that is made here: zeros)."""
    c, dev = _cache(cache)
    qp, ldq, ldqh = _rows("q", q, dev, None, None, c[6])
    rows, heads, dim = q.shape
    if heads == 0 or heads % max(c[4], 1):
        _refuse(f"q: {heads} heads over {c[4]} of the cache")
    t, ldt, width, l, s, seqs = _seqs(table, lens, starts, dev)
    if out is None:
        out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    op, ldo, ldoh = _rows("out", out, dev, rows, heads, dim, q.dtype)
    stream = _raw_stream(dev)
    need = C.c_size_t()
    rc = _entry("kv8_attention_bytes")(dev, _DTYPES[q.dtype], heads, c[4], dim, seqs, rows, max_rows, C.byref(need))
    if rc:
        _failed(rc)
    work = torch.empty(need.value, dtype=torch.uint8, device=q.device)
    rc = _entry("kv8_attention")(dev, qp, ldq, ldqh, op, ldo, ldoh, _DTYPES[q.dtype], heads, dim ** -0.5 if scale is None else scale, *c, t, ldt, width, l, s, seqs, rows, max_rows,
                                 work.data_ptr(), need.value, stream)
    if rc:
        _failed(rc)
    return out
