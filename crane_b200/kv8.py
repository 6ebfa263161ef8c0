"""A paged key/value cache in 8 bits on CUDA tensors: e4m3 codes with a scale for every page and head, and attention over it.

    cache = kv8.pages(4096, kv_heads=8, dim=128)                      # (k codes, v codes, scales); any page may be any sequence's
    kv8.append(k, v, cache, table, lens, starts)                      # the new rows of all sequences into their pages
    out = kv8.attention(q, cache, table, lens, starts)                # each new row over what its sequence holds, itself included

`table` [sequences, pages] int32 has the pages of each sequence (the rest: any number outside the cache; a row of its own for each: expanded and overlapping tables are refused), `lens` [sequences] int32 the positions it holds, new rows included, and
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
_sizes = {}                # bytes of workspaces by what they depend on


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
        shape, dev = k.shape, k.get_device()
        n, h, p, d = shape
        if (k.dtype is CODES and v.dtype is CODES and scales.dtype is _F32 and v.shape == shape and scales.shape == (n, h, 2) and dev >= 0 and dev == v.get_device() == scales.get_device()
                and k.is_contiguous() and v.is_contiguous() and scales.is_contiguous()):
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


# As in fp8.py: one look tells that all is in order; what it does not find goes through the checks one by one, which name what is wrong or find the rarer layouts good.
def _seqs(table, lens, starts, dev: int):
    try:
        seqs, width = table.shape
        ldt, step = table.stride()
        if (step == 1 and ldt >= width and table.dtype is _I32 and lens.dtype is _I32 and starts.dtype is _I32 and lens.shape == (seqs,) and starts.shape == (seqs + 1,)
                and lens.is_contiguous() and starts.is_contiguous() and dev == table.get_device() == lens.get_device() == starts.get_device()):
            return table.data_ptr(), ldt, width, lens.data_ptr(), starts.data_ptr(), seqs
    except (AttributeError, ValueError):
        pass
    t = _ints("table", table, dev, (None, None))
    seqs, width = table.shape
    return t, table.stride(0) if seqs > 1 else width, width, _ints("lens", lens, dev, (seqs,)), _ints("starts", starts, dev, (seqs + 1,)), seqs


def _rows(what: str, x, dev: int, rows, heads, dim: int, dtype=None):
    """(address, row distance, head distance, type) of [rows, heads, dim] with contiguous columns."""
    try:
        (r, h, d), (ld, ldh, step), t = x.shape, x.stride(), x.dtype
        code = _DTYPES.get(t)
        if step == 1 and d == dim and code is not None and (dtype is None or t is dtype) and x.get_device() == dev and (rows is None or r == rows) and (heads is None or h == heads):
            return x.data_ptr(), ld, ldh if h > 1 else dim, code
    except (AttributeError, ValueError):
        pass
    if isinstance(x, torch.Tensor) and x.dim() == 3 and x.stride(2) != 1 and x.shape[2] == dim:
        _refuse(f"{what}: its columns are not contiguous")
    _refuse(f"{what}: [{'rows' if rows is None else rows}, {'heads' if heads is None else heads}, {dim}] of {dtype or 'f32, bf16 or f16'} on cuda:{dev} is wanted")


def append(k, v, cache, table, lens, starts):
    """Rows k and v [rows, kv_heads, dim] (f32, bf16 or f16; rows and heads at any distance from dim on) into the pages of their sequences."""
    c, dev = _cache(cache)
    kp, ldk, ldkh, code = _rows("k", k, dev, None, c[4], c[6])
    rows = k.shape[0]
    vp, ldv, ldvh, _ = _rows("v", v, dev, rows, c[4], c[6], k.dtype)
    rc = _entry("kv8_append")(dev, kp, ldk, ldkh, vp, ldv, ldvh, code, *c, *_seqs(table, lens, starts, dev), rows, _raw_stream(dev))
    if rc:
        _failed(rc)
    return cache


def attention(q, cache, table, lens, starts, *, scale: float = None, max_rows: int = 0, out=None):
    """q [rows, heads, dim] (f32, bf16 or f16) over the cache -> out of q's shape and type.  `scale`: None is dim ** -0.5.  `max_rows`: the most rows that any sequence brings, 0 if
    not known: decode rounds run faster when it is (16-bit ones of 64 or 128 columns take half the launches, and a workspace that may be 39 MB smaller).  `out` may be q.  Rows of no sequence are left as they are (in a result that is made here: zeros)."""
    c, dev = _cache(cache)
    kv_heads, dim = c[4], c[6]
    qp, ldq, ldqh, code = _rows("q", q, dev, None, None, dim)
    rows, heads, _ = q.shape
    s = _seqs(table, lens, starts, dev)
    if out is None:
        out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    op, ldo, ldoh, _ = _rows("out", out, dev, rows, heads, dim, q.dtype)
    key = (dev, code, heads, kv_heads, dim, s[5], rows, max_rows)
    need = _sizes.get(key)
    if need is None:
        n = C.c_size_t()
        rc = _entry("kv8_attention_bytes")(*key, C.byref(n))
        if rc:
            _failed(rc)
        if len(_sizes) >= 4096:
            _sizes.clear()
        need = _sizes[key] = n.value
    work = torch.empty(need, dtype=torch.uint8, device=q.device)
    rc = _entry("kv8_attention")(dev, qp, ldq, ldqh, op, ldo, ldoh, code, heads, dim ** -0.5 if scale is None else scale, *c, *s, rows, max_rows, work.data_ptr(), need, _raw_stream(dev))
    if rc:
        _failed(rc)
    return out
