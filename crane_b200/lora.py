"""Low-rank adapters of many requests beside a shared projection, on CUDA tensors:

    y = fp8.linear(codes, code_scales, weight, weight_scales)         # every request's rows through the shared weight
    lora.linear(x, a, b, which, scales=alphas, add=y, out=y)          # each row's own adapter on top

Row i goes through adapter which[i]; numbers outside the adapters mean none.  Calls run on the tensors' device and its current stream, wait for nothing, keep nothing and may be
captured into graphs; `which` is read on the device only.
"""
from __future__ import annotations

import torch

from .fp8 import _DTYPES, _F32, _failed, _matrix, _raw_stream, _refuse, _rows_in
from .kv8 import _entry, _ints


def linear(x, a, b, which, *, scales=None, add=None, out=None):
    """out[i] = add[i] + scales[w] * (x[i] @ a[w].T) @ b[w].T, w = which[i].

    x [m, k] f32, bf16 or f16; a [adapters, rank, k] and b [adapters, n, rank], contiguous, of x's type or, beside f32 rows, any of the three; rank up to 128; which [m] int32;
    scales [adapters] f32 (None: ones); add [m, n] (None: zeros; may be out) and out of x's type.  An infinity of x or of an adapter becomes an infinity or a NaN of the results that it reaches."""
    dev, m, k, ldx, dtype = _rows_in("x", x)
    for what, w in (("a", a), ("b", b)):
        if not isinstance(w, torch.Tensor) or w.dim() != 3 or w.dtype not in _DTYPES or w.get_device() != dev or not w.is_contiguous():
            _refuse(f"{what}: a contiguous 3-D tensor of f32, bf16 or f16 on cuda:{dev} is wanted")
    adapters, rank, ka = a.shape
    n = b.shape[1]
    if ka != k or b.shape != (adapters, n, rank) or a.dtype is not b.dtype:
        _refuse(f"a {tuple(a.shape)} {a.dtype}, b {tuple(b.shape)} {b.dtype}: [adapters, rank, {k}] and [adapters, n, rank] of one type are wanted")
    wp = _ints("which", which, dev, (m,))
    if scales is not None and (not isinstance(scales, torch.Tensor) or scales.dtype is not _F32 or scales.shape != (adapters,) or scales.get_device() != dev
                               or (adapters > 1 and scales.stride(0) != 1)):
        _refuse(f"scales: {adapters} contiguous f32 values on cuda:{dev} are wanted")
    if out is None:
        out = torch.empty((m, n), dtype=x.dtype, device=x.device)
    ldo = _matrix("out", out, (x.dtype,), x.device, (m, n))
    ldadd = 0 if add is None else ldo if add is out else _matrix("add", add, (x.dtype,), x.device, (m, n))
    rc = _entry("lora_linear")(dev, x.data_ptr(), ldx, dtype, a.data_ptr(), b.data_ptr(), _DTYPES[a.dtype], adapters, rank, wp, None if scales is None else scales.data_ptr(),
                               None if add is None else add.data_ptr(), ldadd, out.data_ptr(), ldo, m, n, k, _raw_stream(dev))
    if rc:
        _failed(rc)
    return out
