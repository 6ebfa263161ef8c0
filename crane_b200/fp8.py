"""Linears in 8-bit floating point on CUDA tensors: rows to e4m3 codes with an f32 scale for every 128 columns, and codes x codes^T.

A model of an fp8 checkpoint (`quantization_config` {"quant_method": "fp8", "weight_block_size": [128, 128]}) runs its projections like this by itself
(`Qwen3Model`); these are the same kernels for programs that keep their tensors on the device:

    codes, scales = fp8.rms_norm(x, weight, eps, residual=stream, residual_out=stream)       # stream += x; rows of its norm
    gate_up = fp8.linear(codes, scales, w_gate_up, w_gate_up_scales)
    codes, scales = fp8.silu_mul(gate_up)
    stream = fp8.linear(codes, scales, w_down, w_down_scales, add=stream, out=stream)

Calls run on the tensors' device and its current stream, wait for nothing, keep nothing and may be captured into graphs (`status` waits, and tells of a linear that gave up a wait).  Given `out` they allocate nothing.
As everywhere in this package there is no CPU path.
"""
from __future__ import annotations

import torch

from . import BF16, F16, F32, INVALID_ARG, CraneB200Error, load_library

BLOCK = 128
CODES = torch.float8_e4m3fn
_F32 = torch.float32
_DTYPES = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_fn = {}


def _entry(name: str):
    fn = _fn.get(name)
    if fn is None:
        fn = _fn[name] = getattr(load_library(), "crane_b200_fp8_" + name)
    return fn


def _failed(rc: int):
    raise CraneB200Error(rc, (load_library().crane_b200_fp8_last_error() or b"").decode("utf-8", "replace"))


def _refuse(msg: str):
    raise CraneB200Error(INVALID_ARG, msg)


def _matrix(what: str, t, dtypes, device, shape) -> int:
    """Checks a row-major matrix -> the distance of its rows in elements."""
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        _refuse(f"{what}: a tensor of {' / '.join(str(d) for d in dtypes)} is wanted")
    if t.shape != shape:
        _refuse(f"{what}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.device != device:
        _refuse(f"{what} is on {t.device}, expected {device}")
    ld, step = t.stride()
    if step != 1 and shape[1] > 1:
        _refuse(f"{what}: its columns are not contiguous")
    return ld if shape[0] > 1 else max(ld, shape[1])       # (one row's own distance says nothing)


def _row_scales(what: str, t, device, m: int, k: int) -> int:
    """Checks the scales of m rows of k columns, stored block by block -> the distance of two blocks."""
    blocks = (k + BLOCK - 1) // BLOCK
    if not isinstance(t, torch.Tensor) or t.dtype != _F32:
        _refuse(f"{what}: an f32 tensor is wanted")
    if t.shape != (m, blocks):
        _refuse(f"{what}: shape {tuple(t.shape)}, expected {(m, blocks)}")
    if t.device != device:
        _refuse(f"{what} is on {t.device}, expected {device}")
    step, ld = t.stride()
    if step != 1 and m > 1:
        _refuse(f"{what}: the scales of a block are not contiguous (a tensor like rows() gives is wanted)")
    return ld if blocks > 1 else max(ld, m)


def _codes(what: str, t, device, shape) -> int:
    ld = _matrix(what, t, (CODES,), device, shape)
    return ld if shape[0] > 1 else (shape[1] + 15) // 16 * 16


def _input(what: str, x):
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dim() != 2:
        _refuse(f"{what}: a 2-D CUDA tensor is wanted")
    return x.device, x.shape[0], x.shape[1]


def rows(m: int, k: int, device="cuda"):
    """Uninitialised codes [m, k] and scales [m, ceil(k / 128)] as the calls below take them: rows of codes start on 16 bytes, a block's scales lie side by side."""
    codes = torch.empty((m, (k + 15) // 16 * 16), dtype=CODES, device=device)[:, :k]
    return codes, torch.empty(((k + BLOCK - 1) // BLOCK, (m + 3) // 4 * 4), dtype=_F32, device=device)[:, :m].t()


# A small kernel takes no longer than the checks around it.  So the calls look their tensors over in as few attribute reads as tell that all is in order; whatever that does not
# find goes through the checks above, one by one, which name what is wrong or find the rarer layouts good.  (Distances of rows and alignment are checked by the library.)
def _out(out, m: int, k: int, dev: int):
    """(codes, scales, ld, lds) of a result."""
    if out is None:
        out = rows(m, k, dev)
    codes, scales = out
    try:
        (ld, step), (sstep, lds) = codes.stride(), scales.stride()
        if (step == 1 and sstep == 1 and codes.dtype is CODES and scales.dtype is _F32 and codes.shape == (m, k) and scales.shape == (m, (k + 127) // 128)
                and codes.get_device() == dev and scales.get_device() == dev and ld >= k and not ld & 15 and lds >= m):
            return codes, scales, ld, lds
    except (AttributeError, ValueError):
        pass
    device = torch.device("cuda", dev)
    return codes, scales, _codes("out[0]", codes, device, (m, k)), _row_scales("out[1]", scales, device, m, k)


def _rows_in(what: str, x):
    """(device index, rows, columns, row distance, type) of an input."""
    try:
        (m, k), (ld, step), dtype, dev = x.shape, x.stride(), _DTYPES.get(x.dtype), x.get_device()
        if step == 1 and dtype is not None and dev >= 0 and ld >= k:
            return dev, m, k, ld, dtype
    except (AttributeError, ValueError):
        pass
    device, m, k = _input(what, x)
    return device.index, m, k, _matrix(what, x, _DTYPES, device, (m, k)), _DTYPES[x.dtype]


def quantize(x, out=None):
    """Rows x [m, k] (f32, bf16 or f16) -> (codes, scales)."""
    dev, m, k, ldx, dtype = _rows_in("x", x)
    codes, scales, ld, lds = _out(out, m, k, dev)
    rc = _entry("quantize")(dev, x.data_ptr(), dtype, ldx, m, k, codes.data_ptr(), ld, scales.data_ptr(), lds, _raw_stream(dev))
    if rc:
        _failed(rc)
    return codes, scales


def silu_mul(gate_up, out=None):
    """Rows [gate | up] of 2 k columns -> (codes, scales) of SiLU(gate) * up."""
    dev, m, k, ldx, dtype = _rows_in("gate_up", gate_up)
    if k % 2:
        _refuse(f"gate_up: {k} columns are not gates and as many ups")
    k //= 2
    codes, scales, ld, lds = _out(out, m, k, dev)
    rc = _entry("silu_mul")(dev, gate_up.data_ptr(), dtype, ldx, m, k, codes.data_ptr(), ld, scales.data_ptr(), lds, _raw_stream(dev))
    if rc:
        _failed(rc)
    return codes, scales


def rms_norm(x, weight, eps: float = 1e-6, *, residual=None, residual_out=None, out=None):
    """(codes, scales) of the RMS norm of h = x, or of h = x + residual, which is stored to `residual_out` (None: in place of `residual`) in the residual's type and
    normalised as stored.  `weight` [k] f32, bf16 or f16."""
    dev, m, k, ldx, dtype = _rows_in("x", x)
    wtype = _DTYPES.get(weight.dtype) if isinstance(weight, torch.Tensor) else None
    if wtype is None or weight.shape != (k,) or weight.get_device() != dev or (k > 1 and weight.stride(0) != 1):
        _refuse(f"weight: {k} contiguous f32, bf16 or f16 values on cuda:{dev} are wanted")
    res = res_out = None
    rtype = ldr = 0
    if residual is not None:
        rdev, rm, rk, ldr, rtype = _rows_in("residual", residual)
        if (rdev, rm, rk) != (dev, m, k):
            _refuse(f"residual: shape {(rm, rk)} on cuda:{rdev}, expected {(m, k)} on cuda:{dev}")
        res = res_out = residual.data_ptr()
        if residual_out is not None and residual_out is not residual:
            if (not isinstance(residual_out, torch.Tensor) or residual_out.dtype is not residual.dtype or residual_out.get_device() != dev or residual_out.shape != residual.shape
                    or (m > 1 and residual_out.stride() != residual.stride()) or (k > 1 and residual_out.stride(1) != 1)):
                _refuse("residual_out: a tensor of the residual's type, device, shape and strides is wanted")
            res_out = residual_out.data_ptr()
    elif residual_out is not None:
        _refuse("residual_out without a residual")
    codes, scales, ld, lds = _out(out, m, k, dev)
    rc = _entry("rms_norm")(dev, x.data_ptr(), dtype, ldx, res, res_out, rtype, ldr, weight.data_ptr(), wtype, eps, m, k, codes.data_ptr(), ld,
                            scales.data_ptr(), lds, _raw_stream(dev))
    if rc:
        _failed(rc)
    return codes, scales


def linear(x, x_scales, weight, weight_scales, *, add=None, out=None, dtype=torch.bfloat16):
    """x [m, k] codes x weight [n, k] codes transposed, each with its scales (weight_scales [ceil(n / 128), ceil(k / 128)] f32), + add -> [m, n] of `out`'s or
    `dtype`'s type (f32, bf16, f16).  Sums are f32, rounded once.  `add` has the result's type and may be `out`."""
    if out is None:
        try:
            out = torch.empty((x.shape[0], weight.shape[0]), dtype=dtype, device=x.device)
        except (AttributeError, IndexError, TypeError):
            _refuse("x and weight: 2-D tensors are wanted")
    try:
        (m, k), (n, kw) = x.shape, weight.shape
        (ldx, a), (ldw, b), (c, lds), (ldws, d), (ldo, e) = x.stride(), weight.stride(), x_scales.stride(), weight_scales.stride(), out.stride()
        dev, blocks = x.get_device(), (k + 127) // 128
        good = (a == b == c == d == e == 1 and kw == k and x_scales.shape == (m, blocks) and weight_scales.shape == ((n + 127) // 128, blocks) and out.shape == (m, n)
                and x.dtype is CODES and weight.dtype is CODES and x_scales.dtype is _F32 and weight_scales.dtype is _F32 and out.dtype in _DTYPES
                and dev >= 0 and dev == weight.get_device() == x_scales.get_device() == weight_scales.get_device() == out.get_device()
                and ldx >= k and ldw >= k and not (ldx | ldw) & 15 and lds >= m and ldws >= blocks and ldo >= n)
    except (AttributeError, ValueError):
        good = False
    if not good:
        device, m, k = _input("x", x)
        if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
            _refuse("weight: a 2-D tensor is wanted")
        dev, n = device.index, weight.shape[0]
        ldx, ldw = _codes("x", x, device, (m, k)), _codes("weight", weight, device, (n, k))
        lds = _row_scales("x_scales", x_scales, device, m, k)
        ldws = _matrix("weight_scales", weight_scales, (_F32,), device, ((n + BLOCK - 1) // BLOCK, (k + BLOCK - 1) // BLOCK))
        ldo = _matrix("out", out, _DTYPES, device, (m, n))
    ldadd = 0 if add is None else ldo if add is out else _matrix("add", add, (out.dtype,), x.device, (m, n))
    rc = _entry("linear")(dev, x.data_ptr(), ldx, x_scales.data_ptr(), lds, weight.data_ptr(), ldw, weight_scales.data_ptr(), ldws, m, n, k,
                          None if add is None else add.data_ptr(), ldadd, out.data_ptr(), _DTYPES[out.dtype], ldo, _raw_stream(dev))
    if rc:
        _failed(rc)
    return out


def status(device=None):
    """Waits for the current stream of `device`; raises when its work failed, or when a linear on the device, captured or not, gave up a wait on the GPU since
    the last call for that stream (whichever stream it ran on: each is told once)."""
    index = None if device is None else torch.device(device).index
    dev = torch.cuda.current_device() if index is None else index
    rc = _entry("status")(dev, _raw_stream(dev))
    if rc:
        _failed(rc)
