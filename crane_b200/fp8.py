"""Linears in 8-bit floating point on CUDA tensors: rows to e4m3 codes with an f32 scale for every 128 columns, and codes x codes^T.

A model of an fp8 checkpoint (`quantization_config` {"quant_method": "fp8", "weight_block_size": [128, 128]}) runs its projections like this by itself
(`Qwen3Model`); these are the same kernels for programs that keep their tensors on the device:

    codes, scales = fp8.rms_norm(x, weight, eps, residual=stream, residual_out=stream)       # stream += x; rows of its norm
    gate_up = fp8.linear(codes, scales, w_gate_up, w_gate_up_scales)
    codes, scales = fp8.silu_mul(gate_up)
    stream = fp8.linear(codes, scales, w_down, w_down_scales, add=stream, out=stream)

Calls run on the tensors' device and its current stream, wait for nothing, keep nothing and may be captured into graphs.  Given `out` they allocate nothing.
As everywhere in this package there is no CPU path.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import BF16, F16, F32, INVALID_ARG, OK, CraneB200Error, load_library

BLOCK = 128
CODES = torch.float8_e4m3fn
_DTYPES = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
_fn = {}


def _call(name: str, *args):
    fn = _fn.get(name)
    if fn is None:
        fn = _fn[name] = getattr(load_library(), "crane_b200_fp8_" + name)
    rc = fn(*args)
    if rc != OK:
        raise CraneB200Error(rc, (load_library().crane_b200_fp8_last_error() or b"").decode("utf-8", "replace"))


def _refuse(msg: str):
    raise CraneB200Error(INVALID_ARG, msg)


def _matrix(what: str, t, dtypes, device, shape) -> int:
    """Checks a row-major matrix -> the distance of its rows in elements."""
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        _refuse(f"{what}: a tensor of {' / '.join(str(d) for d in dtypes)} is wanted")
    if t.dim() != 2 or t.shape != shape:
        _refuse(f"{what}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.device != device:
        _refuse(f"{what} is on {t.device}, expected {device}")
    ld, step = t.stride()
    if step != 1 and shape[1] > 1:
        _refuse(f"{what}: its columns are not contiguous")
    return ld if shape[0] > 1 else max(ld, shape[1])


def _row_scales(what: str, t, device, m: int, blocks: int) -> int:
    """Checks rows' scales [m, blocks], stored block by block -> the distance of two blocks."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32:
        _refuse(f"{what}: an f32 tensor is wanted")
    if t.dim() != 2 or t.shape != (m, blocks):
        _refuse(f"{what}: shape {tuple(t.shape)}, expected {(m, blocks)}")
    if t.device != device:
        _refuse(f"{what} is on {t.device}, expected {device}")
    step, ld = t.stride()
    if step != 1 and m > 1:
        _refuse(f"{what}: the scales of a block are not contiguous (a tensor like rows() gives is wanted)")
    return ld if blocks > 1 else max(ld, m)


def _codes_ld(t, k: int) -> int:
    """Row distance of codes in memory that starts rows on 16 bytes: one row says nothing by its own stride."""
    ld = t.stride(0) if t.shape[0] > 1 else (k + 15) // 16 * 16
    return ld


def rows(m: int, k: int, device="cuda"):
    """Uninitialised codes [m, k] and scales [m, ceil(k / 128)] as the calls below take them: rows of codes start on 16 bytes, a block's scales lie side by side."""
    codes = torch.empty((m, (k + 15) // 16 * 16), dtype=CODES, device=device)[:, :k]
    return codes, torch.empty(((k + BLOCK - 1) // BLOCK, (m + 3) // 4 * 4), dtype=torch.float32, device=device)[:, :m].t()


def _out(out, m: int, k: int, device):
    if out is None:
        out = rows(m, k, device)
    codes, scales = out
    _matrix("out[0]", codes, (CODES,), device, (m, k))
    lds = _row_scales("out[1]", scales, device, m, (k + BLOCK - 1) // BLOCK)
    return codes, scales, _codes_ld(codes, k), lds


def _input(what: str, x):
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dim() != 2:
        _refuse(f"{what}: a 2-D CUDA tensor is wanted")
    return x.device, x.shape[0], x.shape[1]


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def quantize(x, out=None):
    """Rows x [m, k] (f32, bf16 or f16) -> (codes, scales)."""
    dev, m, k = _input("x", x)
    ldx = _matrix("x", x, _DTYPES, dev, (m, k))
    codes, scales, ld, lds = _out(out, m, k, dev)
    _call("quantize", dev.index, x.data_ptr(), _DTYPES[x.dtype], ldx, m, k, codes.data_ptr(), ld, scales.data_ptr(), lds, _stream(dev))
    return codes, scales


def silu_mul(gate_up, out=None):
    """Rows [gate | up] of 2 k columns -> (codes, scales) of SiLU(gate) * up."""
    dev, m, k = _input("gate_up", gate_up)
    if k % 2:
        _refuse(f"gate_up: {k} columns are not gates and as many ups")
    k //= 2
    ldx = _matrix("gate_up", gate_up, _DTYPES, dev, (m, 2 * k))
    codes, scales, ld, lds = _out(out, m, k, dev)
    _call("silu_mul", dev.index, gate_up.data_ptr(), _DTYPES[gate_up.dtype], ldx, m, k, codes.data_ptr(), ld, scales.data_ptr(), lds, _stream(dev))
    return codes, scales


def rms_norm(x, weight, eps: float = 1e-6, *, residual=None, residual_out=None, out=None):
    """(codes, scales) of the RMS norm of h = x, or of h = x + residual, which is stored to `residual_out` (None: in place of `residual`) in the residual's type and
    normalised as stored.  `weight` [k] f32, bf16 or f16."""
    dev, m, k = _input("x", x)
    ldx = _matrix("x", x, _DTYPES, dev, (m, k))
    if not isinstance(weight, torch.Tensor) or weight.dtype not in _DTYPES or weight.shape != (k,) or weight.device != dev or (k > 1 and weight.stride(0) != 1):
        _refuse(f"weight: {k} contiguous f32, bf16 or f16 values on {dev} are wanted")
    res = res_out = None
    rtype = ldr = 0
    if residual is not None:
        if residual_out is None:
            residual_out = residual
        ldr, rtype = _matrix("residual", residual, _DTYPES, dev, (m, k)), _DTYPES[residual.dtype]
        if _matrix("residual_out", residual_out, (residual.dtype,), dev, (m, k)) != ldr:
            _refuse("residual_out: its rows lie as far apart as the residual's")
        res, res_out = residual.data_ptr(), residual_out.data_ptr()
    elif residual_out is not None:
        _refuse("residual_out without a residual")
    codes, scales, ld, lds = _out(out, m, k, dev)
    _call("rms_norm", dev.index, x.data_ptr(), _DTYPES[x.dtype], ldx, res, res_out, rtype, ldr, weight.data_ptr(), _DTYPES[weight.dtype], eps, m, k, codes.data_ptr(), ld,
          scales.data_ptr(), lds, _stream(dev))
    return codes, scales


def linear(x, x_scales, weight, weight_scales, *, add=None, out=None, dtype=torch.bfloat16):
    """x [m, k] codes x weight [n, k] codes transposed, each with its scales (weight_scales [ceil(n / 128), ceil(k / 128)] f32), + add -> [m, n] of `out`'s or
    `dtype`'s type (f32, bf16, f16).  Sums are f32, rounded once.  `add` has the result's type and may be `out`."""
    dev, m, k = _input("x", x)
    _matrix("x", x, (CODES,), dev, (m, k))
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        _refuse("weight: a 2-D tensor is wanted")
    n, blocks = weight.shape[0], (k + BLOCK - 1) // BLOCK
    _matrix("weight", weight, (CODES,), dev, (n, k))
    lds = _row_scales("x_scales", x_scales, dev, m, blocks)
    ldws = _matrix("weight_scales", weight_scales, (torch.float32,), dev, ((n + BLOCK - 1) // BLOCK, blocks))
    if out is None:
        out = torch.empty((m, n), dtype=dtype, device=dev)
    ldo = _matrix("out", out, _DTYPES, dev, (m, n))
    ldadd = 0 if add is None else _matrix("add", add, (out.dtype,), dev, (m, n))
    _call("linear", dev.index, x.data_ptr(), _codes_ld(x, k), x_scales.data_ptr(), lds, weight.data_ptr(), _codes_ld(weight, k), weight_scales.data_ptr(), ldws, m, n, k,
          None if add is None else add.data_ptr(), ldadd, out.data_ptr(), _DTYPES[out.dtype], ldo, _stream(dev))
    return out


def status(device=None):
    """Waits for the current stream of `device`; raises when its work failed, or when a linear gave up a wait on the GPU."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    _call("status", dev.index if dev.index is not None else torch.cuda.current_device(), _stream(dev))
