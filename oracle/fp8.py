"""CPU oracle of fp8 checkpoints -- TEST INFRASTRUCTURE ONLY: the dense decoder of oracle/qwen3.py with its projections from e4m3 codes.

Weights are codes times a scale for each 128 x 128 (`weight_scale_inv`), activation rows codes with a scale for each 128 columns:
a = max(max |y|, 2^-100), scale = a / 448, code = e4m3(y * (448 / a)).
"""
from __future__ import annotations

import numpy as np
import torch

from crane_b200 import synth
from .qwen3 import Qwen3Oracle


def quantise_rows(y: np.ndarray):
    """f32 rows [m, k], k a multiple of 128 -> (values of the codes [m, k], scales [m, k / 128])."""
    b = np.asarray(y, np.float32).reshape(y.shape[0], -1, 128)
    a = np.maximum(np.abs(b).max(2), np.float32(2.0 ** -100))
    t = b * (np.float32(448) / a)[:, :, None]
    return synth.e4m3_decode(synth.e4m3_encode(t)).reshape(y.shape), a / np.float32(448)


class Fp8Oracle(Qwen3Oracle):
    """`tensors`: those of synth.fp8_checkpoint.  `plain`: activations stay as they are, weights alone are rounded."""

    def __init__(self, cfg: dict, tensors: dict, plain: bool = False, **kw):
        self.f8, w, self.plain = {}, {}, plain
        for name, arr in tensors.items():
            if name.endswith(".weight_scale_inv"):
                continue
            scale = tensors.get(name + "_scale_inv")
            if scale is None:
                w[name] = arr
            else:
                full = synth.e4m3_decode(arr).astype(np.float64) * np.repeat(np.repeat(scale.astype(np.float64), 128, 0), 128, 1)
                self.f8[name] = torch.from_numpy(full)
        super().__init__(cfg, w, **kw)

    def _linear(self, full_name: str, x: torch.Tensor, w=None) -> torch.Tensor:
        if full_name not in self.f8:
            return super()._linear(full_name, x, w)
        rows = x.reshape(-1, x.shape[-1])
        if self.plain:
            y = rows.double()
        else:
            codes, scales = quantise_rows(rows.numpy())
            y = torch.from_numpy(codes.astype(np.float64) * np.repeat(scales.astype(np.float64), 128, 1))
        return (y @ self.f8[full_name].T).float().reshape(*x.shape[:-1], -1)
