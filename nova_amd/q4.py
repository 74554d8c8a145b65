"""The 4-bit format of weights and cache: groups of 32 values of a row share a scale.

With ``amax`` a group's largest magnitude, ``s = max(amax / 7, 2^-24)`` rounded to 8 significant bits and
held in fp16, ``code = clamp(rint(x / s), -7, 7)`` and the value is ``code * s``, which fp16 holds exactly:
4.5 bits a value. ``quantize_q4`` makes a weight of it once; ``nova_amd.gemv.rms_gemv_q4`` and
``swiglu_gemv_q4`` multiply tokens with it; ``nova_amd.paged.PagedKVQ4Cache`` holds keys and values so.

The reference extracts 4-bit weights of another format (src/nova/quant.py:39-135, a table of 16 values per
64 weights) and multiplies one token with them (src/nova/kernels.py:243-289).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from .chunks import launch
from .kvquant import _DT

GROUP = 32


@dataclass(frozen=True)
class Q4Weight:
    """A weight ``[out_features, in_features]`` in 4 bits: ``codes`` uint8 ``[out, in / 2]`` (byte i of a row holds
    code + 8 of inputs 2 i, low half, and 2 i + 1), ``scales`` fp16 ``[out, in / 32]``."""

    codes: torch.Tensor
    scales: torch.Tensor

    def __post_init__(self):
        c, s = self.codes, self.scales
        if c.dim() != 2 or c.dtype != torch.uint8 or not c.is_cuda or not c.is_contiguous() or c.data_ptr() % 16 or c.shape[1] % 16:
            raise ValueError("codes must be a contiguous, 16-byte aligned uint8 CUDA tensor [out, in / 2], in a multiple of 32")
        if (s.dim() != 2 or s.shape != (c.shape[0], c.shape[1] // 16) or s.dtype != torch.float16 or s.device != c.device
                or not s.is_contiguous()):
            raise ValueError(f"scales must be a contiguous fp16 tensor [{c.shape[0]}, {c.shape[1] // 16}] on {c.device}")

    @property
    def shape(self) -> tuple[int, int]:
        return self.codes.shape[0], 2 * self.codes.shape[1]

    def nbytes(self) -> int:
        return self.codes.numel() + 2 * self.scales.numel()


def quantize_q4(w: torch.Tensor) -> Q4Weight:
    """``w`` ``[out_features, in_features]`` (fp16 / bf16 / fp32, on the GPU; ``in_features`` a multiple of 32) in 4 bits."""
    if w.dim() != 2 or w.dtype not in _DT or not w.is_cuda:
        raise ValueError(f"w must be a 2-d fp16 / bf16 / fp32 CUDA tensor, got {tuple(w.shape)} {w.dtype} on {w.device}")
    rows, n = w.shape
    if n == 0 or n % GROUP:
        raise ValueError(f"in_features {n} must be a positive multiple of {GROUP}")
    w = w.detach()
    w = w if w.is_contiguous() and w.data_ptr() % 16 == 0 else w.clone(memory_format=torch.contiguous_format)
    codes = torch.empty((rows, n // 2), dtype=torch.uint8, device=w.device)
    scales = torch.empty((rows, n // GROUP), dtype=torch.float16, device=w.device)
    launch(w.device, "nkv_quantize_q4", w.data_ptr(), _DT[w.dtype], rows, n, codes.data_ptr(), scales.data_ptr())
    return Q4Weight(codes, scales)


def dequantize_q4(w: Q4Weight, dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """The values of ``w`` as ``[out_features, in_features]`` of ``dtype`` (exact in fp16 and fp32)."""
    if dtype not in _DT:
        raise ValueError(f"unsupported dtype {dtype}")
    out = torch.empty(w.shape, dtype=dtype, device=w.codes.device)
    launch(out.device, "nkv_dequantize_q4", w.codes.data_ptr(), w.scales.data_ptr(), *w.shape, out.data_ptr(), _DT[dtype])
    return out
