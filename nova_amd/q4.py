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
from .chunks import launch, overlap
from .kvquant import _DT

GROUP = 32


@dataclass(frozen=True, eq=False)
class Q4Weight:
    """A weight ``[out_features, in_features]`` in 4 bits, as ``quantize_q4`` lays it out: ``data`` uint8 in blocks of 16 rows
    and 128 columns, each 1024 bytes of codes and 64 fp16 scales (``nkv_quantize_q4``)."""

    data: torch.Tensor
    shape: tuple[int, int]

    def __post_init__(self):
        d, (rows, n) = self.data, self.shape
        if rows < 0 or n <= 0 or n % GROUP:
            raise ValueError(f"shape {self.shape}: in_features must be a positive multiple of {GROUP}")
        size = -(-rows // 16) * -(-n // 128) * 1152
        if d.dtype != torch.uint8 or not d.is_cuda or not d.is_contiguous() or d.numel() != size or d.data_ptr() % 16:
            raise ValueError(f"data must be a contiguous, 16-byte aligned uint8 CUDA tensor of {size} elements")

    def nbytes(self) -> int:
        return self.data.numel()


def quantize_q4(w: torch.Tensor, out: Q4Weight | None = None) -> Q4Weight:
    """``w`` ``[out_features, in_features]`` (fp16 / bf16 / fp32, on the GPU; ``in_features`` a multiple of 32) in 4 bits.
    ``out``: a weight of the same shape to overwrite (captured graphs that read it go on)."""
    if w.dim() != 2 or w.dtype not in _DT or not w.is_cuda:
        raise ValueError(f"w must be a 2-d fp16 / bf16 / fp32 CUDA tensor, got {tuple(w.shape)} {w.dtype} on {w.device}")
    rows, n = w.shape
    if n == 0 or n % GROUP:
        raise ValueError(f"in_features {n} must be a positive multiple of {GROUP}")
    w = w.detach()
    w = w if w.is_contiguous() and w.data_ptr() % 16 == 0 else w.clone(memory_format=torch.contiguous_format)
    if out is None:
        out = Q4Weight(torch.empty(_lib.load().nkv_q4_weight_bytes(rows, n), dtype=torch.uint8, device=w.device), (rows, n))
    elif out.shape != (rows, n) or out.data.device != w.device or overlap(out.data, w):
        raise ValueError(f"out must be a Q4Weight of {(rows, n)} on {w.device} apart from w")
    launch(w.device, "nkv_quantize_q4", w.data_ptr(), _DT[w.dtype], rows, n, out.data.data_ptr())
    return out


def dequantize_q4(w: Q4Weight, dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """The values of ``w`` as ``[out_features, in_features]`` of ``dtype`` (exact in fp16 and fp32)."""
    if dtype not in _DT:
        raise ValueError(f"unsupported dtype {dtype}")
    out = torch.empty(w.shape, dtype=dtype, device=w.data.device)
    launch(out.device, "nkv_dequantize_q4", w.data.data_ptr(), *w.shape, out.data_ptr(), _DT[dtype])
    return out
