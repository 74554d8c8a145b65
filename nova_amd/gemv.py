"""Batch-1 decode-step projections of the synthetic decoder, on the HIP kernels of
``libnova_kv.so`` (``nkv_gemv``, ``nkv_swiglu_gemv``, ``nkv_qk_norm_rope``).

They fuse what a decoder layer runs around the int8 KV path for one token: the RMSNorm
(src/nova/norm.py:35-41) into the projection that reads its output, the residual add into
the projection that produces it, SwiGLU (``LeanMLP``, src/nova/layers.py:173-174) into the
gate/up projection, and the q/k head norms plus RoPE into one launch. Each function takes
fp16 CUDA tensors and the caller's preallocated ``out`` (graph capture), and raises when
the library is missing: there is no torch fallback here.

``rms_gemv_q4`` and ``swiglu_gemv_q4`` are the same projections with 4-bit weights (``nova_amd.q4``), for any number of
tokens in fp16 or bf16.
"""

from __future__ import annotations

import functools

import torch

from . import _lib
from .chunks import launch
from .kvquant import _DT
from .q4 import Q4Weight


def _vec(t: torch.Tensor, name: str, n: int | None = None) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.float16 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous fp16 CUDA tensor")
    if n is not None and t.numel() != n:
        raise ValueError(f"{name} has {t.numel()} elements, expected {n}")


def rms_gemv(x: torch.Tensor, w: torch.Tensor, gamma: torch.Tensor | None = None, eps: float = 1e-6,
             residual: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``W @ rms_norm(x) (+ residual)`` for one token: ``x`` has ``in`` elements, ``w`` is
    ``[out, in]``; the result has ``out`` elements and the shape of ``residual`` (when given)
    or ``x.shape[:-1] + (out,)``. ``gamma=None`` skips the norm. ``out`` may be ``residual``."""
    if w.dim() != 2:
        raise ValueError("w must be [out_features, in_features]")
    n_out, n_in = w.shape
    _vec(x, "x", n_in)
    _vec(w, "w")
    if gamma is not None:
        _vec(gamma, "gamma", n_in)
    if residual is not None:
        _vec(residual, "residual", n_out)
    if out is None:
        out = torch.empty(residual.shape if residual is not None else (*x.shape[:-1], n_out), dtype=x.dtype,
                          device=x.device)
    _vec(out, "out", n_out)
    if out.data_ptr() == x.data_ptr():
        raise ValueError("out must not alias x")
    _lib.call("nkv_gemv", x.data_ptr(), _lib.ptr(gamma), float(eps), w.data_ptr(), n_out, n_in, _lib.ptr(residual),
              out.data_ptr(), _lib.stream_ptr(x.device))
    return out


def swiglu_gemv(x: torch.Tensor, w_gate_up: torch.Tensor, gamma: torch.Tensor | None = None, eps: float = 1e-6,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """``silu(G @ xn) * (U @ xn)`` for one token with ``w_gate_up = cat([G, U])`` of
    ``[2 * intermediate, in]`` and ``xn = rms_norm(x)`` (``gamma=None``: ``x``)."""
    if w_gate_up.dim() != 2 or w_gate_up.shape[0] % 2:
        raise ValueError("w_gate_up must be [2 * intermediate, in_features]")
    inter, n_in = w_gate_up.shape[0] // 2, w_gate_up.shape[1]
    _vec(x, "x", n_in)
    _vec(w_gate_up, "w_gate_up")
    if gamma is not None:
        _vec(gamma, "gamma", n_in)
    if out is None:
        out = torch.empty((*x.shape[:-1], inter), dtype=x.dtype, device=x.device)
    _vec(out, "out", inter)
    _lib.call("nkv_swiglu_gemv", x.data_ptr(), _lib.ptr(gamma), float(eps), w_gate_up.data_ptr(), inter, n_in,
              out.data_ptr(), _lib.stream_ptr(x.device))
    return out


def qk_norm_rope_(qkv: torch.Tensor, hq: int, hkv: int, q_gamma: torch.Tensor, k_gamma: torch.Tensor,
                  eps: float, inv_freq: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
    """In place on one token's ``qkv`` (``(hq + 2 hkv) * 128`` elements, q then k then v heads):
    per-head RMSNorm of q and k, then RoPE at the device position ``pos`` (int64, one element)
    with ``inv_freq`` (fp32, 64 elements). Returns ``qkv``."""
    d = 128
    _vec(qkv, "qkv", (hq + 2 * hkv) * d)
    _vec(q_gamma, "q_gamma", d)
    _vec(k_gamma, "k_gamma", d)
    if inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous() or inv_freq.numel() != d // 2:
        raise ValueError("inv_freq must be a contiguous fp32 tensor of 64 elements")
    if pos.dtype != torch.int64 or pos.numel() != 1:
        raise ValueError("pos must be a one-element int64 tensor")
    _lib.call("nkv_qk_norm_rope", qkv.data_ptr(), hq, hkv, d, q_gamma.data_ptr(), k_gamma.data_ptr(), float(eps),
              inv_freq.data_ptr(), pos.data_ptr(), _lib.stream_ptr(qkv.device))
    return qkv


# ---- 4-bit weights (``nova_amd.q4``), one token or a few


def _q4_args(x: torch.Tensor, w: Q4Weight, gamma: torch.Tensor | None, n_out: int, out: torch.Tensor | None,
             residual: torch.Tensor | None = None) -> tuple[int, torch.Tensor]:
    """The checked arguments of a product: the number of tokens and the output."""
    if not isinstance(w, Q4Weight):
        raise ValueError("w must be a Q4Weight (nova_amd.q4.quantize_q4)")
    n_in, dev, dtype, shape = w.shape[1], w.data.device, x.dtype, x.shape
    if dtype not in (torch.float16, torch.bfloat16) or not shape or shape[-1] != n_in or x.device != dev:
        raise ValueError(f"x must be fp16 / bf16 [.., {n_in}] on {dev}, got {tuple(shape)} {dtype} on {x.device}")
    if not x.is_contiguous() or x.data_ptr() % 16:
        raise ValueError("x must be contiguous and 16-byte aligned")
    if gamma is not None and (gamma.dtype != dtype or gamma.shape != (n_in,) or gamma.device != dev
                              or not gamma.is_contiguous() or gamma.data_ptr() % 16):
        raise ValueError(f"gamma must be a contiguous, 16-byte aligned {dtype} tensor of {n_in} elements on {dev}")
    shape = (*shape[:-1], n_out)
    if residual is not None and (residual.dtype != dtype or residual.shape != shape or residual.device != dev
                                 or not residual.is_contiguous()):
        raise ValueError(f"residual must be a contiguous {dtype} tensor {list(shape)} on {dev}")
    if out is None:
        out = x.new_empty(shape)
    else:
        if out.dtype != dtype or out.shape != shape or out.device != dev or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {dtype} tensor {list(shape)} on {dev}")
        first = out.data_ptr()
        end = first + out.nbytes
        for name, t in (("x", x), ("gamma", gamma), ("w", w.data), ("residual, unless it is the same", residual)):
            if t is not None and first < (at := t.data_ptr()) + t.nbytes and at < end and not (t is residual and at == first):
                raise ValueError(f"out must not overlap {name}")
    return x.numel() // n_in, out


@functools.lru_cache(maxsize=4096)  # (the sizes decide; 1 of a call's 7.5 us on the host)
def _q4_bytes(*sizes: int) -> int:
    return _lib.load().nkv_gemv_q4_workspace_bytes(*sizes)


def _q4_scratch(x: torch.Tensor, tokens: int, n_out: int, n_in: int, gamma: torch.Tensor | None,
                swiglu: bool) -> tuple[int | None, int]:
    """Memory of the call's own for the normalized input, where one launch does not make it itself."""
    n = _q4_bytes(_DT[x.dtype], tokens, n_out, n_in, gamma is not None, swiglu)
    return (_lib.scratch(x.device, n).data_ptr(), n) if n else (None, 0)


def rms_gemv_q4(x: torch.Tensor, w: Q4Weight, gamma: torch.Tensor | None = None, eps: float = 1e-6,
                residual: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``W @ rms_norm(x) (+ residual)`` for each token of ``x`` ``[.., in]`` (fp16 or bf16, contiguous) with a 4-bit
    weight; ``gamma=None`` skips the norm. Returns ``[.., out]`` of x's type; ``out`` may be ``residual``.

    The normalized input is rounded once, to 11 bits of bf16 inputs and 22 of fp16, as the matrix cores' operands; all
    else is fp32 with one rounding of the result. Made for one token to a few dozen (each 16 to 64 tokens read the weight again, from the
    caches where it fits them). The number of tokens chooses the kernel, and so the last bits."""
    tokens, out = _q4_args(x, w, gamma, w.shape[0], out, residual)
    launch(x.device, "nkv_gemv_q4", x.data_ptr(), _DT[x.dtype], tokens, _lib.ptr(gamma), float(eps), w.data.data_ptr(),
           *w.shape, _lib.ptr(residual), out.data_ptr(), *_q4_scratch(x, tokens, *w.shape, gamma, False))
    return out


def swiglu_gemv_q4(x: torch.Tensor, w_gate_up: Q4Weight, gamma: torch.Tensor | None = None, eps: float = 1e-6,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """``silu(G @ xn) * (U @ xn)`` for each token with the 4-bit ``w_gate_up = cat([G, U])`` of
    ``[2 * intermediate, in]`` and ``xn = rms_norm(x)`` (``gamma=None``: ``x``), as :func:`rms_gemv_q4`."""
    if not isinstance(w_gate_up, Q4Weight) or w_gate_up.shape[0] % 2:
        raise ValueError("w_gate_up must be a Q4Weight [2 * intermediate, in_features] (nova_amd.q4.quantize_q4)")
    inter = w_gate_up.shape[0] // 2
    tokens, out = _q4_args(x, w_gate_up, gamma, inter, out)
    launch(x.device, "nkv_swiglu_gemv_q4", x.data_ptr(), _DT[x.dtype], tokens, _lib.ptr(gamma), float(eps),
           w_gate_up.data.data_ptr(), inter, w_gate_up.shape[1], out.data_ptr(),
           *_q4_scratch(x, tokens, inter, w_gate_up.shape[1], gamma, True))
    return out
