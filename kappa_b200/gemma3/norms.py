"""RMSNorm with Gemma's ``(1 + scale)`` (kappa/gemma3/norms.py:8-13) on the B200 kernel."""

from __future__ import annotations

import torch

from kappa_b200 import _lib, _norm
from kappa_b200.qwen3.quant import Q8Rows


def rms_norm(x: torch.Tensor, scale: torch.Tensor, *, epsilon: float = 1e-6,
             out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x * rsqrt(mean(x^2) + eps) * (1 + scale)`` in fp32, rounded to bf16."""
    return _norm.rms_norm(x, scale, kind=_lib.NORM_GEMMA, epsilon=epsilon, out_dtype=out_dtype)


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, scale: torch.Tensor, *,
                 epsilon: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """``h = x + residual`` in bf16 and ``rms_norm(h, scale)``, in one pass: ``(h, y)``, both bf16."""
    return _norm.add_rms_norm(x, residual, scale, kind=_lib.NORM_GEMMA, epsilon=epsilon, quantize=False)


def add_rms_norm_q8(x: torch.Tensor, residual: torch.Tensor, scale: torch.Tensor, *,
                    epsilon: float = 1e-6) -> tuple[torch.Tensor, Q8Rows]:
    """``h = x + residual`` in bf16 and the fp32 norm of ``h`` as 8-bit rows (one scale per row, absmax / 127)."""
    return _norm.add_rms_norm(x, residual, scale, kind=_lib.NORM_GEMMA, epsilon=epsilon, quantize=True)


def rms_norm_q8(x: torch.Tensor, scale: torch.Tensor, *, epsilon: float = 1e-6) -> Q8Rows:
    """The fp32 norm of ``x`` as 8-bit rows; nothing to add first."""
    return _norm.add_rms_norm(x, None, scale, kind=_lib.NORM_GEMMA, epsilon=epsilon, quantize=True)[1]
