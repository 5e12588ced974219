"""Attention projections (kappa/qwen3/linear.py:11-25) as W8 linears.

Same signatures and layouts as kappa: ``q_w`` / ``k_w`` / ``v_w``
``[heads, model_dim, head_dim]``, ``o_w`` ``[heads, head_dim, model_dim]``.
Each projection is one ``kw8_linear`` call (the tensor-core GEMM for
prefill, the weight-streaming kernel for decode) on the weight viewed
K-major: ``[heads * head_dim, model_dim]`` for Q/K/V (the storage
``quantize_weight`` produces for ``in_axis=-2``) and ``[model_dim, heads *
head_dim]`` for O (the storage :func:`quantize_attn_out` produces).
kappa computes ``einsum(x, to_compute_dtype(w, x.dtype))``: a bf16 product
of bf16 dequantised weights; here the int8 values are widened exactly, the
products accumulate in fp32 and the scale is applied to the sum.

The projections also take 8-bit rows (``Q8Rows``, made by ``add_rms_norm_q8``)
in place of bf16 ones, and :func:`linear_q8` is that product for any W8
weight: int8 x int8 on the tensor core with exact int32 sums
(``kw8_linear_q8``).
"""

from __future__ import annotations

import torch

from kappa_b200 import _dense, _lib
from kappa_b200.qwen3.quant import KMajor, Q8Rows, Q8Weight, Weight, is_q8_weight, kmajor, quantize_weight

__all__ = ["project_q", "project_kv", "project_attn_out", "quantize_attn_out", "attn_out_kmajor",
           "linear_q8"]


def linear_q8(x: Q8Rows, w: Weight | KMajor, *, in_axis: int = -1,
              out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """8-bit rows ``[.., K]`` times a W8 weight ``[.., N, K]`` (``in_axis=-1``) or ``[.., K, N]`` (``-2``): ``[.., N]``.

    ``out[t, n] = (sum_k x.values[t, k] * w.values[n, k]) * x.scale[t] * w.scale[n]``; N counts the leading axes of a
    stacked weight too.  A weight that is K-major already (``attn_out_kmajor``'s, for the output projection on heads
    flattened to ``[.., n * h]``) is taken as it is.
    """
    if not isinstance(x, Q8Rows):
        raise TypeError("x: linear_q8 takes 8-bit rows (add_rms_norm_q8, rms_norm_q8)")
    if isinstance(w, KMajor):
        return _dense.linear_q8(x, w, out_dtype=out_dtype)
    if type(w) is Q8Weight and in_axis == -1:
        # A weight [N, K] as it is stored: no views to make (kmajor's take as long as the launch).
        q, s = w
        if (q.is_cuda and q.dtype is torch.int8 and q.dim() == 2 and q.is_contiguous() and s.is_contiguous()
                and s.get_device() == q.get_device()):
            N, K = q.shape
            n, dt = s.numel(), _dense._OUT_DT.get(s.dtype)
            if dt is not None and (n == 1 or n == N):
                weight = _lib.KW8Weight(q.data_ptr(), s.data_ptr(), dt, 1 if n > 1 else 0, _lib.LAYOUT_KMAJOR, 0)
                return _dense.linear_q8_rows(x, weight, q, N, K, out_dtype)
    return _dense.linear_q8(x, kmajor(w, in_axis, "w"), out_dtype=out_dtype)


def _project_heads(x: torch.Tensor | Q8Rows, w: Weight, name: str) -> torch.Tensor:
    """``einsum("btd,ndh->btnh", x, w)`` for a W8 ``w`` ``[n, d, h]``."""
    km = kmajor(w, -2, name)
    if len(km.shape) != 3:
        raise ValueError(f"{name} must be [heads, model_dim, head_dim], got {tuple(w.values.shape)}")
    n, h, d = (int(s) for s in km.shape)
    if isinstance(x, Q8Rows):
        return _dense.linear_q8(x, km).unflatten(-1, (n, h))
    _dense.check_x(x, d)
    b, t = int(x.shape[0]), int(x.shape[1])
    return _dense.linear(x.reshape(b * t, d), km).reshape(b, t, n, h)


def project_q(x: torch.Tensor | Q8Rows, q_w: Weight) -> torch.Tensor:
    """kappa/qwen3/linear.py:11-13: ``q_w`` ``[num_heads, model_dim, head_dim]``."""
    return _project_heads(x, q_w, "q_w")


def project_kv(x: torch.Tensor | Q8Rows, k_w: Weight, v_w: Weight) -> tuple[torch.Tensor, torch.Tensor]:
    """kappa/qwen3/linear.py:16-20: ``k_w``, ``v_w`` each ``[num_kv, model_dim, head_dim]``."""
    return _project_heads(x, k_w, "k_w"), _project_heads(x, v_w, "v_w")


def attn_out_kmajor(o_w: Weight) -> KMajor:
    """``o_w`` ``[n, h, d]`` as the K-major ``[d, n*h]`` weight of the output projection.

    A per-channel scale must hold one value per model-dim channel (the form
    :func:`quantize_attn_out` makes); values stored otherwise are copied.
    """
    if not is_q8_weight(o_w):
        raise TypeError("o_w: kappa_b200 implements the W8 path; quantize the weight first")
    v = o_w.values
    if v.dim() != 3:
        raise ValueError(f"o_w must be [heads, head_dim, model_dim], got {tuple(v.shape)}")
    n, h, d = (int(s) for s in v.shape)
    s = o_w.scale
    if s.numel() not in (1, d):
        raise ValueError(
            f"o_w: per-channel scales must be one per model-dim channel ({d}), got {s.numel()} "
            "(quantize the output projection with quantize_attn_out)"
        )
    flat = Q8Weight(values=v.reshape(n * h, d), scale=s.reshape(1, d) if s.numel() == d else s.reshape(()))
    return kmajor(flat, -2, "o_w")


def project_attn_out(encoded: torch.Tensor, o_w: Weight) -> torch.Tensor:
    """kappa/qwen3/linear.py:23-25: ``einsum("btnh,nhd->btd", encoded, o_w)``."""
    if isinstance(encoded, Q8Rows):
        raise TypeError("encoded: the output projection takes bf16 heads (8-bit rows: linear_q8 on attn_out_kmajor's weight)")
    km = attn_out_kmajor(o_w)
    d, nh = (int(s) for s in km.shape)
    if encoded.dim() != 4 or int(encoded.shape[2]) * int(encoded.shape[3]) != nh:
        raise ValueError(f"encoded {tuple(encoded.shape)} does not match o_w {tuple(o_w.values.shape)}")
    b, t = int(encoded.shape[0]), int(encoded.shape[1])
    x = encoded.reshape(b, t, nh)
    _dense.check_x(x, nh)
    return _dense.linear(x.reshape(b * t, nh), km).reshape(b, t, d)


def quantize_attn_out(o_w: torch.Tensor, *, scale_dtype: torch.dtype = torch.bfloat16,
                      per_channel: bool = False) -> Q8Weight:
    """``quantize_weight`` of an output projection ``[n, h, d]`` over its whole
    contraction ``(n, h)``: per tensor this is kappa's result; per channel
    it gives one scale per model-dim channel.  ``values`` keeps the ``[n, h,
    d]`` shape as a view of the K-major ``[d, n*h]`` storage."""
    if o_w.dim() != 3:
        raise ValueError(f"o_w must be [heads, head_dim, model_dim], got {tuple(o_w.shape)}")
    n, h, d = (int(s) for s in o_w.shape)
    q = quantize_weight(o_w.reshape(n * h, d), scale_dtype=scale_dtype, per_channel=per_channel, in_axis=-2)
    scale = q.scale.reshape(1, 1, d) if per_channel else q.scale
    return Q8Weight(values=q.values.reshape(n, h, d), scale=scale)
