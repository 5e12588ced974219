"""Tokens from logits: temperature, top-k, top-p and min-p, from given random numbers.

kappa's sampling (kappa/gemma3/sampling.py) draws from a JAX key inside; here
the caller brings one uniform number per row, so a draw can be repeated and
checked.  One ``kw8_sample`` launch takes the logits of
``logits_from_hidden`` (bf16 or fp32) to token ids.
"""

from __future__ import annotations

import ctypes

import torch

from kappa_b200 import _lib

__all__ = ["sample_tokens"]

_DT = {torch.float32: _lib.DT_F32, torch.bfloat16: _lib.DT_BF16}


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _setting(v, name: str, lead: torch.Size, device: int, dtype: torch.dtype):
    """(the tensor of one value per row or None, the one value or 0)."""
    if not isinstance(v, torch.Tensor):
        if dtype == torch.int32:
            if int(v) != v:
                raise ValueError(f"{name} must be a whole number, got {v}")
            return None, max(-1, min(int(v), 2**31 - 1))
        if v != v:
            raise ValueError(f"{name} is NaN")
        return None, float(v)
    if v.shape != lead or v.get_device() != device:
        raise ValueError(f"{name}: one value per row wants shape {tuple(lead)} on cuda:{device}, got {tuple(v.shape)} "
                         f"on {v.device}")
    if v.is_floating_point() != (dtype == torch.float32) or v.dtype == torch.bool:
        raise ValueError(f"{name}: unsupported dtype {v.dtype}")
    if dtype == torch.int32 and v.dtype == torch.int64:
        v = v.clamp(-1, 2**31 - 1)
    return v.to(dtype).contiguous(), 0


def sample_tokens(
    logits: torch.Tensor,
    u: torch.Tensor,
    *,
    temperature: float | torch.Tensor = 1.0,
    top_k: int | torch.Tensor = 0,
    top_p: float | torch.Tensor = 1.0,
    min_p: float | torch.Tensor = 0.0,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``logits`` ``[.., V]`` (bf16 or fp32) and uniform ``u`` ``[..]`` fp32 -> token ids int32 and log-probabilities fp32 ``[..]``.

    Each setting is one number or a tensor of one per row.  A row's tokens are
    ordered by logit (ties: the lower id first); kept are the first ``top_k``
    (below 1: all), of these the shortest prefix with at least ``top_p`` of
    their probability, of these the ones at least ``min_p`` times as likely as
    the first.  The token is drawn from the kept ones in the order of their ids
    by ``u``, and the log-probability is its share of them.  ``temperature <=
    0`` takes the first token (greedy).  NaN logits are never drawn, ``+inf``
    counts as the largest finite number; a row without any logit above ``-inf`` gives token ``-1`` and ``-inf``.
    """
    _lib.require_cuda(logits, "logits")
    _lib.require_cuda(u, "u")
    if logits.dtype not in _DT:
        raise ValueError(f"logits must be bfloat16 or float32, got {logits.dtype}")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must be [.., V], got {tuple(logits.shape)}")
    if _lib.elsewhere(logits):
        with torch.cuda.device(logits.device):
            return sample_tokens(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    shape, dev = logits.shape, logits.get_device()
    lead, V = shape[:-1], shape[-1]
    if u.dtype != torch.float32 or u.shape != lead or u.get_device() != dev:
        raise ValueError(f"u must be float32 {tuple(lead)} on {logits.device}, got {u.dtype} {tuple(u.shape)} on {u.device}")
    t, t0 = _setting(temperature, "temperature", lead, dev, torch.float32)
    k, k0 = _setting(top_k, "top_k", lead, dev, torch.int32)
    p, p0 = _setting(top_p, "top_p", lead, dev, torch.float32)
    m, m0 = _setting(min_p, "min_p", lead, dev, torch.float32)
    # Rows may be strided (the last positions of [B, T, V]); the vocabulary may not.
    x = logits if len(shape) == 2 else logits.reshape(-1, V)
    if V > 1 and x.stride(-1) != 1:
        x = x.contiguous()
    B = x.shape[0]
    uc = u.contiguous()
    token = torch.empty_like(uc, dtype=torch.int32)
    logprob = torch.empty_like(uc)
    settings = _lib.KW8Sampling(_ptr(t), _ptr(k), _ptr(p), _ptr(m), t0, k0, p0, m0)
    code = _lib.load().kw8_sample(x.data_ptr(), _DT[x.dtype], B, V, x.stride(0) if B > 1 else V, uc.data_ptr(),
                                  ctypes.byref(settings), token.data_ptr(), logprob.data_ptr(), _lib.stream_of(x))
    if code:
        _lib.check(code)
    return token, logprob
