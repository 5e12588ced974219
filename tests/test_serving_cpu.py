"""Host-side refusals of the serving entry points: they fail before any launch, so they need no GPU.

The pointers are never dereferenced on the host.
"""

from __future__ import annotations

import pytest

import kappa_b200._lib as L

P = 1 << 20  # a 16-byte aligned address that nothing reads


def _norm(x=P, residual=P + (1 << 16), T=4, D=64, scale=P + (1 << 17), dt=L.DT_F32, kind=L.NORM_QWEN, eps=1e-6,
          h=P + (1 << 18), y=None, q=P + (1 << 19), qs=P + (1 << 20)):
    return L.load().kw8_add_rms_norm(x, residual, T, D, scale, dt, kind, eps, h, y, q, qs, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(x=None), L.KW8_ERR_INVALID_ARG, "null"),
    (dict(scale=None), L.KW8_ERR_INVALID_ARG, "null"),
    (dict(D=60), L.KW8_ERR_UNSUPPORTED, "D %"),
    (dict(D=16392), L.KW8_ERR_UNSUPPORTED, "D %"),
    (dict(T=-1), L.KW8_ERR_UNSUPPORTED, "RMSNorm"),
    (dict(T=1 << 31), L.KW8_ERR_UNSUPPORTED, "too many"),
    (dict(dt=5), L.KW8_ERR_INVALID_ARG, "dtype"),
    (dict(kind=3), L.KW8_ERR_INVALID_ARG, "kind"),
    (dict(eps=-1.0), L.KW8_ERR_INVALID_ARG, "eps"),
    (dict(eps=float("nan")), L.KW8_ERR_INVALID_ARG, "eps"),
    (dict(q=None), L.KW8_ERR_INVALID_ARG, "either"),
    (dict(qs=None), L.KW8_ERR_INVALID_ARG, "either"),
    (dict(y=P + (1 << 21)), L.KW8_ERR_INVALID_ARG, "either"),
    (dict(q=None, qs=None), L.KW8_ERR_INVALID_ARG, "either"),
    (dict(x=P + 8), L.KW8_ERR_UNSUPPORTED, "aligned"),
    (dict(q=P + (1 << 19) + 4), L.KW8_ERR_UNSUPPORTED, "aligned"),
    (dict(h=P + 16), L.KW8_ERR_INVALID_ARG, "overlap"),
    (dict(q=P), L.KW8_ERR_INVALID_ARG, "overlap"),
    (dict(q=None, qs=None, y=P), L.KW8_ERR_INVALID_ARG, "overlap"),
    (dict(qs=P + (1 << 18)), L.KW8_ERR_INVALID_ARG, "overlap"),
    (dict(scale=P + (1 << 19)), L.KW8_ERR_INVALID_ARG, "overlap"),
])
def test_add_rms_norm_refuses(kw, code, text):
    assert _norm(**kw) == code
    assert text in L.last_error()


def test_add_rms_norm_of_no_rows_is_nothing():
    assert _norm(T=0, x=None, residual=None, scale=None, h=None, q=None, qs=None) == L.KW8_OK
