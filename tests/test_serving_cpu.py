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
    (dict(scale=P + (1 << 17) + 8), L.KW8_ERR_UNSUPPORTED, "aligned"),
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


def _linear(q=P, qs=P + (1 << 16), T=4, K=64, N=32, w=None, dt=L.DT_BF16, out=P + (1 << 18)):
    w = w or L.KW8Weight(P + (1 << 17), P + (1 << 19), L.DT_F32, 1, L.LAYOUT_KMAJOR, 0)
    return L.load().kw8_linear_q8(q, qs, T, K, N, w, dt, out, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(q=None), L.KW8_ERR_INVALID_ARG, "null"),
    (dict(qs=None), L.KW8_ERR_INVALID_ARG, "null"),
    (dict(out=None), L.KW8_ERR_INVALID_ARG, "null"),
    (dict(T=-1), L.KW8_ERR_INVALID_ARG, "bad shape"),
    (dict(K=0), L.KW8_ERR_INVALID_ARG, "bad shape"),
    (dict(N=0), L.KW8_ERR_INVALID_ARG, "bad shape"),
    (dict(K=72), L.KW8_ERR_UNSUPPORTED, "multiple of 16"),
    (dict(K=131072), L.KW8_ERR_UNSUPPORTED, "131056"),
    (dict(T=1 << 31), L.KW8_ERR_UNSUPPORTED, "range"),
    (dict(N=1 << 31), L.KW8_ERR_UNSUPPORTED, "range"),
    (dict(dt=4), L.KW8_ERR_INVALID_ARG, "out dtype"),
    (dict(q=P + 8), L.KW8_ERR_UNSUPPORTED, "aligned"),
    (dict(out=P + (1 << 18) + 1), L.KW8_ERR_UNSUPPORTED, "aligned"),
    (dict(out=P + (1 << 18) + 2, dt=L.DT_F32), L.KW8_ERR_UNSUPPORTED, "aligned"),
    (dict(out=P), L.KW8_ERR_INVALID_ARG, "overlap"),
    (dict(out=P + (1 << 17) + 64), L.KW8_ERR_INVALID_ARG, "overlap"),
    (dict(out=P + (1 << 16)), L.KW8_ERR_INVALID_ARG, "overlap"),
    (dict(out=P + (1 << 19)), L.KW8_ERR_INVALID_ARG, "overlap"),
    (dict(w=L.KW8Weight(None, P, L.DT_F32, 1, 0, 0)), L.KW8_ERR_INVALID_ARG, "null"),
    (dict(w=L.KW8Weight(P, P, 9, 1, 0, 0)), L.KW8_ERR_INVALID_ARG, "scale dtype"),
    (dict(w=L.KW8Weight(P, P, L.DT_F32, 1, 7, 0)), L.KW8_ERR_INVALID_ARG, "layout"),
    (dict(w=L.KW8Weight(P + 4, P, L.DT_F32, 1, 0, 0)), L.KW8_ERR_UNSUPPORTED, "aligned"),
])
def test_linear_q8_refuses(kw, code, text):
    assert _linear(**kw) == code
    assert text in L.last_error()


def test_linear_q8_of_no_rows_is_nothing():
    assert _linear(T=0, q=None, qs=None, out=None) == L.KW8_OK


def _sample(logits=P, dt=L.DT_F32, B=4, V=100, ld=100, u=P + (1 << 16), s=0, token=P + (1 << 17), logprob=P + (1 << 18),
            **kw):
    import ctypes

    s = L.KW8Sampling(None, None, None, None, kw.get("temperature", 1.0), 0, kw.get("top_p", 1.0), kw.get("min_p", 0.0)) \
        if s == 0 else s
    if s is not None and "temperatures" in kw:
        s.temperatures = kw["temperatures"]
    return L.load().kw8_sample(logits, dt, B, V, ld, u, None if s is None else ctypes.byref(s), token, logprob, None)


NAN = float("nan")


@pytest.mark.parametrize("kw,code,text", [
    (dict(logits=None), L.KW8_ERR_INVALID_ARG, "null"),
    (dict(u=None), L.KW8_ERR_INVALID_ARG, "null"),
    (dict(token=None), L.KW8_ERR_INVALID_ARG, "null"),
    (dict(s=None), L.KW8_ERR_INVALID_ARG, "settings"),
    (dict(dt=2), L.KW8_ERR_INVALID_ARG, "f32 or bf16"),
    (dict(V=0), L.KW8_ERR_INVALID_ARG, "bad shape"),
    (dict(B=-1), L.KW8_ERR_INVALID_ARG, "bad shape"),
    (dict(V=393217, ld=393217), L.KW8_ERR_UNSUPPORTED, "393216"),
    (dict(B=1 << 28), L.KW8_ERR_UNSUPPORTED, "too many"),
    (dict(ld=-1), L.KW8_ERR_INVALID_ARG, "stride"),
    (dict(ld=1 << 41), L.KW8_ERR_INVALID_ARG, "stride"),
    (dict(temperature=NAN), L.KW8_ERR_INVALID_ARG, "temperature"),
    (dict(top_p=NAN), L.KW8_ERR_INVALID_ARG, "top_p"),
    (dict(min_p=NAN), L.KW8_ERR_INVALID_ARG, "min_p"),
    (dict(logits=P + 2), L.KW8_ERR_UNSUPPORTED, "aligned"),
    (dict(logits=P + 1, dt=L.DT_BF16), L.KW8_ERR_UNSUPPORTED, "aligned"),
    (dict(token=P + 2), L.KW8_ERR_UNSUPPORTED, "aligned"),
    (dict(temperatures=P + 1), L.KW8_ERR_UNSUPPORTED, "aligned"),
    (dict(token=P + 1596), L.KW8_ERR_INVALID_ARG, "overlap"),
    (dict(logprob=P + (1 << 17) + 12), L.KW8_ERR_INVALID_ARG, "overlap"),
    (dict(logprob=P + (1 << 16)), L.KW8_ERR_INVALID_ARG, "overlap"),
])
def test_sample_refuses(kw, code, text):
    assert _sample(**kw) == code
    assert text in L.last_error()


def test_sample_of_no_rows_is_nothing():
    assert _sample(B=0, logits=None, u=None, token=None) == L.KW8_OK


def _dequant(q=P, s=P + (1 << 16), T=4, D=64, dt=L.DT_BF16, out=P + (1 << 18)):
    return L.load().kw8_dequantize_rows(q, s, T, D, dt, out, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(q=None), L.KW8_ERR_INVALID_ARG, "null"),
    (dict(s=None), L.KW8_ERR_INVALID_ARG, "null"),
    (dict(out=None), L.KW8_ERR_INVALID_ARG, "null"),
    (dict(T=-1), L.KW8_ERR_INVALID_ARG, "bad shape"),
    (dict(T=1 << 31), L.KW8_ERR_UNSUPPORTED, "range"),
    (dict(dt=3), L.KW8_ERR_INVALID_ARG, "dtype"),
    (dict(out=P + (1 << 18) + 1), L.KW8_ERR_UNSUPPORTED, "misaligned"),
    (dict(out=P + 128), L.KW8_ERR_INVALID_ARG, "overlap"),
])
def test_dequantize_rows_refuses(kw, code, text):
    assert _dequant(**kw) == code
    assert text in L.last_error()


def test_dequantize_rows_of_nothing():
    assert _dequant(T=0, q=None, s=None, out=None) == L.KW8_OK
    assert _dequant(D=0, q=None, s=None, out=None) == L.KW8_OK
