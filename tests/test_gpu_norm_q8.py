"""The residual norm (``add_rms_norm``, ``add_rms_norm_q8``, ``rms_norm_q8``) against a 64-bit evaluation.

Tolerances.  ``h`` is one fp32 addition of two bf16 numbers and one rounding: bit exact.  The fp32 chain behind it
(at most 64 serial and 8 tree additions of squares, a divide, a reciprocal square root, two products) is off by less
than 80 * 2^-24 / 2 + 6 * 2^-24 < 2^-18 relative; a bf16 result adds half a step (2^-8), the scale two roundings
(still < 2^-17).  ``y / s`` is at most 127, so its error is below 127 * (2^-18 + 2^-17 + 2^-23) < 2^-8 steps, on top
of the half step that rounding to int8 may be off.
"""

from __future__ import annotations

import pytest
import torch

from kappa_b200 import _lib
from kappa_b200.gemma3 import norms as gemma
from kappa_b200.qwen3 import norms as qwen
from kappa_b200.qwen3.quant import Q8Rows, dequantize_rows

pytestmark = pytest.mark.gpu

FP32 = 2.0 ** -18
TINY = 1.1754943508222875e-38


@pytest.fixture(autouse=True)
def _status():
    yield
    assert _lib.device_status(torch.zeros(1, device="cuda")) == 0, "a kernel reported a device-side error"


def _inputs(T, D, seed, scale_dtype=torch.float32, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(T, D, generator=g, device="cuda") * std).to(torch.bfloat16)
    r = (torch.randn(T, D, generator=g, device="cuda") * 3 * std).to(torch.bfloat16)
    s = (torch.randn(D, generator=g, device="cuda") * 0.3 + 0.2).to(scale_dtype)
    return x, r, s


def _norm64(h, scale, is_gemma, eps=1e-6):
    h = h.double()
    g = scale.double() + (1.0 if is_gemma else 0.0)
    return h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * g


def _check_rows(q, y):
    """Q8Rows ``q`` against the 64-bit rows ``y``."""
    s = (y.abs().amax(-1, keepdim=True) / 127).clamp_min(TINY)
    assert q.values.dtype == torch.int8 and q.scale.dtype == torch.float32
    assert tuple(q.scale.shape) == tuple(q.values.shape[:-1]) + (1,)
    assert ((q.scale.double() - s).abs() <= 2 * FP32 * s).all()
    assert ((q.values.double() - y / s).abs() <= 0.5 + 2.0 ** -8).all()
    assert (q.values.int().abs() <= 127).all()
    if y.shape[0] and y.shape[-1]:
        big = y.abs().amax(-1) > 127 * TINY
        assert (q.values.int().abs().amax(-1)[big] == 127).all()


def _within_bf16(y, ref):
    assert ((y.double() - ref).abs() <= (2.0 ** -8 + FP32) * ref.abs() + 1e-38).all()


SHAPES = [(1, 8), (1, 2048), (2, 2560), (3, 264), (7, 5128), (33, 1032), (64, 2560), (5, 16384), (301, 128), (1200, 2048),
          (700, 8200)]


@pytest.mark.parametrize("T,D", SHAPES)
@pytest.mark.parametrize("fam", [gemma, qwen], ids=["gemma", "qwen"])
@pytest.mark.parametrize("sd", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_add_rms_norm(T, D, fam, sd):
    x, r, s = _inputs(T, D, 7 * T + D, sd)
    h_ref = (x.float() + r.float()).to(torch.bfloat16)
    y_ref = _norm64(h_ref, s, fam is gemma)
    h, y = fam.add_rms_norm(x, r, s)
    assert torch.equal(h, h_ref)
    _within_bf16(y, y_ref)
    h, q = fam.add_rms_norm_q8(x, r, s)
    assert torch.equal(h, h_ref)
    _check_rows(q, y_ref)
    _check_rows(fam.rms_norm_q8(x, s), _norm64(x, s, fam is gemma))


def test_same_bits_as_the_norm_of_the_stored_sum():
    """add_rms_norm is the addition followed by rms_norm, to the bf16 rounding of both."""
    x, r, s = _inputs(96, 2560, 5)
    h, y = gemma.add_rms_norm(x, r, s)
    assert ((y.double() - gemma.rms_norm(h, s).double()).abs() <= 2.0 ** -7 * y.double().abs()).all()


def test_leading_axes_strides_and_offsets():
    x, r, s = _inputs(2 * 3 * 5, 256, 11, torch.bfloat16)
    x3, r3 = x.reshape(2, 3, 5, 256), r.reshape(2, 3, 5, 256)
    h, q = qwen.add_rms_norm_q8(x3.transpose(0, 2), r3.transpose(0, 2), s)
    h_ref = (x3.float() + r3.float()).to(torch.bfloat16).transpose(0, 2)
    assert torch.equal(h, h_ref) and tuple(q.scale.shape) == (5, 3, 2, 1)
    _check_rows(q, _norm64(h_ref, s, False))
    # Rows and a scale that start off a 16-byte boundary.
    flat = torch.cat([x.reshape(-1)[:1], x.reshape(-1)])[1:].reshape(x.shape)
    sc = torch.cat([s[:1], s])[1:]
    assert flat.data_ptr() % 16 and sc.data_ptr() % 16
    _check_rows(qwen.rms_norm_q8(flat, sc), _norm64(x, s, False))
    h, y = qwen.add_rms_norm(flat, flat, sc)
    _within_bf16(y, _norm64((2 * x.float()).to(torch.bfloat16), s, False))


def test_zero_rows_tiny_rows_and_no_rows():
    x, r, s = _inputs(4, 512, 3)
    x[1], r[1] = 0, 0
    x[2], r[2] = 1e-30, 0
    h, q = qwen.add_rms_norm_q8(x, r, s, epsilon=1e-6)
    assert (q.values[1] == 0).all() and float(q.scale[1]) == pytest.approx(TINY)
    _check_rows(q, _norm64(h, s, False))
    # epsilon 0 on a zero row: 0 * inf is not a number, and the row says so.  Squares are taken in fp32, as kappa
    # takes them: (1e-30)^2 = 1e-60 is below 2^-150, half the least fp32 number, so row 2 sums to zero too and
    # 1e-30 * inf = inf.
    h, q = qwen.add_rms_norm_q8(x, r, s, epsilon=0.0)
    assert torch.isnan(q.scale[[1, 2]]).all() and (q.values[1] == 0).all() and (q.values[2] == 0).all()
    assert torch.isfinite(q.scale[[0, 3]]).all()
    for T in (0,):
        h, q = gemma.add_rms_norm_q8(x[:T], r[:T], s)
        assert tuple(h.shape) == (0, 512) and tuple(q.values.shape) == (0, 512) and tuple(q.scale.shape) == (0, 1)
        assert tuple(gemma.add_rms_norm(x[:T], r[:T], s)[1].shape) == (0, 512)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_rows_that_are_not_finite_stand_alone(bad):
    x, r, s = _inputs(5, 1000 // 8 * 8, 9)
    x[2, 17] = bad
    h, q = gemma.add_rms_norm_q8(x, r, s)
    assert torch.isnan(q.scale[2]).all() and (q.values[2] == 0).all()
    keep = [0, 1, 3, 4]
    _check_rows(type(q)(q.values[keep], q.scale[keep]), _norm64(h[keep], s, True))


def test_in_place_and_overlap_at_the_c_entry():
    x, r, s = _inputs(40, 2048, 21)
    h_ref = (x.float() + r.float()).to(torch.bfloat16)
    y_ref = _norm64(h_ref, s, False)
    lib = _lib.load()
    for which in ("x", "residual"):
        a, b = x.clone(), r.clone()
        h = a if which == "x" else b
        y = torch.empty_like(x)
        _lib.check(lib.kw8_add_rms_norm(a.data_ptr(), b.data_ptr(), 40, 2048, s.data_ptr(), _lib.DT_F32, _lib.NORM_QWEN,
                                        1e-6, h.data_ptr(), y.data_ptr(), None, None, _lib.stream_of(x)))
        assert torch.equal(h, h_ref)
        _within_bf16(y, y_ref)


def test_on_another_stream_and_in_a_graph():
    x, r, s = _inputs(48, 2560, 31)
    want = gemma.add_rms_norm_q8(x, r, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gemma.add_rms_norm_q8(x, r, s)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1].values, want[1].values)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = gemma.add_rms_norm_q8(x, r, s)
    x2, r2, _ = _inputs(48, 2560, 32)
    x.copy_(x2)
    r.copy_(r2)
    graph.replay()
    want = gemma.add_rms_norm_q8(x2, r2, s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1].values, want[1].values)
    assert torch.equal(got[1].scale, want[1].scale)


@pytest.mark.parametrize("T,D", [(1, 16), (3, 2560), (17, 33), (9, 1000), (0, 64), (4097, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_dequantize_rows(T, D, dtype):
    """One fp32 product and one rounding: bit exact."""
    g = torch.Generator(device="cuda").manual_seed(T + D)
    q = torch.randint(-128, 128, (T, D), generator=g, device="cuda").to(torch.int8)
    s = torch.rand(T, 1, generator=g, device="cuda") + 1e-3
    assert torch.equal(dequantize_rows(Q8Rows(q, s), dtype), (q.float() * s).to(dtype))
    flat = torch.cat([q.reshape(-1)[:1] if T else q.reshape(-1), q.reshape(-1)])[1 if T else 0:].reshape(T, D)
    assert torch.equal(dequantize_rows(Q8Rows(flat, s), dtype), (q.float() * s).to(dtype))
    with pytest.raises(ValueError, match="one scale per row"):
        dequantize_rows(Q8Rows(q, s.reshape(-1)[:, None, None]))
    with pytest.raises(ValueError, match="dtype"):
        dequantize_rows(Q8Rows(q, s), torch.float16)


def test_refusals():
    x, r, s = _inputs(4, 64, 1)
    with pytest.raises(ValueError, match="bfloat16"):
        qwen.add_rms_norm(x.float(), r, s)
    with pytest.raises(ValueError, match="residual"):
        qwen.add_rms_norm_q8(x, r[:3], s)
    with pytest.raises(ValueError, match="residual"):
        qwen.add_rms_norm_q8(x, r.float(), s)
    with pytest.raises(ValueError, match="features"):
        qwen.rms_norm_q8(x, s[:32])
    with pytest.raises(ValueError, match="CUDA"):
        qwen.rms_norm_q8(x.cpu(), s)
    with pytest.raises(ValueError, match="D %"):
        qwen.rms_norm_q8(x[:, :36], s[:36])
    with pytest.raises(ValueError, match="eps"):
        qwen.rms_norm_q8(x, s, epsilon=-1.0)
