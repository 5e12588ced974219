"""8-bit rows at the entry points around ``linear_q8``, bit for bit (the argument of test_gpu_linear_q8.py)."""

from __future__ import annotations

import pytest
import torch

from kappa_b200 import _lib
from kappa_b200.gemma3 import norms
from kappa_b200.qwen3 import linear as qlin
from kappa_b200.qwen3 import transformer as QT
from kappa_b200.qwen3.quant import Q8Rows, Q8Weight, kmajor, pack_weight
from test_gpu_linear_q8 import _ref, _rows, _weight
from test_gpu_norm_q8 import _norm64

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    yield
    assert _lib.device_status(torch.zeros(1, device="cuda")) == 0, "a kernel reported a device-side error"


@pytest.mark.parametrize("per_channel", [False, True], ids=["tensor", "channel"])
@pytest.mark.parametrize("B,T", [(1, 1), (2, 33), (3, 200)])
def test_the_output_projection_on_8_bit_rows(B, T, per_channel):
    """The way that project_attn_out's refusal names: linear_q8 on attn_out_kmajor's weight."""
    n, h, d = 4, 64, 520
    g = torch.Generator(device="cuda").manual_seed(B + T)
    o = qlin.quantize_attn_out(torch.randn(n, h, d, generator=g, device="cuda") * 0.05, per_channel=per_channel,
                               scale_dtype=torch.float32)
    x = _rows(B * T, n * h, T)
    x3 = Q8Rows(x.values.reshape(B, T, n * h), x.scale.reshape(B, T, 1))
    flat = type(o)(o.values.reshape(n * h, d).t(), o.scale.reshape(-1, 1) if per_channel else o.scale)
    for dtype in (torch.bfloat16, torch.float32):
        y = qlin.linear_q8(x3, qlin.attn_out_kmajor(o), out_dtype=dtype)
        assert torch.equal(y, _ref(x, flat, dtype).reshape(B, T, d))
    with pytest.raises(TypeError, match="attn_out_kmajor"):
        qlin.project_attn_out(x3, o)
    with pytest.raises(ValueError, match="features"):
        qlin.linear_q8(Q8Rows(x3.values[..., :-16], x3.scale), qlin.attn_out_kmajor(o))


@pytest.mark.parametrize("dtype", [None, torch.float32])
@pytest.mark.parametrize("B,L", [(1, 1), (3, 7), (40, 5)])
def test_last_positions_of_8_bit_rows(B, L, dtype):
    """Positions as JAX's gather takes them: negative ones count from the end, all are clamped."""
    D, V = 256, 1001
    x, w = _rows(B * L, D, L), _weight(V, D, 3)
    x3 = Q8Rows(x.values.reshape(B, L, D), x.scale.reshape(B, L, 1))
    last = torch.tensor([(3 * i) % (2 * L + 3) - L - 1 for i in range(B)], device="cuda")
    at = [min(max(int(i) + L if int(i) < 0 else int(i), 0), L - 1) for i in last]
    rows = torch.arange(B, device="cuda") * L + torch.tensor(at, device="cuda")
    want = _ref(Q8Rows(x.values[rows], x.scale[rows]), w, dtype or torch.bfloat16)
    assert torch.equal(QT.logits_from_hidden_last_positions(x3, w, last, out_dtype=dtype), want)
    strided = Q8Rows(x3.values.transpose(0, 1).contiguous().transpose(0, 1), x3.scale)
    assert torch.equal(QT.logits_from_hidden_last_positions(strided, w, last, out_dtype=dtype), want)


def test_last_positions_refuses():
    w = _weight(96, 64, 1)
    for x in (_rows(6, 64, 2), torch.zeros(6, 64, dtype=torch.bfloat16, device="cuda")):
        def shaped(*s, x=x):
            return Q8Rows(x.values.reshape(*s), x.scale.reshape(*s[:-1], 1)) if isinstance(x, Q8Rows) else x.reshape(*s)

        def empty(x=x):
            return Q8Rows(x.values[:0].reshape(2, 0, 64), x.scale[:0].reshape(2, 0, 1)) if isinstance(x, Q8Rows) \
                else x[:0].reshape(2, 0, 64)

        two = torch.zeros(2, dtype=torch.int64, device="cuda")
        with pytest.raises(ValueError, match="last_idx"):
            QT.logits_from_hidden_last_positions(shaped(3, 2, 64), w, two)
        with pytest.raises(ValueError, match="must be"):
            QT.logits_from_hidden_last_positions(shaped(6, 64), w, two)
        with pytest.raises(ValueError):
            QT.logits_from_hidden_last_positions(shaped(2, 3, 64), _weight(96, 32, 1), two)
        with pytest.raises(ValueError, match="no positions"):
            QT.logits_from_hidden_last_positions(empty(), w, two)


def test_a_packed_weight_brings_a_scale_that_fits():
    """Refused as a K-major weight's is, before anything reads it."""
    w = pack_weight(_weight(48, 64, 1), in_axis=-1)
    for scale, text in ((w.scale.cpu(), "devices"), (w.scale.half(), "dtype"), (w.scale[:-1], "expected 1 or 48"),
                        (torch.cat([w.scale, w.scale]), "expected 1 or 48"), (w.scale[:0], "expected 1 or 48")):
        with pytest.raises(ValueError, match=text):
            kmajor(w._replace(scale=scale), -1)
    x = _rows(3, 64, 2)
    with pytest.raises(ValueError, match="devices"):
        qlin.linear_q8(x, w._replace(scale=w.scale.cpu()))
    assert torch.equal(qlin.linear_q8(x, w), _ref(x, _weight(48, 64, 1), torch.bfloat16))


@pytest.mark.parametrize("N,K", [(32, 0), (0, 64), (0, 0)])
@pytest.mark.parametrize("T", [0, 4])
def test_weights_without_rows_or_features_are_refused(T, N, K):
    x = Q8Rows(torch.zeros(T, K, dtype=torch.int8, device="cuda"), torch.ones(T, 1, device="cuda"))
    w = Q8Weight(torch.zeros(N, K, dtype=torch.int8, device="cuda"), torch.ones((), device="cuda"))
    with pytest.raises(ValueError, match="bad shape"):
        qlin.linear_q8(x, w)


@pytest.mark.parametrize("loud", [0.0, 20.0, 100.0])
def test_what_8_bit_rows_cost_in_accuracy(loud):
    """The norm's rows in 8 bits, multiplied, against the product of the rows in 64 bits.

    A value of a row is off by at most half a step and what test_gpu_norm_q8.py derives (2^-8 steps, and 127 * 2^-17 for
    the scale): below 0.505 steps of max|y| / 127, whatever its own size.  So features that are far larger than the others
    cost the others their accuracy, and an output is off by at most 0.505 max|y| / 127 times the sum of its weights'
    sizes (and three fp32 roundings).  The bound is kept to; the rows of loud features do cost.
    """
    g = torch.Generator(device="cuda").manual_seed(1)
    T, D, N = 64, 1024, 512
    m = 1 + loud * (torch.rand(D, generator=g, device="cuda") < 0.004)
    x = (torch.randn(T, D, generator=g, device="cuda") * m).to(torch.bfloat16)
    r = (3 * torch.randn(T, D, generator=g, device="cuda") * m).to(torch.bfloat16)
    gain = 0.1 * torch.randn(D, generator=g, device="cuda")
    w = _weight(N, D, 5)
    h, q = norms.add_rms_norm_q8(x, r, gain)
    y = _norm64(h, gain, True)
    ws = w.values.double() * w.scale.double()
    want = y @ ws.t()
    step = y.abs().amax(-1, keepdim=True) / 127
    far = (qlin.linear_q8(q, w, out_dtype=torch.float32).double() - want).abs()
    assert (far <= 0.505 * step * ws.abs().sum(-1) + 2.0 ** -22 * want.abs()).all()
