"""8-bit rows at the entry points around ``linear_q8``, bit for bit (the argument of test_gpu_linear_q8.py)."""

from __future__ import annotations

import pytest
import torch

from kappa_b200 import _lib
from kappa_b200.qwen3 import linear as qlin
from kappa_b200.qwen3.quant import Q8Rows
from test_gpu_linear_q8 import _ref, _rows

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
