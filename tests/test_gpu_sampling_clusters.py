"""Sampling over clusters of every size, with settings of one per row.

Tokens are compared with the 64-bit evaluation of test_gpu_sampling.py (equal, by the argument made there: 16384 draws and
fewer, so a draw that two correct exps decide differently has a probability below 0.003), or with one another.
"""

from __future__ import annotations

import pytest
import torch

from kappa_b200 import _lib
from kappa_b200.qwen3.sampling import sample_tokens
from test_gpu_sampling import check, make

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    yield
    assert _lib.device_status(torch.zeros(1, device="cuda")) == 0, "a kernel reported a device-side error"


@pytest.mark.parametrize("B,V", [(1, 32768), (9, 32768), (18, 16384), (37, 8192), (74, 4096), (3, 32769)])
def test_short_slices_of_wide_clusters(B, V):
    """Two thousand logits a CTA: the CTAs of a cluster meet right after their start.  The maximum comes from any of them."""
    x, u = make(B, V, B + V)
    first = torch.empty(B, dtype=torch.int64, device="cuda")
    for i in range(16):
        at = (torch.arange(B, device="cuda") * 2053 + i * (V // 16) + 7) % V
        y = x.scatter(1, at[:, None], 50.0)
        first.copy_(at)
        for _ in range(20):
            greedy, _ = sample_tokens(y, u, temperature=0.0)
            likely, _ = sample_tokens(y, u, top_k=40)
            assert torch.equal(greedy.long(), first) and torch.equal(likely.long(), first)
    check(x, u)
    check(x, u, top_k=40, top_p=0.9)
