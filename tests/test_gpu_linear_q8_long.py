"""A product that runs longer than the limit of a wait inside a kernel (2 s): the limit bounds what does not go on, not work.

Nothing here is rounded differently from test_gpu_linear_q8.py: sampled outputs are equal to the exact ones.
"""

from __future__ import annotations

import pytest
import torch

from kappa_b200 import _lib
from kappa_b200.qwen3 import linear as qlin
from kappa_b200.qwen3.quant import Q8Rows, Q8Weight

pytestmark = pytest.mark.gpu

LIMIT_MS = 2000.0


def test_a_launch_longer_than_the_wait_limit_reports_nothing():
    # 2 * 180224^2 * 131056 operations: 2.5 s at twice the bf16 rate.  The rows are the weight's (24 GB, and 65 GB of outputs).
    T = N = 180224
    K = 131056
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 100e9:
        pytest.skip("needs 100 GB of device memory")
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.empty(N, K, dtype=torch.int8, device="cuda")
    for i in range(0, N, 16384):
        q[i:i + 16384].random_(-127, 128, generator=g)
    xs = torch.rand(T, 1, generator=g, device="cuda") * 0.02 + 1e-3
    ws = torch.rand(N, 1, generator=g, device="cuda") * 0.02 + 1e-4
    assert _lib.device_status(q) == 0
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    y = qlin.linear_q8(Q8Rows(q, xs), Q8Weight(q, ws))
    end.record()
    torch.cuda.synchronize()
    status = _lib.device_status(q)
    rows = torch.randint(0, T, (61,), generator=g, device="cuda")
    cols = torch.randint(0, N, (67,), generator=g, device="cuda")
    rows[:2], cols[:2] = torch.tensor([0, T - 1]), torch.tensor([0, N - 1])
    got = y[rows][:, cols]
    del y
    acc = q[rows].double() @ q[cols].double().t()
    want = (acc.float() * xs[rows] * ws[cols].reshape(1, -1)).to(torch.bfloat16)
    del q
    torch.cuda.empty_cache()
    assert torch.equal(got, want)
    assert start.elapsed_time(end) > LIMIT_MS, "the product no longer runs longer than the limit"
    assert status == 0, "a wait that went on was reported as a timeout"
