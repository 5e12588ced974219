"""``kw8_linear`` over SM pairs (``OPT_TC_PAIR``) on a product that runs longer than the limit of a wait inside a kernel (2 s).

Rows of -1, 0 and 1: every partial sum is a whole number below 98304 * 128 < 2^24, so fp32 sums in any order are exact and
the outputs are equal to the exact ones, rounded once.
"""

from __future__ import annotations

import pytest
import torch

from kappa_b200 import _dense, _lib
from kappa_b200.qwen3.quant import Q8Weight, kmajor

pytestmark = pytest.mark.gpu

LIMIT_MS = 2000.0


def test_a_pair_launch_longer_than_the_wait_limit_reports_nothing():
    T = N = 114688
    K = 98304
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 110e9:
        pytest.skip("needs 110 GB of device memory")
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.empty(T, K, dtype=torch.bfloat16, device="cuda")
    q = torch.empty(N, K, dtype=torch.int8, device="cuda")
    for i in range(0, T, 16384):
        x[i:i + 16384].random_(-1, 2, generator=g)
        q[i:i + 16384].random_(-127, 128, generator=g)
    w = kmajor(Q8Weight(q, torch.ones((), device="cuda")), -1)
    assert _lib.device_status(q) == 0
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    _lib.set_option(_lib.OPT_TC_PAIR, 2)
    try:
        start.record()
        y = _dense.linear(x, w)
        end.record()
    finally:
        _lib.set_option(_lib.OPT_TC_PAIR, 0)
    torch.cuda.synchronize()
    status = _lib.device_status(q)
    rows = torch.randint(0, T, (61,), generator=g, device="cuda")
    cols = torch.randint(0, N, (67,), generator=g, device="cuda")
    rows[:2], cols[:2] = torch.tensor([0, T - 1]), torch.tensor([0, N - 1])
    got = y[rows][:, cols]
    want = (x[rows].double() @ q[cols].double().t()).to(torch.bfloat16)
    del x, q, w, y
    torch.cuda.empty_cache()
    assert torch.equal(got, want)
    assert start.elapsed_time(end) > LIMIT_MS, "the product no longer runs longer than the limit"
    assert status == 0, "a wait that went on was reported as a timeout"
