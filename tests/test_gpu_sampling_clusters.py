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


def _per_row(B, V, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def pick(*v, dtype=torch.float32):
        return torch.tensor(v, device="cuda", dtype=dtype)[torch.randint(0, len(v), (B,), generator=g, device="cuda")]

    return dict(temperature=pick(0.0, 0.6, 1.0, 1.7), top_k=pick(0, 3, 300, 1500, V // 2, V - 1, 10 * V, dtype=torch.int64),
                top_p=pick(1.0, 0.95, 0.5), min_p=pick(0.0, 0.0, 1e-6, 0.05))


# Rows of two to eight CTAs, held in shared memory or read again (37 x 262144, 150 x 65521 and 600 x 100003 fp32: slices too
# large for two of them on an SM).
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,V", [(3, 40000), (64, 40000), (3, 151643), (64, 151643), (37, 262144), (7, 393216), (150, 65521),
                                 (600, 100003)])
def test_settings_of_one_per_row(B, V, dtype):
    """Among them cuts by top-k beyond what one CTA lists, alone and in front of a top-p cut."""
    for seed, std in ((1, 2.0), (2, 0.3), (3, 0.0)):
        x, u = make(B, V, seed, dtype, std)
        x[:, V - V // 50:] = float("-inf")
        kw = _per_row(B, V, seed)
        token, logprob = sample_tokens(x, u, **kw)
        rows = sorted({0, 1, 2, B // 2, B - 1})
        for k in (1500, V // 2):  # rows of every kind of cut, whatever the draw of the settings
            for p in (1.0, 0.95):
                at = ((kw["top_k"] == k) & (kw["top_p"] == torch.tensor(p)) & (kw["temperature"] > 0)).nonzero().reshape(-1)
                rows += [int(i) for i in at[:1]]
        for b in rows:
            check(x[b:b + 1], u[b:b + 1], (token[b:b + 1], logprob[b:b + 1]), **{n: v[b:b + 1] for n, v in kw.items()})


@pytest.mark.parametrize("V", [40000, 151643])
def test_a_top_k_per_row_is_the_top_k_as_a_number(V):
    """One kernel takes the settings of each row, another one setting for all: the same bits."""
    x, u = make(24, V, V)
    for kw in (dict(top_k=1500), dict(top_k=V // 2), dict(top_k=1500, top_p=0.9), dict(top_k=V // 2, top_p=0.9, min_p=1e-5),
               dict(top_k=40, min_p=0.1)):
        want = sample_tokens(x, u, temperature=1.3, **kw)
        rows = {n: torch.full((24,), v, device="cuda") for n, v in kw.items()}
        got = sample_tokens(x, u, temperature=torch.full((24,), 1.3, device="cuda"), **rows)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
