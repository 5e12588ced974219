"""Sampling against a 64-bit evaluation of its definition on the host.

Tokens are whole numbers and must be equal.  The weights are floor(2^44 exp(.)) on both sides; where the two exps round
differently a weight moves by one unit of 2^-44, so a token could only differ where u * sum falls within about V units
of a border: less than 2^18 * V / 2^44 of the draws, 0.003 over every draw made here.  The log-probability is a 64-bit
quotient and logarithm rounded once to fp32: half a step (2^-24) relative, and 1e-9 absolute where it is near 0.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from kappa_b200 import _lib
from kappa_b200.gemma3 import sampling as gemma_sampling
from kappa_b200.qwen3.sampling import sample_tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    yield
    assert _lib.device_status(torch.zeros(1, device="cuda")) == 0, "a kernel reported a device-side error"


def reference_row(x, u, T, k, p, m):
    """(token, logprob, number of tokens kept) of one row; x in float64."""
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return -1, -math.inf, 0
    order = np.lexsort((np.arange(len(x)), -x))
    if not T > 0 or not p > 0 or not m <= 1:
        return int(order[0]), 0.0, 1
    if 0 < k < len(x):
        order = order[:k]
    if top == np.inf:
        w = np.where(x[order] == np.inf, 1 << 44, 0)
    else:
        with np.errstate(over="ignore", invalid="ignore", under="ignore"):
            e = np.where(x[order] == -np.inf, 0.0, np.exp((x[order] - top) / T))
        w = np.floor(e * 2.0**44).astype(np.int64)
    run = np.cumsum(w)
    n = len(order)
    if p < 1:
        n = 1 + int(np.count_nonzero((run[:-1].astype(np.float64) < p * float(run[-1]))))
    n = min(n, max(1, int(np.count_nonzero(w.astype(np.float64) >= m * 2.0**44))))
    ids = np.sort(order[:n])
    weight = np.zeros(len(x), np.int64)
    weight[order[:n]] = w[:n]
    cum = np.cumsum(weight[ids])
    total = int(cum[-1])
    goal = min(int(min(max(u, 0.0), 1.0) * float(total)), total - 1)
    j = int(np.searchsorted(cum, goal, side="right"))
    return int(ids[j]), math.log(float(weight[ids[j]]) / float(total)), n


def check(logits, u, got=None, **kw):
    token, logprob = got or sample_tokens(logits, u, **kw)
    assert token.dtype == torch.int32 and logprob.dtype == torch.float32
    assert token.shape == logits.shape[:-1] == logprob.shape
    x = logits.double().cpu().numpy().reshape(-1, logits.shape[-1])
    B = x.shape[0]

    def per_row(name, default):
        v = kw.get(name, default)
        v = v.cpu().numpy().reshape(-1) if isinstance(v, torch.Tensor) else np.full(B, v)
        return v.astype(np.int64) if name == "top_k" else v.astype(np.float32).astype(np.float64)

    T, k, p, m = per_row("temperature", 1.0), per_row("top_k", 0), per_row("top_p", 1.0), per_row("min_p", 0.0)
    uu = u.double().cpu().numpy().reshape(-1)
    tk, lp = token.cpu().numpy().reshape(-1), logprob.cpu().numpy().reshape(-1)
    kept = []
    for b in range(B):
        t, l, n = reference_row(x[b], uu[b], T[b], k[b], p[b], m[b])
        assert tk[b] == t, f"row {b}: token {tk[b]}, expected {t}"
        assert lp[b] == l or abs(lp[b] - l) <= 2.0**-24 * abs(l) + 1e-9, (b, lp[b], l)
        kept.append(n)
    return kept


def make(B, V, seed, dtype=torch.float32, std=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, V, generator=g, device="cuda") * std
    x.scatter_add_(1, torch.randint(0, V, (B, 8), generator=g, device="cuda"), 6 * torch.rand(B, 8, generator=g, device="cuda"))
    return x.to(dtype), torch.rand(B, generator=g, device="cuda")


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7), dict(top_k=1), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.1),
            dict(temperature=0.8, top_k=50, top_p=0.95), dict(temperature=1.3, top_k=400, top_p=0.7, min_p=0.02),
            dict(top_p=0.999), dict(top_k=1000000, top_p=1.5, min_p=-1.0), dict(temperature=4.0, top_p=0.5),
            dict(top_p=1e-6), dict(top_p=-1.0), dict(min_p=2.0), dict(temperature=-3.0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (2, 3), (5, 31), (2, 513), (4, 1000), (3, 2049), (2, 32000), (2, 151643)])
def test_settings(B, V, dtype):
    for i, kw in enumerate(SETTINGS):
        x, u = make(B, V, 100 * V + i, dtype)
        check(x, u, **kw)


@pytest.mark.parametrize("B", [1, 8, 37, 75, 149, 300, 700])
def test_batches(B):
    """Every split of a row over CTAs, with settings of one per row."""
    for V, dtype in ((5003, torch.float32), (6000, torch.bfloat16)):
        x, u = make(B, V, B + V, dtype)
        g = torch.Generator(device="cuda").manual_seed(B)
        pick = lambda *v: torch.tensor(v, device="cuda")[torch.randint(0, len(v), (B,), generator=g, device="cuda")]  # noqa: E731
        check(x, u, temperature=pick(0.0, 0.5, 1.0, 2.0), top_k=pick(0, 1, 7, 300, 9999, -5), top_p=pick(1.0, 0.9, 0.3),
              min_p=pick(0.0, 0.01, 0.3))


@pytest.mark.parametrize("V", [262144, 393216])
def test_large_vocabularies(V):
    for dtype in (torch.float32, torch.bfloat16):
        x, u = make(2, V, V, dtype)
        for kw in (dict(), dict(top_k=50, top_p=0.95), dict(temperature=0.9, top_p=0.8)):
            check(x, u, **kw)


@pytest.mark.parametrize("B", [10, 18, 19, 40])
def test_batches_of_the_largest_vocabulary(B):
    """Whatever the batch leaves of the CTAs, the slices of a row fit."""
    x, u = make(B, 393216, B)
    for kw in (dict(), dict(top_k=20, top_p=0.9), dict(temperature=torch.full((B,), 0.7, device="cuda"), top_p=0.9)):
        token, logprob = sample_tokens(x, u, **kw)
        kw = {name: v[:1] if isinstance(v, torch.Tensor) else v for name, v in kw.items()}
        for b in (0, B - 1):
            check(x[b:b + 1], u[b:b + 1], (token[b:b + 1], logprob[b:b + 1]), **kw)


@pytest.mark.parametrize("V", [1, 7, 1025, 40000])
def test_ties(V):
    """All logits equal, two values only, and bf16 steps: the lower ids stay."""
    u = torch.tensor([0.0, 0.25, 0.5, 0.999999, 1.0], device="cuda")
    x = torch.full((5, V), -1.5, device="cuda")
    for kw in (dict(), dict(top_k=max(1, V // 3)), dict(top_p=0.5), dict(top_k=max(1, V // 2), top_p=0.3), dict(min_p=1.0)):
        check(x, u, **kw)
        check(x.bfloat16(), u, **kw)
        two = x.clone()
        two[:, ::3] = 0.25
        check(two, u, **kw)
        check((torch.arange(V, device="cuda") % 5).float().expand(5, V) * 0.5, u, **kw)


def test_zeros_of_either_sign_tie():
    x = torch.tensor([[-0.0, 0.0, -0.0, 0.0, -1.0]], device="cuda")
    for uu in (0.0, 0.3, 0.6, 0.99):
        u = torch.tensor([uu], device="cuda")
        for kw in (dict(top_k=1), dict(top_k=2), dict(top_k=3), dict(temperature=0.0), dict(top_p=0.4)):
            check(x, u, **kw)


def test_masked_rows():
    """-inf, NaN and +inf logits, rows with one token left, rows with none."""
    V = 5000
    x, u = make(10, V, 7)
    x[0, :] = -math.inf
    x[1, :] = math.nan
    x[2, :] = -math.inf
    x[2, 4321] = -2.0
    x[3, ::2] = math.nan
    x[4, 17] = math.inf
    x[5, [5, 900, 4000]] = math.inf
    x[6, 100:] = -math.inf
    x[7, :] = torch.finfo(torch.float32).min
    x[8, :-1] = torch.finfo(torch.float32).min
    x[9, :2500] = math.nan
    x[9, 2500:] = -math.inf
    for kw in (dict(), dict(temperature=0.0), dict(top_k=3), dict(top_k=200, top_p=0.9), dict(top_p=0.9), dict(min_p=0.1)):
        check(x, u, **kw)
        check(x.bfloat16(), u, **kw)
    token, logprob = sample_tokens(x, u)
    assert token[[0, 1, 9]].tolist() == [-1, -1, -1] and (logprob[[0, 1, 9]] == -math.inf).all()


def test_values_over_the_whole_range():
    """Huge, tiny and subnormal logits and temperatures."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(6, 3000, generator=g, device="cuda") * 10.0 ** torch.randint(-44, 38, (6, 3000), generator=g, device="cuda")
    x[1] *= 1e-30
    x[2] = x[2].clamp(-1e-38, 1e-38)
    u = torch.rand(6, generator=g, device="cuda")
    for T in (1e-42, 1e-30, 1.0, 1e30, math.inf):
        for kw in (dict(), dict(top_k=10), dict(top_p=0.8), dict(top_k=100, top_p=0.5)):
            check(x, u, temperature=T, **kw)


@pytest.mark.parametrize("offset,T", [(1e6, 1.0), (-1e6, 0.1), (3e7, 4.0), (1e5, 1e-3), (1e4, 30.0)])
def test_logits_whose_steps_are_wider_than_a_bin(offset, T):
    """Far from zero a step of the format spans several histogram bins, or a bin many tokens."""
    for V in (3000, 40000):
        g = torch.Generator(device="cuda").manual_seed(int(abs(offset)) + V)
        x = torch.randn(3, V, generator=g, device="cuda") * 4 * T + offset
        u = torch.rand(3, generator=g, device="cuda")
        for kw in (dict(), dict(top_k=5), dict(top_k=700), dict(top_p=0.5), dict(top_p=0.97), dict(min_p=0.05),
                   dict(top_p=0.9, min_p=0.3), dict(top_k=1500, top_p=0.8)):
            check(x, u, temperature=T, **kw)


@pytest.mark.parametrize("top_p", [0.01, 0.3, 0.7, 0.9, 0.99, 0.999999])
@pytest.mark.parametrize("std", [0.0, 0.02, 0.5, 2.0, 8.0])
def test_nuclei_of_every_width(top_p, std):
    """From one token to nearly all: lists, windows of the histogram, and cuts among equal logits."""
    for V, dtype in ((1500, torch.float32), (60000, torch.float32), (60000, torch.bfloat16)):
        g = torch.Generator(device="cuda").manual_seed(int(100 * std) + V)
        x = (torch.randn(3, V, generator=g, device="cuda") * std).to(dtype)
        u = torch.rand(3, generator=g, device="cuda")
        check(x, u, top_p=top_p)
        check(x, u, top_p=top_p, min_p=0.2)
        check(x, u, top_p=top_p, top_k=V // 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("min_p", [0.0, 1e-7], ids=["top_p", "min_p"])
def test_wide_nuclei_of_many_rows(dtype, min_p):
    """Rows that are read again from global memory, at rows of every alignment; sampled rows are compared."""
    B, V = 64, 151643
    for std, top_p in ((2.0, 0.9), (3.0, 0.98), (1.0, 0.5), (2.0, 0.9999)):
        x, u = make(B, V, int(10 * std), dtype, std)
        x[:, V - 999:] = -math.inf
        token, logprob = sample_tokens(x, u, top_p=top_p, min_p=min_p)
        for b in (0, 1, 2, 3, 31, 63):
            check(x[b:b + 1], u[b:b + 1], (token[b:b + 1], logprob[b:b + 1]), top_p=top_p, min_p=min_p)


@pytest.mark.parametrize("ties", [2, 300, 5000, 100000])
def test_nucleus_that_ends_inside_ties(ties):
    """The cut falls into equal logits: a few of them, more than a list holds, and more than a CTA holds."""
    V = 151643
    for seed, (top_p, std) in enumerate(((0.3, 1.0), (0.6, 1.0), (0.85, 0.2))):
        x, u = make(2, V, seed, std=std)
        at = torch.randperm(V, generator=torch.Generator().manual_seed(seed))[:ties].cuda()
        for b in range(2):
            order = x[b].double().sort(descending=True).values
            mass = (order - order[0]).exp().cumsum(0)
            x[b, at] = order[int((mass < top_p * mass[-1]).sum())].float()
        check(x, u, top_p=top_p)
        check(x.to(torch.bfloat16), u, top_p=top_p)


@pytest.mark.parametrize("temperature", [1e-30, 1e-32, 1e-36])
def test_temperatures_near_the_smallest_number(temperature):
    """Steps between the logits of the same order as the temperature."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x = -30.0 * torch.rand(3, 5003, generator=g, device="cuda", dtype=torch.float64) * temperature
    u = torch.rand(3, generator=g, device="cuda")
    for kw in (dict(), dict(top_p=0.9), dict(top_p=0.9999), dict(top_k=2000), dict(top_k=3000, top_p=0.8)):
        check(x.float(), u, temperature=temperature, **kw)


@pytest.mark.parametrize("temperature", [9e35, 2e36, 1e37, 2e37, 3e38])
def test_temperatures_near_the_largest_number(temperature):
    g = torch.Generator(device="cuda").manual_seed(6)
    x = 3e38 * (2 * torch.rand(3, 5003, generator=g, device="cuda") - 1)
    u = torch.rand(3, generator=g, device="cuda")
    for kw in (dict(), dict(top_p=0.9), dict(top_p=0.9999), dict(top_k=2000), dict(top_k=3000, top_p=0.8), dict(top_p=0.7, min_p=0.01)):
        check(x, u, temperature=temperature, **kw)
        check(x.to(torch.bfloat16), u, temperature=temperature, **kw)


def test_settings_that_are_not_numbers_take_the_first_token():
    x, u = make(4, 3000, 5)
    nan, one = torch.full((4,), math.nan, device="cuda"), torch.ones(4, device="cuda")
    first = x.argmax(-1).int()
    for kw in (dict(temperature=nan), dict(top_p=nan), dict(min_p=nan)):
        token, logprob = sample_tokens(x, u, **kw)
        assert torch.equal(token, first) and (logprob == 0).all()
    assert torch.equal(sample_tokens(x, nan, top_k=40)[0], sample_tokens(x, 0 * one, top_k=40)[0])
    assert torch.equal(sample_tokens(x, -one)[0], sample_tokens(x, 0 * one)[0])
    assert torch.equal(sample_tokens(x, 7 * one)[0], sample_tokens(x, one)[0])


def test_shapes_and_strides():
    x, u = make(12, 1003, 9)
    want = sample_tokens(x, u, top_k=20)
    kw = dict(top_k=20)
    x3, u3 = x.reshape(3, 4, 1003), u.reshape(3, 4)
    check(x3, u3, **kw)
    check(x3[:, -1], u3[:, -1], **kw)  # rows 4 * V apart
    check(x3[:, 1, 1:], u3[:, 1], **kw)  # rows that start at an odd address
    check(x.t().contiguous().t(), u, **kw)
    check(x[0], u[0], **kw)
    check(x[:1].expand(12, 1003), u, **kw)
    check(x3.transpose(0, 1), u3.transpose(0, 1), **kw)
    t = sample_tokens(x[:0], u[:0])
    assert t[0].shape == t[1].shape == (0,)
    assert torch.equal(gemma_sampling.sample_tokens(x, u, top_k=20)[0], want[0])


def test_draws_follow_the_distribution():
    """20000 draws of a 6-token row: each share within 5 standard deviations."""
    x = torch.tensor([1.0, 0.0, -1.0, 2.0, 0.5, -3.0], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    N = 20000
    token, logprob = sample_tokens(x.expand(N, 6), torch.rand(N, generator=g, device="cuda"), top_k=4)
    p = torch.softmax(x.double(), 0).cpu().numpy()
    p[[2, 5]] = 0
    p /= p.sum()
    share = np.bincount(token.cpu().numpy(), minlength=6) / N
    assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / N)).all() and share[2] == share[5] == 0
    assert np.allclose(logprob.cpu().numpy(), np.log(p[token.cpu().numpy()]), rtol=1e-6, atol=1e-9)


def test_same_tokens_on_every_call_stream_and_replay():
    x, u = make(20, 50000, 21, torch.bfloat16)
    kw = dict(temperature=0.9, top_p=0.9)
    want = sample_tokens(x, u, **kw)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(sample_tokens(x, u, **kw))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want[0]) and torch.equal(l, want[1]) for t, l in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sample_tokens(x, u, **kw)
    x2, u2 = make(20, 50000, 22, torch.bfloat16)
    x.copy_(x2)
    u.copy_(u2)
    graph.replay()
    check(x2, u2, got=out, **kw)


def test_refusals():
    x, u = make(4, 100, 1)
    with pytest.raises(ValueError, match="bfloat16 or float32"):
        sample_tokens(x.half(), u)
    with pytest.raises(ValueError, match="u must be"):
        sample_tokens(x, u[:3])
    with pytest.raises(ValueError, match="u must be"):
        sample_tokens(x, u.double())
    with pytest.raises(ValueError, match="temperature"):
        sample_tokens(x, u, temperature=u[:2])
    with pytest.raises(ValueError, match="NaN"):
        sample_tokens(x, u, top_p=math.nan)
    with pytest.raises(ValueError, match="top_k"):
        sample_tokens(x, u, top_k=2.5)
    with pytest.raises(ValueError, match="dtype"):
        sample_tokens(x, u, top_k=u)
    with pytest.raises(ValueError, match="CUDA"):
        sample_tokens(x.cpu(), u)
    with pytest.raises(ValueError, match="above"):
        sample_tokens(torch.zeros(1, 393217, device="cuda"), u[:1])
    with pytest.raises(ValueError, match="V"):
        sample_tokens(x[:, :0], u)
