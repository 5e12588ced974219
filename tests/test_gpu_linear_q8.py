"""The W8 linear on 8-bit rows (``linear_q8`` and the projections and head on ``Q8Rows``), bit for bit.

The sum is a whole number below 2^31, exact in 64 bits; what follows is one rounding to fp32, two fp32 products and
one rounding to the output type, each of which torch does alike.  So no tolerance: the outputs are equal.
"""

from __future__ import annotations

import pytest
import torch

from kappa_b200 import _lib
from kappa_b200.gemma3 import linear as glin
from kappa_b200.qwen3 import linear as qlin
from kappa_b200.qwen3 import transformer as QT
from kappa_b200.qwen3.quant import Q8Rows, Q8Weight, pack_weight

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    yield
    assert _lib.device_status(torch.zeros(1, device="cuda")) == 0, "a kernel reported a device-side error"


def _rows(T, K, seed, lo=-127, hi=128):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(lo, hi, (T, K), generator=g, device="cuda").to(torch.int8)
    return Q8Rows(q, torch.rand(T, 1, generator=g, device="cuda") * 0.02 + 1e-3)


def _weight(N, K, seed, per_channel=True, sd=torch.float32, lo=-128, hi=128):
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = torch.randint(lo, hi, (N, K), generator=g, device="cuda").to(torch.int8)
    s = (torch.rand(N, 1, generator=g, device="cuda") * 0.02 + 1e-4) if per_channel else torch.tensor(0.0123, device="cuda")
    return Q8Weight(q, s.to(sd))


def _ref(x, w, dtype):
    acc = x.values.double().reshape(-1, x.values.shape[-1]) @ w.values.double().reshape(-1, w.values.shape[-1]).t()
    return ((acc.float() * x.scale.reshape(-1, 1)) * w.scale.float().reshape(1, -1)).to(dtype)


SHAPES = [(1, 16, 16), (1, 16, 1), (1, 64, 128), (2, 48, 100), (5, 144, 257), (16, 2048, 512), (17, 2064, 129), (33, 4096, 2048),
          (1, 9728, 2560), (64, 256, 3001), (100, 640, 1000), (128, 128, 128), (129, 272, 130), (200, 1040, 700),
          (255, 128, 255), (256, 512, 256), (257, 528, 513), (300, 2048, 1030), (512, 96, 2048), (1000, 2560, 1544),
          (2049, 1024, 777)]


@pytest.mark.parametrize("T,K,N", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_linear_q8(T, K, N, dtype):
    x = _rows(T, K, T + K + N)
    for per_channel, sd in ((True, torch.float32), (True, torch.bfloat16), (False, torch.bfloat16)):
        w = _weight(N, K, T + K, per_channel, sd)
        y = qlin.linear_q8(x, w, out_dtype=dtype)
        assert y.dtype == dtype and torch.equal(y, _ref(x, w, dtype))


@pytest.mark.parametrize("T,K,N", [(1100, 64, 1000), (1100, 272, 1021), (1100, 2064, 1025), (2049, 64, 1024), (2049, 272, 511),
                                   (2049, 2576, 1090), (4100, 144, 2049), (4100, 2048, 640),
                                   (257, 9728, 10240), (300, 9728, 10243), (513, 5136, 20480)])
def test_many_rows(T, K, N):
    """Sizes that go to the pair kernel: several tiles a pair, ends inside them, one and two output boxes a warp, a few rows
    behind the last whole tile."""
    x, w = _rows(T, K, N), _weight(N, K, T)
    for dtype in (torch.bfloat16, torch.float32):
        assert torch.equal(qlin.linear_q8(x, w, out_dtype=dtype), _ref(x, w, dtype))


@pytest.mark.parametrize("T,K,N", [(1, 208, 100), (16, 2048, 512), (50, 1040, 257), (256, 512, 256), (300, 2048, 1030), (700, 272, 2000),
                                   (2049, 272, 1030), (30000, 64, 48)])
def test_packed_weights_give_the_same_bits(T, K, N):
    x, w = _rows(T, K, 5), _weight(N, K, 6)
    for dtype in (torch.bfloat16, torch.float32):
        assert torch.equal(qlin.linear_q8(x, pack_weight(w, in_axis=-1), out_dtype=dtype), _ref(x, w, dtype))


@pytest.mark.parametrize("T,K,N", [(300, 64, 1), (300, 64, 3), (300, 64, 8), (260, 64, 16), (300, 64, 24), (257, 64, 72), (257, 64, 63), (257, 64, 65), (270, 80, 127), (513, 64, 255), (258, 64, 258),
                                   (400, 48, 301)]
                         + [(30000, 64, N) for N in (1, 2, 3, 7, 8, 15, 16, 17, 63, 64, 65, 66)])
def test_widths_around_the_tiles(T, K, N):
    """Output rows that start at every alignment, ends inside a word, a box and a tile."""
    x, w = _rows(T, K, N), _weight(N, K, N)
    for dtype in (torch.bfloat16, torch.float32):
        buf = torch.full((T * N + 8,), 7.0, dtype=dtype, device="cuda")
        for shift in (0, 1, 4):
            out = buf[shift:shift + T * N].reshape(T, N)
            wk = _lib.KW8Weight(w.values.data_ptr(), w.scale.data_ptr(), _lib.DT_F32, 1, 0, 0)
            _lib.check(_lib.load().kw8_linear_q8(x.values.data_ptr(), x.scale.data_ptr(), T, K, N, wk,
                                                 _lib.DT_F32 if dtype == torch.float32 else _lib.DT_BF16, out.data_ptr(),
                                                 _lib.stream_of(out)))
            assert torch.equal(out, _ref(x, w, dtype))
            assert (buf[:shift] == 7).all() and (buf[shift + T * N:] == 7).all()
            buf.fill_(7.0)


def test_largest_sums():
    """Every product at its extreme: the sum reaches 128 * 128 * K just below 2^31."""
    K = 131056
    for T, N in ((3, 20), (300, 300), (1000, 1000)):
        for a, b in ((-128, -128), (-128, 127), (127, 127)):
            x = Q8Rows(torch.full((T, K), a, dtype=torch.int8, device="cuda"), torch.ones(T, 1, device="cuda"))
            w = Q8Weight(torch.full((N, K), b, dtype=torch.int8, device="cuda"), torch.ones(N, 1, device="cuda"))
            y = qlin.linear_q8(x, w, out_dtype=torch.float32)
            assert (y == torch.tensor(a * b * K, dtype=torch.float64).float().item()).all()


def test_scales_that_are_not_finite_stay_in_their_row():
    x, w = _rows(40, 512, 8), _weight(300, 512, 9)
    x.scale[7] = float("nan")
    x.scale[9] = float("inf")
    x.values[9] = 1
    y = qlin.linear_q8(x, w)
    assert torch.isnan(y[7]).all() and not torch.isfinite(y[9]).any()
    keep = [i for i in range(40) if i not in (7, 9)]
    assert torch.equal(y[keep], _ref(Q8Rows(x.values[keep], x.scale[keep]), w, torch.bfloat16))


def test_leading_axes_layouts_and_no_rows():
    x = _rows(2 * 3 * 4, 256, 3)
    w = _weight(96, 256, 4)
    want = _ref(x, w, torch.bfloat16)
    x4 = Q8Rows(x.values.reshape(2, 3, 4, 256), x.scale.reshape(2, 3, 4, 1))
    assert torch.equal(qlin.linear_q8(x4, w), want.reshape(2, 3, 4, 96))
    xt = Q8Rows(x4.values.transpose(0, 2), x4.scale.transpose(0, 2))
    assert torch.equal(qlin.linear_q8(xt, w), want.reshape(2, 3, 4, 96).transpose(0, 2))
    wt = Q8Weight(w.values.t(), w.scale.reshape(1, 96))
    assert torch.equal(qlin.linear_q8(x, wt, in_axis=-2), want)
    off = torch.cat([x.values.reshape(-1)[:1], x.values.reshape(-1)])[1:].reshape(24, 256)
    assert off.data_ptr() % 16 and torch.equal(qlin.linear_q8(Q8Rows(off, x.scale), w), want)
    assert tuple(qlin.linear_q8(Q8Rows(x.values[:0], x.scale[:0]), w).shape) == (0, 96)


def test_projections_and_head_take_8_bit_rows():
    x = _rows(2 * 5, 512, 13)
    x3 = Q8Rows(x.values.reshape(2, 5, 512), x.scale.reshape(2, 5, 1))

    def heads(n, h, seed):
        w = _weight(n * h, 512, seed)
        return w, Q8Weight(w.values.reshape(n, h, 512).transpose(1, 2), w.scale.reshape(n, 1, h))

    wq, q = heads(4, 64, 20)
    assert torch.equal(qlin.project_q(x3, q), _ref(x, wq, torch.bfloat16).reshape(2, 5, 4, 64))
    (wk, k), (wv, v) = heads(2, 64, 21), heads(2, 64, 22)
    got = qlin.project_kv(x3, k, v)
    assert torch.equal(got[0], _ref(x, wk, torch.bfloat16).reshape(2, 5, 2, 64))
    assert torch.equal(got[1], _ref(x, wv, torch.bfloat16).reshape(2, 5, 2, 64))
    kv = Q8Weight(torch.stack([k.values.transpose(1, 2), v.values.transpose(1, 2)]).transpose(2, 3),
                  torch.stack([k.scale, v.scale]))
    for a, b in zip(glin.project_kv(x3, kv), got):
        assert torch.equal(a, b)
    head = _weight(1001, 512, 23)
    for dt in (None, torch.float32):
        want = _ref(x, head, dt or torch.bfloat16).reshape(2, 5, 1001)
        assert torch.equal(QT.logits_from_hidden(x3, head, out_dtype=dt), want)
        assert torch.equal(QT.logits_from_hidden_tied(x3, head, out_dtype=dt), want)


def test_rows_behind_the_last_are_left_alone():
    """The kernel writes T rows of N values and nothing else."""
    lib = _lib.load()
    for T, K, N in ((3, 256, 100), (130, 256, 136), (300, 256, 520), (2100, 256, 1036), (2100, 256, 1037)):
        x, w = _rows(T, K, 1), _weight(N, K, 2)
        out = torch.full((T + 8, N), 7.0, dtype=torch.bfloat16, device="cuda")
        wk = _lib.KW8Weight(w.values.data_ptr(), w.scale.data_ptr(), _lib.DT_F32, 1, 0, 0)
        _lib.check(lib.kw8_linear_q8(x.values.data_ptr(), x.scale.data_ptr(), T, K, N, wk, _lib.DT_BF16, out[4:].data_ptr(),
                                     _lib.stream_of(out)))
        assert torch.equal(out[4:T + 4], _ref(x, w, torch.bfloat16))
        assert (out[:4] == 7).all() and (out[T + 4:] == 7).all()


def test_two_streams_and_a_graph():
    cases = [(_rows(T, K, T), _weight(N, K, N)) for T, K, N in ((1, 2048, 4096), (16, 2048, 6000), (300, 1024, 2048))]
    want = [_ref(x, w, torch.bfloat16) for x, w in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(qlin.linear_q8(*cases[i]))
    torch.cuda.synchronize()
    for ys, r in zip(got, want):
        assert all(torch.equal(y, r) for y in ys)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ys = [qlin.linear_q8(*c) for c in cases]
    for x, _ in cases:
        x.values.copy_(x.values.flip(0).roll(3, 1))
    graph.replay()
    for y, (x, w) in zip(ys, cases):
        assert torch.equal(y, _ref(x, w, torch.bfloat16))


def test_refusals():
    x, w = _rows(4, 64, 1), _weight(32, 64, 2)
    with pytest.raises(TypeError, match="8-bit rows"):
        qlin.linear_q8(x.values, w)
    with pytest.raises(TypeError, match="W8"):
        qlin.linear_q8(x, w.values)
    with pytest.raises(ValueError, match="features"):
        qlin.linear_q8(x, _weight(32, 80, 2))
    with pytest.raises(ValueError, match="out_dtype"):
        qlin.linear_q8(x, w, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="one scale per row"):
        qlin.linear_q8(Q8Rows(x.values, x.scale[:, 0]), w)
    with pytest.raises(ValueError, match="fp32 scales"):
        qlin.linear_q8(Q8Rows(x.values, x.scale.bfloat16()), w)
    with pytest.raises(ValueError, match="CUDA"):
        qlin.linear_q8(Q8Rows(x.values.cpu(), x.scale.cpu()), w)
    with pytest.raises(ValueError, match="multiple of 16"):
        qlin.linear_q8(Q8Rows(x.values[:, :40].contiguous(), x.scale), Q8Weight(w.values[:, :40].contiguous(), w.scale))
