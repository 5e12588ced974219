"""The serving operators in a row, as a decode step uses them: the residual stream through the norm into 8-bit rows, the
projections on them, the output projection and the FFN half in bf16, the final norm into 8-bit rows, the LM head, the
next token.  Every stage is checked against a 64-bit evaluation of its own inputs (tolerances as in the operators' own
tests: one bf16 half step for norms, equality for products and tokens), and the captured step gives the eager one's bits.
"""

from __future__ import annotations

import pytest
import torch

from kappa_b200 import _lib
from kappa_b200.gemma3 import norms as gnorms
from kappa_b200.qwen3 import linear as lin
from kappa_b200.qwen3 import norms as qnorms
from kappa_b200.qwen3 import transformer as QT
from kappa_b200.qwen3.ffn import swiglu_ffn
from kappa_b200.qwen3.quant import quantize_weight
from kappa_b200.qwen3.sampling import sample_tokens
from test_gpu_norm_q8 import _check_rows, _norm64, _within_bf16
from test_gpu_sampling import check as check_tokens

pytestmark = pytest.mark.gpu

D, H, HD, KV, I, V = 512, 8, 64, 2, 1024, 5003


class Layer:
    def __init__(self, gemma):
        g = torch.Generator(device="cuda").manual_seed(17)

        def w(*shape):
            return torch.randn(shape, generator=g, device="cuda") * 0.03

        q = dict(per_channel=True, scale_dtype=torch.float32)
        self.norms = gnorms if gemma else qnorms
        self.gemma = gemma
        self.n1, self.n2, self.n3 = (1.0 * (not gemma) + 0.1 * w(D) for _ in range(3))
        self.q = quantize_weight(w(H, D, HD), **q)
        self.k, self.v = quantize_weight(w(KV, D, HD), **q), quantize_weight(w(KV, D, HD), **q)
        self.o = lin.quantize_attn_out(w(H, HD, D), **q)
        self.gate, self.up = quantize_weight(w(D, I), **q), quantize_weight(w(D, I), **q)
        self.down = quantize_weight(w(I, D), **q)
        self.head = quantize_weight(w(V, D) * 4, in_axis=-1, **q)

    def step(self, x, residual, u, stages=None):
        n = self.norms
        h1, r1 = n.add_rms_norm_q8(x, residual, self.n1)
        q = lin.project_q(r1, self.q)
        k, v = lin.project_kv(r1, self.k, self.v)
        attn = lin.project_attn_out(q + v.repeat_interleave(H // KV, 2), self.o)  # stands for the attention itself
        h2, r2 = n.add_rms_norm(attn, h1, self.n2)
        ffn = swiglu_ffn(r2, self.gate, self.up, self.down)
        h3, r3 = n.add_rms_norm_q8(ffn, h2, self.n3)
        logits = QT.logits_from_hidden(r3, self.head, out_dtype=torch.float32)
        tokens, logprobs = sample_tokens(logits, u, temperature=0.8, top_k=100, top_p=0.9)
        if stages is not None:
            stages.update(h1=h1, r1=r1, q=q, k=k, v=v, attn=attn, h2=h2, r2=r2, ffn=ffn, h3=h3, r3=r3, logits=logits)
        return tokens, logprobs, h3


def _inputs(B, T, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, T, D, generator=g, device="cuda").bfloat16()
    r = (torch.randn(B, T, D, generator=g, device="cuda") * 2).bfloat16()
    return x, r, torch.rand(B, T, generator=g, device="cuda")


def _product(rows, w, axis, dtype):
    """Exactly what the product of 8-bit rows is: whole sums, two fp32 scales, one rounding."""
    wq, ws = w.values.double(), w.scale.float()
    wk = (wq.transpose(-1, -2) if axis == -2 else wq).reshape(-1, D)
    acc = rows.values.double().reshape(-1, D) @ wk.t()
    return ((acc.float() * rows.scale.reshape(-1, 1)) * ws.reshape(1, -1)).to(dtype)


@pytest.mark.parametrize("B,T", [(1, 1), (16, 1), (3, 50)], ids=["token", "batch", "chunk"])
@pytest.mark.parametrize("gemma", [False, True], ids=["qwen", "gemma"])
def test_step(B, T, gemma):
    m = Layer(gemma)
    x, r, u = _inputs(B, T, B + T)
    s = {}
    tokens, logprobs, _ = m.step(x, r, u, s)
    assert torch.equal(s["h1"], (x.float() + r.float()).bfloat16())
    _check_rows(s["r1"], _norm64(s["h1"], m.n1, gemma))
    for name, w in (("q", m.q), ("k", m.k), ("v", m.v)):
        assert torch.equal(s[name].reshape(B * T, -1), _product(s["r1"], w, -2, torch.bfloat16))
    assert torch.equal(s["h2"], (s["attn"].float() + s["h1"].float()).bfloat16())
    _within_bf16(s["r2"], _norm64(s["h2"], m.n2, gemma))
    assert torch.equal(s["h3"], (s["ffn"].float() + s["h2"].float()).bfloat16())
    _check_rows(s["r3"], _norm64(s["h3"], m.n3, gemma))
    assert torch.equal(s["logits"].reshape(B * T, V), _product(s["r3"], m.head, -1, torch.float32))
    check_tokens(s["logits"], u, got=(tokens, logprobs), temperature=0.8, top_k=100, top_p=0.9)
    assert _lib.device_status(x) == 0


def test_captured_steps_replay_with_the_eager_bits():
    """Two captured steps of different sizes, replayed in turn on new inputs."""
    m = Layer(False)
    graphs = []
    for B, T in ((1, 1), (24, 1)):
        x, r, u = _inputs(B, T, 1)
        m.step(x, r, u)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = m.step(x, r, u)
        graphs.append((g, (x, r, u), out))
    for seed in (5, 6, 7):
        for g, (x, r, u), out in graphs:
            new = _inputs(x.shape[0], x.shape[1], seed)
            for a, b in zip((x, r, u), new):
                a.copy_(b)
            g.replay()
            want = m.step(*new)
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert _lib.device_status(graphs[0][1][0]) == 0
