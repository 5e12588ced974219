"""What is measured of the serving operators: the residual norm with 8-bit rows, the W8 linear on such rows, and sampling.

A case names its operator in ``op``:

* ``norm``: ``h = x + residual`` in bf16, then the RMSNorm of ``h`` as bf16 rows or as int8 rows with one fp32 scale
  each (Gemma's gain is ``1 + scale``, Qwen's ``scale``);
* ``linear``: int8 rows times int8 weights with one scale per row and one per output channel;
* ``sample``: one token per row of logits under temperature, top-k, top-p and min-p, from given random numbers.
"""

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_ONE = float(1 << 44)  # the fixed-point weight of the most likely token
_TINY = 1.1754943508222875e-38  # smallest normal fp32: the least scale of a quantised row


def listed():
    return [
        # One decode step of one sequence: the norm before a projection, 2048 wide.
        dict(name="norm_q8_1x2048", op="norm", T=1, D=2048, gemma=False, residual=True, out="q8", scale="bf16"),
        # A decode batch on 2560-wide rows with Gemma's gain, bf16 rows out.
        dict(name="norm_bf16_64x2560", op="norm", T=64, D=2560, gemma=True, residual=True, out="bf16", scale="f32"),
        # A ragged chunk of wide rows, the first norm of a stack (nothing to add yet).
        dict(name="norm_q8_777x5128_first", op="norm", T=777, D=5128, gemma=True, residual=False, out="q8", scale="f32"),
        # A prefill chunk.
        dict(name="norm_q8_8192x2560", op="norm", T=8192, D=2560, gemma=True, residual=True, out="q8", scale="bf16"),
        # Query projection of one decoded token (2048 -> 32 heads of 128).
        dict(name="linear_1x2048x4096", op="linear", T=1, K=2048, N=4096, out="bf16", scale="f32", per_channel=True),
        # LM head over a decode batch: the largest weight of a step, logits kept in fp32.
        dict(name="linear_16x2048x151936", op="linear", T=16, K=2048, N=151936, out="f32", scale="f32", per_channel=True),
        # A ragged batch of short requests, odd output width, one scale for the whole weight.
        dict(name="linear_77x2560x10243", op="linear", T=77, K=2560, N=10243, out="bf16", scale="bf16", per_channel=False),
        # Prefill chunk through an MLP-wide product: the largest one.
        dict(name="linear_8192x2560x10240", op="linear", T=8192, K=2560, N=10240, out="bf16", scale="f32", per_channel=True),
        # Next token of one sequence with the usual filters.
        dict(name="sample_1x151936", op="sample", B=1, V=151936, dtype="bf16", top_k=50, top_p=0.95, min_p=0.0, mixed=False),
        # A batch of requests that each bring their own settings (greedy ones among them), a vocabulary of odd size.
        dict(name="sample_64x151643_mixed", op="sample", B=64, V=151643, dtype="f32", top_k=0, top_p=0.0, min_p=0.0, mixed=True),
        # Nucleus and min-p sampling over a large vocabulary.
        dict(name="sample_16x262144_top_p", op="sample", B=16, V=262144, dtype="bf16", top_k=0, top_p=0.9, min_p=0.02, mixed=False),
        # Plain sampling of many rows (rollouts).
        dict(name="sample_256x32000_all", op="sample", B=256, V=32000, dtype="f32", top_k=0, top_p=1.0, min_p=0.0, mixed=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "linear", "sample"])
    if op == "norm":
        D = 8 * _log_int(rng, 16, 1024)
        T = min(_log_int(rng, 1, 8192), max(1, 8192 * 2560 // D))
        return dict(op=op, T=T, D=D, gemma=rng.random() < 0.5, residual=rng.random() < 0.75, out=rng.choice(["q8", "q8", "bf16"]),
                    scale=rng.choice(["f32", "bf16"]))
    if op == "linear":
        K = 16 * _log_int(rng, 4, 640)
        N = min(_log_int(rng, 16, 151936), 2048 * 151936 // K)
        T = min(_log_int(rng, 1, 8192), max(1, 8192 * 2560 * 10240 // (K * N)), max(1, 8192 * 10240 // N))
        return dict(op=op, T=T, K=K, N=N, out=rng.choice(["bf16", "f32"]), scale=rng.choice(["f32", "bf16"]),
                    per_channel=rng.random() < 0.75)
    V = _log_int(rng, 1000, 262144)
    B = min(_log_int(rng, 1, 256), max(1, 64 * 151643 // V))
    return dict(op=op, B=B, V=V, dtype=rng.choice(["bf16", "f32"]), top_k=rng.choice([0, 0, 1, 40, 1000]),
                top_p=rng.choice([1.0, 0.95, 0.6]), min_p=rng.choice([0.0, 0.0, 0.05]), mixed=rng.random() < 0.3)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda") * std

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    s = dict(case)
    if case["op"] == "norm":
        T, D = case["T"], case["D"]
        # A residual stream: a few features far larger than the others, as trained models have them.
        loud = 1.0 + 20.0 * (uniform(D) < 0.004)
        s["x"] = (normal(1, T, D) * loud).to(torch.bfloat16)
        s["residual"] = (normal(1, T, D, std=3.0) * loud).to(torch.bfloat16) if case["residual"] else None
        s["g"] = ((0.0 if case["gemma"] else 1.0) + normal(D, std=0.1)).to(_DT[case["scale"]])
    elif case["op"] == "linear":
        T, K, N = case["T"], case["K"], case["N"]
        # Rows as the norm makes them: the largest value of each is 127.
        x = normal(T, K)
        s["xs"] = x.abs().amax(-1, keepdim=True) / 127.0
        s["xq"] = (x / s["xs"]).round().to(torch.int8)
        s["wq"] = (normal(N, K) * 32.0).round().clamp(-127, 127).to(torch.int8)
        ws = 0.02 * (0.5 + uniform(N, 1)) / 32.0
        s["ws"] = (ws if case["per_channel"] else ws[0, 0].clone()).to(_DT[case["scale"]])
        if own:
            from kappa_b200.qwen3.quant import Q8Weight

            s["w"] = Q8Weight(values=s["wq"], scale=s["ws"])
    else:
        B, V = case["B"], case["V"]
        x = normal(B, V, std=2.0)
        # A handful of likely tokens in each row, and a banned range as a grammar or a padded vocabulary has it.
        hot = torch.randint(0, V, (B, 24), generator=g, device="cuda")
        x.scatter_add_(1, hot, 4.0 + 6.0 * uniform(B, 24))
        x[:, V - V // 50:] = -math.inf
        s["logits"] = x.to(_DT[case["dtype"]])
        s["u"] = uniform(B)
        if case["mixed"]:
            pick = lambda *v: torch.tensor(v, device="cuda")[torch.randint(0, len(v), (B,), generator=g, device="cuda")]  # noqa: E731
            s["temperature"] = pick(0.0, 0.6, 0.8, 1.0, 1.3)
            s["k"] = pick(0, 1, 20, 50, 400).to(torch.int32)
            s["p"] = pick(1.0, 0.95, 0.8)
            s["m"] = pick(0.0, 0.0, 0.05)
        else:
            s["temperature"], s["k"], s["p"], s["m"] = 0.8, case["top_k"], case["top_p"], case["min_p"]
    return s


def _norm_own(s):
    from kappa_b200.gemma3 import norms as gemma
    from kappa_b200.qwen3 import norms as qwen
    from kappa_b200.qwen3.quant import dequantize_rows

    n = gemma if s["gemma"] else qwen
    if s["out"] == "bf16":
        return n.add_rms_norm(s["x"], s["residual"], s["g"]) if s["residual"] is not None else n.rms_norm(s["x"], s["g"])
    if s["residual"] is None:
        q = n.rms_norm_q8(s["x"], s["g"])
        return dequantize_rows(q), q.scale
    h, q = n.add_rms_norm_q8(s["x"], s["residual"], s["g"])
    return h, dequantize_rows(q), q.scale


def _norm_plain(s):
    h = s["x"]
    if s["residual"] is not None:
        h = (h.float() + s["residual"].float()).to(torch.bfloat16)
    f, gain = h.float(), s["g"].float()
    if s["gemma"]:
        gain = gain + 1.0
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6) * gain
    if s["out"] == "bf16":
        y = y.to(torch.bfloat16)
        return (h, y) if s["residual"] is not None else y
    scale = (y.abs().amax(-1, keepdim=True) / 127.0).clamp_min(_TINY)
    v = ((y / scale).round().clamp(-127, 127) * scale).to(torch.bfloat16)
    return (h, v, scale) if s["residual"] is not None else (v, scale)


def _linear_own(s):
    from kappa_b200.qwen3.linear import linear_q8
    from kappa_b200.qwen3.quant import Q8Rows

    return linear_q8(Q8Rows(s["xq"], s["xs"]), s["w"], out_dtype=_DT[s["out"]])


def _linear_plain(s):
    acc = s["xq"].float() @ s["wq"].float().t()
    return (acc * s["xs"] * s["ws"].float().reshape(1, -1)).to(_DT[s["out"]])


def _sample_own(s):
    from kappa_b200.qwen3.sampling import sample_tokens

    return sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["k"], top_p=s["p"], min_p=s["m"])


def _column(v, B, dtype):
    if isinstance(v, torch.Tensor):
        return v.to(dtype).reshape(B, 1)
    # Settings given as numbers are 32-bit ones, as those of a tensor are.
    return torch.full((B, 1), v, dtype=torch.float32, device="cuda").to(dtype)


def _sample_plain(s):
    # In 64 bits: a token changes where a running sum passes a border.
    x = s["logits"].double()
    B, V = x.shape
    x = torch.where(x.isnan(), -math.inf, x)
    T = _column(s["temperature"], B, torch.float64)
    k = _column(s["k"], B, torch.int64)
    order = torch.sort(x, dim=-1, descending=True, stable=True)
    top = order.values[:, :1]
    greedy = ~(T > 0)
    w = (torch.exp((x - top) / torch.where(greedy, 1.0, T)) * _ONE).floor().to(torch.int64)
    ws = w.gather(1, order.indices)
    place = torch.arange(V, device=x.device).reshape(1, V)
    k = torch.where(greedy, 1, torch.where((k <= 0) | (k > V), V, k))
    ws = torch.where(place < k, ws, 0)
    run_ = ws.cumsum(-1)
    p = _column(s["p"], B, torch.float64)
    before = (run_ - ws).double()
    keep = (place < k) & ((before < p * run_[:, -1:].double()) | (p >= 1.0) | (place == 0))
    keep &= (ws.double() >= _column(s["m"], B, torch.float64) * _ONE) | (place == 0)
    kept = torch.zeros_like(w).scatter_(1, order.indices, torch.where(keep, ws, 0))
    total = kept.sum(-1, keepdim=True)
    at = torch.minimum((s["u"].double().reshape(B, 1) * total.double()).to(torch.int64), total - 1)
    token = (kept.cumsum(-1) <= at).sum(-1)
    mass = kept.gather(1, token.reshape(B, 1)).double() / total.double()
    return token.to(torch.int32), mass.log().reshape(B).float()


def run(state):
    if own:
        return {"norm": _norm_own, "linear": _linear_own, "sample": _sample_own}[state["op"]](state)
    return {"norm": _norm_plain, "linear": _linear_plain, "sample": _sample_plain}[state["op"]](state)


def work(case):
    if case["op"] == "norm":
        T, D = case["T"], case["D"]
        out = (T * D + 4 * T) if case["out"] == "q8" else 2 * T * D
        moved = 2 * T * D * (3 if case["residual"] else 1) + out + D * (4 if case["scale"] == "f32" else 2)
        return {"bytes": moved, "flops": 6 * T * D}
    if case["op"] == "linear":
        T, K, N = case["T"], case["K"], case["N"]
        channels = (N if case["per_channel"] else 1) * (4 if case["scale"] == "f32" else 2)
        return {"bytes": T * K + N * K + 4 * T + channels + T * N * (4 if case["out"] == "f32" else 2), "flops": 2 * T * K * N}
    B, V = case["B"], case["V"]
    return {"bytes": B * V * (4 if case["dtype"] == "f32" else 2) + 12 * B, "flops": 3 * B * V}


def _exact_norm(s):
    h = s["x"][0].double()
    if s["residual"] is not None:
        h = (h + s["residual"][0].double()).to(torch.bfloat16).double()
    gain = s["g"].double() + (1.0 if s["gemma"] else 0.0)
    length = torch.linalg.vector_norm(h, dim=-1) / math.sqrt(h.shape[-1])
    y = h * gain / torch.sqrt(length * length + 1e-6)[:, None]
    outs = [h[None]] if s["residual"] is not None else []
    if s["out"] == "bf16":
        return tuple(outs + [y[None]]) if outs else y[None]
    scale = torch.linalg.vector_norm(y, ord=math.inf, dim=-1).div(torch.tensor(127.0, dtype=torch.float64, device=y.device))
    scale = scale.clamp_min(_TINY)[:, None]
    return tuple(outs + [(torch.round(y / scale) * scale)[None], scale[None]])


def _exact_linear(s):
    a = s["xq"].double() * s["xs"].double()
    b = s["wq"].double() * s["ws"].double()
    return torch.einsum("tk,nk->tn", a, b)


def _exact_sample(s):
    import numpy as np

    x = s["logits"].double().cpu().numpy()
    B, V = x.shape

    def per_row(v, kind):
        return v.cpu().numpy().astype(kind) if isinstance(v, torch.Tensor) else np.full(B, np.float32(v)).astype(kind)

    T, p, m = (per_row(s[n], np.float64) for n in ("temperature", "p", "m"))
    k, u = per_row(s["k"], np.int64), s["u"].double().cpu().numpy()
    token, logprob = np.zeros(B, np.int32), np.zeros(B)
    for b in range(B):
        rank = np.lexsort((np.arange(V), -x[b]))
        if T[b] > 0:
            if 0 < k[b] < V:
                rank = rank[: k[b]]
        else:
            rank = rank[:1]
        w = np.floor(np.exp((x[b, rank] - x[b, rank[0]]) / (T[b] if T[b] > 0 else 1.0)) * 2.0**44).astype(np.int64)
        run_ = np.cumsum(w)
        n = len(rank) if p[b] >= 1 else max(1, int(np.searchsorted(run_.astype(np.float64), p[b] * float(run_[-1]), side="left")) + 1)
        n = min(n, max(1, int(np.count_nonzero(w >= m[b] * 2.0**44))))
        by_place = np.argsort(rank[:n])
        cum = np.cumsum(w[:n][by_place])
        j = int(np.searchsorted(cum, min(int(u[b] * float(cum[-1])), int(cum[-1]) - 1), side="right"))
        token[b] = rank[:n][by_place][j]
        logprob[b] = math.log(float(w[:n][by_place][j]) / float(cum[-1]))
    return torch.from_numpy(token), torch.from_numpy(logprob)


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "linear": _exact_linear, "sample": _exact_sample}[case["op"]](s)
