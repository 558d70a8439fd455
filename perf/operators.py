"""The operators of 8-bit training and distillation as cases that can be timed and compared: their plain forms, the
library's calls, and their definitions in 64 bits.

Four operators, as a student decoder in 8 bits uses them:

  quantize  ops.quantize_fp8: e4m3 values with one power-of-two scale for each block of 128 elements of a row (or of
            128 x 128), optionally with the transpose quantised along the other dimension as well
  product   ops.gemm_fp8: C[M, N] = A[M, K] * B[N, K]^T from such operands, each block's partial sum times its scales
  linear    ops.linear_fp8, forward and backward: a training step's use of the two above
  distill   ops.distillation_loss, forward and backward: cross-entropy of a student against a teacher's top logits
"""
import math

import torch

own = False   # False: the plain forms; True: the library's calls

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}
E4M3 = torch.float8_e4m3fn
BLOCK = 128

MOST_QUANTIZED = 14336 * 4096
MOST_PRODUCT = 4096 * 14336 * 4096
MOST_LINEAR = 8192 * 1024 * 4096
MOST_LOGITS = 8192 * 50257


def listed():
    return [
        # Activations of a decode batch on their way into an 8-bit product: all latency.
        {"name": "quantize_16x4096", "kind": "quantize", "m": 16, "k": 4096, "type": "bf16", "rows": 1, "both": False},
        # FFN activations of eight sequences of 1024 tokens, for the product of the forward pass and, transposed, for
        # the gradient of the weight.
        {"name": "quantize_8192x4096_both", "kind": "quantize", "m": 8192, "k": 4096, "type": "bf16", "rows": 1, "both": True},
        # An FFN weight in fp32 as a checkpoint or an optimizer's master copy holds it, 128 x 128 blocks.
        {"name": "quantize_weight_fp32", "kind": "quantize", "m": 14336, "k": 4096, "type": "fp32", "rows": 128, "both": False},
        # One token through a square projection: weight traffic and latency.
        {"name": "product_1", "kind": "product", "m": 1, "n": 4096, "k": 4096, "out": "bf16", "bias": False, "b_rows": 128},
        # A decode batch of 16 through the FFN's first weight.
        {"name": "product_16", "kind": "product", "m": 16, "n": 14336, "k": 4096, "out": "bf16", "bias": True, "b_rows": 128},
        # A ragged middle-sized product, no dimension of which divides into tiles, a scale for every row of B.
        {"name": "product_ragged_777", "kind": "product", "m": 777, "n": 1003, "k": 1544, "out": "fp16", "bias": True, "b_rows": 1},
        # Prefill: 4096 tokens through the FFN's first weight.
        {"name": "product_4096", "kind": "product", "m": 4096, "n": 14336, "k": 4096, "out": "bf16", "bias": False, "b_rows": 128},
        # The first FFN layer of the GPT-2 shaped decoder (1024 features) on eight sequences of 1024 tokens.
        {"name": "linear_8192", "kind": "linear", "m": 8192, "n": 4096, "k": 1024, "type": "bf16", "bias": True},
        # A batch with padding removed: an odd number of tokens, a width that is no multiple of a block.
        {"name": "linear_ragged_1001", "kind": "linear", "m": 1001, "n": 5000, "k": 1288, "type": "fp16", "bias": False},
        # The last positions of 64 sequences against a teacher's 8 best tokens, logits in rows padded to eight.
        {"name": "distill_64x50257", "kind": "distill", "t": 64, "v": 50257, "k": 8, "type": "bf16", "tau": 1.0, "reduction": "mean",
         "padded": True},
        # The decoder's training batch against 64 entries a token, dense rows that start anywhere; prompt tokens
        # have no entry.
        {"name": "distill_8192x50257", "kind": "distill", "t": 8192, "v": 50257, "k": 64, "type": "bf16", "tau": 2.0, "reduction": "mean",
         "padded": False},
        # Logits in fp32, a loss for every token (weighted by the caller).
        {"name": "distill_fp32_2000x32000", "kind": "distill", "t": 2000, "v": 32000, "k": 100, "type": "fp32", "tau": 1.5,
         "reduction": "none", "padded": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "product", "product", "linear", "distill"])
    while True:
        if kind == "quantize":
            case = {"kind": kind, "m": _log_int(rng, 1, 16384), "k": _log_int(rng, 16, 16384), "type": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    "rows": rng.choice([1, 1, 128]), "both": rng.random() < 0.5}
            if case["m"] * case["k"] * SIZES[case["type"]] <= 2 * MOST_QUANTIZED:
                return case
        elif kind == "product":
            case = {"kind": kind, "m": _log_int(rng, 1, 8192), "n": _log_int(rng, 64, 14336), "k": _log_int(rng, 64, 14336),
                    "out": rng.choice(["bf16", "bf16", "fp16"]), "bias": rng.random() < 0.5, "b_rows": rng.choice([128, 128, 1])}
            if rng.random() < 0.5:   # a layer's width more often than not divides into blocks
                case["n"], case["k"] = max(128, case["n"] // 128 * 128), max(128, case["k"] // 128 * 128)
            if case["m"] * case["n"] * case["k"] <= MOST_PRODUCT:
                return case
        elif kind == "linear":
            case = {"kind": kind, "m": _log_int(rng, 1, 16384), "n": _log_int(rng, 64, 8192), "k": _log_int(rng, 64, 8192),
                    "type": rng.choice(["bf16", "bf16", "fp16"]), "bias": rng.random() < 0.5}
            if case["m"] * case["n"] * case["k"] <= MOST_LINEAR:
                return case
        else:
            case = {"kind": kind, "t": _log_int(rng, 1, 8192), "v": _log_int(rng, 1000, 131072), "k": _log_int(rng, 1, 512),
                    "type": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "tau": rng.choice([0.7, 1.0, 2.0, 4.0]),
                    "reduction": rng.choice(["mean", "mean", "sum", "none"]), "padded": rng.random() < 0.5}
            if case["t"] * case["v"] * SIZES[case["type"]] <= 2 * MOST_LOGITS:
                return case


# ---- inputs


def _activations(gen, m, k, dtype):
    """Rows of different sizes, a few features far above the others, now and then a row of zeros (a padding token)."""
    x = torch.randn(m, k, generator=gen, device="cuda")
    x *= torch.exp(torch.randn(m, 1, generator=gen, device="cuda") * 0.5)
    x *= torch.where(torch.rand(1, k, generator=gen, device="cuda") < 0.01, 20.0, 1.0)
    if m > 8:
        x[torch.randint(0, m, (m // 64 + 1,), generator=gen, device="cuda")] = 0.0
    return x.to(dtype)


def _weight(gen, n, k, dtype):
    return (torch.randn(n, k, generator=gen, device="cuda") * 0.02).to(dtype)


def _checkpoint(gen, n, k, rows):
    """An 8-bit weight as a checkpoint has it: scales of any value, not powers of two alone."""
    w = _weight(gen, n, k, torch.float32)
    scale = _block_max(w, rows).clamp_min(1e-12) / 448.0
    q = torch.empty(n, (k + 15) // 16 * 16, dtype=E4M3, device="cuda")[:, :k]
    return q.copy_((w / _spread(scale, rows, n, k)).to(E4M3)), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, state = case["kind"], {"case": case}
    if kind == "quantize":
        if case["rows"] == 128:
            state["x"] = _weight(gen, case["m"], case["k"], TYPES[case["type"]])
        else:
            state["x"] = _activations(gen, case["m"], case["k"], TYPES[case["type"]])
    elif kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        q, scale = _quantize(_activations(gen, m, k, torch.bfloat16), 1)
        a = torch.empty(m, (k + 15) // 16 * 16, dtype=E4M3, device="cuda")[:, :k]   # rows on 16 bytes
        state["a"], state["a_scale"] = a.copy_(q), scale.t().contiguous().t()       # a column of scales for a block of K
        state["b"], state["b_scale"] = _checkpoint(gen, n, k, case["b_rows"])
        state["bias"] = torch.randn(n, generator=gen, device="cuda").to(TYPES[case["out"]]) if case["bias"] else None
    elif kind == "linear":
        m, n, k, dtype = case["m"], case["n"], case["k"], TYPES[case["type"]]
        state["x"] = _activations(gen, m, k, dtype).requires_grad_()
        state["weight"] = _weight(gen, n, k, dtype).requires_grad_()
        state["bias"] = torch.randn(n, generator=gen, device="cuda").to(dtype).requires_grad_() if case["bias"] else None
        state["grad"] = (_activations(gen, m, n, torch.float32) * 1e-3).to(dtype)
    else:
        t, v, k = case["t"], case["v"], case["k"]
        wide = (v + 7) // 8 * 8 if case["padded"] else v
        start = torch.randint(0, v, (t, 1), generator=gen, device="cuda")
        step = torch.randint(1, max(1, v // k) + 1, (t, 1), generator=gen, device="cuda")
        ids = (start + step * torch.arange(k, device="cuda")) % v
        logits = torch.randn(t, wide, generator=gen, device="cuda") * 2
        gap = torch.rand(t, k, generator=gen, device="cuda") * (8.0 / k)
        top = 14.0 - gap.cumsum(1)
        logits.scatter_add_(1, ids, top * 0.7)
        # entries that a nucleus cut off, and tokens of the prompt, which have none (the first token has one)
        ids[torch.rand(t, k, generator=gen, device="cuda") < 0.1] = -1
        ids[torch.rand(t, generator=gen, device="cuda") < 0.15] = -1
        ids[0, 0] = start[0, 0]
        state["logits"] = logits.to(TYPES[case["type"]])[:, :v].requires_grad_()
        state["ids"], state["top"] = ids, top
        state["grad"] = torch.rand((t,) if case["reduction"] == "none" else (), generator=gen, device="cuda") + 0.5
    return state


# ---- plain forms


def _block_max(x, rows):
    """Largest magnitude of each block of `rows` x 128, in fp32."""
    m, k = x.shape
    x = torch.nn.functional.pad(x.float().abs(), (0, -k % BLOCK, 0, -m % rows))
    return x.view(x.shape[0] // rows, rows, x.shape[1] // BLOCK, BLOCK).amax((1, 3))


def _spread(scale, rows, m, k):
    return scale.repeat_interleave(rows, 0)[:m].repeat_interleave(BLOCK, 1)[:, :k]


def _quantize(x, rows):
    """Values and scales: the smallest power of two that brings a block's largest magnitude to 448 or less."""
    top = _block_max(x, rows)
    half, e = torch.frexp(top)   # top = half * 2^e, half in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(top == 0, -126, (e - 9 + (half > 0.875).int()).clamp_min(-126))
    scale = ((e + 127) << 23).to(torch.int32).view(torch.float32)
    return (x.float() / _spread(scale, rows, *x.shape)).to(E4M3), scale


def _values(q, scale, rows):
    return q.float() * _spread(scale, rows, *q.shape)


def _plain_linear(x, weight, bias, grad):
    m, (n, k) = x.shape[0], weight.shape
    w = _values(*_quantize(weight, 128), 128)
    y = _values(*_quantize(x, 1), 1) @ w.t()
    if bias is not None:
        y = y + bias.float()
    dx = _values(*_quantize(grad, 1), 1) @ w
    dw = _values(*_quantize(grad.t(), 1), 1) @ _values(*_quantize(x.t(), 1), 1).t()
    out = [y.to(x.dtype), dx.to(x.dtype), dw.to(x.dtype)]
    return out if bias is None else out + [grad.float().sum(0).to(x.dtype)]


def _plain_distill(logits, ids, top, tau, reduction, grad):
    z = logits.float()
    there = ids >= 0
    at = ids.clamp_min(0)
    t = torch.where(there, top, -math.inf)
    counts = there.any(1)
    t = (t - torch.where(counts, t.amax(1), 0.0).unsqueeze(1)) / tau
    e = torch.exp(t)
    total = torch.where(counts, e.sum(1), 1.0).unsqueeze(1)
    p = e / total
    high = z.amax(1, keepdim=True)
    e = torch.exp((z - high) / tau)
    s = e.sum(1, keepdim=True)
    log_q = (z.gather(1, at) - high) / tau - torch.log(s)
    rows = tau * tau * torch.where(p > 0, p * (t - torch.log(total) - log_q), 0.0).sum(1)
    n = counts.sum()
    loss = rows if reduction == "none" else rows.sum() if reduction == "sum" else rows.sum() / n
    factor = grad * tau / (n if reduction == "mean" else 1)
    d = (e / s).scatter_add_(1, at, -p) * torch.where(counts, factor, 0.0).unsqueeze(1)
    return [loss, d.to(logits.dtype)]


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from mini_nccl_b200 import ops

        if kind == "quantize":
            return list(ops.quantize_fp8(state["x"], block_rows=case["rows"], transposed=case["both"]))
        if kind == "product":
            return ops.gemm_fp8(state["a"], state["a_scale"], state["b"], state["b_scale"], bias=state["bias"], out_dtype=TYPES[case["out"]])
        if kind == "linear":
            leaves = [t for t in (state["x"], state["weight"], state["bias"]) if t is not None]
            y = ops.linear_fp8(state["x"], state["weight"], state["bias"])
            return [y.detach(), *torch.autograd.grad(y, leaves, state["grad"])]
        loss = ops.distillation_loss(state["logits"], state["ids"], state["top"], temperature=case["tau"], reduction=case["reduction"])
        return [loss.detach(), *torch.autograd.grad(loss, [state["logits"]], state["grad"])]
    with torch.no_grad():
        if kind == "quantize":
            q, scale = _quantize(state["x"], case["rows"])
            if not case["both"]:
                return [q, scale]
            if case["rows"] == 128:
                return [q, scale, q.t().contiguous(), scale.t().contiguous()]
            return [q, scale, *_quantize(state["x"].t(), 1)]
        if kind == "product":
            y = _values(state["a"], state["a_scale"], 1) @ _values(state["b"], state["b_scale"], case["b_rows"]).t()
            if state["bias"] is not None:
                y = y + state["bias"].float()
            return y.to(TYPES[case["out"]])
        if kind == "linear":
            return _plain_linear(state["x"], state["weight"], state["bias"], state["grad"])
        return _plain_distill(state["logits"], state["ids"], state["top"], case["tau"], case["reduction"], state["grad"])


def work(case):
    kind = case["kind"]
    blocks = lambda n: -(-n // BLOCK)  # noqa: E731
    if kind == "quantize":
        m, k = case["m"], case["k"]
        scales = -(-m // case["rows"]) * blocks(k) + (blocks(m) * (k if case["rows"] == 1 else blocks(k)) if case["both"] else 0)
        return {"bytes": m * k * (SIZES[case["type"]] + (2 if case["both"] else 1)) + 4 * scales, "flops": 3.0 * m * k}
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        scales = (m + -(-n // case["b_rows"])) * blocks(k)
        return {"bytes": m * k + n * k + 4 * scales + SIZES[case["out"]] * (m * n + (n if case["bias"] else 0)), "flops": 2.0 * m * n * k}
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        size = SIZES[case["type"]]
        return {"bytes": size * (2 * m * k + 2 * n * k + 2 * m * n + (2 * n if case["bias"] else 0)), "flops": 6.0 * m * n * k}
    t, v = case["t"], case["v"]
    return {"bytes": 2 * t * v * SIZES[case["type"]] + 12 * t * case["k"] + (8 * t if case["reduction"] == "none" else 8), "flops": 8.0 * t * v}


# ---- definitions in 64 bits


def _exact_quantize(x, rows):
    """(values / scale, scale) by arithmetic: no conversion to 8 bits, no bit patterns."""
    x = x.double()
    m, k = x.shape
    top = torch.zeros(-(-m // rows), -(-k // BLOCK), dtype=torch.float64, device=x.device)
    at = (torch.arange(m, device=x.device) // rows)[:, None] * top.shape[1] + torch.arange(k, device=x.device)[None, :] // BLOCK
    top.view(-1).scatter_reduce_(0, at.reshape(-1), x.abs().reshape(-1), "amax")
    near = torch.exp2(torch.round(torch.log2(top / 448.0)).clamp_min(-126.0))
    scale = torch.where(448.0 * near >= top, near, 2.0 * near)   # (a logarithm may come out above a whole number)
    v = x / scale.view(-1)[at]
    near = torch.exp2(torch.round(torch.log2(v.abs())).clamp_min(-7.0))
    step = torch.where(near <= v.abs(), near, 0.5 * near).clamp_min(2.0 ** -6) / 8.0   # e4m3: three bits behind the leading one
    return torch.round(v / step) * step, scale, at


def _exact_values(x, rows):
    q, scale, at = _exact_quantize(x, rows)
    return q * scale.view(-1)[at]


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    with torch.no_grad():
        if kind == "quantize":
            q, scale, _ = _exact_quantize(state["x"], case["rows"])
            if not case["both"]:
                return [q, scale]
            if case["rows"] == 128:
                return [q, scale, q.t().contiguous(), scale.t().contiguous()]
            return [q, scale, *_exact_quantize(state["x"].t().contiguous(), 1)[:2]]
        if kind == "product":
            def values(q, scale, rows):
                i, j = torch.arange(q.shape[0], device="cuda") // rows, torch.arange(q.shape[1], device="cuda") // BLOCK
                return q.double() * scale.double()[i][:, j]

            y = torch.einsum("mk,nk->mn", values(state["a"], state["a_scale"], 1), values(state["b"], state["b_scale"], case["b_rows"]))
            return y if state["bias"] is None else y + state["bias"].double()
        if kind == "linear":
            x, weight, grad = state["x"], state["weight"], state["grad"]
            w = _exact_values(weight, 128)
            y = torch.einsum("mk,nk->mn", _exact_values(x, 1), w)
            dx = torch.einsum("mn,nk->mk", _exact_values(grad, 1), w)
            dw = torch.einsum("nm,km->nk", _exact_values(grad.t().contiguous(), 1), _exact_values(x.t().contiguous(), 1))
            if state["bias"] is None:
                return [y, dx, dw]
            return [y + state["bias"].double(), dx, dw, grad.double().sum(0)]
        z, ids, tau = state["logits"].double() / case["tau"], state["ids"], case["tau"]
        counts = (ids >= 0).any(1)
        t = (state["top"].double() / tau).masked_fill(ids < 0, -math.inf)
        log_p = (t - torch.logsumexp(t, 1, keepdim=True)).masked_fill(ids < 0, 0.0)
        p = log_p.exp().masked_fill(ids < 0, 0.0)
        lse = torch.logsumexp(z, 1, keepdim=True)
        rows = tau ** 2 * (p * (log_p - z.gather(1, ids.clamp_min(0)) + lse)).sum(1)
        n = int(counts.sum())
        loss = {"none": rows, "sum": rows.sum(), "mean": rows.sum() / n}[case["reduction"]]
        d = torch.exp(z - lse)
        del z
        d.scatter_add_(1, ids.clamp_min(0), -p)
        d *= ((state["grad"].double() * tau / (n if case["reduction"] == "mean" else 1)) * counts).reshape(-1, 1)
        return [loss, d]
