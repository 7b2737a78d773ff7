"""Workloads of the operators that close a mixture-of-experts block: the dense W8A8 product (shared expert, projections, head), the norm
behind the block with its gate and scaled residual sum and the next block's norm in int8 rows, and the experts' load with its balance loss
and gradient.

``run`` computes them in elementary torch operations in fp32 (64 bits for long sums and for differences of nearly equal numbers), or, with
``own``, through this package.  ``exact`` computes them in 64 bits.  Sizes follow ``perf/cases.py`` and ``synth.CONFIGS`` (hidden 7168,
intermediate 2048, gate/up 4096, 256 experts, top-8; the small model's 2048 / 768 / 64 experts; 611 tokens of 1424 x 2976 and their odd
neighbours as sizes that fill no tile).
"""
from __future__ import annotations

import math

import torch

DEV = "cuda:0"
_TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}

#: False: plain torch operations.  True: the operators of this package.
own = False


def listed():
    return [
        # the small model's shared down projection while 16 sequences decode: one short launch, latency counts
        dict(name="matmul_small", op="matmul", tokens=16, K=768, N=2048, layout="kn", out="bf16", bias="none", per_token=True),
        # the large model's shared gate/up width while 16 sequences decode: 29 MB of weights stream through, as a checkpoint stores them
        dict(name="matmul_decode", op="matmul", tokens=16, K=7168, N=4096, layout="nk", out="bf16", bias="none", per_token=True),
        # a prefill of 4096 tokens over the same weights
        dict(name="matmul_prefill", op="matmul", tokens=4096, K=7168, N=4096, layout="kn", out="bf16", bias="none", per_token=True),
        # a middling batch whose sizes are odd in every direction, with bias, fp32 rows for what follows
        dict(name="matmul_ragged", op="matmul", tokens=611, K=1423, N=2977, layout="nk", out="f32", bias="f32", per_token=True),
        # the block's exit on the small model, 16 sequences decode: fp32 sums of the experts, no gate
        dict(name="sandwich_decode", op="sandwich", tokens=16, h=2048, x="f32", dtype="bf16", post=True, gate="none", act="none",
             smooth=False, quant=True, normed=True),
        # the same with 128 sequences of the large model, a sigmoid gate for each token and smoothing scales
        dict(name="sandwich_decode_gate", op="sandwich", tokens=128, h=7168, x="f16", dtype="f16", post=True, gate="token", act="sigmoid",
             smooth=True, quant=True, normed=False),
        # a prefill of 4096 tokens whose next block takes 16-bit rows; a learned gate for each channel
        dict(name="sandwich_prefill", op="sandwich", tokens=4096, h=7168, x="f32", dtype="bf16", post=True, gate="channel", act="none",
             smooth=False, quant=False, normed=True),
        # rows of an odd length, a gate for each element, residual scaling without a norm behind the block
        dict(name="sandwich_ragged", op="sandwich", tokens=611, h=1423, x="bf16", dtype="bf16", post=False, gate="full", act="tanh",
             smooth=False, quant=True, normed=True),
        # the load of one decoding step, for placement and for moving the balancing bias
        dict(name="balance_decode", op="balance", tokens=16, experts=64, top_k=8, dtype="bf16", scoring="softmax", sequences=0, masked=False,
             grad=False),
        # one training step of the router over 4096 tokens, loss and gradient
        dict(name="balance_step", op="balance", tokens=4096, experts=256, top_k=8, dtype="bf16", scoring="softmax", sequences=0, masked=False,
             grad=True),
        # a long packed batch: the loss of each of 16 sequences, sigmoid scores in fp32
        dict(name="balance_packed", op="balance", tokens=16384, experts=256, top_k=8, dtype="f32", scoring="sigmoid", sequences=16,
             masked=False, grad=True),
        # a padded batch (rows without a token, experts that are switched off), a count of experts that fills no lane evenly
        dict(name="balance_ragged", op="balance", tokens=3001, experts=155, top_k=6, dtype="f16", scoring="softmax", sequences=7, masked=True,
             grad=True),
    ]


def _span(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """1 to 4096 tokens (16384 for the load) over widths of 256 to 8192, odd ones among them, 8 to 256 experts, whole batches and up to 64
    packed sequences; never more work than the largest listed case of the operator."""
    op = rng.choice(["matmul", "sandwich", "balance"])
    while True:
        tokens = _span(rng, 1, 16384 if op == "balance" else 4096)
        if op == "matmul":
            K, N = (_span(rng, 256, 8192) if rng.random() < 0.25 else 16 * _span(rng, 16, 512) for _ in range(2))
            out = rng.choice(["bf16", "bf16", "f16", "f32"])
            if tokens * K * N > 4096 * 7168 * 4096 or tokens * (K + _BYTES[out] * N) + K * N > 4096 * (7168 + 2 * 4096) + 7168 * 4096:
                continue
            return dict(op=op, tokens=tokens, K=K, N=N, layout=rng.choice(["kn", "nk"]), out=out,
                        bias=rng.choice(["none", "none", "f32", "out"]), per_token=rng.random() < 0.9)
        if op == "sandwich":
            h = _span(rng, 256, 8192) if rng.random() < 0.4 else 16 * _span(rng, 16, 512)
            dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
            c = dict(op=op, tokens=tokens, h=h, x=rng.choice(["f32", dtype]), dtype=dtype, post=rng.random() < 0.8,
                     gate=rng.choice(["none", "none", "channel", "token", "full"]), act=rng.choice(["none", "sigmoid", "tanh"]),
                     smooth=rng.random() < 0.3, quant=rng.random() < 0.7, normed=rng.random() < 0.5)
            if work(c)["bytes"] > 4096 * 7168 * 10:
                continue
            return c
        experts = _span(rng, 8, 256)
        if tokens * experts > 16384 * 256:
            continue
        return dict(op=op, tokens=tokens, experts=experts, top_k=rng.randint(1, min(8, experts)), dtype=rng.choice(["f32", "bf16", "f16"]),
                    scoring=rng.choice(["softmax", "sigmoid"]), sequences=rng.choice([0, 0, min(_span(rng, 1, 64), tokens)]),
                    masked=rng.random() < 0.3, grad=rng.random() < 0.7)


def work(case):
    """Bytes: every input read and every output written once (the gradient reads the logits again: it needs the counts of all tokens)."""
    t = case["tokens"]
    if case["op"] == "matmul":
        K, N, e = case["K"], case["N"], _BYTES[case["out"]]
        return {"bytes": t * K + K * N + t * N * e + 4 * N + 4 * t, "flops": 2 * t * K * N}
    if case["op"] == "sandwich":
        h, e = case["h"], _BYTES[case["dtype"]]
        gate = {"none": 0, "channel": e * h, "token": e * t, "full": e * t * h}[case["gate"]]
        planes = _BYTES[case["x"]] + (2 + case["normed"]) * e + case["quant"]
        return {"bytes": t * h * planes + gate + 4 * t * case["quant"] + h * e * (1 + case["post"]) + 4 * h * case["smooth"], "flops": 12 * t * h}
    E, e = case["experts"], _BYTES[case["dtype"]]
    return {"bytes": t * E * e * (3 if case["grad"] else 1) + 4 * t * case["top_k"] + 12 * E * max(1, case["sequences"]),
            "flops": t * E * (12 if case["grad"] else 6)}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------

def _gen(seed, i):
    return torch.Generator(DEV).manual_seed(seed * 1000 + i)


def _normal(shape, seed, i, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, device=DEV, generator=_gen(seed, i)) * scale).to(dtype)


def _int8(shape, seed, i):
    # what per-row quantisation makes of activations and weights
    return _normal(shape, seed, i, scale=32).round_().clamp_(-127, 127).to(torch.int8)


def prepare(case, seed):
    s = {"case": case}
    t = case["tokens"]
    if case["op"] == "matmul":
        K, N = case["K"], case["N"]
        s["x"] = _int8((t, K), seed, 1)
        # [K, N], or the view of a weight that is stored [N, K]
        s["w"] = _int8((K, N), seed, 2) if case["layout"] == "kn" else _int8((N, K), seed, 2).t()
        s["scale"] = (torch.rand(N, device=DEV, generator=_gen(seed, 3)) * 0.5 + 0.75) / (32 * math.sqrt(K))
        s["token"] = (torch.rand(t, device=DEV, generator=_gen(seed, 4)) + 0.5) / 32 if case["per_token"] else None
        bias = {"none": None, "f32": torch.float32, "out": _TORCH[case["out"]]}[case["bias"]]
        s["bias"] = None if bias is None else _normal((N,), seed, 5, bias, 0.5)
    elif case["op"] == "sandwich":
        h, dtype = case["h"], _TORCH[case["dtype"]]
        # activations of a residual stream: normal with a few channels that are an order of magnitude larger
        wide = 1 + 15 * (torch.rand(h, device=DEV, generator=_gen(seed, 1)) < 0.004)
        s["x"] = _normal((t, h), seed, 2, _TORCH[case["x"]], 3.0)
        s["residual"] = (_normal((t, h), seed, 3) * wide).to(dtype)
        s["gamma"] = _normal((h,), seed, 4, scale=0.2).add_(1).to(dtype)
        s["post"] = _normal((h,), seed, 5, scale=0.2).add_(0.7).to(dtype) if case["post"] else None
        s["smooth"] = torch.rand(h, device=DEV, generator=_gen(seed, 6)) + 0.5 if case["smooth"] else None
        shape = {"none": None, "channel": (h,), "token": (t, 1), "full": (t, h)}[case["gate"]]
        s["gate"] = None if shape is None else _normal(shape, seed, 7, dtype)
    else:
        E, k, n = case["experts"], case["top_k"], case["sequences"]
        logits = _normal((t, E), seed, 1) + _normal((E,), seed, 2, scale=0.5)
        if case["masked"]:  # experts that are switched off for a token
            logits.masked_fill_(torch.rand(t, E, device=DEV, generator=_gen(seed, 3)) < 0.05, -math.inf)
        s["logits"] = logits.to(_TORCH[case["dtype"]])
        s["mask"] = torch.rand(t, device=DEV, generator=_gen(seed, 4)) < 0.8 if case["masked"] else None
        # the router's choices, shifted by a balancing bias; -1 where there is no token or no expert
        best, ids = (logits + _normal((E,), seed, 5, scale=0.1)).topk(k, dim=1)
        ids = torch.where(best > -math.inf, ids, -1)
        s["ids"] = (torch.where(s["mask"][:, None], ids, -1) if case["masked"] else ids).to(torch.int32)
        s["cu"] = None
        if n:
            cuts = torch.randint(0, t + 1, (n + 1,), device=DEV, generator=_gen(seed, 6)).sort().values
            cuts[0] = 0
            if not case["masked"]:  # a padded batch ends before its rows do
                cuts[-1] = t
            s["cu"] = cuts.to(torch.int32)
        # what the loss is multiplied by on its way into the total; with fp16 the loss scale that keeps gradients out of the subnormals
        s["grad_loss"] = (torch.rand((), device=DEV, generator=_gen(seed, 7)) + 0.5) * (256 * t if case["dtype"] == "f16" else 1) if case["grad"] else None
    return s


COEFFICIENT = 1e-2
RESIDUAL_SCALE, BLOCK_SCALE = 0.875, 0.5
EPS = 1e-6


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms: fp32, rounded once at the end
# ---------------------------------------------------------------------------------------------------------------------

def _plain_matmul(s):
    y = (s["x"].float() @ s["w"].float()) * s["scale"]
    if s["token"] is not None:
        y = y * s["token"][:, None]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(_TORCH[s["case"]["out"]])


def _values(q, scale):
    """The int8 rows as the values that they stand for, in 16 bits."""
    return q.to(torch.bfloat16).mul_(scale.to(torch.bfloat16)[:, None])


def _plain_sandwich(s):
    case, n = s["case"], s["x"].float()
    dtype = _TORCH[case["dtype"]]
    if case["post"]:
        n = n * torch.rsqrt(n.square().mean(1, keepdim=True) + EPS) * s["post"].float()
    if s["gate"] is not None:
        g = s["gate"].float()
        if case["act"] == "sigmoid":
            g = 1.0 / (1.0 + torch.exp(-g))
        elif case["act"] == "tanh":
            e = torch.exp(-2.0 * g.abs())
            g = torch.sign(g) * (1.0 - e) / (1.0 + e)
        n = n * g
    h = s["residual"].float() * RESIDUAL_SCALE + n * BLOCK_SCALE
    rms = torch.rsqrt(h.square().mean(1, keepdim=True) + EPS)
    u = h * s["gamma"].float()
    normed = (u * rms).to(dtype) if case["normed"] else None
    if not case["quant"]:
        return None, None, h.to(dtype), normed
    if case["smooth"]:
        u = u * s["smooth"]
    amax = u.abs().amax(1, keepdim=True)
    step = amax / torch.full_like(amax, 127.0)
    q = torch.where(step > 0, torch.round(u / step), torch.zeros_like(u))
    scale = (step * rms).squeeze(1)
    return _values(q, scale), scale, h.to(dtype), normed


def _plain_balance(s):
    case, l = s["case"], s["logits"].float()
    t, E, k = case["tokens"], case["experts"], case["top_k"]
    gone = ~(l > -math.inf)
    if case["scoring"] == "sigmoid":
        score = torch.where(gone, 0.0, 1.0 / (1.0 + torch.exp(-l)))
    else:
        top = torch.where(gone, -math.inf, l).amax(1, keepdim=True)
        score = torch.where(gone, 0.0, torch.exp(torch.where(l == top, 0.0, l - top)))
    total = score.sum(1, keepdim=True)
    p = torch.where(total > 0, score / total, 0.0)
    # which sequence a row belongs to, as one row of ones and zeros for each sequence
    row = torch.arange(t, device=l.device)
    member = torch.ones(1, t, dtype=torch.bool, device=l.device)
    if s["cu"] is not None:
        member = (row >= s["cu"][:-1, None]) & (row < s["cu"][1:, None])
    if s["mask"] is not None:
        member = member & s["mask"]
    # 64 bits for the sums over all tokens and for the differences that the gradient is made of
    member = member.double()
    tokens = member.sum(1, keepdim=True)
    chosen = (s["ids"][:, :, None] == torch.arange(E, device=l.device)).sum(1)
    counts = member @ chosen.double()
    some = (tokens > 0).sum()
    slope = torch.where(tokens > 0, COEFFICIENT * E / k * counts / (tokens * tokens * some), 0.0)
    loss = (slope * (member @ p.double())).sum().float()
    counts = counts.to(torch.int64)
    if s["cu"] is None:
        counts = counts[0]
    if not case["grad"]:
        return loss, counts, None
    d = member.t() @ slope
    d = d - (p * d).sum(1, keepdim=True)
    grad = p * d * s["grad_loss"]
    if case["scoring"] == "sigmoid":
        grad = grad * (1.0 - score)
    return loss, counts, (grad * member.sum(0)[:, None]).to(s["logits"].dtype)


def _own(s):
    import ops_transformer_b200 as ops
    case = s["case"]
    if case["op"] == "matmul":
        return ops.quant_matmul(s["x"], s["w"], s["scale"], s["token"], bias=s["bias"], out_dtype=_TORCH[case["out"]])
    if case["op"] == "sandwich":
        q, scale, h, y = ops.sandwich_norm_quant(s["x"], s["residual"], s["gamma"], post_gamma=s["post"], gate=s["gate"], gate_act=case["act"],
                                                 residual_scale=RESIDUAL_SCALE, block_scale=BLOCK_SCALE, smooth=s["smooth"], eps=EPS,
                                                 quant=case["quant"], normed=case["normed"])
        return (None, None, h, y) if q is None else (_values(q, scale), scale, h, y)
    loss, counts, weight = ops.expert_balance(s["logits"], s["ids"], scoring=case["scoring"], coefficient=COEFFICIENT, token_mask=s["mask"],
                                              cu_seqlens=s["cu"])
    if not case["grad"]:
        return loss, counts, None
    return loss, counts, ops.expert_balance_grad(s["logits"], counts, weight, scoring=case["scoring"], token_mask=s["mask"], cu_seqlens=s["cu"],
                                                 grad_loss=s["grad_loss"])


def run(s):
    """One pass: the product's rows; (int8 rows as values, their scales, the residual stream, normed rows); (loss, counts, gradient)."""
    if own:
        return _own(s)
    return {"matmul": _plain_matmul, "sandwich": _plain_sandwich, "balance": _plain_balance}[s["case"]["op"]](s)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "matmul":
        y = torch.mm(s["x"].double(), s["w"].double()) * s["scale"].double()
        y = y * s["token"].double().unsqueeze(1) if s["token"] is not None else y
        return y if s["bias"] is None else y + s["bias"].double()
    if case["op"] == "sandwich":
        h = BLOCK_SCALE * s["x"].double()
        if case["post"]:
            x = s["x"].double()
            h = h / ((x * x).sum(1, keepdim=True) / case["h"] + EPS).sqrt() * s["post"].double()
        if s["gate"] is not None:
            h = h * {"none": lambda v: v, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[case["act"]](s["gate"].double())
        h = h + RESIDUAL_SCALE * s["residual"].double()
        y = h / ((h * h).sum(1, keepdim=True) / case["h"] + EPS).sqrt() * s["gamma"].double()
        out = h, y if case["normed"] else None
        if not case["quant"]:
            return (None, None) + out
        z = y * s["smooth"].double() if case["smooth"] else y
        scale = z.abs().max(1, keepdim=True).values / 127
        return ((z / scale).round() * scale, scale[:, 0]) + out
    l = s["logits"].double().clone()
    t, E, k = case["tokens"], case["experts"], case["top_k"]
    live = torch.ones(t, dtype=torch.bool, device=l.device) if s["mask"] is None else s["mask"]
    cuts = [0, t] if s["cu"] is None else s["cu"].tolist()
    parts = [torch.arange(a, b, device=l.device)[live[a:b]] for a, b in zip(cuts[:-1], cuts[1:])]
    parts = [at for at in parts if len(at)]
    l.requires_grad_(True)
    loss = l.nan_to_num(neginf=0.0).sum() * 0   # no token at all: no loss, and a gradient of zeros
    for at in parts:
        row = l[at]
        p = torch.softmax(row, 1) if case["scoring"] == "softmax" else torch.sigmoid(row) / torch.sigmoid(row).sum(1, keepdim=True)
        ids = s["ids"][at].reshape(-1).long()
        share = torch.bincount(ids[ids >= 0], minlength=E).double() * E / (k * len(at))
        loss = loss + COEFFICIENT * (share * p.mean(0)).sum() / len(parts)
    if case["grad"]:
        loss.backward(s["grad_loss"].double())
    return loss.detach(), None, torch.nan_to_num(l.grad) if case["grad"] else None
