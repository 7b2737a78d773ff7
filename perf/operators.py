"""Workloads of the operators that stand around the quantised expert FFN in a mixture-of-experts block: the norm that makes its
int8 rows, the choice of experts, and low-rank adapters of many requests beside a shared projection.

``run`` computes them in elementary torch operations in fp32, or, with ``own``, through this package.  ``exact`` computes them in 64
bits.  Sizes follow ``perf/cases.py`` and ``synth.CONFIGS`` (hidden 7168, intermediate 2048, 256 experts, top-8; the small model's
2048 / 768 / 64 experts; 611 tokens of 1424 x 2976 as the size that fills no tile).
"""
from __future__ import annotations

import math

import torch

DEV = "cuda:0"
_TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4, "int8": 1}

#: False: plain torch operations in fp32.  True: the operators of this package.
own = False


def listed():
    return [
        # decoding with 16 sequences on a small model: one short launch, latency counts
        dict(name="norm_decode", op="norm", tokens=16, h=2048, dtype="bf16", residual=True, smooth=False, normed=True),
        # decoding with 128 sequences of the large model, smoothing scales in front of the quantisation
        dict(name="norm_decode_smooth", op="norm", tokens=128, h=7168, dtype="f16", residual=True, smooth=True, normed=False),
        # a prefill of 4096 tokens: the residual stream, the router's rows and the int8 rows are written in one pass
        dict(name="norm_prefill", op="norm", tokens=4096, h=7168, dtype="bf16", residual=True, smooth=False, normed=True),
        # rows of an odd length in fp32, without a residual
        dict(name="norm_ragged", op="norm", tokens=611, h=1423, dtype="f32", residual=False, smooth=False, normed=True),
        # the small model's router while decoding: softmax over 64 experts
        dict(name="route_decode", op="route", tokens=16, experts=64, top_k=8, dtype="bf16", scoring="softmax", bias=False, groups=1,
             top_groups=1, group_score="max", masked=False),
        # the large model's: sigmoid scores, a balancing bias, the four best of eight groups
        dict(name="route_decode_groups", op="route", tokens=128, experts=256, top_k=8, dtype="f32", scoring="sigmoid", bias=True,
             groups=8, top_groups=4, group_score="top2", masked=False),
        # the same for a prefill of 16384 tokens
        dict(name="route_prefill_groups", op="route", tokens=16384, experts=256, top_k=8, dtype="f32", scoring="sigmoid", bias=True,
             groups=8, top_groups=4, group_score="top2", masked=False),
        # a padded batch (rows without a token, experts that are switched off), biased softmax scores, a count of experts that fills no
        # lane evenly
        dict(name="route_ragged", op="route", tokens=3001, experts=155, top_k=6, dtype="f16", scoring="softmax", bias=True, groups=5,
             top_groups=3, group_score="max", masked=True),
        # the small model's gate/up projection while decoding: 16 sequences, 4 tenants
        dict(name="adapter_decode", op="adapter", tokens=16, requests=16, adapters=4, rank=16, K=2048, N=1536, dtype="bf16", x="bf16",
             without=0.0),
        # the large model's shared down projection, 128 sequences of 64 tenants, int8 rows as the SwiGLU operator returns them
        dict(name="adapter_decode_many", op="adapter", tokens=128, requests=128, adapters=64, rank=32, K=2048, N=7168, dtype="bf16",
             x="int8", without=0.1),
        # a prefill of 4096 tokens in 16 prompts over 8 tenants
        dict(name="adapter_prefill", op="adapter", tokens=4096, requests=16, adapters=8, rank=64, K=7168, N=4096, dtype="bf16", x="bf16",
             without=0.0),
        # sizes that fill no tile, a rank that is no power of two, a quarter of the prompts without an adapter
        dict(name="adapter_ragged", op="adapter", tokens=611, requests=37, adapters=13, rank=12, K=1424, N=2976, dtype="f16", x="f16",
             without=0.25),
    ]


def _span(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """1 to 4096 tokens (16384 for the router) over widths of 256 to 8192, odd ones among them, 8 to 256 experts, 1 to 64 adapters of
    rank 4 to 64; never more work than the largest listed case of the operator."""
    op = rng.choice(["norm", "route", "adapter"])
    while True:
        tokens = _span(rng, 1, 16384 if op == "route" else 4096)
        if op == "norm":
            h = _span(rng, 256, 8192) if rng.random() < 0.5 else 16 * _span(rng, 16, 512)
            dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
            if tokens * h * _BYTES[dtype] > 4096 * 7168 * 2:
                continue
            return dict(op=op, tokens=tokens, h=h, dtype=dtype, residual=rng.random() < 0.7, smooth=rng.random() < 0.3,
                        normed=rng.random() < 0.6)
        if op == "route":
            groups = rng.choice([1, 1, 4, 8])
            experts = groups * max(2, _span(rng, 8, 256) // groups)
            if tokens * experts > 16384 * 256:
                continue
            top_groups = groups if groups == 1 else rng.randint(1, groups - 1)
            return dict(op=op, tokens=tokens, experts=experts, top_k=rng.randint(1, min(8, top_groups * experts // groups)),
                        dtype=rng.choice(["f32", "bf16", "f16"]), scoring=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5,
                        groups=groups, top_groups=top_groups, group_score=rng.choice(["max", "top2"]), masked=rng.random() < 0.3)
        K, N = (_span(rng, 256, 8192) if rng.random() < 0.3 else 16 * _span(rng, 16, 512) for _ in range(2))
        adapters, rank = _span(rng, 1, 64), _span(rng, 4, 64)
        if tokens * adapters * rank * (K + N) > 4096 * 512 * (7168 + 4096) or tokens * (K + 2 * N) > 4096 * (7168 + 2 * 4096):
            continue
        dtype = rng.choice(["bf16", "bf16", "f16"])
        return dict(op=op, tokens=tokens, requests=min(tokens, _span(rng, 1, 128)), adapters=adapters, rank=rank, K=K, N=N, dtype=dtype,
                    x=rng.choice([dtype, dtype, "int8"]), without=rng.choice([0.0, 0.0, 0.25]))


def work(case):
    """Bytes: every input read and every output written once (of the adapters, those that some token can name)."""
    t = case["tokens"]
    if case["op"] == "norm":
        h, e = case["h"], _BYTES[case["dtype"]]
        planes = 1 + (2 if case["residual"] else 0) + (1 if case["normed"] else 0)
        return {"bytes": t * h * (planes * e + 1) + 4 * t + h * (e + (4 if case["smooth"] else 0)), "flops": 8 * t * h}
    if case["op"] == "route":
        return {"bytes": t * case["experts"] * _BYTES[case["dtype"]] + 8 * t * case["top_k"], "flops": 4 * t * case["experts"]}
    K, N, r, used = case["K"], case["N"], case["rank"], min(case["adapters"], case["requests"])
    return {"bytes": t * K * _BYTES[case["x"]] + 4 * t * N + 2 * used * r * (K + N) + 4 * t, "flops": 2 * t * r * (K + N)}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------

def _gen(seed, i):
    return torch.Generator(DEV).manual_seed(seed * 1000 + i)


def _normal(shape, seed, i, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, device=DEV, generator=_gen(seed, i)) * scale).to(dtype)


def prepare(case, seed):
    s = {"case": case}
    t = case["tokens"]
    if case["op"] == "norm":
        h, dtype = case["h"], _TORCH[case["dtype"]]
        # activations of a residual stream: normal with a few channels that are an order of magnitude larger
        wide = 1 + 15 * (torch.rand(h, device=DEV, generator=_gen(seed, 1)) < 0.004)
        s["x"] = _normal((t, h), seed, 2, dtype)
        s["residual"] = (_normal((t, h), seed, 3) * wide).to(dtype) if case["residual"] else None
        s["gamma"] = _normal((h,), seed, 4, scale=0.2).add_(1).to(dtype)
        s["smooth"] = torch.rand(h, device=DEV, generator=_gen(seed, 5)) + 0.5 if case["smooth"] else None
    elif case["op"] == "route":
        E = case["experts"]
        logits = _normal((t, E), seed, 1) + _normal((E,), seed, 2, scale=0.5)
        if case["masked"]:  # experts that are switched off for a token
            logits.masked_fill_(torch.rand(t, E, device=DEV, generator=_gen(seed, 3)) < 0.05, -math.inf)
        s["logits"] = logits.to(_TORCH[case["dtype"]])
        # a bias that load balancing has moved up and down by steps of a thousandth
        s["bias"] = torch.randint(-60, 61, (E,), device=DEV, generator=_gen(seed, 4)) * 1e-3 if case["bias"] else None
        s["mask"] = torch.rand(t, device=DEV, generator=_gen(seed, 5)) < 0.8 if case["masked"] else None
    else:
        K, N, r, L, dtype = case["K"], case["N"], case["rank"], case["adapters"], _TORCH[case["dtype"]]
        if case["x"] == "int8":
            s["x"] = _normal((t, K), seed, 1, scale=32).round_().clamp_(-127, 127).to(torch.int8)
            s["x_scale"] = (torch.rand(t, device=DEV, generator=_gen(seed, 2)) + 0.5) / 32
        else:
            s["x"], s["x_scale"] = _normal((t, K), seed, 1, dtype), None
        s["a"] = _normal((L, r, K), seed, 3, dtype, 1 / math.sqrt(K))
        s["b"] = _normal((L, N, r), seed, 4, dtype, 0.25 / math.sqrt(r))
        s["base"] = _normal((t, N), seed, 5, dtype)
        s["scaling"] = torch.rand(L, device=DEV, generator=_gen(seed, 6)) + 1
        # the tokens of a request stand together and share its adapter, -1 where it has none
        adapter = torch.randint(0, L, (case["requests"],), device=DEV, generator=_gen(seed, 7))
        none = torch.rand(case["requests"], device=DEV, generator=_gen(seed, 8)) < case["without"]
        adapter = torch.where(none, -1, adapter)
        s["ids"] = adapter[torch.arange(t, device=DEV) * case["requests"] // t].to(torch.int32)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms: fp32, rounded once at the end
# ---------------------------------------------------------------------------------------------------------------------

def _plain_norm(s):
    case, x = s["case"], s["x"]
    h = x.float()
    if case["residual"]:
        h = h + s["residual"].float()
    rms = torch.rsqrt(h.square().mean(1, keepdim=True) + 1e-6)
    u = h * s["gamma"].float()
    normed = u * rms
    if case["smooth"]:
        u = u * s["smooth"]
    amax = u.abs().amax(1, keepdim=True)
    step = amax / torch.full_like(amax, 127.0)
    q = torch.where(step > 0, torch.round(u / step), torch.zeros_like(u))
    # the int8 rows as the values that they stand for
    return ((q * (step * rms)).to(x.dtype), (step * rms).squeeze(1), h.to(x.dtype) if case["residual"] else None,
            normed.to(x.dtype) if case["normed"] else None)


def _plain_route(s):
    case, l = s["case"], s["logits"].float()
    t, E, G, k = case["tokens"], case["experts"], case["groups"], case["top_k"]
    gone = ~(l > -math.inf)
    if case["scoring"] == "sigmoid":
        scores = 1.0 / (1.0 + torch.exp(-l))
    else:
        top = torch.where(gone, -math.inf, l).amax(1, keepdim=True)
        e = torch.where(gone, 0.0, torch.exp(torch.where(l == top, 0.0, l - top)))
        # 64 bits for the one sum that a choice can hang on: which expert wins must not go by the order of its terms
        total = e.sum(1, keepdim=True, dtype=torch.float64).float()
        scores = torch.where(total > 0, e / total, 0.0)
    scores = torch.where(gone, 0.0, scores)
    choice = scores + s["bias"] if case["bias"] else scores
    if not case["bias"] and (G == 1 or case["group_score"] == "max"):
        choice = l  # the scores grow with the logits
    choice = torch.where(gone | torch.isnan(choice), -math.inf, choice)
    if G > 1:
        best = choice.view(t, G, E // G).sort(dim=2, descending=True).values
        group = best[:, :, 0]
        if case["group_score"] == "top2":
            second = best[:, :, 1]
            group = group + torch.where(second > -math.inf, second, 0.0)
        stays = torch.zeros(t, G, dtype=torch.bool, device=l.device)
        stays.scatter_(1, group.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]], True)
        choice = torch.where(stays.repeat_interleave(E // G, dim=1), choice, -math.inf)
    value, ids = (v[:, :k] for v in choice.sort(dim=1, descending=True, stable=True))
    there = value > -math.inf
    if case["masked"]:
        there = there & s["mask"][:, None]
    w = torch.where(there, scores.gather(1, ids), 0.0)
    total = w.sum(1, keepdim=True)
    w = torch.where(total > 0, w / total, 0.0) * 2.5
    return w, torch.where(there, ids, -1).to(torch.int32)


def _plain_adapter(s):
    case, x = s["case"], s["x"].float()
    L, r = case["adapters"], case["rank"]
    if s["x_scale"] is not None:
        x = x * s["x_scale"][:, None]
    v = (x @ s["a"].float().view(L * r, -1).t()).view(-1, L, r)
    mine = s["ids"][:, None] == torch.arange(L, device=x.device)
    v = v * (mine * s["scaling"])[:, :, None]
    delta = v.view(-1, L * r) @ s["b"].float().transpose(1, 2).reshape(L * r, -1)
    return (s["base"].float() + delta).to(s["base"].dtype)


def _own(s):
    import ops_transformer_b200 as ops
    case = s["case"]
    if case["op"] == "norm":
        q, scale, h, y = ops.add_rms_norm_quant(s["x"], s["gamma"], residual=s["residual"], smooth=s["smooth"], eps=1e-6,
                                                normed=case["normed"])
        return torch.mul(q, scale[:, None], out=torch.empty_like(s["x"])), scale, h, y
    if case["op"] == "route":
        return ops.route_top_k(s["logits"], case["top_k"], scoring=case["scoring"], bias=s["bias"], n_group=case["groups"],
                               topk_group=case["top_groups"], group_score=case["group_score"], renormalize=True, scale=2.5,
                               token_mask=s["mask"])
    return ops.adapter_add(s["base"], s["x"], s["a"], s["b"], s["ids"], x_scale=s["x_scale"], scaling=s["scaling"])


def run(s):
    """One pass: (int8 rows as values, their scales, residual sum, normed rows), (weights, expert ids) or the projection's rows."""
    if own:
        return _own(s)
    return {"norm": _plain_norm, "route": _plain_route, "adapter": _plain_adapter}[s["case"]["op"]](s)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h = h + s["residual"].double()
        y = h / ((h * h).sum(1, keepdim=True) / case["h"] + 1e-6).sqrt() * s["gamma"].double()
        z = y * s["smooth"].double() if s["smooth"] is not None else y
        scale = z.abs().max(1, keepdim=True).values / 127
        return ((z / scale).round() * scale, scale[:, 0], h if s["residual"] is not None else None, y if case["normed"] else None)
    if case["op"] == "route":
        l = s["logits"].double()
        t, E, G = case["tokens"], case["experts"], case["groups"]
        scores = torch.sigmoid(l) if case["scoring"] == "sigmoid" else torch.nan_to_num(torch.softmax(l, 1), nan=0.0)
        choice = scores + (s["bias"].double() if s["bias"] is not None else 0)
        choice = torch.where(l == -math.inf, -math.inf, choice)
        if G > 1:
            rank = choice.view(t, G, -1).topk(2, dim=2).values
            rank = rank[..., 0] if case["group_score"] == "max" else rank[..., 0] + torch.nan_to_num(rank[..., 1], neginf=0.0)
            place = rank.argsort(dim=1, descending=True, stable=True).argsort(dim=1)  # equal groups: the first one is the better one
            choice = torch.where((place < case["top_groups"]).repeat_interleave(E // G, 1), choice, -math.inf)
        at = choice.argsort(dim=1, descending=True, stable=True)[:, :case["top_k"]]
        w = scores.gather(1, at) * (choice.gather(1, at) > -math.inf)
        if s["mask"] is not None:
            w = w * s["mask"][:, None]
        return 2.5 * w / w.sum(1, keepdim=True).clamp_min(1e-300), None
    out = s["base"].double()
    for i in range(case["adapters"]):
        at = (s["ids"] == i).nonzero()[:, 0]
        x = s["x"][at].double() * (s["x_scale"][at, None].double() if s["x_scale"] is not None else 1)
        out[at] += s["scaling"][i].double() * ((x @ s["a"][i].double().t()) @ s["b"][i].double().t())
    return out
