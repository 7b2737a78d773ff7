"""The mixture-of-experts block that runs the norm, the router, the adapters and the W8A8 operators together, against the same block in 64
bits without quantised activations."""
import math

import pytest
import torch

from ops_transformer_b200.block import random_block

pytestmark = pytest.mark.gpu
DEV = "cuda"


def reference(block, x, residual, ids, weights, adapter_ids, unquantised):
    """The block's output in 64 bits for the experts that it chose."""
    h = (x.float() + residual.float()).double()
    y = h / (h.square().mean(1, keepdim=True) + block.eps).sqrt() * block.gamma.double()
    down = unquantised["w_down"]

    def expert(v, w1, s1, w2, s2):
        t = v @ (w1.double() * s1.double())
        gate, up = t.chunk(2, dim=-1)
        return torch.nn.functional.silu(gate) * up, w2.double() * s2.double()

    act, w2 = expert(y, block.shared[0][0], block.shared[1][0], block.shared[2][0], block.shared[3][0])
    out = act @ w2
    if adapter_ids is not None:
        for i in range(block.adapters.a.shape[0]):
            at = (adapter_ids == i).nonzero()[:, 0]
            out[at] += block.adapters.scaling[i].double() * (act[at] @ block.adapters.a[i].double().t() @ block.adapters.b[i].double().t())
    for e in range(block.experts):
        token, slot = (ids == e).nonzero(as_tuple=True)
        if len(token):
            act, w2 = expert(y[token], block.w_gate_up[e], block.s_gate_up[e], down[e], block.s_down[e])
            out.index_add_(0, token, weights[token, slot, None].double() * (act @ w2))
    return out


@pytest.mark.parametrize("tokens,hidden,inter,experts,top_k,adapters,routing", [
    (1, 512, 256, 8, 2, 3, dict(scoring="softmax")),
    (40, 1024, 512, 16, 4, 5, dict(scoring="sigmoid", n_group=4, topk_group=2, group_score="top2", routed_scale=2.5)),
    (300, 768, 256, 12, 3, 0, dict(scoring="softmax", n_group=3, topk_group=2)),
])
def test_block_against_64_bits(monkeypatch, tokens, hidden, inter, experts, top_k, adapters, routing):
    from ops_transformer_b200 import block as module
    seen, kept = {}, {}
    monkeypatch.setattr(module, "route_top_k", lambda *a, _f=module.route_top_k, **k: seen.setdefault("r", _f(*a, **k)))
    monkeypatch.setattr(module, "format_cast_nz", lambda w, _f=module.format_cast_nz: _f(kept.setdefault("w_down", w)))
    if routing["scoring"] == "sigmoid":
        routing = dict(routing, router_bias=torch.randn(experts, device=DEV, generator=torch.Generator(DEV).manual_seed(3)) * 0.05)
    b = random_block(hidden, inter, experts, top_k, adapters=adapters, **routing)
    g = torch.Generator(DEV).manual_seed(1)
    x, residual = (torch.randn(tokens, hidden, device=DEV, generator=g).to(torch.bfloat16) for _ in range(2))
    adapter_ids = torch.randint(-1, adapters, (tokens,), device=DEV, generator=g).to(torch.int32) if adapters else None
    mask = torch.rand(tokens, device=DEV, generator=g) < 0.8
    mask[0] = True
    out, stream = b(x, residual, adapter_ids=adapter_ids, token_mask=mask)
    assert torch.equal(stream, (x.float() + residual.float()).to(torch.bfloat16))
    weights, ids = seen["r"]
    assert (ids[~mask] == -1).all() and (ids[mask] >= 0).all()
    want = reference(b, x, residual, ids, weights, adapter_ids, kept)
    # Two quantisations of rows, each with a step of their largest value / 127: for normal rows of these lengths at most 4.5 sigma, so an
    # error of 4.5 / 127 / sqrt(12) = 1.02 % of the row; the products of gate and up double the first one.  sqrt(2^2 + 1) * 1.02 % = 2.3 %,
    # and 0.4 % for each of two 16-bit roundings: below 4 %.
    assert (out.double() - want).norm() / want.norm() < 0.04


def test_block_can_be_captured():
    b = random_block(512, 256, 8, 2, adapters=2, scoring="softmax")
    x, residual = (torch.randn(24, 512, device=DEV).to(torch.bfloat16) for _ in range(2))
    ids = (torch.arange(24, device=DEV) % 3 - 1).to(torch.int32)
    b(x, residual, adapter_ids=ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, stream = b(x, residual, adapter_ids=ids)
    x.copy_(torch.randn(24, 512, device=DEV))
    graph.replay()
    torch.cuda.synchronize()
    got = out.clone(), stream.clone()
    want = b(x, residual, adapter_ids=ids)
    assert torch.equal(got[1], want[1])
    # rows are added into the result in no fixed order: a few units in the last place of fp32 sums of order one
    assert (got[0] - want[0]).abs().max() < 64 * 2.0 ** -24 * math.sqrt(512)


@pytest.mark.parametrize("tokens,hidden,inter,experts,top_k,adapters,masked,routing", [
    (1, 512, 256, 8, 2, 3, "none", dict(scoring="softmax")),
    (40, 1024, 512, 16, 4, 5, "some", dict(scoring="sigmoid", n_group=4, topk_group=2, group_score="top2", routed_scale=2.5)),
    (300, 768, 256, 12, 3, 3, "some", dict(scoring="softmax", n_group=3, topk_group=2)),
    (300, 768, 256, 12, 3, 40, "first", dict(scoring="softmax")),
    (65, 512, 256, 8, 2, 2, "all", dict(scoring="sigmoid")),
])
def test_block_row_by_row(monkeypatch, tokens, hidden, inter, experts, top_k, adapters, masked, routing):
    """Every row by itself: one pair of token and expert that goes astray is a third of its token's row and next to nothing of all rows.  Rows
    that the mask takes out are the shared expert with its adapter alone."""
    from ops_transformer_b200 import block as module
    seen, kept = {}, {}
    monkeypatch.setattr(module, "route_top_k", lambda *a, _f=module.route_top_k, **k: seen.setdefault("r", _f(*a, **k)))
    monkeypatch.setattr(module, "format_cast_nz", lambda w, _f=module.format_cast_nz: _f(kept.setdefault("w_down", w)))
    b = random_block(hidden, inter, experts, top_k, adapters=adapters, **routing)
    g = torch.Generator(DEV).manual_seed(2)
    x, residual = (torch.randn(tokens, hidden, device=DEV, generator=g).to(torch.bfloat16) for _ in range(2))
    adapter_ids = torch.randint(-1, adapters, (tokens,), device=DEV, generator=g).to(torch.int32)
    at = torch.arange(tokens, device=DEV)
    mask = {"none": at >= 0, "some": torch.rand(tokens, device=DEV, generator=g) < 0.6, "first": at >= tokens // 2, "all": at < 0}[masked]
    out, _ = b(x, residual, adapter_ids=adapter_ids, token_mask=mask)
    weights, ids = seen["r"]
    assert (ids[~mask] == -1).all() and (ids[mask] >= 0).all()
    want = reference(b, x, residual, ids, weights, adapter_ids, kept)
    # A row's two quantisations have steps of its largest value / 127.  Its normed values are normal: the largest of all rows is below 5.5
    # sigma, 5.5 / 127 / sqrt(12) = 1.25 %, which gate times up doubles.  Products of two such have larger ones, up to 20 sigma: 4.6 %.
    # With two 16-bit roundings of 0.4 % below 8 % if all of it added up.
    off = (out.double() - want).norm(dim=1) / want.norm(dim=1)
    assert (off < 0.08).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_block_weights_as_they_are(monkeypatch, scoring):
    from ops_transformer_b200 import block as module
    seen, kept = {}, {}
    monkeypatch.setattr(module, "route_top_k", lambda logits, k, _f=module.route_top_k, **kw: seen.setdefault("r", (logits, *_f(logits, k, **kw)))[1:])
    monkeypatch.setattr(module, "format_cast_nz", lambda w, _f=module.format_cast_nz: _f(kept.setdefault("w_down", w)))
    b = random_block(512, 256, 8, 2, scoring=scoring, routed_scale=1.5, renormalize=False)
    x, residual = (torch.randn(50, 512, device=DEV, generator=torch.Generator(DEV).manual_seed(i)).to(torch.bfloat16) for i in (1, 2))
    out, _ = b(x, residual)
    logits, weights, ids = seen["r"]
    scores = (torch.softmax(logits.double(), 1) if scoring == "softmax" else torch.sigmoid(logits.double())).gather(1, ids.long())
    assert torch.allclose(weights.double(), 1.5 * scores, rtol=1e-5, atol=0)
    want = reference(b, x, residual, ids, 1.5 * scores, None, kept)
    assert ((out.double() - want).norm(dim=1) / want.norm(dim=1) < 0.08).all()   # as in test_block_row_by_row
