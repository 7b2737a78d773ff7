"""A mixture-of-experts block of a quantised decoder layer on one GPU, from the residual stream to the sum of the experts:

  1. ``add_rms_norm_quant``: residual sum, int8 rows with per-token scales for every W8A8 operator, 16-bit rows for the router
  2. router projection (a matrix product of torch) and ``route_top_k``
  3. ``moe_init_routing_v3``: the int8 rows and their scales grouped by expert, without another quantisation
  4. ``grouped_matmul_swiglu_quant`` over the experts' rows, and over all rows for the shared expert
  5. ``quant_matmul``: the shared expert's down projection, with ``adapter_add`` for the requests that bring an adapter to it
  6. ``grouped_matmul_finalize_routing``: the experts' down projection, weighted and added onto the shared expert's rows
  7. where the next block's weights are at hand, ``sandwich_norm_quant``: what this block puts out, through its own norm, gate and residual
     sum, into the int8 rows that the next one begins with at step 3
  8. on request, ``expert_balance``: how the step's tokens load the experts, and the loss that evens them out

Nothing is read back to the host, so a step can be captured in a CUDA graph; padded rows of such a batch are named by ``token_mask``.
``python -m ops_transformer_b200.block`` runs a small one.
"""
from __future__ import annotations

import dataclasses
from typing import NamedTuple, Optional

import torch

from .acl import (adapter_add, add_rms_norm_quant, expert_balance, expert_balance_grad, format_cast_nz, grouped_matmul_finalize_routing,
                  grouped_matmul_swiglu_quant, moe_init_routing_v3, quant_matmul, route_top_k, sandwich_norm_quant)


@dataclasses.dataclass
class Adapters:
    """Low-rank adapters of the shared expert's down projection: a [adapters, rank, inter], b [adapters, hidden, rank] in the type of the
    hidden states, scaling fp32 [adapters] (1 without it)."""
    a: torch.Tensor
    b: torch.Tensor
    scaling: Optional[torch.Tensor] = None


class Entered(NamedTuple):
    """What a block begins with once its norm is done: int8 rows, their scales, the residual stream and the rows in 16 bits."""
    rows: torch.Tensor
    scales: torch.Tensor
    stream: torch.Tensor
    normed: torch.Tensor


class Load(tuple):
    """(loss, counts, weight) of ``expert_balance`` for the tokens of one call of a block, with what the gradient takes beside them.  ``loss`` is a
    number without an autograd history; what trains the router is ``load.logits.backward(load.grad())``, whose logits have one if the block's
    router requires gradients."""

    def __new__(cls, result, logits, scoring, token_mask):
        self = super().__new__(cls, result)
        self.logits, self.scoring, self.token_mask = logits, scoring, token_mask
        return self

    loss, counts, weight = (property(lambda self, i=i: self[i]) for i in range(3))

    def grad(self, grad_loss=None):
        """The gradient of ``loss``, times ``grad_loss`` (one fp32 number on the device), with respect to ``logits``."""
        return expert_balance_grad(self.logits, self.counts, self.weight, scoring=self.scoring, token_mask=self.token_mask, grad_loss=grad_loss)


@dataclasses.dataclass
class BlockExit:
    """The way from a block's output into the next block: ``gamma`` of the next block's norm, and the optional parts of
    ``sandwich_norm_quant`` that the model has (the block's own norm, its gate, the scales of the residual sum, the scales that the next block's
    int8 weights were smoothed with)."""
    gamma: torch.Tensor
    post_gamma: Optional[torch.Tensor] = None
    gate: Optional[torch.Tensor] = None
    gate_act: str = "none"
    residual_scale: float = 1.0
    block_scale: float = 1.0
    eps: float = 1e-6
    post_eps: Optional[float] = None
    smooth: Optional[torch.Tensor] = None

    def __call__(self, out, stream) -> Entered:
        return Entered(*sandwich_norm_quant(out, stream, self.gamma, post_gamma=self.post_gamma, gate=self.gate, gate_act=self.gate_act,
                                            residual_scale=self.residual_scale, block_scale=self.block_scale, eps=self.eps,
                                            post_eps=self.post_eps, smooth=self.smooth, normed=True))


class QuantMoeBlock:
    """Weights of the experts: w_gate_up int8 [E, hidden, 2 * inter], w_down int8 [E, inter, hidden], scales fp32 per channel; of the shared
    expert: the same with E = 1.  ``router`` bf16 [E, hidden], ``router_bias`` fp32 [E] or None.  Hidden states are bf16.  Without
    ``renormalize`` the chosen experts' weights are their scores as they are (times ``routed_scale``)."""

    def __init__(self, gamma, router, w_gate_up, s_gate_up, w_down, s_down, shared_gate_up, shared_s_gate_up, shared_down, shared_s_down, *,
                 top_k: int, router_bias=None, scoring: str = "softmax", n_group: int = 1, topk_group: int = 1, group_score: str = "max",
                 routed_scale: float = 1.0, renormalize: bool = True, eps: float = 1e-6, adapters: Optional[Adapters] = None):
        self.gamma, self.router, self.router_bias = gamma, router.t(), router_bias
        self.w_gate_up, self.s_gate_up = w_gate_up, s_gate_up
        self.w_down, self.s_down = format_cast_nz(w_down), s_down      # the layout that the combining operator takes
        self.shared = shared_gate_up, shared_s_gate_up, shared_down, shared_s_down
        self.experts, self.top_k = router.shape[0], top_k
        self.routing = dict(scoring=scoring, n_group=n_group, topk_group=topk_group, group_score=group_score, scale=routed_scale,
                            renormalize=renormalize)
        self.eps, self.adapters = eps, adapters

    def __call__(self, x, residual=None, *, adapter_ids=None, token_mask=None, leave: Optional[BlockExit] = None,
                 balance: Optional[float] = None):
        """(the block's output fp32 [tokens, hidden], the new residual stream) for the layer's hidden states ``x`` and ``residual``; without a
        residual the stream is ``x`` itself, as in a model's first layer.  ``x`` may be what the block before left as ``Entered``, without a
        residual; with ``leave`` that is what this one returns for the next, in the place of the two.  ``adapter_ids`` (int32 [tokens]): the
        adapter of every token, negative for none.  ``token_mask``: rows without a token, which take part in no expert.  With ``balance``, a
        coefficient, the load of the experts follows: ``expert_balance``'s (loss, counts, weight) as a ``Load``."""
        if isinstance(x, Entered):
            if residual is not None:
                raise ValueError("rows that have entered the block bring their residual stream")
            rows, scales, stream, normed = x
        else:
            rows, scales, stream, normed = add_rms_norm_quant(x, self.gamma, residual=residual, eps=self.eps, normed=True)
            if residual is None:
                stream = x
        tokens, E = rows.shape[0], self.experts
        logits = normed @ self.router
        weights, ids = route_top_k(logits, self.top_k, bias=self.router_bias, token_mask=token_mask, **self.routing)

        pairs = tokens * self.top_k
        # pairs without an expert leave rows behind, which must name a pair all the same
        outs = (rows.new_empty((pairs, rows.shape[1])), ids.new_zeros(pairs), ids.new_empty(E, dtype=torch.int64), scales.new_empty(pairs))
        ex, pair_of_row, counts, ex_scales = moe_init_routing_v3(rows, ids, expert_num=E, active_expert_range=(0, E), quant_mode=-1, scale=scales,
                                                                 outputs=outs)
        pair_of_row = pair_of_row.long()
        act, act_scales = grouped_matmul_swiglu_quant(ex, self.w_gate_up, self.s_gate_up, ex_scales, counts.cumsum(0))

        gate_up, s_gate_up, down, s_down = self.shared
        every = torch.full((1,), tokens, dtype=torch.int64, device=rows.device)
        shared_act, shared_scales = grouped_matmul_swiglu_quant(rows, gate_up, s_gate_up, scales, every)
        shared = quant_matmul(shared_act, down[0], s_down[0], shared_scales)
        if self.adapters is not None and adapter_ids is not None:
            adapter_add(shared, shared_act, self.adapters.a, self.adapters.b, adapter_ids, x_scale=shared_scales, scaling=self.adapters.scaling,
                        out=shared)
        out = grouped_matmul_finalize_routing(act, self.w_down, self.s_down, counts, pair_of_row // self.top_k, tokens, pertoken_scale=act_scales,
                                              logit=weights.view(-1)[pair_of_row], shared_input=shared)
        result = (out, stream) if leave is None else leave(out, stream)
        if balance is None:
            return result
        scoring = self.routing["scoring"]
        load = Load(expert_balance(logits, ids, scoring=scoring, coefficient=balance, token_mask=token_mask), logits, scoring, token_mask)
        return (*result, load) if leave is None else (result, load)


def random_block(hidden: int, inter: int, experts: int, top_k: int, *, adapters: int = 0, rank: int = 16, seed: int = 0, device="cuda", **routing):
    """A block with random weights whose outputs are of order one."""
    g = torch.Generator(device).manual_seed(seed)
    int8 = lambda *s: (torch.randn(s, device=device, generator=g) * 32).round().clamp(-127, 127).to(torch.int8)  # noqa: E731
    scale = lambda e, n, k: (torch.rand(e, n, device=device, generator=g) * 0.5 + 0.75) / (32 * k ** 0.5)          # noqa: E731
    normal = lambda s, by: (torch.randn(s, device=device, generator=g) * by).to(torch.bfloat16)                    # noqa: E731
    weights = []
    for e in (experts, 1):
        weights += [int8(e, hidden, 2 * inter), scale(e, 2 * inter, hidden), int8(e, inter, hidden), scale(e, hidden, inter)]
    own = Adapters(normal((adapters, rank, inter), inter ** -0.5), normal((adapters, hidden, rank), rank ** -0.5),
                   torch.rand(adapters, device=device, generator=g) + 0.5) if adapters else None
    return QuantMoeBlock(normal((hidden,), 0.1) + 1, normal((experts, hidden), hidden ** -0.5), *weights, top_k=top_k, adapters=own, **routing)


def main():
    tokens, hidden, adapters = 128, 2048, 8
    first, second = (random_block(hidden, 768, 64, 8, adapters=adapters, scoring="sigmoid", n_group=8, topk_group=4, group_score="top2",
                                  router_bias=torch.zeros(64, device="cuda"), routed_scale=2.5, seed=seed) for seed in (0, 1))
    between = BlockExit(second.gamma, post_gamma=torch.ones_like(second.gamma))
    g = torch.Generator("cuda").manual_seed(1)
    x, residual = (torch.randn(tokens, hidden, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    adapter_ids = (torch.arange(tokens, device="cuda") % (adapters + 1) - 1).to(torch.int32)
    mask = torch.arange(tokens, device="cuda") < 120

    def step():
        entered, load = first(x, residual, adapter_ids=adapter_ids, token_mask=mask, leave=between, balance=0.01)
        return *second(entered, adapter_ids=adapter_ids, token_mask=mask), load

    step()
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, stream, (loss, counts, _) = step()
    for _ in range(3):
        graph.replay()
    start.record()
    for _ in range(20):
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    print(f"two blocks, {tokens} tokens of {hidden}, 64 experts (top 8) and {adapters} adapters: {start.elapsed_time(end) / 20 * 1e3:.1f} us a step, "
          f"rms of the output {out.square().mean().sqrt().item():.3f}, finite {bool(out.isfinite().all())}, "
          f"busiest expert of the first {int(counts.max())} of {int(counts.sum())} choices, balance loss {loss.item():.4f}")


if __name__ == "__main__":
    main()
