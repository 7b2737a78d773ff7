"""The mixture-of-experts block as a model's layers call it: the first one, the way from one into the next, the load of its experts in training."""
import pytest
import torch

import ops_transformer_b200 as ops
from ops_transformer_b200.block import BlockExit, random_block

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32
U32 = 2.0 ** -24


def randn(shape, seed, dtype=F32, scale=1.0):
    return (torch.randn(shape, device=DEV, generator=torch.Generator(DEV).manual_seed(seed)) * scale).to(dtype)


def near(a, b, tokens_hidden):
    """Outputs of two runs: rows are added up in no fixed order, a few units of fp32 of the partial sums, which are about sqrt(hidden)."""
    return (a - b).abs().max() < 64 * U32 * tokens_hidden ** 0.5


@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_first_block_has_no_residual(tokens):
    """Hidden states that nothing is added to are the residual stream, and go on into the next block as such."""
    first, second = (random_block(512, 256, 8, 2, seed=s) for s in (0, 1))
    x = randn((tokens, 512), 1, BF16)
    want, want_stream = first(x, torch.zeros_like(x))
    out, stream = first(x)
    assert torch.equal(want_stream, x) and torch.equal(stream, x) and near(out, want, 512)
    leave = BlockExit(second.gamma, post_gamma=randn((512,), 2, BF16, 0.1) + 1)
    entered = first(x, leave=leave)
    # the stream holds the first block's output behind its norm, rounded once: two runs of that output differ as above, by a 2^-16th of a row's largest
    other = leave(want, x)
    assert ((entered.stream.double() - other.stream.double()).abs() <= other.stream.double().abs() * 2.0 ** -7 + 2.0 ** -15 * other.stream.double().abs().amax(1, keepdim=True)).all()
    out, stream = second(entered)
    assert torch.equal(stream, entered.stream) and out.isfinite().all()


@pytest.mark.parametrize("tokens", [3, 300])
def test_way_into_a_block_with_smoothed_weights(tokens):
    """The smoothing scales multiply what is quantised, and neither the stream nor the rows that the router reads."""
    first, second = (random_block(512, 256, 8, 2, seed=s) for s in (0, 1))
    x, residual = randn((tokens, 512), 1, BF16), randn((tokens, 512), 2, BF16)
    out, stream = first(x, residual)
    smooth = 2.0 ** torch.randint(-1, 2, (512,), device=DEV, generator=torch.Generator(DEV).manual_seed(3)).float()
    plain, smoothed = BlockExit(second.gamma)(out, stream), BlockExit(second.gamma, smooth=smooth)(out, stream)
    assert torch.equal(plain.stream, smoothed.stream) and torch.equal(plain.normed, smoothed.normed)
    s = 1.0 * stream.double() + out.double()
    u = s * (s.square().mean(1, keepdim=True) + 1e-6).rsqrt() * second.gamma.double() * smooth.double()
    top = u.abs().amax(1, keepdim=True)
    # half a step of 127, and a hundred units of fp32 for the norm (512 / 32 + 16 additions) and its products
    assert ((smoothed.rows * smoothed.scales.double()[:, None] - u).abs() <= top / 127 * 0.5 + top * 100 * U32).all()
    assert not torch.equal(plain.rows, smoothed.rows)
    assert second(smoothed)[1] is smoothed.stream


@pytest.mark.parametrize("tokens,scoring", [(1, "softmax"), (50, "sigmoid"), (700, "softmax")])
@pytest.mark.parametrize("last", [True, False])
def test_a_router_is_trained_by_the_load_of_its_block(tokens, scoring, last):
    """The block hands out what the balance loss is differentiated with: the router's gradient is the formula's."""
    block, after = (random_block(512, 256, 16, 2, seed=s, scoring=scoring) for s in (0, 1))
    router = block.router.t().detach().clone().requires_grad_(True)
    block.router = router.t()
    x, residual = randn((tokens, 512), 1, BF16), randn((tokens, 512), 2, BF16)
    mask = torch.arange(tokens, device=DEV) % 4 != 3
    *_, load = block(x, residual, token_mask=mask, balance=0.01, leave=None if last else BlockExit(after.gamma))
    loss, counts, weight = load
    assert loss is load.loss and counts is load.counts and weight is load.weight and not loss.requires_grad
    scale = torch.tensor(1000.0, device=DEV)
    grad = load.grad(scale)
    load.logits.backward(grad)

    normed = ops.add_rms_norm_quant(x, block.gamma, residual=residual, normed=True)[3]
    logits = load.logits.detach().double().requires_grad_(True)
    assert torch.equal(load.logits, normed @ block.router)
    p = logits.softmax(1) if scoring == "softmax" else logits.sigmoid() / logits.sigmoid().sum(1, keepdim=True)
    n = int(mask.sum())
    want = 0.01 * 16 / (2 * n * n) * (counts * (p * mask[:, None]).sum(0)).sum()
    (1000.0 * want).backward()
    # p's errors are some units of fp32 (logits of about 3), a sum over `tokens` of them
    assert abs(loss.item() - want.item()) <= want.item() * (tokens + 100) * U32
    # every element within half a unit of bf16 of its own, and some units of fp32 of the largest of its row's products before they cancel
    size = (p * 0.01 * 16 / (2 * n * n) * counts.max() * 1000).detach()
    assert ((grad.double() - logits.grad).abs() <= logits.grad.abs() * 2.0 ** -8 + size * 100 * U32).all()
    # the product with `normed` in bf16, fp32 sums of up to 700 terms, one rounding
    want_router = grad.double().t() @ normed.double()
    assert (router.grad.double() - want_router).norm() <= want_router.norm() * 2.0 ** -7
    assert (grad[~mask] == 0).all()


def test_load_of_a_captured_block():
    """Loss, counts and gradient of a replay are those of its inputs."""
    block = random_block(512, 256, 16, 2)
    x, residual = randn((24, 512), 1, BF16), randn((24, 512), 2, BF16)
    mask = torch.arange(24, device=DEV) < 20

    def step():
        out, stream, load = block(x, residual, token_mask=mask, balance=0.01)
        return (*load, load.grad())
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (3, 4):
        x.copy_(randn((24, 512), seed, BF16))
        mask[:seed] = False
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
