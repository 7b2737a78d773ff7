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
