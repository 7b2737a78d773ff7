"""The operators of a block's exit where kernels wait: for other CTAs of a cluster, for copies that do not come, beside other work on the GPU."""
import pytest
import torch

import ops_transformer_b200 as ops

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F16, F32, I8, I32, I64 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.int32, torch.int64


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def randn(shape, seed, dtype=F32, scale=1.0):
    return (torch.randn(shape, device=DEV, generator=gen(seed)) * scale).to(dtype)


# ---------------------------------------------------------------------------------------------------------------------
# expert_balance: the cluster whose CTAs send one another their parts of the loss
# ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,experts,sequences", [(3000, 64, None), (700, 256, 1), (900, 40, 7), (2000, 1000, 32), (40, 1024, 16)])
def test_balance_clusters_beside_other_work(rows, experts, sequences):
    """Calls among products of another stream, whose CTAs keep the SMs busy while those of a cluster come: the same bits each time, and the loss
    that the counts and the scores' sums give."""
    logits = randn((rows, experts), 1)
    ids = (logits + randn((experts,), 2)).topk(4, 1).indices
    cu = None if sequences is None else torch.linspace(0, rows, sequences + 1, device=DEV).to(I32)
    first = ops.expert_balance(logits, ids, cu_seqlens=cu)
    bounds = [0, rows] if cu is None else cu.tolist()
    p, want = logits.double().softmax(1), 0.0
    for a, b in zip(bounds[:-1], bounds[1:]):
        want += experts / (4 * (b - a) ** 2) * (torch.bincount(ids[a:b].flatten(), minlength=experts) * p[a:b].sum(0)).sum().item() / (len(bounds) - 1)
    # a score: its exponent's argument and size (logits within 10), the row's sum of E / 32 + 5 steps; over tokens at most rows / 148 + 80 additions
    assert abs(first[0].item() - want) <= want * (10 + experts / 32 + 12 + rows / 148 + 80) * 2.0 ** -24
    a = randn((2048, 2048), 3, BF16)
    torch.cuda.synchronize()
    busy, side = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(30):
        with torch.cuda.stream(busy):
            b = a @ a
        with torch.cuda.stream(side):
            got += [ops.expert_balance(logits, ids, cu_seqlens=cu) for _ in range(3)]
    torch.cuda.synchronize()
    assert b.isfinite().all()
    for again in got:
        assert all(torch.equal(x, y) for x, y in zip(again, first))


# ---------------------------------------------------------------------------------------------------------------------
# waits that run out
# ---------------------------------------------------------------------------------------------------------------------

def int8(shape, seed):
    return torch.randint(-128, 128, shape, device=DEV, generator=gen(seed)).to(I8)


@pytest.mark.parametrize("m,k,n", [(16, 4096, 2048), (256, 512, 18944), (3, 100, 77)])
def test_matmul_records_of_limited_waits(m, k, n):
    """A workspace that holds anything, a limit of the caller's: the record is that of this call, whatever order its CTAs come in."""
    x, w, scale = int8((m, k), 1), int8((k, n), 2), torch.rand(n, device=DEV, generator=gen(3)) + 0.5
    want, ws = ops.quant_matmul(x, w, scale, return_workspace=True)
    for fill in (0, 1, 2, 255):
        mine = torch.full((ws.numel(),), fill, dtype=torch.uint8, device=DEV)
        ops.quant_matmul(x, w, scale, workspace=mine, options=ops.LaunchOptions(wait_limit_cycles=2_000_000, test_skip_k_blocks=1))
        with pytest.raises(ops.AclnnError) as info:
            ops.check_status(mine)
        code, cta, role, parity = info.value.record
        assert code == 1 and cta >= 0 and 200 <= role < 500 and parity in (0, 1)
        got = ops.quant_matmul(x, w, scale, workspace=mine, options=ops.LaunchOptions(wait_limit_cycles=1 << 31))
        ops.check_status(mine)
        assert torch.equal(got, want)


@pytest.mark.parametrize("m,k,n,nk", [(16, 7168, 4096, True), (64, 4096, 512, False), (256, 7168, 1024, True), (300, 1000, 640, False), (5, 128, 100, True)])
def test_matmul_leaves_nothing_under_way_when_a_wait_runs_out(m, k, n, nk):
    """Waits that give up while copies, products and sums of other CTAs are still on their way: the kernel ends only when these have landed, and what
    runs next, in the same places of the GPU, is right.  With K blocks left out the call says that it failed; rows that it does not finish stay."""
    x, scale, token = int8((m, k), 1), torch.rand(n, device=DEV, generator=gen(3)) + 0.5, torch.rand(m, device=DEV, generator=gen(4)) + 0.5
    w = int8((n, k), 2).t() if nk else int8((k, n), 2)
    want = (x.double() @ w.double()).float() * scale * token[:, None]
    got, ws = ops.quant_matmul(x, w, scale, token, out_dtype=F32, return_workspace=True)
    ops.check_status(ws)
    assert torch.equal(got, want)
    mine = torch.zeros(ws.numel(), dtype=torch.uint8, device=DEV)
    for limit in (100, 1000, 3000, 10_000, 100_000):
        for skip in (0, 1):
            room = torch.full((m, n), 7.0, device=DEV)
            ops.quant_matmul(x, w, scale, token, out=room, workspace=mine, options=ops.LaunchOptions(wait_limit_cycles=limit, test_skip_k_blocks=skip))
            again = [ops.quant_matmul(x, w, scale, token, out_dtype=F32) for _ in range(3)]
            assert all(torch.equal(a, want) for a in again)
            if skip:
                with pytest.raises(ops.AclnnError) as info:
                    ops.check_status(mine)
                assert info.value.record[0] == 1
                assert (room == 7).all()   # every CTA misses a block of its own
            else:
                try:
                    ops.check_status(mine)
                except ops.AclnnError:
                    continue
                assert torch.equal(room, want)
