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


def sandwich_inputs(rows, h, x_dtype=F32, dtype=BF16):
    return dict(x=randn((rows, h), 1, x_dtype, 3.0), residual=randn((rows, h), 2, dtype), gamma=randn((h,), 3, dtype, 0.2) + 1)


def right_or_nan(got, want):
    """Whether every element is the right one, or NaN."""
    return ((got == want) | got.isnan()).all()


SANDWICH_WAITS = [(4096, 7168, F32, BF16, dict(post_gamma=True, gate="channel", normed=True)), (3000, 5001, F32, F16, dict(post_gamma=True, normed=True)),
                  (4000, 2100, BF16, BF16, dict(gate="full", normed=True)), (600, 9000, F32, F32, dict(post_gamma=True, gate="token")),
                  (600, 7000, F32, F32, dict(post_gamma=True, gate="token")),
                  (2500, 7168, F16, F16, dict(post_gamma=True, smooth=True)), (2000, 6000, F32, BF16, dict(stream_only=True)),
                  (2000, 6001, BF16, BF16, dict(stream_only=True, post_gamma=True))]


def in_turn(h, dtype):
    """Whether rows of that length fit a group of threads with two packs each, as the kernel with waits takes them: up to 1024 threads.  (9000 values
    of fp32 are 2250 packs, for 1125.)"""
    v = 16 // dtype.itemsize
    packs = h // v if h % v == 0 else (h + 2 * v - 2) // v
    return (packs + 1) // 2 <= 1024


def sandwich_call(rows, h, x_dtype, dtype, how):
    t = sandwich_inputs(rows, h, x_dtype, dtype)
    kw = dict(normed=how.get("normed", False))
    if how.get("post_gamma"):
        kw["post_gamma"] = randn((h,), 4, dtype, 0.2) + 0.7
    if "gate" in how:
        kw["gate"] = randn({"channel": (h,), "token": (rows, 1), "full": (rows, h)}[how["gate"]], 5, dtype)
        kw["gate_act"] = "sigmoid"
    if how.get("smooth"):
        kw["smooth"] = torch.rand(h, device=DEV, generator=gen(6)) + 0.5
    if how.get("stream_only"):
        kw["quant"] = False
        t["gamma"] = None
    return lambda **more: ops.sandwich_norm_quant(**t, **kw, **more)


@pytest.mark.parametrize("rows,h,x_dtype,dtype,how", SANDWICH_WAITS)
def test_sandwich_reports_a_wait_that_runs_out(rows, h, x_dtype, dtype, how):
    """Rows at the end are not fetched and waits last about 1 ms: the call ends, says so, and what it could not work on is NaN through and through;
    the next one on the same workspace is right."""
    call = sandwich_call(rows, h, x_dtype, dtype, how)
    want = call()
    for skip in (1, rows // 2, rows):
        for fill in (0, 255):
            mine = torch.full((256,), fill, dtype=torch.uint8, device=DEV)
            *got, ws = call(workspace=mine, return_workspace=True, options=ops.LaunchOptions(wait_limit_cycles=2_000_000, test_skip_k_blocks=skip))
            assert ws is mine
            if not in_turn(h, dtype):
                ops.check_status(mine)
                assert all(a is b if a is None else torch.equal(a, b) for a, b in zip(got, want))
                continue
            with pytest.raises(ops.AclnnError) as info:
                ops.check_status(mine)
            code, cta, role, parity = info.value.record
            assert code == 1 and 0 <= cta < 148 and role in (1000, 1001) and parity in (0, 1)
            q, scale, stream, normed = got
            lost = stream.isnan().all(1)
            assert lost[rows - skip:].all() and torch.equal(stream[~lost], want[2][~lost])
            if scale is not None:
                assert scale[lost].isnan().all() and (q[lost] == 0).all()
                assert torch.equal(scale[~lost], want[1][~lost]) and torch.equal(q[~lost], want[0][~lost])
            if normed is not None:
                assert normed[lost].isnan().all() and torch.equal(normed[~lost], want[3][~lost])
            *again, ws = call(workspace=mine, return_workspace=True)
            ops.check_status(ws)
            assert all(a is b if a is None else torch.equal(a, b) for a, b in zip(again, want))


@pytest.mark.parametrize("rows,h,x_dtype,dtype,how", SANDWICH_WAITS)
def test_sandwich_leaves_nothing_under_way_when_a_wait_runs_out(rows, h, x_dtype, dtype, how):
    """Waits that give up while rows are on their way: these land before the kernel ends, and what runs next in its place is right."""
    call = sandwich_call(rows, h, x_dtype, dtype, how)
    want = call()
    mine = torch.empty(256, dtype=torch.uint8, device=DEV)
    for limit in (100, 1000, 3000, 10_000, 100_000):
        got = call(workspace=mine, options=ops.LaunchOptions(wait_limit_cycles=limit))
        again = [call() for _ in range(2)]
        for a in again:
            assert all(x is y if x is None else torch.equal(x, y) for x, y in zip(a, want))
        assert right_or_nan(got[2], want[2])
        if got[3] is not None:
            assert right_or_nan(got[3], want[3])
        if got[1] is not None:
            assert right_or_nan(got[1], want[1]) and ((got[0] == want[0]) | (got[0] == 0)).all()
        try:
            ops.check_status(mine)
        except ops.AclnnError:
            continue
        assert all(x is y if x is None else torch.equal(x, y) for x, y in zip(got, want))


def test_sandwich_status_of_calls_without_waits():
    """Few rows and rows on no pack have kernels without waits, and a clean record."""
    for rows, h, offset in ((1, 8, 0), (16, 2048, 0), (9, 40000, 0), (700, 1000, 1)):
        t = sandwich_inputs(rows, h)
        t["x"] = randn((rows * h + 8,), 7)[offset:offset + rows * h].view(rows, h)
        for options in (None, ops.LaunchOptions(wait_limit_cycles=1000)):
            mine = torch.full((256,), 255, dtype=torch.uint8, device=DEV)
            *got, ws = ops.sandwich_norm_quant(**t, workspace=mine, return_workspace=True, options=options)
            assert ws is mine
            ops.check_status(ws)
            assert all(a is b if a is None else torch.equal(a, b) for a, b in zip(got, ops.sandwich_norm_quant(**t)))
    t = sandwich_inputs(0, 64)
    assert ops.sandwich_norm_quant(**t, return_workspace=True)[4] is None


# ---------------------------------------------------------------------------------------------------------------------
# launch options
# ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("m,k,n", [(16, 768, 2048), (100, 1000, 640), (4096, 2048, 4096), (3000, 1001, 4096)])
def test_matmul_options_do_not_hang_on_the_size(m, k, n):
    """Events are recorded around the product whatever kernel takes the call, and a cap on the CTAs is followed by none."""
    x, w, scale = int8((m, k), 1), int8((k, n), 2), torch.rand(n, device=DEV, generator=gen(3)) + 0.5
    want = ops.quant_matmul(x, w, scale)
    took = {}
    for cap in (0, 2):
        for _ in range(3):
            start, stop = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()   # creates it; what the two say until they are recorded anew is about 10 ms
            torch.cuda._sleep(20_000_000)
            stop.record()
            torch.cuda.synchronize()
            got = ops.quant_matmul(x, w, scale, options=ops.LaunchOptions(max_ctas=cap, start_event=start.cuda_event, stop_event=stop.cuda_event))
            stop.synchronize()
            took[cap] = min(took.get(cap, 1e9), start.elapsed_time(stop))
            assert torch.equal(got, want)
    assert 0 < took[0] < 1 and took[2] < 4 * took[0] + 0.01   # two CTAs of 148 would take 70 times as long for the large ones


# ---------------------------------------------------------------------------------------------------------------------
# scales and biases that leave the result's type, element by element
# ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,k,n", [(4, 65535, 64), (40, 2048, 512), (3, 100, 77), (1500, 1536, 4096)])
@pytest.mark.parametrize("special", ["scale", "token", "bias", "all"])
def test_matmul_extreme_scales_element_by_element(m, k, n, dtype, special):
    """Overflow, infinities, NaN and zeros in scales and bias: every element as the same steps in fp32 give it, with its sign."""
    x, w = int8((m, k), 1), int8((k, n), 2)
    x[0], w[:, 0] = -128, -128
    x[1], w[:, 1] = 127, 127
    scale, token, bias = torch.ones(n, device=DEV), torch.ones(m, device=DEV), torch.zeros(n, device=DEV)
    odd = torch.tensor([float("inf"), -float("inf"), float("nan"), 0.0, -0.0, 1e38, -3e38, 1e-38], device=DEV)
    if special in ("scale", "all"):
        scale[:64] = odd.repeat(8)
    if special in ("token", "all"):
        token[:min(m, 8)] = odd[:min(m, 8)]
    if special in ("bias", "all"):
        bias[8:72 if n >= 72 else n] = odd.repeat(8)[:min(64, n - 8)]
    got = ops.quant_matmul(x, w, scale, token, bias=bias, out_dtype=dtype)
    want = ((x.double() @ w.double()).float() * scale * token[:, None] + bias).to(dtype)
    torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)
    if special == "scale":   # the same without what the calls need not have
        torch.testing.assert_close(ops.quant_matmul(x, w, scale, out_dtype=dtype), ((x.double() @ w.double()).float() * scale).to(dtype), rtol=0, atol=0, equal_nan=True)


# ---------------------------------------------------------------------------------------------------------------------
# adapter_add: limits that are shorter than what is under way takes
# ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("is_int8", [False, True])
@pytest.mark.parametrize("tokens,adapters,k,n,rank", [(300, 2, 4096, 4096, 16), (300, 60, 2048, 520, 16), (2100, 2, 512, 3000, 64), (300, 2, 1001, 3001, 61)])
def test_adapter_leaves_nothing_under_way_when_a_wait_runs_out(tokens, adapters, k, n, rank, is_int8):
    """The kernels end only when their products have, and what runs next in the same tensor memory is right."""
    base, a, b = randn((tokens, n), 1, BF16), randn((adapters, rank, k), 2, BF16, k ** -0.5), randn((adapters, n, rank), 3, BF16, rank ** -0.5)
    x = int8((tokens, k), 4) if is_int8 else randn((tokens, k), 4, BF16)
    kw = dict(x_scale=torch.rand(tokens, device=DEV, generator=gen(5)) / 64 if is_int8 else None)
    ids = (torch.arange(tokens, device=DEV) % adapters).to(I32)
    want, ws = ops.adapter_add(base, x, a, b, ids, return_workspace=True, **kw)
    ops.check_status(ws)
    mine = torch.zeros(ws.numel(), dtype=torch.uint8, device=DEV)
    for limit in (100, 1000, 3000, 10_000, 100_000):
        got = ops.adapter_add(base, x, a, b, ids, workspace=mine, options=ops.LaunchOptions(wait_limit_cycles=limit), **kw)
        again = [ops.adapter_add(base, x, a, b, ids, **kw) for _ in range(2)]
        assert all(torch.equal(t, want) for t in again)
        try:
            ops.check_status(mine)
        except ops.AclnnError as error:
            assert error.record[0] == 1
            continue
        assert torch.equal(got, want)
