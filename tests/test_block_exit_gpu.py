"""quant_matmul, sandwich_norm_quant, expert_balance and its gradient on the GPU against plain implementations in 64 bits (and in fp32 where a
result has to be bit-identical), at the sizes, strides, masks and special values where they can go wrong.

Tolerances come from the operators' arithmetic: u = 2^-24 is half a unit in the last place of fp32, and a result in a 16-bit type may
be off by half of one of its own units."""
import math

import pytest
import torch

import ops_transformer_b200 as ops

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U32 = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # of 24, 11 and 8 significant bits
TINY = {torch.float32: 1e-38, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-38}   # half a subnormal step, or nothing
BF16, F16, F32, I8, I32, I64 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.int32, torch.int64


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def randn(shape, seed, dtype=F32, scale=1.0):
    return (torch.randn(shape, device=DEV, generator=gen(seed)) * scale).to(dtype)


def rand(shape, seed):
    return torch.rand(shape, device=DEV, generator=gen(seed))


def int8(shape, seed, lo=-128, hi=128):
    return torch.randint(lo, hi, shape, device=DEV, generator=gen(seed)).to(I8)


# ---------------------------------------------------------------------------------------------------------------------
# quant_matmul: every step is an exact sum or one rounding, so results are bit-identical to the same steps in torch
# ---------------------------------------------------------------------------------------------------------------------

def plain_matmul(x, w, scale, token, bias, dtype):
    acc = x.double() @ w.double()   # exact: below 2^53
    y = acc.float() * scale.float()
    if token is not None:
        y = y * token[:, None]
    if bias is not None:
        y = y + bias.float()
    return y.to(dtype)


def check_matmul(m, k, n, nk=False, dtype=BF16, bias=None, scale_dtype=F32, token=True, seed=0):
    x = int8((m, k), seed + 1)
    w = int8((n, k), seed + 2).t() if nk else int8((k, n), seed + 2)
    scale = ((rand((n,), seed + 3) + 0.5) / 1024).to(scale_dtype)
    per_token = (rand((m,), seed + 4) + 0.5) / 16 if token else None
    b = randn((n,), seed + 5, bias) if bias else None
    got = ops.quant_matmul(x, w, scale, per_token, bias=b, out_dtype=dtype)
    assert got.shape == (m, n) and got.dtype == dtype
    assert torch.equal(got, plain_matmul(x, w, scale, per_token, b, dtype))


MATMUL_SIZES = [(1, 1, 1), (1, 16, 16), (1, 7168, 128), (2, 17, 33), (3, 128, 129), (5, 127, 255), (16, 768, 2048), (16, 2048, 160), (31, 1000, 1008),
                (33, 4096, 384), (64, 512, 1536), (65, 2048, 2064), (100, 144, 7000), (128, 640, 129), (129, 1423, 300), (200, 16, 2000), (257, 1424, 2976),
                (611, 1423, 2977), (700, 300, 512), (1025, 2048, 1040), (2000, 1000, 1999)]


@pytest.mark.parametrize("nk", [False, True])
@pytest.mark.parametrize("m,k,n", MATMUL_SIZES)
def test_matmul_sizes(m, k, n, nk):
    check_matmul(m, k, n, nk)
    check_matmul(m, k, n, nk, dtype=F32, bias=F32, token=False, seed=10)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("bias", [None, F32, BF16, F16])
@pytest.mark.parametrize("m,k,n", [(16, 1024, 1024), (7, 100, 77), (1500, 1536, 4096)])
def test_matmul_types(m, k, n, bias, dtype):
    for scale_dtype in (F32, BF16, F16):
        check_matmul(m, k, n, nk=bias is None, dtype=dtype, bias=bias, scale_dtype=scale_dtype)


def test_matmul_large():
    check_matmul(4096, 2048, 4096)
    check_matmul(1, 2048, 129280, nk=True, dtype=F32)     # a head
    check_matmul(70, 512, 100003, dtype=F32)
    check_matmul(70000, 64, 272, nk=True)
    check_matmul(3, 65535, 48)


def test_matmul_extreme_values():
    """The largest sums that 65535 products make stay in int32; scales that leave the result's type."""
    m, k, n = 4, 65535, 64
    x, w = torch.full((m, k), -128, device=DEV, dtype=I8), torch.full((k, n), -128, device=DEV, dtype=I8)
    one = torch.ones(n, device=DEV)
    assert (ops.quant_matmul(x, w, one, out_dtype=F32) == 65535 * 16384).all()
    w[:, 1::2] = 127
    got = ops.quant_matmul(x, w, one, out_dtype=F32)
    assert (got[:, ::2] == 65535.0 * 16384).all() and (got[:, 1::2] == -float(torch.tensor(65535 * 16256).float())).all()
    scale = one.clone()
    scale[:4] = torch.tensor([math.inf, math.nan, 0.0, 1e38], device=DEV)
    got = ops.quant_matmul(x, w, scale, out_dtype=F16)
    assert torch.equal(got, plain_matmul(x, w, scale, None, None, F16)) or (got[:, 0].isinf().all() and got[:, 1].isnan().all() and (got[:, 2] == 0).all() and got[:, 3].isinf().all())
    token = torch.tensor([1.0, math.inf, math.nan, 0.0], device=DEV)
    got = ops.quant_matmul(x, w, one, token, out_dtype=F32)
    assert got[1].isinf().all() and got[2].isnan().all() and (got[3] == 0).all()


def test_matmul_equals_one_group():
    for m, k, n in ((1, 512, 256), (40, 2048, 4096), (300, 1024, 512)):
        x, w = int8((m, k), 1), int8((k, n), 2)
        scale, token = rand((n,), 3) / 256, rand((m,), 4)
        for dtype in (BF16, F16):
            one = ops.grouped_matmul_v4(x, w[None], scale[None], token, torch.full((1,), m, device=DEV, dtype=I64), out_dtype=dtype)
            assert torch.equal(ops.quant_matmul(x, w, scale, token, out_dtype=dtype), one)


@pytest.mark.parametrize("m", [5, 150, 1300])
def test_matmul_strided_operands(m):
    k, n = 400, 528
    scale, token, bias = rand((n,), 1), rand((m,), 2), randn((n,), 3)
    dense_x, dense_w = int8((m, k), 4), int8((k, n), 5)
    want = plain_matmul(dense_x, dense_w, scale, token, bias, BF16)

    def padded(t, left, right):   # the same values inside wider rows
        wide = torch.full((t.shape[0], left + t.shape[1] + right), 77, device=DEV, dtype=t.dtype)
        wide[:, left:left + t.shape[1]] = t
        return wide[:, left:left + t.shape[1]]

    xs = [padded(dense_x, 16, 32), padded(dense_x, 3, 0), padded(dense_x, 0, 5), dense_x.t().contiguous().t(), dense_x.repeat_interleave(2, 1)[:, ::2]]
    ws = [padded(dense_w, 16, 32), padded(dense_w, 1, 2), dense_w.t().contiguous().t(), padded(dense_w.t(), 32, 16).t(), padded(dense_w.t(), 5, 2).t(),
          dense_w.repeat_interleave(2, 1)[:, ::2]]
    for x in xs:
        assert torch.equal(ops.quant_matmul(x, dense_w, scale, token, bias=bias), want)
    for w in ws:
        assert torch.equal(ops.quant_matmul(dense_x, w, scale, token, bias=bias), want)
    assert torch.equal(ops.quant_matmul(xs[1], ws[4], scale, token, bias=bias), want)
    row = torch.ones(1, k, device=DEV, dtype=I8).expand(m, k)
    assert torch.equal(ops.quant_matmul(row, dense_w, scale, token), plain_matmul(row, dense_w, scale, token, None, BF16))
    # results into wider rows, on and off the boundaries of packs, and into columns apart; what lies between stays as it was
    for left, right in ((8, 8), (1, 2), (0, 3)):
        wide = torch.full((m, left + n + right), 5.0, device=DEV, dtype=BF16)
        ops.quant_matmul(dense_x, dense_w, scale, token, bias=bias, out=wide[:, left:left + n])
        assert torch.equal(wide[:, left:left + n], want) and (wide[:, :left] == 5).all() and (wide[:, left + n:] == 5).all()
    apart = torch.full((m, 2 * n), 5.0, device=DEV, dtype=BF16)
    ops.quant_matmul(dense_x, dense_w, scale, token, bias=bias, out=apart[:, ::2])
    assert torch.equal(apart[:, ::2], want) and (apart[:, 1::2] == 5).all()


def test_matmul_no_rows_and_rows_behind():
    assert ops.quant_matmul(int8((0, 64), 1), int8((64, 48), 2), rand((48,), 3)).shape == (0, 48)
    y, ws = ops.quant_matmul(int8((0, 64), 1), int8((64, 48), 2), rand((48,), 3), return_workspace=True)
    assert ws is None
    room = torch.full((70, 256), 9.0, device=DEV, dtype=BF16)
    ops.quant_matmul(int8((33, 128), 1), int8((128, 256), 2), rand((256,), 3), out=room[:33])
    assert (room[33:] == 9).all()


def test_matmul_same_bits_every_time_and_status():
    x, w, scale = int8((77, 3000), 1), int8((3000, 1111), 2), rand((1111,), 3)
    first, ws = ops.quant_matmul(x, w, scale, out_dtype=F32, return_workspace=True)
    ops.check_status(ws)
    for _ in range(5):
        assert torch.equal(ops.quant_matmul(x, w, scale, out_dtype=F32), first)


# ---------------------------------------------------------------------------------------------------------------------
# sandwich_norm_quant
# ---------------------------------------------------------------------------------------------------------------------

def gate_of(gate, act):
    return {"none": lambda g: g, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[act](gate.double())


def check_sandwich(x, residual, gamma, got, *, post_gamma=None, gate=None, gate_act="none", residual_scale=1.0, block_scale=1.0, smooth=None, eps=1e-6,
                   post_eps=None, quant=True, normed=False):
    q, scale, stream, y = got
    dtype, h = residual.dtype, residual.shape[1]
    post_eps = eps if post_eps is None else post_eps
    f32 = lambda v: torch.tensor(v, dtype=F32).item()  # noqa: E731  (numbers travel as fp32)
    # an fp32 sum of h squares by at most h / 32 + 10 steps in a row (each relative u, halved by the root), quotient, root, reciprocal
    rel_r = (h / 32 + 16) * U32
    n = x.double()
    if post_gamma is not None:
        n = n / (n.square().mean(1, keepdim=True) + f32(post_eps)).sqrt() * post_gamma.double()
    if gate is not None:
        n = n * gate_of(gate, gate_act)
    n = n * f32(block_scale)
    s = f32(residual_scale) * residual.double() + n
    # n: the first norm, three products; a gate's exponential and quotient or hyperbolic tangent below 8 units
    rel_n = (rel_r if post_gamma is not None else 0) + (4 + 16) * U32
    off_s = n.abs() * rel_n + s.abs() * U32
    if stream is not None:
        assert stream.dtype == dtype
        assert ((stream.double() - s).abs() <= s.abs() * HALF_ULP[dtype] + off_s * (1 + HALF_ULP[dtype]) + TINY[dtype]).all()
    if gamma is None:
        assert q is None and scale is None and y is None
        return
    r = 1 / (s.square().mean(1, keepdim=True) + f32(eps)).sqrt()
    # the root mean square moves by no more than the 2-norm of what its elements move by
    rel_r2 = rel_r + off_s.norm(dim=1, keepdim=True) / (s.norm(dim=1, keepdim=True) + 1e-30) * 1.01
    g = gamma.double()
    if normed:
        want = s * r * g
        assert ((y.double() - want).abs() <= want.abs() * (HALF_ULP[dtype] * (1 + 1e-3) + rel_r2 + 3 * U32) + off_s * r * g.abs() * 1.01 + TINY[dtype]).all()
    else:
        assert y is None
    if not quant:
        assert q is None and scale is None
        return
    m = smooth.double() if smooth is not None else 1
    z, off_z = s * g * m, (off_s + 3 * U32 * s.abs()) * (g * m).abs() * 1.01
    top = z.abs().amax(1, keepdim=True)
    off_top = off_z.amax(1, keepdim=True)
    exact = (top / 127 * r)[:, 0]
    off_scale = (off_top / 127 * r)[:, 0] + exact * (rel_r2[:, 0] + 4 * U32)
    assert ((scale.double() - exact).abs() <= off_scale * 1.01 + 1e-38).all()
    # every element is the nearest step; the quotient's own error is what its parts make of it
    t = torch.where(top > 0, z / (top / 127), torch.zeros_like(z))
    off_t = torch.where(top > 0, (off_z + z.abs() * (off_top / (top + 1e-300) + 4 * U32)) / (top / 127), torch.zeros_like(z))
    assert ((q.double() - t).abs() <= 0.5 + off_t * 1.01).all()
    assert (q.abs().amax(1) == torch.where(top[:, 0] > 0, 127, 0)).all()


def sandwich_inputs(rows, h, dtype, x_dtype, seed=0):
    return dict(x=randn((rows, h), seed + 1, x_dtype, 3.0), residual=randn((rows, h), seed + 2, dtype), gamma=randn((h,), seed + 3, dtype, 0.2) + 1)


def run_sandwich(x, residual, gamma, **kw):
    got = ops.sandwich_norm_quant(x, residual, gamma, **kw)
    kw.setdefault("normed", False)
    check_sandwich(x, residual, gamma, got, **kw)
    return got


SANDWICH_SIZES = [(1, 1), (1, 8), (3, 7), (5, 16), (2, 255), (17, 256), (4, 1000), (1, 2048), (33, 1423), (150, 2048), (300, 1424), (7, 7168), (700, 7168), (1300, 1423),
                  (3, 8200), (2, 16384), (700, 5001), (2, 20001), (1, 65535), (2, 65528), (640, 9000)]


@pytest.mark.parametrize("dtype,x_dtype", [(BF16, F32), (BF16, BF16), (F16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("rows,h", SANDWICH_SIZES)
def test_sandwich_sizes(rows, h, dtype, x_dtype):
    t = sandwich_inputs(rows, h, dtype, x_dtype)
    post, smooth = randn((h,), 4, dtype, 0.2) + 0.7, rand((h,), 5) + 0.5
    run_sandwich(**t, post_gamma=post, normed=True, eps=1e-5)
    run_sandwich(**t, gate=randn((h,), 6, dtype), smooth=smooth, residual_scale=0.75, block_scale=0.4)
    run_sandwich(**t, post_gamma=post, gate=randn((rows, 1), 7, dtype), gate_act="sigmoid", quant=False, normed=True, post_eps=1e-3)
    run_sandwich(**t, post_gamma=post, gate=randn((rows, h), 8, dtype), gate_act="tanh", smooth=smooth, normed=True, block_scale=-1.5)
    run_sandwich(t["x"], t["residual"], None, post_gamma=post, quant=False)


@pytest.mark.parametrize("dtype,x_dtype", [(BF16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("rows,h", [(149, 7168), (200, 5001), (2500, 2047), (5000, 2048), (7000, 1431), (450, 8200), (150, 16384), (150, 33000)])
def test_sandwich_many_rows(rows, h, dtype, x_dtype):
    """Groups of threads with rows in turn, at every start of a row; what is too long for them."""
    t = sandwich_inputs(rows, h, dtype, x_dtype)
    post, smooth = randn((h,), 4, dtype, 0.2) + 0.7, rand((h,), 5) + 0.5
    run_sandwich(**t, post_gamma=post)
    run_sandwich(**t, gate=randn((h,), 6, dtype), gate_act="tanh", smooth=smooth, normed=True, residual_scale=0.75, block_scale=0.4)
    run_sandwich(**t, post_gamma=post, gate=randn((rows, h), 8, dtype), gate_act="sigmoid", smooth=smooth, normed=True)
    run_sandwich(**t, gate=randn((rows, 1), 7, dtype), quant=False, normed=True)
    run_sandwich(t["x"], t["residual"], None, post_gamma=post, quant=False)
    want = ops.sandwich_norm_quant(**t, post_gamma=post, normed=True)
    for into in ("residual", "x") if x_dtype == dtype else ("residual",):
        mine = {k: v.clone() for k, v in t.items()}
        got = ops.sandwich_norm_quant(**mine, post_gamma=post, normed=True, residual_out=mine[into])
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[2] is mine[into]


@pytest.mark.parametrize("offset,pitch", [(0, 2 * 5000), (8, 5008), (1, 5003), (4, 5004)])
def test_sandwich_many_strided_rows(offset, pitch):
    rows, h = 333, 5000
    wide = lambda seed, dt=BF16: randn((rows * pitch + 64,), seed, dt)[offset:].as_strided((rows, h), (pitch, 1))  # noqa: E731
    x, residual, gate, stream, normed = wide(1, F32), wide(2), wide(3), wide(4), wide(5)
    gamma, post = randn((h + 8,), 3, BF16)[offset:offset + h], randn((h + 8,), 4, BF16)[offset:offset + h]
    room = torch.full((rows * pitch + 64,), 5, dtype=I8, device=DEV)
    q = room[offset:].as_strided((rows, h), (pitch, 1))
    before = [v.as_strided((rows * pitch,), (1,)).clone() for v in (stream, normed)]
    got = ops.sandwich_norm_quant(x, residual, gamma, post_gamma=post, gate=gate, q=q, residual_out=stream, normed_out=normed)
    check_sandwich(x, residual, gamma, got, post_gamma=post, gate=gate, normed=True)
    gap = torch.arange(rows * pitch, device=DEV) % pitch >= h   # between the rows nothing is written
    for was, now in zip(before, (stream, normed)):
        assert torch.equal(was[gap], now.as_strided((rows * pitch,), (1,))[gap])
    assert (room[offset:offset + rows * pitch][gap] == 5).all() and (room[:offset] == 5).all()


def test_sandwich_many_special_rows():
    for h in (7168, 5003):
        t = sandwich_inputs(400, h, BF16, F32)
        gamma = torch.ones(h, device=DEV, dtype=BF16)
        t["x"][1], t["residual"][1] = 0, 0
        t["x"][2, 5], t["x"][3, h - 1], t["residual"][399, 0] = math.inf, math.nan, -math.inf
        q, scale, stream, y = got = ops.sandwich_norm_quant(t["x"], t["residual"], gamma, post_gamma=gamma, normed=True)
        assert (q[1] == 0).all() and scale[1] == 0 and (y[1] == 0).all() and all(scale[i].isnan() and (q[i] == 0).all() for i in (2, 3, 399))
        good = torch.tensor([0] + list(range(4, 399)), device=DEV)
        check_sandwich(t["x"][good], t["residual"][good], gamma, [v[good] for v in got], post_gamma=gamma, normed=True)


@pytest.mark.parametrize("act", ["none", "sigmoid", "tanh"])
@pytest.mark.parametrize("rows,h", [(6, 520), (400, 1001)])
def test_sandwich_gates(rows, h, act):
    t = sandwich_inputs(rows, h, BF16, F32)
    wide = randn((rows, 2 * h + 3), 9, BF16, 4.0)
    for gate in (wide[0, :h], wide[:1, :h], wide[:, :1], wide[:, 5:6], wide[:, 3:3 + h], wide[:, :2 * h:2], wide[:1, 4:5], randn((h, rows), 3, BF16).t()):
        run_sandwich(**t, post_gamma=t["gamma"], gate=gate, gate_act=act, normed=True)
    # gates that saturate
    gate = randn((h,), 10, BF16, 60.0)
    gate[0], gate[1], gate[2] = 0, 1e4, -1e4
    run_sandwich(**t, gate=gate, gate_act=act)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_sandwich_gammas_in_fp32(dtype):
    for rows, h in ((9, 512), (700, 1000), (4, 333)):
        t = sandwich_inputs(rows, h, dtype, F32)
        t["gamma"] = randn((h,), 6)
        run_sandwich(**t, post_gamma=randn((h,), 7), normed=True)


@pytest.mark.parametrize("offset,pitch", [(0, 2 * 1024), (8, 1024 + 8), (1, 1024 + 3), (4, 1024 + 4)])
@pytest.mark.parametrize("rows", [37, 700])
def test_sandwich_strided_rows_and_offsets(offset, pitch, rows):
    h = 1024
    wide = lambda seed, dt=BF16: randn((rows * pitch + 64,), seed, dt)[offset:].as_strided((rows, h), (pitch, 1))  # noqa: E731
    x, residual, gate = wide(1, F32), wide(2), wide(3)
    gamma, post = randn((h + 8,), 3, BF16)[offset:offset + h], randn((h + 8,), 4, BF16)[offset:offset + h]
    stream, normed = wide(4), wide(5)
    q = torch.zeros(rows * pitch + 64, dtype=I8, device=DEV)[offset:].as_strided((rows, h), (pitch, 1))
    got = ops.sandwich_norm_quant(x, residual, gamma, post_gamma=post, gate=gate, q=q, residual_out=stream, normed_out=normed)
    assert got[0] is q and got[2] is stream and got[3] is normed
    check_sandwich(x, residual, gamma, got, post_gamma=post, gate=gate, normed=True)
    dense = [v.contiguous() for v in (x, residual, gate)]
    for i, v in enumerate((randn((rows, 2 * h), 7, F32)[:, ::2], randn((h, rows), 8, BF16).t(), randn((1, h), 9, BF16).expand(rows, h))):
        args = list(dense)
        args[i] = v
        run_sandwich(args[0], args[1], gamma, post_gamma=post, gate=args[2], normed=True)
    # inputs whose rows are differently far apart
    run_sandwich(dense[0], residual, gamma, post_gamma=post, gate=gate, normed=True)
    run_sandwich(x, dense[1], gamma, post_gamma=post, gate=gate, normed=True)


def test_sandwich_in_place():
    for rows, h, dtype in ((40, 2048, BF16), (3, 40000, BF16), (5, 77, F32), (700, 1423, BF16), (800, 512, F16)):
        t = sandwich_inputs(rows, h, dtype, dtype)
        kw = dict(post_gamma=t["gamma"], gate=randn((rows, h), 5, dtype), gate_act="sigmoid", normed=True)
        want = ops.sandwich_norm_quant(**t, **kw)
        for into in ("residual", "x"):
            a, b = t["x"].clone(), t["residual"].clone()
            got = ops.sandwich_norm_quant(a, b, t["gamma"], residual_out=b if into == "residual" else a, normed_out=a if into == "residual" else None, **kw)
            assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_sandwich_special_rows():
    h = 1040
    for dtype in (BF16, F32):
        for rows in (9, 700):
            t = sandwich_inputs(rows, h, dtype, F32)
            x, residual = t["x"], t["residual"]
            gamma = torch.ones(h, device=DEV, dtype=dtype)
            x[1], residual[1] = 0, 0              # no step to divide by
            x[2, 5] = math.inf
            x[3, h - 1] = math.nan
            residual[4, 7] = math.inf
            x[5] = 0                              # nothing comes out of the block
            residual[6] = 0
            residual[7, 3] = 1e4                  # one value dwarfs the rest
            q, scale, stream, y = got = ops.sandwich_norm_quant(x, residual, gamma, post_gamma=gamma, normed=True)
            assert (q[1] == 0).all() and scale[1] == 0 and (y[1] == 0).all() and (stream[1] == 0).all()
            assert all(scale[i].isnan() and (q[i] == 0).all() for i in (2, 3, 4))
            good = torch.tensor([0, 5, 6, 7] + list(range(8, rows)), device=DEV)
            check_sandwich(x[good], residual[good], gamma, [v[good] for v in got], post_gamma=gamma, normed=True)
            # without the norm behind the block an infinity stays where it is
            stream = ops.sandwich_norm_quant(x, residual, None, quant=False)[2]
            assert stream[2, 5].isinf() and stream[2, :5].isfinite().all() and stream[3, h - 1].isnan() and stream[4, 7].isinf()
    # gammas of zeros
    t = sandwich_inputs(4, 64, BF16, F32)
    q, scale, _, y = ops.sandwich_norm_quant(t["x"], t["residual"], torch.zeros_like(t["gamma"]), normed=True)
    assert (q == 0).all() and (scale == 0).all() and (y == 0).all()
    run_sandwich(**t, post_gamma=torch.zeros_like(t["gamma"]))


def test_sandwich_no_rows_and_rows_behind():
    q, scale, stream, y = ops.sandwich_norm_quant(randn((0, 64), 1), randn((0, 64), 2, BF16), randn((64,), 3, BF16), normed=True)
    assert q.shape == stream.shape == y.shape == (0, 64) and scale.shape == (0,)
    t = sandwich_inputs(700, 512, BF16, F32)
    outs = dict(q=torch.full((710, 512), 7, device=DEV, dtype=I8), scale=torch.full((710,), 7.0, device=DEV), residual_out=torch.full((710, 512), 7.0, device=DEV, dtype=BF16),
                normed_out=torch.full((710, 512), 7.0, device=DEV, dtype=BF16))
    ops.sandwich_norm_quant(**t, **{k: v[:700] for k, v in outs.items()})
    assert all((v[700:] == 7).all() for v in outs.values())


def test_sandwich_agrees_with_add_rms_norm_quant():
    """Without norm, gate and scales it is that operator, bit for bit."""
    for rows, h, dtype in ((3, 2048, BF16), (700, 1423, F16), (500, 1024, F32), (2, 40000, BF16)):
        x, residual, gamma, smooth = randn((rows, h), 1, dtype), randn((rows, h), 2, dtype), randn((h,), 3, dtype), rand((h,), 4)
        a = ops.sandwich_norm_quant(x, residual, gamma, smooth=smooth, normed=True)
        b = ops.add_rms_norm_quant(x, gamma, residual=residual, smooth=smooth, normed=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
        assert ((a[1] - b[1]).abs() <= b[1] * (h / 16 + 8) * U32).all()   # two orders of one sum


# ---------------------------------------------------------------------------------------------------------------------
# expert_balance
# ---------------------------------------------------------------------------------------------------------------------

def plain_balance(logits, ids, scoring, coefficient, mask=None, cu=None, upstream=1.0):
    """(loss, counts, gradient, p, c, p's tokens' weights) in 64 bits, the gradient from the formula."""
    l = logits.double()
    t, E = l.shape
    k = ids.shape[1]
    gone = ~(l > -math.inf)
    if scoring == "softmax":
        top = l.masked_fill(gone, -math.inf).amax(1, keepdim=True)
        e = torch.where(l == top, torch.ones_like(l), (l - top).exp()).masked_fill(gone, 0)
        rest = torch.ones_like(l)
    else:
        e = torch.sigmoid(l).masked_fill(gone, 0)
        rest = torch.sigmoid(-l).masked_fill(gone, 1)
    total = e.sum(1, keepdim=True)
    p = torch.where(total > 0, e / total, torch.zeros_like(e))
    cuts = [0, t] if cu is None else cu.tolist()
    row = torch.arange(t, device=DEV)
    member = torch.stack([(row >= a) & (row < b) for a, b in zip(cuts[:-1], cuts[1:])])
    if mask is not None:
        member &= mask.bool()
    n = member.sum(1)
    chosen = torch.stack([(ids == j).sum(1) for j in range(E)], 1)
    counts = (member.double() @ chosen.double()).long()
    some = int((n > 0).sum())
    weight = torch.where(n > 0, coefficient * E / (k * n.double().clamp(min=1) ** 2 * max(some, 1)), 0.0)
    c = weight[:, None] * counts
    loss = ((member.double() @ p) * c).sum()
    of_row = member.double().t() @ c
    grad = p * (of_row - (p * of_row).sum(1, keepdim=True)) * rest * upstream * member.any(0)[:, None]
    return loss, counts, weight, grad, p, of_row


def error_of_scores(logits, scoring):
    # p: the argument of the exponential is off by u of its size, the exponential and the quotient by 4 units, the sum of the row's by
    # E / 32 + 5, two products
    finite = logits.double()[torch.isfinite(logits)]
    span = float(finite.max() - finite.min()) if len(finite) and scoring == "softmax" else float(finite.abs().max()) if len(finite) else 0.0
    return (span + 4 + logits.shape[1] / 32 + 5 + 3) * U32


def check_grad(grad, logits, scoring, want, p, c, upstream):
    assert grad.dtype == logits.dtype and grad.shape == logits.shape
    # g = p (c - sum p c): p's own error, and that of a sum of E terms no larger than the largest c (and of c's own mean, taken off before)
    rel_p, terms = error_of_scores(logits, scoring), logits.shape[1] / 32 + 12
    size = p * (c - c.mean(1, keepdim=True)).abs().amax(1, keepdim=True) * abs(upstream)
    bound = want.abs() * (rel_p + 8 * U32) + 2 * size * (rel_p + terms * U32)
    assert ((grad.double() - want).abs() <= bound + want.abs() * HALF_ULP[grad.dtype] * 1.01 + TINY[grad.dtype]).all()


def check_balance(logits, ids, scoring="softmax", coefficient=0.01, mask=None, cu=None, grad_loss=None):
    t, E = logits.shape
    kw = dict(scoring=scoring, token_mask=mask, cu_seqlens=cu)
    loss, counts, weight = ops.expert_balance(logits, ids, coefficient=coefficient, **kw)
    up = 1.0 if grad_loss is None else grad_loss.item()
    f32 = torch.tensor(coefficient, dtype=F32).item()
    want, want_counts, want_weight, want_grad, p, c = plain_balance(logits, ids, scoring, f32, mask, cu, up)
    assert loss.shape == () and loss.dtype == F32 and weight.dtype == F32
    assert torch.equal(counts, want_counts[0] if cu is None else want_counts)
    assert ((weight.double() - want_weight).abs() <= want_weight.abs() * 2 * U32).all()
    # additions that a score's sum over tokens goes through: a warp's rows (of 32 warps on 148 SMs), the 32 warps, a warp's share of at most
    # 148 + 1 pieces, the 32 warps
    chain = t / 148 / 32 + 1 + 32 + 149 / 32 + 1 + 32
    assert abs(loss.item() - want.item()) <= abs(want.item()) * (error_of_scores(logits, scoring) + (chain + 4) * U32) + 1e-38
    grad = ops.expert_balance_grad(logits, counts, weight, grad_loss=grad_loss, **kw)
    check_grad(grad, logits, scoring, want_grad, p, c, up)
    return loss, counts, weight, grad


def balance_inputs(t, E, k, dtype, seed=0):
    logits = (randn((t, E), seed + 1) + randn((E,), seed + 2, scale=0.5)).to(dtype)
    return logits, (logits.float() + randn((E,), seed + 3, scale=0.1)).topk(k, dim=1).indices


BALANCE_SIZES = [(1, 1, 1), (1, 8, 2), (16, 64, 8), (17, 31, 3), (64, 256, 8), (65, 33, 4), (300, 100, 6), (512, 160, 8), (1000, 161, 8), (611, 512, 4), (300, 1024, 8),
                 (77, 1000, 2), (48, 256, 8), (49, 256, 8), (1024, 256, 8), (1025, 256, 8), (500, 512, 8), (4000, 40, 5), (129, 1024, 4), (3001, 155, 6), (5000, 256, 8), (16384, 64, 8), (9000, 8, 1), (2500, 257, 5)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t,E,k", BALANCE_SIZES)
def test_balance_sizes(t, E, k, dtype):
    logits, ids = balance_inputs(t, E, k, dtype)
    scale = torch.tensor(float(t) * 100, device=DEV)
    for scoring in ("softmax", "sigmoid"):
        check_balance(logits, ids.to(I32), scoring, grad_loss=scale)
        mask = rand((t,), 5) < 0.7
        check_balance(logits, torch.where(mask[:, None], ids, -1), scoring, mask=mask, grad_loss=scale)


def cuts(t, n, seed, last=None):
    c = torch.randint(0, t + 1, (n + 1,), device=DEV, generator=gen(seed)).sort().values.to(I32)
    c[0] = 0
    c[-1] = t if last is None else last
    return c


@pytest.mark.parametrize("t,E,k,n", [(1, 8, 2, 1), (40, 64, 4, 3), (40, 64, 4, 40), (700, 33, 3, 16), (5000, 256, 8, 5), (5000, 128, 8, 300), (16384, 256, 8, 16), (300, 16, 2, 2000), (2000, 1000, 3, 20), (900, 600, 2, 32),
                                     (900, 8, 2, 33), (19, 172, 4, 19), (150, 256, 8, 32), (600, 64, 8, 7), (40, 1024, 8, 16), (40, 1024, 8, 17), (320, 121, 5, 3),
                                     (80, 512, 4, 32), (1, 64, 4, 32)])
def test_balance_sequences(t, E, k, n):
    for dtype, scoring in ((F32, "softmax"), (BF16, "sigmoid")):
        logits, ids = balance_inputs(t, E, k, dtype, seed=7)
        check_balance(logits, ids, scoring, cu=cuts(t, n, 1), grad_loss=torch.tensor(100.0, device=DEV))
        mask = rand((t,), 5) < 0.5
        check_balance(logits, torch.where(mask[:, None], ids, -1).to(I32), scoring, mask=mask, cu=cuts(t, n, 2))


def test_balance_of_one_sequence_is_that_of_all_rows():
    logits, ids = balance_inputs(2000, 64, 4, F32)
    cu = torch.tensor([0, 2000], device=DEV, dtype=I32)
    a, b = ops.expert_balance(logits, ids), ops.expert_balance(logits, ids, cu_seqlens=cu)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1][0]) and torch.equal(a[2], b[2])
    assert torch.equal(ops.expert_balance_grad(logits, *a[1:]), ops.expert_balance_grad(logits, *b[1:], cu_seqlens=cu))


def test_balance_few_rows_outside_and_between():
    """Sequences that begin and end inside and on the borders of what a group of lanes holds, empty ones among them, rows before and behind."""
    for rows, E in ((97, 64), (160, 256), (33, 1000)):
        logits, ids = balance_inputs(rows, E, 4, F32)
        for cu in ([0, rows], [5, 5, 6, 6, rows - 3], [0, 0, 0, rows, rows], [rows, rows], [0, 0], [1, 2, 3, 4, 5, 6, 7, 8, 16, 24, 25, 32], list(range(0, 33)),
                   [0, 8, 16, 32], [31, 32, 33]):
            check_balance(logits, ids, cu=torch.tensor(cu, device=DEV, dtype=I32), mask=rand((rows,), 3) < 0.8)


def test_balance_rows_outside_the_sequences():
    """Rows in front of the first and behind the last sequence, and empty sequences at either end and between, as in a padded batch."""
    logits, ids = balance_inputs(1000, 40, 4, F32)
    for c in ([0, 0, 10, 10, 10, 700, 700], [5, 5, 300, 301], [1000, 1000, 1000], [0, 0], [999, 1000], [0, 1, 2, 3, 1000, 1000]):
        cu = torch.tensor(c, device=DEV, dtype=I32)
        *_, grad = check_balance(logits, ids, cu=cu)
        assert (grad[:c[0]] == 0).all() and (grad[c[-1]:] == 0).all()
    # offsets beyond the rows are cut to them
    a = ops.expert_balance(logits, ids, cu_seqlens=torch.tensor([-5, 400, 2000], device=DEV, dtype=I32))
    b = ops.expert_balance(logits, ids, cu_seqlens=torch.tensor([0, 400, 1000], device=DEV, dtype=I32))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_balance_no_rows_and_no_tokens():
    for cu in (None, torch.zeros(4, device=DEV, dtype=I32)):
        loss, counts, weight = ops.expert_balance(randn((0, 24), 1), torch.empty((0, 3), device=DEV, dtype=I32), cu_seqlens=cu)
        assert loss == 0 and (counts == 0).all() and (weight == 0).all()
        assert counts.shape == ((24,) if cu is None else (3, 24))
    for t in (10, 500):
        logits, ids = balance_inputs(t, 24, 3, BF16)
        none = torch.zeros(t, device=DEV, dtype=torch.bool)
        loss, counts, weight, grad = check_balance(logits, ids, mask=none)
        assert loss == 0 and (counts == 0).all() and (weight == 0).all() and (grad == 0).all()


def test_balance_special_logits_and_ids():
    for t in (30, 3000):
        for scoring in ("softmax", "sigmoid"):
            logits, ids = balance_inputs(t, 72, 4, F32, seed=3)
            logits[rand((t, 72), 1) < 0.1] = -math.inf
            logits[1] = -math.inf               # no expert at all
            logits[2] = math.nan
            logits[3, 5], logits[3, 6] = math.nan, -math.inf
            logits[4] = torch.finfo(F32).min    # a mask of the type's lowest value
            logits[5, :40] = torch.finfo(F32).min
            logits[6] *= 30
            logits[7] -= 60
            if scoring == "softmax":
                logits[8, 3] = logits[8, 9] = math.inf
            ids[9:12] = -1
            ids[12] = 72                        # names no expert
            ids[13] = 5                         # the same one in every slot
            ids[14] = 1 << 40
            # rows whose scores span the whole of fp32 have bounds of their own; here only that nothing is wrong beyond them
            loss, counts, weight = ops.expert_balance(logits, ids, scoring=scoring, coefficient=0.01)
            want = plain_balance(logits, ids, scoring, 0.01)
            assert torch.equal(counts, want[1][0]) and abs(loss - want[0]) <= 1e-5 * want[0]
            grad = ops.expert_balance_grad(logits, counts, weight, scoring=scoring)
            assert grad.isfinite().all() and (grad[1] == 0).all() and (grad[2] == 0).all()
            # Logits of up to 250 make exponentials that are 250 u off.  Where one score is all but 1 the gradient p (c - sum p c) is the small
            # difference of two numbers of c's size, each of them rounded: its error goes by p times the largest |c - mean c|, as in
            # check_balance, and not by the gradient, which vanishes with 1 - p (row 6: 1 - p is below u).
            p, c = want[4:]
            size = p * (c - c.mean(1, keepdim=True)).abs().amax(1, keepdim=True)
            assert ((grad.double() - want[3]).abs() <= 2 * (size + want[3].abs()) * (250 + 4 + 8 + 72 / 32 + 12) * U32 + 1e-38).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E", [72, 71])
def test_balance_logits_far_out(scoring, E):
    """Rows whose logits are all far from zero, on both sides of what the plain way of forming scores takes."""
    base = randn((40, E), 1)
    for shift in ([-700, -300, -104, -90, -61, -59, -47, -45, -20, 30, 88, 89, 104] if scoring == "sigmoid" else
                  [-3e5, -700, -90, 90, 1e5, 2.0 ** 20 - 8, 2.0 ** 20, 2.0 ** 21, 2.0 ** 22]):
        logits = base + shift
        ids = logits.topk(3, dim=1).indices
        loss, counts, weight = ops.expert_balance(logits, ids, scoring=scoring)
        grad = ops.expert_balance_grad(logits, counts, weight, scoring=scoring, grad_loss=torch.tensor(1e3, device=DEV))
        want, want_counts, _, want_grad, p, c = plain_balance(logits, ids, scoring, 1.0, upstream=1e3)
        if scoring == "sigmoid" and shift == -700:      # around the border below which there is no score
            assert loss.isfinite() and grad.isfinite().all()
            continue
        # softmax depends on differences alone, which fp32 forms exactly this near to one another; sigmoids on the logits themselves
        rel = (float(logits.abs().max() if scoring == "sigmoid" else (logits.max() - logits.min())) + 4 + E / 32 + 8) * U32
        assert torch.equal(counts, want_counts[0]) and abs(loss.item() - want.item()) <= abs(want.item()) * (rel + 60 * U32)
        size = p * (c - c.mean(1, keepdim=True)).abs().amax(1, keepdim=True) * 1e3
        assert ((grad.double() - want_grad).abs() <= want_grad.abs() * (rel + 8 * U32) + 2 * size * (rel + (E / 32 + 12) * U32) + 1e-38).all()
    huge = torch.full((3, E), -3e38, device=DEV)
    huge[0, 3], huge[1, :2], huge[2, 1] = 3e38, 1e30, -1e38
    grad = ops.expert_balance_grad(huge, *ops.expert_balance(huge, torch.tensor([[3], [0], [1]], device=DEV), scoring=scoring)[1:], scoring=scoring)
    assert grad.isfinite().all()


def test_balance_gradient_against_differences():
    """(L(l + h v) - L(l - h v)) / 2h = <grad, v> + h^2 / 6 L'''; the counts stay, as the ids do."""
    for scoring in ("softmax", "sigmoid"):
        for cu in (None, torch.tensor([0, 30, 30, 90, 120], device=DEV, dtype=I32)):
            logits, ids = balance_inputs(120, 24, 3, F32, seed=11)
            mask = rand((120,), 6) < 0.9
            kw = dict(scoring=scoring, token_mask=mask, cu_seqlens=cu)
            _, counts, weight = ops.expert_balance(logits, ids, coefficient=1.0, **kw)
            grad = ops.expert_balance_grad(logits, counts, weight, **kw).double()
            for i in range(5):
                v, h = randn((120, 24), 20 + i, torch.float64), 1e-4
                up, down = (plain_balance(logits.double() + d * v, ids, scoring, 1.0, mask, cu)[0] for d in (h, -h))
                # third derivatives of scores along v are below |v|^3 of a row, some 24 ** 1.5 of them: 1e-8 / 6 * 118 < 2e-7 a unit of loss;
                # rounding 2^-53 / h = 1e-12; the gradient's own error 1e-6 of the sum of its terms
                assert abs((up - down) / (2 * h) - (grad * v).sum()) <= 2e-7 * 3 + 1e-6 * (grad * v).abs().sum()


def test_balance_strided_rows():
    wide = randn((600, 3 * 64), 1, BF16)
    ids = balance_inputs(600, 64, 4, BF16)[1]
    for logits in (wide[:, 64:128], wide[:, 1:65], wide[:, 3:3 + 62], wide[:, :128:2], randn((64, 600), 2, BF16).t(), wide[:1, :64].expand(600, 64)):
        _, counts, weight, grad = check_balance(logits, ids.clamp(max=logits.shape[1] - 1), grad_loss=torch.tensor(600.0, device=DEV))
        room = torch.full((600, 200), 3.0, device=DEV, dtype=BF16)
        for left in (0, 1, 8):
            out = room[:, left:left + logits.shape[1]]
            assert ops.expert_balance_grad(logits, counts, weight, grad_loss=torch.tensor(600.0, device=DEV), grad=out) is out
            check_grad(out, logits, "softmax", *plain_balance(logits, ids.clamp(max=logits.shape[1] - 1), "softmax", 0.01, upstream=600.0)[3:], 600.0)
            assert (room[:, :left] == 3).all()
            assert (room[:, left + logits.shape[1]:] == 3).all()
            room.fill_(3.0)
    logits = wide[:, :64].contiguous()
    _, counts, weight = ops.expert_balance(logits, ids.repeat_interleave(2, 1)[:, ::2])
    want = ops.expert_balance_grad(logits, counts, weight)
    assert torch.equal(ops.expert_balance_grad(logits, counts, weight, grad=logits), want) and torch.equal(logits, want)   # in place


def test_balance_same_bits_every_time():
    logits, ids = balance_inputs(12345, 256, 8, F32)
    first = ops.expert_balance(logits, ids, cu_seqlens=cuts(12345, 7, 3))
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, ops.expert_balance(logits, ids, cu_seqlens=cuts(12345, 7, 3))))


def test_balance_feeds_a_router_that_torch_differentiates():
    """One step against the gradient lowers the loss of the same choices; the router's gradient is that of the formula."""
    h, w = randn((400, 96), 1), randn((40, 96), 2, scale=0.1).requires_grad_(True)
    logits = h @ w.t()
    ids = ops.route_top_k(logits.detach(), 4)[1]
    loss, counts, weight = ops.expert_balance(logits.detach(), ids, coefficient=1.0)
    logits.backward(ops.expert_balance_grad(logits.detach(), counts, weight))
    want = plain_balance(logits.detach(), ids, "softmax", 1.0)[3].t() @ h.double()
    assert (w.grad.double() - want).norm() <= 1e-4 * want.norm()   # fp32 products of 400 terms
    assert (counts == torch.bincount(ids.flatten().long(), minlength=40)).all()


# ---------------------------------------------------------------------------------------------------------------------
# streams, graphs, threads
# ---------------------------------------------------------------------------------------------------------------------

def every_op(seed=0, rows=300):
    x, w, scale, token = int8((rows, 512), seed + 1), int8((512, 640), 2), rand((640,), 3), rand((rows,), seed + 4)
    t = sandwich_inputs(rows, 640, BF16, F32, seed)
    logits, ids = balance_inputs(rows, 64, 4, F32, seed)
    return dict(x=x, w=w, scale=scale, token=token, logits=logits, ids=ids, **{"n_" + k: v for k, v in t.items()})


def run_every_op(s, stream=None):
    y = ops.quant_matmul(s["x"], s["w"], s["scale"], s["token"], stream=stream)
    normed = ops.sandwich_norm_quant(s["n_x"], s["n_residual"], s["n_gamma"], post_gamma=s["n_gamma"], normed=True, stream=stream)
    loss, counts, weight = ops.expert_balance(s["logits"], s["ids"], stream=stream)
    return (y, *normed, loss, counts, weight, ops.expert_balance_grad(s["logits"], counts, weight, stream=stream))


def test_operators_on_another_stream():
    s = every_op()
    want = run_every_op(s)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = run_every_op(s, stream=side)
    with torch.cuda.stream(side):
        again = run_every_op(s)
    side.synchronize()
    assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(got, want, again))


@pytest.mark.parametrize("rows", [3, 300])
def test_operators_can_be_captured(rows):
    """Two graphs that are replayed in turn, with calls outside between them, on inputs that change."""
    states, graphs, outs = [every_op(i, rows) for i in (0, 50)], [], []
    for s in states:
        run_every_op(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run_every_op(s))
        graphs.append(g)
    for i, fresh in ((0, 100), (1, 150), (0, 200), (1, 250)):
        new = every_op(fresh, rows)
        for k, v in states[i].items():
            v.copy_(new[k])
        graphs[i].replay()
        want = run_every_op(new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[i], want))


def test_operators_from_several_threads():
    import threading
    states = [every_op(10 * i, rows=100 + 50 * i) for i in range(4)]
    want = [run_every_op(s) for s in states]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = run_every_op(states[i])
            torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                failed.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


@pytest.mark.parametrize("m,k,n", [(16, 1024, 256), (256, 512, 18944), (600, 384, 640)])
def test_matmul_reports_a_wait_that_runs_out(m, k, n):
    """The producer leaves out the last K block of every CTA and the others wait for about 1 ms: the call ends, says so in its status, and the next
    one on the same workspace is right.  Cluster of several CTAs, and one CTA a tile."""
    x, w, scale = int8((m, k), 1), int8((k, n), 2), rand((n,), 3) + 0.5
    want = plain_matmul(x, w, scale, None, None, BF16)
    y, ws = ops.quant_matmul(x, w, scale, return_workspace=True)
    ops.check_status(ws)
    assert torch.equal(y, want)
    ws = torch.zeros(ws.numel(), dtype=torch.uint8, device=DEV)
    ops.quant_matmul(x, w, scale, out=torch.empty_like(y), workspace=ws, options=ops.LaunchOptions(wait_limit_cycles=2_000_000, test_skip_k_blocks=1))
    with pytest.raises(ops.AclnnError):
        ops.check_status(ws)
    again = ops.quant_matmul(x, w, scale, out=torch.zeros_like(y), workspace=ws)
    ops.check_status(ws)
    assert torch.equal(again, want)


# ---------------------------------------------------------------------------------------------------------------------
# all of them as a decoder layer runs them: block, exit, next block, load
# ---------------------------------------------------------------------------------------------------------------------

def chain(tokens, hidden=512, inter=256, experts=8, top_k=2, scoring="softmax"):
    from ops_transformer_b200.block import BlockExit, random_block
    first, second = (random_block(hidden, inter, experts, top_k, adapters=2, scoring=scoring, seed=s) for s in (0, 1))
    leave = BlockExit(second.gamma, post_gamma=randn((hidden,), 5, BF16, 0.1) + 1, gate=randn((hidden,), 6, BF16), gate_act="sigmoid", residual_scale=0.75,
                      block_scale=1.25)
    return first, second, leave


@pytest.mark.parametrize("tokens,scoring", [(1, "softmax"), (40, "sigmoid"), (300, "softmax")])
def test_blocks_in_a_row(monkeypatch, tokens, scoring):
    from ops_transformer_b200 import block as module
    first, second, leave = chain(tokens, scoring=scoring)
    x, residual = randn((tokens, 512), 1, BF16), randn((tokens, 512), 2, BF16)
    adapter_ids, mask = (torch.arange(tokens, device=DEV) % 3 - 1).to(I32), torch.arange(tokens, device=DEV) % 5 != 3
    kw = dict(adapter_ids=adapter_ids, token_mask=mask)
    out, stream = first(x, residual, **kw)
    routed = []
    with monkeypatch.context() as m:
        m.setattr(module, "route_top_k", lambda logits, k, _f=module.route_top_k, **kw: routed.append((logits, *_f(logits, k, **kw))) or routed[-1][1:])
        entered, (loss, counts, weight) = first(x, residual, leave=leave, balance=0.01, **kw)
        got, got_stream, load = second(entered, balance=0.02, **kw)
    # the way out, from `out` as another run of the block gives it: its rows are added up in no fixed order, a few units of fp32 of their
    # size, below 2^-16 of the largest value, which the norms pass on about as large
    n = out.double() * (out.double().square().mean(1, keepdim=True) + 1e-6).rsqrt() * leave.post_gamma.double()
    s = 0.75 * stream.double() + 1.25 * torch.sigmoid(leave.gate.double()) * n
    u = s * (s.square().mean(1, keepdim=True) + 1e-6).rsqrt() * second.gamma.double()
    near = 2.0 ** -15 * s.abs().amax(1, keepdim=True)
    assert ((entered.stream.double() - s).abs() <= s.abs() * 2.0 ** -8 + near).all()
    near = 2.0 ** -14 * u.abs().amax(1, keepdim=True)
    assert ((entered.normed.double() - u).abs() <= u.abs() * 2.0 ** -8 * 1.01 + near).all()
    assert ((entered.rows * entered.scales.double()[:, None] - u).abs() <= entered.scales.double()[:, None] * 0.501 + near).all()
    # the next block takes the rows as its own norm would have left them
    want = second(module.Entered(*entered), **kw)
    assert torch.equal(got_stream, entered.stream) and torch.equal(want[1], entered.stream)
    assert (got - want[0]).abs().max() < 64 * U32 * math.sqrt(512)
    for (logits, _, ids), (loss, counts, weight), coefficient in ((routed[0], (loss, counts, weight), 0.01), (routed[1], load, 0.02)):
        f32 = torch.tensor(coefficient, dtype=F32).item()
        want = plain_balance(logits, ids, scoring, f32, mask)
        assert torch.equal(counts, want[1][0]) and int(counts.sum()) == int(mask.sum()) * 2
        assert abs(loss.item() - want[0].item()) <= abs(want[0].item()) * (error_of_scores(logits, scoring) + 80 * U32)


def test_blocks_in_a_row_can_be_captured():
    first, second, leave = chain(24)
    x, residual = randn((24, 512), 1, BF16), randn((24, 512), 2, BF16)
    mask = torch.arange(24, device=DEV) < 20

    def step():
        entered, load = first(x, residual, token_mask=mask, leave=leave, balance=0.01)
        return *second(entered, token_mask=mask), *load
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    x.copy_(randn((24, 512), 3, BF16))
    mask[:4] = False
    graph.replay()
    got = [o.clone() for o in outs]
    want = step()
    # rows are added into the first block's result in no fixed order, which an int8 row of the second may round to its other neighbour
    assert torch.equal(got[3], want[3]) and torch.equal(got[4], want[4]) and torch.equal(got[2], want[2])
    assert ((got[1].double() - want[1].double()).abs() <= want[1].double().abs() * 2.0 ** -7 + 2.0 ** -15).all()
    assert (got[0] - want[0]).norm() <= 0.01 * want[0].norm()


def test_block_takes_one_residual_stream():
    first, second, leave = chain(4)
    entered = first(randn((4, 512), 1, BF16), randn((4, 512), 2, BF16), leave=leave)
    with pytest.raises(ValueError, match="residual"):
        second(entered, randn((4, 512), 2, BF16))


def test_shared_expert_as_the_grouped_product_gives_it():
    """The block's shared expert goes through quant_matmul; its rows are those of the grouped product with one group."""
    for m, k, n in ((1, 256, 512), (40, 512, 1024), (300, 256, 768)):
        x, w, scale, token = int8((m, k), 1), int8((1, k, n), 2), rand((1, n), 3) * 0.01, rand((m,), 4)
        group = torch.full((1,), m, dtype=I64, device=DEV)
        assert torch.equal(ops.quant_matmul(x, w[0], scale[0], token), ops.grouped_matmul_v4(x, w, scale, token, group))


# ---------------------------------------------------------------------------------------------------------------------
# sizes and arguments at the edge of what is allowed
# ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("m,k,n,nk", [(600_000, 128, 4096, False), (300_000, 8192, 160, True), (300_001, 7170, 20, False)])
def test_matmul_beyond_32_bits(m, k, n, nk):
    """Rows of the result, or of x, behind the 2^31st element: as a call of their own gives them."""
    x = torch.zeros((m, k), dtype=I8, device=DEV)
    x[-300:] = int8((300, k), 1)
    w = int8((n, k), 2).t() if nk else int8((k, n), 2)
    scale, token, bias = rand((n,), 3), rand((m,), 4), rand((n,), 5)
    got = ops.quant_matmul(x, w, scale, token, bias=bias)
    assert torch.equal(got[-300:], ops.quant_matmul(x[-300:].clone(), w, scale, token[-300:].clone(), bias=bias))
    assert (got[:1000] == bias.to(BF16)).all() and (got[m // 2:m // 2 + 1000] == bias.to(BF16)).all()


@pytest.mark.parametrize("rows,h", [(310_000, 7168), (310_001, 7001), (40_000, 65535), (9_000_000, 256)])
def test_sandwich_beyond_32_bits(rows, h):
    x, residual = (torch.zeros((rows, h), dtype=F16, device=DEV) for _ in range(2))
    t = sandwich_inputs(200, h, F16, F16)
    x[-200:], residual[-200:] = t["x"], t["residual"]
    got = ops.sandwich_norm_quant(x, residual, t["gamma"], post_gamma=t["gamma"], normed=True)
    check_sandwich(t["x"], t["residual"], t["gamma"], [v[-200:] for v in got], post_gamma=t["gamma"], normed=True)
    assert all((v[:1000] == 0).all() and (v[rows // 2:rows // 2 + 1000] == 0).all() for v in got)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_balance_beyond_32_bits(scoring):
    """The same 4096 tokens 1100 times over: their loss is that of them once, and a gradient the 1100th part."""
    times, E = 1100, 512
    logits, ids = balance_inputs(4096, E, 8, BF16)
    loss, counts, weight = ops.expert_balance(logits, ids, scoring=scoring)
    grad = ops.expert_balance_grad(logits, counts, weight, scoring=scoring, grad_loss=torch.tensor(4096.0, device=DEV))
    many, many_ids = logits.repeat(times, 1), ids.repeat(times, 1)
    assert many.numel() > 1 << 31
    got = ops.expert_balance(many, many_ids, scoring=scoring)
    assert torch.equal(got[1], counts * times)
    # sums of 4.5 million scores: a warp's rows, its groups, the pieces
    assert abs(got[0].item() / loss.item() - 1) <= (4096 * times / 148 / 16 + 80) * U32
    g = ops.expert_balance_grad(many, got[1], got[2], scoring=scoring, grad_loss=torch.tensor(4096.0 * times, device=DEV))
    for part in (g[:4096], g[-4096:]):
        # the same steps with factors that are rounded apart: half a unit of bf16 each, and single ones of fp32
        assert ((part.double() - grad.double()).abs() <= grad.double().abs() * 2.0 ** -7 + 1e-30).all()


def test_balance_arguments_of_other_strides_and_places():
    logits, ids = balance_inputs(700, 64, 4, F32)
    mask = rand((1400,), 1) < 0.6
    cu = torch.tensor([0, 9, 100, 9, 350, 9, 700, 9], device=DEV, dtype=I32)
    for kw in (dict(token_mask=mask[::2]), dict(cu_seqlens=cu[::2]), dict(token_mask=mask[::2].to(I8), cu_seqlens=cu[::2])):
        dense = {k: v.contiguous() for k, v in kw.items()}
        want = ops.expert_balance(logits, ids, **dense)
        want_grad = ops.expert_balance_grad(logits, *want[1:], **dense)
        n = 3 if "cu_seqlens" in kw else 1
        room = torch.full((9,), 7.0, device=DEV)
        counts = torch.full((n, 2 * 64) if n > 1 else (2 * 64,), 5, device=DEV, dtype=I64)[..., ::2]
        weight = torch.full((2 * n,), 3.0, device=DEV)
        loss, c, w = ops.expert_balance(logits, ids, loss=room[4], counts=counts, weight=weight[::2], **kw)
        assert torch.equal(loss, want[0]) and room[4] == want[0] and (room[:4] == 7).all() and (room[5:] == 7).all()
        assert torch.equal(c, want[1]) and torch.equal(w, want[2]) and (weight[1::2] == 3).all()
        assert torch.equal(ops.expert_balance_grad(logits, c, w, grad_loss=torch.ones(3, device=DEV)[1], **kw), want_grad)
        # counts on no 16-byte boundary
        off = torch.zeros(want[1].numel() + 1, dtype=I64, device=DEV)[1:].view_as(want[1]).copy_(want[1])
        # (other lanes have the experts then: two sums of 64 terms a row in another order, 6 additions each, and what is formed from them)
        assert (ops.expert_balance_grad(logits, off, w.clone(), **dense) - want_grad).abs().max() <= 2 * (6 + 6 + 4) * U32 * want_grad.abs().max()


def test_sandwich_normed_rows_in_place_of_x():
    for rows, h in ((20, 512), (400, 5001), (300, 7168), (3, 40000)):
        t = sandwich_inputs(rows, h, BF16, BF16)
        want = ops.sandwich_norm_quant(**t, post_gamma=t["gamma"], normed=True)
        x = t["x"].clone()
        got = ops.sandwich_norm_quant(x, t["residual"], t["gamma"], post_gamma=t["gamma"], normed_out=x)
        assert got[3] is x and all(torch.equal(a, b) for a, b in zip(got, want))
