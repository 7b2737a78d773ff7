"""add_rms_norm_quant, route_top_k and adapter_add on the GPU against plain implementations in 64 bits (and in fp32 where a result has
to be bit-identical), at the sizes, strides, masks and special values where they can go wrong.

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
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def randn(shape, seed, dtype=F32, scale=1.0):
    return (torch.randn(shape, device=DEV, generator=gen(seed)) * scale).to(dtype)


# ---------------------------------------------------------------------------------------------------------------------
# add_rms_norm_quant
# ---------------------------------------------------------------------------------------------------------------------

def check_norm(x, gamma, residual, smooth, eps, got):
    q, scale, res_out, normed = got
    n = x.shape[1]
    h32 = x.float() + residual.float() if residual is not None else x.float()
    if residual is not None:
        assert torch.equal(res_out, h32.to(x.dtype))
    else:
        assert res_out is None
    h = x.double() + residual.double() if residual is not None else x.double()
    h = h32.double()   # the operator's h is the fp32 sum
    r = 1 / (h.square().mean(1, keepdim=True) + eps).sqrt()
    # fp32 sum of n squares by at most n / 32 + 10 steps in a row (each relative u, halved by the root), quotient, root, reciprocal
    rel_r = (n / 32 + 16) * U32
    if normed is not None:
        y = h * r * gamma.double()
        assert ((normed.double() - y).abs() <= y.abs() * (HALF_ULP[x.dtype] * (1 + 1e-3) + rel_r + 3 * U32) + TINY[x.dtype]).all()
    u = h32 * gamma.float()
    if smooth is not None:
        u = u * smooth
    step = u.abs().amax(1, keepdim=True)
    step = step / torch.full_like(step, 127.0)
    want = torch.where(step > 0, torch.round(u / step), torch.zeros_like(u)).clamp(-127, 127)
    assert torch.equal(q.float(), want)
    exact = step.double()[:, 0] * r[:, 0]
    assert ((scale.double() - exact).abs() <= exact * (rel_r + 3 * U32)).all()
    # the dequantised row is within half a step of the normed row
    z = h * r * gamma.double() * (smooth.double() if smooth is not None else 1)
    assert ((q.double() * scale.double()[:, None] - z).abs() <= scale.double()[:, None] * (0.5 + 127 * (rel_r + 8 * U32))).all()


NORM_SIZES = [(1, 1), (1, 8), (3, 7), (5, 16), (2, 255), (17, 256), (4, 1000), (1, 2048), (33, 1423), (150, 2048), (7, 7168), (200, 7168),
              (3, 8200), (2, 16384), (2, 20001), (1, 65535), (2, 65528)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,h", NORM_SIZES)
def test_norm_sizes(rows, h, dtype):
    x, res = randn((rows, h), 1, dtype), randn((rows, h), 2, dtype, 3.0)
    gamma = randn((h,), 3, dtype, 0.2) + 1
    smooth = torch.rand(h, device=DEV, generator=gen(4)) + 0.5
    for residual, sm, normed in ((res, None, True), (None, smooth, False), (res, smooth, True), (None, None, False)):
        got = ops.add_rms_norm_quant(x, gamma, residual=residual, smooth=sm, eps=1e-5, normed=normed)
        check_norm(x, gamma, residual, sm, 1e-5, got)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_norm_gamma_in_fp32(dtype):
    for rows, h in ((9, 512), (300, 1000), (4, 333)):
        x, gamma = randn((rows, h), 5, dtype), randn((h,), 6)
        check_norm(x, gamma, None, None, 1e-6, ops.add_rms_norm_quant(x, gamma, eps=1e-6, normed=True))


@pytest.mark.parametrize("offset,pitch", [(0, 2 * 1024), (8, 1024 + 8), (1, 1024 + 3), (4, 1024 + 4)])
def test_norm_strided_rows_and_offsets(offset, pitch):
    rows, h = 37, 1024
    wide = lambda seed, dt=BF16: randn((rows * pitch + 64,), seed, dt)[offset:].as_strided((rows, h), (pitch, 1))  # noqa: E731
    x, res, gamma = wide(1), wide(2), randn((h + 8,), 3, BF16)[offset:offset + h]
    res_out, normed = wide(4), wide(5)
    q = torch.zeros(rows * pitch + 64, dtype=torch.int8, device=DEV)[offset:].as_strided((rows, h), (pitch, 1))
    got = ops.add_rms_norm_quant(x, gamma, residual=res, q=q, residual_out=res_out, normed_out=normed)
    check_norm(x, gamma, res, None, 1e-6, got)
    # columns apart and transposed views go through copies
    x2 = randn((rows, 2 * h), 7, BF16)[:, ::2]
    x3 = randn((h, rows), 8, BF16).t()
    for v in (x2, x3, randn((1, h), 9, BF16).expand(rows, h)):
        check_norm(v, gamma, None, None, 1e-6, ops.add_rms_norm_quant(v, gamma, normed=True))


def test_norm_in_place():
    for rows, h in ((40, 2048), (3, 40000), (5, 77)):
        x, res, gamma = randn((rows, h), 1, BF16), randn((rows, h), 2, BF16), randn((h,), 3, BF16)
        want = ops.add_rms_norm_quant(x, gamma, residual=res, normed=True)
        for into in ("residual", "x"):
            a, b = x.clone(), res.clone()
            got = ops.add_rms_norm_quant(a, gamma, residual=b, residual_out=b if into == "residual" else a,
                                         normed_out=a if into == "residual" else None)
            assert all(torch.equal(g, w) for g, w in zip(got[:3], want[:3]))
            if into == "residual":
                assert torch.equal(a, want[3])


def test_norm_special_rows():
    h = 1040
    for dtype in (BF16, F32):
        x = randn((8, h), 1, dtype)
        gamma = torch.ones(h, device=DEV, dtype=dtype)
        x[1] = 0                       # no step to divide by
        x[2, 5] = math.inf
        x[3, h - 1] = math.nan
        x[4] = 0
        x[4, 9] = -1e-30               # a step far below the others
        x[5, 3] = 1e4                  # one value dwarfs the rest
        x[6] = 1e-41 if dtype == F32 else 1e-40   # subnormal values
        q, scale, _, y = ops.add_rms_norm_quant(x, gamma, eps=1e-6, normed=True)
        assert (q[1] == 0).all() and scale[1] == 0 and (y[1] == 0).all()
        assert scale[2].isnan() and (q[2] == 0).all() and scale[3].isnan() and (q[3] == 0).all()
        assert q[4, 9] == -127 and (q[4].abs().sum() == 127)
        good = torch.tensor([0, 4, 5, 7], device=DEV)
        check_norm(x[good], gamma, None, None, 1e-6, (q[good], scale[good], None, y[good]))
        assert q[6].abs().max() <= 127 and scale[6].isfinite()
    # gamma with zeros, and all zeros
    x, gamma = randn((4, 64), 2, BF16), torch.zeros(64, device=DEV, dtype=BF16)
    q, scale, _, _ = ops.add_rms_norm_quant(x, gamma)
    assert (q == 0).all() and (scale == 0).all()


def test_norm_no_rows_and_many_rows():
    x = torch.empty((0, 512), dtype=BF16, device=DEV)
    q, scale, r, y = ops.add_rms_norm_quant(x, torch.ones(512, dtype=BF16, device=DEV), residual=x, normed=True)
    assert q.shape == (0, 512) and scale.shape == (0,) and r.shape == (0, 512) and y.shape == (0, 512)
    x = randn((70001, 32), 1, BF16)
    check_norm(x, randn((32,), 2, BF16), None, None, 1e-6, ops.add_rms_norm_quant(x, randn((32,), 2, BF16)))


def test_norm_offsets_beyond_32_bits():
    rows, h, pitch = 3, 64, 1 << 30
    x = torch.zeros(rows * pitch, dtype=BF16, device=DEV).as_strided((rows, h), (pitch, 1))
    x.copy_(randn((rows, h), 1, BF16))
    gamma = randn((h,), 2, BF16)
    check_norm(x, gamma, None, None, 1e-6, ops.add_rms_norm_quant(x, gamma, normed=True))


# ---------------------------------------------------------------------------------------------------------------------
# route_top_k
# ---------------------------------------------------------------------------------------------------------------------

def route_reference(logits, k, scoring, bias, G, topk_group, group_score, mask):
    """(scores, choices with what is out at -inf, rows that are there) in 64 bits; the rules written out."""
    l = logits.double()
    gone = torch.isnan(l) | (l == -math.inf)
    if scoring == "sigmoid":
        s = torch.sigmoid(l)
    else:
        s = torch.softmax(torch.where(gone, -math.inf, l), 1)
        inf = l == math.inf
        s = torch.where(inf.any(1, keepdim=True), inf / inf.sum(1, keepdim=True).clamp_min(1), s)
    s = torch.where(gone, 0.0, s)
    scored = bias is not None or (G > 1 and group_score == "top2")
    c = s + bias.double() if bias is not None else s if scored else l.clone()
    c = torch.where(gone | torch.isnan(c), -math.inf, c)
    return s, c, scored


def check_route(logits, k, got, *, scoring="softmax", bias=None, n_group=1, topk_group=1, group_score="max", renormalize=True, scale=1.0,
                token_mask=None):
    w, ids = got
    T, E = logits.shape
    s, c, scored = route_reference(logits, k, scoring, bias, n_group, topk_group, group_score, token_mask)
    # a choice is off by the score's rounding (exp, sum, quotient: 4 u of at most 1), the bias's addition and a group's sum
    slack = 1e-6 * max(1.0, float(bias.abs().nan_to_num(0, 0, 0).max()) if bias is not None else 1.0) if scored else 0.0
    ids = ids.long()
    live = token_mask.bool() if token_mask is not None else torch.ones(T, dtype=torch.bool, device=DEV)
    assert (ids[~live] == -1).all() and (w[~live] == 0).all()
    there = ids >= 0
    assert (ids < E).all() and (w[~there] == 0).all()
    assert (there[:, 1:] <= there[:, :-1]).all(), "free slots come last"
    cc = c.gather(1, ids.clamp_min(0))
    assert (cc[there] > -math.inf).all()
    if n_group > 1:
        gs = E // n_group
        top = c.view(T, n_group, gs).topk(min(2, gs), dim=2).values
        rank = top[..., 0]
        if group_score == "top2" and gs > 1:
            rank = rank + top[..., 1].nan_to_num(neginf=0.0)
        used = (torch.nn.functional.one_hot(ids.clamp_min(0) // gs, n_group) * there[..., None]).sum(1) > 0
        # every used group is among the best ones: at most topk_group - 1 others are better by more than the slack
        better = (rank[:, None, :] > rank[:, :, None] + 2 * slack).sum(2)
        assert (better[used & live[:, None]] < topk_group).all()
        assert (used.sum(1) <= topk_group).all()
        surely = (rank[:, None, :] >= rank[:, :, None] - 2 * slack).sum(2) <= topk_group   # among the best whatever the rounding
        out = torch.where(surely.repeat_interleave(gs, 1), c, -math.inf)                    # experts that were surely candidates
    else:
        out = c
    # none that was left out beats one that was taken; taken ones stand in order
    left = out.scatter(1, ids.clamp_min(0), torch.where(there, -math.inf, out.gather(1, ids.clamp_min(0))))
    worst = torch.where(there, cc, math.inf).amin(1)
    full = there.all(1)
    best_left = left.amax(1)
    assert (best_left <= worst + 2 * slack)[live & full].all()
    assert (best_left == -math.inf)[live & ~full].all(), "a slot stayed free although an expert was left"
    d = cc[:, 1:] - cc[:, :-1]
    both = there[:, 1:] & there[:, :-1]
    assert (d[both & ~torch.isnan(d)] <= 2 * slack).all()
    if not scored:   # by the logits: exactly the stable order
        ties = (cc[:, 1:] == cc[:, :-1]) & both
        assert (ids[:, 1:] > ids[:, :-1])[ties].all()
    assert all(len(set(r[r >= 0].tolist())) == int((r >= 0).sum()) for r in ids.cpu()[:64])
    want = torch.where(there, s.gather(1, ids.clamp_min(0)), 0.0)
    if renormalize:
        total = want.sum(1, keepdim=True)
        want = torch.where(total > 0, want / total, 0.0)
    want = want * scale
    finite = logits.double()[logits.double().isfinite()]
    spread = float(finite.abs().max()) if finite.numel() else 0.0   # exp's argument is rounded: relative u times its size
    assert ((w.double() - want).abs() <= want.abs() * (2 * spread + 24) * U32 + 1e-37).all()


def route(logits, k, **kw):
    got = ops.route_top_k(logits, k, **kw)
    check_route(logits, k, got, **kw)
    return got


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 2, 1), (5, 8, 8), (33, 31, 3), (16, 64, 8), (7, 100, 32), (129, 256, 8), (50, 257, 6),
                                   (9, 512, 1), (3, 1000, 10), (5, 1024, 32)])
def test_route_sizes(T, E, k, scoring):
    bias = randn((E,), 2, scale=0.1)
    for dtype in (F32, BF16, F16):
        logits = randn((T, E), 1, dtype, 2.0)
        for renorm in (True, False):
            route(logits, k, scoring=scoring, renormalize=renorm)
            route(logits, k, scoring=scoring, renormalize=renorm, bias=bias, scale=2.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("T,E,G,kg,k", [(40, 256, 8, 4, 8), (17, 160, 8, 3, 6), (9, 155, 5, 3, 6), (21, 96, 32, 7, 5), (3, 1024, 2, 1, 8),
                                        (11, 1023, 31, 30, 16), (8, 7, 7, 2, 2), (13, 30, 3, 3, 30), (4, 999, 3, 2, 9)])
def test_route_groups(T, E, G, kg, k, group_score, scoring):
    for seed, dtype in ((1, F32), (2, BF16)):
        logits = randn((T, E), seed, dtype)
        for bias in (None, randn((E,), 5, scale=0.05)):
            route(logits, k, scoring=scoring, bias=bias, n_group=G, topk_group=kg, group_score=group_score)


def test_route_ties_take_the_lowest_id():
    logits = torch.randint(-2, 3, (200, 96), device=DEV, generator=gen(1)).float()
    logits[0] = 0.0
    logits[1, ::2], logits[1, 1::2] = -0.0, 0.0          # the two zeros are equal
    for scoring in ("softmax", "sigmoid"):
        w, ids = route(logits, 12, scoring=scoring)
        assert torch.equal(ids.long(), logits.sort(dim=1, descending=True, stable=True).indices[:, :12])
        w, ids = route(logits, 4, scoring=scoring, n_group=8, topk_group=2)
        assert ids[0].tolist() == [0, 1, 2, 3] and ids[1].tolist() == [0, 1, 2, 3]
        # equal scores and equal biases are ties as well
        _, ids = route(logits, 12, scoring=scoring, bias=torch.full((96,), 0.25, device=DEV))
        assert ids[0].tolist() == list(range(12))


def test_route_masks_and_special_values():
    T, E = 64, 40
    logits = randn((T, E), 1)
    logits[0] = -math.inf                       # no expert at all
    logits[1] = math.nan
    logits[2, 3:] = -math.inf                   # fewer than k
    logits[3, 7] = math.inf
    logits[4, 7] = logits[4, 9] = math.inf
    logits[5, ::2] = math.nan
    logits[6] = torch.finfo(F32).min            # the type's lowest value is a value
    logits[7, 1:] = torch.finfo(F32).min
    logits[8] = 200.0
    logits[9] = -200.0
    mask = torch.rand(T, device=DEV, generator=gen(2)) < 0.7
    mask[:10] = True
    bias = randn((E,), 3, scale=0.1)
    bias[11], bias[12], bias[13] = -math.inf, math.nan, math.inf
    for scoring in ("softmax", "sigmoid"):
        for kw in (dict(), dict(bias=bias), dict(n_group=4, topk_group=2), dict(n_group=4, topk_group=2, group_score="top2"),
                   dict(renormalize=False), dict(renormalize=False, bias=bias)):
            kw = dict(kw, scoring=scoring, token_mask=mask)
            w, ids = ops.route_top_k(logits, 6, **kw)
            assert w.isfinite().all()
            assert (ids[:2] == -1).all() and (w[:2] == 0).all()
            assert (ids[2] >= 0).sum() == 3
            assert (ids[~mask] == -1).all()
            if "bias" in kw:
                assert not ((ids == 11) | (ids == 12)).any() and (ids[mask][8:, 0] == 13).all()
            elif scoring == "softmax":
                assert ids[3, 0] == 7 and ids[4, :2].tolist() == [7, 9] and not (ids[5] % 2 == 0).any()
            rest = torch.arange(T, device=DEV) >= 10
            kw2 = {k: v for k, v in kw.items() if k != "token_mask"}
            if "bias" not in kw:
                check_route(logits[rest], 6, (w[rest], ids[rest]), token_mask=mask[rest], **kw2)
    assert ops.route_top_k(logits, 6, token_mask=mask.to(torch.int8))[1].equal(ops.route_top_k(logits, 6, token_mask=mask)[1])


def test_route_outputs_strides_and_empty():
    wide = randn((50, 300), 1)
    logits = wide[:, 20:148]
    w, ids = route(logits, 8)
    w2, i2 = route(logits.contiguous(), 8)
    assert torch.equal(w, w2) and torch.equal(ids, i2)
    w3, i3 = ops.route_top_k(wide.t().contiguous().t()[:, 20:148], 8, ids_dtype=torch.int64)
    assert i3.dtype == torch.int64 and torch.equal(i3, ids.long()) and torch.equal(w3, w)
    out = torch.zeros(50, 16, device=DEV)[:, ::2], torch.zeros(50, 16, dtype=torch.int32, device=DEV)[:, ::2]
    ops.route_top_k(logits, 8, weights=out[0], ids=out[1])
    assert torch.equal(out[0], w) and torch.equal(out[1], ids)
    w, ids = ops.route_top_k(torch.empty((0, 16), device=DEV), 4)
    assert w.shape == (0, 4) and ids.shape == (0, 4)
    one = randn((1, 64), 3, BF16).expand(9, 64)
    w, ids = route(one, 5)
    assert (ids == ids[0]).all()


# ---------------------------------------------------------------------------------------------------------------------
# adapter_add
# ---------------------------------------------------------------------------------------------------------------------

def adapter_case(T, K, N, L, r, dtype=BF16, x_i8=False, seed=0, ids=None, scaling=True):
    x = randn((T, K), seed + 1, F32, 30).round().clamp(-127, 127).to(torch.int8) if x_i8 else randn((T, K), seed + 1, dtype)
    xs = (torch.rand(T, device=DEV, generator=gen(seed + 2)) + 0.5) / 32 if x_i8 else None
    a, b = randn((L, r, K), seed + 3, dtype, 1 / math.sqrt(K)), randn((L, N, r), seed + 4, dtype, 1 / math.sqrt(r))
    if ids is None:
        ids = torch.randint(-1, L, (T,), device=DEV, generator=gen(seed + 5)).to(torch.int32)
    sc = torch.rand(L, device=DEV, generator=gen(seed + 6)) + 0.5 if scaling else None
    return dict(base=randn((T, N), seed + 7, dtype), x=x, a=a, b=b, adapter_ids=ids, x_scale=xs, scaling=sc)


def check_adapter(c, out):
    K, r, L = c["x"].shape[1], c["a"].shape[1], c["a"].shape[0]
    want, mag = c["base"].double(), torch.zeros_like(c["base"], dtype=torch.float64)
    for i in range(L):
        at = (c["adapter_ids"] == i).nonzero()[:, 0]
        if not len(at):
            continue
        x = c["x"][at].double()
        if c["x_scale"] is not None:
            x = x * c["x_scale"][at, None].double()
        s = c["scaling"][i].double() if c["scaling"] is not None else 1.0
        want[at] += s * ((x @ c["a"][i].double().t()) @ c["b"][i].double().t())
        mag[at] = s * ((x.abs() @ c["a"][i].double().abs().t()) @ c["b"][i].double().abs().t())
    # a fp32 accumulation of K / 16 + rank / 16 steps, each off by a unit of the partial sum at most, two factors, the split of the
    # product's first part in two 16-bit halves (2^-16 in bf16); and the rounding of the result
    tol = mag * ((K / 16 + r / 16 + 8) * 2 * U32 + 2.0 ** -16) + want.abs() * HALF_ULP[out.dtype] * 1.001 + TINY[out.dtype]
    assert out.isfinite().all()
    assert ((out.double() - want).abs() <= tol).all()
    none = (c["adapter_ids"] < 0) | (c["adapter_ids"] >= L)
    assert torch.equal(out[none], c["base"][none])


ADAPTER_SIZES = [(1, 1, 1, 1, 1), (1, 64, 64, 1, 16), (3, 7, 5, 2, 3), (16, 2048, 1536, 4, 16), (5, 256, 300, 3, 8), (128, 512, 1024, 64, 32),
                 (100, 1424, 2976, 13, 12), (300, 1040, 520, 5, 64), (64, 129, 131, 7, 17), (200, 4096, 256, 1, 128), (1000, 256, 256, 300, 4),
                 (257, 264, 1000, 3, 128), (40, 8192, 16, 2, 1), (1500, 512, 640, 6, 24)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,K,N,L,r", ADAPTER_SIZES)
def test_adapter_sizes(T, K, N, L, r, dtype):
    for x_i8 in (False, True):
        c = adapter_case(T, K, N, L, r, dtype, x_i8)
        check_adapter(c, ops.adapter_add(**c))


def test_adapter_one_adapter_none_and_out_of_range():
    for ids in (torch.full((70,), 2), torch.full((70,), -1), torch.full((70,), 5), torch.arange(70) % 9 - 2, torch.full((70,), 2 ** 31 - 1)):
        c = adapter_case(70, 512, 384, 5, 16, ids=ids.to(torch.int32).to(DEV), scaling=False)
        check_adapter(c, ops.adapter_add(**c))


def test_adapter_prompts_of_many_lengths():
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 300, 5, 1, 1]
    ids = torch.cat([torch.full((n,), i % 5 - 1) for i, n in enumerate(lens)]).to(torch.int32).to(DEV)
    for x_i8 in (False, True):
        c = adapter_case(len(ids), 640, 1000, 4, 48, x_i8=x_i8, ids=ids)
        check_adapter(c, ops.adapter_add(**c))


def test_adapter_in_place_strides_and_empty():
    c = adapter_case(90, 512, 768, 4, 16)
    want = ops.adapter_add(**c)
    base = c["base"].clone()
    got = ops.adapter_add(**dict(c, base=base), out=base)
    assert got is base and torch.equal(base, want)
    for off, pitch in ((0, 1536), (8, 776), (3, 771)):
        wide = lambda t, p: torch.empty(90 * p + 16, dtype=t.dtype, device=DEV)[off:].as_strided(t.shape, (p, 1)).copy_(t)  # noqa: E731
        s = dict(c, base=wide(c["base"], pitch), x=wide(c["x"], pitch))
        out = torch.empty(90 * pitch + 16, dtype=BF16, device=DEV)[off:].as_strided((90, 768), (pitch, 1))
        assert torch.equal(ops.adapter_add(**s, out=out), want) or off == 3   # other loads, the same sums up to their order
        check_adapter(s, out)
    check_adapter(c, ops.adapter_add(**dict(c, a=c["a"].transpose(1, 2).contiguous().transpose(1, 2))))
    one = dict(c, x=c["x"][:1].expand(90, 512))
    check_adapter(one, ops.adapter_add(**one))
    e = adapter_case(0, 64, 64, 2, 8)
    assert ops.adapter_add(**e).shape == (0, 64)


def test_adapter_nan_stays_in_its_row():
    c = adapter_case(60, 512, 384, 3, 16)
    c["x"][7, 100] = math.nan
    c["x"][8, 3] = math.inf
    c["base"][9, 5] = math.inf
    c["adapter_ids"][7:9] = 1
    out = ops.adapter_add(**c)
    keep = torch.ones(60, dtype=torch.bool, device=DEV)
    keep[7:10] = False
    assert out[7].isnan().all() and not out[8].isfinite().any() and not out[9, 5].isfinite()
    k = {n: (v[keep] if n in ("base", "x", "adapter_ids") else v) for n, v in c.items()}
    check_adapter(k, out[keep])
    # weights of an adapter that no token names do no harm
    c = adapter_case(60, 512, 384, 3, 16, ids=torch.zeros(60, dtype=torch.int32, device=DEV))
    c["a"][2], c["b"][1] = math.nan, math.inf
    check_adapter(c, ops.adapter_add(**c))


def test_adapter_offsets_beyond_32_bits():
    c = adapter_case(3, 64, 64, 2, 8, ids=torch.tensor([1, 0, 1], dtype=torch.int32, device=DEV))
    pitch = 1 << 30
    big = torch.zeros(3 * pitch, dtype=BF16, device=DEV).as_strided((3, 64), (pitch, 1))
    want = ops.adapter_add(**c)
    assert torch.equal(ops.adapter_add(**dict(c, x=big.copy_(c["x"]))), want)
    assert torch.equal(ops.adapter_add(**dict(c, base=big.copy_(c["base"]))), want)


def test_adapter_large_values_fp16():
    """The product of the first part may pass what fp16 holds; the result does not."""
    c = adapter_case(33, 512, 256, 2, 16, F16, ids=torch.arange(33, device=DEV, dtype=torch.int32) % 2)
    c["a"].mul_(2000)
    c["x"].mul_(40)
    c["b"].mul_(1e-3)
    check_adapter(c, ops.adapter_add(**c))


# ---------------------------------------------------------------------------------------------------------------------
# streams, graphs, repeated calls
# ---------------------------------------------------------------------------------------------------------------------

def calls():
    x, res, gamma = randn((70, 1024), 1, BF16), randn((70, 1024), 2, BF16), randn((1024,), 3, BF16)
    logits, bias = randn((70, 64), 4), randn((64,), 5, scale=0.1)
    c = adapter_case(70, 1024, 512, 5, 16)
    return [lambda s=None: ops.add_rms_norm_quant(x, gamma, residual=res, normed=True, stream=s),
            lambda s=None: ops.route_top_k(logits, 6, scoring="sigmoid", bias=bias, n_group=4, topk_group=2, group_score="top2", stream=s),
            lambda s=None: (ops.adapter_add(**c, stream=s),)]


def test_another_stream_and_repeated_calls_give_the_same():
    s = torch.cuda.Stream()
    for call in calls():
        want = call()
        torch.cuda.synchronize()
        got = call(s)
        s.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))
        with torch.cuda.stream(s):
            got = call()
        s.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))
        assert all(all(torch.equal(g, w) for g, w in zip(call(), want)) for _ in range(3))


def test_captured_calls_replay():
    for call in calls():
        want = call()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = call()
        for t in got:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_tensors_elsewhere_are_refused():
    x, gamma = torch.zeros(2, 8, dtype=BF16, device=DEV), torch.zeros(8, dtype=BF16)
    with pytest.raises(ValueError, match="CUDA device"):
        ops.add_rms_norm_quant(x, gamma)
    with pytest.raises(ValueError, match="CUDA device"):
        ops.route_top_k(x, 2, bias=torch.zeros(8))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("r", [8, 16, 24, 32, 64, 120, 128])
@pytest.mark.parametrize("T,K,N,L", [(1, 8, 8, 1), (4, 264, 256, 1), (7, 2048, 1000, 64), (128, 1024, 2976, 64), (256, 520, 264, 300), (200, 256, 8, 50)])
def test_adapter_few_tokens_of_many_adapters(T, K, N, L, r, dtype):
    for x_i8 in (False, True):
        c = adapter_case(T, K, N, L, r, dtype, x_i8, seed=T + r)
        check_adapter(c, ops.adapter_add(**c))
    # all tokens of one adapter, all without one
    for i in (0, -1):
        c["adapter_ids"] = torch.full_like(c["adapter_ids"], i)
        check_adapter(c, ops.adapter_add(**c))


@pytest.mark.parametrize("T,L,r", [(2048, 1, 64), (2500, 8, 16), (4100, 9, 40), (3000, 2, 128), (2048, 30, 8)])
def test_adapter_large_tiles(T, L, r):
    for x_i8 in (False, True):
        c = adapter_case(T, 1032, 520, L, r, BF16, x_i8)
        check_adapter(c, ops.adapter_add(**c))


def test_route_choices_that_hang_on_the_last_bits():
    """Sigmoid scores with a bias whose differences are of the size of their rounding: the choice is the one of scores that are rounded as
    the definition says (torch's elementwise operations round the same), ties go to the lowest id."""
    T, E = 512, 256
    base = randn((T, 1), 1) * 2
    for step in (0.0, 1e-7, 3e-7, 1e-6, 4e-6):
        logits = base + step * torch.randint(-3, 4, (T, E), device=DEV, generator=gen(2))
        for bias in (torch.zeros(E, device=DEV), torch.randint(-2, 3, (E,), device=DEV, generator=gen(3)) * 1e-7, torch.full((E,), 3.0, device=DEV)):
            choice = 1.0 / (1.0 + torch.exp(-logits)) + bias
            want = choice.sort(dim=1, descending=True, stable=True).indices[:, :8]
            assert torch.equal(ops.route_top_k(logits, 8, scoring="sigmoid", bias=bias)[1].long(), want)
            for score in ("max", "top2"):
                best = choice.view(T, 8, 32).sort(dim=2, descending=True).values
                rank = best[..., 0] if score == "max" else best[..., 0] + best[..., 1]
                place = rank.argsort(dim=1, descending=True, stable=True).argsort(dim=1)
                kept = torch.where((place < 3).repeat_interleave(32, 1), choice, -math.inf)
                want = kept.sort(dim=1, descending=True, stable=True).indices[:, :8]
                got = ops.route_top_k(logits, 8, scoring="sigmoid", bias=bias, n_group=8, topk_group=3, group_score=score)[1]
                assert torch.equal(got.long(), want)


@pytest.mark.parametrize("group_score", ["max", "top2"])
def test_route_groups_with_special_biases(group_score):
    T, E = 300, 64
    logits = randn((T, E), 1)
    logits[7, 8:24] = -math.inf
    bias = randn((E,), 2, scale=0.1)
    bias[3] = bias[9] = math.nan
    bias[17] = -math.inf
    bias[32:40] = math.nan       # a group without an expert
    for scoring in ("sigmoid", "softmax"):
        w, ids = route(logits, 5, scoring=scoring, bias=bias, n_group=8, topk_group=3, group_score=group_score)
        assert not torch.isin(ids.long(), torch.tensor([3, 9, 17] + list(range(32, 40)), device=DEV)).any()
        big = bias.nan_to_num(0.0, 0.0, 0.0)
        big[20] = math.inf
        _, ids = ops.route_top_k(logits, 5, scoring=scoring, bias=big, n_group=8, topk_group=3, group_score=group_score)
        live = torch.arange(T, device=DEV) != 7
        assert (ids[live, 0] == 20).all() and not (ids[7] == 20).any()
        big[60] = math.inf       # two groups without bounds, one of which stays
        _, ids = ops.route_top_k(logits, 5, scoring=scoring, bias=big, n_group=8, topk_group=1, group_score=group_score)
        assert ((ids[live] >= 16) & (ids[live] < 24)).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,r", [(40, 1), (40, 17), (8, 8)])
def test_adapter_infinite_activations(T, r, dtype):
    # one infinite element makes the row's first product infinite, and every result of the row with it, of the sign of b
    c = adapter_case(T, 64, 200, 2, r, dtype, ids=torch.arange(T, device=DEV, dtype=torch.int32) % 2)
    c["a"][:, :, 5] = 0.5
    c["b"] = c["b"].abs() + 0.25
    c["b"][:, 1::2] *= -1
    clean = ops.adapter_add(**c)
    c["x"][3, 5] = float("inf")
    out = ops.adapter_add(**c)
    want = torch.tensor([float("inf"), -float("inf")], device=DEV, dtype=dtype).repeat(100)
    assert torch.equal(out[3], want)
    others = torch.arange(T, device=DEV) != 3
    assert torch.equal(out[others], clean[others])


@pytest.mark.parametrize("x_i8", [False, True])
@pytest.mark.parametrize("T,K,N,L,r", [(1, 1, 1, 1, 1), (1, 1001, 133, 1, 7), (5, 264, 200, 2, 31), (30, 77, 136, 4, 65), (9, 1500, 64, 3, 12),
                                       (250, 17, 40, 20, 3), (16, 513, 96, 16, 127), (4, 6, 8, 1, 2), (70, 2047, 264, 9, 5)])
def test_adapter_few_tokens_on_any_boundary(T, K, N, L, r, x_i8):
    for dtype in (BF16, F16):
        c = adapter_case(T, K, N, L, r, dtype, x_i8)
        check_adapter(c, ops.adapter_add(**c))
        # the same rows farther apart, from the second element on, with NaN around them; weights that begin at an odd place
        wide = torch.full((T, K + 4), 99 if x_i8 else math.nan, device=DEV, dtype=c["x"].dtype)
        wide[:, 1:K + 1] = c["x"]
        moved = {}
        for n in ("a", "b"):
            store = torch.full((c[n].numel() + 2,), math.nan, device=DEV, dtype=dtype)
            store[1:-1] = c[n].flatten()
            moved[n] = store[1:-1].view(c[n].shape)
        check_adapter(c, ops.adapter_add(**{**c, **moved, "x": wide[:, 1:K + 1]}))


@pytest.mark.parametrize("T,L", [(300, 3), (1000, 60), (2100, 2)])
@pytest.mark.parametrize("r", [1, 7, 30, 61, 67, 127])
def test_adapter_ranks_on_any_boundary(T, L, r):
    for dtype, N in ((BF16, 264), (F16, 1000)):
        c = adapter_case(T, 520, N, L, r, dtype)
        check_adapter(c, ops.adapter_add(**c))
        store = torch.full((c["b"].numel() + 2,), math.nan, device=DEV, dtype=dtype)
        store[1:-1] = c["b"].flatten()
        check_adapter(c, ops.adapter_add(**{**c, "b": store[1:-1].view(c["b"].shape)}))


@pytest.mark.parametrize("size", [20.0, 50.0, 200.0, 1000.0, 3e4])
def test_route_groups_whose_largest_choices_cancel(size):
    """Groups are ranked by best + second, each rounded on the grid of its own size, which cancels out of the sum: two experts of a group with
    biases of +size and -size.  Ranks then differ by a few units of that grid or are equal, and must order as the definition rounds them."""
    T, G, E = 4096, 8, 64
    near = randn((T, 1, 2), 1) + 2e-6 * randn((T, G, 2), 2)
    logits = torch.full((T, G, E // G), -math.inf, device=DEV)
    logits[:, :, 2], logits[:, :, 5] = near[..., 0], near[..., 1]
    logits = logits.view(T, E)
    bias = torch.zeros(G, E // G, device=DEV)
    bias[:, 2], bias[:, 5] = size, -size
    bias = bias.view(E)
    choice = 1.0 / (1.0 + torch.exp(-logits)) + bias
    choice = torch.where(logits > -math.inf, choice, -math.inf)
    best = choice.view(T, G, -1).sort(dim=2, descending=True).values
    rank = best[..., 0] + best[..., 1]
    place = rank.argsort(dim=1, descending=True, stable=True).argsort(dim=1)
    for kept in (1, 3):
        left = torch.where((place < kept).repeat_interleave(E // G, 1), choice, -math.inf)
        want = left.sort(dim=1, descending=True, stable=True).indices[:, :kept]
        got = ops.route_top_k(logits, kept, scoring="sigmoid", bias=bias, n_group=G, topk_group=kept, group_score="top2")[1]
        assert torch.equal(got.long(), want)


def test_route_one_group_of_large_choices_among_small_ones():
    """The error of another group's rank counts as much as a group's own: one whose two choices are large and cancel, among small ones."""
    T, E = 4096, 32
    near = torch.rand(T, 1, device=DEV, generator=gen(1)) - 0.5
    logits = near + 3e-6 * randn((T, E), 2)
    bias = torch.zeros(E, device=DEV)
    logits[:, 8:16] = -math.inf
    logits[:, [9, 14]] = near + 3e-6 * randn((T, 2), 3)
    bias[9], bias[14] = 100.0, -100.0
    choice = torch.where(logits > -math.inf, 1.0 / (1.0 + torch.exp(-logits)) + bias, -math.inf)
    best = choice.view(T, 4, 8).sort(dim=2, descending=True).values
    rank = best[..., 0] + best[..., 1]
    place = rank.argsort(dim=1, descending=True, stable=True).argsort(dim=1)
    left = torch.where((place < 2).repeat_interleave(8, 1), choice, -math.inf)
    want = left.sort(dim=1, descending=True, stable=True).indices[:, :4]
    got = ops.route_top_k(logits, 4, scoring="sigmoid", bias=bias, n_group=4, topk_group=2, group_score="top2")[1].long()
    there = left.gather(1, want) > -math.inf
    assert torch.equal(got, torch.where(there, want, -1))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("r", [16, 61, 128])
@pytest.mark.parametrize("T,K,L", [(300, 136, 3), (300, 137, 80), (2100, 64, 4)])
def test_adapter_small_components_beside_large_ones(T, K, L, r, dtype):
    """x a^T is held in fp32 on its way into the second product: an output whose b has weight only on components that are 2^-20 of the row's
    largest is as exact as any other (fp16), and one in which large components nearly cancel too (bf16)."""
    N = 264
    ids = (torch.arange(T, device=DEV) % L).to(torch.int32)
    c = adapter_case(T, K, N, L, r, dtype, ids=ids)
    c["base"].zero_()
    if dtype == F16:
        c["a"].normal_(generator=gen(3))
        c["a"][:, 0] *= 2.0 ** 7
        c["a"][:, 1:] *= 2.0 ** -13
        c["b"].normal_(generator=gen(4)).mul_(16)
        c["b"][:, ::2, 0] = 0                       # every other channel hangs on the small components alone
    else:
        c["a"][:, 1:2] = c["a"][:, :1]
        c["a"][:, 1, 3::7] *= 1 + 2.0 ** -7         # the two components differ by about 2^-9
        c["b"][:, :, 1] = -c["b"][:, :, 0]
        c["b"][:, :, 2:] *= 2.0 ** -9
    check_adapter_fp32(c, ops.adapter_add(**c))


def check_adapter_fp32(c, out):
    """As check_adapter, without an allowance for fewer bits than fp32 has between the products: v of a row is off by its own sum's rounding, a
    result by that times |b|, by the second sum's and by its own rounding."""
    K, r, L = c["x"].shape[1], c["a"].shape[1], c["a"].shape[0]
    want, tol = c["base"].double(), torch.zeros_like(c["base"], dtype=torch.float64)
    for i in range(L):
        at = (c["adapter_ids"] == i).nonzero()[:, 0]
        x, a, b, s = c["x"][at].double(), c["a"][i].double(), c["b"][i].double(), c["scaling"][i].double()
        v, mag = s * (x @ a.t()), s * (x.abs() @ a.abs().t())
        want[at] += v @ b.t()
        # K / 16 + 8 steps of the first sum (one unit of the partial sum each), rank / 16 + 8 of the second, which the largest product bounds
        tol[at] = (mag @ b.abs().t()) * (K / 16 + 8) * 2 * U32 + (v.abs() @ b.abs().t()) * (r / 16 + 8) * 2 * U32
    tol += want.abs() * HALF_ULP[out.dtype] * 1.001 + TINY[out.dtype]
    # what passes the largest number of the type by more than its own error is an infinity
    most = torch.finfo(out.dtype).max
    over, fits = want.abs() - tol > most, want.abs() + tol < most
    assert torch.equal(out[over].double(), want[over].sign() * math.inf) and out[fits].isfinite().all()
    assert ((out.double() - want).abs() <= tol)[fits].all()


# More rows than find a place on the GPU together: a CTA goes through several, with the copies of the next under way.  Rows of one pack and of
# four a thread, of one warp and of many, on pack boundaries and off them.
NORM_MANY_ROWS = [(4096, 7168), (4096, 3500), (1500, 5001), (5000, 20), (2500, 1423), (6000, 1), (9500, 255), (2600, 2049), (1800, 4097)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,h", NORM_MANY_ROWS)
def test_norm_many_rows(rows, h, dtype):
    x, res = randn((rows, h), 1, dtype), randn((rows, h), 2, dtype, 3.0)
    gamma = randn((h,), 3, dtype, 0.2) + 1
    smooth = torch.rand(h, device=DEV, generator=gen(4)) + 0.5
    for residual, sm, normed in ((res, None, True), (None, smooth, False), (res, smooth, True), (None, None, False)):
        got = ops.add_rms_norm_quant(x, gamma, residual=residual, smooth=sm, eps=1e-5, normed=normed)
        check_norm(x, gamma, residual, sm, 1e-5, got)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,h", [(4096, 3584), (2500, 1423), (5000, 20)])
def test_norm_many_rows_in_place(rows, h, dtype):
    x, res, gamma = randn((rows, h), 1, dtype), randn((rows, h), 2, dtype), randn((h,), 3, dtype)
    want = ops.add_rms_norm_quant(x, gamma, residual=res, normed=True)
    check_norm(x, gamma, res, None, 1e-6, want)
    for into in ("residual", "x"):
        a, b = x.clone(), res.clone()
        got = ops.add_rms_norm_quant(a, gamma, residual=b, residual_out=b if into == "residual" else a, normed_out=a if into == "residual" else None)
        assert all(torch.equal(g, w) for g, w in zip(got[:3], want[:3]))
        if into == "residual":
            assert torch.equal(a, want[3])
    alone = x.clone()
    got = ops.add_rms_norm_quant(alone, gamma, normed_out=alone)
    check_norm(x, gamma, None, None, 1e-6, got)


@pytest.mark.parametrize("rows,h,pitch", [(5000, 100, 103), (5000, 100, 96), (2500, 1423, 1429), (1200, 7000, 7007), (3000, 1024, 2048)])
def test_norm_many_rows_apart(rows, h, pitch):
    """Rows that do not begin where the last one ends, behind one another or into one another; nothing lies behind the last one."""
    for dtype in (BF16, F32):
        at = lambda seed, p, n: randn(((rows - 1) * p + n,), seed, dtype).as_strided((rows, n), (p, 1))  # noqa: E731
        x, res, gamma = at(1, pitch, h), at(2, pitch, h), randn((h,), 3, dtype)
        check_norm(x, gamma, res, None, 1e-6, ops.add_rms_norm_quant(x, gamma, residual=res, normed=True))
        if pitch >= h:   # outputs between the rows of which nothing may be written
            out = torch.full((rows * pitch,), 7.0, dtype=dtype, device=DEV)
            view = out[:(rows - 1) * pitch + h].as_strided((rows, h), (pitch, 1))
            check_norm(x, gamma, res, None, 1e-6, ops.add_rms_norm_quant(x, gamma, residual=res, normed_out=view))
            assert (out.view(rows, pitch)[:, h:] == 7.0).all()


# ---------------------------------------------------------------------------------------------------------------------
# adapter_add's two ways: a few tokens on the CUDA cores, tiles of 16, 64 or 128 tokens on the tensor cores
# ---------------------------------------------------------------------------------------------------------------------

def adapter_way(c):
    """"few", or the tokens of a tile, for calls of these sizes (the way does not hang on the ids), from what one leaves in its workspace: behind
    the status (256 bytes) the tiles' way keeps the number of tiles, in 256 bytes of their own; the other way keeps x a^T there."""
    T, c = len(c["base"]), dict(c, adapter_ids=torch.zeros_like(c["adapter_ids"]))
    need = ops.adapter_add(**c, return_workspace=True)[1].numel()
    ws = torch.full((need,), 0x5a, dtype=torch.uint8, device=DEV)
    ops.adapter_add(**c, workspace=ws)
    ops.check_status(ws)
    head = ws[256:512].cpu()
    if not (head[4:] == 0x5a).all():
        return "few"
    return next(t for t in (16, 64, 128) if (T + t - 1) // t == int(head[:4].view(torch.int32)))


# tokens, K, adapters, rank and the way that these sizes take; a K that is no multiple of 8 keeps few tokens off the CUDA cores
ADAPTER_WAYS = [(60, 512, 3, 16, "few"), (60, 511, 3, 16, 64), (70, 511, 5, 16, 16), (300, 512, 60, 16, 16), (400, 512, 3, 16, 64), (400, 513, 3, 31, 64),
                (300, 512, 3, 128, 64), (2100, 512, 2, 16, 128), (2300, 512, 4, 61, 128)]


@pytest.mark.parametrize("T,K,L,r,way", ADAPTER_WAYS)
def test_adapter_ways_are_the_ones_that_are_meant(T, K, L, r, way):
    for dtype, x_i8 in ((BF16, False), (F16, True)):
        c = adapter_case(T, K, 264, L, r, dtype, x_i8, ids=(torch.arange(T, device=DEV) % L).to(torch.int32))
        assert adapter_way(c) == way
        check_adapter(c, ops.adapter_add(**c))


@pytest.mark.parametrize("T,K,L,r,way", ADAPTER_WAYS)
def test_adapter_ways_nan_and_infinities_stay_in_their_rows(T, K, L, r, way):
    for x_i8 in (False, True):
        ids = (torch.arange(T, device=DEV) % (L + 1) - 1).to(torch.int32)
        c = adapter_case(T, K, 264, L, r, x_i8=x_i8, ids=ids)
        ops.adapter_add(**dict(c, x=torch.full_like(c["x"], 127) if x_i8 else torch.full_like(c["x"], math.nan)))   # NaN left behind on the chip
        clean = ops.adapter_add(**c)
        ids[7], ids[8], ids[9] = 0, 1, 1
        if x_i8:
            c["x_scale"][7], c["x_scale"][8] = math.nan, math.inf
        else:
            c["x"][7, 100], c["x"][8, 3] = math.nan, math.inf
        c["base"][9, 5] = math.inf
        out = ops.adapter_add(**c)
        assert out[7].isnan().all() and not out[8].isfinite().any() and out[9, 5] == math.inf
        keep = torch.ones(T, dtype=torch.bool, device=DEV)
        keep[7:10] = False
        assert torch.equal(out[keep], clean[keep])
        check_adapter({n: (v[keep] if n in ("base", "x", "adapter_ids", "x_scale") and v is not None else v) for n, v in c.items()}, out[keep])
        # weights of adapters that no token names
        c = adapter_case(T, K, 264, L, r, x_i8=x_i8, ids=torch.full_like(ids, 1))
        want = ops.adapter_add(**c)
        c["a"][0], c["b"][0], c["scaling"][0] = math.nan, math.inf, math.nan
        assert torch.equal(ops.adapter_add(**c), want)
        check_adapter(dict(c, a=c["a"].nan_to_num(), b=c["b"].nan_to_num(), scaling=c["scaling"].nan_to_num()), want)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,K,L,r,way", ADAPTER_WAYS)
def test_adapter_ways_infinite_activations(T, K, L, r, way, dtype):
    c = adapter_case(T, K, 200, L, r, dtype, ids=(torch.arange(T, device=DEV) % L).to(torch.int32))
    c["a"][:, :, 5] = 0.5
    c["b"] = c["b"].abs() + 0.25
    c["b"][:, 1::2] *= -1
    clean = ops.adapter_add(**c)
    c["x"][3, 5] = math.inf
    out = ops.adapter_add(**c)
    assert torch.equal(out[3], torch.tensor([math.inf, -math.inf], device=DEV, dtype=dtype).repeat(100))
    others = torch.arange(T, device=DEV) != 3
    assert torch.equal(out[others], clean[others])


@pytest.mark.parametrize("T,K,L,r,way", ADAPTER_WAYS)
def test_adapter_ways_large_values_fp16(T, K, L, r, way):
    c = adapter_case(T, K, 264, L, r, F16, ids=(torch.arange(T, device=DEV) % L).to(torch.int32))
    c["a"].mul_(2000)
    c["x"].mul_(40)
    c["b"].mul_(1e-3)
    check_adapter(c, ops.adapter_add(**c))


@pytest.mark.parametrize("T,K,L,r,way", ADAPTER_WAYS)
def test_adapter_ways_one_adapter_none_and_out_of_range(T, K, L, r, way):
    for ids in (torch.full((T,), L - 1), torch.full((T,), -1), torch.full((T,), L), torch.arange(T) % (L + 4) - 2, torch.full((T,), 2 ** 31 - 1),
                torch.full((T,), -2 ** 31)):
        c = adapter_case(T, K, 264, L, r, ids=ids.to(torch.int32).to(DEV), scaling=False)
        check_adapter(c, ops.adapter_add(**c))


@pytest.mark.parametrize("T,K,L,r,way", ADAPTER_WAYS)
def test_adapter_ways_in_place_and_strides(T, K, L, r, way):
    for N in (264, 261):
        c = adapter_case(T, K, N, L, r)
        want = ops.adapter_add(**c)
        check_adapter(c, want)
        base = c["base"].clone()
        assert ops.adapter_add(**dict(c, base=base), out=base) is base and torch.equal(base, want)
        for off, pitch in ((0, 1024), (8, 1040), (3, 777)):
            wide = lambda t: torch.full((T * pitch + 16,), 3.0, dtype=t.dtype, device=DEV)[off:off + T * pitch]  # noqa: E731
            rows = lambda t, n: t.view(T, pitch)[:, :n]  # noqa: E731
            x, base = rows(wide(c["x"]), K).copy_(c["x"]), wide(c["base"])
            out = rows(base, N).copy_(c["base"])
            assert ops.adapter_add(**dict(c, base=out, x=x), out=out) is out
            check_adapter(c, out)
            assert (base.view(T, pitch)[:, N:] == 3.0).all()


@pytest.mark.parametrize("T,K,L,r,pitch", [(3, 63, 2, 8, 1 << 30), (300, 64, 2, 8, 1 << 23), (300, 64, 60, 8, 1 << 23)])
def test_adapter_ways_offsets_beyond_32_bits(T, K, L, r, pitch):
    c = adapter_case(T, K, 64, L, r, ids=(torch.arange(T, device=DEV) % (L + 1) - 1).to(torch.int32))
    assert adapter_way(c) == (16 if L == 60 or T == 3 else 64)
    big = torch.zeros((T - 1) * pitch + 64, dtype=BF16, device=DEV)
    rows = lambda n: big.as_strided((T, n), (pitch, 1))  # noqa: E731
    want = ops.adapter_add(**c)
    check_adapter(c, want)
    assert torch.equal(ops.adapter_add(**dict(c, x=rows(K).copy_(c["x"]))), want)
    rows(64).copy_(c["base"])
    assert torch.equal(ops.adapter_add(**dict(c, base=rows(64))), want)
    assert torch.equal(ops.adapter_add(**dict(c, base=rows(64)), out=rows(64)), want)


@pytest.mark.parametrize("T,K,L,r,way", ADAPTER_WAYS)
def test_adapter_ways_streams_and_replays_with_other_ids(T, K, L, r, way):
    c = adapter_case(T, K, 264, L, r)
    want = ops.adapter_add(**c)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = ops.adapter_add(**c, stream=s)
    s.synchronize()
    assert torch.equal(got, want)
    with torch.cuda.stream(s):
        got = ops.adapter_add(**c)
    s.synchronize()
    assert torch.equal(got, want) and all(torch.equal(ops.adapter_add(**c), want) for _ in range(3))
    torch.cuda.synchronize()
    # which tokens share an adapter is found anew in every replay, for any distribution of them
    live = dict(c, adapter_ids=c["adapter_ids"].clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.adapter_add(**live)
    at = torch.arange(T, device=DEV)
    for ids in (c["adapter_ids"], at % L, at * 0, at * 0 - 1, at * (L + 2) // T - 1, at % (L + 1) - 1, c["adapter_ids"].flip(0), at * 0 + L - 1):
        live["adapter_ids"].copy_(ids)
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        fresh = dict(c, adapter_ids=ids.to(torch.int32))
        assert torch.equal(got, ops.adapter_add(**fresh))
        check_adapter(fresh, got)


@pytest.mark.parametrize("T,L,r", [(8192, 5, 8), (8193, 3, 8), (16384, 40, 8), (20000, 1500, 4), (9000, 1024, 4), (3000, 16384, 2), (300, 12000, 4)])
def test_adapter_many_tokens_and_many_adapters(T, L, r):
    """More tokens than the plan keeps in registers, more adapters than it has threads, and than its counters fit the usual shared memory."""
    for ids in (torch.randint(-1, L, (T,), device=DEV, generator=gen(1)), torch.arange(T, device=DEV) * L // T, torch.arange(T, device=DEV) % 2 * (L - 1)):
        c = adapter_case(T, 72, 72, L, r, ids=ids.to(torch.int32))
        # as check_adapter, without a loop over thousands of adapters
        at = c["adapter_ids"].long().clamp_min(0)
        x, a, b, s = c["x"].double(), c["a"].double()[at], c["b"].double()[at], c["scaling"].double()[at, None]
        s = torch.where(c["adapter_ids"][:, None] < 0, 0.0, s)
        delta = lambda x, a, b: s * torch.einsum("tr,tnr->tn", torch.einsum("tk,trk->tr", x, a), b)  # noqa: E731
        want, mag = c["base"].double() + delta(x, a, b), delta(x.abs(), a.abs(), b.abs())
        out = ops.adapter_add(**c)
        tol = mag * (72 / 16 + r / 16 + 8) * 2 * U32 + want.abs() * HALF_ULP[BF16] * 1.001 + TINY[BF16]
        assert ((out.double() - want).abs() <= tol).all()
        assert torch.equal(out[c["adapter_ids"] < 0], c["base"][c["adapter_ids"] < 0])


def test_results_that_do_not_fit_raise_what_torch_raises():
    x = torch.zeros((1, 65528), dtype=BF16, device=DEV).expand(1 << 29, 65528)   # 32 TiB of results
    with pytest.raises(torch.OutOfMemoryError):
        ops.add_rms_norm_quant(x, x[0])
    with pytest.raises(torch.OutOfMemoryError):
        ops.route_top_k(torch.zeros((1, 64), device=DEV).expand(1 << 40, 64), 32)
    assert torch.isfinite(ops.route_top_k(torch.zeros((2, 64), device=DEV), 2)[0]).all()
