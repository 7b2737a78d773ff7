"""Refusals of add_rms_norm_quant, route_top_k and adapter_add: what their first phases, which need no device, check and report.  Host
tensors stand in for device tensors; a call whose arguments are in order is refused for that at the end."""
import ctypes as C

import pytest
import torch

import ops_transformer_b200 as ops
from ops_transformer_b200 import _lib, acl

NULLPTR, INVALID = 161001, 161002
BF16, F16, F32, I8, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.int32


def status(call):
    """The aclnnStatus of a refused call, 0 if only the tensors' place is wrong."""
    try:
        call()
    except acl.AclnnError as err:
        return err.status
    except ValueError as err:
        assert "CUDA device" in str(err)
        return 0
    raise AssertionError("host tensors were accepted")


def e(*shape, dtype=BF16):
    return torch.empty(shape, dtype=dtype)


def norm(**kw):
    args = dict(x=e(4, 64), gamma=e(64), residual=e(4, 64), smooth=e(64, dtype=F32), eps=1e-6, normed=True)
    args.update(kw)
    return status(lambda: ops.add_rms_norm_quant(**args))


@pytest.mark.parametrize("kw", [
    {}, dict(residual=None), dict(smooth=None), dict(normed=False), dict(gamma=e(64, dtype=F32)), dict(x=e(4, 128)[:, ::2]),
    dict(x=e(0, 64), residual=None), dict(x=e(1, 64).expand(4, 64)), dict(q=e(4, 128, dtype=I8)[:, ::2]),
    dict(x=e(2, 1, dtype=F32), gamma=e(1, dtype=F32), residual=None, smooth=None), dict(x=e(1, 65535), gamma=e(65535), residual=None, smooth=None)])
def test_norm_accepts(kw):
    assert norm(**kw) == 0


@pytest.mark.parametrize("kw", [
    dict(x=e(4, 8, 8)), dict(x=e(64)), dict(x=e(4, 64, dtype=torch.int32)), dict(x=e(4, 64, dtype=F16)), dict(gamma=e(63)), dict(gamma=e(1, 64)),
    dict(gamma=e(64, dtype=F16)), dict(residual=e(5, 64)), dict(residual=e(4, 64, dtype=F32)), dict(smooth=e(64)), dict(smooth=e(32, dtype=F32)),
    dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(q=e(4, 64)), dict(q=e(4, 32, dtype=I8)),
    dict(scale=e(4)), dict(scale=e(5, dtype=F32)), dict(residual_out=e(4, 64, dtype=F32)), dict(normed_out=e(4, 65)),
    dict(x=e(4, 0), gamma=e(0), residual=None, smooth=None), dict(x=e(1, 65536), gamma=e(65536), residual=None, smooth=None)])
def test_norm_refuses(kw):
    assert norm(**kw) == INVALID


def test_norm_refuses_what_is_missing():
    assert norm(residual=None, residual_out=e(4, 64)) == NULLPTR
    for gone in ("x", "gamma", "q", "scale"):
        t = dict(x=e(4, 64), gamma=e(64), q=e(4, 64, dtype=I8), scale=e(4, dtype=F32))
        t[gone] = None
        words = _lib.describe_call("tttttttti", t["x"], None, t["gamma"], None, t["q"], t["scale"], None, None, acl._float_bits(1e-6))
        res = _lib.CallResult()
        rc = _lib.lib().gmmB200Call(_lib.OP_ADD_RMS_NORM_QUANT | _lib.OP_PLAN_ONLY, words, len(words) // 8, None, 0, None, None, C.byref(res))
        assert rc == NULLPTR and gone in _lib.last_error()


def route(logits=None, top_k=4, **kw):
    return status(lambda: ops.route_top_k(e(6, 32, dtype=F32) if logits is None else logits, top_k, **kw))


@pytest.mark.parametrize("kw", [
    {}, dict(logits=e(6, 32)), dict(logits=e(6, 32, dtype=F16)), dict(logits=e(0, 32)), dict(scoring="sigmoid"), dict(bias=e(32, dtype=F32)),
    dict(n_group=4, topk_group=2), dict(n_group=32, topk_group=4, group_score="top2"), dict(token_mask=e(6, dtype=torch.bool)),
    dict(token_mask=e(6, dtype=I8)), dict(ids_dtype=torch.int64), dict(logits=e(6, 64)[:, 1:33]), dict(logits=e(2, 1024), top_k=32),
    dict(logits=e(2, 1), top_k=1)])
def test_route_accepts(kw):
    assert route(**kw) == 0


@pytest.mark.parametrize("kw", [
    dict(logits=e(32)), dict(logits=e(6, 32, dtype=I32)), dict(logits=e(6, 1025), top_k=2), dict(logits=e(6, 0), top_k=1), dict(top_k=0), dict(top_k=33),
    dict(logits=e(6, 3)), dict(bias=e(32)), dict(bias=e(31, dtype=F32)), dict(n_group=5, topk_group=2), dict(n_group=0), dict(n_group=4, topk_group=0),
    dict(n_group=4, topk_group=5), dict(n_group=8, topk_group=1, top_k=5), dict(logits=e(6, 64), n_group=64, topk_group=8), dict(token_mask=e(5, dtype=I8)),
    dict(token_mask=e(6, dtype=F32)), dict(ids_dtype=torch.int8), dict(scale=float("inf")), dict(weights=e(6, 4)), dict(weights=e(6, 5, dtype=F32)),
    dict(ids=e(7, 4, dtype=I32))])
def test_route_refuses(kw):
    assert route(**kw) == INVALID


def test_route_names_are_checked():
    for kw in (dict(scoring="relu"), dict(group_score="mean")):
        with pytest.raises(ValueError, match="unknown"):
            ops.route_top_k(e(6, 32), 4, **kw)


def adapter(**kw):
    args = dict(base=e(6, 48), x=e(6, 64), a=e(3, 16, 64), b=e(3, 48, 16), adapter_ids=e(6, dtype=I32), x_scale=None, scaling=e(3, dtype=F32))
    args.update(kw)
    return status(lambda: ops.adapter_add(**args))


@pytest.mark.parametrize("kw", [
    {}, dict(scaling=None), dict(x=e(6, 64, dtype=I8), x_scale=e(6, dtype=F32)), dict(x=e(6, 128)[:, :64]), dict(out=e(6, 96)[:, 48:]),
    dict(base=e(0, 48), x=e(0, 64), adapter_ids=e(0, dtype=I32)), dict(a=e(3, 128, 64), b=e(3, 48, 128)), dict(a=e(3, 1, 64), b=e(3, 48, 1)),
    dict(base=e(6, 48, dtype=F16), x=e(6, 64, dtype=F16), a=e(3, 16, 64, dtype=F16), b=e(3, 48, 16, dtype=F16))])
def test_adapter_accepts(kw):
    assert adapter(**kw) == 0


@pytest.mark.parametrize("kw", [
    dict(base=e(6, 48, dtype=F32)), dict(x=e(6, 64, dtype=F16)), dict(x=e(6, 64, dtype=F32)), dict(x=e(5, 64)), dict(x=e(6, 65)), dict(x_scale=e(6, dtype=F32)),
    dict(x=e(6, 64, dtype=I8), x_scale=e(5, dtype=F32)), dict(x=e(6, 64, dtype=I8), x_scale=e(6)), dict(a=e(3, 16, 64, dtype=F16)),
    dict(b=e(3, 48, 16, dtype=F32)), dict(b=e(2, 48, 16)), dict(b=e(3, 16, 48)), dict(a=e(3, 129, 64), b=e(3, 48, 129)), dict(a=e(3, 0, 64), b=e(3, 48, 0)),
    dict(a=e(0, 16, 64), b=e(0, 48, 16)), dict(adapter_ids=e(6, dtype=torch.int64)), dict(adapter_ids=e(7, dtype=I32)), dict(scaling=e(3)),
    dict(scaling=e(4, dtype=F32)), dict(out=e(6, 49)), dict(out=e(6, 48, dtype=F16)), dict(a=e(3, 16)), dict(base=e(48))])
def test_adapter_refuses(kw):
    assert adapter(**kw) == INVALID


def test_adapter_refuses_what_is_missing():
    assert adapter(x=e(6, 64, dtype=I8)) == NULLPTR


@pytest.mark.parametrize("op", [_lib.OP_ADD_RMS_NORM_QUANT, _lib.OP_ROUTE_TOP_K, _lib.OP_ADAPTER_ADD])
@pytest.mark.parametrize("words", [[], [2, 0, 2, 2, 4], [9], [1, 0, 2, 2, 4, 1, 12], [-1] * 40])
def test_malformed_descriptions_are_refused(op, words):
    res = _lib.CallResult()
    packed = (C.c_int64 * max(len(words), 1))(*words)
    assert _lib.lib().gmmB200Call(op, packed, len(words), None, 0, None, None, C.byref(res)) == INVALID
    assert "malformed" in _lib.last_error()


def test_second_phase_takes_an_executor_once_and_of_its_own_operator():
    L = _lib.lib()

    def plan():
        x, gamma, q, scale = e(0, 64), e(64), e(0, 64, dtype=I8), e(0, dtype=F32)
        words = _lib.describe_call("tttttttti", x, None, gamma, None, q, scale, None, None, acl._float_bits(1e-6))
        res = _lib.CallResult()
        assert L.gmmB200Call(_lib.OP_ADD_RMS_NORM_QUANT | _lib.OP_PLAN_ONLY, words, len(words) // 8, None, 0, None, None, C.byref(res)) == 0
        assert res.stage == _lib.STAGE_PLANNED and res.workspaceSize == 0
        return C.c_void_p(res.executor)

    ex = plan()   # no rows: nothing is enqueued
    assert L.gmmB200AddRmsNormQuant(None, 0, ex, None) == 0
    assert L.gmmB200AddRmsNormQuant(None, 0, ex, None) == INVALID
    assert L.gmmB200RouteTopK(None, 0, plan(), None) == INVALID
    assert L.gmmB200AdapterAdd(None, 0, None, None) == NULLPTR


def test_numbers_are_read_anew_in_every_call():
    """eps and scale may be anything that is a number; a tensor's value is the one that it has at the call."""
    import struct
    bits = lambda v: struct.unpack("<I", struct.pack("<f", v))[0]  # noqa: E731
    t = torch.tensor(2.5)
    assert acl._float_bits(t) == bits(2.5)
    t.fill_(1.0)
    assert acl._float_bits(t) == bits(1.0)
    assert [acl._float_bits(v) for v in (0.0, -0.0, 0.0, 1, True, 1.0)] == [0, 1 << 31, 0] + [bits(1.0)] * 3
    with pytest.raises(struct.error):
        acl._float_bits("1")


def _planned(op, words):
    res = _lib.CallResult()
    assert _lib.lib().gmmB200Call(op | _lib.OP_PLAN_ONLY, words, len(words) // 8, None, 0, None, None, C.byref(res)) == 0, _lib.last_error()
    return C.c_void_p(res.executor), res.workspaceSize


@pytest.mark.parametrize("shift", [1, 2, 4, 8])
def test_workspaces_that_kernels_cannot_use_are_refused_before_anything_is_enqueued(shift):
    """Copies of strided views and partial sums are read and written by whole elements and packs."""
    apart = lambda *s, dtype=BF16: torch.empty(s[:-1] + (2 * s[-1],), dtype=dtype)[..., ::2]  # noqa: E731
    x, gamma, q, scale = apart(4, 64), e(64), e(4, 64, dtype=I8), e(4, dtype=F32)
    logits, weights, ids = apart(6, 32, dtype=F32), e(6, 4, dtype=F32), e(6, 4, dtype=I32)
    base, ax, a, b = e(6, 48), apart(6, 64), e(3, 16, 64), e(3, 48, 16)
    calls = [("gmmB200AddRmsNormQuant", _lib.OP_ADD_RMS_NORM_QUANT,
              _lib.describe_call("tttttttti", x, None, gamma, None, q, scale, None, None, acl._float_bits(1e-6))),
             ("gmmB200RouteTopK", _lib.OP_ROUTE_TOP_K, _lib.describe_call("tttttiiiiii", logits, None, None, weights, ids, 0, 1, 1, 0, 1, acl._float_bits(1.0))),
             ("gmmB200AdapterAdd", _lib.OP_ADAPTER_ADD, _lib.describe_call("tttttttt", base, ax, None, a, b, e(6, dtype=I32), None, base))]
    if shift < 4:   # the copy of the scales, for an operator whose workspace may begin on any boundary of 4 bytes
        calls.append(("aclnnGroupedMatmulV4", _lib.OP_GMM["V4"], _lib.describe_call(
            "tftttttiiiiil", e(4, 32, dtype=I8), (e(1, 32, 64, dtype=I8), 2, None), None, e(1, 64, dtype=F32), apart(4, dtype=F32),
            e(1, dtype=torch.int64), e(4, 64), 3, 0, 0, 0, 0, None)))
    for name, op, words in calls:
        ex, need = _planned(op, words)
        assert need > 0
        room = torch.empty(need + 64, dtype=torch.uint8)
        at = (room.data_ptr() + 15) // 16 * 16 + shift
        assert getattr(_lib.lib(), name)(at, need, ex, None) == INVALID
        assert "aligned" in _lib.last_error()


def test_tensors_off_their_elements_boundaries_are_refused():
    room = torch.empty(4096, dtype=torch.uint8)
    at = (room.data_ptr() + 15) // 16 * 16 + 1
    def moved(words, place):   # the tensor of `place` begins at an odd address
        w = list((C.c_int64 * (len(words) // 8)).from_buffer_copy(words))
        i = 0
        for _ in range(place):
            i += 1 if w[i] < 0 else 4 + 2 * w[i] + 1 + w[i + 4 + 2 * w[i]]
        w[i + 1] = at
        return (C.c_int64 * len(w))(*w), len(w)

    res = _lib.CallResult()
    for op, words, places in [
            (_lib.OP_ADD_RMS_NORM_QUANT, _lib.describe_call("tttttttti", e(2, 8), e(2, 8), e(8), e(8, dtype=F32), e(2, 8, dtype=I8), e(2, dtype=F32), e(2, 8),
                                                            e(2, 8), acl._float_bits(1e-6)), (0, 1, 2, 3, 5, 6, 7)),
            (_lib.OP_ROUTE_TOP_K, _lib.describe_call("tttttiiiiii", e(2, 8), e(8, dtype=F32), None, e(2, 2, dtype=F32), e(2, 2, dtype=I32), 0, 1, 1, 0, 1,
                                                     acl._float_bits(1.0)), (0, 1, 3, 4)),
            (_lib.OP_ADAPTER_ADD, _lib.describe_call("tttttttt", e(2, 8), e(2, 8, dtype=I8), e(2, dtype=F32), e(1, 4, 8), e(1, 8, 4), e(2, dtype=I32),
                                                     e(1, dtype=F32), e(2, 8)), (0, 2, 3, 4, 5, 6, 7))]:
        for place in places:
            w, n = moved(words, place)
            assert _lib.lib().gmmB200Call(op | _lib.OP_PLAN_ONLY, w, n, None, 0, None, None, C.byref(res)) == INVALID, place
            assert "aligned" in _lib.last_error()


def test_a_workspace_in_pieces_is_refused():
    with pytest.raises(ValueError, match="contiguous"):
        ops.adapter_add(e(6, 48), e(6, 64), e(3, 16, 64), e(3, 48, 16), e(6, dtype=I32), workspace=torch.empty(1, dtype=torch.uint8).expand(1 << 24))


def test_route_outputs_of_another_width_are_refused():
    for n in (3, 8):
        with pytest.raises(ValueError, match="top_k"):
            ops.route_top_k(e(6, 32, dtype=F32), 4, weights=e(6, n, dtype=F32), ids=e(6, n, dtype=I32))
    assert route(top_k=4, weights=e(6, 4, dtype=F32), ids=e(6, 4, dtype=I32)) == 0
    assert route(top_k=4, weights=e(6, 4, dtype=F32), ids=e(6, 8, dtype=I32)) == INVALID
