"""Refusals of quant_matmul, sandwich_norm_quant, expert_balance and expert_balance_grad: what their first phases, which need no device, check
and report.  Host tensors stand in for device tensors; a call whose arguments are in order is refused for that at the end."""
import ctypes as C

import pytest
import torch

import ops_transformer_b200 as ops
from ops_transformer_b200 import _lib, acl

NULLPTR, INVALID = 161001, 161002
BF16, F16, F32, I8, I32, I64 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.int32, torch.int64


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


def far(*shape, dtype):
    """A tensor of that shape with next to no memory: sizes at the limits."""
    return torch.empty(1, dtype=dtype).expand(shape)


def matmul(**kw):
    args = dict(x=e(6, 64, dtype=I8), weight=e(64, 48, dtype=I8), scale=e(48, dtype=F32), per_token_scale=e(6, dtype=F32), bias=None)
    args.update(kw)
    return status(lambda: ops.quant_matmul(**args))


@pytest.mark.parametrize("kw", [
    {}, dict(per_token_scale=None), dict(bias=e(48, dtype=F32)), dict(bias=e(48)), dict(bias=e(48, dtype=F16)), dict(scale=e(48)), dict(scale=e(48, dtype=F16)),
    dict(out_dtype=F16), dict(out_dtype=F32), dict(out=e(6, 96)[:, 48:]), dict(weight=e(48, 64, dtype=I8).t()), dict(weight=e(48, 128, dtype=I8)[:, 64:].t()),
    dict(weight=e(64, 96, dtype=I8)[:, ::2]), dict(x=e(6, 128, dtype=I8)[:, ::2]), dict(x=e(0, 64, dtype=I8), per_token_scale=e(0, dtype=F32)),
    dict(x=e(6, 1, dtype=I8), weight=e(1, 1, dtype=I8), scale=e(1, dtype=F32)), dict(x=far(1, 65535, dtype=I8), weight=far(65535, 2, dtype=I8), scale=e(2), per_token_scale=None)])
def test_matmul_accepts(kw):
    assert matmul(**kw) == 0


@pytest.mark.parametrize("kw", [
    dict(x=e(6, 64)), dict(weight=e(64, 48)), dict(weight=e(63, 48, dtype=I8)), dict(weight=e(48, 64, dtype=I8)), dict(weight=e(1, 64, 48, dtype=I8), out=e(6, 48)),
    dict(x=e(2, 3, 64, dtype=I8), out=e(6, 48)), dict(scale=e(47, dtype=F32)), dict(scale=e(1, 48, dtype=F32)), dict(scale=e(48, dtype=I32)),
    dict(per_token_scale=e(5, dtype=F32)), dict(per_token_scale=e(6)), dict(bias=e(47)), dict(bias=e(48, dtype=I32)), dict(out=e(6, 47)), dict(out=e(5, 48)),
    dict(out=e(6, 48, dtype=I32)), dict(out_dtype=I32), dict(x=e(6, 0, dtype=I8), weight=e(0, 48, dtype=I8)), dict(weight=e(64, 0, dtype=I8), scale=e(0, dtype=F32)),
    dict(x=far(1, 65536, dtype=I8), weight=far(65536, 48, dtype=I8), per_token_scale=None)])
def test_matmul_refuses(kw):
    assert matmul(**kw) == INVALID


def sandwich(**kw):
    args = dict(x=e(4, 64, dtype=F32), residual=e(4, 64), gamma=e(64), post_gamma=e(64), gate=e(64), smooth=e(64, dtype=F32), normed=True)
    args.update(kw)
    return status(lambda: ops.sandwich_norm_quant(**args))


@pytest.mark.parametrize("kw", [
    {}, dict(x=e(4, 64)), dict(post_gamma=None), dict(gate=None), dict(smooth=None), dict(normed=False), dict(quant=False), dict(gate=e(4, 1)), dict(gate=e(4, 64)),
    dict(gate=e(1, 64)), dict(gate=e(1, 1)), dict(gate=e(4, 8)[:, 3:4]), dict(gate=e(64, 4).t()), dict(gamma=e(64, dtype=F32), post_gamma=e(64, dtype=F32)),
    dict(gamma=None, quant=False, normed=False, smooth=None), dict(gate_act="sigmoid"), dict(gate_act="tanh"), dict(post_eps=1e-3),
    dict(x=e(0, 64, dtype=F32), residual=e(0, 64)), dict(x=e(4, 128, dtype=F32)[:, ::2]), dict(residual=e(4, 128)[:, :64]), dict(residual_scale=0, block_scale=-2),
    dict(x=far(2, 65535, dtype=F32), residual=far(2, 65535, dtype=BF16), gamma=e(65535), post_gamma=None, gate=None, smooth=None)])
def test_sandwich_accepts(kw):
    assert sandwich(**kw) == 0


@pytest.mark.parametrize("kw", [
    dict(residual=e(64)), dict(residual=e(4, 64, dtype=I32)), dict(x=e(4, 64, dtype=F16)), dict(x=e(5, 64)), dict(x=e(4, 63)), dict(gamma=e(63)), dict(gamma=e(64, dtype=F32)),
    dict(gamma=e(64, dtype=F16), post_gamma=e(64, dtype=F16)), dict(post_gamma=e(1, 64)), dict(gate=e(63)), dict(gate=e(3, 64)), dict(gate=e(4, 2)), dict(gate=e(64, dtype=F32)),
    dict(gate=e(4, 64, 1)), dict(smooth=e(64)), dict(eps=0.0), dict(eps=float("nan")), dict(post_eps=-1.0), dict(post_eps=float("inf")), dict(residual_scale=float("inf")),
    dict(block_scale=float("nan")), dict(q=e(4, 64)), dict(q=e(4, 63, dtype=I8)), dict(scale=e(4)), dict(residual_out=e(4, 64, dtype=F32)), dict(normed_out=e(4, 65)),
    dict(x=e(4, 0, dtype=F32), residual=e(4, 0), gamma=e(0), post_gamma=None, gate=None, smooth=None)])
def test_sandwich_refuses(kw):
    assert sandwich(**kw) == INVALID


def plan(op, kinds, *items):
    words = _lib.describe_call(kinds, *items)
    res = _lib.CallResult()
    return _lib.lib().gmmB200Call(op | _lib.OP_PLAN_ONLY, words, len(words) // 8, None, 0, None, None, C.byref(res)), res


SANDWICH_KINDS = "ttttttttttiiiii"


def sandwich_items(**kw):
    t = dict(x=e(4, 64), residual=e(4, 64), gamma=e(64), post=None, gate=None, smooth=None, q=e(4, 64, dtype=I8), scale=e(4, dtype=F32), out=e(4, 64), normed=None)
    t.update(kw)
    one, eps = acl._float_bits(1.0), acl._float_bits(1e-6)
    return (*t.values(), 0, one, one, eps, eps)


def test_sandwich_refuses_what_is_missing():
    assert sandwich(gamma=None, normed=False) == NULLPTR and sandwich(gamma=None, quant=False) == NULLPTR
    for kw in (dict(x=None), dict(residual=None), dict(q=None), dict(scale=None), dict(q=None, scale=None, out=None)):
        rc, _ = plan(_lib.OP_SANDWICH_NORM_QUANT, SANDWICH_KINDS, *sandwich_items(**kw))
        assert rc == NULLPTR, kw
    for act in (-1, 3):
        items = list(sandwich_items())
        items[10] = act
        assert plan(_lib.OP_SANDWICH_NORM_QUANT, SANDWICH_KINDS, *items)[0] == INVALID
    with pytest.raises(ValueError, match="gate_act"):
        ops.sandwich_norm_quant(e(4, 64), e(4, 64), e(64), gate_act="silu")


def test_matmul_refuses_what_is_missing():
    for gone in range(6):
        items = [e(6, 64, dtype=I8), e(64, 48, dtype=I8), e(48, dtype=F32), e(6, dtype=F32), None, e(6, 48)]
        items[gone] = None
        assert plan(_lib.OP_QUANT_MATMUL, "tttttt", *items)[0] == (0 if gone in (3, 4) else NULLPTR)


def balance(logits=None, ids=None, **kw):
    return status(lambda: ops.expert_balance(e(6, 32, dtype=F32) if logits is None else logits, e(6, 4, dtype=I32) if ids is None else ids, **kw))


@pytest.mark.parametrize("kw", [
    {}, dict(logits=e(6, 32)), dict(logits=e(6, 32, dtype=F16)), dict(ids=e(6, 4, dtype=I64)), dict(scoring="sigmoid"), dict(coefficient=0), dict(token_mask=e(6, dtype=torch.bool)),
    dict(token_mask=e(6, dtype=I8)), dict(cu_seqlens=e(4, dtype=I32)), dict(cu_seqlens=e(2, dtype=I32)), dict(logits=e(0, 32), ids=e(0, 4, dtype=I32)),
    dict(logits=e(6, 64)[:, 1:33]), dict(ids=e(6, 8, dtype=I32)[:, ::2]), dict(logits=e(6, 1024)), dict(logits=e(6, 1), ids=e(6, 1, dtype=I32)),
    dict(cu_seqlens=far(65536, dtype=I32))])
def test_balance_accepts(kw):
    assert balance(**kw) == 0


@pytest.mark.parametrize("kw", [
    dict(logits=e(32)), dict(logits=e(6, 32, dtype=I32)), dict(logits=e(6, 1025)), dict(logits=e(6, 0)), dict(ids=e(6, dtype=I32)), dict(ids=e(5, 4, dtype=I32)), dict(ids=e(6, 0, dtype=I32)),
    dict(ids=e(6, 4, dtype=I8)), dict(ids=e(6, 4, dtype=F32)), dict(ids=far(6, 1025, dtype=I32)), dict(token_mask=e(5, dtype=I8)), dict(token_mask=e(6, dtype=F32)),
    dict(cu_seqlens=e(1, dtype=I32)), dict(cu_seqlens=e(0, dtype=I32)), dict(cu_seqlens=e(4, dtype=I64)), dict(cu_seqlens=e(2, 2, dtype=I32)), dict(cu_seqlens=far(65537, dtype=I32)),
    dict(coefficient=float("inf")), dict(loss=e(2, dtype=F32)), dict(loss=e(1)), dict(counts=e(31, dtype=I64)), dict(counts=e(32, dtype=I32)), dict(weight=e(2, dtype=F32)),
    dict(weight=e(1)), dict(cu_seqlens=e(4, dtype=I32), counts=e(32, dtype=I64)), dict(cu_seqlens=e(4, dtype=I32), weight=e(4, dtype=F32))])
def test_balance_refuses(kw):
    assert balance(**kw) == INVALID


def grad(**kw):
    args = dict(logits=e(6, 32, dtype=F32), counts=e(32, dtype=I64), weight=e(1, dtype=F32))
    args.update(kw)
    return status(lambda: ops.expert_balance_grad(**args))


@pytest.mark.parametrize("kw", [
    {}, dict(logits=e(6, 32)), dict(scoring="sigmoid"), dict(grad_loss=e(dtype=F32)), dict(grad_loss=e(1, dtype=F32)), dict(grad=e(6, 64, dtype=F32)[:, :32]),
    dict(cu_seqlens=e(4, dtype=I32), counts=e(3, 32, dtype=I64), weight=e(3, dtype=F32)), dict(logits=e(0, 32, dtype=F32)), dict(token_mask=e(6, dtype=torch.bool))])
def test_balance_grad_accepts(kw):
    assert grad(**kw) == 0


@pytest.mark.parametrize("kw", [
    dict(logits=e(32, dtype=F32)), dict(counts=e(32, dtype=I32)), dict(counts=e(1, 32, dtype=I64)), dict(weight=e(dtype=F32)), dict(weight=e(2, dtype=F32)), dict(grad=e(6, 32)),
    dict(grad=e(6, 31, dtype=F32)), dict(grad_loss=e(2, dtype=F32)), dict(grad_loss=e(1)), dict(token_mask=e(7, dtype=I8)),
    dict(cu_seqlens=e(4, dtype=I32)), dict(cu_seqlens=e(4, dtype=I32), counts=e(4, 32, dtype=I64), weight=e(3, dtype=F32))])
def test_balance_grad_refuses(kw):
    assert grad(**kw) == INVALID


def test_balance_names_and_what_is_missing():
    for call in (ops.expert_balance, ops.expert_balance_grad):
        with pytest.raises(ValueError, match="scoring"):
            call(e(6, 32, dtype=F32), e(6, 4, dtype=I32), *([e(1, dtype=F32)] if call is ops.expert_balance_grad else []), scoring="relu")
    items = [e(6, 32, dtype=F32), e(6, 4, dtype=I32), None, None, e(dtype=F32), e(32, dtype=I64), e(1, dtype=F32)]
    for gone in range(7):
        these = list(items)
        these[gone] = None
        assert plan(_lib.OP_EXPERT_BALANCE, "tttttttii", *these, 0, acl._float_bits(1.0))[0] == (0 if gone in (2, 3) else NULLPTR)
    assert plan(_lib.OP_EXPERT_BALANCE, "tttttttii", *items, 2, acl._float_bits(1.0))[0] == INVALID
    items = [e(6, 32, dtype=F32), e(32, dtype=I64), e(1, dtype=F32), None, None, None, e(6, 32, dtype=F32)]
    for gone in (0, 1, 2, 6):
        these = list(items)
        these[gone] = None
        assert plan(_lib.OP_EXPERT_BALANCE_GRAD, "ttttttti", *these, 0)[0] == NULLPTR


NEW = [_lib.OP_QUANT_MATMUL, _lib.OP_SANDWICH_NORM_QUANT, _lib.OP_EXPERT_BALANCE, _lib.OP_EXPERT_BALANCE_GRAD]


@pytest.mark.parametrize("op", NEW)
@pytest.mark.parametrize("words", [[], [2, 0, 2, 2, 4], [9], [1, 0, 2, 2, 4, 1, 12], [-1] * 40])
def test_malformed_descriptions_are_refused(op, words):
    res = _lib.CallResult()
    packed = (C.c_int64 * max(len(words), 1))(*words)
    assert _lib.lib().gmmB200Call(op, packed, len(words), None, 0, None, None, C.byref(res)) == INVALID
    assert "malformed" in _lib.last_error()


def calls():
    """(operator, symbol, kinds, items) of a valid call of each; the tensors among the items that are wider than a byte."""
    one = acl._float_bits(1.0)
    return [(_lib.OP_QUANT_MATMUL, "gmmB200QuantMatmul", "tttttt", [e(6, 64, dtype=I8), e(64, 48, dtype=I8), e(48, dtype=F32), e(6, dtype=F32), e(48), e(6, 48)]),
            (_lib.OP_SANDWICH_NORM_QUANT, "gmmB200SandwichNormQuant", SANDWICH_KINDS,
             list(sandwich_items(post=e(64), gate=e(64), smooth=e(64, dtype=F32), normed=e(4, 64)))),
            (_lib.OP_EXPERT_BALANCE, "gmmB200ExpertBalance", "tttttttii",
             [e(200, 32, dtype=F32), e(200, 4, dtype=I32), None, e(3, dtype=I32), e(1, dtype=F32), e(2, 32, dtype=I64), e(2, dtype=F32), 0, one]),
            (_lib.OP_EXPERT_BALANCE_GRAD, "gmmB200ExpertBalanceGrad", "ttttttti",
             [e(6, 32, dtype=F32), e(2, 32, dtype=I64), e(2, dtype=F32), None, e(3, dtype=I32), e(1, dtype=F32), e(6, 32, dtype=F32), 0])]


def test_tensors_off_their_elements_boundaries_are_refused():
    for op, _, kinds, items in calls():
        for place, t in enumerate(items):
            if not isinstance(t, torch.Tensor) or t.element_size() == 1:
                continue
            room = torch.empty(t.numel() * t.element_size() + 64, dtype=torch.uint8)
            at = (room.data_ptr() + 15) // 16 * 16 + 1
            words = _lib.describe_call(kinds, *items)
            w = list((C.c_int64 * (len(words) // 8)).from_buffer_copy(words))
            i = 0
            for _ in range(place):
                i += 1 if w[i] < 0 else 4 + 2 * w[i] + 1 + w[i + 4 + 2 * w[i]]
            w[i + 1] = at
            res = _lib.CallResult()
            assert _lib.lib().gmmB200Call(op | _lib.OP_PLAN_ONLY, (C.c_int64 * len(w))(*w), len(w), None, 0, None, None, C.byref(res)) == INVALID, place
            assert "aligned" in _lib.last_error()


@pytest.mark.parametrize("shift", [1, 4, 8])
def test_workspaces_that_kernels_cannot_use_are_refused_before_anything_is_enqueued(shift):
    for op, name, kinds, items in calls():
        if op == _lib.OP_SANDWICH_NORM_QUANT:
            items[0] = e(4, 128)[:, ::2]   # its workspace holds copies of views
        if op == _lib.OP_EXPERT_BALANCE_GRAD:
            items[0] = e(6, 64, dtype=F32)[:, ::2]
        rc, res = plan(op, kinds, *items)
        assert rc == 0 and res.workspaceSize > 0, (name, _lib.last_error())
        room = torch.empty(res.workspaceSize + 64, dtype=torch.uint8)
        at = (room.data_ptr() + 15) // 16 * 16 + shift
        assert getattr(_lib.lib(), name)(at, res.workspaceSize, C.c_void_p(res.executor), None) == INVALID
        assert "aligned" in _lib.last_error()
        rc, res = plan(op, kinds, *items)
        assert getattr(_lib.lib(), name)(None, 0, C.c_void_p(res.executor), None) == INVALID
        assert "smaller" in _lib.last_error()


def test_calls_without_rows_plan_nothing():
    assert plan(_lib.OP_QUANT_MATMUL, "tttttt", e(0, 64, dtype=I8), e(64, 48, dtype=I8), e(48, dtype=F32), None, None, e(0, 48))[1].workspaceSize == 0
    assert plan(_lib.OP_EXPERT_BALANCE_GRAD, "ttttttti", e(0, 32), e(32, dtype=I64), e(1, dtype=F32), None, None, None, e(0, 32), 0)[1].workspaceSize == 0
