"""What the first phases of the operators of a block's exit say of workspaces and options, without a device."""
import ctypes as C

import pytest
import torch

import ops_transformer_b200 as ops
from ops_transformer_b200 import _lib, acl

INVALID = 161002
BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


def e(*shape, dtype=BF16):
    return torch.empty(shape, dtype=dtype)


def plan(op, kinds, *items):
    words = _lib.describe_call(kinds, *items)
    res = _lib.CallResult()
    assert _lib.lib().gmmB200Call(op | _lib.OP_PLAN_ONLY, words, len(words) // 8, None, 0, None, None, C.byref(res)) == 0, _lib.last_error()
    return res


@pytest.mark.parametrize("rows,h", [(1, 8), (16, 2048), (4096, 7168), (700, 5001), (3, 65535)])
def test_sandwich_keeps_a_status_record(rows, h):
    """256 bytes at the start of its workspace whatever kernel takes the call, in front of the copies of strided views; none without rows."""
    one, eps = acl._float_bits(1.0), acl._float_bits(1e-6)

    def size(rows, x):
        res = plan(_lib.OP_SANDWICH_NORM_QUANT, "ttttttttttiiiii", x, e(rows, h), e(h), None, None, None, e(rows, h, dtype=I8), e(rows, dtype=F32), e(rows, h), None,
                   0, one, one, eps, eps)
        options = ops.LaunchOptions(wait_limit_cycles=1000, test_skip_k_blocks=1)
        assert _lib.lib().gmmB200SetExecutorOptions(C.c_void_p(res.executor), C.byref(options)) == 0
        rc = _lib.lib().gmmB200SandwichNormQuant(None, max(res.workspaceSize - 1, 0), C.c_void_p(res.executor), None) if res.workspaceSize else INVALID
        assert rc == INVALID
        if not res.workspaceSize:
            _lib.lib().aclDestroyAclOpExecutor(C.c_void_p(res.executor))
        return res.workspaceSize

    assert size(rows, e(rows, h)) == 256 and size(0, e(0, h)) == 0
    staged = (rows * h * 2 + 255) // 256 * 256
    if h > 1:
        assert size(rows, e(rows, 2 * h)[:, ::2]) == 256 + staged
