"""Host-side mirror of the reference operator interface on top of the C ABI.

``grouped_matmul_v4`` follows aclnnGroupedMatmulV4 (gmm/grouped_matmul/op_host/op_api/aclnn_grouped_matmul_v4.h:66-86
of the reference) and ``grouped_matmul_swiglu_quant`` follows aclnnGroupedMatmulSwigluQuant
(gmm/grouped_matmul_swiglu_quant/op_host/op_api/aclnn_grouped_matmul_swiglu_quant.h:37-52): same argument
names and meaning, same two-phase sequence (GetWorkspaceSize -> allocate -> launch on a stream), same status
codes raised as ``AclnnError``.  torch is used for device memory and streams only.
"""
from __future__ import annotations

import array
import contextlib
import ctypes as C
import struct
import threading
from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import LaunchOptions  # noqa: F401  (re-exported: the per-call options of include/gmm_b200.h)
from ._lib import (ACL_BF16, ACL_FLOAT, ACL_FLOAT16, ACL_FORMAT_FRACTAL_NZ, ACL_FORMAT_ND, ACL_INT8, ACL_INT32, ACL_INT64,
                   ACLNN_SUCCESS)

_DTYPES = {
    torch.float32: ACL_FLOAT, torch.float16: ACL_FLOAT16, torch.int8: ACL_INT8, torch.int32: ACL_INT32,
    torch.int64: ACL_INT64, torch.bfloat16: ACL_BF16,
}


class AclnnError(RuntimeError):
    """A non-zero aclnnStatus.  ``status`` holds the code, the text comes from aclGetRecentErrMsg."""

    def __init__(self, status: int, where: str):
        self.status = int(status)
        super().__init__(f"{where} failed with aclnnStatus {status}: {_lib.last_error()}")


def _i64(values: Sequence[int]):
    return (C.c_int64 * len(values))(*values)


def create_tensor(t: torch.Tensor, fmt: int = ACL_FORMAT_ND, dtype: Optional[int] = None,
                  view_dims: Optional[Sequence[int]] = None) -> int:
    """aclCreateTensor over a torch tensor's view (dims, strides, device address).  The caller destroys it.
    ``view_dims``: the tensor is the storage (its shape becomes the storage shape) and is viewed with these dimensions,
    as a FRACTAL_NZ weight is: storage [E, N/32, K/16, 16, 32], view [E, K, N]."""
    storage = list(t.shape)
    if view_dims is None:
        dims, strides = storage, list(t.stride())
    else:
        dims = list(view_dims)
        strides = [1] * len(dims)
        for i in range(len(dims) - 2, -1, -1):
            strides[i] = strides[i + 1] * dims[i + 1]
    code = _DTYPES[t.dtype] if dtype is None else dtype
    h = _lib.lib().aclCreateTensor(_i64(dims), len(dims), code, _i64(strides), 0, fmt, _i64(storage), len(storage),
                                   C.c_void_p(t.data_ptr()))
    if not h:
        raise MemoryError("aclCreateTensor returned null")
    return h


def format_cast_nz(weight: torch.Tensor) -> torch.Tensor:
    """int8 [E, K, N] -> the FRACTAL_NZ storage [E, N/32, K/16, 16, 32] (a copy; K % 16 == 0, N % 32 == 0): element
    (k, n) moves to [n // 32, k // 16, k % 16, n % 32].  What a caller of the reference does once per weight with its
    framework's format cast before calling the WeightNZ operators; a set-up step, not part of the hot path."""
    E, K, N = weight.shape
    if K % 16 or N % 32:
        raise ValueError("FRACTAL_NZ needs K % 16 == 0 and N % 32 == 0")
    return weight.reshape(E, K // 16, 16, N // 32, 32).permute(0, 3, 1, 2, 4).contiguous()


def create_tensor_list(tensors: Sequence[torch.Tensor], fmt: int = ACL_FORMAT_ND) -> int:
    """aclCreateTensorList; the list owns its tensor handles (aclDestroyTensorList frees them)."""
    hs = [create_tensor(t, fmt) for t in tensors]
    arr = (C.c_void_p * len(hs))(*hs)
    h = _lib.lib().aclCreateTensorList(arr, len(hs))
    if not h:
        raise MemoryError("aclCreateTensorList returned null")
    return h


class _Slot:
    """The pooled workspace of one stream.  ``lock`` is held while a call is enqueued with ``buf``: the clear and the kernels of
    two calls must not interleave on the stream."""
    __slots__ = ("lock", "buf")

    def __init__(self):
        self.lock = threading.RLock()
        self.buf: Optional[torch.Tensor] = None


class _Workspace:
    """Growing device buffers for the calls that bring no workspace, one per device and stream: a call uses its buffer until
    its last kernel is done, so calls that may run at the same time must not share one.  The buffers are allocated on their
    own stream; one that is outgrown or evicted goes back to the allocator, which reuses it in that stream's order."""
    MAX_SLOTS = 16   # streams with a buffer; with more of them the oldest slot's goes

    def __init__(self):
        self._slots = {}
        self._lock = threading.Lock()
        self._replayed = {}   # address -> buffer a replay will use (see for_capture)

    def slot(self, device: torch.device, handle: int) -> _Slot:
        # the per-thread default stream has one handle and is another stream in every thread
        key = (device.type, device.index, handle, threading.get_ident() if handle == _STREAM_PER_THREAD else 0)
        s = self._slots.get(key)
        if s is None:
            with self._lock:
                s = self._slots.setdefault(key, _Slot())
                while len(self._slots) > self.MAX_SLOTS:
                    del self._slots[next(iter(self._slots))]
        return s

    def slot_of(self, index: int, handle: int) -> _Slot:
        """The same by a GPU's number."""
        s = self._slots.get(("cuda", index, handle, 0)) if handle != _STREAM_PER_THREAD else None
        return s if s is not None else self.slot(torch.device("cuda", index), handle)

    def lend(self, slot: _Slot, device: torch.device, stream, nbytes: int) -> torch.Tensor:
        """A workspace of at least ``nbytes`` for the call that is about to be enqueued with the slot's lock held."""
        return (self.for_capture if device.type == "cuda" and _capturing(stream) else self.grown)(slot, device, stream, nbytes)

    @staticmethod
    def grown(slot: _Slot, device: torch.device, stream, nbytes: int) -> torch.Tensor:
        """The slot's buffer with room for ``nbytes``."""
        if slot.buf is None or slot.buf.numel() < nbytes:
            with _on_stream(stream, device):
                slot.buf = torch.empty(int(nbytes), dtype=torch.uint8, device=device)
        return slot.buf

    def for_capture(self, slot: _Slot, device: torch.device, stream, nbytes: int) -> torch.Tensor:
        """A workspace for a call that is being captured.  A buffer from the memory pool of a torch graph belongs to that graph
        as long as it lives, so that its replays share it neither with other graphs nor with calls outside.  A capture that
        has no such pool gets the stream's buffer, which is kept from then on even if the stream's calls outgrow it."""
        with _on_stream(stream, device):
            b = torch.empty(int(nbytes), dtype=torch.uint8, device=device)
        if _in_graph_pool(b):
            return b
        b = self.grown(slot, device, stream, nbytes)
        self._replayed[b.data_ptr()] = b
        return b


_WS = _Workspace()
_STREAM_PER_THREAD = 2   # cudaStreamPerThread


def _on_stream(stream, device: torch.device):
    """Context in which torch's current stream is ``stream``."""
    if stream is None or device.type != "cuda":
        return contextlib.nullcontext()
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(int(stream.cuda_stream), device=device)
    return torch.cuda.stream(stream)


def _capturing(stream) -> bool:
    if stream is None:
        return torch.cuda.is_current_stream_capturing()
    return _lib.lib().gmmB200StreamIsCapturing(int(stream.cuda_stream)) != 0


def _in_graph_pool(t: torch.Tensor) -> bool:
    p = t.data_ptr()
    return any(tuple(seg["segment_pool_id"]) != (0, 0) for seg in torch.cuda.memory_snapshot()
               if seg["address"] <= p < seg["address"] + seg["total_size"])


def _with_pooled(device: torch.device, stream, handle: int, nbytes: int, call):
    """``call(workspace)``, which enqueues on ``stream``, with a pooled workspace of ``nbytes``; returns the workspace."""
    slot = _WS.slot(device, handle)
    with slot.lock:
        workspace = _WS.lend(slot, device, stream, nbytes)
        call(workspace)
        return workspace


def _stream_handle(stream) -> int:
    if stream is None:
        stream = torch.cuda.current_stream()
    return int(stream.cuda_stream)


def _gpu_stream_handle(stream) -> int:
    """The same where CUDA is known to be up, without the stream object that torch.cuda.current_stream builds."""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice()) if stream is None else int(stream.cuda_stream)


def check_status(workspace: Optional[torch.Tensor], stream=None) -> None:
    """Synchronise the stream and raise if a kernel recorded a problem in the workspace status word."""
    rec = (C.c_int32 * 4)()
    ptr = C.c_void_p(workspace.data_ptr()) if workspace is not None else None
    size = workspace.numel() if workspace is not None else 0
    rc = _lib.lib().gmmB200CheckStatus(ptr, size, C.c_void_p(_stream_handle(stream)), rec)
    if rc != ACLNN_SUCCESS:
        err = AclnnError(rc, "gmmB200CheckStatus")
        err.record = tuple(int(v) for v in rec)   # (code, CTA, waiting role, detail)
        raise err


def _put(words: list, t: Optional[torch.Tensor], fmt: int = ACL_FORMAT_ND, view_dims: Optional[Sequence[int]] = None) -> None:
    """Append one tensor to a packed description (gmmB200Call, include/gmm_b200.h); the same view as ``create_tensor``."""
    words += array.array("q", _lib.describe((t, fmt, view_dims)))


def _ints(values: Optional[Sequence[int]]) -> Optional[list]:
    return None if values is None else list(values)


def _call(op: int, name: str, words, device: torch.device, workspace: Optional[torch.Tensor], stream,
          options: Optional[LaunchOptions]) -> Optional[torch.Tensor]:
    """Both phases of operator ``name`` on the packed description (bytes or a list of its words); returns the workspace that was
    used (None if none)."""
    if not isinstance(words, bytes):
        words = array.array("q", words).tobytes()
    on_gpu = device.type == "cuda"
    handle = _gpu_stream_handle(stream) if on_gpu else 0
    if workspace is not None:
        return _enqueue(op, name, words, device, workspace, stream, handle, options, None)
    slot = _WS.slot(device, handle)
    with slot.lock:
        return _enqueue(op, name, words, device, None, stream, handle, options, slot)


def _enqueue(op: int, name: str, words: bytes, device: torch.device, workspace: Optional[torch.Tensor], stream, handle: int,
             options: Optional[LaunchOptions], slot: Optional[_Slot]) -> Optional[torch.Tensor]:
    L = _lib.lib()
    res = _lib.CallResult()
    # validation needs no device: tensors that are not on one are planned only, so that what is wrong with them is reported first
    on_gpu = device.type == "cuda"
    buf = None if not on_gpu else workspace if slot is None else slot.buf
    rc = L.gmmB200Call(op if slot is None else op | _lib.OP_POOLED, words, len(words) // 8, buf.data_ptr() if buf is not None else None,
                       buf.numel() if buf is not None else 0, C.byref(options) if options is not None else None, handle, C.byref(res))
    if rc == ACLNN_SUCCESS and res.stage == _lib.STAGE_PLANNED:
        ex = C.c_void_p(res.executor)
        if workspace is not None and workspace.numel() < res.workspaceSize:
            L.aclDestroyAclOpExecutor(ex)
            raise ValueError(f"workspace of {workspace.numel()} bytes is smaller than the {res.workspaceSize} required")
        try:
            buf = workspace if slot is None else _WS.lend(slot, device, stream, res.workspaceSize)
            handle = handle if on_gpu else _stream_handle(stream)
        except Exception:
            L.aclDestroyAclOpExecutor(ex)
            raise
        rc = getattr(L, name)(buf.data_ptr(), res.workspaceSize, ex, handle)
        res.stage = _lib.STAGE_RUN
    if rc != ACLNN_SUCCESS:
        raise AclnnError(rc, name + ("GetWorkspaceSize" if res.stage == _lib.STAGE_PLAN else
                                     ": gmmB200SetExecutorOptions" if res.stage == _lib.STAGE_OPTIONS else ""))
    return workspace if slot is None else buf if res.workspaceSize else None


def grouped_matmul_v4(x: torch.Tensor, weight: torch.Tensor, scale: Optional[torch.Tensor],
                      per_token_scale: Optional[torch.Tensor], group_list: torch.Tensor, *,
                      bias: Optional[torch.Tensor] = None, split_item: int = 3, group_type: int = 0,
                      group_list_type: int = 0, act_type: int = 0, out: Optional[torch.Tensor] = None,
                      out_dtype: torch.dtype = torch.bfloat16, stream=None, workspace: Optional[torch.Tensor] = None,
                      return_workspace: bool = False, out_row_index: Optional[torch.Tensor] = None,
                      out_peers: Optional[Sequence[int]] = None, weight_format: int = ACL_FORMAT_ND,
                      api: str = "V4", tuning_config: Optional[Sequence[int]] = None, quant_group_size: int = 0,
                      options: Optional[LaunchOptions] = None, out_rows: int = 0):
    """y = bf16(act((x @ weight[e]) * scale[e] * per_token_scale)) per expert row range (W8A8), a float16 result with
    ``out_dtype`` torch.float16, or the raw int32 accumulators with torch.int32.  Rows not covered by ``group_list``
    keep their contents.  ``weight_format`` ACL_FORMAT_FRACTAL_NZ: ``weight`` is the 5-D storage of ``format_cast_nz``.
    ``api`` picks the entry point: "V4", "V5" (adds ``tuning_config``) or "WeightNz" (adds ``quant_group_size`` and
    treats the weight as FRACTAL_NZ) - aclnn_grouped_matmul_v5.h:49-58, aclnn_grouped_matmul_weight_nz.h:50-59 of the
    reference.  ``out_row_index`` (int64 [M], an extension of this library) scatters result row r to row
    out_row_index[r]; it goes through the flat entry point gmmB200GroupedMatmulW8A8.  ``options``: per-call
    ``LaunchOptions`` (CTA cap, timing events)."""
    nz = weight_format == ACL_FORMAT_FRACTAL_NZ or api == "WeightNz"
    if out is None and not out_peers:
        n_out = weight.shape[1] * 32 if (nz and weight.dim() == 5) else weight.shape[2]
        out = x.new_empty((x.shape[0], n_out), dtype=out_dtype)
    if out_row_index is not None:
        return _grouped_matmul_flat(x, weight, scale, per_token_scale, group_list, bias, group_list_type, act_type, out,
                                    out_row_index, stream, workspace, return_workspace, out_peers, nz, options, out_rows)
    if api not in _lib.OP_GMM:
        raise ValueError(f"unknown api {api!r}")
    words = _lib.describe_call("tftttttiiiiil", x, (weight, ACL_FORMAT_FRACTAL_NZ if nz else ACL_FORMAT_ND, None), bias, scale, per_token_scale,
                               group_list, out, split_item, group_type, group_list_type, act_type, quant_group_size, _ints(tuning_config))
    workspace = _call(_lib.OP_GMM[api], "aclnnGroupedMatmul" + api, words, x.device, workspace, stream, options)
    return (out, workspace) if return_workspace else out


def _grouped_matmul_flat(x, weight, scale, per_token_scale, group_list, bias, group_list_type, act_type, out, out_row_index,
                         stream, workspace, return_workspace, out_peers=None, nz=False, options=None, out_rows=0):
    """Flat entry point.  ``out_peers`` (device addresses, one [rows, N] bf16 buffer per GPU) makes out_row_index hold
    (gpu << 40) | row; ``out`` may then be None.  ``out_rows``: rows of ``out`` / of every peer buffer (0 = taken from
    ``out``, unbounded without it); rows scattered outside are skipped and reported by ``check_status``."""
    L = _lib.lib()
    M, K = x.shape
    if nz and weight.dim() == 5:
        E, N = weight.shape[0], weight.shape[1] * 32
    else:
        E, _, N = weight.shape
    trans = 2 if nz else int((not weight.is_contiguous()) and weight.transpose(1, 2).is_contiguous())
    for t in (x, scale, per_token_scale, group_list, bias, out, out_row_index):
        if t is not None and not t.is_contiguous():
            raise ValueError("the flat entry point needs contiguous tensors")
    if out_row_index.dtype != torch.int64 or out_row_index.numel() != M:
        raise ValueError("out_row_index must be int64 [M]")
    ydt = _DTYPES[out.dtype] if out is not None else ACL_BF16
    if not out_rows and out is not None:
        out_rows = out.shape[0]
    n_peers = len(out_peers) if out_peers else 0
    peers = (C.c_void_p * max(n_peers, 1))(*[C.c_void_p(a) for a in (out_peers or [])])
    size = C.c_uint64(0)
    rc = L.gmmB200GroupedMatmulW8A8WorkspaceSize(M, K, N, E, ydt, C.byref(size))
    if rc != ACLNN_SUCCESS:
        raise AclnnError(rc, "gmmB200GroupedMatmulW8A8WorkspaceSize")
    p = lambda t: C.c_void_p(t.data_ptr()) if t is not None else None  # noqa: E731
    handle = _gpu_stream_handle(stream) if x.device.type == "cuda" else _stream_handle(stream)

    def enqueue(workspace):
        rc = L.gmmB200GroupedMatmulW8A8(p(x), p(weight), p(scale), _DTYPES[scale.dtype] if scale is not None else 0, p(per_token_scale),
                                        p(bias), _DTYPES[bias.dtype] if bias is not None else 0, p(group_list), group_list.numel(),
                                        group_list_type, M, K, N, E, trans, act_type, p(out_row_index), peers if n_peers else None, n_peers, out_rows,
                                        p(out), ydt, p(workspace), workspace.numel(), handle,
                                        C.byref(options) if options is not None else None)
        if rc != ACLNN_SUCCESS:
            raise AclnnError(rc, "gmmB200GroupedMatmulW8A8")
    if workspace is None:
        workspace = _with_pooled(x.device, stream, handle, size.value, enqueue)
    else:
        enqueue(workspace)
    return (out, workspace) if return_workspace else out


def grouped_matmul_swiglu_quant(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, x_scale: torch.Tensor,
                                group_list: torch.Tensor, *, bias: Optional[torch.Tensor] = None,
                                offset: Optional[torch.Tensor] = None, output: Optional[torch.Tensor] = None,
                                output_scale: Optional[torch.Tensor] = None, stream=None,
                                workspace: Optional[torch.Tensor] = None, return_workspace: bool = False,
                                weight_format: int = ACL_FORMAT_ND, api: str = "", options: Optional[LaunchOptions] = None):
    """(output int8 [M, N/2], output_scale fp32 [M]) = per-token int8 requant of SwiGLU of the dequantised grouped
    GEMM.  ``group_list`` holds running totals.  Rows at and beyond group_list[-1] keep their contents.
    ``weight_format`` ACL_FORMAT_FRACTAL_NZ: ``weight`` is the 5-D storage of ``format_cast_nz``; ``api`` "WeightNZ"
    calls aclnnGroupedMatmulSwigluQuantWeightNZ (aclnn_grouped_matmul_swiglu_quant_weight_nz.h:37-54 of the reference),
    which takes the storage as FRACTAL_NZ whatever the format says."""
    M = x.shape[0]
    N = weight_scale.shape[1] if weight_scale.dim() == 2 else 0
    if output is None:
        output = x.new_empty((M, N // 2), dtype=torch.int8)
    if output_scale is None:
        output_scale = x.new_empty((M,), dtype=torch.float32)
    words = _lib.describe_call("tfttttttt", x, (weight, weight_format, None), bias, offset, weight_scale, x_scale, group_list, output, output_scale)
    workspace = _call(_lib.OP_SWIGLU_QUANT[api], "aclnnGroupedMatmulSwigluQuant" + api, words, x.device, workspace, stream, options)
    return (output, output_scale, workspace) if return_workspace else (output, output_scale)


def grouped_matmul_finalize_routing(x: torch.Tensor, weight_nz: torch.Tensor, scale: torch.Tensor, group_list: torch.Tensor,
                                    row_index: torch.Tensor, batch: int, *, bias: Optional[torch.Tensor] = None,
                                    pertoken_scale: Optional[torch.Tensor] = None, shared_input: Optional[torch.Tensor] = None,
                                    logit: Optional[torch.Tensor] = None, shared_input_weight: float = 1.0,
                                    shared_input_offset: int = 0, group_list_type: int = 1, out: Optional[torch.Tensor] = None,
                                    view_3d: bool = True, api: str = "", tuning_config: Optional[Sequence[int]] = None,
                                    stream=None, workspace: Optional[torch.Tensor] = None, return_workspace: bool = False,
                                    options: Optional[LaunchOptions] = None):
    """aclnnGroupedMatmulFinalizeRoutingWeightNz (``api`` "") or ...WeightNzV2 (``api`` "V2"): W8A8 grouped GEMM whose fp32
    result rows, weighted by ``logit``, are added into row ``row_index[i]`` of ``out`` [batch, N] on top of the weighted
    ``shared_input`` rows (gmm/grouped_matmul_finalize_routing/op_host/op_api/aclnn_grouped_matmul_finalize_routing_weight_nz.h:48-64
    of the reference).  ``weight_nz`` is the FRACTAL_NZ storage [E, N/32, K/16, 16, 32] (``format_cast_nz``); with
    ``view_3d`` it is described to the operator as the reference's callers do, a view [E, K, N] over that storage."""
    E, n1, k1 = weight_nz.shape[0], weight_nz.shape[1], weight_nz.shape[2]
    N, K = n1 * 32, k1 * 16
    if out is None:
        out = x.new_empty((batch, N), dtype=torch.float32)
    words = _lib.describe_call("tfttttttttiiil", x, (weight_nz, ACL_FORMAT_FRACTAL_NZ, [E, K, N] if view_3d else None), scale, bias,
                               pertoken_scale, group_list, shared_input, logit, row_index, out,
                               struct.unpack("<I", bytes(C.c_float(shared_input_weight)))[0], shared_input_offset, group_list_type, _ints(tuning_config))
    workspace = _call(_lib.OP_FINALIZE_ROUTING[api], "aclnnGroupedMatmulFinalizeRoutingWeightNz" + api, words, x.device, workspace, stream,
                      options)
    return (out, workspace) if return_workspace else out


def grouped_matmul_finalize_routing_flat(x, weight, weight_layout, scale, group_list, row_index, out, *, bias=None,
                                         pertoken_scale=None, shared_input=None, logit=None, shared_input_weight=1.0,
                                         shared_input_offset=0, group_list_type=1, stream=None, workspace=None, options=None):
    """gmmB200GroupedMatmulFinalizeRouting: the same operator without handles; ``weight_layout`` 0 takes the ND [E, K, N]
    weight (the faster layout here), 2 the FRACTAL_NZ storage."""
    L = _lib.lib()
    M, K = x.shape
    if weight_layout == 2:
        E, N = weight.shape[0], weight.shape[1] * 32
    else:
        E, _, N = weight.shape
    p = lambda t: C.c_void_p(t.data_ptr()) if t is not None else None  # noqa: E731
    handle = _gpu_stream_handle(stream) if x.device.type == "cuda" else _stream_handle(stream)

    def enqueue(workspace):
        rc = L.gmmB200GroupedMatmulFinalizeRouting(
            p(x), p(weight), weight_layout, p(scale), _DTYPES[scale.dtype], p(bias), p(pertoken_scale), p(group_list),
            group_list.numel(), group_list_type, p(shared_input), 0 if shared_input is None else shared_input.shape[0],
            shared_input_offset, shared_input_weight, p(logit), p(row_index), _DTYPES[row_index.dtype], M, K, N, E, p(out),
            out.shape[0], p(workspace), workspace.numel(), handle,
            C.byref(options) if options is not None else None)
        if rc != ACLNN_SUCCESS:
            raise AclnnError(rc, "gmmB200GroupedMatmulFinalizeRouting")
    if workspace is None:
        _with_pooled(x.device, stream, handle, 256, enqueue)
    else:
        enqueue(workspace)
    return out


def moe_init_routing_v3(x: torch.Tensor, expert_idx: torch.Tensor, *, expert_num: int, active_expert_range: Sequence[int],
                        quant_mode: int = 1, scale: Optional[torch.Tensor] = None, offset: Optional[torch.Tensor] = None,
                        active_num: Optional[int] = None, expert_capacity: int = 0, drop_pad_mode: int = 0,
                        expert_tokens_num_type: int = 1, expert_tokens_num_flag: bool = True, row_idx_type: int = 1,
                        outputs=None, stream=None, workspace: Optional[torch.Tensor] = None):
    """aclnnMoeInitRoutingV3 (moe/moe_init_routing_v3/op_host/op_api/aclnn_moe_init_routing_v3.h:24-47 of the reference):
    returns (expandedX, expandedRowIdx, expertTokensCountOrCumsum, expandedScale).  With ``quant_mode`` 1 expandedX is int8
    and expandedScale the per-row scale, i.e. the x / per-token scale of the grouped GEMM operators."""
    n, h = x.shape
    k = expert_idx.shape[1]
    start, end = active_expert_range
    if outputs is None:
        ex = x.new_empty((n * k, h), dtype=torch.int8 if quant_mode == 1 else x.dtype)
        ri = x.new_empty((n * k,), dtype=torch.int32)
        cnt = x.new_empty((end - start,) if expert_tokens_num_type == 1 else (expert_num, 2), dtype=torch.int64)
        es = x.new_empty((n * k,), dtype=torch.float32)
    else:
        ex, ri, cnt, es = outputs
    words = _lib.describe_call("ttttttttiiiiiiiil", x, expert_idx, scale, offset, ex, ri, cnt, es, n * k if active_num is None else active_num,
                               expert_capacity, expert_num, drop_pad_mode, expert_tokens_num_type, 1 if expert_tokens_num_flag else 0, quant_mode,
                               row_idx_type, _ints(active_expert_range))
    _call(_lib.OP_MOE_INIT_ROUTING, "aclnnMoeInitRoutingV3", words, x.device, workspace, stream, None)
    return ex, ri, cnt, es


# ---------------------------------------------------------------------------------------------------------------------
# Operators around the expert FFN (include/gmm_b200.h)
# ---------------------------------------------------------------------------------------------------------------------

_FLOAT, _WORD = struct.Struct("<f"), struct.Struct("<I")


def _float_bits(v: float) -> int:
    return _WORD.unpack(_FLOAT.pack(v))[0]


_current_device, _raw_stream = (getattr(torch._C, name, None) for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"))
_POOLED = frozenset((_lib.OP_ADAPTER_ADD, _lib.OP_QUANT_MATMUL, _lib.OP_SANDWICH_NORM_QUANT, _lib.OP_EXPERT_BALANCE))


def _block_call(op: int, name: str, workspace: Optional[torch.Tensor], stream, options: Optional[LaunchOptions], kinds: str,
                *items) -> Optional[torch.Tensor]:
    """The call of an operator around the expert FFN, natively.  Its tensors all have to be on one GPU; elsewhere the arguments are
    checked and the call is refused.  It runs on that GPU, whichever is the current one.  A call that needs no workspace (all but those of
    ``_POOLED`` and strided views) takes none.  Returns the workspace that the call uses (None if none)."""
    module, call = _lib.native()
    x, buf = items[0], workspace
    if workspace is None and stream is None and options is None and x.get_device() >= 0 and x.get_device() == _current_device():
        # what most calls are, with as little on the way as can be: their kernels are often shorter
        handle = _raw_stream(x.get_device())
        if op not in _POOLED:
            done = module.launch(call, op, handle, None, 0, kinds, *items)
        else:
            slot = _WS.slot_of(x.get_device(), handle)
            with slot.lock:   # the clear and the kernels of two calls must not interleave on the stream
                buf = slot.buf
                done = module.launch(call, op | _lib.OP_POOLED, handle, buf, 0, kinds, *items)
        return buf if done is None else _block_rest(op, name, workspace, stream, handle, kinds, items, done)
    if x.is_cuda and x.get_device() != torch._C._cuda_getDevice():
        with torch.cuda.device(x.device):
            return _block_call(op, name, workspace, stream, options, kinds, *items)
    how = 0 if options is None else C.addressof(options)
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    pooled = workspace is None and op in _POOLED
    handle = None
    if not x.is_cuda:
        done = False
    else:
        handle = _gpu_stream_handle(stream)
        if pooled:
            slot = _WS.slot(x.device, handle)
            with slot.lock:   # the clear and the kernels of two calls must not interleave on the stream
                buf = slot.buf
                done = module.launch(call, op | _lib.OP_POOLED, handle, buf, how, kinds, *items)
        else:
            done = module.launch(call, op, handle, workspace, how, kinds, *items)
    return buf if done is None else _block_rest(op, name, workspace, stream, handle, kinds, items, done)


def _block_rest(op: int, name: str, workspace, stream, handle, kinds: str, items, done) -> Optional[torch.Tensor]:
    """What a call that was not enqueued at once still needs: its refusal, or a workspace."""
    x = items[0]
    if done is False:
        words = _lib.describe_call(kinds, *items)
        res = _lib.CallResult()
        rc = _lib.lib().gmmB200Call(op | _lib.OP_PLAN_ONLY, words, len(words) // 8, None, 0, None, None, C.byref(res))
        if rc != ACLNN_SUCCESS:
            raise AclnnError(rc, name + "GetWorkspaceSize")
        _lib.lib().aclDestroyAclOpExecutor(C.c_void_p(res.executor))
        raise ValueError(f"{name}: all tensors must be on one CUDA device")
    rc, stage, need, executor = done
    if rc != ACLNN_SUCCESS:
        raise AclnnError(rc, name + ("GetWorkspaceSize" if stage == _lib.STAGE_PLAN else
                                     ": gmmB200SetExecutorOptions" if stage == _lib.STAGE_OPTIONS else ""))
    # planned only: the pool's buffer is too small or not for this call, or strided views need one
    if workspace is not None:
        _lib.lib().aclDestroyAclOpExecutor(C.c_void_p(executor))
        raise ValueError(f"workspace of {workspace.numel()} bytes is smaller than the {need} required")
    slot = _WS.slot(x.device, handle)
    with slot.lock:
        try:
            workspace = _WS.lend(slot, x.device, stream, need)
        except Exception:
            _lib.lib().aclDestroyAclOpExecutor(C.c_void_p(executor))
            raise
        rc = getattr(_lib.lib(), name)(workspace.data_ptr(), need, C.c_void_p(executor), handle)
    if rc != ACLNN_SUCCESS:
        raise AclnnError(rc, name)
    return workspace


def add_rms_norm_quant(x: torch.Tensor, gamma: torch.Tensor, *, residual: Optional[torch.Tensor] = None,
                       smooth: Optional[torch.Tensor] = None, eps: float = 1e-6, normed: bool = False,
                       q: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                       residual_out: Optional[torch.Tensor] = None, normed_out: Optional[torch.Tensor] = None, stream=None,
                       workspace: Optional[torch.Tensor] = None):
    """(q int8 [rows, h], scale fp32 [rows], residual_out, normed_out): the norm of ``h = x + residual`` in 8 bits with per-token scales,
    as the W8A8 operators take their rows, ``h`` itself (None without a residual) and, with ``normed`` or a ``normed_out`` to write to,
    the normed rows in x's type.  ``smooth`` (fp32 [h]) multiplies what is quantised, not ``normed_out``.  ``residual_out`` may be
    ``residual`` or ``x``.  gmmB200AddRmsNormQuant (include/gmm_b200.h) has the formulas."""
    empty = _lib.native()[0].empty
    if q is None:
        q = empty(x, "b")
    if scale is None:
        scale = empty(x, "f", x.shape[0])
    if residual_out is None and residual is not None:
        residual_out = empty(x, "=")
    if normed_out is None and normed:
        normed_out = empty(x, "=")
    _block_call(_lib.OP_ADD_RMS_NORM_QUANT, "gmmB200AddRmsNormQuant", workspace, stream, None, "tttttttti", x, residual, gamma, smooth, q, scale,
                residual_out, normed_out, _float_bits(eps))
    return q, scale, residual_out, normed_out


_SCORING = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORE = {"max": 0, "top2": 1}
_ID_LETTER = {torch.int32: "i", torch.int64: "l"}


def route_top_k(logits: torch.Tensor, top_k: int, *, scoring: str = "softmax", bias: Optional[torch.Tensor] = None, n_group: int = 1,
                topk_group: int = 1, group_score: str = "max", renormalize: bool = True, scale: float = 1.0,
                token_mask: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None, ids: Optional[torch.Tensor] = None,
                ids_dtype: torch.dtype = torch.int32, stream=None, workspace: Optional[torch.Tensor] = None):
    """(weights fp32 [rows, top_k], ids [rows, top_k]): the experts of every row, largest choice first, ties to the lowest id.
    ``scoring`` "softmax" or "sigmoid"; ``bias`` (fp32 [experts]) is added for the choice and is no part of the weights; with ``n_group``
    only the ``topk_group`` best groups stay, ranked by their largest choice ("max") or the sum of the two largest ("top2").
    ``token_mask`` (bool or int8 [rows]): rows without a token.  Slots without an expert have id -1 and weight 0.  ``ids_dtype`` int32 is
    what ``moe_init_routing_v3`` takes, int64 the expert-parallel layer.  gmmB200RouteTopK (include/gmm_b200.h) has the rules."""
    if scoring not in _SCORING or group_score not in _GROUP_SCORE:
        raise ValueError(f"unknown scoring {scoring!r} or group_score {group_score!r}")
    if weights is not None and ids is not None and weights.shape == ids.shape and weights.shape[-1:] != (top_k,):
        raise ValueError(f"weights and ids must have top_k = {top_k} columns")
    empty = _lib.native()[0].empty
    if weights is None:
        weights = empty(logits, "f", logits.shape[0], top_k)
    if ids is None:
        letter = _ID_LETTER.get(ids_dtype)
        shape = logits.shape[0], top_k
        ids = empty(logits, letter, *shape) if letter else logits.new_empty(shape, dtype=ids_dtype)   # refused by the operator
    if token_mask is not None and token_mask.dtype == torch.bool:
        token_mask = token_mask.view(torch.int8)
    _block_call(_lib.OP_ROUTE_TOP_K, "gmmB200RouteTopK", workspace, stream, None, "tttttiiiiii", logits, bias, token_mask, weights, ids,
                _SCORING[scoring], n_group, topk_group, _GROUP_SCORE[group_score], 1 if renormalize else 0, _float_bits(scale))
    return weights, ids


def adapter_add(base: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, adapter_ids: torch.Tensor, *,
                x_scale: Optional[torch.Tensor] = None, scaling: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                stream=None, workspace: Optional[torch.Tensor] = None, return_workspace: bool = False,
                options: Optional[LaunchOptions] = None):
    """out [rows, n] = base + scaling[i] * (x a[i]^T) b[i]^T with the adapter i = adapter_ids[row] of every row (int32, negative: none):
    low-rank adapters of many requests beside one shared projection, whose result is ``base``.  ``x`` has base's type or is int8 with
    ``x_scale`` (fp32 [rows]); a [adapters, rank, k], b [adapters, n, rank].  ``out`` may be ``base``.  With
    ``return_workspace`` (out, workspace), for ``check_status`` (no rows: None); ``options``: per-call ``LaunchOptions`` (wait bound).  gmmB200AdapterAdd
    (include/gmm_b200.h)."""
    if out is None:
        out = _lib.native()[0].empty(base, "=")
    workspace = _block_call(_lib.OP_ADAPTER_ADD, "gmmB200AdapterAdd", workspace, stream, options, "tttttttt", base, x, x_scale, a, b, adapter_ids,
                            scaling, out)
    return (out, workspace if base.shape[0] else None) if return_workspace else out


_FLOAT_LETTER = {torch.float32: "f", torch.float16: "h", torch.bfloat16: "w"}


def quant_matmul(x: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, per_token_scale: Optional[torch.Tensor] = None, *,
                 bias: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16, stream=None,
                 workspace: Optional[torch.Tensor] = None, return_workspace: bool = False, options: Optional[LaunchOptions] = None):
    """y [rows, n] = ((x @ weight) * scale) * per_token_scale + bias of int8 ``x`` [rows, k] and ``weight`` [k, n] (or the transposed view of
    one stored [n, k]), with one scale a channel and, where given, one a token: the W8A8 product without groups.  ``scale`` and ``bias`` [n]
    fp32 or 16-bit, ``per_token_scale`` fp32 [rows]; the result is ``out_dtype`` (bf16, fp16 or fp32) or ``out``.  With ``return_workspace``
    (y, workspace), for ``check_status`` (no rows: None); ``options``: per-call ``LaunchOptions`` (wait bound, timing events).
    gmmB200QuantMatmul (include/gmm_b200.h)."""
    if stream is not None:   # what a call returns belongs to the stream that writes it
        with _on_stream(stream, x.device):
            return quant_matmul(x, weight, scale, per_token_scale, bias=bias, out=out, out_dtype=out_dtype, workspace=workspace,
                                return_workspace=return_workspace, options=options)
    if out is None:
        letter = _FLOAT_LETTER.get(out_dtype)
        if letter and x.dim() == 2 and weight.dim() == 2:
            out = _lib.native()[0].empty(x, letter, x.shape[0], weight.shape[1])
        else:   # refused by the operator
            out = x.new_empty((x.shape[0], weight.shape[-1]), dtype=out_dtype)
    workspace = _block_call(_lib.OP_QUANT_MATMUL, "gmmB200QuantMatmul", workspace, None, options, "tttttt", x, weight, scale, per_token_scale, bias, out)
    return (out, workspace if x.shape[0] else None) if return_workspace else out


_GATE_ACT = {"none": 0, "sigmoid": 1, "tanh": 2}


def sandwich_norm_quant(x: torch.Tensor, residual: torch.Tensor, gamma: Optional[torch.Tensor] = None, *,
                        post_gamma: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, gate_act: str = "none",
                        residual_scale: float = 1.0, block_scale: float = 1.0, smooth: Optional[torch.Tensor] = None, eps: float = 1e-6,
                        post_eps: Optional[float] = None, quant: bool = True, normed: bool = False, q: Optional[torch.Tensor] = None,
                        scale: Optional[torch.Tensor] = None, residual_out: Optional[torch.Tensor] = None,
                        normed_out: Optional[torch.Tensor] = None, stream=None, workspace: Optional[torch.Tensor] = None,
                        return_workspace: bool = False, options: Optional[LaunchOptions] = None):
    """(q int8 [rows, h], scale fp32 [rows], residual_out, normed_out): the way from a block's output ``x`` into the next block.  The residual
    stream ``s = residual_scale * residual + block_scale * act(gate) * n`` with the block's output behind its norm, ``n = rms_norm(x) *
    post_gamma`` (x itself without ``post_gamma``), and the norm of s with ``gamma`` in 8 bits with per-token scales (None without ``quant``)
    and, with ``normed`` or a ``normed_out`` to write to, in residual's type.  ``x`` has residual's type or is fp32; ``gate`` is one for each
    channel [h], each token [rows, 1] or each element, and goes through ``gate_act`` ("none", "sigmoid", "tanh"); ``smooth`` (fp32 [h])
    multiplies what is quantised, not ``normed_out``; ``post_eps`` is ``eps`` unless given.  ``residual_out`` may be ``residual``.
    With ``return_workspace`` the workspace follows, for ``check_status`` (no rows: None); ``options``: per-call
    ``LaunchOptions`` (wait bound).  gmmB200SandwichNormQuant (include/gmm_b200.h) has the formulas."""
    if stream is not None:   # what a call returns belongs to the stream that writes it
        with _on_stream(stream, x.device):
            return sandwich_norm_quant(x, residual, gamma, post_gamma=post_gamma, gate=gate, gate_act=gate_act, residual_scale=residual_scale,
                                       block_scale=block_scale, smooth=smooth, eps=eps, post_eps=post_eps, quant=quant, normed=normed, q=q,
                                       scale=scale, residual_out=residual_out, normed_out=normed_out, workspace=workspace,
                                       return_workspace=return_workspace, options=options)
    if gate_act not in _GATE_ACT:
        raise ValueError(f"unknown gate_act {gate_act!r}")
    empty = _lib.native()[0].empty
    if quant or q is not None or scale is not None:
        if q is None:
            q = empty(x, "b")
        if scale is None:
            scale = empty(x, "f", x.shape[0])
    if residual_out is None:
        residual_out = empty(residual, "=")
    if normed_out is None and normed:
        normed_out = empty(residual, "=")
    eps = _float_bits(eps)
    workspace = _block_call(_lib.OP_SANDWICH_NORM_QUANT, "gmmB200SandwichNormQuant", workspace, None, options, "ttttttttttiiiii", x, residual, gamma,
                            post_gamma, gate, smooth, q, scale, residual_out, normed_out, _GATE_ACT[gate_act], _float_bits(residual_scale),
                            _float_bits(block_scale), eps, eps if post_eps is None else _float_bits(post_eps))
    if return_workspace:
        return q, scale, residual_out, normed_out, workspace if residual.shape[0] else None
    return q, scale, residual_out, normed_out


def expert_balance(logits: torch.Tensor, ids: torch.Tensor, *, scoring: str = "softmax", coefficient: float = 1.0,
                   token_mask: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None, loss: Optional[torch.Tensor] = None,
                   counts: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None, stream=None,
                   workspace: Optional[torch.Tensor] = None):
    """(loss, counts, weight): how the choices ``ids`` [rows, top_k] of ``route_top_k`` load the experts, and the loss that evens them out,
    ``coefficient * experts / top_k * sum_e (share of the tokens' choices that are e) * (mean of the tokens' scores of e)``, the mean of it
    over the sequences where ``cu_seqlens`` (int32 [sequences + 1]) names some.  ``loss`` is one fp32 number on the device, ``counts`` int64
    [experts] or [sequences, experts], ``weight`` fp32 [sequences]: what ``expert_balance_grad`` takes.  ``scoring`` "softmax" or "sigmoid" (divided
    by the row's sum); ``token_mask`` (bool or int8 [rows]): rows without a token; negative ids are not counted.  The loss has no autograd history,
    also where ``logits`` have one: added to another loss it brings no gradient, which is ``expert_balance_grad``'s.  gmmB200ExpertBalance
    (include/gmm_b200.h) has the formulas."""
    if stream is not None:   # what a call returns belongs to the stream that writes it
        with _on_stream(stream, logits.device):
            return expert_balance(logits, ids, scoring=scoring, coefficient=coefficient, token_mask=token_mask, cu_seqlens=cu_seqlens, loss=loss,
                                  counts=counts, weight=weight, workspace=workspace)
    if scoring not in _SCORING:
        raise ValueError(f"unknown scoring {scoring!r}")
    empty = _lib.native()[0].empty
    sequences = 1 if cu_seqlens is None else max(cu_seqlens.shape[0] - 1, 0)
    if loss is None:
        loss = empty(logits, "s")
    if counts is None:
        counts = empty(logits, "l", logits.shape[-1]) if cu_seqlens is None else empty(logits, "l", sequences, logits.shape[-1])
    if weight is None:
        weight = empty(logits, "f", sequences)
    _block_call(_lib.OP_EXPERT_BALANCE, "gmmB200ExpertBalance", workspace, None, None, "tttttttii", logits, ids, token_mask, cu_seqlens, loss, counts,
                weight, _SCORING[scoring], _float_bits(coefficient))
    return loss, counts, weight


def expert_balance_grad(logits: torch.Tensor, counts: torch.Tensor, weight: torch.Tensor, *, scoring: str = "softmax",
                        token_mask: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None,
                        grad_loss: Optional[torch.Tensor] = None, grad: Optional[torch.Tensor] = None, stream=None,
                        workspace: Optional[torch.Tensor] = None):
    """The gradient of ``expert_balance``'s loss with respect to ``logits``, in their type, from the ``counts`` and ``weight`` that it returned and
    the same ``scoring``, ``token_mask`` and ``cu_seqlens``; ``grad_loss`` (one fp32 number on the device) multiplies it.  ``logits.backward(grad)``
    hands it on to a router that torch differentiates.  ``grad`` may be ``logits``.  gmmB200ExpertBalanceGrad (include/gmm_b200.h)."""
    if stream is not None:   # what a call returns belongs to the stream that writes it
        with _on_stream(stream, logits.device):
            return expert_balance_grad(logits, counts, weight, scoring=scoring, token_mask=token_mask, cu_seqlens=cu_seqlens, grad_loss=grad_loss,
                                       grad=grad, workspace=workspace)
    if scoring not in _SCORING:
        raise ValueError(f"unknown scoring {scoring!r}")
    if grad is None:
        grad = _lib.native()[0].empty(logits, "=")
    _block_call(_lib.OP_EXPERT_BALANCE_GRAD, "gmmB200ExpertBalanceGrad", workspace, None, None, "ttttttti", logits, counts, weight,
                token_mask, cu_seqlens, grad_loss, grad, _SCORING[scoring])
    return grad
