"""Host layer of sliding-window attention with sinks: validation, allocation, torch ops and the autograd Function. The
conditions are those of the other attention functions (`ops.py`), whose checks name the fault when a call does not meet
them; see `dispatch.py` for the way to the C entries."""
from __future__ import annotations

import ctypes
import functools

import torch

from . import lib as _lib
from . import ops
from .dispatch import PACK_BWD, PACK_FWD, define, entry, on_device, readable, refuse_tangents, stream_of

BF16, INT32 = torch.bfloat16, torch.int32


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(direction, sink, packed, *problem):
    names = ("batch", "seqlen_q", "seqlen_k", "heads_q", "heads_kv", "head_dim", "window_left", "window_right")
    args = _lib.Problem(**dict(zip(names, problem)), softmax_scale=1.0, cu_seqlens_q=packed or None, cu_seqlens_k=packed or None)
    return getattr(_lib.library(), f"b200fa_sink_{direction}_workspace_bytes")(args, sink)


def _fits(q, k, v, cu_seqlens_q, cu_seqlens_k):
    """Whether the tensors are what the kernels take; ops.check_inputs says what is wrong when they are not."""
    shape_q, shape_k, device = q.shape, k.shape, q.get_device()
    rank = 4 if cu_seqlens_q is None else 3
    return (
        q.dtype is BF16 and k.dtype is BF16 and v.dtype is BF16 and len(shape_q) == rank == len(shape_k) and v.shape == shape_k
        and shape_q[-1] == shape_k[-1] and shape_q[-1] in ops.CANDIDATE_HEAD_DIMS
        and shape_q[-2] > 0 and shape_k[-2] > 0 and shape_q[-2] % shape_k[-2] == 0
        and device == k.get_device() == v.get_device()
        and (
            cu_seqlens_k is None and shape_q[0] == shape_k[0]
            if cu_seqlens_q is None
            else cu_seqlens_k is not None and cu_seqlens_q.dtype is INT32 and cu_seqlens_k.dtype is INT32 and cu_seqlens_q.dim() == 1
            and cu_seqlens_q.shape == cu_seqlens_k.shape and cu_seqlens_q.shape[0] > 0
            and device == cu_seqlens_q.get_device() == cu_seqlens_k.get_device()
        )
    )


def _strides(tensor, packed):
    stride = tensor.stride()
    return (0, stride[0], stride[1]) if packed else stride[:3]


def _problem(q, k, cu_seqlens_q, window_left, window_right):
    if cu_seqlens_q is None:
        sizes = q.shape[0], q.shape[1], k.shape[1]
    else:
        sizes = cu_seqlens_q.shape[0] - 1, q.shape[0], k.shape[0]
    return *sizes, q.shape[-2], k.shape[-2], q.shape[-1], window_left, window_right


def _check_tensors(q, k, v, cu_seqlens_q, cu_seqlens_k, direction):
    ops.check_same_device(q, k=k, v=v, cu_seqlens_q=cu_seqlens_q, cu_seqlens_k=cu_seqlens_k)
    ops.check_inputs(q, k, v, cu_seqlens_q, cu_seqlens_k, direction)
    if k.shape[-2] == 0 or q.shape[-2] == 0:
        raise ValueError("the head counts must be positive")
    if cu_seqlens_q is not None and cu_seqlens_q.shape[0] == 0:
        raise ValueError("cu_seqlens_q must hold at least one boundary")


def _forward(q, k, v, cu_seqlens_q, cu_seqlens_k, softmax_scale, window_left, window_right, sink_size):
    if not _fits(q, k, v, cu_seqlens_q, cu_seqlens_k):
        _check_tensors(q, k, v, cu_seqlens_q, cu_seqlens_k, ops.FORWARD)
    packed, device = cu_seqlens_q is not None, q.get_device()
    q, k, v = readable(q), readable(k), readable(v)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    softmax_lse = q.new_empty(ops.lse_shape(q, packed), dtype=torch.float32)
    if packed:
        cu_seqlens_q, cu_seqlens_k = ops._contiguous_int(cu_seqlens_q), ops._contiguous_int(cu_seqlens_k)
    problem = _problem(q, k, cu_seqlens_q, window_left, window_right)
    nbytes = _workspace_bytes("fwd", sink_size, packed, *problem)
    workspace = q.new_empty((nbytes,), dtype=torch.uint8) if nbytes else None
    lse_stride = softmax_lse.stride()
    arguments = PACK_FWD(
        *problem, softmax_scale, cu_seqlens_q.data_ptr() if packed else 0, cu_seqlens_k.data_ptr() if packed else 0, 0, 0, 0, 0, 0,
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), softmax_lse.data_ptr(), *_strides(q, packed),
        *_strides(k, packed), *_strides(v, packed), *_strides(out, packed), 0 if packed else lse_stride[0], lse_stride[-2],
        workspace.data_ptr() if nbytes else 0, nbytes,
    )
    on_device(device, entry("b200fa_sink_fwd_all_rows", ctypes.c_int32, ctypes.c_void_p), arguments, sink_size, stream_of(device))
    return out, softmax_lse


sink_forward = define(
    "sink_forward(Tensor q, Tensor k, Tensor v, Tensor? cu_seqlens_q, Tensor? cu_seqlens_k, float softmax_scale, "
    "int window_size_left, int window_size_right, int sink_size) -> (Tensor, Tensor)",
    _forward,
    lambda q, k, v, cu_seqlens_q, *unused: (
        q.new_empty(q.shape), q.new_empty(ops.lse_shape(q, cu_seqlens_q is not None), dtype=torch.float32)),
)


def _backward(dout, q, k, v, out, softmax_lse, cu_seqlens_q, cu_seqlens_k, softmax_scale, window_left, window_right, sink_size):
    packed, device = cu_seqlens_q is not None, q.get_device()
    if not _fits(q, k, v, cu_seqlens_q, cu_seqlens_k):
        _check_tensors(q, k, v, cu_seqlens_q, cu_seqlens_k, ops.BACKWARD)
    if not (
        dout.dtype is BF16 and out.dtype is BF16 and dout.shape == q.shape == out.shape and softmax_lse.dtype is torch.float32
        and softmax_lse.shape == ops.lse_shape(q, packed)
        and device == dout.get_device() == out.get_device() == softmax_lse.get_device()
    ):
        ops.check_same_device(q, dout=dout, out=out, softmax_lse=softmax_lse)
        ops.check_backward_operands(dout, q, k, v, out, softmax_lse, q, k, v, packed)
    dout, q, k, v, out, softmax_lse = readable(dout), readable(q), readable(k), readable(v), readable(out), softmax_lse.contiguous()
    dq = torch.empty_like(q, memory_format=torch.contiguous_format)
    dk = torch.empty_like(k, memory_format=torch.contiguous_format)
    dv = torch.empty_like(v, memory_format=torch.contiguous_format)
    if packed:
        cu_seqlens_q, cu_seqlens_k = ops._contiguous_int(cu_seqlens_q), ops._contiguous_int(cu_seqlens_k)
    problem = _problem(q, k, cu_seqlens_q, window_left, window_right)
    nbytes = _workspace_bytes("bwd", sink_size, packed, *problem)
    workspace = q.new_empty((max(nbytes, 1),), dtype=torch.uint8)
    lse_stride, stride_dk = softmax_lse.stride(), _strides(dk, packed)
    arguments = PACK_BWD(
        *problem, softmax_scale, cu_seqlens_q.data_ptr() if packed else 0, cu_seqlens_k.data_ptr() if packed else 0, 0, 0, 0, 0, 0,
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr(), softmax_lse.data_ptr(), dq.data_ptr(),
        dk.data_ptr(), dv.data_ptr(), *_strides(q, packed), *_strides(k, packed), *_strides(v, packed), *_strides(out, packed),
        *_strides(dout, packed), *_strides(dq, packed), *stride_dk, *stride_dk, 0 if packed else lse_stride[0], lse_stride[-2],
        workspace.data_ptr(), nbytes,
    )
    on_device(device, entry("b200fa_sink_bwd_all_rows", ctypes.c_int32, ctypes.c_void_p), arguments, sink_size, stream_of(device))
    return dq, dk, dv


sink_backward = define(
    "sink_backward(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor out, Tensor softmax_lse, Tensor? cu_seqlens_q, "
    "Tensor? cu_seqlens_k, float softmax_scale, int window_size_left, int window_size_right, int sink_size) -> "
    "(Tensor, Tensor, Tensor)",
    _backward,
    lambda dout, q, k, v, *unused: (q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)),
)


class FlashAttnSinkFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens_q, cu_seqlens_k, softmax_scale, window_left, window_right, sink_size, return_softmax):
        out, softmax_lse = sink_forward(q, k, v, cu_seqlens_q, cu_seqlens_k, softmax_scale, window_left, window_right, sink_size)
        ctx.save_for_backward(q, k, v, out, softmax_lse, cu_seqlens_q, cu_seqlens_k)
        ctx.options = (softmax_scale, window_left, window_right, sink_size)
        if not return_softmax:
            return out
        ctx.mark_non_differentiable(softmax_lse)
        return out, softmax_lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, *unused):
        return *sink_backward(dout, *ctx.saved_tensors, *ctx.options), None, None, None, None, None, None, None


def flash_attn_sink(q, k, v, cu_seqlens_q, cu_seqlens_k, sink_size, softmax_scale, causal, window_size, deterministic, return_softmax):
    ops.reject_unsupported(deterministic=deterministic)
    ops.check_sink_size(sink_size)
    left, right = window_size
    ops.require_window(left, right)
    refuse_tangents("attention with sinks", q, k, v)
    softmax_scale = ops.default_softmax_scale(softmax_scale, q.shape[-1])
    if not softmax_scale > 0:
        raise ValueError(f"attention with sinks needs a positive softmax_scale, got {softmax_scale}")
    # a bound of 2^30 keys is none for any sequence, and leaves room for the kernels' sums of positions in 32 bits
    window = tuple(min(int(bound), 2**30) for bound in (left, 0 if causal else right))
    arguments = (q, k, v, cu_seqlens_q, cu_seqlens_k, softmax_scale, *window, min(int(sink_size), 2**30))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return FlashAttnSinkFunc.apply(*arguments, return_softmax)
    result = sink_forward(*arguments)
    return result if return_softmax else result[0]
