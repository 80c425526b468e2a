"""Short way from the public functions to the C entries, for operators that are called once per layer and token.

An operator is registered with the dispatcher (schema, CUDA implementation, fake implementation for tracing), but plain
arguments in eager mode go straight to the implementation, which the host needs for calls that take it longer than the GPU:
appending one token to 64 sequences 11.2 us instead of 22.8, paged attention of one sequence 3 us less than through it.
Argument structures are packed with `struct` (0.3 us for 30 fields) in the layout of include/b200fa.h.
"""
from __future__ import annotations

import ctypes
import functools
import struct

import torch
from torch.autograd import forward_ad

from . import lib as _lib

_library = torch.library.Library("zigfa", "FRAGMENT")
_PLAIN = {torch.Tensor, torch.nn.Parameter, type(None), int, float}
_is_compiling = torch.compiler.is_compiling
_modes = torch._C._len_torch_dispatch_stack
_increment = torch._C._increment_version
_transform = torch._C._functorch.peek_interpreter_stack  # the innermost of torch.vmap, torch.func.grad, ...; None outside

PROBLEM = "8if7P"  # b200fa_problem
PACK_FWD = struct.Struct(f"@{PROBLEM}5P14qPN").pack
PACK_BWD = struct.Struct(f"@{PROBLEM}9P26qPN").pack
PACK_PAGED = struct.Struct("@9if7P11qPN").pack
KV_CACHE = "4i2P6q"
PACK_KV_CACHE = struct.Struct(f"@{KV_CACHE}").pack
PACK_APPEND = struct.Struct(f"@{KV_CACHE}2P6qq3Pq2i").pack
PACK_PAGES = struct.Struct("@5iPq7PN").pack


def raise_versions(tensors):
    try:
        _increment(tensors)
    except RuntimeError:  # tensors made in inference mode have no version counter
        for tensor in tensors:
            if not tensor.is_inference():
                _increment((tensor,))


def define(schema, implementation, fake, written=()):
    """Registers zigfa::<schema> and returns the function that the host layer calls. `written` = (position, name) of the
    arguments that the operator writes into, which stand next to each other: their version counters go up, as with any
    in-place operation, so that a backward pass that has saved one of them raises instead of reading the new values."""
    name = schema.split("(")[0]
    if written:  # as the other operators that write into their arguments: the registration counts the versions
        op = torch.library.custom_op(f"zigfa::{name}", implementation, mutates_args=[argument for _, argument in written],
                                     device_types="cuda", schema=schema[len(name):])
        op.register_fake(fake)
    else:
        _library.define(schema)
        _library.impl(name, implementation, "CUDA")
        torch.library.register_fake(f"zigfa::{name}", fake, lib=_library)
    op = getattr(torch.ops.zigfa, name).default
    where = slice(written[0][0], written[-1][0] + 1) if written else None

    @functools.wraps(implementation)
    def call(*arguments):
        # Every argument counts: the implementation takes addresses, which a tensor subclass or a batch of tensors lacks.
        if (
            _PLAIN.issuperset(map(type, arguments)) and arguments[0].is_cuda and not _is_compiling() and not _modes()
            and _transform() is None
        ):
            result = implementation(*arguments)
            if written:
                raise_versions(arguments[where])
            return result
        return op(*arguments)  # traced, transformed, or without a kernel for the device

    return call


@functools.cache
def entry(name, *arguments):
    """The C function `name` taking a packed structure first, then `arguments`."""
    function = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_char_p, *arguments)((name, _lib.library()))
    return function


def on_device(index, function, *arguments):
    """function(*arguments) with the device made current; raises what its status says."""
    if torch._C._cuda_getDevice() == index:
        status = function(*arguments)
    else:
        with torch.cuda.device(index):
            status = function(*arguments)
    if status:
        _lib.check(status)


stream_of = torch._C._cuda_getCurrentRawStream


def readable(tensor):
    """`tensor`, or a contiguous copy where the kernels cannot address it (ops.kernel_ready) -- of three dimensions or more."""
    stride = tensor.stride()
    if stride[-1] == 1 and not (stride[0] | stride[1] | stride[-2]) & 7 and not tensor.data_ptr() & 15:
        return tensor
    return tensor.clone(memory_format=torch.contiguous_format)


def refuse_tangents(what, *tensors):
    """Forward-mode derivatives: a call that does not go through an autograd Function would drop them silently."""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(tensor).tangent is not None for tensor in tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def refuse_gradients(what, *tensors):
    refuse_tangents(what, *tensors)
    if torch.is_grad_enabled():
        for tensor in tensors:
            if tensor.requires_grad:
                raise NotImplementedError(f"{what} has no backward pass: call it under torch.no_grad()")
