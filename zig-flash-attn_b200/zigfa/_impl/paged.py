"""Host layer of the paged key-value cache: validation, allocation and torch ops for attention of one new token over the
pages, for writing tokens into them, copying them, and keeping the books of which sequence holds which page.

The checks look at shapes, types, strides and devices only; what stands in the integer tensors (lengths, page numbers)
stays on the device and is bounds-checked by the kernels. Each operation tests the whole of its conditions in one expression
and turns to the check that names the fault only when that fails. Work is enqueued on the current stream of the tensors'
device and never synchronises.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import lib as _lib
from . import ops
from .dispatch import (PACK_APPEND, PACK_KV_CACHE, PACK_PAGED, PACK_PAGES, define, entry, on_device, readable,
                       refuse_gradients, stream_of)

BF16, INT32 = torch.bfloat16, torch.int32


# ------------------------------------------------------------------------------------------------ validation
def check_ints(name, tensor, *shape):
    """An int32 tensor of this shape (None: any size); a table's columns are contiguous, vectors may be strided."""
    if tensor.dtype != torch.int32 or tensor.dim() != len(shape) or any(
            want is not None and want != size for want, size in zip(shape, tensor.shape)):
        wanted = ", ".join("n" if want is None else str(want) for want in shape)
        raise ValueError(f"{name} must be an int32 tensor of shape ({wanted}), got {tensor.dtype} {tuple(tensor.shape)}")
    if len(shape) == 2 and tensor.stride(-1) != 1 and tensor.shape[-1] > 1:
        raise ValueError(f"{name} must have contiguous columns")


def check_cache(k_cache, v_cache):
    for name, tensor in (("k_cache", k_cache), ("v_cache", v_cache)):
        if tensor.dtype != torch.bfloat16:
            raise ValueError(f"{name} must be bfloat16, got {tensor.dtype}")
        if tensor.dim() != 4:
            raise ValueError(f"{name} must have 4 dimensions (pages, page size, heads, head_dim), got {tensor.dim()}")
    if k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must have the same shape")
    if 0 in k_cache.shape[1:]:
        raise ValueError("the pages of a cache must not be empty")
    for name, tensor in (("k_cache", k_cache), ("v_cache", v_cache)):
        if tensor.numel() and not ops.kernel_ready(tensor):  # a cache is read and written in place, never copied
            raise ValueError(f"{name} must be 16-byte aligned with a contiguous last dimension and strides that are multiples of 8 elements")


def check_page_size(page_size):
    if not isinstance(page_size, int) or not 0 < page_size < 2**31:
        raise ValueError(f"page_size must be a positive integer, got {page_size!r}")


def check_paged(q, k_cache, v_cache, block_table, cache_seqlens, window_left, sink_size):
    if q.dtype != torch.bfloat16:
        raise ValueError(f"q must be bfloat16, got {q.dtype}")
    if q.dim() != 3:
        raise ValueError(f"q must have 3 dimensions (sequences, heads, head_dim), got {q.dim()}")
    check_cache(k_cache, v_cache)
    supported = ops.head_dims()
    if q.shape[-1] != k_cache.shape[-1] or q.shape[-1] not in supported:
        raise ValueError(f"head_dim must be one of {list(supported)} and equal for q and the caches")
    if q.shape[1] == 0 or q.shape[1] % k_cache.shape[2]:
        raise ValueError("the query head count must be a multiple of the key head count (num_heads_q % num_heads_k)")
    check_ints("block_table", block_table, q.shape[0], None)
    check_ints("cache_seqlens", cache_seqlens, q.shape[0])
    ops.require_window(window_left, -1)
    ops.check_sink_size(sink_size)
    ops.check_same_device(q, k_cache=k_cache, v_cache=v_cache, block_table=block_table, cache_seqlens=cache_seqlens)


def check_append(k, v, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens):
    check_cache(k_cache, v_cache)
    rank = 4 if cu_seqlens is None else 3
    for name, tensor in (("k", k), ("v", v)):
        if tensor.dtype != torch.bfloat16:
            raise ValueError(f"{name} must be bfloat16, got {tensor.dtype}")
        if tensor.dim() != rank:
            raise ValueError(f"{name} must have {rank} dimensions, got {tensor.dim()}")
    if k.shape != v.shape:
        raise ValueError("k and v must have the same shape")
    if k.shape[-2:] != k_cache.shape[-2:]:
        raise ValueError("k and v must have the heads and the head_dim of the caches")
    if k.shape[-1] % 8 or k.shape[-1] > 1024:
        raise ValueError(f"head_dim must be a multiple of 8 of at most 1024, got {k.shape[-1]}")
    batch = cache_seqlens.shape[0] if cache_seqlens.dim() == 1 else -1
    check_ints("cache_seqlens", cache_seqlens, None)
    check_ints("block_table", block_table, batch, None)
    if cu_seqlens is not None:
        check_ints("cu_seqlens", cu_seqlens, batch + 1)
    elif k.shape[0] != batch:
        raise ValueError("k, block_table and cache_seqlens must have the same number of sequences")
    ops.check_same_device(k, v=v, k_cache=k_cache, v_cache=v_cache, block_table=block_table, cache_seqlens=cache_seqlens,
                      cu_seqlens=cu_seqlens)


def check_copy(k_cache, v_cache, source_pages, target_pages):
    check_cache(k_cache, v_cache)
    if k_cache.shape[-1] % 8 or k_cache.shape[-1] > 1024:
        raise ValueError(f"head_dim must be a multiple of 8 of at most 1024, got {k_cache.shape[-1]}")
    check_ints("source_pages", source_pages, None)
    check_ints("target_pages", target_pages, source_pages.shape[0])
    ops.check_same_device(k_cache, v_cache=v_cache, source_pages=source_pages, target_pages=target_pages)


def check_books(block_table, page_refs, **per_sequence):
    check_ints("block_table", block_table, None, None)
    check_ints("page_refs", page_refs, None)
    for name, tensor in per_sequence.items():
        check_ints(name, tensor, block_table.shape[0])
    ops.check_same_device(block_table, page_refs=page_refs, **per_sequence)


# ------------------------------------------------------------------------------------------------ launches
def _table_stride(block_table):
    return block_table.stride(0) if block_table.shape[0] > 1 else block_table.shape[1]


def _is_table(block_table):
    return block_table.dtype is INT32 and block_table.dim() == 2 and (block_table.stride(1) == 1 or block_table.shape[1] <= 1)


def _is_vector(tensor, size):
    return tensor.dtype is INT32 and tensor.shape == (size,)


def _is_cache(k_cache, v_cache):
    shape, k_stride, v_stride = k_cache.shape, k_cache.stride(), v_cache.stride()
    return (
        k_cache.dtype is BF16 and v_cache.dtype is BF16 and len(shape) == 4 and v_cache.shape == shape
        and shape[1] > 0 and shape[2] > 0 and shape[3] > 0 and k_stride[3] == 1 == v_stride[3]
        and not (k_stride[0] | k_stride[1] | k_stride[2] | v_stride[0] | v_stride[1] | v_stride[2]) & 7
        and not (k_cache.data_ptr() | v_cache.data_ptr()) & 15
    )


@functools.lru_cache(maxsize=4096)
def _paged_workspace(batch, heads_q, heads_kv, head_dim, page_size, max_pages, window_left, sink_size):
    args = _lib.PagedArgs(batch=batch, heads_q=heads_q, heads_kv=heads_kv, head_dim=head_dim, page_size=page_size,
                          max_pages=max_pages, window_left=window_left, sink_size=sink_size)
    return _lib.library().b200fa_paged_decode_workspace_bytes(args)


def _paged_forward(q, k_cache, v_cache, block_table, cache_seqlens, softmax_scale, window_left, sink_size):
    shape, cache_shape, device = q.shape, k_cache.shape, q.get_device()
    if not (
        q.dtype is BF16 and len(shape) == 3 and _is_cache(k_cache, v_cache) and shape[2] == cache_shape[3]
        and _is_table(block_table) and block_table.shape[0] == shape[0] and _is_vector(cache_seqlens, shape[0])
        and device == k_cache.get_device() == v_cache.get_device() == block_table.get_device() == cache_seqlens.get_device()
        and type(sink_size) is int and 0 <= sink_size < 2**31
    ):
        check_paged(q, k_cache, v_cache, block_table, cache_seqlens, window_left, sink_size)
    batch, heads_q, head_dim = shape
    num_pages, page_size, heads_kv, _ = cache_shape
    max_pages = block_table.shape[1]
    if not cache_seqlens.is_contiguous():
        cache_seqlens = cache_seqlens.contiguous()
    q = readable(q)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    softmax_lse = q.new_empty((batch, heads_q), dtype=torch.float32)
    nbytes = _paged_workspace(batch, heads_q, heads_kv, head_dim, page_size, max_pages, window_left, sink_size)
    workspace = q.new_empty((nbytes,), dtype=torch.uint8) if nbytes else None
    q_stride, k_stride, v_stride = q.stride(), k_cache.stride(), v_cache.stride()
    packed = PACK_PAGED(
        batch, heads_q, heads_kv, head_dim, num_pages, page_size, max_pages, window_left, sink_size, softmax_scale,
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), cache_seqlens.data_ptr(), out.data_ptr(),
        softmax_lse.data_ptr(), q_stride[0], q_stride[1], k_stride[0], k_stride[1], k_stride[2],
        v_stride[0], v_stride[1], v_stride[2], heads_q * head_dim, head_dim, _table_stride(block_table),
        workspace.data_ptr() if nbytes else 0, nbytes,
    )
    on_device(device, entry("b200fa_paged_decode", ctypes.c_void_p), packed, stream_of(device))
    return out, softmax_lse


paged_forward = define(
    "paged_forward(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor cache_seqlens, float softmax_scale, "
    "int window_left, int sink_size) -> (Tensor, Tensor)",
    _paged_forward,
    lambda q, *unused: (q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)),
)


def _append_kv(k, v, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens):
    packed, shape, device, batch = cu_seqlens is not None, k.shape, k.get_device(), cache_seqlens.shape[0] if cache_seqlens.dim() else 0
    if not (
        k.dtype is BF16 and v.dtype is BF16 and v.shape == shape and len(shape) == (3 if packed else 4)
        and _is_cache(k_cache, v_cache) and shape[-2:] == k_cache.shape[-2:] and not shape[-1] & 7 and shape[-1] <= 1024
        and _is_vector(cache_seqlens, batch) and _is_table(block_table) and block_table.shape[0] == batch
        and (_is_vector(cu_seqlens, batch + 1) and cu_seqlens.get_device() == device if packed else shape[0] == batch)
        and device == v.get_device() == k_cache.get_device() == v_cache.get_device() == block_table.get_device() == cache_seqlens.get_device()
    ):
        check_append(k, v, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens)
    k, v, cache_seqlens, cu_seqlens = readable(k), readable(v), ops._contiguous_int(cache_seqlens), ops._contiguous_int(cu_seqlens)
    num_pages, page_size, heads, head_dim = k_cache.shape
    arguments = PACK_APPEND(
        num_pages, page_size, heads, head_dim, k_cache.data_ptr(), v_cache.data_ptr(), *k_cache.stride()[:3],
        *v_cache.stride()[:3], k.data_ptr(), v.data_ptr(), *((0, *k.stride()[:2]) if packed else k.stride()[:3]),
        *((0, *v.stride()[:2]) if packed else v.stride()[:3]), shape[0] if packed else shape[1],
        cu_seqlens.data_ptr() if packed else 0, cache_seqlens.data_ptr(), block_table.data_ptr(), _table_stride(block_table),
        batch, block_table.shape[1],
    )
    on_device(device, entry("b200fa_append_kv", ctypes.c_void_p), arguments, stream_of(device))


append_kv = define(
    "append_kv(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor block_table, Tensor cache_seqlens, "
    "Tensor? cu_seqlens) -> ()",
    _append_kv,
    lambda *unused: None,
    written=((2, "k_cache"), (3, "v_cache")),
)


def _copy_pages(k_cache, v_cache, source_pages, target_pages):
    device, count = k_cache.get_device(), source_pages.numel()
    if not (
        _is_cache(k_cache, v_cache) and not k_cache.shape[3] & 7 and k_cache.shape[3] <= 1024 and _is_vector(source_pages, count)
        and _is_vector(target_pages, count)
        and device == v_cache.get_device() == source_pages.get_device() == target_pages.get_device()
    ):
        check_copy(k_cache, v_cache, source_pages, target_pages)
    source_pages, target_pages = ops._contiguous_int(source_pages), ops._contiguous_int(target_pages)
    cache = PACK_KV_CACHE(*k_cache.shape, k_cache.data_ptr(), v_cache.data_ptr(), *k_cache.stride()[:3], *v_cache.stride()[:3])
    call = entry("b200fa_copy_pages", ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32, ctypes.c_void_p)
    on_device(device, call, cache, source_pages.data_ptr(), target_pages.data_ptr(), count, stream_of(device))


copy_pages = define(
    "copy_pages(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor source_pages, Tensor target_pages) -> ()",
    _copy_pages,
    lambda *unused: None,
    written=((0, "k_cache"), (1, "v_cache")),
)


def _are_books(block_table, page_refs, *per_sequence):
    sequences, device = block_table.shape[0] if block_table.dim() else 0, block_table.get_device()
    return (
        _is_table(block_table) and page_refs.dtype is INT32 and page_refs.dim() == 1 and page_refs.get_device() == device
        and all(_is_vector(tensor, sequences) and tensor.get_device() == device for tensor in per_sequence)
    )


def _like(tensor):
    return torch.empty_like(tensor, memory_format=torch.contiguous_format)


def _keep_books(name, block_table, page_refs, cache_seqlens, page_size, table_out, source, target, *extra):
    """Runs one of the bookkeeping calls; returns the new page_refs."""
    sequences, max_pages = block_table.shape
    num_pages, device = page_refs.shape[0], block_table.get_device()
    page_refs = ops._contiguous_int(page_refs)
    refs_out = _like(page_refs)
    scratch = None if name == "free" else _like(page_refs)
    arguments = PACK_PAGES(
        sequences, table_out.shape[0], max_pages, num_pages, page_size, block_table.data_ptr(), _table_stride(block_table),
        page_refs.data_ptr(), 0 if cache_seqlens is None else cache_seqlens.data_ptr(), table_out.data_ptr(), refs_out.data_ptr(),
        0 if source is None else source.data_ptr(), 0 if target is None else target.data_ptr(),
        0 if scratch is None else scratch.data_ptr(), 0 if scratch is None else 4 * num_pages,
    )
    call = entry(f"b200fa_{name}_pages", *([ctypes.c_void_p] * (len(extra) + 1)))
    on_device(device, call, arguments, *(tensor.data_ptr() for tensor in extra), stream_of(device))
    return refs_out


def _reserve_pages(block_table, cache_seqlens, new_tokens, page_refs, page_size):
    if not (_are_books(block_table, page_refs, cache_seqlens, new_tokens) and type(page_size) is int and page_size > 0):
        check_books(block_table, page_refs, cache_seqlens=cache_seqlens, new_tokens=new_tokens)
        check_page_size(page_size)
    table = _like(block_table)
    refs = _keep_books("reserve", block_table, page_refs, ops._contiguous_int(cache_seqlens), page_size, table, None, None,
                       ops._contiguous_int(new_tokens))
    return table, refs


def _fork_pages(block_table, cache_seqlens, page_refs, parents, page_size):
    if not (
        _are_books(block_table, page_refs, cache_seqlens) and type(page_size) is int and page_size > 0
        and _is_vector(parents, parents.numel()) and parents.get_device() == block_table.get_device()
    ):
        check_books(block_table, page_refs, cache_seqlens=cache_seqlens)
        check_ints("parents", parents, None)
        ops.check_same_device(block_table, parents=parents)
        check_page_size(page_size)
    table = block_table.new_empty((parents.shape[0], block_table.shape[1]))
    parents = ops._contiguous_int(parents)
    lengths, source, target = _like(parents), _like(parents), _like(parents)
    refs = _keep_books("fork", block_table, page_refs, ops._contiguous_int(cache_seqlens), page_size, table, source, target,
                       parents, lengths)
    return table, lengths, refs, source, target


def _free_pages(block_table, page_refs, first_entry, last_entry):
    if not _are_books(block_table, page_refs, first_entry, last_entry):
        check_books(block_table, page_refs, first_entry=first_entry, last_entry=last_entry)
    table = _like(block_table)
    refs = _keep_books("free", block_table, page_refs, None, 1, table, None, None, ops._contiguous_int(first_entry),
                       ops._contiguous_int(last_entry))
    return table, refs


def _compact_pages(block_table, page_refs):
    if not _are_books(block_table, page_refs):
        check_books(block_table, page_refs)
    table, pairs = _like(block_table), (page_refs.shape[0] // 2,)
    source, target = page_refs.new_empty(pairs), page_refs.new_empty(pairs)
    refs = _keep_books("compact", block_table, page_refs, None, 1, table, source, target)
    return table, refs, source, target


reserve_pages = define(
    "reserve_pages(Tensor block_table, Tensor cache_seqlens, Tensor new_tokens, Tensor page_refs, int page_size) -> (Tensor, Tensor)",
    _reserve_pages,
    lambda table, lengths, new, refs, page_size: (table.new_empty(table.shape), refs.new_empty(refs.shape)),
)
fork_pages = define(
    "fork_pages(Tensor block_table, Tensor cache_seqlens, Tensor page_refs, Tensor parents, int page_size) -> "
    "(Tensor, Tensor, Tensor, Tensor, Tensor)",
    _fork_pages,
    lambda table, lengths, refs, parents, page_size: (
        table.new_empty((parents.shape[0], table.shape[1])), parents.new_empty(parents.shape), refs.new_empty(refs.shape),
        parents.new_empty(parents.shape), parents.new_empty(parents.shape)),
)
free_pages = define(
    "free_pages(Tensor block_table, Tensor page_refs, Tensor first_entry, Tensor last_entry) -> (Tensor, Tensor)",
    _free_pages,
    lambda table, refs, *unused: (table.new_empty(table.shape), refs.new_empty(refs.shape)),
)
compact_pages = define(
    "compact_pages(Tensor block_table, Tensor page_refs) -> (Tensor, Tensor, Tensor, Tensor)",
    _compact_pages,
    lambda table, refs: (table.new_empty(table.shape), refs.new_empty(refs.shape), refs.new_empty((refs.shape[0] // 2,)),
                         refs.new_empty((refs.shape[0] // 2,))),
)


# ------------------------------------------------------------------------------------------------ public entry points
def flash_attn_paged(q, k_cache, v_cache, block_table, cache_seqlens, softmax_scale, window_size, sink_size, return_lse):
    left, right = window_size
    if not (type(left) is int and type(right) is int and -1 <= left < 2**31 and right >= -1):
        ops.require_window(left, right)
        left = min(int(left), 2**31 - 1)
    if type(sink_size) is not int:
        ops.check_sink_size(sink_size)
        sink_size = int(sink_size)
    refuse_gradients("paged attention", q, k_cache, v_cache)
    softmax_scale = ops.default_softmax_scale(softmax_scale, q.shape[-1])
    result = paged_forward(q, k_cache, v_cache, block_table, cache_seqlens, softmax_scale, left, sink_size)
    return result if return_lse else result[0]


def append_paged_kv(k, v, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens):
    refuse_gradients("writing into a cache", k, v, k_cache, v_cache)
    append_kv(k, v, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens)


def copy_kv_pages(k_cache, v_cache, source_pages, target_pages):
    refuse_gradients("copying pages", k_cache, v_cache)
    copy_pages(k_cache, v_cache, source_pages, target_pages)
