"""Host layer of the paged key-value cache: validation, allocation and torch ops for attention of one new token over the
pages, for writing tokens into them, copying them, and keeping the books of which sequence holds which page.

The checks look at shapes, types, strides and devices only; what stands in the integer tensors (lengths, page numbers)
stays on the device and is bounds-checked by the kernels. Work is enqueued on the current stream of the tensors' device
and never synchronises. The ops are defined straight on the dispatcher: a decoding step calls them once per layer, and
the wrapper that `torch.library.custom_op` puts around a function costs more host time than the small kernels take.
"""
from __future__ import annotations

import torch

from . import lib as _lib
from . import ops

_library = torch.library.Library("zigfa", "FRAGMENT")


def _define(schema, implementation, fake):
    name = schema.split("(")[0]
    _library.define(schema)
    _library.impl(name, implementation, "CUDA")
    torch.library.register_fake(f"zigfa::{name}", fake, lib=_library)


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
    if not isinstance(page_size, int) or page_size < 1:
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


def _kv_cache(k_cache, v_cache):
    num_pages, page_size, heads, head_dim = k_cache.shape
    return _lib.KvCache(num_pages, page_size, heads, head_dim, k_cache.data_ptr(), v_cache.data_ptr(),
                        _lib.Stride3(*k_cache.stride()[:3]), _lib.Stride3(*v_cache.stride()[:3]))


def paged_forward(q, k_cache, v_cache, block_table, cache_seqlens, softmax_scale, window_left, sink_size):
    check_paged(q, k_cache, v_cache, block_table, cache_seqlens, window_left, sink_size)
    q, cache_seqlens = ops.readable(q), cache_seqlens.contiguous()
    batch, heads_q, head_dim = q.shape
    num_pages, page_size, heads_kv, _ = k_cache.shape
    out = torch.empty((batch, heads_q, head_dim), dtype=torch.bfloat16, device=q.device)
    softmax_lse = torch.empty((batch, heads_q), dtype=torch.float32, device=q.device)
    library = _lib.library()
    args = _lib.PagedArgs(
        batch, heads_q, heads_kv, head_dim, num_pages, page_size, block_table.shape[1], window_left, sink_size,
        softmax_scale, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(),
        cache_seqlens.data_ptr(), out.data_ptr(), softmax_lse.data_ptr(), _lib.Stride2(*q.stride()[:2]),
        _lib.Stride3(*k_cache.stride()[:3]), _lib.Stride3(*v_cache.stride()[:3]), _lib.Stride2(*out.stride()[:2]),
        _table_stride(block_table),
    )
    with torch.cuda.device(q.device):
        workspace = ops._workspace(library.b200fa_paged_decode_workspace_bytes(args), q.device)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), workspace.numel()
        _lib.check(library.b200fa_paged_decode(args, ops._stream(q.device)))
    return out, softmax_lse


_define(
    "paged_forward(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor cache_seqlens, float softmax_scale, "
    "int window_left, int sink_size) -> (Tensor, Tensor)",
    paged_forward,
    lambda q, *unused: (q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)),
)


def append_kv(k, v, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens):
    check_append(k, v, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens)
    k, v, cache_seqlens = ops.readable(k), ops.readable(v), cache_seqlens.contiguous()
    packed = cu_seqlens is not None
    cu_seqlens = ops._contiguous_int(cu_seqlens)
    args = _lib.AppendArgs(
        _kv_cache(k_cache, v_cache), k.data_ptr(), v.data_ptr(), _lib.strides3(k, packed), _lib.strides3(v, packed),
        k.shape[0] if packed else k.shape[1], _lib.pointer(cu_seqlens), cache_seqlens.data_ptr(), block_table.data_ptr(),
        _table_stride(block_table), cache_seqlens.shape[0], block_table.shape[1],
    )
    with torch.cuda.device(k.device):
        _lib.check(_lib.library().b200fa_append_kv(args, ops._stream(k.device)))


_define(
    "append_kv(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor block_table, Tensor cache_seqlens, "
    "Tensor? cu_seqlens) -> ()",
    append_kv,
    lambda *unused: None,
)


def copy_pages(k_cache, v_cache, source_pages, target_pages):
    check_copy(k_cache, v_cache, source_pages, target_pages)
    source_pages, target_pages = source_pages.contiguous(), target_pages.contiguous()
    with torch.cuda.device(k_cache.device):
        _lib.check(_lib.library().b200fa_copy_pages(
            _kv_cache(k_cache, v_cache), source_pages.data_ptr(), target_pages.data_ptr(), source_pages.shape[0],
            ops._stream(k_cache.device)))


_define(
    "copy_pages(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor source_pages, Tensor target_pages) -> ()",
    copy_pages,
    lambda *unused: None,
)


def _keep_books(name, block_table, page_refs, cache_seqlens, page_size, rows, pairs, *extra):
    """Runs one of the bookkeeping calls; returns (block_table, page_refs, source_pages, target_pages)."""
    sequences, max_pages = block_table.shape
    num_pages, device = page_refs.shape[0], block_table.device
    page_refs = page_refs.contiguous()
    cache_seqlens = ops._contiguous_int(cache_seqlens)
    extra = [tensor.contiguous() for tensor in extra]

    def ints(*shape):
        return torch.empty(shape, dtype=torch.int32, device=device)

    table_out, refs_out = ints(rows, max_pages), ints(num_pages)
    source, target = (ints(pairs), ints(pairs)) if pairs is not None else (None, None)
    outputs = [ints(rows)] if name == "fork" else []
    library = _lib.library()
    nbytes = 0 if name == "free" else library.b200fa_pages_workspace_bytes(num_pages)
    with torch.cuda.device(device):
        workspace = ops._workspace(nbytes, device)
        args = _lib.PagesArgs(
            sequences, rows, max_pages, num_pages, page_size, block_table.data_ptr(), _table_stride(block_table),
            page_refs.data_ptr(), _lib.pointer(cache_seqlens), table_out.data_ptr(), refs_out.data_ptr(),
            _lib.pointer(source), _lib.pointer(target), workspace.data_ptr(), nbytes,
        )
        function = getattr(library, f"b200fa_{name}_pages")
        _lib.check(function(args, *(tensor.data_ptr() for tensor in (*extra, *outputs)), ops._stream(device)))
    return table_out, refs_out, source, target, *outputs


def reserve_pages(block_table, cache_seqlens, new_tokens, page_refs, page_size):
    check_books(block_table, page_refs, cache_seqlens=cache_seqlens, new_tokens=new_tokens)
    check_page_size(page_size)
    return _keep_books("reserve", block_table, page_refs, cache_seqlens, page_size, block_table.shape[0], None, new_tokens)[:2]


def fork_pages(block_table, cache_seqlens, page_refs, parents, page_size):
    check_books(block_table, page_refs, cache_seqlens=cache_seqlens)
    check_ints("parents", parents, None)
    ops.check_same_device(block_table, parents=parents)
    check_page_size(page_size)
    rows = parents.shape[0]
    table, refs, source, target, lengths = _keep_books("fork", block_table, page_refs, cache_seqlens, page_size, rows, rows, parents)
    return table, lengths, refs, source, target


def free_pages(block_table, page_refs, first_entry, last_entry):
    check_books(block_table, page_refs, first_entry=first_entry, last_entry=last_entry)
    return _keep_books("free", block_table, page_refs, None, 1, block_table.shape[0], None, first_entry, last_entry)[:2]


def compact_pages(block_table, page_refs):
    check_books(block_table, page_refs)
    return _keep_books("compact", block_table, page_refs, None, 1, block_table.shape[0], page_refs.shape[0] // 2)


def _like(table, *shape):
    return table.new_empty(shape)


_define(
    "reserve_pages(Tensor block_table, Tensor cache_seqlens, Tensor new_tokens, Tensor page_refs, int page_size) -> (Tensor, Tensor)",
    reserve_pages,
    lambda table, lengths, new, refs, page_size: (_like(table, *table.shape), _like(refs, *refs.shape)),
)
_define(
    "fork_pages(Tensor block_table, Tensor cache_seqlens, Tensor page_refs, Tensor parents, int page_size) -> "
    "(Tensor, Tensor, Tensor, Tensor, Tensor)",
    fork_pages,
    lambda table, lengths, refs, parents, page_size: (
        _like(table, parents.shape[0], table.shape[1]), _like(parents, *parents.shape), _like(refs, *refs.shape),
        _like(parents, *parents.shape), _like(parents, *parents.shape)),
)
_define(
    "free_pages(Tensor block_table, Tensor page_refs, Tensor first_entry, Tensor last_entry) -> (Tensor, Tensor)",
    free_pages,
    lambda table, refs, *unused: (_like(table, *table.shape), _like(refs, *refs.shape)),
)
_define(
    "compact_pages(Tensor block_table, Tensor page_refs) -> (Tensor, Tensor, Tensor, Tensor)",
    compact_pages,
    lambda table, refs: (_like(table, *table.shape), _like(refs, *refs.shape), _like(refs, refs.shape[0] // 2),
                         _like(refs, refs.shape[0] // 2)),
)


# ------------------------------------------------------------------------------------------------ public entry points
def flash_attn_paged(q, k_cache, v_cache, block_table, cache_seqlens, softmax_scale, window_size, sink_size, return_lse):
    left, right = window_size
    ops.require_window(left, right)
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        raise NotImplementedError("paged attention has no backward pass: call it under torch.no_grad()")
    softmax_scale = ops.default_softmax_scale(softmax_scale, q.shape[-1])
    out, softmax_lse = torch.ops.zigfa.paged_forward(q, k_cache, v_cache, block_table, cache_seqlens, softmax_scale, left,
                                                     sink_size)
    return (out, softmax_lse) if return_lse else out
