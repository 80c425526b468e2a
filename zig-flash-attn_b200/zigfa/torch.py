"""Public attention functions. Signatures, defaults and return values follow the reference API
(reference src/zigfa/torch.py:17-298) so that callers can switch packages without edits. Each function hands its
arguments, in declaration order, to the autograd Function of the same family in `_impl.ops`; torch is imported only
when a function is first called.
"""
from __future__ import annotations

import dataclasses
from typing import TYPE_CHECKING

if TYPE_CHECKING:
    from torch import Tensor


@dataclasses.dataclass(frozen=True, slots=True)
class InterSequenceMetadata:
    """Prepared visibility of an inter-sequence batch: (transposed bits, visible-key prefix sums, visible-query
    prefix sums). Treat as read-only; reuse while boundaries, bits and device stay the same."""

    _tensors: tuple[Tensor, Tensor, Tensor]


def flash_attn_func(
    q: Tensor, k: Tensor, v: Tensor, softmax_scale: float | None = None, causal: bool = False,
    qv: Tensor | None = None, q_descale: Tensor | None = None, k_descale: Tensor | None = None,
    v_descale: Tensor | None = None, window_size: tuple[int, int] = (-1, -1), attention_chunk: int = 0,
    softcap: float = 0.0, num_splits: int = 1, pack_gqa: bool | None = None, deterministic: bool = False,
    sm_margin: int = 0, return_attn_probs: bool = False,
) -> Tensor | tuple[Tensor, Tensor]:
    from ._impl import ops

    arguments = (q, k, v, softmax_scale, causal, qv, q_descale, k_descale, v_descale, window_size, attention_chunk, softcap, num_splits, pack_gqa, deterministic, sm_margin, return_attn_probs)
    return ops.FlashAttnFunc.apply(*arguments)


def flash_attn_varlen_func(
    q: Tensor, k: Tensor, v: Tensor, cu_seqlens_q: Tensor, cu_seqlens_k: Tensor, max_seqlen_q: int,
    max_seqlen_k: int, seqused_q: Tensor | None = None, seqused_k: Tensor | None = None,
    softmax_scale: float | None = None, causal: bool = False, qv: Tensor | None = None,
    q_descale: Tensor | None = None, k_descale: Tensor | None = None, v_descale: Tensor | None = None,
    window_size: tuple[int, int] = (-1, -1), attention_chunk: int = 0, softcap: float = 0.0, num_splits: int = 1,
    pack_gqa: bool | None = None, deterministic: bool = False, sm_margin: int = 0, return_attn_probs: bool = False,
) -> Tensor | tuple[Tensor, Tensor]:
    from ._impl import ops

    arguments = (q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, seqused_q, seqused_k, softmax_scale, causal, qv, q_descale, k_descale, v_descale, window_size, attention_chunk, softcap, num_splits, pack_gqa, deterministic, sm_margin, return_attn_probs)
    return ops.FlashAttnVarlenFunc.apply(*arguments)


def flash_attn_qkvpacked_func(
    qkv: Tensor, softmax_scale: float | None = None, causal: bool = False, q_descale: Tensor | None = None,
    k_descale: Tensor | None = None, v_descale: Tensor | None = None, window_size: tuple[int, int] = (-1, -1),
    attention_chunk: int = 0, softcap: float = 0.0, deterministic: bool = False, num_heads_q: int | None = None,
    sm_margin: int = 0, return_attn_probs: bool = False,
) -> Tensor | tuple[Tensor, Tensor]:
    from ._impl import ops

    arguments = (qkv, softmax_scale, causal, q_descale, k_descale, v_descale, window_size, attention_chunk, softcap, deterministic, num_heads_q, sm_margin, return_attn_probs)
    return ops.FlashAttnQKVPackedFunc.apply(*arguments)


def flash_attn_kvpacked_func(
    q: Tensor, kv: Tensor, dropout_p: float = 0.0, softmax_scale: float | None = None, causal: bool = False,
    window_size: tuple[int, int] = (-1, -1), softcap: float = 0.0, alibi_slopes: Tensor | None = None,
    deterministic: bool = False, return_attn_probs: bool = False,
) -> Tensor | tuple[Tensor, Tensor]:
    from ._impl import ops

    arguments = (q, kv, dropout_p, softmax_scale, causal, window_size, softcap, alibi_slopes, deterministic, return_attn_probs)
    return ops.FlashAttnKVPackedFunc.apply(*arguments)


def flash_attn_varlen_kvpacked_func(
    q: Tensor, kv: Tensor, cu_seqlens_q: Tensor, cu_seqlens_k: Tensor, max_seqlen_q: int, max_seqlen_k: int,
    dropout_p: float = 0.0, softmax_scale: float | None = None, causal: bool = False,
    window_size: tuple[int, int] = (-1, -1), softcap: float = 0.0, alibi_slopes: Tensor | None = None,
    deterministic: bool = False, return_attn_probs: bool = False,
) -> Tensor | tuple[Tensor, Tensor]:
    from ._impl import ops

    arguments = (q, kv, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, dropout_p, softmax_scale, causal, window_size, softcap, alibi_slopes, deterministic, return_attn_probs)
    return ops.FlashAttnVarlenKVPackedFunc.apply(*arguments)


def flash_attn_inter_sequence_func(
    q: Tensor, k: Tensor, v: Tensor, cu_seqlens_q: Tensor, cu_seqlens_k: Tensor, max_seqlen_q: int,
    max_seqlen_k: int, visibility_bits: Tensor, softmax_scale: float | None = None, causal: bool = False,
    window_size: tuple[int, int] = (-1, -1), window_sizes: Tensor | None = None,
    metadata: InterSequenceMetadata | None = None, deterministic: bool = False, return_attn_probs: bool = False,
) -> Tensor | tuple[Tensor, Tensor]:
    from ._impl import ops

    arguments = (q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, visibility_bits, softmax_scale, causal, window_size, window_sizes, metadata, deterministic, return_attn_probs)
    return ops.FlashAttnInterSequenceFunc.apply(*arguments)


def flash_attn_inter_sequence_kvpacked_func(
    q: Tensor, kv: Tensor, cu_seqlens_q: Tensor, cu_seqlens_k: Tensor, max_seqlen_q: int, max_seqlen_k: int,
    visibility_bits: Tensor, softmax_scale: float | None = None, causal: bool = False,
    window_size: tuple[int, int] = (-1, -1), window_sizes: Tensor | None = None,
    metadata: InterSequenceMetadata | None = None, deterministic: bool = False, return_attn_probs: bool = False,
) -> Tensor | tuple[Tensor, Tensor]:
    from ._impl import ops

    arguments = (q, kv, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, visibility_bits, softmax_scale, causal, window_size, window_sizes, metadata, deterministic, return_attn_probs)
    return ops.FlashAttnInterSequenceKVPackedFunc.apply(*arguments)


def prepare_inter_sequence_metadata(
    cu_seqlens_q: Tensor, cu_seqlens_k: Tensor, visibility_bits: Tensor,
) -> InterSequenceMetadata:
    """Builds the reusable metadata of an inter-sequence batch on the current CUDA stream. Prepare it again when
    sequence boundaries, visibility bits or the device change."""
    from ._impl import ops

    return ops.prepare_inter_sequence_metadata(cu_seqlens_q, cu_seqlens_k, visibility_bits)


def flash_attn_sink_func(
    q: Tensor, k: Tensor, v: Tensor, sink_size: int, softmax_scale: float | None = None, causal: bool = False,
    window_size: tuple[int, int] = (-1, -1), deterministic: bool = False, return_attn_probs: bool = False,
) -> Tensor | tuple[Tensor, Tensor]:
    """flash_attn_func with a sliding window whose first `sink_size` keys stay visible: query row i sees key j when the
    right bound (or `causal`) allows it and j is within window_size[0] of it or below sink_size. Head dims as flash_attn_func,
    forward and backward. Keys and values that no row sees still have to be finite."""
    from ._impl import sink

    return sink.flash_attn_sink(q, k, v, None, None, sink_size, softmax_scale, causal, window_size, deterministic, return_attn_probs)


def flash_attn_varlen_sink_func(
    q: Tensor, k: Tensor, v: Tensor, cu_seqlens_q: Tensor, cu_seqlens_k: Tensor, max_seqlen_q: int, max_seqlen_k: int,
    sink_size: int, softmax_scale: float | None = None, causal: bool = False, window_size: tuple[int, int] = (-1, -1),
    deterministic: bool = False, return_attn_probs: bool = False,
) -> Tensor | tuple[Tensor, Tensor]:
    """flash_attn_sink_func for packed batches (flash_attn_varlen_func): the first `sink_size` keys of every sequence stay
    visible to its own rows. What rows in front of the first or behind the last sequence hold (NaN included) has no effect on
    any result; they come out as zeros, with a log-sum-exp of -inf and gradients of zero."""
    from ._impl import sink

    return sink.flash_attn_sink(q, k, v, cu_seqlens_q, cu_seqlens_k, sink_size, softmax_scale, causal, window_size, deterministic, return_attn_probs)


def flash_attn_paged_func(
    q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, cache_seqlens: Tensor,
    softmax_scale: float | None = None, window_size: tuple[int, int] = (-1, -1), sink_size: int = 0,
    return_attn_probs: bool = False,
) -> Tensor | tuple[Tensor, Tensor]:
    """Attention of one new token per sequence over a paged key-value cache (inference only).

    q (sequences, heads_q, head_dim); k_cache, v_cache (pages, page_size, heads_kv, head_dim), any strides the kernels can
    read; block_table (sequences, max_pages) int32, the page of every page_size keys, where an entry outside the cache
    holds no keys; cache_seqlens (sequences) int32, the keys of each sequence with those of the new token, which is the
    last one. It sees the last window_size[0] + 1 keys (-1: all) and the first `sink_size`; window_size[1] has no effect.
    A sequence without visible keys gets zeros and a log-sum-exp of -inf. Returns out, and with `return_attn_probs`
    (out, softmax_lse), softmax_lse (sequences, heads_q) float32."""
    from ._impl import paged

    return paged.flash_attn_paged(q, k_cache, v_cache, block_table, cache_seqlens, softmax_scale, window_size, sink_size, return_attn_probs)


def append_paged_kv(
    k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, cache_seqlens: Tensor,
    cu_seqlens: Tensor | None = None,
) -> None:
    """Writes the keys and values of new tokens into the pages of their sequences, in place.

    k, v (sequences, tokens, heads_kv, head_dim), or packed (total, heads_kv, head_dim) with cu_seqlens (sequences + 1);
    token i of sequence b becomes key cache_seqlens[b] + i, so cache_seqlens counts the keys held before the call. Tokens
    whose position lies outside the table, in front of key 0 included, or whose entry holds no page are dropped. Sequences must
    not share the pages that are written to. The version counters of the caches go up: a backward pass that has saved one of
    them raises."""
    from ._impl import paged

    paged.append_paged_kv(k, v, k_cache, v_cache, block_table, cache_seqlens, cu_seqlens)


def copy_kv_pages(k_cache: Tensor, v_cache: Tensor, source_pages: Tensor, target_pages: Tensor) -> None:
    """Copies page source_pages[i] of both caches to page target_pages[i], in place; a pair with an entry outside the cache
    (-1) is skipped. The targets must differ from one another and from every source."""
    from ._impl import paged

    paged.copy_kv_pages(k_cache, v_cache, source_pages, target_pages)


def reserve_kv_pages(
    block_table: Tensor, cache_seqlens: Tensor, new_tokens: Tensor, page_refs: Tensor, page_size: int,
) -> tuple[Tensor, Tensor]:
    """Pages for the next new_tokens[b] tokens of every sequence: the table entries behind those that cache_seqlens[b]
    tokens fill get a free page (page_refs <= 0) where they hold none, lowest pages first, in the order (sequence, entry);
    -1 stays where no page is left. Returns the new (block_table, page_refs)."""
    from ._impl import paged

    return paged.reserve_pages(block_table, cache_seqlens, new_tokens, page_refs, page_size)


def fork_kv_pages(
    block_table: Tensor, cache_seqlens: Tensor, page_refs: Tensor, parents: Tensor, page_size: int,
) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """New sequences that continue those named by `parents` (children) int32. A child shares its parent's full pages,
    whose page_refs count it, and gets a free page for the partly filled last one, to be copied in every layer with
    copy_kv_pages. Returns (child_table, child_seqlens, page_refs, source_pages, target_pages); a pair is -1 where nothing
    has to be copied or no page was left (the child's table entry is then -1 too)."""
    from ._impl import paged

    return paged.fork_pages(block_table, cache_seqlens, page_refs, parents, page_size)


def free_kv_pages(
    block_table: Tensor, page_refs: Tensor, first_entry: Tensor, last_entry: Tensor,
) -> tuple[Tensor, Tensor]:
    """Gives the table entries [first_entry[b], last_entry[b]) of every sequence back: they become -1 and their pages lose
    a reference each; a page without references is free. Whole sequences (0 to max_pages) and pages that a window has left
    go the same way. Returns the new (block_table, page_refs)."""
    from ._impl import paged

    return paged.free_pages(block_table, page_refs, first_entry, last_entry)


def compact_kv_pages(block_table: Tensor, page_refs: Tensor) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """Moves the pages in use to the front of the pool: with n of them, the i-th page in use at or behind n goes to the
    i-th free page in front of n. Returns the new (block_table, page_refs) and the pairs (source_pages, target_pages),
    -1 behind the last one, to be copied in every layer with copy_kv_pages."""
    from ._impl import paged

    return paged.compact_pages(block_table, page_refs)


__all__ = [
    "InterSequenceMetadata",
    "append_paged_kv",
    "compact_kv_pages",
    "copy_kv_pages",
    "flash_attn_func",
    "flash_attn_inter_sequence_func",
    "flash_attn_inter_sequence_kvpacked_func",
    "flash_attn_kvpacked_func",
    "flash_attn_paged_func",
    "flash_attn_qkvpacked_func",
    "flash_attn_sink_func",
    "flash_attn_varlen_func",
    "flash_attn_varlen_kvpacked_func",
    "flash_attn_varlen_sink_func",
    "fork_kv_pages",
    "free_kv_pages",
    "prepare_inter_sequence_metadata",
    "reserve_kv_pages",
]
