"""Sliding-window attention with sinks, without a GPU: the key and query blocks the kernels visit, workspace sizes, and what
the host layer and the C entries refuse."""
import ctypes
import itertools
import time

import pytest
import torch

import zigfa
from zigfa._impl import lib, ops


def visible(lq, lk, left, right, sink):
    """(lq, lk) mask: row i sees column j when j <= i + lk - lq + right and (j >= i + lk - lq - left or j < sink)."""
    row, column = torch.arange(lq)[:, None] + (lk - lq), torch.arange(lk)[None]
    mask = torch.ones(lq, lk, dtype=torch.bool)
    if left >= 0:
        mask &= (column >= row - left) | (column < sink)
    if right >= 0:
        mask &= column <= row + right
    return mask


def problem(lq, lk, left, right, **changes):
    return lib.Problem(**{**dict(batch=1, seqlen_q=lq, seqlen_k=lk, heads_q=4, heads_kv=2, head_dim=128, window_left=left,
                                 window_right=right, softmax_scale=0.1), **changes})


def blocks(function, *arguments):
    out = (ctypes.c_int32 * 4096)()
    count = function(*arguments, out, 1024)
    return [tuple(out[4 * i:4 * i + 4]) for i in range(count)]


SIZES = [(1, 1), (1, 700), (130, 130), (600, 600), (300, 900), (900, 300), (1500, 1500), (700, 0), (0, 700)]


@pytest.mark.parametrize("lq, lk", SIZES)
def test_key_and_query_blocks_cover_exactly_the_blocks_with_visible_keys(lq, lk):
    library = lib.library()
    for left, right, sink in itertools.product((0, 1, 100, 127, 128, 500), (-1, 0, 3, 200), (1, 4, 127, 128, 129, 400, 5000)):
        mask, p = visible(lq, lk, left, right, sink), problem(lq, lk, left, right)
        for m0 in range(0, lq, 256):
            got = blocks(library.b200fa_sink_key_blocks_host, ctypes.byref(p), sink, 0, m0, m0 + 256)
            columns = [b[1] for b in got]
            assert columns == sorted(set(columns)) and all(c % 128 == 0 for c in columns)
            assert all((row, limit, banded) == (c, lk, 1) for row, c, limit, banded in got)
            seen = mask[m0:m0 + 256].any(0)
            needed = [c for c in range(0, lk, 128) if seen[c:c + 128].any()]
            assert set(needed) <= set(columns), (left, right, sink, m0)
            extra = set(columns) - set(needed)  # the window and the sinks of the tile's rows together may leave a gap open
            assert not extra or max(columns) == max(needed, default=-1), (left, right, sink, m0, extra)
        for c0 in range(0, lk, 128):
            got = [b[1] for b in blocks(library.b200fa_sink_query_blocks_host, ctypes.byref(p), sink, 0, c0, c0 + 128)]
            seen = mask[:, c0:c0 + 128].any(1)
            assert set(r for r in range(0, lq, 128) if seen[r:r + 128].any()) <= set(got), (left, right, sink, c0)
            assert got == list(range(got[0], got[0] + 128 * len(got), 128)) if got else True


def test_without_a_left_bound_or_sinks_nothing_changes():
    library = lib.library()
    for left, right, sink in ((-1, 0, 5), (-1, -1, 300), (200, 0, 0)):
        p = problem(900, 1300, left, right)
        assert library.b200fa_sink_fwd_workspace_bytes(ctypes.byref(p), sink) == library.b200fa_fwd_workspace_bytes(ctypes.byref(p))
        for m0 in range(0, 900, 256):
            assert blocks(library.b200fa_sink_key_blocks_host, ctypes.byref(p), sink, 0, m0, m0 + 256) == blocks(
                library.b200fa_key_blocks_host, ctypes.byref(p), 0, m0, m0 + 256)


def test_short_queries_over_a_long_window_are_split_with_the_sinks_counted():
    library = lib.library()
    p = problem(64, 20000, 300, 0)
    assert library.b200fa_fwd_workspace_bytes(ctypes.byref(p)) == 0  # four key blocks, too few for two shares
    assert library.b200fa_sink_fwd_workspace_bytes(ctypes.byref(p), 4000) > 0


def test_c_entries_refuse_without_a_launch():
    library = lib.library()
    for function, arguments in ((library.b200fa_sink_fwd, lib.FwdArgs), (library.b200fa_sink_bwd, lib.BwdArgs)):
        assert function(ctypes.byref(arguments(problem=problem(64, 64, 10, 0))), -1, None) == -1
        assert "sink_size" in lib.last_error()
        bits = problem(64, 64, 10, 0, cu_seqlens_q=8, cu_seqlens_k=8, visibility_bits=8, visibility_bits_t=8, cu_visible_k=8, cu_visible_q=8)
        assert function(ctypes.byref(arguments(problem=bits)), 4, None) == -1
        assert "inter-sequence" in lib.last_error()
        assert function(None, 4, None) == -1
        assert function(ctypes.byref(arguments(problem=problem(64, 64, 10, 0, softmax_scale=0.0))), 4, None) == -1
        assert "positive softmax_scale" in lib.last_error()


def test_host_layer_refusals():
    for bad in (-1, 2**31):
        with pytest.raises(ValueError, match="sink_size"):
            ops.check_sink_size(bad)
    for bad in (1.0, None, "4"):
        with pytest.raises(TypeError, match="sink_size"):
            ops.check_sink_size(bad)
    q = torch.zeros(1, 8, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="sink_size"):
        zigfa.flash_attn_sink_func(q, q, q, -1)
    with pytest.raises(ValueError, match="window bounds"):
        zigfa.flash_attn_sink_func(q, q, q, 4, window_size=(-2, 0))
    for scale in (0.0, -0.1, float("nan")):  # a masked score of -inf times these is no -inf
        with pytest.raises(ValueError, match="positive softmax_scale"):
            zigfa.flash_attn_sink_func(q, q, q, 4, softmax_scale=scale, window_size=(9, 0))
    with pytest.raises(NotImplementedError, match="deterministic"):
        zigfa.flash_attn_sink_func(q, q, q, 4, deterministic=True)
    with pytest.raises(ValueError, match="is on meta"):
        ops.check_same_device(q, k=q.to("meta"))


def test_the_reference_gradients_match_differences():
    """The formulas that the GPU tests compare with, against automatic and numeric differentiation in 64 bits."""
    import sink_reference as plain

    torch.manual_seed(0)
    for lq, lk, left, right, sink in ((9, 9, 3, 0, 2), (5, 12, 2, 1, 4), (8, 3, 1, 0, 1)):
        mask = plain.visible(lq, lk, left, right, sink, device="cpu")
        q, k, v = (torch.randn(n, h, 5, dtype=torch.float64, requires_grad=True) for n, h in ((lq, 4), (lk, 2), (lk, 2)))
        dout = torch.randn(lq, 4, 5, dtype=torch.float64)
        results = plain.with_tolerances(q.detach(), k.detach(), v.detach(), dout, mask, 0.7)
        seen = mask.any(1)  # a row without keys has no derivative in the softmax below; it takes no part

        def loss(q, k, v):
            return (plain.attention(q[seen], k, v, mask[seen], 0.7)[0] * dout[seen]).sum()

        assert torch.autograd.gradcheck(loss, (q, k, v))
        for name, gradient in zip(("dq", "dk", "dv"), torch.autograd.grad(loss(q, k, v), (q, k, v))):
            assert torch.allclose(results[name][0], gradient, rtol=1e-9, atol=1e-12), name


@pytest.mark.parametrize("seqlen", [512, 4096, 131072])
def test_plan_of_a_window_wider_than_any_sequence_is_quick(seqlen):
    # A bound of 2^30 keys, which the host layer makes of any larger one, must not make the backward plan search for a share
    # size of that many blocks (267 ms a call at 128 k tokens); the workspace is that of a window as long as the sequence.
    library = lib.library()

    def workspace(left):
        p = problem(seqlen, seqlen, left, 0, batch=2, heads_q=16, heads_kv=4)
        return library.b200fa_sink_bwd_workspace_bytes(ctypes.byref(p), 4)

    start = time.perf_counter()
    for _ in range(20):
        size = workspace(2**30)
    assert time.perf_counter() - start < 0.5  # 20 plans: 0.7 to 5 s with the search, below a millisecond without
    assert size == workspace(seqlen)


def test_forward_mode_derivatives_are_refused_not_dropped():
    q = torch.randn(1, 8, 2, 64, dtype=torch.bfloat16)
    cache = torch.randn(4, 16, 2, 64, dtype=torch.bfloat16)
    table, lengths = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        for arguments in ((dual, q, q), (q, dual, q), (q, q, dual)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                zigfa.flash_attn_sink_func(*arguments, 2, causal=True, window_size=(3, 0))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            zigfa.flash_attn_paged_func(dual[:, 0], cache, cache, table, lengths)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            zigfa.append_paged_kv(dual, q, cache, cache, table, lengths)


def test_entries_that_fill_all_rows_want_contiguous_results():
    library = lib.library()
    aligned = 1 << 20  # passes the alignment checks; nothing dereferences it on these paths
    packed = problem(64, 64, 10, 0, batch=0, cu_seqlens_q=aligned, cu_seqlens_k=aligned)
    row, heads = lib.Stride3(0, 4 * 128, 128), lib.Stride3(0, 2 * 128, 128)
    good = dict(problem=packed, out=aligned, softmax_lse=aligned, out_stride=row, lse_stride=lib.Stride2(0, 64))
    for changes, message in [(dict(out_stride=lib.Stride3(0, 8 * 128, 128)), "contiguous"), (dict(out_stride=lib.Stride3(0, 4 * 128, 256)), "contiguous"),
                             (dict(lse_stride=lib.Stride2(0, 72)), "contiguous"), (dict(out=None), "pointer"), (dict(out=aligned + 8), "aligned"),
                             (dict(softmax_lse=None), "null")]:
        assert library.b200fa_sink_fwd_all_rows(ctypes.byref(lib.FwdArgs(**{**good, **changes})), 4, None) == -1, changes
        assert message in lib.last_error(), changes
    good = dict(problem=packed, dq=aligned, dk=aligned, dv=aligned, dq_stride=row, dk_stride=heads, dv_stride=heads)
    for changes, message in [(dict(dq_stride=heads), "contiguous"), (dict(dv_stride=row), "contiguous"), (dict(dk=None), "pointer"),
                             (dict(dv=aligned + 4), "aligned")]:
        assert library.b200fa_sink_bwd_all_rows(ctypes.byref(lib.BwdArgs(**{**good, **changes})), 4, None) == -1, changes
        assert message in lib.last_error(), changes
    for function in (library.b200fa_sink_fwd_all_rows, library.b200fa_sink_bwd_all_rows):
        assert function(None, 4, None) == -1
    empty = problem(0, 0, 10, 0, batch=0, cu_seqlens_q=aligned, cu_seqlens_k=aligned)
    assert library.b200fa_sink_fwd_all_rows(ctypes.byref(lib.FwdArgs(problem=empty, out_stride=row)), 4, None) == 0  # no rows, no launch
    fixed = lib.FwdArgs(problem=problem(0, 0, 10, 0, batch=0))  # nothing stands between the sequences of a fixed-length batch
    assert library.b200fa_sink_fwd_all_rows(ctypes.byref(fixed), 4, None) == 0


@pytest.mark.parametrize("tokens, heads_q, heads_kv, d, left, sink", [
    (131072, 32, 8, 128, 1023, 4), (131072, 32, 8, 128, 1023, 500), (131072, 16, 8, 256, 1023, 500), (16384, 8, 8, 64, 255, 512),
    (131072, 8, 8, 128, 255, 17), (65536, 32, 8, 128, 255, 4), (4000, 2, 2, 72, 50, 300), (131072, 1, 1, 64, 100, 4)])
def test_workspace_of_a_packed_backward_pass_does_not_grow_with_the_number_of_documents(tokens, heads_q, heads_kv, d, left, sink):
    """The FP32 parts of dK and dV belong to sequences of two shares or more, however many short ones there are; and they are
    no larger than what the pass keeps anyway (1024 documents in 131072 tokens once took 8 GB of parts next to 3 GB)."""
    library = lib.library()

    def parts(documents):
        p = problem(tokens, tokens, left, 0, batch=documents, heads_q=heads_q, heads_kv=heads_kv, head_dim=d, cu_seqlens_q=8, cu_seqlens_k=8)
        plain = library.b200fa_bwd_workspace_bytes(ctypes.byref(p))
        return library.b200fa_sink_bwd_workspace_bytes(ctypes.byref(p), sink) - plain, plain

    extra, plain = parts(1)
    assert 0 <= extra <= 1.5 * plain
    for documents in (2, 100, 1000, 4096):
        # the list of shares holds 8 bytes per sequence of more than `least` rows, 512 or more; both lists are aligned to 256
        assert abs(parts(documents)[0] - extra) <= 8 * (tokens // 512) + 512, documents


def test_the_plan_counts_both_halves_of_the_head_dimension():
    """At head_dim 256 a key block is two CTAs' work, so a share may be twice as large as with half the columns: the parts of
    a long batch take the same memory per key head (twice the width, half the shares)."""
    library = lib.library()

    def parts(d):
        p = problem(131072, 131072, 1023, 0, heads_q=16, heads_kv=8, head_dim=d)
        return library.b200fa_sink_bwd_workspace_bytes(ctypes.byref(p), 4) - library.b200fa_bwd_workspace_bytes(ctypes.byref(p))

    assert 0 < parts(256) <= 1.1 * parts(128)


def test_results_without_rows_may_have_any_strides():
    library = lib.library()
    empty = problem(0, 0, 10, 0, batch=0, cu_seqlens_q=8, cu_seqlens_k=8)  # torch: a (heads, 0) tensor has the strides (1, 1)
    args = lib.FwdArgs(problem=empty, out_stride=lib.Stride3(8, 8, 8), lse_stride=lib.Stride2(0, 1))
    assert library.b200fa_sink_fwd_all_rows(ctypes.byref(args), 4, None) == 0
    args = lib.BwdArgs(problem=empty, dq_stride=lib.Stride3(8, 8, 8), dk_stride=lib.Stride3(8, 8, 8), dv_stride=lib.Stride3(8, 8, 8))
    assert library.b200fa_sink_bwd_all_rows(ctypes.byref(args), 4, None) == 0
