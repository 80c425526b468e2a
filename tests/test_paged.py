"""The paged key-value cache without a GPU: which keys a token sees (host twin of the kernel's walk), and what the host
layer and the C entries refuse."""
import ctypes
import itertools

import pytest
import torch

import paged_reference as plain
import zigfa
from zigfa._impl import lib, paged

ALIGNED = 1 << 20  # a pointer value that passes the alignment checks; nothing dereferences it on these paths


def test_visible_keys_match_the_definition():
    library = lib.library()
    keys = (ctypes.c_int32 * 4096)()
    lengths = (-7, 0, 1, 2, 15, 16, 17, 31, 32, 33, 100, 129, 300, 1000)
    for length, left, sink, capacity in itertools.product(lengths, (-1, 0, 1, 14, 15, 16, 17, 40, 127, 2000),
                                                          (0, 1, 15, 16, 17, 40, 2000), (0, 5, 112, 4096)):
        count = library.b200fa_paged_keys_host(length, capacity, left, sink, keys, 4096)
        assert keys[:count] == plain.visible_keys(length, capacity, left, sink), (length, left, sink, capacity)


def cache(pages=6, page_size=16, heads=2, d=64, **options):
    return torch.zeros(pages, page_size, heads, d, dtype=torch.bfloat16, **options)


def ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def decode_arguments(**changes):
    arguments = dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), k_cache=cache(), v_cache=cache(), block_table=ints(3, 5),
                     cache_seqlens=ints(3), window_left=-1, sink_size=0)
    return {**arguments, **changes}


@pytest.mark.parametrize("changes, message", [
    (dict(q=torch.zeros(3, 4, 64)), "q must be bfloat16"),
    (dict(q=torch.zeros(3, 4, 1, 64, dtype=torch.bfloat16)), "q must have 3 dimensions"),
    (dict(q=torch.zeros(3, 4, 80, dtype=torch.bfloat16), k_cache=cache(d=80), v_cache=cache(d=80)), "head_dim must be one of"),
    (dict(q=torch.zeros(3, 4, 128, dtype=torch.bfloat16)), "head_dim must be one of"),
    (dict(q=torch.zeros(3, 5, 64, dtype=torch.bfloat16)), "multiple of the key head count"),
    (dict(q=torch.zeros(3, 0, 64, dtype=torch.bfloat16)), "multiple of the key head count"),
    (dict(k_cache=cache().half()), "k_cache must be bfloat16"),
    (dict(v_cache=cache()[0]), "v_cache must have 4 dimensions"),
    (dict(v_cache=cache(pages=7)), "same shape"),
    (dict(k_cache=cache(page_size=0), v_cache=cache(page_size=0)), "must not be empty"),
    (dict(k_cache=cache(d=128)[..., ::2], v_cache=cache(d=128)[..., ::2]), "16-byte aligned"),
    (dict(k_cache=torch.zeros(6 * 16 * 2 * 64 + 1, dtype=torch.bfloat16)[1:].view(6, 16, 2, 64)), "16-byte aligned"),
    (dict(block_table=ints(4, 5)), "block_table must be an int32 tensor"),
    (dict(block_table=ints(3, 5).long()), "block_table must be an int32 tensor"),
    (dict(block_table=ints(5, 3).T), "contiguous columns"),
    (dict(cache_seqlens=ints(2)), "cache_seqlens must be an int32 tensor"),
    (dict(window_left=-2), "window bounds"),
    (dict(sink_size=-1), "sink_size"),
    (dict(cache_seqlens=ints(3).to("meta")), "is on meta"),
])
def test_decode_refusals(changes, message):
    paged.check_paged(**decode_arguments())
    with pytest.raises(ValueError, match=message):
        paged.check_paged(**decode_arguments(**changes))


def test_decode_refuses_a_sink_size_that_is_no_integer():
    with pytest.raises(TypeError, match="sink_size"):
        paged.check_paged(**decode_arguments(sink_size=1.5))


def test_decode_refuses_gradients():
    arguments = decode_arguments(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16, requires_grad=True))
    arguments = [arguments[n] for n in ("q", "k_cache", "v_cache", "block_table", "cache_seqlens")]
    with pytest.raises(NotImplementedError, match="no backward"):
        zigfa.flash_attn_paged_func(*arguments)


def append_arguments(**changes):
    arguments = dict(k=torch.zeros(3, 2, 2, 64, dtype=torch.bfloat16), v=torch.zeros(3, 2, 2, 64, dtype=torch.bfloat16),
                     k_cache=cache(), v_cache=cache(), block_table=ints(3, 5), cache_seqlens=ints(3), cu_seqlens=None)
    return {**arguments, **changes}


@pytest.mark.parametrize("changes, message", [
    (dict(k=torch.zeros(3, 2, 2, 64)), "k must be bfloat16"),
    (dict(cu_seqlens=ints(4)), "k must have 3 dimensions"),
    (dict(v=torch.zeros(3, 1, 2, 64, dtype=torch.bfloat16)), "same shape"),
    (dict(k_cache=cache(heads=3), v_cache=cache(heads=3)), "heads and the head_dim"),
    (dict(cache_seqlens=ints(3).long()), "cache_seqlens must be an int32"),
    (dict(cache_seqlens=ints(4), block_table=ints(4, 5)), "same number of sequences"),
    (dict(block_table=ints(2, 5)), "block_table must be an int32"),
    (dict(k=torch.zeros(6, 2, 64, dtype=torch.bfloat16), v=torch.zeros(6, 2, 64, dtype=torch.bfloat16), cu_seqlens=ints(3)), "cu_seqlens must be"),
    (dict(block_table=ints(3, 5).to("meta")), "is on meta"),
])
def test_append_refusals(changes, message):
    paged.check_append(**append_arguments())
    with pytest.raises(ValueError, match=message):
        paged.check_append(**append_arguments(**changes))


def test_bookkeeping_refusals():
    table, refs, lengths = ints(3, 5), ints(6), ints(3)
    paged.check_books(table, refs, cache_seqlens=lengths)
    for arguments, message in [((table.long(), refs), "block_table"), ((table[0], refs), "block_table"),
                               ((table, refs.long()), "page_refs"), ((table, refs[None]), "page_refs"),
                               ((table, refs.to("meta")), "is on meta")]:
        with pytest.raises(ValueError, match=message):
            paged.check_books(*arguments)
    with pytest.raises(ValueError, match="cache_seqlens"):
        paged.check_books(table, refs, cache_seqlens=ints(4))
    for size in (0, -3, 2.0, None):
        with pytest.raises(ValueError, match="page_size"):
            paged.check_page_size(size)
    with pytest.raises(ValueError, match="target_pages"):
        paged.check_copy(cache(), cache(), ints(3), ints(4))
    with pytest.raises(ValueError, match="multiple of 8"):
        paged.check_copy(cache(d=2048), cache(d=2048), ints(3), ints(3))


def test_c_entries_refuse_without_a_launch():
    library = lib.library()

    def decode(**changes):
        fields = dict(batch=2, heads_q=8, heads_kv=2, head_dim=128, num_pages=10, page_size=16, max_pages=4, window_left=-1,
                      sink_size=0, softmax_scale=0.1, **{name: ALIGNED for name in (
                          "q", "k_cache", "v_cache", "block_table", "cache_seqlens", "out", "softmax_lse")})
        return library.b200fa_paged_decode(lib.PagedArgs(**{**fields, **changes}), None)

    for changes, message in [(dict(batch=-1), "negative"), (dict(page_size=0), "page_size"), (dict(heads_q=7), "multiple"),
                             (dict(head_dim=80), "head_dim 80"), (dict(window_left=-2), "window"), (dict(sink_size=-1), "sink"),
                             (dict(max_pages=1 << 28), "2\\^31"), (dict(q=None), "null"), (dict(block_table=None), "null"),
                             (dict(k_cache=ALIGNED + 8), "16-byte"), (dict(q_stride=lib.Stride2(4, 8)), "multiples of 8"),
                             (dict(v_stride=lib.Stride3(8, 8, 4)), "multiples of 8")]:
        assert decode(**changes) < 0, changes
        with pytest.raises((ValueError, NotImplementedError), match=message):
            lib.check(-1)
    assert decode(batch=0) == 0

    kv = dict(num_pages=10, page_size=16, heads_kv=2, head_dim=64, k_cache=ALIGNED, v_cache=ALIGNED)
    for changes, message in [(dict(page_size=0), "page size"), (dict(head_dim=60), "multiple of 8"), (dict(k_cache=None), "null"),
                             (dict(v_cache=ALIGNED + 4), "16-byte"), (dict(k_stride=lib.Stride3(1, 8, 8)), "multiples of 8")]:
        bad = lib.KvCache(**{**kv, **changes})
        assert library.b200fa_copy_pages(bad, ALIGNED, ALIGNED, 3, None) == -1
        with pytest.raises(ValueError, match=message):
            lib.check(-1)
        append = lib.AppendArgs(cache=bad, k=ALIGNED, v=ALIGNED, rows=1, batch=1, max_pages=1, cache_seqlens=ALIGNED, block_table=ALIGNED)
        assert library.b200fa_append_kv(append, None) == -1
    assert library.b200fa_copy_pages(lib.KvCache(**kv), ALIGNED, ALIGNED, -1, None) == -1
    assert library.b200fa_copy_pages(lib.KvCache(**kv), ALIGNED, None, 1, None) == -1
    assert library.b200fa_copy_pages(lib.KvCache(**kv), None, None, 0, None) == 0
    append = dict(cache=lib.KvCache(**kv), k=ALIGNED, v=ALIGNED, rows=1, batch=1, max_pages=1, cache_seqlens=ALIGNED, block_table=ALIGNED)
    for changes in (dict(k=None), dict(v=ALIGNED + 8), dict(rows=-1), dict(batch=-1), dict(k_stride=lib.Stride3(4, 8, 8)),
                    dict(rows=1 << 31), dict(max_pages=1 << 28)):
        assert library.b200fa_append_kv(lib.AppendArgs(**{**append, **changes}), None) == -1, changes
    assert library.b200fa_append_kv(lib.AppendArgs(**{**append, "rows": 0}), None) == 0

    books = dict(sequences=2, rows=2, max_pages=4, num_pages=10, page_size=16, block_table=ALIGNED, page_refs=ALIGNED,
                 cache_seqlens=ALIGNED, block_table_out=ALIGNED, page_refs_out=ALIGNED, source_pages=ALIGNED,
                 target_pages=ALIGNED, workspace=ALIGNED, workspace_bytes=40)
    calls = dict(reserve=(ALIGNED,), fork=(ALIGNED, ALIGNED), free=(ALIGNED, ALIGNED), compact=())
    assert library.b200fa_pages_workspace_bytes(10) == 40
    for name, extra in calls.items():
        function = getattr(library, f"b200fa_{name}_pages")
        for changes in (dict(sequences=-1), dict(page_size=0), dict(page_refs=None), dict(block_table=None),
                        dict(block_table_out=None), dict(max_pages=1 << 28), dict(page_refs_out=None)):
            assert function(lib.PagesArgs(**{**books, **changes}), *extra, None) == -1, (name, changes)
        if name != "free":
            assert function(lib.PagesArgs(**{**books, "workspace_bytes": 39}), *extra, None) == -1
            assert "workspace" in lib.last_error()
        if name != "fork":
            assert function(lib.PagesArgs(**{**books, "rows": 1}), *extra, None) == -1
        if extra:
            assert function(lib.PagesArgs(**books), *([None] * len(extra)), None) == -1


def test_ops_have_fake_implementations():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode(), torch.device("cuda"):
        q, k = torch.empty(3, 8, 64, dtype=torch.bfloat16), torch.empty(9, 16, 2, 64, dtype=torch.bfloat16)
        table, lengths, refs = (torch.empty(*s, dtype=torch.int32) for s in ((3, 5), (3,), (9,)))
        out, lse = zigfa.flash_attn_paged_func(q, k, k, table, lengths, return_attn_probs=True)
        assert out.shape == (3, 8, 64) and lse.shape == (3, 8) and lse.dtype == torch.float32
        assert [tuple(t.shape) for t in zigfa.fork_kv_pages(table, lengths, refs, torch.empty(7, dtype=torch.int32), 16)] == [
            (7, 5), (7,), (9,), (7,), (7,)]
        assert [tuple(t.shape) for t in zigfa.compact_kv_pages(table, refs)] == [(3, 5), (9,), (4,), (4,)]
        assert [tuple(t.shape) for t in zigfa.free_kv_pages(table, refs, lengths, lengths)] == [(3, 5), (9,)]
        assert [tuple(t.shape) for t in zigfa.reserve_kv_pages(table, lengths, lengths, refs, 16)] == [(3, 5), (9,)]
        assert zigfa.append_paged_kv(torch.empty(3, 1, 2, 64, dtype=torch.bfloat16), torch.empty(3, 1, 2, 64, dtype=torch.bfloat16),
                                     k, k, table, lengths) is None


def test_packed_arguments_have_the_layout_of_the_structures():
    """The host layer packs the argument structures with `struct`; their sizes and field offsets are those of ctypes."""
    import struct

    from zigfa._impl import dispatch

    for name, structure in (("fwd", lib.FwdArgs), ("bwd", lib.BwdArgs), ("paged", lib.PagedArgs), ("kv_cache", lib.KvCache),
                            ("append", lib.AppendArgs), ("pages", lib.PagesArgs)):
        pack = getattr(dispatch, f"PACK_{name.upper()}")
        layout = pack.__self__

        def values(fields):  # every scalar of the structure, in order, numbered
            for _, kind in fields:
                if hasattr(kind, "_fields_"):
                    yield from values(kind._fields_)
                elif hasattr(kind, "_length_"):
                    yield from [kind._type_] * kind._length_
                else:
                    yield kind

        kinds = list(values(structure._fields_))
        data = pack(*range(1, len(kinds) + 1))
        assert layout.size <= ctypes.sizeof(structure) < layout.size + 8, name  # a structure may end in padding
        filled = structure.from_buffer_copy(data.ljust(ctypes.sizeof(structure), b"\0"))

        def read(value):
            for field, kind in value._fields_:
                item = getattr(value, field)
                if hasattr(kind, "_fields_"):
                    yield from read(item)
                elif hasattr(kind, "_length_"):
                    yield from item
                else:
                    yield item

        assert list(read(filled)) == list(range(1, len(kinds) + 1)), name


def test_writing_into_a_cache_is_seen_by_autograd():
    """A backward pass that has saved a cache must not read what was written into it afterwards."""
    def fill(*caches):
        for tensor in caches:
            tensor.data.fill_(7)  # as a kernel does, without telling autograd

    with torch.library._scoped_library("zigfa", "IMPL") as stand_in:  # CPU kernels in the operators' place, for this test
        stand_in.impl("append_kv", lambda k, v, k_cache, v_cache, *unused: fill(k_cache, v_cache), "CPU")
        stand_in.impl("copy_pages", lambda k_cache, v_cache, *unused: fill(k_cache, v_cache), "CPU")
        rows, table, lengths = torch.ones(1, 1, 2, 64, dtype=torch.bfloat16), ints(1, 4), ints(1)
        for write in (lambda k, v: zigfa.append_paged_kv(rows, rows, k, v, table, lengths),
                      lambda k, v: zigfa.copy_kv_pages(k, v, ints(1), ints(1))):
            for saved in (0, 1):
                caches = [cache(), cache()]
                weight = torch.ones(1, requires_grad=True)
                product = (weight * caches[saved]).sum()
                write(*caches)
                assert (caches[saved] == 7).all()
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    product.backward()
            with torch.inference_mode():
                write(cache(), cache())


def test_the_short_way_counts_the_versions_too(monkeypatch):
    """The same for plain CUDA tensors, which do not pass through the dispatcher; here with the launch left out."""
    from zigfa._impl import dispatch

    calls = []
    schema = "version_probe(Tensor x, Tensor(a!) y) -> ()"
    probe = dispatch.define(schema, lambda x, y: calls.append(1) and None, lambda *unused: None, written=((1, "y"),))

    class Plain(torch.Tensor):
        is_cuda = True

    monkeypatch.setattr(dispatch, "_PLAIN", {Plain, torch.Tensor})
    x, y = torch.zeros(3).as_subclass(Plain), torch.zeros(3)
    before = y._version
    probe(x, y)
    assert calls == [1] and y._version == before + 1 and x._version == 0
    with torch.inference_mode():
        frozen = torch.zeros(3)
        probe(torch.zeros(3).as_subclass(Plain), frozen)
    assert calls == [1, 1]


def test_the_short_way_is_for_plain_arguments_only(monkeypatch):
    """The implementations take addresses. A subclass in any place, or a transform around the call, goes to the dispatcher;
    a subclass that wraps other tensors has the address 0."""
    from torch.utils._python_dispatch import TorchDispatchMode

    from zigfa._impl import dispatch

    direct, wrapped = [], []
    probe = dispatch.define("short_way_probe(Tensor x, Tensor? y, int n) -> Tensor", lambda x, y, n: direct.append(1) or x.clone(),
                            lambda x, *unused: torch.empty_like(x))

    class Cuda(torch.Tensor):  # stands for a plain tensor on a device, whose implementation may be called
        is_cuda = True

    class Wrapper(torch.Tensor):
        @staticmethod
        def __new__(cls, inner):
            return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype)

        def __init__(self, inner):
            self.inner = inner

        @classmethod
        def __torch_dispatch__(cls, function, types, arguments=(), options=None):
            wrapped.append(str(function))
            return torch.zeros(3)

    monkeypatch.setattr(dispatch, "_PLAIN", {*dispatch._PLAIN, Cuda})
    x = torch.zeros(3).as_subclass(Cuda)
    probe(x, None, 1)
    probe(x, torch.zeros(3), 1)
    assert len(direct) == 2
    with torch._C.DisableTorchFunctionSubclass():
        probe(x, Wrapper(torch.zeros(3)), 1)
        assert wrapped == ["zigfa.short_way_probe.default"]
        with pytest.raises(NotImplementedError, match="short_way_probe"):  # no kernel for the CPU behind the dispatcher
            torch.vmap(lambda y: probe(x, y, 1))(torch.zeros(2, 3))
    assert len(direct) == 2


@pytest.mark.parametrize("d, heads_kv, batch, keys, whole", [
    (128, 8, 1, 512, True), (128, 8, 1, 528, False), (128, 8, 16, 1280, True), (128, 8, 16, 1296, False), (64, 8, 37, 1536, True), (128, 8, 37, 1552, False), (128, 8, 24, 1296, False),
    (128, 8, 38, 512, True), (128, 8, 38, 528, False),  # 304 pairs: a second round for eight of them
    (128, 8, 56, 1280, True), (128, 8, 74, 1280, True), (64, 8, 76, 528, False), (128, 8, 100, 1280, True), (128, 8, 74, 1296, False),
    (256, 4, 2, 256, True), (256, 4, 2, 272, False), (256, 4, 32, 512, True), (256, 4, 32, 528, False), (256, 4, 76, 272, False),
    (256, 4, 148, 512, False), (512, 2, 64, 512, True), (512, 2, 80, 272, False)])
def test_which_pairs_of_sequence_and_key_head_are_cut(d, heads_kv, batch, keys, whole):
    args = lib.PagedArgs(batch=batch, heads_q=4 * heads_kv, heads_kv=heads_kv, head_dim=d, page_size=16, max_pages=keys // 16, window_left=-1)
    assert (lib.library().b200fa_paged_decode_workspace_bytes(args) == 0) == whole
    if whole:  # a window bounds the pairs whatever the table holds
        args.max_pages, args.window_left, args.sink_size = 4096, keys // 2 - 16, keys // 2 - 32
        assert lib.library().b200fa_paged_decode_workspace_bytes(args) == 0
