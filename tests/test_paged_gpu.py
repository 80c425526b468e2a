"""GPU tests of the paged key-value cache: one-token attention against 64-bit attention over the keys that the table
names, and writing, copying and bookkeeping against plain lists (equal to the last bit)."""
import itertools
import random

import pytest
import torch

import paged_reference as plain
import zigfa

pytestmark = pytest.mark.gpu


def randn(*shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device="cuda", dtype=dtype)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def scattered(lengths, page_size, spare=3, columns=None):
    """(table, number of pages): pages of the sequences scattered over a pool, unused entries -1."""
    counts = [-(-max(n, 0) // page_size) for n in lengths]
    pages = sum(counts) + spare
    order = iter(torch.randperm(pages).tolist())
    columns = max([columns or 0, 1, *counts])
    return ints([[next(order) if e < c else -1 for e in range(columns)] for c in counts]), pages


def poisoned(table, lengths, page_size, pages, heads, d, left=-1, sink=0):
    """Caches whose rows are finite where some sequence's token sees them and NaN everywhere else."""
    k, v = (torch.full((pages, page_size, heads, d), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    rows = table.tolist()
    for b, length in enumerate(lengths):
        slots = [(rows[b][j // page_size], j % page_size) for j in plain.visible_keys(length, len(rows[b]) * page_size, left, sink)]
        slots = [s for s in slots if 0 <= s[0] < pages]
        if slots:
            page, row = (torch.tensor(x, device="cuda") for x in zip(*slots))
            k[page, row], v[page, row] = randn(len(slots), heads, d), randn(len(slots), heads, d)
    return k, v


def check_decode(q, k_cache, v_cache, table, lengths, left=-1, sink=0, scale=None, note=""):
    result = zigfa.flash_attn_paged_func(q, k_cache, v_cache, table, lengths, softmax_scale=scale, window_size=(left, -1),
                                         sink_size=sink, return_attn_probs=True)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    plain.assert_decode(result, plain.decode(q, k_cache, v_cache, table, lengths, scale, left, sink), note)
    return result


LENGTHS = (0, 1, 2, 15, 16, 17, 63, 64, 65, 130, 333, 1100)


@pytest.mark.parametrize("d", [64, 72, 96, 128, 256, 512])
@pytest.mark.parametrize("heads", [(1, 1), (4, 4), (6, 2), (8, 1), (9, 1), (16, 2), (32, 2), (40, 1), (64, 1)])
def test_decode_matches_64_bits(d, heads):
    torch.manual_seed(d + heads[0])
    for page_size in (1, 7, 16, 64):
        table, pages = scattered(LENGTHS, page_size)
        k, v = poisoned(table, LENGTHS, page_size, pages, heads[1], d)
        check_decode(randn(len(LENGTHS), heads[0], d), k, v, table, ints(LENGTHS), note=(d, heads, page_size))


@pytest.mark.parametrize("left, sink", [(0, 0), (0, 1), (5, 3), (15, 16), (16, 17), (64, 0), (100, 40), (127, 2000), (2000, 5), (-1, 9)])
def test_decode_windows_and_sinks(left, sink):
    torch.manual_seed(left + sink + 2)
    for (d, heads), page_size in itertools.product([((128), (8, 2)), (64, (8, 1)), (256, (4, 4))], (3, 16, 128)):
        table, pages = scattered(LENGTHS, page_size)
        k, v = poisoned(table, LENGTHS, page_size, pages, heads[1], d, left, sink)
        check_decode(randn(len(LENGTHS), heads[0], d), k, v, table, ints(LENGTHS), left, sink, note=(d, page_size))


def test_decode_bad_table_entries_and_lengths_are_bounds_checked():
    """Entries outside the cache hold no keys; lengths beyond the table (or negative) are cut."""
    torch.manual_seed(3)
    page_size, d = 16, 128
    lengths = [5000, 200, 200, -4, 64, 97, 2**31 - 1, 80]
    table, pages = scattered([80, 200, 200, 0, 64, 97, 128, 80], page_size)
    table[0, 5:] = 2**31 - 1
    table[1, 2:6] = -1
    table[2, 0], table[2, 3], table[2, 7] = pages, -(2**31), 10**9
    table[4] = -1
    table[7] = pages + 5
    held = [min(max(n, 0), table.shape[1] * page_size) for n in lengths]
    k, v = poisoned(table, held, page_size, pages, 2, d)
    out, lse = check_decode(randn(8, 8, d), k, v, table, ints(lengths))
    for b in (3, 4, 7):  # nothing to see
        assert (out[b] == 0).all() and (lse[b] == float("-inf")).all()
    empty = zigfa.flash_attn_paged_func(randn(2, 4, 64), randn(0, 16, 2, 64), randn(0, 16, 2, 64), ints([[0], [3]]), ints([5, 5]))
    assert (empty == 0).all()
    no_columns = torch.empty(2, 0, dtype=torch.int32, device="cuda")
    assert (zigfa.flash_attn_paged_func(randn(2, 4, 64), randn(4, 16, 2, 64), randn(4, 16, 2, 64), no_columns, ints([5, 5])) == 0).all()
    assert zigfa.flash_attn_paged_func(randn(0, 4, 64), randn(4, 16, 2, 64), randn(4, 16, 2, 64), ints([]).view(0, 3), ints([])).shape == (0, 4, 64)


def test_decode_strides_and_shared_pages():
    """Heads-first pools, one buffer for K and V, sliced queries, tables with longer rows, and a prefix that every sequence
    shares (the same page in several tables)."""
    torch.manual_seed(4)
    lengths, page_size, d, heads_kv = [100, 64, 333], 16, 128, 2
    table, pages = scattered(lengths, page_size)
    table[1, :3] = table[0, :3]
    table[2, :3] = table[0, :3]
    wide = torch.full((3, 40), 10**8, dtype=torch.int32, device="cuda")
    wide[:, 1:1 + table.shape[1]] = table
    q = randn(3, 3, 8, d)[:, 1]
    heads_first = randn(2, pages, heads_kv, page_size, d)
    interleaved = randn(pages, 2, page_size, heads_kv, d)
    for k, v in ((heads_first[0].transpose(1, 2), heads_first[1].transpose(1, 2)), (interleaved[:, 0], interleaved[:, 1])):
        check_decode(q, k, v, wide[:, 1:1 + table.shape[1]], ints(lengths))
    odd = randn(3 * 8 * d + 1)[1:].view(3, 8, d)  # not 16-byte aligned: copied by the host layer
    check_decode(odd, *heads_first.transpose(2, 3), table, ints([n for x in lengths for n in (x, 0)])[::2])


def test_decode_scores_of_every_size():
    """Peaked rows, equal scores, a scale of zero and a negative one, scores far apart between the shares of a long cache."""
    torch.manual_seed(5)
    lengths, page_size, d = [40, 700, 9000], 16, 64
    table, pages = scattered(lengths, page_size)
    k, v = randn(pages, page_size, 2, d), randn(pages, page_size, 2, d)
    q = randn(3, 4, d)
    for scale in (8.0, 1.0, 0.0, -0.3):
        check_decode(q, k, v, table, ints(lengths), scale=scale, note=scale)
    k[table[2, 300]] *= 30
    check_decode(q, k, v, table, ints(lengths))
    check_decode(q * 0, k, v, table, ints(lengths))


@pytest.mark.parametrize("d, heads, lengths, page_size, left", [
    (128, (32, 8), [30011], 16, -1), (128, (8, 1), [70001, 3], 64, -1), (64, (4, 4), [9000] * 3, 24, -1),
    (256, (16, 2), [20000, 12], 32, -1), (512, (8, 1), [6000], 16, -1), (128, (16, 2), [50000, 40000, 100], 16, 20000),
    (128, (8, 2), list(range(0, 3000, 7)), 16, -1),
])
def test_decode_long_caches_and_large_batches(d, heads, lengths, page_size, left):
    torch.manual_seed(lengths[0])
    table, pages = scattered(lengths, page_size)
    k, v = randn(pages, page_size, heads[1], d), randn(pages, page_size, heads[1], d)
    first = check_decode(randn(len(lengths), heads[0], d), k, v, table, ints(lengths), left, 5 if left >= 0 else 0)
    assert torch.isfinite(first[0]).all()


def test_decode_offsets_past_32_bits():
    pages, page_size, d = 70000, 16, 128
    k = torch.empty(pages, page_size, 16, d, dtype=torch.bfloat16, device="cuda")  # 2.3e9 elements
    table = ints([[pages - 1, 3, pages - 2], [pages - 5, pages - 4, 7]])
    k[table.flatten().long()] = randn(6, page_size, 16, d)
    small = torch.arange(6, device="cuda", dtype=torch.int32).view(2, 3)
    q, lengths = randn(2, 32, d), ints([40, 48])
    out = zigfa.flash_attn_paged_func(q, k, k, table, lengths)
    compact = k[table.flatten().long()].contiguous()
    assert torch.equal(out, zigfa.flash_attn_paged_func(q, compact, compact, small, lengths))
    rows = randn(2, 3, 16, d)
    zigfa.append_paged_kv(rows, rows, k, k, table, ints([0, 30]))
    assert torch.equal(k[pages - 1, :3], rows[0]) and torch.equal(k[pages - 4, 14:], rows[1, :2]) and torch.equal(k[7, 0], rows[1, 2])
    zigfa.copy_kv_pages(k, k, ints([pages - 1]), ints([pages - 30]))
    assert torch.equal(k[pages - 1], k[pages - 30])


def test_decode_repeats_bit_for_bit_on_streams_and_in_graphs():
    torch.manual_seed(6)
    lengths, page_size, d = [3000, 17, 900, 0], 16, 128
    table, pages = scattered(lengths, page_size, columns=300)
    k, v, q, held = randn(pages, page_size, 2, d), randn(pages, page_size, 2, d), randn(4, 8, d), ints(lengths)

    def call():
        return zigfa.flash_attn_paged_func(q, k, v, table, held, return_attn_probs=True)

    want = call()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for stream in streams:
            with torch.cuda.stream(stream):
                got.append(call())
    torch.cuda.synchronize()
    for out, lse in got:
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    # Graphs with pools of their own may be replayed in any order, each with a workspace that nobody else writes; graphs
    # that share a pool in the order of their capture (torch hands the second one the memory that the first has freed).
    # Replays read the tensors as they are then.
    for pool, order in ((None, (0, 1, 1, 0)), (torch.cuda.graph_pool_handle(), (0, 1, 0, 1))):
        graphs, results = [], []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, pool=pool):
                results.append(call())
            graphs.append(graph)
        held.copy_(ints([2999, 18, 850, 5] if pool is None else [1, 300, 2, 9]))
        table[3, 0], table[1] = table[0, 4], table[0].flip(0)
        want = call()
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        for out, lse in results:
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    torch.cuda.set_sync_debug_mode("error")
    try:
        call()
    finally:
        torch.cuda.set_sync_debug_mode("default")


# ------------------------------------------------------------------------------------------------ append and copy
@pytest.mark.parametrize("heads, d, page_size", [(1, 64, 16), (2, 72, 1), (8, 128, 64), (3, 96, 7), (1, 512, 24), (2, 8, 16)])
def test_append_matches_lists(heads, d, page_size):
    torch.manual_seed(heads * d)
    held, new = [0, 1, 15, 40, 100, 3], [0, 1, 70, 33, 16, 5]
    table, pages = scattered([h + n for h, n in zip(held, new)], page_size)
    table[4, -1] = -1
    k_cache, v_cache = randn(pages, page_size, heads, d), randn(pages, page_size, heads, d)
    total = sum(new)
    k, v = randn(total + 9, heads, d), randn(total + 9, heads, d)  # rows behind the last sequence are left out
    cu = ints([0, *torch.tensor(new).cumsum(0).tolist()])
    want = plain.append(k, v, k_cache, v_cache, table, ints(held), cu.tolist())
    zigfa.append_paged_kv(k, v, k_cache, v_cache, table, ints(held), cu)
    assert torch.equal(k_cache, want[0]) and torch.equal(v_cache, want[1])
    for tokens in (0, 1, 3):
        k, v = randn(6, heads, tokens, d).transpose(1, 2), randn(6, tokens, heads, d)
        want = plain.append(k, v, k_cache, v_cache, table, ints(held))
        zigfa.append_paged_kv(k, v, k_cache, v_cache, table, ints(held))
        assert torch.equal(k_cache, want[0]) and torch.equal(v_cache, want[1])


def test_append_drops_what_has_no_page():
    torch.manual_seed(8)
    k_cache, v_cache = randn(5, 16, 2, 64), randn(5, 16, 2, 64)
    table = ints([[0, -1], [5, 1], [2**31 - 1, -(2**31)], [2, 3], [4, 4]])
    held = ints([10, 10, 0, 30, -3])
    k, v = randn(5, 12, 2, 64), randn(5, 12, 2, 64)
    want = plain.append(k, v, k_cache, v_cache, table, held)
    zigfa.append_paged_kv(k, v, k_cache, v_cache, table, held)
    assert torch.equal(k_cache, want[0]) and torch.equal(v_cache, want[1])


def test_copy_pages():
    torch.manual_seed(9)
    for heads, d, page_size in ((1, 64, 16), (2, 72, 3), (8, 128, 64), (5, 8, 1)):
        buffer = randn(20, 2, page_size, heads, d)
        for k, v in ((buffer[:, 0], buffer[:, 1]), (randn(20, heads, page_size, d).transpose(1, 2), randn(20, page_size, heads, d))):
            source, target = [3, -1, 7, 3, 19, 20, 2**31 - 1, 5, 6], [0, 1, -1, 2, 4, 8, 9, 20, 6]
            want_k, want_v = k.clone(), v.clone()
            for s, t in zip(source, target):
                if 0 <= s < 20 and 0 <= t < 20:
                    want_k[t], want_v[t] = k[s], v[s]
            zigfa.copy_kv_pages(k, v, ints(source), ints(target))
            assert torch.equal(k, want_k) and torch.equal(v, want_v)
            zigfa.copy_kv_pages(k, v, ints([]), ints([]))


# ------------------------------------------------------------------------------------------------ bookkeeping
def books(generator, sequences, columns, pages, page_size):
    """A consistent state with some free pages, shared pages and entries that hold nothing."""
    rows, refs = [], [0] * pages
    order = list(range(pages))
    generator.shuffle(order)
    order = order[:int(pages * generator.uniform(0.2, 1.0))]
    lengths = []
    for b in range(sequences):
        length = generator.randint(0, columns * page_size)
        row = [-1] * columns
        for e in range(-(-length // page_size)):
            if order and generator.random() < 0.9:
                row[e] = order.pop()
            elif rows and generator.random() < 0.5:
                row[e] = rows[0][0]
        lengths.append(length)
        rows.append(row)
    for row in rows:
        for e in row:
            if e >= 0:
                refs[e] += 1
    return rows, lengths, refs


def as_lists(result):
    return [t.tolist() for t in result]


@pytest.mark.parametrize("sequences, columns, pages, page_size", [
    (1, 1, 1, 1), (1, 4, 2, 16), (3, 5, 12, 16), (9, 33, 200, 7), (70, 20, 900, 64), (300, 9, 5000, 16), (1500, 3, 3000, 8),
    (5, 2, 20000, 16), (9000, 1, 30, 16), (2, 700, 1025, 16)])
def test_bookkeeping_matches_lists(sequences, columns, pages, page_size):
    generator = random.Random(sequences * 7 + pages)
    for _ in range(3):
        rows, lengths, refs = books(generator, sequences, columns, pages, page_size)
        for row in rows[::5]:  # entries that hold nothing come in every form
            row[-1] = generator.choice([row[-1], -5, pages, 2**31 - 1, -(2**31)])
        wide = ints([[7] + row + [7, 7] for row in rows])
        table = wide[:, 1:1 + columns]
        counts = ints(refs)
        new = [generator.choice([0, 1, 1, 2, page_size, 5 * page_size, -3]) for _ in rows]
        assert as_lists(zigfa.reserve_kv_pages(table, ints(lengths), ints(new), counts, page_size)) == list(
            plain.reserve(rows, lengths, new, refs, page_size))
        parents = [generator.randint(-1, sequences) for _ in range(generator.choice([0, 1, 7, 150, 1300]))]
        child, held, refs_out, source, target = zigfa.fork_kv_pages(table, ints(lengths), counts, ints(parents), page_size)
        want = plain.fork(rows, lengths, refs, parents, page_size)
        assert child.shape == (len(parents), columns)
        assert as_lists((child, held, refs_out, source, target)) == list(want)
        first = [generator.choice([0, 0, 1, -2, columns]) for _ in rows]
        last = [generator.choice([0, columns, 2**31 - 1, 1, columns // 2]) for _ in rows]
        assert as_lists(zigfa.free_kv_pages(table, counts, ints(first), ints(last))) == list(plain.free(rows, refs, first, last))
        assert as_lists(zigfa.compact_kv_pages(table, counts)) == list(plain.compact(rows, refs))
        assert counts.tolist() == refs and wide.tolist() == [[7] + row + [7, 7] for row in rows]  # nothing in place


def test_bookkeeping_of_nothing():
    none, refs = torch.empty(0, 3, dtype=torch.int32, device="cuda"), ints([0, 1, 0, 2])
    assert as_lists(zigfa.compact_kv_pages(none, refs)) == [[], [2, 1, 0, 0], [3, -1], [0, -1]]  # page 3 (two references) goes to page 0
    assert as_lists(zigfa.free_kv_pages(none, refs, ints([]), ints([])))[1] == refs.tolist()
    assert as_lists(zigfa.reserve_kv_pages(none, ints([]), ints([]), refs, 4))[1] == refs.tolist()
    child = zigfa.fork_kv_pages(none, ints([]), refs, ints([0, -1]), 4)
    assert as_lists(child) == [[[-1] * 3] * 2, [0, 0], refs.tolist(), [-1, -1], [-1, -1]]
    no_columns = torch.empty(2, 0, dtype=torch.int32, device="cuda")
    assert as_lists(zigfa.reserve_kv_pages(no_columns, ints([0, 5]), ints([9, 9]), refs, 4))[1] == refs.tolist()
    assert as_lists(zigfa.compact_kv_pages(ints([[2, 0]]), ints([])))[0] == [[-1, -1]]


def test_bookkeeping_at_the_size_of_a_server():
    """A million pages: every choice follows from prefix sums over them."""
    torch.manual_seed(11)
    pages, page_size, sequences, columns = 1 << 20, 16, 512, 600
    order = torch.randperm(pages, device="cuda").int()
    table = order[:sequences * columns].view(sequences, columns).clone()
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[table.flatten().long()] = 1
    moved, counts, source, target = zigfa.compact_kv_pages(table, refs)
    live = sequences * columns
    assert torch.equal(counts, (torch.arange(pages, device="cuda") < live).int())
    assert torch.equal(moved.flatten().sort().values, torch.arange(live, device="cuda").int())
    pairs = int((source >= 0).sum())
    assert (source[pairs:] == -1).all() and (target[pairs:] == -1).all()
    assert torch.equal(source[:pairs], (refs > 0).nonzero().flatten().int()[-pairs:])
    assert torch.equal(target[:pairs], (refs[:live] <= 0).nonzero().flatten().int())
    to = torch.arange(pages, device="cuda").int()
    to[source[:pairs].long()] = target[:pairs]
    assert torch.equal(moved, to[table.long()])
    lengths = torch.full((sequences,), 500 * page_size, dtype=torch.int32, device="cuda")
    table[:, 500:] = -1
    refs = torch.zeros_like(refs)
    refs[table[:, :500].flatten().long()] = 1
    grown, counts = zigfa.reserve_kv_pages(table, lengths, torch.full_like(lengths, 100 * page_size), refs, page_size)
    assert torch.equal(grown[:, 500:].flatten(), (refs == 0).nonzero().flatten().int()[:sequences * 100])
    assert int(counts.sum()) == sequences * 600


# ------------------------------------------------------------------------------------------------ together
def test_a_server_that_appends_decodes_forks_frees_and_compacts():
    """The operators as they are used together: prompts are written, tokens decoded under a window with sinks, pages that the
    window has left given back, sequences forked and ended, the pool compacted. Next to it a plain list holds every
    sequence's keys and values, and each step's attention is compared with 64 bits over them."""
    torch.manual_seed(12)
    generator = random.Random(12)
    page_size, heads_q, heads_kv, d, columns, pages, left, sink = 16, 8, 2, 128, 40, 160, 100, 5
    k_cache, v_cache = randn(pages, page_size, heads_kv, d), randn(pages, page_size, heads_kv, d)
    sequences = 6
    table = torch.full((sequences, columns), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    history = [(randn(n, heads_kv, d), randn(n, heads_kv, d)) for n in (5, 16, 130, 300, 1, 0)]

    def lengths():
        return ints([len(k) for k, _ in history])

    new = lengths()
    table, refs = zigfa.reserve_kv_pages(table, torch.zeros_like(new), new, refs, page_size)
    cu = ints([0, *new.cumsum(0).tolist()])
    zigfa.append_paged_kv(torch.cat([k for k, _ in history]), torch.cat([v for _, v in history]), k_cache, v_cache, table,
                          torch.zeros_like(new), cu)
    for step in range(60):
        held = lengths()
        table, refs = zigfa.reserve_kv_pages(table, held, torch.ones_like(held), refs, page_size)
        k, v, q = randn(sequences, 1, heads_kv, d), randn(sequences, 1, heads_kv, d), randn(sequences, heads_q, d)
        zigfa.append_paged_kv(k, v, k_cache, v_cache, table, held)
        history = [(torch.cat([hk, nk]), torch.cat([hv, nv])) for (hk, hv), nk, nv in zip(history, k, v)]
        out = zigfa.flash_attn_paged_func(q, k_cache, v_cache, table, held + 1, window_size=(left, 0), sink_size=sink,
                                          return_attn_probs=True)
        longest = max(len(hk) for hk, _ in history)
        dense_k, dense_v = (torch.zeros(sequences, longest, heads_kv, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        for b, (hk, hv) in enumerate(history):
            dense_k[b, :len(hk)], dense_v[b, :len(hv)] = hk, hv
        identity = torch.arange(sequences, device="cuda", dtype=torch.int32)[:, None]
        plain.assert_decode(out, plain.decode(q, dense_k, dense_v, identity, held + 1, d**-0.5, left, sink), step)
        kind = step % 6
        if kind == 1:  # the window moves on
            behind = (lengths() - left).clamp(min=0) // page_size
            table, refs = zigfa.free_kv_pages(table, refs, torch.full_like(behind, -(-sink // page_size)), behind)
        elif kind == 3:  # one sequence ends, a fork of another takes its place
            ended, parent = generator.sample(range(sequences), 2)
            gone = torch.zeros(sequences, dtype=torch.int32, device="cuda")
            gone[ended] = columns
            table, refs = zigfa.free_kv_pages(table, refs, torch.zeros_like(gone), gone)
            child, child_length, refs, source, target = zigfa.fork_kv_pages(table, lengths(), refs, ints([parent]), page_size)
            zigfa.copy_kv_pages(k_cache, v_cache, source, target)
            table[ended] = child[0]
            history[ended] = history[parent]
            assert child_length.tolist() == [len(history[parent][0])]
        elif kind == 5:
            table, refs, source, target = zigfa.compact_kv_pages(table, refs)
            zigfa.copy_kv_pages(k_cache, v_cache, source, target)
            used = int((refs > 0).sum())
            assert (refs[:used] > 0).all() and int(table.max()) < used
        entries = table[table >= 0].long()
        assert torch.equal(torch.bincount(entries, minlength=pages).int(), refs.clamp(min=0))


def test_the_books_and_the_writes_run_in_a_captured_graph():
    torch.manual_seed(13)
    page_size, pages = 16, 64
    table, refs = torch.full((4, 8), -1, dtype=torch.int32, device="cuda"), torch.zeros(pages, dtype=torch.int32, device="cuda")
    held, one = ints([0, 0, 0, 0]), ints([1, 1, 1, 1])
    k_cache, v_cache = torch.zeros(pages, page_size, 2, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(pages, page_size, 2, 64, device="cuda", dtype=torch.bfloat16)
    k, q = randn(4, 1, 2, 64), randn(4, 4, 64)

    def step():
        new_table, new_refs = zigfa.reserve_kv_pages(table, held, one, refs, page_size)
        zigfa.append_paged_kv(k, k, k_cache, v_cache, new_table, held)
        table.copy_(new_table)
        refs.copy_(new_refs)
        held.add_(one)
        return zigfa.flash_attn_paged_func(q, k_cache, v_cache, table, held)

    step()  # warm-up, also step 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(40):
        graph.replay()
    torch.cuda.synchronize()
    assert held.tolist() == [41] * 4 and int((refs > 0).sum()) == 4 * 3
    # every value ever written is the same k: softmax over equal rows gives that row back
    assert torch.allclose(out.float(), k[:, 0].float().repeat_interleave(2, 1), rtol=2.0**-7, atol=0)


def test_other_device_than_the_current_one_is_refused_or_used():
    q, k, table, lengths = randn(2, 4, 64), randn(4, 16, 2, 64), ints([[0], [1]]), ints([5, 6])
    with pytest.raises((ValueError, NotImplementedError)):
        zigfa.flash_attn_paged_func(q, k, k, table.cpu(), lengths)
    with pytest.raises((ValueError, NotImplementedError)):
        zigfa.flash_attn_paged_func(q.cpu(), k.cpu(), k.cpu(), table.cpu(), lengths.cpu())
    with pytest.raises((ValueError, NotImplementedError)):
        zigfa.copy_kv_pages(k, k, lengths.cpu(), lengths.cpu())


def test_ops_pass_the_library_checks_and_compile():
    utils = ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic")
    torch.manual_seed(14)
    table, lengths, refs = ints([[0, 2], [1, 3]]), ints([20, 7]), ints([1, 1, 1, 1, 0, 0])
    q, k_cache, v_cache = randn(2, 4, 64), randn(6, 16, 2, 64), randn(6, 16, 2, 64)
    k = randn(2, 1, 2, 64)
    zigfa.flash_attn_paged_func(q, k_cache, v_cache, table, lengths)
    for op, arguments in [
        ("paged_forward", (q, k_cache, v_cache, table, lengths, 0.1, 5, 2)), ("append_kv", (k, k, k_cache, v_cache, table, lengths, None)),
        ("copy_pages", (k_cache, v_cache, ints([0, -1]), ints([5, -1]))), ("reserve_pages", (table, lengths, lengths, refs, 16)),
        ("fork_pages", (table, lengths, refs, ints([1, 0, 1]), 16)), ("free_pages", (table, refs, ints([0, 0]), ints([1, 2]))),
        ("compact_pages", (table, refs)),
    ]:
        torch.library.opcheck(getattr(torch.ops.zigfa, op).default, arguments, test_utils=utils)

    def step(q, k, k_cache, v_cache, table, lengths, refs):
        table, refs = zigfa.reserve_kv_pages(table, lengths, torch.ones_like(lengths), refs, 16)
        zigfa.append_paged_kv(k, k, k_cache, v_cache, table, lengths)
        return zigfa.flash_attn_paged_func(q, k_cache, v_cache, table, lengths + 1, window_size=(9, 0), sink_size=2), table, refs

    torch._dynamo.reset()
    with torch.no_grad():
        caches = [(k_cache.clone(), v_cache.clone()) for _ in range(2)]
        want = step(q, k, *caches[0], table, lengths, refs)
        got = torch.compile(step, fullgraph=True)(q, k, *caches[1], table, lengths, refs)
    torch._dynamo.reset()
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and all(torch.equal(a, b) for a, b in zip(*caches))


def test_writes_raise_the_version_of_the_caches():
    torch.manual_seed(15)
    table, held, rows = ints([[0, 1]]), ints([3]), randn(1, 1, 2, 64)
    writes = (lambda k, v: zigfa.append_paged_kv(rows, rows, k, v, table, held), lambda k, v: zigfa.copy_kv_pages(k, v, ints([0]), ints([2])),
              lambda k, v: torch.ops.zigfa.append_kv(rows, rows, k, v, table, held, None),
              lambda k, v: torch.ops.zigfa.copy_pages(k, v, ints([0]), ints([2])))
    for write in writes:
        k, v = randn(4, 16, 2, 64), randn(4, 16, 2, 64)
        before = k._version, v._version
        write(k, v)
        assert k._version > before[0] and v._version > before[1]
        # training over a cached prefix: the attention has saved views of the cache
        q = randn(1, 32, 2, 64).requires_grad_()
        out = zigfa.flash_attn_func(q, k[:2].reshape(1, 32, 2, 64), v[:2].reshape(1, 32, 2, 64), causal=True)
        write(k, v)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()
        with torch.inference_mode():
            write(randn(4, 16, 2, 64), randn(4, 16, 2, 64))


@pytest.mark.parametrize("d, heads, lengths, page_size", [(128, (8, 2), [40, 300, 20000, 9], 16), (64, (4, 4), [40, 300, 9], 7),
                                                         (256, (4, 2), [2000, 5, 9], 16), (512, (2, 1), [30, 5, 9], 16)])
def test_decode_reports_what_is_no_number(d, heads, lengths, page_size):
    """A NaN among the queries or the visible keys makes that head's output and log-sum-exp NaN, not "sees no key" (-inf)."""
    torch.manual_seed(d)
    table, pages = scattered(lengths, page_size)
    k, v = randn(pages, page_size, heads[1], d), randn(pages, page_size, heads[1], d)
    q = randn(len(lengths), heads[0], d)
    want, want_lse, tolerance, lse_tolerance = plain.decode(q, k, v, table, lengths, d**-0.5, -1, 0)
    group = heads[0] // heads[1]
    bad = torch.zeros(len(lengths), heads[0], dtype=torch.bool)
    bad[0, 0] = bad[1, :group] = True
    for value in (float("nan"), float("inf")):
        bad_q, bad_k = q.clone(), k.clone()
        bad_q[0, 0, 3] = value
        page = table[1, lengths[1] // page_size // 2]
        bad_k[page, 1, 0, 5], bad_k[page, 2, 0, 5] = value, -value  # seen by the first key head's queries of sequence 1
        out, lse = (x.cpu() for x in zigfa.flash_attn_paged_func(bad_q, bad_k, v, table, ints(lengths), return_attn_probs=True))
        assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all()
        assert ((out.double() - want).abs() <= tolerance)[~bad].all()  # nobody else's
        assert ((lse.double() - want_lse).abs() <= lse_tolerance)[~bad].all()


def test_vmap_takes_the_dispatcher():
    torch.manual_seed(16)
    table, lengths = ints([[0, 1], [2, 3]]), ints([20, 7])
    q, k, v = randn(3, 2, 4, 64), randn(4, 16, 2, 64), randn(4, 16, 2, 64)
    want = torch.stack([zigfa.flash_attn_paged_func(x, k, v, table, lengths) for x in q])
    assert torch.equal(torch.vmap(lambda x: zigfa.flash_attn_paged_func(x, k, v, table, lengths))(q), want)
    rows = randn(3, 2, 1, 2, 64)
    before = k.clone()
    with pytest.raises(RuntimeError, match="append_kv|vmap|[Bb]atch"):
        torch.vmap(lambda x: zigfa.append_paged_kv(x, x, k, v, table, lengths))(rows)
    assert torch.equal(k, before)
    q, k, v = randn(3, 1, 40, 2, 64), randn(1, 40, 2, 64), randn(1, 40, 2, 64)
    want = torch.stack([zigfa.flash_attn_sink_func(x, k, v, 4, causal=True, window_size=(9, -1)) for x in q])
    assert torch.equal(torch.vmap(lambda x: zigfa.flash_attn_sink_func(x, k, v, 4, causal=True, window_size=(9, -1)))(q), want)
