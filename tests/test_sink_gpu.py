"""GPU tests of sliding-window attention with sinks: output, log-sum-exp and gradients against 64 bits with tolerances that
count the kernels' roundings (sink_reference.py)."""
import itertools

import pytest
import torch

import sink_reference as plain
import zigfa
from zigfa._impl import ops

pytestmark = pytest.mark.gpu


def randn(*shape, requires_grad=False):
    return torch.randn(*shape, device="cuda", dtype=torch.bfloat16).requires_grad_(requires_grad)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def check_fixed(batch, lq, lk, heads, d, left, right, sink, backward=True, scale=None, note=""):
    note = note or (batch, lq, lk, heads, d, left, right, sink)
    q, k, v = randn(batch, lq, heads[0], d, requires_grad=True), randn(batch, lk, heads[1], d, requires_grad=True), randn(batch, lk, heads[1], d, requires_grad=True)
    dout = randn(batch, lq, heads[0], d) if backward else None
    out, lse = zigfa.flash_attn_sink_func(q, k, v, sink, softmax_scale=scale, window_size=(left, right), return_attn_probs=True)
    got = {"out": out.detach(), "lse": lse}
    if backward:
        got.update(zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), dout)))
    mask = plain.visible(lq, lk, left, right, sink)
    for b in range(batch):
        want = plain.with_tolerances(q[b].detach(), k[b].detach(), v[b].detach(), dout[b] if backward else None, mask,
                                     d**-0.5 if scale is None else scale)
        for name, (value, tolerance) in want.items():
            plain.assert_within(name, got[name][b], value, tolerance, note)
    return got


@pytest.mark.parametrize("d", [64, 72, 96, 128, 256, 512])
@pytest.mark.parametrize("left, sink", [(0, 1), (1, 4), (63, 1), (100, 4), (127, 128), (128, 129), (200, 17), (400, 300), (1000, 5)])
def test_fixed_length_matches_64_bits(d, left, sink):
    torch.manual_seed(d + left + sink)
    for lq, lk in ((1, 1), (130, 130), (257, 513), (700, 700), (300, 90)):
        check_fixed(1, lq, lk, (2, 2) if lq % 2 else (6, 2), d, left, 0, sink, backward=d < 512)


@pytest.mark.parametrize("heads", [(1, 1), (4, 4), (6, 1), (8, 2), (32, 2), (3, 3)])
def test_head_layouts(heads):
    torch.manual_seed(heads[0])
    for d, right in itertools.product((64, 128), (-1, 0, 50)):
        check_fixed(2, 333, 450, heads, d, 77, right, 9)


def test_long_sequences():
    torch.manual_seed(1)
    check_fixed(1, 3000, 3000, (4, 2), 128, 511, 0, 4)
    check_fixed(1, 2500, 2900, (4, 1), 64, 300, 0, 200)
    check_fixed(2, 2100, 2100, (2, 2), 96, 20, 0, 1)
    check_fixed(1, 2000, 2000, (2, 1), 256, 200, 0, 5)
    check_fixed(1, 1300, 1500, (2, 2), 512, 200, 0, 5, backward=False)


def test_short_queries_over_long_keys_take_the_split_path():
    torch.manual_seed(2)
    for d in (64, 128):
        check_fixed(1, 40, 9000, (4, 2), d, 5000, 0, 300)
        check_fixed(1, 1, 6000, (8, 1), d, 3000, 0, 4)


def test_peaked_rows_scales_and_the_pivot_setting():
    torch.manual_seed(3)
    for scale in (1.5, 1e-6, 0.02):
        check_fixed(1, 400, 400, (4, 2), 64, 64, 0, 4, scale=scale)
    before = zigfa.set_pivot_gradients(True)
    try:
        check_fixed(1, 700, 700, (4, 2), 128, 100, 0, 4)
        check_fixed(1, 300, 300, (2, 1), 64, 30, 0, 130, scale=0.5)
        check_fixed(1, 1500, 1500, (2, 1), 256, 100, 0, 4, scale=0.3)
    finally:
        zigfa.set_pivot_gradients(before)


PACKED = [([5], [5]), ([300, 0, 1, 513, 77], [300, 5, 1, 600, 0]), ([129, 127, 128], [129, 300, 128]), ([1000, 30], [1000, 700]),
          ([0, 0], [0, 0]), ([200, 333, 64, 65, 1, 1, 2], [100, 333, 64, 65, 1, 2, 1])]


@pytest.mark.parametrize("lengths", PACKED)
@pytest.mark.parametrize("heads, d", [((4, 4), 128), ((8, 2), 64), ((3, 1), 96), ((16, 1), 128), ((4, 2), 256), ((2, 1), 512)])
def test_packed_batches_match_64_bits_whatever_stands_behind_them(lengths, heads, d):
    """Rows behind the last sequence hold NaN, and are left as they were."""
    torch.manual_seed(sum(lengths[0]) + d)
    lengths_q, lengths_k = lengths
    padding, (total_q, total_k) = 70, (sum(lengths_q), sum(lengths_k))
    cu_q, cu_k = (ints([0, *torch.tensor(x).cumsum(0).tolist()]) for x in lengths)
    for left, right, sink in ((100, 0, 4), (15, -1, 140), (0, 0, 1)):
        q, k, v, dout = randn(total_q + padding, heads[0], d), randn(total_k + padding, heads[1], d), randn(total_k + padding, heads[1], d), randn(total_q + padding, heads[0], d)
        for x, total in ((q, total_q), (k, total_k), (v, total_k), (dout, total_q)):
            x[total:] = float("nan")
        leaves = [x.requires_grad_(d < 512) for x in (q, k, v)]
        out, lse = zigfa.flash_attn_varlen_sink_func(*leaves, cu_q, cu_k, max(lengths_q), max(lengths_k), sink, window_size=(left, right),
                                                     return_attn_probs=True)
        got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout) if d < 512 else ()), out=out.detach())
        row_q = row_k = 0
        for lq, lk in zip(lengths_q, lengths_k):
            rows, keys = slice(row_q, row_q + lq), slice(row_k, row_k + lk)
            want = plain.with_tolerances(q[rows].detach(), k[keys].detach(), v[keys].detach(), dout[rows] if d < 512 else None, plain.visible(lq, lk, left, right, sink), d**-0.5)
            plain.assert_within("lse", lse[:, rows], *want.pop("lse"), (lengths, heads, left))
            for name, (value, tolerance) in want.items():
                plain.assert_within(name, got[name][keys if name in ("dk", "dv") else rows], value, tolerance, (lengths, heads, left, lq, lk))
            row_q, row_k = row_q + lq, row_k + lk


def test_rows_behind_the_last_sequence_are_not_written():
    torch.manual_seed(5)
    total, padding, d = 400, 64, 128
    q, k, v, dout = (randn(total + padding, 4, d) for _ in range(4))
    cu = ints([0, 150, 400])
    out, lse = torch.full_like(q, float("nan")), torch.full((4, total + padding), float("nan"), device="cuda")
    ops.launch_forward(q, k, v, out, lse, cu, cu, d**-0.5, 50, 0, sink=4)
    assert torch.isnan(out[total:]).all() and torch.isnan(lse[:, total:]).all() and torch.isfinite(out[:total]).all()
    gradients = [torch.full_like(q, float("nan")) for _ in range(3)]
    ops.launch_backward(dout, q, k, v, out, lse, *gradients, cu, cu, d**-0.5, 50, 0, sink=4)
    for gradient in gradients:
        assert torch.isnan(gradient[total:]).all() and torch.isfinite(gradient[:total]).all()


def test_without_a_window_or_sinks_it_is_plain_attention_to_the_last_bit():
    torch.manual_seed(6)
    q, k, v = randn(2, 300, 8, 128), randn(2, 500, 2, 128), randn(2, 500, 2, 128)
    for sink, window, causal in ((0, (60, 0), False), (7, (-1, -1), True), (500, (-1, 30), False)):
        got = zigfa.flash_attn_sink_func(q, k, v, sink, causal=causal, window_size=window, return_attn_probs=True)
        want = zigfa.flash_attn_func(q, k, v, causal=causal, window_size=window, return_attn_probs=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # as many sinks as keys: nothing of the causal triangle is hidden
    got = zigfa.flash_attn_sink_func(q, k, v, 500, window_size=(10, 0), return_attn_probs=True)
    want = zigfa.flash_attn_func(q, k, v, causal=True, return_attn_probs=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_strided_inputs_and_expanded_gradients():
    torch.manual_seed(7)
    qkv = randn(2, 300, 3, 4, 64, requires_grad=True)
    q, k, v = qkv.unbind(2)
    out = zigfa.flash_attn_sink_func(q, k, v, 4, causal=True, window_size=(50, -1))
    out.sum().backward()  # the gradient of a sum is an expanded one
    dense = [x.detach().contiguous().requires_grad_() for x in (q, k, v)]
    other = zigfa.flash_attn_sink_func(*dense, 4, causal=True, window_size=(50, -1))
    assert torch.equal(out, other)
    gradients = torch.autograd.grad(other, dense, torch.ones_like(other))
    for i in (1, 2):  # dq is summed by atomic additions, dk and dv are not
        assert torch.equal(qkv.grad[:, :, i], gradients[i])
    assert torch.allclose(qkv.grad[:, :, 0].float(), gradients[0].float(), rtol=2.0**-6, atol=1e-4)


def test_streams_graphs_and_no_synchronisation():
    torch.manual_seed(8)
    cu = ints([0, 130, 700])
    q, k, v = (randn(700, 4, 64, requires_grad=True) for _ in range(3))
    dout = randn(700, 4, 64)

    def step():
        out, lse = zigfa.flash_attn_varlen_sink_func(q, k, v, cu, cu, 570, 570, 6, causal=True, window_size=(90, 0), return_attn_probs=True)
        return out.detach(), lse, *torch.autograd.grad(out, (q, k, v), dout)

    want = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # no eager autograd graph of the leaves is alive here: torch would join its stream
        captured = step()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    for result in (again, captured):
        for i in (0, 1, 3, 4):
            assert torch.equal(result[i], want[i]), i
        assert torch.allclose(result[2].float(), want[2].float(), rtol=2.0**-6, atol=1e-4)
    torch.cuda.set_sync_debug_mode("error")
    try:
        step()
    finally:
        torch.cuda.set_sync_debug_mode("default")


def test_head_dims_without_a_kernel_are_refused():
    q = randn(1, 64, 2, 80)
    with pytest.raises(ValueError, match="head_dim"):
        zigfa.flash_attn_sink_func(q, q, q, 4, window_size=(10, 0))
    q = randn(1, 64, 2, 512, requires_grad=True)
    out = zigfa.flash_attn_sink_func(q, q, q, 4, window_size=(10, 0))
    with pytest.raises(NotImplementedError, match="512"):  # forward only, as everywhere
        out.sum().backward()
    with pytest.raises(ValueError, match="cuda|cpu"):
        zigfa.flash_attn_varlen_sink_func(*(randn(64, 2, 64) for _ in range(3)), ints([0, 64]).cpu(), ints([0, 64]).cpu(), 64, 64, 4, window_size=(9, 0))


OPCHECK = ("test_schema", "test_autograd_registration", "test_faketensor", "test_aot_dispatch_dynamic")


def test_ops_pass_the_library_checks():
    q, k = randn(1, 40, 2, 64), randn(1, 40, 2, 64)
    arguments = (q, k, k, None, None, 0.1, 9, 0, 3)
    torch.library.opcheck(torch.ops.zigfa.sink_forward.default, arguments, test_utils=OPCHECK)
    out, lse = torch.ops.zigfa.sink_forward(*arguments)
    torch.library.opcheck(torch.ops.zigfa.sink_backward.default, (randn(1, 40, 2, 64), q, k, k, out, lse, *arguments[3:]), test_utils=OPCHECK)
    cu = ints([0, 10, 40])
    torch.library.opcheck(torch.ops.zigfa.sink_forward.default, (q[0], k[0], k[0], cu, cu, 0.1, 9, 0, 3), test_utils=OPCHECK)


def test_compiled_attention_matches_eager():
    torch._dynamo.reset()
    torch.manual_seed(9)
    q, k, v = (randn(2, 256, h, 128, requires_grad=True) for h in (4, 2, 2))

    def attention(q, k, v):
        return zigfa.flash_attn_sink_func(q, k, v, 4, causal=True, window_size=(60, -1))

    compiled = torch.compile(attention, fullgraph=True, dynamic=True)
    out, eager = compiled(q, k, v), attention(q, k, v)
    dout = randn(*out.shape)
    got, want = torch.autograd.grad(out, (q, k, v), dout), torch.autograd.grad(eager, (q, k, v), dout)
    assert torch.equal(out, eager) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    assert torch.allclose(got[0].float(), want[0].float(), rtol=2.0**-6, atol=1e-4)
    torch._dynamo.reset()


def test_a_second_derivative_is_refused():
    q, k, v = (randn(1, 40, 2, 64, requires_grad=True) for _ in range(3))
    out = zigfa.flash_attn_sink_func(q, k, v, 4, causal=True, window_size=(9, -1))
    gradient, = torch.autograd.grad(out.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gradient.sum().backward()


def test_two_streams_at_once():
    """Calls in flight on two streams share nothing: the same values as one after the other."""
    torch.manual_seed(10)
    cu = ints([0, 700, 1500])
    inputs = [[randn(1500, 8, 128), randn(1500, 2, 128), randn(1500, 2, 128)] for _ in range(2)]
    calls = [lambda x=x: zigfa.flash_attn_varlen_sink_func(*x, cu, cu, 800, 800, 5, causal=True, window_size=(200, 0)) for x in inputs]
    want = [call() for call in calls]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for stream, call in zip(streams, calls):
            with torch.cuda.stream(stream):
                got.append(call())
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert torch.equal(out, want[i % 2])


@pytest.mark.parametrize("left, right, sink", [(100, 0, 0), (-1, 0, 4), (-1, -1, 0), (-1, 30, 200), (0, -1, 0)])
@pytest.mark.parametrize("heads, d", [((4, 4), 128), ((8, 2), 64), ((3, 1), 96), ((4, 2), 256), ((2, 1), 512)])
def test_packed_batches_without_sinks_or_a_left_bound_do_not_see_what_stands_behind_them(left, right, sink, heads, d):
    """The promise about rows behind the last sequence holds whatever the window and the sinks are."""
    torch.manual_seed(d + left + sink)
    lengths_q, lengths_k, padding = (300, 0, 77, 129), (300, 5, 200, 130), 70
    total_q, total_k = sum(lengths_q), sum(lengths_k)
    cu_q, cu_k = (ints([0, *torch.tensor(x).cumsum(0).tolist()]) for x in (lengths_q, lengths_k))
    q, k, v, dout = (randn(total + padding, h, d) for total, h in ((total_q, heads[0]), (total_k, heads[1]), (total_k, heads[1]), (total_q, heads[0])))
    for x, total in ((q, total_q), (k, total_k), (v, total_k), (dout, total_q)):
        x[total:] = float("nan")
    leaves = [x.requires_grad_(d < 512) for x in (q, k, v)]
    out, lse = zigfa.flash_attn_varlen_sink_func(*leaves, cu_q, cu_k, 300, 300, sink, window_size=(left, right), return_attn_probs=True)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout) if d < 512 else ()), out=out.detach())
    row_q = row_k = 0
    for lq, lk in zip(lengths_q, lengths_k):
        rows, keys = slice(row_q, row_q + lq), slice(row_k, row_k + lk)
        want = plain.with_tolerances(q[rows].detach(), k[keys].detach(), v[keys].detach(), dout[rows] if d < 512 else None, plain.visible(lq, lk, left, right, sink), d**-0.5)
        plain.assert_within("lse", lse[:, rows], *want.pop("lse"), (heads, lq, lk))
        for name, (value, tolerance) in want.items():
            plain.assert_within(name, got[name][keys if name in ("dk", "dv") else rows], value, tolerance, (heads, d, lq, lk))
        row_q, row_k = row_q + lq, row_k + lk


@pytest.mark.parametrize("d", [64, 72, 128, 256, 512])
@pytest.mark.parametrize("window, sink", [((50, 0), 4), ((50, 0), 0), ((-1, 0), 0)])
def test_rows_of_no_sequence_come_out_as_zeros(d, window, sink):
    """What the functions return for rows in front of the first and behind the last sequence is defined: zeros, a log-sum-exp
    of -inf, and gradients of zero, so that a layer in front may sum over all rows."""
    torch.manual_seed(d)
    for cu_q, cu_k, total_q, total_k in (([0, 150, 400], [0, 20, 300], 1000, 333), ([3, 100], [40, 200], 101, 900), ([0, 64], [0, 64], 64, 64),
                                         ([7], [9], 50, 60), ([0, 0], [0, 30], 40, 30), ([0, 5, 5], [0, 0, 0], 6, 3)):
        leftover = [torch.full((n,), float("nan"), device="cuda", dtype=torch.bfloat16) for n in (total_q * 4 * d, total_k * 2 * d) * 4]
        del leftover  # the allocator hands this memory out next
        q, k, v = (randn(n, h, d, requires_grad=d < 512) for n, h in ((total_q, 4), (total_k, 2), (total_k, 2)))
        dout = torch.ones(total_q, 4, d, device="cuda", dtype=torch.bfloat16)
        out, lse = zigfa.flash_attn_varlen_sink_func(q, k, v, ints(cu_q), ints(cu_k), 300, 300, sink, window_size=window, return_attn_probs=True)
        results = [(out.detach(), cu_q)]
        if d < 512:
            results += zip(torch.autograd.grad(out, (q, k, v), dout), (cu_q, cu_k, cu_k))
        for tensor, cu in results:
            assert torch.isfinite(tensor).all()
            assert (tensor[:cu[0]] == 0).all() and (tensor[cu[-1]:] == 0).all()
            if len(cu) > 1 and cu_q[-1] > cu_q[0] and cu_k[-1] > cu_k[0]:
                assert (tensor[cu[0]:cu[-1]] != 0).any()
        assert (lse[:, :cu_q[0]] == float("-inf")).all() and (lse[:, cu_q[-1]:] == float("-inf")).all()
        assert not torch.isnan(lse).any()


@pytest.mark.parametrize("heads, d, left, sink", [((4, 2), 64, 100, 4), ((2, 2), 128, 300, 300), ((4, 1), 256, 60, 17), ((3, 1), 72, 0, 500)])
def test_many_short_documents_next_to_long_ones(heads, d, left, sink):
    """Documents below, at and above the size of a share (512 query rows here and more) in one packed batch."""
    torch.manual_seed(d + sink)
    lengths = [int(n) for n in torch.randint(0, 60, (40,))]
    for place, length in ((0, 513), (5, 2100), (11, 512), (12, 511), (20, 1025), (30, 1024), (40, 3000), (44, 640), (46, 641)):
        lengths.insert(place, length)
    other = [n + (i % 3) * 17 if i % 5 else n // 2 for i, n in enumerate(lengths)]
    lengths[25] = other[25] = 0
    other[10], lengths[33] = 0, 0
    cu_q, cu_k = (ints([0, *torch.tensor(x).cumsum(0).tolist()]) for x in (lengths, other))
    q, k, v = (randn(sum(x), h, d, requires_grad=True) for x, h in ((lengths, heads[0]), (other, heads[1]), (other, heads[1])))
    dout = randn(sum(lengths), heads[0], d)
    out = zigfa.flash_attn_varlen_sink_func(q, k, v, cu_q, cu_k, 3000, 3100, sink, window_size=(left, 0))
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), dout)), out=out.detach())
    again = torch.autograd.grad(zigfa.flash_attn_varlen_sink_func(q, k, v, cu_q, cu_k, 3000, 3100, sink, window_size=(left, 0)), (k, v), dout)
    assert torch.equal(again[0], got["dk"]) and torch.equal(again[1], got["dv"])  # parts are added in order
    row_q = row_k = 0
    for lq, lk in zip(lengths, other):
        rows, keys = slice(row_q, row_q + lq), slice(row_k, row_k + lk)
        want = plain.with_tolerances(q[rows].detach(), k[keys].detach(), v[keys].detach(), dout[rows], plain.visible(lq, lk, left, 0, sink), d**-0.5)
        want.pop("lse")
        for name, (value, tolerance) in want.items():
            plain.assert_within(name, got[name][keys if name in ("dk", "dv") else rows], value, tolerance, (d, lq, lk))
        row_q, row_k = row_q + lq, row_k + lk


@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("sink, window", [(4, (3, 0)), (0, (-1, -1))])
def test_packed_batches_of_no_rows(d, sink, window):
    for total_q, total_k, cu_q, cu_k in ((0, 5, [0, 0], [0, 5]), (5, 0, [0, 5], [0, 0]), (0, 0, [0], [0]), (0, 0, [0, 0, 0], [0, 0, 0]),
                                         (6, 7, [0, 3, 3], [2, 2, 7])):
        q, k, v = (randn(n, h, d, requires_grad=d < 512) for n, h in ((total_q, 4), (total_k, 2), (total_k, 2)))
        out, lse = zigfa.flash_attn_varlen_sink_func(q, k, v, ints(cu_q), ints(cu_k), 9, 9, sink, window_size=window, return_attn_probs=True)
        assert out.shape == q.shape and lse.shape == (4, total_q)
        assert (out == 0).all() and (lse == float("-inf")).all()  # no row sees a key
        if d < 512:
            for gradient, x in zip(torch.autograd.grad(out, (q, k, v), torch.ones_like(out)), (q, k, v)):
                assert gradient.shape == x.shape and (gradient == 0).all()
