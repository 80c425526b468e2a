"""Plain statements of the paged operators for the tests: lists and loops for the bookkeeping, 64-bit attention over the
keys that a sequence's table entries name."""
import torch

EPS = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}  # half a step, relative


def visible_keys(length, capacity, left, sink):
    length = min(max(length, 0), capacity)
    return [j for j in range(length) if left < 0 or j >= length - 1 - left or j < sink]


def decode(q, k_cache, v_cache, table, lengths, scale, left, sink):
    """(out, lse, tolerance of out, tolerance of lse) in 64 bits on the CPU. The tolerances add up the roundings of the
    kernels: the output is rounded to BF16 (half a step of itself), the probabilities enter the product with V in BF16 (half
    a step of sum p |v|), a score is a sum of head_dim products in FP32 (head_dim + 2 half steps of scale * sum |q k|, the
    last two for the scale and the subtraction of the maximum, whose size that sum bounds), exp2 has 2 steps, and the sums
    over n keys run in at most n / 16 + 64 FP32 additions one behind the other."""
    q, k_cache, v_cache, table = (x.cpu() for x in (q, k_cache, v_cache, table))
    batch, heads_q, d = q.shape
    pages, page_size, heads_kv, _ = k_cache.shape
    capacity, group = table.shape[1] * page_size, heads_q // heads_kv
    out = torch.zeros(batch, heads_q, d, dtype=torch.float64)
    lse = torch.full((batch, heads_q), float("-inf"), dtype=torch.float64)
    out_tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(batch):
        keys = visible_keys(int(lengths[b]), capacity, left, sink)
        slots = [(int(table[b, j // page_size]), j % page_size) for j in keys]
        slots = [(page, row) for page, row in slots if 0 <= page < pages]
        if not slots:
            continue
        page, row = (torch.tensor(x) for x in zip(*slots))
        k = k_cache[page, row].double().repeat_interleave(group, 1)  # (keys, heads_q, d)
        v = v_cache[page, row].double().repeat_interleave(group, 1)
        qb = q[b].double()
        s = torch.einsum("hd,khd->hk", qb, k) * scale
        lse[b] = torch.logsumexp(s, 1)
        p = torch.exp(s - lse[b][:, None])
        out[b] = torch.einsum("hk,khd->hd", p, v)
        half = EPS[torch.float32]
        score = (d + 2) * half * abs(scale) * torch.einsum("hd,khd->hk", qb.abs(), k.abs()).amax(1) * 2 + 4 * half
        chain = (len(slots) / 16 + 64) * half
        weight = torch.einsum("hk,khd->hd", p, v.abs())
        out_tol[b] = EPS[torch.bfloat16] * out[b].abs() + weight * (EPS[torch.bfloat16] + 2 * score[:, None] + 2 * chain) * 1.01
        lse_tol[b] = score + chain + 4 * half * lse[b].abs()
    return out, lse, out_tol, lse_tol


def assert_decode(result, reference, note=""):
    out, lse = (x.double().cpu() for x in result)
    want, want_lse, tol, lse_tol = reference
    assert not torch.isnan(out).any() and not torch.isnan(lse).any(), note
    assert torch.equal(lse == float("-inf"), want_lse == float("-inf")), note
    finite = torch.isfinite(want_lse)
    assert ((lse - want_lse).abs()[finite] <= lse_tol[finite]).all(), (note, (lse - want_lse).abs()[finite].max())
    excess = (out - want).abs() - tol
    assert (excess <= 0).all(), (note, excess.max())


def append(k, v, k_cache, v_cache, table, lengths, cu=None):
    """The caches (copies) after the call."""
    k_cache, v_cache = k_cache.clone(), v_cache.clone()
    pages, page_size = k_cache.shape[:2]
    table, lengths = table.tolist(), lengths.tolist()
    for b in range(len(lengths)):
        count = k.shape[1] if cu is None else int(cu[b + 1] - cu[b])
        for i in range(count):
            position = lengths[b] + i
            if not 0 <= position < len(table[b]) * page_size:
                continue
            page = table[b][position // page_size]
            if 0 <= page < pages:
                at = (b, i) if cu is None else (int(cu[b]) + i,)
                k_cache[page, position % page_size] = k[at]
                v_cache[page, position % page_size] = v[at]
    return k_cache, v_cache


def _clean(table, pages):
    return [[e if 0 <= e < pages else -1 for e in row] for row in table]


def reserve(table, lengths, new, refs, page_size):
    table, refs = _clean(table, len(refs)), list(refs)
    free = [i for i, r in enumerate(refs) if r <= 0]
    for b, row in enumerate(table):
        length = max(lengths[b], 0)
        first, last = -(-length // page_size), -(-(length + max(new[b], 0)) // page_size)
        for e in range(first, min(last, len(row))):
            if row[e] < 0 and free:
                row[e] = free.pop(0)
                refs[row[e]] = 1
    return table, refs


def fork(table, lengths, refs, parents, page_size):
    table, new_refs = _clean(table, len(refs)), list(refs)
    columns = len(table[0]) if table else 0
    free = [i for i, r in enumerate(refs) if r <= 0]
    children, held, source, target = [], [], [], []
    for parent in parents:
        row, n, pair = [-1] * columns, 0, (-1, -1)
        if 0 <= parent < len(table):
            n = min(max(lengths[parent], 0), columns * page_size)
            for e in range(n // page_size):
                row[e] = table[parent][e]
            if n % page_size and table[parent][n // page_size] >= 0 and free:
                pair = (table[parent][n // page_size], free.pop(0))
                row[n // page_size] = pair[1]
                new_refs[pair[1]] = 1
        children.append(row), held.append(n), source.append(pair[0]), target.append(pair[1])
    for row, n in zip(children, held):
        for e in row[:n // page_size]:
            if e >= 0:
                new_refs[e] += 1
    return children, held, new_refs, source, target


def free(table, refs, first, last):
    table, refs = _clean(table, len(refs)), list(refs)
    for b, row in enumerate(table):
        for e in range(max(first[b], 0), min(last[b], len(row))):
            if row[e] >= 0:
                refs[row[e]] -= 1
                row[e] = -1
    return table, refs


def compact(table, refs):
    table, old = _clean(table, len(refs)), list(refs)
    live = [i for i, r in enumerate(refs) if r > 0]
    count = len(live)
    pairs = list(zip([i for i in live if i >= count], [i for i in range(count) if refs[i] <= 0]))
    moved, new = dict(pairs), [r if i < count else 0 for i, r in enumerate(refs)]
    for s, t in pairs:
        new[t] = old[s]
    table = [[moved.get(e, e) if e >= 0 and old[e] > 0 else -1 for e in row] for row in table]
    fill = [-1] * (len(refs) // 2 - len(pairs))
    return table, new, [s for s, _ in pairs] + fill, [t for _, t in pairs] + fill
