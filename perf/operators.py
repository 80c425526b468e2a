"""Workloads for measuring the serving and sink-attention operators: attention with a sliding window and sinks
(forward, and forward with backward), one-token attention over a paged key-value cache, writing new tokens into the
pages, and forking, compacting, freeing and reserving pages.

`run` computes each operator in plain torch operations in 32 bits, or, with `own` set, through the public functions of
the package. `exact` states the same definitions once more in 64 bits. Nothing here synchronises with the device."""
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parent.parent / "zig-flash-attn_b200")


def _zigfa():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import zigfa

    return zigfa


# ------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # A prompt of 8 k tokens on its way into a model with a window of 1024 tokens and four sinks (prefill).
        dict(name="sink prefill 8k d128", kind="sink", backward=False, packed=False, batch=1, shortest=8192, longest=8192,
             extra=0, hq=32, hkv=8, d=128, left=1023, sink=4),
        # A training step of the same layer: two rows of 4 k tokens, forward and gradients.
        dict(name="sink train 2x4k d128", kind="sink", backward=True, packed=False, batch=2, shortest=4096, longest=4096,
             extra=0, hq=16, hkv=4, d=128, left=511, sink=4),
        # A packed batch of documents of odd lengths, three query heads per key head, the training step.
        dict(name="sink train packed d64", kind="sink", backward=True, packed=True, batch=5, shortest=37, longest=1501,
             extra=0, hq=6, hkv=2, d=64, left=200, sink=17),
        # The first answer tokens of one short conversation: nothing but latency.
        dict(name="decode 1x400", kind="decode", batch=1, shortest=400, longest=400, hq=32, hkv=8, d=128, page=16, left=-1,
             sink=0),
        # A serving batch of conversations of very different lengths, full attention.
        dict(name="decode 64 ragged 8k", kind="decode", batch=64, shortest=100, longest=8192, hq=32, hkv=8, d=128, page=64,
             left=-1, sink=0),
        # Two very long contexts: the cache is split over the whole GPU.
        dict(name="decode 2x128k", kind="decode", batch=2, shortest=125001, longest=131072, hq=16, hkv=2, d=128, page=16,
             left=-1, sink=0),
        # Many bounded conversations: window and sinks, one key head, the pages in between already given back.
        dict(name="decode window 128x30k d64", kind="decode", batch=128, shortest=2000, longest=30000, hq=8, hkv=1, d=64,
             page=16, left=1023, sink=16),
        # The write of one decoding step.
        dict(name="append 64x1", kind="append", packed=False, batch=64, shortest=100, longest=8000, new=1, hkv=8, d=128,
             page=16),
        # The write of a batch of prompts, behind what their sequences hold already.
        dict(name="append prompts 8x4k", kind="append", packed=True, batch=8, shortest=0, longest=3000, new=4096, hkv=8,
             d=128, page=64),
        # Sixteen conversations forked into four continuations each; the partly filled pages of two layers are copied.
        dict(name="fork 16 to 64", kind="fork", batch=16, children=64, shortest=501, longest=4000, spare=400, hkv=8, d=128,
             page=64, layers=2),
        # Defragmentation of a large pool before its tail is handed back: two layers are moved.
        dict(name="compact 16k pages", kind="compact", batch=256, pages=16384, live=0.6, hkv=8, d=128, page=16, layers=2),
        # The bookkeeping of one decoding step of a busy server: pages that left the window and those of finished
        # sequences are given back, the next tokens get theirs.
        dict(name="turnover 512 of 64k pages", kind="turnover", batch=512, pages=65536, shortest=17, longest=8000, hkv=8,
             d=128, page=16, left=1023, sink=16),
    ]


def _log_int(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    kind = rng.choice(["sink", "sink", "decode", "decode", "decode", "append", "fork", "compact", "turnover"])
    hkv = rng.choice([1, 2, 3, 4, 8])
    if kind == "sink":
        hq = hkv * rng.choice([1, 2, 3, 4, 8])
        longest = _log_int(rng, 60, 4000)
        packed = rng.random() < 0.5
        batch = max(1, min(_log_int(rng, 1, 16), 40000000 // (longest * longest * hq) + 1))
        return dict(kind=kind, backward=rng.random() < 0.6, packed=packed, batch=batch,
                    shortest=rng.randint(0, longest) if packed else longest, longest=longest,
                    extra=rng.choice([0, 0, rng.randint(1, 300)]), hq=hq, hkv=hkv, d=rng.choice([64, 72, 96, 128]),
                    left=_log_int(rng, 1, 1500), sink=_log_int(rng, 1, 300))
    if kind == "decode":
        hq = hkv * rng.choice([1, 2, 3, 4, 6, 8, 16])
        d = rng.choice([64, 72, 96, 128, 128, 256])
        longest = _log_int(rng, 20, 100000)
        batch = max(1, min(_log_int(rng, 1, 200), 200000000 // (longest * hkv * d)))
        windowed = rng.random() < 0.4
        return dict(kind=kind, batch=batch, shortest=rng.randint(0, longest), longest=longest, hq=hq, hkv=hkv, d=d,
                    page=rng.choice([8, 16, 16, 24, 32, 64, 128]), left=_log_int(rng, 20, 3000) if windowed else -1,
                    sink=_log_int(rng, 1, 100) if windowed else 0)
    if kind == "append":
        new = _log_int(rng, 1, 3000)
        return dict(kind=kind, packed=rng.random() < 0.5, batch=max(1, min(_log_int(rng, 1, 256), 16000 // new)),
                    shortest=0, longest=_log_int(rng, 10, 5000), new=new, hkv=hkv, d=rng.choice([64, 72, 96, 128, 256]),
                    page=rng.choice([8, 16, 24, 32, 64, 128]))
    if kind == "fork":
        batch = _log_int(rng, 1, 64)
        return dict(kind=kind, batch=batch, children=_log_int(rng, 1, 200), shortest=1, longest=_log_int(rng, 20, 4000),
                    spare=rng.randint(100, 500), hkv=hkv, d=rng.choice([64, 96, 128]), page=rng.choice([8, 16, 24, 32, 64]),
                    layers=rng.randint(1, 3))
    if kind == "compact":
        return dict(kind=kind, batch=_log_int(rng, 1, 500), pages=_log_int(rng, 50, 6000),
                    live=round(rng.uniform(0.1, 0.95), 3), hkv=hkv, d=rng.choice([64, 96, 128]),
                    page=rng.choice([8, 16, 24, 32]), layers=rng.randint(1, 2))
    return dict(kind=kind, batch=_log_int(rng, 1, 500), pages=_log_int(rng, 3000, 60000), shortest=1,
                longest=_log_int(rng, 50, 8000), hkv=hkv, d=128, page=rng.choice([8, 16, 24, 32, 64]),
                left=_log_int(rng, 20, 3000), sink=_log_int(rng, 1, 100))


# ------------------------------------------------------------------------------------------------------ the inputs
def _spread(count, shortest, longest, salt=0):
    """`count` lengths between shortest and longest: the same for every seed, so that work() knows them."""
    return [shortest + (((i + 1 + salt) * 2654435761) % 4294967296) * (longest - shortest + 1) // 4294967296 for i in range(count)]


def _pages_of(length, page):
    return -(-length // page)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cu(lengths):
    return _int([0, *np.cumsum(lengths).tolist()])


def _tables(lengths, page, columns, num_pages, generator):
    """Block tables that hold `lengths` tokens on pages scattered over the pool, and the reference counts."""
    order = torch.randperm(num_pages, generator=generator, device="cuda").to(torch.int32)
    counts = torch.tensor([_pages_of(n, page) for n in lengths], device="cuda")
    starts = counts.cumsum(0) - counts
    entry = torch.arange(columns, device="cuda")
    taken = entry[None] < counts[:, None]
    table = torch.where(taken, order[((starts[:, None] + entry[None]) * taken).long()], -1).to(torch.int32)
    refs = torch.zeros(num_pages, dtype=torch.int32, device="cuda")
    refs[table[taken].long()] = 1
    return table, refs


def _turnover_lengths(case):
    """Lengths of a busy server's sequences, as many as the pool has pages for."""
    lengths, left = [], case["pages"] - case["batch"]
    for n in _spread(case["batch"], case["shortest"], case["longest"]):
        n = min(n, max(left, 0) * case["page"])
        left -= _pages_of(n, case["page"])
        lengths.append(n)
    return lengths


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=generator, device="cuda", dtype=torch.bfloat16)

    kind, state = case["kind"], dict(case=case)
    if kind == "sink":
        lengths_q = _spread(case["batch"], case["shortest"], case["longest"])
        lengths_k = [n + case["extra"] for n in lengths_q]
        if case["packed"]:
            lead_q, lead_k = (sum(lengths_q),), (sum(lengths_k),)
            state.update(cu_q=_cu(lengths_q), cu_k=_cu(lengths_k), longest_q=max(lengths_q), longest_k=max(lengths_k))
        else:
            lead_q, lead_k = (case["batch"], lengths_q[0]), (case["batch"], lengths_k[0])
        q, k, v = randn(*lead_q, case["hq"], case["d"]), randn(*lead_k, case["hkv"], case["d"]), randn(*lead_k, case["hkv"], case["d"])
        state.update(q=q, k=k, v=v)
        if case["backward"]:
            for x in (q, k, v):
                x.requires_grad_(True)
            state["dout"] = randn(*lead_q, case["hq"], case["d"])
        return state
    page, hkv, d = case["page"], case["hkv"], case["d"]
    if kind in ("decode", "append"):
        held = _spread(case["batch"], case["shortest"], case["longest"])
        new = _spread(case["batch"], 0, case["new"], 7) if kind == "append" and case["packed"] else [case.get("new", 0)] * case["batch"]
        total = [h + n for h, n in zip(held, new)]
        columns = max(1, max(_pages_of(n, page) for n in total))
        num_pages = max(1, sum(_pages_of(n, page) for n in total)) + 3
        table, _ = _tables(total, page, columns, num_pages, generator)
        state.update(table=table, seqlens=_int(held), k_cache=randn(num_pages, page, hkv, d), v_cache=randn(num_pages, page, hkv, d))
        if kind == "decode":
            if case["left"] >= 0:  # what lies between the sinks and the window has been given back
                entry = torch.arange(columns, device="cuda")[None]
                first = _pages_of(case["sink"], page)
                last = ((state["seqlens"] - 1 - case["left"]).clamp(min=0) // page)[:, None]
                state["table"] = torch.where((entry >= first) & (entry < last), -1, table).to(torch.int32)
            state["q"] = randn(case["batch"], case["hq"], d)
        elif case["packed"]:
            state.update(cu=_cu(new), k=randn(sum(new), hkv, d), v=randn(sum(new), hkv, d))
        else:
            state.update(cu=None, k=randn(case["batch"], case["new"], hkv, d), v=randn(case["batch"], case["new"], hkv, d))
        return state
    if kind == "fork":
        lengths = _spread(case["batch"], case["shortest"], case["longest"])
        num_pages = sum(_pages_of(n, page) for n in lengths) + case["spare"]
        table, refs = _tables(lengths, page, _pages_of(max(lengths), page) + 4, num_pages, generator)
        parents = torch.randint(0, case["batch"], (case["children"],), generator=generator, device="cuda").to(torch.int32)
        state.update(table=table, refs=refs, seqlens=_int(lengths), parents=parents)
    elif kind == "compact":
        num_pages = case["pages"]
        each = int(num_pages * case["live"]) // case["batch"]
        table, refs = _tables([each * page] * case["batch"], page, each + 1, num_pages, generator)
        state.update(table=table, refs=refs)
    else:
        lengths = _turnover_lengths(case)
        table, refs = _tables(lengths, page, _pages_of(case["longest"], page) + 2, case["pages"], generator)
        seqlens = _int(lengths)
        finished = torch.rand(case["batch"], generator=generator, device="cuda") < 0.1
        state.update(table=table, refs=refs, seqlens=seqlens, finished=finished, new_tokens=torch.ones_like(seqlens))
    if "layers" in case:
        state["caches"] = [(randn(num_pages, page, hkv, d), randn(num_pages, page, hkv, d)) for _ in range(case["layers"])]
    return state


# ------------------------------------------------------------------------------------------------------ the plain forms
def _softmax(scores, visible):
    """(probabilities, log-sum-exp) over the last axis; a row without a visible entry gets zeros and -inf."""
    scores = torch.where(visible, scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = weights.sum(-1, keepdim=True)
    return weights / torch.where(total == 0, 1.0, total), (top + torch.log(total))[..., 0]


def _padded(x, cu, longest):
    """Packed (total, heads, d) as (batch, longest, heads, d) in 32 bits, with the places taken from it."""
    place = cu[:-1, None].long() + torch.arange(longest, device=x.device)[None]
    inside = place < cu[1:, None]
    return torch.where(inside[..., None, None], x[place.clamp(max=max(x.shape[0] - 1, 0))].float(), 0.0), inside


def _plain_sink(state):
    case = state["case"]
    q, k, v, dout = (state[n].detach() if n in state else None for n in ("q", "k", "v", "dout"))
    scale, group = case["d"] ** -0.5, case["hq"] // case["hkv"]
    if case["packed"]:
        (q, in_q), (k, in_k), (v, _) = _padded(q, state["cu_q"], state["longest_q"]), _padded(k, state["cu_k"], state["longest_k"]), _padded(v, state["cu_k"], state["longest_k"])
        dout = _padded(dout, state["cu_q"], state["longest_q"])[0] if dout is not None else None
        lq, lk = (state["cu_q"].diff()[:, None, None], state["cu_k"].diff()[:, None, None])
    else:
        q, k, v, dout = (x.float() if x is not None else None for x in (q, k, v, dout))
        lq, lk = q.shape[1], k.shape[1]
    row = torch.arange(q.shape[1], device="cuda")[None, :, None] + (lk - lq)
    column = torch.arange(k.shape[1], device="cuda")[None, None, :]
    visible = (column <= row) & (column < lk) & ((column >= row - case["left"]) | (column < case["sink"]))

    def grouped(x):  # (batch, rows, heads, d) -> (batch, key heads, group * rows, d)
        return x.unflatten(2, (case["hkv"], -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)

    def ungrouped(x, heads):  # the reverse
        return x.unflatten(2, (heads // case["hkv"], -1)).permute(0, 3, 1, 2, 4).flatten(2, 3)

    visible = visible[:, None].expand(-1, -1, q.shape[1], -1).repeat(1, 1, group, 1)
    qg, kg, vg = grouped(q), grouped(k), grouped(v)
    p, lse = _softmax(qg @ kg.transpose(-1, -2) * scale, visible)
    out = p @ vg
    results = [ungrouped(out, case["hq"])]
    if dout is not None:
        dg = grouped(dout)
        dv = p.transpose(-1, -2) @ dg
        ds = p * (dg @ vg.transpose(-1, -2) - (out * dg).sum(-1, keepdim=True)) * scale
        results += [ungrouped(ds @ kg, case["hq"]), ungrouped(ds.transpose(-1, -2) @ qg, case["hkv"]), ungrouped(dv, case["hkv"])]
    if case["packed"]:
        results = [x[inside] for x, inside in zip(results, (in_q, in_q, in_k, in_k))]
    results = [x.to(torch.bfloat16) for x in results]
    if dout is not None:
        return results
    lse = lse.unflatten(2, (group, -1)).flatten(1, 2)  # (batch, query heads, rows)
    return results + [lse.transpose(1, 2)[in_q].transpose(0, 1).contiguous() if case["packed"] else lse]


def _plain_decode(state):
    case, table, lengths = state["case"], state["table"], state["seqlens"]
    position = torch.arange(table.shape[1] * case["page"], device="cuda")
    entry = table.long()[:, position // case["page"]]
    row = (lengths - 1)[:, None]
    visible = (position <= row) & (entry >= 0)
    if case["left"] >= 0:
        visible = visible & ((position >= row - case["left"]) | (position < case["sink"]))
    k, v = (torch.where(visible[..., None, None], cache[entry.clamp(min=0), position % case["page"]].float(), 0.0)
            for cache in (state["k_cache"], state["v_cache"]))
    q = state["q"].float().unflatten(1, (case["hkv"], -1))
    p, lse = _softmax(q @ k.permute(0, 2, 3, 1) * case["d"] ** -0.5, visible[:, None, None])
    return (p @ v.permute(0, 2, 1, 3)).flatten(1, 2).to(torch.bfloat16), lse.flatten(1, 2)


def _plain_append(state):
    case, cu = state["case"], state["cu"]
    if cu is None:
        k, v = state["k"].flatten(0, 1), state["v"].flatten(0, 1)
        sequence = torch.arange(case["batch"], device="cuda").repeat_interleave(case["new"])
        offset = torch.arange(case["new"], device="cuda").repeat(case["batch"])
    else:
        k, v = state["k"], state["v"]
        token = torch.arange(k.shape[0], device="cuda", dtype=torch.int32)
        sequence = torch.bucketize(token, cu[1:], right=True)
        offset = token - cu[sequence]
    position = (state["seqlens"][sequence] + offset).long()
    entry = state["table"][sequence, position // case["page"]].long()
    state["k_cache"][entry, position % case["page"]] = k
    state["v_cache"][entry, position % case["page"]] = v
    return state["k_cache"], state["v_cache"]


def _plain_free_pages(refs):
    """The free pages, lowest first, behind them num_pages for 'none'."""
    page = torch.arange(refs.shape[0], device="cuda")
    return torch.sort(torch.where(refs <= 0, page, refs.shape[0])).values


def _plain_handout(refs, wanted):
    """A page for each True of `wanted`, in its order, lowest free pages first; -1 where none is left. New references too."""
    free = _plain_free_pages(refs)
    rank = wanted.flatten().long().cumsum(0) - 1
    given = torch.where(wanted.flatten() & (rank < free.shape[0]), free[rank.clamp(0, free.shape[0] - 1)], refs.shape[0])
    refs = torch.cat([refs, refs.new_zeros(1)]).index_fill(0, given, 1)[:-1]
    return torch.where(given < refs.shape[0], given, -1).to(torch.int32).view(wanted.shape), refs


def _plain_copy(caches, source, target):
    kept = target >= 0
    many = caches[0][0].shape[0]
    # A pair of -1 copies a page onto itself, so that the shapes hold without asking the device how many pairs there are.
    fallback = torch.arange(source.shape[0], device="cuda") % many
    if source.shape[0]:
        filled = torch.where(kept, source, source[:1].clamp(min=0)).long()
        place = torch.where(kept, target, target[:1].clamp(min=0)).long()
        none = ~kept[:1].expand_as(kept)
        filled, place = torch.where(none, fallback, filled), torch.where(none, fallback, place)
        for pair in caches:
            for cache in pair:
                cache[place] = cache[filled]
    return caches


def _plain_fork(state):
    case, table, refs = state["case"], state["table"], state["refs"]
    parents = state["parents"].long()
    lengths = state["seqlens"][parents]
    entry = torch.arange(table.shape[1], device="cuda")[None]
    full, rest = (lengths // case["page"])[:, None], (lengths % case["page"])[:, None]
    rows = table[parents]
    shared = (entry < full) & (rows >= 0)
    shares = torch.zeros(refs.shape[0] + 1, dtype=torch.int32, device="cuda")
    shares.index_add_(0, torch.where(shared, rows, refs.shape[0]).flatten().long(), torch.ones_like(rows).flatten())
    partial = (entry == full) & (rest > 0) & (rows >= 0)
    source = torch.where(partial, rows, -1).amax(1)
    target, refs = _plain_handout(refs, source >= 0)
    child = torch.where(shared, rows, torch.where(partial, target[:, None], -1)).to(torch.int32)
    refs = refs + shares[:-1]
    source = torch.where(target >= 0, source, -1)
    # Pairs without a copy go to the end as far as the copy is concerned: an order by 'has none' that keeps the rest.
    order = torch.sort((target < 0).to(torch.int8), stable=True).indices
    caches = _plain_copy(state["caches"], source[order], target[order])
    return child, lengths, refs, source.to(torch.int32), target, caches


def _plain_compact(state):
    table, refs = state["table"], state["refs"]
    many = refs.shape[0]
    live = refs > 0
    page = torch.arange(many, device="cuda")
    count = live.sum()
    moves = live & (page >= count)
    pairs = many // 2
    source = torch.sort(torch.where(moves, page, many)).values[:pairs]
    target = torch.sort(torch.where(~live & (page < count), page, many)).values[:pairs]
    to = torch.cat([page, page.new_full((1,), -1)])
    to[source] = target
    to[-1] = -1
    bad = (table < 0) | ~live[table.clamp(min=0).long()]
    moved = torch.where(bad, -1, to[table.clamp(min=0).long()]).to(torch.int32)
    packed = torch.where(page < count, refs, 0)
    packed = torch.cat([packed, packed.new_zeros(1)])
    packed[target] = torch.cat([refs, refs.new_zeros(1)])[source]
    source, target = (torch.where(x < many, x, -1).to(torch.int32) for x in (source, target))
    return moved, packed[:-1].contiguous(), source, target, _plain_copy(state["caches"], source, target)


def _plain_turnover(state):
    case, table, refs, lengths = state["case"], state["table"], state["refs"], state["seqlens"]
    first, last, kept, new = _turnover_ranges(state)
    entry = torch.arange(table.shape[1], device="cuda")[None]
    freed = (entry >= first[:, None]) & (entry < last[:, None])
    gone = torch.zeros(refs.shape[0] + 1, dtype=torch.int32, device="cuda")
    gone.index_add_(0, torch.where(freed & (table >= 0), table, refs.shape[0]).flatten().long(), torch.ones_like(table).flatten())
    refs = refs - gone[:-1]
    table = torch.where(freed, -1, table)
    need = (kept + new + case["page"] - 1) // case["page"]
    have = (kept + case["page"] - 1) // case["page"]
    wanted = (entry >= have[:, None]) & (entry < need[:, None]) & (table < 0)
    given, refs = _plain_handout(refs, wanted)
    return torch.where(wanted, given, table), refs


def _turnover_ranges(state):
    """What the program asks for: entries [first, last) to give back, lengths that stay, tokens to come."""
    case, lengths = state["case"], state["seqlens"]
    behind = (lengths - case["left"]).clamp(min=0) // case["page"]  # pages that the next token no longer sees
    first = torch.where(state["finished"], 0, _pages_of(case["sink"], case["page"])).to(torch.int32)
    last = torch.where(state["finished"], state["table"].shape[1], behind).to(torch.int32)
    kept = torch.where(state["finished"], 0, lengths)
    return first, last, kept, state["new_tokens"]


# ------------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        plain = {"sink": _plain_sink, "decode": _plain_decode, "append": _plain_append, "fork": _plain_fork,
                 "compact": _plain_compact, "turnover": _plain_turnover}
        return plain[kind](state)
    zigfa = _zigfa()
    if kind == "sink":
        options = dict(sink_size=case["sink"], causal=True, window_size=(case["left"], -1))
        q, k, v = state["q"], state["k"], state["v"]
        if case["packed"]:
            arguments = (q, k, v, state["cu_q"], state["cu_k"], state["longest_q"], state["longest_k"])
            function = zigfa.flash_attn_varlen_sink_func
        else:
            arguments, function = (q, k, v), zigfa.flash_attn_sink_func
        if not case["backward"]:
            return list(function(*arguments, return_attn_probs=True, **options))
        out = function(*arguments, **options)
        return [out.detach(), *torch.autograd.grad(out, (q, k, v), state["dout"])]
    if kind == "decode":
        return zigfa.flash_attn_paged_func(state["q"], state["k_cache"], state["v_cache"], state["table"], state["seqlens"],
                                           window_size=(case["left"], -1), sink_size=case["sink"], return_attn_probs=True)
    if kind == "append":
        zigfa.append_paged_kv(state["k"], state["v"], state["k_cache"], state["v_cache"], state["table"], state["seqlens"],
                              state["cu"])
        return state["k_cache"], state["v_cache"]
    if kind == "fork":
        child, lengths, refs, source, target = zigfa.fork_kv_pages(state["table"], state["seqlens"], state["refs"],
                                                                   state["parents"], case["page"])
        for k_cache, v_cache in state["caches"]:
            zigfa.copy_kv_pages(k_cache, v_cache, source, target)
        return child, lengths, refs, source, target, state["caches"]
    if kind == "compact":
        table, refs, source, target = zigfa.compact_kv_pages(state["table"], state["refs"])
        for k_cache, v_cache in state["caches"]:
            zigfa.copy_kv_pages(k_cache, v_cache, source, target)
        return table, refs, source, target, state["caches"]
    first, last, kept, new = _turnover_ranges(state)
    table, refs = zigfa.free_kv_pages(state["table"], state["refs"], first, last)
    return zigfa.reserve_kv_pages(table, kept, new, refs, case["page"])


# ------------------------------------------------------------------------------------------------------ what it costs
def _visible_pairs(lq, lk, left, sink):
    row = np.arange(lq) + (lk - lq)
    low, high = np.maximum(row - left, 0) if left >= 0 else 0 * row, row + 1
    return int(np.where(high > 0, high - low + np.minimum(np.minimum(sink, low), high), 0).sum())


def work(case):
    kind, d = case["kind"], case["d"]
    if kind == "sink":
        lengths = _spread(case["batch"], case["shortest"], case["longest"])
        pairs = sum(_visible_pairs(n, n + case["extra"], case["left"], case["sink"]) for n in lengths)
        rows_q, rows_k = sum(lengths), sum(lengths) + case["extra"] * case["batch"]
        q_bytes, k_bytes = rows_q * case["hq"] * d * 2, rows_k * case["hkv"] * d * 2
        if case["backward"]:  # q, k, v, dout in; out, dq, dk, dv out
            return dict(bytes=max(1, 4 * q_bytes + 4 * k_bytes), flops=14 * d * pairs * case["hq"])
        return dict(bytes=max(1, 2 * q_bytes + 2 * k_bytes + 4 * rows_q * case["hq"]), flops=4 * d * pairs * case["hq"])
    token = case["hkv"] * d * 2  # bytes of one token in one cache
    if kind == "decode":
        keys = sum(_visible_pairs(1, n, case["left"], case["sink"]) for n in _spread(case["batch"], case["shortest"], case["longest"]) if n)
        rows = case["batch"] * case["hq"]
        return dict(bytes=2 * keys * token + rows * (4 * d + 4) + 4 * keys // case["page"], flops=4 * d * keys * case["hq"])
    if kind == "append":
        new = sum(_spread(case["batch"], 0, case["new"], 7)) if case["packed"] else case["batch"] * case["new"]
        return dict(bytes=max(1, 4 * new * token), flops=0)
    if kind == "fork":
        lengths = _spread(case["batch"], case["shortest"], case["longest"])
        many = sum(_pages_of(n, case["page"]) for n in lengths) + case["spare"]
        row = 4 * (_pages_of(max(lengths), case["page"]) + 4)
        return dict(bytes=8 * many + 2 * case["children"] * row + 4 * case["layers"] * case["children"] * case["page"] * token, flops=0)
    if kind == "compact":
        each = int(case["pages"] * case["live"]) // case["batch"]
        live = each * case["batch"]
        moves = live * (case["pages"] - live) // case["pages"]  # what is expected of pages scattered at random
        return dict(bytes=8 * case["pages"] + 8 * case["batch"] * (each + 1) + 4 * case["layers"] * moves * case["page"] * token, flops=0)
    return dict(bytes=8 * case["pages"] + 8 * case["batch"] * (_pages_of(case["longest"], case["page"]) + 2), flops=0)


# ------------------------------------------------------------------------------------------------------ in 64 bits
def _exact_head(q, k, v, dout, seen, scale):
    """One head of one sequence: rows x d against keys x d, with the mask as a matrix."""
    e = torch.exp2((q @ k.T * (scale * 1.4426950408889634)).masked_fill(~seen, -torch.inf))
    z = e.sum(1)
    some = z > 0
    p = e / torch.where(some, z, 1)[:, None]
    out = p @ v
    if dout is None:
        return out, z.log()
    pull = dout @ v.T
    ds = p * (pull - (p * pull).sum(1, keepdim=True))
    return out, ds @ k * scale, ds.T @ q * scale, p.T @ dout


def _exact_sink(case, state):
    q, k, v = (state[n].detach().double() for n in "qkv")
    dout = state["dout"].double() if case["backward"] else None
    lengths = _spread(case["batch"], case["shortest"], case["longest"])
    answers = [torch.zeros_like(q)] + ([torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)] if case["backward"] else [])
    if not case["backward"]:
        answers.append(torch.zeros(*((case["hq"], q.shape[0]) if case["packed"] else (case["batch"], case["hq"], q.shape[1])), dtype=torch.float64, device="cuda"))
    at = 0
    for b, n in enumerate(lengths):
        m = n + case["extra"]
        i, j = torch.arange(n, device="cuda")[:, None] + case["extra"], torch.arange(m, device="cuda")[None]
        seen = (j <= i) & ((i - j <= case["left"]) | (j < case["sink"]))
        for h in range(case["hq"]):
            g = h * case["hkv"] // case["hq"]
            if case["packed"]:
                rows, keys = (slice(at, at + n), h), (slice(at + b * case["extra"], at + b * case["extra"] + m), g)
            else:
                rows, keys = (b, slice(None), h), (b, slice(None), g)
            got = _exact_head(q[rows], k[keys], v[keys], None if dout is None else dout[rows], seen, case["d"] ** -0.5)
            answers[0][rows] = got[0]
            if case["backward"]:
                answers[1][rows] = got[1]
                answers[2][keys] += got[2]
                answers[3][keys] += got[3]
            elif case["packed"]:
                answers[1][h, at:at + n] = got[1]
            else:
                answers[1][b, h] = got[1]
        at += n
    return answers


def _exact_decode(case, state):
    out = torch.zeros(case["batch"], case["hq"], case["d"], dtype=torch.float64, device="cuda")
    lse = torch.full((case["batch"], case["hq"]), -torch.inf, dtype=torch.float64, device="cuda")
    table, group = state["table"].tolist(), case["hq"] // case["hkv"]
    for b, n in enumerate(_spread(case["batch"], case["shortest"], case["longest"])):
        seen = [j for j in range(n) if case["left"] < 0 or n - 1 - j <= case["left"] or j < case["sink"]]
        if not seen:
            continue
        where = torch.tensor([table[b][j // case["page"]] * case["page"] + j % case["page"] for j in seen], device="cuda")
        k, v = (state[c].flatten(0, 1)[where].double() for c in ("k_cache", "v_cache"))
        for g in range(case["hkv"]):
            heads = slice(g * group, (g + 1) * group)
            s = state["q"][b, heads].double() @ k[:, g].T * case["d"] ** -0.5
            lse[b, heads] = torch.logsumexp(s, 1)
            out[b, heads] = torch.exp(s - lse[b, heads, None]) @ v[:, g]
    return out, lse


def _exact_copies(caches, pairs):
    moved = []
    for pair in caches:
        moved.append([cache.double() for cache in pair])
        for cache, old in zip(moved[-1], pair):
            if pairs:
                source, target = (torch.tensor(x, device="cuda") for x in zip(*pairs))
                cache[target] = old[source].double()
    return moved


def _exact_append(case, state):
    table, held = state["table"].tolist(), state["seqlens"].tolist()
    cu = state["cu"].tolist() if case["packed"] else [i * case["new"] for i in range(case["batch"] + 1)]
    slots = [table[b][(held[b] + t) // case["page"]] * case["page"] + (held[b] + t) % case["page"]
             for b in range(case["batch"]) for t in range(cu[b + 1] - cu[b])]
    answers = []
    for cache, fresh in ((state["k_cache"], state["k"]), (state["v_cache"], state["v"])):
        whole = cache.double()
        whole.flatten(0, 1)[torch.tensor(slots, dtype=torch.long, device="cuda")] = fresh.reshape(-1, *fresh.shape[-2:]).double()
        answers.append(whole)
    return answers


def _exact_fork(case, state):
    table, refs, held = state["table"].tolist(), state["refs"].tolist(), state["seqlens"].tolist()
    free = [i for i, r in enumerate(refs) if r <= 0]
    child, lengths, sources, targets = [], [], [], []
    for parent in state["parents"].tolist():
        n, row = held[parent], [-1] * len(table[0])
        for e in range(n // case["page"]):
            row[e] = table[parent][e]
            refs[row[e]] += 1
        source = target = -1
        if n % case["page"] and free:
            source, target = table[parent][n // case["page"]], free.pop(0)
            row[n // case["page"]], refs[target] = target, 1
        child.append(row), lengths.append(n), sources.append(source), targets.append(target)
    pairs = [(s, t) for s, t in zip(sources, targets) if t >= 0]
    return _int(child), _int(lengths), _int(refs), _int(sources), _int(targets), _exact_copies(state["caches"], pairs)


def _exact_compact(case, state):
    table, refs = state["table"].tolist(), state["refs"].tolist()
    live = [i for i, r in enumerate(refs) if r > 0]
    holes = [i for i in range(len(live)) if refs[i] <= 0]
    pairs = list(zip([i for i in live if i >= len(live)], holes))
    to = dict(pairs)
    for s, t in pairs:
        refs[t], refs[s] = refs[s], 0
    table = [[to.get(e, e) for e in row] for row in table]
    fill = [(-1, -1)] * (len(refs) // 2 - len(pairs))
    sources, targets = zip(*(pairs + fill)) if pairs or fill else ((), ())
    return _int(table), _int(refs), _int(sources), _int(targets), _exact_copies(state["caches"], pairs)


def _exact_turnover(case, state):
    table, refs = state["table"].tolist(), state["refs"].tolist()
    first, last, kept, new = (x.tolist() for x in _turnover_ranges(state))
    for b, row in enumerate(table):
        for e in range(first[b], min(last[b], len(row))):
            if row[e] >= 0:
                refs[row[e]] -= 1
                row[e] = -1
    free = iter([i for i, r in enumerate(refs) if r <= 0])
    for b, row in enumerate(table):
        for e in range(_pages_of(kept[b], case["page"]), min(_pages_of(kept[b] + new[b], case["page"]), len(row))):
            if row[e] < 0:
                row[e] = next(free, -1)
                if row[e] >= 0:
                    refs[row[e]] = 1
    return _int(table), _int(refs)


def exact(case, seed):
    state = prepare(case, seed)
    forms = {"sink": _exact_sink, "decode": _exact_decode, "append": _exact_append, "fork": _exact_fork,
             "compact": _exact_compact, "turnover": _exact_turnover}
    with torch.no_grad():
        return forms[case["kind"]](case, state)
