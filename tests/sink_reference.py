"""64-bit statement of sliding-window attention with sinks and its gradients, with elementwise tolerances that add up the
roundings of the kernels."""
import torch

HALF_BF16, HALF_FP32 = 2.0**-8, 2.0**-24  # half a step, relative


def visible(lq, lk, left, right, sink, device="cuda"):
    row, column = torch.arange(lq, device=device)[:, None] + (lk - lq), torch.arange(lk, device=device)[None]
    mask = torch.ones(lq, lk, dtype=torch.bool, device=device)
    if left >= 0:
        mask &= (column >= row - left) | (column < sink)
    if right >= 0:
        mask &= column <= row + right
    return mask


def attention(q, k, v, mask, scale):
    """(out, lse) of one sequence in the type of its inputs: q (lq, heads_q, d), k and v (lk, heads_kv, d)."""
    group = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.einsum("qhd,khd->hqk", q, k) * scale
    s = s.masked_fill(~mask, float("-inf"))
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(lse == float("-inf"), 0.0, lse)[..., None])
    return torch.einsum("hqk,khd->qhd", p, v), lse


def with_tolerances(q, k, v, dout, mask, scale):
    """{name: (value, tolerance)} for out, lse and, with dout, dq, dk, dv of one sequence.

    A score is a sum of d products in FP32: at most d + 2 half steps of scale * sum |q k| each way (the last two for the
    scale and the subtraction of the maximum or the log-sum-exp), counted twice because a tensor core may cut instead of
    round. exp2 and the sums add a few half steps; a sum over n terms is a chain of n / 16 + 64 additions at most (16 products
    at a time). P and dS enter the products rounded to BF16, the outputs are rounded to BF16, and D = sum out * dout is
    formed from the rounded output."""
    q, k, v = q.double(), k.double(), v.double()
    heads_kv, group = k.shape[1], q.shape[1] // k.shape[1]
    out = torch.zeros_like(q)
    lse = torch.empty(q.shape[1], q.shape[0], dtype=torch.float64, device=q.device)
    results = {"out": (out, torch.zeros_like(q)), "lse": (lse, torch.zeros_like(lse))}
    if dout is not None:
        dout = dout.double()
        results.update({n: (torch.zeros_like(x), torch.zeros_like(x)) for n, x in (("dq", q), ("dk", k), ("dv", v))})
    d = q.shape[-1]
    chain_k, chain_q = (mask.shape[1] / 16 + 64) * 2 * HALF_FP32, (mask.shape[0] * group / 16 + 64) * 2 * HALF_FP32
    for h in range(q.shape[1]):
        g = h // group
        qh, kh, vh = q[:, h], k[:, g], v[:, g]
        s = (qh @ kh.T * scale).masked_fill(~mask, float("-inf"))
        lse[h] = torch.logsumexp(s, -1)
        shift = torch.where(lse[h] == float("-inf"), 0.0, lse[h])[:, None]
        p = torch.exp(s - shift)
        out[:, h] = p @ vh
        size = (qh.abs() @ kh.abs().T * abs(scale)).masked_fill(~mask, 0.0).amax(-1, keepdim=True) if mask.shape[1] else torch.zeros_like(shift)
        score = 2 * (d + 2) * HALF_FP32 * size + 8 * HALF_FP32
        results["lse"][1][h] = (score + chain_k + 4 * HALF_FP32 * shift.abs())[:, 0]
        relative = 2 * score + 4 * HALF_FP32 * shift.abs() + chain_k  # of a probability
        out_tol = HALF_BF16 * out[:, h].abs() + (p @ vh.abs()) * (HALF_BF16 + 2 * relative) * 1.01
        results["out"][1][:, h] = out_tol
        if dout is None:
            continue
        oh = dout[:, h]
        results["dv"][0][:, g] += p.T @ oh
        results["dv"][1][:, g] += (p * (HALF_BF16 + relative)).T @ oh.abs() * 1.01 + chain_q * (p.T @ oh.abs())
        delta = (out[:, h] * oh).sum(-1, keepdim=True)
        dp = oh @ vh.T
        ds = p * (dp - delta)
        dp_tol = 2 * d * HALF_FP32 * (oh.abs() @ vh.abs().T) + (out_tol * oh.abs()).sum(-1, keepdim=True) + d * HALF_FP32 * (
            out[:, h].abs() * oh.abs()).sum(-1, keepdim=True)
        ds_tol = p * dp_tol + (ds.abs() + p * dp_tol) * (HALF_BF16 + relative) * 1.01
        results["dq"][0][:, h] = ds @ kh * scale
        results["dq"][1][:, h] = abs(scale) * (ds_tol @ kh.abs() + chain_k * (ds.abs() @ kh.abs()))
        results["dk"][0][:, g] += ds.T @ qh * scale
        results["dk"][1][:, g] += abs(scale) * (ds_tol.T @ qh.abs() + chain_q * (ds.abs().T @ qh.abs()))
    for name in ("dq", "dk", "dv"):
        if name in results:
            results[name][1].add_(HALF_BF16 * results[name][0].abs() * 1.01)
    return results


def assert_within(name, got, want, tolerance, note=""):
    got = got.double()
    assert not torch.isnan(got).any(), (name, note)
    infinite = torch.isinf(want)
    assert torch.equal(torch.isinf(got), infinite), (name, note)
    excess = torch.where(infinite, 0.0, (got - want).abs() - tolerance)
    # values below BF16's normal range keep fewer bits: an absolute step of 2^-133
    assert excess.numel() == 0 or excess.max().item() <= 2.0**-133, (name, note, excess.max().item(), tolerance.max().item())
