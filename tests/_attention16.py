"""Plain attention in 64 bits, and how far 16-bit attention may be from it.

Weights are rounded to the cache's type, at most u = eps / 2 of each, and the output once more, u of itself.  So an
output is within u (sum of w |v|) + u |o| of the exact one, w the normalised weights; 1/16 of the first term is allowed
on top for scores, exponentials and sums in 32 bits (2^-12 of the weights for scores up to 2^6).  float16 has no value
below 2^-24 (relative to the row's largest weight, 1): 2^-25 of each visible |v|, and of an output, come on top.
"""

from __future__ import annotations

import torch


def attention64(q, k, v, scale):
    """(out, bound) of the last q.shape[0] tokens of k and v, causal; q [n, Hq, D], k and v [m, H, D], CPU."""

    n, m, group = q.shape[0], k.shape[0], q.shape[1] // k.shape[1]
    u = torch.finfo(q.dtype).eps / 2
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    qd = q.double().transpose(0, 1)
    kd, vd = (x.double().transpose(0, 1).repeat_interleave(group, 0) for x in (k, v))
    if m == 0 or n == 0:
        return torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    hidden = torch.arange(m)[None, :] > torch.arange(n)[:, None] + (m - n)
    scores = (qd @ kd.transpose(1, 2) * scale).masked_fill(hidden, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    w = torch.exp(scores - torch.where(top == -torch.inf, torch.zeros_like(top), top))
    w = torch.where(hidden, torch.zeros_like(w), w)
    total = w.sum(-1, keepdim=True)
    w = torch.where(total == 0, torch.zeros_like(w), w / total)

    def times(weights, values):  # masked places weigh nothing, whatever they hold
        if values.isfinite().all():
            return weights @ values
        out = torch.zeros(*weights.shape[:2], values.shape[2], dtype=torch.float64)
        for t in range(m):
            seen = ~hidden[:, t]
            out[:, seen] += weights[:, seen, t, None] * values[:, t, None, :]
        return out

    out = times(w, vd)
    spread = times(w, vd.abs())
    bound = u * (1 + 1 / 16) * spread + u * out.abs() + tiny * (1 + times((~hidden).double().expand_as(w), vd.abs()))
    return out.transpose(0, 1), bound.transpose(0, 1)


def packed_attention64(q, k, v, cu_q, cu_k, scale):
    """The same for packed sequences; rows outside them are 0."""

    out, bound = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(2))
    for i in range(len(cu_q) - 1):
        rows, keys = slice(cu_q[i], cu_q[i + 1]), slice(cu_k[i], cu_k[i + 1])
        out[rows], bound[rows] = attention64(q[rows], k[keys], v[keys], scale)
    return out, bound


def assert_within(got, want, bound, label=""):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (label, got.shape, want.shape)
    same = (got == want) | (got.isnan() & want.isnan())  # infinities and NaN
    off = torch.where(same, torch.zeros_like(want), (got - want).abs() - bound)
    assert not (off > 0).any() and not (got.isnan() ^ want.isnan()).any(), (
        f"{label}: {int((~(off <= 0)).sum())} of {off.numel()} outside, the worst by {off.nan_to_num(torch.inf).max().item():.3e}")


def offsets(lens, start=0):
    cu = [start]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu
