"""float16: a first key that outweighs tens of thousands of others, whose weights together still count.

Weights are rounded to float16, whose values end at 2^-24, as 2^7 times themselves: each is off by at most u = 2^-11 of
itself or 2^-25 2^-7 of the row's largest.  With the bound of _attention16 (1/16 of u on top for 32-bit steps; the
output's own rounding, u of itself or 2^-25):

  |error| <= u (1 + 1/16) sum of w |v| + 2^-32 sum of |v| + u |o| + 2^-25
"""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from _helpers import require_gpu

pytestmark = pytest.mark.gpu

KEYS, TOP = 40000, 17.046875  # exp(-TOP) = 0.66 2^-24


def _values(kv_heads, dim):
    v = 0.5 + torch.rand(KEYS, kv_heads, dim, generator=torch.Generator().manual_seed(1))
    v[0] = 0
    return v.half()


def _want(v, rows, group):
    """The last ``rows`` tokens: key 0 scores TOP, the others 0."""

    light = torch.exp(torch.tensor(-TOP, dtype=torch.float64))
    sums = v.double().cumsum(0)[KEYS - rows:]  # (key 0's value is 0)
    seen = torch.arange(KEYS - rows + 1, KEYS + 1, dtype=torch.float64)[:, None, None]
    out = (light * sums / (1 + light * (seen - 1))).repeat_interleave(group, 1)
    u = 2.0 ** -11
    return out, u * (2 + 1 / 16) * out + 2.0 ** -32 * sums.repeat_interleave(group, 1) + 2.0 ** -25


def _check(got, rows, v, group):
    want, bound = _want(v, rows, group)
    off = (got.cpu().double() - want).abs()
    assert (off <= bound).all(), f"off by {(off / want).max():.3f} of the output"


def _queries(rows, heads, kv_heads, dim):
    q, k = torch.zeros(rows, heads, dim, dtype=torch.float16), torch.zeros(KEYS, kv_heads, dim, dtype=torch.float16)
    q[:, :, 0], k[0, :, 0] = 1, TOP
    return q, k


@pytest.mark.parametrize("rows,heads,kv_heads,dim", [(1, 4, 1, 128), (1024, 64, 8, 64), (300, 16, 8, 128)])
def test_packed(rows, heads, kv_heads, dim):
    require_gpu()
    from prism_infer.ops.prompt_attention import prompt_attention

    (q, k), v = _queries(rows, heads, kv_heads, dim), _values(kv_heads, dim)
    cq, ck = (torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (rows, KEYS))
    got = prompt_attention(q.cuda(), k.cuda(), v.cuda(), cq, num_heads=heads, num_kv_heads=kv_heads, scale=1.0, cu_seqlens_k=ck)
    _check(got, rows, v, heads // kv_heads)


@pytest.mark.parametrize("page", [16, 64])
def test_pages(page):
    require_gpu()
    from prism_infer.ops.paged_prefill import paged_prefill_attention

    rows, heads, kv_heads, dim = 1024, 64, 8, 64
    (q, k), v = _queries(rows, heads, kv_heads, dim), _values(kv_heads, dim)
    caches = [x.view(KEYS // page, page, kv_heads, dim).cuda() for x in (k, v)]
    context = SimpleNamespace(block_tables=torch.arange(KEYS // page, dtype=torch.int32, device="cuda")[None],
                              context_lens=torch.tensor([KEYS], dtype=torch.int32, device="cuda"),
                              cu_seqlens_q=torch.tensor([0, rows], dtype=torch.int32, device="cuda"))
    got = paged_prefill_attention(q.cuda(), *caches, context, num_heads=heads, num_kv_heads=kv_heads, scale=1.0)
    _check(got, rows, v, heads // kv_heads)
