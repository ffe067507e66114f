"""Decode of float16 queries over 4-bit caches whose keys are no float16 numbers, or only just: small, large, and both in one step."""

from __future__ import annotations

import math

import pytest
import torch

from _fp4 import Pool, attend, check
from _helpers import require_gpu
from test_gpu_fp4_attention import decode

pytestmark = pytest.mark.gpu
F16 = torch.float16


def expected(pool, q, scale):
    """Output and bound: `attend`'s, with scores that are sums of up to 256 exact products.

    A float16 query is the sum of two bf16 numbers there, the second at most 2^-8 of the first: 2 * 128 products, whose
    magnitudes sum to at most 1 + 2^-8 of sum |q| |k|.  `attend` counts 132 roundings of 2^-24 of that, 136 more cover it.
    """

    q = q.double().cpu()
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(q.shape[0]):
        k, v, keep = pool.rows(i)
        group = q.shape[1] // k.shape[1]
        for h in range(k.shape[1]):
            rows = slice(h * group, (h + 1) * group)
            seen = torch.ones(group, keep.numel(), dtype=torch.bool)
            out[i, rows], bound[i, rows] = attend(q[i, rows], k[:, h], v[:, h], scale, seen, 2.0 ** -16)
            more = 136 * 2.0 ** -24 * abs(scale) * (q[i, rows].abs() @ k[:, h].abs().t()).amax(1, keepdim=True)
            bound[i, rows] += 2 * more * (torch.softmax(scale * q[i, rows] @ k[:, h].t(), 1) @ v[:, h].abs())
    return out, bound


GEOMETRIES = [(32, 8, 128, 256), (16, 4, 64, 16), (8, 1, 128, 16), (16, 2, 128, 64), (16, 1, 128, 64), (16, 1, 64, 48), (3, 3, 64, 128)]


def make(heads, kv_heads, dim, page, low, high):
    """Keys with exponent bytes low to high, and a scale that makes scores of these a few units."""

    pool = Pool([300, 65, 1], page=page, kv_heads=kv_heads, dim=dim, seed=heads + dim, spread=False)
    g = torch.Generator().manual_seed(low)
    e = pool.ks.view(torch.uint8)
    e.copy_(torch.randint(low, high + 1, e.shape, generator=g))
    q = (torch.randn(3, heads, dim, generator=g) * 2.0 ** 8).to(F16)
    scale = 2.0 ** (127 - high) / 2.0 ** 8 / math.sqrt(dim)
    return pool, q, scale


# (0.5 to 6 times 2^(byte - 127): 2 to 23 are below 2^-100, 104 begins at float16's smallest number, 108 at 2^4 of it, 141
# and more exceed its largest, 145 and more 2^4 of it)
@pytest.mark.parametrize("low,high", [(24, 30), (90, 99), (104, 107), (106, 106), (108, 109), (141, 144), (145, 148), (190, 200)])
@pytest.mark.parametrize("geometry", GEOMETRIES, ids=lambda c: "-".join(map(str, c)))
def test_keys_beside_float16s_range(geometry, low, high):
    require_gpu()
    pool, q, scale = make(*geometry, low, high)
    want, bound = expected(pool, q, scale)
    check(decode(pool, q.cuda(), scale), want, bound, f"bytes {low} to {high}")


@pytest.mark.parametrize("geometry", GEOMETRIES, ids=lambda c: "-".join(map(str, c)))
def test_small_keys_beside_large_ones(geometry):
    """32 dims of large keys that meet zeros of the queries: the scores are the small keys' alone."""

    require_gpu()
    pool, q, scale = make(*geometry, 100, 105)
    pool.ks.view(torch.uint8)[..., 0] = 160
    q[..., :32] = 0
    want, bound = expected(pool, q, scale)
    check(decode(pool, q.cuda(), scale), want, bound, "small beside large")
    # one step of large keys among steps of ordinary ones
    pool, q, scale = make(*geometry, 126, 128)
    table, e = pool.tables[0].cpu(), pool.ks.view(torch.uint8)
    for t in range(130, 140):
        e[int(table[t // pool.page]), t % pool.page] = 152
    q *= 2.0 ** -24
    want, bound = expected(pool, q, 2.0 ** 24 * scale)
    check(decode(pool, q.cuda(), 2.0 ** 24 * scale), want, bound, "a step of large keys")


def test_bad_queries_over_small_keys_leave_the_others_alone():
    require_gpu()
    pool, q, scale = make(8, 2, 128, 64, 100, 105)
    want, bound = expected(pool, q, scale)
    q[0, 1, 5], q[0, 7, 100], q[1, 2, 0] = torch.inf, torch.nan, -torch.inf
    bad = torch.zeros(3, 8, dtype=torch.bool)
    bad[0, 1] = bad[0, 7] = bad[1, 2] = True
    got = decode(pool, q.cuda(), scale)
    assert torch.equal(got.isnan().all(-1).cpu(), bad) and torch.equal(got.isnan().any(-1).cpu(), bad)
    check(got.cpu()[~bad], want[~bad], bound[~bad], "the others")
